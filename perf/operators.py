"""The serving operators of the decoder library, measured: page plans, the 8-bit
paged K/V cache (written, read back, attended over) and token sampling.

Each case names one operator ("op") and its sizes; prepare() makes what a
serving program holds before the call, run() makes one call. With `own` false
run() computes the operator in plain torch operations, with it true through
the framework's entry points (whisper.go_b200/wgdec.py)."""
import math
import pathlib
import random
import sys

import torch

own = False

ROOT = pathlib.Path(__file__).resolve().parents[1]
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}


def _wgdec():
    if str(ROOT / "whisper.go_b200") not in sys.path:
        sys.path.insert(0, str(ROOT / "whisper.go_b200"))
    import wgdec
    return wgdec


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # one token for each of 48 live streams: the plan of every decode step
        {"name": "plan_step_48", "op": "plan", "requests": 48, "max_len": 448, "max_new": 1, "page": 16},
        # admission of a large batch: whole prompts of up to a text context each
        {"name": "plan_prompts_1500", "op": "plan", "requests": 1500, "max_len": 448, "max_new": 448, "page": 32},
        # one decode step's K and V of 64 streams, large-v3 heads, pages partly filled before
        {"name": "cache_step_64", "op": "cache", "requests": 64, "max_len": 448, "max_new": 1, "heads": 20, "dim": 64,
         "page": 16, "dtype": "f16"},
        # ragged prompts of a small model in bf16, some continuing a page that is already begun
        {"name": "cache_prompts_24", "op": "cache", "requests": 24, "max_len": 448, "max_new": 224, "heads": 12,
         "dim": 64, "page": 32, "dtype": "bf16"},
        # the encoder's K and V of 64 utterances of 1500 frames, one large-v3 layer
        {"name": "cache_encoder_64", "op": "cache", "requests": 64, "max_len": 1500, "max_new": 1500, "heads": 20,
         "dim": 64, "page": 64, "dtype": "f16", "full": True},
        # one stream of a tiny model: latency
        {"name": "attn_one_tiny", "op": "attn", "requests": 1, "max_q": 1, "max_len": 229, "heads": 6, "group": 1,
         "dim": 64, "page": 16, "causal": True, "dtype": "f16", "full": True},
        # cross-attention of 64 utterances, five beams each, over 1500 frames, large-v3
        {"name": "attn_cross_64x5", "op": "attn", "requests": 64, "max_q": 5, "max_len": 1500, "heads": 20, "group": 1,
         "dim": 64, "page": 64, "causal": False, "dtype": "f16", "full": True},
        # ragged prompts attending to themselves
        {"name": "attn_prompts_16", "op": "attn", "requests": 16, "max_q": 448, "max_len": 448, "heads": 20, "group": 1,
         "dim": 64, "page": 32, "causal": True, "dtype": "bf16", "full": False},
        # single tokens over a long history with shared K/V heads and wide heads
        {"name": "attn_long_2", "op": "attn", "requests": 2, "max_q": 1, "max_len": 60001, "heads": 8, "group": 4,
         "dim": 128, "page": 64, "causal": True, "dtype": "bf16", "full": False},
        # one row of the multilingual vocabulary: latency
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 51865, "dtype": "f32"},
        # a middling batch of 16-bit logits
        {"name": "sample_48_f16", "op": "sample", "rows": 48, "vocab": 51864, "dtype": "f16"},
        # 64 utterances of five candidates, large-v3 vocabulary
        {"name": "sample_320", "op": "sample", "rows": 320, "vocab": 51866, "dtype": "f32"},
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["plan", "cache", "cache", "attn", "attn", "attn", "sample", "sample"])
    page = rng.choice([16, 32, 64])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 1500), "max_len": _log(rng, 1, 1500),
                "max_new": rng.choice([1, 1, _log(rng, 2, 448)]), "page": page}
    if op == "cache":
        heads, dim = rng.choice([6, 8, 12, 16, 20]), rng.choice([64, 64, 128])
        tokens = 64 * 1500 * 20 * 64 // (heads * dim)
        requests = _log(rng, 1, 64)
        max_len = _log(rng, 1, max(1, min(2900, tokens // requests)))
        return {"op": op, "requests": requests, "max_len": max_len, "max_new": rng.choice([1, max_len]), "heads": heads,
                "dim": dim, "page": page, "dtype": rng.choice(["f16", "bf16", "f32"])}
    if op == "attn":
        heads, dim, group = rng.choice([2, 6, 8, 12, 20]), rng.choice([64, 64, 128]), rng.choice([1, 1, 2, 4])
        room = 64 * 1500 * 20 * 64 // (heads * dim)
        requests = _log(rng, 1, 64)
        max_len = _log(rng, 1, max(1, min(60000, room // requests)))
        max_q = rng.choice([1, 1, rng.randint(2, 5), _log(rng, 6, 448)])
        # no more scores than the prompts' and no more work than the largest listed case
        max_q = max(1, min(max_q, 64 * 5 * 1500 * 20 * 64 // (requests * max_len * heads * group * dim)))
        return {"op": op, "requests": requests, "max_q": max_q, "max_len": max_len, "heads": heads, "group": group,
                "dim": dim, "page": page, "causal": rng.random() < 0.6, "dtype": rng.choice(["f16", "bf16"]),
                "full": rng.random() < 0.3}
    vocab = _log(rng, 1000, 131072)
    return {"op": op, "rows": _log(rng, 1, max(1, min(320, 320 * 51866 // vocab))), "vocab": vocab,
            "dtype": rng.choice(["f32", "f16", "bf16"])}


# ---- inputs -------------------------------------------------------------------
def _lens(case):
    """Lengths after the step and new tokens of each request: plain numbers of the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    R, most = case["requests"], case["max_len"]
    if case.get("full"):
        lens = [most] * R
    else:
        lens = [rng.randint(max(1, most // 8), most) for _ in range(R)]
        lens[rng.randrange(R)] = most
    new = case.get("max_new", case.get("max_q", 1))
    fresh = [min(n, new) if new == 1 or case.get("full") else min(n, rng.randint(max(1, new // 2), new)) for n in lens]
    return lens, fresh


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32).to(dev)


def _layout(case, seed, dev):
    """Block table with each request's pages in a shuffled pool; entries past a request's pages are -1."""
    lens, fresh = _lens(case)
    need = _pages(lens, case["page"])
    pool = sum(need) + 3
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    return lens, fresh, pool, table.to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op = case["op"]
    s = {"case": case}
    if op == "plan":
        lens, fresh, pool, table = _layout(case, seed, dev)
        held = _pages([n - m for n, m in zip(lens, fresh)], case["page"])
        s["lens"], s["new"] = _i32(lens, dev), _i32(fresh, dev)
        cols = torch.arange(table.shape[1], device=dev)
        s["table"] = torch.where(cols[None, :] < _i32(held, dev)[:, None], table, torch.full_like(table, -1))
        used = sum(held)
        gc = torch.Generator().manual_seed(seed + 1)
        s["free"] = (torch.randperm(sum(_pages(lens, case["page"])) + 5, generator=gc) + used).to(torch.int32).to(dev)
        s["cursor"] = _i32([5], dev)
        s["cap"] = sum(fresh) + 7
        s["slots"] = torch.empty(s["cap"], dtype=torch.int32, device=dev)
        s["cu"] = torch.empty(len(lens) + 1, dtype=torch.int32, device=dev)
        s["cursor_out"] = torch.empty(1, dtype=torch.int32, device=dev)
        s["status"] = torch.empty(2, dtype=torch.int32, device=dev)
        return s
    if op == "sample":
        R, V = case["rows"], case["vocab"]
        logits = torch.randn(R, V, generator=g, device=dev) * 2.5
        at = torch.randint(0, V, (R, 8), generator=g, device=dev)
        logits.scatter_add_(1, at, 6.0 + 3.0 * torch.randn(R, 8, generator=g, device=dev))
        logits[:, torch.randint(0, V, (90,), generator=g, device=dev)] = -math.inf  # suppressed tokens
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        s["u"] = torch.rand(R, generator=g, device=dev)
        row = torch.arange(R, device=dev)
        # the settings of the rows of one serving batch: nucleus, top-k, min-p, all three, none, the first maximum
        pick = lambda *v: torch.tensor(v, device=dev)[row % 6]  # noqa: E731
        s["temperature"] = pick(0.7, 1.0, 0.8, 0.9, 1.0, 0.0).float()
        s["top_k"] = pick(0, 50, 0, 200, 0, 0).int()
        s["top_p"] = pick(0.9, 1.0, 1.0, 0.95, 1.0, 1.0).float()
        s["min_p"] = pick(0.0, 0.0, 0.05, 0.02, 0.0, 0.0).float()
        s["tokens"] = torch.empty(R, dtype=torch.int32, device=dev)
        s["logprobs"] = torch.empty(R, dtype=torch.float32, device=dev)
        return s
    # the 8-bit cache
    lens, fresh, pool, table = _layout(case, seed, dev)
    page, H, D = case["page"], case["heads"], case["dim"]
    codes = torch.empty(pool, 2, H, page, D, dtype=torch.int8, device=dev)
    for a in range(0, pool, 2048):  # in parts: the intermediate is four times the codes
        part = torch.randn(codes[a:a + 2048].shape, generator=g, device=dev)
        codes[a:a + 2048] = (part * 34).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.exp2(torch.randint(-7, -4, (pool, 2, H), generator=g, device=dev).float())
    s["codes"], s["scales"], s["table"] = codes, scales, table
    s["lens"] = _i32(lens, dev)
    s["max_len"] = max(lens)
    if own:
        s["cache"] = _wgdec().Kv8Cache(codes, scales)
    cu = [0]
    for n in fresh if op == "cache" else [min(case["max_q"], n) if not case.get("full") else case["max_q"] for n in lens]:
        cu.append(cu[-1] + n)
    s["cu"], s["max_q"] = _i32(cu, dev), max(b - a for a, b in zip(cu, cu[1:]))
    T = cu[-1]
    dt = DTYPES[case["dtype"]]
    if op == "cache":
        rows = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(fresh))
        pos = torch.arange(T) - torch.tensor(cu)[rows] + (torch.tensor(lens) - torch.tensor(fresh))[rows]
        rows, pos = rows.to(dev), pos.to(dev)
        s["slots"] = (table[rows, pos // page] * page + pos % page).to(torch.int32)
        # K and V of a fused projection: each token's row is q | k | v
        qkv = torch.randn(T, 3 * H * D, generator=g, device=dev, dtype=torch.float32).to(dt)
        s["k"], s["v"] = qkv[:, H * D:2 * H * D].view(T, H, D), qkv[:, 2 * H * D:].view(T, H, D)
        s["k_out"] = torch.empty(T, H, D, dtype=torch.bfloat16, device=dev)
        s["v_out"] = torch.empty(T, H, D, dtype=torch.bfloat16, device=dev)
    else:
        s["q"] = (2.0 * torch.randn(T, H * case["group"], D, generator=g, device=dev)).to(dt)
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(D)
    return s


# ---- plain forms ----------------------------------------------------------------
def _plan(s):
    page = s["case"]["page"]
    lens, new, table, free = s["lens"].long(), s["new"].long(), s["table"], s["free"].long()
    R, cols = table.shape
    held = (lens - new + page - 1) // page
    need = (lens + page - 1) // page
    zero = torch.zeros(1, dtype=torch.int64, device=lens.device)
    off = torch.cat([zero, torch.cumsum(need - held, 0)])
    cu = torch.cat([zero, torch.cumsum(new, 0)])
    col = torch.arange(cols, device=lens.device)[None, :]
    take = (col >= held[:, None]) & (col < need[:, None])
    at = s["cursor"].long() + off[:-1, None] + col - held[:, None]
    full = torch.where(take, free[at.clamp(0, free.numel() - 1)], table.long())
    i = torch.arange(s["cap"], device=lens.device)
    r = (torch.searchsorted(cu, i, right=True) - 1).clamp(0, R - 1)
    pos = (lens - new)[r] + i - cu[r]
    slot = full[r, (pos // page).clamp(0, cols - 1)] * page + pos % page
    s["table"].copy_(full)
    s["slots"].copy_(torch.where(i < cu[-1], slot, -torch.ones_like(slot)))
    s["cu"].copy_(cu)
    s["cursor_out"].copy_(s["cursor"] + off[-1:])
    s["status"].copy_(torch.cat([zero, off[-1:]]))
    return {"table": s["table"], "slots": s["slots"], "cu": s["cu"], "cursor": s["cursor_out"], "status": s["status"]}


def _needed(amax):
    """The power of two that takes amax to at most 127 steps (0 for 0)."""
    mant, exp = torch.frexp(amax)  # amax = mant * 2^exp, mant in [0.5, 1)
    e = torch.clamp(torch.where(mant <= 127 / 128, exp - 7, exp - 6), min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.zeros_like(amax))


def _append(s):
    codes, scales, page = s["codes"], s["scales"], s["case"]["page"]
    slots = s["slots"].long()
    pages = slots // page
    x = torch.stack([s["k"], s["v"]], 1).float()  # [T, 2, H, D]
    first = torch.full((codes.shape[0],), page, dtype=torch.int64, device=slots.device)
    first.scatter_reduce_(0, pages, slots % page, "amin")  # page: untouched
    amax = torch.zeros_like(scales)
    amax.scatter_reduce_(0, pages[:, None, None].expand(-1, *scales.shape[1:]), x.abs().amax(-1), "amax")
    begun = (first > 0)[:, None, None]
    new = torch.where(begun, torch.maximum(scales, _needed(amax)), _needed(amax))
    grown = new > scales
    ratio = torch.where(begun & grown, scales / new, torch.ones_like(new))
    early = torch.arange(page, device=slots.device)[None, :] < first[:, None]
    shrunk = torch.round(codes.float() * ratio[..., None, None]).to(torch.int8)
    codes.copy_(torch.where(early[:, None, None, :, None], shrunk, codes))
    scales.copy_(new)
    step = new[pages]
    q = torch.where(step[..., None] > 0, x / step[..., None], torch.zeros_like(x))
    codes[pages, :, :, slots % page] = torch.round(q).clamp(-127, 127).to(torch.int8)


def _read(s):
    slots, page = s["slots"].long(), s["case"]["page"]
    x = s["codes"][slots // page, :, :, slots % page].float() * s["scales"][slots // page][..., None]
    s["k_out"].copy_(x[:, 0])
    s["v_out"].copy_(x[:, 1])


def _attention(s):
    case, table, lens, cu = s["case"], s["table"], s["lens"].long(), s["cu"].long()
    page, H, G, D = case["page"], case["heads"], case["group"], case["dim"]
    R, L, Q = lens.numel(), s["max_len"], s["max_q"]
    dev = lens.device
    pos = torch.arange(L, device=dev)
    ids = table[:, pos // page].long().clamp(min=0)  # [R, L]
    at = (pos % page)[None, :].expand(R, L)
    qlen = cu[1:] - cu[:-1]
    i = torch.arange(Q, device=dev)
    there = i[None, :] < qlen[:, None]  # [R, Q]
    rows = (cu[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(R, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(R, H, G * Q, D)
    k = s["codes"][ids, 0, :, at].float().mul_(s["scales"][ids, 0][..., None])  # [R, L, H, D]
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    del k
    last = lens[:, None] - qlen[:, None] + i[None, :] if case["causal"] else (lens - 1)[:, None].expand(R, Q)
    seen = pos[None, None, :] <= torch.minimum(last, (lens - 1)[:, None])[:, :, None]  # [R, Q, L]
    sc = sc.view(R, H, G, Q, L).masked_fill(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    v = s["codes"][ids, 1, :, at].float().mul_(s["scales"][ids, 1][..., None])
    o = torch.matmul(p.view(R, H, G * Q, L), v.permute(0, 2, 1, 3)).view(R, H, G, Q, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(R, Q, H * G, D)
    s["out"][rows[there]] = o[there].to(s["out"].dtype)
    return s["out"]


def _sample(s):
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    V = x.shape[1]
    t = s["temperature"].double()[:, None]
    z = x / torch.where(t > 0, t, torch.ones_like(t))
    top = z.amax(-1, keepdim=True)
    w = torch.where(z == top, torch.ones_like(z), torch.exp(z - top))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = s["top_k"].long()[:, None]
    rank = torch.arange(V, device=x.device)[None, :]
    keep = rank < torch.where((k > 0) & (t > 0), k, torch.full_like(k, V))
    keep &= (t > 0) | (rank == 0)
    ws = torch.where(keep, ws, torch.zeros_like(ws))
    mass = torch.cumsum(ws, -1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (mass - ws < p * mass[:, -1:]) | (rank == 0)
    keep &= (ws >= s["min_p"].double()[:, None]) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = torch.where(kept, w, torch.zeros_like(w))
    cum = torch.cumsum(w, -1)
    over = cum > s["u"].double()[:, None] * cum[:, -1:]
    token = over.to(torch.int8).argmax(-1, keepdim=True)
    logz = torch.log(torch.exp(z - top).sum(-1, keepdim=True)) + top
    s["tokens"].copy_(token[:, 0])
    s["logprobs"].copy_((z.gather(1, token) - logz)[:, 0])
    return {"tokens": s["tokens"], "logprobs": s["logprobs"]}


# ---- one pass ---------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        if op == "plan":
            return _plan(s)
        if op == "attn":
            return _attention(s)
        if op == "sample":
            return _sample(s)
        _append(s)
        _read(s)
        return {"k": s["k_out"], "v": s["v_out"], "scales": s["scales"]}
    wgdec = _wgdec()
    if op == "plan":
        wgdec.kv_plan(s["lens"], s["new"], case["page"], s["free"], s["cursor"], s["table"], s["slots"], s["cu"],
                      s["status"], cursor_out=s["cursor_out"])
        return {"table": s["table"], "slots": s["slots"], "cu": s["cu"], "cursor": s["cursor_out"],
                "status": s["status"]}
    if op == "attn":
        s["cache"].attention(s["q"], s["cu"], s["lens"], s["table"], max_q=s["max_q"], max_kv=s["max_len"],
                             causal=case["causal"], scale=s["scale"], out=s["out"])
        return s["out"]
    if op == "sample":
        wgdec.sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"], tokens=s["tokens"], logprobs=s["logprobs"])
        return {"tokens": s["tokens"], "logprobs": s["logprobs"]}
    s["cache"].append(s["k"], s["v"], s["slots"])
    # what the cache now holds of these tokens, as values
    s["cache"].read(s["slots"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"], "scales": s["scales"]}


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * ITEM[case["dtype"]] + case["rows"] * 28, "flops": 4 * n}
    lens, fresh = _lens(case)
    if op == "plan":
        new = sum(_pages(lens, case["page"])) - sum(_pages([a - b for a, b in zip(lens, fresh)], case["page"]))
        return {"bytes": 4 * (2 * len(lens) + 2 * new + sum(fresh) + len(lens) + 1 + 4), "flops": 0}
    H, D, page = case["heads"], case["dim"], case["page"]
    if op == "cache":  # K and V in, codes out, codes in again, values out (16 bits), scales
        n = 2 * sum(fresh) * H * D
        return {"bytes": n * (ITEM[case["dtype"]] + 1 + 1 + 2) + 16 * H * sum(_pages(fresh, page)), "flops": 4 * n}
    q = [case["max_q"] if case.get("full") else min(case["max_q"], n) for n in lens]
    pairs = 0
    for n, m in zip(lens, q):
        pairs += sum(max(0, n - m + 1 + i) for i in range(m)) if case["causal"] else n * m
    held = sum(lens) * 2 * H * D + sum(_pages(lens, page)) * 2 * H * 4
    return {"bytes": held + 2 * 2 * sum(q) * H * case["group"] * D, "flops": 4 * pairs * H * case["group"] * D}


# ---- the operators' definitions in 64 bits ---------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    s = prepare(case, seed)
    if op == "cache":
        page = case["page"]
        slots = s["slots"].cpu().tolist()
        runs, at = [], 0  # (first token, one past the last) of the tokens that share a page
        for i in range(1, len(slots) + 1):
            if i == len(slots) or slots[i] // page != slots[at] // page:
                runs.append((at, i))
                at = i
        page_of = torch.tensor([slots[a] // page for a, _ in runs], device=s["k"].device)
        begun = torch.tensor([slots[a] % page > 0 for a, _ in runs], device=s["k"].device)
        run_of = torch.repeat_interleave(torch.arange(len(runs)), torch.tensor([b - a for a, b in runs])).to(begun.device)
        scales = s["scales"].double()
        found = []
        for j, x in enumerate((s["k"], s["v"])):
            size = x.abs().amax(-1).double()  # [T, H]
            most = torch.zeros(len(runs), size.shape[1], dtype=torch.float64, device=size.device)
            most.index_reduce_(0, run_of, size, "amax")
            step = torch.exp2(torch.ceil(torch.log2(most / 127)).clamp(min=-126))
            step = torch.where(step / 2 * 127 >= most, step / 2, step)  # log2's rounding at a border
            step = torch.where(step * 127 < most, step * 2, step)
            step = torch.where(most > 0, step, torch.zeros_like(most))
            step = torch.where(begun[:, None], torch.maximum(step, scales[page_of, j]), step)
            scales[page_of, j] = step
            own_step = step[run_of][..., None]
            # rounded to 32 bits here only to hold less: codes of at most 7 bits times powers of two are exact
            found.append((torch.round(x.float() / own_step.float()).clamp(-127, 127) * own_step.float()).nan_to_num(0.0))
        return {"k": found[0], "v": found[1], "scales": _untouched(scales, page_of, s["scales"])}
    if op == "attn":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        page, H, G = case["page"], case["heads"], case["group"]
        cu, lens = s["cu"].cpu().tolist(), s["lens"].cpu().tolist()
        for r, n in enumerate(lens):
            ids = s["table"][r, :-(-n // page)].long()
            kv = s["codes"][ids].double() * s["scales"][ids].double()[..., None, None]  # [pages, 2, H, P, D]
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, H, -1, kv.shape[-1])[:, :, :n]
            m = cu[r + 1] - cu[r]
            q = s["q"][cu[r]:cu[r + 1]].double()  # [m, H * G, D]
            col, row = torch.arange(n, device=q.device)[None, :], torch.arange(m, device=q.device)[:, None]
            hidden = col > n - m + row if case["causal"] else torch.zeros(m, n, dtype=torch.bool, device=q.device)
            for h in range(H):
                for g in range(G):
                    sc = (q[:, h * G + g] @ kv[0, h].T * s["scale"]).masked_fill(hidden, -math.inf)
                    a = torch.softmax(sc, -1).masked_fill(hidden.all(-1, keepdim=True), 0.0)
                    out[cu[r]:cu[r + 1], h * G + g] = a @ kv[1, h]
        return out
    tokens, logprobs = [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        t = float(s["temperature"][r])
        z = x / (t if t > 0 else 1.0)
        logp = z - torch.logsumexp(z, 0)
        if t <= 0:
            token = int(torch.nonzero(x == x.max())[0])
        else:
            vals, idx = torch.sort(x, descending=True, stable=True)
            w = torch.exp((vals - vals[0]) / t)
            n = int(s["top_k"][r])
            n = n if 0 < n < x.numel() else x.numel()
            total = w[:n].sum()
            p = float(s["top_p"][r])
            if p < 1:
                n = min(n, 1 + int((torch.cumsum(w[:n], 0) < p * total).sum()))
            n = max(1, min(n, int((w >= float(s["min_p"][r])).sum())))
            ids = torch.sort(idx[:n]).values
            mass = torch.cumsum(torch.exp((x[ids] - vals[0]) / t), 0)
            token = int(ids[min(n - 1, int((mass <= float(s["u"][r]) * mass[-1]).sum()))])
        tokens.append(token)
        logprobs.append(float(logp[token]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}


def _untouched(scales, pages, before):
    """Scales of the pages that were written; the others as they were."""
    kept = before.double().clone()
    kept[pages] = scales[pages]
    return kept
