"""The serving operators (page plans, the 8-bit paged cache, attention over
it, token sampling) against plain 64-bit forms (serving_ref.py)."""
import numpy as np
import pytest

import serving_ref as ref
import wgdec

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DEV = "cuda:0"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)


def host(t):
    return t.detach().cpu().to(torch.float64).numpy() if t.is_floating_point() else t.detach().cpu().numpy()


# ---- wg_kv_plan ---------------------------------------------------------------
def run_plan(lens, new, page, free, cursor, table, n_slots, in_place=False, shift=0):
    R = len(lens)
    t, c = i32(table), i32([cursor])
    out = c if in_place else i32([-7])
    buf = torch.full((n_slots + shift,), -9, dtype=torch.int32, device=DEV)
    slots = buf[shift:]
    cu, st = i32(np.full(R + 1, -9)), i32([-9, -9])
    wgdec.kv_plan(i32(lens), i32(new), page, i32(free), c, t, slots, cu, st, cursor_out=None if in_place else out)
    return [host(x) for x in (st, t, slots, cu, out)]


def check_plan(lens, new, page, free, cursor, table, n_slots, **kw):
    code, t, s, cu, c, taken = ref.plan(lens, new, page, free, cursor, table, n_slots)
    got = run_plan(lens, new, page, free, cursor, table, n_slots, **kw)
    assert list(got[0]) == [code, taken]
    np.testing.assert_array_equal(got[1], t)
    np.testing.assert_array_equal(got[2], s)
    np.testing.assert_array_equal(got[3], cu)
    assert list(got[4]) == [c]
    return code


@pytest.mark.parametrize("R,page,most,new_most", [(1, 16, 1, 1), (1, 128, 5000, 5000), (5, 16, 100, 7),
                                                  (64, 32, 448, 1), (1023, 16, 40, 40), (1024, 64, 90, 2),
                                                  (2500, 16, 70, 33), (3, 64, 9000, 9000)])
@pytest.mark.parametrize("shift", [0, 1])
def test_plan(R, page, most, new_most, shift):
    rng = np.random.default_rng(R * 7 + page)
    lens = rng.integers(0, most + 1, R)
    lens[rng.integers(R)] = most
    new = np.minimum(lens, rng.integers(0, new_most + 1, R))
    cols = -(-most // page) + 2
    table = rng.permutation(R * cols).reshape(R, cols).astype(np.int32)
    free = (rng.permutation(R * cols) + R * cols).astype(np.int32)
    assert check_plan(lens, new, page, free, 3, table, int(new.sum()) + 5, in_place=bool(shift), shift=shift) == 0 or \
        len(free) - 3 < sum(-(-lens // page)) - sum(-(-(lens - new) // page))


@pytest.mark.parametrize("change", ["negative length", "negative new", "new past length", "table", "slots", "pages",
                                    "too few pages", "cursor", "several"])
def test_plan_that_cannot_be_made(change):
    lens, new = [40, 5, 0, 17], [20, 5, 0, 1]
    free, cursor, n_slots = np.arange(100, 110), 0, 26
    table = np.arange(12).reshape(4, 3)
    if change == "negative length":
        lens[2] = -1
    if change == "negative new":
        new[1] = -1
    if change == "new past length":
        new[3] = 18
    if change in ("table", "several"):
        lens[0], new[0] = 49, 29
    if change in ("slots", "several"):
        n_slots = 25
    if change == "pages":
        free = free[:3]  # requests 0, 1 and 3 take one page each: just enough
    if change == "too few pages":
        free = free[:2]
    if change == "cursor":
        cursor = -1
    for in_place in (False, True):
        code = check_plan(np.array(lens), np.array(new), 16, free, cursor, table, n_slots, in_place=in_place)
        assert (code > 0) == (change != "pages")


def test_plan_page_numbers_without_slots():
    """A page number that is negative, or whose slots are past 32 bits, goes into the table and gives -1 for its slots."""
    free = np.array([5, 2 ** 31 - 1, -7, 2 ** 27 - 1, 2 ** 27, 9])
    st, t, slots, cu, c = run_plan([16 * 6], [16 * 6], 16, free, 0, np.zeros((1, 6), int), 100)
    assert list(st) == [0, 6] and t[0].tolist() == free.tolist()
    want = -np.ones(100, np.int64)
    for i, pg in enumerate(free):
        if 0 <= pg < 2 ** 27:
            want[16 * i:16 * i + 16] = pg * 16 + np.arange(16)
    np.testing.assert_array_equal(slots, want)


def test_plan_exactly_full():
    """The last free page, the last slot and the last table column are usable."""
    assert check_plan(np.array([48, 16]), np.array([48, 16]), 16, np.arange(7, 11), 0, np.zeros((2, 3), int), 64) == 0


# ---- wg_kv8_append / wg_kv8_read ------------------------------------------------
def make_cache(rng, pages, page, H, D):
    codes = rng.integers(-127, 128, (pages, 2, H, page, D)).astype(np.int8)
    scales = (2.0 ** rng.integers(-9, -2, (pages, 2, H))).astype(np.float32)
    return codes, scales, wgdec.Kv8Cache(torch.tensor(codes, device=DEV), torch.tensor(scales, device=DEV))


def rows(rng, n, H, D, dt, pad=0, off=0, spread=True):
    """A [n, H, D] view with rows pad elements further apart, off elements into its storage."""
    x = rng.standard_normal((n, H, D))
    if spread:
        x *= 2.0 ** rng.integers(-6, 7, (n, 1, 1))
    buf = torch.zeros(n * (H * D + pad) + off, dtype=DT[dt], device=DEV)
    v = buf[off:].view(n, H * D + pad)[:, :H * D].view(n, H, D)
    v.copy_(torch.tensor(x))
    return v


SLOT_CASES = {
    "one token": lambda page: [3 * page + 5],
    "first of a page": lambda page: [3 * page],
    "last of a page": lambda page: [4 * page - 1],
    "a whole page": lambda page: list(range(2 * page, 3 * page)),
    "a run over three pages": lambda page: list(range(2 * page - 3, 2 * page)) + list(range(5 * page, 6 * page)) + [3 * page],
    "many singles": lambda page: [p * page + (p * 5) % page for p in range(7)],
    "padding between": lambda page: [-1, 7, 8, -1, -1, page * 6, page * 6 + 1, -1],
    "outside": lambda page: [page * 7, 9, 2 ** 31 - 1, -2 ** 31, page * 7 - 1],
}


@pytest.mark.parametrize("case", SLOT_CASES)
@pytest.mark.parametrize("dt,D,page,H,pad,off", [("f16", 64, 16, 3, 0, 0), ("bf16", 128, 32, 1, 64, 8),
                                                 ("f32", 64, 64, 2, 3, 1), ("f16", 128, 128, 5, 1, 3),
                                                 ("bf16", 64, 128, 20, 8, 0)])
def test_append_and_read(case, dt, D, page, H, pad, off):
    """Codes and scales equal the definition's bit for bit (powers of two: no
    step but the rounding to the code is inexact); values read back equal
    code * scale, exact in fp32 and bf16."""
    rng = np.random.default_rng(len(case) + D + page)
    codes, scales, cache = make_cache(rng, 7, page, H, D)
    slots = SLOT_CASES[case](page)
    n = len(slots)
    k, v = rows(rng, n, H, D, dt, pad, off), rows(rng, n, H, D, dt, pad, off)
    cache.append(k, v, i32(slots))
    ref.append(codes, scales, host(k), host(v), slots)
    np.testing.assert_array_equal(host(cache.scales).astype(np.float32), scales)
    np.testing.assert_array_equal(host(cache.codes), codes)
    for rd in ("f32", "bf16", "f16"):
        ko, vo = rows(rng, n, H, D, rd, pad, off), rows(rng, n, H, D, rd, pad, off)
        want = [host(ko).copy(), host(vo).copy()]
        cache.read(i32(slots), ko, vo)
        for t, s in enumerate(slots):
            if 0 <= s < 7 * page:
                for j in range(2):
                    val = codes[s // page, j, :, s % page].astype(np.float64) * scales[s // page, j, :, None]
                    want[j][t] = host(torch.tensor(val).to(DT[rd]))
        np.testing.assert_array_equal(host(ko), want[0])
        np.testing.assert_array_equal(host(vo), want[1])


def test_append_special_values():
    page, H, D = 16, 2, 64
    rng = np.random.default_rng(5)
    codes, scales, cache = make_cache(rng, 4, page, H, D)
    k, v = rows(rng, 12, H, D, "f32"), rows(rng, 12, H, D, "f32")
    k[0, 0] = float("nan")
    k[1, 0, :5] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0, -0.0])
    v[0:4, 1] = 0.0
    v[4:8, 1] = 1e-42        # subnormal: the scale stops at 2^-126
    v[8:12, 0] = 3.0e38
    k[8:12, 1] = torch.tensor(127 * 2.0 ** -20)  # exactly 127 steps
    k[8, 1, 3] = 127 * 2.0 ** -20 * (1 + 2.0 ** -23)  # just past them
    slots = list(range(0, 4)) + list(range(16, 20)) + list(range(36, 40))
    cache.append(k, v, i32(slots))
    ref.append(codes, scales, host(k), host(v), slots)
    np.testing.assert_array_equal(host(cache.scales).astype(np.float32), scales)
    np.testing.assert_array_equal(host(cache.codes), codes)


def test_append_token_by_token_grows_the_scale():
    """A page filled one token at a time with growing magnitudes: every token
    stays within one step of its value (each of the g growths rounds the code
    by at most half a step of that moment: 1/2 + 1/4 + ... < 1 final step)."""
    page, H, D = 32, 2, 64
    rng = np.random.default_rng(6)
    cache = wgdec.Kv8Cache.alloc(1, page, H, D, device=DEV)  # not initialised
    x = rng.standard_normal((page, H, D)) * np.exp(np.linspace(-4, 4, page))[:, None, None]
    k = torch.tensor(x, dtype=torch.float32, device=DEV)
    for i in range(page):
        cache.append(k[i:i + 1], -k[i:i + 1], i32([i]))
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    cache.read(i32(np.arange(page)), ko, vo)
    step = host(cache.scales)[0]
    assert (np.abs(host(ko) - host(k)) <= step[0][None, :, None]).all()
    assert (np.abs(host(vo) + host(k)) <= step[1][None, :, None]).all()


@pytest.mark.parametrize("H,n_seq,page", [(9, 420, 32), (20, 280, 128)])
def test_append_large_equals_its_parts(H, n_seq, page):
    """A long call gives each CTA more tokens and more heads than a short one:
    the same sequences appended a few at a time give the same bits."""
    rng = np.random.default_rng(H + page)
    lens = rng.integers(1, 200, n_seq)
    first = np.concatenate([[0], np.cumsum(-(-lens // page))])
    order = rng.permutation(first[-1])  # pages anywhere
    slots, starts = [], []
    for r, n in enumerate(lens):
        starts.append(len(slots))
        t = np.arange(n)
        slots += list(order[first[r] + t // page] * page + t % page) + [-1] * (r % 3)
    starts.append(len(slots))
    n, D = len(slots), 64
    k, v = (torch.tensor(rng.standard_normal((n, H, D), dtype=np.float32), device=DEV).half() for _ in range(2))
    codes, scales = torch.zeros(len(order), 2, H, page, D, dtype=torch.int8, device=DEV), torch.zeros(len(order), 2, H, device=DEV)
    whole, parts = wgdec.Kv8Cache(codes, scales), wgdec.Kv8Cache(codes.clone(), scales.clone())
    at = i32(slots)
    whole.append(k, v, at)
    for r in range(0, n_seq, 5):
        a, b = starts[r], starts[min(r + 5, n_seq)]
        parts.append(k[a:b], v[a:b], at[a:b])
    assert torch.equal(whole.scales, parts.scales) and torch.equal(whole.codes, parts.codes)
    assert (whole.scales != 0).all()


# ---- wg_kv8_attention -------------------------------------------------------------
EPS = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def attn_case(rng, lens, nq, page, H, G, D, qdt, causal, odt=None, max_q=None, bad=(), table_pad=2, extra_rows=0,
              ld_pad=0, q_scale=1.5):
    R = len(lens)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    codes, scales, cache = make_cache(rng, pages, page, H, D)
    perm = rng.permutation(pages)
    table = np.full((R, max(need + [1]) + table_pad), -1)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    for r, c, to in bad:
        table[r, c] = to
    cu = np.concatenate([[0], np.cumsum(nq)])
    n_q = int(cu[-1]) + extra_rows
    q = rows(rng, n_q, H * G, D, qdt, pad=ld_pad, spread=False)
    q.mul_(q_scale)
    odt = odt or ("f16" if qdt == "f32" else qdt)
    buf = torch.full((n_q, H * G * D + ld_pad), 77.0, dtype=DT[odt], device=DEV)
    out = buf[:, :H * G * D].view(n_q, H * G, D)
    scale = D ** -0.5
    cache.attention(q, i32(cu), i32(lens), i32(table), max_q=max(nq) if max_q is None else max_q,
                    max_kv=max(list(lens) + [0]), causal=causal, scale=scale, out=out)
    qh = host(q)
    want, most = ref.attention(codes, scales, qh, cu, lens, table, H * G, causal, scale, max_q)
    check_attn(host(out), want, most, odt, qdt, qh, codes, scales, scale, max(list(lens) + [1]))
    return want


def check_attn(got, want, most, odt, qdt, q, codes, scales, scale, n):
    """Error of one output, relative to the largest |v| it sums: each weight is
    rounded to f16 (2^-11, or 2^-25 where subnormal, n of them against a sum
    of at least 1); the fp32 sums, exponentials and scores within 2^-13; for
    fp32 queries every q element is rounded by 2^-11, which moves a score by
    at most ds and a weight by exp(2 ds); last the rounding of the output."""
    kmax = 127.0 * float(scales[:, 0].max())
    for row, o in want.items():
        ds = scale * 2.0 ** -11 * kmax * np.abs(q[row]).sum(-1, keepdims=True) if qdt == "f32" else 0.0
        tol = EPS[odt] * np.abs(o) + most[row] * (2.0 ** -11 + n * 2.0 ** -25 + 2.0 ** -13 + np.expm1(2 * ds)) + 2.0 ** -25
        assert (np.abs(got[row] - o) <= tol).all(), (row, np.abs(got[row] - o).max())
    for row in range(got.shape[0]):
        if row not in want:
            assert (got[row] == 77.0).all(), row


@pytest.mark.parametrize("H,G,D,page,qdt", [(3, 1, 64, 16, "f16"), (2, 4, 128, 32, "bf16"), (1, 8, 64, 64, "f32"),
                                            (2, 3, 64, 128, "bf16"), (1, 1, 128, 16, "f16"), (1, 20, 64, 32, "f16")])
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [31, 32, 33, 64, 65], [0, 5, 0], [700, 3, 259], [2300]], ids=str)
def test_attention_single_tokens(lens, H, G, D, page, qdt):
    rng = np.random.default_rng(sum(lens) + H * D + page)
    attn_case(rng, lens, [1] * len(lens), page, H, G, D, qdt, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,G,D,page,qdt", [(2, 1, 64, 16, "bf16"), (1, 2, 128, 64, "f16"), (2, 5, 64, 32, "f16")])
@pytest.mark.parametrize("lens,nq", [([40, 7, 100], [5, 5, 5]), ([130, 64, 17], [130, 64, 17]), ([33], [16]),
                                     ([200, 300, 3], [17, 0, 9]), ([10, 0, 70], [25, 4, 70])], ids=str)
def test_attention_prompts(lens, nq, H, G, D, page, qdt, causal):
    """Prompts and beams; more queries than tokens leaves causal rows that see
    nothing (zeros); a request without queries has no rows."""
    rng = np.random.default_rng(sum(lens) + sum(nq) + D)
    attn_case(rng, lens, nq, page, H, G, D, qdt, causal, extra_rows=3)


def test_attention_long_prompt_over_a_longer_history():
    attn_case(np.random.default_rng(1), [1111, 640], [300, 129], 64, 1, 2, 64, "f16", True)


def test_attention_strides_and_types():
    rng = np.random.default_rng(2)
    attn_case(rng, [50, 90], [1, 3], 16, 2, 1, 64, "f16", True, odt="bf16", ld_pad=5)
    attn_case(rng, [50, 90], [1, 3], 16, 2, 1, 64, "bf16", True, odt="f16", ld_pad=64)
    attn_case(rng, [50, 90], [40, 33], 32, 2, 1, 128, "f32", False, odt="bf16", ld_pad=1)


@pytest.mark.parametrize("page", [16, 32, 64])
def test_attention_bad_pages_hide_their_tokens(page):
    """Page numbers outside the cache are never read; a row left with nothing gives zeros."""
    rng = np.random.default_rng(3)
    n = 5 * page
    bad = [(0, 1, -1), (0, 3, 10 ** 9), (1, 0, -5), (1, 1, 2 ** 31 - 1)]
    for nq in ([1, 1], [4, 20]):
        want = attn_case(rng, [n, page + 3], nq, page, 2, 1, 64, "f16", False, bad=bad)
        assert (want[nq[0]] == 0).all()


def test_attention_ragged_descriptors():
    """Lengths past the table are cut to it, negative ones hold nothing, a
    descending or outside cu_q pair has no rows, rows past max_q stay as they were."""
    rng = np.random.default_rng(4)
    page, H, D = 16, 2, 64
    codes, scales, cache = make_cache(rng, 12, page, H, D)
    table = rng.permutation(12).reshape(4, 3)
    q = rows(rng, 9, H, D, "f16", spread=False)
    lens = [1000, -3, 20, 48]
    for cu in ([0, 2, 4, 6, 9], [5, 7, 1, 3, 5], [0, 3, 5, 50, 9], [-1, 2, 4, 6, 9]):
        out = torch.full((9, H, D), 77.0, dtype=torch.float16, device=DEV)
        cache.attention(q, i32(cu), i32(lens), i32(table), max_q=2, max_kv=48, causal=True, out=out)
        want, most = ref.attention(codes, scales, host(q), cu, lens, table, H, True, D ** -0.5, max_q=2)
        check_attn(host(out), want, most, "f16", "f16", host(q), codes, scales, D ** -0.5, 48)


def test_attention_extreme_scores():
    """Sharp softmaxes (one token takes all), zero scales, and bf16 queries far outside f16's range."""
    rng = np.random.default_rng(7)
    attn_case(rng, [300], [1], 32, 1, 1, 64, "f16", True, q_scale=300.0)
    page, H, D = 16, 1, 64
    codes, scales, cache = make_cache(rng, 4, page, H, D)
    scales[1] = 0.0
    scales[2] *= 2.0 ** 20
    cache.scales.copy_(torch.tensor(scales))
    table = np.array([[0, 1, 2, 3]])
    for mul in (2.0 ** 60, 2.0 ** -60):
        q = (torch.randn(1, 1, D, device=DEV) * mul).to(torch.bfloat16)
        out = torch.full((1, 1, D), 77.0, dtype=torch.bfloat16, device=DEV)
        cache.attention(q, i32([0, 1]), i32([60]), i32(table), max_q=1, max_kv=60, scale=1.0 / mul / 64, out=out)
        want, most = ref.attention(codes, scales, host(q), [0, 1], [60], table, 1, True, 1.0 / mul / 64)
        check_attn(host(out), want, most, "bf16", "bf16", host(q), codes, scales, 1.0 / mul / 64, 60)


def test_attention_nan_and_infinite_queries_stay_in_their_rows():
    rng = np.random.default_rng(8)
    page, H, D = 16, 1, 64
    codes, scales, cache = make_cache(rng, 8, page, H, D)
    table = rng.permutation(8).reshape(2, 4)
    q = rows(rng, 6, H, D, "bf16", spread=False)
    clean = torch.empty_like(q)
    cache.attention(q, i32([0, 3, 6]), i32([50, 61]), i32(table), max_q=3, max_kv=61, out=clean)
    q[1, 0, 3], q[4, 0, 9] = float("nan"), float("inf")
    out = torch.empty_like(q)
    cache.attention(q, i32([0, 3, 6]), i32([50, 61]), i32(table), max_q=3, max_kv=61, out=out)
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[4]).any()
    for r in (0, 2, 3, 5):
        assert torch.equal(out[r], clean[r])


@pytest.mark.parametrize("nq,page", [(6, 32), (13, 16), (13, 64), (40, 16), (40, 64)])
@pytest.mark.parametrize("qdt", ["f16", "f32"])
def test_attention_nan_and_infinite_queries_in_every_kernel(nq, page, qdt):
    """Rows with a NaN or an infinity give no number, the rows around them their own."""
    rng = np.random.default_rng(nq + page)
    H, D = 1, 64
    codes, scales, cache = make_cache(rng, 8, page, H, D)
    table = i32(rng.permutation(8)[:6][None])
    q = rows(rng, nq, H, D, qdt, spread=False)
    clean = torch.empty(nq, H, D, dtype=torch.bfloat16, device=DEV)
    cache.attention(q, i32([0, nq]), i32([90]), table, max_q=nq, max_kv=90, out=clean)
    q[1, 0, 3], q[4, 0, 9], q[nq - 1, 0, 0] = float("nan"), float("inf"), -float("inf")
    out = torch.empty_like(clean)
    cache.attention(q, i32([0, nq]), i32([90]), table, max_q=nq, max_kv=90, out=out)
    bad = [1, 4, nq - 1]
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[bad]).any()
    for r in range(nq):
        if r not in bad:
            assert torch.equal(out[r], clean[r]), r


@pytest.mark.parametrize("log2", [5, 20, 24, 27, 30, 34, 50, 90])
@pytest.mark.parametrize("nq,G,D,page", [(1, 1, 64, 64), (3, 2, 64, 16), (2, 2, 128, 32), (12, 1, 64, 32), (3, 4, 128, 16),
                                         (40, 1, 64, 64), (24, 1, 128, 16)])
def test_attention_of_any_size_of_scores(nq, G, D, page, log2):
    """Scores so far apart that one token takes all, up to sizes where fp32 has
    no digits left behind the point: the output is that token's value."""
    rng = np.random.default_rng(nq + G + log2)
    H, n = 1, 150
    codes, scales, cache = make_cache(rng, -(-n // page), page, H, D)
    # queries along dim 0 alone: the best token's code there leads the others' by 47
    codes[:, 0] = rng.integers(-3, 4, codes[:, 0].shape)
    codes[:, 0, :, :, 0] = 8 * rng.integers(-10, 11, codes.shape[0] * page).reshape(-1, 1, page)
    best = int(rng.integers(0, n))
    codes[best // page, 0, :, best % page, 0] = 127
    scales[:, 0] = 1.0
    cache.codes.copy_(torch.tensor(codes))
    cache.scales.copy_(torch.tensor(scales))
    x = np.zeros((nq, H * G, D))
    x[..., 0] = 2.0 ** log2 * (1 + rng.integers(0, 128, (nq, H * G)) / 128)
    q = torch.tensor(x, dtype=torch.bfloat16, device=DEV)
    table = np.arange(codes.shape[0])[None]
    out = torch.full((nq, H * G, D), 77.0, dtype=torch.float16, device=DEV)
    cache.attention(q, i32([0, nq]), i32([n]), i32(table), max_q=nq, max_kv=n, causal=False, scale=0.25, out=out)
    want, most = ref.attention(codes, scales, x, [0, nq], [n], table, H * G, False, 0.25)
    v = codes[best // page, 1, 0, best % page].astype(np.float64) * scales[best // page, 1, 0]
    assert np.abs(want[0][0] - v).max() <= 1e-9  # 2^5 * 0.25 * 47 steps above the next: all others under e^-376
    check_attn(host(out), want, most, "f16", "bf16", x, codes, scales, 0.25, n)


@pytest.mark.parametrize("nq", [[30, 9], [3, 2]], ids=str)
def test_attention_bounds_far_above_the_queries(nq):
    """max_q is a bound: "no limit" computes the same rows as n_q does, bit for
    bit (and as the tight value, where that chooses the same kernel), and
    nothing around them is touched."""
    rng = np.random.default_rng(sum(nq))
    page, H, G, D, lens = 16, 1, 2, 64, [37, 20]
    codes, scales, cache = make_cache(rng, 8, page, H, D)
    table = i32(rng.permutation(8)[:6].reshape(2, 3))
    cu = np.concatenate([[0], np.cumsum(nq)])
    q = rows(rng, int(cu[-1]), H * G, D, "f16", spread=False)
    outs = []
    for max_q in (max(nq), 2 ** 31 - 1, int(cu[-1])):
        buf = torch.full((256 + int(cu[-1]) + 256, H * G, D), 77.0, dtype=torch.float16, device=DEV)
        cache.attention(q, i32(cu), i32(lens), table, max_q=max_q, max_kv=37, out=buf[256:-256])
        assert (buf[:256] == 77.0).all() and (buf[-256:] == 77.0).all()
        outs.append(host(buf[256:-256]))
    want, most = ref.attention(codes, scales, host(q), cu, lens, host(table), H * G, True, D ** -0.5)
    for out in outs:
        check_attn(out, want, most, "f16", "f16", host(q), codes, scales, D ** -0.5, 37)
    np.testing.assert_array_equal(outs[1], outs[2])
    if max(nq) * G > 16:
        np.testing.assert_array_equal(outs[0], outs[2])


@pytest.mark.parametrize("nq,G,page", [(1, 1, 64), (5, 1, 16), (1, 4, 32), (3, 4, 16), (16, 1, 64), (30, 1, 32)])
def test_attention_queries_of_one_sign(nq, G, page):
    """Queries far from zero on one side, keys whose sums nearly cancel: every
    product and partial sum of codes and these queries fits 24 bits, so scores
    carry no rounding of the sum of the queries."""
    rng = np.random.default_rng(nq * G + page)
    H, D, n = 2, 128, 100
    codes, scales, cache = make_cache(rng, 8, page, H, D)
    codes[:, 0, :, :, 1::2] = -codes[:, 0, :, :, 0::2]
    scales[:, 0] = 1.0
    cache.codes.copy_(torch.tensor(codes))
    cache.scales.copy_(torch.tensor(scales))
    table = rng.permutation(8)[None]
    q = rows(rng, nq, H * G, D, "f16", spread=False)
    q.copy_(q.float().clamp(-3, 3) * 0.05 + 8.0)  # steps of 2^-7 below 8, 2^-8 above
    out = torch.full_like(q, 77.0)
    cache.attention(q, i32([0, nq]), i32([n]), i32(table), max_q=nq, max_kv=n, causal=False, out=out)
    want, most = ref.attention(codes, scales, host(q), [0, nq], [n], table, H * G, False, D ** -0.5)
    check_attn(host(out), want, most, "f16", "f16", host(q), codes, scales, D ** -0.5, n)


@pytest.mark.parametrize("nq,G,D,page", [(1, 1, 64, 64), (1, 8, 64, 16), (1, 2, 128, 32), (12, 1, 64, 64), (4, 4, 128, 16),
                                         (40, 1, 64, 32)])
def test_attention_small_values_beside_a_strong_zero(nq, G, D, page):
    """A token 9.6 nats above 63 others, its value 0 and theirs one step: the
    output is their weights alone (each an f16 of 11 bits, all alike, 2^-11),
    with the scores and fp32 sums within 2^-13 and the output rounded by
    2^-11. No rounding of the strong token's weight times an offset is in it."""
    pages = 64 // page
    codes = np.zeros((pages, 2, 1, page, D), np.int8)
    codes[:, 1] = 1
    codes[0, 0, 0, 7, 0], codes[0, 1, 0, 7] = 127, 0
    scales = np.ones((pages, 2, 1), np.float32)
    scales[:, 1] = 16.0
    cache = wgdec.Kv8Cache(torch.tensor(codes, device=DEV), torch.tensor(scales, device=DEV))
    q = torch.zeros(nq, G, D, dtype=torch.float16, device=DEV)
    q[:, :, 0] = 9.6 / (127 * D ** -0.5)
    top = 127 * D ** -0.5 * float(q[0, 0, 0])
    out = torch.empty_like(q)
    cache.attention(q, i32([0, nq]), i32([64]), i32(np.arange(pages)[None]), max_q=nq, max_kv=64, causal=False, out=out)
    want = 16.0 * 63 * np.exp(-top) / (1 + 63 * np.exp(-top))
    assert np.abs(host(out) / want - 1).max() <= 2.0 ** -11 + 2.0 ** -13 + 2.0 ** -11


@pytest.mark.parametrize("gap", [9.0, 17.5, 19.0, 23.0])
@pytest.mark.parametrize("nq,G,D,page", [(1, 1, 64, 64), (1, 4, 128, 16), (1, 12, 64, 16), (1, 16, 128, 32), (5, 1, 64, 16),
                                         (33, 1, 64, 16), (20, 1, 128, 64)])
def test_attention_many_weak_tokens_under_a_strong_one(nq, G, D, page, gap):
    """One token `gap` nats above n others that share what is left of the mass,
    and all of the output: its own value is 0. The weak weights are all alike,
    so their rounding to f16 shows as it is: by 2^-11 where they are normal
    numbers (2^-28 of the largest and up), else by 2^-39 of the largest. The
    scores (25 to 33 octaves in fp32, products and sums of one term) and the
    fp32 sums stay within 2^-13, the output is rounded by 2^-11."""
    n = 60000
    pages = -(-n // page)
    strong = 31 * page + 7
    codes = np.zeros((pages, 2, 1, page, D), np.int8)
    codes[:, 1] = 100
    codes[31, 0, 0, 7, 0], codes[31, 1, 0, 7] = 127, 0
    scales = np.ones((pages, 2, 1), np.float32)
    scales[:, 1] = 2.0 ** 6
    cache = wgdec.Kv8Cache(torch.tensor(codes, device=DEV), torch.tensor(scales, device=DEV))
    q = torch.zeros(nq, G, D, dtype=torch.float16, device=DEV)
    q[:, :, 0] = gap / (127 * D ** -0.5)
    top = 127 * D ** -0.5 * float(q[0, 0, 0])
    out = torch.empty_like(q)
    cache.attention(q, i32([0, nq]), i32([n]), i32(np.arange(pages)[None]), max_q=nq, max_kv=n, causal=False, out=out)
    weak = np.exp(-top) * (n - 1)
    want = 6400.0 * weak / (1 + weak)
    tol = 2.0 ** -11 if np.exp(-top) >= 2.0 ** -28 else 2.0 ** -39 / np.exp(-top)
    assert strong < n and np.abs(host(out) / want - 1).max() <= tol + 2.0 ** -13 + 2.0 ** -11


@pytest.mark.parametrize("qdt", ["bf16", "f32"])
@pytest.mark.parametrize("nq,G,D,page", [(1, 1, 64, 16), (2, 3, 128, 64), (11, 1, 64, 32), (24, 1, 128, 16), (24, 1, 64, 64)])
def test_attention_queries_of_a_wide_range(nq, G, D, page, qdt):
    """A query's largest value meets codes of 0; the rest, 2^-22 of it, make the
    scores. 8 bits (bf16) or 11 bits (fp32) of every value reach the product."""
    rng = np.random.default_rng(nq + D)
    H, n = 1, 90
    codes, scales, cache = make_cache(rng, 8, page, H, D)
    codes[:, 0, ..., 3] = 0
    scales[:, 0] = 2.0 ** -5
    cache.codes.copy_(torch.tensor(codes))
    cache.scales.copy_(torch.tensor(scales))
    table = rng.permutation(8)[None]
    steps = 128 if qdt == "bf16" else 1024
    x = (1 + rng.integers(0, steps, (nq, H * G, D)) / steps) * rng.choice([-1, 1], (nq, H * G, D)) * 2.0 ** -22
    x[..., 3] = 1.0
    q = torch.tensor(x, dtype=DT[qdt], device=DEV)
    np.testing.assert_array_equal(host(q), x)
    scale = 2.0 ** 22 * D ** -0.5
    out = torch.full((nq, H * G, D), 77.0, dtype=torch.float16, device=DEV)
    cache.attention(q, i32([0, nq]), i32([n]), i32(table), max_q=nq, max_kv=n, causal=False, scale=scale, out=out)
    want, most = ref.attention(codes, scales, x, [0, nq], [n], table, H * G, False, scale)
    check_attn(host(out), want, most, "f16", "exact", x, codes, scales, scale, n)


@pytest.mark.parametrize("mul", [2.0 ** 126, 2.0 ** -100, 2.0 ** -120])
@pytest.mark.parametrize("nq", [1, 10, 20])
def test_attention_queries_at_the_ends_of_bf16(nq, mul):
    rng = np.random.default_rng(nq)
    H, D, n, page = 1, 64, 60, 16
    codes, scales, cache = make_cache(rng, 4, page, H, D)
    table = rng.permutation(4)[None]
    x = np.clip(rng.standard_normal((nq, H, D)), -1.9, 1.9)
    q = (torch.tensor(x, dtype=torch.bfloat16, device=DEV).double() * mul).to(torch.bfloat16)
    # scores of order 1: the scale takes back what it can, the page's steps the rest
    scale = min(max(1.0 / mul, 2.0 ** -120), 2.0 ** 100) / 8
    scales[:, 0] = 1.0 / (mul * scale * 64 * 8)
    cache.scales.copy_(torch.tensor(scales))
    out = torch.full((nq, H, D), 77.0, dtype=torch.bfloat16, device=DEV)
    cache.attention(q, i32([0, nq]), i32([n]), i32(table), max_q=nq, max_kv=n, causal=False, scale=scale, out=out)
    want, most = ref.attention(codes, scales, host(q), [0, nq], [n], table, H, False, float(np.float32(scale)))
    check_attn(host(out), want, most, "bf16", "bf16", host(q), codes, scales, scale, n)


def test_offsets_past_32_bits():
    """A cache of 4.6 GB: pages whose codes lie beyond 2^32 bytes are written, read and attended to."""
    page, H, D = 64, 20, 64
    pages = 28100  # x 163,840 bytes
    cache = wgdec.Kv8Cache.alloc(pages, page, H, D, device=DEV)
    rng = np.random.default_rng(9)
    ids = [pages - 1, 1, 26300, 13107]  # ends, and either side of 2^31 and 2^32 bytes
    n = 4 * page - 3
    slots = np.concatenate([np.arange(i * page, (i + 1) * page) for i in ids])[:n]
    k, v = rows(rng, n, H, D, "f16"), rows(rng, n, H, D, "f16")
    cache.append(k, v, i32(slots))
    ko, vo = torch.zeros(n, H, D, device=DEV), torch.zeros(n, H, D, device=DEV)
    cache.read(i32(slots), ko, vo)
    codes, scales = np.zeros((4, 2, H, page, D), np.int8), np.zeros((4, 2, H), np.float32)
    ref.append(codes, scales, host(k), host(v), np.arange(n))
    val = codes.astype(np.float64) * scales[..., None, None]
    np.testing.assert_array_equal(host(ko), val[:, 0].transpose(0, 2, 1, 3).reshape(-1, H, D)[:n])
    np.testing.assert_array_equal(host(vo), val[:, 1].transpose(0, 2, 1, 3).reshape(-1, H, D)[:n])
    q = rows(rng, 2, H, D, "f16", spread=False)
    q.mul_(2.0 ** -6)
    out = torch.full_like(q, 77.0)
    cache.attention(q, i32([0, 2]), i32([n]), i32([ids]), max_q=2, max_kv=n, out=out)
    want, most = ref.attention(codes, scales, host(q), [0, 2], [n], np.arange(4)[None], H, True, D ** -0.5)
    check_attn(host(out), want, most, "f16", "f16", host(q), codes, scales, D ** -0.5, n)


# ---- wg_sample_rows -----------------------------------------------------------------
def check_sample(x, u, T, k, p, m, dt="f32", ld_pad=0):
    """Tokens equal; log-probs within the rounding to fp32 and 2^-15 for a sum
    of up to 2^18 fp32 weights (each within 2^-18 relative where it matters)."""
    R, V = x.shape
    buf = torch.zeros(R, V + ld_pad, dtype=DT[dt], device=DEV)
    lg = buf[:, :V]
    lg.copy_(torch.tensor(x))
    f = lambda a: None if a is None else torch.tensor(np.asarray(a, np.float32), device=DEV)  # noqa: E731
    uu = np.asarray(u, np.float32)
    before = lg.clone()
    tok, lp = wgdec.sample_rows(lg, f(u), f(T), None if k is None else i32(k), f(p), f(m))
    assert torch.equal(torch.nan_to_num(before.float()), torch.nan_to_num(lg.float()))
    xs = host(lg)
    g = lambda a, r, d: d if a is None else float(np.float32(a[r]))  # noqa: E731
    for r in range(R):
        t, l = ref.sample(xs[r], float(uu[r]), g(T, r, 1.0), 0 if k is None else int(k[r]), g(p, r, 1.0), g(m, r, 0.0))
        assert int(tok[r]) == t, r
        if t >= 0 and np.isfinite(l):
            assert abs(float(lp[r]) - l) <= 2.0 ** -24 * abs(l) + 2.0 ** -15, r
        else:
            assert float(lp[r]) == l, r


SETTINGS = [dict(), dict(T=0.7), dict(T=0.0), dict(T=-1.0), dict(k=1), dict(k=50), dict(k=10 ** 6), dict(p=0.9),
            dict(p=0.0), dict(p=1.5), dict(m=0.05), dict(m=1.0), dict(m=2.0), dict(T=0.8, k=200, p=0.95, m=0.02),
            dict(T=30.0, p=0.5), dict(T=0.01, k=40), dict(T=1e-30, p=0.3), dict(k=500, p=0.999), dict(T=1.3, p=0.9999)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 8191, 51865])
def test_sample(V, dt):
    rng = np.random.default_rng(V)
    R = len(SETTINGS)
    x = rng.standard_normal((R, V)) * 2.5
    x[:, rng.integers(0, V, 8)] += 6
    get = lambda n, d: np.array([s.get(n, d) for s in SETTINGS])  # noqa: E731
    for j in range(2):
        check_sample(x, rng.random(R), get("T", 1.0), get("k", 0), get("p", 1.0), get("m", 0.0), dt, ld_pad=3 * j)


WIDE = [dict(k=1000), dict(k=1500), dict(k=30000, T=2.0), dict(k=5000, p=0.999, T=1.5), dict(p=0.99, T=2.5),
        dict(p=0.9, T=5.0, m=1e-4), dict(m=1e-6), dict(m=1e-3, T=4.0), dict(k=1024, m=0.3, T=3.0), dict(p=0.9999999)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", ["normal", "flat", "steps", "far"])
def test_sample_keeps_many(dt, shape):
    """Kept sets of thousands: no short list, cuts by descents; flat rows, rows
    of few distinct values, and rows whose tail lies far below the rest."""
    V, R = 51865, len(WIDE)
    rng = np.random.default_rng(len(shape))
    x = rng.standard_normal((R, V)) * {"normal": 2.5, "flat": 0.05, "steps": 2.0, "far": 1.0}[shape]
    if shape == "steps":
        x = np.round(x)
    if shape == "far":
        x[:, ::2] -= 200.0
    get = lambda n, d: np.array([s.get(n, d) for s in WIDE])  # noqa: E731
    check_sample(x, rng.random(R), get("T", 1.0), get("k", 0), get("p", 1.0), get("m", 0.0), dt)


@pytest.mark.parametrize("n", [256, 257, 1023, 1024, 1025])
def test_sample_lists_of_every_length(n):
    """Exactly n candidates: ordered by counting, by sorting, and too many for either."""
    V = 20000
    rng = np.random.default_rng(n)
    x = np.full((6, V), -90.0)
    for r in range(6):
        x[r, rng.permutation(V)[:n]] = rng.standard_normal(n)
    check_sample(x, rng.random(6), [1.0] * 6, [0, n, n - 1, 0, 0, 100], [0.95, 1.0, 0.9, 1.0, 0.9999, 0.5],
                 [0, 0, 0, 1e-9, 1e-9, 0])


def test_sample_defaults_and_many_rows():
    rng = np.random.default_rng(11)
    x = rng.standard_normal((400, 777)) * 3
    check_sample(x, rng.random(400), None, None, None, None)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [2049, 3001, 4095, 4096])
def test_sample_vocabularies_of_two_slices(V, dt):
    """Short and long kept sets, exact masses, ties and edges of rows that two CTAs share."""
    sets = SETTINGS + [dict(k=1025), dict(k=V - 3), dict(k=1500, p=0.999, T=2.0), dict(p=0.99, T=4.0), dict(p=0.5, T=9.0, m=1e-3),
                       dict(m=1e-6), dict(m=1e-3, T=5.0), dict(k=1024, m=0.2, T=3.0), dict(p=0.9999999)]
    get = lambda n, d: np.array([s.get(n, d) for s in sets])  # noqa: E731
    rng = np.random.default_rng(V)
    R = len(sets)
    for shape in range(3):
        x = rng.standard_normal((R, V)) * (2.5, 0.05, 2.0)[shape]
        if shape == 2:
            x = np.round(x)  # ties by the hundred, at every cut
        check_sample(x, rng.random(R), get("T", 1.0), get("k", 0), get("p", 1.0), get("m", 0.0), dt, ld_pad=shape)


@pytest.mark.parametrize("V", [130001, 262144])
def test_sample_wide_vocabularies(V):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((4, V)) * 2
    check_sample(x, rng.random(4), [1.0, 0.8, 1.0, 1.2], [0, 64, 0, 0], [1.0, 0.9, 0.95, 1.0], [0, 0, 0.01, 0.1])


def test_sample_ties():
    """Equal logits: the lowest indices stay, and the draw is by exact counts."""
    V = 4099
    x = np.zeros((8, V))
    x[4:, 7::3] = 1.0
    x[6] = np.round(np.random.default_rng(1).standard_normal(V) * 2) / 2
    x[7] = x[6]
    check_sample(x, [0.0, 0.5, 0.9999999, 0.25, 0.3, 0.6, 0.4, 0.8], [1.0] * 8, [0, 0, 0, 100, 50, 0, 700, 0],
                 [1.0, 0.25, 1.0, 0.5, 1.0, 0.6, 0.7, 0.31], [0] * 8)


def test_sample_masked_rows():
    """Masks of -inf and of the type's lowest value, NaN, +inf, rows with nothing, rows with one token."""
    V = 2000
    rng = np.random.default_rng(2)
    x = rng.standard_normal((10, V)) * 2
    low = float(np.finfo(np.float32).min)
    x[0] = -np.inf
    x[1, :] = -np.inf
    x[1, 1234] = -3.0
    x[2, 100:] = low
    x[3] = low
    x[4, 5:500] = np.nan
    x[5] = np.nan
    x[6, [30, 700]] = np.inf
    x[7, 1500:] = -np.inf
    x[8, :] = -np.inf
    x[8, 3] = low
    x[9, 4:] = low
    check_sample(x, [0.5, 0.2, 0.99, 0.75, 0.4, 0.1, 0.7, 0.999, 0.3, 0.8], [1, 1, 0.5, 1, 2, 1, 1, 1, 1, 1],
                 [0, 0, 150, 0, 900, 0, 0, 0, 5, 10], [0.9, 0.9, 0.99, 0.5, 1.0, 1, 0.9, 0.97, 1.0, 1.0],
                 [0, 0, 0, 0, 0.1, 0, 0.5, 0, 0, 0])


@pytest.mark.parametrize("gap", [4.0, 9.0, 15.0, 19.0])
def test_sample_logprob_of_a_nearly_certain_token(gap):
    """log-prob = -log(1 + rest): the rest of the row is summed apart from the
    maximum, so its digits stay: every weight exp(-gap - d) is within
    2^-22 + 3 * 2^-24 * (its octaves, at most 60) and the sum's adds within 2^-18."""
    V = 30000
    rng = np.random.default_rng(int(gap))
    x = (rng.standard_normal((2, V)) - gap - np.log(V)).astype(np.float32)
    x[:, 77] = 0.0
    x[1, 78] = 0.0
    tok, lp = wgdec.sample_rows(torch.tensor(x, device=DEV), torch.tensor([0.5, 0.25], device=DEV))
    for r in range(2):
        _, want = ref.sample(x[r].astype(np.float64), 0.5 if r == 0 else 0.25)
        assert int(tok[r]) == 77 and abs(float(lp[r]) - want) <= abs(want) * (2.0 ** -22 + 180 * 2.0 ** -24 + 2.0 ** -18)


@pytest.mark.parametrize("V,C", [(300, 1.5), (3001, 2.5), (51865, 2.5), (51865, 0.1)])
def test_sample_at_the_edges_of_elements(V, C):
    """Rows without filters, numbers as near to a running mass as fp32 has
    them: beside every edge the 64-bit sums decide. The exact units (2^-45 of
    the largest weight) are off by less than V 2^-46 <= 2^-30 of a row's mass;
    numbers nearer than 2^-29 to an edge are not used."""
    R = 96
    rng = np.random.default_rng(V)
    x = (rng.standard_normal(V) * C).astype(np.float32)
    cum = np.cumsum(np.exp(x.astype(np.float64) - x.max()))
    edge = cum / cum[-1]
    u, want = [], []
    for j in rng.integers(0, V - 1, 4 * R):
        for step in (-1, 0, 1, 20, -20):  # ulps off the edge's fp32 value
            v = np.float32(edge[j]) * np.float32(1 + step * 2.0 ** -23)
            i = int(np.searchsorted(edge, float(v), side="right"))
            near = min(abs(edge[q] - float(v)) for q in (max(0, i - 1), min(i, V - 1)))
            if v < 1 and near > 2.0 ** -29:
                u.append(v)
                want.append(i)
    u, want = u[:R], want[:R]
    assert len(u) == R
    lg = torch.tensor(x, device=DEV).expand(R, V).contiguous()
    tok, _ = wgdec.sample_rows(lg, torch.tensor(np.array(u), device=DEV))
    np.testing.assert_array_equal(host(tok), want)


@pytest.mark.parametrize("V", [300, 1000, 3001, 4099, 51865])
@pytest.mark.parametrize("depth", [25.0, 31.9, 33.0, 40.0, 300.0])
def test_sample_the_number_zero(V, depth):
    """u = 0 is the first kept token in index order, also where its weight is
    far below the units in which masses are held; with and without filters,
    beside rows whose number is not 0."""
    sets = [dict(), dict(k=40), dict(k=V - 7), dict(p=0.9), dict(m=1e-20), dict(m=1e-12), dict(k=200, m=1e-16), dict(T=0.5),
            dict(k=30, p=0.5), dict(k=V // 2, p=0.999999), dict(m=1e-44), dict(T=0.0), dict(k=V // 2, T=3.0, m=1e-17)]
    R = 2 * len(sets)
    rng = np.random.default_rng(V + int(depth))
    x = rng.standard_normal((R, V)) * 2 - depth
    x[:, V // 2] = 0.0
    x[3, :5] = -np.inf
    x[4, 0] = np.nan
    get = lambda n, d: np.array([s.get(n, d) for s in sets + sets])  # noqa: E731
    u = np.where(np.arange(R) < len(sets), 0.0, rng.random(R))
    check_sample(x, u, get("T", 1.0), get("k", 0), get("p", 1.0), get("m", 0.0))


@pytest.mark.parametrize("n", [300, 1000])
def test_sample_list_in_one_bin(n):
    """Candidates that share a histogram bin, equal or an ulp apart."""
    V = 9000
    rng = np.random.default_rng(n)
    x = np.full((4, V), -60.0)
    for r in range(4):
        x[r, rng.permutation(V)[:n]] = 5.0 + (np.arange(n) % (r + 1)) * 2.0 ** -10
    check_sample(x, rng.random(4), [1.0] * 4, [n // 2, 0, 0, n // 3], [1.0, 0.6, 0.9, 0.5], [0, 0, 0, 0])


def test_sample_distribution():
    """Drawn frequencies follow the kept weights: 40,000 stratified draws of
    one row, so each token's count is within 1 of its share."""
    rng = np.random.default_rng(3)
    V, n = 300, 40000
    row = rng.standard_normal(V) * 1.5
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    lg = torch.tensor(row, dtype=torch.float32, device=DEV).expand(n, V).contiguous()
    tok, _ = wgdec.sample_rows(lg, torch.tensor(u, device=DEV), top_k=i32(np.full(n, 20)))
    x = host(lg[0])
    keep = np.sort(np.argsort(-x, kind="stable")[:20])
    share = np.exp(x[keep] - x[keep].max())
    share = share / share.sum() * n
    count = np.bincount(host(tok), minlength=V)
    # a stratum whose u lies within 2^-24 of a border may fall on either side
    assert count.sum() == count[keep].sum() and (np.abs(count[keep] - share) <= 2).all()


# ---- together -------------------------------------------------------------------------
def test_other_stream_and_two_at_once():
    """Calls follow the current torch stream; two streams with their own tensors do not disturb each other."""
    rng = np.random.default_rng(12)
    page, H, D, L = 16, 4, 64, 500
    sets = []
    for _ in range(2):
        codes, scales, cache = make_cache(rng, 40, page, H, D)
        table = rng.permutation(40)[:32].reshape(1, 32)
        q = rows(rng, 3, H, D, "f16", spread=False)
        want, most = ref.attention(codes, scales, host(q), [0, 3], [L], table, H, True, D ** -0.5)
        sets.append((cache, i32(table), q, torch.empty_like(q), want, most, codes, scales, torch.cuda.Stream()))
    cu, lens = i32([0, 3]), i32([L])
    torch.cuda.synchronize()
    for _ in range(20):
        for cache, table, q, out, *_, st in sets:
            with torch.cuda.stream(st):
                cache.attention(q, cu, lens, table, max_q=3, max_kv=L, out=out)
    torch.cuda.synchronize()
    for cache, table, q, out, want, most, codes, scales, _ in sets:
        check_attn(host(out), want, most, "f16", "f16", host(q), codes, scales, D ** -0.5, L)


class Server:
    """A token loop over the operators: streams of different ages, padded to a fixed batch."""

    def __init__(self, R, page, H, G, D, pages, cols, V, seed):
        rng = np.random.default_rng(seed)
        self.R, self.page, self.H, self.G, self.D, self.V = R, page, H, G, D, V
        self.cache = wgdec.Kv8Cache.alloc(pages, page, H, D, device=DEV)
        self.table = i32(np.full((R, cols), -1))
        self.free, self.cursor = i32(rng.permutation(pages)), i32([0])
        self.lens, self.new = i32(np.zeros(R)), i32(np.zeros(R))
        self.status = i32([0, 0])
        self.rng = rng

    def buffers(self, n):
        H, G, D = self.H, self.G, self.D
        f16 = dict(dtype=torch.float16, device=DEV)
        self.slots, self.cu = i32(np.zeros(n)), i32(np.zeros(self.R + 1))
        self.q, self.k, self.v = torch.zeros(n, H * G, D, **f16), torch.zeros(n, H, D, **f16), torch.zeros(n, H, D, **f16)
        self.out = torch.full((n, H * G, D), 77.0, **f16)
        self.logits = torch.zeros(self.R, self.V, device=DEV)
        self.u = torch.zeros(self.R, device=DEV)
        self.T, self.p = torch.full((self.R,), 0.8, device=DEV), torch.full((self.R,), 0.9, device=DEV)
        self.tokens, self.lp = i32(np.zeros(self.R)), torch.zeros(self.R, device=DEV)

    def step(self, max_q, max_kv):
        wgdec.kv_plan(self.lens, self.new, self.page, self.free, self.cursor, self.table, self.slots, self.cu, self.status)
        self.cache.append(self.k, self.v, self.slots)
        self.cache.attention(self.q, self.cu, self.lens, self.table, max_q=max_q, max_kv=max_kv, out=self.out)
        wgdec.sample_rows(self.logits, self.u, temperature=self.T, top_p=self.p, tokens=self.tokens, logprobs=self.lp)


@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(graph):
    """Prompts, then single tokens of streams that come and go, planned,
    cached, attended to and sampled step by step (the single-token steps also
    as one captured graph, replayed), against the plain forms kept alongside."""
    R, page, H, G, D, V = 5, 16, 2, 2, 64, 1000
    s = Server(R, page, H, G, D, 64, 8, V, 21)
    codes, scales = np.zeros((64, 2, H, page, D), np.int8), np.zeros((64, 2, H), np.float32)
    free, table, cursor = host(s.free), np.full((R, 8), -1), 0
    lens = np.zeros(R, int)
    captured = None
    for step in range(9):
        if step == 0:
            new = np.array([20, 1, 0, 33, 16])
            s.buffers(int(new.sum()) + 3)
        else:
            new = np.array([1, 1, step % 2, 0 if step > 5 else 1, 1])
            if step == 1:
                s.buffers(R)
        lens = lens + new
        n = s.slots.shape[0]
        for t in (s.q, s.k, s.v):
            t.copy_(torch.tensor(s.rng.standard_normal(t.shape)))
        s.k[int(new.sum()):] = float("nan")  # rows behind the last sequence hold anything
        s.logits.copy_(torch.tensor(s.rng.standard_normal((R, V)) * 3))
        s.u.copy_(torch.tensor(s.rng.random(R)))
        s.out.fill_(77.0)
        s.lens.copy_(i32(lens))
        s.new.copy_(i32(new))
        if graph and step >= 2:
            if captured is None:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=side):
                    s.step(1, 128)
                torch.cuda.synchronize()
            captured.replay()
        else:
            s.step(int(new.max()), int(lens.max()))
        torch.cuda.synchronize()
        code, table, slots, cu, cursor, _ = ref.plan(lens, new, page, free, cursor, table, n)
        assert code == 0 and host(s.status)[0] == 0
        np.testing.assert_array_equal(host(s.table), table)
        np.testing.assert_array_equal(host(s.slots), slots)
        ref.append(codes, scales, host(s.k), host(s.v), slots)
        want, most = ref.attention(codes, scales, host(s.q), cu, lens, table, H * G, True, D ** -0.5)
        check_attn(host(s.out), want, most, "f16", "f16", host(s.q), codes, scales, D ** -0.5, int(lens.max()))
        for r in range(R):
            tok, _ = ref.sample(host(s.logits[r]), float(s.u[r]), float(s.T[r]), 0, float(s.p[r]), 0.0)
            assert int(s.tokens[r]) == tok
