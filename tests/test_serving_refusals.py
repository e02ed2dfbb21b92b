"""Argument checks of the serving operators (no GPU needed): every refusal
comes before any device work, with the documented status and a message that
names the call."""
import ctypes

import pytest

import wgdec

INVALID, UNSUPPORTED, NO_DEVICE = 1, 4, 8
PTR = 4096  # a plausible, 16-byte aligned address that no refused call touches


def last():
    return wgdec.last_error()


def cache(**kw):
    f = dict(codes=PTR, scales=PTR, num_pages=8, page=16, n_kv_head=2, head_dim=64)
    f.update(kw)
    return wgdec.WgKv8(**f)


def attn(**kw):
    f = dict(q=PTR, ldq=128, q_dtype=1, n_head=2, cu_q=PTR, n_q=4, n_requests=2, kv_lens=PTR, block_table=PTR,
             ld_table=4, max_pages=4, max_q=2, max_kv=64, causal=1, scale=0.125, out_dtype=1, out=PTR, ldo=128)
    f.update(kw)
    return wgdec.WgKv8Attn(**f)


def smp(**kw):
    f = dict(logits=PTR, ld=100, dtype=0, R=2, V=100, u=PTR, tokens=PTR)
    f.update(kw)
    return wgdec.WgSample(**f)


BAD_CACHES = [dict(codes=None), dict(scales=None), dict(num_pages=0), dict(page=8), dict(page=48), dict(page=256),
              dict(n_kv_head=0), dict(head_dim=32), dict(head_dim=96), dict(codes=PTR + 8), dict(scales=PTR + 2),
              dict(num_pages=1 << 27, page=16)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches(bad):
    L, c = wgdec.lib(), cache(**bad)
    assert L.wg_kv8_append(ctypes.byref(c), PTR, PTR, 1, 128, 128, PTR, 4, 0, None) == INVALID
    assert last().startswith("wg_kv8_append")
    assert L.wg_kv8_read(ctypes.byref(c), PTR, 4, PTR, PTR, 1, 128, 128, 0, None) == INVALID
    assert last().startswith("wg_kv8_read")
    assert L.wg_kv8_attention(ctypes.byref(c), ctypes.byref(attn()), 0, None) == INVALID
    assert last().startswith("wg_kv8_attention")


@pytest.mark.parametrize("args", [(None, PTR, 1, 128, 128, PTR, 4), (PTR, None, 1, 128, 128, PTR, 4),
                                  (PTR, PTR, 8, 128, 128, PTR, 4), (PTR, PTR, 1, 127, 128, PTR, 4),
                                  (PTR, PTR, 1, 128, 127, PTR, 4), (PTR, PTR, 1, 128, 128, None, 4),
                                  (PTR, PTR, 1, 128, 128, PTR, -1), (PTR + 1, PTR, 1, 128, 128, PTR, 4)], ids=str)
def test_bad_rows(args):
    L, c = wgdec.lib(), cache()
    k, v, dt, ldk, ldv, slots, n = args
    assert L.wg_kv8_append(ctypes.byref(c), k, v, dt, ldk, ldv, slots, n, 0, None) == INVALID
    assert L.wg_kv8_read(ctypes.byref(c), slots, n, k, v, dt, ldk, ldv, 0, None) == INVALID


@pytest.mark.parametrize("bad,status", [(dict(n_head=3), INVALID), (dict(n_head=0), INVALID), (dict(ldq=127), INVALID),
                                        (dict(ldo=127), INVALID), (dict(ld_table=3), INVALID), (dict(n_q=-1), INVALID),
                                        (dict(n_requests=-1), INVALID), (dict(max_q=-1), INVALID),
                                        (dict(max_kv=-1), INVALID), (dict(max_pages=-1), INVALID),
                                        (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
                                        (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(cu_q=None), INVALID),
                                        (dict(kv_lens=None), INVALID), (dict(block_table=None), INVALID),
                                        (dict(q=PTR + 1), INVALID), (dict(q_dtype=8), UNSUPPORTED),
                                        (dict(out_dtype=0), UNSUPPORTED)], ids=str)
def test_bad_attention(bad, status):
    assert wgdec.lib().wg_kv8_attention(ctypes.byref(cache()), ctypes.byref(attn(**bad)), 0, None) == status
    assert last().startswith("wg_kv8_attention")


def test_bad_plan():
    L = wgdec.lib()
    good = [PTR, PTR, 3, 16, PTR, 10, PTR, PTR, PTR, 4, 4, PTR, 8, PTR, PTR, 0, None]
    for at, v in [(0, None), (1, None), (2, 0), (3, 8), (3, 24), (4, None), (5, -1), (6, None), (7, None), (8, None),
                  (9, 3), (10, 0), (11, None), (12, -1), (13, None), (14, None)]:
        args = list(good)
        args[at] = v
        assert L.wg_kv_plan(*args) == INVALID, at
        assert last().startswith("wg_kv_plan")


@pytest.mark.parametrize("bad,status", [(dict(V=0), INVALID), (dict(V=(1 << 18) + 1, ld=1 << 19), INVALID),
                                        (dict(ld=99), INVALID), (dict(R=-1), INVALID), (dict(logits=None), INVALID),
                                        (dict(u=None), INVALID), (dict(tokens=None), INVALID),
                                        (dict(logits=PTR + 2), INVALID), (dict(dtype=8), UNSUPPORTED)], ids=str)
def test_bad_sample(bad, status):
    assert wgdec.lib().wg_sample_rows(ctypes.byref(smp(**bad)), 0, None) == status
    assert last().startswith("wg_sample_rows")


def test_null_descriptors():
    L = wgdec.lib()
    assert L.wg_kv8_append(None, PTR, PTR, 1, 128, 128, PTR, 4, 0, None) == INVALID
    assert L.wg_kv8_attention(None, ctypes.byref(attn()), 0, None) == INVALID
    assert L.wg_kv8_attention(ctypes.byref(cache()), None, 0, None) == INVALID
    assert L.wg_sample_rows(None, 0, None) == INVALID


def test_empty_calls_do_nothing():
    L = wgdec.lib()
    assert L.wg_kv8_append(ctypes.byref(cache()), None, None, 1, 128, 128, None, 0, 0, None) == 0
    assert L.wg_kv8_read(ctypes.byref(cache()), None, 0, None, None, 1, 128, 128, 0, None) == 0
    for kw in (dict(n_requests=0), dict(n_q=0), dict(max_q=0)):
        assert L.wg_kv8_attention(ctypes.byref(cache()), ctypes.byref(attn(**kw)), 0, None) == 0
    assert L.wg_sample_rows(ctypes.byref(smp(R=0)), 0, None) == 0


@pytest.mark.skipif(wgdec.device_count() > 0, reason="a CUDA device is visible")
def test_no_device():
    L = wgdec.lib()
    assert L.wg_kv8_append(ctypes.byref(cache()), PTR, PTR, 1, 128, 128, PTR, 4, 0, None) == NO_DEVICE
    assert L.wg_kv8_attention(ctypes.byref(cache()), ctypes.byref(attn()), 0, None) == NO_DEVICE
    assert L.wg_sample_rows(ctypes.byref(smp()), 0, None) == NO_DEVICE
    assert L.wg_kv_plan(PTR, PTR, 3, 16, PTR, 10, PTR, PTR, PTR, 4, 4, PTR, 8, PTR, PTR, 0, None) == NO_DEVICE


def test_mirror_refuses_host_tensors_and_wrong_shapes():
    torch = pytest.importorskip("torch")
    with pytest.raises(wgdec.DecodeError):
        wgdec.Kv8Cache(torch.zeros(2, 2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 2, 1))  # not on a device
    with pytest.raises(wgdec.DecodeError):
        wgdec.Kv8Cache(torch.zeros(2, 2, 1, 16, 64), torch.zeros(2, 2, 1))  # not int8
    with pytest.raises(wgdec.DecodeError):
        wgdec.sample_rows(torch.zeros(2, 10), torch.zeros(2))
    with pytest.raises(wgdec.DecodeError):
        wgdec.sample_rows(torch.zeros(10), torch.zeros(1))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(wgdec.DecodeError):
        wgdec.kv_plan(i, i, 16, i, i[:1], torch.zeros(2, 2, dtype=torch.int32), i, torch.zeros(3, dtype=torch.int32), i)


@pytest.mark.parametrize("n_q,max_q,n_head,refused", [(1 << 29, 1 << 30, 6, True), (1 << 30, (1 << 30) - 1, 4, True),
                                                      (1 << 29, 2 ** 31 - 1, 4, False), (1, 2 ** 31 - 1, 64, False),
                                                      (2 ** 31 - 1, 1 << 29, 4, False)])
def test_attention_rows_are_counted_in_32_bits(n_q, max_q, n_head, refused):
    """(query, grouped head) rows of one K/V head: the lesser of max_q and n_q counts, and at most 2^30 of them pass."""
    p = attn(n_q=n_q, max_q=max_q, n_head=n_head, ldq=64 * n_head, ldo=64 * n_head, n_requests=0)
    assert wgdec.lib().wg_kv8_attention(ctypes.byref(cache()), ctypes.byref(p), 0, None) == 0  # no request: no work
    if refused or wgdec.device_count() == 0:  # what passes would run
        p.n_requests = 2
        status = wgdec.lib().wg_kv8_attention(ctypes.byref(cache()), ctypes.byref(p), 0, None)
        assert status == (INVALID if refused else NO_DEVICE) and (not refused or "too many" in last())


@pytest.mark.parametrize("R,n_slots", [((1 << 30) + 1, 8), (2 ** 31 - 1, 8), (3, (1 << 30) + 1), (3, 2 ** 31 - 1)])
def test_plan_refuses_what_its_indices_cannot_step_over(R, n_slots):
    """The kernel steps 32-bit indices by up to 2^18 past R and n_slots, so both end at 2^30."""
    assert wgdec.lib().wg_kv_plan(PTR, PTR, R, 16, PTR, 10, PTR, PTR, PTR, 4, 4, PTR, n_slots, PTR, PTR, 0, None) == INVALID
    assert last().startswith("wg_kv_plan")


def test_tensors_off_their_types_alignment():
    """Every int32 and fp32 tensor is checked: a kernel that met one of these would fault."""
    L, off = wgdec.lib(), PTR + 2
    good = [PTR, PTR, 3, 16, PTR, 10, PTR, PTR, PTR, 4, 4, PTR, 8, PTR, PTR, 0, None]
    for at in (0, 1, 4, 6, 7, 8, 11, 13, 14):
        args = list(good)
        args[at] = off
        assert L.wg_kv_plan(*args) == INVALID and "aligned" in last(), at
    assert L.wg_kv8_append(ctypes.byref(cache()), PTR, PTR, 1, 128, 128, off, 4, 0, None) == INVALID
    assert L.wg_kv8_read(ctypes.byref(cache()), off, 4, PTR, PTR, 1, 128, 128, 0, None) == INVALID
    for name in ("cu_q", "kv_lens", "block_table"):
        assert L.wg_kv8_attention(ctypes.byref(cache()), ctypes.byref(attn(**{name: off})), 0, None) == INVALID, name
    for name in ("u", "temperature", "top_k", "top_p", "min_p", "tokens", "logprobs"):
        assert L.wg_sample_rows(ctypes.byref(smp(**{name: off})), 0, None) == INVALID, name
