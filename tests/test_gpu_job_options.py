"""Decode jobs with options: the cross K/V cache in 8 bits, and drawn tokens.

The 8-bit cross cache is checked against the decoder's layers written out in
numpy (float64) around the same quantised cache; drawn tokens against the
64-bit definition of the draw on the oracle's logits."""
import numpy as np
import pytest

import oracle
import serving_ref as ref
import wgdec

pytestmark = pytest.mark.gpu
PROMPT = [50258, 50259, 50357, 50363]
ATOL, RTOL = 2e-2, 1e-3  # the gates of the f16 cache's parity tests


def weights(model, mat):
    """A descriptor matrix as float64 [rows, cols]."""
    import ctypes
    rb = wgdec.gen().wg_gen_row_bytes(mat.qtype, mat.cols)
    raw = ctypes.string_at(mat.data, mat.rows * rb)
    return oracle.dequant(mat.qtype, raw, mat.rows * mat.cols).astype(np.float64).reshape(mat.rows, mat.cols)


def vec(p, n):
    return np.ctypeslib.as_array(p, (n,)).astype(np.float64)


def layer_norm(x, w, b):
    m = x.mean(-1, keepdims=True)
    return (x - m) / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + 1e-5) * w + b


def gelu(x):
    return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))


def softmax(s):
    e = np.exp(s - s.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def heads(x, H):
    return x.reshape(x.shape[0], H, -1).transpose(1, 0, 2)


def quantised(x):
    """[T, H, 64] through the 8-bit cache's definition, pages of 64 frames."""
    T, H, D = x.shape
    pages = -(-T // 64)
    codes, scales = np.zeros((pages, 2, H, 64, D), np.int8), np.zeros((pages, 2, H), np.float32)
    ref.append(codes, scales, x, x, np.arange(T))
    v = codes[:, 0].astype(np.float64) * scales[:, 0, :, None, None]
    return v.transpose(0, 2, 1, 3).reshape(-1, H, D)[:T]


def forward(m, enc, tokens):
    """Logits of the last position (decoder.go:745-833) with the cross K/V of `enc` in the 8-bit cache."""
    d = wgdec._desc_ptr(m).contents
    n, H = d.n_state, d.n_head
    emb = weights(m, d.token_embedding)
    pos = np.ctypeslib.as_array(d.positional_embedding, (d.n_text_ctx, n)).astype(np.float64)
    x = emb[np.asarray(tokens)] + pos[:len(tokens)]
    P = len(tokens)
    mask = np.where(np.arange(P)[None, :] > np.arange(P)[:, None], -np.inf, 0.0)
    e16 = enc.astype(np.float16).astype(np.float64)  # the encoder output enters the products as f16
    for i in range(d.n_layer):
        L = d.layers[i]
        y = layer_norm(x, vec(L.self_ln_w, n), vec(L.self_ln_b, n))
        q, k, v = y @ weights(m, L.self_q).T + vec(L.self_q_b, n), y @ weights(m, L.self_k).T, \
            y @ weights(m, L.self_v).T + vec(L.self_v_b, n)
        a = softmax(heads(q, H) @ heads(k, H).transpose(0, 2, 1) / 8 + mask) @ heads(v, H)
        x = x + a.transpose(1, 0, 2).reshape(P, n) @ weights(m, L.self_o).T + vec(L.self_o_b, n)
        y = layer_norm(x, vec(L.cross_ln_w, n), vec(L.cross_ln_b, n))
        q = y @ weights(m, L.cross_q).T + vec(L.cross_q_b, n)
        k = (e16 @ weights(m, L.cross_k).T).astype(np.float16).astype(np.float64)
        v = (e16 @ weights(m, L.cross_v).T + vec(L.cross_v_b, n)).astype(np.float16).astype(np.float64)
        k, v = quantised(k.reshape(-1, H, 64)), quantised(v.reshape(-1, H, 64))
        a = softmax(heads(q, H) @ k.transpose(1, 2, 0) / 8) @ v.transpose(1, 0, 2)
        x = x + a.transpose(1, 0, 2).reshape(P, n) @ weights(m, L.cross_o).T + vec(L.cross_o_b, n)
        y = layer_norm(x, vec(L.mlp_ln_w, n), vec(L.mlp_ln_b, n))
        h = gelu(y @ weights(m, L.mlp0).T + vec(L.mlp0_b, 4 * n))
        x = x + h @ weights(m, L.mlp2).T + vec(L.mlp2_b, n)
    return layer_norm(x[-1:], vec(d.ln_w, n), vec(d.ln_b, n))[0] @ emb.T


@pytest.mark.parametrize("qtype,T", [("Q8_0", 1500), ("Q5_1", 130), ("F16", 64)])
def test_cross_cache8_logits(qtype, T):
    """Teacher-forced logits with the 8-bit cross cache, several layers and
    utterances, the frames ending inside a page or at its end."""
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, qtype, seed=31)
    dec = wgdec.WhisperDecoder(m)
    encs = [m.encoder_output(u, T) for u in (0, 1)]
    forced = np.random.default_rng(3).integers(0, 50257, size=(2, 3))
    got = dec.teacher_forced_logits(encs, PROMPT, forced, cross_cache8=True)
    for u in range(2):
        for s in (0, 2):
            want = forward(m, encs[u], PROMPT + [int(t) for t in forced[u, :s]])
            err = np.abs(got[s, u] - want).max()
            assert err <= ATOL and err <= RTOL * np.abs(want).max(), (u, s, err)
    dec.close()
    m.close()


@pytest.mark.parametrize("beam", [1, 5])
def test_cross_cache8_decodes(beam):
    """Whole decodes through the job and its graph: repeatable, several
    utterances at once as each alone, and beside a job with the f16 cache."""
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, "Q8_0", seed=33)
    dec = wgdec.WhisperDecoder(m)
    encs = [m.encoder_output(u) for u in range(3)]
    p8 = wgdec.DecoderParams(prompt=PROMPT, beam_size=beam, max_tokens=12, cross_cache8=True, suppress_eot=True)
    p16 = wgdec.DecoderParams(prompt=PROMPT, beam_size=beam, max_tokens=12, suppress_eot=True)
    before = dec.decode_tokens(encs, p16)[0]
    a = dec.decode_tokens(encs, p8)[0]
    b = dec.decode_tokens(encs, p8)[0]
    np.testing.assert_array_equal(a, b)
    np.testing.assert_array_equal(dec.decode_tokens(encs, p16)[0], before)
    assert a.shape == before.shape and (a[:, :4] == PROMPT).all()
    dec.close()
    m.close()


def coarse_encoders(m, n, T):
    """Encoder outputs with a frame eight times as large in every page of 64: the
    page's steps are coarse, so logits with the 8-bit cache lie an order of
    magnitude further from those without it than the gates are wide."""
    encs = []
    for u in range(n):
        e = m.encoder_output(u, T).copy()
        e[5::64] *= 8
        encs.append(e)
    return encs


def gate_of(want):
    return min(ATOL, RTOL * float(np.abs(want).max()))


class Quantised:
    """The numpy decoder's penalised logits by token prefix, and how far a device logit may be off."""

    def __init__(self, m, dec, encs):
        self.m, self.dec, self.encs, self.seen = m, dec, encs, {}

    def __call__(self, u, tokens):
        key = (u, tuple(int(t) for t in tokens))
        if key not in self.seen:
            raw = forward(self.m, self.encs[u], list(key[1]))
            x = oracle.apply_penalty(raw.astype(np.float32), np.asarray(key[1], np.int32)).astype(np.float64)
            x[self.dec.eot] = -np.inf
            self.seen[key] = x, gate_of(raw)
        return self.seen[key]


def test_cross_cache8_logits_are_not_the_f16_cache_s(monkeypatch):
    """Where the two caches' logits differ by many gates, the device's with the option are the quantised ones."""
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, "Q8_0", seed=33)
    dec = wgdec.WhisperDecoder(m)
    encs = coarse_encoders(m, 2, 130)
    forced = np.random.default_rng(4).integers(0, 50257, size=(2, 2))
    got8 = dec.teacher_forced_logits(encs, PROMPT, forced, cross_cache8=True)
    got16 = dec.teacher_forced_logits(encs, PROMPT, forced)
    for u in range(2):
        tokens = PROMPT + [int(forced[u, 0])]
        want8 = forward(m, encs[u], tokens)
        with monkeypatch.context() as mp:
            mp.setitem(globals(), "quantised", lambda x: x)
            want16 = forward(m, encs[u], tokens)
        g = gate_of(want8)
        assert np.abs(want8 - want16).max() > 8 * g
        assert np.abs(got8[1, u] - want8).max() <= g and np.abs(got16[1, u] - want16).max() <= g
    dec.close()
    m.close()


def test_cross_cache8_greedy_tokens():
    """Each token of three utterances decoded at once is the numpy decoder's
    maximum (to twice the logits' gate), and each utterance alone gives the
    same tokens up to such a tie."""
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, "Q8_0", seed=33)
    dec = wgdec.WhisperDecoder(m)
    encs = coarse_encoders(m, 3, 130)
    logits = Quantised(m, dec, encs)
    p8 = wgdec.DecoderParams(prompt=PROMPT, max_tokens=6, cross_cache8=True, suppress_eot=True, no_fallback=True)
    toks, lens, _ = dec.decode_tokens(encs, p8)
    assert (lens == 10).all() and len({tuple(t) for t in toks.tolist()}) == 3
    for u in range(3):
        for s in range(4, 10):
            x, g = logits(u, toks[u, :s])
            assert x[toks[u, s]] >= x.max() - 2 * g, (u, s)
        alone = dec.decode_tokens([encs[u]], p8)[0][0]
        off = np.flatnonzero(alone[:10] != toks[u, :10])
        if off.size:
            x, g = logits(u, toks[u, :off[0]])
            assert abs(x[alone[off[0]]] - x[toks[u, off[0]]]) <= 4 * g, u
    dec.close()
    m.close()


def test_cross_cache8_beams():
    """Five beams of three utterances, step by step: every hypothesis' score is
    the sum of its tokens' log-probs in the numpy decoder (each off by at most
    twice the logits' gate), the first token of all of them its maximum (the five
    equal prompts of the start each offer it, and it ranks first), and each
    utterance alone finds hypotheses of the same scores."""
    B, M, U = 5, 3, 3
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, "Q8_0", seed=33)
    dec = wgdec.WhisperDecoder(m)
    encs = coarse_encoders(m, U, 130)
    logits = Quantised(m, dec, encs)
    params = wgdec.DecoderParams(prompt=PROMPT, beam_size=B, max_tokens=M, cross_cache8=True, suppress_eot=True)

    def steps_of(which):
        job, out = wgdec.Job(dec, len(which), 130, params), []
        job.upload([encs[u] for u in which])
        job.start()
        for _ in range(M):
            job.step(1)
            out.append([a.copy() for a in job.beams()])
        job.close()
        return out

    together, alone = steps_of(range(U)), [steps_of([u]) for u in range(U)]
    for st in range(M):
        toks, lens, scores = together[st]
        for u in range(U):
            for b in range(B):
                assert lens[u, b] == len(PROMPT) + st + 1
                seq, want, slack = toks[u, b, :lens[u, b]], 0.0, 0.0
                for s in range(len(PROMPT), len(seq)):
                    x, g = logits(u, seq[:s])
                    want += x[seq[s]] - x.max() - np.log(np.exp(x - x.max()).sum())
                    slack += 2 * g
                assert abs(scores[u, b] - want) <= slack + 1e-5 * abs(want), (st, u, b)
            x, g = logits(u, PROMPT)
            assert x[toks[u, :, 4]].min() >= x.max() - 2 * g
            # sorted by score and length alike, near-ties may swap tokens but not move a rank's score
            assert np.abs(alone[u][st][2][0] - scores[u]).max() <= 2 * slack
    dec.close()
    m.close()


@pytest.mark.parametrize("settings", [dict(top_k=5), dict(top_p=0.8, temperature=0.7), dict(min_p=0.1),
                                      dict(top_k=40, top_p=0.95, min_p=0.01, temperature=1.5), dict(cross_cache8=True)],
                         ids=str)
def test_drawn_tokens(settings):
    """Every drawn token is the one its random number falls on in the
    definition's distribution of the oracle's penalised logits. The device's
    logits are within ATOL of the oracle's, so a weight is off by at most
    exp(2 ATOL / T) - 1 and the running mass before a token, relative to the
    kept mass, by twice that; a token whose interval, so widened, misses the
    number is wrong. With the 8-bit cache only the draw's repeatability and
    validity are asked."""
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, "Q8_0", seed=35)
    dec = wgdec.WhisperDecoder(m)
    encs = [m.encoder_output(u) for u in range(3)]
    params = wgdec.DecoderParams(prompt=PROMPT, max_tokens=10, sample=True, seed=77, suppress_eot=True, **settings)
    toks, lens, _ = dec.decode_tokens(encs, params)
    again, _, _ = dec.decode_tokens(encs, params)
    np.testing.assert_array_equal(toks, again)
    assert (lens == len(PROMPT) + 10).all() and (toks >= 0).all() and (toks < m.n_vocab).all()
    if not params.cross_cache8:
        T = params.temperature or 1.0
        for u in range(3):
            lg = oracle.teacher_forced(m, encs[u], PROMPT, toks[u, 4:], wgdec.MODE_CORRECT, m.n_vocab)
            for s in range(10):
                x = oracle.apply_penalty(lg[s], toks[u, :4 + s]).astype(np.float64)
                x[dec.eot] = -np.inf
                t, un = int(toks[u, 4 + s]), oracle.uniform(77, u, s)
                slack = 2 * np.expm1(2 * ATOL / T)
                order = np.argsort(-x, kind="stable")
                w = np.exp((x[order] - x[order[0]]) / T)
                n = params.top_k if params.top_k > 0 else x.size
                before = np.concatenate([[0], np.cumsum(w[:n])[:-1]])
                if params.top_p < 1:
                    n = max(1, int((before < params.top_p * w[:n].sum()).sum()))
                n = max(1, min(n, int((w >= params.min_p).sum())))
                near = int((x >= x[order[n - 1]] - 2 * ATOL).sum())  # what a logit error may add to the kept ones
                assert t in set(order[:near].tolist()), (u, s)
                kept = np.sort(order[:n])
                cum = np.cumsum(np.exp((x[kept] - x[order[0]]) / T))
                i = int(np.searchsorted(kept, t))
                lo, hi = (cum[i - 1] if i else 0.0) / cum[-1], cum[min(i, n - 1)] / cum[-1]
                edge = slack + (near - n) * float(np.exp((x[order[n - 1]] - x[order[0]]) / T)) / cum[-1]
                assert lo - edge <= un <= hi + edge, (u, s, lo, un, hi)
    other = dec.decode_tokens(encs, wgdec.DecoderParams(prompt=PROMPT, max_tokens=10, sample=True, seed=78,
                                                        suppress_eot=True, **settings))[0]
    assert (other != toks).any()
    dec.close()
    m.close()


def test_top_1_draws_are_the_greedy_tokens():
    """top_k = 1 keeps the first maximum: the decode is the greedy one, token for token."""
    m = wgdec.SyntheticModel(51864, 384, 6, 2, 448, "Q8_0", seed=37)
    dec = wgdec.WhisperDecoder(m)
    encs = [m.encoder_output(u) for u in range(2)]
    g = dec.decode_tokens(encs, wgdec.DecoderParams(prompt=PROMPT, max_tokens=20, no_fallback=True))
    d = dec.decode_tokens(encs, wgdec.DecoderParams(prompt=PROMPT, max_tokens=20, sample=True, top_k=1))
    np.testing.assert_array_equal(g[0], d[0])
    np.testing.assert_array_equal(g[1], d[1])
    dec.close()
    m.close()


def test_refused_options():
    m = wgdec.SyntheticModel(1000, 64, 2, 1, 64, "Q8_0", seed=39)  # 32-wide heads
    dec = wgdec.WhisperDecoder(m)
    enc = m.encoder_output(0, 20)
    P = [1, 2]
    for kw, status in ((dict(cross_cache8=True), 4), (dict(sample=True, beam_size=2), 4),
                       (dict(sample=True, suppress_nst=True), 4), (dict(sample=True, top_p=float("nan")), 1),
                       (dict(sample=True, min_p=float("nan")), 1)):
        with pytest.raises(wgdec.DecodeError) as ei:
            dec.decode_tokens([enc], wgdec.DecoderParams(prompt=P, max_tokens=2, **kw))
        assert ei.value.status == status, kw
    b = wgdec.Batcher(dec)
    with pytest.raises(wgdec.DecodeError):
        b.decode_tokens(enc, wgdec.DecoderParams(prompt=P, max_tokens=2, sample=True))
    b.close()
    dec.close()
    m.close()
