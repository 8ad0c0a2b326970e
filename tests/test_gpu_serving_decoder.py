"""A serving decoder (caches in f16 or 8 bits, a shared prefix, sampled tokens) against the plain decoder and, with a
prefix, against the model in 64 bits over the stored K and V.

Bars: the plain decoder's own against its reference, 5e-3 of the largest logit (f16 operands in every projection), for
the model in 64 bits.  Between the two decoders: with f16 caches both hold the same halves and differ in the rounding of
attention alone (the plain one rounds q and the probabilities to f16), 2e-3; 8-bit caches add the rounding of K and V, at
most 1/254 of a row's largest (i8) or 1/16 of a value (e4m3) in each of two layers, 5e-2 and 0.3.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_decoder import B, D, E, EPS, H, HD, HKV, I, LOGIT_TOL, NL, S0, STEPS, THETA, TOPK, V, _weights  # noqa: E402
from test_gpu_serving import code, encode, values  # noqa: E402


def _decoder(um, backend, W, max_seq, **kw):
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    blocks, keep = [], []
    for b in W["blocks"]:
        d = {k: dev(v) for k, v in b.items()}
        keep.append(d)
        moe = um.make_layer(D, E, I, TOPK, 1, d["router"], d["gate"], um.Q4_K, d["up"], um.Q4_K, d["down"], um.Q6_K)
        blocks.append({"attn_norm": d["attn_norm"], "ffn_norm": d["ffn_norm"], "wq": d["wq"], "wq_fmt": um.Q8_0,
                       "wk": d["wk"], "wk_fmt": um.Q8_0, "wv": d["wv"], "wv_fmt": um.Q8_0, "wo": d["wo"],
                       "wo_fmt": um.Q8_0, "moe": moe})
    dec = um.Decoder(backend, NL, D, H, HKV, V, B, max_seq, blocks, dev(W["out_norm"]), dev(W["emb"]), um.Q8_0,
                     rope_theta=THETA, rms_eps=EPS, **kw)
    dec._keep.append(keep)
    return dec


def _logits(dec, tokens):
    out = np.empty((B, V), np.float32)
    dec.step(tokens, out, None)
    return out.astype(np.float64)


def _tokens(seed):
    return np.random.default_rng(seed).integers(0, V, size=(STEPS, B)).astype(np.int32)


@pytest.mark.parametrize("fmt,bar", [("f16", 2e-3), ("i8", 5e-2), ("e4m3", 0.3)])
def test_matches_the_plain_decoder(um, backend, fmt, bar):
    W, kv = _weights(um)
    plain, serving = _decoder(um, backend, W, S0 + STEPS), _decoder(um, backend, W, S0 + STEPS, kv_fmt=code(um, fmt))
    try:
        for dec in (plain, serving):
            for l, (k, v) in enumerate(kv):
                dec.set_kv(l, k, v, S0)
        for s, tok in enumerate(_tokens(3)):
            a, b = _logits(plain, tok), _logits(serving, tok)
            assert np.abs(a - b).max() <= bar * np.abs(a).max(), s
            assert serving.position == S0 + s + 1
    finally:
        plain.close()
        serving.close()


def _stored(rows, fmt):
    """What a cache returns for K or V rows, in 64 bits."""
    return rows.astype(np.float16).astype(np.float64) if fmt == "f16" else values(*encode(rows, fmt), fmt)


def _rotated(x, pos):
    c = np.exp(-np.log(THETA) * np.arange(0, HD, 2) / HD) * pos
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * np.cos(c) - x[..., 1::2] * np.sin(c)
    out[..., 1::2] = x[..., 0::2] * np.sin(c) + x[..., 1::2] * np.cos(c)
    return out


def _plain_step(um, oracle, W, tokens, pos, past, fmt):
    """One step in 64 bits; past[l] = (K, V) [B, HKV, positions, HD] as stored, extended in place."""
    full = lambda q, n, k: oracle.dequant(um.Q8_0, q, n, k).astype(np.float64)  # noqa: E731
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w  # noqa: E731
    x = full(W["emb"], V, D)[tokens]
    for l, b in enumerate(W["blocks"]):
        n = norm(x, b["attn_norm"])
        q = _rotated((n @ full(b["wq"], H * HD, D).T).reshape(B, H, HD), pos)
        k = _rotated((n @ full(b["wk"], HKV * HD, D).T).reshape(B, HKV, 1, HD), pos)
        v = (n @ full(b["wv"], HKV * HD, D).T).reshape(B, HKV, 1, HD)
        past[l] = K, U = tuple(np.concatenate([p, _stored(r, fmt)], 2) for p, r in zip(past[l], (k, v)))
        s = np.einsum("bghd,bgnd->bghn", q.reshape(B, HKV, H // HKV, HD), K) / np.sqrt(HD)
        e = np.exp(s - s.max(-1, keepdims=True))
        a = np.einsum("bghn,bgnd->bghd", e / e.sum(-1, keepdims=True), U).reshape(B, H * HD)
        x = x + a @ full(b["wo"], D, H * HD).T
        n2 = norm(x, b["ffn_norm"]).astype(np.float32)
        _, probs, _ = oracle.router(n2, b["router"])
        x = x + oracle.experts_packed(n2, b["gate"], um.Q4_K, b["up"], um.Q4_K, b["down"], um.Q6_K, probs, E, I, TOPK,
                                      1)[0]
    return norm(x, W["out_norm"]) @ full(W["emb"], V, D).T


@pytest.mark.parametrize("fmt", ["f16", "i8", "e4m3"])
def test_a_shared_prefix_matches_the_plain_model(um, backend, oracle, fmt):
    W, _ = _weights(um)
    P = 70
    f = lambda s: um.fill_normal((HKV, P, HD), 9, s)  # noqa: E731
    kv = [(f(2 * l), f(2 * l + 1)) for l in range(NL)]
    past = [tuple(np.broadcast_to(_stored(a, fmt), (B, HKV, P, HD)) for a in pair) for pair in kv]
    dec = _decoder(um, backend, W, STEPS, kv_fmt=code(um, fmt), prefix_max=P + 3)
    try:
        for l, (k, v) in enumerate(kv):
            dec.set_prefix(l, k, v, P)
        for s, tok in enumerate(_tokens(6)):  # no token near a tie of experts
            want, got = _plain_step(um, oracle, W, tok, P + s, past, fmt), _logits(dec, tok)
            assert np.abs(got - want).max() <= LOGIT_TOL * np.abs(want).max(), s
    finally:
        dec.close()


def test_sampled_steps(um, backend):
    """Greedy settings give the arg-max; a sampled token is the operator's on the step's logits."""
    W, kv = _weights(um)
    dec = _decoder(um, backend, W, S0 + STEPS, kv_fmt=um.KV_I8)
    f = lambda *v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    try:
        for l, (k, v) in enumerate(kv):
            dec.set_kv(l, k, v, S0)
        heat, k, p, least, u = f(0.0, 0.9, 1.2), i(0, 20, 0), f(1.0, 0.9, 0.8), f(0.0, 0.0, 0.05), f(0.4, 0.7, 0.2)
        nxt, probs, logits = i(0, 0, 0), f(0, 0, 0), torch.empty((B, V), device="cuda")
        tok = torch.from_numpy(_tokens(5)[0]).cuda()
        for s in range(STEPS):
            dec.step_sampled(tok, heat, k, p, least, u, nxt, probs, logits)
            again, prob2 = i(-9, -9, -9), f(0, 0, 0)
            backend.sample(logits, heat, k, p, least, u, again, prob2)
            backend.synchronize()
            assert torch.equal(nxt, again) and torch.equal(probs, prob2)
            assert int(nxt[0]) == int(logits[0].argmax()) and float(probs[0]) == 1.0
            tok = nxt.clone()
        with pytest.raises(um.UaiiMoeError) as e:
            dec.step_sampled(tok, heat, k, p, least, u, nxt)
        assert "full" in e.value.message
    finally:
        dec.close()


def test_serving_refusals(um, backend):
    W, _ = _weights(um)
    with pytest.raises(um.UaiiMoeError) as e:
        _decoder(um, backend, W, 8, kv_fmt=um.Q8_0)
    assert e.value.status == um.NOT_IMPLEMENTED
    with pytest.raises(ValueError):
        _decoder(um, backend, W, 8, prefix_max=4)
    dec = _decoder(um, backend, W, 8, kv_fmt=um.KV_I8, prefix_max=4)
    try:
        k = np.zeros((HKV, 5, HD), np.float32)
        for call in (lambda: dec.set_prefix(0, k, k, 5), lambda: dec.set_prefix(NL, k, k, 4), lambda: dec.fill_kv(2)):
            with pytest.raises(um.UaiiMoeError):
                call()
    finally:
        dec.close()


def test_rope_pairs_of_halves(um, backend):
    """rope_mode 2 (halves of a head are the pairs) turns q and k as the plain decoder does."""
    W, kv = _weights(um)
    plain = _decoder(um, backend, W, S0 + STEPS, rope_mode=2)
    serving = _decoder(um, backend, W, S0 + STEPS, rope_mode=2, kv_fmt=um.F16)
    try:
        for dec in (plain, serving):
            for l, (k, v) in enumerate(kv):
                dec.set_kv(l, k, v, S0)
        for s, tok in enumerate(_tokens(3)):
            a, b = _logits(plain, tok), _logits(serving, tok)
            assert np.abs(a - b).max() <= 2e-3 * np.abs(a).max(), s
    finally:
        plain.close()
        serving.close()


def test_generate_equals_stepping(um, backend):
    W, kv = _weights(um)
    tok = _tokens(7)[0]
    a, b = (_decoder(um, backend, W, S0 + STEPS, kv_fmt=um.KV_E4M3) for _ in range(2))
    try:
        for dec in (a, b):
            for l, (k, v) in enumerate(kv):
                dec.set_kv(l, k, v, S0)
        out = np.empty((STEPS, B), np.int32)
        a.generate(tok, STEPS, out)
        for s in range(STEPS):
            nxt = np.empty(B, np.int32)
            b.step(tok, None, nxt)
            assert np.array_equal(nxt, out[s]), s
            tok = nxt
    finally:
        a.close()
        b.close()


def test_refused_settings_leave_the_position(um, backend):
    W, _ = _weights(um)
    dec = _decoder(um, backend, W, 4, kv_fmt=um.F16)
    f, i = torch.zeros(B, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    try:
        with pytest.raises(um.UaiiMoeError) as e:
            dec.step_sampled(i, f.cpu(), i, f, f, f, i)
        assert e.value.status == um.INVALID_ARGUMENT and dec.position == 0
    finally:
        dec.close()
