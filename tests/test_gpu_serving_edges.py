"""More of the serving operators' edges: batches of many hundred sequences, items of many rows (sharp scores, faults,
hidden keys), logits that lie together or at the ends of their type, and the sizes at which a row changes its split.

Tolerances are those of the first file (see its head).  An item of many rows keeps probabilities in f16 with 2^8 in front
of the largest: each loses at most 2^-33 of it beneath f16's last place, n 2^-32 max|v| over a row's n positions with
both parts of a split.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_serving import FMTS, Cache, attention64, check_attention, dev, interval, sample  # noqa: E402


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("b,g,t,p_len", [(513, 2, 1, 0), (1100, 1, 1, 40), (520, 9, 2, 0), (600, 1, 20, 70)])
def test_attention_hundreds_of_sequences(um, backend, fmt, b, g, t, p_len):
    lens = [(i * 29) % 71 if i % 5 else 0 for i in range(b)]
    check_attention(um, backend, fmt, fmt != "i8", 64, 1, g, t, lens, p_len)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("g,t,p_len", [(17, 1, 0), (4, 5, 129), (8, 40, 63), (3, 100, 0)])
def test_attention_many_rows(um, backend, fmt, half, hd, g, t, p_len):
    check_attention(um, backend, fmt, half, hd, 2, g, t, [0, 1, t, 64, 65, 200], p_len)


@pytest.mark.parametrize("fmt", ["f16", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("gain", [8.0, 40.0])
def test_attention_many_rows_sharp(um, backend, fmt, half, rising, gain):
    """Scores that spread over hundreds; rising: the running maximum grows with nearly every key."""
    rng = np.random.default_rng(3)
    b, h, g, t, hd, p_len, lens = 2, 1, 6, 9, 128, 150, [211, 9]
    own, prefix = Cache(um, fmt, b, h, 220, hd, rng, lens=lens), Cache(um, fmt, 1, h, 160, hd, rng, lens=[p_len])
    q = gain * rng.standard_normal((b, t, h * g, hd))
    if rising:  # along the keys' own trend: one dimension grows with the position
        for c, n in ((own, 220), (prefix, 160)):
            c.enc["k"][0][..., 0] = np.linspace(0, 3, n) if fmt == "f16" else 1 + np.arange(n) // 3
            c.t["k"][0].copy_(dev(c.enc["k"][0]))
        q[..., 0] = np.abs(q[..., 0])
    q = q.astype(np.float16 if half else np.float32)
    out = torch.empty(q.shape, dtype=torch.float16 if half else torch.float32, device="cuda")
    backend.prefix_attention(dev(q), own.view, dev(np.array(lens, np.int32)), out, prefix=prefix.view, prefix_len=p_len)
    backend.synchronize()
    want, tol, mag = attention64(q.astype(np.float64), own, lens, prefix, p_len, 1 / np.sqrt(hd))
    top = max(np.nanmax(np.abs(c.values("v"))[:, :, :n]) for c, n in ((own, 9), (own, 211), (prefix, p_len)))
    tol = tol + (p_len + 211) * 2.0 ** -32 * top
    if half:
        tol = tol + 2.0 ** -11 * mag + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    bad = np.abs(out.cpu().numpy().astype(np.float64) - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(out.cpu().numpy() - want).max())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
def test_attention_many_rows_keep_a_fault_to_its_sequence(um, backend, fmt, half):
    own = Cache(um, fmt, 3, 2, 100, 128, np.random.default_rng(5))
    if fmt == "f16":
        own.t["v"][0][1, 0, 17, 3] = float("nan")
    else:
        own.t["v"][1][1, 0, 17] = float("nan")
    q = torch.randn((3, 6, 8, 128), device="cuda").to(torch.float16 if half else torch.float32)
    out = torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(np.array([60, 60, 10], np.int32)), out)
    backend.synchronize()
    nan = out.isnan()
    assert nan[1, :, :4].any(-1).all()
    nan[1, :, :4] = False
    assert not nan.any()


@pytest.mark.parametrize("half", [False, True])
def test_attention_many_rows_with_hidden_keys(um, backend, half):
    """Keys whose scores are -inf carry no weight; a row that sees nothing else is zero."""
    t = 20
    own = Cache(um, "f16", 1, 1, 80, 64, np.random.default_rng(1))
    k = own.t["k"][0]
    k[..., 0] = float("-inf")
    k[0, 0, 66, 0] = 0.5
    q = torch.zeros((1, t, 1, 64), dtype=torch.float16 if half else torch.float32, device="cuda")
    q[..., 0] = 1.0
    out = torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(np.array([76], np.int32)), out)
    backend.synchronize()
    first = t - (76 - 66)  # token j sees positions up to 76 - t + j
    assert (out[0, :first] == 0).all()
    assert torch.allclose(out[0, first:, 0].float(), own.t["v"][0][0, 0, 66].float().expand(t - first, 64), rtol=1e-3)


@pytest.mark.parametrize("fmt,bad", [("f16", "nan"), ("f16", "inf"), ("f16", "-inf"), ("e4m3", "byte"), ("e4m3", "scale"),
                                     ("i8", "scale")])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,g,t,last", [(128, 2, 4, 40), (64, 2, 8, 33), (128, 6, 9, 66), (64, 4, 90, 130), (128, 1, 7, 5)])
def test_attention_faults_that_some_tokens_do_not_see(um, backend, fmt, bad, half, hd, g, t, last):
    """An infinity or a NaN at a position that only the later tokens see: the earlier ones' results are as without it,
    bit for bit, and so are the later ones' in the other dimensions."""
    own = Cache(um, fmt, 2, 2, last + 6, hd, np.random.default_rng(t))
    q = torch.randn((2, t, 2 * g, hd), device="cuda").to(torch.float16 if half else torch.float32)
    lens, clean, out = dev(np.array([last, last], np.int32)), torch.empty_like(q), torch.empty_like(q)
    at = max(0, last - t // 2 - 1)  # sequence 1, kv head 0
    backend.prefix_attention(q, own.view, lens, clean)
    data, scale = own.t["v"]
    if fmt == "f16":
        data[1, 0, at, 3] = float(bad)
    elif bad == "byte":
        data[1, 0, at, 3] = 0xff
    else:
        scale[1, 0, at] = float("nan")
    backend.prefix_attention(q, own.view, lens, out)
    backend.synchronize()
    first = max(0, t - (last - at))  # token j sees positions below last - t + 1 + j
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[1, first:, :g, slice(None) if bad == "scale" else slice(3, 4)] = True
    assert torch.equal(out[~hit], clean[~hit])
    if bad in ("inf", "-inf") and half:
        assert (out[hit] == float(bad)).all()
    else:
        assert not out[hit].isfinite().any()


# ---------------------------------------------------------------- sampling


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("v", [4095, 4096, 4097, 8193, 16384, 16385, 32769, 400000])
def test_sample_where_the_split_changes(um, backend, half, v):
    rng = np.random.default_rng(v)
    b = 6
    x = (3 * rng.standard_normal((b, v))).astype(np.float16 if half else np.float32)
    heat = np.array([0.5, 1, 1, 2, 1, 0.9], np.float32)
    k = np.array([0, 50, 0, 700, v - 1, v], np.int32)
    p = np.array([0.9, 1, 0.99, 0.5, 1, 0.3], np.float32)
    least = np.array([0, 0, 0.05, 0, 0, 1e-6], np.float32)
    u = rng.random(b).astype(np.float32)
    tok, prob, kept = sample(um, backend, x, heat, k, p, least, u)
    for i in range(b):
        lo, hi, n, want = interval(x[i], float(heat[i]), int(k[i]), float(p[i]), float(least[i]), tok[i])
        assert lo - 2e-6 <= u[i] <= hi + 2e-6, (i, lo, hi, u[i])
        assert abs(int(kept[i]) - n) <= (0 if p[i] >= 1 and least[i] == 0 else 1), (i, kept[i], n)
        assert abs(prob[i] - want) <= 1e-5 * want + (1e-6 if p[i] < 1 else 0)


@pytest.mark.parametrize("v", [900, 5000, 60000])
def test_sample_equal_weights_of_unequal_logits(um, backend, v):
    """At a huge temperature every weight rounds to the same whole number: the ranking is still the logits'."""
    rng = np.random.default_rng(v)
    x = rng.permutation(np.linspace(-4, 4, v)).astype(np.float32)
    order = np.argsort(-x.astype(np.float64), kind="stable")
    u = np.linspace(0, 0.999, 8).astype(np.float32)
    for k in (1, 2, v // 3, v - 1):
        tok, prob, kept = sample(um, backend, np.broadcast_to(x, (8, v)), 1e30, top_k=k, u=u)
        idx = np.sort(order[:k])
        assert (kept == k).all() and np.allclose(prob, 1 / k, rtol=1e-6)
        assert tok.tolist() == [int(idx[int(np.float64(z) * k)]) for z in u]


@pytest.mark.parametrize("v", [300, 40000])
def test_sample_the_types_lowest_values(um, backend, v):
    """Logits masked with the type's lowest value weigh nothing beside others, and are equal among themselves."""
    for t in (np.float16, np.float32):
        low = np.finfo(t).min
        x = np.full((4, v), low, t)
        x[0, [7, 9, v - 1]] = [1.0, 0.0, 1.0]
        x[1, [0, v // 2]] = np.finfo(t).max
        x[3, 5] = -np.inf
        tok, prob, kept = sample(um, backend, x, [1.0, 1e-3, 0.7, 2.0], top_k=[3, 0, 0, 0],
                                 top_p=[1.0, 0.9, 1.0, 1.0], u=[0.999, 0.999, 0.5, 0.0])
        assert tok.tolist() == [v - 1, v // 2, v // 2, 0]
        e = np.exp(-1.0)
        assert np.allclose(prob, [1 / (2 + e), 0.5, 1 / v, 1 / (v - 1)], rtol=1e-5)
        assert kept.tolist()[:3] == [3, 2, v]


def test_sizes_that_are_refused(um, backend):
    def refused(status, part, call, *args):
        with pytest.raises(um.UaiiMoeError) as e:
            call(*args)
        assert e.value.status == status and part in e.value.message, e.value.message

    f, i = torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    refused(um.NOT_IMPLEMENTED, "vocab", backend.sample, torch.zeros((1, 400001), device="cuda"), f, i, f, f, f, i)
    own = Cache(um, "i8", 1, 2, 4, 64, np.random.default_rng(0))
    many = um.KVCache.from_buffer_copy(own.view)
    many.batch, many._keep = 32768, own.t
    pos = torch.zeros(32768, dtype=torch.int32, device="cuda")
    x = torch.zeros((32768, 1, 2, 64), device="cuda")
    refused(um.INVALID_ARGUMENT, "cache sizes", backend.kv_append, many, x, x, pos)
    refused(um.INVALID_ARGUMENT, "cache sizes", backend.prefix_attention, x, many, pos, x)
    backend.synchronize()


@pytest.mark.parametrize("fmt,hd", [("e4m3", 128), ("f16", 64)])
def test_attention_long_f32_sums_do_not_shrink(um, backend, fmt, hd):
    """Many rows over thousands of keys: an accumulator that is cut off at each addition loses 2^-24 of itself on average,
    so 40 additions to a sum that grows from nothing lose 40 / 2 * 2^-24 of it, 1.2e-6; scores (8 additions, up to 4
    in magnitude) and the roundings of the reference's rows add as much again.  Bar on the whole result: 2.5e-6."""
    rng = np.random.default_rng(9)
    b, h, g, t, p_len, own_len = 64, 8, 7, 4, 7741, 70
    prefix = Cache(um, fmt, 1, h, p_len, hd, rng)
    own = Cache(um, fmt, b, h, own_len, hd, rng)
    q = torch.randn((b, t, h * g, hd), device="cuda")
    out = torch.empty_like(q)
    lens = dev(np.full(b, own_len, np.int32))
    backend.prefix_attention(q, own.view, lens, out, prefix=prefix.view, prefix_len=p_len)
    backend.synchronize()
    sees = torch.arange(own_len, device="cuda")[None, :] <= own_len - t + torch.arange(t, device="cuda")[:, None]
    off = whole = 0.0
    (pk, ok), (pv, ov) = ((dev(prefix.values(n)), dev(own.values(n))) for n in "kv")
    for kh in range(h):
        for i in range(b):
            k, v = torch.cat([pk[0, kh], ok[i, kh]]), torch.cat([pv[0, kh], ov[i, kh]])
            x = q[i, :, kh * g:(kh + 1) * g].double()
            s = torch.einsum("tgd,nd->tgn", x, k) / hd ** 0.5
            s[:, :, p_len:].masked_fill_(~sees[:, None, :], float("-inf"))
            want = torch.softmax(s, -1) @ v
            off += float((out[i, :, kh * g:(kh + 1) * g].double() - want).square().sum())
            whole += float(want.square().sum())
    assert (off / whole) ** 0.5 <= 2.5e-6
