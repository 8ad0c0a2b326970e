"""The serving operators (KV cache in f16 / 8 bits, attention over a shared prefix, sampling) against their
definitions in 64 bits (numpy), at the sizes, strides and masks where such kernels go wrong.

Tolerances, fixed before the first run:
  cache      bytes and scales equal the f32 formula exactly (one IEEE operation per step); values within half a
             step of the source (i8: scale / 2 and the roundings of x * (127 / a) and of the scale; e4m3: 2^-4 of the value, or 2^-10 of the scale below the normals).
  attention  a score's error is at most d = 2^-18 * scale * |q|.|k| (f32 sums of 16-element products: at most 16
             roundings of 2^-23 of the summed magnitudes, and a split of q to 2^-22), a probability's 2 d relative,
             the sum over n positions at most (n / 16 + 64) * 2^-23 of sum p |v|, exponentials and row scales
             2^-20.  f16 results add one rounding of p and one of the result, 2^-11 each.
  sampling   with integer-exact weights the result is exact; elsewhere the chosen token's interval of the running
             mass must hold u to 2e-6 of the whole (an exponential is good to 2 ulp; sums are exact).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FMTS = ("f16", "i8", "e4m3")
I8_STEP = 0.5 + 127 * 3 * 2.0 ** -24  # of the scale: rint's half, and three f32 roundings of a number up to 127


def code(um, fmt):
    return {"f16": um.F16, "i8": um.KV_I8, "e4m3": um.KV_E4M3}[fmt]


def e4m3_values():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


E4M3 = e4m3_values()


def encode(x, fmt):
    """The f32 formula: rows of x -> (bytes, scale)."""
    x = x.astype(np.float32)
    a = np.abs(x).max(-1, keepdims=True)
    top = np.float32(127 if fmt == "i8" else 448)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        ok = a >= np.float32(2.0 ** -100)
        scale = np.where(ok, a / top, np.float32(0)).astype(np.float32)
        y = np.where(ok, x * (top / a).astype(np.float32), np.float32(0)).astype(np.float32)
    if fmt == "i8":
        return (np.rint(y) + 128).astype(np.uint8), scale[..., 0]
    return torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), scale[..., 0]


def values(c, s, fmt):
    """64-bit values of stored rows."""
    if fmt == "f16":
        return c.astype(np.float64)
    q = c.astype(np.float64) - 128 if fmt == "i8" else E4M3[c]
    return q * s.astype(np.float64)[..., None]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Cache:
    """A cache of random rows; rows at and beyond lens[b] hold NaNs (f16, e4m3) or stray bytes and NaN scales."""

    def __init__(self, um, fmt, b, h, s, d, rng, lens=None, gain=1.0):
        self.fmt = fmt
        self.k, self.v = (gain * rng.standard_normal((b, h, s, d)).astype(np.float32) for _ in range(2))
        self.enc = {}
        for n, x in (("k", self.k), ("v", self.v)):
            c, sc = (x.astype(np.float16), None) if fmt == "f16" else encode(x, fmt)
            if lens is not None:
                past = np.arange(s)[None, :] >= np.asarray(lens)[:, None]
                c = np.where(past[:, None, :, None], np.float16(np.nan) if fmt == "f16" else np.uint8(255), c)
                if sc is not None:
                    sc = np.where(past[:, None, :], np.float32(np.nan), sc)
            self.enc[n] = (c, sc)
        self.t = {n: (dev(c), None if sc is None else dev(sc)) for n, (c, sc) in self.enc.items()}
        self.view = um.kv_cache(code(um, fmt), self.t["k"][0], self.t["v"][0], self.t["k"][1], self.t["v"][1])

    def values(self, n):
        return values(*self.enc[n], self.fmt)


# ---------------------------------------------------------------- the cache


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("b,t,h,shift,wide", [(1, 1, 1, 0, 0), (3, 1, 8, 0, 4), (2, 37, 3, 1, 0), (5, 6, 2, 4, 1)])
def test_append_writes_the_formula_and_nothing_else(um, backend, fmt, half, hd, b, t, h, shift, wide):
    rng = np.random.default_rng(hd + t + h)
    s = t + 9
    c = Cache(um, fmt, b, h, s, hd, rng)
    before = {n: (x.cpu().numpy().copy(), None if y is None else y.cpu().numpy().copy()) for n, (x, y) in c.t.items()}
    # K and V as parts of one buffer with `wide` heads before them, starting `shift` elements in
    row = (wide + 2 * h) * hd + shift
    buf = rng.standard_normal(b * t * row + shift).astype(np.float16 if half else np.float32)
    buf[shift + wide * hd:][:hd] = 0                     # a row of zeros
    src = dev(buf)[shift:].unflatten(0, (b, t, row))[..., :(wide + 2 * h) * hd].unflatten(-1, (wide + 2 * h, hd))
    k, v = src[:, :, wide:wide + h], src[:, :, wide + h:]
    pos = np.array([(7 * i) % 10 for i in range(b)], np.int32)
    count = np.array([t if i % 2 == 0 else max(0, t - 1 - i) for i in range(b)], np.int32)
    backend.kv_append(c.view, k, v, dev(pos), dev(count))
    backend.synchronize()
    for n, x in (("k", k), ("v", v)):
        x = x.float().cpu().numpy()
        want, want_s = before[n]
        want = want.copy()
        for i in range(b):
            rows = x[i, :count[i]].transpose(1, 0, 2)
            at = slice(pos[i], pos[i] + count[i])
            if fmt == "f16":
                want[i, :, at] = rows.astype(np.float16)
            else:
                q, sc = encode(rows, fmt)
                want[i, :, at], want_s[i, :, at] = q, sc
                got = values(q, sc, fmt)
                step = sc[..., None] * I8_STEP if fmt == "i8" else np.maximum(np.abs(rows) / 16, sc[..., None] / 1024)
                assert (np.abs(got - rows) <= step * (1 + 2.0 ** -18)).all()
        got_c = c.t[n][0].cpu().numpy()
        assert np.array_equal(got_c.view(np.uint8), want.view(np.uint8)), n
        if fmt != "f16":
            assert np.array_equal(c.t[n][1].cpu().numpy().view(np.uint32), want_s.view(np.uint32)), n


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_extreme_rows(um, backend, fmt):
    hd, rows = 128, 9
    x = np.random.default_rng(3).standard_normal((1, rows, 1, hd)).astype(np.float32)
    x[0, 0] = 0
    x[0, 1] *= np.float32(1e-38)          # under 2^-100: kept as zeros
    x[0, 2] *= np.float32(1e30)
    x[0, 3, 0, 5] = np.inf
    x[0, 4, 0, 127] = np.nan
    x[0, 5] = 0
    x[0, 5, 0, 77] = -3e38
    x[0, 6, 0, :] = np.float32(2.0 ** -100)
    x[0, 7, 0, 0] = -np.inf
    x[0, 8, 0, :] = -0.0
    c = Cache(um, fmt, 1, 1, rows, hd, np.random.default_rng(4))
    xd = dev(x)
    backend.kv_append(c.view, xd, xd, dev(np.zeros(1, np.int32)))
    out = [torch.empty((1, 1, rows, hd), device="cuda") for _ in range(2)]
    backend.kv_read(c.view, 0, rows, *out)
    backend.synchronize()
    assert torch.equal(out[0].isnan(), out[1].isnan())
    got = out[0].cpu().numpy()[0, 0]
    bad = [3, 4, 7]
    assert np.isnan(got[bad]).all() and np.isfinite(np.delete(got, bad, 0)).all()
    assert (got[[0, 1, 8]] == 0).all()
    for r in (2, 5, 6):
        want = x[0, r, 0].astype(np.float64)
        amax = np.abs(want).max()
        assert np.abs(got[r] - want).max() <= amax * (I8_STEP / 127 if fmt == "i8" else 1 / 16) * (1 + 2.0 ** -18)


def test_append_reports_positions_outside_the_cache(um, backend):
    c = Cache(um, "i8", 2, 2, 8, 64, np.random.default_rng(0))
    before = c.t["k"][0].clone()
    x = torch.randn((2, 3, 2, 64), device="cuda")
    backend.kv_append(c.view, x, x, dev(np.array([6, -2], np.int32)))
    with pytest.raises(um.UaiiMoeError) as e:
        backend.synchronize()
    assert e.value.status == um.INVALID_ARGUMENT and "position" in e.value.message
    after = c.t["k"][0]
    assert torch.equal(after[0, :, :6], before[0, :, :6]) and torch.equal(after[1, :, 1:], before[1, :, 1:])
    assert not torch.equal(after[0, :, 6:], before[0, :, 6:]) and not torch.equal(after[1, :, 0], before[1, :, 0])
    backend.synchronize()  # reported once


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,b,h,s,pos0,n", [(128, 1, 1, 1, 0, 1), (64, 3, 2, 70, 5, 61), (128, 2, 3, 300, 299, 1),
                                             (128, 2, 1, 1025, 0, 1025), (64, 1, 1, 10, 10, 0)])
def test_read_gives_the_stored_values(um, backend, fmt, half, hd, b, h, s, pos0, n):
    c = Cache(um, fmt, b, h, s, hd, np.random.default_rng(s))
    out = [torch.full((b, h, n, hd), 7.0, dtype=torch.float16 if half else torch.float32, device="cuda") for _ in range(2)]
    backend.kv_read(c.view, pos0, n, *out)
    backend.synchronize()
    for name, got in zip(("k", "v"), out):
        want = c.values(name)[:, :, pos0:pos0 + n].astype(np.float32)
        if half:
            want = want.astype(np.float16)
        assert np.array_equal(got.cpu().numpy(), want)


def test_a_row_beyond_32_bit_offsets(um, backend):
    """A cache of more than 2^32 bytes: its last rows are written, read and attended to like any other."""
    h, s, d = 8, 4_300_000, 128
    k = torch.zeros((1, h, s, d), dtype=torch.uint8, device="cuda")
    sc = torch.zeros((1, h, s), device="cuda")
    view = um.kv_cache(um.KV_I8, k, k, sc, sc)
    x = torch.randn((1, 2, h, d), device="cuda")
    backend.kv_append(view, x, x, dev(np.array([s - 2], np.int32)))
    out = [torch.empty((1, h, 2, d), device="cuda") for _ in range(2)]
    backend.kv_read(view, s - 2, 2, *out)
    backend.synchronize()
    q, want_s = encode(x.cpu().numpy(), "i8")
    want = values(q, want_s, "i8").astype(np.float32)[0].transpose(1, 0, 2)
    assert np.array_equal(out[0].cpu().numpy()[0], want) and torch.equal(out[0], out[1])
    # attention over a short prefix view of the far end: the last 2 positions of head 7 alone carry weight
    own = Cache(um, "i8", 1, h, 4, d, np.random.default_rng(1), lens=[0])
    res = torch.empty((1, 1, h, d), device="cuda")
    backend.prefix_attention(torch.zeros((1, 1, h, d), device="cuda"), own.view, dev(np.zeros(1, np.int32)), res,
                             prefix=view, prefix_len=s)
    backend.synchronize()
    expect = want.astype(np.float64).sum(1) / s  # equal weights: zeros everywhere but in the last two rows
    assert np.abs(res.cpu().numpy()[0, 0] - expect).max() <= 1e-4 * np.abs(expect).max()


# ---------------------------------------------------------------- attention


def attention64(q, own, lens, prefix, p_len, scale):
    """(out, tolerance for f32, sum p |v|) from the definition: q [B, T, H, d] in 64 bits."""
    b, t, hq, d = q.shape
    h = own.k.shape[1]
    g = hq // h
    ok, ov = own.values("k"), own.values("v")
    out, tol, mag = (np.zeros(q.shape) for _ in range(3))
    for i in range(b):
        for kh in range(h):
            k, v = ok[i, kh, :lens[i]], ov[i, kh, :lens[i]]
            if p_len:
                k = np.concatenate([prefix.values("k")[0, kh, :p_len], k])
                v = np.concatenate([prefix.values("v")[0, kh, :p_len], v])
            for j in range(t):
                n = p_len + max(0, lens[i] - t + j + 1)
                if n == 0:
                    continue
                x = q[i, j, kh * g:(kh + 1) * g]
                s = scale * x @ k[:n].T
                e = np.exp(s - s.max(-1, keepdims=True))
                e /= e.sum(-1, keepdims=True)
                err = (2.0 ** -18 * scale * np.abs(x) @ np.abs(k[:n]).T).max(-1, keepdims=True)
                at = (i, j, slice(kh * g, (kh + 1) * g))
                out[at], mag[at] = e @ v[:n], e @ np.abs(v[:n])
                tol[at] = (2 * err + (n / 16 + 64) * 2.0 ** -23 + 2.0 ** -20) * mag[at]
    return out, tol, mag


def check_attention(um, backend, fmt, half, hd, h, g, t, lens, p_len, gain=1.0, room=3, scale=0.0):
    rng = np.random.default_rng(len(lens) * 1000 + p_len + g + t)
    b = len(lens)
    own = Cache(um, fmt, b, h, max(max(lens), 1) + room, hd, rng, lens=lens)
    prefix = Cache(um, fmt, 1, h, p_len + room, hd, rng, lens=[p_len]) if p_len else None
    np_t = np.float16 if half else np.float32
    wide = (gain * rng.standard_normal((b, t, h * g + 2, hd))).astype(np_t)  # heads of a wider buffer
    q = dev(wide)[:, :, 1:-1]
    out = torch.full((b, t, h * g, hd), 9.0, dtype=q.dtype, device="cuda")
    backend.prefix_attention(q, own.view, dev(np.array(lens, np.int32)), out, prefix=prefix.view if prefix else None,
                             prefix_len=p_len, scale=scale)
    again = torch.empty_like(out)
    backend.prefix_attention(q, own.view, dev(np.array(lens, np.int32)), again,
                             prefix=prefix.view if prefix else None, prefix_len=p_len, scale=scale)
    backend.synchronize()
    assert torch.equal(out.view(torch.int16 if half else torch.int32), again.view(torch.int16 if half else torch.int32))
    want, tol, mag = attention64(wide[:, :, 1:-1].astype(np.float64), own, lens, prefix, p_len, scale or 1 / np.sqrt(hd))
    got = out.cpu().numpy().astype(np.float64)
    if half:  # one rounding of p and one of the result (2^-25: half the smallest f16 step)
        tol = tol + 2.0 ** -11 * mag + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want).max(), np.abs(want).max())
    empty = want == 0
    assert (got[empty] == 0).all()


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_own_lengths(um, backend, fmt, half, hd):
    check_attention(um, backend, fmt, half, hd, 2, 4, 1, EDGES, 0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("p_len", [1, 31, 64, 65, 130, 1027])
def test_attention_prefix_lengths(um, backend, fmt, half, p_len):
    check_attention(um, backend, fmt, half, 128, 2, 4, 1, [0, 3, 64, 0, 129], p_len)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,g,t", [(1, 1, 1), (3, 1, 2), (2, 3, 1), (1, 7, 4), (1, 8, 5), (2, 5, 3), (1, 16, 1), (1, 12, 11),
                                   (4, 8, 16), (1, 2, 33), (1, 33, 1), (1, 1, 130)])
def test_attention_heads_and_tokens(um, backend, half, hd, h, g, t):
    check_attention(um, backend, "i8", half, hd, h, g, t, [0, 1, 5, 40, 131], 70)


@pytest.mark.parametrize("fmt", FMTS)
def test_attention_many_sequences(um, backend, fmt):
    lens = [(i * 37) % 180 for i in range(70)]
    check_attention(um, backend, fmt, True, 128, 1, 4, 1, lens, 517)
    check_attention(um, backend, fmt, False, 64, 2, 2, 2, lens, 133)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("gain", [0.0, 30.0])
def test_attention_flat_and_sharp_scores(um, backend, half, gain):
    check_attention(um, backend, "f16", half, 128, 2, 4, 1, [1, 70, 300], 100, gain=gain)
    check_attention(um, backend, "i8", half, 64, 2, 4, 2, [0, 70, 300], 0, gain=gain, scale=0.25)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("p_len", [0, 90])
def test_attention_keeps_a_fault_to_its_sequence(um, backend, fmt, p_len):
    rng = np.random.default_rng(5)
    own = Cache(um, fmt, 3, 2, 100, 128, rng)
    prefix = Cache(um, fmt, 1, 2, 100, 128, rng) if p_len else None
    if fmt == "f16":
        own.t["v"][0][1, 0, 17, 3] = float("nan")
    else:
        own.t["v"][1][1, 0, 17] = float("nan")
    q = torch.randn((3, 1, 8, 128), device="cuda")
    out = torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(np.array([60, 60, 10], np.int32)), out,
                             prefix=prefix.view if prefix else None, prefix_len=p_len)
    backend.synchronize()
    nan = out.isnan()
    assert nan[1, 0, :4].any(-1).all()
    nan[1, 0, :4] = False
    assert not nan.any()


def test_attention_infinite_key_scores(um, backend):
    """A K row of -inf scores carries no weight; a row whose every visible score is -inf is 0, not NaN."""
    own = Cache(um, "f16", 1, 1, 8, 64, np.random.default_rng(1))
    own.t["k"][0][0, 0, :, 0] = float("-inf")
    q = torch.zeros((1, 1, 1, 64), device="cuda")
    q[..., 0] = 1.0
    own.t["k"][0][0, 0, 3, 0] = 0.5
    out = torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(np.array([8], np.int32)), out)
    backend.synchronize()
    assert torch.allclose(out[0, 0, 0], own.t["v"][0][0, 0, 3].float(), rtol=1e-6)
    backend.prefix_attention(q, own.view, dev(np.array([3], np.int32)), out)
    backend.synchronize()
    assert (out == 0).all()


def test_attention_reports_lengths_outside_the_cache(um, backend):
    own = Cache(um, "i8", 2, 1, 16, 64, np.random.default_rng(2))
    q = torch.randn((2, 1, 2, 64), device="cuda")
    out, full = torch.empty_like(q), torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(np.array([17, -1], np.int32)), out)
    with pytest.raises(um.UaiiMoeError) as e:
        backend.synchronize()
    assert e.value.status == um.INVALID_ARGUMENT and "length" in e.value.message
    backend.prefix_attention(q, own.view, dev(np.array([16, 0], np.int32)), full)
    backend.synchronize()
    assert torch.equal(out, full)


# ---------------------------------------------------------------- sampling


def sample(um, backend, logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):
    b = logits.shape[0]
    f = lambda v: torch.as_tensor(np.broadcast_to(np.asarray(v, np.float32), (b,)).copy()).cuda()  # noqa: E731
    k = torch.as_tensor(np.broadcast_to(np.asarray(top_k, np.int32), (b,)).copy()).cuda()
    tok, kept = (torch.full((b,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    p = torch.empty(b, device="cuda")
    x = logits if torch.is_tensor(logits) else dev(logits)
    backend.sample(x, f(temperature), k, f(top_p), f(min_p), f(u), tok, p, kept)
    backend.synchronize()
    return tok.cpu().numpy(), p.cpu().numpy(), kept.cpu().numpy()


@pytest.mark.parametrize("v", [1, 2, 3, 31, 1000, 4097, 32000])
def test_sample_ties_are_exact(um, backend, v):
    """Equal logits have equal whole weights: the k first indices are kept and u picks among them exactly."""
    u = np.array([0.0, 0.25, 0.5, 0.999999, 0.75], np.float32)
    x = np.full((5, v), 2.5, np.float32)
    for k in sorted({1, min(v, 7), v, v + 9}):
        tok, p, kept = sample(um, backend, x, 0.7, top_k=k, u=u)
        n = min(k, v)
        want = [min(n - 1, int(np.float64(z) * n * 2.0 ** 31 // 2 ** 31)) for z in u]
        assert tok.tolist() == want and (kept == n).all() and np.allclose(p, 1 / n, rtol=1e-7)
    tok, p, kept = sample(um, backend, x, 0.7, top_p=0.5, u=u)  # ceil(half the mass) of equal tokens
    assert (kept == -(-v // 2)).all()


def test_sample_two_levels_with_cuts_inside_the_ties(um, backend):
    """Logits 0 and -inf and a tie at the cut: exact whole numbers throughout."""
    v = 257
    x = np.full((1, v), -np.inf, np.float32)
    x[0, [5, 9, 100, 255]] = 1.0
    for k, n in ((0, 4), (2, 2), (3, 3), (4, 4)):
        for u, which in ((0.0, 0), (0.49, None), (0.9999, n - 1)):
            tok, p, kept = sample(um, backend, x, 1.3, top_k=k, u=u)
            at = [5, 9, 100, 255]
            assert tok[0] == at[int(u * n)] and p[0] == np.float32(1 / n)
            assert kept[0] == (n if k else v), (k, kept)  # without a cut the -inf tokens are kept, with no mass
    tok, p, kept = sample(um, backend, x, 1.0, top_p=0.6, u=0.999)
    assert kept[0] == 3 and tok[0] == 100  # 3/4 is the first leading part that reaches 0.6
    x[0, 200] = 0.0
    tok, p, kept = sample(um, backend, x, 1.0, min_p=0.5, u=0.999)
    assert kept[0] == 4 and tok[0] == 255


def interval(x, heat, k, p, least, tok):
    """(start, end) of the token's share of the kept mass in index order, and the kept count, in 64 bits."""
    x = x.astype(np.float64)
    e = np.exp((x - x.max()) / heat)
    order = np.argsort(-x, kind="stable")
    if k > 0:
        order = order[:k]
    if p < 1:
        m = e[order]
        before = np.cumsum(m) - m
        order = order[before < p * m.sum()]
    order = np.concatenate([order[:1], order[1:][e[order[1:]] >= least]])
    idx = np.sort(order)
    c = np.cumsum(e[idx]) / e[idx].sum()
    j = np.searchsorted(idx, tok)
    assert idx[j] == tok, "a token outside the kept set"
    return (c[j - 1] if j else 0.0), c[j], len(idx), e[tok] / e[idx].sum()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("v,ld", [(33, 33), (1000, 1003), (32000, 32000), (50257, 50304), (151937, 151937)])
def test_sample_against_the_definition(um, backend, half, v, ld):
    rng = np.random.default_rng(v)
    b = 24
    full = (3 * rng.standard_normal((b, ld))).astype(np.float16 if half else np.float32)
    full[rng.random((b, ld)) < 0.02] = -np.inf
    heat = rng.choice([0.3, 0.8, 1.0, 1.7], b).astype(np.float32)
    k = rng.choice([0, 1, 2, 40, 999, v + 1], b).astype(np.int32)
    p = rng.choice([0.1, 0.5, 0.9, 0.999, 1.0], b).astype(np.float32)
    least = rng.choice([0.0, 0.01, 0.3], b).astype(np.float32)
    u = rng.random(b).astype(np.float32)
    tok, prob, kept = sample(um, backend, dev(full)[:, :v], heat, k, p, least, u)
    for i in range(b):
        x = full[i, :v].astype(np.float64)
        lo, hi, n, want_p = interval(x, float(heat[i]), int(k[i]), float(p[i]), float(least[i]), tok[i])
        assert lo - 2e-6 <= u[i] <= hi + 2e-6, (i, lo, hi, u[i])
        # a cut by mass or by min_p may fall one token to either side where two masses agree to the rounding
        assert abs(int(kept[i]) - n) <= (0 if p[i] >= 1 and least[i] == 0 else 1), (i, kept[i], n)
        assert abs(prob[i] - want_p) <= 1e-5 * want_p + (1e-6 if p[i] < 1 else 0)


def test_sample_frequencies(um, backend):
    """A grid of u over one distribution: each token's share of the grid is its probability."""
    v, n = 50, 20000
    x = (2 * np.random.default_rng(1).standard_normal(v)).astype(np.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tok, _, _ = sample(um, backend, np.broadcast_to(x, (n, v)), 0.9, u=u)
    e = np.exp(x.astype(np.float64) / np.float32(0.9))
    assert np.abs(np.bincount(tok, minlength=v) / n - e / e.sum()).max() <= 1.5 / n


def test_sample_greedy_and_odd_settings(um, backend):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((9, 700)).astype(np.float32)
    x[:, 300] = x[:, 611] = 9.0  # the first of two largest
    heat = [0.0, -1.0, np.nan, 1.0, 1.0, 1.0, 1e-30, 1.0, 1.0]
    k = [0, 5, 0, 1, 0, 0, 0, 0, -3]
    p = [0.5, 1.0, 0.9, 1.0, 0.0, 1.0, 1.0, np.nan, 1.0]
    least = [0.0, 0.0, 0.5, 0.0, 0.0, 1.5, 1.0, 0.0, np.nan]
    tok, prob, kept = sample(um, backend, x, heat, k, p, least, u=[0.999, 0.5, 0.2, 0.7, 0.9, 0.9, 0.9, 0.9, 0.9])
    assert tok.tolist() == [300] * 6 + [611] + [300] * 2
    assert kept.tolist() == [1] * 6 + [2] + [1] * 2 and prob.tolist() == [1.0] * 6 + [0.5] + [1.0] * 2


def test_sample_rows_without_or_with_infinite_logits(um, backend):
    x = np.zeros((5, 40), np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 7], x[2, 30] = np.inf, np.inf
    x[3, :39] = np.nan
    x[4, 3] = np.nan
    tok, prob, kept = sample(um, backend, x, u=0.6)
    assert tok[:4].tolist() == [-1, -1, 30, 39] and prob[:4].tolist() == [0.0, 0.0, 0.5, 1.0]
    assert kept[:2].tolist() == [0, 0]
    assert tok[4] == 24 and prob[4] == np.float32(1 / 39)  # 39 equal tokens, index 3 without mass


def test_sample_signed_zeros_tie(um, backend):
    x = np.full((1, 64), -5.0, np.float32)
    x[0, 10], x[0, 20] = -0.0, 0.0
    tok, _, kept = sample(um, backend, x, top_k=1, u=0.5)
    assert tok[0] == 10 and kept[0] == 1


def test_sample_outside_uniforms(um, backend):
    x = np.zeros((4, 8), np.float32)
    tok, _, _ = sample(um, backend, x, u=[1.0, 2.0, -1.0, np.nan])
    assert tok.tolist() == [7, 7, 0, 0]


# ---------------------------------------------------------------- refusals


def test_refusals(um, backend):
    rng = np.random.default_rng(0)
    own = Cache(um, "i8", 2, 2, 16, 64, rng)
    one = Cache(um, "i8", 1, 2, 16, 64, rng)
    f16 = Cache(um, "f16", 1, 2, 16, 64, rng)
    x = torch.zeros((2, 1, 2, 64), device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros((2, 2, 16, 64), device="cuda")

    def refused(status, part, call, *args, **kw):
        with pytest.raises(um.UaiiMoeError) as e:
            call(*args, **kw)
        assert e.value.status == status and part in e.value.message, e.value.message

    def bent(**kw):
        c = um.KVCache.from_buffer_copy(own.view)
        for n, v in kw.items():
            setattr(c, n, v)
        c._keep = own.t
        return c

    bad = um.INVALID_ARGUMENT
    wide = torch.zeros((2, 1, 2, 80), device="cuda")
    refused(um.NOT_IMPLEMENTED, "head_dim", backend.kv_append, bent(head_dim=80), wide, wide, pos)
    refused(um.NOT_IMPLEMENTED, "format", backend.kv_append, bent(fmt=um.Q8_0), x, x, pos)
    refused(bad, "out of range", backend.kv_read, bent(max_seq=0), 0, 0, out[:, :, :0], out[:, :, :0])
    refused(bad, "device memory", backend.kv_append, bent(k=own.enc["k"][0].ctypes.data), x, x, pos)
    refused(bad, "scales", backend.kv_append, bent(k_scale=None), x, x, pos)
    refused(bad, "16-byte", backend.kv_append, bent(k=own.view.k + 8), x, x, pos)
    refused(bad, "device memory", backend.kv_append, own.view, x.cpu(), x.cpu(), pos)
    refused(bad, "device memory", backend.kv_append, own.view, x, x, pos.cpu())
    long = torch.zeros((2, 17, 2, 64), device="cuda")
    refused(bad, "token count", backend.kv_append, own.view, long, long, pos)
    refused(bad, "outside", backend.kv_read, own.view, 1, 16, out, out)
    refused(bad, "outside", backend.kv_read, own.view, -1, 16, out, out)
    q, o = torch.zeros((2, 1, 4, 64), device="cuda"), torch.zeros((2, 1, 4, 64), device="cuda")
    att = backend.prefix_attention
    refused(bad, "multiple", att, x.new_zeros((2, 1, 3, 64)), own.view, pos, x.new_zeros((2, 1, 3, 64)))
    refused(bad, "prefix_len", att, q, own.view, pos, o, prefix_len=3)
    refused(bad, "exceeds", att, q, own.view, pos, o, prefix=one.view, prefix_len=17)
    refused(bad, "negative", att, q, own.view, pos, o, prefix=one.view, prefix_len=-1)
    refused(bad, "share format", att, q, own.view, pos, o, prefix=f16.view, prefix_len=3)
    refused(bad, "one sequence", att, q, own.view, pos, o, prefix=own.view, prefix_len=3)
    refused(bad, "finite", att, q, own.view, pos, o, scale=float("inf"))
    refused(bad, "device memory", att, q.cpu(), own.view, pos, o)
    s = torch.zeros((2, 8), device="cuda")
    f, i = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    refused(bad, "vocab", backend.sample, s[:, :0], f, i, f, f, f, i)
    refused(bad, "device memory", backend.sample, s.cpu(), f, i, f, f, f, i)
    refused(bad, "device memory", backend.sample, s, f, i, f, f, f, i, kept=i.cpu())
    # the binding's own checks
    with pytest.raises(TypeError):
        backend.sample(s.double(), f, i, f, f, f, i)
    with pytest.raises(ValueError):
        backend.sample(s, f[:1], i, f, f, f, i)
    with pytest.raises(TypeError):
        backend.sample(s, f, f, f, f, f, i)
    with pytest.raises(ValueError):
        backend.sample(s.t(), f, i, f, f, f, i)
    with pytest.raises(ValueError):
        backend.kv_append(own.view, x, x.transpose(1, 2).contiguous().transpose(1, 2)[:, :, :1], pos)
    with pytest.raises(TypeError):
        um.kv_cache(um.KV_I8, own.t["k"][0].view(torch.int8), own.t["v"][0], own.t["k"][1], own.t["v"][1])
    backend.synchronize()


def test_empty_calls_do_nothing(um, backend):
    own = Cache(um, "i8", 2, 2, 16, 64, np.random.default_rng(0))
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.zeros((2, 0, 2, 64), device="cuda")
    backend.kv_append(own.view, x, x, pos)
    backend.prefix_attention(x, own.view, pos, x)
    z = torch.zeros((0, 8), device="cuda")
    f, i = torch.zeros(0, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    backend.sample(z, f, i, f, f, f, i)
    backend.synchronize()


def test_calls_on_a_stream_of_the_caller(um):
    """A backend on the caller's stream: producers and consumers there need no synchronization in between."""
    st = torch.cuda.Stream()
    be = um.Backend(0, stream=st.cuda_stream)
    try:
        with torch.cuda.stream(st):
            big = torch.randn((4096, 4096), device="cuda")
            for _ in range(4):
                big = big @ big * 1e-2
            x = (big[:2, :4 * 64].reshape(2, 2, 2, 64) * 0 + torch.randn((2, 2, 2, 64), device="cuda")).nan_to_num(0.25)
            k = torch.zeros((2, 2, 8, 64), dtype=torch.uint8, device="cuda")
            v, s1, s2 = torch.zeros_like(k), torch.zeros((2, 2, 8), device="cuda"), torch.zeros((2, 2, 8), device="cuda")
            pos = torch.zeros(2, dtype=torch.int32, device="cuda")
            c = um.kv_cache(um.KV_I8, k, v, s1, s2)
            be.kv_append(c, x, x, pos)
            out = torch.empty((2, 2, 2, 64), device="cuda")
            be.kv_read(c, 0, 2, out, torch.empty_like(out))
            got = out + 0
        st.synchronize()
        q, sc = encode(x.cpu().numpy(), "i8")
        assert np.array_equal(got.cpu().numpy(), values(q, sc, "i8").astype(np.float32).transpose(0, 2, 1, 3))
        be.synchronize()
    finally:
        be.close()
