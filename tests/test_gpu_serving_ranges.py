"""Attention where rows, scores and lengths are far from alike: V rows of very unequal size, keys that weigh nothing, long
walks of one warp.

Reference: the definition in 64 bits over the stored rows.  With p_j the probabilities and e_j the bound of a score's error,
2^-18 * scale * sum_d |q_d k_jd| (f32 sums of 16-element products: at most 16 roundings of 2^-23 of the summed magnitudes,
and a split of q to 2^-22), a result may be off by
    sum_j p_j e_j |v_j|  +  (sum_j p_j e_j) sum_j p_j |v_j|          the scores' errors, in weights and denominator
  + ((n / 16 + 64) 2^-23 + 2^-20) sum_j p_j |v_j|                    sums over n positions; exponentials and scales
  + n 2^-32 max_j (p_j max_d |v_jd|)                                 weights that f16's smallest step cuts: at most 2^-25
                                                                     in each of two parts, where the largest product of
                                                                     a weight and a row's scale is 2^8 or more
f16 results add a rounding of p and of the result: 2^-11 (sum_j p_j |v_j| + |result|) + 2^-25; where the test says so, of
the result alone: 2^-11 |result| + 2^-25.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_serving import FMTS, code, dev, encode, values  # noqa: E402


class Rows:
    """A cache of given rows: k, v [batch, heads, positions, head_dim]."""

    def __init__(self, um, fmt, k, v):
        self.val, t = {}, {}
        for n, x in (("k", k), ("v", v)):
            c, s = (x.astype(np.float16), None) if fmt == "f16" else encode(x, fmt)
            self.val[n] = dev(values(c, s, fmt))
            t[n], t[n + "s"] = dev(c), None if s is None else dev(s)
        self.view = um.kv_cache(code(um, fmt), t["k"], t["v"], t["ks"], t["vs"])

    def rows(self, n, i, kh, end):
        return self.val[n][i, kh, :end]


class DeviceRows:
    """The same of rows made on the device, where they may be many."""

    def __init__(self, um, fmt, k, v):
        self.fmt, self.t = fmt, {}
        for n, x in (("k", k), ("v", v)):
            if fmt == "f16":
                self.t[n] = x.half(), None
                continue
            scale = x.abs().amax(-1) / (127 if fmt == "i8" else 448)
            y = x / scale[..., None]
            self.t[n] = ((y.round() + 128).to(torch.uint8) if fmt == "i8" else y.to(torch.float8_e4m3fn).view(torch.uint8)), scale
        self.view = um.kv_cache(code(um, fmt), *(self.t[n][j] for j in (0, 1) for n in "kv"))

    def rows(self, n, i, kh, end):
        c, s = self.t[n]
        c = c[i, kh, :end]
        if self.fmt == "f16":
            return c.double()
        c = c.double() - 128 if self.fmt == "i8" else c.view(torch.float8_e4m3fn).double()
        return c * s[i, kh, :end, None].double()


def definition(q, own, lens, prefix=None, p_len=0, scale=None):
    """(result, tolerance for f32 results, sum p |v|), all in 64 bits on the device; q [B, T, H, d]."""
    b, t, hq, d = q.shape
    h = own.view.n_kv_heads
    g = hq // h
    scale = scale or d ** -0.5
    q = q.double().view(b, t, h, g, d)
    out, tol, mag = (torch.zeros_like(q) for _ in range(3))
    for i in range(b):
        for kh in range(h):
            k, v = own.rows("k", i, kh, lens[i]), own.rows("v", i, kh, lens[i])
            if p_len:
                k, v = torch.cat([prefix.rows("k", 0, kh, p_len), k]), torch.cat([prefix.rows("v", 0, kh, p_len), v])
            n = len(k)
            if n == 0:
                continue
            x = q[i, :, kh]
            sees = torch.arange(n, device="cuda") < p_len + torch.arange(t, device="cuda")[:, None] + lens[i] - t + 1
            sees |= torch.arange(n, device="cuda") < p_len
            s = (scale * x @ k.T).masked_fill(~sees[:, None], float("-inf"))
            p = torch.softmax(s, -1).nan_to_num(0.0)
            e = p * (2.0 ** -18 * scale * x.abs() @ k.abs().T)
            w, peak = p @ v.abs(), (p * v.abs().amax(-1)).amax(-1, keepdim=True)
            out[i, :, kh], mag[i, :, kh] = p @ v, w
            tol[i, :, kh] = (e @ v.abs() + e.sum(-1, keepdim=True) * w + ((n / 16 + 64) * 2.0 ** -23 + 2.0 ** -20) * w
                             + n * 2.0 ** -32 * peak)
    return tuple(x.view(b, t, hq, d) for x in (out, tol, mag))


def check(um, backend, q, own, lens, prefix=None, p_len=0, scale=0.0, weights=2.0 ** -11):
    out = torch.full_like(q, 9.0)
    backend.prefix_attention(q, own.view, dev(np.array(lens, np.int32)), out, prefix=prefix.view if prefix else None,
                             prefix_len=p_len, scale=scale)
    backend.synchronize()
    want, tol, mag = definition(q, own, lens, prefix, p_len, scale)
    if q.dtype is torch.float16:
        tol = tol + weights * mag + 2.0 ** -11 * want.abs() + 2.0 ** -25
        over = want.abs() - tol >= 65520.0  # beyond the type: an infinity (and near its end, either)
        assert (out[over] == torch.copysign(torch.full_like(want[over], float("inf")), want[over])).all()
        edge = want.abs() + tol >= 65520.0
        out, want, tol = (torch.where(edge, torch.zeros_like(x), x) for x in (out, want, tol))
    off = (out.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), float((off / tol).nan_to_num(1e30).max()),
                           float((off.amax() / want.abs().amax())))


def queries(b, t, hq, d, half, rng, lead=4.0):
    """Random queries whose dimension 0 is `lead`: a key's dimension 0 then moves all their scores alike."""
    q = rng.standard_normal((b, t, hq, d))
    q[..., 0] = lead
    return dev(q.astype(np.float16 if half else np.float32))


def random_rows(rng, *shape):
    k, v = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    k[..., 0] = 0
    return k, v


SHAPES = [(4, 1), (4, 4), (7, 4)]  # query heads of a kv head, tokens: items of 4, 16 and 28 rows


# ---------------------------------------------------------------- V rows of unequal size


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("g,t", SHAPES)
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("nats", [4.0, 18.0, 100.0])
def test_a_large_v_row_of_little_weight(um, backend, fmt, half, g, t, ratio, nats):
    """One V row is `ratio` times larger than the others, its key `nats` below them: whatever it weighs, the others keep
    their bits (in the own positions at three places, and in the prefix)."""
    rng = np.random.default_rng(int(nats) + g + t)
    b, h, d, n, p_len = 3, 2, 128, 200, 140
    k, v = random_rows(rng, b, h, n, d)
    pk, pv = random_rows(rng, 1, h, p_len, d)
    for x, y, at in ((k[0], v[0], 0), (k[1], v[1], n // 2), (k[2], v[2], n - t - 1), (pk[0], pv[0], 70)):
        x[:, at] = 0
        x[:, at, 0] = -nats * d ** 0.5 / 4.0
        y[:, at] *= ratio
    own, prefix = Rows(um, fmt, k, v), Rows(um, fmt, pk, pv)
    q = queries(b, t, g * h, d, half, rng)
    check(um, backend, q, own, [n] * b)
    check(um, backend, q, own, [n, n, n - 70], prefix, 70)   # (the prefix's large row is its first unseen one)
    check(um, backend, q, own, [n, 60, n - 70], prefix, p_len)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("g,t", SHAPES)
def test_a_large_v_row_that_earlier_tokens_do_not_see(um, backend, fmt, half, g, t):
    """The last token's V row is 1e8 times larger: the tokens before it, which do not see it, keep their bits."""
    rng = np.random.default_rng(g)
    b, h, d, n = 2, 2, 64, 90
    k, v = random_rows(rng, b, h, n, d)
    v[:, :, -1] *= 1e8
    check(um, backend, queries(b, t, g * h, d, half, rng), Rows(um, fmt, k, v), [n, n])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("g,t", SHAPES)
@pytest.mark.parametrize("v_up", [-24, 24])
@pytest.mark.parametrize("k_up", [-120.0, 0.0, 120.0])
def test_v_rows_that_grow_or_shrink_along_the_sequence(um, backend, fmt, half, g, t, v_up, k_up):
    """V's size changes by 2^v_up from the first position to the last, the scores by k_up nats: the largest product of both
    moves along the sequence, with and against the largest score."""
    rng = np.random.default_rng(g + t)
    b, h, d, n = 2, 1, 64, 420
    k, v = random_rows(rng, b, h, n, d)
    along = np.linspace(0, 1, n)
    v *= 2.0 ** (v_up * along)[:, None].astype(np.float32)
    k = (0.5 * k).astype(np.float32)
    k[..., 0] = k_up * along * d ** 0.5 / 4.0
    check(um, backend, queries(b, t, g * h, d, half, rng), Rows(um, fmt, k, v), [n, n - 130])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("g,t", SHAPES)
@pytest.mark.parametrize("nats", [12.0, 40.0])
def test_a_heavy_position_whose_v_is_zero(um, backend, fmt, half, g, t, nats):
    """Nearly all weight lies on a position whose V row is zero: the result is the others' small share, to its own bits."""
    rng = np.random.default_rng(g)
    b, h, d, n = 2, 2, 128, 150
    k, v = random_rows(rng, b, h, n, d)
    k[0, :, 0, 0] = k[1, :, 77, 0] = nats * d ** 0.5 / 4.0
    v[0, :, 0] = v[1, :, 77] = 0
    check(um, backend, queries(b, t, g * h, d, half, rng), Rows(um, fmt, k, v), [n, n])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("g,t", SHAPES)
@pytest.mark.parametrize("size", [1e-20, 1e-3, 1e15])
def test_v_of_any_size(um, backend, fmt, half, g, t, size):
    """All V rows tiny or huge (f16 results: within their type)."""
    rng = np.random.default_rng(g)
    b, h, d, n = 2, 2, 64, 150
    k, v = random_rows(rng, b, h, n, d)
    if half and size > 1:
        size = 1e4
    check(um, backend, queries(b, t, g * h, d, half, rng), Rows(um, fmt, k, (v * size).astype(np.float32)), [n, n - 7])


# ---------------------------------------------------------------- keys that weigh nothing


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("g,t", [(4, 1), (3, 4), (7, 4)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lead", [1e-9, -3e-8, 1e-12, 0.7])
def test_infinite_keys_against_small_query_values(um, backend, half, g, t, d, lead):
    """Keys masked by an infinity in one dimension, where the queries hold a value that may be far below the row's largest:
    the masked positions lose their weight and nothing else changes."""
    rng = np.random.default_rng(g + d)
    b, h, n = 2, 2, 130
    k, v = random_rows(rng, b, h, n, d)
    hidden = rng.random(n) < 0.4
    hidden[-t:] = False  # (every token sees the same finite keys but its own last ones)
    if half:
        lead = np.copysign(max(abs(lead), 6e-8), lead)  # f16's smallest
    k[:, :, hidden, 0] = np.copysign(np.inf, -lead)
    q = queries(b, t, g * h, d, half, rng, lead=lead)
    own, left = Rows(um, "f16", k, v), Rows(um, "f16", k[:, :, ~hidden], v[:, :, ~hidden])
    out = torch.full_like(q, 9.0)
    backend.prefix_attention(q, own.view, dev(np.array([n] * b, np.int32)), out)
    backend.synchronize()
    want, tol, mag = definition(q, left, [int((~hidden).sum())] * b)
    if half:
        tol = tol + 2.0 ** -11 * (mag + want.abs()) + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()


# ---------------------------------------------------------------- long walks


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("half,g,t", [(False, 4, 1), (True, 4, 1), (True, 4, 4)])
def test_many_steps_of_one_warp(um, backend, fmt, d, half, g, t):
    """Thousands of positions of many sequences, so that a warp walks some thirty to seventy steps of one item: copies reuse
    their places, references rise while sums are not zero, small weights follow large ones.  By turns, sequences are plain,
    their scores rise by 60 nats along the positions, their V grows 2^12-fold, and both at once with V falling."""
    gen = torch.Generator(device="cuda").manual_seed(d + g + t)
    b, h, n = 64, 8, 3900
    k, v = (torch.randn((b, h, n, d), generator=gen, device="cuda") for _ in range(2))
    along, kind = torch.linspace(0, 1, n, device="cuda"), torch.arange(b, device="cuda") % 4
    k[..., 0] = 60 * d ** 0.5 / 4.0 * along * (kind % 2 == 1)[:, None, None]
    turn = torch.where(kind == 2, 1.0, torch.where(kind == 3, -1.0, 0.0))[:, None, None]
    v *= torch.exp2(12 * turn * (along - 0.5))[..., None]
    own = DeviceRows(um, fmt, k, v)
    del k, v
    q = torch.randn((b, t, g * h, d), generator=gen, device="cuda")
    q[..., 0] = 4.0
    check(um, backend, q.half() if half else q, own, [n - 61 * (i % 7) for i in range(b)])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
def test_many_tiles_of_one_block(um, backend, fmt, half):
    """Items of 160 rows over a prefix of thousands of positions: a block walks some tens of tiles of one item, with scores
    that rise and V that grows, then falls."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    b, h, g, d, n = 40, 8, 4, 128, 31000
    k, v = (torch.randn((1, h, n, d), generator=gen, device="cuda") for _ in range(2))
    along = torch.linspace(0, 1, n, device="cuda")
    k[..., 0] = 40 * d ** 0.5 / 4.0 * along * (torch.arange(h, device="cuda") % 2)[:, None]
    v *= torch.exp2(12 * (1 - (2 * along - 1).abs()))[:, None]
    prefix = DeviceRows(um, fmt, k, v)
    own = DeviceRows(um, fmt, *(torch.randn((b, h, 30, d), generator=gen, device="cuda") for _ in range(2)))
    q = torch.randn((b, 1, g * h, d), generator=gen, device="cuda")
    q[..., 0] = 4.0
    check(um, backend, q.half() if half else q, own, [i % 31 for i in range(b)], prefix, n)


@pytest.mark.parametrize("fmt,d", [("i8", 64), ("e4m3", 128), ("f16", 64), ("f16", 128)])
def test_long_f32_sums_of_few_rows_do_not_shrink(um, backend, fmt, d):
    """Few rows over tens of thousands of positions, hundreds of steps of one warp: an accumulator that is cut off at each
    addition loses 2^-24 of itself on average, so 32 additions to a sum that grows from nothing lose 32 / 2 * 2^-24 of it,
    1e-6; scores (8 additions) and the roundings of the rows as much again.  Bar on the whole result: 2.5e-6."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    b, h, g, n = 96, 4 if fmt == "f16" else 8, 2, 24000
    k = torch.empty((b, h, n, d), dtype=torch.float16 if fmt == "f16" else torch.uint8, device="cuda")
    own = DeviceRows.__new__(DeviceRows)
    own.fmt, own.t = fmt, {}
    for name in "kv":
        if fmt == "f16":
            own.t[name] = torch.randn(k.shape, generator=gen, dtype=torch.float16, device="cuda"), None
        else:  # any bytes are rows; e4m3's two NaNs are not
            c = torch.randint(1, 126, k.shape, generator=gen, dtype=torch.uint8, device="cuda")
            c += 128 * torch.randint(0, 2, k.shape, generator=gen, dtype=torch.uint8, device="cuda")
            own.t[name] = c, (0.015 if fmt == "i8" else 0.01) * (0.5 + torch.rand((b, h, n), generator=gen, device="cuda"))
    own.view = um.kv_cache(code(um, fmt), *(own.t[x][j] for j in (0, 1) for x in "kv"))
    q = torch.randn((b, 1, g * h, d), generator=gen, device="cuda")
    out = torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(np.full(b, n, np.int32)), out)
    backend.synchronize()
    off = whole = 0.0
    for i in range(b):
        for kh in range(h):
            x = q[i, 0, kh * g:(kh + 1) * g].double()
            want = torch.softmax(x @ own.rows("k", i, kh, n).T / d ** 0.5, -1) @ own.rows("v", i, kh, n)
            off += float((out[i, 0, kh * g:(kh + 1) * g].double() - want).square().sum())
            whole += float(want.square().sum())
    assert (off / whole) ** 0.5 <= 2.5e-6, (off / whole) ** 0.5


# ---------------------------------------------------------------- f16 queries


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,g,t,p_len,n", [(3, 4, 1, 0, 300), (3, 4, 3, 0, 300), (3, 4, 4, 200, 70), (3, 7, 4, 200, 70),
                                           (70, 4, 1, 900, 40), (2, 2, 90, 0, 200)])
def test_f16_results_are_rounded_once(um, backend, fmt, d, b, g, t, p_len, n):
    """Whatever the rows of an item (4, 12, 16, 28, 280 over a prefix, 180), the weights keep f32's bits and the result is
    rounded once."""
    rng = np.random.default_rng(b + g + t)
    h = 2
    own = Rows(um, fmt, *(rng.standard_normal((b, h, n, d)).astype(np.float32) for _ in range(2)))
    prefix = Rows(um, fmt, *(rng.standard_normal((1, h, p_len, d)).astype(np.float32) for _ in range(2))) if p_len else None
    q = dev(rng.standard_normal((b, t, g * h, d)).astype(np.float16))
    check(um, backend, q, own, [n - i % 30 for i in range(b)], prefix, p_len, weights=0.0)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("g,t", [(4, 1), (4, 4), (3, 5), (7, 4)])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_infinite_v_that_every_token_sees(um, backend, half, d, g, t, where):
    """An infinity of V at a position of weight makes an infinity of its sign of that dimension and nothing of the others,
    whether its weight has a rest beside f16's leading part or none (equal scores: a weight of 2^8)."""
    rng = np.random.default_rng(g)
    b, h, n, p_len = 2, 2, 80, 90
    for k_gain in (0.0, 0.5):
        (k, v), (pk, pv) = random_rows(rng, b, h, n, d), random_rows(rng, 1, h, p_len, d)
        k, pk = k_gain * k, k_gain * pk
        clean = definition(q := queries(b, t, g * h, d, half, rng), Rows(um, "f16", k, v), [n] * b, Rows(um, "f16", pk, pv), p_len)
        y = pv if where == "prefix" else v
        y[:, :, 20, 3], y[:, :, 41, 17] = np.inf, -np.inf
        out = torch.empty_like(q)
        backend.prefix_attention(q, Rows(um, "f16", k, v).view, dev(np.array([n] * b, np.int32)), out,
                                 prefix=Rows(um, "f16", pk, pv).view, prefix_len=p_len)
        backend.synchronize()
        assert (out[..., 3] == np.inf).all() and (out[..., 17] == -np.inf).all()
        rest = [x for x in range(d) if x not in (3, 17)]
        want, tol, _ = (x[..., rest] for x in clean)
        tol = tol + (2.0 ** -11 * want.abs() + 2.0 ** -25 if half else 0)
        assert ((out[..., rest].double() - want).abs() <= tol).all()
