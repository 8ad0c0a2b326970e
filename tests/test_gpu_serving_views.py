"""Views that the serving operators take: dimensions of one element, whose strides say nothing.

The cache's bytes are those of the contiguous call, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_serving import Cache, dev  # noqa: E402


@pytest.mark.parametrize("fmt", ["f16", "i8", "e4m3"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("b,t,h", [(4, 1, 8), (1, 5, 3), (3, 4, 1), (1, 1, 4), (1, 1, 1)])
def test_append_of_views_that_differ_in_dimensions_of_one(um, backend, fmt, half, b, t, h):
    rng = np.random.default_rng(b + t + h)
    dtype = torch.float16 if half else torch.float32
    k, v = (torch.randn((b, t, h, 128), device="cuda").to(dtype) for _ in range(2))
    other = v
    for i, n in enumerate((b, t, h)):  # the same memory order, other strides where a dimension has one element
        if n == 1:
            s = list(other.stride())
            s[i] = 7 + 2 * i
            other = other.as_strided(other.shape, s)
    assert other.stride() != k.stride() and torch.equal(other, v)
    pos = dev(np.zeros(b, np.int32))
    one, two = (Cache(um, fmt, b, h, t + 2, 128, np.random.default_rng(1)) for _ in range(2))
    backend.kv_append(one.view, k, v, pos)
    backend.kv_append(two.view, k, other, pos)
    backend.synchronize()
    for n in "kv":
        for x, y in zip(one.t[n], two.t[n]):
            assert x is y is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    lens, q = dev(np.full(b, t, np.int32)), torch.randn((b, t, 2 * h, 128), device="cuda").to(dtype)
    outs = [torch.empty_like(q) for _ in range(2)]
    s = [7 if n == 1 else z for n, z in zip(q.shape[:3], q.stride())] + [1]
    backend.prefix_attention(q, one.view, lens, outs[0])
    backend.prefix_attention(q.as_strided(q.shape, s), one.view, lens, outs[1])
    backend.synchronize()
    assert torch.equal(*outs)


def test_append_still_refuses_views_of_another_layout(um, backend):
    c = Cache(um, "i8", 2, 3, 8, 64, np.random.default_rng(1))
    k = torch.zeros((2, 4, 3, 64), device="cuda")
    pos = dev(np.zeros(2, np.int32))
    for v in (torch.zeros((2, 3, 4, 64), device="cuda").transpose(1, 2), torch.zeros((2, 4, 6, 64), device="cuda")[:, :, :3],
              k[:, :, :, :32], k.half()):
        with pytest.raises(ValueError):
            backend.kv_append(c.view, k, v, pos)
