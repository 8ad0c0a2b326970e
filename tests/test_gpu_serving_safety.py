"""Serving operators where blocks, warps and calls meet one another: sampling rows whose blocks have little to read, and
faults that one lane clears for the others.

Sampled tokens are held to the definition's exactly (whole-number weights).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_serving import FMTS, Cache, check_attention, dev, sample  # noqa: E402


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("b,v", [(3000, 4097), (1500, 8200), (1100, 16385), (600, 32769)])
def test_sample_rows_of_many_short_blocks(um, backend, half, b, v):
    """Thousands of clusters whose blocks read a few thousand logits each and start at different times: the largest
    logit, wherever it lies, reaches every block, and equal logits are drawn exactly."""
    rng = np.random.default_rng(v)
    x = rng.standard_normal((b, v)).astype(np.float16 if half else np.float32)
    at = rng.integers(0, v, b)
    x[np.arange(b), at] = 9.0
    two = (at + 1 + rng.integers(0, v - 1, b)) % v
    x[np.arange(b), two] = 9.0
    u = rng.random(b).astype(np.float32)
    xd = dev(x)
    tok, prob, kept = sample(um, backend, xd, 0.0, u=u)
    assert np.array_equal(tok, np.minimum(at, two)) and (kept == 1).all() and (prob == 1).all()
    tok, prob, kept = sample(um, backend, xd, 1.0, min_p=0.9, u=u)  # the next logit is far below 9
    assert np.array_equal(tok, np.where(u < 0.5, np.minimum(at, two), np.maximum(at, two)))
    assert (kept == 2).all() and (prob == 0.5).all()


@pytest.mark.parametrize("fmt,half,hd,g,t", [("f16", False, 128, 2, 4), ("f16", True, 64, 2, 8), ("e4m3", False, 64, 1, 7),
                                             ("e4m3", True, 128, 4, 4), ("f16", True, 128, 4, 2)])
def test_attention_faults_in_every_position_that_some_tokens_do_not_see(um, backend, fmt, half, hd, g, t):
    """NaNs in V of every position that only later tokens see, in all dimensions and many sequences: whichever lane of a
    warp clears a byte, no other lane reads it as it was.  The first tokens' results are as without them, bit for bit."""
    rng = np.random.default_rng(t)
    b = 96
    lens = np.array([t + (i * 7) % 90 for i in range(b)], np.int32)
    own = Cache(um, fmt, b, 2, int(lens.max()) + 1, hd, rng)
    q = torch.randn((b, t, 2 * g, hd), device="cuda").to(torch.float16 if half else torch.float32)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    backend.prefix_attention(q, own.view, dev(lens), clean)
    for i, n in enumerate(lens):
        own.t["v"][0][i, :, n - t + 1:] = float("nan") if fmt == "f16" else 0xff
    for _ in range(3):
        backend.prefix_attention(q, own.view, dev(lens), out)
        backend.synchronize()
        assert torch.equal(out[:, 0], clean[:, 0]) and out[:, 1:].isnan().all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("half", [False, True])
def test_attention_many_items_of_one_tile(um, backend, fmt, half):
    """Items of many rows whose keys are one tile (or none): one of the two warps that issue products has nothing to issue
    between the pieces, and keeps step with them."""
    lens = [(i * 23) % 65 for i in range(300)]
    check_attention(um, backend, fmt, half, 128, 3, 8, 3, lens, 0)


@pytest.mark.parametrize("g,t,p_len", [(4, 1, 0), (4, 1, 100), (8, 4, 100)])
def test_attention_calls_in_a_row_with_other_lengths(um, backend, g, t, p_len):
    """Calls queued back to back share the workspace: each joins the pieces that its own lengths give."""
    rng = np.random.default_rng(g)
    b, h, hd = 40, 2, 64
    own, prefix = Cache(um, "i8", b, h, 400, hd, rng), Cache(um, "i8", 1, h, 128, hd, rng)
    q = torch.randn((b, t, h * g, hd), device="cuda")
    lens = [dev(x.astype(np.int32)) for x in (np.full(b, 400), np.arange(b) * 3 % 7, rng.integers(0, 400, b),
                                             np.where(np.arange(b) % 2, 399, 0))]
    kw = dict(prefix=prefix.view, prefix_len=p_len) if p_len else {}
    alone = []
    for n in lens:
        out = torch.empty_like(q)
        backend.prefix_attention(q, own.view, n, out, **kw)
        backend.synchronize()
        alone.append(out)
    order = [0, 1, 0, 2, 3, 1, 2, 0, 3] * 20
    outs = [torch.empty_like(q) for _ in order]
    for i, out in zip(order, outs):
        backend.prefix_attention(q, own.view, lens[i], out, **kw)
    backend.synchronize()
    assert all(torch.equal(out, alone[i]) for i, out in zip(order, outs))


def test_sample_refuses_misaligned_arrays(um, backend):
    """Addresses that are no multiple of an element's size are refused on the host, one argument at a time."""
    b, v = 2, 8
    x = torch.zeros((b, v), device="cuda")
    f, i = torch.zeros(b + 1, device="cuda"), torch.zeros(b + 1, dtype=torch.int32, device="cuda")
    good = [f, i, f, f, f, i.clone(), f.clone(), i.clone()]  # temperature, top_k, top_p, min_p, u, tokens, probs, kept
    for at in range(len(good)):
        for shift in (1, 2, 3):
            ptrs = [a.data_ptr() + (shift if k == at else 0) for k, a in enumerate(good)]
            st = um.lib.uaii_moe_sample(backend._h, x.data_ptr(), um.DTYPE_F32, b, v, v, *ptrs)
            assert st == um.INVALID_ARGUMENT and b"misaligned" in um.lib.uaii_moe_last_error(), (at, shift)
    st = um.lib.uaii_moe_sample(backend._h, x.data_ptr() + 2, um.DTYPE_F32, b, v, v, *[a.data_ptr() for a in good])
    assert st == um.INVALID_ARGUMENT
    st = um.lib.uaii_moe_sample(backend._h, x.data_ptr(), um.DTYPE_F32, b, v, v, *[a.data_ptr() for a in good])
    assert st == um.OK
    backend.synchronize()


def test_sample_from_several_threads_with_other_vocabularies(um):
    """Backends sample in threads of their own, rows of the largest vocabulary and short ones: no call's launch depends on
    the shared memory that another one asks for."""
    import threading

    errors, start = [], threading.Barrier(4)

    def work(v, b, n):
        be = um.Backend(0)
        try:
            x = torch.zeros((b, v), device="cuda")
            f, i = torch.ones(b, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            tok, zero, u = torch.empty(b, dtype=torch.int32, device="cuda"), f * 0, f * 0.5
            args = (be._h, x.data_ptr(), um.DTYPE_F32, b, v, v, f.data_ptr(), i.data_ptr(), f.data_ptr(), zero.data_ptr(),
                    u.data_ptr(), tok.data_ptr(), None, None)
            start.wait()
            for _ in range(n):
                st = um.lib.uaii_moe_sample(*args)
                assert st == um.OK, um.lib.uaii_moe_last_error()
            be.synchronize()
            assert (tok == v // 2).all()
        except Exception as e:  # noqa: BLE001 (reported by the test)
            errors.append((v, repr(e)))
        finally:
            be.close()

    threads = [threading.Thread(target=work, args=a) for a in ((400000, 1, 20000), (600, 1, 20000), (60000, 1, 20000), (20, 1, 20000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_calls_captured_in_a_graph(um):
    """A decode step's operators captured in a CUDA graph on the backend's stream: a replay gives what the calls gave."""
    st = torch.cuda.Stream()
    be = um.Backend(0, stream=st.cuda_stream)
    try:
        rng = np.random.default_rng(0)
        b, h, hd = 40, 2, 128
        own, prefix = Cache(um, "i8", b, h, 400, hd, rng), Cache(um, "i8", 1, h, 600, hd, rng)
        lens = dev((np.arange(b) * 9 % 400).astype(np.int32))
        q, drafts = torch.randn((b, 1, 8, hd), device="cuda"), torch.randn((b, 4, 16, hd), device="cuda").half()
        outs = [torch.empty_like(q), torch.empty_like(drafts), torch.empty(b, dtype=torch.int32, device="cuda")]
        x, f, i = torch.randn((b, 32000), device="cuda"), torch.ones(b, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
        settings = f, i + 40, f * 0.9, f * 0, f * 0.5
        row, pos = torch.randn((b, 1, h, hd), device="cuda"), i + 399
        torch.cuda.synchronize()

        def step():
            be.kv_append(own.view, row, row, pos)
            be.prefix_attention(q, own.view, lens, outs[0], prefix=prefix.view, prefix_len=600)
            be.prefix_attention(drafts, own.view, lens, outs[1], prefix=prefix.view, prefix_len=600)
            be.sample(x, *settings, outs[2])

        with torch.cuda.stream(st):
            step()
        be.synchronize()
        want = [t.clone() for t in outs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step()
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, t) for a, t in zip(want, outs))
        be.synchronize()
    finally:
        be.close()
