"""More of the serving decoder's refusals: misaligned settings, prefixes of different lengths."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_decoder import B, HD, HKV, NL, _weights  # noqa: E402
from test_gpu_serving_decoder import _decoder  # noqa: E402


def test_misaligned_settings_leave_the_position(um, backend):
    W, _ = _weights(um)
    dec = _decoder(um, backend, W, 4, kv_fmt=um.F16)
    f, i = torch.zeros(B + 1, device="cuda"), torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    good = [f, i, f, f, f, i.clone(), f.clone()]  # temperature, top_k, top_p, min_p, u, next, probs
    tok = np.zeros(B, np.int32)
    try:
        for at in range(len(good)):
            ptrs = [a.data_ptr() + (2 if k == at else 0) for k, a in enumerate(good)]
            st = um.lib.uaii_moe_decoder_step_sampled(dec._h, tok.ctypes.data, *ptrs, None)
            assert st == um.INVALID_ARGUMENT and b"misaligned" in um.lib.uaii_moe_last_error(), at
        assert dec.position == 0
    finally:
        dec.close()


def test_prefixes_of_different_lengths_are_refused(um, backend):
    """A step while the layers hold prefixes of different lengths would give weight to rows that nothing was written to."""
    W, _ = _weights(um)
    dec = _decoder(um, backend, W, 4, kv_fmt=um.KV_I8, prefix_max=9)
    k = um.fill_normal((HKV, 9, HD), 4, 1)
    tok, out = np.zeros(B, np.int32), np.empty(B, np.int32)
    f, i = torch.zeros(B, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    try:
        dec.set_prefix(0, k, k, 9)
        for call in (lambda: dec.step(tok, None, out), lambda: dec.generate(tok, 2, np.empty((2, B), np.int32)),
                     lambda: dec.step_sampled(tok, f, i, f, f, f, i)):
            with pytest.raises(um.UaiiMoeError) as e:
                call()
            assert e.value.status == um.INVALID_ARGUMENT and "prefix" in e.value.message and dec.position == 0
        for l in range(1, NL):
            dec.set_prefix(l, k[:, :5].copy(), k[:, :5].copy(), 5)
        with pytest.raises(um.UaiiMoeError):
            dec.step(tok, None, out)
        dec.set_prefix(0, k[:, :5].copy(), k[:, :5].copy(), 5)
        dec.step(tok, None, out)
        backend.synchronize()
        assert dec.position == 1
    finally:
        dec.close()
