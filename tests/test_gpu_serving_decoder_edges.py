"""More of the serving decoder's refusals: misaligned settings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_decoder import B, _weights  # noqa: E402
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
