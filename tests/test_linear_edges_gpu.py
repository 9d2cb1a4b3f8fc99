"""Linear attention and the single-token steps where it is easy to go wrong:
widths narrower than a vector beside wide ones, infinities and NaN in states,
values and keys, factors far above and below the range of f16, launches at the
limits, and tokens that are views of different buffers.

References and bounds as in test_linear_gpu; where they are narrower here, the
text of the test says why.
"""
import numpy as np
import pytest
import torch

from test_linear_gpu import _cuda, _inputs, _randn, _slopes, check, reference

gpu = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def clef():
    import clef_hip
    clef_hip.lib()
    return clef_hip


# ---------------------------------------------------------------------------- widths
@gpu
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dk,dv", [(100, 5), (12, 4), (4, 13), (33, 3), (3, 33), (127, 1), (1, 127), (128, 2),
                                   (2, 128)])
def test_one_narrow_width(clef, dk, dv, dtype):
    """One width below a 16-byte vector, the other above it and mostly no multiple of one."""
    Hk, Hv, lens = 2, 4, [70, 1, 0, 130]
    T = sum(lens)
    q, k, v = _inputs(dk, T, Hk, Hv, dk, dv, dtype)
    g, init = _slopes(Hv), _randn(5, Hv, dk, dv)
    scan = clef.LinearScan(dk, dv)
    cq, ck, cv, cg, ci = _cuda(q, k, v, g, init)
    out, final = scan.prefill(cq, ck, cv, cg, initial=ci, out_dtype=dtype)
    check(out, final, q, k, v, g, scan.scale, init)
    cu = np.concatenate([[0], np.cumsum(lens)])
    out, final = scan.prefill_varlen(cq, ck, cv, cg, torch.tensor(cu, dtype=torch.int32, device="cuda"), initial=ci,
                                     out_dtype=dtype)
    for s, n in enumerate(lens):
        a = int(cu[s])
        if n:
            check(out[a:a + n], final[s], q[a:a + n], k[a:a + n], v[a:a + n], g, scan.scale, init)
        else:
            assert torch.equal(final[s].cpu(), init)
