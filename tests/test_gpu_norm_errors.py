"""GPU test: the norms' entry points report their own launches' errors, and leave an
error that somebody else's call has left behind where it is."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_an_earlier_error_is_not_the_norms(fms):
    L = fms.load_library()
    rt = ctypes.CDLL("libcudart.so.12")  # the copy that torch and the library share
    x = torch.randn(5, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    z, y, dx, dh = (torch.zeros_like(x) for _ in range(4))
    dw = torch.empty_like(w)
    stats = torch.empty(4, 5, device="cuda")
    nb = L.fms_norm_residual_bwd_workspace_size(5, 1, 64)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    want = fms.norm_residual(x, x, w, w)
    p = lambda t: t.data_ptr()  # noqa: E731
    torch.cuda.synchronize()
    s = torch.cuda.current_stream().cuda_stream
    assert rt.cudaSetDevice(10 ** 6) == 101  # no such device
    try:
        fwd = L.fms_norm_residual_fwd(0, 0, 0, p(x), p(x), p(w), None, p(w), None, None, 1, 5, 64, 1e-6, 1.0, p(z),
                                      p(y), p(stats), s)
        bwd = L.fms_norm_residual_bwd(0, 0, 0, p(x), p(x), p(w), None, p(w), None, 1, 5, 64, 1.0, p(stats), p(x), p(x),
                                      p(dx), p(dh), p(dw), None, None, None, None, p(ws), nb, s)
        left = rt.cudaPeekAtLastError()
    finally:
        rt.cudaGetLastError()
    assert (fwd, bwd, left) == (0, 0, 101)
    torch.cuda.synchronize()
    assert torch.equal(z, want[0]) and torch.equal(y, want[1])
