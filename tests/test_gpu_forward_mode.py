"""GPU test: a tensor that carries a forward-mode tangent is refused, not computed on
without its tangent."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def calls(fms):
    r = lambda *s, dtype=torch.float16: torch.randn(*s, device="cuda").to(dtype)  # noqa: E731
    x, w, v = r(6, 16), r(8, 16), r(16)
    index = fms.quantize_int8_symmetric(r(8, 16, dtype=torch.float32))
    q, d = r(2, 4, 16), r(2, 5, 16)
    return {"gated_ffn": (lambda x, w: fms.gated_ffn(x, w, w), [x, w]),
            "norm_residual": (lambda x, h, v: fms.norm_residual(x, h, v, v), [x, r(6, 16), v]),
            "norm_residual gate": (lambda g: fms.norm_residual(x, x, v, v, gate=g), [v]),
            "int8_linear": (lambda x, b: fms.int8_linear(x, index, bias=b), [x, r(8)]),
            "maxsim": (lambda q, d: fms.maxsim(q, d), [q, d])}


@pytest.mark.parametrize("name", ["gated_ffn", "norm_residual", "norm_residual gate", "int8_linear", "maxsim"])
def test_dual_tensors_are_refused(fms, name):
    f, args = calls(fms)[name]
    f(*args)
    with forward_ad.dual_level():
        f(*args)  # no tangent: as ever
        for k in range(len(args)):
            dual = list(args)
            dual[k] = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(fms.ArgumentError, match="forward"):
                f(*dual)
            with torch.no_grad(), pytest.raises(fms.ArgumentError, match="forward"):
                f(*dual)
    f(*args)
