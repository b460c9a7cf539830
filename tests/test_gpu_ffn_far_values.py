"""GPU tests of the gated feed-forward block's activations far from zero, one product per
value (dim 1), so that g and u are exact: there an activation is its argument or zero and
its derivative one or zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FAR = [40.0, 1e3, 3e4, 1e6, 2.0 ** 25, 1e9, 1e12, 1e14, 1e20, 1e30]


def grads(fms, x, wg, wu, act):
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    h = fms.gated_ffn(*leaves, act=act)
    return (h.detach(), *torch.autograd.grad(h, leaves, torch.ones_like(h)))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_derivative_is_one_or_zero(fms, act):
    """x = 1 and w_up = 1: dw_gate is the derivative itself, dw_up the activation; at -40 both
    are below 40 e^-40 < 1e-15."""
    wg = torch.tensor([s * v for v in FAR for s in (1, -1)], device="cuda").bfloat16()[:, None]
    one = torch.ones_like(wg)
    h, dx, dg, du = grads(fms, one[:1], wg, one, act)
    on = (wg > 0).to(wg.dtype)
    for got, want in ((h.T, wg * on), (dg, on), (du, wg * on)):
        assert ((got.double() - want.double()).abs() <= 1e-15).all()
    # dx adds dg w_gate + du w_up over the columns: the largest counts, the others are below its rounding
    assert dx.item() == pytest.approx(2 * float((wg * on).double().sum()), rel=2.0 ** -7)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_derivative_of_thousands_in_float16(fms, act):
    """g between 1e3 and 8e4 with a fraction: dw_gate = x dg with dg = u rounded to float16,
    two roundings of half a unit (2^-11) and 2^-18 for the derivative."""
    x = torch.tensor([[1.3701]], device="cuda").half()
    wg = torch.logspace(3, 4.78, 200, device="cuda").half()[:, None]
    wu = torch.full_like(wg, 0.731)
    _, _, dg, _ = grads(fms, x, wg, wu, act)
    want = float(x.double()) ** 2 * wu.double()
    assert ((dg.double() - want).abs() <= (2 * 2.0 ** -11 + 2.0 ** -18) * 1.001 * want).all()
