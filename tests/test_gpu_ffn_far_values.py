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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 40])
def test_the_small_side_of_gelu(fms, dtype, rows):
    """g from -12.5 to 0 and to 4, where Phi(g) falls to 4e-36: h and the derivative are right
    relative to their own size.  2^-13 of Phi(g) covers the fit's 6.1e-5 with the float32
    roundings around it, against half a unit of the last place (float16: of its smallest)."""
    wg = torch.cat([torch.linspace(-12.5, 0, 400, device="cuda"), torch.linspace(0, 4, 100, device="cuda")]).to(dtype)[:, None]
    one = torch.ones_like(wg)
    x = torch.zeros(rows, 1, device="cuda", dtype=dtype)
    x[-1] = 1
    leaf = wg.clone().requires_grad_()
    h = fms.gated_ffn(x, leaf, one, act="gelu")
    dh = torch.zeros_like(h)
    dh[-1] = 1
    dg, = torch.autograd.grad(h, leaf, dh)
    g = wg.double()[:, 0]
    ndtr = lambda v: 0.5 * torch.erfc(-v * 0.5 ** 0.5)  # noqa: E731  (torch's own is 1 + erf: nothing below 1e-16)
    cdf, slope = ndtr(g), g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    hu, tiny = (2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -8, 2.0 ** -134)
    near = torch.minimum(cdf, ndtr(-g))
    for got, want, size in ((h[-1], g * cdf, g.abs() * near), (dg[:, 0], cdf + slope, near + slope.abs())):
        off = (got.double() - want).abs() - (2.0 ** -13 * size + 2.0 ** -20 * want.abs() + hu * 1.01 * want.abs() + tiny)
        assert not (off > 0).any(), (g[off > 0], got[off > 0], want[off > 0])
