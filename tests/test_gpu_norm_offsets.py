"""GPU tests of the layer norm on rows whose values lie far from zero and close together
(constant rows are what padding gives): the mean has to come off before the reciprocal
deviation, up to 1 / sqrt(eps), goes on."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DIMS = [1, 2, 40, 257, 768, 1000, 1024, 1536, 5120, 8200, 16384]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("eps", [1e-6, 1e-5])
def test_constant_rows(fms, dtype, dim, eps):
    """Constants of eight bits: every partial sum of a row is exact, so is the mean, and the
    norm of the row is its bias."""
    c = torch.tensor([0.0, 1.0, -3.0, 100.0, 1016.0, -2.0 ** 15, 0.0078125, 51200.0, 89.0], device="cuda")
    rows = c[:, None].expand(-1, dim).to(dtype).contiguous()
    ones = torch.ones(dim, device="cuda", dtype=dtype)
    z, y = fms.norm_residual(rows, rows.flip(0).contiguous(), ones, ones, kind="layer", eps=eps)
    assert torch.equal(z, rows) and not y.any()
    b = torch.linspace(-1, 1, dim, device="cuda").to(dtype)
    z, y = fms.norm_residual(torch.zeros_like(rows), rows, ones, ones, b_post=b, b_pre=b, kind="layer", eps=eps)
    assert torch.equal(z, b.expand_as(rows))
    z, y = fms.norm_residual(rows, rows, ones, ones, b_pre=b, kind="layer", eps=eps)
    assert torch.equal(y, b.expand_as(rows))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("eps", [1e-6, 1e-5])
def test_gradients_of_constant_rows(fms, dtype, dim, eps):
    """Normalised values of zero: the weights' gradients are zero, and the rows' are the
    centred cotangents times 1 / sqrt(eps): float32 sums of `dim` terms near one, against
    (dim + 16) 2^-24, and half a unit of the last place."""
    gen = torch.Generator(device="cuda").manual_seed(dim)
    c = torch.tensor([100.0, 1016.0, -2.0 ** 15, 89.0, 7.0], device="cuda")
    x = c[:, None].expand(-1, dim).to(dtype).contiguous().requires_grad_()
    h = x.detach().flip(0).contiguous().requires_grad_()
    wp, wq = (torch.ones(dim, device="cuda", dtype=dtype).requires_grad_() for _ in range(2))
    dz, dy = (torch.randn(5, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    out = fms.norm_residual(x, h, wp, wq, kind="layer", eps=eps)
    dx, dh, dwp, dwq = torch.autograd.grad(out, (x, h, wp, wq), (dz, dy))
    assert not dwp.any() and not dwq.any()
    centre = lambda v: v - v.mean(-1, keepdim=True)  # noqa: E731
    r = eps ** -0.5
    hu = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    want = dz.double() + r * centre(dy.double())
    tol = (dim + 16) * 2.0 ** -24 * 6
    assert ((dx.double() - want).abs() <= r * tol + hu * 1.01 * want.abs()).all()
    want = r * centre(want)
    assert ((dh.double() - want).abs() <= 2 * r * r * tol + hu * 1.01 * want.abs()).all()
