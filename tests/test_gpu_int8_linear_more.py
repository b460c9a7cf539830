"""GPU tests of the INT8 linear layer: gradients it does not have are refused whatever the
features are, and its own quantiser beside the index's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_bias_that_wants_a_gradient_is_refused(fms):
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(4, 32, generator=gen, device="cuda")
    w = fms.quantize_int8_symmetric(torch.randn(16, 32, generator=gen, device="cuda"))
    b = torch.randn(16, generator=gen, device="cuda").requires_grad_()
    for features in (x, fms.quantize_int8_symmetric(x)):
        with pytest.raises(fms.ArgumentError, match="forward-only"):
            fms.int8_linear(features, w, bias=b)
        with torch.no_grad():
            y = fms.int8_linear(features, w, bias=b)
        assert torch.equal(y, fms.int8_linear(features, w, bias=b.detach()))
    trained = fms.Int8Index(w.codes, w.scales.clone().requires_grad_())
    for features, weight in ((x, trained), (trained, w)):
        with pytest.raises(fms.ArgumentError, match="forward-only"):
            fms.int8_linear(features, weight)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,out", [(1, 768, 64), (7, 129, 40), (300, 768, 128), (2000, 100, 33)])
def test_beside_the_index_of_the_same_features(fms, dtype, rows, dim, out):
    """The layer's scale is absmax times fl(1/127), the index's absmax / 127: three roundings
    apart at most, 3 2^-24 of it.  A code can differ, by one, only where x / scale lies within
    as much of its size of a half; each such code moves an output by one weight code."""
    gen = torch.Generator(device="cuda").manual_seed(rows + dim)
    x = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    w = fms.quantize_int8_symmetric(torch.randn(out, dim, generator=gen, device="cuda"))
    q = fms.quantize_int8_symmetric(x.float())
    a = fms.int8_linear(x, w, out_dtype=torch.float32).double()
    b = fms.int8_linear(q, w).double()
    t = (x.double() / q.scales.double()[:, None]).abs()
    doubtful = ((t - torch.floor(t) - 0.5).abs() <= 127 * 5 * 2.0 ** -24).double()
    unit = q.scales.double()[:, None] * w.scales.double()[None, :]
    # the sums in units of the last place: 3 for the scales, 3 for the products of either side
    bound = (doubtful @ w.codes.double().abs().T) * unit * 1.001 + 9 * 2.0 ** -24 * b.abs()
    assert ((a - b).abs() <= bound).all()
