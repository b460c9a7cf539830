"""The token-encoder operators on tensors of more than 2^31 values: the last rows, whose
offsets pass 32 bits, equal those of a call on these rows alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _room():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    yield
    torch.cuda.empty_cache()


def tail(t, n=300):
    return t[-n:].contiguous()


def test_gated_ffn(fms):
    rows, dim, hidden = 1_060_001, 64, 2048
    x = torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16)
    wg, wu = (torch.randn(hidden, dim, device="cuda").bfloat16() / 8 for _ in range(2))
    h = fms.gated_ffn(x, wg, wu)
    assert h.numel() > 2 ** 31
    # the same sums in the same order, whatever the tile
    assert torch.equal(tail(h), fms.gated_ffn(tail(x), wg, wu)) and torch.equal(h[:300], fms.gated_ffn(x[:300], wg, wu))


def test_norm_residual(fms):
    rows, dim = 2_900_003, 768
    x = torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16)
    h = torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(dim, device="cuda").bfloat16()
    leaf = x.requires_grad_()
    z, y = fms.norm_residual(leaf, h, w, w, kind="layer")
    assert z.numel() > 2 ** 31
    dz = torch.zeros_like(z)
    dz[-300:] = 1.0
    dx, = torch.autograd.grad(z, leaf, dz)
    xs, hs = tail(x.detach()).requires_grad_(), tail(h)
    zs, ys = fms.norm_residual(xs, hs, w, w, kind="layer")
    assert torch.equal(tail(z), zs) and torch.equal(tail(y), ys)
    assert torch.equal(tail(dx), torch.autograd.grad(zs, xs, torch.ones_like(zs))[0])
    assert not dx[:300].any()


def test_int8_linear(fms):
    rows, dim, out = 1_060_001, 64, 2048
    x = torch.randn(rows, dim, device="cuda", dtype=torch.float16)
    w = fms.quantize_int8_symmetric(torch.randn(out, dim, device="cuda"))
    y = fms.int8_linear(x, w)
    assert y.numel() > 2 ** 31
    assert torch.equal(tail(y), fms.int8_linear(tail(x), w))


def test_adamw(fms):
    n = 2 ** 31 + 1001
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    g[-3:] = -0.25
    m, v = fms.moments8(p), fms.moments8(p)
    fms.adamw_step([p], [g], [m], [v], step=1, lr=1.0, weight_decay=0.0, eps=0.0)
    # the first step is lr times the gradient's sign
    assert p[-4:].tolist() == [-1.0, 1.0, 1.0, 1.0] and p[:3].tolist() == [-1.0] * 3 and float(p[2 ** 31]) == -1.0
    # past 2^32 the random bits take the value's high word: here the codes of the last block
    assert float(m[0][-1].float() * m[1][-1]) == pytest.approx(-0.025, rel=0.13)
    assert float(v[0][2 ** 31].float() * v[1][2 ** 31 // 256]) == pytest.approx(0.5 * 0.001 ** 0.5, rel=1e-5)
