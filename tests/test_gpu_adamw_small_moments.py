"""GPU tests of the AdamW step with second moments near and below float32's smallest
normal value (gradients of 1e-22 to 1e-15): the square root of a small moment decides the
whole step when eps is zero."""
import math

import pytest
import torch

from test_gpu_adamw import decode, encode, random16

pytestmark = pytest.mark.gpu


def test_32_bits(fms):
    """Moments that halve exactly (b1 = b2 = 1/2, zero gradients), so that the new second
    moment is a float32 value known in advance; lr 1, eps 0, parameters zero.  The step is
    then -2 m / (sqrt(v) sqrt 2): a root, two products and a quotient in float32, each off by
    2^-24 at most, against 8 2^-24."""
    v = torch.logspace(-44.8, -29, 4096, dtype=torch.float64).float()
    m = (v.double().sqrt() * torch.linspace(-3, 3, 4096, dtype=torch.float64)).float()
    p, g = torch.zeros(4096, device="cuda"), torch.zeros(4096, device="cuda")
    m2, v2 = (2 * m).cuda(), (2 * v).cuda()
    fms.adamw_step([p], [g], [m2], [v2], step=1, lr=1.0, betas=(0.5, 0.5), eps=0.0, weight_decay=0.0)
    assert torch.equal(m2.cpu(), m) and torch.equal(v2.cpu(), v)
    want = -2 * m.double() / (v.double().sqrt() * math.sqrt(2))
    off = (p.cpu().double() - want).abs() / want.abs()
    assert off.max() <= 8 * 2.0 ** -24, f"{int((off > 8 * 2.0 ** -24).sum())} outside, worst {off.max()}"


def test_8_bits(fms):
    """The first step of moments in 8 bits: codes and scales equal the formula evaluated
    operation by operation in float32, the parameter moves by lr in the gradient's direction
    (b1 = b2 = 0: m = g, v = g g, whose own rounding below 1e-38 is up to 2^-149 of v)."""
    gen = torch.Generator().manual_seed(1)
    g = torch.cat([10.0 ** e * (1 + torch.rand(256, generator=gen)) * torch.sign(torch.randn(256, generator=gen))
                   for e in (-22, -21, -20, -19.5, -19, -18, -17, -16, -15)])
    n = g.numel()
    p = torch.zeros(n, device="cuda")
    m, v = fms.moments8(p), fms.moments8(p)
    fms.adamw_step([p], [g.cuda()], [m], [v], step=1, seed=9, lr=0.5, betas=(0.0, 0.0), eps=0.0, weight_decay=0.0)
    square = g * g
    root = torch.sqrt(square.double()).float()
    rm, rv = random16(9, 1, 0, n)
    for got, x, r, positive in ((m, g, rm, False), (v, root, rv, True)):
        codes, scales = encode(x, r, positive)
        assert torch.equal(got[1].cpu(), scales)
        assert torch.equal(got[0].view(torch.uint8).cpu(), codes)
        assert torch.isfinite(decode(*got, n)).all()
    want = -0.5 * g.double() / root.double()
    assert ((p.cpu().double() - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()


def test_zeros_beside_small_ones(fms):
    """Values that have never had a gradient beside tiny ones: with an eps they stay where
    they are, the others take the formula's step."""
    for bits in (32, 8):
        g = torch.zeros(1024)
        g[::3] = 1e-20
        p = torch.ones(1024, device="cuda")
        m, v = (fms.moments8(p) if bits == 8 else torch.zeros_like(p) for _ in range(2))
        fms.adamw_step([p], [g.cuda()], [m], [v], step=1, lr=0.25, betas=(0.0, 0.0), eps=1e-20, weight_decay=0.0)
        want = 1 - 0.25 * g.double() / ((g * g).double().sqrt() + 1e-20)
        assert ((p.cpu().double() - want).abs() <= 4 * 2.0 ** -24).all()
        assert (p.cpu()[g == 0] == 1).all()
