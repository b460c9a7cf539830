"""GPU tests of the AdamW step.  32-bit moments: each value is a few float32
operations, so 8 2^-24 of the magnitudes that enter it bounds its error (and half a
unit of the last place of a 16-bit parameter).  8-bit moments: the codes are those of
the formula evaluated operation by operation in float32, equal bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SHAPES = [(128, 25), (7,), (1,), (255,), (256,), (257,), (3, 1001), (0,), (2, 5, 64), (4096,)]
H = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def make(shapes, P, G, C, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    p = [(0.1 * r(s)).to(P) for s in shapes]
    return p, [(1e-2 * r(s)).to(G) for s in shapes], None if C is None else [t.to(C) for t in p]


def step64(p, g, m, v, t, scale=1.0):
    b1, b2 = H["betas"]
    g = g.double() * scale
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - H["lr"] * H["weight_decay"]) - H["lr"] / (1 - b1 ** t) * m / \
        (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + H["eps"]), m, v


@pytest.mark.parametrize("P,G,C", [(torch.float32, torch.float32, None),
                                   (torch.float32, torch.bfloat16, torch.bfloat16),
                                   (torch.float32, torch.float16, torch.float16),
                                   (torch.bfloat16, torch.bfloat16, None),
                                   (torch.float16, torch.float32, None)])
def test_32_bits_against_64(fms, P, G, C):
    p, g, c = make(SHAPES, P, G, C)
    m, v = ([torch.zeros(t.shape, device="cuda") for t in p] for _ in range(2))
    scale = torch.tensor([0.37], device="cuda")
    for t in (1, 2, 3):
        want = [step64(a.double(), b, x.double(), y.double(), t, float(scale)) for a, b, x, y in zip(p, g, m, v)]
        fms.adamw_step(p, g, m, v, step=t, copies=c, grad_scale=scale, **H)
        for k, (wp, wm, wv) in enumerate(want):
            # v a sum of two positive terms; m can cancel: against its terms
            assert ((v[k].double() - wv).abs() <= 8 * 2.0 ** -24 * wv + 2.0 ** -140).all()
            terms = wm.abs() + 0.2 * g[k].double().abs()
            assert ((m[k].double() - wm).abs() <= 8 * 2.0 ** -24 * terms).all()
            # |update| <= lr m / sqrt(v) <= 4 lr here, its m off by its terms / sqrt(v) < 10
            bound = 8 * 2.0 ** -24 * (wp.abs() + 40 * H["lr"]) + HALF_ULP[P] * 1.01 * wp.abs() + \
                (2.0 ** -25 if P == torch.float16 else 0)
            assert ((p[k].double() - wp).abs() <= bound).all(), (t, k)
            if c is not None:
                assert torch.equal(c[k], p[k].to(C))


MASK = 0xFFFFFFFF


def mix(h):
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & MASK
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & MASK
    return h ^ (h >> 16)


def random16(seed, step, k, n):
    key = mix((mix((seed + step * 0x9E3779B1) & MASK) + k * 0x3C6EF373) & MASK)
    r = mix(torch.arange(n, dtype=torch.int64) ^ key)
    return r & 0xFFFF, r >> 16


def blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)


def encode(x, r16, positive):
    a = blocks(x.abs())
    top = a.amax(1)
    sc = torch.where(top < 1e-30, torch.full_like(top, 1e-30), top) * (1 / 448)
    a = (a * (1.0 / sc)[:, None]).clamp(max=448.0).view(-1)[:x.numel()]
    r16 = r16.int()
    big = ((a.view(torch.int32) + (r16 << 4)) >> 20) - 960
    small = (a * 512.0 + r16.float() * (1.0 / 65536.0)).int()
    k = torch.where(a < 0.015625, small, big).clamp(max=126)
    k = torch.where(x > 0, k.clamp(min=1), k) if positive else k + 128 * (x < 0)
    return k.to(torch.uint8), sc


def decode(codes, sc, n):
    return (blocks(codes.view(-1).cpu().view(torch.float8_e4m3fn).float()) * sc.cpu()[:, None]).view(-1)[:n]


@pytest.mark.parametrize("P,G,C", [(torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32, None),
                                   (torch.bfloat16, torch.bfloat16, None)])
def test_8_bits_operation_by_operation(fms, P, G, C):
    """Codes, scales, parameters and copies equal the formula in float32 on the host."""
    p, g, c = make(SHAPES, P, G, C, 1)
    m, v = ([fms.moments8(t) for t in p] for _ in range(2))
    b1, b2 = H["betas"]
    for t in (1, 2, 3):
        want = []
        for k in range(len(p)):
            n = p[k].numel()
            pk, gk = p[k].cpu().view(-1).float(), g[k].cpu().view(-1).float()
            mk, root = decode(*m[k], n), decode(*v[k], n)
            mk = mk * b1 + gk * (1 - b1)
            vk = (root * root) * b2 + (gk * gk) * (1 - b2)
            root = torch.sqrt(vk.double()).float()  # correctly rounded, which the host's vector sqrt is not
            w = pk * (1.0 - H["lr"] * H["weight_decay"]) - (mk * (H["lr"] / (1 - b1 ** t))) / \
                (root * (1 / math.sqrt(1 - b2 ** t)) + H["eps"])
            rm, rv = random16(77, t, k, n)
            want.append((w.to(P), encode(mk, rm, False), encode(root, rv, True)))
        fms.adamw_step(p, g, m, v, step=t, seed=77, copies=c, **H)
        for k, (w, (mc, ms), (vc, vs)) in enumerate(want):
            assert torch.equal(p[k].cpu().view(-1), w), (t, k)
            assert torch.equal(m[k][0].view(-1).view(torch.uint8).cpu(), mc) and torch.equal(m[k][1].cpu(), ms)
            assert torch.equal(v[k][0].view(-1).view(torch.uint8).cpu(), vc) and torch.equal(v[k][1].cpu(), vs)
            if C is not None:
                assert torch.equal(c[k].cpu().view(-1), w.to(C))


def test_rounding_is_without_bias(fms):
    """The mean over seeds of a code between two neighbours: 256 values, 600 seeds, each
    draw off by half a code step (at most 1/16 of the value) at most; five standard
    errors of that."""
    n, seeds = 256, 600
    x = torch.linspace(0.02, 1.0, n, device="cuda")
    total = torch.zeros(n, device="cuda", dtype=torch.float64)
    for seed in range(seeds):
        p, m, v = torch.zeros(n, device="cuda"), fms.moments8(x), fms.moments8(x)
        fms.adamw_step([p], [x], [m], [v], step=1, seed=seed, betas=(0.0, 0.0))
        total += m[0].double() * m[1].double()
    assert ((total / seeds - x.double()).abs() <= 5 * x.double() / 16 / math.sqrt(seeds) + 1e-6).all()


def test_second_moment_moves(fms):
    """A constant gradient: b2 = 0.999 moves a moment by far less than a code each step,
    and the expectation still follows.  r = sqrt(v) converges to |g|, its codes spread
    by sqrt(step / 2) = 0.25 of it at most for each value; 4096 values."""
    n, steps = 4096, 3000
    g = torch.full((n,), 0.5, device="cuda")
    g[::256] = 1.0  # each block's largest, so that the others lie inside the codes
    p, m, v = torch.zeros(n, device="cuda"), fms.moments8(g), fms.moments8(g)
    for t in range(1, steps + 1):
        fms.adamw_step([p], [g], [m], [v], step=t, lr=0.0, seed=5)
    r = v[0].float() * v[1].repeat_interleave(256)
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[::256] = False
    want = 0.5 * math.sqrt(1 - 0.999 ** steps)
    # the square is what is averaged, so the root's own mean lies below by its spread
    assert abs(float((r[rest] ** 2).mean()) ** 0.5 / want - 1) < 0.1


def test_both_widths_train_alike(fms):
    """A least-squares problem: 8-bit moments end near where 32-bit ones do."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    A = torch.randn(2048, 64, generator=gen, device="cuda")
    X = torch.randn(64, 32, generator=gen, device="cuda")
    Y = A @ X + 0.1 * torch.randn(2048, 32, generator=gen, device="cuda")
    loss = {}
    for bits in (32, 8):
        W = torch.zeros(64, 32, device="cuda", requires_grad=True)
        opt = fms.AdamW([W], lr=2e-2, weight_decay=0.0, bits=bits)
        for _ in range(400):
            opt.zero_grad()
            out = (A @ W - Y).pow(2).mean()
            out.backward()
            opt.step()
        loss[bits] = float(out.detach())
    assert loss[32] < 0.0102 and loss[8] < 0.0102 * 1.1


def test_optimizer_object(fms):
    """A parameter without a gradient is left alone and counts its own steps; the state
    is saved and taken up again."""
    p, g, _ = make([(300,), (40, 8)], torch.float32, torch.float32, None, 4)
    for bits in (32, 8):
        a = [t.clone().requires_grad_() for t in p]
        opt = fms.AdamW(a, bits=bits, seed=1, **H)
        opt.step([g[0], None])
        assert torch.equal(a[1], p[1]) and opt.exp_avgs[1] is None
        opt.step([g[0], g[1]])
        assert opt.steps == [2, 1]
        other = fms.AdamW([t.detach().clone() for t in a], bits=bits, seed=1, **H)
        other.load_state_dict({k: ([tuple(u.clone() for u in s) if bits == 8 else s.clone() for s in v]
                                   if k.startswith("exp") else v) for k, v in opt.state_dict().items()})
        opt.step([g[0], g[1]])
        other.step([g[0], g[1]])
        assert all(torch.equal(x, y) for x, y in zip(a, other.params))
        with pytest.raises(fms.ArgumentError):
            fms.AdamW(a, bits=40 - bits).load_state_dict(opt.state_dict())


def test_views_off_alignment_and_repeats(fms):
    """Tensors that start anywhere in a flat buffer give what aligned ones do."""
    for bits in (32, 8):
        p, g, c = make(SHAPES, torch.float32, torch.bfloat16, torch.bfloat16, 5)
        state = lambda t: fms.moments8(t) if bits == 8 else torch.zeros(t.shape, device="cuda")  # noqa: E731
        m, v = [state(t) for t in p], [state(t) for t in p]

        def shifted(t):
            return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

        p2, g2, c2 = [shifted(t) for t in p], [shifted(t) for t in g], [shifted(t) for t in c]
        m2, v2 = ([tuple(shifted(u) for u in state(t)) if bits == 8 else shifted(state(t)) for t in p] for _ in range(2))
        for t in (1, 2):
            fms.adamw_step(p, g, m, v, step=t, copies=c, seed=3, **H)
            fms.adamw_step(p2, g2, m2, v2, step=t, copies=c2, seed=3, **H)
        flat = lambda s: [u for t in s for u in (t if isinstance(t, tuple) else (t,))]  # noqa: E731
        for a, b in zip(p + c + flat(m) + flat(v), p2 + c2 + flat(m2) + flat(v2)):
            assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a,
                               b.view(torch.uint8) if b.element_size() == 1 else b)


def test_many_tensors(fms):
    """More tensors than one launch's table holds."""
    n = 900
    p = [torch.full((1 + k % 7,), float(k), device="cuda") for k in range(n)]
    g = [torch.full_like(t, 1.0) for t in p]
    m, v = ([torch.zeros_like(t) for t in p] for _ in range(2))
    fms.adamw_step(p, g, m, v, step=1, lr=0.5, weight_decay=0.0, eps=0.0)
    for k in range(n):
        assert torch.allclose(p[k], torch.full_like(p[k], k - 0.5), rtol=1e-6, atol=1e-6)


def test_not_a_number_is_kept(fms):
    """A NaN gradient reaches its parameter and shows in its block's moments, not beyond."""
    for bits in (32, 8):
        p, g = torch.ones(600, device="cuda"), torch.full((600,), 0.1, device="cuda")
        g[300] = float("nan")
        m, v = (fms.moments8(p) if bits == 8 else torch.zeros_like(p) for _ in range(2))
        fms.adamw_step([p], [g], [m], [v], step=1)
        assert torch.isnan(p[300]) and torch.isfinite(p).sum() == 599
        if bits == 8:
            assert torch.isnan(m[1]).tolist() == [False, True, False]
        else:
            assert torch.isnan(m).sum() == 1


def test_autograd_sees_the_update(fms):
    w = torch.ones(4, device="cuda", requires_grad=True)
    y = (w * w).sum()
    fms.adamw_step([w], [torch.ones(4, device="cuda")], [torch.zeros(4, device="cuda")],
                   [torch.zeros(4, device="cuda")], step=1)
    with pytest.raises(RuntimeError):  # w was needed and has been changed in place
        y.backward()


def test_another_stream(fms):
    p, g, _ = make(SHAPES, torch.float32, torch.float32, None, 6)
    q = [t.clone() for t in p]
    m, v, m2, v2 = ([torch.zeros_like(t) for t in p] for _ in range(4))
    fms.adamw_step(p, g, m, v, step=1, **H)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fms.adamw_step(q, g, m2, v2, step=1, **H)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(p, q))


def test_refusals(fms):
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    p, g, m, v = z(8), z(8), z(8), z(8)
    e = fms.moments8(p)
    A, D = fms.ArgumentError, fms.DimensionMismatch
    call = fms.adamw_step
    for err, f in [(D, lambda: call([p], [], [m], [v], step=1)),
                   (D, lambda: call([p], [z(9)], [m], [v], step=1)),
                   (D, lambda: call([p], [g], [z(7)], [v], step=1)),
                   (D, lambda: call([p], [g], [(e[0], z(2))], [e], step=1)),
                   (A, lambda: call([p], [g], [m], [v], step=0)),
                   (A, lambda: call([p], [g], [m], [v], step=1, betas=(1.0, 0.9))),
                   (A, lambda: call([p], [g], [m], [v], step=1, eps=-1e-8)),
                   (A, lambda: call([p], [g], [m.half()], [v], step=1)),
                   (A, lambda: call([p], [g], [m], [e], step=1)),
                   (A, lambda: call([p], [g], [(e[0].float(), e[1])], [e], step=1)),
                   (A, lambda: call([p.double()], [g], [m], [v], step=1)),
                   (A, lambda: call([z(16)[::2]], [g], [m], [v], step=1)),
                   (A, lambda: call([p], [g.cpu()], [m], [v], step=1)),
                   (A, lambda: call([p], [g], [m], [v], step=1, copies=[z(8)])),
                   (A, lambda: call([p], [g], [m], [v], step=1, grad_scale=z(2))),
                   (A, lambda: fms.AdamW([p], bits=16))]:
        with pytest.raises(err):
            f()
    call([], [], [], [], step=1)
