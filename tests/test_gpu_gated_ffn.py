"""GPU tests of the gated feed-forward block against its formulas in 64 bits.

The bounds are elementwise and follow the arithmetic: a float32 sum of K products
is off by at most K 2^-24 times the sum of their magnitudes, the activations by
2^-18 relative plus 2^-22 absolute (fast exponentials, error function), each
rounding to the features' type by half a unit of its last place."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def act64(g, act):
    """a(g), a'(g) in 64 bits."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    if act == "gelu":
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def make(rows, dim, hidden, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    sd = 1 / math.sqrt(max(dim, 1))
    return (r(rows, dim).to(dtype), (r(hidden, dim) * sd).to(dtype), (r(hidden, dim) * sd).to(dtype),
            r(rows, hidden).to(dtype))


def reference(x, wg, wu, dh, act):
    """Values and elementwise error bounds of h, dx, dw_gate, dw_up."""
    T = x.dtype
    hu, tiny = HALF_ULP[T], TINY[T]
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    K = x.shape[1]
    acc = lambda n: (n + 2) * 2.0 ** -24  # noqa: E731
    g, u = x @ wg.T, x @ wu.T
    eg, eu = acc(K) * (x.abs() @ wg.abs().T), acc(K) * (x.abs() @ wu.abs().T)
    a, da = act64(g, act)
    # |a'| <= 1.13 and |a''| <= 1.2 for these (relu: a' jumps at 0, inputs avoid it)
    ea = 1.13 * eg + a.abs() * 2.0 ** -18 + 2.0 ** -22 * (1 + g.abs())
    eda = (0 if act == "relu" else 1.2) * eg + da.abs() * 2.0 ** -18 + 2.0 ** -22 * (1 + g.abs())
    h = a * u
    eh = ea * u.abs() + (a.abs() + ea) * eu
    out = {"h": (h, eh + hu * (h.abs() + eh) + tiny)}
    dg, du = dh * u * da, dh * a
    edg = dh.abs() * (eda * (u.abs() + eu) + da.abs() * eu) * 1.01
    edu = dh.abs() * ea * 1.01
    edg = edg + hu * (dg.abs() + edg) + tiny
    edu = edu + hu * (du.abs() + edu) + tiny

    def product(pairs):
        v = sum(p @ q for p, _, q in pairs)
        n = sum(p.shape[1] for p, _, _ in pairs)
        e = sum(ep @ q.abs() + acc(n) * ((p.abs() + ep) @ q.abs()) for p, ep, q in pairs)
        return v, e + hu * (v.abs() + e) + tiny

    out["dx"] = product([(dg, edg, wg), (du, edu, wu)])
    out["dw_gate"] = product([(dg.T, edg.T, x)])
    out["dw_up"] = product([(du.T, edu.T, x)])
    return out


def check(got, ref):
    for name, t in got.items():
        v, bound = ref[name]
        assert t.shape == v.shape, name
        off = (t.double() - v).abs() - bound
        assert not (off > 0).any() and torch.isfinite(t).all(), \
            f"{name}: {int((off > 0).sum())} of {t.numel()} outside their bound, worst by {off.max()}"


def run_all(fms, x, wg, wu, dh, act):
    leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu)]
    h = fms.gated_ffn(*leaves, act=act)
    d = torch.autograd.grad(h, leaves, dh)
    return {"h": h.detach(), "dx": d[0], "dw_gate": d[1], "dw_up": d[2]}


SIZES = [(1, 1, 1), (1, 768, 256), (2, 8, 5), (7, 33, 130), (8, 64, 64), (9, 100, 65), (17, 72, 257), (64, 256, 8),
         (129, 128, 128), (130, 129, 127), (300, 264, 520), (513, 768, 136), (33, 1000, 300)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,hidden", SIZES)
def test_against_64_bits(fms, dtype, rows, dim, hidden):
    x, wg, wu, dh = make(rows, dim, hidden, dtype, rows + dim)
    got = run_all(fms, x, wg, wu, dh, "silu")
    check(got, reference(x, wg, wu, dh, "silu"))
    # without gradients the same values
    assert torch.equal(fms.gated_ffn(x, wg, wu), got["h"])


# Enough tiles for pairs of SMs, at widths that end inside a tile, inside a store's 64
# columns and off 16 bytes; few rows and many columns, whose input gradient is summed in
# parts; many rows and few columns, whose weights' gradients are.
TILES = [(1500, 64, 1500), (900, 72, 2603), (1020, 136, 1067), (1301, 201, 1800), (100, 264, 2048), (2049, 72, 1161),
         (9000, 40, 70), (700, 1000, 1601)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,hidden", TILES)
def test_tiles_against_64_bits(fms, dtype, rows, dim, hidden):
    x, wg, wu, dh = make(rows, dim, hidden, dtype, rows + hidden)
    check(run_all(fms, x, wg, wu, dh, "gelu"), reference(x, wg, wu, dh, "gelu"))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_activations_in_tiles(fms, act):
    x, wg, wu, dh = make(1030, 64, 1600, torch.float16, 17)
    x = (x.float() * 4).to(x.dtype)
    check(run_all(fms, x, wg, wu, dh, act), reference(x, wg, wu, dh, act))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("rows", [1, 5, 140])
def test_activations(fms, act, rows):
    x, wg, wu, dh = make(rows, 96, 72, torch.bfloat16, 3)
    if rows == 140:
        x = (x.float() * 6).to(x.dtype)  # far into both tails
    check(run_all(fms, x, wg, wu, dh, act), reference(x, wg, wu, dh, act))


def test_many_rows_for_the_weights(fms):
    """A long sum over rows: the weights' gradients, which several tiles share."""
    x, wg, wu, dh = make(5000, 72, 136, torch.bfloat16, 5)
    check(run_all(fms, x, wg, wu, dh, "gelu"), reference(x, wg, wu, dh, "gelu"))


def test_repeats_bit_for_bit(fms):
    x, wg, wu, dh = make(3001, 136, 264, torch.float16, 6)
    a, b = run_all(fms, x, wg, wu, dh, "silu"), run_all(fms, x, wg, wu, dh, "silu")
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_gradient_against_differences(fms):
    """Along one direction in every input: the central difference of sum(dh * h).

    A 16-bit h is off by its rounding alone; those errors, taken as independent,
    give the noise of the quotient, and the 64-bit difference at the same step
    gives its curvature."""
    x, wg, wu, dh = make(200, 96, 136, torch.float16, 8)
    got = run_all(fms, x, wg, wu, dh, "silu")
    step = 2.0 ** -5
    gen = torch.Generator(device="cuda").manual_seed(9)
    for k, name in enumerate(("dx", "dw_gate", "dw_up")):
        base = [x, wg, wu]
        v = torch.randn(base[k].shape, generator=gen, device="cuda") * base[k].float().std()
        up, down = list(base), list(base)
        up[k], down[k] = (base[k].float() + step * v).half(), (base[k].float() - step * v).half()
        move = up[k].double() - down[k].double()
        value = lambda t: float((dh.double() * fms.gated_ffn(*t).double()).sum())  # noqa: E731

        def value64(t):
            a, _ = act64(t[0].double() @ t[1].double().T, "silu")
            return float((dh.double() * a * (t[0].double() @ t[2].double().T)).sum())

        quotient = value(up) - value(down)
        slope = float((got[name].double() * move).sum())
        bent = abs(value64(up) - value64(down) - float((reference(x, wg, wu, dh, "silu")[name][0] * move).sum()))
        noise = 2.0 ** -11 * float((dh.double() * got["h"].double()).norm()) * math.sqrt(2) * 5
        rounded = 2.0 ** -11 * float((got[name].double() * move).norm()) * 2 * 5
        assert abs(quotient - slope) <= bent + noise + rounded, (name, quotient, slope, bent, noise)


def test_layouts_and_shapes(fms):
    x, wg, wu, dh = make(24, 64, 48, torch.bfloat16, 10)
    h = fms.gated_ffn(x, wg, wu)
    # leading dimensions
    assert torch.equal(fms.gated_ffn(x.view(2, 3, 4, 64), wg, wu), h.view(2, 3, 4, 48))
    assert torch.equal(fms.gated_ffn(x[0], wg, wu), fms.gated_ffn(x[:1], wg, wu)[0])
    # strided features, transposed weights, a start that is off 16 bytes
    wide = torch.empty(24, 130, dtype=x.dtype, device="cuda")
    wide[:, 1:129:2] = x
    assert torch.equal(fms.gated_ffn(wide[:, 1:129:2], wg, wu), h)
    assert torch.equal(fms.gated_ffn(x, wg.T.contiguous().T, wu), h)
    off = torch.empty(24 * 64 + 1, dtype=x.dtype, device="cuda")[1:].view(24, 64)
    off.copy_(x)
    got = run_all(fms, off, wg, wu, dh, "silu")
    check(got, reference(x, wg, wu, dh, "silu"))
    # a cotangent that is a broadcast
    leaf = x.clone().requires_grad_()
    fms.gated_ffn(leaf, wg, wu).sum().backward()
    one = run_all(fms, x, wg, wu, torch.ones_like(dh), "silu")
    assert torch.equal(leaf.grad, one["dx"])


def test_empty(fms):
    for rows, dim, hidden in ((0, 16, 8), (4, 16, 0), (4, 0, 8)):
        x, wg, wu, dh = make(rows, dim, hidden, torch.bfloat16)
        got = run_all(fms, x, wg, wu, dh, "silu")
        assert got["h"].shape == (rows, hidden) and not got["h"].any()
        assert got["dx"].shape == x.shape and not got["dx"].any()
        assert got["dw_gate"].shape == wg.shape and not got["dw_gate"].any() and not got["dw_up"].any()


def test_only_wanted_gradients(fms):
    x, wg, wu, dh = make(40, 64, 72, torch.bfloat16, 11)
    ref = run_all(fms, x, wg, wu, dh, "silu")
    for k, name in enumerate(("dx", "dw_gate", "dw_up")):
        t = [x.clone(), wg.clone(), wu.clone()]
        t[k].requires_grad_()
        fms.gated_ffn(*t).backward(dh)
        assert torch.equal(t[k].grad, ref[name])


@pytest.mark.parametrize("rows", [3, 200])
def test_not_a_number_stays_in_its_rows(fms, rows):
    x, wg, wu, _ = make(rows, 80, 96, torch.float16, 12)
    clean = fms.gated_ffn(x, wg, wu)
    x[1, 7] = float("nan")
    x[2, 3] = float("inf")
    h = fms.gated_ffn(x, wg, wu)
    assert torch.isnan(h[1]).all() and not torch.isfinite(h[2]).any()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    assert torch.equal(h[keep], clean[keep])


def test_another_stream(fms):
    x, wg, wu, dh = make(700, 128, 192, torch.bfloat16, 13)
    ref = run_all(fms, x, wg, wu, dh, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_all(fms, x, wg, wu, dh, "silu")
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(got[k], ref[k]) for k in ref)


def test_a_thread_without_a_context(fms):
    """A new host thread, memory from torch's cache: the call is the thread's first of CUDA."""
    import threading
    x, wg, wu, _ = make(700, 128, 192, torch.bfloat16, 16)
    ref = fms.gated_ffn(x, wg, wu)
    spare = [torch.empty_like(ref), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")]  # noqa: F841
    torch.cuda.synchronize()
    del spare
    got = []

    def work():
        try:
            got.append(fms.gated_ffn(x, wg, wu))
        except Exception as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert isinstance(got[0], torch.Tensor), got[0]
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref)


def test_in_a_cuda_graph(fms):
    x, wg, wu, _ = make(65, 128, 192, torch.bfloat16, 14)
    fms.gated_ffn(x, wg, wu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = fms.gated_ffn(x, wg, wu)
    x.copy_(make(65, 128, 192, torch.bfloat16, 15)[0])
    graph.replay()
    assert torch.equal(h, fms.gated_ffn(x, wg, wu))


def test_refusals(fms):
    x, wg, wu, _ = make(4, 16, 8, torch.bfloat16)
    bad = [(fms.ArgumentError, lambda: fms.gated_ffn(x, wg, wu, act="tanh")),
           (fms.ArgumentError, lambda: fms.gated_ffn(x.float(), wg.float(), wu.float())),
           (fms.ArgumentError, lambda: fms.gated_ffn(x, wg.half(), wu)),
           (fms.ArgumentError, lambda: fms.gated_ffn(x, wg.cpu(), wu)),
           (fms.DimensionMismatch, lambda: fms.gated_ffn(x[:, :8], wg, wu)),
           (fms.DimensionMismatch, lambda: fms.gated_ffn(x, wg, wu[:4])),
           (fms.DimensionMismatch, lambda: fms.gated_ffn(x, wg[0], wu[0]))]
    for err, call in bad:
        with pytest.raises(err):
            call()
