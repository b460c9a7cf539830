"""GPU tests of the norms around a block (gate, residual scale) against their
formulas in 64 bits, with torch's differentiation of them for the gradients.

Bounds: a row's sums run over `dim` float32 terms, taken against the row's largest
magnitudes with (dim + 16) 2^-24 (a bound on the error of any summation order, and of
the handful of operations around it), the vectors' gradients over all rows; then
half a unit of the last place of the output's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
NAMES = ("x", "h", "w_post", "w_pre", "b_post", "b_pre", "gate")
EPS = 1e-6


def make(batch, tokens, dim, dtype, kind, gate, vdtype=None, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    V = vdtype or dtype
    t = {"x": (2 * r(batch, tokens, dim)).to(dtype), "h": (0.5 * r(batch, tokens, dim) + 0.2).to(dtype),
         "w_post": (1 + 0.2 * r(dim)).to(V), "w_pre": (1 + 0.2 * r(dim)).to(V)}
    if bias:
        t["b_post"], t["b_pre"] = (0.1 * r(dim)).to(V), (0.1 * r(dim)).to(V)
    if gate == "dim":
        t["gate"] = (0.5 + 0.3 * r(dim)).to(V)
    elif gate == "sequence":
        t["gate"] = (0.5 + 0.3 * r(batch, dim)).to(V)
    return t, r(batch, tokens, dim).to(dtype), r(batch, tokens, dim).to(dtype)


def norm64(t, w, b, kind):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    out = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + EPS) * w
    return out if b is None else out + b


def formula(t, scale, kind):
    p = norm64(t["h"], t["w_post"], t.get("b_post"), kind)
    if "gate" in t:
        p = p * (t["gate"] if t["gate"].dim() == 1 else t["gate"][:, None])
    z = scale * t["x"] + p
    return z, norm64(z, t["w_pre"], t.get("b_pre"), kind)


def run_all(fms, t, dz, dy, scale, kind):
    leaf = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
    z, y = fms.norm_residual(**leaf, scale=scale, kind=kind, eps=EPS)
    names = [k for k in NAMES if k in t]
    grads = torch.autograd.grad((z, y), [leaf[k] for k in names], (dz, dy))
    return {"z": z.detach(), "y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def reference(t, dz, dy, scale, kind):
    d = {k: v.detach().double().requires_grad_() for k, v in t.items()}
    z, y = formula(d, scale, kind)
    names = [k for k in NAMES if k in t]
    grads = torch.autograd.grad((z, y), [d[k] for k in names], (dz.double(), dy.double()))
    return {"z": z.detach(), "y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def check(got, ref, t, dz, dy, kind):
    """Rows against their own largest values, vectors against the sums of magnitudes."""
    dim = t["x"].shape[-1]
    per_row = (dim + 16) * 2.0 ** -24
    # a norm, and its gradient, amplify an error by one over the row's deviation
    centre = (lambda v: v - v.mean(-1, keepdim=True)) if kind == "layer" else (lambda v: v)
    narrow = 1.0
    for v in (t["h"].double(), ref["z"]):
        narrow = narrow * (1 + torch.rsqrt(centre(v).pow(2).mean(-1, keepdim=True) + EPS))
    for name, v in ref.items():
        o = got[name]
        assert o.shape == v.shape and torch.isfinite(o).all(), name
        hu = HALF_ULP[o.dtype]
        if name in ("z", "y", "dx", "dh"):
            bound = per_row * 16 * narrow * (v.abs().amax(-1, keepdim=True) + 1) + hu * v.abs() * 1.01
        else:
            # every term is of the size of a normal times ten and off as its row is
            n = narrow if v.dim() == 1 else narrow.sum(1)
            rows = t["x"].numel() // dim if v.dim() == 1 else t["x"].shape[1]
            total = narrow.sum() if v.dim() == 1 else n
            bound = ((rows + 16) * 2.0 ** -24 + per_row * 16) * 10 * total + hu * v.abs() * 1.01
        off = (o.double() - v).abs() - bound
        assert not (off > 0).any(), f"{name}: {int((off > 0).sum())} outside, worst by {off.max()}"


SHAPES = [(1, 1, 768), (3, 5, 2), (2, 7, 33), (4, 9, 64), (3, 50, 128), (2, 40, 129), (5, 17, 768), (2, 31, 1001),
          (1, 200, 1024), (2, 3, 2056), (1, 5, 4104), (2, 2, 8200), (1, 3, 4099),
          (1, 2, 9001), (1, 2, 16384)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,tokens,dim", SHAPES)
def test_against_64_bits(fms, kind, dtype, batch, tokens, dim):
    for gate in ("none", "dim", "sequence"):
        t, dz, dy = make(batch, tokens, dim, dtype, kind, gate, seed=dim, bias=kind == "layer")
        scale = {"none": 1.0, "dim": 0.7, "sequence": 1.25}[gate]
        got = run_all(fms, t, dz, dy, scale, kind)
        check(got, reference(t, dz, dy, scale, kind), t, dz, dy, kind)
        z, y = fms.norm_residual(**t, scale=scale, kind=kind, eps=EPS)  # without gradients: the same
        assert torch.equal(z, got["z"]) and torch.equal(y, got["y"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_float32_vectors(fms, dtype, kind):
    """Float32 weights beside 16-bit features; the bias of an rms norm too."""
    t, dz, dy = make(3, 21, 136, dtype, kind, "sequence", vdtype=torch.float32, seed=4)
    check(run_all(fms, t, dz, dy, 1.0, kind), reference(t, dz, dy, 1.0, kind), t, dz, dy, kind)


def test_many_rows(fms):
    """Rows over more blocks than the device holds, and groups that share a block's work."""
    for batch, tokens, gate in ((1, 9001, "dim"), (700, 13, "sequence"), (3000, 1, "sequence")):
        t, dz, dy = make(batch, tokens, 72, torch.float32, "layer", gate, seed=5)
        check(run_all(fms, t, dz, dy, 1.0, "layer"), reference(t, dz, dy, 1.0, "layer"), t, dz, dy, "layer")


def test_repeats_bit_for_bit(fms):
    t, dz, dy = make(30, 111, 768, torch.bfloat16, "layer", "sequence", seed=6)
    a, b = run_all(fms, t, dz, dy, 1.0, "layer"), run_all(fms, t, dz, dy, 1.0, "layer")
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradient_against_differences(fms, kind):
    """Central differences in float32 along one direction of every argument: the sum's
    float32 error over the step, and the 64-bit difference's own curvature."""
    t, dz, dy = make(3, 20, 96, torch.float32, kind, "sequence", seed=7)
    got = run_all(fms, t, dz, dy, 0.9, kind)
    ref = reference(t, dz, dy, 0.9, kind)
    gen = torch.Generator(device="cuda").manual_seed(8)

    def value(f, a):
        z, y = f(a)
        return float((dz.double() * z.double()).sum() + (dy.double() * y.double()).sum())

    kernel = lambda a: fms.norm_residual(**a, scale=0.9, kind=kind, eps=EPS)  # noqa: E731
    plain = lambda a: formula({k: v.double() for k, v in a.items()}, 0.9, kind)  # noqa: E731
    for name in t:
        v = torch.randn(t[name].shape, generator=gen, device="cuda")
        up, down = dict(t), dict(t)
        up[name], down[name] = t[name] + 2.0 ** -8 * v, t[name] - 2.0 ** -8 * v
        move = up[name].double() - down[name].double()
        quotient = value(kernel, up) - value(kernel, down)
        slope = float((got["d" + name].double() * move).sum())
        bent = abs(value(plain, up) - value(plain, down) - float((ref["d" + name] * move).sum()))
        noise = 112 * 2.0 ** -24 * 2 * (float(dz.double().norm()) * float(got["z"].double().abs().max())
                                        + float(dy.double().norm()) * float(got["y"].double().abs().max()))
        assert abs(quotient - slope) <= bent + noise + 1e-5 * abs(slope), (name, quotient, slope)


def test_one_cotangent(fms):
    """Only z or only y goes on: the other's cotangent is zero."""
    t, dz, dy = make(2, 30, 64, torch.bfloat16, "rms", "dim", seed=9)
    zero = torch.zeros_like(dz)
    for which in (0, 1):
        leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
        out = fms.norm_residual(**leaf, kind="rms", eps=EPS)
        out[which].backward((dz, dy)[which])
        full = run_all(fms, t, dz if which == 0 else zero, zero if which == 0 else dy, 1.0, "rms")
        for k in t:
            assert torch.equal(leaf[k].grad, full["d" + k]), (which, k)


def test_rows_of_zeros_and_of_one_value(fms):
    """A row without spread: the norm's eps alone keeps it finite."""
    for kind in ("rms", "layer"):
        t, dz, dy = make(2, 6, 40, torch.float32, kind, "dim", seed=10)
        t["x"][0], t["h"][0] = 0, 0
        t["h"][1] = 3.0
        got = run_all(fms, t, dz, dy, 1.0, kind)
        ref = reference(t, dz, dy, 1.0, kind)
        for k in ("z", "y"):
            assert torch.allclose(got[k].double(), ref[k], rtol=1e-5, atol=1e-4)
        assert all(torch.isfinite(v).all() for v in got.values())


def test_large_and_small_values(fms):
    """Squares that a 16-bit sum would not hold, and an offset that cancels in a variance."""
    t, dz, dy = make(1, 40, 768, torch.float16, "layer", "none", seed=11)
    t["h"] = (t["h"].float() * 2 + 3000).half()  # neighbouring values 2 apart
    z, y = fms.norm_residual(**t, kind="layer", eps=EPS)
    rz, ry = formula({k: v.double() for k, v in t.items()}, 1.0, "layer")
    # the mean is off by 3000 * 784 * 2^-24 = 0.14 at most against a deviation near 1
    assert (z.double() - rz).abs().max() < 0.14 * 1.7 + 0.01 * float(rz.abs().max())
    t, dz, dy = make(1, 40, 768, torch.bfloat16, "rms", "none", seed=12, bias=False)
    t["h"] = (t["h"].float() * 1e15).bfloat16()  # squares near 1e30, their sum near 1e32
    z, y = fms.norm_residual(**t, kind="rms", eps=EPS)
    rz, ry = formula({k: v.double() for k, v in t.items()}, 1.0, "rms")
    assert (z.double() - rz).abs().max() < 2.0 ** -8 * float(rz.abs().max()) * 1.02


def test_not_a_number_stays_in_its_row(fms):
    t, dz, dy = make(2, 9, 96, torch.float32, "layer", "dim", seed=13)
    z0, y0 = fms.norm_residual(**t, kind="layer")
    t["h"][0, 3, 5] = float("nan")
    t["x"][1, 2, 0] = float("inf")
    z, y = fms.norm_residual(**t, kind="layer")
    assert torch.isnan(z[0, 3]).all() and torch.isnan(y[0, 3]).all() and torch.isnan(y[1, 2]).all()
    keep = torch.ones(2, 9, dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[1, 2] = False
    assert torch.equal(z[keep], z0[keep]) and torch.equal(y[keep], y0[keep])


def test_layouts(fms):
    t, dz, dy = make(2, 12, 80, torch.bfloat16, "layer", "sequence", seed=14)
    z, y = fms.norm_residual(**t, kind="layer")
    odd = dict(t)
    wide = torch.empty(2, 12, 161, dtype=torch.bfloat16, device="cuda")
    wide[..., 1::2] = t["x"]
    odd["x"] = wide[..., 1::2]
    odd["h"] = t["h"].transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.empty(2 * 80 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 80)
    odd["gate"] = off.copy_(t["gate"])
    z1, y1 = fms.norm_residual(**odd, kind="layer")
    assert torch.equal(z, z1) and torch.equal(y, y1)
    got, ref = run_all(fms, odd, dz, dy, 1.0, "layer"), run_all(fms, t, dz, dy, 1.0, "layer")
    assert all(torch.equal(got[k], ref[k]) for k in ref)
    # starts that are off 16 bytes give the same values
    flat = {k: v for k, v in t.items()}
    for k in ("x", "h"):
        flat[k] = torch.empty(t[k].numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(t[k]).copy_(t[k])
    z2, y2 = fms.norm_residual(**flat, kind="layer")
    assert torch.allclose(z2.float(), z.float(), rtol=2.0 ** -7) and torch.allclose(y2.float(), y.float(), rtol=2.0 ** -6, atol=1e-4)
    # two dimensions, and one row alone
    two = {k: (v.view(24, 80) if k in ("x", "h") else v) for k, v in t.items() if k != "gate"}
    za, ya = fms.norm_residual(**two, kind="layer")
    one = {k: (v[7] if k in ("x", "h") else v) for k, v in two.items()}
    zb, yb = fms.norm_residual(**one, kind="layer")
    assert torch.equal(za[7], zb) and torch.equal(ya[7], yb)


def test_empty(fms):
    t, dz, dy = make(0, 5, 16, torch.float32, "layer", "sequence")
    got = run_all(fms, t, dz, dy, 1.0, "layer")
    assert got["z"].shape == (0, 5, 16) and got["dgate"].shape == (0, 16)
    assert not got["dw_post"].any() and not got["db_pre"].any()
    t, dz, dy = make(3, 0, 16, torch.float32, "rms", "sequence")
    got = run_all(fms, t, dz, dy, 1.0, "rms")
    assert got["dgate"].shape == (3, 16) and not got["dgate"].any() and not got["dw_pre"].any()


def test_another_stream(fms):
    t, dz, dy = make(20, 60, 256, torch.bfloat16, "rms", "dim", seed=15)
    ref = run_all(fms, t, dz, dy, 1.0, "rms")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_all(fms, t, dz, dy, 1.0, "rms")
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(got[k], ref[k]) for k in ref)


def test_refusals(fms):
    t, _, _ = make(2, 3, 16, torch.bfloat16, "rms", "dim")
    with_ = lambda **kw: (lambda: fms.norm_residual(**{**t, **kw}))  # noqa: E731
    for err, call in [(fms.ArgumentError, with_(kind="batch")),
                      (fms.ArgumentError, with_(eps=-1.0)),
                      (fms.ArgumentError, with_(h=t["h"].float())),
                      (fms.ArgumentError, with_(w_pre=t["w_pre"].float())),
                      (fms.ArgumentError, with_(x=t["x"].double(), h=t["h"].double())),
                      (fms.ArgumentError, with_(gate=t["gate"].cpu())),
                      (fms.DimensionMismatch, with_(h=t["h"][:1])),
                      (fms.DimensionMismatch, with_(w_post=t["w_post"][:8])),
                      (fms.DimensionMismatch, with_(gate=t["gate"].expand(3, 16))),
                      (fms.DimensionMismatch, lambda: fms.norm_residual(*[torch.zeros(n, 16385, device="cuda").squeeze(0)
                                                                          for n in (2, 2, 1, 1)])),
                      (fms.DimensionMismatch, with_(b_pre=t["b_pre"][None]))]:
        with pytest.raises(err):
            call()
