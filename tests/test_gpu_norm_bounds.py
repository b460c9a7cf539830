"""GPU tests of the norms around a block with bounds that a missing term, a lost part of a
sum or a statistic in fewer bits would break, and the proof of it: for each shape the
checks reject such outputs.

Derivation.  A kernel adds at most 16 values in a thread, 6 levels in a warp and 32 warps'
sums in turn for a row's statistic: 54 roundings of half a unit of 2^-23 in float32, each
spread evenly, a standard deviation of sqrt(54 / 12) 2^-23 = 2.1 2^-23 of the sum of
magnitudes; six of these and the handful of operations around them are 16 2^-23 = 2^-19.
A norm and its gradient amplify an error by the row's reciprocal deviations (`narrow`).
A vector's gradient sums one such term per row, independent from row to row, each below
8 in size (six deviations of its normal factors are larger, but their errors add in
squares): 8 2^-19 sqrt(sum narrow^2), which also holds the 2^-24 sqrt(rows) of the sum's
own roundings.  Then half a unit of the last place of the output's type."""
import pytest
import torch

from test_gpu_norm_residual import EPS, HALF_ULP, NAMES, make, reference, run_all

pytestmark = pytest.mark.gpu

U = 2.0 ** -19
SHAPES = [(1, 3, 96), (2, 7, 33), (3, 50, 128), (2, 40, 129), (5, 17, 768), (2, 31, 1001), (1, 200, 1024), (2, 3, 2056),
          (1, 5, 4104), (2, 2, 8200), (1, 3, 4099), (1, 2, 9001), (1, 4, 16384), (1, 9001, 72), (700, 13, 72),
          (3000, 1, 72), (40, 180, 256)]


def stats(v, kind):
    m = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    return m, torch.rsqrt((v - m).pow(2).mean(-1, keepdim=True) + EPS)


def bounds(t, ref, kind):
    h, z = t["h"].double(), ref["z"]
    narrow = (1 + stats(h, kind)[1]) * (1 + stats(z, kind)[1])
    out = {}
    for name, v in ref.items():
        hu = HALF_ULP[t["x"].dtype if name in ("z", "y", "dx", "dh") else t["w_post"].dtype] * 1.01
        if name in ("z", "y", "dx", "dh"):
            out[name] = U * narrow * (1 + v.abs().amax(-1, keepdim=True)) + hu * v.abs()
        else:
            total = narrow.pow(2).sum(dim=(0, 1) if v.dim() == 1 else 1).sqrt()
            out[name] = 8 * U * total + hu * v.abs()
    return out


def outside(got, ref, bound):
    return {k: int(((got[k].double() - ref[k]).abs() > bound[k]).sum()) for k in ref}


def gradient(dout, w, hat, rstd, kind, drop=()):
    """A norm's gradient, without the terms named in `drop`."""
    d = dout * w
    e = d
    if "product" not in drop:
        e = e - hat * (d * hat).mean(-1, keepdim=True)
    if kind == "layer" and "mean" not in drop:
        e = e - d.mean(-1, keepdim=True)
    return e * rstd


def rows_gradients(t, dz, dy, scale, kind, ref, drop_pre=(), drop_post=()):
    d = {k: v.double() for k, v in t.items()}
    mh, rh = stats(d["h"], kind)
    mz, rz = stats(ref["z"], kind)
    hhat, zhat = (d["h"] - mh) * rh, (ref["z"] - mz) * rz
    g = 1.0 if "gate" not in d else d["gate"] if d["gate"].dim() == 1 else d["gate"][:, None]
    dzt = dz.double() + gradient(dy.double(), d["w_pre"], zhat, rz, kind, drop_pre)
    return {"dx": scale * dzt, "dh": gradient(dzt * g, d["w_post"], hhat, rh, kind, drop_post)}


CASES = [(kind, gate, b, n, d) for b, n, d in SHAPES for kind, gate in
         (("layer", "sequence"), ("rms", "dim"), ("layer", "none"))]


@pytest.mark.parametrize("kind,gate,batch,tokens,dim", CASES)
def test_float32(fms, kind, gate, batch, tokens, dim):
    scale = 0.75
    t, dz, dy = make(batch, tokens, dim, torch.float32, kind, gate, seed=dim + tokens, bias=kind == "layer")
    ref = reference(t, dz, dy, scale, kind)
    bound = bounds(t, ref, kind)
    none = {k: 0 for k in ref}
    assert outside(run_all(fms, t, dz, dy, scale, kind), ref, bound) == none

    # what the checks have to reject: a vector's gradient left out, or one row of it
    for k in ["d" + n for n in NAMES[2:] if n in t]:
        assert outside({**ref, k: torch.zeros_like(ref[k])}, ref, bound)[k] > 0, k
    # a gradient of the rows without one of its terms
    right = rows_gradients(t, dz, dy, scale, kind, ref)
    assert outside({**ref, **right}, ref, bound) == none
    for drop in (("product",), ("mean",)) if kind == "layer" else (("product",),):
        wrong = rows_gradients(t, dz, dy, scale, kind, ref, drop_pre=drop)["dx"]
        assert outside({**ref, "dx": wrong}, ref, bound)["dx"] > 0, drop
        wrong = rows_gradients(t, dz, dy, scale, kind, ref, drop_post=drop)["dh"]
        assert outside({**ref, "dh": wrong}, ref, bound)["dh"] > 0, drop
    # outputs from inputs in bfloat16, as a product or a statistic in fewer bits would give
    fewer = reference({k: v.bfloat16() for k, v in t.items()}, dz, dy, scale, kind)
    assert outside(fewer, ref, bound)["z"] > 0 and outside(fewer, ref, bound)["y"] > 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind,gate,batch,tokens,dim", CASES)
def test_16_bits(fms, dtype, kind, gate, batch, tokens, dim):
    t, dz, dy = make(batch, tokens, dim, dtype, kind, gate, seed=dim + tokens, bias=kind == "layer")
    ref = reference(t, dz, dy, 1.25, kind)
    bound = bounds(t, ref, kind)
    assert outside(run_all(fms, t, dz, dy, 1.25, kind), ref, bound) == {k: 0 for k in ref}
    for k in ["d" + n for n in NAMES[2:] if n in t]:
        assert outside({**ref, k: torch.zeros_like(ref[k])}, ref, bound)[k] > 0, k
