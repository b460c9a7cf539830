"""GPU test: where the vectors of a norm start (a slice of a flat buffer of parameters)
does not change its results, for rows that start on 16 bytes."""
import pytest
import torch

from test_gpu_norm_residual import make, run_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,vdtype", [(torch.float32, None), (torch.float16, None), (torch.bfloat16, None),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dim", [64, 768, 1536, 5120])
def test_vectors_off_16_bytes(fms, dtype, vdtype, kind, dim):
    t, dz, dy = make(3, 37, dim, dtype, kind, "sequence", vdtype=vdtype, seed=dim, bias=kind == "layer")
    want = run_all(fms, t, dz, dy, 0.75, kind)
    off = {k: v if k in ("x", "h") else torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")[1:].view(v.shape).copy_(v)
           for k, v in t.items()}
    leaf = {k: v.requires_grad_() for k, v in off.items()}
    z, y = fms.norm_residual(**leaf, scale=0.75, kind=kind, eps=1e-6)
    names = list(leaf)
    grads = torch.autograd.grad((z, y), [leaf[k] for k in names], (dz, dy))
    got = {"z": z, "y": y, **{"d" + k: g for k, g in zip(names, grads)}}
    for k in want:
        assert torch.equal(got[k], want[k]), k
