"""A token encoder trained through MaxSim and served from an INT8 index.

Queries are shortened copies of documents under noise, as synthetic token features.  The
encoder is two residual blocks (norm, gated feed-forward, norm, gate) and a projection
to 128 values per token; in-batch late-interaction scores are trained with a softmax
over the batch, gradients come back through maxsim's argmax tape, and AdamW steps
float32 weights with 8-bit moments beside the bfloat16 copies that the model computes
with.  Then the projection runs in INT8, its output becomes an Int8Index, and each
query searches all documents.

    python examples/train_token_encoder.py
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import flashmaxsim_b200 as fms  # noqa: E402


SIGNAL = 24


class Encoder:
    """Weights in float32 (`masters`), the bfloat16 copies that compute (`w`), names alike."""

    def __init__(self, dim, hidden, out, blocks, gen, dev):
        r = lambda *s: torch.randn(*s, generator=gen, device=dev) / math.sqrt(s[-1])  # noqa: E731
        self.masters = {"norm": torch.ones(dim, device=dev), "proj": r(out, dim)}
        for b in range(blocks):
            self.masters |= {f"gate{b}": r(hidden, dim), f"up{b}": r(hidden, dim), f"down{b}": r(dim, hidden),
                             f"post{b}": torch.ones(dim, device=dev), f"pre{b}": torch.ones(dim, device=dev),
                             f"mix{b}": torch.full((dim,), 0.1, device=dev)}
        self.blocks = blocks
        self.w = {k: v.bfloat16().requires_grad_() for k, v in self.masters.items()}

    def features(self, x):
        """(B, T, dim) bfloat16 -> the same, normalised."""
        w = self.w
        # the first norm has no block before it
        y = torch.nn.functional.rms_norm(x, x.shape[-1:], w["norm"], 1e-6)
        for b in range(self.blocks):
            h = fms.gated_ffn(y, w[f"gate{b}"], w[f"up{b}"], act="silu") @ w[f"down{b}"].T
            x, y = fms.norm_residual(x, h, w[f"post{b}"], w[f"pre{b}"], gate=w[f"mix{b}"])
        return y

    def tokens(self, x):
        """(B, T, dim) -> (B, T, out), each token of length one."""
        return torch.nn.functional.normalize((self.features(x) @ self.w["proj"].T).float(), dim=-1).bfloat16()


def batch(gen, dev, n, tq, td, basis, noise):
    """n documents, and a query from some of each one's tokens.  What both share lies in the
    first SIGNAL directions of `basis`; the others are noise, new for every token."""
    dim = basis.shape[0]
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    d = r(n, td, SIGNAL)
    at = torch.rand(n, td, generator=gen, device=dev).argsort(1)[:, :tq]
    q = torch.gather(d, 1, at[..., None].expand(-1, -1, SIGNAL))
    q, d = (torch.cat([t, noise * r(*t.shape[:2], dim - SIGNAL)], -1) @ basis for t in (q, d))
    return q.bfloat16(), d.bfloat16()


def main(steps=60, n=64, tq=8, td=40, dim=192, hidden=512, out=128, blocks=2, noise=1.0, lr=2e-3, scale=3.0, seed=0,
         bits=8, say=print):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    basis = torch.linalg.qr(torch.randn(dim, dim, generator=gen, device=dev))[0]
    enc = Encoder(dim, hidden, out, blocks, gen, dev)
    names = list(enc.w)
    opt = fms.AdamW([enc.masters[k] for k in names], lr=lr, bits=bits, seed=seed,
                    copies=[enc.w[k].detach() for k in names])
    target = torch.arange(n, device=dev)
    losses = []
    for step in range(steps):
        q, d = batch(gen, dev, n, tq, td, basis, noise)
        scores = fms.maxsim(enc.tokens(q), enc.tokens(d), fms.InBatch(), backward=fms.InvGrid())
        loss = torch.nn.functional.cross_entropy(scores * scale, target)
        grads = torch.autograd.grad(loss, [enc.w[k] for k in names])
        opt.step(grads)
        losses.append(loss.detach())
        if step % 20 == 0 or step == steps - 1:
            say(f"step {step:3d}  loss {float(losses[-1]):.3f}")

    # serving: the projection in INT8, its output an INT8 index of every document
    with torch.no_grad():
        proj = fms.quantize_int8_symmetric(enc.masters["proj"])
        q, d = batch(gen, dev, 4 * n, tq, td, basis, noise)
        project = lambda x: torch.nn.functional.normalize(  # noqa: E731
            fms.int8_linear(enc.features(x), proj, out_dtype=torch.float32), dim=-1)
        index = fms.quantize_int8_symmetric(project(d))
        _, ids = fms.maxsim(project(q), index, topk=10)
        right = ids == torch.arange(1, 4 * n + 1, device=dev)[:, None]
        top1, top10 = float(right[:, 0].float().mean()), float(right.any(1).float().mean())
    say(f"INT8 index of {4 * n} documents: right document first for {top1:.0%} of the queries, in the first 10 for {top10:.0%}")
    return [float(x) for x in losses], top1, top10


if __name__ == "__main__":
    main()
