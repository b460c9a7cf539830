"""GPU test of the gated feed-forward block on operands that start two bytes off a word:
views into buffers whose other values are NaN."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def inside(t):
    """t in the middle of a buffer of NaN, one element after an aligned start."""
    buf = torch.full((t.numel() + 3,), float("nan"), dtype=t.dtype, device="cuda")
    v = buf[1:1 + t.numel()].view(t.shape)
    return buf, v.copy_(t)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,hidden", [(9, 1, 1), (10, 2, 3), (17, 3, 2), (33, 64, 48), (40, 65, 49), (200, 130, 257)])
def test_operands_off_a_word(fms, dtype, rows, dim, hidden):
    g = torch.Generator(device="cuda").manual_seed(rows)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    args = [r(rows, dim), r(hidden, dim), r(hidden, dim)]
    dh = r(rows, hidden)

    def run(args, dh):
        leaves = [t.detach().requires_grad_() for t in args]
        h = fms.gated_ffn(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    want = run(args, dh)
    kept = [inside(t) for t in (*args, dh)]
    got = run([v for _, v in kept[:3]], kept[3][1])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for buf, v in kept:  # and nothing was written beside them
        assert torch.isnan(buf[0]) and torch.isnan(buf[1 + v.numel():]).all()
