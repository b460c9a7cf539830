"""GPU tests of what AdamW keeps between steps: its counters and moments when a step is
refused, saved and loaded state, version counters, tensors named twice."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
BITS = pytest.mark.parametrize("bits", [32, 8])


def parts(s):
    return list(s) if isinstance(s, tuple) else [s]


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def same(a, b):
    return len(a) == len(b) and all(
        (x is None) == (y is None) and (x is None or all(torch.equal(raw(u), raw(v)) for u, v in zip(parts(x), parts(y))))
        for x, y in zip(a, b))


def make(fms, bits, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    p = [torch.randn(s, generator=gen, device="cuda") for s in ((300,), (40, 8))]
    g = [1e-2 * torch.randn(t.shape, generator=gen, device="cuda") for t in p]
    return fms.AdamW(p, bits=bits, seed=1, **H), g


@BITS
def test_a_refused_step_changes_nothing(fms, bits):
    """A step that is refused is not counted: the next one is the one it would have been."""
    opt, g = make(fms, bits)
    ref, _ = make(fms, bits)
    bad = [g[0], g[1].double()]
    for _ in range(2):
        with pytest.raises(fms.ArgumentError):
            opt.step(bad)
        assert opt.steps == [0, 0] and opt.exp_avgs == [None, None] and opt.exp_avg_sqs == [None, None]
    opt.step(g), ref.step(g)
    with pytest.raises(fms.DimensionMismatch):
        opt.step([g[0], g[1][:1]])
    opt.step(g), ref.step(g)
    assert opt.steps == ref.steps == [2, 2]
    assert same(opt.params, ref.params) and same(opt.exp_avgs, ref.exp_avgs) and same(opt.exp_avg_sqs, ref.exp_avg_sqs)


def test_versions_of_all_that_is_written(fms):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    c = p.bfloat16()
    m, v = fms.moments8(p), fms.moments8(p)
    written = [p, c, *m, *v]
    before = [t._version for t in written]
    fms.adamw_step([p], [g], [m], [v], step=1, copies=[c])
    assert all(t._version > b for t, b in zip(written, before))
    assert g._version == 0
