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


@BITS
def test_a_saved_state_is_taken_up_twice(fms, bits):
    """Two optimisers from one dict step independently, and the dict keeps what it held."""
    opt, g = make(fms, bits)
    opt.step(g)
    saved = opt.state_dict()
    kept = [[tuple(u.clone() for u in s) if bits == 8 else s.clone() for s in saved[k]] for k in ("exp_avgs", "exp_avg_sqs")]
    start = [t.clone() for t in opt.params]

    def taken_up():
        o = fms.AdamW([t.clone() for t in start], bits=bits, seed=1, **H)
        o.load_state_dict(saved)
        return o

    a, b = taken_up(), taken_up()
    for o in (opt, a, b):
        for _ in range(2):
            o.step(g)
    assert opt.steps == a.steps == b.steps == [3, 3]
    assert same(opt.params, a.params) and same(opt.params, b.params)
    assert same(opt.exp_avgs, a.exp_avgs) and same(opt.exp_avgs, b.exp_avgs)
    assert same(saved["exp_avgs"], kept[0]) and same(saved["exp_avg_sqs"], kept[1]) and saved["steps"] == [1, 1]
    # back to the saved step
    for t, s in zip(opt.params, start):
        t.copy_(s)
    opt.load_state_dict(saved)
    for _ in range(2):
        opt.step(g)
    assert same(opt.params, a.params) and same(opt.exp_avgs, a.exp_avgs) and same(opt.exp_avg_sqs, a.exp_avg_sqs)


@BITS
def test_a_state_read_on_the_host(fms, bits):
    """Moments that were loaded to the host go to their parameter's device."""
    opt, g = make(fms, bits)
    opt.step(g)
    host = {k: [tuple(u.cpu() for u in s) if bits == 8 else s.cpu() for s in v] if k.startswith("exp") else v
            for k, v in opt.state_dict().items()}
    other = fms.AdamW([t.clone() for t in opt.params], bits=bits, seed=1, **H)
    other.load_state_dict(host)
    opt.step(g), other.step(g)
    assert same(opt.params, other.params)


@BITS
def test_a_state_that_does_not_fit_is_refused(fms, bits):
    opt, g = make(fms, bits)
    opt.step(g)
    good = opt.state_dict()
    short = lambda s: tuple(u[:-1] for u in s) if bits == 8 else s[:-1]  # noqa: E731
    other = lambda s: (s[0].float(), s[1]) if bits == 8 else s.half()  # noqa: E731
    m = good["exp_avgs"]
    before = [opt.steps, opt.exp_avgs, opt.exp_avg_sqs]
    for err, bad in [(fms.ArgumentError, dict(good, steps=[1])),
                     (fms.ArgumentError, dict(good, steps=[1, -1])),
                     (fms.ArgumentError, dict(good, exp_avgs=m[:1])),
                     (fms.ArgumentError, dict(good, exp_avg_sqs=good["exp_avg_sqs"][:1])),
                     (fms.ArgumentError, dict(good, exp_avgs=[m[0], None])),
                     (fms.ArgumentError, dict(good, exp_avgs=[m[0], other(m[1])])),
                     (fms.DimensionMismatch, dict(good, exp_avgs=[short(m[0]), m[1]]))]:
        with pytest.raises(err):
            opt.load_state_dict(bad)
        assert all(x is y for x, y in zip(before, [opt.steps, opt.exp_avgs, opt.exp_avg_sqs]))


def test_versions_of_all_that_is_written(fms):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    c = p.bfloat16()
    m, v = fms.moments8(p), fms.moments8(p)
    written = [p, c, *m, *v]
    before = [t._version for t in written]
    fms.adamw_step([p], [g], [m], [v], step=1, copies=[c])
    assert all(t._version > b for t, b in zip(written, before))
    assert g._version == 0


def test_a_tensor_named_twice_is_refused(fms):
    """Two entries of one launch that write the same memory would race."""
    z = lambda n=512: torch.zeros(n, device="cuda")  # noqa: E731
    p, q, g = z(), z(), torch.ones(512, device="cuda")
    m, v = [z(), z()], [z(), z()]
    e = fms.moments8(p)
    for f in (lambda: fms.adamw_step([p, p], [g, g], m, v, step=1),
              lambda: fms.adamw_step([p, q], [g, g], [m[0], m[0]], v, step=1),
              lambda: fms.adamw_step([p, q], [g, g], m, [v[0], m[1]], step=1),
              lambda: fms.adamw_step([p], [g], [(e[0], e[1])], [(fms.moments8(p)[0], e[1])], step=1),
              lambda: fms.adamw_step([p.bfloat16()] * 2, [g, g], m, v, step=1),
              lambda: fms.AdamW([p, p]).step([g, g])):
        with pytest.raises(fms.ArgumentError, match="twice"):
            f()
    assert not p.any() and not m[0].any()
    # shared gradients are only read; empty tensors may have any address
    fms.adamw_step([p, q, z(0), z(0)], [g, g, z(0), z(0)], m + [z(0), z(0)], v + [z(0), z(0)], step=1)
    assert torch.equal(p, q) and p.any()


def test_a_copy_may_be_its_parameter(fms):
    p, g = torch.ones(300, device="cuda").bfloat16(), torch.ones(300, device="cuda")
    q = p.clone()
    m, v, m2, v2 = (torch.zeros(300, device="cuda") for _ in range(4))
    fms.adamw_step([p], [g], [m], [v], step=1, copies=[p])
    fms.adamw_step([q], [g], [m2], [v2], step=1)
    assert torch.equal(p, q)
