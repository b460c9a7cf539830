"""GPU tests of the INT8 linear layer.  The integer sums are exact, so the result is
(sx * sw) * sum + b with three float32 roundings and one to the output's type: the
bound is 3 2^-24 of the product and of the bias, and half a unit of the last place
(the codes of float features are those of the float32 formula, bit for bit)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def make(fms, rows, dim, out, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    w = fms.quantize_int8_symmetric(torch.randn(out, dim, generator=g, device="cuda") / dim ** 0.5)
    return x, w, torch.randn(out, generator=g, device="cuda").to(dtype)


def codes32(x):
    """The codes and scales of the float32 formula, on the host."""
    x = x.float().cpu().numpy()
    top = np.abs(x).max(1) if x.shape[1] else np.zeros(len(x), np.float32)
    sc = (np.maximum(top, np.float32(1e-8)) * np.float32(1 / 127)).astype(np.float32)
    return np.rint(np.clip(x / sc[:, None], -127, 127)).astype(np.int64), sc


def check(y, xc, xs, w, bias):
    acc = xc.astype(np.float64) @ w.codes.cpu().numpy().astype(np.float64).T  # whole numbers below 2^53: exact
    v = acc * (xs.astype(np.float64)[:, None] * w.scales.cpu().numpy().astype(np.float64)[None, :])
    b = 0.0 if bias is None else bias.double().cpu().numpy()[None, :]
    bound = 3 * 2.0 ** -24 * (np.abs(v) + np.abs(b)) + HALF_ULP[y.dtype] * 1.01 * np.abs(v + b) + TINY[y.dtype]
    off = np.abs(y.double().cpu().numpy() - (v + b)) - bound
    assert y.shape == v.shape and np.isfinite(off).all() and not (off > 0).any(), \
        f"{(off > 0).sum()} outside, worst by {off.max()}"


SIZES = [(1, 1, 1), (1, 768, 256), (2, 100, 33), (3, 16, 7), (5, 129, 130), (8, 4096, 64), (9, 128, 300), (16, 64, 128),
         (31, 768, 128), (32, 200, 1), (33, 256, 257), (64, 17, 48), (127, 777, 129), (129, 128, 128), (300, 272, 520),
         (1000, 768, 136), (257, 1040, 512)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,out", SIZES)
def test_against_exact_sums(fms, dtype, rows, dim, out):
    x, w, b = make(fms, rows, dim, out, dtype, rows + dim + out)
    xc, xs = codes32(x)
    check(fms.int8_linear(x, w), xc, xs, w, None)
    check(fms.int8_linear(x, w, bias=b), xc, xs, w, b)


# Enough tiles for pairs of SMs, at widths that end inside a tile and off 16 bytes; rows of
# codes and of features that do not start on 16 bytes.
TILES = [(1500, 256, 3001), (1301, 101, 2600), (2600, 64, 1500), (1020, 1500, 2056), (999, 2051, 1100)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,out", TILES)
def test_tiles_against_exact_sums(fms, dtype, rows, dim, out):
    x, w, b = make(fms, rows, dim, out, dtype, rows + out)
    xc, xs = codes32(x)
    check(fms.int8_linear(x, w, bias=b), xc, xs, w, b)


# Narrow layers over many tokens: whole and part tiles of tokens, widths inside a block of the
# sum and at its end, outputs inside a tile and off 16 bytes; a token of zeros.
NARROW = [(18944, 128, 128), (19000, 48, 64), (20001, 768, 128), (18951, 752, 100), (19072, 1024, 33), (40000, 512, 256),
          (19100, 272, 200), (18945, 16, 1), (19333, 640, 65), (18944, 1040, 64), (18943, 256, 128), (57000, 144, 48)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,out", NARROW)
def test_narrow_against_exact_sums(fms, dtype, rows, dim, out):
    x, w, b = make(fms, rows, dim, out, dtype, rows + dim + out)
    x[rows - 3] = 0
    xc, xs = codes32(x)
    y = fms.int8_linear(x, w, bias=b)
    check(y, xc, xs, w, b)
    other = torch.float32 if dtype != torch.float32 else torch.bfloat16
    check(fms.int8_linear(x, w, out_dtype=other), xc, xs, w, None)
    assert torch.equal(y, fms.int8_linear(x, w, bias=b))
    assert torch.equal(y[-70:], fms.int8_linear(x[-70:].contiguous(), w, bias=b))  # another tile's bits


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [60, 700])
def test_scales_and_bias_off_16_bytes(fms, dtype, rows):
    x, w, b = make(fms, rows, 192, 161, dtype, rows)
    tail = fms.Int8Index(w.codes[1:].contiguous(), w.scales[1:])
    xc, xs = codes32(x)
    y = fms.int8_linear(x, tail, bias=b[1:])
    check(y, xc, xs, tail, b[1:])
    whole = fms.Int8Index(tail.codes, tail.scales.clone())
    for bias in (b[1:], b[1:].clone()):
        assert torch.equal(fms.int8_linear(x, whole, bias=bias), y)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_narrow_layer_keeps_a_bad_token_to_itself(fms, bad):
    x, w, b = make(fms, 19000, 256, 96, torch.bfloat16)
    good = fms.int8_linear(x, w, bias=b)
    x[18000, 77] = bad
    y = fms.int8_linear(x, w, bias=b)
    assert y[18000].isnan().all()
    keep = torch.arange(19000, device="cuda") != 18000
    assert torch.equal(y[keep], good[keep])


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_quantised_features(fms, rows):
    """An Int8Index of features, scores in every type; equal to the float call on its codes."""
    x, w, _ = make(fms, rows, 384, 160, torch.float32, rows)
    q = fms.quantize_int8_symmetric(x)
    xc, xs = q.codes.cpu().numpy().astype(np.int64), q.scales.cpu().numpy()
    for T in (torch.float32, torch.float16, torch.bfloat16):
        check(fms.int8_linear(q, w, out_dtype=T), xc, xs, w, None)
    same = fms.Int8Index(*(torch.from_numpy(a).cuda() for a in (codes32(x)[0].astype(np.int8), codes32(x)[1])))
    assert torch.equal(fms.int8_linear(same, w), fms.int8_linear(x, w))
    assert fms.int8_linear(x.half(), w, out_dtype=torch.float32).dtype == torch.float32


@pytest.mark.parametrize("rows", [1, 12, 150])
def test_extreme_codes(fms, rows):
    """Sums past 2^24, at both ends of the codes (-128 too), stay exact."""
    dim, out = 8191, 40
    xc = torch.full((rows, dim), 127, dtype=torch.int8, device="cuda")
    wc = torch.full((out, dim), -128, dtype=torch.int8, device="cuda")
    xc[0, ::3] = -128
    wc[1::2] = 127
    ones = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    w = fms.Int8Index(wc, ones(out))
    y = fms.int8_linear(fms.Int8Index(xc, ones(rows)), w)
    check(y, xc.cpu().numpy().astype(np.int64), np.ones(rows, np.float32), w, None)


def test_ties_round_to_even(fms):
    """absmax 127 makes the scale 1, so the halves are exact ties."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 3.0]], device="cuda")
    eye = fms.Int8Index(torch.eye(8, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda"))
    for rows in (1, 50):
        y = fms.int8_linear(x.expand(rows, 8), eye)
        assert y[0].tolist() == [127, 0, 2, 2, 0, -2, -126, 3]
        assert torch.equal(y, y[:1].expand(rows, 8))


@pytest.mark.parametrize("rows", [4, 100])
def test_zero_infinite_and_nan_tokens(fms, rows):
    x, w, b = make(fms, rows, 96, 72, torch.bfloat16, 5)
    clean = fms.int8_linear(x, w, bias=b)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 9] = float("-inf")
    y = fms.int8_linear(x, w, bias=b)
    assert torch.equal(y[0], b) and torch.isnan(y[1:3]).all() and torch.equal(y[3:], clean[3:])


def test_layouts_and_shapes(fms):
    x, w, b = make(fms, 24, 80, 48, torch.float16, 6)
    y = fms.int8_linear(x, w, bias=b)
    assert torch.equal(fms.int8_linear(x.view(2, 3, 4, 80), w, bias=b), y.view(2, 3, 4, 48))
    assert torch.equal(fms.int8_linear(x[3], w, bias=b), y[3])
    wide = torch.empty(24, 161, dtype=x.dtype, device="cuda")
    wide[:, 1::2] = x
    assert torch.equal(fms.int8_linear(wide[:, 1::2], w, bias=b), y)
    turned = fms.Int8Index(w.codes.T.contiguous().T, w.scales)
    assert torch.equal(fms.int8_linear(x, turned, bias=b), y)
    # starts that are off 16 bytes
    codes = torch.empty(48 * 80 + 1, dtype=torch.int8, device="cuda")[1:].view(48, 80).copy_(w.codes)
    off = torch.empty(24 * 80 + 1, dtype=x.dtype, device="cuda")[1:].view(24, 80).copy_(x)
    assert torch.equal(fms.int8_linear(off, fms.Int8Index(codes, w.scales), bias=b), y)


def test_empty(fms):
    x, w, b = make(fms, 0, 32, 16, torch.float16)
    assert fms.int8_linear(x, w, bias=b).shape == (0, 16)
    none = fms.Int8Index(w.codes[:0], w.scales[:0])
    assert fms.int8_linear(torch.zeros(3, 32, device="cuda"), none).shape == (3, 0)


def test_another_stream_and_graph(fms):
    x, w, b = make(fms, 300, 256, 160, torch.bfloat16, 7)
    y = fms.int8_linear(x, w, bias=b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = fms.int8_linear(x, w, bias=b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, z)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = fms.int8_linear(x[:1], w, bias=b)
    x[:1] = make(fms, 1, 256, 160, torch.bfloat16, 8)[0]
    graph.replay()
    assert torch.equal(z, fms.int8_linear(x[:1], w, bias=b))


def test_feeds_the_index(fms):
    """Features projected in INT8, quantised into an index and searched: the scores are
    those of the same index scored pair by pair."""
    g = torch.Generator(device="cuda").manual_seed(9)
    feats = torch.randn(12, 20, 96, generator=g, device="cuda").half()
    w = fms.quantize_int8_symmetric(torch.randn(128, 96, generator=g, device="cuda"))
    d = torch.nn.functional.normalize(fms.int8_linear(feats, w, out_dtype=torch.float32), dim=-1)
    index = fms.quantize_int8_symmetric(d)
    q = d[:2, :8].contiguous()
    vals, ids = fms.maxsim(q, index, topk=3)
    assert ids[0, 0] == 1 and ids[1, 0] == 2
    one = fms.maxsim(q[1], fms.Int8Index(index.codes[1], index.scales[1]))
    assert torch.allclose(one, vals[1, :1], rtol=1e-6)


def test_refusals(fms):
    x, w, b = make(fms, 4, 32, 16, torch.float16)
    I = fms.Int8Index
    for err, call in [(fms.DimensionMismatch, lambda: fms.int8_linear(x[:, :16], w)),
                      (fms.DimensionMismatch, lambda: fms.int8_linear(x, w, bias=b[:8])),
                      (fms.DimensionMismatch, lambda: fms.int8_linear(x, I(w.codes, w.scales[:8]))),
                      (fms.DimensionMismatch, lambda: fms.int8_linear(x, I(w.codes[None], w.scales[None]))),
                      (fms.ArgumentError, lambda: fms.int8_linear(x, I(w.codes.short(), w.scales))),
                      (fms.ArgumentError, lambda: fms.int8_linear(x, I(w.codes, w.scales.half()))),
                      (fms.ArgumentError, lambda: fms.int8_linear(x.double(), w)),
                      (fms.ArgumentError, lambda: fms.int8_linear(x, w, bias=b.float())),
                      (fms.ArgumentError, lambda: fms.int8_linear(x.cpu(), w)),
                      (fms.ArgumentError, lambda: fms.int8_linear(x, w, out_dtype=torch.int8)),
                      (fms.ArgumentError, lambda: fms.int8_linear(x.clone().requires_grad_(), w))]:
        with pytest.raises(err):
            call()
    # an int32 sum could overflow past this width: refused before any launch
    L = fms.load_library()
    assert L.fms_int8_linear_fwd(4, None, None, None, None, None, 1, 131072, 1, 0, None, None, 0, None) == -6
