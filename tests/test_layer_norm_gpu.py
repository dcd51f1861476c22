"""GPU tests of layer norm and its backward pass (k3_layer_norm_*, cumatrix.LayerNormPerRow / DiffLayerNormPerRow) against the formulas in float64, and of the derivatives against
differences.

Bounds.  Every result is computed in float32 and rounded once to the matrix's type: half a step of the result, plus what the float32 steps can be off.  A sum of n terms taken as
n / 64 terms by each of 64 lanes or more and then over the lanes is off by at most (n / 64 + 16) half steps of the sum of the magnitudes; call that factor C(n).  Two dozen further
roundings (differences, products, the root) are covered by adding 24 to it.  float16 has steps of 2^-24 below 2^-14, which adds 2^-25."""
import pytest, torch
from tests.rowop_cases import TYPES, U32, half_step, matrix, empty_like, untouched, assert_within, generator
pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 2), (1, 768), (17, 63), (5, 64), (33, 65), (64, 129), (300, 257), (7, 768), (129, 1023), (40, 1536), (9, 2047), (12, 2050), (70, 4096), (3, 8191), (4, 8200),
         (5, 20011), (3, 40007), (2, 70001)]

def C(n): return (n / 64 + 40) * U32

def reference(x, scale, offset, eps):
    x = x.double(); mean = x.mean(1, keepdim=True); d = x - mean
    inv = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + eps); xhat = d * inv
    y = xhat * (1.0 if scale is None else scale.double()) + (0.0 if offset is None else offset.double())
    return y, mean, inv, xhat

def reference_backward(x, dy, scale, mean, inv):
    xhat = (x.double() - mean.double()[:, None]) * inv.double()[:, None]
    g = dy.double() * (1.0 if scale is None else scale.double())
    a, b = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    return inv.double()[:, None] * (g - a - xhat * b), (dy.double() * xhat).sum(0), dy.double().sum(0), xhat, g

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward_matches_the_formula(rows, cols, dtype):
    from kaldi_amd.cumatrix import LayerNormPerRow
    g = generator(rows * 100003 + cols)
    for pad, first, affine, shift in ((0, 0, True, 0.0), (3, 1, False, 30.0), (8, 0, True, 30.0)):
        x = matrix(g, rows, cols, dtype, pad, 2.0, first); x += shift
        scale = torch.randn(cols, generator=g, device="cuda") if affine else None; offset = torch.randn(cols, generator=g, device="cuda") if affine else None
        y = empty_like(x); mean = torch.empty(rows, device="cuda"); inv = torch.empty(rows, device="cuda")
        LayerNormPerRow(x, scale, offset, 1e-5, y, mean, inv)
        want, m, r, xhat = reference(x, scale, offset, 1e-5)
        assert untouched(y)
        assert_within(mean, m[:, 0], C(cols) * x.double().abs().mean(1) + 1e-30, "mean")
        # the square root halves the relative error of var + eps, whose terms' magnitudes sum to themselves.  cols = 1 (var = 0): x - mean is 0 exactly
        assert_within(inv, r[:, 0], C(cols) * r[:, 0], "inv_std")
        # the difference from the mean is off by at most C(cols) of the mean magnitude of the differences (the first mean's error is taken out by the second sum), and a step of itself
        off = C(cols) * ((xhat.abs() + xhat.abs().mean(1, keepdim=True)) * (1.0 if scale is None else scale.double().abs())) + 4 * U32 * want.abs()
        if offset is not None: off = off + 2 * U32 * offset.double().abs()
        assert_within(y, want, half_step(dtype) * (want.abs() + off) + off + (2.0 ** -25 if dtype == torch.float16 else 0.0), "y")
        z = x.clone() if pad == 0 else x
        LayerNormPerRow(z, scale, offset, 1e-5, z)      # in place, and without keeping the statistics
        assert torch.equal(z, y)

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES + [(1000, 96), (2500, 768), (600, 1537)])
def test_backward_matches_the_formula(rows, cols, dtype):
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    g = generator(rows * 100003 + cols + 1)
    for pad, affine in ((0, True), (5, False)):
        x = matrix(g, rows, cols, dtype, pad, 2.0, pad // 5); dy = matrix(g, rows, cols, dtype, 2 * pad, 0.5); scale = torch.randn(cols, generator=g, device="cuda") if affine else None
        mean = torch.empty(rows, device="cuda"); inv = torch.empty(rows, device="cuda"); LayerNormPerRow(x, scale, None, 1e-5, empty_like(x), mean, inv)
        dx = empty_like(x); ds = torch.full((cols,), 5.0, device="cuda"); do = torch.full((cols,), 5.0, device="cuda")
        DiffLayerNormPerRow(x, dy, scale, mean, inv, dx, ds, do)
        want, wds, wdo, xhat, gg = reference_backward(x, dy, scale, mean, inv)
        assert untouched(dx)
        r = inv.double()[:, None]; sums = gg.abs().mean(1, keepdim=True) + xhat.abs() * (gg * xhat).abs().mean(1, keepdim=True)
        # x - mean loses a step of x, relative to a difference that may be small: counted as 2 U32 |x| inv_std in xhat
        hat = 2 * U32 * x.double().abs() * r
        off = r * (C(cols) * (gg.abs() + sums) + hat * (gg * xhat).abs().mean(1, keepdim=True) + xhat.abs() * (gg.abs() * hat).mean(1, keepdim=True))
        assert_within(dx, want, half_step(dtype) * (want.abs() + off) + off + (2.0 ** -25 if dtype == torch.float16 else 0.0), "dx")
        # sums over rows: at most rows / 4 + 300 terms one after another
        R = (rows / 4 + 300) * U32
        assert_within(ds, wds, R * (dy.double() * xhat).abs().sum(0) + (dy.double().abs() * hat).sum(0) + 1e-30, "scale_deriv")
        assert_within(do, wdo, R * dy.double().abs().sum(0) + 1e-30, "offset_deriv")
        again = torch.ones_like(ds); DiffLayerNormPerRow(x, dy, scale, mean, inv, None, again, None, accumulate=True)
        assert_within(again, ds.double() + 1.0, 2 * U32 * (ds.double().abs() + 2.0), "accumulated")
        only = torch.empty_like(do); DiffLayerNormPerRow(x, dy, scale, mean, inv, offset_deriv=only); assert torch.equal(only, do)
        place = empty_like(dy); place.copy_(dy); DiffLayerNormPerRow(x, place, scale, mean, inv, place, ds2 := torch.empty_like(ds)); assert torch.equal(place, dx) and torch.equal(ds2, ds)      # over out_deriv
        xx = empty_like(x); xx.copy_(x); DiffLayerNormPerRow(xx, dy, scale, mean, inv, xx, ds2, do2 := torch.empty_like(do)); assert torch.equal(xx, dx) and torch.equal(ds2, ds) and torch.equal(do2, do)      # over in_value

def test_derivatives_match_differences():
    """f = sum(c y) along random directions of x, scale and offset, by central differences of the float64 formula: truncation h^2 f''' / 6, taken as 1e-6 of the terms' magnitude at
    h = 1e-4, above the float32 error of the derivatives (C)"""
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    g = generator(5); rows, cols, h = 6, 77, 1e-4
    x = torch.randn(rows, cols, generator=g, device="cuda"); scale = torch.randn(cols, generator=g, device="cuda"); offset = torch.randn(cols, generator=g, device="cuda"); c = torch.randn(rows, cols, generator=g, device="cuda")
    mean = torch.empty(rows, device="cuda"); inv = torch.empty(rows, device="cuda"); LayerNormPerRow(x, scale, offset, 1e-5, torch.empty_like(x), mean, inv)
    dx = torch.empty_like(x); ds = torch.empty(cols, device="cuda"); do = torch.empty(cols, device="cuda"); DiffLayerNormPerRow(x, c, scale, mean, inv, dx, ds, do)
    f = lambda x, s, o: (reference(x, s, o, 1e-5)[0] * c.double()).sum()  # noqa: E731
    for _ in range(4):
        vx, vs, vo = (torch.randn(t.shape, generator=g, device="cuda").double() for t in (x, scale, offset))
        diff = (f(x.double() + h * vx, scale.double() + h * vs, offset.double() + h * vo) - f(x.double() - h * vx, scale.double() - h * vs, offset.double() - h * vo)) / (2 * h)
        terms = torch.cat([(dx.double() * vx).reshape(-1), ds.double() * vs, do.double() * vo])
        assert abs(terms.sum() - diff) <= (1e-6 + C(cols)) * terms.abs().sum()

def test_edges():
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    # rows of one value: y = offset exactly, finite derivative; no rows; a NaN stays in its row
    x = torch.full((4, 100), 3.25, device="cuda"); o = torch.randn(100, device="cuda"); y = torch.empty_like(x); m = torch.empty(4, device="cuda"); r = torch.empty(4, device="cuda")
    LayerNormPerRow(x, None, o, 1e-5, y, m, r); assert torch.equal(y, o.expand(4, 100)) and (m == 3.25).all()
    x[2, 5] = float("nan"); LayerNormPerRow(x, None, o, 1e-5, y, m, r); assert torch.isnan(y[2]).all() and torch.equal(y[[0, 1, 3]], o.expand(3, 100))
    e = torch.empty(0, 100, device="cuda"); none = torch.empty(0, device="cuda"); LayerNormPerRow(e, None, None, 1e-5, e, none, none)
    ds = torch.full((100,), 3.0, device="cuda"); DiffLayerNormPerRow(e, e, None, none, none, e, ds, None, accumulate=True); assert (ds == 3.0).all()
    DiffLayerNormPerRow(e, e, None, none, none, e, ds, None); assert (ds == 0.0).all()
    # a large mean beside a small spread: the spread survives (the sum of the squared differences, not of the squares)
    x = 4096.0 + torch.randn(8, 768, generator=generator(1), device="cuda") * 0.5; y = torch.empty_like(x); LayerNormPerRow(x, None, None, 1e-5, y)
    want, _, _, xhat = reference(x, None, None, 1e-5); assert_within(y, want, C(768) * (xhat.abs() + 1.0), "large mean")

def test_long_matrix_offsets_pass_32_bits():
    """more than 2^32 bytes and 2^31 elements into a matrix: the last rows are as those of a short one"""
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    rows, cols = 300000, 8192; x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda"); x[:-8].fill_(1.0); x[-8:].normal_(generator=generator(3)); dy = torch.empty_like(x); dy[:-8].zero_(); dy[-8:].normal_(generator=generator(4))
    m = torch.empty(rows, device="cuda"); r = torch.empty(rows, device="cuda"); y = torch.empty_like(x); LayerNormPerRow(x, None, None, 1e-5, y, m, r)
    t = x[-8:].clone(); y2 = torch.empty_like(t); m2 = torch.empty(8, device="cuda"); r2 = torch.empty(8, device="cuda"); LayerNormPerRow(t, None, None, 1e-5, y2, m2, r2); assert torch.equal(y[-8:], y2) and torch.equal(m[-8:], m2)
    dx = torch.empty_like(x); ds = torch.empty(cols, device="cuda"); DiffLayerNormPerRow(x, dy, None, m, r, dx, ds); _, wds, _, xhat, _ = reference_backward(t, dy[-8:], None, m2, r2)
    assert_within(ds, wds, 400 * U32 * (dy[-8:].double() * xhat).abs().sum(0) + 1e-30, "scale_deriv"); dx2 = torch.empty_like(t); DiffLayerNormPerRow(t, dy[-8:].contiguous(), None, m2, r2, dx2); assert torch.equal(dx[-8:], dx2)

def test_captured_and_replayed_on_a_side_stream():
    """forward and backward in a graph, replayed with new inputs and with eager calls of the same shapes between the replays"""
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    g = generator(9); rows, cols = 333, 770
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda"); dy = torch.empty_like(x); scale = torch.randn(cols, generator=g, device="cuda")
    def buffers(): return [torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")]
    def step(b): LayerNormPerRow(x, scale, None, 1e-5, b[0], b[1], b[2]); DiffLayerNormPerRow(x, dy, scale, b[1], b[2], b[3], b[4], b[5])
    a, b = buffers(), buffers(); x.normal_(generator=g); dy.normal_(generator=g); step(a); torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph): step(a)
    for _ in range(4):
        x.normal_(generator=g); dy.normal_(generator=g); torch.cuda.synchronize(); graph.replay(); step(b); torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream()); c = buffers()
    with torch.cuda.stream(s): step(c)
    torch.cuda.current_stream().wait_stream(s); torch.cuda.synchronize(); assert all(torch.equal(p, q) for p, q in zip(c, b))
