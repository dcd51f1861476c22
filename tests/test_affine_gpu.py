"""GPU tests of the half-precision affine layer (k3_affine_*, cumatrix.AffinePerRow / DiffAffinePerRow) against the formulas in float64, and of its derivatives against differences.

Bounds.  Products of two halves are exact in float32; a sum of k of them, in whatever order, is off by at most k half steps U of float32 times the sum of their magnitudes |x| |W|^T (the
matrix cores may cut instead of rounding: 2 k U).  An activation changes by at most 1.2 of that (the largest slope, swish's and gelu's, is below 1.2), is itself within 16 U of its
argument's size, and the result is rounded once.  Where an activation is undone, dz = dy act'(pre) is rounded before the products: half a step of the type times |dz| |W| (or |dz|^T |x|)."""
import math, pytest, torch
from tests.rowop_cases import U32, half_step, matrix, empty_like, untouched, assert_within, generator
pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
# rows, inner, cols: one of each, below a matrix instruction, odd everywhere, at and around the tiles, long contractions in parts, few rows by many columns and the other way round
SIZES = [(1, 1, 1), (1, 64, 6024), (2, 7, 5), (17, 768, 129), (16, 32, 64), (33, 65, 66), (64, 64, 64), (65, 63, 130), (5, 4000, 24), (128, 128, 128), (129, 200, 255), (250, 72, 264), (256, 192, 256),
         (300, 96, 1000), (1000, 160, 40), (513, 520, 776), (40, 6024, 96), (4096, 64, 3), (2500, 256, 700)]

def act64(name, z):
    return {"none": z, "relu": z.clamp(min=0), "sigmoid": torch.sigmoid(z), "tanh": torch.tanh(z), "swish": z * torch.sigmoid(z), "gelu": 0.5 * z * torch.erfc(-z / math.sqrt(2))}[name]
def slope64(name, z):
    s = torch.sigmoid(z)
    return {"none": torch.ones_like(z), "relu": (z > 0).double(), "sigmoid": s * (1 - s), "tanh": 1 / torch.cosh(z) ** 2, "swish": s * (1 + z * (1 - s)),
            "gelu": 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[name]

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,inner,cols", SIZES)
def test_forward_matches_the_formula(rows, inner, cols, dtype):
    from kaldi_amd.cumatrix import AffinePerRow
    g = generator(rows * 10007 + inner * 101 + cols)
    for pad, act, bias, residual in ((0, "none", False, False), (8, "relu", True, True), (3, "gelu", True, False), (0, "swish", True, True), (1, "tanh", False, True), (0, "sigmoid", True, False)):
        x = matrix(g, rows, inner, dtype, pad); w = matrix(g, cols, inner, dtype, pad, inner ** -0.5, pad % 2); b = torch.randn(cols, generator=g, device="cuda") if bias else None
        r = matrix(g, rows, cols, dtype, pad) if residual else None; y = matrix(g, rows, cols, dtype, pad); y._base.fill_(77.0); pre = empty_like(y) if act != "none" else None
        AffinePerRow(x, w, b, act, r, y, pre); assert untouched(y)
        z = x.double() @ w.double().t(); size = x.double().abs() @ w.double().abs().t()
        if b is not None: z = z + b.double(); size = size + b.double().abs()
        off = 2 * (inner + 4) * U32 * size
        if pre is not None: assert untouched(pre); assert_within(pre, z, half_step(dtype) * (z.abs() + off) + off + TINY[dtype], "pre")
        want = act64(act, z); off = 1.2 * off + 16 * U32 * (z.abs() + 1)
        if r is not None: want = want + r.double(); off = off + 2 * U32 * r.double().abs()
        assert_within(y, want, half_step(dtype) * (want.abs() + off) + off + TINY[dtype], "y")
        if r is not None: AffinePerRow(x, w, b, act, r, r); assert torch.equal(r, y)      # over the residual, and without keeping what goes into the activation

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,inner,cols", SIZES)
def test_backward_matches_the_formula(rows, inner, cols, dtype):
    from kaldi_amd.cumatrix import DiffAffinePerRow
    g = generator(rows * 10007 + inner * 101 + cols + 1)
    for pad, act in ((0, "none"), (3, "none"), (0, "relu"), (8, "gelu"), (1, "swish"), (0, "tanh"), (0, "sigmoid")):
        x = matrix(g, rows, inner, dtype, pad); w = matrix(g, cols, inner, dtype, pad, inner ** -0.5); dy = matrix(g, rows, cols, dtype, pad, 0.5); pre = matrix(g, rows, cols, dtype, pad) if act != "none" else None
        dx, dw, db = empty_like(x), empty_like(w), torch.full((cols,), 5.0, device="cuda"); DiffAffinePerRow(x, w, pre, act, dy, dx, dw, db); assert untouched(dx) and untouched(dw)
        s = torch.ones_like(dy, dtype=torch.float64) if pre is None else slope64(act, pre.double()); dz = dy.double() * s
        # an activation's slope is off by 16 U of 1 + |z|
        rough = torch.zeros_like(dz) if act == "none" else 16 * U32 * dy.double().abs() * (1 + pre.double().abs()); rounded = rough if act in ("none", "relu") else rough + half_step(dtype) * (dz.abs() + rough) + TINY[dtype]
        want = dz @ w.double(); off = (2 * (cols + 4) * U32 * dz.abs() + rounded * 1.01) @ w.double().abs()
        assert_within(dx, want, half_step(dtype) * (want.abs() + off) + off + TINY[dtype], "dx")
        want = dz.t() @ x.double(); off = (2 * (rows + 4) * U32 * dz.abs() + rounded * 1.01).t() @ x.double().abs()
        assert_within(dw, want, half_step(dtype) * (want.abs() + off) + off + TINY[dtype], "dw")
        assert_within(db, dz.sum(0), ((rows + 4) * U32 * dz.abs() + rough * 1.01).sum(0) + 1e-30, "db")
        only = torch.empty_like(db); DiffAffinePerRow(x, w, pre, act, dy, bias_params_deriv=only); assert torch.equal(only, db)
        a = empty_like(dx); DiffAffinePerRow(x, w, pre, act, dy, a); assert torch.equal(a, dx)
        a = empty_like(dw); DiffAffinePerRow(x, w, pre, act, dy, None, a); assert torch.equal(a, dw)

@pytest.mark.parametrize("dtype", HALVES)
def test_values_behind_the_edges_do_not_come_in(dtype):
    """NaNs and infinities around every operand (in the padding of the rows, behind the last one): results are those of clean surroundings"""
    from kaldi_amd.cumatrix import AffinePerRow, DiffAffinePerRow
    g = generator(11)
    for rows, inner, cols in ((70, 72, 136), (33, 40, 50), (257, 264, 300), (129, 100, 127)):
        for pad in (8, 3):
            def dirty(r, c, value):
                base = torch.full((r + 2, c + pad), value, dtype=dtype, device="cuda"); v = base[:r, :c]; v.copy_(torch.randn(r, c, generator=g, device="cuda")); return v
            for value in (float("nan"), float("inf")):
                x, w, dy = dirty(rows, inner, value), dirty(cols, inner, value), dirty(rows, cols, value); cx, cw, cdy = x.contiguous(), w.contiguous(), dy.contiguous()
                y, cy = torch.empty(rows, cols, dtype=dtype, device="cuda"), torch.empty(rows, cols, dtype=dtype, device="cuda"); AffinePerRow(x, w, None, "none", None, y); AffinePerRow(cx, cw, None, "none", None, cy)
                assert torch.equal(y, cy)
                d, c = [torch.empty_like(cx), torch.empty_like(cw), torch.empty(cols, device="cuda")], [torch.empty_like(cx), torch.empty_like(cw), torch.empty(cols, device="cuda")]
                DiffAffinePerRow(x, w, None, "none", dy, *d); DiffAffinePerRow(cx, cw, None, "none", cdy, *c); assert all(torch.equal(p, q) for p, q in zip(d, c))

def test_values_that_are_not_finite_stay_where_they_belong():
    from kaldi_amd.cumatrix import AffinePerRow, DiffAffinePerRow
    g = generator(12); x = torch.randn(200, 96, generator=g, device="cuda").bfloat16(); w = torch.randn(80, 96, generator=g, device="cuda").bfloat16(); x[7, 3] = float("nan"); w[5, 2] = float("inf"); x[:, 2] = 1.0
    for act in ("none", "relu", "sigmoid", "tanh", "swish", "gelu"):
        y = torch.empty(200, 80, dtype=torch.bfloat16, device="cuda"); pre = torch.empty_like(y); AffinePerRow(x, w, None, act, None, y, pre); keep = torch.ones(200, dtype=torch.bool, device="cuda"); keep[7] = False
        assert torch.isnan(y[7].float()).all() and torch.isfinite(y[keep][:, 6:]).all() and (y[keep][:, 5] == (1.0 if act in ("sigmoid", "tanh") else float("inf"))).all()
    big = torch.tensor([[-300.0, -88.0, -20.0, -5.0, 0.0, 5.0, 20.0, 88.0, 300.0, 60000.0, -60000.0]], device="cuda").half(); one = torch.ones(1, 11, device="cuda").half(); x1 = torch.ones(1, 1, device="cuda").half(); w1 = torch.ones(11, 1, device="cuda").half()
    for act in ("relu", "sigmoid", "tanh", "swish", "gelu"):
        db = torch.empty(11, device="cuda"); DiffAffinePerRow(x1, w1, big, act, one, bias_params_deriv=db); want = slope64(act, big.double())[0].nan_to_num(); assert_within(db, want, 16 * U32 * (1 + big.double()[0].abs().clamp(max=100)) , act)

def test_derivatives_match_differences():
    """f = sum(c y) along random directions of x, W and b through gelu and a residual, by central differences of the float64 formula with h = 1e-4 (h^2 f''' / 6 within 1e-6 of the terms), against the
    derivatives in float16: their rounding, half a step each way of dz and of the result, adds up to at most 2^-10 of the terms' magnitudes"""
    from kaldi_amd.cumatrix import AffinePerRow, DiffAffinePerRow
    g = generator(5); rows, inner, cols, h = 9, 33, 21, 1e-4
    x = torch.randn(rows, inner, generator=g, device="cuda").half(); w = (torch.randn(cols, inner, generator=g, device="cuda") / 6).half(); b = torch.randn(cols, generator=g, device="cuda"); c = torch.randn(rows, cols, generator=g, device="cuda").half()
    y, pre = torch.empty_like(c), torch.empty_like(c); AffinePerRow(x, w, b, "gelu", c, y, pre); dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(cols, device="cuda"); DiffAffinePerRow(x, w, pre, "gelu", c, dx, dw, db)
    f = lambda x, w, b: (act64("gelu", x @ w.t() + b) * c.double()).sum()  # noqa: E731
    for _ in range(4):
        vx, vw, vb = (torch.randn(t.shape, generator=g, device="cuda").double() for t in (x, w, b))
        diff = (f(x.double() + h * vx, w.double() + h * vw, b.double() + h * vb) - f(x.double() - h * vx, w.double() - h * vw, b.double() - h * vb)) / (2 * h)
        terms = torch.cat([(dx.double() * vx).reshape(-1), (dw.double() * vw).reshape(-1), db.double() * vb])
        # pre is rounded too: half a step of it times the second derivative (below 0.8) times |c| |direction|
        size = (vx.abs() @ w.double().abs().t() + x.double().abs() @ vw.abs().t() + vb.abs()) * c.double().abs()
        assert abs(terms.sum() - diff) <= 2.0 ** -10 * (size * 1.2).sum() + 2.0 ** -11 * (pre.double().abs() * 0.8 * size).sum() + 1e-6 * terms.abs().sum()

def test_no_rows():
    from kaldi_amd.cumatrix import AffinePerRow, DiffAffinePerRow
    x = torch.empty(0, 8, device="cuda").half(); y = torch.empty(0, 24, device="cuda").half(); w = torch.ones(24, 8, device="cuda").half(); AffinePerRow(x, w, None, "relu", None, y, y)
    dw, db = torch.ones_like(w), torch.ones(24, device="cuda"); DiffAffinePerRow(x, w, y, "relu", y, x, dw, db); assert not dw.any() and not db.any()

def test_captured_replayed_and_on_a_side_stream():
    from kaldi_amd.cumatrix import AffinePerRow, DiffAffinePerRow
    g = generator(9)
    for rows, inner, cols in ((17, 768, 1000), (700, 200, 520)):
        x = torch.empty(rows, inner, dtype=torch.bfloat16, device="cuda"); w = torch.randn(cols, inner, generator=g, device="cuda").bfloat16(); bias = torch.randn(cols, generator=g, device="cuda"); dy = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
        def buffers(): return [torch.empty_like(dy), torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w), torch.empty_like(bias)]
        def step(b): AffinePerRow(x, w, bias, "gelu", dy, b[0], b[1]); DiffAffinePerRow(x, w, b[1], "gelu", dy, b[2], b[3], b[4])
        a, b = buffers(), buffers(); x.normal_(generator=g); dy.normal_(generator=g); step(a); torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph): step(a)
        for _ in range(4):
            x.normal_(generator=g); dy.normal_(generator=g); torch.cuda.synchronize(); graph.replay(); step(b); torch.cuda.synchronize(); assert all(torch.equal(p, q) for p, q in zip(a, b))
        s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream()); c = buffers()
        with torch.cuda.stream(s): step(c)
        torch.cuda.synchronize(); assert all(torch.equal(p, q) for p, q in zip(c, b))
