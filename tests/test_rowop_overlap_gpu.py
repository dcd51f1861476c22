"""GPU tests of the operators on rows of matrices with operands that share a buffer without sharing an element of it: results are those of operands of their own."""
import torch, pytest
from tests.rowop_cases import generator
pytestmark = pytest.mark.gpu

def beside(*shapes, dtype, gap=0):
    """matrices of equal numbers of rows as columns of one buffer, `gap` elements apart"""
    base = torch.full((shapes[0][0], sum(c + gap for _, c in shapes)), 77.0, dtype=dtype, device="cuda"); at = 0; out = []
    for _, c in shapes: out.append(base[:, at:at + c]); at += c + gap
    return out

def test_affine_layer_within_one_buffer():
    from kaldi_amd.cumatrix import AffinePerRow, DiffAffinePerRow
    for dtype in (torch.float16, torch.bfloat16):
        for R, K, C, gap in ((300, 64, 136, 0), (37, 41, 19, 3), (1, 64, 8, 0)):
            g = generator(R); x, y, pre, r, dx, dy = beside((R, K), (R, C), (R, C), (R, C), (R, K), (R, C), dtype=dtype, gap=gap); w = torch.randn(C, K, generator=g, device="cuda").to(dtype); b = torch.randn(C, generator=g, device="cuda")
            for t in (x, r, dy): t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            own = [t.clone() for t in (x, r, dy)]; y2, pre2, dx2 = (torch.empty_like(t.contiguous()) for t in (y, pre, dx)); AffinePerRow(x, w, b, "gelu", r, y, pre); AffinePerRow(own[0], w, b, "gelu", own[1], y2, pre2)
            assert torch.equal(y, y2) and torch.equal(pre, pre2)
            dw, db, dw2, db2 = torch.empty_like(w), torch.empty_like(b), torch.empty_like(w), torch.empty_like(b); DiffAffinePerRow(x, w, pre, "gelu", dy, dx, dw, db); DiffAffinePerRow(own[0], w, pre2, "gelu", own[2], dx2, dw2, db2)
            assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2) and all(torch.equal(p, q) for p, q in zip((x, r, dy), own))
            # every second row of a buffer, and rows in front of each other
            rows = torch.empty(2 * R, C, dtype=dtype, device="cuda"); rows[::2] = r; AffinePerRow(x, w, b, "gelu", rows[::2], rows[1::2]); assert torch.equal(rows[1::2], y2) and torch.equal(rows[::2], own[1])
            rows = torch.empty(2 * R, C, dtype=dtype, device="cuda"); rows[R:] = r; AffinePerRow(x, w, b, "gelu", rows[R:], rows[:R]); assert torch.equal(rows[:R], y2)
            AffinePerRow(x, w, b, "gelu", r, r); assert torch.equal(r, y2)

def test_affine_layer_in_the_gaps_of_another_stride():
    """a matrix of two wide rows, and the other one's rows of another stride between and behind them"""
    from kaldi_amd.cumatrix import AffinePerRow
    g = generator(1); base = torch.full((400,), 77.0, dtype=torch.float16, device="cuda"); x = base.as_strided((2, 40), (200, 1), 0); y = base.as_strided((2, 24), (220, 1), 50); x.copy_(torch.randn(2, 40, generator=g, device="cuda")); w = torch.randn(24, 40, generator=g, device="cuda").half()
    own, want = x.contiguous(), torch.empty(2, 24, dtype=torch.float16, device="cuda"); AffinePerRow(own, w, None, "none", None, want); AffinePerRow(x, w, None, "none", None, y); assert torch.equal(y, want) and torch.equal(x, own)

def test_layer_norm_within_one_buffer():
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for R, C, gap in ((50, 136, 0), (37, 19, 3), (1, 64, 0), (9, 20011, 1)):
            g = generator(C); x, y, dy, dx = beside((R, C), (R, C), (R, C), (R, C), dtype=dtype, gap=gap); x.copy_(torch.randn(R, C, generator=g, device="cuda")); dy.copy_(torch.randn(R, C, generator=g, device="cuda")); stats = torch.empty(2, R, device="cuda"); vectors = torch.randn(4, C, generator=g, device="cuda")
            ox, ody, oy, odx = x.clone(), dy.clone(), torch.empty_like(x.contiguous()), torch.empty_like(x.contiguous()); om, oi, ods, odo = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
            LayerNormPerRow(ox, vectors[0].clone(), vectors[1].clone(), 1e-5, oy, om, oi); DiffLayerNormPerRow(ox, ody, vectors[0].clone(), om, oi, odx, ods, odo)
            LayerNormPerRow(x, vectors[0], vectors[1], 1e-5, y, stats[0], stats[1]); DiffLayerNormPerRow(x, dy, vectors[0], stats[0], stats[1], dx, vectors[2], vectors[3])      # the vectors are neighbours too
            assert torch.equal(y, oy) and torch.equal(stats[0], om) and torch.equal(stats[1], oi) and torch.equal(dx, odx) and torch.equal(vectors[2], ods) and torch.equal(vectors[3], odo) and torch.equal(x, ox) and torch.equal(dy, ody)
            DiffLayerNormPerRow(x, dy, vectors[0], stats[0], stats[1], dy); assert torch.equal(dy, odx); LayerNormPerRow(x, vectors[0], vectors[1], 1e-5, x); assert torch.equal(x, oy)

def test_scores_and_distillation_within_one_buffer():
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs, ComputeDistillObjfAndDeriv, DistillationOptions
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for R, C, gap in ((50, 136, 0), (37, 19, 3), (1, 6024, 0), (9, 20011, 1), (2, 140001, 0)):
            g = generator(C); z, dz, v, dd = beside((R, C), (R, C), (R, 5), (R, C), dtype=dtype, gap=gap); z.copy_(torch.randn(R, C, generator=g, device="cuda")); v.copy_(torch.randn(R, 5, generator=g, device="cuda"))
            i = torch.randint(-1, C, (R, 5), generator=g, device="cuda").to(torch.int32); y = i[:, 0].contiguous(); vectors = torch.rand(6, R, generator=g, device="cuda"); st = torch.empty(R, 2, device="cuda")
            oz, ov, o = z.clone(), v.clone(), [t.clone() for t in vectors]; odz, odd, ost = torch.empty_like(z.contiguous()), torch.empty_like(z.contiguous()), torch.empty_like(st); opt = DistillationOptions(2.0)
            LabelLogProbs(oz, y, o[0], o[1], ost); DiffLabelLogProbs(oz, y, ost, o[1], o[2], o[3], odz); ComputeDistillObjfAndDeriv(opt, oz, ov, i, o[4], o[5], odd)
            LabelLogProbs(z, y, vectors[0], vectors[1], st); DiffLabelLogProbs(z, y, st, vectors[1], vectors[2], vectors[3], dz); ComputeDistillObjfAndDeriv(opt, z, v, i, vectors[4], vectors[5], dd)
            assert torch.equal(vectors, torch.stack(o)) and torch.equal(st, ost) and torch.equal(dz, odz) and torch.equal(dd, odd) and torch.equal(z, oz) and torch.equal(v, ov)
            DiffLabelLogProbs(z, y, st, vectors[1], vectors[2], vectors[3], z); assert torch.equal(z, odz); z.copy_(oz); ComputeDistillObjfAndDeriv(opt, z, v, i, vectors[4], vectors[5], z); assert torch.equal(z, odd)
