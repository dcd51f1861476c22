"""GPU tests of the operators on rows of matrices with more rows than one dimension of a launch has wavefronts or workgroups for: every row is as in a call on a part of the rows."""
import torch, pytest
from tests.rowop_cases import generator
pytestmark = pytest.mark.gpu

@pytest.fixture(autouse=True)
def memory_given_back():
    yield
    torch.cuda.empty_cache()

def test_scores_and_distillation_of_short_rows():
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs, ComputeDistillObjfAndDeriv, DistillationOptions
    R, C = (1 << 26) + 77, 3; half = R // 2; g = generator(1); z = torch.randn(R, C, generator=g, device="cuda", dtype=torch.float16); y = torch.randint(-1, C, (R,), generator=g, device="cuda", dtype=torch.int32); t = torch.randn(R, 1, generator=g, device="cuda", dtype=torch.float16)
    lp, h, st, ai = torch.full((R,), 7.0, device="cuda"), torch.full((R,), 7.0, device="cuda"), torch.full((R, 2), 7.0, device="cuda"), torch.full((R, 1), 7, dtype=torch.int32, device="cuda"); LabelLogProbs(z, y, lp, h, st, None, ai)
    dz = torch.full_like(z, 7.0); DiffLabelLogProbs(z, y, st, h, lp, h, dz); f, dd = torch.full((R,), 7.0, device="cuda"), torch.full_like(z, 7.0); ComputeDistillObjfAndDeriv(DistillationOptions(), z, t, y[:, None], None, f, dd)
    for s in (slice(0, half), slice(half, R)):
        n = s.stop - s.start; lp2, h2, st2, ai2 = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda"), torch.empty(n, 1, dtype=torch.int32, device="cuda"); LabelLogProbs(z[s], y[s], lp2, h2, st2, None, ai2)
        assert torch.equal(lp[s], lp2) and torch.equal(h[s], h2) and torch.equal(st[s], st2) and torch.equal(ai[s], ai2)
        dz2 = torch.empty(n, C, device="cuda", dtype=torch.float16); DiffLabelLogProbs(z[s], y[s], st2, h2, lp2, h2, dz2); assert torch.equal(dz[s], dz2); ComputeDistillObjfAndDeriv(DistillationOptions(), z[s], t[s], y[s][:, None], None, lp2, dz2); assert torch.equal(f[s], lp2) and torch.equal(dd[s], dz2)

def test_scores_of_rows_that_take_a_workgroup():
    from kaldi_amd.objective import LabelLogProbs
    R, C = (1 << 24) + 5, 4097; z = torch.zeros(R, C, dtype=torch.bfloat16, device="cuda"); pick = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, 5 << 20, (1 << 24) - 1, 1 << 24, R - 1], device="cuda"); z[pick] = torch.randn(len(pick), C, generator=generator(2), device="cuda").bfloat16()
    y = torch.full((R,), 9, dtype=torch.int32, device="cuda"); lp, h = torch.full((R,), 7.0, device="cuda"), torch.full((R,), 7.0, device="cuda"); LabelLogProbs(z, y, lp, h)
    # (as many rows as make the call on a part take one workgroup per row too)
    part = z[: 1 << 10].clone(); part[: len(pick)] = z[pick]; lp2, h2 = torch.empty(1 << 10, device="cuda"), torch.empty(1 << 10, device="cuda"); LabelLogProbs(part, y[: 1 << 10], lp2, h2)
    assert torch.equal(lp[pick], lp2[: len(pick)]) and torch.equal(h[pick], h2[: len(pick)]); keep = torch.ones(R, dtype=torch.bool, device="cuda"); keep[pick] = False; assert (lp[keep] == lp2[-1]).all() and (h[keep] == h2[-1]).all()

def test_affine_layer_of_one_column():
    from kaldi_amd.cumatrix import AffinePerRow
    R = (1 << 29) + 77; x = torch.empty(R, 1, dtype=torch.float16, device="cuda"); x.normal_(generator=generator(3)); w = torch.full((1, 1), 0.5, dtype=torch.float16, device="cuda"); y = torch.full_like(x, 7.0); AffinePerRow(x, w, torch.ones(1, device="cuda"), "none", None, y)
    for s in range(0, R, 1 << 27): assert torch.equal(y[s:s + (1 << 27)], (x[s:s + (1 << 27)].float() * 0.5 + 1.0).half())      # (x / 2 is exact, and the sum is rounded to float32 and then to float16 on both sides)
