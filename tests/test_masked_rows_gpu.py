"""GPU tests of the label scores and of distillation on rows of which a range of columns holds the type's lowest value, as masks do that are added or filled in (kaldi_amd.objective), against
the formulas in float64.

Bounds: those of the tests with ordinary values, S(n, D) = (n / 64 + 2 D + 40) half steps of float32, with D = 40 (a column further below the row's largest adds less than 2^-57 of the
sum, masked ones nothing)."""
import pytest, torch
from tests.rowop_cases import TYPES, U32, half_step, empty_like, untouched, assert_within, generator
pytestmark = pytest.mark.gpu

def S(n, D=40): return (n / 64 + 2 * D + 40) * U32
def tiny(dtype): return 2.0 ** -25 if dtype == torch.float16 else 1e-30

def masked_rows(cols, dtype):
    """rows with a masked head, tail, middle, everything but the first or the last column, every third range of 2048 columns, everything, and nothing; the rest is of unit size"""
    z = torch.randn(8, cols, generator=generator(cols), device="cuda").to(dtype); low = torch.finfo(dtype).min; c = torch.arange(cols, device="cuda"); third = cols // 3
    for r, m in enumerate((c < third, c >= cols - third, (c >= third) & (c < 2 * third), c > 0, c < cols - 1, c // 2048 % 3 == 1, c >= 0)): z[r] = torch.where(m, torch.full_like(z[r], low), z[r])
    return z

# one part per row; parts of few rows (2048 columns and more); parts that a workgroup holds of float32, of halves; the most columns
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [300, 4096, 9001, 16385, 40000, 70001, 131073, 1 << 19])
def test_scores_and_their_derivative(cols, dtype):
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs
    z = masked_rows(cols, dtype); n = z.shape[0]; y = torch.tensor([cols - 1, 0, cols // 2, 0, cols - 1, 1, 7, -1], dtype=torch.int32, device="cuda"); y[2] = 0
    lp, h, st = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, 2, device="cuda"); LabelLogProbs(z, y, lp, h, st)
    # (the largest value is taken away first: beside the lowest number even float64 has no room for a logarithm)
    m = z.double().amax(1); x = z.double() - m[:, None]; ls = torch.logsumexp(x, 1); lq = x - ls[:, None]; q = lq.exp(); H = -torch.where(q > 0, q * lq, 0.0).sum(1); err = S(cols) + 4 * U32 * ls.abs()
    assert torch.equal(st[:, 0].double(), m); assert_within(st[:, 1], ls, err, "log sum")
    want = torch.where(y >= 0, lq.gather(1, y.long().clamp(min=0)[:, None])[:, 0], 0.0); assert_within(lp, want, err + 3 * U32 * want.abs(), "log prob")
    assert_within(h, H, err + (S(cols) + 8 * U32) * (H + ls), "entropy")
    a, b = torch.randn(n, generator=generator(1), device="cuda"), torch.randn(n, generator=generator(2), device="cuda"); dz = empty_like(z); DiffLabelLogProbs(z, y, st, h, a, b, dz); assert untouched(dz)
    ga, gb = torch.where(y >= 0, a, 0.0).double()[:, None], b.double()[:, None]; inner = lq.clamp(min=-1e4) + H[:, None]; want = -q * (ga + gb * inner); want[torch.arange(n, device="cuda"), y.long().clamp(min=0)] += ga[:, 0]
    e = S(cols) + 4 * U32 * (ls[:, None].abs() + 101.0); off = q * (e + 4 * U32) * (ga.abs() + gb.abs() * (inner.abs() + H[:, None] + ls[:, None].abs() + 2)) + 4 * U32 * want.abs() + 2 * U32 * ga.abs() * (want.abs() > 0)
    assert_within(dz, want, half_step(dtype) * (want.abs() + off) + off + tiny(dtype), "dz")

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [300, 4096, 9001, 70001, 140001])
def test_distillation_with_entries_at_masked_columns(cols, dtype):
    """the objective there is w T p (z - M), within the range of float32 for the probabilities chosen, though not (z - M) / T for T < 1.44.  The differences are off by a few half steps
    of their sizes, which S covers as it does for ordinary ones"""
    from kaldi_amd.objective import ComputeDistillObjfAndDeriv, DistillationOptions
    z = masked_rows(cols, dtype); n, c = z.shape[0], cols // 2; g = generator(cols + 1); third = cols // 3
    # columns in every range: most of each row's entries are at masked ones in some row, with probabilities of a tenth or less; the teacher has a masked entry of its own
    idx = torch.tensor([[0, c, cols - 1, 1, c + 1, cols - 2, third, -1]], dtype=torch.int32, device="cuda").repeat(n, 1); idx[7, 0] = 5
    t = torch.tensor([[4.0, 1.0, 0.5, 0.2, 0.1, float(torch.finfo(dtype).min), 0.3, 9.0]], device="cuda").to(dtype).repeat(n, 1); order = torch.tensor([2, 0, 0, 0, 2, 0, 1, 0])
    for r in range(n): k = int(order[r]); t[r, [0, k]] = t[r, [k, 0]]
    w = torch.tensor([1.0, 0.5, -0.25, 1.0, 0.5, 1.0, 1.0, 2.0], device="cuda"); f, dz, alone = torch.empty(n, device="cuda"), empty_like(z), torch.empty(n, device="cuda")
    for T in (0.5, 1.0, 1.4, 2.0):
        o = DistillationOptions(T); ComputeDistillObjfAndDeriv(o, z, t, idx, w, f, dz); ComputeDistillObjfAndDeriv(o, z, t, idx, w, alone); assert untouched(dz)
        used = idx >= 0; at = idx.long().clamp(min=0); tt = torch.where(used, t.double(), -float("inf")) / T; tt = tt - tt.amax(1, keepdim=True); lp = tt - torch.logsumexp(tt, 1, keepdim=True); p = torch.where(used, lp.exp(), 0.0)
        x = (z.double() - z.double().amax(1, keepdim=True)) / T; lq = x - torch.logsumexp(x, 1, keepdim=True); lqk = lq.gather(1, at); D = 40.0 + 8.0 / T; e = S(cols, D) + S(64, D)
        want = w.double() * T * T * torch.where(p > 0, p * (lqk - lp), 0.0).sum(1); mag = w.double().abs() * T * T * torch.where(p > 0, p * (lqk.abs() + lp.abs() + 1), 0.0).sum(1); assert (want.abs() < 3.4e38).all()
        if dtype != torch.float16: assert (want.abs() > 1e30).sum() >= 4      # (masked columns do count: ordinary ones give less than 100)
        assert_within(f, want, e * mag, "objf"); assert_within(alone, want, e * mag, "objf alone")
        P = torch.zeros_like(lq).scatter_add_(1, at, p); d = w.double()[:, None] * T * (P - lq.exp()); off = e * w.double().abs()[:, None] * T * (P + lq.exp())
        assert_within(dz, d, half_step(dtype) * (d.abs() + off) + off + tiny(dtype), "dz")

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [67, 489, 9001, 20794, 140001])
def test_distillation_with_all_entries_at_masked_columns(cols, dtype):
    """the probabilities add up to 1 but for their roundings, and the objective to w T (lowest - M): finite, as the bounds above have it, where w T is below 1"""
    from kaldi_amd.objective import ComputeDistillObjfAndDeriv, DistillationOptions
    g = generator(cols); n, N, c = 64, 40, cols // 2; z = torch.randn(n, cols, generator=g, device="cuda").to(dtype); z[:, c:] = torch.finfo(dtype).min; idx = torch.randint(c, cols, (n, N), generator=g, device="cuda").to(torch.int32)
    t = torch.randn(n, N, generator=g, device="cuda").to(dtype); w = (0.1 + 0.3 * torch.rand(n, generator=g, device="cuda")); f, dz, alone = torch.empty(n, device="cuda"), empty_like(z), torch.empty(n, device="cuda")
    for T in (0.5, 1.0, 2.0):
        o = DistillationOptions(T); ComputeDistillObjfAndDeriv(o, z, t, idx, w, f, dz); ComputeDistillObjfAndDeriv(o, z, t, idx, w, alone); D = 40.0 + 8.0 / T; e = S(cols, D) + S(64, D)
        lp = torch.log_softmax(t.double() / T, 1); x = (z.double() - z.double().amax(1, keepdim=True)) / T; lq = x - torch.logsumexp(x, 1, keepdim=True); p = lp.exp(); lqk = lq.gather(1, idx.long())
        want = w.double() * T * T * (p * (lqk - lp)).sum(1); off = e * w.double() * T * T * (p * (lqk.abs() + lp.abs() + 1)).sum(1); assert (want.abs() < 2.8e38).all(); assert_within(f, want, off, "objf"); assert_within(alone, want, off, "objf alone")
        P = torch.zeros_like(lq).scatter_add_(1, idx.long(), p); d = w.double()[:, None] * T * (P - lq.exp()); off = e * w.double()[:, None] * T * (P + lq.exp()); assert_within(dz, d, half_step(dtype) * (d.abs() + off) + off + tiny(dtype), "dz")
