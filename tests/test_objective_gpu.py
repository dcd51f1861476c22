"""GPU tests of kaldi_amd.objective (k3_label_logprobs*, k3_distill_objf_and_deriv) against the formulas in float64, and of the derivatives against differences.

Bounds.  With |z - M| <= D over the elements that matter, the exponent's fma and its constant are off by 2 half steps of D, so an exponential is off by (2 D + 4) U relative (v_exp_f32: one
step); a sum of n positive terms taken by 64 lanes or more adds (n / 64 + 16) U.  So s, and what is divided by it, is off by S(n, D) = (n / 64 + 2 D + 40) U relative, a logarithm of it
by S + 4 U of itself; two dozen roundings are within the 40."""
import pytest, torch
from tests.rowop_cases import TYPES, U32, half_step, matrix, empty_like, untouched, assert_within, generator
pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 2), (5, 63), (64, 64), (33, 200), (130, 257), (9, 1000), (40, 2048), (7, 2049), (12, 4097), (50, 6024), (1, 6024), (600, 6024), (6, 8193), (3, 16385), (2, 33000), (700, 10007),
         (3, 65537), (1, 131073), (2, 200003), (600, 20001)]

def S(n, D): return (n / 64 + 2 * D + 40) * U32

def logits(g, rows, cols, dtype, pad=0, scale=2.0, masked=True):
    z = matrix(g, rows, cols, dtype, pad, scale)
    if masked and cols > 4: z[:, 2] = -float("inf"); z[rows // 2, cols // 2:] = -float("inf")
    return z

def scores64(z):
    z = z.double(); m = z.amax(1); lz = torch.logsumexp(z, 1); lq = z - lz[:, None]; q = lq.exp()
    return m, lz - m, lq, q, -torch.where(q > 0, q * lq, 0.0).sum(1)

def best64(z, n):
    """the n largest columns, ties to the lowest: a stable sort of the exact values"""
    return torch.sort(z.double().cpu() + 0.0, dim=1, descending=True, stable=True).indices[:, :n].to(z.device)

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_scores_match_the_formulas(rows, cols, dtype):
    from kaldi_amd.objective import LabelLogProbs
    g = generator(rows * 1000003 + cols)
    for pad, top in ((0, min(cols, 5)), (3, 0), (8, min(cols, 64))):
        z = logits(g, rows, cols, dtype, pad); labels = torch.randint(0, cols, (rows,), generator=g, device="cuda").to(torch.int32); labels[::3] = -1; labels[1::7] = cols
        lp, h, st = (torch.full(s, 7.0, device="cuda") for s in ((rows,), (rows,), (rows, 2)))
        al, ai = (torch.full((rows, top), 7.0, device="cuda"), torch.full((rows, top), 7, dtype=torch.int32, device="cuda")) if top else (None, None)
        LabelLogProbs(z, labels, lp, h, st, al, ai)
        m, ls, lq, q, want_h = scores64(z)
        D = 40.0; e = S(cols, D)      # further below the maximum than 40 an element adds less than 2^-57 of the sum
        assert torch.equal(st[:, 0].double(), m)
        err = e + 4 * U32 * ls.abs() + 1e-30
        assert_within(st[:, 1], ls, err, "log sum")
        has = (labels >= 0) & (labels < cols); at = labels.long().clamp(0, cols - 1)[:, None]
        want = torch.where(has, lq.gather(1, at)[:, 0], 0.0)
        assert_within(lp, want, err + 3 * U32 * (want.abs() + (z.double().gather(1, at)[:, 0] - m).abs().nan_to_num(posinf=0.0)), "log prob")
        # ln s and sum q (M - z) are both positive
        assert_within(h, want_h, err + (e + 8 * U32) * (want_h + ls), "entropy")
        if top:
            idx = best64(z, top); assert torch.equal(ai.long(), idx)
            w = lq.gather(1, idx); assert_within(al, w, err[:, None] + 3 * U32 * (w.abs() + (z.double().gather(1, idx) - m[:, None]).abs()).nan_to_num(posinf=0.0), "alternatives")
        only = torch.empty_like(lp); LabelLogProbs(z, labels, only); assert torch.equal(only, lp)
        if top: b = torch.empty_like(ai); LabelLogProbs(z, None, alt_labels=b); assert torch.equal(b, ai)

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 700, 6024, 50000])
def test_alternatives_of_equal_values_go_by_column(cols, dtype):
    """rows of one value, of two, of a rising and a falling staircase, with zeros of both signs, and with fewer finite values than alternatives: more equal values than are gathered"""
    from kaldi_amd.objective import LabelLogProbs
    g = generator(cols); c = torch.arange(cols, device="cuda").float()
    rows = [torch.full((cols,), 1.5, device="cuda"), (torch.rand(cols, generator=g, device="cuda") < 0.5).float(), torch.floor(c / 50), -torch.floor(c / 50), torch.where(torch.rand(cols, generator=g, device="cuda") < 0.5, 0.0, -0.0),
            torch.where(c % (cols // 3 + 1) == 5, c / cols, -float("inf")), torch.where(c == cols - 1, 1.0, -float("inf")), torch.where(c < 900, 2.0, 1.0) + torch.where(c == 63, 1.0, 0.0)]
    z = torch.stack(rows).to(dtype)
    for n in (1, 7, 64):
        ai = torch.empty(len(rows), n, dtype=torch.int32, device="cuda"); al = torch.empty(len(rows), n, device="cuda"); LabelLogProbs(z, None, alt_log_probs=al, alt_labels=ai)
        idx = best64(z, n); assert torch.equal(ai.long(), idx)
        lq = scores64(z)[2].gather(1, idx); assert_within(al, lq, S(cols, 40) + 8 * U32 * lq.abs().nan_to_num(posinf=0.0), "alternatives")

def test_rows_without_values_and_rows_that_are_not_finite():
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs
    inf, nan = float("inf"), float("nan")
    for dtype in TYPES:
        for cols in (5, 300, 9000, 40000):
            z = torch.randn(6, cols, generator=generator(cols), device="cuda").to(dtype); z[0] = -inf; z[1, 3] = nan; z[2, 4] = inf; z[3] = -inf; z[3, cols - 2] = nan; z[4] = torch.finfo(dtype).min
            labels = torch.full((6,), 3, dtype=torch.int32, device="cuda"); lp, h = torch.empty(6, device="cuda"), torch.empty(6, device="cuda"); st = torch.empty(6, 2, device="cuda")
            al, ai = torch.empty(6, 4, device="cuda"), torch.empty(6, 4, dtype=torch.int32, device="cuda"); LabelLogProbs(z, labels, lp, h, st, al, ai)
            assert lp[0] == -inf and h[0] == 0 and (al[0] == -inf).all() and ai[0].tolist() == [0, 1, 2, 3]
            for r in (1, 2, 3): assert torch.isnan(lp[r]) and torch.isnan(h[r]) and torch.isnan(al[r]).all() and (ai[r] == -1).all()
            # the type's lowest value in every column is a uniform row
            ln = torch.log(torch.tensor(float(cols), dtype=torch.float64, device="cuda")); assert_within(lp[4:5], -ln[None], S(cols, 1) + 4 * U32 * ln, "lowest"); assert_within(h[4:5], ln[None], S(cols, 1) + 4 * U32 * ln, "lowest"); assert ai[4].tolist() == [0, 1, 2, 3]
            assert torch.isfinite(lp[5]) and torch.isfinite(h[5])
            one = torch.ones(6, device="cuda"); dz = empty_like(z); DiffLabelLogProbs(z, labels, st, h, one, one, dz)
            assert (dz[0] == 0).all() and torch.isfinite(dz[4:]).all()
            for r in (1, 2): assert torch.isnan(dz[r].float()).any()

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_score_derivatives_match_the_formulas(rows, cols, dtype):
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs
    g = generator(rows * 1000003 + cols + 1)
    for pad, with_h in ((0, True), (5, False)):
        z = logits(g, rows, cols, dtype, pad); labels = torch.randint(0, cols, (rows,), generator=g, device="cuda").to(torch.int32); labels[::3] = -1; labels[1::7] = cols + 5
        h, st = torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda"); LabelLogProbs(z, None, None, h, st)
        a, b = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda"); dz = empty_like(z)
        DiffLabelLogProbs(z, labels, st, h if with_h else None, a, b if with_h else None, dz); assert untouched(dz)
        m, ls, lq, q, H = scores64(z); has = (labels >= 0) & (labels < cols)
        ga = torch.where(has, a.double(), 0.0)[:, None]; gb = b.double()[:, None] if with_h else torch.zeros_like(ga)
        lq0 = lq.nan_to_num(neginf=-1e4)
        want = -q * (ga + gb * (lq0 + H[:, None]))
        want[torch.arange(rows, device="cuda")[has], labels[has].long()] += ga[has, 0]
        # log q carries the errors of the kept statistics (S) and its own two roundings; q the same relative
        D = 40.0; e = S(cols, D) + 4 * U32 * (ls.abs()[:, None] + lq0.abs().clamp(max=100.0) + m.abs()[:, None] * 0 + 1)
        off = q * (e * (ga.abs() + gb.abs() * (lq0.abs() + H[:, None].abs() + ls.abs()[:, None] + 2)) + 4 * U32 * (ga.abs() + gb.abs() * (lq0.abs() + H[:, None]))) + 4 * U32 * want.abs() + 2 * U32 * ga.abs() * (want.abs() > 0) + 1e-30
        assert_within(dz, want, half_step(dtype) * (want.abs() + off) + off + (2.0 ** -25 if dtype == torch.float16 else 0.0), "dz")
        DiffLabelLogProbs(z, labels, st, h if with_h else None, a, b if with_h else None, z); assert torch.equal(z, dz)      # in place

def distill64(z, t, idx, w, T):
    cols = z.shape[1]; used = (idx >= 0) & (idx < cols) ; at = idx.long().clamp(0, cols - 1)
    t = torch.where(used, t.double() / T, -float("inf")); live = (t > -float("inf")).any(1) & (w != 0)
    lp = t - torch.logsumexp(t, 1, keepdim=True); p = torch.where(used & live[:, None], lp.exp(), 0.0)
    lq = torch.log_softmax(z.double() / T, 1); lqk = lq.gather(1, at)
    terms = torch.where(p > 0, p * (lqk - lp), 0.0)
    objf = torch.where(live, w.double() * T * T * terms.sum(1), 0.0)
    d = -lq.exp(); d.scatter_add_(1, at, p); d = torch.where(live[:, None], w.double()[:, None] * T * d, 0.0)
    return objf, d, p, lq, terms, live

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_distillation_matches_the_formulas(rows, cols, dtype):
    from kaldi_amd.objective import ComputeDistillObjfAndDeriv, DistillationOptions
    g = generator(rows * 1000003 + cols + 2)
    for pad, top, T, weighted in ((0, 1, 1.0, False), (3, 17, 2.0, True), (8, 130, 0.5, True)) + (((0, 700, 1.5, True),) if cols < 7000 and rows < 200 else ()):
        z = logits(g, rows, cols, dtype, pad, masked=False); t = matrix(g, rows, top, dtype, pad, 2.0); idx = torch.randint(0, cols, (rows, top + pad), generator=g, device="cuda").to(torch.int32)[:, :top]
        idx[torch.rand(rows, top, generator=g, device="cuda") < 0.2] = -1; idx[0, 0] = cols; t[rows // 2, 0] = -float("inf")
        if rows > 2: idx[2] = -1; z[2] = float("nan")      # a row of padding: whatever is in it
        w = None
        if weighted: w = torch.randn(rows, generator=g, device="cuda"); w[rows // 3] = 0.0; z[rows // 3] = float("inf")
        objf = torch.full((rows,), 7.0, device="cuda"); dz = empty_like(z); ComputeDistillObjfAndDeriv(DistillationOptions(T), z, t, idx, w, objf, dz); assert untouched(dz)
        zz = z.double().nan_to_num(nan=0.0, posinf=0.0)
        want, d, p, lq, terms, live = distill64(zz, t, idx, torch.ones(rows, device="cuda") if w is None else w, T); ww = (torch.ones(rows, device="cuda") if w is None else w).double()
        D = 30.0 / T; e = S(cols, D) + S(top * 64, D); mag = T * T * ww.abs() * (torch.where(p > 0, p * (lq.gather(1, idx.long().clamp(0, cols - 1)).abs() + D + 10), 0.0).sum(1))
        assert_within(objf, want, e * mag + e * T * T * ww.abs() + 1e-30, "objf")
        off = e * ww.abs()[:, None] * T * (lq.exp() + (d / (ww[:, None] * T)).nan_to_num().abs() + (d != 0) * 0) + 1e-30
        P = torch.zeros_like(d).scatter_add_(1, idx.long().clamp(0, cols - 1), p); off = off + e * ww.abs()[:, None] * T * P
        assert_within(dz, d, half_step(dtype) * (d.abs() + off) + off + (2.0 ** -25 if dtype == torch.float16 else 0.0), "dz")
        o2 = torch.empty_like(objf); ComputeDistillObjfAndDeriv(DistillationOptions(T), z, t, idx, w, o2)      # without the derivative (wide rows take another way)
        assert_within(o2, want, e * mag + e * T * T * ww.abs() + 1e-30, "objf alone")
        ComputeDistillObjfAndDeriv(DistillationOptions(T), z, t, idx, w, o2, z); assert torch.equal(z, dz) and torch.equal(o2, objf)      # in place

@pytest.mark.parametrize("dtype", TYPES)
def test_the_widest_rows(dtype):
    """2^19 columns, the last of them the label, an alternative and a teacher's entry: every part of the row comes in"""
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs, ComputeDistillObjfAndDeriv, DistillationOptions
    rows, cols = 3, 1 << 19; g = generator(19); z = torch.randn(rows, cols, generator=g, device="cuda").to(dtype); z[:, -1] = 9.0; z[:, 0] = 8.0; z[1, cols // 2 + 1] = 10.0
    y = torch.full((rows,), cols - 1, dtype=torch.int32, device="cuda"); lp, h, st = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda"); al, ai = torch.empty(rows, 40, device="cuda"), torch.empty(rows, 40, dtype=torch.int32, device="cuda")
    LabelLogProbs(z, y, lp, h, st, al, ai); m, ls, lq, q, H = scores64(z); e = S(cols, 40) + 8 * U32 * ls; idx = best64(z, 40)
    assert_within(lp, lq[:, -1], e, "log prob"); assert_within(h, H, e + S(cols, 40) * (H + ls), "entropy"); assert torch.equal(ai.long(), idx); assert_within(al, lq.gather(1, idx), e[:, None].expand(rows, 40), "alternatives")
    t = torch.tensor([[1.0, 0.0]], device="cuda").expand(rows, 2).contiguous().to(dtype); ti = torch.tensor([[cols - 1, 5]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous(); f, dz = torch.empty(rows, device="cuda"), torch.empty_like(z)
    ComputeDistillObjfAndDeriv(DistillationOptions(), z, t, ti, None, f, dz); want, d, _, _, _, _ = distill64(z, t, ti, torch.ones(rows, device="cuda"), 1.0)
    assert_within(f, want, S(cols, 40) * 40 * torch.ones_like(want), "objf"); off = S(cols, 40) * (q + d.abs()) + S(cols, 40) * (d > 0); assert_within(dz, d, half_step(dtype) * (d.abs() + off) + off + (2.0 ** -25 if dtype == torch.float16 else 0.0), "dz")

def test_rows_with_nothing_to_pass_on_get_zeros():
    """padding with NaNs and infinities in it, no label and no derivative of the entropy: zeros"""
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs
    for cols in (100, 5000):
        z = torch.randn(4, cols, generator=generator(cols), device="cuda"); z[1, 3] = float("nan"); z[2] = float("inf"); y = torch.tensor([1, -1, -1, 2], dtype=torch.int32, device="cuda"); h, st = torch.empty(4, device="cuda"), torch.empty(4, 2, device="cuda"); LabelLogProbs(z, y, None, h, st)
        dz = torch.empty_like(z); DiffLabelLogProbs(z, y, st, None, torch.ones(4, device="cuda"), None, dz); assert (dz[1:3] == 0).all() and torch.isfinite(dz).all() and dz[0, 1] > 0 and dz[3, 2] > 0

def test_distillation_edges():
    from kaldi_amd.objective import ComputeDistillObjfAndDeriv, DistillationOptions
    inf = float("inf"); o = DistillationOptions()
    for dtype in TYPES:
        for cols in (40, 3000, 30000, 150000):
            z = torch.randn(4, cols, generator=generator(cols), device="cuda").to(dtype); z[0] = -inf; z[1, 7] = -inf; z[2, 9] = float("nan")
            t = torch.tensor([[1.0, 2.0]], device="cuda").expand(4, 2).contiguous().to(dtype); idx = torch.tensor([[7, 7], [7, 8], [1, 2], [3, 3]], dtype=torch.int32, device="cuda")
            f = torch.empty(4, device="cuda"); dz = empty_like(z); ComputeDistillObjfAndDeriv(o, z, t, idx, None, f, dz)
            assert f[0] == -inf and (dz[0] == 0).all()                                        # a row that can be nothing
            assert f[1] == -inf and torch.isfinite(dz[1]).all() and dz[1, 7] > 0               # an entry at a column that cannot be: the derivative is finite
            assert torch.isnan(f[2]) and torch.isnan(dz[2].float()).any()
            q = torch.softmax(z[3].double(), 0); assert abs(dz[3, 3].double() - (1 - q[3])) <= half_step(dtype) + S(cols, 20)      # the same column twice: the probabilities add up to 1
            want = torch.log_softmax(z[3].double(), 0)[3] - (torch.log_softmax(t[3].double(), 0).exp() * torch.log_softmax(t[3].double(), 0)).sum(); assert abs(f[3].double() - want) <= S(cols, 20) * 20

def test_derivatives_match_differences():
    """along random directions, by central differences of the float64 formulas with h = 1e-4: h^2 f''' / 6 is within 1e-6 of the terms' magnitudes"""
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs, ComputeDistillObjfAndDeriv, DistillationOptions
    g = generator(17); rows, cols, h, T = 5, 90, 1e-4, 2.0
    z = torch.randn(rows, cols, generator=g, device="cuda"); y = torch.randint(0, cols, (rows,), generator=g, device="cuda").to(torch.int32); a, b = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    H, st, dz = torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda"), torch.empty_like(z); LabelLogProbs(z, y, None, H, st); DiffLabelLogProbs(z, y, st, H, a, b, dz)
    def f(z): lq = torch.log_softmax(z, 1); return (a.double() * lq.gather(1, y.long()[:, None])[:, 0] - b.double() * (lq.exp() * lq).sum(1)).sum()
    t = torch.randn(rows, 6, generator=g, device="cuda"); idx = torch.randint(0, cols, (rows, 6), generator=g, device="cuda").to(torch.int32); w = torch.rand(rows, generator=g, device="cuda"); o, dd = torch.empty(rows, device="cuda"), torch.empty_like(z)
    ComputeDistillObjfAndDeriv(DistillationOptions(T), z, t, idx, w, o, dd)
    for deriv, func in ((dz, f), (dd, lambda z: distill64(z, t, idx, w, T)[0].sum())):
        for _ in range(4):
            v = torch.randn(rows, cols, generator=g, device="cuda").double(); diff = (func(z.double() + h * v) - func(z.double() - h * v)) / (2 * h); terms = deriv.double() * v
            assert abs(terms.sum() - diff) <= (1e-6 + S(cols, 10)) * terms.abs().sum()

def test_long_matrix_offsets_pass_32_bits():
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs, ComputeDistillObjfAndDeriv, DistillationOptions
    rows, cols = 17000, 131072; z = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda"); z[-4:].normal_(generator=generator(2)); y = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    lp, h, st = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda"); ai = torch.empty(rows, 3, dtype=torch.int32, device="cuda"); LabelLogProbs(z, y, lp, h, st, None, ai)
    s = z[-4:].clone(); m, ls, lq, q, H = scores64(s); assert_within(lp[-4:], lq[:, 77], S(cols, 10) + 4 * U32 * ls, "log prob"); assert torch.equal(ai[-4:].long(), best64(s, 3)); assert ai[5].tolist() == [0, 1, 2]
    g = torch.zeros(rows, device="cuda"); g[-4:] = 1.0; DiffLabelLogProbs(z, y, st, None, g, None, z); want = -q; want[:, 77] += 1; off = 2 * S(cols, 20); assert_within(z[-4:], want, half_step(torch.bfloat16) * want.abs() * 1.01 + off * q + off * (want > 0), "dz"); assert (z[-5] == 0).all()
    z[-4:] = s; t = torch.zeros(rows, 2, dtype=torch.bfloat16, device="cuda"); idx = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda"); idx[-4:, 0] = 77; f = torch.empty(rows, device="cuda"); ComputeDistillObjfAndDeriv(DistillationOptions(), z, t, idx, None, f, z)
    assert_within(f[-4:], lq[:, 77], S(cols, 10) + 4 * U32 * ls, "objf"); assert_within(z[-4:], want, half_step(torch.bfloat16) * want.abs() * 1.01 + off * q + off * (want > 0), "dz"); assert (f[:-4] == 0).all()

def test_captured_replayed_and_on_a_side_stream():
    from kaldi_amd.objective import LabelLogProbs, DiffLabelLogProbs, ComputeDistillObjfAndDeriv, DistillationOptions
    g = generator(3)
    for rows, cols, dtype in ((70, 6024, torch.float32), (3, 70001, torch.float32), (5, 140001, torch.bfloat16)):
        z = torch.empty(rows, cols, dtype=dtype, device="cuda"); y = torch.randint(0, cols, (rows,), generator=g, device="cuda").to(torch.int32); t = torch.randn(rows, 9, generator=g, device="cuda").to(dtype); idx = torch.randint(-1, cols, (rows, 9), generator=g, device="cuda").to(torch.int32); one = torch.ones(rows, device="cuda")
        def buffers(): return [torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda"), torch.empty(rows, 8, device="cuda"), torch.empty(rows, 8, dtype=torch.int32, device="cuda"), torch.empty_like(z), torch.empty(rows, device="cuda"), torch.empty_like(z), torch.empty(rows, device="cuda")]
        def step(b):
            LabelLogProbs(z, y, *b[:5]); DiffLabelLogProbs(z, y, b[2], b[1], one, one, b[5]); ComputeDistillObjfAndDeriv(DistillationOptions(2.0), z, t, idx, one, b[6], b[7]); ComputeDistillObjfAndDeriv(DistillationOptions(2.0), z, t, idx, one, b[8])
        a, b = buffers(), buffers(); z.normal_(generator=g); step(a); torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph): step(a)
        for _ in range(3):
            z.normal_(generator=g); torch.cuda.synchronize(); graph.replay(); step(b); torch.cuda.synchronize(); assert all(torch.equal(p, q) for p, q in zip(a, b))
        s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream()); c = buffers()
        with torch.cuda.stream(s): step(c)
        torch.cuda.synchronize(); assert all(torch.equal(p, q) for p, q in zip(c, b))
