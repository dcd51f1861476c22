"""What the Python calls of the operators on rows of matrices refuse of tensors on a GPU: missing ones, others than tensors, and wrong types, shapes, devices and strides.  Nothing is queued."""
import pytest, torch
from kaldi_amd.lib import K3Error
pytestmark = pytest.mark.gpu

def wrong_vectors(n):
    yield "x"
    yield torch.zeros(n)                                              # not on the GPU
    yield torch.zeros(n + 1, device="cuda")
    yield torch.zeros(n, dtype=torch.float64, device="cuda")
    yield torch.zeros(2 * n, device="cuda")[::2]

def test_objectives():
    from kaldi_amd import objective as ob
    R, C, N = 4, 40, 3; z = torch.randn(R, C, device="cuda"); y = torch.zeros(R, dtype=torch.int32, device="cuda"); v = lambda *s: torch.zeros(s, device="cuda"); i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for bad in wrong_vectors(R):
        for k in ("log_prob", "entropy", "stats"):
            with pytest.raises(K3Error): ob.LabelLogProbs(z, y, **{k: bad})
        for k in range(5):
            a = [y, v(R, 2), v(R), v(R), v(R)]; a[k] = bad
            with pytest.raises(K3Error): ob.DiffLabelLogProbs(z, *a, v(R, C))
        for w, f in ((bad, v(R)), (None, bad)):
            with pytest.raises(K3Error): ob.ComputeDistillObjfAndDeriv(ob.DistillationOptions(), z, v(R, N), i(R, N), w, f)
    for labels in (None, "x", y.long(), y.cpu(), y[:3], v(R)):
        with pytest.raises(K3Error): ob.LabelLogProbs(z, labels, v(R))
    for al, ai in (("x", None), (None, "x"), (v(R, N), "x"), (v(R, N), i(R, N + 1)), (v(R, N), i(R + 1, N)), (v(), None), (v(R, 65), None), (i(R, N), i(R, N)), (v(R, N), v(R, N)), (v(R, C + 1), None)):
        with pytest.raises(K3Error): ob.LabelLogProbs(z, y, None, None, None, al, ai)
    o = ob.DistillationOptions()
    for t, k in ((None, i(R, N)), ("x", i(R, N)), (v(R, N).half(), i(R, N)), (v(R + 1, N), i(R, N)), (v(R, N), None), (v(R, N), "x"), (v(R, N), i(R, N).long()), (v(R, N), i(R, N + 1)), (v(R, N), i(R, N).cpu()), (v(R, N), i(N, R).t()), (v(R, N), i(1, N).expand(R, N)), (v(N, R).t(), i(R, N)), (v(R, 0), i(R, 0))):
        with pytest.raises(K3Error): ob.ComputeDistillObjfAndDeriv(o, z, t, k, None, v(R))
    with pytest.raises(K3Error): ob.ComputeDistillObjfAndDeriv(o, z, v(R, N), i(R, N), None, None)
    for d in ("x", v(R, C + 1), v(R, C).half(), v(C, R).t(), v(1, C).expand(R, C), v(R, C).cpu()):
        with pytest.raises(K3Error): ob.ComputeDistillObjfAndDeriv(o, z, v(R, N), i(R, N), None, v(R), d)
        with pytest.raises(K3Error): ob.DiffLabelLogProbs(z, y, v(R, 2), None, v(R), None, d)

def test_layers():
    from kaldi_amd import cumatrix as cm
    R, K, C = 4, 24, 40; x = torch.randn(R, K, device="cuda").half(); w = torch.randn(C, K, device="cuda").half(); y = torch.zeros(R, C, device="cuda").half(); v = lambda n: torch.zeros(n, device="cuda")  # noqa: E731
    for bad in wrong_vectors(C):
        with pytest.raises(K3Error): cm.AffinePerRow(x, w, bad, "relu", None, y)
        with pytest.raises(K3Error): cm.DiffAffinePerRow(x, w, y, "relu", y.clone(), bias_params_deriv=bad)
        for k in range(2):
            a = [None, None]; a[k] = bad
            with pytest.raises(K3Error): cm.LayerNormPerRow(y, *a, 1e-5, y.clone())
            with pytest.raises(K3Error): cm.DiffLayerNormPerRow(y, y, None, v(R), v(R), None, *a)
        with pytest.raises(K3Error): cm.DiffLayerNormPerRow(y, y, bad, v(R), v(R), y.clone())
    for bad in list(wrong_vectors(R)) + [None]:
        for k in range(2):
            a = [v(R), v(R)]; a[k] = bad
            with pytest.raises(K3Error): cm.DiffLayerNormPerRow(y, y, None, *a, y.clone())
            if bad is not None:
                with pytest.raises(K3Error): cm.LayerNormPerRow(y, None, None, 1e-5, y.clone(), *a)
    for bad in (None, "x", y.float(), y.bfloat16(), y[:3], y[:, :-1], y.cpu(), y.t().contiguous().t(), y[:1].expand(R, C)):
        with pytest.raises(K3Error): cm.AffinePerRow(x, w, None, "relu", None, bad)
        with pytest.raises(K3Error): cm.DiffAffinePerRow(x, w, bad, "relu", y, x.clone())
        with pytest.raises(K3Error): cm.DiffAffinePerRow(x, w, y, "relu", bad, x.clone())
        with pytest.raises(K3Error): cm.LayerNormPerRow(y, None, None, 1e-5, bad)
        with pytest.raises(K3Error): cm.DiffLayerNormPerRow(y, bad, None, v(R), v(R), y.clone())
        if bad is not None:
            with pytest.raises(K3Error): cm.AffinePerRow(x, w, None, "relu", bad, y)
            with pytest.raises(K3Error): cm.AffinePerRow(x, w, None, "relu", None, y, bad)
            with pytest.raises(K3Error): cm.DiffAffinePerRow(x, w, y, "relu", y.clone(), bad)
    for act in (None, "swiglu", 1):
        with pytest.raises(K3Error): cm.AffinePerRow(x, w, None, act, None, y)
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(K3Error): cm.LayerNormPerRow(y, None, None, eps, y.clone())
