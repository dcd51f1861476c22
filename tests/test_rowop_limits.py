"""Sizes that the operators on rows of float32 / float16 / bfloat16 matrices refuse (on the host, before anything is queued; no GPU is needed for any of it)."""
import pytest, torch
from kaldi_amd import lib as _l
from tests.test_rowop_refusals import P, refused

def test_layer_norm_of_rows_whose_column_numbers_pass_32_bits():
    L = _l.load(); most = (1 << 31) - 1024; wide = 1 << 32
    fwd = lambda cols: L.k3_layer_norm_forward(1, P, wide, None, None, 1e-5, P, wide, None, None, 0, cols, None)  # noqa: E731
    bwd = lambda cols, ds=None, do=None: L.k3_layer_norm_backward(1, P, wide, P, wide, None, P, P, P, wide, ds, do, 0, None, 0, 0 if ds is None and do is None else 1, cols, None)  # noqa: E731
    for cols in (most + 1, (1 << 31) - 256, (1 << 31) - 1): refused(fwd(cols), "at most"); refused(bwd(cols), "at most")
    assert fwd(most) == 0 and bwd(most) == 0      # (without rows: nothing is queued)
    for cols in ((1 << 28) - 63, 1 << 30, most): refused(bwd(cols, P), "at most"); refused(bwd(cols, None, P), "at most")
    refused(bwd((1 << 28) - 64, P), "workspace")      # (gets as far as that)

def test_sizes_that_do_not_fit_32_bits():
    """on tensors without memory: what does not fit is refused before where they are is looked at"""
    from kaldi_amd import cumatrix as cm, objective as ob
    from kaldi_amd.lib import K3Error
    for shape in ((1 << 31, 1), ((1 << 32) + 4, 8), (1, 1 << 31), (4, (1 << 32) + 8)):
        t = torch.empty(shape, dtype=torch.float16, device="meta")
        for call in (lambda: cm.LayerNormPerRow(t, None, None, 1e-5, t), lambda: cm.AffinePerRow(t, t, None, "none", None, t), lambda: cm.DiffAffinePerRow(t, t, None, "none", t), lambda: ob.LabelLogProbs(t, None),
                     lambda: cm.DiffLayerNormPerRow(t, t, None, None, None), lambda: ob.DiffLabelLogProbs(t, None, None, None, None, None, t), lambda: ob.ComputeDistillObjfAndDeriv(ob.DistillationOptions(), t, t, t, None, None)):
            with pytest.raises(K3Error, match="2\\^31"): call()

def test_label_derivative_of_rows_whose_column_numbers_pass_32_bits():
    L = _l.load(); most = (1 << 31) - 4096; wide = 1 << 32
    for dtype in (0, 1, 2):
        f = lambda cols: L.k3_label_logprobs_deriv(dtype, P, wide, None, P, None, None, None, P, wide, 0, cols, None)  # noqa: E731
        for cols in (most + 1, (1 << 31) - 2048, (1 << 31) - 1): refused(f(cols), "at most")
        assert f(most) == 0      # (without rows: nothing is queued)
