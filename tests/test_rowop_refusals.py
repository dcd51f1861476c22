"""What the operators on rows of float32 / float16 / bfloat16 matrices refuse: on the host, before anything is queued (no GPU is needed for any of it)."""
import ctypes, pytest, torch
from kaldi_amd import lib as _l
from kaldi_amd.lib import K3Error

P = 1 << 20      # stands for a device pointer: never dereferenced by a call that is refused

def refused(status, *words):
    assert status < 0
    text = _l.load().k3_last_error().decode()
    assert all(w in text for w in words), text

def test_layer_norm_entry_points():
    L = _l.load()
    fwd = lambda dtype=0, ldx=8, eps=1e-5, ldy=8, rows=4, cols=8, x=P, y=P: L.k3_layer_norm_forward(dtype, x, ldx, None, None, eps, y, ldy, None, None, rows, cols, None)  # noqa: E731
    refused(fwd(dtype=3), "type"); refused(fwd(dtype=-1), "type"); refused(fwd(ldx=7), "bad argument"); refused(fwd(ldy=7), "bad argument"); refused(fwd(rows=-1), "bad argument")
    refused(fwd(cols=-1), "bad argument"); refused(fwd(eps=-1.0), "bad argument"); refused(fwd(eps=float("nan")), "bad argument"); refused(fwd(x=None), "null"); refused(fwd(y=None), "null")
    assert fwd(rows=0) == 0 and fwd(cols=0) == 0
    need = L.k3_layer_norm_backward_workspace(4, 8); assert need > 0 and L.k3_layer_norm_backward_workspace(0, 8) == 0
    bwd = lambda dtype=0, ldx=8, ldg=8, ldd=8, mean=P, ds=P, ws=P, n=need, rows=4, cols=8, x=P: L.k3_layer_norm_backward(dtype, x, ldx, P, ldg, None, mean, P, P, ldd, ds, None, 0, ws, n, rows, cols, None)  # noqa: E731
    refused(bwd(dtype=9), "type"); refused(bwd(ldx=7), "bad argument"); refused(bwd(ldg=7), "bad argument"); refused(bwd(ldd=7), "bad argument"); refused(bwd(mean=None), "null"); refused(bwd(x=None), "null")
    refused(bwd(ws=None), "workspace"); refused(bwd(n=need - 1), "workspace")

def test_matrices_that_are_no_rows_on_a_gpu():
    from kaldi_amd import cumatrix as cm
    t = torch.zeros(4, 8)
    for bad, word in ((t, "GPU"), (torch.zeros(4), "matrix"), (torch.zeros(4, 8, dtype=torch.float64), "matrix"), (torch.zeros(4, 8, dtype=torch.int32), "matrix"), ("x", "matrix")):
        with pytest.raises(K3Error, match=word): cm.LayerNormPerRow(bad, None, None, 1e-5, bad)
