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

def test_label_entry_points():
    L = _l.load()
    f = lambda dtype=0, z=P, ld=8, y=P, lp=P, n=0, al=None, ai=None, ws=None, nb=0, rows=4, cols=8: L.k3_label_logprobs(dtype, z, ld, y, lp, None, None, n, al, ai, ws, nb, rows, cols, None)  # noqa: E731
    refused(f(dtype=3), "type"); refused(f(ld=7), "bad argument"); refused(f(rows=-1), "bad argument"); refused(f(cols=0), "bad argument"); refused(f(n=-1), "bad argument"); refused(f(z=None), "null"); refused(f(y=None), "null")
    refused(f(n=65, al=P, cols=100, ld=100), "at most"); refused(f(cols=(1 << 19) + 1, ld=1 << 22), "at most"); refused(f(n=9, al=P), "more alternatives"); refused(f(n=3), "do not go together"); refused(f(al=P), "do not go together")
    assert f(rows=0) == 0
    need = L.k3_label_logprobs_workspace(0, 4, 100000, 5); assert need > 0 and L.k3_label_logprobs_workspace(0, 4000, 6024, 5) == 0
    refused(f(cols=100000, ld=100000, n=5, al=P, ws=P, nb=need - 1), "workspace"); refused(f(cols=100000, ld=100000, n=5, al=P, ws=P + 4, nb=need), "workspace"); refused(f(cols=100000, ld=100000, n=5, al=P), "workspace")
    g = lambda dtype=0, z=P, ld=8, y=P, st=P, h=P, a=P, b=P, dz=P, ldd=8, rows=4, cols=8: L.k3_label_logprobs_deriv(dtype, z, ld, y, st, h, a, b, dz, ldd, rows, cols, None)  # noqa: E731
    refused(g(dtype=-1), "type"); refused(g(ld=7), "bad argument"); refused(g(ldd=7), "bad argument"); refused(g(cols=0), "bad argument"); refused(g(rows=-1), "bad argument")
    for k in ("z", "st", "dz", "y", "h"): refused(g(**{k: None}), "null")
    assert g(rows=0) == 0

def test_distillation_entry_point():
    L = _l.load()
    f = lambda dtype=0, T=1.0, z=P, ld=8, v=P, ldv=3, i=P, ldi=3, n=3, o=P, dz=P, ldd=8, ws=None, nb=0, rows=4, cols=8: L.k3_distill_objf_and_deriv(dtype, T, z, ld, v, ldv, i, ldi, n, None, o, dz, ldd, ws, nb, rows, cols, None)  # noqa: E731
    refused(f(dtype=3), "type")
    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-4): refused(f(T=T), "temperature")
    for k in ("ld", "ldv", "ldi", "ldd"): refused(f(**{k: 2}), "bad argument")
    refused(f(n=0), "bad argument"); refused(f(cols=0), "bad argument"); refused(f(rows=-1), "bad argument"); refused(f(n=1025, ldv=2000, ldi=2000), "at most"); refused(f(cols=(1 << 19) + 1, ld=1 << 22, ldd=1 << 22), "at most")
    for k in ("z", "v", "i", "o"): refused(f(**{k: None}), "null")
    assert f(rows=0) == 0
    need = L.k3_distill_workspace(0, 4, 200000, 3, 1); assert need > 0 and L.k3_distill_workspace(0, 4, 6024, 3, 1) == 0
    refused(f(cols=200000, ld=200000, ldd=200000, ws=P, nb=need - 1), "workspace"); refused(f(cols=200000, ld=200000, ldd=200000), "workspace"); refused(f(cols=200000, ld=200000, ldd=200000, ws=P + 8, nb=need), "workspace")

def test_affine_entry_points():
    L = _l.load()
    need = L.k3_affine_forward_workspace(4, 4096, 8); assert need > 0
    f = lambda dtype=1, act=0, x=P, ldx=4096, w=2 * P, ldw=4096, r=None, ldr=8, y=3 * P, ldy=8, pre=None, ldp=8, ws=P, n=need, rows=4, inner=4096, cols=8: L.k3_affine_forward(dtype, act, x, ldx, w, ldw, None, r, ldr, y, ldy, pre, ldp, ws, n, rows, inner, cols, None)  # noqa: E731
    for d in (0, 3, -1): refused(f(dtype=d), "float16 and bfloat16")
    refused(f(act=6), "activation"); refused(f(act=-1), "activation")
    for k in ("ldx", "ldw", "ldy"): refused(f(**{k: 7}), "bad argument")
    refused(f(r=P, ldr=7), "bad argument"); refused(f(pre=P, ldp=7), "bad argument"); refused(f(rows=-1), "bad argument"); refused(f(inner=0), "bad argument"); refused(f(cols=0), "bad argument")
    refused(f(inner=1 << 21, ldx=1 << 21, ldw=1 << 21), "too large"); refused(f(rows=(1 << 31) - 1, cols=4096, ldy=4096), "too large")
    for k in ("x", "w", "y"): refused(f(**{k: None}), "null")
    refused(f(ws=None), "workspace"); refused(f(n=need - 1), "workspace"); refused(f(ws=P + 4), "workspace"); assert f(rows=0) == 0
    for k in (dict(y=P), dict(y=2 * P), dict(pre=3 * P), dict(pre=P), dict(pre=2 * P), dict(pre=5 * P, r=5 * P)): refused(f(**k), "lies on")
    need = L.k3_affine_backward_workspace(1, 4, 4096, 8); assert need > 0
    b = lambda dtype=1, act=1, x=P, ldx=4096, w=2 * P, ldw=4096, pre=3 * P, ldp=8, dy=4 * P, lddy=8, dx=5 * P, lddx=4096, dw=6 * P, lddw=4096, ws=P, n=need, rows=4, inner=4096, cols=8: L.k3_affine_backward(dtype, act, x, ldx, w, ldw, pre, ldp, dy, lddy, dx, lddx, dw, lddw, P, ws, n, rows, inner, cols, None)  # noqa: E731
    refused(b(dtype=0), "float16 and bfloat16"); refused(b(act=9), "activation")
    for k in ("ldx", "ldw", "ldp", "lddy", "lddx", "lddw"): refused(b(**{k: 7}), "bad argument")
    refused(b(rows=-1), "bad argument"); refused(b(inner=0), "bad argument"); refused(b(cols=0), "bad argument"); refused(b(inner=1 << 21, ldx=1 << 21, ldw=1 << 21, lddx=1 << 21, lddw=1 << 21), "too large")
    for k in ("x", "w", "pre", "dy"): refused(b(**{k: None}), "null")
    refused(b(ws=None), "workspace"); refused(b(n=need - 1), "workspace"); refused(b(ws=P + 4), "workspace")
    for at in (1, 2, 3, 4): refused(b(dx=at * P), "lies on"); refused(b(dw=at * P), "lies on")
    refused(b(dw=5 * P), "lie on each other")

def test_matrices_that_are_no_rows_on_a_gpu():
    from kaldi_amd import cumatrix as cm, objective as ob
    t = torch.zeros(4, 8)
    for bad, word in ((t, "GPU"), (torch.zeros(4), "matrix"), (torch.zeros(4, 8, dtype=torch.float64), "matrix"), (torch.zeros(4, 8, dtype=torch.int32), "matrix"), ("x", "matrix")):
        with pytest.raises(K3Error, match=word): cm.LayerNormPerRow(bad, None, None, 1e-5, bad)
        with pytest.raises(K3Error, match=word): ob.LabelLogProbs(bad, None)
        with pytest.raises(K3Error, match=word): cm.AffinePerRow(bad, bad, None, "none", None, bad)
        with pytest.raises(K3Error, match=word): ob.ComputeDistillObjfAndDeriv(ob.DistillationOptions(), bad, bad, bad, None, None)
