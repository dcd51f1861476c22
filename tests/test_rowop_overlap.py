"""Operands that share memory: which calls of the operators on rows of matrices refuse it (on the host, with addresses that are never used; no GPU is needed for those)."""
import torch
from kaldi_amd import lib as _l
from tests.test_rowop_refusals import P, refused

def test_affine_layer():
    L = _l.load(); R, K, C = 6, 40, 24; n = L.k3_affine_forward_workspace(R, K, C)
    f = lambda x=P, ldx=K, w=2 * P, ldw=K, b=3 * P, r=4 * P, ldr=C, y=5 * P, ldy=C, pre=6 * P, ldp=C, rows=R: L.k3_affine_forward(1, 1, x, ldx, w, ldw, b, r, ldr, y, ldy, pre, ldp, 9 * P, n, rows, K, C, None)  # noqa: E731
    end = 2 * ((R - 1) * K + K)      # of x
    for at in (P + 2, P + 2 * K, P + end - 2, P - 2 * ((R - 1) * C + C) + 2): refused(f(y=at), "lies on"); refused(f(pre=at), "lies on")
    for at in (2 * P + 2, 2 * P + 2 * C * K - 2, 3 * P, 3 * P + 4 * C - 2): refused(f(y=at), "lies on"); refused(f(pre=at), "lies on")      # the weights, the bias
    refused(f(y=4 * P, ldy=C + 1), "lies on"); refused(f(y=4 * P, ldr=C + 8), "lies on"); refused(f(y=4 * P + 2), "lies on"); refused(f(y=4 * P + 2 * C), "lies on"); refused(f(pre=4 * P), "lies on")      # the residual, but for its own place
    refused(f(y=5 * P, pre=5 * P + 2 * C * R - 2), "lies on")
    refused(f(ldx=100, ldy=100, y=P + 2 * (K - 1)), "lies on"); refused(f(ldx=100, ldy=100, y=P + 2 * (100 - C + 1)), "lies on")      # columns of one buffer that reach into each other, in one row or the next
    refused(f(ldx=100, ldy=90, y=P + 2 * K), "lies on"); refused(f(rows=2, ldx=100, ldy=50, y=P + 2 * 60), "lies on")                 # strides that differ: the second row meets x
    n = L.k3_affine_backward_workspace(1, R, K, C)
    b = lambda x=P, ldx=K, w=2 * P, pre=3 * P, dy=4 * P, lddy=C, dx=5 * P, lddx=K, dw=6 * P, lddw=K, db=7 * P: L.k3_affine_backward(1, 1, x, ldx, w, K, pre, C, dy, lddy, dx, lddx, dw, lddw, db, 9 * P, n, R, K, C, None)  # noqa: E731
    for at in (P + 2, P + end - 2, 2 * P + 2 * C * K - 2, 3 * P + 2 * C * R - 2, 4 * P + 2): refused(b(dx=at), "lies on"); refused(b(dw=at), "lies on"); refused(b(db=at), "lies on")
    refused(b(dx=4 * P + 2 * (C - 1), lddy=100, lddx=100), "lies on"); refused(b(dw=5 * P + end - 2), "lie on each other"); refused(b(db=5 * P + 4), "lie on each other"); refused(b(db=6 * P), "lie on each other")

def test_layer_norm():
    L = _l.load(); R, C, X = 6, 40, 4
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        f = lambda x=P, ldx=C, sc=2 * P, of=3 * P, y=5 * P, ldy=C, m=6 * P, i=7 * P: L.k3_layer_norm_forward(dtype, x, ldx, sc, of, 1e-5, y, ldy, m, i, R, C, None)  # noqa: E731
        for at in (P + size, P + size * (R * C - 1), 2 * P, 3 * P + 4 * C - size, 6 * P, 7 * P + 4 * R - size): refused(f(y=at), "lies on")
        for k in ("m", "i"):
            for at in (P, P + size * R * C - 4, 2 * P + 4, 3 * P): refused(f(**{k: at}), "lies on")
        refused(f(y=P, ldy=C + 1), "lies on"); refused(f(y=P, ldx=C + 8), "lies on"); refused(f(ldx=100, ldy=100, y=P + size * (C - 1)), "lies on"); refused(f(ldx=100, ldy=100, y=P - size * (C - 1)), "lies on")
        n = L.k3_layer_norm_backward_workspace(R, C)
        b = lambda x=P, ldx=C, dy=2 * P, lddy=C, sc=3 * P, m=4 * P, i=5 * P, dx=6 * P, lddx=C, ds=7 * P, do=8 * P: L.k3_layer_norm_backward(dtype, x, ldx, dy, lddy, sc, m, i, dx, lddx, ds, do, 0, 9 * P, n, R, C, None)  # noqa: E731
        for at in (P + size, 2 * P + size, P + size * (R * C - 1), 2 * P - size, 3 * P, 4 * P, 5 * P + 4 * R - size, 7 * P, 8 * P + 4 * C - size): refused(b(dx=at), "lies on")
        for k in (dict(dx=P, lddx=C + 1), dict(dx=2 * P, lddx=C + 8), dict(dx=P, ldx=C + 1), dict(dx=2 * P, lddy=C + 1), dict(ds=8 * P), dict(do=7 * P + 4 * C - 4)): refused(b(**k), "lies on")

def test_label_scores():
    L = _l.load(); R, C, N = 6, 40, 4
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        f = lambda y=2 * P, lp=3 * P, h=4 * P, st=5 * P, al=6 * P, ai=7 * P: L.k3_label_logprobs(dtype, P, C, y, lp, h, st, N, al, ai, None, 0, R, C, None)  # noqa: E731
        for k, n in (("lp", R), ("h", R), ("st", 2 * R), ("al", N * R), ("ai", N * R)):
            for at in (P, P + size * R * C - 4, P - 4 * n + 4, 2 * P, 2 * P + 4 * R - 4): refused(f(**{k: at}), "lies on")
        g = lambda z=P, ld=C, dz=8 * P, ldd=C: L.k3_label_logprobs_deriv(dtype, z, ld, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P, dz, ldd, R, C, None)  # noqa: E731
        for at in (P + size, P - size, P + size * (R * C - 1), 2 * P, 3 * P + 8 * R - size, 4 * P, 5 * P, 6 * P + 4 * R - size): refused(g(dz=at), "lies on")
        refused(g(dz=P, ldd=C + 1), "lies on"); refused(g(dz=P, ld=C + 8), "lies on"); refused(g(ld=100, ldd=100, dz=P + size * (C - 1)), "lies on")

def test_distillation():
    L = _l.load(); R, C, N = 6, 40, 4
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        f = lambda z=P, ld=C, v=2 * P, i=3 * P, w=4 * P, o=5 * P, dz=6 * P, ldd=C: L.k3_distill_objf_and_deriv(dtype, 1.0, z, ld, v, N, i, N, N, w, o, dz, ldd, None, 0, R, C, None)  # noqa: E731
        for at in (P + size, P - size, P + size * (R * C - 1), 2 * P, 2 * P + size * (R * N - 1), 3 * P + 4 * R * N - size, 4 * P, 5 * P): refused(f(dz=at), "lies on")
        for at in (P, P + size * R * C - 4, 2 * P, 3 * P + 4, 4 * P, 6 * P): refused(f(o=at), "lies on")
        refused(f(dz=P, ldd=C + 1), "lies on"); refused(f(dz=P, ld=C + 8), "lies on"); refused(f(ld=100, ldd=100, dz=P + size * (C - 1)), "lies on")
