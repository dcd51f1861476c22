"""Objectives and scores from the rows of a network's output, in float32, float16 or bfloat16: the log-probability of one given label per row with the row's entropy and best
alternatives, and distillation from a teacher's top logits; with their derivatives.  They stand beside the LF-MMI objective (kaldi_amd.chain) and CuMatrixBase::LogSoftMaxPerRow, and like
them write into matrices and vectors that the caller has.  ctypes plumbing over libk3hip.so (include/k3hip.h: k3_label_logprobs*, k3_distill_*); nothing is waited for."""
from . import lib as _l
from .cumatrix import _rows, _like_rows, _vec, _table, _workspace, _run, _refuse, _I32

def LabelLogProbs(nnet_output, labels, log_prob=None, entropy=None, stats=None, alt_log_probs=None, alt_labels=None):
    """nnet_output: [rows, cols] logits; labels: int32 [rows], one column per row, anything outside 0 .. cols - 1 (-1) = none (its log_prob is 0); None only if log_prob is.
    Receive, where given: log_prob, entropy: float32 [rows]; stats: float32 [rows, 2] (what DiffLabelLogProbs takes); alt_log_probs: float32 and alt_labels: int32 [rows, n], n <= 64: the
    row's n most probable columns, best first, equal ones by column.  -inf in nnet_output = a column that cannot be; a row with a NaN or +inf has NaN scores and alternatives -1."""
    dt, z, ld, r, c, i = _rows(nnet_output, "nnet_output")
    alt = alt_log_probs if alt_log_probs is not None else alt_labels
    try: n = 0 if alt is None else alt.shape[-1]
    except (AttributeError, IndexError): _refuse("alternatives: tensors of shape [rows, n] are wanted")
    if n > 64: _refuse(f"alternatives: {n}, at most 64 are kept")
    L = _l.load(); nw = L.k3_label_logprobs_workspace(dt, r, c, n); w = _workspace(nw, i)
    _run(i, L.k3_label_logprobs, dt, z, ld, _vec(labels, r, i, "labels", _I32), _vec(log_prob, r, i, "log_prob"), _vec(entropy, r, i, "entropy"), _table(stats, r, 2, i, "stats"), n,
         _table(alt_log_probs, r, n, i, "alt_log_probs"), _table(alt_labels, r, n, i, "alt_labels", _I32), w.data_ptr() if nw else None, nw, r, c)

def DiffLabelLogProbs(nnet_output, labels, stats, entropy, log_prob_deriv, entropy_deriv, nnet_output_deriv):
    """nnet_output_deriv (overwritten; may be nnet_output) = the derivative of sum(log_prob_deriv log_prob + entropy_deriv entropy) with respect to nnet_output.  stats and entropy: what
    LabelLogProbs gave; entropy may be None where entropy_deriv is, and either derivative may be None."""
    x = _rows(nnet_output, "nnet_output"); dt, z, ld, r, c, i = x; d, ldd = _like_rows(nnet_output_deriv, x, "nnet_output_deriv")
    _run(i, _l.load().k3_label_logprobs_deriv, dt, z, ld, _vec(labels, r, i, "labels", _I32), _table(stats, r, 2, i, "stats"), _vec(entropy, r, i, "entropy"),
         _vec(log_prob_deriv, r, i, "log_prob_deriv"), _vec(entropy_deriv, r, i, "entropy_deriv"), d, ldd, r, c)

class DistillationOptions:
    """temperature: both softmaxes are taken at it (and the objective is scaled by its square, which keeps the derivatives' size)"""
    __slots__ = ("temperature",)
    def __init__(self, temperature=1.0): self.temperature = float(temperature)

def ComputeDistillObjfAndDeriv(opts, nnet_output, teacher_values, teacher_indexes, weights, objf, nnet_output_deriv=None):
    """Distillation from a teacher's top logits.  teacher_values [rows, n] (nnet_output's type), teacher_indexes int32 [rows, n], n <= 1024: a row's teacher logits and their columns, -1 =
    unused; weights: float32 [rows] or None (1).  objf: float32 [rows] receives w T^2 sum_k p_k (log q - log p_k) (to be maximised, 0 at best), p the teacher's softmax over the row's
    entries, q the network's over all columns, both at the temperature T; nnet_output_deriv (where given; overwritten; may be nnet_output) its derivative with respect to
    nnet_output.  Rows without an entry or of weight 0: 0 and zeros.  One entry per row: the cross entropy."""
    x = _rows(nnet_output, "nnet_output"); dt, z, ld, r, c, i = x
    vt, v, ldv, vr, n, vi = _rows(teacher_values, "teacher_values")
    if vr != r or vt != dt or vi != i: _refuse(f"teacher_values: {vr} rows of type {vt} on device {vi} do not go with {r} of type {dt} on device {i}")
    t = teacher_indexes
    if getattr(t, "dtype", None) is not _I32 or t.shape != (r, n) or t.get_device() != i: _refuse(f"teacher_indexes: an int32 matrix of shape {(r, n)} on device {i} is wanted")
    s0, s1 = t.stride()
    if r <= 1: s0 = n
    if (s1 != 1 and n > 1) or s0 < n: _refuse(f"teacher_indexes: rows must be contiguous and must not overlap (strides {s0}, {s1})")
    d, ldd = (None, c) if nnet_output_deriv is None else _like_rows(nnet_output_deriv, x, "nnet_output_deriv")
    L = _l.load(); nw = L.k3_distill_workspace(dt, r, c, n, 0 if d is None else 1); w = _workspace(nw, i)
    _run(i, L.k3_distill_objf_and_deriv, dt, opts.temperature, z, ld, v, ldv, t.data_ptr(), s0, n, _vec(weights, r, i, "weights"), _vec(objf, r, i, "objf"), d, ldd,
         w.data_ptr() if nw else None, nw, r, c)
