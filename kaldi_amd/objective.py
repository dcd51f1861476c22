"""Objectives and scores from the rows of a network's output, in float32, float16 or bfloat16: the log-probability of one given label per row with the row's entropy and best
alternatives, and distillation from a teacher's top logits; with their derivatives.  They stand beside the LF-MMI objective (kaldi_amd.chain) and CuMatrixBase::LogSoftMaxPerRow, and like
them write into matrices and vectors that the caller has.  ctypes plumbing over libk3hip.so (include/k3hip.h: k3_label_logprobs*, k3_distill_*); nothing is waited for."""
import torch
from . import lib as _l
from .cumatrix import _rows, _like_rows, _vec, _run, _refuse, _DTYPES

def _workspace(n, ref): return None if n == 0 else torch.empty(n, dtype=torch.uint8, device=ref.device)
def _ws(w): return (None, 0) if w is None else (w.data_ptr(), w.numel())

def LabelLogProbs(nnet_output, labels, log_prob=None, entropy=None, stats=None, alt_log_probs=None, alt_labels=None):
    """nnet_output: [rows, cols] logits; labels: int32 [rows], one column per row, anything outside 0 .. cols - 1 (-1) = none (its log_prob is 0); None only if log_prob is.
    Receive, where given: log_prob, entropy: float32 [rows]; stats: float32 [rows, 2] (what DiffLabelLogProbs takes); alt_log_probs: float32 and alt_labels: int32 [rows, n], n <= 64: the
    row's n most probable columns, best first, equal ones by column.  -inf in nnet_output = a column that cannot be; a row with a NaN or +inf has NaN scores and alternatives -1."""
    z, ld = _rows(nnet_output, "nnet_output"); r, c = z.shape
    alt = alt_log_probs if alt_log_probs is not None else alt_labels
    n = 0
    if alt is not None:
        if alt.dim() != 2: _refuse("alternatives: [rows, n] is wanted")
        n = alt.shape[1]
    L = _l.load(); dt = _DTYPES[z.dtype]
    w = _workspace(L.k3_label_logprobs_workspace(dt, r, c, n), z)
    _run(z, L.k3_label_logprobs, dt, z.data_ptr(), ld, _vec(labels, (r,), z, "labels", torch.int32), _vec(log_prob, (r,), z, "log_prob"), _vec(entropy, (r,), z, "entropy"),
         _vec(stats, (r, 2), z, "stats"), n, _vec(alt_log_probs, (r, n), z, "alt_log_probs"), _vec(alt_labels, (r, n), z, "alt_labels", torch.int32), *_ws(w), r, c)

def DiffLabelLogProbs(nnet_output, labels, stats, entropy, log_prob_deriv, entropy_deriv, nnet_output_deriv):
    """nnet_output_deriv (overwritten; may be nnet_output) = the derivative of sum(log_prob_deriv log_prob + entropy_deriv entropy) with respect to nnet_output.  stats and entropy: what
    LabelLogProbs gave; entropy may be None where entropy_deriv is, and either derivative may be None."""
    z, ld = _rows(nnet_output, "nnet_output"); d, ldd = _like_rows(nnet_output_deriv, z, "nnet_output_deriv"); r, c = z.shape
    _run(z, _l.load().k3_label_logprobs_deriv, _DTYPES[z.dtype], z.data_ptr(), ld, _vec(labels, (r,), z, "labels", torch.int32), _vec(stats, (r, 2), z, "stats"), _vec(entropy, (r,), z, "entropy"),
         _vec(log_prob_deriv, (r,), z, "log_prob_deriv"), _vec(entropy_deriv, (r,), z, "entropy_deriv"), d.data_ptr(), ldd, r, c)

class DistillationOptions:
    """temperature: both softmaxes are taken at it (and the objective is scaled by its square, which keeps the derivatives' size)"""
    __slots__ = ("temperature",)
    def __init__(self, temperature=1.0): self.temperature = float(temperature)

def ComputeDistillObjfAndDeriv(opts, nnet_output, teacher_values, teacher_indexes, weights, objf, nnet_output_deriv=None):
    """Distillation from a teacher's top logits.  teacher_values [rows, n] (nnet_output's type), teacher_indexes int32 [rows, n], n <= 1024: a row's teacher logits and their columns, -1 =
    unused; weights: float32 [rows] or None (1).  objf: float32 [rows] receives w T^2 sum_k p_k (log q - log p_k) (to be maximised, 0 at best), p the teacher's softmax over the row's
    entries, q the network's over all columns, both at the temperature T; nnet_output_deriv (where given; overwritten; may be nnet_output) its derivative with respect to
    nnet_output.  Rows without an entry or of weight 0: 0 and zeros.  One entry per row: the cross entropy."""
    z, ld = _rows(nnet_output, "nnet_output"); r, c = z.shape
    v, ldv = _rows(teacher_values, "teacher_values"); n = v.shape[1]
    if v.shape[0] != r or v.dtype != z.dtype or v.device != z.device: _refuse(f"teacher_values: {tuple(v.shape)} {v.dtype} on {v.device} does not go with {tuple(z.shape)} {z.dtype} on {z.device}")
    i = teacher_indexes
    if not isinstance(i, torch.Tensor) or i.dtype != torch.int32 or i.shape != v.shape or i.device != z.device or (n > 1 and i.stride(1) != 1) or (r > 1 and i.stride(0) < n):
        _refuse(f"teacher_indexes: an int32 matrix of shape {tuple(v.shape)} on {z.device} with contiguous rows is wanted")
    if objf is None: _refuse("objf: a float32 vector is wanted")
    d, ldd = (None, c) if nnet_output_deriv is None else _like_rows(nnet_output_deriv, z, "nnet_output_deriv")
    L = _l.load(); dt = _DTYPES[z.dtype]
    w = _workspace(L.k3_distill_workspace(dt, r, c, n, int(d is not None)), z)
    _run(z, L.k3_distill_objf_and_deriv, dt, opts.temperature, z.data_ptr(), ld, v.data_ptr(), ldv, i.data_ptr(), i.stride(0) if r > 1 else n, n, _vec(weights, (r,), z, "weights"),
         _vec(objf, (r,), z, "objf"), None if d is None else d.data_ptr(), ldd, *_ws(w), r, c)
