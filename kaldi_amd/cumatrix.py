"""CuMatrix-style view over a torch CUDA tensor whose methods call the k3_mat_* C ABI (include/k3hip.h): the Python mirror of
the adapter a Kaldi build would put under cudamatrix/cu-matrix.cc.  Method names and argument order follow CuMatrixBase
(cudamatrix/cu-matrix.h:79-791); kTrans/kNoTrans as booleans."""
import ctypes, torch
from . import lib as _l

def _st(): return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

# ---- arguments of the operators that take matrices of any k3_dtype: CuMatrix objects or 2-dimensional tensors whose rows are contiguous, all on one device (which need not be
# the current one); the kernels run on that device's current stream.  What a call writes shares no element with its other operands, unless it may be one of them (K3Error otherwise)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # k3_dtype
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda index: torch.cuda.current_stream(index).cuda_stream

_current_device = torch.cuda.current_device
_F32, _I32 = torch.float32, torch.int32
_MOST = 0x7fffffff      # the C entries' sizes are int32, and ctypes would cut what is larger
_devices = [torch.device("cuda", i) for i in range(64)]

def _refuse(what): raise _l.K3Error(what)
def _rows(m, name):
    """a matrix argument, checked: (k3_dtype, pointer, leading dimension, rows, columns, device index)"""
    t = m.t if type(m) is CuMatrix else m
    try: dt = _DTYPES[t.dtype]; r, c = t.shape; s0, s1 = t.stride(); i = t.get_device()
    except (AttributeError, KeyError, ValueError, RuntimeError): _refuse(f"{name}: a matrix of float32, float16 or bfloat16 is wanted")
    if not 1 < r <= _MOST: s0 = c if r <= 1 else -1
    if (s1 != 1 and c > 1) or not s0 >= c <= _MOST:
        if r > _MOST or c > _MOST: _refuse(f"{name}: {r} x {c}: at most 2^31 - 1 rows and columns")
        _refuse(f"{name}: rows must be contiguous and must not overlap (strides {s0}, {s1})")
    if i < 0: _refuse(f"{name}: not on a GPU")
    return dt, t.data_ptr(), s0, r, c, i
def _like_rows(m, x, name):
    """a second matrix of x's shape, type and device (x: what _rows gave): (pointer, leading dimension)"""
    y = _rows(m, name)
    if y[3] != x[3] or y[4] != x[4] or y[0] != x[0] or y[5] != x[5]: _refuse(f"{name}: {y[3]} x {y[4]} of type {y[0]} on device {y[5]} does not go with {x[3]} x {x[4]} of type {x[0]} on device {x[5]}")
    return y[1], y[2]
def _vec(t, n, i, name, dtype=_F32):
    """pointer of a contiguous vector of n elements on device i (None: null)"""
    if t is None: return None
    try:
        if t.dtype is dtype and t.numel() == n and t.get_device() == i and t.is_contiguous(): return t.data_ptr()
    except AttributeError: pass
    _refuse(f"{name}: a contiguous {dtype} tensor of {n} elements on device {i} is wanted")
def _table(t, r, c, i, name, dtype=_F32):
    """pointer of a contiguous [r, c] tensor on device i (None: null)"""
    if t is not None and getattr(t, "shape", None) != (r, c): _refuse(f"{name}: a tensor of shape {(r, c)} is wanted, not {tuple(getattr(t, 'shape', ()))}")
    return _vec(t, r * c, i, name, dtype)
def _workspace(n, i):
    """n bytes on device i, of the current stream (or of the graph that is being captured); None for none"""
    return torch.empty(n, dtype=torch.uint8, device=_devices[i]) if n else None
def _run(i, f, *args):
    """f(*args, stream) on device i and its current stream"""
    if i == _current_device(): status = f(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i): status = f(*args, _raw_stream(i))
    if status: _l.check(status)

class CuMatrix:
    def __init__(self, t):
        assert t.is_cuda and t.dtype == torch.float32 and t.dim() == 2 and t.stride(1) == 1
        self.t = t; self._L = _l.load()
    def NumRows(self): return self.t.shape[0]
    def NumCols(self): return self.t.shape[1]
    def Stride(self): return self.t.stride(0)
    def _a(self): return (self.t.data_ptr(), self.Stride(), self.NumRows(), self.NumCols())
    def AddMatMat(self, alpha, A, transA, B, transB, beta):
        M, N = self.NumRows(), self.NumCols(); K = A.NumRows() if transA else A.NumCols()
        assert (A.NumCols() if transA else A.NumRows()) == M and (B.NumRows() if transB else B.NumCols()) == N and (B.NumCols() if transB else B.NumRows()) == K
        _l.check(self._L.k3_mat_add_mat_mat(alpha, A.t.data_ptr(), A.Stride(), int(transA), B.t.data_ptr(), B.Stride(), int(transB), beta, self.t.data_ptr(), self.Stride(), M, N, K, _st()))
    def SetZero(self): self.Set(0.0)
    def Set(self, v): _l.check(self._L.k3_mat_set(*self._a(), v, _st()))
    def Scale(self, v): _l.check(self._L.k3_mat_scale(*self._a(), v, _st()))
    def Add(self, v): _l.check(self._L.k3_mat_add(*self._a(), v, _st()))
    def ApplyFloor(self, v): _l.check(self._L.k3_mat_apply_floor(*self._a(), v, _st()))
    def ApplyCeiling(self, v): _l.check(self._L.k3_mat_apply_ceiling(*self._a(), v, _st()))
    def CopyRowsFromVec(self, v): _l.check(self._L.k3_mat_copy_rows_from_vec(*self._a(), v.data_ptr(), _st()))
    def MulColsVec(self, v): _l.check(self._L.k3_mat_mul_cols_vec(*self._a(), v.data_ptr(), _st()))
    def MulRowsVec(self, v): _l.check(self._L.k3_mat_mul_rows_vec(*self._a(), v.data_ptr(), _st()))
    def AddVecToRows(self, alpha, row, beta=1.0): _l.check(self._L.k3_mat_add_vec_to_rows(alpha, row.data_ptr(), beta, *self._a(), _st()))
    def AddVecToCols(self, alpha, col, beta=1.0): _l.check(self._L.k3_mat_add_vec_to_cols(alpha, col.data_ptr(), beta, *self._a(), _st()))
    def CopyFromMat(self, M, trans=False): _l.check(self._L.k3_mat_copy_from_mat(*self._a(), M.t.data_ptr(), M.Stride(), int(trans), _st()))
    def AddMat(self, alpha, A, transA=False): _l.check(self._L.k3_mat_add_mat(alpha, A.t.data_ptr(), A.Stride(), int(transA), *self._a(), _st()))
    def CopyRows(self, src, indexes): _l.check(self._L.k3_mat_copy_rows(*self._a(), src.t.data_ptr(), src.Stride(), indexes.data_ptr(), _st()))
    def AddRows(self, alpha, src, indexes): _l.check(self._L.k3_mat_add_rows(alpha, src.t.data_ptr(), src.Stride(), indexes.data_ptr(), *self._a(), _st()))
    # ---- the parameter update's operations (natural gradient, max-change, orthonormal constraint)
    def SymAddMat2(self, alpha, A, transA, beta): self.AddMatMat(alpha, A, transA, A, not transA, beta)      # both triangles
    def CopyLowerToUpper(self): assert self.NumRows() == self.NumCols(); _l.check(self._L.k3_mat_copy_lower_to_upper(self.t.data_ptr(), self.Stride(), self.NumRows(), _st()))
    def AddToDiag(self, v): _l.check(self._L.k3_mat_add_to_diag(*self._a(), v, _st()))
    def AddVecVec(self, alpha, x, y): _l.check(self._L.k3_mat_add_vec_vec(alpha, x.data_ptr(), y.data_ptr(), *self._a(), _st()))
    def DivElements(self, A): _l.check(self._L.k3_mat_div_elements(*self._a(), A.t.data_ptr(), A.Stride(), _st()))
    def AddDiagVecMat(self, alpha, v, M, transM, beta):
        _l.check(self._L.k3_mat_add_diag_vec_mat(alpha, v.data_ptr(), M.t.data_ptr(), M.Stride(), int(transM), beta, self.t.data_ptr(), self.Stride(), self.NumRows(), self.NumCols(), _st()))
    # ---- the remaining nonlinearities of nnet3's simple components and their derivatives (cu-matrix.h:288-307,:386-396,:501-511; cu-math.h:272-300)
    def _map(self, op, src, a=0.0, flag=0): _l.check(self._L.k3_mat_apply_map(op, *self._a(), src.t.data_ptr(), src.Stride(), a, flag, _st()))
    def Sigmoid(self, src): self._map(0, src)
    def Tanh(self, src): self._map(1, src)
    def Log(self, src): self._map(2, src)
    def Pow(self, src, power): self._map(3, src, power)
    def PowAbs(self, src, power, include_sign=False): self._map(4, src, power, int(include_sign))
    def MaxMat(self, A): self._map(5, A)      # CuMatrixBase::Max(const CuMatrixBase &A) (Max() without an argument is the scalar reduction)
    def DiffSigmoid(self, value, diff): _l.check(self._L.k3_mat_diff_activation(0, *self._a(), value.t.data_ptr(), value.Stride(), diff.t.data_ptr(), diff.Stride(), _st()))
    def DiffTanh(self, value, diff): _l.check(self._L.k3_mat_diff_activation(1, *self._a(), value.t.data_ptr(), value.Stride(), diff.t.data_ptr(), diff.Stride(), _st()))
    def DivRowsVec(self, div): _l.check(self._L.k3_mat_div_rows_vec(*self._a(), div.data_ptr(), _st()))
    def CopyColsFromVec(self, v):
        if v.numel() == self.NumRows() * self.NumCols(): _l.check(self._L.k3_mat_copy_from_mat(*self._a(), v.data_ptr(), self.NumRows(), 1, _st()))      # the vector is the matrix column by column
        else: assert v.numel() == self.NumRows(); _l.check(self._L.k3_mat_copy_cols_from_vec(*self._a(), v.data_ptr(), _st()))
    def CopyColFromVec(self, v, col): assert v.numel() == self.NumRows(); _l.check(self._L.k3_mat_copy_from_mat(self.t.data_ptr() + 4 * col, self.Stride(), self.NumRows(), 1, v.data_ptr(), 1, 0, _st()))
    def CopyCols(self, src, indexes): _l.check(self._L.k3_mat_copy_cols(0, *self._a(), src.t.data_ptr(), src.Stride(), indexes.data_ptr(), _st()))
    def MulRows(self, src, indexes): _l.check(self._L.k3_mat_mul_rows(*self._a(), src.t.data_ptr(), src.Stride(), indexes.data_ptr(), _st()))
    def SetMatMatDivMat(self, A, B, C): _l.check(self._L.k3_mat_elements3(0, *self._a(), 1.0, A.t.data_ptr(), A.Stride(), B.t.data_ptr(), B.Stride(), C.t.data_ptr(), C.Stride(), 0.0, _st()))
    def AddMatMatElements(self, alpha, A, B, beta): _l.check(self._L.k3_mat_elements3(1, *self._a(), alpha, A.t.data_ptr(), A.Stride(), B.t.data_ptr(), B.Stride(), None, 0, beta, _st()))
    def AddCols(self, src, indexes): _l.check(self._L.k3_mat_copy_cols(1, *self._a(), src.t.data_ptr(), src.Stride(), indexes.data_ptr(), _st()))
    def _reduce(self, op, B=None):
        r = ctypes.c_double(0.0)
        _l.check(self._L.k3_mat_reduce_scalar(op, self.t.data_ptr(), self.Stride(), B.t.data_ptr() if B is not None else None, B.Stride() if B is not None else 0, self.NumRows(), self.NumCols(), ctypes.byref(r), _st()))
        return r.value
    def Trace(self): return self._reduce(2)
    def Sum(self): return self._reduce(3)
    def Max(self): return self._reduce(4)
    def Min(self): return self._reduce(5)

def TraceMatMat(A, B, trans=False): return A._reduce(0 if trans else 1, B)

def NormalizePerRow(inp, target_rms, add_log_stddev, out):      # cu::NormalizePerRow (cudamatrix/cu-math.h:272)
    assert out.NumRows() == inp.NumRows() and out.NumCols() == inp.NumCols() + int(add_log_stddev)
    _l.check(out._L.k3_mat_normalize_rows(0, out.t.data_ptr(), out.Stride(), inp.t.data_ptr(), inp.Stride(), None, 0, inp.NumRows(), inp.NumCols(), target_rms, int(add_log_stddev), _st()))
def DiffNormalizePerRow(in_value, out_deriv, target_rms, add_log_stddev, in_deriv):      # cu::DiffNormalizePerRow (cudamatrix/cu-math.h:296): ADDS to in_deriv unless it is out_deriv
    assert out_deriv.NumCols() == in_value.NumCols() + int(add_log_stddev) and in_deriv.NumCols() == in_value.NumCols()
    _l.check(in_deriv._L.k3_mat_normalize_rows(1, in_deriv.t.data_ptr(), in_deriv.Stride(), in_value.t.data_ptr(), in_value.Stride(), out_deriv.t.data_ptr(), out_deriv.Stride(), in_value.NumRows(), in_value.NumCols(), target_rms, int(add_log_stddev), _st()))

def LayerNormPerRow(inp, scale, offset, eps, out, mean=None, inv_std=None):
    """Layer norm: out = (inp - mean) inv_std scale + offset row by row, inv_std = 1 / sqrt(var + eps).  inp, out: matrices of one type (float32, float16, bfloat16), out may be inp;
    scale, offset: float32 vectors of the row length or None; mean, inv_std: float32 vectors of the number of rows that receive the statistics DiffLayerNormPerRow takes, or None."""
    x = _rows(inp, "inp"); dt, px, ldx, r, c, i = x; y, ldy = _like_rows(out, x, "out")
    if not 0.0 <= eps < float("inf"): _refuse(f"eps: {eps}")
    _run(i, _l.load().k3_layer_norm_forward, dt, px, ldx, _vec(scale, c, i, "scale"), _vec(offset, c, i, "offset"), eps, y, ldy, _vec(mean, r, i, "mean"), _vec(inv_std, r, i, "inv_std"), r, c)
def DiffLayerNormPerRow(in_value, out_deriv, scale, mean, inv_std, in_deriv=None, scale_deriv=None, offset_deriv=None, accumulate=False):
    """The backward pass of LayerNormPerRow from its input, its kept statistics and the derivative with respect to its output.  in_deriv (may be out_deriv or in_value) is overwritten;
    scale_deriv, offset_deriv (float32 vectors) are overwritten, or added to with accumulate.  What is None is not computed."""
    x = _rows(in_value, "in_value"); dt, px, ldx, r, c, i = x; g, ldg = _like_rows(out_deriv, x, "out_deriv")
    if mean is None or inv_std is None: _refuse("mean, inv_std: the statistics of the forward pass are wanted")
    d, ldd = (None, c) if in_deriv is None else _like_rows(in_deriv, x, "in_deriv")
    L = _l.load(); ws = None; n = 0
    if scale_deriv is not None or offset_deriv is not None: n = L.k3_layer_norm_backward_workspace(r, c); ws = _workspace(n, i)
    _run(i, L.k3_layer_norm_backward, dt, px, ldx, g, ldg, _vec(scale, c, i, "scale"), _vec(mean, r, i, "mean"), _vec(inv_std, r, i, "inv_std"), d, ldd,
         _vec(scale_deriv, c, i, "scale_deriv"), _vec(offset_deriv, c, i, "offset_deriv"), 1 if accumulate else 0, ws.data_ptr() if n else None, n, r, c)

ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "swish": 4, "gelu": 5}      # k3_activation
def _half_rows(m, name):
    x = _rows(m, name)
    if x[0] == 0: _refuse(f"{name}: float16 or bfloat16 is wanted (float32 products: CuMatrix.AddMatMat)")
    return x
def _rows_of(m, r, c, x, name):
    """a matrix of r x c of x's type and device (None: none): (pointer, leading dimension)"""
    if m is None: return None, c
    y = _rows(m, name)
    if y[3] != r or y[4] != c or y[0] != x[0] or y[5] != x[5]: _refuse(f"{name}: {y[3]} x {y[4]} of type {y[0]} on device {y[5]}: {r} x {c} of type {x[0]} on device {x[5]} is wanted")
    return y[1], y[2]
def AffinePerRow(inp, linear_params, bias_params, activation, residual, out, pre_activation=None):
    """An affine layer in float16 or bfloat16: out = activation(inp linear_params^T + bias_params) + residual.  inp [rows, inner], linear_params [cols, inner]; bias_params: float32 vector of
    cols or None; activation: one of ACTIVATIONS; residual [rows, cols] or None (out may be it); pre_activation [rows, cols] receives inp linear_params^T + bias_params, which
    DiffAffinePerRow takes, or None."""
    x = _half_rows(inp, "inp"); dt, px, ldx, r, k, i = x; act = ACTIVATIONS.get(activation)
    if act is None: _refuse(f"activation: {activation!r} is none of {', '.join(ACTIVATIONS)}")
    wt, pw, ldw, c, wk, wi = _rows(linear_params, "linear_params")
    if wt != dt or wk != k or wi != i: _refuse(f"linear_params: {c} x {wk} of type {wt} on device {wi} does not go with an input of {k} columns of type {dt} on device {i}")
    res, ldr = _rows_of(residual, r, c, x, "residual")
    if out is None: _refuse("out: a matrix is wanted")
    y, ldy = _rows_of(out, r, c, x, "out"); pre, ldp = _rows_of(pre_activation, r, c, x, "pre_activation")
    L = _l.load(); n = L.k3_affine_forward_workspace(r, k, c); ws = _workspace(n, i)
    _run(i, L.k3_affine_forward, dt, act, px, ldx, pw, ldw, _vec(bias_params, c, i, "bias_params"), res, ldr, y, ldy, pre, ldp, ws.data_ptr() if n else None, n, r, k, c)
def DiffAffinePerRow(in_value, linear_params, pre_activation, activation, out_deriv, in_deriv=None, linear_params_deriv=None, bias_params_deriv=None):
    """The backward pass of AffinePerRow from its input, its weights, the kept pre_activation (None for the activation "none") and the derivative with respect to its output, which is the
    residual's derivative too.  in_deriv, linear_params_deriv (matrices) and bias_params_deriv (float32 vector) are overwritten; what is None is not computed."""
    x = _half_rows(in_value, "in_value"); dt, px, ldx, r, k, i = x; act = ACTIVATIONS.get(activation)
    if act is None: _refuse(f"activation: {activation!r} is none of {', '.join(ACTIVATIONS)}")
    wt, pw, ldw, c, wk, wi = _rows(linear_params, "linear_params")
    if wt != dt or wk != k or wi != i: _refuse(f"linear_params: {c} x {wk} of type {wt} on device {wi} does not go with an input of {k} columns of type {dt} on device {i}")
    if out_deriv is None: _refuse("out_deriv: a matrix is wanted")
    if pre_activation is None and act: _refuse("pre_activation: what the forward pass kept is wanted")
    pre, ldp = _rows_of(pre_activation, r, c, x, "pre_activation"); g, ldg = _rows_of(out_deriv, r, c, x, "out_deriv")
    dx, lddx = _rows_of(in_deriv, r, k, x, "in_deriv"); dw, lddw = _rows_of(linear_params_deriv, c, k, x, "linear_params_deriv")
    L = _l.load(); n = L.k3_affine_backward_workspace(act, r, k, c); ws = _workspace(n, i)
    _run(i, L.k3_affine_backward, dt, act, px, ldx, pw, ldw, pre, ldp, g, ldg, dx, lddx, dw, lddw, _vec(bias_params_deriv, c, i, "bias_params_deriv"), ws.data_ptr() if n else None, n, r, k, c)

class CuRand:
    """CuRand<BaseFloat> (cudamatrix/cu-rand.h:31-64) over k3_mat_set_rand: one seed per object, the counter position advances by what each fill consumes"""
    def __init__(self, seed=0): self.seed, self.offset, self._L = int(seed), 0, _l.load()
    def _fill(self, kind, M):
        _l.check(self._L.k3_mat_set_rand(kind, M.t.data_ptr(), M.Stride(), M.NumRows(), M.NumCols(), self.seed, self.offset, _st())); self.offset += (M.NumRows() * M.NumCols() + 3) // 4
    def RandUniform(self, M): self._fill(0, M)
    def RandGaussian(self, M): self._fill(1, M)
