"""Tensor-level calls of the serving operators (include/ecog2txt_hip.h: e2t_quant_rows_i8, e2t_gemm_nt_i8, e2t_linear_i8,
e2t_sample_rows): argument checks, outputs and workspaces; everything runs on the calling thread's current stream of the
tensors' device.  Workspaces come from torch's allocator per call, so calls on different streams, and graphs captured from them,
share none.  Weights are quantised once (`quantize_rows`) and kept by the caller as an `Int8Rows`.

Nothing here has a gradient: tensors that ask for one are refused."""
import ctypes as C

import torch

from . import hip_lib as H

_DTYPE = {torch.float32: H.DT_F32, torch.bfloat16: H.DT_BF16}
_FLOATS, _INT8 = (torch.float32, torch.bfloat16), (torch.int8,)
# the calling thread's current stream of a device, as an integer (one C call; torch.cuda.current_stream builds a Stream object: 3 us)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _bad(what):
    raise ValueError('ecog2txt_amd.serving: ' + what)


class _Native:
    """The library's functions, looked up once (loading it on the first use)."""

    def __getattr__(self, name):
        fn = getattr(H.load(), name)
        setattr(self, name, fn)
        return fn


_c = _Native()


def _call(index, fn, *args):
    """fn(*args, the current stream) with device `index` current."""
    was = torch.cuda.current_device()
    if was == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        raise RuntimeError('%s failed (%d): %s' % (fn.__name__, rc, _c.e2t_last_error().decode()))


def _matrix(x, name, dtypes):
    """Row stride of a 2-D device tensor with contiguous rows."""
    if isinstance(x, torch.Tensor) and x.dtype in dtypes and x.is_cuda and x.dim() == 2 and not (x.requires_grad and torch.is_grad_enabled()):
        (rows, cols), (s0, s1) = x.shape, x.stride()
        if s1 == 1 and s0 >= cols > 0:
            return s0
        if cols == 0:
            _bad('%s has no columns' % name)
        if s1 != 1 and cols > 1:
            _bad('%s must have contiguous rows (stride 1 along the last dimension)' % name)
        if s0 < cols and rows > 1:
            _bad('rows of %s overlap' % name)
        return max(s0, cols)
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        _bad('%s asks for a gradient: the serving operators have none (use torch.no_grad())' % name)
    _bad('%s must be a 2-D device tensor of %s' % (name, ' / '.join(str(d).replace('torch.', '') for d in dtypes)))


def _vector(v, n, dtype, index, name):
    if not isinstance(v, torch.Tensor) or v.dtype is not dtype or v.get_device() != index or v.dim() != 1 or v.shape[0] != n or not v.is_contiguous():
        _bad('%s must be a contiguous %s tensor of %d on device %d' % (name, str(dtype).replace('torch.', ''), n, index))
    return v.data_ptr()


def _out(out, rows, cols, dtype, like):
    """(tensor, row stride) of the output."""
    if out is None:
        return torch.empty((rows, cols), dtype=dtype, device=like.device), cols
    ld = _matrix(out, 'out', (dtype,))
    if out.get_device() != like.get_device() or out.shape[0] != rows or out.shape[1] != cols:
        _bad('out must be (%d, %d) on %s' % (rows, cols, like.device))
    return out, ld


class Int8Rows:
    """A matrix in 8 bits: row i stands for scale[i] * q[i, :cols].  q int8 [rows, >= cols rounded up to 64] (zeros from `cols` up
    to that), rows 16-byte aligned; scale fp32 [rows]."""
    __slots__ = ('q', 'scale', 'cols', 'ld')

    def __init__(self, q, scale, cols):
        ld = _matrix(q, 'q', _INT8)
        width = q.shape[1]
        if not 0 < cols <= width - (-cols) % 64:
            _bad('q needs %d columns (the %d of the matrix, rounded up to 64)' % ((cols + 63) // 64 * 64, cols))
        if cols > 131071:
            _bad('more than 131071 columns overflow the 32-bit sums')
        if q.shape[0] <= 1:
            ld = width // 64 * 64
        if (ld | q.data_ptr()) & 15:
            _bad('the rows of q must start on 16-byte boundaries')
        _vector(scale, q.shape[0], torch.float32, q.get_device(), 'scale')
        self.q, self.scale, self.cols, self.ld = q, scale, int(cols), ld

    @property
    def rows(self):
        return self.q.shape[0]

    def float(self):
        """The values it stands for, fp32 [rows, cols]."""
        return self.q[:, :self.cols].float() * self.scale[:, None]


def quantize_rows(x):
    """Symmetric 8-bit rows of a [rows, cols] fp32 or bf16 tensor: activations (a scale for each token) or a weight matrix stored as
    [outputs, inputs] (a scale for each output channel)."""
    ldx = _matrix(x, 'x', _FLOATS)
    rows, cols = x.shape
    q = torch.empty(rows, (cols + 63) // 64 * 64, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    r = Int8Rows(q, scale, cols)
    if rows:
        _call(x.get_device(), _c.e2t_quant_rows_i8, x.data_ptr(), _DTYPE[x.dtype], ldx, rows, cols, q.data_ptr(), q.shape[1], scale.data_ptr())
    return r


def _weights(w, cols, bias, out_dtype, relu, index):
    if not isinstance(w, Int8Rows) or w.q.get_device() != index:
        _bad('the weights must be Int8Rows on device %d' % index)
    n = w.q.shape[0]
    if w.cols != cols:
        _bad('%d columns of activations, %d of weights' % (cols, w.cols))
    if n == 0:
        _bad('the weights have no rows')
    if out_dtype not in _DTYPE:
        _bad('out_dtype must be float32 or bfloat16')
    b = None if bias is None else _vector(bias, n, torch.float32, index, 'bias')
    return n, b, (H.GEMM_RELU if relu else 0) | (H.GEMM_OUT_BF16 if out_dtype is torch.bfloat16 else 0)


def matmul_i8(a, w, bias=None, out_dtype=torch.float32, relu=False, out=None):
    """a . w^T (+ bias) of two Int8Rows: [a.rows, w.rows], the integer sums exact.  out (or None): where to, overlapping no input."""
    if not isinstance(a, Int8Rows):
        _bad('a must be Int8Rows')
    q, index = a.q, a.q.get_device()
    n, b, flags = _weights(w, a.cols, bias, out_dtype, relu, index)
    m = q.shape[0]
    y, ldy = _out(out, m, n, out_dtype, q)
    if m:
        _call(index, _c.e2t_gemm_nt_i8, q.data_ptr(), a.ld, a.scale.data_ptr(), w.q.data_ptr(), w.ld, w.scale.data_ptr(), b, y.data_ptr(), ldy,
              m, n, a.cols, flags)
    return y


def linear_i8(x, w, bias=None, out_dtype=torch.float32, relu=False, out=None):
    """quantize_rows(x) . w^T (+ bias) in one call: x fp32 or bf16 [rows, cols], w Int8Rows.  out (or None): where to, overlapping no input."""
    ldx = _matrix(x, 'x', _FLOATS)
    (m, cols), index = x.shape, x.get_device()
    n, b, flags = _weights(w, cols, bias, out_dtype, relu, index)
    y, ldy = _out(out, m, n, out_dtype, x)
    if m:
        need = _c.e2t_linear_i8_ws_bytes(m, n, cols)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        _call(index, _c.e2t_linear_i8, x.data_ptr(), _DTYPE[x.dtype], ldx, w.q.data_ptr(), w.ld, w.scale.data_ptr(), b, y.data_ptr(), ldy,
              m, n, cols, flags, ws.data_ptr() if need else None, need)
    return y


def sample_config(rows, index, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """e2t_sample_cfg from numbers (all rows alike) or tensors of `rows` on device `index` (fp32; top_k int32), which must outlive the
    call it is used in."""
    c = H.SampleCfg()
    if isinstance(temperature, torch.Tensor):
        c.temperature_rows = _vector(temperature, rows, torch.float32, index, 'temperature')
    else:
        c.temperature = temperature
    if isinstance(top_k, torch.Tensor):
        c.top_k_rows = _vector(top_k, rows, torch.int32, index, 'top_k')
    else:
        c.top_k = max(0, min(int(top_k), 2 ** 31 - 1))
    if isinstance(top_p, torch.Tensor):
        c.top_p_rows = _vector(top_p, rows, torch.float32, index, 'top_p')
    else:
        c.top_p = top_p
    if isinstance(min_p, torch.Tensor):
        c.min_p_rows = _vector(min_p, rows, torch.float32, index, 'min_p')
    else:
        c.min_p = min_p
    return c


def sample_rows(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token for each row of logits [rows, vocabulary] (fp32 or bf16) from one uniform number a row, u fp32 [rows] in [0, 1):
    (token int32 [rows], log-probability among the kept tokens fp32 [rows]).  Settings are numbers or device tensors of one value
    a row; temperature <= 0 takes the largest logit, top_k <= 0, top_p >= 1 and min_p <= 0 keep everything."""
    ldl = _matrix(logits, 'logits', _FLOATS)
    (rows, vocab), index, dev = logits.shape, logits.get_device(), logits.device
    up = _vector(u, rows, torch.float32, index, 'u')
    cfg = sample_config(rows, index, temperature, top_k, top_p, min_p)
    token = torch.empty(rows, dtype=torch.int32, device=dev)
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    if rows:
        need = _c.e2t_sample_ws_bytes(rows, vocab)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _call(index, _c.e2t_sample_rows, logits.data_ptr(), _DTYPE[logits.dtype], ldl, rows, vocab, up, C.byref(cfg), token.data_ptr(),
              logprob.data_ptr(), ws.data_ptr() if need else None, need)
    return token, logprob
