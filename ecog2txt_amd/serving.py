"""Tensor-level calls of the serving operators (include/ecog2txt_hip.h: e2t_quant_rows_i8, e2t_gemm_nt_i8, e2t_linear_i8,
e2t_sample_rows): argument checks, outputs and workspaces; everything runs on the calling thread's current stream of the
tensors' device.  Workspaces come from torch's allocator per call, so calls on different streams, and graphs captured from them,
share none.  Weights are quantised once (`quantize_rows`) and kept by the caller as an `Int8Rows`.

Nothing here has a gradient: tensors that ask for one are refused."""
import ctypes as C

import torch

from . import hip_lib as H
from .hip_lib import lib

_DTYPE = {torch.float32: H.DT_F32, torch.bfloat16: H.DT_BF16}


def _bad(what):
    raise ValueError('ecog2txt_amd.serving: ' + what)


def _stream_of(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _matrix(x, name, dtypes):
    """Row stride of a 2-D device tensor with contiguous rows."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.device.type != 'cuda' or x.dtype not in dtypes:
        _bad('%s must be a 2-D device tensor of %s' % (name, ' / '.join(str(d).replace('torch.', '') for d in dtypes)))
    if x.requires_grad and torch.is_grad_enabled():
        _bad('%s asks for a gradient: the serving operators have none (use torch.no_grad())' % name)
    rows, cols = x.shape
    if cols == 0:
        _bad('%s has no columns' % name)
    if x.stride(1) != 1 and cols > 1:
        _bad('%s must have contiguous rows (stride 1 along the last dimension)' % name)
    if rows > 1 and x.stride(0) < cols:
        _bad('rows of %s overlap' % name)
    return x.stride(0) if rows > 1 else max(x.stride(0), cols)


def _vector(v, n, dtype, dev, name):
    if not isinstance(v, torch.Tensor) or v.dtype != dtype or v.device != dev or v.dim() != 1 or v.shape[0] != n or not v.is_contiguous():
        _bad('%s must be a contiguous %s tensor of %d on %s' % (name, str(dtype).replace('torch.', ''), n, dev))
    return v.data_ptr()


def _out(out, shape, dtype, dev):
    """(tensor, row stride) of the output."""
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    elif out.device != dev or tuple(out.shape) != tuple(shape):
        _bad('out must be %s on %s' % (tuple(shape), dev))
    return out, _matrix(out, 'out', (dtype,))


class Int8Rows:
    """A matrix in 8 bits: row i stands for scale[i] * q[i, :cols].  q int8 [rows, >= cols rounded up to 64] (zeros from `cols` up
    to that), rows 16-byte aligned; scale fp32 [rows]."""
    __slots__ = ('q', 'scale', 'cols', 'ld')

    def __init__(self, q, scale, cols):
        self.ld = _matrix(q, 'q', (torch.int8,))
        if not 0 < cols or q.shape[1] < (cols + 63) // 64 * 64:
            _bad('q needs %d columns (the %d of the matrix, rounded up to 64)' % ((cols + 63) // 64 * 64, cols))
        if cols > 131071:
            _bad('more than 131071 columns overflow the 32-bit sums')
        if self.ld % 16 or q.data_ptr() % 16:
            _bad('the rows of q must start on 16-byte boundaries')
        _vector(scale, q.shape[0], torch.float32, q.device, 'scale')
        self.q, self.scale, self.cols = q, scale, int(cols)

    @property
    def rows(self):
        return self.q.shape[0]

    def float(self):
        """The values it stands for, fp32 [rows, cols]."""
        return self.q[:, :self.cols].float() * self.scale[:, None]


def quantize_rows(x):
    """Symmetric 8-bit rows of a [rows, cols] fp32 or bf16 tensor: activations (a scale for each token) or a weight matrix stored as
    [outputs, inputs] (a scale for each output channel)."""
    ldx = _matrix(x, 'x', (torch.float32, torch.bfloat16))
    rows, cols = x.shape
    q = torch.empty(rows, (cols + 63) // 64 * 64, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    r = Int8Rows(q, scale, cols)
    if rows:
        with torch.cuda.device(x.device):
            lib.e2t_quant_rows_i8(x.data_ptr(), _DTYPE[x.dtype], ldx, rows, cols, q.data_ptr(), q.shape[1], scale.data_ptr(), _stream_of(x.device))
    return r


def _weights(w, cols, bias, out_dtype, relu, dev):
    if not isinstance(w, Int8Rows) or w.q.device != dev:
        _bad('the weights must be Int8Rows on %s' % (dev,))
    if w.cols != cols:
        _bad('%d columns of activations, %d of weights' % (cols, w.cols))
    if w.rows == 0:
        _bad('the weights have no rows')
    if out_dtype not in _DTYPE:
        _bad('out_dtype must be float32 or bfloat16')
    b = None if bias is None else _vector(bias, w.rows, torch.float32, dev, 'bias')
    return b, (H.GEMM_RELU if relu else 0) | (H.GEMM_OUT_BF16 if out_dtype == torch.bfloat16 else 0)


def matmul_i8(a, w, bias=None, out_dtype=torch.float32, relu=False, out=None):
    """a . w^T (+ bias) of two Int8Rows: [a.rows, w.rows], the integer sums exact."""
    if not isinstance(a, Int8Rows):
        _bad('a must be Int8Rows')
    dev = a.q.device
    b, flags = _weights(w, a.cols, bias, out_dtype, relu, dev)
    y, ldy = _out(out, (a.rows, w.rows), out_dtype, dev)
    if a.rows:
        with torch.cuda.device(dev):
            lib.e2t_gemm_nt_i8(a.q.data_ptr(), a.ld, a.scale.data_ptr(), w.q.data_ptr(), w.ld, w.scale.data_ptr(), b, y.data_ptr(), ldy,
                               a.rows, w.rows, a.cols, flags, _stream_of(dev))
    return y


def linear_i8(x, w, bias=None, out_dtype=torch.float32, relu=False, out=None):
    """quantize_rows(x) . w^T (+ bias) in one call: x fp32 or bf16 [rows, cols], w Int8Rows."""
    ldx = _matrix(x, 'x', (torch.float32, torch.bfloat16))
    rows, cols = x.shape
    dev = x.device
    b, flags = _weights(w, cols, bias, out_dtype, relu, dev)
    y, ldy = _out(out, (rows, w.rows), out_dtype, dev)
    if rows:
        n = lib.e2t_linear_i8_ws_bytes(rows, cols)
        with torch.cuda.device(dev):
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            lib.e2t_linear_i8(x.data_ptr(), _DTYPE[x.dtype], ldx, w.q.data_ptr(), w.ld, w.scale.data_ptr(), b, y.data_ptr(), ldy, rows,
                              w.rows, cols, flags, ws.data_ptr(), n, _stream_of(dev))
    return y


def sample_config(rows, dev, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """e2t_sample_cfg from numbers (all rows alike) or device tensors of `rows` (fp32; top_k int32).  The tensors must outlive the
    call it is used in."""
    c = H.SampleCfg()
    for name, v, dtype in (('temperature', temperature, torch.float32), ('top_k', top_k, torch.int32), ('top_p', top_p, torch.float32),
                           ('min_p', min_p, torch.float32)):
        if isinstance(v, torch.Tensor):
            setattr(c, name + '_rows', _vector(v, rows, dtype, dev, name))
        elif dtype is torch.int32:
            setattr(c, name, max(0, min(int(v), 2 ** 31 - 1)))
        else:
            setattr(c, name, float(v))
    return c


def sample_rows(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token for each row of logits [rows, vocabulary] (fp32 or bf16) from one uniform number a row, u fp32 [rows] in [0, 1):
    (token int32 [rows], log-probability among the kept tokens fp32 [rows]).  Settings are numbers or device tensors of one value
    a row; temperature <= 0 takes the largest logit, top_k <= 0, top_p >= 1 and min_p <= 0 keep everything."""
    ldl = _matrix(logits, 'logits', (torch.float32, torch.bfloat16))
    rows, vocab = logits.shape
    dev = logits.device
    up = _vector(u, rows, torch.float32, dev, 'u')
    cfg = sample_config(rows, dev, temperature, top_k, top_p, min_p)
    token = torch.empty(rows, dtype=torch.int32, device=dev)
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    if rows:
        n = lib.e2t_sample_ws_bytes(rows, vocab)
        with torch.cuda.device(dev):
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            lib.e2t_sample_rows(logits.data_ptr(), _DTYPE[logits.dtype], ldl, rows, vocab, up, C.byref(cfg), token.data_ptr(),
                                logprob.data_ptr(), ws.data_ptr(), n, _stream_of(dev))
    return token, logprob
