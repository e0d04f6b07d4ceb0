"""Tensor-level calls of the serving operators (include/ecog2txt_hip.h: e2t_quant_rows_i8, e2t_gemm_nt_i8, e2t_linear_i8,
e2t_sample_rows): argument checks, outputs and workspaces; everything runs on the calling thread's current stream of the
tensors' device.  Workspaces come from torch's allocator per call, so calls on different streams, and graphs captured from them,
share none.  Weights are quantised once (`quantize_rows`) and kept by the caller as an `Int8Rows`.

The checks and the calls themselves are native (csrc/serving_host.cpp).  What cannot be served raises ValueError; nothing here has a
gradient: tensors that ask for one, operands, scales, bias and settings alike, are refused, in forward mode too."""
import ctypes as C

import torch

from . import hip_lib as H

_host = None


def _bind():
    """The native host module, with the library's functions handed to it (on the first use)."""
    global _host
    lib = H.load()
    try:
        from . import _serving_host as host
    except ImportError as e:
        raise RuntimeError('ecog2txt_amd/_serving_host.so is not built or does not fit this torch (%s). Run `python -c "import __graft_entry__ as g; '
                           'g.build()"` or ecog2txt_amd/csrc/build.sh.' % e) from e
    names = ('e2t_quant_rows_i8', 'e2t_gemm_nt_i8', 'e2t_linear_i8_ws_bytes', 'e2t_linear_i8', 'e2t_sample_ws_bytes', 'e2t_sample_rows', 'e2t_last_error')
    stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
    host.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in names}, stream, Int8Rows)
    _host = host
    return host


class Int8Rows:
    """A matrix in 8 bits: row i stands for scale[i] * q[i, :cols].  q int8 [rows, >= cols rounded up to 64] (zeros from `cols` up
    to that), rows 16-byte aligned and at most 8388608 bytes apart; scale fp32 [rows].  At most 131071 columns.  (Checked again in every
    call that it is used in.)"""
    __slots__ = ('q', 'scale', 'cols', 'ld')

    def __init__(self, q, scale, cols):
        self.ld = (_host or _bind()).check_rows(q, scale, cols)
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
    q, scale = (_host or _bind()).quantize(x)
    return Int8Rows(q, scale, x.shape[1])


def matmul_i8(a, w, bias=None, out_dtype=torch.float32, relu=False, out=None):
    """a . w^T (+ bias) of two Int8Rows: [a.rows, w.rows], the integer sums exact.  out (or None): where to, overlapping no input."""
    return (_host or _bind()).matmul(a, w, bias, out_dtype, relu, out)


def linear_i8(x, w, bias=None, out_dtype=torch.float32, relu=False, out=None):
    """quantize_rows(x) . w^T (+ bias) in one call: x fp32 or bf16 [rows, cols], w Int8Rows.  out (or None): where to, overlapping no input."""
    return (_host or _bind()).linear(x, w, bias, out_dtype, relu, out)


def _rows_array(v, rows, dtype, index, name):
    if v.requires_grad and torch.is_grad_enabled():
        raise ValueError('ecog2txt_amd.serving: %s asks for a gradient: the serving operators have none (use torch.no_grad())' % name)
    if v.dtype is not dtype or v.get_device() != index or v.dim() != 1 or v.shape[0] != rows or not v.is_contiguous():
        raise ValueError('ecog2txt_amd.serving: %s must be a contiguous %s tensor of %d on device %d' % (name, str(dtype).replace('torch.', ''), rows, index))
    return v.data_ptr()


def sample_config(rows, index, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """e2t_sample_cfg from numbers (all rows alike) or tensors of `rows` on device `index` (fp32; top_k int32), which must outlive the
    call it is used in."""
    c = H.SampleCfg()
    if isinstance(temperature, torch.Tensor):
        c.temperature_rows = _rows_array(temperature, rows, torch.float32, index, 'temperature')
    else:
        c.temperature = temperature
    if isinstance(top_k, torch.Tensor):
        c.top_k_rows = _rows_array(top_k, rows, torch.int32, index, 'top_k')
    else:
        c.top_k = max(0, min(int(top_k), 2 ** 31 - 1))
    if isinstance(top_p, torch.Tensor):
        c.top_p_rows = _rows_array(top_p, rows, torch.float32, index, 'top_p')
    else:
        c.top_p = top_p
    if isinstance(min_p, torch.Tensor):
        c.min_p_rows = _rows_array(min_p, rows, torch.float32, index, 'min_p')
    else:
        c.min_p = min_p
    return c


def sample_rows(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token for each row of logits [rows, vocabulary] (fp32 or bf16) from one uniform number a row, u fp32 [rows] in [0, 1):
    (token int32 [rows], log-probability among the kept tokens fp32 [rows]).  Settings are numbers or device tensors of one value
    a row; temperature <= 0 takes the largest logit, top_k <= 0, top_p >= 1 and min_p <= 0 keep everything.  At most 1048576 tokens a row, any number of rows."""
    return (_host or _bind()).sample(logits, u, temperature, top_k, top_p, min_p)
