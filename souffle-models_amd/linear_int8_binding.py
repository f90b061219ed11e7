"""linear_int8_binding: linear layers in 8-bit integers (a wrapper over the C ABI; the reference has no counterpart).

    w = quantize_weight(weight)                     # once per model: [K, N] fp16 / bf16 / fp32 -> Int8Weight
    y = linear_int8(x, w, bias=b, act="gelu")       # rows of x quantised as they come, y of x's type
    q, s = quantize_rows(x)                         # the two steps apart, where q feeds more than one product
    y = gemm_int8(q, s, w, dtype=torch.float16)     #   (or comes from gated_norm_binding.gated_norm_int8)

A row x is held as q = round_half_even(x / s), s = max(max|x| / 127, 2^-100) in fp32, a weight column likewise; products
sum in exact 32-bit integers.  A row with a NaN or an infinity gives a row of NaN.  Work is queued on the current
stream of the tensors' device; nothing is kept between calls, so calls may overlap on several streams and be captured.
"""
from typing import NamedTuple

import torch

import souffle_hip as sh

_DTYPES = {torch.float16: sh.F16, torch.bfloat16: sh.BF16, torch.float32: sh.F32}
_ACTS = {None: sh.ACT_NONE, "relu": sh.ACT_RELU, "gelu": sh.ACT_GELU_ERF, "gelu_tanh": sh.ACT_GELU_TANH}


class Int8Weight(NamedTuple):
    """A weight matrix [in_features, out_features] in 8 bits: the packed bytes (layout: include/souffle_hip.h) and the
    fp32 scale of each output channel."""
    packed: torch.Tensor
    scale: torch.Tensor
    in_features: int
    out_features: int


def _check_cuda(name, t, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))


def _rows(name, t):
    """(t as [rows, columns] with adjacent columns, distance of its rows in elements)."""
    if t.dim() < 1 or (t.dim() > 2 and not t.is_contiguous()):
        raise ValueError("%s must be [rows, columns], or contiguous with more dimensions" % name)
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((t.shape[:-1].numel(), t.shape[-1]))
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("the columns of %s must be adjacent" % name)
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if ld < t.shape[1]:
        raise ValueError("the rows of %s overlap" % name)
    return t, ld


def _check_weight(w, device):
    if not isinstance(w, Int8Weight):
        raise TypeError("weight must be an Int8Weight (quantize_weight, pack_weight)")
    _check_cuda("weight.packed", w.packed, device)
    _check_cuda("weight.scale", w.scale, device)
    if w.packed.dtype != torch.int8 or not w.packed.is_contiguous() or w.packed.numel() != -(-w.in_features // 64) * -(-w.out_features // 64) * 4096:
        raise ValueError("weight.packed must hold the packed [%d, %d] matrix as contiguous int8" % (w.in_features, w.out_features))
    if w.scale.dtype != torch.float32 or not w.scale.is_contiguous() or w.scale.numel() != w.out_features:
        raise ValueError("weight.scale must hold %d contiguous float32" % w.out_features)


def _epilogue(bias, act, n, dtype, device):
    if act not in _ACTS:
        raise ValueError("act must be None, 'relu', 'gelu' or 'gelu_tanh', got %r" % (act,))
    if bias is None:
        return None, _ACTS[act]
    _check_cuda("bias", bias, device)
    if bias.dtype != dtype or not bias.is_contiguous() or bias.numel() != n:
        raise ValueError("bias must be %d contiguous values of %s" % (n, dtype))
    return bias.data_ptr(), _ACTS[act]


def _output(out, rows, n, dtype, device):
    if out is None:
        return torch.empty((rows, n), dtype=dtype, device=device), n
    _check_cuda("out", out, device)
    if out.dtype != dtype or out.dim() != 2 or tuple(out.shape) != (rows, n):
        raise ValueError("out must be [%d, %d] of %s" % (rows, n, dtype))
    return _rows("out", out)


def pack_weight(weight_q, scale):
    """Int8Weight of an int8 matrix [K, N] and the float32 scale [N] of its columns."""
    _check_cuda("weight_q", weight_q)
    _check_cuda("scale", scale, weight_q.device)
    if weight_q.dtype != torch.int8 or weight_q.dim() != 2:
        raise TypeError("weight_q must be an int8 matrix [K, N]")
    (w, ld), (K, N) = _rows("weight_q", weight_q), weight_q.shape
    if scale.dtype != torch.float32 or scale.dim() != 1 or scale.numel() != N:
        raise ValueError("scale must be [%d] float32" % N)
    with torch.cuda.device(w.device):
        packed = torch.empty(sh.lib().souffle_int8_packed_bytes(K, N), dtype=torch.int8, device=w.device)
        sh.check(sh.lib().souffle_int8_pack_weight(w.data_ptr(), ld, packed.data_ptr(), K, N, sh.current_stream()))
    return Int8Weight(packed, scale.contiguous(), K, N)


def quantize_weight(weight):
    """Int8Weight of a matrix [K, N] in fp16, bf16 or fp32, quantised per output channel.  Once per model."""
    _check_cuda("weight", weight)
    if weight.dtype not in _DTYPES or weight.dim() != 2:
        raise TypeError("weight must be a float16, bfloat16 or float32 matrix [K, N]")
    (w, ld), (K, N) = _rows("weight", weight), weight.shape
    with torch.cuda.device(w.device):
        packed = torch.empty(sh.lib().souffle_int8_packed_bytes(K, N), dtype=torch.int8, device=w.device)
        scale = torch.empty(N, dtype=torch.float32, device=w.device)
        sh.check(sh.lib().souffle_int8_quantize_weight(w.data_ptr(), _DTYPES[w.dtype], ld, packed.data_ptr(), scale.data_ptr(), K, N,
                                                       sh.current_stream()))
    return Int8Weight(packed, scale, K, N)


def quantize_rows(x):
    """(q, row_scale) of x [..., K] (more than two dimensions: contiguous): q [rows, K] int8 in rows that lie K rounded
    up to 64 bytes apart, row_scale [rows] float32."""
    _check_cuda("x", x)
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float16, bfloat16 or float32")
    x, ld = _rows("x", x)
    M, K = x.shape
    with torch.cuda.device(x.device):
        ldq = -(-K // 64) * 64
        q = torch.empty((M, ldq), dtype=torch.int8, device=x.device)
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
        sh.check(sh.lib().souffle_quantize_rows(x.data_ptr(), _DTYPES[x.dtype], ld, q.data_ptr(), ldq, scale.data_ptr(), M, K,
                                                sh.current_stream()))
    return q[:, :K], scale


def gemm_int8(q, row_scale, weight, *, bias=None, act=None, dtype=torch.float16, out=None):
    """act(row_scale * weight.scale * (q . W) + bias) as [rows, N] of `dtype`.  q [rows, K] int8: rows that start at
    multiples of 16 bytes and can be read up to K rounded up to 64 bytes (as quantize_rows and gated_norm_int8 make
    them; what lies behind K does not matter).  bias is of `dtype`; out: a [rows, N] tensor to write to."""
    _check_cuda("q", q)
    dev = q.device
    _check_cuda("row_scale", row_scale, dev)
    _check_weight(weight, dev)
    K, N = weight.in_features, weight.out_features
    if q.dtype != torch.int8 or q.dim() != 2 or q.shape[1] != K:
        raise ValueError("q must be [rows, %d] int8" % K)
    if dtype not in _DTYPES:
        raise TypeError("dtype must be float16, bfloat16 or float32")
    M = q.shape[0]
    if row_scale.dtype != torch.float32 or not row_scale.is_contiguous() or row_scale.numel() != M:
        raise ValueError("row_scale must hold %d contiguous float32" % M)
    if K > 1 and q.stride(1) != 1:
        raise ValueError("the columns of q must be adjacent")
    need = -(-K // 64) * 64
    ldq = q.stride(0) if M > 1 else need
    if M > 0 and q.untyped_storage().nbytes() < q.storage_offset() + (M - 1) * ldq + need:
        raise ValueError("the rows of q must be readable up to %d bytes each (quantize_rows makes such rows)" % need)
    b, a = _epilogue(bias, act, N, dtype, dev)
    with torch.cuda.device(dev):
        out, ldy = _output(out, M, N, dtype, dev)
        sh.check(sh.lib().souffle_gemm_int8(q.data_ptr(), ldq, row_scale.data_ptr(), weight.packed.data_ptr(), weight.scale.data_ptr(),
                                            b, a, out.data_ptr(), _DTYPES[dtype], ldy, M, N, K, sh.current_stream()))
    return out


def linear_int8(x, weight, *, bias=None, act=None, out=None):
    """act(x . W + bias) with the rows of x [..., K] in 8 bits: quantize_rows and gemm_int8 in one call, bit for bit.
    Returns [rows, N] of x's type; bias is of that type too."""
    _check_cuda("x", x)
    dev = x.device
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float16, bfloat16 or float32")
    _check_weight(weight, dev)
    K, N = weight.in_features, weight.out_features
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError("x must be [..., %d]" % K)
    x, ld = _rows("x", x)
    M = x.shape[0]
    b, a = _epilogue(bias, act, N, x.dtype, dev)
    with torch.cuda.device(dev):
        out, ldy = _output(out, M, N, x.dtype, dev)
        nbytes = sh.lib().souffle_linear_int8_workspace_bytes(M, K)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        sh.check(sh.lib().souffle_linear_int8(x.data_ptr(), ld, weight.packed.data_ptr(), weight.scale.data_ptr(), b, a, out.data_ptr(),
                                              _DTYPES[x.dtype], ldy, M, N, K, sh.ptr(ws), nbytes, sh.current_stream()))
    return out
