"""linear_int8_binding: linear layers in 8-bit integers (a wrapper over the C ABI; the reference has no counterpart).

    w = quantize_weight(weight)                     # once per model: [K, N] fp16 / bf16 / fp32 -> Int8Weight
    y = linear_int8(x, w, bias=b, act="gelu")       # rows of x quantised as they come, y of x's type
    q, s = quantize_rows(x)                         # the two steps apart, where q feeds more than one product
    y = gemm_int8(q, s, w, dtype=torch.float16)     #   (or comes from gated_norm_binding.gated_norm_int8)

A row x is held as q = round_half_even(x / s), s = max(max|x| / 127, 2^-100) in fp32, a weight column likewise; products
sum in exact 32-bit integers.  x [..., K] may be any slice whose rows lie at one distance (x[..., a:b], x[:, -1:]).  A row with a NaN or an infinity gives a row of NaN.  Work is queued on the current
stream of the tensors' device; nothing is kept between calls, so calls may overlap on several streams and be captured.
They are for inference: autograd does not record them, so their results require no gradient, whatever x requires.
"""
import functools
from typing import NamedTuple

import torch

import souffle_hip as sh

# Index of the current device, and hipStream_t of a device's current stream, without the objects that torch.cuda makes of them
# (they take 1.3 and 2.8 us, a call of one row some 8).
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream

_DTYPES = {torch.float16: sh.F16, torch.bfloat16: sh.BF16, torch.float32: sh.F32}
_ACTS = {None: sh.ACT_NONE, "relu": sh.ACT_RELU, "gelu": sh.ACT_GELU_ERF, "gelu_tanh": sh.ACT_GELU_TANH}


class Int8Weight(NamedTuple):
    """A weight matrix [in_features, out_features] in 8 bits: the packed bytes (layout: include/souffle_hip.h) and the
    fp32 scale of each output channel."""
    packed: torch.Tensor
    scale: torch.Tensor
    in_features: int
    out_features: int


def _check_cuda(name, t, index=None):
    """The index of t's device, which has to be `index` where one is given."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    at = t.get_device()
    if index is not None and at != index:
        raise ValueError("%s is on cuda:%d, expected cuda:%d" % (name, at, index))
    return at


def _rows(name, t):
    """(t as [rows, columns] with adjacent columns, distance of its rows in elements)."""
    if t.dim() != 2:
        if t.dim() < 1:
            raise ValueError("%s must have at least one dimension" % name)
        if t.is_contiguous():
            return t.view(t.shape[:-1].numel(), t.shape[-1]), t.shape[-1]
        try:
            t = t.view(t.shape[:-1].numel(), t.shape[-1])
        except RuntimeError:
            raise ValueError("the rows of %s must lie at one distance" % name) from None
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError("the columns of %s must be adjacent" % name)
    ld = t.stride(0) if rows > 1 else cols
    if ld < cols:
        raise ValueError("the rows of %s overlap" % name)
    return t, ld


def _check_weight(w, index):
    if type(w) is not Int8Weight:
        raise TypeError("weight must be an Int8Weight (quantize_weight, pack_weight)")
    packed, scale, K, N = w
    _check_cuda("weight.packed", packed, index)
    if packed.dtype is not torch.int8 or packed.numel() != -(-K // 64) * -(-N // 64) * 4096 or not packed.is_contiguous():
        raise ValueError("weight.packed must hold the packed [%d, %d] matrix as contiguous int8" % (K, N))
    _check_cuda("weight.scale", scale, index)
    if scale.dtype is not torch.float32 or scale.numel() != N or not scale.is_contiguous():
        raise ValueError("weight.scale must hold %d contiguous float32" % N)
    return packed.data_ptr(), scale.data_ptr(), K, N


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(M, N, K):
    return sh.lib().souffle_linear_int8_workspace_bytes(M, N, K)


def _epilogue(bias, act, n, dtype, index):
    if act not in _ACTS:
        raise ValueError("act must be None, 'relu', 'gelu' or 'gelu_tanh', got %r" % (act,))
    if bias is None:
        return None, _ACTS[act]
    _check_cuda("bias", bias, index)
    if bias.dtype != dtype or not bias.is_contiguous() or bias.numel() != n:
        raise ValueError("bias must be %d contiguous values of %s" % (n, dtype))
    return bias.data_ptr(), _ACTS[act]


def _output(out, like, rows, n, dtype, index):
    if out is None:
        return like.new_empty((rows, n), dtype=dtype), n
    _check_cuda("out", out, index)
    if out.dtype != dtype or tuple(out.shape) != (rows, n):
        raise ValueError("out must be [%d, %d] of %s" % (rows, n, dtype))
    return _rows("out", out)


def _overlap(a, rows_a, width_a, pitch_a, b, rows_b, width_b, pitch_b):
    """Whether two sets of rows have a byte in common (address, rows, bytes of a row, distance of the rows).  Sets that lie within
    each other count as apart only where their rows do as columns side by side in one buffer."""
    if not rows_a or not rows_b or a + (rows_a - 1) * pitch_a + width_a <= b or b + (rows_b - 1) * pitch_b + width_b <= a:
        return False
    if rows_a == 1:
        pitch_a = pitch_b
    elif rows_b == 1:
        pitch_b = pitch_a
    gap = (b - a) % pitch_a
    return pitch_a != pitch_b or gap < width_a or gap + width_b > pitch_a


def _check_apart(at, M, width, pitch, named, *others):
    """out (address, rows, bytes of a row, distance of the rows) has no byte in common with an input, as some are still read when
    it is written: `named`, rows like out's with a name in front, and the others (name, address or None, bytes)."""
    end = at + (M - 1) * pitch + width
    if named[1] < end and at < named[1] + (M - 1) * named[3] + named[2] and _overlap(named[1], M, named[2], named[3], at, M, width, pitch):
        raise ValueError("out must not overlap " + named[0])
    for name, address, nbytes in others:
        if address and address < end and at < address + nbytes and _overlap(address, 1, nbytes, nbytes, at, M, width, pitch):
            raise ValueError("out must not overlap " + name)


def pack_weight(weight_q, scale):
    """Int8Weight of an int8 matrix [K, N] and the float32 scale [N] of its columns."""
    index = _check_cuda("weight_q", weight_q)
    _check_cuda("scale", scale, index)
    if weight_q.dtype != torch.int8 or weight_q.dim() != 2:
        raise TypeError("weight_q must be an int8 matrix [K, N]")
    (w, ld), (K, N) = _rows("weight_q", weight_q), weight_q.shape
    if scale.dtype != torch.float32 or scale.dim() != 1 or scale.numel() != N:
        raise ValueError("scale must be [%d] float32" % N)
    with torch.cuda.device(index):
        packed = w.new_empty(sh.lib().souffle_int8_packed_bytes(K, N))
        sh.check(sh.lib().souffle_int8_pack_weight(w.data_ptr(), ld, packed.data_ptr(), K, N, _stream(index)))
    return Int8Weight(packed, scale.contiguous(), K, N)


def quantize_weight(weight):
    """Int8Weight of a matrix [K, N] in fp16, bf16 or fp32, quantised per output channel.  Once per model."""
    index = _check_cuda("weight", weight)
    if weight.dtype not in _DTYPES or weight.dim() != 2:
        raise TypeError("weight must be a float16, bfloat16 or float32 matrix [K, N]")
    (w, ld), (K, N) = _rows("weight", weight), weight.shape
    with torch.cuda.device(index):
        packed = w.new_empty(sh.lib().souffle_int8_packed_bytes(K, N), dtype=torch.int8)
        scale = w.new_empty(N, dtype=torch.float32)
        sh.check(sh.lib().souffle_int8_quantize_weight(w.data_ptr(), _DTYPES[w.dtype], ld, packed.data_ptr(), scale.data_ptr(), K, N,
                                                       _stream(index)))
    return Int8Weight(packed, scale, K, N)


def quantize_rows(x):
    """(q, row_scale) of x [..., K] (rows at one distance): q [rows, K] int8 in rows that lie K rounded
    up to 64 bytes apart, row_scale [rows] float32."""
    index = _check_cuda("x", x)
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float16, bfloat16 or float32")
    if index != _device():
        with torch.cuda.device(index):
            return quantize_rows(x)
    x, ld = _rows("x", x)
    M, K = x.shape
    ldq = -(-K // 64) * 64
    q = x.new_empty((M, ldq), dtype=torch.int8)
    scale = x.new_empty(M, dtype=torch.float32)
    sh.check(sh.lib().souffle_quantize_rows(x.data_ptr(), _DTYPES[x.dtype], ld, q.data_ptr(), ldq, scale.data_ptr(), M, K, _stream(index)))
    return (q if K == ldq else q[:, :K]), scale


def gemm_int8(q, row_scale, weight, *, bias=None, act=None, dtype=torch.float16, out=None):
    """act(row_scale * weight.scale * (q . W) + bias) as [rows, N] of `dtype`.  q [rows, K] int8: rows that start at
    multiples of 16 bytes and can be read up to K rounded up to 64 bytes (as quantize_rows and gated_norm_int8 make
    them; what lies behind K does not matter).  bias is of `dtype`; out: a [rows, N] tensor to write to, apart from all inputs."""
    index = _check_cuda("q", q)
    if index != _device():
        with torch.cuda.device(index):
            return gemm_int8(q, row_scale, weight, bias=bias, act=act, dtype=dtype, out=out)
    _check_cuda("row_scale", row_scale, index)
    packed, scale, K, N = _check_weight(weight, index)
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
    b, a = _epilogue(bias, act, N, dtype, index)
    given = out is not None
    out, ldy = _output(out, q, M, N, dtype, index)
    q_ptr, scale_ptr, out_ptr = q.data_ptr(), row_scale.data_ptr(), out.data_ptr()
    if given:
        size = dtype.itemsize
        _check_apart(out_ptr, M, N * size, ldy * size, ("q", q_ptr, K, ldq), ("row_scale", scale_ptr, 4 * M), ("bias", b, size * N),
                     ("weight.packed", packed, weight.packed.numel()), ("weight.scale", scale, 4 * N))
    sh.check(sh.lib().souffle_gemm_int8(q_ptr, ldq, scale_ptr, packed, scale, b, a, out_ptr, _DTYPES[dtype], ldy, M, N, K, _stream(index)))
    return out


def linear_int8(x, weight, *, bias=None, act=None, out=None):
    """act(x . W + bias) with the rows of x [..., K] in 8 bits: quantize_rows and gemm_int8 in one call, bit for bit.
    Returns [rows, N] of x's type; bias is of that type too.  out must not overlap an input."""
    index = _check_cuda("x", x)
    if index != _device():
        with torch.cuda.device(index):
            return linear_int8(x, weight, bias=bias, act=act, out=out)
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float16, bfloat16 or float32")
    packed, scale, K, N = _check_weight(weight, index)
    x, ld = _rows("x", x)
    M = x.shape[0]
    if x.shape[1] != K:
        raise ValueError("x must be [..., %d]" % K)
    b, a = _epilogue(bias, act, N, x.dtype, index)
    given = out is not None
    out, ldy = _output(out, x, M, N, x.dtype, index)
    x_ptr, out_ptr = x.data_ptr(), out.data_ptr()
    if given:
        size = x.dtype.itemsize
        _check_apart(out_ptr, M, N * size, ldy * size, ("x", x_ptr, K * size, ld * size), ("bias", b, size * N),
                     ("weight.packed", packed, weight.packed.numel()), ("weight.scale", scale, 4 * N))
    nbytes = _workspace_bytes(M, N, K)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    sh.check(sh.lib().souffle_linear_int8(x_ptr, ld, packed, scale, b, a, out_ptr, _DTYPES[x.dtype], ldy, M, N, K, sh.ptr(ws), nbytes, _stream(index)))
    return out
