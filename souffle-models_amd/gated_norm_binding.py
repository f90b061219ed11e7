"""gated_norm_binding: the norms on both sides of a transformer block with the block's gate and the residual scale in
between, forward and backward (a wrapper over the C ABI; the reference has no counterpart).

    y, h = gated_norm(x, f, gate=g, ...)            # y = residual_scale x + g N_post(f),  h = N_pre(y)
    y, q, s = gated_norm_int8(x, f, gate=g, ...)    # h as 8-bit rows for linear_int8_binding.gemm_int8
    grads = gated_norm_backward(dy, dh, x, f, gate=g, ...)

x is the residual stream and f the block's output, [..., D] in fp16, bf16 or fp32, rows at one distance (contiguous, or a slice such as
x[..., a:b] or x[:, -1:]); every vector has their type.  Keywords
of all three:
    post_norm, pre_norm     "layer", "rms"; post_norm also None
    post_gamma, post_beta, pre_gamma, pre_beta      [D] or None
    gate                    [D], or [G, D]: one row for each of G equal runs of rows (a sequence), or None
    residual_scale, post_eps, pre_eps               numbers
Statistics and sums are in fp32, h comes from y before y is rounded, and two calls give the same bits.  Work is queued on
the current stream of the tensors' device and nothing is kept between calls.  Where gradients are on and an input
requires one, autograd records gated_norm, and its backward pass is gated_norm_backward; that pass cannot be captured into a
graph through autograd (gated_norm_backward itself can).  gated_norm_int8 is not recorded.
"""
import ctypes as C
import functools

import torch

import souffle_hip as sh
from linear_int8_binding import _DTYPES, _check_cuda, _device, _rows, _stream

_NORMS = {None: sh.NORM_NONE, "layer": sh.NORM_LAYER, "rms": sh.NORM_RMS}


@functools.lru_cache(maxsize=256)
def _cfg(*fields):
    """The configuration struct of these sizes and numbers (building it takes as long as the call itself)."""
    return sh.GatedNormCfg(*fields)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(M, D, per_gate):
    """Of a gradient call; the kinds of the norms and the type do not matter."""
    return sh.lib().souffle_gated_norm_backward_workspace_bytes(_cfg(M, D, sh.F32, sh.NORM_RMS, sh.NORM_RMS, per_gate, 1.0, 0.0, 0.0, D, D, D, D))


def _on_device(position):
    """Runs a function with the device of its argument `x`, at that position, as the current one."""
    def decorate(fn):
        @functools.wraps(fn)
        def call(*args, **kw):
            x = args[position] if len(args) > position else kw.get("x")
            if not isinstance(x, torch.Tensor) or not x.is_cuda or x.get_device() == _device():
                return fn(*args, **kw)
            with torch.cuda.device(x.get_device()):
                return fn(*args, **kw)
        return call
    return decorate


def _vector(name, v, x, D, index):
    """Address of a vector [D] of x's type, or None."""
    if v is None:
        return None
    if not isinstance(v, torch.Tensor) or v.get_device() != index or v.dtype is not x.dtype or v.shape != (D,) or not v.is_contiguous():
        _check_cuda(name, v, index)
        raise ValueError("%s must be contiguous, of x's type and [%d]" % (name, D))
    return v.data_ptr()


def _gate(gate, x, M, D, index):
    """(address of a gate [D] or [G, D], rows that share one of its rows; 0: all)."""
    if gate is None or not isinstance(gate, torch.Tensor) or gate.dim() != 2:
        return _vector("gate", gate, x, D, index), 0
    G = gate.shape[0]
    if G < 1 or M % G:
        raise ValueError("a gate of %d rows does not divide %d rows" % (G, M))
    if gate.get_device() != index or gate.dtype is not x.dtype or gate.shape[1] != D or not gate.is_contiguous():
        _check_cuda("gate", gate, index)
        raise ValueError("gate must be contiguous, of x's type and [%d] or [G, %d]" % (D, D))
    return gate.data_ptr(), M // G


def _like(x):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps):
    """(x and f as rows, index of their device, cfg, vectors)."""
    index = _check_cuda("x", x)
    if not isinstance(f, torch.Tensor) or f.get_device() != index:
        _check_cuda("f", f, index)
    dtype = x.dtype
    if dtype not in _DTYPES or f.dtype != dtype:
        raise TypeError("x and f must both be float16, bfloat16 or float32")
    if x.shape != f.shape:
        raise ValueError("x and f must have one shape, got %s and %s" % (tuple(x.shape), tuple(f.shape)))
    if post_norm not in _NORMS or pre_norm not in ("layer", "rms"):
        raise ValueError("post_norm must be 'layer', 'rms' or None, pre_norm 'layer' or 'rms'")
    x, ldx = _rows("x", x)
    f, ldf = _rows("f", f)
    M, D = x.shape
    gate_ptr, per_gate = _gate(gate, x, M, D, index)
    if post_norm is None and (post_gamma is not None or post_beta is not None):
        raise ValueError("post_gamma and post_beta need a post_norm")
    w = sh.GatedNormW(_vector("post_gamma", post_gamma, x, D, index), _vector("post_beta", post_beta, x, D, index), gate_ptr,
                      _vector("pre_gamma", pre_gamma, x, D, index), _vector("pre_beta", pre_beta, x, D, index))
    cfg = _cfg(M, D, _DTYPES[dtype], _NORMS[post_norm], _NORMS[pre_norm], per_gate, float(residual_scale), float(post_eps), float(pre_eps), ldx, ldf, D, D)
    return x, f, index, cfg, w


class _Recorded(torch.autograd.Function):
    """gated_norm for autograd; `numbers` are the keywords that are no tensors."""

    @staticmethod
    def forward(ctx, want_y, numbers, x, f, gate, post_gamma, post_beta, pre_gamma, pre_beta):
        ctx.numbers = numbers
        ctx.set_materialize_grads(False)      # (None for an output that the loss does not use)
        ctx.save_for_backward(x, f, gate, post_gamma, post_beta, pre_gamma, pre_beta)
        return gated_norm(x, f, gate=gate, post_gamma=post_gamma, post_beta=post_beta, pre_gamma=pre_gamma, pre_beta=pre_beta, want_y=want_y, **numbers)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        # What autograd adds to a captured pass (the leaves' accumulation, on the streams of eager graphs that are still there) may end the process.
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("autograd's backward pass through gated_norm cannot be captured into a graph: capture gated_norm_backward")
        x, f, gate, post_gamma, post_beta, pre_gamma, pre_beta = ctx.saved_tensors
        dy, dh = (None if d is None else d.contiguous() for d in (dy, dh))      # (a sum's gradient is one element, expanded)
        g = gated_norm_backward(dy, dh, x, f, gate=gate, post_gamma=post_gamma, post_beta=post_beta, pre_gamma=pre_gamma, pre_beta=pre_beta, **ctx.numbers)
        return (None, None) + tuple(g[name] for name in ("x", "f", "gate", "post_gamma", "post_beta", "pre_gamma", "pre_beta"))


@_on_device(0)
def gated_norm(x, f, *, gate=None, residual_scale=1.0, post_norm="layer", post_gamma=None, post_beta=None, post_eps=1e-5,
               pre_norm="layer", pre_gamma=None, pre_beta=None, pre_eps=1e-5, want_y=True):
    """(y, h), of x's shape and type; y is None with want_y=False (a post-norm encoder only keeps h).  Differentiable."""
    xr, fr, index, cfg, w = _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps)
    if torch.is_grad_enabled():
        for v in (x, f, gate, post_gamma, post_beta, pre_gamma, pre_beta):
            if v is not None and v.requires_grad:
                numbers = dict(residual_scale=residual_scale, post_norm=post_norm, post_eps=post_eps, pre_norm=pre_norm, pre_eps=pre_eps)
                return _Recorded.apply(want_y, numbers, x, f, gate, post_gamma, post_beta, pre_gamma, pre_beta)
    y = _like(x) if want_y else None
    h = _like(x)
    sh.check(sh.lib().souffle_gated_norm_forward(cfg, w, xr.data_ptr(), fr.data_ptr(), sh.ptr(y), h.data_ptr(), _stream(index)))
    return y, h


@_on_device(0)
def gated_norm_int8(x, f, *, gate=None, residual_scale=1.0, post_norm="layer", post_gamma=None, post_beta=None, post_eps=1e-5,
                    pre_norm="layer", pre_gamma=None, pre_beta=None, pre_eps=1e-5, want_y=True):
    """(y, q, row_scale): h in 8 bits by the rule of linear_int8_binding.quantize_rows (without rounding h to x's type
    first), q [rows, D] int8 in rows D rounded up to 64 bytes apart, row_scale [rows] float32."""
    xr, fr, index, cfg, w = _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps)
    M, D = xr.shape
    ldq = -(-D // 64) * 64
    y = _like(x) if want_y else None
    q = x.new_empty((M, ldq), dtype=torch.int8)
    scale = x.new_empty(M, dtype=torch.float32)
    sh.check(sh.lib().souffle_gated_norm_forward_int8(cfg, w, xr.data_ptr(), fr.data_ptr(), sh.ptr(y), q.data_ptr(), ldq, scale.data_ptr(),
                                                      _stream(index)))
    return y, (q if D == ldq else q[:, :D]), scale


@_on_device(2)
def gated_norm_backward(dy, dh, x, f, *, gate=None, residual_scale=1.0, post_norm="layer", post_gamma=None, post_beta=None,
                        post_eps=1e-5, pre_norm="layer", pre_gamma=None, pre_beta=None, pre_eps=1e-5):
    """The gradients for incoming dy and dh (one of them may be None: zero) as a dict: "x", "f", and "gate", "post_gamma",
    "post_beta", "pre_gamma", "pre_beta" for the vectors that were given (None for the others), each of its input's shape
    and type.  x and f are the forward call's inputs; nothing else of it is needed."""
    xr, fr, index, cfg, w = _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps)
    if dy is None and dh is None:
        raise ValueError("one of dy and dh must be given")
    M, D = xr.shape
    incoming = []
    for name, d in (("dy", dy), ("dh", dh)):
        if d is None:
            incoming.append((None, D))
            continue
        _check_cuda(name, d, index)
        if d.dtype != x.dtype or d.shape != x.shape:
            raise ValueError("%s must have x's shape and type" % name)
        d, ld = _rows(name, d)
        incoming.append((d.data_ptr(), ld))
    vector_gate = gate if gate is not None and gate.dim() == 1 else None
    given = [n for n, v in (("gate", vector_gate), ("post_gamma", post_gamma), ("post_beta", post_beta), ("pre_gamma", pre_gamma), ("pre_beta", pre_beta))
             if v is not None]
    vectors = x.new_empty((len(given), D)) if M else x.new_zeros((len(given), D))      # (one allocation: each takes as long as a check of all)
    g = {"x": _like(x), "f": _like(x), "gate": None, "post_gamma": None, "post_beta": None, "pre_gamma": None, "pre_beta": None}
    g.update(zip(given, vectors.unbind(0)))
    if gate is not vector_gate:
        g["gate"] = gate.new_empty(gate.shape) if M else gate.new_zeros(gate.shape)
    if M == 0:
        return g
    (dy_ptr, ld_dy), (dh_ptr, ld_dh) = incoming
    grad = sh.GatedNormGrad(g["x"].data_ptr(), g["f"].data_ptr(), sh.ptr(g["pre_gamma"]), sh.ptr(g["pre_beta"]), sh.ptr(g["gate"]),
                            sh.ptr(g["post_gamma"]), sh.ptr(g["post_beta"]), ld_dy, ld_dh, D, D)
    nbytes = _workspace_bytes(M, D, cfg.rows_per_gate)
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    sh.check(sh.lib().souffle_gated_norm_backward(cfg, w, dy_ptr, dh_ptr, xr.data_ptr(), fr.data_ptr(), grad, ws.data_ptr(), nbytes, _stream(index)))
    return g
