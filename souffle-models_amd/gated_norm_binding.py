"""gated_norm_binding: the norms on both sides of a transformer block with the block's gate and the residual scale in
between, forward and backward (a wrapper over the C ABI; the reference has no counterpart).

    y, h = gated_norm(x, f, gate=g, ...)            # y = residual_scale x + g N_post(f),  h = N_pre(y)
    y, q, s = gated_norm_int8(x, f, gate=g, ...)    # h as 8-bit rows for linear_int8_binding.gemm_int8
    grads = gated_norm_backward(dy, dh, x, f, gate=g, ...)

x is the residual stream and f the block's output, [..., D] in fp16, bf16 or fp32; every vector has their type.  Keywords
of all three:
    post_norm, pre_norm     "layer", "rms"; post_norm also None
    post_gamma, post_beta, pre_gamma, pre_beta      [D] or None
    gate                    [D], or [G, D]: one row for each of G equal runs of rows (a sequence), or None
    residual_scale, post_eps, pre_eps               numbers
Statistics and sums are in fp32, h comes from y before y is rounded, and two calls give the same bits.  Work is queued on
the current stream of the tensors' device and nothing is kept between calls.
"""
import ctypes as C

import torch

import souffle_hip as sh
from linear_int8_binding import _DTYPES, _check_cuda, _rows

_NORMS = {None: sh.NORM_NONE, "layer": sh.NORM_LAYER, "rms": sh.NORM_RMS}


def _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps):
    """(x and f as rows, cfg, vectors)."""
    _check_cuda("x", x)
    _check_cuda("f", f, x.device)
    if x.dtype not in _DTYPES or f.dtype != x.dtype:
        raise TypeError("x and f must both be float16, bfloat16 or float32")
    if x.shape != f.shape:
        raise ValueError("x and f must have one shape, got %s and %s" % (tuple(x.shape), tuple(f.shape)))
    if post_norm not in _NORMS or pre_norm not in ("layer", "rms"):
        raise ValueError("post_norm must be 'layer', 'rms' or None, pre_norm 'layer' or 'rms'")
    x, ldx = _rows("x", x)
    f, ldf = _rows("f", f)
    M, D = x.shape
    per_gate = 0
    if gate is not None:
        _check_vector("gate", gate, x, gate.shape if gate.dim() == 2 else (D,), D)
        if gate.dim() == 2:
            if gate.shape[0] < 1 or M % gate.shape[0]:
                raise ValueError("a gate of %d rows does not divide %d rows" % (gate.shape[0], M))
            per_gate = M // gate.shape[0]
    for name, v in (("post_gamma", post_gamma), ("post_beta", post_beta), ("pre_gamma", pre_gamma), ("pre_beta", pre_beta)):
        if v is not None:
            _check_vector(name, v, x, (D,), D)
    if post_norm is None and (post_gamma is not None or post_beta is not None):
        raise ValueError("post_gamma and post_beta need a post_norm")
    cfg = sh.GatedNormCfg(M, D, _DTYPES[x.dtype], _NORMS[post_norm], _NORMS[pre_norm], per_gate, residual_scale, post_eps, pre_eps, ldx, ldf, D, D)
    return x, f, cfg, sh.GatedNormW(sh.ptr(post_gamma), sh.ptr(post_beta), sh.ptr(gate), sh.ptr(pre_gamma), sh.ptr(pre_beta))


def _check_vector(name, v, x, shape, D):
    _check_cuda(name, v, x.device)
    if v.dtype != x.dtype or not v.is_contiguous() or tuple(v.shape) != tuple(shape) or v.shape[-1] != D:
        raise ValueError("%s must be contiguous, of x's type and %s" % (name, "[%d] or [G, %d]" % (D, D) if name == "gate" else "[%d]" % D))


def gated_norm(x, f, *, gate=None, residual_scale=1.0, post_norm="layer", post_gamma=None, post_beta=None, post_eps=1e-5,
               pre_norm="layer", pre_gamma=None, pre_beta=None, pre_eps=1e-5, want_y=True):
    """(y, h), of x's shape and type; y is None with want_y=False (a post-norm encoder only keeps h)."""
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x, f, cfg, w = _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps)
    with torch.cuda.device(x.device):
        y = torch.empty(shape, dtype=x.dtype, device=x.device) if want_y else None
        h = torch.empty(shape, dtype=x.dtype, device=x.device)
        sh.check(sh.lib().souffle_gated_norm_forward(C.byref(cfg), C.byref(w), x.data_ptr(), f.data_ptr(), sh.ptr(y), h.data_ptr(),
                                                     sh.current_stream()))
    return y, h


def gated_norm_int8(x, f, *, gate=None, residual_scale=1.0, post_norm="layer", post_gamma=None, post_beta=None, post_eps=1e-5,
                    pre_norm="layer", pre_gamma=None, pre_beta=None, pre_eps=1e-5, want_y=True):
    """(y, q, row_scale): h in 8 bits by the rule of linear_int8_binding.quantize_rows (without rounding h to x's type
    first), q [rows, D] int8 in rows D rounded up to 64 bytes apart, row_scale [rows] float32."""
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x, f, cfg, w = _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps)
    M, D = x.shape
    ldq = -(-D // 64) * 64
    with torch.cuda.device(x.device):
        y = torch.empty(shape, dtype=x.dtype, device=x.device) if want_y else None
        q = torch.empty((M, ldq), dtype=torch.int8, device=x.device)
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
        sh.check(sh.lib().souffle_gated_norm_forward_int8(C.byref(cfg), C.byref(w), x.data_ptr(), f.data_ptr(), sh.ptr(y), q.data_ptr(), ldq,
                                                          scale.data_ptr(), sh.current_stream()))
    return y, q[:, :D], scale


def gated_norm_backward(dy, dh, x, f, *, gate=None, residual_scale=1.0, post_norm="layer", post_gamma=None, post_beta=None,
                        post_eps=1e-5, pre_norm="layer", pre_gamma=None, pre_beta=None, pre_eps=1e-5):
    """The gradients for incoming dy and dh (one of them may be None: zero) as a dict: "x", "f", and "gate", "post_gamma",
    "post_beta", "pre_gamma", "pre_beta" for the vectors that were given (None for the others), each of its input's shape
    and type.  x and f are the forward call's inputs; nothing else of it is needed."""
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x, f, cfg, w = _setup(x, f, gate, residual_scale, post_norm, post_gamma, post_beta, post_eps, pre_norm, pre_gamma, pre_beta, pre_eps)
    if dy is None and dh is None:
        raise ValueError("one of dy and dh must be given")
    rows = {}
    for name, d in (("dy", dy), ("dh", dh)):
        if d is not None:
            _check_cuda(name, d, x.device)
            if d.dtype != x.dtype or d.shape != shape:
                raise ValueError("%s must have x's shape and type" % name)
            rows[name] = _rows(name, d)
    M, D = x.shape
    with torch.cuda.device(x.device):
        g = {"x": torch.empty(shape, dtype=x.dtype, device=x.device), "f": torch.empty(shape, dtype=x.dtype, device=x.device)}
        for name, v in (("gate", gate), ("post_gamma", post_gamma), ("post_beta", post_beta), ("pre_gamma", pre_gamma), ("pre_beta", pre_beta)):
            g[name] = None if v is None else torch.empty_like(v) if M else torch.zeros_like(v)
        if M == 0:
            return g
        grad = sh.GatedNormGrad(g["x"].data_ptr(), g["f"].data_ptr(), sh.ptr(g["pre_gamma"]), sh.ptr(g["pre_beta"]), sh.ptr(g["gate"]),
                                sh.ptr(g["post_gamma"]), sh.ptr(g["post_beta"]), rows["dy"][1] if dy is not None else D,
                                rows["dh"][1] if dh is not None else D, D, D)
        nbytes = sh.lib().souffle_gated_norm_backward_workspace_bytes(C.byref(cfg))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        sh.check(sh.lib().souffle_gated_norm_backward(C.byref(cfg), C.byref(w), rows["dy"][0].data_ptr() if dy is not None else None,
                                                      rows["dh"][0].data_ptr() if dh is not None else None, x.data_ptr(), f.data_ptr(),
                                                      C.byref(grad), ws.data_ptr(), nbytes, sh.current_stream()))
    return g
