"""The gated norm and the 8-bit linear layer in 64 bits on the CPU, and bounds on what fp32 arithmetic may add.

Bounds count roundings.  EPS32 = 2^-24 is half a step of fp32 relative to the value; a sum over a row passes through at
most 16 additions in a thread, 6 across a wave and 16 across the waves, the products and the final scaling add a few:
C = 64 roundings per row statistic.  Sums over rows have up to one rounding per row of a chunk and 64 behind it.  The result is rounded once to its
type: half a step."""
import torch

EPS32 = 2.0 ** -24
C = 64 * EPS32
ACTS = {None: lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
        "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}


def half_step(ref, dtype):
    """Half a step of `dtype` at the values of ref (with the smallest subnormal's half below its normal range)."""
    f = torch.finfo(dtype)
    return ref.abs() * (f.eps / 2) * (1 + f.eps) + f.tiny * f.eps / 2


def check(name, got, ref, tol):
    got, ref = got.detach().double().cpu(), ref.double()
    assert got.shape == ref.shape, "%s: shape %s, expected %s" % (name, tuple(got.shape), tuple(ref.shape))
    assert torch.isfinite(got).all(), "%s: non-finite values" % name
    over = (got - ref).abs() - tol
    worst = int(over.reshape(-1).argmax()) if over.numel() else 0
    assert over.numel() == 0 or over.max() <= 0, "%s: off by %.4g where %.4g is allowed (at %d, value %.6g)" % (
        name, (got - ref).abs().reshape(-1)[worst], tol.reshape(-1)[worst], worst, ref.reshape(-1)[worst])


# ------------------------------------------------------------------------------------------------- rows ----
def quantize(x):
    """(q, scale) in 64 bits of the definition; the scale is a 32-bit number."""
    x = x.double()
    scale = (x.abs().amax(-1) / 127).float().double().clamp_min(2.0 ** -100)
    return torch.round(x / scale[:, None]), scale


def linear(q, row_scale, wq, col_scale, bias, act):
    """(y, bound without the final rounding): exact sums; conversion, two scalings and the bias are 4 roundings, and the
    activations (slope at most 1.13, own error a few roundings of their argument) stay within 16 in all."""
    p = (q.double() @ wq.double()) * col_scale.double() * row_scale.double()[:, None]
    v = p if bias is None else p + bias.double()
    return ACTS[act](v), 16 * EPS32 * (p.abs() + v.abs())


# ------------------------------------------------------------------------------------------------- norms ----
def norm(v, kind, eps, gamma, beta):
    if kind is None:
        return v, v, torch.ones_like(v[:, :1])
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    hat = c * r
    out = hat if gamma is None else hat * gamma
    return out if beta is None else out + beta, hat, r


def gate_rows(gate, rows):
    return gate if gate is None or gate.dim() == 1 else gate.repeat_interleave(rows // gate.shape[0], 0)


def wide(p):
    return {k: v.detach().double().cpu() if isinstance(v, torch.Tensor) else v for k, v in p.items()}


def forward(x, f, p):
    """(y, h, bound of y, bound of h) without the final roundings."""
    p = {"residual_scale": 1.0, "post_norm": "layer", "pre_norm": "layer", "post_eps": 1e-5, "pre_eps": 1e-5, **wide(p)}
    x, f = x.double().cpu(), f.double().cpu()
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    post, fhat, fr = norm(f, p["post_norm"], p["post_eps"], p.get("post_gamma"), p.get("post_beta"))
    g = gate_rows(p.get("gate"), x.shape[0])
    g = torch.ones_like(x[:1]) if g is None else g
    y = p["residual_scale"] * x + g * post
    h, yhat, yr = norm(y, p["pre_norm"], p["pre_eps"], p.get("pre_gamma"), p.get("pre_beta"))
    one = lambda v: 1.0 if v is None else v.abs()  # noqa: E731
    zero = lambda v: 0.0 if v is None else v.abs()  # noqa: E731
    e_post = C * ((fhat.abs() + fr * mean(f.abs())) * one(p.get("post_gamma")) + zero(p.get("post_beta")))
    e_y = g.abs() * e_post + C * (y.abs() + (p["residual_scale"] * x).abs())
    e_h = one(p.get("pre_gamma")) * (yr * (e_y + mean(e_y) + C * mean(y.abs())) + yhat.abs() * (C + yr * mean(e_y * yhat.abs()))) + C * h.abs()
    return y, h, e_y, e_h


def backward(dy, dh, x, f, p):
    """({name: gradient}, {name: bound}) by the formulas."""
    p = {"residual_scale": 1.0, "post_norm": "layer", "pre_norm": "layer", "post_eps": 1e-5, "pre_eps": 1e-5, **wide(p)}
    x, f = x.double().cpu(), f.double().cpu()
    dy = torch.zeros_like(x) if dy is None else dy.double().cpu()
    dh = torch.zeros_like(x) if dh is None else dh.double().cpu()
    rows, cols = x.shape
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    post, fhat, fr = norm(f, p["post_norm"], p["post_eps"], p.get("post_gamma"), p.get("post_beta"))
    gate = p.get("gate")
    g = gate_rows(gate, rows)
    g = torch.ones_like(x[:1]) if g is None else g
    y = p["residual_scale"] * x + g * post
    _, yhat, yr = norm(y, p["pre_norm"], p["pre_eps"], None, None)
    _, _, e_y, _ = forward(x, f, p)
    e_yhat = yr * (e_y + mean(e_y) + C * mean(y.abs())) + yhat.abs() * (C + yr * mean(e_y * yhat.abs()))
    e_fhat = C * (fhat.abs() + fr * mean(f.abs()))

    def through(d, e_d, hat, e_hat, r, kind):      # (gradient of the norm's input, bound)
        if kind is None:
            return d, e_d
        layer = kind == "layer"
        m = mean(d * hat)
        out = r * (d - hat * m - (mean(d) if layer else 0))
        a = d.abs() + mean(d.abs()) + hat.abs() * mean((d * hat).abs())
        e = e_d + mean(e_d) + hat.abs() * mean(e_d * hat.abs() + d.abs() * e_hat) + e_hat * m.abs()
        return out, r * (4 * C * a + e) + out.abs() * mean(e_hat)

    grads, bounds = {}, {}
    over_rows = lambda name, v, e: (grads.__setitem__(name, v.sum(0)), bounds.__setitem__(name, (e + (rows + 64) * EPS32 * v.abs()).sum(0)))  # noqa: E731
    over_rows("pre_gamma", dh * yhat, dh.abs() * e_yhat)
    over_rows("pre_beta", dh, 0 * dh)
    dhat = dh if p.get("pre_gamma") is None else dh * p["pre_gamma"]
    dn, e_dn = through(dhat, EPS32 * dhat.abs(), yhat, e_yhat, yr, p["pre_norm"])
    d, e_d = dy + dn, e_dn + 2 * EPS32 * (dy.abs() + dn.abs())
    grads["x"], bounds["x"] = p["residual_scale"] * d, abs(p["residual_scale"]) * (e_d + EPS32 * d.abs())
    one = lambda v: 1.0 if v is None else v.abs()  # noqa: E731
    if gate is not None:
        dg = d * post
        e_dg = e_d * post.abs() + d.abs() * (e_fhat * one(p.get("post_gamma")) + 4 * EPS32 * post.abs())
        if gate.dim() == 1:
            over_rows("gate", dg, e_dg)
        else:
            by = lambda v: v.view(gate.shape[0], -1, cols).sum(1)  # noqa: E731
            grads["gate"], bounds["gate"] = by(dg), by(e_dg + (rows + 64) * EPS32 * dg.abs())
    dp, e_dp = d * g, e_d * g.abs() + EPS32 * (d * g).abs()
    over_rows("post_gamma", dp * fhat, e_dp * fhat.abs() + dp.abs() * e_fhat)
    over_rows("post_beta", dp, e_dp)
    df = dp if p.get("post_gamma") is None else dp * p["post_gamma"]
    grads["f"], bounds["f"] = through(df, e_dp * one(p.get("post_gamma")) + EPS32 * df.abs(), fhat, e_fhat, fr, p["post_norm"])
    return grads, bounds
