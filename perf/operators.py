"""The 8-bit linear layer and the gated double norm, as cases that can be timed and compared.

Two families that a transformer block uses next to each other:

* linear       y = act(dequantised(int8(x) . Wq) + bias): x is quantised row by row while it is taken in, Wq holds
               8-bit integers with one scale per output channel;
* norm         y = a x + g * N_post(f), h = N_pre(y): the norm behind a block, its gate and residual scale, and the norm in
               front of the next block;
* norm_grad    the gradients of that operator;
* norm_linear  the same norm with h handed over as 8-bit rows, and the linear layer that reads them.

run() computes either the plain torch form or, where `own` is set, makes the framework's calls.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SMALLEST_SCALE = 2.0 ** -100          # of a quantised row: keeps its reciprocal finite
LARGEST = {"linear": 2.0 * 8192 * 4096 * 4096, "norm": 16384 * 4096, "norm_grad": 8192 * 4096, "norm_linear": 2.0 * 3136 * 1024 * 4096}


# ------------------------------------------------------------------------------------------------- cases ----
def _linear(name, rows, k, n, dtype, act=None, bias=True, extra=0):
    """extra: columns that x's rows have beyond k, where x is a slice of a wider activation."""
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "extra": extra}


def _norm(name, kind, sequences, tokens, d, dtype, post, pre, gate, a=1.0, n=0, act=None):
    """gate: "channel" (one vector for all rows), "sequence" (one vector for each sequence) or None.  n: columns of
    the linear layer behind a norm_linear."""
    return {"name": name, "kind": kind, "sequences": sequences, "tokens": tokens, "d": d, "dtype": dtype, "post": post, "pre": pre,
            "gate": gate, "a": a, "n": n, "act": act}


def listed():
    return [
        # the QKV projection of a 768-wide encoder for a single token: latency
        _linear("linear one token", 1, 768, 2304, "f16"),
        # 24 sequences that each produce one token: the weights are the traffic
        _linear("linear decode", 24, 4096, 8192, "bf16", bias=False),
        # one sequence of 384 tokens through a 768-wide output projection
        _linear("linear one sequence", 384, 768, 768, "f16"),
        # sizes that fit no tile, rows cut out of a wider activation, full precision around the 8-bit product
        _linear("linear ragged", 333, 1000, 1111, "f32", "gelu", True, 7),
        # a large batch: bound by the matrix cores
        _linear("linear large batch", 8192, 4096, 4096, "bf16"),
        # between two blocks of a 768-wide encoder, one token
        _norm("norm one token", "norm", 1, 1, 768, "f16", "layer", "layer", "channel"),
        # the same for 32 sequences of 128 tokens
        _norm("norm batch", "norm", 32, 128, 768, "f16", "layer", "layer", "channel"),
        # long sequences, wide rows, a gate that each sequence brings: bound by memory
        _norm("norm long", "norm", 4, 4096, 4096, "bf16", "rms", "rms", "sequence", 0.5),
        # fine tuning on 197 image tokens with an odd width in full precision
        _norm("norm gradient ragged", "norm_grad", 6, 197, 1001, "f32", "layer", "layer", "sequence"),
        # a training step's rows: bound by memory
        _norm("norm gradient large", "norm_grad", 4, 2048, 4096, "bf16", "rms", "rms", "channel", 0.7),
        # the way into a 1024-wide block's MLP, one token
        _norm("norm and linear one token", "norm_linear", 1, 1, 1024, "f16", "layer", "layer", "channel", 1.0, 4096, "gelu_tanh"),
        # the same for 64 images of 49 tokens
        _norm("norm and linear batch", "norm_linear", 64, 49, 1024, "f16", "layer", "layer", "channel", 1.0, 4096, "gelu_tanh"),
    ]


def _spread(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi; half of them multiples of 64 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v > 64 and rng.random() < 0.5:
        v -= v % 64
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "norm_grad", "norm_linear"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    act = rng.choice([None, "gelu", "gelu_tanh", "relu"])
    if kind == "linear":
        k, n = _spread(rng, 32, 8192), _spread(rng, 32, 8192)
        rows = _spread(rng, 1, min(8192, int(LARGEST[kind] / (2.0 * k * n))))
        case = _linear("", rows, k, n, dtype, act, rng.random() < 0.7, rng.choice([0, 0, 7, 64]))
    else:
        d = _spread(rng, 32, 8192)
        n = _spread(rng, 32, 4096) if kind == "norm_linear" else 0
        if kind == "norm_linear":      # (8-bit rows of full-precision activations are the linear layer's own business)
            dtype = rng.choice(["f16", "bf16"])
        most = int(LARGEST[kind] / (2.0 * d * n if n else d))
        sequences = _spread(rng, 1, min(64, most))
        tokens = _spread(rng, 1, max(1, min(4096, most // sequences)))
        case = _norm("", kind, sequences, tokens, d, dtype, rng.choice(["layer", "rms", None]), rng.choice(["layer", "rms"]),
                     rng.choice([None, "channel", "sequence"]), rng.choice([1.0, 0.5]), n, act if n else None)
    del case["name"]
    return case


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": size * m * (k + n) + k * n + 4 * n + (size * n if case["bias"] else 0), "flops": 2.0 * m * k * n + 4.0 * m * k}
    m, d, n = case["sequences"] * case["tokens"], case["d"], case["n"]
    vectors = _vectors(case) * d + (d * case["sequences"] if case["gate"] == "sequence" else 0)
    if case["kind"] == "norm":
        return {"bytes": size * (4 * m * d + vectors), "flops": 20.0 * m * d}
    if case["kind"] == "norm_grad":    # reads x, f and the two incoming gradients, writes two
        return {"bytes": size * (6 * m * d + 2 * vectors), "flops": 50.0 * m * d}
    return {"bytes": size * (3 * m * d + vectors + m * n + n) + d * n + 4 * n, "flops": 2.0 * m * d * n + 24.0 * m * d}


def _vectors(case):
    """How many vectors of d values the norms and a channel gate have."""
    return {"layer": 2, "rms": 1, None: 0}[case["post"]] + {"layer": 2, "rms": 1}[case["pre"]] + (case["gate"] == "channel")


# ------------------------------------------------------------------------------------------------ inputs ----
def _activation(g, rows, cols, std=1.0):
    """Normal values with a few channels that stand out, as in a residual stream."""
    x = torch.randn(rows, cols, generator=g, device="cuda") * std
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return x * torch.where(loud, 6.0, 1.0)


def packed_weight(wq):
    """Wq [K][N] in the order that the framework's product reads it (zeros up to multiples of 64): per 64 columns and
    64 of K four KB, one for each of the four matrix-core operands t; lane 16 c + 4 g + v of an operand holds the 16
    values k = 16 c .. 16 c + 15 of column 16 g + 4 t + v."""
    k, n = wq.shape
    kb, nb = -(-k // 64), -(-n // 64)
    w = torch.zeros(kb * 64, nb * 64, dtype=torch.int8, device=wq.device)
    w[:k, :n] = wq
    return w.view(kb, 4, 16, nb, 4, 4, 4).permute(3, 0, 5, 1, 4, 6, 2).contiguous().view(-1)   # [N/64][K/64][t][c][g][v][16]


def _weight(g, k, n):
    """(Wq [K][N], packed, scale [N]): a normal weight matrix, quantised per output channel when the model was loaded."""
    w = torch.randn(k, n, generator=g, device="cuda") / math.sqrt(k)
    scale = w.abs().amax(0) / 127
    wq = (w / scale).round().clamp(-127, 127).to(torch.int8)
    return wq, packed_weight(wq), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "linear":
        wide = _activation(g, case["rows"], case["k"] + case["extra"]).to(t)
        state["x"] = wide[:, :case["k"]]
        state["wq"], state["packed"], state["scale"] = _weight(g, case["k"], case["n"])
        state["bias"] = (0.1 * torch.randn(case["n"], generator=g, device="cuda")).to(t) if case["bias"] else None
        return state
    m, d = case["sequences"] * case["tokens"], case["d"]
    vector = lambda mean, std, *shape: (mean + std * torch.randn(*shape, generator=g, device="cuda")).to(t)  # noqa: E731
    state["x"], state["f"] = _activation(g, m, d, 2.0).to(t), _activation(g, m, d).to(t)
    p = {"residual_scale": case["a"], "post_norm": case["post"], "pre_norm": case["pre"]}
    if case["post"]:
        p["post_gamma"] = vector(1.0, 0.1, d)
    if case["post"] == "layer":
        p["post_beta"] = vector(0.0, 0.1, d)
    p["pre_gamma"] = vector(1.0, 0.1, d)
    if case["pre"] == "layer":
        p["pre_beta"] = vector(0.0, 0.1, d)
    if case["gate"]:
        p["gate"] = vector(0.5, 0.2, *((d,) if case["gate"] == "channel" else (case["sequences"], d)))
    state["p"] = p
    if case["kind"] == "norm_grad":
        state["dy"], state["dh"] = vector(0.0, 0.1, m, d), vector(0.0, 0.1, m, d)
    if case["kind"] == "norm_linear":
        state["wq"], state["packed"], state["scale"] = _weight(g, d, case["n"])
        state["bias"] = vector(0.0, 0.1, case["n"])
    return state


# -------------------------------------------------------------------------------------------- plain forms ----
def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.7071067811865476))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    return v


def _quantized(h):
    """h (32 bits) as whole numbers -127..127 and one scale per row.  The scale is a 32-bit number, the quotient is
    taken in 64 bits: halves are common (any value that is half its row's largest one)."""
    scale = (h.abs().amax(-1, keepdim=True).double() / 127).float().clamp_min(SMALLEST_SCALE)
    return (h.double() / scale.double()).round().float(), scale


def _plain_linear(q, row_scale, wq, scale, bias, act, t):
    v = (q @ wq.float()) * row_scale * scale
    if bias is not None:
        v = v + bias.float()
    return _act(v, act).to(t)


def _normalized(v, kind, eps=1e-5):
    """(normalised rows, 1 / their deviation) of v."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    return v * r, r


def _affine(v, gamma, beta):
    v = v if gamma is None else v * gamma.float()
    return v if beta is None else v + beta.float()


def _gate_rows(gate, rows):
    """The gate as [rows][d] or [d], in 32 bits."""
    if gate is None:
        return None
    return gate.float() if gate.dim() == 1 else gate.float().repeat_interleave(rows // gate.shape[0], 0)


def _plain_norm(x, f, p):
    f = f.float()
    post = _affine(_normalized(f, p["post_norm"])[0], p.get("post_gamma"), p.get("post_beta")) if p["post_norm"] else f
    gate = _gate_rows(p.get("gate"), x.shape[0])
    y = p["residual_scale"] * x.float() + (post if gate is None else gate * post)
    return y, _affine(_normalized(y, p["pre_norm"])[0], p.get("pre_gamma"), p.get("pre_beta"))


def _norm_grad(d, hat, r, kind):
    """The gradient of a norm's input from that of its normalised rows."""
    g = d - hat * (d * hat).mean(-1, keepdim=True)
    return r * (g - d.mean(-1, keepdim=True) if kind == "layer" else g)


def _plain_norm_grad(dy, dh, x, f, p):
    t, rows = x.dtype, x.shape[0]
    dy, dh, x, f = dy.float(), dh.float(), x.float(), f.float()
    fhat, fr = _normalized(f, p["post_norm"]) if p["post_norm"] else (f, None)
    post = _affine(fhat, p.get("post_gamma"), p.get("post_beta"))
    gate = _gate_rows(p.get("gate"), rows)
    yhat, yr = _normalized(p["residual_scale"] * x + (post if gate is None else gate * post), p["pre_norm"])
    out = {"pre_gamma": (dh * yhat).sum(0)}
    if "pre_beta" in p:
        out["pre_beta"] = dh.sum(0)
    dy = dy + _norm_grad(_affine(dh, p["pre_gamma"], None), yhat, yr, p["pre_norm"])
    out["x"] = p["residual_scale"] * dy
    if gate is not None:
        dg = dy * post
        out["gate"] = dg.sum(0) if p["gate"].dim() == 1 else dg.view(p["gate"].shape[0], -1, dg.shape[1]).sum(1)
        dy = dy * gate
    if p["post_norm"]:
        out["post_gamma"] = (dy * fhat).sum(0)
        if "post_beta" in p:
            out["post_beta"] = dy.sum(0)
        dy = _norm_grad(_affine(dy, p["post_gamma"], None), fhat, fr, p["post_norm"])
    out["f"] = dy
    return {name: v.to(t) for name, v in out.items()}


def run(state):
    case = state["case"]
    return _run_own(case, state) if own else _run_plain(case, state)


def _run_plain(case, s):
    t = s["x"].dtype
    if case["kind"] == "linear":
        q, row_scale = _quantized(s["x"].float())
        return _plain_linear(q, row_scale, s["wq"], s["scale"], s["bias"], case["act"], t)
    if case["kind"] == "norm_grad":
        return _plain_norm_grad(s["dy"], s["dh"], s["x"], s["f"], s["p"])
    y, h = _plain_norm(s["x"], s["f"], s["p"])
    if case["kind"] == "norm":
        return {"y": y.to(t), "h": h.to(t)}
    q, row_scale = _quantized(h)
    return {"y": y.to(t), "out": _plain_linear(q, row_scale, s["wq"], s["scale"], s["bias"], case["act"], t)}


# --------------------------------------------------------------------------------- the framework's calls ----
_bindings = None


def _framework():
    global _bindings
    if _bindings is None:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "souffle-models_amd")
        if here not in sys.path:
            sys.path.insert(0, here)
        import gated_norm_binding
        import linear_int8_binding
        _bindings = linear_int8_binding, gated_norm_binding
    return _bindings


def _run_own(case, s):
    linear, norm = _framework()
    if case["kind"] == "linear":
        weight = linear.Int8Weight(s["packed"], s["scale"], case["k"], case["n"])
        return linear.linear_int8(s["x"], weight, bias=s["bias"], act=case["act"])
    if case["kind"] == "norm":
        y, h = norm.gated_norm(s["x"], s["f"], **s["p"])
        return {"y": y, "h": h}
    if case["kind"] == "norm_grad":
        g = norm.gated_norm_backward(s["dy"], s["dh"], s["x"], s["f"], **s["p"])
        return {name: v for name, v in g.items() if v is not None}
    y, q, row_scale = norm.gated_norm_int8(s["x"], s["f"], **s["p"])
    weight = linear.Int8Weight(s["packed"], s["scale"], case["d"], case["n"])
    return {"y": y, "out": linear.gemm_int8(q, row_scale, weight, bias=s["bias"], act=case["act"], dtype=s["x"].dtype)}


# --------------------------------------------------------------------------------- the definitions, 64 bits ----
def _exact_linear(h, s, act):
    scale = torch.clamp((h.abs().amax(1) / 127).to(torch.float32).to(torch.float64), min=SMALLEST_SCALE)
    q = torch.round(h / scale[:, None])
    v = torch.matmul(q, s["wq"].to(torch.float64)) * torch.outer(scale, s["scale"].to(torch.float64))
    v = v if s["bias"] is None else v + s["bias"].to(torch.float64)
    return {None: lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
            "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[act](v)


def _exact_norm(x, f, p):
    def norm(v, kind, gamma, beta):
        if kind == "layer":
            return torch.nn.functional.layer_norm(v, v.shape[-1:], gamma, beta, 1e-5)
        return v / torch.sqrt(torch.mean(v * v, -1, True) + 1e-5) * gamma
    post = norm(f, p["post_norm"], p["post_gamma"], p.get("post_beta")) if p["post_norm"] else f
    if p.get("gate") is not None:
        sequences = p["gate"].shape[0] if p["gate"].dim() == 2 else 1
        post = (post.view(sequences, -1, post.shape[-1]) * p["gate"].view(sequences, 1, -1)).view(post.shape)
    y = p["residual_scale"] * x + post
    return y, norm(y, p["pre_norm"], p["pre_gamma"], p.get("pre_beta"))


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda v: v.double() if isinstance(v, torch.Tensor) else v  # noqa: E731
    if case["kind"] == "linear":
        return _exact_linear(wide(s["x"]), s, case["act"])
    leaves = {name: wide(v) for name, v in s["p"].items()}
    leaves["x"], leaves["f"] = wide(s["x"]), wide(s["f"])
    tensors = {name: v for name, v in leaves.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "norm_grad":    # automatic differentiation of the definition
        for v in tensors.values():
            v.requires_grad_(True)
        outputs = _exact_norm(leaves["x"], leaves["f"], leaves)
        return dict(zip(tensors, torch.autograd.grad(outputs, list(tensors.values()), [wide(s["dy"]), wide(s["dh"])])))
    y, h = _exact_norm(leaves["x"], leaves["f"], leaves)
    if case["kind"] == "norm":
        return {"y": y, "h": h}
    return {"y": y, "out": _exact_linear(h, s, case["act"])}
