"""The gated norm: forward, 8-bit rows and gradients against 64 bits with counted roundings, gradients against
differences, refusals; and a block of gated norms and 8-bit linear layers as they are used together."""
import ctypes as C

import pytest
import torch

import norm_int8_ref as ref
import souffle_hip as sh
from gpu_util import announce

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
gpu = pytest.mark.gpu


def values(seed, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (mean + std * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def params(seed, rows, cols, dtype, post, pre, gate, affine=True):
    """Keywords of the operator, tensors on the CPU.  gate: None, "channel", or a number of gate rows."""
    p = {"residual_scale": 0.75, "post_norm": post, "pre_norm": pre, "post_eps": 1e-5, "pre_eps": 1e-6}
    vec = lambda i, mean, *shape: values(seed + i, *shape, dtype=dtype, std=0.3, mean=mean)  # noqa: E731
    if affine and post:
        p["post_gamma"], p["post_beta"] = vec(1, 1.0, cols), vec(2, 0.0, cols)
    if affine:
        p["pre_gamma"], p["pre_beta"] = vec(3, 1.0, cols), vec(4, 0.0, cols)
    if gate:
        p["gate"] = vec(5, 0.5, cols) if gate == "channel" else vec(5, 0.5, gate, cols)
    return p


def cuda(p):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in p.items()}


def run_forward(x, f, p):
    import gated_norm_binding as gn
    t = x.dtype
    y, h = gn.gated_norm(x.cuda(), f.cuda(), **cuda(p))
    ry, rh, ey, eh = ref.forward(x, f, p)
    ref.check("y", y, ry, ey + ref.half_step(ry, t))
    ref.check("h", h, rh, eh + ref.half_step(rh, t))
    y8, q, s = gn.gated_norm_int8(x.cuda(), f.cuda(), **cuda(p))
    assert torch.equal(y8, y) and q.shape == h.shape
    s, amax = s.double().cpu(), rh.abs().amax(-1)
    assert ((s * 127 - amax).abs() <= eh.amax(-1) + 2 * ref.EPS32 * amax + 2.0 ** -93).all()
    # rounded to the nearest step: half of one, what h may be off, and the quotient's last digit
    assert ((q.double().cpu() * s[:, None] - rh).abs() <= 0.5 * s[:, None] * (1 + 2.0 ** -20) + eh).all()


def run_backward(dy, dh, x, f, p):
    import gated_norm_binding as gn
    c = lambda v: None if v is None else v.cuda()  # noqa: E731
    got = gn.gated_norm_backward(c(dy), c(dh), x.cuda(), f.cuda(), **cuda(p))
    again = gn.gated_norm_backward(c(dy), c(dh), x.cuda(), f.cuda(), **cuda(p))
    grads, bounds = ref.backward(dy, dh, x, f, p)
    for name in ("x", "f", "gate", "post_gamma", "post_beta", "pre_gamma", "pre_beta"):
        if name not in ("x", "f") and p.get(name) is None:
            assert got[name] is None, name
            continue
        assert got[name].dtype == x.dtype
        ref.check("gradient of " + name, got[name], grads[name], bounds[name] + ref.half_step(grads[name], x.dtype))
        assert torch.equal(got[name], again[name]), "two calls differ: " + name
    return got


# ------------------------------------------------------------------------------------------------- CPU ----
@pytest.mark.parametrize("post,pre,gate", [("layer", "layer", "channel"), ("rms", "rms", 3), (None, "layer", 2), ("layer", "rms", None)])
def test_reference_gradients_are_those_of_automatic_differentiation(post, pre, gate):
    x, f, dy, dh = (values(i, 6, 10, dtype=torch.float64) for i in range(4))
    p = params(7, 6, 10, torch.float64, post, pre, gate)
    leaves = {k: v.clone().requires_grad_(True) for k, v in {"x": x, "f": f, **p}.items() if isinstance(v, torch.Tensor)}
    po = ref.norm(leaves["f"], post, 1e-5, leaves.get("post_gamma"), leaves.get("post_beta"))[0]
    g = ref.gate_rows(leaves.get("gate"), 6)
    y = 0.75 * leaves["x"] + (po if g is None else g * po)
    h = ref.norm(y, pre, 1e-6, leaves.get("pre_gamma"), leaves.get("pre_beta"))[0]
    auto = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [dy, dh])))
    grads, bounds = ref.backward(dy, dh, x, f, p)
    for name, v in auto.items():
        assert (v - grads[name]).abs().max() < 1e-12, name
        assert (bounds[name] < 1e-3 * (1 + grads[name].abs())).all(), "the bound of %s says nothing" % name


def cfg(**k):
    return sh.GatedNormCfg(*{**dict(rows=4, cols=32, dtype=0, post=1, pre=1, rpg=0, a=1.0, e1=1e-5, e2=1e-5, ldx=32, ldf=32, ldy=32, ldh=32), **k}.values())


def test_refusals_without_gpu():
    lib, P = sh.lib(), 4096
    w = sh.GatedNormW()
    fw = lambda c, w=w, x=P, f=P, y=P, h=P: lib.souffle_gated_norm_forward(C.byref(c), C.byref(w), x, f, y, h, None)  # noqa: E731
    for bad in (dict(rows=-1), dict(cols=0), dict(cols=16385), dict(dtype=3), dict(post=3), dict(pre=0), dict(rpg=3), dict(rpg=-1), dict(e1=-1.0),
                dict(e2=float("nan")), dict(ldx=31), dict(ldf=31), dict(ldy=31), dict(ldh=31)):
        assert fw(cfg(**bad)) == -2, bad
        assert sh.last_error()
    assert lib.souffle_gated_norm_forward(None, C.byref(w), P, P, P, P, None) == -1
    assert lib.souffle_gated_norm_forward(C.byref(cfg()), None, P, P, P, P, None) == -1
    assert fw(cfg(), x=None) == -1 and fw(cfg(), f=None) == -1 and fw(cfg(), h=None) == -1
    assert fw(cfg(), x=P + 1) == -3 and fw(cfg(dtype=2), h=P + 2) == -3 and fw(cfg(rows=0), x=None, f=None, y=None, h=None) == 0
    assert fw(cfg(post=0), w=sh.GatedNormW(post_gamma=P)) == -2 and fw(cfg(), w=sh.GatedNormW(gate=P + 1)) == -3
    f8 = lambda c, q=P, ldq=64, s=P: lib.souffle_gated_norm_forward_int8(C.byref(c), C.byref(w), P, P, None, q, ldq, s, None)  # noqa: E731
    assert f8(cfg(), q=None) == -1 and f8(cfg(), s=None) == -1 and f8(cfg(), ldq=48) == -2 and f8(cfg(), ldq=72) == -3 and f8(cfg(), q=P + 8) == -3
    n = lib.souffle_gated_norm_backward_workspace_bytes(C.byref(cfg()))
    assert n >= 4 * 5 * 32 * 4 and lib.souffle_gated_norm_backward_workspace_bytes(C.byref(cfg(cols=0))) == 0
    full = dict(dx=P, df=P, pre_gamma=P, pre_beta=P, gate=None, post_gamma=P, post_beta=P, ld_dy=32, ld_dh=32, ld_dx=32, ld_df=32)
    bw = lambda c=cfg(), w=w, dy=P, dh=P, x=P, ws=P, n=n, **k: lib.souffle_gated_norm_backward(C.byref(c), C.byref(w), dy, dh, x, P, C.byref(sh.GatedNormGrad(**{**full, **k})), ws, n, None)  # noqa: E731
    assert bw(dy=None, dh=None) == -1 and bw(x=None) == -1 and bw(gate=P) == -1
    assert bw(ws=None) == -4 and bw(n=n - 1) == -4 and bw(ws=P + 8) == -3
    assert bw(ld_dy=31) == -2 and bw(ld_dx=31) == -2 and bw(c=cfg(rows=0)) == -2 and bw(c=cfg(post=0)) == -2 and bw(df=P + 1) == -3 and bw(pre_beta=P + 1) == -3


def test_bindings_refuse_cpu_tensors():
    import gated_norm_binding as gn
    z = torch.zeros(2, 8)
    for call in (lambda: gn.gated_norm(z, z), lambda: gn.gated_norm_int8(z, z), lambda: gn.gated_norm_backward(z, z, z, z)):
        with pytest.raises(TypeError, match="CUDA"):
            call()


# ------------------------------------------------------------------------------------------------- GPU ----
@gpu
def test_bindings_refuse_wrong_tensors():
    announce("gated norm: refusals of the bindings")
    import gated_norm_binding as gn
    x = torch.zeros(6, 32, device="cuda")
    v = torch.zeros(32, device="cuda")
    bad = [(ValueError, (x, x[:5]), {}), (TypeError, (x, x.half()), {}), (TypeError, (x.double(), x.double()), {}), (ValueError, (x, x), dict(post_norm="batch")),
           (ValueError, (x, x), dict(pre_norm=None)), (ValueError, (x, x), dict(gate=v[:31])), (ValueError, (x, x), dict(gate=torch.zeros(4, 32, device="cuda"))),
           (ValueError, (x, x), dict(gate=v.half())), (ValueError, (x, x), dict(pre_gamma=v.view(1, 32))), (ValueError, (x, x), dict(post_norm=None, post_gamma=v)),
           (ValueError, (x.t(), x.t()), {}), (ValueError, (x[:1].expand(6, 32), x), {}), (TypeError, (x, x), dict(gate=v.cpu())), (sh.SouffleError, (x, x), dict(pre_eps=-1.0))]
    for error, args, kw in bad:
        with pytest.raises(error):
            gn.gated_norm(*args, **kw)
    for dy, dh in ((None, None), (x[:5], x), (x, x.half())):
        with pytest.raises(ValueError):
            gn.gated_norm_backward(dy, dh, x, x)


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 513), (7, 768), (4, 1001), (3, 2048), (2, 2049), (3, 4096), (2, 4099), (2, 8192), (1, 8200), (2, 16384)]


@gpu
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_sizes(dtype, rows, cols):
    announce("gated norm %s %dx%d" % (dtype, rows, cols))
    x, f = values(1, rows, cols, dtype=TYPES[dtype], std=2.0), values(2, rows, cols, dtype=TYPES[dtype])
    run_forward(x, f, params(3, rows, cols, TYPES[dtype], "layer", "layer", "channel"))


@gpu
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_sizes(dtype, rows, cols):
    announce("gated norm gradient %s %dx%d" % (dtype, rows, cols))
    x, f, dy, dh = (values(i, rows, cols, dtype=TYPES[dtype]) for i in range(4))
    run_backward(dy, dh, x, f, params(5, rows, cols, TYPES[dtype], "layer", "layer", "channel"))


@gpu
@pytest.mark.parametrize("post", ["layer", "rms", None])
@pytest.mark.parametrize("pre", ["layer", "rms"])
@pytest.mark.parametrize("gate", [None, "channel", 3, 12])
@pytest.mark.parametrize("affine", [True, False])
def test_every_form(post, pre, gate, affine):
    announce("gated norm post=%s pre=%s gate=%s affine=%s" % (post, pre, gate, affine))
    for dtype, cols in (("f32", 200), ("bf16", 1100)):
        t = TYPES[dtype]
        x, f, dy, dh = (values(10 + i, 12, cols, dtype=t, mean=0.2) for i in range(4))
        p = params(9, 12, cols, t, post, pre, gate, affine)
        run_forward(x, f, p)
        run_backward(dy, dh, x, f, p)


@gpu
@pytest.mark.parametrize("rows,cols,gate", [(700, 96, "channel"), (1111, 520, None), (600, 64, 300), (600, 64, 600), (260, 1032, 4), (515, 256, 5), (300, 4096, 2), (9000, 40, 9)])
def test_many_rows(rows, cols, gate):
    """Chunks of rows: inside one gate row, across several, as many gate rows as rows."""
    announce("gated norm %dx%d gate=%s" % (rows, cols, gate))
    x, f, dy, dh = (values(i, rows, cols) for i in range(4))
    p = params(5, rows, cols, torch.float32, "layer", "rms", gate)
    run_forward(x, f, p)
    run_backward(dy, dh, x, f, p)


@gpu
@pytest.mark.parametrize("gate", [None, 7, "channel"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 16, 100, 128, 129, 200, 250, 256, 257])
def test_rows_that_share_a_wave(cols, dtype, gate):
    announce("gated norm %s of %d columns, gate=%s" % (dtype, cols, gate))
    rows = 77 * 7
    x, f, dy, dh = (values(60 + i, rows, cols, dtype=TYPES[dtype], mean=0.1) for i in range(4))
    p = params(65, rows, cols, TYPES[dtype], "layer" if gate else "rms", "layer" if cols > 1 else "rms", gate)
    x[5] = 0 if cols > 1 else x[5]
    run_forward(x, f, p)
    run_backward(dy, dh, x, f, p)
    x[9] = float("nan")      # stays in its row
    import gated_norm_binding as gn
    y, h = gn.gated_norm(x.cuda(), f.cuda(), **cuda(p))
    y8, q, s = gn.gated_norm_int8(x.cuda(), f.cuda(), **cuda(p))
    g = gn.gated_norm_backward(dy.cuda(), dh.cuda(), x.cuda(), f.cuda(), **cuda(p))
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[9] = True
    for v in (h.isnan().all(1), s.isnan(), g["x"].isnan().all(1)):
        assert torch.equal(v, bad)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [5, 40, 203, 1000, 1033, 2056, 4100, 8200])
@pytest.mark.parametrize("gates,per_gate", [(300, 1), (261, 3), (256, 7), (257, 8), (90, 2)])
def test_gradient_with_few_rows_per_gate(gates, per_gate, cols, dtype):
    """Gate rows of one row and of several, more and fewer than there are chunks, the last chunk not full."""
    announce("gated norm gradient %s %d gate rows of %d rows, %d columns" % (dtype, gates, per_gate, cols))
    rows = gates * per_gate if cols < 4000 else min(gates, 258) * min(per_gate, 2)
    gates = rows // (per_gate if cols < 4000 else min(per_gate, 2))
    x, f, dy, dh = (values(20 + i, rows, cols, dtype=TYPES[dtype]) for i in range(4))
    run_backward(dy, dh, x, f, params(25, rows, cols, TYPES[dtype], "layer", "rms", gates))


@gpu
@pytest.mark.parametrize("gates,rows,cols", [(128, 512, 1033), (2, 600, 40), (60, 600, 2100), (300, 600, 72)])
def test_gate_rows_with_several_chunks_and_gradients_not_wanted(gates, rows, cols):
    """Gate rows made of few and of many chunks; and the other gradients keep their bits where the gate's is not wanted
    (its sums are then of other chunks: those of the vectors may differ, dx and df may not)."""
    import gated_norm_binding as gn
    announce("gated norm gradient %d gate rows of %d rows, %d columns" % (gates, rows, cols))
    x, f, dy, dh = (values(40 + i, rows, cols) for i in range(4))
    p = params(45, rows, cols, torch.float32, "rms", "layer", gates)
    got = run_backward(dy, dh, x, f, p)
    grads, bounds = ref.backward(dy, dh, x, f, p)
    x, f, dy, dh, p = x.cuda(), f.cuda(), dy.cuda(), dh.cuda(), cuda(p)
    dx, df, gamma = torch.empty_like(x), torch.empty_like(x), torch.empty(cols, device="cuda")
    cfg = gn._cfg(rows, cols, sh.F32, sh.NORM_RMS, sh.NORM_LAYER, rows // gates, 0.75, 1e-5, 1e-6, cols, cols, cols, cols)
    w = sh.GatedNormW(*[p[k].data_ptr() for k in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")])
    grad = sh.GatedNormGrad(dx.data_ptr(), df.data_ptr(), gamma.data_ptr(), None, None, None, None, cols, cols, cols, cols)
    ws = torch.empty(sh.lib().souffle_gated_norm_backward_workspace_bytes(cfg), dtype=torch.uint8, device="cuda")
    sh.check(sh.lib().souffle_gated_norm_backward(cfg, w, dy.data_ptr(), dh.data_ptr(), x.data_ptr(), f.data_ptr(), grad, ws.data_ptr(), ws.numel(),
                                                  torch.cuda.current_stream().cuda_stream))
    assert torch.equal(dx, got["x"]) and torch.equal(df, got["f"])
    ref.check("gradient of pre_gamma alone", gamma, grads["pre_gamma"], bounds["pre_gamma"])


@gpu
def test_one_incoming_gradient():
    announce("gated norm gradient: dy or dh alone")
    x, f, d = (values(i, 20, 72) for i in range(3))
    p = params(5, 20, 72, torch.float32, "rms", "layer", 4)
    run_backward(d, None, x, f, p)
    run_backward(None, d, x, f, p)


@gpu
@pytest.mark.parametrize("post,pre,gate", [("layer", "layer", "channel"), ("rms", "rms", 3), (None, "layer", 3), ("layer", "rms", None)])
def test_gradients_against_differences(post, pre, gate):
    """The change of sum(dy y + dh h) along a random direction of every input, by central differences in 64 bits: with
    steps of 1e-4 they are good to 1e-7, the gradients in fp32 to 1e-5 of the terms' size (here about one per element)."""
    announce("gated norm gradient against differences: %s %s %s" % (post, pre, gate))
    import gated_norm_binding as gn
    rows, cols = 6, 50
    x, f, dy, dh = (values(20 + i, rows, cols) for i in range(4))
    p = params(30, rows, cols, torch.float32, post, pre, gate)
    got = gn.gated_norm_backward(dy.cuda(), dh.cuda(), x.cuda(), f.cuda(), **cuda(p))
    inputs = {"x": x, "f": f, **{k: v for k, v in p.items() if isinstance(v, torch.Tensor)}}

    def loss(inputs):
        y, h, _, _ = ref.forward(inputs["x"], inputs["f"], {**p, **{k: v for k, v in inputs.items() if k not in ("x", "f")}})
        return float((dy.double() * y + dh.double() * h).sum())
    for i, (name, v) in enumerate(inputs.items()):
        u = values(40 + i, *v.shape, dtype=torch.float64)
        at = lambda e: loss({**inputs, name: v.double() + e * u})  # noqa: E731
        diff = (at(1e-4) - at(-1e-4)) / 2e-4
        along = float((got[name].double().cpu() * u).sum())
        size = float((got[name].double().cpu() * u).abs().sum())
        assert abs(diff - along) <= 1e-5 * size + 1e-6, (name, diff, along)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("post,pre,gate", [("layer", "layer", "channel"), ("rms", "rms", 3), (None, "layer", 6), ("layer", "rms", None)])
def test_autograd_gives_the_gradient(dtype, post, pre, gate):
    """loss.backward() through gated_norm is gated_norm_backward, bit for bit, with and without another path to the loss."""
    import gated_norm_binding as gn
    announce("gated norm by autograd: %s %s %s %s" % (dtype, post, pre, gate))
    t = TYPES[dtype]
    x, f, dy, dh = (values(90 + i, 2, 3, 72, dtype=t).cuda() for i in range(4))
    p = cuda(params(95, 6, 72, t, post, pre, gate))
    leaves = {"x": x, "f": f, **{k: v for k, v in p.items() if isinstance(v, torch.Tensor)}}
    expect = gn.gated_norm_backward(dy, dh, x, f, **p)
    plain = gn.gated_norm(x, f, **p)
    assert not plain[0].requires_grad and not plain[1].requires_grad
    for v in leaves.values():
        v.requires_grad_(True)
    with torch.no_grad():
        assert not gn.gated_norm(x, f, **p)[1].requires_grad
    y, h = gn.gated_norm(x, f, **p)
    assert torch.equal(y, plain[0]) and torch.equal(h, plain[1]) and y.requires_grad and h.requires_grad
    for name, got in zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [dy, dh], retain_graph=True)):
        assert got.dtype == t and torch.equal(got, expect[name]), name
    y.backward(dy, retain_graph=True)      # one output alone, accumulated into the leaves
    alone = gn.gated_norm_backward(dy, None, x.detach(), f.detach(), **{k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in p.items()})
    for name, v in leaves.items():
        assert torch.equal(v.grad, alone[name]), name
        v.grad = None
    (h * dh).sum().backward()
    alone = gn.gated_norm_backward(None, dh, x.detach(), f.detach(), **{k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in p.items()})
    for name, v in leaves.items():
        assert torch.equal(v.grad, alone[name]), name
    # beside another path, the expanded gradient of a sum, y not wanted, and only some inputs that require a gradient
    f, frozen = f.detach(), {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    x.grad = None
    _, h = gn.gated_norm(x, f, **frozen, want_y=False)
    assert _ is None
    (h.sum() + x.sum()).backward()
    one = torch.ones_like(x)
    assert torch.equal(x.grad, one + gn.gated_norm_backward(None, one, x.detach(), f, **frozen)["x"])


@gpu
def test_autograd_refuses_what_it_cannot_do():
    """A second derivative, inputs written over before the backward pass, and a captured backward pass; the leaves stay usable."""
    import gated_norm_binding as gn
    announce("gated norm by autograd: refusals")
    x, f, d = (values(i, 6, 72).cuda() for i in range(3))
    x.requires_grad_(True)
    y, h = gn.gated_norm(x, f)
    first, = torch.autograd.grad(h, x, d, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)
    y, h = gn.gated_norm(x, f)
    f.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.backward(d)
    expect = gn.gated_norm(x.detach(), f)[1]
    kept = gn.gated_norm(x, f)      # an eager graph of the same leaf stays alive
    x.grad = None
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _, held = gn.gated_norm(x, f)
        with pytest.raises(RuntimeError, match="capture gated_norm_backward"):
            held.backward(d)
    assert x.grad is None
    for _ in range(3):
        held.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, expect)
    kept[1].backward(d)
    assert torch.equal(x.grad, gn.gated_norm_backward(None, d, x.detach(), f)["x"])


@gpu
def test_rows_apart_in_place_and_what_lies_around():
    """Slices of wider tensors that start anywhere as inputs; through the C ABI: y over x and h over f in place, outputs in
    rows apart, columns and rows around them left as they were."""
    announce("gated norm: strides, in place, canaries")
    import gated_norm_binding as gn
    for t in TYPES.values():
        for rows, cols in ((5, 77), (3, 1500)):
            wide = [values(i, rows + 2, cols + 9, dtype=t).cuda() for i in range(2)]
            x, f = (w[1:rows + 1, 3:cols + 3] for w in wide)
            p = cuda(params(5, rows, cols, t, "layer", "rms", "channel"))
            y0, h0 = gn.gated_norm(x.contiguous(), f.contiguous(), **p)
            y1, h1 = gn.gated_norm(x, f, **p)
            assert torch.equal(y0, y1) and torch.equal(h0, h1)
            y2, h2 = gn.gated_norm(x, f, **p, want_y=False)
            assert y2 is None and torch.equal(h0, h2)
            d = values(8, rows, cols, dtype=t).cuda()
            for a, b in zip(gn.gated_norm_backward(d, y0, x, f, **p).values(), gn.gated_norm_backward(d, y0, x.contiguous(), f.contiguous(), **p).values()):
                assert (a is None and b is None) or torch.equal(a, b)
            before = [w.clone() for w in wide]
            c = sh.GatedNormCfg(rows, cols, {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[t], 1, 2, 0, p["residual_scale"], p["post_eps"], p["pre_eps"],
                                cols + 9, cols + 9, cols + 9, cols + 9)
            w = sh.GatedNormW(*(sh.ptr(p.get(n)) for n in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")))
            sh.check(sh.lib().souffle_gated_norm_forward(C.byref(c), C.byref(w), x.data_ptr(), f.data_ptr(), x.data_ptr(), f.data_ptr(), sh.current_stream()))
            torch.cuda.synchronize()
            assert torch.equal(x, y0) and torch.equal(f, h0)
            for now, old, inner in zip(wide, before, (y0, h0)):
                old[1:rows + 1, 3:cols + 3] = inner
                assert torch.equal(now, old), "written outside the rows"


# (type, rows, columns, gate rows): more rows than the forward launch has slots for, so that a slot walks over two or three of them, for every
# count of threads per row; an odd number of rows per gate row, so that its border falls inside a slot's run.
WALKS = [("f16", 33000, 7, 40), ("f32", 33000, 40, 40), ("bf16", 70000, 24, 16), ("f16", 33000, 250, 40), ("bf16", 9000, 300, 8), ("f16", 8200, 520, 8),
         ("f32", 4100, 1001, 4), ("bf16", 2100, 1100, 4), ("f32", 2100, 1104, 4), ("f16", 2100, 2056, 4), ("f32", 1030, 2056, 2), ("bf16", 1030, 4104, 2),
         ("f32", 1100, 4099, 4), ("f16", 520, 8200, 8), ("f32", 520, 8200, 8)]


def threads_per_row(dtype, cols):
    """Of the forward kernel."""
    if dtype == "f32":
        return next(t for t, most in ((16, 256), (64, 512), (128, 1024), (256, 2048), (512, 4096), (1024, 16384)) if cols <= most)
    return next(t for t, most in ((16, 256), (64, 1024), (256, 4096), (512, 8192), (1024, 16384)) if cols <= most)


def abi(x, p, gates):
    """(cfg, vectors, (ld, dtype)) of the C calls on contiguous rows like x's with the keywords p."""
    rows, cols = x.shape
    kinds = {None: sh.NORM_NONE, "layer": sh.NORM_LAYER, "rms": sh.NORM_RMS}
    c = sh.GatedNormCfg(rows, cols, {torch.float16: sh.F16, torch.bfloat16: sh.BF16, torch.float32: sh.F32}[x.dtype], kinds[p["post_norm"]], kinds[p["pre_norm"]],
                        rows // gates if gates else 0, p["residual_scale"], p["post_eps"], p["pre_eps"], cols, cols, cols, cols)
    return c, sh.GatedNormW(*(sh.ptr(p.get(n)) for n in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")))


@gpu
@pytest.mark.parametrize("dtype,rows,cols,gates", WALKS)
def test_forward_walks_over_several_rows(dtype, rows, cols, gates):
    """The next row asked for while the present one is reduced, the gate changed on the way: against 64 bits, and in place."""
    import gated_norm_binding as gn
    announce("gated norm %s %dx%d, %d gate rows: several rows a slot" % (dtype, rows, cols, gates))
    slots = sh.device_info()["num_cus"] * 2048 // threads_per_row(dtype, cols)
    per_slot = -(-rows // slots)
    assert per_slot > 1 and rows // gates % per_slot, "this case does not test what it is for"
    x, f = values(70, rows, cols, dtype=TYPES[dtype], std=2.0, mean=0.1), values(71, rows, cols, dtype=TYPES[dtype])
    post, pre = [("layer", "rms"), ("rms", "layer"), (None, "layer"), ("layer", "layer")][cols % 4]
    p = params(72, rows, cols, TYPES[dtype], post, pre, gates)
    run_forward(x, f, p)
    x, f, p = x.cuda(), f.cuda(), cuda(p)
    y, h = gn.gated_norm(x, f, **p)
    for over in ((0, 1), (1, 0)):      # y over x and h over f, and the other way round
        a = [x.clone(), f.clone()]
        c, w = abi(x, p, gates)
        sh.check(sh.lib().souffle_gated_norm_forward(C.byref(c), C.byref(w), a[0].data_ptr(), a[1].data_ptr(), a[over[0]].data_ptr(), a[over[1]].data_ptr(),
                                                     sh.current_stream()))
        torch.cuda.synchronize()
        assert torch.equal(a[over[0]], y) and torch.equal(a[over[1]], h)


@gpu
@pytest.mark.parametrize("dtype,rows,cols,gates", [("f32", 3001, 200, None), ("bf16", 2100, 1001, None), ("f16", 6000, 64, 8), ("f16", 515, 300, 515), ("f32", 783, 520, 261),
                                                   ("bf16", 90, 2100, 90), ("f16", 600, 4100, 4), ("f32", 520, 5000, None), ("f32", 300, 8200, 300), ("bf16", 270, 8200, 1)])
def test_gradient_in_place(dtype, rows, cols, gates):
    """dx over dy and df over dh gives the bits of outputs of their own: slots without a row, several turns, a gate row a token, wide rows."""
    announce("gated norm gradient in place %s %dx%d, gate rows: %s" % (dtype, rows, cols, gates))
    x, f, dy, dh = (values(80 + i, rows, cols, dtype=TYPES[dtype]).cuda() for i in range(4))
    p = cuda(params(85, rows, cols, TYPES[dtype], "layer", "layer" if gates else "rms", gates or "channel"))
    c, w = abi(x, p, gates)
    names = ("pre_gamma", "pre_beta", "gate", "post_gamma", "post_beta")
    ws = torch.empty(sh.lib().souffle_gated_norm_backward_workspace_bytes(C.byref(c)), dtype=torch.uint8, device="cuda")

    def call(dx, df, dy, dh):
        vectors = [torch.empty_like(p[n]) for n in names]
        grad = sh.GatedNormGrad(dx.data_ptr(), df.data_ptr(), *(v.data_ptr() for v in vectors), cols, cols, cols, cols)
        sh.check(sh.lib().souffle_gated_norm_backward(C.byref(c), C.byref(w), sh.ptr(dy), sh.ptr(dh), x.data_ptr(), f.data_ptr(), C.byref(grad), ws.data_ptr(),
                                                      ws.numel(), sh.current_stream()))
        return [dx, df] + vectors
    for given in ((dy, dh), (dy, None), (None, dh)):
        apart = call(torch.empty_like(x), torch.empty_like(x), *given)
        mine = [None if d is None else d.clone() for d in given]
        over = call(*(torch.empty_like(x) if d is None else d for d in mine), *mine)
        torch.cuda.synchronize()
        for name, a, b in zip(("x", "f") + names, apart, over):
            assert torch.isfinite(a).all() and torch.equal(a, b), name


@gpu
def test_hard_rows():
    """Constant rows, zero rows, a mean a thousand times the deviation; NaN and infinity stay in their rows."""
    announce("gated norm: constant, shifted and non-finite rows")
    import gated_norm_binding as gn
    x, f = values(1, 6, 300), values(2, 6, 300)
    x[0], f[0] = 0, 0
    x[1], f[1] = 3.0, -2.0
    x[2] += 1000
    f[2] += 1000
    p = params(3, 6, 300, torch.float32, "layer", "layer", "channel")
    run_forward(x, f, p)
    run_backward(values(4, 6, 300), values(5, 6, 300), x, f, p)
    y0, h0 = gn.gated_norm(x.cuda(), f.cuda(), **cuda(p))
    x[3, 7], f[4, 299] = float("nan"), float("inf")
    y, h = gn.gated_norm(x.cuda(), f.cuda(), **cuda(p))
    _, q, s = gn.gated_norm_int8(x.cuda(), f.cuda(), **cuda(p))
    assert torch.isnan(h[3]).all() and torch.isnan(h[4]).all() and torch.isnan(s[3:5]).all() and not q[3:5].any()
    keep = [0, 1, 2, 5]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(h[keep], h0[keep]) and torch.isfinite(s[keep]).all()


@gpu
def test_no_rows_and_leading_dimensions():
    announce("gated norm: no rows, three dimensions")
    import gated_norm_binding as gn
    e, v = torch.empty(0, 40, device="cuda"), torch.ones(40, device="cuda")
    y, h = gn.gated_norm(e, e, gate=v)
    assert y.shape == h.shape == (0, 40)
    y, q, s = gn.gated_norm_int8(e, e)
    assert q.shape == (0, 40) and s.shape == (0,)
    g = gn.gated_norm_backward(e, e, e, e, gate=v, pre_gamma=v)
    assert g["x"].shape == (0, 40) and not g["gate"].any() and not g["pre_gamma"].any() and g["post_gamma"] is None
    x, f = values(1, 2, 3, 40).cuda(), values(2, 2, 3, 40).cuda()
    gate = values(3, 2, 40).cuda()
    y, h = gn.gated_norm(x, f, gate=gate)
    y2, h2 = gn.gated_norm(x.view(6, 40), f.view(6, 40), gate=gate)
    assert y.shape == x.shape and torch.equal(y.view(6, 40), y2) and torch.equal(h.view(6, 40), h2)


def test_rows_at_one_distance():
    """Which tensors are rows at one distance, without a copy."""
    import linear_int8_binding as lb
    t = torch.arange(4 * 6 * 10).view(4, 6, 10)
    for v, ld in ((t, 10), (t[..., 2:7], 10), (t[:, -1:], 60), (t[:, -1], 60), (t[:1, 1:3, :9], 10), (t[2, 3], 10), (t[2:3, 4:5, 3:5], 2), (t[:, :, :1], 10),
                  (t.view(2, 2, 6, 10)[..., 1:4], 10), (t[:0, :, 1:3], None), (t[:, :, 3:3], None)):
        rows, got = lb._rows("t", v)
        assert rows.dim() == 2 and torch.equal(rows, v.reshape(v.shape[:-1].numel(), v.shape[-1])) and (not v.numel() or rows.data_ptr() == v.data_ptr())
        assert ld is None or got == ld
        if v.numel():
            assert torch.equal(torch.as_strided(v, rows.shape, (got, 1), v.storage_offset()), rows)
    for bad in (t[:, 1:3], t.transpose(0, 1), t.transpose(1, 2), t[:1].expand(4, 6, 10), t[..., ::2], t.flip(0)[0, 0, 0], t[0, 0, ::2]):
        with pytest.raises(ValueError):
            lb._rows("t", bad)


@gpu
def test_slices_of_three_dimensions():
    announce("gated norm and 8-bit layer: slices of [B, S, D]")
    import gated_norm_binding as gn
    import linear_int8_binding as lb
    wide = [values(50 + i, 4, 6, 90, dtype=torch.float16).cuda() for i in range(4)]
    w = lb.quantize_weight(values(60, 77, 40).cuda())
    gate = values(61, 4, 77, dtype=torch.float16).cuda()
    for at in (lambda v: v[..., 5:82], lambda v: v[:, -1:, 5:82], lambda v: v[1:2, 2:4, :77].expand(1, 2, 77)):
        x, f, dy, dh = (at(v) for v in wide)
        near = [v.contiguous() for v in (x, f, dy, dh)]
        p = dict(gate=gate if x.shape[0] == 4 else gate[0])
        for a, b in ((gn.gated_norm(x, f, **p), gn.gated_norm(*near[:2], **p)), (gn.gated_norm_int8(x, f, **p), gn.gated_norm_int8(*near[:2], **p)),
                     (gn.gated_norm_backward(dy, dh, x, f, **p).values(), gn.gated_norm_backward(near[2], near[3], *near[:2], **p).values()),
                     (lb.quantize_rows(x), lb.quantize_rows(near[0])), ((lb.linear_int8(x, w),), (lb.linear_int8(near[0], w),))):
            for u, v in zip(a, b):
                assert (u is None and v is None) or (u.shape == v.shape and torch.equal(u, v))
        assert gn.gated_norm(x, f)[0].shape == x.shape


@gpu
def test_rows_beyond_two_gib():
    announce("gated norm: offsets beyond 2^31")
    import gated_norm_binding as gn
    rows, wide, cols = 70000, 32800, 48
    big = torch.empty((rows, wide), dtype=torch.float16, device="cuda")
    x, src, f = big[:, 32700:32700 + cols], values(9, rows, cols, dtype=torch.float16).cuda(), values(8, rows, cols, dtype=torch.float16).cuda()
    x.copy_(src)
    for a, b in zip(gn.gated_norm(x, f), gn.gated_norm(src, f)):
        assert torch.equal(a, b)
    for a, b in zip(gn.gated_norm_backward(f, f, x, f).values(), gn.gated_norm_backward(f, f, src, f).values()):
        assert (a is None and b is None) or torch.equal(a, b)


# ------------------------------------------------------------------------------- together, as they are used ----
def block(x, f, p1, w1, b1, w2, b2, p2):
    """The MLP of a transformer block: the norm in front of it hands over 8-bit rows, the norm behind it takes its output."""
    import gated_norm_binding as gn
    import linear_int8_binding as lb
    y, q, s = gn.gated_norm_int8(x, f, **p1)
    u = lb.gemm_int8(q, s, w1, bias=b1, act="gelu_tanh", dtype=x.dtype)
    m = lb.linear_int8(u, w2, bias=b2)
    y2, h2 = gn.gated_norm(y, m, **p2)
    return y, q, s, u, m, y2, h2


def block_inputs(rows, D, F, t, seed):
    import linear_int8_binding as lb
    x, f = values(seed, rows, D, dtype=t).cuda(), values(seed + 1, rows, D, dtype=t).cuda()
    p1, p2 = (cuda(params(seed + 10 * i, rows, D, t, "layer", "layer", "channel")) for i in (1, 2))
    w1, w2 = lb.quantize_weight(values(seed + 2, D, F, std=D ** -0.5).cuda()), lb.quantize_weight(values(seed + 3, F, D, std=F ** -0.5).cuda())
    return x, f, p1, w1, values(seed + 4, F, dtype=t).cuda(), w2, values(seed + 5, D, dtype=t).cuda(), p2


def unpack(w):
    K, N = w.in_features, w.out_features
    from test_linear_int8 import packed_index
    return w.packed.cpu()[torch.from_numpy(packed_index(K, N))]


@gpu
@pytest.mark.parametrize("rows,D,F,dtype", [(1, 768, 1000, "f16"), (49, 256, 1024, "bf16"), (300, 130, 500, "f32")])
def test_block_step_by_step(rows, D, F, dtype):
    """Every step of the block against 64 bits from what the step before handed over."""
    announce("block of gated norms and 8-bit layers %d x %d x %d %s" % (rows, D, F, dtype))
    t = TYPES[dtype]
    x, f, p1, w1, b1, w2, b2, p2 = block_inputs(rows, D, F, t, 100)
    y, q, s, u, m, y2, h2 = block(x, f, p1, w1, b1, w2, b2, p2)
    ry, rh, ey, eh = ref.forward(x, f, p1)
    ref.check("y", y, ry, ey + ref.half_step(ry, t))
    assert ((q.double().cpu() * s.double().cpu()[:, None] - rh).abs() <= 0.5 * s.double().cpu()[:, None] * (1 + 2.0 ** -20) + eh).all()
    r, e = ref.linear(q.cpu(), s.cpu(), unpack(w1), w1.scale.cpu(), b1.cpu(), "gelu_tanh")
    ref.check("first layer", u, r, e + ref.half_step(r, t))
    r, e = ref.linear(*ref.quantize(u.cpu()), unpack(w2), w2.scale.cpu(), b2.cpu(), None)
    ref.check("second layer", m, r, e + ref.half_step(r, t))
    ry, rh, ey, eh = ref.forward(y.cpu(), m.cpu(), p2)
    ref.check("y of the next block", y2, ry, ey + ref.half_step(ry, t))
    ref.check("h of the next block", h2, rh, eh + ref.half_step(rh, t))


@gpu
@pytest.mark.parametrize("rows", [1, 80])
def test_block_and_gradient_in_a_graph_and_on_another_stream(rows):
    """Captured once and replayed on new inputs with eager work in between, and on a stream of its own: the eager bits."""
    announce("block in a graph, rows=%d" % rows)
    import gated_norm_binding as gn
    x, f, p1, w1, b1, w2, b2, p2 = block_inputs(rows, 192, 320, torch.float16, 200)

    def everything(x, f):
        out = block(x, f, p1, w1, b1, w2, b2, p2)
        g = gn.gated_norm_backward(out[5], out[6], x, f, **p1)
        return list(out) + [v for v in g.values() if v is not None]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = everything(x, f)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, everything(x, f)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything(x, f)
    for i in range(4):
        nx, nf = values(300 + i, rows, 192, dtype=torch.float16).cuda(), values(400 + i, rows, 192, dtype=torch.float16).cuda()
        eager = everything(nx, nf)
        x.copy_(nx)
        f.copy_(nf)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b), "replay %d" % i


@gpu
def test_calls_at_once_from_two_threads_and_two_graphs():
    """Calls of different sizes on two streams at once, from two threads and as two captured graphs replayed side by side,
    give what each gives alone."""
    import threading

    import gated_norm_binding as gn
    import linear_int8_binding as lb
    announce("two threads and two graphs at once")

    def work(seed, rows, d, n):
        x, f, dy, dh = (values(seed + i, rows, d, dtype=torch.float16).cuda() for i in range(4))
        p = cuda(params(seed + 4, rows, d, torch.float16, "layer", "rms", "channel"))
        w, b = lb.quantize_weight(values(seed + 9, d, n).cuda()), values(seed + 10, n, dtype=torch.float16).cuda()

        def step():
            y, q, s = gn.gated_norm_int8(x, f, **p)
            z = lb.gemm_int8(q, s, w, bias=b, act="gelu")
            z2 = lb.linear_int8(y, w, bias=b, act="relu")
            g = gn.gated_norm_backward(dy, dh, x, f, **p)
            return [y, q.contiguous(), s, z, z2] + [v for v in g.values() if v is not None]
        return step
    steps = [work(1, 300, 520, 700), work(31, 2000, 1100, 300)]
    alone = [s() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    wrong = []

    def many(k):
        try:
            with torch.cuda.stream(streams[k]):
                for _ in range(20):
                    got = steps[k]()
                    if not all(torch.equal(a, b) for a, b in zip(got, alone[k])):
                        wrong.append(k)
        except Exception as e:      # (a thread's own errors do not reach the test)
            wrong.append(e)
    threads = [threading.Thread(target=many, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, s in zip(graphs, steps):
        with torch.cuda.graph(g):
            outs.append(s())
    for turn in range(4):
        for out in outs:
            for v in out:
                v.zero_()
        torch.cuda.synchronize()
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        eager = steps[turn % 2]()      # and the same work beside them
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], alone[k])), "graph %d, replay %d" % (k, turn)
        assert all(torch.equal(a, b) for a, b in zip(eager, alone[turn % 2]))


@gpu
def test_post_norm_encoder_form():
    """LN(x + f) of a post-norm encoder: no norm behind the block, no gate, y not kept."""
    announce("gated norm as LN(x + f)")
    import gated_norm_binding as gn
    x, f, g, b = values(1, 64, 768, dtype=torch.float16), values(2, 64, 768, dtype=torch.float16), values(3, 768, dtype=torch.float16), values(4, 768, dtype=torch.float16)
    y, h = gn.gated_norm(x.cuda(), f.cuda(), post_norm=None, pre_gamma=g.cuda(), pre_beta=b.cuda(), pre_eps=1e-12, want_y=False)
    p = {"post_norm": None, "pre_gamma": g, "pre_beta": b, "pre_eps": 1e-12}
    _, rh, _, eh = ref.forward(x, f, p)
    ref.check("h", h, rh, eh + ref.half_step(rh, torch.float16))
    r = torch.nn.functional.layer_norm(x.double() + f.double(), (768,), g.double(), b.double(), 1e-12)
    assert y is None and (rh - r).abs().max() < 1e-10
