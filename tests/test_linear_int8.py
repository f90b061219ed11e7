"""8-bit linear layers: row and weight quantisation and the packed layout (exact), the product with its epilogue against
64 bits, and what the entry points refuse.  CPU: the reference against the definition, refusals.  GPU: the kernels."""
import ctypes as C

import numpy as np
import pytest
import torch

import norm_int8_ref as ref
import souffle_hip as sh
from gpu_util import announce

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
gpu = pytest.mark.gpu


def values(seed, *shape, dtype=torch.float32, std=1.0):
    return (std * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def weight(seed, K, N):
    """(Wq int8, scale) of a random matrix, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (K, N), generator=g, dtype=torch.int8), 0.001 + 0.01 * torch.rand(N, generator=g)


def packed_index(K, N):
    """Offset of weight (k, n) in the packed copy, as include/souffle_hip.h states it."""
    k, n = np.arange(K)[:, None], np.arange(N)[None, :]
    return ((n // 64 * -(-K // 64) + k // 64) * 4 + n // 4 % 4) * 1024 + (k // 16 % 4 * 16 + n // 16 % 4 * 4 + n % 4) * 16 + k % 16


def test_packed_layout_covers_every_byte_once():
    for K, N in [(64, 64), (128, 192), (192, 64)]:
        assert sorted(packed_index(K, N).reshape(-1).tolist()) == list(range(K * N))


def test_reference_rounds_halves_to_even():
    q, s = ref.quantize(torch.tensor([[127.0, 0.5, 1.5, -2.5, 63.5, -63.5]]))
    assert s.item() == 1.0 and q.tolist() == [[127, 0, 2, -2, 64, -64]]


def test_refusals_without_gpu():
    lib, P = sh.lib(), 4096      # an aligned address that no refused call reads
    assert lib.souffle_int8_packed_bytes(100, 65) == 128 * 128
    assert lib.souffle_int8_packed_bytes(0, 64) == 0 and "K must be" in sh.last_error()
    assert lib.souffle_int8_packed_bytes(131072, 64) == 0 and lib.souffle_int8_packed_bytes(131071, 64) == 131072 * 64
    assert lib.souffle_linear_int8_workspace_bytes(300, 8000, 1100) >= 300 * (1152 + 4) and lib.souffle_linear_int8_workspace_bytes(-1, 64, 100) == 0
    q = lambda **k: lib.souffle_quantize_rows(*{**dict(x=P, t=0, ldx=100, q=P, ldq=128, s=P, M=2, K=100, st=None), **k}.values())  # noqa: E731
    assert q(x=None) == -1 and q(q=None) == -1 and q(s=None) == -1
    assert q(t=3) == -2 and "dtype" in sh.last_error()
    assert q(ldx=99) == -2 and "overlap" in sh.last_error()
    assert q(ldq=112) == -2 and q(ldq=120) == -3 and q(q=P + 8) == -3 and q(x=P + 1) == -3 and q(s=P + 2) == -3
    assert q(M=-1) == -2 and q(K=0) == -2 and q(M=0, x=None) == 0
    g = lambda **k: lib.souffle_gemm_int8(*{**dict(q=P, ldq=128, rs=P, w=P, cs=P, b=None, act=3, y=P, t=0, ldy=50, M=2, N=50, K=100, st=None), **k}.values())  # noqa: E731
    for name in ("q", "rs", "w", "cs", "y"):
        assert g(**{name: None}) == -1, name
    assert g(act=4) == -2 and "activation" in sh.last_error()
    assert g(t=-1) == -2 and g(ldy=49) == -2 and g(ldq=64) == -2 and g(N=0) == -2 and g(K=131072) == -2 and g(M=-1) == -2
    assert g(ldq=136) == -3 and g(w=P + 8) == -3 and g(b=P + 1) == -3 and g(y=P + 1) == -3 and g(M=0, q=None, y=None) == 0
    l = lambda **k: lib.souffle_linear_int8(*{**dict(x=P, ldx=2000, w=P, cs=P, b=None, act=3, y=P, t=2, ldy=50, M=200, N=50, K=2000, ws=P, n=1 << 20, st=None), **k}.values())  # noqa: E731
    assert l(ws=None) == -4 and l(n=100) == -4 and "workspace" in sh.last_error()
    assert l(x=None) == -1 and l(ldx=1999) == -2 and l(x=P + 2) == -3 and l(ws=P + 4) == -3 and l(M=0, ws=None, n=0) == 0
    p = lambda **k: lib.souffle_int8_pack_weight(*{**dict(w=P, ldw=50, p=P, K=100, N=50, st=None), **k}.values())  # noqa: E731
    assert p(w=None) == -1 and p(p=None) == -1 and p(ldw=49) == -2 and p(p=P + 8) == -3 and p(N=0) == -2
    z = lambda **k: lib.souffle_int8_quantize_weight(*{**dict(w=P, t=0, ldw=50, p=P, s=P, K=100, N=50, st=None), **k}.values())  # noqa: E731
    assert z(w=None) == -1 and z(s=None) == -1 and z(t=7) == -2 and z(ldw=49) == -2 and z(w=P + 1) == -3 and z(s=P + 1) == -3


def test_bindings_refuse_cpu_tensors():
    import linear_int8_binding as lb
    w = lb.Int8Weight(torch.zeros(4096, dtype=torch.int8), torch.zeros(8), 8, 8)
    for call in (lambda: lb.linear_int8(torch.zeros(2, 8), w), lambda: lb.quantize_rows(torch.zeros(2, 8)), lambda: lb.quantize_weight(torch.zeros(8, 8)),
                 lambda: lb.gemm_int8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2), w), lambda: lb.pack_weight(torch.zeros(8, 8, dtype=torch.int8), torch.zeros(8))):
        with pytest.raises(TypeError, match="CUDA"):
            call()


def test_overlap_of_rows():
    """Against the sets of bytes themselves.  Rows at one distance whose columns meet count as overlapping wherever the spans do, which
    is more than the bytes say only where one set begins behind the other's last row, or the distances differ."""
    import linear_int8_binding as lb

    def touched(a, rows, width, pitch):
        return {a + r * pitch + c for r in range(rows) for c in range(width)}
    for rows_a, width_a, pitch_a in ((0, 3, 8), (1, 5, 5), (3, 3, 8), (2, 8, 8)):
        for rows_b, width_b, pitch_b in ((1, 2, 2), (1, 20, 20), (3, 4, 8), (3, 3, 8), (2, 3, 7)):
            for b in range(60, 140):
                both = touched(100, rows_a, width_a, pitch_a) & touched(b, rows_b, width_b, pitch_b)
                got = lb._overlap(100, rows_a, width_a, pitch_a, b, rows_b, width_b, pitch_b)
                assert got or not both, (rows_a, width_a, rows_b, width_b, b)
                if got and not both:
                    spans = rows_a and 100 < b + (rows_b - 1) * pitch_b + width_b and b < 100 + (rows_a - 1) * pitch_a + width_a
                    assert spans and (pitch_a != pitch_b or rows_a != rows_b), (rows_a, width_a, rows_b, width_b, b)
    # columns side by side, and one row in the gap between another's rows
    assert not lb._overlap(100, 5, 16, 64, 116, 5, 48, 64) and not lb._overlap(116, 5, 48, 64, 100, 5, 16, 64) and lb._overlap(100, 5, 16, 64, 115, 5, 16, 64)
    assert not lb._overlap(120, 1, 30, 30, 100, 5, 16, 64) and lb._overlap(120, 1, 50, 50, 100, 5, 16, 64)


@gpu
@pytest.mark.parametrize("M", [1, 3, 200])
def test_out_over_an_input_is_refused(M):
    """The product reads all of its inputs while it writes: out over the 8-bit rows, a scale, the bias or the weights."""
    announce("8-bit product: out over an input, M=%d" % M)
    import linear_int8_binding as lb
    w = lb.quantize_weight(values(3, 64, 64).cuda())
    x, b = values(4, M, 64).cuda(), values(5, 64).cuda()
    room = torch.zeros(M * 320, dtype=torch.uint8, device="cuda")
    q = room[:M * 64].view(torch.int8).view(M, 64)
    q0, s = lb.quantize_rows(x)
    q.copy_(q0)
    y = lb.gemm_int8(q, s, w, bias=b, dtype=torch.float32)
    over = lambda at: room[at:at + M * 256].view(torch.float32).view(M, 64)  # noqa: E731
    with pytest.raises(ValueError, match="overlap q"):
        lb.gemm_int8(q, s, w, bias=b, dtype=torch.float32, out=over(0))
    with pytest.raises(ValueError, match="overlap q"):
        lb.gemm_int8(q, s, w, bias=b, dtype=torch.float32, out=over(M * 64 - 4))
    assert torch.equal(lb.gemm_int8(q, s, w, bias=b, dtype=torch.float32, out=over(M * 64)), y)
    out = torch.empty(M, 64, device="cuda")
    inside = out.view(-1)
    packed = torch.empty(4096 + M * 256, dtype=torch.int8, device="cuda")
    packed[:4096] = w.packed
    bad = [("bias", w, inside[:64], out), ("weight.scale", w._replace(scale=inside[-64:]), b, out),
           ("weight.packed", w._replace(packed=packed[:4096]), b, packed[4092:4092 + M * 256].view(torch.float32).view(M, 64))]
    for name, weight, bias, o in bad:
        with pytest.raises(ValueError, match="overlap " + name):
            lb.gemm_int8(q, s, weight, bias=bias, dtype=torch.float32, out=o)
        with pytest.raises(ValueError, match="overlap " + name):
            lb.linear_int8(x, weight, bias=bias, out=o)
    with pytest.raises(ValueError, match="overlap row_scale"):
        lb.gemm_int8(q, inside[:M], w, bias=b, dtype=torch.float32, out=out)
    # inputs between the rows of an output that lie apart are fine
    wide = torch.zeros(M, 192, device="cuda")
    wide[0, 64:128] = b
    assert torch.equal(lb.linear_int8(x, w, bias=wide[0, 64:128], out=wide[:, 128:]), y) and torch.equal(wide[0, 64:128], b)


@gpu
def test_bindings_refuse_wrong_tensors():
    announce("8-bit linear layer: refusals of the bindings")
    import linear_int8_binding as lb
    w = lb.quantize_weight(values(1, 100, 50).cuda())
    x, b = values(2, 4, 100, dtype=torch.float16).cuda(), torch.zeros(50, dtype=torch.float16, device="cuda")
    q, s = lb.quantize_rows(x)
    bad = [
        (TypeError, lambda: lb.linear_int8(x.double(), w)), (ValueError, lambda: lb.linear_int8(x[:, :99], w)),
        (ValueError, lambda: lb.linear_int8(x.t().contiguous().t(), w)), (ValueError, lambda: lb.linear_int8(x, w, act="tanh")),
        (ValueError, lambda: lb.linear_int8(x, w, bias=b.float())), (ValueError, lambda: lb.linear_int8(x, w, bias=b[:49])),
        (ValueError, lambda: lb.linear_int8(x, w, out=torch.empty(4, 51, dtype=torch.float16, device="cuda"))),
        (ValueError, lambda: lb.linear_int8(x, w, out=torch.empty(4, 50, device="cuda"))),
        (ValueError, lambda: lb.linear_int8(x[:1].expand(4, 100), w)),
        (TypeError, lambda: lb.linear_int8(x, (w.packed, w.scale))), (ValueError, lambda: lb.linear_int8(x, w._replace(packed=w.packed[:-1]))),
        (ValueError, lambda: lb.linear_int8(x, w._replace(scale=w.scale[:-1]))), (ValueError, lambda: lb.linear_int8(x, w._replace(scale=w.scale.half()))),
        (ValueError, lambda: lb.gemm_int8(q[:, :99], s, w)), (ValueError, lambda: lb.gemm_int8(q, s[:3], w)), (TypeError, lambda: lb.gemm_int8(q, s, w, dtype=torch.float64)),
        (ValueError, lambda: lb.gemm_int8(q[:, :100].contiguous(), s, w)), (sh.SouffleError, lambda: lb.gemm_int8(q.contiguous().repeat(2, 1)[:4], s, w)),
        (TypeError, lambda: lb.pack_weight(x, s)), (ValueError, lambda: lb.pack_weight(torch.zeros(8, 9, dtype=torch.int8, device="cuda"), s)),
        (TypeError, lambda: lb.quantize_weight(x[0])),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (1, 8), (5, 64), (2, 511), (9, 512), (2, 513), (3, 1001), (2, 2048), (2, 2056), (2, 4097), (3, 8192), (2, 8193), (1, 20000)])
def test_quantize_rows_is_exact(dtype, M, K):
    announce("quantize_rows %s %dx%d" % (dtype, M, K))
    import linear_int8_binding as lb
    x = values(K, M, K + 3, dtype=TYPES[dtype])[:, 1:K + 1]          # rows that start anywhere
    big = x.abs().amax(-1)
    x[:, K // 2] = big / 2                                           # a half, where the type holds it
    x[:, -1] = big
    q, s = lb.quantize_rows(x.cuda())
    rq, rs = ref.quantize(x)
    assert q.shape == (M, K) and torch.equal(s.cpu().double(), rs)
    assert torch.equal(q.cpu().double(), rq)


@gpu
def test_quantize_rows_at_the_borders():
    """Halves of the step on both sides, subnormal rows, zeros, and rows that hold a NaN or an infinity."""
    announce("quantize_rows: halves, tiny rows, non-finite rows")
    import linear_int8_binding as lb
    top = torch.tensor([127.0, 100.0, 1.0, 3.0 ** 20, 2.0 ** -60, 1e-30, 2.0 ** -140, 3e38])
    k = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    scale = (top.double() / 127).float().double().clamp_min(2.0 ** -100)
    half = (k[None, :] * scale[:, None]).float()                     # the fp32 values next to every half
    inf = torch.tensor(float("inf"))
    x = torch.cat([half, torch.nextafter(half, inf), torch.nextafter(half, -inf)], 1).clamp(-top[:, None], top[:, None])
    x = torch.cat([x, top[:, None], torch.zeros(8, 2)], 1)
    q, s = lb.quantize_rows(x.cuda())
    rq, rs = ref.quantize(x)
    assert torch.equal(s.cpu().double(), rs) and torch.equal(q.cpu().double(), rq)
    for t in TYPES.values():
        x = torch.ones(4, 70, dtype=t)
        x[0] = 0
        x[1, 69] = float("nan")
        x[2, 3] = float("-inf")
        q, s = lb.quantize_rows(x.cuda())
        assert s[0].item() == 2.0 ** -100 and torch.isnan(s[1:3]).all() and s[3].item() == np.float32(1) / np.float32(127)
        assert not q[:3].any() and (q[3] == 127).all()


@gpu
@pytest.mark.parametrize("K,N", [(1, 1), (64, 64), (65, 63), (100, 130), (333, 70)])
def test_packed_weights(K, N):
    announce("packed weights %dx%d" % (K, N))
    import linear_int8_binding as lb
    wq, scale = weight(K, K, N)
    for w in (wq, torch.nn.functional.pad(wq, (0, 5))[:, :N]):       # rows apart
        p = lb.pack_weight(w.cuda(), scale.cuda())
        expect = torch.zeros(lb.sh.lib().souffle_int8_packed_bytes(K, N), dtype=torch.int8)
        expect[torch.from_numpy(packed_index(K, N))] = wq
        assert torch.equal(p.packed.cpu(), expect) and torch.equal(p.scale.cpu(), scale)
    for t in TYPES.values():
        w = values(N, K, N, dtype=t)
        p = lb.quantize_weight(w.cuda())
        rq, rs = ref.quantize(w.t())
        expect = torch.zeros_like(p.packed, device="cpu")
        expect[torch.from_numpy(packed_index(K, N))] = rq.t().to(torch.int8)
        assert torch.equal(p.scale.cpu().double(), rs) and torch.equal(p.packed.cpu(), expect)


def run_linear(dtype, M, K, N, act, bias, seed=0, ldx=0, ldy=0):
    """linear_int8 and the two steps apart against 64 bits, with canaries around the output."""
    import linear_int8_binding as lb
    t = TYPES[dtype]
    x = values(seed, M, K + ldx, dtype=t, std=2.0).cuda()[:, :K]
    wq, cs = weight(seed + 1, K, N)
    b = values(seed + 2, N, dtype=t) if bias else None
    w = lb.pack_weight(wq.cuda(), cs.cuda())
    room = torch.full((M + 2, N + ldy), 77.0, dtype=t, device="cuda")
    out = room[1:M + 1, :N]
    y = lb.linear_int8(x, w, bias=None if b is None else b.cuda(), act=act, out=out)
    q, s = lb.quantize_rows(x)
    y2 = lb.gemm_int8(q, s, w, bias=None if b is None else b.cuda(), act=act, dtype=t)
    torch.cuda.synchronize()
    rq, rs = ref.quantize(x.cpu())
    r, bound = ref.linear(rq, rs, wq, cs, b, act)
    ref.check("linear_int8", y, r, bound + ref.half_step(r, t))
    assert torch.equal(y, y2), "the call and its two steps differ"
    assert (room[0] == 77).all() and (room[M + 1] == 77).all() and (room[:, N:] == 77).all(), "written outside the output"


@gpu
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128, 130, 257])
@pytest.mark.parametrize("K,N", [(1, 1), (64, 64), (65, 3), (200, 130), (1000, 65), (1152, 320)])
def test_linear_sizes(M, K, N):
    announce("linear_int8 M=%d K=%d N=%d" % (M, K, N))
    run_linear("f16", M, K, N, None, True, seed=M + K + N)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N,ldx,ldy", [(1, 768, 100, 0, 0), (7, 129, 77, 5, 3), (70, 256, 192, 64, 64), (300, 520, 257, 1, 1)])
def test_linear_types_and_epilogues(dtype, act, M, K, N, ldx, ldy):
    announce("linear_int8 %s act=%s M=%d K=%d N=%d" % (dtype, act, M, K, N))
    run_linear(dtype, M, K, N, act, act != "relu", seed=M, ldx=ldx, ldy=ldy)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 16384, 40), (1, 16385, 40), (2, 4100, 5000), (3, 5461, 20), (4, 4096, 4200), (5, 777, 4101), (8, 2048, 64), (9, 1820, 65), (16, 1024, 300), (16, 1025, 300), (17, 1024, 300), (33, 1024, 4000), (40, 1025, 300), (300, 1017, 1000), (31, 8, 70), (47, 7, 70), (512, 1000, 2040), (513, 1000, 2040)])
def test_linear_few_rows(dtype, M, K, N):
    """Around the size up to which the product's workgroups quantise the rows themselves, for every split of the waves."""
    announce("linear_int8 %s M=%d K=%d N=%d" % (dtype, M, K, N))
    run_linear(dtype, M, K, N, None, True, seed=M + K, ldx=1)


@gpu
@pytest.mark.parametrize("M,K,N", [(1024, 512, 768), (2048, 1024, 1100), (4099, 320, 520), (4099, 1088, 2300), (600, 64, 4096), (1500, 200, 1024), (1100, 4160, 70)])
def test_linear_many_rows(M, K, N):
    announce("linear_int8 M=%d K=%d N=%d" % (M, K, N))
    run_linear("bf16", M, K, N, "gelu_tanh", True, seed=M)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(17, 3, 70), (31, 8, 64), (32, 9, 200), (33, 64, 33), (64, 511, 640), (100, 513, 1000), (250, 1000, 400), (384, 1023, 768),
                                   (47, 1024, 4100), (300, 1025, 300), (640, 520, 832), (672, 520, 832)])
def test_linear_rows_quantised_on_the_way(dtype, M, K, N):
    """Tiles of 32 rows with their last rows missing, up to the longest row that is quantised there and one beyond."""
    run_linear(dtype, M, K, N, "gelu", True, seed=M + K, ldx=K + 5)


@gpu
@pytest.mark.parametrize("M", [1, 40, 4096])
def test_gelu_keeps_its_digits_in_the_tails(M):
    """Rows of zeros, so that the activation's argument is the bias itself.  Up to |v| = 4 the error is relative to the
    result: the exponent, at most 8 log2(e), is rounded twice (9.5e-7 in the power), nine steps of a polynomial, four
    products and two functions of one unit each add 9 + 4 + 4 roundings of 2^-24 and the fit 1e-7: 2.1e-6."""
    import linear_int8_binding as lb
    announce("gelu of %d rows" % M)
    v = torch.cat([torch.linspace(-4, 4, 3000), torch.linspace(-30, 30, 1000), torch.logspace(-30, 30, 400), -torch.logspace(-30, 30, 400),
                   torch.tensor([0.0, float("inf"), float("nan")])])
    w = lb.quantize_weight(torch.ones(64, v.numel(), device="cuda"))
    y = lb.linear_int8(torch.zeros(M, 64, device="cuda"), w, bias=v.cuda(), act="gelu").double().cpu()
    assert torch.equal(y[:, :-1], y[:1, :-1].expand(M, -1))      # (without the NaN)
    y, v = y[0], v.double()
    assert y[-2] == float("inf") and torch.isnan(y[-1]) and y[-3] == 0
    y, v = y[:-3], v[:-3]
    exact = v.clamp_min(0) - 0.5 * v.abs() * torch.special.erfc(v.abs() / 2 ** 0.5)
    error = (y - exact).abs()
    near = v.abs() <= 4
    # (v - w near 0 for positive v: the difference of the two is rounded, half a step of v)
    assert (error[near] <= 2.1e-6 * exact[near].abs() + ref.EPS32 * v[near].clamp_min(0)).all()
    assert (error <= 16 * ref.EPS32 * v.abs()).all()


@gpu
def test_longest_sums_stay_exact():
    """K = 131071 with every factor -128: the sum is 2147467264, 16384 short of what 32 bits hold."""
    announce("gemm_int8 K=131071")
    import linear_int8_binding as lb
    K = 131071
    q = torch.full((2, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = lb.pack_weight(torch.full((K, 2), -128, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"))
    y = lb.gemm_int8(q, torch.ones(2, device="cuda"), w, dtype=torch.float32)
    assert (y == float(np.float32(2147467264))).all()


@gpu
def test_bytes_behind_k_do_not_matter():
    announce("gemm_int8: bytes behind K")
    import linear_int8_binding as lb
    for M in (3, 40, 200):
        wq, cs = weight(5, 70, 40)
        w = lb.pack_weight(wq.cuda(), cs.cuda())
        a = torch.randint(-127, 128, (M, 128), dtype=torch.int8, generator=torch.Generator().manual_seed(M)).cuda()
        s = torch.rand(M, device="cuda")
        y = lb.gemm_int8(a[:, :70], s, w)
        b = a.clone()
        b[:, 70:] = -128
        assert torch.equal(y, lb.gemm_int8(b[:, :70], s, w))


@gpu
def test_non_finite_rows_stay_in_their_rows():
    announce("linear_int8: rows with NaN and infinity")
    import linear_int8_binding as lb
    for M in (8, 48, 300):
        for act in (None, "relu", "gelu", "gelu_tanh"):
            w = lb.quantize_weight(values(3, 96, 80).cuda())
            x = values(4, M, 96, dtype=torch.bfloat16).cuda()
            clean = lb.linear_int8(x, w, act=act)
            x[2, 5], x[5, 95], x[6] = float("nan"), float("inf"), 0
            y = lb.linear_int8(x, w, act=act)
            assert torch.isnan(y[2]).all() and torch.isnan(y[5]).all() and not y[6].any()
            keep = [i for i in range(M) if i not in (2, 5, 6)]
            assert torch.equal(y[keep], clean[keep])


@gpu
def test_empty_and_leading_dimensions():
    announce("linear_int8: no rows, three dimensions")
    import linear_int8_binding as lb
    w = lb.quantize_weight(values(3, 96, 80).cuda())
    assert lb.linear_int8(torch.empty(0, 96, device="cuda"), w).shape == (0, 80)
    q, s = lb.quantize_rows(torch.empty(0, 96, device="cuda"))
    assert q.shape == (0, 96) and s.shape == (0,) and lb.gemm_int8(q, s, w).shape == (0, 80)
    x = values(4, 2, 3, 96).cuda()
    assert torch.equal(lb.linear_int8(x, w), lb.linear_int8(x.view(6, 96), w))
    assert torch.equal(lb.linear_int8(x[0, 0], w), lb.linear_int8(x.view(6, 96)[:1], w))


@gpu
def test_out_beside_x_in_one_buffer_and_never_over_it():
    announce("linear_int8: out and x in one buffer")
    import linear_int8_binding as lb
    for M in (3, 200):
        w = lb.quantize_weight(values(3, 64, 48).cuda())
        buf = values(4, M, 128, dtype=torch.float16).cuda()
        y = lb.linear_int8(buf[:, :64].contiguous(), w)
        for bad in (buf[:, :48], buf[:, 63:111], buf.view(-1)[64 * M:64 * M + 48 * M].view(M, 48)):
            with pytest.raises(ValueError, match="overlap"):
                lb.linear_int8(buf[:, :64], w, out=bad)
        assert lb.linear_int8(buf[:, :64], w, out=buf[:, 80:]) is not None
        assert torch.equal(buf[:, 80:], y)
        big = values(5, 2 * M, 64, dtype=torch.float16).cuda()
        assert torch.equal(lb.linear_int8(big[M:], w, out=big[:M, :48]), lb.linear_int8(big[M:], w))


@gpu
def test_rows_beyond_two_gib():
    """Offsets of a long activation pass 31 bits: rows 70000 apart by 32800 elements."""
    announce("linear_int8: offsets beyond 2^31")
    import linear_int8_binding as lb
    rows, wide, K, N = 70000, 32800, 64, 8
    big = torch.empty((rows, wide), dtype=torch.float16, device="cuda")
    x = big[:, :K]
    src = values(9, rows, K, dtype=torch.float16).cuda()
    x.copy_(src)
    w = lb.quantize_weight(values(3, K, N).cuda())
    assert torch.equal(lb.linear_int8(x, w), lb.linear_int8(src, w))
