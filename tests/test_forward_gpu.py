"""GPU tests of the forward operators on EXL3 tensors against 64-bit values.

The dense weight comes from the oracle's decode (pinned to the reference), in fp64.

Tolerance of one product, per output: with xh = (x suh) B the rotated activations and
V = W_inner B diag(svh), y_j = sum_i xh_i V_ij.  The kernel rounds each xh_i once to
fp16, off by at most 2^-11 |xh_i| (half a step; the block scale keeps fp16 normal), with
a variance of at most a third of that squared; the roundings are independent, so the
error has a standard deviation below 2^-11 / sqrt(3) * s_j, s_j = sqrt(sum_i xh_i^2
V_ij^2), and eight of those are allowed.  The fp32 sums add at most 2^-22 of a partial sum (a few
s_j) for each of the k / 16 steps: k / 16 * 2^-20 * s_j covers them.  The epilogue's
few fp32 operations add 2^-20 of the magnitudes they see, and the result is rounded
once, half a step of its type: eps / 2 of its magnitude.  The activations' slopes are
below 1.13."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CODES = ("exl3_mul1", "exl3_3inst", "exl3_mcg")


@pytest.fixture(scope="module")
def fw():
    from exl3b import forward
    return forward


def _had(blocks):
    h = np.ones((1, 1))
    while h.shape[0] < 128:
        h = np.block([[h, h], [h, -h]])
    return np.kron(np.eye(blocks), h / math.sqrt(128.0))


class Problem:
    """A random EXL3 tensor and its fp64 pieces."""

    def __init__(self, oracle, k, n, K, code="exl3_mul1", seed=0, scale=None):
        rng = np.random.default_rng(seed)
        self.k, self.n, self.K, self.code = k, n, K, code
        tr = rng.integers(-32768, 32768, (k // 16, n // 16, 16 * K)).astype(np.int16)
        std = 1.0 / math.sqrt(k) if scale is None else scale
        sgn = lambda m: rng.choice([-1.0, 1.0], m) * np.exp(0.3 * rng.standard_normal(m))
        self.suh = (sgn(k) * std / 1.24).astype(np.float16)
        self.svh = sgn(n).astype(np.float16)
        self.trellis = tr
        inner = oracle.decode_trellis(tr, oracle.code_lut(code), K, k, n).astype(np.float64)
        self.V = inner @ _had(n // 128) * self.svh.astype(np.float64)[None, :]
        self.B = _had(k // 128)

    def weight(self, fw):
        t = lambda a: torch.from_numpy(a).cuda()
        return fw.TrellisWeight(t(self.trellis), t(self.suh), t(self.svh), self.K, self.code)

    def product(self, x):
        """x (fp64 numpy [M, k]) -> (x W, its tolerance)"""
        xh = (x * self.suh.astype(np.float64)) @ self.B
        s = np.sqrt((xh ** 2) @ (self.V ** 2))
        return xh @ self.V, s * (8 * 2.0 ** -11 / math.sqrt(3) + self.k / 16 * 2.0 ** -20)


def act64(v, act):
    t = torch.from_numpy(v)
    if act == "relu":
        t = t.clamp(min=0)
    elif act == "silu":
        t = t * torch.sigmoid(t)
    elif act == "gelu":
        t = torch.nn.functional.gelu(t)
    elif act == "gelu_tanh":
        t = torch.nn.functional.gelu(t, approximate="tanh")
    return t.numpy()


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def expect(prob, x, bias=None, act=None, mul=None, residual=None):
    """(value, tolerance) of linear in fp64"""
    y, tol = prob.product(f64(x))
    if bias is not None:
        y = y + f64(bias)
    tol = tol + 2.0 ** -20 * np.abs(y)
    y, tol = act64(y, act), tol * (1.13 if act else 1.0)
    if mul is not None:
        y, tol = y * f64(mul), tol * np.abs(f64(mul))
    if residual is not None:
        y = y + f64(residual)
        tol = tol + 2.0 ** -23 * np.abs(f64(residual))
    half = torch.finfo(x.dtype).eps / 2
    return y, tol + half * (np.abs(y) + tol) + torch.finfo(x.dtype).smallest_normal * half


def check(got, want, tol):
    d = np.abs(f64(got) - want)
    bad = ~(d <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(d / tol)), np.argwhere(bad)[:4])


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * scale
    if x.dim() > 1:
        x[..., ::97] *= 15.0                     # a few loud channels
    return x.to(dtype).cuda()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("K", range(2, 8))
def test_linear_codes(fw, oracle, K, code):
    prob = Problem(oracle, 384, 256, K, code, seed=K)
    w = prob.weight(fw)
    for M in (3, 40):
        x = rnd((M, 384), torch.float16, M)
        check(fw.linear(x, w), *expect(prob, x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 65, 128, 129, 223, 225,
                               300, 517])
def test_linear_rows(fw, oracle, M, dtype):
    prob = Problem(oracle, 640, 384, 4, seed=7)
    x = rnd((M, 640), dtype, M)
    check(fw.linear(x, prob.weight(fw)), *expect(prob, x))


@pytest.mark.parametrize("k,n", [(128, 128), (128, 1152), (1152, 128), (4992, 256), (256, 2176),
                                 (17408, 128)])
def test_linear_shapes(fw, oracle, k, n):
    prob = Problem(oracle, k, n, 5, seed=k + n)
    w = prob.weight(fw)
    for M in (1, 11, 70):
        x = rnd((M, k), torch.bfloat16, M)
        check(fw.linear(x, w), *expect(prob, x))


@pytest.mark.parametrize("M", [5, 50])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_linear_epilogue(fw, oracle, act, dtype, M):
    prob = Problem(oracle, 256, 384, 3, seed=3)
    w = prob.weight(fw)
    x, bias = rnd((M, 256), dtype, 1), rnd((384,), dtype, 2)
    mul, res = rnd((M, 384), dtype, 3), rnd((M, 384), dtype, 4)
    for kw in ({}, {"bias": bias}, {"mul": mul}, {"residual": res},
               {"bias": bias, "mul": mul, "residual": res}):
        got = fw.linear(x, w, activation=act, **kw)
        check(got, *expect(prob, x, act=act, **kw))


@pytest.mark.parametrize("M", [3, 40])
@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e30])
def test_linear_range_of_bf16(fw, oracle, scale, M):
    """Activations far outside fp16's range are no matter: blocks are scaled."""
    prob = Problem(oracle, 384, 128, 4, seed=9)
    x = rnd((M, 384), torch.bfloat16, 5, scale)
    x[:, 128:256] *= 1e-3                     # blocks of different magnitude
    x[1] = 0                                  # and a row of zeros
    got = fw.linear(x, prob.weight(fw))
    check(got, *expect(prob, x))
    assert not got[1].any()


@pytest.mark.parametrize("M", [4, 48])
def test_linear_rows_are_independent(fw, oracle, M):
    """A NaN or infinite row spoils itself only; rows do not depend on the batch."""
    prob = Problem(oracle, 512, 256, 6, seed=11)
    w = prob.weight(fw)
    x = rnd((M, 512), torch.bfloat16, 6)
    clean = fw.linear(x, w)
    x[1, 130] = float("inf")
    x[2, 5] = float("nan")
    got = fw.linear(x, w)
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[1]).any() and torch.isnan(got[2]).all()


@pytest.mark.parametrize("M", [6, 60])
def test_linear_layouts(fw, oracle, M):
    prob = Problem(oracle, 256, 128, 4, seed=13)
    w = prob.weight(fw)
    dt = torch.float16
    x, res = rnd((M, 256), dt, 1), rnd((M, 128), dt, 2)
    ref = fw.linear(x, w, residual=res)
    check(ref, *expect(prob, x, residual=res))
    # row pitch, odd offset, transposed storage, expanded rows, leading dimensions
    wide = torch.zeros(M, 520, dtype=dt, device="cuda")
    for off in (0, 4, 3):
        v = wide[:, off:off + 256]
        v.copy_(x)
        assert torch.equal(fw.linear(v, w, residual=res), ref)
    assert torch.equal(fw.linear(x.t().contiguous().t(), w,
                                 residual=res.t().contiguous().t()), ref)
    assert torch.equal(fw.linear(x[:1].expand(M, 256), w), fw.linear(x[:1], w).expand(M, 128))
    assert torch.equal(fw.linear(x.view(2, M // 2, 256), w, residual=res.view(2, M // 2, 128)),
                       ref.view(2, M // 2, 128))
    assert torch.equal(fw.linear(x[0], w), fw.linear(x[:1], w)[0])
    assert fw.linear(x[:0], w).shape == (0, 128)
    # out: a column range of a wider buffer, whose other columns stay
    buf = torch.full((M + 2, 384), 7.0, dtype=dt, device="cuda")
    o = buf[1:M + 1, 128:256]
    assert fw.linear(x, w, residual=res, out=o) is o
    assert torch.equal(o, ref)
    o.fill_(7.0)
    assert bool((buf == 7.0).all())
    # in place on the residual, and on mul
    r2 = res.clone()
    fw.linear(x, w, residual=r2, out=r2)
    assert torch.equal(r2, ref)
    m2 = res.clone()
    fw.linear(x, w, mul=m2, out=m2)
    assert torch.equal(m2, fw.linear(x, w, mul=res))
    with pytest.raises(ValueError, match="overlaps"):
        fw.linear(wide[:, :256], w, out=wide[:, 128:256])


@pytest.mark.parametrize("M", [1, 9, 90, 260])
def test_linear_repeats_and_streams(fw, oracle, M):
    """The same bits every time: on another stream, and from a replayed graph."""
    prob = Problem(oracle, 1280, 512, 5, seed=17)
    w = prob.weight(fw)
    x, res = rnd((M, 1280), torch.bfloat16, 1), rnd((M, 512), torch.bfloat16, 2)
    ref = fw.linear(x, w, residual=res, activation="silu")
    for _ in range(3):
        assert torch.equal(fw.linear(x, w, residual=res, activation="silu"), ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fw.linear(x, w, residual=res, activation="silu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref)
    graphs, outs = [], []
    xs = x.clone()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fw.linear(xs, w, residual=res, activation="silu"))
        graphs.append(g)
    xs.copy_(x.flip(0))
    for g in graphs:
        g.replay()
    want = fw.linear(xs, w, residual=res, activation="silu")
    assert all(torch.equal(o, want) for o in outs)


def test_linear_refuses_gradients_and_devices(fw, oracle):
    prob = Problem(oracle, 128, 128, 4)
    w = prob.weight(fw)
    x = rnd((2, 128), torch.bfloat16, 1).requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        fw.linear(x, w)
    with torch.no_grad():
        assert not fw.linear(x, w).requires_grad
    with pytest.raises(ValueError, match="is on"):
        fw.linear(x.detach().cpu(), w)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("M,k,n,K", [(768, 128, 128, 2), (769, 256, 384, 3), (1100, 640, 256, 4),
                                     (2050, 128, 640, 5), (1280, 1152, 128, 6), (900, 384, 256, 7)])
def test_linear_long(fw, oracle, M, k, n, K, code):
    prob = Problem(oracle, k, n, K, code, seed=M)
    w = prob.weight(fw)
    dt = torch.float16 if K % 2 else torch.bfloat16
    x, bias = rnd((M, k), dt, 1), rnd((n,), dt, 2)
    x[5] = 0
    x[7] *= 1e-4
    mul, res = rnd((M, n), dt, 3), rnd((M, n), dt, 4)
    check(fw.linear(x, w), *expect(prob, x))
    kw = {"bias": bias, "mul": mul, "residual": res}
    ref = fw.linear(x, w, activation="silu", **kw)
    check(ref, *expect(prob, x, act="silu", **kw))
    # rows on 8-byte boundaries only, and in place on the residual
    buf = torch.zeros(M, n + 4, dtype=dt, device="cuda")
    o = buf[:, 4:]
    o.copy_(res)
    fw.linear(x, w, bias=bias, activation="silu", mul=mul, residual=o, out=o)
    assert torch.equal(o, ref)
    assert not buf[:, :4].any()
    x[9, 3] = float("nan")
    got = fw.linear(x, w, activation="silu", **kw)
    assert torch.isnan(got[9]).all()
    keep = [i for i in range(M) if i != 9]
    assert torch.equal(got[keep], ref[keep])


def test_linear_long_graphs(fw, oracle):
    prob = Problem(oracle, 256, 384, 4, seed=21)
    w = prob.weight(fw)
    x = rnd((1000, 256), torch.bfloat16, 1)
    ref = fw.linear(x, w)
    outs, graphs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fw.linear(x, w))
        graphs.append(g)
    for _ in range(2):
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
            assert torch.equal(o, ref)


@pytest.mark.parametrize("channel_scales", [False, True])
def test_linear_of_a_quantized_layer(fw, tmp_path, channel_scales):
    """quantize_linear_fused -> stored fields -> linear: the forward product equals
    x W_hat^T of the quantizer's own W_hat, from the result and from the files."""
    from exl3b import api, export
    g = torch.Generator().manual_seed(0)
    W = torch.randn(256, 128, generator=g) * 0.05
    r = api.quantize_linear(W, torch.eye(128), K=4, channel_scales=channel_scales,
                            out_device="cuda")
    x = rnd((5, 128), torch.float16, 3)
    w = fw.TrellisWeight.from_result(r)
    got = fw.linear(x, w)
    ref = x.double() @ r["W_hat"].double().t()
    # suh is stored in fp16 (its scale folded in): 2^-11 of each weight, the
    # operand's and the result's rounding as much again each
    scale = (x.double() ** 2 @ r["W_hat"].double().t() ** 2).sqrt()
    assert bool(((got.double() - ref).abs() <= 3 * 8 * 2.0 ** -11 * scale + 2.0 ** -11 * ref.abs()).all())
    path = export.save_quantized(tmp_path, 0, "mlp.up_proj", r)
    assert torch.equal(fw.linear(x, fw.TrellisWeight.load(path)), got)


# ------------------------------------------------------------------ mixture of experts
class Layer:
    """Random experts, each tensor at its own K."""

    def __init__(self, oracle, fw, D, F, E, Ks, code="exl3_mul1", seed=0):
        self.D, self.F, self.E = D, F, E
        K = lambda i: Ks[i % len(Ks)]
        self.gate = [Problem(oracle, D, F, K(3 * e), code, 1000 * seed + 3 * e) for e in range(E)]
        self.up = [Problem(oracle, D, F, K(3 * e + 1), code, 1000 * seed + 3 * e + 1) for e in range(E)]
        self.down = [Problem(oracle, F, D, K(3 * e + 2), code, 1000 * seed + 3 * e + 2)
                     for e in range(E)]
        self.experts = fw.TrellisExperts(*([p.weight(fw) for p in ps]
                                           for ps in (self.gate, self.up, self.down)))

    def expect(self, x, router, top_k, normalize=True, residual=None):
        """(value, tolerance) in fp64.  The tolerance of h = silu(g) u follows from
        those of g and u; its errors (each eight deviations, nearly uncorrelated
        over F) reach the output through the down weights as the root of the sum
        of squares, with half as much again for what correlation there is."""
        X, R = f64(x), f64(router)
        logits = X @ R.T
        T = X.shape[0]
        y, tol = np.zeros((T, self.D)), np.zeros((T, self.D))
        for t in range(T):
            order = sorted(range(self.E), key=lambda e: (-logits[t, e], e))[:top_k]
            p = np.exp(logits[t] - logits[t].max())
            p /= p.sum()
            total = p[order].sum() if normalize else 1.0
            for e in order:
                xt = X[t:t + 1]
                g, tg = self.gate[e].product(xt)
                u, tu = self.up[e].product(xt)
                s = act64(g, "silu")
                h = s * u
                th = 1.1 * tg * (np.abs(u) + tu) + np.abs(s) * tu + 2.0 ** -20 * np.abs(h)
                d = self.down[e]
                v, tv = d.product(h)
                W = (d.suh.astype(np.float64)[:, None] * (d.B @ d.V))
                tv = tv + 1.5 * np.sqrt(th ** 2 @ W ** 2)
                y[t] += p[e] / total * v[0]
                tol[t] += p[e] / total * tv[0]
        tol += 2.0 ** -20 * np.abs(y)
        if residual is not None:
            y = y + f64(residual)
        half = torch.finfo(x.dtype).eps / 2
        return y, tol + half * (np.abs(y) + tol) + torch.finfo(x.dtype).smallest_normal


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D,F,E,top_k,code", [
    (1, 128, 128, 4, 1, "exl3_mul1"), (1, 384, 256, 6, 6, "exl3_mcg"),
    (2, 256, 128, 40, 8, "exl3_3inst"), (7, 640, 384, 5, 2, "exl3_mul1"),
    (9, 256, 640, 9, 3, "exl3_mul1"), (40, 256, 128, 2, 1, "exl3_mul1"),
    (70, 384, 256, 3, 3, "exl3_mcg"), (33, 256, 256, 1, 1, "exl3_mul1")])
def test_moe_values(fw, oracle, T, D, F, E, top_k, code, dtype):
    layer = Layer(oracle, fw, D, F, E, [4, 7, 2, 5, 3, 6, 4], code, seed=T)
    x = rnd((T, D), dtype, T)
    router = (rnd((E, D), torch.float32, 99) / math.sqrt(D)).to(dtype)
    res = rnd((T, D), dtype, 5)
    for kw in ({}, {"normalize": False}, {"residual": res}):
        check(fw.moe(x, router, layer.experts, top_k, **kw),
              *layer.expect(x, router, top_k, **kw))
    r32 = router.float() * 1.01
    check(fw.moe(x, r32, layer.experts, top_k), *layer.expect(x, r32, top_k))


def test_moe_ties_take_the_lowest_index(fw, oracle):
    layer = Layer(oracle, fw, 256, 128, 6, [4], seed=3)
    x = rnd((3, 256), torch.float16, 1)
    router = rnd((6, 256), torch.float16, 2) / 16
    router[4] = router[1]
    router[5] = router[1]
    check(fw.moe(x, router, layer.experts, 3), *layer.expect(x, router, 3))
    zero = torch.zeros_like(router)                       # all equal: experts 0 and 1
    check(fw.moe(x, zero, layer.experts, 2), *layer.expect(x, zero, 2))


def test_moe_many_experts_and_long_inputs(fw, oracle):
    """1024 experts; more than 256 tokens are cut."""
    layer = Layer(oracle, fw, 128, 128, 8, [4], seed=4)
    gate, up, down = layer.experts.weights
    many = fw.TrellisExperts(*([ws[e % 8] for e in range(1024)] for ws in (gate, up, down)))
    x = rnd((5, 128), torch.bfloat16, 1)
    router = torch.full((1024, 128), 0.0, dtype=torch.bfloat16, device="cuda")
    pick = [1023, 31, 512, 704, 64]
    for t, e in enumerate(pick):
        router[e] = x[t] * 0.25
    got = fw.moe(x, router, many, 1)
    # the loud channels make some token prefer another token's expert
    for t, e in enumerate((f64(x) @ f64(router).T).argmax(axis=1)):
        one = torch.zeros(8, 128, dtype=torch.bfloat16, device="cuda")
        one[e % 8] = x[t]
        want, tol = layer.expect(x[t:t + 1], one, 1)
        check(got[t:t + 1], want, tol)
    # each token its own expert: one-hot tokens and router rows
    x = torch.zeros(5, 128, dtype=torch.bfloat16, device="cuda")
    router.zero_()
    for t, e in enumerate(pick):
        x[t, 9 * t] = router[e, 9 * t] = 2.0
    got = fw.moe(x, router, many, 1)
    for t, e in enumerate(pick):
        one = torch.zeros(8, 128, dtype=torch.bfloat16, device="cuda")
        one[e % 8] = x[t]
        check(got[t:t + 1], *layer.expect(x[t:t + 1], one, 1))
    x = rnd((517, 128), torch.bfloat16, 2)
    r = rnd((8, 128), torch.float32, 3) / 12
    got = fw.moe(x, r, layer.experts, 2, residual=x)
    check(got[200:300], *layer.expect(x[200:300], r, 2, residual=x[200:300]))
    check(got[500:], *layer.expect(x[500:], r, 2, residual=x[500:]))


def test_moe_rows_are_independent(fw, oracle):
    layer = Layer(oracle, fw, 256, 128, 4, [4], seed=5)
    x = rnd((12, 256), torch.bfloat16, 1)
    router = rnd((4, 256), torch.bfloat16, 2) / 16
    clean = fw.moe(x, router, layer.experts, 2)
    x[3, 7] = float("nan")
    x[8, 200] = float("inf")
    got = fw.moe(x, router, layer.experts, 2)
    keep = [i for i in range(12) if i not in (3, 8)]
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[8]).any()
    # a router row that is NaN or infinite spoils the softmax, and nothing else
    router[2, 0] = float("nan")
    assert torch.isnan(fw.moe(x[:1], router, layer.experts, 2)).all()
    assert not fw.moe(torch.zeros_like(x[:2]), router.nan_to_num(), layer.experts, 2).any()


def test_moe_layouts_graphs_and_streams(fw, oracle):
    layer = Layer(oracle, fw, 384, 256, 5, [3, 5], seed=6)
    x, res = rnd((6, 384), torch.bfloat16, 1), rnd((6, 384), torch.bfloat16, 2)
    router = rnd((5, 384), torch.bfloat16, 3) / 20
    call = lambda x, **kw: fw.moe(x, router, layer.experts, 2, **kw)
    ref = call(x, residual=res)
    for _ in range(3):
        assert torch.equal(call(x, residual=res), ref)
    wide = torch.zeros(6, 900, dtype=torch.bfloat16, device="cuda")
    for off in (0, 8, 4, 1):
        v = wide[:, off:off + 384]
        v.copy_(x)
        assert torch.equal(call(v, residual=res), ref)
    assert torch.equal(call(x.view(2, 3, 384), residual=res.view(2, 3, 384)), ref.view(2, 3, 384))
    assert call(x[:0]).shape == (0, 384)
    assert torch.equal(fw.moe(x, router.t().contiguous().t(), layer.experts, 2, residual=res), ref)
    r2 = res.clone()
    assert call(x, residual=r2, out=r2) is r2 and torch.equal(r2, ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(x, residual=res)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref)
    xs, graphs, outs = x.clone(), [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(xs, residual=res))
        graphs.append(g)
    xs.copy_(x.flip(0))
    for _ in range(2):
        for g in graphs:
            g.replay()
    want = call(xs, residual=res)
    assert all(torch.equal(o, want) for o in outs)


def test_block_of_quantized_layers(fw):
    """Quantized gate, up and down as a user runs them: a dense gated block with its
    residual, then the same tensors as a one-expert layer."""
    from exl3b import api
    g = torch.Generator().manual_seed(1)
    D, F = 256, 384
    mk = lambda o, i, K: fw.TrellisWeight.from_result(api.quantize_linear(
        torch.randn(o, i, generator=g) / math.sqrt(i), None, K=K, out_device="cuda"))
    gate, up, down = mk(F, D, 4), mk(F, D, 5), mk(D, F, 6)
    x = rnd((4, D), torch.float16, 1)
    h = fw.linear(x, gate, activation="silu", mul=fw.linear(x, up))
    y = fw.linear(h, down, residual=x)
    z = fw.moe(x, torch.zeros(1, D, dtype=torch.float16, device="cuda"),
               fw.TrellisExperts([gate], [up], [down]), 1, residual=x)
    # the dense path rounds up(x) and h to fp16 (2^-11 of each) and the moe path
    # rotates and rounds h itself; both sum the same 384 products of down
    scale = (h.double().abs() @ torch.ones(F, 1, dtype=torch.float64, device="cuda")) / math.sqrt(F)
    assert bool(((y.double() - z.double()).abs()
                 <= 2.0 ** -10 * (z.double().abs() + 4 * scale)).all())

@pytest.mark.parametrize("T,E,top_k", [(64, 4, 2), (64, 16, 2)])
def test_moe_fp16_keeps_its_precision(fw, oracle, T, E, top_k):
    """With fp16 tensors the operands of the products hold 22 bits, so that all which
    is lost is the rounding of the result.  That is uniform within half a step, at most
    2^-11 of the value: 2^-11 / sqrt(3) of it as a root of mean squares, and 2% more for
    the operands (2^-22 each), the fp32 sums (2^-20) and the spread of 32768 values."""
    layer = Layer(oracle, fw, 512, 256, E, [4, 6], seed=40 + E)
    x, router = rnd((T, 512), torch.float16, 1), rnd((E, 512), torch.float16, 2) / 60
    want, _ = layer.expect(x, router, top_k)
    d = f64(fw.moe(x, router, layer.experts, top_k)) - want
    assert np.sqrt((d ** 2).sum() / (want ** 2).sum()) <= 1.02 * 2.0 ** -11 / math.sqrt(3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,top_k", [(256, 1024, 8), (64, 1024, 32), (256, 9, 8), (255, 3, 3)])
def test_moe_largest_calls(fw, oracle, T, E, top_k, dtype):
    """All tokens and choices that one call takes, at the widest tensors, with the
    experts spread or crowded: every row equals the row computed by itself, and some
    are checked by value."""
    layer = Layer(oracle, fw, 256, 128, min(E, 12), [7], seed=50 + E)
    many = fw.TrellisExperts(*([ws[e % 12] for e in range(E)] for ws in layer.experts.weights))
    x = rnd((T, 256), dtype, 1)
    router = rnd((E, 256), torch.float32, 2) / 30
    got = fw.moe(x, router, many, top_k)
    for t in (0, 1, T // 2, T - 1):
        one = fw.moe(x[t:t + 1], router, many, top_k)
        half = torch.finfo(dtype).eps / 2
        # the same products in another order of fp32 sums: a step of the result at most
        assert bool(((one - got[t:t + 1]).abs().double()
                     <= 2 * half * got[t:t + 1].abs().double() + 2.0 ** -16 * x[t].abs().max().double()).all())
    if E <= 12:
        check(got[:8], *layer.expect(x[:8], router, top_k))


def test_calls_on_two_streams_at_once(fw, oracle):
    """Two streams work on the same weights and inputs at the same time, each call with
    its own workspace; what they give is what one stream gives."""
    prob = Problem(oracle, 1280, 1024, 4, seed=60)
    w = prob.weight(fw)
    layer = Layer(oracle, fw, 512, 256, 6, [4], seed=61)
    xs = [rnd((M, 1280), torch.bfloat16, M) for M in (1, 6, 40, 300, 1000)]
    xm, router = rnd((9, 512), torch.bfloat16, 1), rnd((6, 512), torch.bfloat16, 2) / 20
    calls = [lambda x=x: fw.linear(x, w, activation="silu") for x in xs]
    calls.append(lambda: fw.moe(xm, router, layer.experts, 2))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(10):
        for i in range(len(calls)):
            for s, j in zip(streams, (i, len(calls) - 1 - i)):
                with torch.cuda.stream(s):
                    outs.append((j, calls[j]()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[j]) for j, o in outs)


def test_first_call_of_a_kernel_may_be_captured(fw, oracle):
    """No eager call before: what a kernel needs set up once is no work on a stream."""
    prob = Problem(oracle, 256, 128, 3, "exl3_mcg", seed=70)
    w = prob.weight(fw)
    cases = [rnd((M, 256), torch.float16, M) for M in (1, 12, 33, 800)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [fw.linear(x, w, activation="gelu") for x in cases]
    g.replay()
    for x, o in zip(cases, outs):
        check(o, *expect(prob, x, act="gelu"))


def test_out_must_not_overlap_what_is_read_whole(fw, oracle):
    prob = Problem(oracle, 128, 128, 4, seed=71)
    w = prob.weight(fw)
    buf = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlaps bias"):
        fw.linear(rnd((2, 128), torch.bfloat16, 1), w, bias=buf[1], out=buf[:2])
    fw.linear(rnd((2, 128), torch.bfloat16, 1), w, bias=buf[0], out=buf[1:3])
    layer = Layer(oracle, fw, 128, 128, 2, [4], seed=72)
    with pytest.raises(ValueError, match="overlaps router"):
        fw.moe(rnd((2, 128), torch.bfloat16, 1), buf[:2], layer.experts, 1, out=buf[1:3])


def test_copies_of_weights_have_their_own_tensors(fw, oracle):
    """deepcopy and pickle give weights that no longer need the original's memory."""
    import copy
    import gc
    import pickle
    prob = Problem(oracle, 256, 128, 4, seed=80)
    w = prob.weight(fw)
    layer = Layer(oracle, fw, 128, 128, 3, [4, 5], seed=81)
    x, xm = rnd((3, 256), torch.bfloat16, 1), rnd((3, 128), torch.bfloat16, 2)
    router = rnd((3, 128), torch.bfloat16, 3) / 12
    ref, mref = fw.linear(x, w), fw.moe(xm, router, layer.experts, 2)
    copies = [copy.deepcopy(w), pickle.loads(pickle.dumps(w))]
    many = [copy.deepcopy(layer.experts), pickle.loads(pickle.dumps(layer.experts))]
    old = {w.trellis.data_ptr(), *(e.trellis.data_ptr() for e in layer.experts.weights[0])}
    for c in copies + [e for m in many for e in m.weights[0]]:
        assert c.trellis.data_ptr() not in old
    for t in (w.trellis, *(e.trellis for ws in layer.experts.weights for e in ws)):
        t.zero_()                       # what a copy must not read
    del w, layer.experts
    gc.collect()
    assert all(torch.equal(fw.linear(x, c), ref) for c in copies)
    assert all(torch.equal(fw.moe(xm, router, m, 2), mref) for m in many)
    with pytest.raises(AttributeError):
        copies[0].trellis = copies[1].trellis
    with pytest.raises(TypeError):
        fw.moe(xm, router, many[0], 2.5)
    o = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        fw.linear(x, copies[0], out=o)


@pytest.mark.parametrize("M,k", [(1, 512), (2, 2048), (5, 512), (13, 640), (37, 512), (150, 384), (300, 256)])
def test_linear_fp16_keeps_its_precision(fw, oracle, M, k):
    """As test_moe_fp16_keeps_its_precision: the rounding of the result is all there is,
    with loud channels too, whose blocks round alike in all their places."""
    prob = Problem(oracle, k, 384, 4, seed=90 + M)
    w = prob.weight(fw)
    num = den = 0.0
    for i in range(1 + 60 // M):
        x = rnd((M, k), torch.float16, i)
        x[:, ::128] *= 40.0
        want = prob.product(f64(x))[0]
        num += ((f64(fw.linear(x, w)) - want) ** 2).sum()
        den += (want ** 2).sum()
    assert np.sqrt(num / den) <= 1.02 * 2.0 ** -11 / math.sqrt(3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_on_8_byte_boundaries(fw, oracle, dtype):
    """suh and svh may start 4 elements into a buffer, which is what the C header asks
    of them; such fields are taken as they are and give the same bits."""
    def shifted(t):
        v = torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")
        at = (8 - v.data_ptr() % 16) // 2 % 8
        v = v[at:at + t.numel()]
        v.copy_(t)
        assert v.data_ptr() % 16 == 8
        return v

    def move(w):
        m = fw.TrellisWeight(w.trellis, shifted(w.suh), shifted(w.svh), w.K, w.code)
        assert m.suh.data_ptr() % 8 == 0 and m.svh.data_ptr() % 8 == 0
        return m

    layer = Layer(oracle, fw, 384, 256, 5, [3, 5], seed=92)
    moved = fw.TrellisExperts(*([move(w) for w in ws] for ws in layer.experts.weights))
    router = rnd((5, 384), dtype, 3) / 20
    for T in (1, 6, 40):
        x = rnd((T, 384), dtype, T)
        got = fw.moe(x, router, moved, 2)
        assert torch.equal(got, fw.moe(x, router, layer.experts, 2))
        check(got, *layer.expect(x, router, 2))
    prob = Problem(oracle, 256, 384, 4, seed=93)
    w = prob.weight(fw)
    for M in (1, 12, 40, 2600):
        x = rnd((M, 256), dtype, M)
        assert torch.equal(fw.linear(x, move(w)), fw.linear(x, w))


@pytest.mark.parametrize("T,E,top_k", [(1, 5, 3), (1, 6, 6), (1, 7, 1), (9, 11, 4), (40, 13, 7),
                                       (200, 3, 2)])
def test_moe_odd_numbers_of_experts(fw, oracle, T, E, top_k):
    """The plan's byte counts ([choices / 32][experts]) end inside a word of the shared
    memory that is cleared for them."""
    assert (T * top_k + 31) // 32 * E % 4
    layer = Layer(oracle, fw, 128, 128, E, [4], seed=94)
    x = rnd((T, 128), torch.bfloat16, 1)
    router = rnd((E, 128), torch.float32, 2) / 12
    check(fw.moe(x, router, layer.experts, top_k), *layer.expect(x, router, top_k))


# ------------------------------------------------------------------ long prompts
# Rows and sizes at which the decoded copy is multiplied, by a margin of two in the
# estimates.  5000 x 1280 x 4480: 20 chunks of k pass through the ring of five stages,
# 20 x 18 tiles of 256 x 256 over the pairs of CTAs give each four or five, and neither
# the rows nor the columns end on a tile.
LONG = (5000, 1280, 4480)


def product_of(M, k, n, dtype):
    from exl3b import forward, native
    return native.lib().exl3b_linear_product(M, k, n, forward.DTYPE_IDS[dtype])


def expect_on_gpu(prob, x, bias=None, act=None, mul=None, residual=None):
    """expect() in fp64 on the device, for many rows"""
    c = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    d = lambda t: t.double()
    V, B, suh = c(prob.V), c(_had(1)), c(prob.suh.astype(np.float64))
    xh = ((d(x) * suh).view(-1, prob.k // 128, 128) @ B).reshape(-1, prob.k)
    y, tol = xh @ V, ((xh ** 2) @ (V ** 2)).sqrt() * (8 * 2.0 ** -11 / math.sqrt(3)
                                                     + prob.k / 16 * 2.0 ** -20)
    if bias is not None:
        y = y + d(bias)
    tol = tol + 2.0 ** -20 * y.abs()
    if act:
        y, tol = {"silu": lambda t: t * torch.sigmoid(t),
                  "gelu": torch.nn.functional.gelu}[act](y), tol * 1.13
    if mul is not None:
        y, tol = y * d(mul), tol * d(mul).abs()
    if residual is not None:
        y = y + d(residual)
        tol = tol + 2.0 ** -23 * d(residual).abs()
    half = torch.finfo(x.dtype).eps / 2
    return y, tol + half * (y.abs() + tol) + torch.finfo(x.dtype).smallest_normal * half


def check_on_gpu(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()),
                           bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,code", [(2, "exl3_mul1"), (3, "exl3_mcg"), (4, "exl3_3inst"),
                                    (5, "exl3_mul1"), (6, "exl3_mcg"), (7, "exl3_3inst")])
def test_long_prompt(fw, oracle, K, code, dtype):
    M, k, n = LONG
    assert product_of(M, k, n, dtype) == 3
    prob = Problem(oracle, k, n, K, code, seed=100 + K)
    w = prob.weight(fw)
    x, bias = rnd((M, k), dtype, 1), rnd((n,), dtype, 2)
    x[5] = 0
    x[300] *= 1e-3
    mul, res = rnd((M, n), dtype, 3), rnd((M, n), dtype, 4)
    check_on_gpu(fw.linear(x, w), *expect_on_gpu(prob, x))
    kw = {"bias": bias, "mul": mul, "residual": res}
    act = "silu" if K % 2 else "gelu"
    ref = fw.linear(x, w, activation=act, **kw)
    check_on_gpu(ref, *expect_on_gpu(prob, x, act=act, **kw))
    # a column range of a wider buffer, in place on the residual; other columns stay
    buf = torch.zeros(M, n + 8, dtype=dtype, device="cuda")
    o = buf[:, 4:-4]
    o.copy_(res)
    fw.linear(x, w, bias=bias, activation=act, mul=mul, residual=o, out=o)
    assert torch.equal(o, ref) and not buf[:, :4].any() and not buf[:, -4:].any()
    x[9, 3], x[4999, 1000] = float("nan"), float("inf")
    got = fw.linear(x, w, activation=act, **kw)
    assert torch.isnan(got[9]).all() and not torch.isfinite(got[4999]).any()
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[[9, 4999]] = False
    assert torch.equal(got[keep], ref[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_prompt_captured_first_then_on_two_streams(fw, oracle, dtype):
    M, k, n = LONG
    prob = Problem(oracle, k, n, 4, "exl3_mcg", seed=110)
    w = prob.weight(fw)
    xs = [rnd((m, k), dtype, m) for m in (M, M - 300)]
    assert all(product_of(len(x), k, n, dtype) == 3 for x in xs)
    outs, graphs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fw.linear(x, w, activation="silu"))
        graphs.append(g)
    for g in graphs:
        g.replay()
    for x, o in zip(xs, outs):
        check_on_gpu(o, *expect_on_gpu(prob, x, act="silu"))
    want = [o.clone() for o in outs]
    for x in xs:                         # the graphs read their inputs anew
        x.copy_(x.flip(0))
    for g in graphs:
        g.replay()
    assert all(torch.equal(o, v.flip(0)) for o, v in zip(outs, want))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(6):
        for s, j in zip(streams, (i % 2, 1 - i % 2)):
            with torch.cuda.stream(s):
                got.append((j, fw.linear(xs[j], w, activation="silu")))
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[j]) for j, o in got)


@pytest.mark.parametrize("M,k,n", [(9000, 256, 4480), (9001, 4992, 1152)])
def test_long_prompt_other_shapes(fw, oracle, M, k, n):
    """Fewer chunks than stages; a long k, whose rows are read twice by their rotation."""
    prob = Problem(oracle, k, n, 5, seed=120)
    w = prob.weight(fw)
    for dtype in (torch.bfloat16, torch.float16):
        assert product_of(M, k, n, dtype) == 3
        x = rnd((M, k), dtype, 1)
        check_on_gpu(fw.linear(x, w), *expect_on_gpu(prob, x))


def test_products_by_rows(fw):
    for dtype in (torch.bfloat16, torch.float16):
        assert [product_of(M, 5120, 5120, dtype) for M in (1, 16, 17, 100, 8192)] == [1, 1, 2, 2, 3]


# ------------------------------------------------------------------ bounded waits
@pytest.fixture
def wait_limit():
    """Sets the limit of device-side waits, in ms; the default returns after the test."""
    from exl3b import native
    yield lambda ms: native.call("exl3b_set_wait_limit_ms", float(ms))
    native.call("exl3b_set_wait_limit_ms", 0.0)


@pytest.mark.parametrize("M,k,n,product", [(64, 1280, 512, 2), (*LONG, 3)])
def test_waits_that_run_out_are_told(fw, oracle, wait_limit, M, k, n, product):
    """With a limit of a nanosecond the first wait for a piece that is not there yet runs
    out: the kernel drains what is in flight and ends, the error is told once, and the
    device goes on working.  Nothing is broken for it; the limit alone is short."""
    from exl3b.native import Exl3bError
    prob = Problem(oracle, k, n, 4, seed=130)
    w = prob.weight(fw)
    x = rnd((M, k), torch.bfloat16, 1)
    assert product_of(M, k, n, x.dtype) == product
    layer = Layer(oracle, fw, 128, 128, 2, [4], seed=131)
    xm, router = rnd((1, 128), torch.bfloat16, 2), rnd((2, 128), torch.bfloat16, 3)
    ref, mref = fw.linear(x, w), fw.moe(xm, router, layer.experts, 1)
    fw.check_waits()
    told = [lambda: fw.linear(x, w), lambda: fw.moe(xm, router, layer.experts, 1), fw.check_waits]
    for tell in told:
        torch.cuda.synchronize()
        wait_limit(1e-6)
        fw.linear(x, w)
        torch.cuda.synchronize()
        wait_limit(0)
        with pytest.raises(Exl3bError, match="ran out") as e:
            tell()
        assert e.value.rc == 4
        fw.check_waits()
        assert torch.equal(fw.linear(x, w), ref)
        assert torch.equal(fw.moe(xm, router, layer.experts, 1), mref)
    # a graph keeps the limit that it was captured with, and is asked about afterwards
    wait_limit(1e-6)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fw.linear(x, w)
    wait_limit(0)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        with pytest.raises(Exl3bError, match="ran out"):
            fw.check_waits()
    assert torch.equal(fw.linear(x, w), ref)


@pytest.mark.parametrize("M,k,n,ms,product", [(100, 32768, 131072, 0.15, 2),
                                              (16384, 8192, 16384, 0.5, 3)])
def test_products_longer_than_the_limit_of_a_wait(fw, wait_limit, M, k, n, ms, product):
    """The limit is one of a handover, not of a whole product: ones that run for several
    times the limit are right (the decoding product some 0.8 ms, the GEMM 3 ms)."""
    assert product_of(M, k, n, torch.bfloat16) == product
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    tr = torch.randint(-32768, 32768, (k // 16, n // 16, 64), generator=g, device="cuda",
                       dtype=torch.int16)
    w = fw.TrellisWeight(tr, r(k).half() / math.sqrt(k), r(n).half(), 4)
    x = r(M, k).bfloat16()
    ref = fw.linear(x, w)
    torch.cuda.synchronize()
    fw.check_waits()
    wait_limit(ms)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    got = fw.linear(x, w)
    b.record()
    torch.cuda.synchronize()
    fw.check_waits()
    assert a.elapsed_time(b) > 3 * ms
    assert torch.equal(got, ref)


@pytest.mark.parametrize("M,k,n", [(160, 2048, 8192), (320, 2560, 2560), (700, 640, 1920), LONG])
def test_fp16_precision_does_not_hang_on_the_rows(fw, oracle, M, k, n):
    """From prompts of some hundred rows on, as test_linear_fp16_keeps_its_precision below
    them: the error is that of rounding the exact values to fp16, and at most 2% more as
    a root of mean squares (operands of 22 bits and fp32 sums add less than 2^-18 of the
    magnitudes that are summed, in quadrature)."""
    rng = np.random.default_rng(140)
    tr = rng.integers(-32768, 32768, (k // 16, n // 16, 64)).astype(np.int16)
    suh = (rng.standard_normal(k) / math.sqrt(k)).astype(np.float16)
    svh = rng.choice([-1.0, 1.0], n).astype(np.float16)
    c = lambda a: torch.from_numpy(a).cuda()
    w = fw.TrellisWeight(c(tr), c(suh), c(svh), 4, "exl3_mcg")
    inner = c(oracle.decode_trellis(tr, oracle.code_lut("exl3_mcg"), 4, k, n)).double()
    B = c(_had(1))
    V = (inner.view(k, n // 128, 128) @ B).view(k, n) * c(svh).double()
    x = rnd((M, k), torch.float16, 1)
    x[:, ::128] *= 40.0
    want = ((x.double() * c(suh).double()).view(M, k // 128, 128) @ B).view(M, k) @ V
    rms = lambda t: float((t.double() - want).square().mean().sqrt())
    assert rms(fw.linear(x, w)) <= 1.02 * rms(want.half())


@pytest.mark.parametrize("k,n,dtype,decoding,copying", [
    # rows at which one product took at least 5% less time than the other
    (5120, 5120, torch.bfloat16, (96, 400, 512, 1024), (768, 1300, 2048, 4096)),
    (5120, 5120, torch.float16, (256, 400), (768, 1300, 4096)),
    (5120, 17408, torch.bfloat16, (256, 400, 512), (768, 1024, 4096)),
    (5120, 17408, torch.float16, (160, 256), (512, 768, 4096)),
    (17408, 5120, torch.bfloat16, (400, 768, 1024), (1536, 2048, 4096)),
    (17408, 5120, torch.float16, (400, 512, 1024), (768, 1300, 4096)),
    (5120, 1024, torch.bfloat16, (1024, 2048), (3000, 4096)),
    (5120, 1024, torch.float16, (1024, 2048), (3000, 4096)),
    (2048, 8192, torch.bfloat16, (96, 256), (512, 768, 2048)),
    (2048, 8192, torch.float16, (160, 256), (400, 512, 1300)),
    (128, 17408, torch.bfloat16, (96, 160), (512, 1024)),
    (128, 17408, torch.float16, (64,), (256, 400)),
    (2048, 768, torch.bfloat16, (512, 2048), (4096,)),
])
def test_the_faster_product_is_taken(fw, k, n, dtype, decoding, copying):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("measured on 148 SMs")
    assert [product_of(M, k, n, dtype) for M in (*decoding, *copying)] \
        == [2] * len(decoding) + [3] * len(copying)
