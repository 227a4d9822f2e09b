"""CPU-side checks of the forward operators: the C ABI refuses bad requests before it
touches a device, and the Python wrappers refuse what the kernels do not take."""
import ctypes

import pytest
import torch

P = 0x7F0000001000          # an aligned address that is never dereferenced


def _linear(**kw):
    from exl3b import native
    a = dict(x=P, dtype=1, ldx=256, M=4, k=256, n=128, tr=P, K=4, code=0, suh=P, svh=P, bias=None,
             act=0, mul=None, ldmul=0, res=None, ldres=0, out=P, ldo=128, ws=None, wsb=0)
    a.update(kw)
    rc = native.lib().exl3b_linear(*a.values(), None)
    return rc, native.last_error()


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(K=1), 8, "K=1"), (dict(K=8), 8, "K=8"),
    (dict(code=3), 7, "code 3"), (dict(code=-1), 7, "code -1"),
    (dict(dtype=0), 7, "dtype 0"), (dict(dtype=3), 7, "dtype 3"),
    (dict(act=5), 7, "activation 5"), (dict(act=-1), 7, "activation -1"),
    (dict(M=-1), 7, "multiples of 128"), (dict(k=192, ldx=192), 7, "multiples of 128"),
    (dict(n=64), 7, "multiples of 128"), (dict(k=0), 7, "multiples of 128"),
    (dict(tr=None), 7, "aligned"), (dict(tr=P + 8), 7, "aligned"),
    (dict(suh=P + 4), 7, "aligned"), (dict(svh=None), 7, "aligned"),
    (dict(bias=P + 2), 7, "aligned"),
    (dict(x=None), 7, "x:"), (dict(x=P + 4), 7, "x:"), (dict(ldx=252), 7, "x:"),
    (dict(ldx=258), 7, "x:"), (dict(out=P + 2), 7, "out:"), (dict(ldo=127), 7, "out:"),
    (dict(mul=P, ldmul=64), 7, "mul:"), (dict(mul=P + 4, ldmul=128), 7, "mul:"),
    (dict(res=P, ldres=130), 7, "residual:"),
    (dict(M=(1 << 24) + 1), 7, "at most"), (dict(k=(1 << 22) + 128, ldx=1 << 23), 7, "at most"),
    (dict(n=(1 << 22) + 128, ldo=1 << 23), 7, "at most"),
    (dict(M=1 << 24, n=1 << 15, ldo=1 << 15), 7, "2^38"),
])
def test_linear_abi_refuses(kw, rc, msg):
    got, text = _linear(**kw)
    assert got == rc and msg in text, (got, text)


def test_linear_abi_empty_is_ok():
    assert _linear(M=0, x=None, out=None)[0] == 0


def test_weight_refuses():
    from exl3b import forward
    tr = torch.zeros(8, 8, 64, dtype=torch.int16)
    s = torch.ones(128).half()
    for args, msg in [((tr, s, s, 1), "K=1"), ((tr, s, s, 8), "K=8"),
                      ((tr, s, s, 5), "int16"), ((tr.int(), s, s, 4), "int16"),
                      ((tr[0], s, s, 4), "int16"), ((tr[:4], s[:64], s, 4), "multiples of 128"),
                      ((tr[:0], s[:0], s, 4), "multiples of 128"),
                      ((tr, s[:64], s, 4), "suh"), ((tr, s, s[:64], 4), "svh"),
                      ((tr, s, s, 4), "CUDA device"), ((tr, s, s, 4, "qtip"), "qtip")]:
        with pytest.raises(ValueError, match=msg):
            forward.TrellisWeight(*args)


class _Weight:
    """Stands for a weight where a call must be refused before any kernel."""
    k, n, K, code_id = 256, 128, 4, 0
    device, index = torch.device("cpu"), -1            # what CPU tensors answer


def test_linear_refuses():
    from exl3b import forward
    w = _Weight()
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    y = torch.zeros(3, 128, dtype=torch.bfloat16)
    big = torch.zeros(3, 512, dtype=torch.bfloat16)
    cases = [
        (dict(x=x.float()), "bf16 or fp16"), (dict(x=x[:, :128]), "in = 256"),
        (dict(activation="swish"), "activation"), (dict(bias=y[0].half()), "bias"),
        (dict(bias=y[0, :64]), "bias"), (dict(mul=y[:1]), "mul"),
        (dict(residual=y.half()), "residual"), (dict(residual=y[:, :64]), "residual"),
        (dict(out=y[:2]), "out"), (dict(out=y.half()), "out"),
        (dict(out=torch.zeros(128, 3, dtype=torch.bfloat16).t()), "out"),
        (dict(x=x.clone().requires_grad_()), "gradient"),
        (dict(residual=y.clone().requires_grad_()), "gradient"),
        # out inside x; out shifted against the residual
        (dict(x=big[:, :256], out=big[:, 128:256]), "overlaps x"),
        (dict(residual=big[:, :128], out=big[:, 64:192]), "overlaps an input"),
    ]
    for kw, msg in cases:
        with pytest.raises(ValueError, match=msg):
            forward.linear(kw.pop("x", x), w, **kw)


def test_overlap_rule():
    from exl3b.forward import _overlap
    buf = torch.zeros(4, 64, dtype=torch.float16)
    assert _overlap(buf[:, :32], buf[:, 16:48])
    assert not _overlap(buf[:, :32], buf[:, 32:])       # interleaved columns
    assert not _overlap(buf[:, 32:], buf[:, :32])
    assert not _overlap(buf[:2], buf[2:])
    assert _overlap(buf[:3], buf[2:])
    assert _overlap(buf, buf)
    assert not _overlap(buf[:0], buf)


def test_load_reads_what_the_writer_stores(tmp_path, monkeypatch):
    """TrellisWeight.load and from_result hold the same fields as the files."""
    from exl3b import export, forward
    g = torch.Generator().manual_seed(0)
    result = {"trellis": torch.randint(-32768, 32768, (8, 16, 80), generator=g, dtype=torch.int16),
              "suh": torch.sign(torch.randn(128, generator=g)).half(),
              "svh": torch.sign(torch.randn(256, generator=g)).half(),
              "Wscale": 0.0173, "K": 5, "code": "exl3_mcg", "channel_scales": False}
    path = export.save_quantized(tmp_path, 3, "mlp.up_proj", result)
    seen = []
    monkeypatch.setattr(forward.TrellisWeight, "__init__",
                        lambda self, *a: seen.append(a))
    forward.TrellisWeight.load(path, device="cpu")
    forward.TrellisWeight.from_result(result, device="cpu")
    stored = export.stored_fields(result)
    for trellis, suh, svh, K, code in seen:
        assert torch.equal(trellis, stored["trellis"]) and torch.equal(suh, stored["suh"])
        assert torch.equal(svh, stored["svh"]) and (K, code) == (5, "exl3_mcg")
    assert len(seen) == 2


def _moe(**kw):
    from exl3b import native
    a = dict(x=P, dtype=1, ldx=256, T=4, D=256, F=128, E=8, top_k=2, norm=1, router=P, rdt=1,
             ldr=256, table=P, Kg=4, Ku=4, Kd=4, code=0, res=None, ldres=0, out=P, ldo=256, ws=P,
             wsb=1 << 30)
    a.update(kw)
    rc = native.lib().exl3b_moe(*a.values(), None)
    return rc, native.last_error()


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(Kg=1), 8, "K=1"), (dict(Kd=8), 8, "K=8"), (dict(code=3), 7, "code 3"),
    (dict(dtype=0), 7, "dtype 0"), (dict(rdt=2), 7, "router dtype 2"),
    (dict(T=257), 7, "257 tokens"), (dict(T=-1), 7, "tokens"), (dict(D=192), 7, "hidden 192"),
    (dict(F=64), 7, "width 64"), (dict(E=0), 7, "0 experts"), (dict(E=1025), 7, "1025 experts"),
    (dict(top_k=0), 7, "top_k 0"), (dict(top_k=9), 7, "top_k 9"),
    (dict(E=64, top_k=33), 7, "top_k 33"), (dict(T=100, E=64, top_k=21), 7, "2048"),
    (dict(x=P + 8), 7, "16-byte"), (dict(ldx=260), 7, "16-byte"), (dict(router=None), 7, "16-byte"),
    (dict(ldr=248), 7, "16-byte"), (dict(table=P + 4), 7, "16-byte"),
    (dict(out=P + 4), 7, "8-byte"), (dict(ldo=128), 7, "8-byte"),
    (dict(res=P, ldres=254), 7, "8-byte"),
    (dict(ws=None), 11, "workspace"), (dict(ws=P + 16), 11, "workspace"),
])
def test_moe_abi_refuses(kw, rc, msg):
    got, text = _moe(**kw)
    assert got == rc and msg in text, (got, text)


def test_moe_workspace_bytes():
    from exl3b import native
    f = native.lib().exl3b_moe_workspace_bytes
    assert f(0, 256, 128, 8, 2) == 0 and f(257, 256, 128, 8, 2) == 0 and f(4, 256, 100, 8, 2) == 0
    assert f(100, 256, 128, 64, 21) == 0
    assert _moe(T=0, x=None, ws=None)[0] == 0


def test_experts_and_moe_refuse():
    from exl3b import forward

    class W:
        def __init__(self, k, n, code="exl3_mul1"):
            self.k, self.n, self.K, self.code, self.code_id = k, n, 4, code, 0
            self.device, self.index = torch.device("cpu"), -1
            self.trellis = self.suh = self.svh = torch.zeros(1)
    g, d = W(256, 128), W(128, 256)
    for args, msg in [(([], [], []), "one of each"), (([g], [g, g], [d]), "one of each"),
                      (([g], [d], [d]), "up of expert 0"), (([g, g], [g, g], [d, g]), "down of expert 1"),
                      (([g, W(256, 128, "exl3_mcg")], [g, g], [d, d]), "gate of expert 1"),
                      (([g] * 1025, [g] * 1025, [d] * 1025), "at most 1024")]:
        with pytest.raises(ValueError, match=msg):
            forward.TrellisExperts(*args)
    ex = forward.TrellisExperts([g] * 4, [g] * 4, [d] * 4)
    assert (ex.D, ex.F, ex.E, ex.Kmax) == (256, 128, 4, (4, 4, 4)) and ex.table.numel() == 12 * 32
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    r = torch.zeros(4, 256, dtype=torch.bfloat16)
    for args, kw, msg in [((x.float(), r, ex, 2), {}, "bf16 or fp16"),
                          ((x[:, :128], r, ex, 2), {}, "in = 256"),
                          ((x, r, ex, 0), {}, "top_k=0"), ((x, r, ex, 5), {}, "top_k=5"),
                          ((x, r[:3], ex, 2), {}, "router"), ((x, r.half(), ex, 2), {}, "router"),
                          ((x, r, ex, 2), dict(residual=x[:2]), "residual"),
                          ((x, r, ex, 2), dict(out=x), "overlaps x"),
                          ((x, r.clone().requires_grad_(), ex, 2), {}, "gradient")]:
        with pytest.raises(ValueError, match=msg):
            forward.moe(*args, **kw)


def test_first_calls_may_come_from_two_threads(monkeypatch):
    """A call that begins while another thread's first call is still being prepared."""
    from types import SimpleNamespace

    from exl3b import forward
    done = []
    fake = SimpleNamespace(exl3b_linear=lambda *a: done.append(a) or 0,
                           exl3b_device_init=lambda index: 0)
    monkeypatch.setattr(forward, "lib", lambda: fake)
    monkeypatch.setattr(forward, "_functions", {})
    monkeypatch.setattr(forward, "_raw_stream", lambda index: 0)
    first = [True]

    def count():                # the second call comes while the first one asks
        if first:
            first.pop()
            forward._call("exl3b_linear", 0, (2,))
        return 1

    monkeypatch.setattr(torch.cuda, "device_count", count)
    forward._call("exl3b_linear", 0, (1,))
    assert done == [(2, 0), (1, 0)]


def test_tangents_are_refused():
    """Forward-mode differentiation: a dual tensor does not require a gradient, and its
    tangent would be lost."""
    from torch.autograd import forward_ad

    from exl3b import forward
    w = _Weight()
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    y = torch.zeros(3, 128, dtype=torch.bfloat16)
    s, tr = torch.ones(128).half(), torch.zeros(8, 8, 64, dtype=torch.int16)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: forward.linear(dual(x), w),
                 lambda: forward.linear(x, w, bias=dual(y[0])),
                 lambda: forward.linear(x, w, mul=dual(y)),
                 lambda: forward.linear(x, w, residual=dual(y)),
                 lambda: forward.linear(x, w, out=dual(y)),
                 lambda: forward.TrellisWeight(tr, dual(s), s, 4),
                 lambda: forward.TrellisWeight(tr, s, dual(s), 4)]
        for call in calls:
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="in = 256"):       # a plain one goes on
            forward.linear(x[:, :128], w)


def test_fields_that_require_a_gradient_are_refused():
    from exl3b import forward
    s, tr = torch.ones(128).half(), torch.zeros(8, 8, 64, dtype=torch.int16)
    for args in ((tr, s.clone().requires_grad_(), s, 4), (tr, s, s.clone().requires_grad_(), 4)):
        with pytest.raises(ValueError, match="gradient"):
            forward.TrellisWeight(*args)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            forward.TrellisWeight(*args)


def test_product_of_refused_sizes():
    from exl3b import native
    f = native.lib().exl3b_linear_product
    for args in [(0, 128, 128, 1), (-1, 128, 128, 1), (4, 64, 128, 1), (4, 128, 192, 1),
                 (4, 128, 128, 0), (4, 128, 128, 3), ((1 << 24) + 1, 128, 128, 1),
                 (4, (1 << 22) + 128, 128, 2)]:
        assert f(*args) == 0
