"""The stack driver's probe: finished tensors applied by the forward operators from
their stored fields.  On CPU the command's refusals and the bookkeeping against a
stand-in product; on the GPU one tensor of the stack and a small gated block."""
import math
from types import SimpleNamespace

import pytest
import torch

from exl3b import forward, stack


def test_probe_refusals():
    with pytest.raises(ValueError, match="rows"):
        stack.Probe(0, 0, "cpu")
    for argv in (["--probe", "-1"], ["--probe", "4", "--split-layers"]):
        with pytest.raises(SystemExit, match="probe"):
            stack.main(argv)


def test_run_rank_passes_the_probe_on():
    seen = []

    def fake(layer, device, out_root=None, probe=0):
        seen.append((layer, probe))
        return []

    stack.run_rank(3, 1, 2, "cpu", quantize=fake, probe=5)
    assert seen == [(1, 5)]


def test_probe_of_a_block_on_cpu(monkeypatch):
    """With exact stand-ins for the operators the errors are those of the weights."""
    class Weight:
        def __init__(self, W):
            self.W, (self.n, self.k) = W, W.shape

        @classmethod
        def from_result(cls, r, device):
            return cls(r["W_hat"])

    monkeypatch.setattr(forward, "TrellisWeight", Weight)
    monkeypatch.setattr(forward, "TrellisExperts",
                        lambda g, u, d: SimpleNamespace(D=g[0].k, w=(g[0], u[0], d[0])))
    monkeypatch.setattr(forward, "linear", lambda x, w: x.float() @ w.W.t())

    def moe(x, router, experts, top_k):
        g, u, d = experts.w
        assert router.shape == (1, x.shape[1]) and top_k == 1
        h = torch.nn.functional.silu(x.float() @ g.W.t()) * (x.float() @ u.W.t())
        return h @ d.W.t()

    monkeypatch.setattr(forward, "moe", moe)
    g = torch.Generator().manual_seed(3)
    W = {"gate": torch.randn(48, 32, generator=g), "up": torch.randn(48, 32, generator=g),
         "down": torch.randn(32, 48, generator=g)}
    p = stack.Probe(7, 2, "cpu")
    for name in ("gate", "up"):
        assert p.tensor(name, W[name], {"W_hat": W[name]}) == 0.0 and p.block() is None
    # twice the weight: twice the product, an error of 1
    assert math.isclose(p.tensor("down", W["down"], {"W_hat": 2 * W["down"]}), 1.0, rel_tol=1e-6)
    assert math.isclose(p.block(), 1.0, rel_tol=1e-6)
    assert p.block() is None
    assert p.x(32) is p.x(32) and torch.equal(stack.Probe(7, 2, "cpu").x(32), p.x(32))
    assert not torch.equal(stack.Probe(7, 3, "cpu").x(32), p.x(32))


@pytest.mark.gpu
def test_probe_of_quantized_tensors():
    """The output error on independent normal inputs has the weight's relative error
    as its expectation: sqrt(sum ||x (W - W_hat)^T||^2 / sum ||x W^T||^2) is within 10%
    of ||W - W_hat|| / ||W|| at 64 rows and 256 and more outputs (its deviation is below
    1 / sqrt(2 * 64)), plus the operators' own rounding (2^-11)."""
    from exl3b import api
    dev = torch.device("cuda", 0)
    g = torch.Generator().manual_seed(5)
    D, F = 256, 512
    p = stack.Probe(64, 0, dev)
    for name, o, i, K in (("gate", F, D, 4), ("up", F, D, 5), ("down", D, F, 6)):
        W = (torch.randn(o, i, generator=g) / math.sqrt(i)).to(dev)
        r = api.quantize_linear(W, None, K=K, out_device="cuda")
        rel = float(((r["W_hat"] - W).square().sum() / W.square().sum()).sqrt())
        assert abs(p.tensor(name, W, r) - rel) <= 0.1 * rel + 2.0 ** -10, name
    # the block's error is that of its parts: K = 4 leaves some 5% in gate
    assert 0.0 < p.block() < 0.2


@pytest.mark.gpu
def test_stack_layer_reports_probe_errors():
    dev = torch.device("cuda", 0)
    stats = stack.quantize_layer(0, dev, tensors=["k", "v"], probe=3)
    assert all(0.0 < s["probe_error"] < 0.1 and "block_error" not in s for s in stats)
    assert "probe_error" not in stack.quantize_layer(0, dev, tensors=["k"])[0]


def test_probe_summary():
    stats = [{"probe_error": 0.25}, {"probe_error": 0.75, "block_error": 0.5}]
    assert stack.probe_summary(stats, 0) == {}
    assert stack.probe_summary(stats, 4) == {"probe_rows": 4, "probe_error_max": 0.75,
                                             "probe_error_mean": 0.5, "block_error_max": 0.5}
    assert stack.probe_summary([], 4)["probe_error_max"] is None
