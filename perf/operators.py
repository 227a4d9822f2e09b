"""Cases of the forward operators on EXL3 tensors: the linear layer with its
epilogue and the mixture-of-experts layer.

A weight is held as the quantizer leaves it: trellis int16 [k/16, n/16, 16 K],
suh fp16 [k] (with the tensor's scale folded in) and svh fp16 [n].  With B the
block-diagonal normalised 128-point Hadamard matrix and C the decoded code
values [k, n], the dequantised weight is diag(suh) B C B diag(svh).

`run` computes an operator in its plain form (elementary torch operations in
fp32, rounded once) or, where `own` is set, through the package.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = ("exl3_mul1", "exl3_3inst", "exl3_mcg")
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")


# ------------------------------------------------------------------ the cases
def _linear(name, M, k, n, K, dtype="bf16", code="exl3_mul1", bias=False, act="none",
            mul=False, residual=False):
    return {"name": name, "op": "linear", "M": M, "k": k, "n": n, "K": K, "dtype": dtype,
            "code": code, "bias": bias, "act": act, "mul": mul, "residual": residual}


def _moe(name, T, D, F, E, top_k, Kg, Ku, Kd, dtype="bf16", code="exl3_mul1", normalize=True,
         residual=False):
    return {"name": name, "op": "moe", "T": T, "D": D, "F": F, "E": E, "top_k": top_k,
            "Kg": Kg, "Ku": Ku, "Kd": Kd, "dtype": dtype, "code": code,
            "normalize": normalize, "residual": residual}


def listed():
    return [
        # one generated token through a small projection: latency only
        _linear("token_kv", 1, 5120, 1024, 7, bias=True),
        # one generated token through the square projection
        _linear("token_square", 1, 5120, 5120, 4),
        # one generated token, the gate of the MLP (its up product already there)
        _linear("token_gate", 1, 5120, 17408, 5, act="silu", mul=True),
        # a few sequences decoding together, MLP down with the residual stream
        _linear("batch_down", 8, 17408, 5120, 4, residual=True),
        # an odd number of sequences, another code and type
        _linear("batch_odd", 37, 6144, 5120, 6, dtype="fp16", code="exl3_mcg", residual=True),
        # a short prompt
        _linear("prompt_short", 203, 5120, 6144, 3, bias=True, act="gelu"),
        # a chunk of a long prompt through the largest projection
        _linear("prompt_chunk", 4096, 5120, 17408, 5, act="silu", mul=True),
        # one generated token through a layer of many small experts
        _moe("moe_token", 1, 2048, 768, 128, 8, 4, 4, 4),
        # a few sequences, mixed bit widths
        _moe("moe_batch", 5, 2048, 768, 128, 8, 3, 5, 6, residual=True),
        # few large experts, probabilities not renormalised
        _moe("moe_large", 9, 5120, 1664, 16, 2, 4, 4, 5, dtype="fp16", normalize=False),
        # a full decode batch: almost every expert is active
        _moe("moe_full", 64, 2048, 768, 128, 8, 4, 4, 4, residual=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))


def draw(rng: random.Random):
    dtype = rng.choice(tuple(DTYPES))
    code = rng.choice(CODES)
    if rng.random() < 0.6:
        while True:
            M = _log_int(rng, 1, 4096)
            k = 128 * _log_int(rng, 1, 136)
            n = 128 * _log_int(rng, 1, 136)
            if M * k * n <= 4096 * 5120 * 17408:
                break
        case = _linear("", M, k, n, rng.randint(2, 7), dtype, code, rng.random() < 0.5,
                       rng.choice(ACTIVATIONS), rng.random() < 0.5, rng.random() < 0.5)
    else:
        while True:
            T = _log_int(rng, 1, 64)
            D = 128 * _log_int(rng, 1, 40)
            F = 128 * _log_int(rng, 1, 13)
            E = _log_int(rng, 4, 128)
            top_k = min(E, _log_int(rng, 1, 8))
            active = E * (1.0 - (1.0 - top_k / E) ** T)
            if E * D * F <= 128 * 2048 * 768 and active * D * F <= 120 * 2048 * 768:
                break
        case = _moe("", T, D, F, E, top_k, rng.randint(2, 7), rng.randint(2, 7),
                    rng.randint(2, 7), dtype, code, rng.random() < 0.5, rng.random() < 0.5)
    del case["name"]
    return case


def work(case):
    if case["op"] == "linear":
        M, k, n = case["M"], case["k"], case["n"]
        act_rows = 1 + (1 if case["mul"] else 0) + (1 if case["residual"] else 0)
        return {"bytes": k * n * case["K"] / 8 + 2 * (k + n) + 2 * M * k + 2 * M * n * act_rows
                + (2 * n if case["bias"] else 0),
                "flops": 2 * M * k * n}
    T, D, F, E, top_k = (case[x] for x in ("T", "D", "F", "E", "top_k"))
    active = E * (1.0 - (1.0 - top_k / E) ** T)          # expected, experts drawn evenly
    bits = case["Kg"] + case["Ku"] + case["Kd"]
    return {"bytes": active * (D * F * bits / 8 + 2 * 3 * (D + F)) + 2 * E * D
            + 2 * T * D * (3 if case["residual"] else 2),
            "flops": 6 * T * top_k * D * F + 2 * T * E * D}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _code_table(code):
    """fp32 [65536]: the value of every 16-bit state (exact in fp16)."""
    s = np.arange(65536, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    if code == "exl3_mul1":
        x = (s * np.uint64(0x83DCD12D)) & low
        total = sum((x >> np.uint64(8 * i)) & np.uint64(255) for i in range(4))
        inv, bias = np.array([0x1EEE, 0xC931], dtype=np.uint16).view(np.float16).astype(np.float64)
        v = (1024.0 + total.astype(np.float64)) * inv + bias
    else:
        if code == "exl3_3inst":
            x = (s * np.uint64(89226354) + np.uint64(64248484)) & low
        else:
            x = (s * np.uint64(0xCBAC1FED)) & low
        x = (x & np.uint64(0x8FFF8FFF)) ^ np.uint64(0x3B603B60)
        a = (x & np.uint64(0xFFFF)).astype(np.uint16).view(np.float16).astype(np.float64)
        b = (x >> np.uint64(16)).astype(np.uint16).view(np.float16).astype(np.float64)
        v = a + b
    return torch.from_numpy(v.astype(np.float16).astype(np.float32)).cuda()


def _signs(g, *shape):
    return torch.randint(0, 2, shape, generator=g, device="cuda").float() * 2 - 1


def _tensors(g, lead, k, n, K, std):
    """Random EXL3 fields (any bitstream is a trellis): entries of the
    dequantised weight have about `std`, channel magnitudes spread by ~20%."""
    tr = torch.randint(-32768, 32768, (*lead, k // 16, n // 16, 16 * K), generator=g,
                       device="cuda", dtype=torch.int16)
    suh = _signs(g, *lead, k) * torch.exp(0.2 * torch.randn(*lead, k, generator=g, device="cuda"))
    svh = _signs(g, *lead, n) * torch.exp(0.2 * torch.randn(*lead, n, generator=g, device="cuda"))
    return tr, (suh * (std / 1.24)).half(), svh.half()


def _activations(g, rows, cols, dt):
    """Normal entries with a few channels an order of magnitude larger, as in
    the residual stream of a trained model."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    big = torch.rand(cols, generator=g, device="cuda") < 0.005
    return torch.where(big, x * 12.0, x).to(dt)


def _package():
    path = os.path.join(os.getcwd(), "exl3xpu-mixedk_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from exl3b import forward
    return forward


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case, "table": _code_table(case["code"])}
    i = torch.arange(128, device="cuda")
    parity = torch.zeros(128, 128, dtype=torch.int64, device="cuda")
    for b in range(7):
        parity ^= ((i[:, None] & i[None, :]) >> b) & 1
    s["had"] = (1.0 - 2.0 * parity.float()) / math.sqrt(128.0)
    if case["op"] == "linear":
        M, k, n = case["M"], case["k"], case["n"]
        s["w"] = _tensors(g, (), k, n, case["K"], 1.0 / math.sqrt(k))
        s["x"] = _activations(g, M, k, dt)
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(dt) if case["bias"] else None
        s["mul"] = torch.randn(M, n, generator=g, device="cuda").to(dt) if case["mul"] else None
        s["residual"] = _activations(g, M, n, dt) if case["residual"] else None
        if own:
            s["weight"] = _package().TrellisWeight(*s["w"], case["K"], case["code"])
        return s
    T, D, F, E = (case[x] for x in ("T", "D", "F", "E"))
    s["gate"] = _tensors(g, (E,), D, F, case["Kg"], 1.0 / math.sqrt(D))
    s["up"] = _tensors(g, (E,), D, F, case["Ku"], 1.0 / math.sqrt(D))
    s["down"] = _tensors(g, (E,), F, D, case["Kd"], 1.0 / math.sqrt(F))
    s["router"] = (torch.randn(E, D, generator=g, device="cuda") / math.sqrt(D)).to(dt)
    s["x"] = _activations(g, T, D, dt)
    s["residual"] = _activations(g, T, D, dt) if case["residual"] else None
    if own:
        fw = _package()
        s["experts"] = fw.TrellisExperts(*(
            [fw.TrellisWeight(*(f[e] for f in s[p]), case[K], case["code"]) for e in range(E)]
            for p, K in (("gate", "Kg"), ("up", "Ku"), ("down", "Kd"))))
    return s


# ------------------------------------------------------------------ plain form
def _rows_of_tile(device):
    """Step t of a tile's sequence -> (row, column) inside the 16 x 16 tile."""
    t = torch.arange(256, device=device)
    lane, q = t // 8, t % 8
    row = (lane % 4) * 2 + (q % 2) + 8 * ((q // 2) % 2)
    col = lane // 4 + 8 * (q // 4)
    return row * 16 + col


def _decode(trellis, K, table):
    """int16 [..., k/16, n/16, 16 K] -> code values fp32 [..., k, n]."""
    *lead, tk, tn, words = trellis.shape
    dev = trellis.device
    # the bit stream, 16 bits at a time (32-bit words, high half first)
    j = torch.arange(words, device=dev)
    stream = trellis.to(torch.int32)[..., j ^ 1] & 0xFFFF
    t = torch.arange(256, device=dev)
    first = (t * K + K - 16) % (256 * K)
    i, r = first // 16, (first % 16).to(torch.int32)
    state = ((stream[..., i] << r) | (stream[..., (i + 1) % words] >> (16 - r))) & 0xFFFF
    step = torch.empty(256, dtype=torch.int64, device=dev)
    step[_rows_of_tile(dev)] = t
    v = table[state[..., step]].reshape(*lead, tk, tn, 16, 16)
    return v.transpose(-3, -2).reshape(*lead, tk * 16, tn * 16)


def _blocks(x, had):
    return (x.reshape(-1, 128) @ had).reshape(x.shape)


def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _product(x, w, K, s):
    """x fp32 [M, k] times the dequantised weight -> fp32 [M, n]."""
    trellis, suh, svh = w
    z = _blocks(x * suh.float(), s["had"]) @ _decode(trellis, K, s["table"])
    return _blocks(z, s["had"]) * svh.float()


def _plain_linear(s):
    case = s["case"]
    v = _product(s["x"].float(), s["w"], case["K"], s)
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, case["act"])
    if s["mul"] is not None:
        v = v * s["mul"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["x"].dtype)


def _plain_moe(s):
    case = s["case"]
    T, D, E, top_k = (case[x] for x in ("T", "D", "E", "top_k"))
    # the choice of experts is made in 64 bits: it must not hang on the order of a sum
    logits = s["x"].double() @ s["router"].double().t()
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]
    e = torch.exp((logits - logits.max(dim=1, keepdim=True).values).float())
    p = e / e.sum(dim=1, keepdim=True)
    p = torch.gather(p, 1, ids)
    if case["normalize"]:
        p = p / p.sum(dim=1, keepdim=True)
    x = s["x"].float()
    y = torch.zeros(T, D, device=x.device)

    def expert(rows, pick):
        parts = [tuple(f[pick] for f in s[name]) for name in ("gate", "up", "down")]
        h = _act(_product(rows, parts[0], case["Kg"], s), "silu") \
            * _product(rows, parts[1], case["Ku"], s)
        return _product(h, parts[2], case["Kd"], s)

    if T * top_k < E:
        for t in range(T):
            for j in range(top_k):
                pick = ids[t, j]
                y[t] += p[t, j] * expert(x[t:t + 1], pick)[0]
    else:
        weight = torch.zeros(T, E, device=x.device).scatter_(1, ids, p)
        for i in range(E):
            y += weight[:, i:i + 1] * expert(x, i)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(state):
    case = state["case"]
    if not own:
        return _plain_linear(state) if case["op"] == "linear" else _plain_moe(state)
    fw = _package()
    if case["op"] == "linear":
        return fw.linear(state["x"], state["weight"], bias=state["bias"],
                         activation=None if case["act"] == "none" else case["act"],
                         mul=state["mul"], residual=state["residual"])
    return fw.moe(state["x"], state["router"], state["experts"], case["top_k"],
                  normalize=case["normalize"], residual=state["residual"])


# ------------------------------------------------------------------ 64-bit values
def _dense(w, K, code):
    """The dequantised weight [k, n] in fp64, from single bits."""
    trellis, suh, svh = w
    tk, tn, words = trellis.shape
    dev = trellis.device
    w16 = trellis.to(torch.int32) & 0xFFFF
    w32 = (w16[..., 1::2].to(torch.int64) << 16) | w16[..., 0::2].to(torch.int64)
    bits = torch.stack([(w32 >> (31 - b)) & 1 for b in range(32)], dim=-1)
    bits = bits.to(torch.uint8).reshape(tk, tn, 256 * K)
    last = (torch.arange(256, device=dev) + 1) * K           # one past a window's last bit
    state = torch.zeros(tk, tn, 256, dtype=torch.int32, device=dev)
    for b in range(16):
        state = state * 2 + bits[:, :, (last - 16 + b) % (256 * K)].to(torch.int32)
    values = _code_table(code).double()[state.long()]
    out = torch.empty(tk, 16, tn, 16, dtype=torch.float64, device=dev)
    for lane in range(32):
        for q in range(8):
            row = 2 * (lane % 4) + (0, 1, 8, 9)[q % 4]
            out[:, row, :, lane // 4 + (8 if q > 3 else 0)] = values[:, :, 8 * lane + q]
    out = out.reshape(tk * 16, tn * 16)
    h = torch.ones(1, 1, dtype=torch.float64, device=dev)
    while h.shape[0] < 128:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    h = h / math.sqrt(128.0)
    k, n = out.shape
    out = torch.matmul(h, out.reshape(k // 128, 128, n)).reshape(k, n)
    out = torch.matmul(out.reshape(k, n // 128, 128), h).reshape(k, n)
    return suh.double()[:, None] * out * svh.double()[None, :]


def _silu64(v):
    return v * torch.sigmoid(v)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "linear":
        v = x @ _dense(s["w"], case["K"], case["code"])
        if s["bias"] is not None:
            v = v + s["bias"].double()
        act = case["act"]
        if act == "relu":
            v = v.clamp(min=0.0)
        elif act == "silu":
            v = _silu64(v)
        elif act == "gelu":
            v = v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
        elif act == "gelu_tanh":
            v = v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
        if s["mul"] is not None:
            v = v * s["mul"].double()
        if s["residual"] is not None:
            v = v + s["residual"].double()
        return v
    p = torch.softmax(x @ s["router"].double().t(), dim=1)
    y = torch.zeros_like(x)
    chosen = {}
    for t, row in enumerate(p.tolist()):
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:case["top_k"]]
        total = sum(row[e] for e in best) if case["normalize"] else 1.0
        for e in best:
            chosen.setdefault(e, []).append((t, row[e] / total))
    for e, uses in chosen.items():
        rows = torch.tensor([t for t, _ in uses], device=x.device)
        share = torch.tensor([w for _, w in uses], dtype=torch.float64, device=x.device)
        gate, up, down = (_dense([f[e] for f in s[name]], case[K], case["code"])
                          for name, K in (("gate", "Kg"), ("up", "Ku"), ("down", "Kd")))
        h = _silu64(x[rows] @ gate) * (x[rows] @ up)
        y[rows] += share[:, None] * (h @ down)
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y
