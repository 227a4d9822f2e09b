"""Forward operators on finished EXL3 tensors.

    linear   act(x W^T + bias) * mul + residual, W an EXL3 tensor
    moe      a mixture-of-experts layer for a few tokens, its experts EXL3 tensors

The consumer's side of the quantizer: what a layer computes from the fields the
quantizer stores (trellis, suh, svh), without writing a dense weight.  Weights
are wrapped once (TrellisWeight); a call takes CUDA tensors, runs on torch's
current stream of their device and allocates its output and workspace through
torch's allocator, so it may be captured into a CUDA graph (make or wrap one
weight on the device first: that initialises the library there).

Inference only: the weights are integers, and a tensor that requires a gradient
is refused while gradients are enabled.
"""
from __future__ import annotations

import json
import struct
from pathlib import Path

import torch

from . import ops
from .native import call, lib

DTYPE_IDS = {torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _aligned(t: torch.Tensor, nbytes: int) -> torch.Tensor:
    """t, contiguous and with its first element on an `nbytes` boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % nbytes == 0 else t.clone()


class TrellisWeight:
    """One EXL3 tensor on a CUDA device: trellis int16 [k/16, n/16, 16 K], suh [k]
    (with the tensor's scale folded in) and svh [n] as fp16 -- the fields that
    export.stored_fields / save_quantized write."""

    def __init__(self, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, K: int,
                 code: str = "exl3_mul1"):
        K = int(K)
        if not 2 <= K <= 7:
            raise ValueError(f"K={K} outside 2..7")
        self.code_id = ops.code_id(code)
        if trellis.dim() != 3 or trellis.dtype != torch.int16 or trellis.shape[2] != 16 * K:
            raise ValueError(f"trellis must be int16 [k/16, n/16, {16 * K}] at K={K}, got "
                             f"{tuple(trellis.shape)} {trellis.dtype}")
        k, n = 16 * trellis.shape[0], 16 * trellis.shape[1]
        if k == 0 or n == 0 or k % 128 or n % 128:
            raise ValueError(f"weight [{k}, {n}]: in and out must be multiples of 128")
        if tuple(suh.shape) != (k,) or tuple(svh.shape) != (n,):
            raise ValueError(f"suh {tuple(suh.shape)} / svh {tuple(svh.shape)} for a "
                             f"[{k}, {n}] weight")
        if not (trellis.is_cuda and suh.device == trellis.device and svh.device == trellis.device):
            raise ValueError("trellis, suh and svh must be on one CUDA device")
        self.k, self.n, self.K, self.code = k, n, K, code
        self.device = trellis.device
        self.trellis = _aligned(trellis.detach(), 16)
        self.suh = _aligned(suh.detach().half(), 8)
        self.svh = _aligned(svh.detach().half(), 8)
        with torch.cuda.device(self.device):
            ops.select_device(self.trellis)

    @classmethod
    def from_result(cls, result: dict, device=None) -> "TrellisWeight":
        """The stored form of one quantize_linear result (export.stored_fields:
        the tensor's scale goes into suh, rounded to fp16) on `device`
        (default: the current CUDA device)."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        suh = result["suh"]
        if not result.get("channel_scales", False):
            suh = suh.float() * float(result["Wscale"])
        return cls(result["trellis"].to(dev), suh.half().to(dev), result["svh"].half().to(dev),
                   result["K"], result.get("code", "exl3_mul1"))

    @classmethod
    def load(cls, path, device=None) -> "TrellisWeight":
        """ROOT/L{nn}/{module}.safetensors as export.save_quantized writes it, with
        K and the code from the .json beside it."""
        from safetensors.torch import load_file
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        fields = load_file(str(path))
        info = json.loads(Path(path).with_suffix(".json").read_text())
        return cls(fields["trellis"].to(dev), fields["suh"].to(dev), fields["svh"].to(dev),
                   info["K"], info.get("code", "exl3_mul1"))

    def __repr__(self):
        return f"TrellisWeight([{self.k}, {self.n}], K={self.K}, {self.code}, {self.device})"


# ------------------------------------------------------------------ arguments
def _no_grad(op: str, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{op} has no gradient: call it under torch.no_grad() or on detached "
                         "tensors")


def _check_input(op: str, what: str, t: torch.Tensor, shape, dtype, device):
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{op}: {what} must be {tuple(shape)} {dtype} on {device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t as [rows, cols] the kernels can read: unit inner stride, rows on 8-byte
    boundaries (a copy where it is not so already)."""
    t = t.reshape(-1, cols)
    if t.stride(1) == 1 and t.data_ptr() % 8 == 0 and \
            (t.shape[0] <= 1 or (t.stride(0) >= cols and t.stride(0) % 4 == 0)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [rows, cols] views of 2-byte elements share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    pa, pb, la, lb = a.data_ptr(), b.data_ptr(), _ld(a), _ld(b)
    if pa >= pb + 2 * ((b.shape[0] - 1) * lb + b.shape[1]) or \
            pb >= pa + 2 * ((a.shape[0] - 1) * la + a.shape[1]):
        return False
    if la == lb:                    # interleaved columns of one buffer
        d = ((pb - pa) // 2) % la
        return d < a.shape[1] or d + b.shape[1] > la
    return True


def _out_rows(op: str, out, lead, cols: int, x: torch.Tensor, sources) -> torch.Tensor:
    """The [rows, cols] view to write: a new tensor, or the caller's `out`.  The
    kernel reads `sources` ([rows, cols], element by element where it writes) and
    x (as a whole): out may be one of the sources, and nothing else of them."""
    if out is None:
        return torch.empty(*lead, cols, dtype=x.dtype, device=x.device).view(-1, cols)
    _check_input(op, "out", out, (*lead, cols), x.dtype, x.device)
    try:
        o = out.view(-1, cols)
    except RuntimeError:
        raise ValueError(f"{op}: out {tuple(out.shape)} with strides {out.stride()} is not "
                         "a matrix of rows") from None
    if o.numel() and (o.stride(1) != 1 or o.data_ptr() % 8 or
                      (o.shape[0] > 1 and (o.stride(0) < cols or o.stride(0) % 4))):
        raise ValueError(f"{op}: out must have unit inner stride and rows on 8-byte boundaries")
    if _overlap(o, x):
        raise ValueError(f"{op}: out overlaps x")
    for s in sources:
        if s is not None and _overlap(o, s) and not (
                s.data_ptr() == o.data_ptr() and s.shape == o.shape and _ld(s) == _ld(o)):
            raise ValueError(f"{op}: out overlaps an input it is not equal to")
    return o


def _workspace(nbytes: int, device):
    """(tensor or None, pointer) of stream-ordered scratch."""
    if not nbytes:
        return None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


# ------------------------------------------------------------------ linear
def linear(x: torch.Tensor, w: TrellisWeight, bias: torch.Tensor | None = None,
           activation: str | None = None, mul: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None
           ) -> torch.Tensor:
    """act(x W^T + bias) * mul + residual for an EXL3 weight W [n, k].

    x [..., k] bf16 or fp16 (any number of rows, one to a long prompt); bias [n];
    mul and residual [..., n]; all of x's dtype and on the weight's device.
    activation: None, "relu", "silu", "gelu" (erf) or "gelu_tanh".  Returns
    [..., n] in x's dtype, or writes `out`, which may be `mul` or `residual`
    themselves.  The sums and the epilogue are fp32, rounded once."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {sorted(map(str, ACTIVATIONS))}")
    if x.dtype not in DTYPE_IDS:
        raise ValueError(f"x must be bf16 or fp16, got {x.dtype}")
    if x.device != w.device:
        raise ValueError(f"x is on {x.device}, the weight on {w.device}")
    if x.dim() < 1 or x.shape[-1] != w.k:
        raise ValueError(f"x {tuple(x.shape)} for a weight with in = {w.k}")
    _no_grad("linear", x, bias, mul, residual)
    lead = x.shape[:-1]
    if bias is not None:
        _check_input("linear", "bias", bias, (w.n,), x.dtype, x.device)
        bias = _aligned(bias, 8)
    for what, t in (("mul", mul), ("residual", residual)):
        if t is not None:
            _check_input("linear", what, t, (*lead, w.n), x.dtype, x.device)
    xr = _rows(x, w.k)
    mr = None if mul is None else _rows(mul, w.n)
    rr = None if residual is None else _rows(residual, w.n)
    o = _out_rows("linear", out, lead, w.n, xr, (mr, rr))
    M = xr.shape[0]
    if M:
        with torch.cuda.device(x.device):
            dev = ops.select_device(xr)
            nbytes = lib().exl3b_linear_workspace_bytes(M, w.k, w.n)
            ws, ws_ptr = _workspace(nbytes, x.device)
            call("exl3b_linear", xr.data_ptr(), DTYPE_IDS[x.dtype], _ld(xr), M, w.k, w.n,
                 w.trellis.data_ptr(), w.K, w.code_id, w.suh.data_ptr(), w.svh.data_ptr(),
                 0 if bias is None else bias.data_ptr(), ACTIVATIONS[activation],
                 0 if mr is None else mr.data_ptr(), 0 if mr is None else _ld(mr),
                 0 if rr is None else rr.data_ptr(), 0 if rr is None else _ld(rr),
                 o.data_ptr(), _ld(o), ws_ptr, nbytes, ops.stream_handle(dev))
    return o.view(*lead, w.n) if out is None else out


# ------------------------------------------------------------------ mixture of experts
MOE_TOKENS, MOE_PAIRS = 256, 2048      # tokens and (token, expert) pairs of one call
MOE_EXPERTS, MOE_TOP_K = 1024, 32


class TrellisExperts:
    """The experts of one mixture-of-experts layer: gate and up [D -> F] and down
    [F -> D], one TrellisWeight per expert each, of one code and on one device;
    bit widths may differ from tensor to tensor."""

    def __init__(self, gate, up, down):
        gate, up, down = list(gate), list(up), list(down)
        if not gate or len(gate) != len(up) or len(gate) != len(down):
            raise ValueError(f"{len(gate)} gate, {len(up)} up and {len(down)} down weights: "
                             "need one of each per expert")
        if len(gate) > MOE_EXPERTS:
            raise ValueError(f"{len(gate)} experts: at most {MOE_EXPERTS}")
        first = gate[0]
        self.D, self.F, self.E = first.k, first.n, len(gate)
        for what, ws, shape in (("gate", gate, (self.D, self.F)), ("up", up, (self.D, self.F)),
                                ("down", down, (self.F, self.D))):
            for e, w in enumerate(ws):
                if (w.k, w.n) != shape or w.code != first.code or w.device != first.device:
                    raise ValueError(f"{what} of expert {e} is {w}, expected [{shape[0]}, "
                                     f"{shape[1]}] {first.code} on {first.device}")
        self.device, self.code_id = first.device, first.code_id
        self.weights = (gate, up, down)
        self.Kmax = tuple(max(w.K for w in ws) for ws in self.weights)
        table = b"".join(struct.pack("<QQQii", w.trellis.data_ptr(), w.suh.data_ptr(),
                                     w.svh.data_ptr(), w.K, 0)
                         for ws in self.weights for w in ws)
        self.table = torch.frombuffer(bytearray(table), dtype=torch.uint8).to(self.device)


def _rows16(t: torch.Tensor, cols: int) -> torch.Tensor:
    """_rows with 16-byte aligned rows (8 elements of 2 bytes, 4 of 4)."""
    t = t.reshape(-1, cols)
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and \
            (t.shape[0] <= 1 or (t.stride(0) >= cols and t.stride(0) % 8 == 0)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def moe(x: torch.Tensor, router: torch.Tensor, experts: TrellisExperts, top_k: int,
        normalize: bool = True, residual: torch.Tensor | None = None, *,
        out: torch.Tensor | None = None) -> torch.Tensor:
    """Mixture-of-experts layer, for the few tokens of a decoding batch:

        l = x router^T; S = the top_k largest (ties: lowest index); p = softmax(l)
        y = sum_{e in S} w_e down_e(silu(gate_e x) * up_e x) + residual

    with w = p, or p / sum_S p if `normalize`.  x [..., D] bf16 or fp16, router
    [E, D] of x's dtype or fp32, residual [..., D].  Returns [..., D] in x's
    dtype, or writes `out`, which may be `residual` itself.  More than 256 tokens
    (or 2048 choices) are taken in pieces of that many; a chosen expert is read once
    for 8 or 16 of its tokens, so long prompts are better served by linear per
    expert."""
    if x.dtype not in DTYPE_IDS:
        raise ValueError(f"x must be bf16 or fp16, got {x.dtype}")
    if x.device != experts.device:
        raise ValueError(f"x is on {x.device}, the experts on {experts.device}")
    if x.dim() < 1 or x.shape[-1] != experts.D:
        raise ValueError(f"x {tuple(x.shape)} for experts with in = {experts.D}")
    top_k = int(top_k)
    if not 1 <= top_k <= min(experts.E, MOE_TOP_K):
        raise ValueError(f"top_k={top_k} with {experts.E} experts (at most {MOE_TOP_K})")
    if router.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"router must be {x.dtype} or float32, got {router.dtype}")
    _check_input("moe", "router", router, (experts.E, experts.D), router.dtype, x.device)
    _no_grad("moe", x, router, residual)
    lead, D = x.shape[:-1], experts.D
    if residual is not None:
        _check_input("moe", "residual", residual, (*lead, D), x.dtype, x.device)
    xr = _rows16(x, D)
    rt = _rows16(router, D)
    rr = None if residual is None else _rows(residual, D)
    o = _out_rows("moe", out, lead, D, xr, (rr,))
    T = xr.shape[0]
    if T:
        with torch.cuda.device(x.device):
            dev = ops.select_device(xr)
            most = min(MOE_TOKENS, MOE_PAIRS // top_k)
            nbytes = lib().exl3b_moe_workspace_bytes(min(T, most), D, experts.F, experts.E, top_k)
            ws, ws_ptr = _workspace(nbytes, x.device)
            for t in range(0, T, most):
                n = min(most, T - t)
                call("exl3b_moe", xr[t:].data_ptr(), DTYPE_IDS[x.dtype], _ld(xr), n, D, experts.F,
                     experts.E, top_k, int(bool(normalize)), rt.data_ptr(),
                     0 if router.dtype == torch.float32 else DTYPE_IDS[x.dtype], _ld(rt),
                     experts.table.data_ptr(), *experts.Kmax, experts.code_id,
                     0 if rr is None else rr[t:].data_ptr(), 0 if rr is None else _ld(rr),
                     o[t:].data_ptr(), _ld(o), ws_ptr, nbytes, ops.stream_handle(dev))
    return o.view(*lead, D) if out is None else out
