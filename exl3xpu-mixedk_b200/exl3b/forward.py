"""Forward operators on finished EXL3 tensors.

    linear   act(x W^T + bias) * mul + residual, W an EXL3 tensor
    moe      a mixture-of-experts layer for a few tokens, its experts EXL3 tensors

The consumer's side of the quantizer: what a layer computes from the fields the
quantizer stores (trellis, suh, svh).  A weight is decoded as it is multiplied;
only for long prompts is it decoded once into the call's workspace, where the copy
takes 2 bytes a weight (exl3b_linear_product in the C header tells when).  Weights
are wrapped once (TrellisWeight); a call takes CUDA tensors, runs on torch's
current stream of their device and allocates its output and workspace through
torch's allocator, so it may be captured into a CUDA graph (make or wrap one
weight on the device first: that initialises the library there).

Inference only: the weights are integers, and a tensor that requires a gradient
is refused while gradients are enabled, one with a tangent (forward-mode
differentiation) always.
"""
from __future__ import annotations

import json
import operator
import struct
from pathlib import Path

import torch
from torch.autograd import forward_ad

from . import ops
from .native import check, lib

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
        _no_grad("TrellisWeight", suh, svh)
        if not (trellis.is_cuda and suh.device == trellis.device and svh.device == trellis.device):
            raise ValueError("trellis, suh and svh must be on one CUDA device")
        self.k, self.n, self.K, self.code = k, n, K, code
        self.device = trellis.device
        self.index = trellis.device.index       # of the device
        self._bytes = {}                        # rows -> workspace bytes of linear
        self._fields = (_aligned(trellis.detach(), 16), _aligned(suh.detach().half(), 8),
                        _aligned(svh.detach().half(), 8))
        # trellis, K, code, suh, svh as the C ABI takes them
        self._args = (self.trellis.data_ptr(), K, self.code_id, self.suh.data_ptr(),
                      self.svh.data_ptr())
        with torch.cuda.device(self.device):
            ops.select_device(self.trellis)

    # fixed, since calls go by their addresses; a copy is made anew
    trellis = property(lambda self: self._fields[0])
    suh = property(lambda self: self._fields[1])
    svh = property(lambda self: self._fields[2])

    def __reduce__(self):
        return TrellisWeight, (*self._fields, self.K, self.code)

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
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{op} has no gradient: call it under torch.no_grad() or on "
                                 "detached tensors")
    if forward_ad._current_level >= 0:          # inside a dual_level: no_grad keeps tangents
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{op} has no gradient: a tensor has a tangent")


def _check_input(op: str, what: str, t: torch.Tensor, shape, dtype, index: int):
    if t.shape != shape or t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{op}: {what} must be {tuple(shape)} {dtype} on device {index}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


def _rows(t: torch.Tensor, cols: int, align: int = 8):
    """(t as [rows, cols], its row pitch) as the kernels can read it: unit inner
    stride, rows on `align`-byte boundaries of 2-byte elements (a copy where it is not
    so already)."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    ld, inner = t.stride()
    if inner == 1 and ld >= cols and ld % (align // 2) == 0 and t.data_ptr() % align == 0:
        return t, ld
    if t.shape[0] <= 1 and inner == 1 and t.data_ptr() % align == 0:
        return t, cols
    return t.clone(memory_format=torch.contiguous_format), cols


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [rows, cols] views of 2-byte elements share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    la = a.stride(0) if a.shape[0] > 1 else a.shape[1]
    lb = b.stride(0) if b.shape[0] > 1 else b.shape[1]
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa >= pb + 2 * ((b.shape[0] - 1) * lb + b.shape[1]) or \
            pb >= pa + 2 * ((a.shape[0] - 1) * la + a.shape[1]):
        return False
    if la == lb:                    # interleaved columns of one buffer
        d = ((pb - pa) // 2) % la
        return d < a.shape[1] or d + b.shape[1] > la
    return True


def _out_rows(op: str, out: torch.Tensor, shape, x: torch.Tensor, index: int, sources,
              other: str, o_t: torch.Tensor | None):
    """([rows, cols] view of the caller's `out`, its pitch).  The kernels read `sources`
    ([rows, cols], element by element where they write) and, as a whole, x and `o_t`
    (named `other`): out may be one of the sources, and nothing else of what is read."""
    cols = shape[-1]
    _check_input(op, "out", out, shape, x.dtype, index)
    try:
        o = out.view(-1, cols)
    except RuntimeError:
        raise ValueError(f"{op}: out {tuple(out.shape)} with strides {out.stride()} is not "
                         "a matrix of rows") from None
    many = o.shape[0] > 1
    if o.numel() and (o.stride(1) != 1 or o.data_ptr() % 8 or
                      (many and (o.stride(0) < cols or o.stride(0) % 4))):
        raise ValueError(f"{op}: out must have unit inner stride and rows on 8-byte boundaries")
    if _overlap(o, x):
        raise ValueError(f"{op}: out overlaps x")
    if o_t is not None and o_t.numel() and o.numel():
        last = sum((d - 1) * st for d, st in zip(o_t.shape, o_t.stride())) + 1
        end = o.data_ptr() + 2 * ((o.shape[0] - 1) * o.stride(0) + cols)
        if o_t.data_ptr() < end and o.data_ptr() < o_t.data_ptr() + o_t.element_size() * last:
            raise ValueError(f"{op}: out overlaps {other}")
    for s in sources:
        if s is not None and _overlap(o, s) and not (
                s.data_ptr() == o.data_ptr() and s.shape == o.shape and
                (not many or s.stride(0) == o.stride(0))):
            raise ValueError(f"{op}: out overlaps an input it is not equal to")
    return o, (o.stride(0) if many else cols)


_functions: dict = {}
# the current stream's handle, without a Stream object where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, index: int, args):
    """A C ABI entry point on torch's current stream of device `index`, which is made
    current in the library (it has its own CUDA runtime) and, where it is not, in torch."""
    f = _functions.get(name)
    if f is None:
        # before the function: another thread that finds it will look for this, too
        if "select" not in _functions:
            _functions["select"] = None if torch.cuda.device_count() == 1 \
                else lib().exl3b_device_init
        f = _functions[name] = getattr(lib(), name)
    select = _functions["select"]
    if select is not None:              # with one device it is always the current one
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                return _call(name, index, args)
        check("exl3b_device_init", select(index))
    check(name, f(*args, _raw_stream(index)))


def _scratch(cache: dict, key, index: int, size, *args) -> int:
    """size(*args) bytes of workspace, remembered for a few keys."""
    nbytes = cache.get(key)
    if nbytes is None:
        with torch.cuda.device(index):
            check("exl3b_device_init", lib().exl3b_device_init(index))
            nbytes = size(*args)
        if len(cache) < 64:
            cache[key] = nbytes
    return nbytes


def check_waits(device=None):
    """Raise if a wait inside a forward kernel that has run on `device` (default: the
    current one) ran out, which makes its results invalid.  The next linear or moe call
    there raises it too; work that none follows, a replayed graph's for instance, is
    asked about here, after synchronising.  Told once."""
    with torch.cuda.device(device):
        check("exl3b_device_init", lib().exl3b_device_init(torch.cuda.current_device()))
        check("exl3b_forward_status", lib().exl3b_forward_status())


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
    themselves.  The sums and the epilogue are fp32, rounded once; x is multiplied as
    fp16 numbers after its rotation, which bf16 results hardly show, and with fp16
    tensors as pairs of them."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r}: one of {sorted(map(str, ACTIVATIONS))}")
    dt, k, n, index = DTYPE_IDS.get(x.dtype), w.k, w.n, w.index
    if dt is None:
        raise ValueError(f"x must be bf16 or fp16, got {x.dtype}")
    if x.get_device() != index:
        raise ValueError(f"x is on {x.device}, the weight on {w.device}")
    shape = x.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"x {tuple(shape)} for a weight with in = {k}")
    _no_grad("linear", x, bias, mul, residual, out)
    shape = (*shape[:-1], n)
    bias_ptr = mul_ptr = res_ptr = ldm = ldr = 0
    mr = rr = None
    if bias is not None:
        _check_input("linear", "bias", bias, (n,), x.dtype, index)
        bias = _aligned(bias, 8)
        bias_ptr = bias.data_ptr()
    if mul is not None:
        _check_input("linear", "mul", mul, shape, x.dtype, index)
        mr, ldm = _rows(mul, n)
        mul_ptr = mr.data_ptr()
    if residual is not None:
        _check_input("linear", "residual", residual, shape, x.dtype, index)
        rr, ldr = _rows(residual, n)
        res_ptr = rr.data_ptr()
    xr, ldx = _rows(x, k)
    if out is None:
        y = o = x.new_empty(shape)
        ldo = n
    else:
        y = out
        o, ldo = _out_rows("linear", out, shape, xr, index, (mr, rr), "bias", bias)
    M = xr.shape[0]
    if M:
        nbytes = _scratch(w._bytes, M, index, lib().exl3b_linear_workspace_bytes, M, k, n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        _call("exl3b_linear", index,
              (xr.data_ptr(), dt, ldx, M, k, n, *w._args, bias_ptr, act, mul_ptr, ldm, res_ptr,
               ldr, o.data_ptr(), ldo, ws.data_ptr(), nbytes))
    return y


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
        self.device, self.index, self.code_id = first.device, first.index, first.code_id
        self.weights = (tuple(gate), tuple(up), tuple(down))
        self._bytes = {}                        # (tokens, top_k) -> workspace bytes of moe
        self.Kmax = tuple(max(w.K for w in ws) for ws in self.weights)
        table = b"".join(struct.pack("<QQQii", w.trellis.data_ptr(), w.suh.data_ptr(),
                                     w.svh.data_ptr(), w.K, 0)
                         for ws in self.weights for w in ws)
        self.table = torch.frombuffer(bytearray(table), dtype=torch.uint8).to(self.device)

    def __reduce__(self):               # the table holds addresses: a copy makes its own
        return TrellisExperts, self.weights


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
    dt, D, index = DTYPE_IDS.get(x.dtype), experts.D, experts.index
    if dt is None:
        raise ValueError(f"x must be bf16 or fp16, got {x.dtype}")
    if x.get_device() != index:
        raise ValueError(f"x is on {x.device}, the experts on {experts.device}")
    shape = x.shape
    if not shape or shape[-1] != D:
        raise ValueError(f"x {tuple(shape)} for experts with in = {D}")
    top_k = operator.index(top_k)
    if not 1 <= top_k <= min(experts.E, MOE_TOP_K):
        raise ValueError(f"top_k={top_k} with {experts.E} experts (at most {MOE_TOP_K})")
    if router.dtype is not x.dtype and router.dtype is not torch.float32:
        raise ValueError(f"router must be {x.dtype} or float32, got {router.dtype}")
    _check_input("moe", "router", router, (experts.E, D), router.dtype, index)
    _no_grad("moe", x, router, residual, out)
    rr, res_ptr, ldr = None, 0, 0
    if residual is not None:
        _check_input("moe", "residual", residual, shape, x.dtype, index)
        rr, ldr = _rows(residual, D)
        res_ptr = rr.data_ptr()
    xr, ldx = _rows(x, D, 16)
    rt, ldt = _rows(router, D, 16)
    if out is None:
        y = o = x.new_empty(shape)
        ldo = D
    else:
        y = out
        o, ldo = _out_rows("moe", out, shape, xr, index, (rr,), "router", rt)
    T = xr.shape[0]
    if T:
        most = min(MOE_TOKENS, MOE_PAIRS // top_k)
        nbytes = _scratch(experts._bytes, (min(T, most), top_k), index,
                          lib().exl3b_moe_workspace_bytes, min(T, most), D, experts.F, experts.E,
                          top_k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        rdt = 0 if router.dtype is torch.float32 else dt
        for t in range(0, T, most):
            _call("exl3b_moe", index,
                  (xr.data_ptr() + 2 * t * ldx, dt, ldx, min(most, T - t), D, experts.F, experts.E,
                   top_k, 1 if normalize else 0, rt.data_ptr(), rdt, ldt,
                   experts.table.data_ptr(), *experts.Kmax, experts.code_id,
                   res_ptr + 2 * t * ldr if res_ptr else 0, ldr, o.data_ptr() + 2 * t * ldo, ldo,
                   ws.data_ptr(), nbytes))
    return y
