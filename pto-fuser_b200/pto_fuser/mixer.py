"""Operators around a recurrent token mixer, on hand-written sm_100a kernels.

The chunked forwards start from ready q, k, v. These are the steps a layer needs next to
them, each in its form for prompts and, where it keeps a state, for single tokens:

  short_conv / short_conv_step   short causal depthwise convolution (+ SiLU)
  ssm_scan / ssm_scan_step       selective state space scan
  add_rms_norm                   root-mean-square norm with the residual's addition,
                                 optionally to 8 bits with scales

Like the chunked forwards they launch on the current CUDA stream of the tensors' device
without synchronising, can be captured in a CUDA graph, raise ``ValueError`` /
``TypeError`` for wrong arguments and ``NativeError`` for a failed launch, and have no
derivatives: a call that would have to record a backward or carry a tangent is refused. Scratch comes from torch's
caching allocator, call by call, so calls on several streams and several captured graphs
never share any. They have no counterpart in the reference package.

Prompts come as ``[N, T, ..]`` (N sequences of T tokens) or packed as ``[T, ..]`` with
``cu_seqlens`` (int32 [N + 1] on the device, non-decreasing): sequence n is tokens
``cu_seqlens[n]`` to ``cu_seqlens[n + 1]``, possibly none. Packed tokens of no sequence get
zeros in a fresh output and are left as they were in ``out``.

Single tokens come as ``[M, ..]`` rows. Row m updates the state slot ``slots[m]`` (int32 [M]
on the device; slot m without it) in place. A slot outside the state is padding: nothing is
touched and the row's output is zero. Rows that share a slot are applied in row order. The
state shares no memory with the other arguments.
"""
from __future__ import annotations

import ctypes
import itertools
import math
from typing import Dict, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import native as nv

_INT_MAX = 2 ** 31 - 1
_byref = ctypes.byref


def _tensor(name: str, t: torch.Tensor, shape: tuple, dtype, like: torch.Tensor) -> None:
    """shape, dtype and device of an argument; its innermost dimension is contiguous and its
    memory holds its values."""
    if t.shape != shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} != expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} dtype {t.dtype} != expected {dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} on {t.device}, expected {like.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if t.is_neg():
        raise ValueError(f"{name} is a negated view of other values: pass {name}.resolve_neg()")


def _dense(name: str, t: torch.Tensor, shape: tuple, dtype, like: torch.Tensor) -> None:
    _tensor(name, t, shape, dtype, like)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _weight_dtype(name: str, t: torch.Tensor, x: torch.Tensor):
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise TypeError(f"{name} dtype {t.dtype}: expected {x.dtype} or torch.float32")
    return t.dtype


def _no_backward(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no backward: call it under torch.no_grad() or on "
                                 "detached tensors")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what} has no forward-mode derivative: call it on the primals")


def _sizes(what: str, *sizes: int) -> None:
    for s in sizes:
        if s > _INT_MAX:
            raise ValueError(f"{what}: size {s} is beyond 2^31 - 1")


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First and last + 1 byte that a tensor can touch."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    a = t.data_ptr()
    return a, a + (last + 1) * t.element_size()


def _pitch(t: torch.Tensor) -> int:
    """Greatest common divisor of the strides between a tensor's rows, in bytes (0: one row)."""
    return math.gcd(*(s * t.element_size() for n, s in zip(t.shape[:-1], t.stride()) if n > 1), 0)


def _disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
    """No byte in common: apart as a whole, or columns of one wider buffer."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    pitch = math.gcd(_pitch(a), _pitch(b))
    if pitch == 0 or a.dim() < 2 or b.dim() < 2:
        return False
    # where b's rows begin, counted from where a's do, within a pitch
    at = (b.data_ptr() - a.data_ptr()) % pitch
    return at >= a.shape[-1] * a.element_size() and at + b.shape[-1] * b.element_size() <= pitch


def _apart(what: str, out: torch.Tensor, *others) -> None:
    """``out`` shares no memory with ``others`` and does not overlap itself."""
    if any(t is not None and not _disjoint(out, t) for t in others):
        raise ValueError(f"{what}: out must not share memory with an input")
    _own_memory(what, "out", out)


def _state_apart(what: str, state: torch.Tensor, *inputs) -> None:
    """``state``, which is written while inputs are read, shares no memory with them."""
    if any(t is not None and not _disjoint(state, t) for t in inputs):
        raise ValueError(f"{what}: state must not share memory with an input")
    _own_memory(what, "state", state)


def _own_memory(what: str, name: str, t: torch.Tensor) -> None:
    """No two elements of a tensor that is written lie at one address."""
    if t.is_contiguous():
        return
    need = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < need:
            raise ValueError(f"{what}: {name} overlaps itself")
        need = s * (n - 1) + need


def _cuda(what: str, x: torch.Tensor) -> None:
    if x.device.type != "cuda":
        raise ValueError(f"{what}: CUDA tensors are needed, x is on {x.device}")


# ------------------------------------------------------------------------- launch ----
# A call that has been checked leaves a launch plan for its signature (shapes, strides, types
# and device of its tensors, and its options); later calls with the signature go straight to
# the plan. ``args`` says where the C entry point's pointers come from: a tensor's index,
# _OUT + i for output i, _NULL, _SCRATCH and _SCRATCH_BYTES.
_NULL, _SCRATCH, _SCRATCH_BYTES, _OUT = -1, -2, -3, 100
_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
_CONV, _CONV_STEP, _SCAN, _SCAN_STEP, _NORM = range(5)


def _failed(code: int):
    return nv.NativeError(code, nv.last_error())


def _run(*call):
    """The results by plan, or None where there is none."""
    r = nv.launcher().run(*call)
    if r is not None and r.__class__ is not tuple:
        raise _failed(r)
    return r


def _launch(call: tuple, name: str, p, args: tuple, outs: tuple, results: tuple, *,
            scratch: int = 0, out: Optional[torch.Tensor] = None, keep: bool = True,
            writes: int = -1) -> tuple:
    """Launch a checked call ``(op, flags, tensors...)`` and, unless it writes into ``out``,
    keep it as the plan of its signature. ``writes``: the index of a tensor that it updates (a
    later call where that one's memory reaches into another's is checked anew)."""
    fn = getattr(nv.lib(), name)
    if out is None and keep:
        addr = ctypes.cast(fn, ctypes.c_void_p).value
        codes = tuple((tuple(shape), _CODES[dt]) for shape, dt in outs)
        if nv.launcher().add(call, addr, bytes(p), args, codes, scratch, results,
                             writes):
            r = _run(*call)
            if r is not None:
                return r
    tensors = call[2:]
    dev = tensors[0].device
    with torch.cuda.device(dev):
        made = [torch.empty(shape, dtype=dt, device=dev) for shape, dt in outs]
        if out is not None:
            made[0] = out
        ws = torch.empty(scratch, dtype=torch.uint8, device=dev) if scratch else None
        special = {_NULL: None, _SCRATCH: nv.ptr(ws), _SCRATCH_BYTES: scratch}
        ptrs = [special[i] if i < 0 else made[i - _OUT].data_ptr() if i >= _OUT
                else nv.ptr(tensors[i]) for i in args]
        nv.check(fn(_byref(p), *ptrs, nv.stream_handle(dev)))
    for t in (out, None if writes < 0 else tensors[writes]):
        if t is not None:
            torch.autograd.graph.increment_version(t)     # a backward that saved it must not use it
    return tuple(None if i < 0 else made[i] for i in results)


def _prompt(what: str, x: torch.Tensor, cu_seqlens: Optional[torch.Tensor]):
    """(packed, sequences, tokens, channels) of a prompt call."""
    if cu_seqlens is None:
        if x.dim() != 3:
            raise ValueError(f"{what}: x shape {tuple(x.shape)}: expected [N, T, D], or [T, D] "
                             "with cu_seqlens")
        N, T, D = x.shape
    else:
        if x.dim() != 2:
            raise ValueError(f"{what}: x shape {tuple(x.shape)}: expected [T, D] with cu_seqlens")
        T, D = x.shape
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            raise ValueError(f"{what}: cu_seqlens shape {tuple(cu_seqlens.shape)}: expected [N + 1]")
        _dense("cu_seqlens", cu_seqlens, cu_seqlens.shape, torch.int32, x)
        N = cu_seqlens.shape[0] - 1
    if D < 1:
        raise ValueError(f"{what}: x has no channels")
    _sizes(what, N, T, D)
    return cu_seqlens is not None, N, T, D


def _strides(t: Optional[torch.Tensor], packed: bool) -> Tuple[int, int]:
    """Batch and token stride of a prompt tensor."""
    if t is None:
        return 0, 0
    return (0, t.stride(0)) if packed else (t.stride(0), t.stride(1))


def _dense_strides(x: torch.Tensor) -> Tuple[int, int]:
    """Batch and token stride of a fresh output like a prompt's x."""
    return (0, x.shape[-1]) if x.dim() == 2 else (x.shape[1] * x.shape[2], x.shape[2])


# -------------------------------------------------------------------- convolution ----
def _silu_flag(activation) -> int:
    return 1 if activation == "silu" else 0 if activation is None else 1 << 20


def _conv_weights(what: str, x, weight, bias, activation):
    D = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != D or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"{what}: weight shape {tuple(weight.shape)}: expected [{D}, 2 to 4]")
    wd = _weight_dtype("weight", weight, x)
    _dense("weight", weight, weight.shape, wd, x)
    if bias is not None:
        _dense("bias", bias, (D,), wd, x)
    if activation not in (None, "silu"):
        raise ValueError(f"{what}: activation {activation!r}: expected None or 'silu'")
    return weight.shape[1], nv.dtype_code(wd), int(activation == "silu")


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
               activation: Optional[str] = "silu", initial_state: Optional[torch.Tensor] = None,
               cu_seqlens: Optional[torch.Tensor] = None, output_final_state: bool = True,
               out: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Short causal depthwise convolution over prompts:
    ``y[t, d] = act(bias[d] + sum_j weight[d, j] x[t - W + 1 + j, d])``, accumulated in fp32.

    x [N, T, D], or [T, D] with cu_seqlens (f16 / bf16 / f32; tokens may be strided);
    weight [D, W], W = 2 to 4, and bias [D] in x's type or fp32; activation "silu" or None.
    initial_state [N, W - 1, D] holds the inputs before each sequence, oldest first (zeros
    without it). Returns (y, final_state): y like x, and the last W - 1 inputs of each
    sequence as [N, W - 1, D] (None with output_final_state=False). ``out`` receives y."""
    flags = _silu_flag(activation) | bool(output_final_state) << 1
    call = (_CONV, flags, x, weight, bias, initial_state, cu_seqlens)
    if out is None:
        r = _run(*call)
        if r is not None:
            return r
    packed, N, T, D = _prompt("short_conv", x, cu_seqlens)
    dt = nv.dtype_code(x.dtype)
    _tensor("x", x, x.shape, x.dtype, x)
    W, wd, silu = _conv_weights("short_conv", x, weight, bias, activation)
    if initial_state is not None:
        _dense("initial_state", initial_state, (N, W - 1, D), x.dtype, x)
    _no_backward("short_conv", x, weight, bias, initial_state, out)
    if out is not None:
        _tensor("out", out, x.shape, x.dtype, x)
        _apart("short_conv", out, x, weight, bias, initial_state, cu_seqlens)
    _cuda("short_conv", x)
    ys = _dense_strides(x) if out is None else _strides(out, packed)
    p = nv.ShortConvParams(*_strides(x, packed), *ys, N, T, D, W, dt, wd, silu, packed,
                           out is None)
    outs = ((x.shape, x.dtype), ((N, W - 1, D), x.dtype))[:1 + bool(output_final_state)]
    final = 1 if output_final_state else _NULL
    return _launch(call, "ptof_short_conv_exec", p,
                   (0, 1, 2, 4, 3, _OUT, _OUT + 1 if output_final_state else _NULL), outs,
                   (0, final), out=out)


def _slots(what: str, slots: Optional[torch.Tensor], M: int, S: int, x: torch.Tensor) -> None:
    if slots is not None:
        _dense("slots", slots, (M,), torch.int32, x)
    elif S < M:
        raise ValueError(f"{what}: {M} rows and {S} state slots: pass slots")


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor,
                    bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = "silu",
                    slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None
                    ) -> torch.Tensor:
    """``short_conv`` for single tokens: x [M, D]; state [slots, W - 1, D] in x's type, the
    last inputs of each sequence, oldest first (``short_conv``'s final state), shifted by
    one in place. Returns y [M, D]; ``out`` may be x."""
    call = (_CONV_STEP, _silu_flag(activation), x, state, weight, bias, slots)
    if out is None:
        r = _run(*call)
        if r is not None:
            return r[0]
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"short_conv_step: x shape {tuple(x.shape)}: expected [M, D]")
    M, D = x.shape
    dt = nv.dtype_code(x.dtype)
    _tensor("x", x, x.shape, x.dtype, x)
    W, wd, silu = _conv_weights("short_conv_step", x, weight, bias, activation)
    if state.dim() != 3:
        raise ValueError(f"state shape {tuple(state.shape)} != expected [slots, {W - 1}, {D}]")
    S = state.shape[0]
    _sizes("short_conv_step", M, D, S)
    _tensor("state", state, (S, W - 1, D), x.dtype, x)
    _slots("short_conv_step", slots, M, S, x)
    _no_backward("short_conv_step", x, state, weight, bias, out)
    if out is not None:
        _tensor("out", out, x.shape, x.dtype, x)
        same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
        _apart("short_conv_step", out, None if same else x, state, weight, bias, slots)
    _state_apart("short_conv_step", state, x, weight, bias, slots)
    _cuda("short_conv_step", x)
    p = nv.ShortConvStepParams(x.stride(0), D if out is None else out.stride(0), state.stride(0),
                               state.stride(1), M, S, D, W, dt, wd, silu)
    return _launch(call, "ptof_short_conv_step_exec", p, (0, 1, 2, 3, 4, _OUT),
                   ((x.shape, x.dtype),), (0,), out=out, writes=1)[0]


# --------------------------------------------------------------------------- scan ----
def _scan_weights(what: str, x, dt, A, B, C, D, z, dt_bias):
    """(states, groups) of a scan call; x, dt, z share a shape, B and C are [.., G, n]."""
    lead, ch = x.shape[:-1], x.shape[-1]
    _tensor("x", x, x.shape, x.dtype, x)
    _tensor("dt", dt, x.shape, x.dtype, x)
    if A.dim() != 2 or A.shape[0] != ch:
        raise ValueError(f"A shape {tuple(A.shape)} != expected [{ch}, n]")
    n = A.shape[1]
    if not 1 <= n <= 128:
        raise ValueError(f"{what}: {n} states: expected 1 to 128")
    _dense("A", A, (ch, n), torch.float32, x)
    G = B.shape[-2] if B.dim() == x.dim() + 1 else 1
    if G < 1 or ch % G:
        raise ValueError(f"{what}: {ch} channels do not divide into {G} groups")
    shape = (*lead, G, n) if B.dim() == x.dim() + 1 else (*lead, n)
    _tensor("B", B, shape, x.dtype, x)
    _tensor("C", C, shape, x.dtype, x)
    if D is not None:
        _dense("D", D, (ch,), torch.float32, x)
    if z is not None:
        _tensor("z", z, x.shape, x.dtype, x)
    if dt_bias is not None:
        _dense("dt_bias", dt_bias, (ch,), torch.float32, x)
    return n, G


def _group_stride(t: torch.Tensor, x: torch.Tensor) -> int:
    return t.stride(-2) if t.dim() == x.dim() + 1 else 0


def ssm_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
             *, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
             dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = True,
             initial_state: Optional[torch.Tensor] = None,
             cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None,
             output_final_state: bool = True, out: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Selective state space scan over prompts, in fp32. With ``dt' = softplus(dt + dt_bias)``
    (``dt + dt_bias`` with dt_softplus=False) and channel d reading group ``d * G // D``:

      h[t, d, k] = exp(dt'[t, d] A[d, k]) h[t - 1, d, k] + dt'[t, d] x[t, d] B[t, g, k]
      y[t, d]    = (sum_k C[t, g, k] h[t, d, k] + D[d] x[t, d]) * silu(z[t, d])

    x, dt, z [N, T, D], or [T, D] with cu_seqlens; B, C [.., G, n] or [.., n]; all of one
    type (f16 / bf16 / f32), tokens may be strided. A [D, n], D [D], dt_bias [D] fp32, n up
    to 128. initial_state [N, D, n] fp32 (zeros without it). max_seqlen: an upper bound of
    the packed lengths, used to plan the launch (a wrong one costs time; results differ by rounding).
    A token's decay below 2^-126 is zero. Returns (y, final_state): y like x and the states after each sequence, [N, D, n] fp32
    (None with output_final_state=False). ``out`` receives y."""
    flags = bool(dt_softplus) | bool(output_final_state) << 1 | min(max_seqlen or 0, _INT_MAX) << 2
    call = (_SCAN, flags, x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens)
    if out is None:
        r = _run(*call)
        if r is not None:
            return r
    packed, N, T, ch = _prompt("ssm_scan", x, cu_seqlens)
    dtc = nv.dtype_code(x.dtype)
    n, G = _scan_weights("ssm_scan", x, dt, A, B, C, D, z, dt_bias)
    if initial_state is not None:
        _dense("initial_state", initial_state, (N, ch, n), torch.float32, x)
    if max_seqlen is not None and max_seqlen < 0:
        raise ValueError(f"ssm_scan: max_seqlen {max_seqlen}")
    _no_backward("ssm_scan", x, dt, A, B, C, D, z, dt_bias, initial_state, out)
    if out is not None:
        _tensor("out", out, x.shape, x.dtype, x)
        _apart("ssm_scan", out, x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens)
    _cuda("ssm_scan", x)
    ys = _dense_strides(x) if out is None else _strides(out, packed)
    p = nv.SsmScanParams(*_strides(x, packed), *_strides(dt, packed), *_strides(z, packed), *ys,
                         *_strides(B, packed), _group_stride(B, x), *_strides(C, packed),
                         _group_stride(C, x), N, T, ch, n, G, dtc, bool(dt_softplus), packed,
                         out is None, min(max_seqlen or 0, T))
    need = nv.lib().ptof_ssm_scan_ws_bytes(_byref(p))
    if need < 0:
        raise _failed(nv.EINVAL)
    outs = ((x.shape, x.dtype), ((N, ch, n), torch.float32))[:1 + bool(output_final_state)]
    final = 1 if output_final_state else _NULL
    return _launch(call, "ptof_ssm_scan_exec", p,
                   (0, 1, 2, 3, 4, 5, 6, 7, 9, 8, _OUT, _OUT + 1 if output_final_state else _NULL,
                    _SCRATCH, _SCRATCH_BYTES), outs, (0, final), scratch=need, out=out)


def ssm_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                  C: torch.Tensor, state: torch.Tensor, *, D: Optional[torch.Tensor] = None,
                  z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                  dt_softplus: bool = True, slots: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``ssm_scan`` for single tokens: x, dt, z [M, D], B, C [M, G, n] or [M, n]; state
    [slots, D, n] fp32 (``ssm_scan``'s final state), updated in place. Returns y [M, D];
    ``out`` may be x, dt or z."""
    call = (_SCAN_STEP, bool(dt_softplus), x, dt, A, B, C, state, D, z, dt_bias, slots)
    if out is None:
        r = _run(*call)
        if r is not None:
            return r[0]
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"ssm_scan_step: x shape {tuple(x.shape)}: expected [M, D]")
    M, ch = x.shape
    dtc = nv.dtype_code(x.dtype)
    n, G = _scan_weights("ssm_scan_step", x, dt, A, B, C, D, z, dt_bias)
    if state.dim() != 3:
        raise ValueError(f"state shape {tuple(state.shape)} != expected [slots, {ch}, {n}]")
    S = state.shape[0]
    _sizes("ssm_scan_step", M, ch, S)
    _tensor("state", state, (S, ch, n), torch.float32, x)
    if S and not state[0].is_contiguous():
        raise ValueError("state must be contiguous within a slot")
    _slots("ssm_scan_step", slots, M, S, x)
    _no_backward("ssm_scan_step", x, dt, A, B, C, state, D, z, dt_bias, out)
    if out is not None:
        _tensor("out", out, x.shape, x.dtype, x)
        one = [t for t in (x, dt, z)
               if t is None or t.data_ptr() != out.data_ptr() or t.stride() != out.stride()]
        _apart("ssm_scan_step", out, *one, A, B, C, state, D, dt_bias, slots)
    _state_apart("ssm_scan_step", state, x, dt, A, B, C, D, z, dt_bias, slots)
    _cuda("ssm_scan_step", x)
    p = nv.SsmScanStepParams(x.stride(0), dt.stride(0), z.stride(0) if z is not None else 0,
                             ch if out is None else out.stride(0), B.stride(0),
                             _group_stride(B, x), C.stride(0), _group_stride(C, x),
                             state.stride(0), M, S, ch, n, G, dtc, bool(dt_softplus))
    return _launch(call, "ptof_ssm_scan_step_exec", p, (0, 1, 2, 3, 4, 6, 7, 8, 9, 5, _OUT),
                   ((x.shape, x.dtype),), (0,), out=out, writes=5)[0]


# --------------------------------------------------------------------------- norm ----
_EPS: Dict[float, int] = {}          # eps of late, each by a number that no other one gets
_EPS_MOST = 256
_EPS_NUMBERS = itertools.count()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[.., D] as [rows, D]: a view where the leading dimensions have one stride, else a copy."""
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 *, eps: float = 1e-6, out_dtype=None, group_size: Optional[int] = None
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Root-mean-square norm with the residual's addition:
    ``h = x + residual`` and ``y = h * rsqrt(mean(h^2) + eps) * weight`` over the last
    dimension, with h kept in fp32 for the norm.

    x [.., D] f16 / bf16 / f32; residual like x, in x's type or fp32; weight [D] in x's type
    or fp32. out_dtype None: y in x's type. ``torch.float8_e4m3fn``: y holds y / scale with
    ``scale = max(amax |y| / 448, 2^-126)`` over each row, or over each ``group_size`` (32, 64
    or 128) columns, the last group of a row possibly shorter (the codes are those of the
    quotient by the scale that is returned, rounded once before it is rounded to 8 bits).
    Returns (y, h, scale): h rounded once to the residual's type (None without a residual),
    scale fp32 [.., 1] or [.., ceil(D / group_size)] (None without an 8-bit output)."""
    if type(eps) is not float:
        eps = float(eps)             # a tensor's value, not the tensor, belongs to a signature
    if not eps >= 0.0:
        raise ValueError(f"add_rms_norm: eps {eps}")
    fp8 = out_dtype is not None and out_dtype != x.dtype
    plain = group_size is None or type(group_size) is int and 0 < group_size <= 128
    flags = -1
    if plain and (not fp8 or out_dtype == torch.float8_e4m3fn):
        number = _EPS.get(eps)
        if number is None:           # two threads take two numbers, one of them stays
            if len(_EPS) >= _EPS_MOST:
                _EPS.clear()
            number = _EPS.setdefault(eps, next(_EPS_NUMBERS))
        flags = number << 10 | (group_size or 0) << 1 | fp8
    call = (_NORM, flags, x, weight, residual)
    if flags >= 0:
        r = _run(*call)
        if r is not None:
            return r
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"add_rms_norm: x shape {tuple(x.shape)}: expected [.., D]")
    D = x.shape[-1]
    dt = nv.dtype_code(x.dtype)
    _tensor("x", x, x.shape, x.dtype, x)
    wd = _weight_dtype("weight", weight, x)
    _dense("weight", weight, (D,), wd, x)
    rd = dt
    if residual is not None:
        rt = _weight_dtype("residual", residual, x)
        _tensor("residual", residual, x.shape, rt, x)
        rd = nv.dtype_code(rt)
    if fp8 and out_dtype != torch.float8_e4m3fn:
        raise TypeError(f"add_rms_norm: out_dtype {out_dtype}: expected {x.dtype} or "
                        "torch.float8_e4m3fn")
    if group_size is not None and (not fp8 or group_size not in (32, 64, 128)):
        raise ValueError(f"add_rms_norm: group_size {group_size}: 32, 64 or 128 with an 8-bit "
                         "output")
    _no_backward("add_rms_norm", x, weight, residual)
    _cuda("add_rms_norm", x)
    xr = _rows(x)
    rr = None if residual is None else _rows(residual)
    M = xr.shape[0]
    _sizes("add_rms_norm", M, D)
    outs = [(x.shape, torch.float8_e4m3fn if fp8 else x.dtype)]
    args, results = [0, 2, 1, _OUT, _NULL, _NULL], [0, _NULL, _NULL]
    if residual is not None:
        args[4], results[1] = _OUT + len(outs), len(outs)
        outs.append((x.shape, residual.dtype))
    if fp8:
        args[5], results[2] = _OUT + len(outs), len(outs)
        outs.append(((*x.shape[:-1], -(-D // group_size) if group_size else 1), torch.float32))
    p = nv.AddRmsNormParams(xr.stride(0), rr.stride(0) if rr is not None else 0, D, D, M, D, dt,
                            rd, nv.dtype_code(wd), fp8, group_size or 0, eps)
    # rows that had to be copied together lie elsewhere in each call: no plan
    moved = xr.data_ptr() != x.data_ptr() or \
        rr is not None and rr.data_ptr() != residual.data_ptr()
    return _launch((_NORM, flags, xr, weight, rr) if moved else call, "ptof_add_rms_norm_exec", p,
                   tuple(args), tuple(outs), tuple(results), keep=not moved)
