"""Gated linear recurrence on the HIP library: whole sequences, their backward pass, and one position at a time.

    a_t = sigmoid(f_t)      h_t = a_t h_{t-1} + (1 - a_t) z_t      y_t = sigmoid(o_t) h_t   (y_t = h_t without o)

The gates do not depend on h, so a sequence is a scan that runs in parallel over time; the LSTM and GRU cells of
``modules`` / ``rnn_impl`` need a hop for every step.  z, f and o are what a projection of the layer's input gives (slices of one
[B, T, 3H] product need no copy).  fp32, bf16 and fp16; gates, state and sums are fp32, results are rounded once.

``ctx`` is a Context, an Engine, or None: torch's current stream on the tensors' device.  Nothing here synchronises, and every
call can be captured into a graph (lengths on the host are refused there: they have to be copied first).

Like the rest of this package these calls are outside torch's autograd: results carry no history whatever their inputs require, and a
state that is updated in place gets no new version.  ``gated_scan_backward`` gives the gradients; hand them on to whatever made z, f
and o.  B is at most 65535, T 2^30, H 2^24, and a call at most 2^32 threads."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import numpy as np
import torch

from . import _lib
from .engine import Context, stream_context

_DTYPES = {torch.float32: _lib.T2_F32, torch.bfloat16: _lib.T2_BF16, torch.float16: _lib.T2_F16}


class ScanTape(NamedTuple):
    """What ``gated_scan_backward`` needs of a forward call: its inputs (not copied: leave them as they are until then) and the
    states in front of every 64th step.  A backward pass on another stream (which the caller orders behind the forward call) keeps
    their memory from being given away before that stream is done with it, so the tape can be dropped at once."""
    z: torch.Tensor
    f: torch.Tensor
    o: Optional[torch.Tensor]
    lens: Optional[torch.Tensor]
    reverse: bool
    states: torch.Tensor
    stream: Optional[int] = None          # the forward call's: torch's current stream then

    def _used(self):
        if self.stream is None or torch._C._cuda_getCurrentRawStream(self.states.get_device()) != self.stream:
            for t in (self.z, self.f, self.o, self.lens, self.states):
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(self.states.device))


def _context(ctx, t: torch.Tensor) -> Context:
    if ctx is None:
        return stream_context(t.get_device())
    ctx = ctx if isinstance(ctx, Context) else ctx.context
    if ctx.device != t.device:
        raise ValueError(f"tensors on {t.device}, context on {ctx.device}")
    return ctx


def _sequence(what: str, t, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what} must be a device tensor")
    if like is None:
        if t.dim() != 3 or t.dtype not in _DTYPES or 0 in t.shape:
            raise ValueError(f"{what} must be a non-empty [B, T, H] tensor of float32, bfloat16 or float16, got {t.dtype} {tuple(t.shape)}")
    elif t.dtype is not like.dtype or t.shape != like.shape or t.get_device() != like.get_device():
        raise ValueError(f"{what} must be {like.dtype} {tuple(like.shape)} on {like.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"the channels of {what} must be contiguous")
    return t


def _output(what: str, t, like: torch.Tensor) -> torch.Tensor:
    if t is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    _sequence(what, t, like)
    B, T, H = t.shape
    sb, st = t.stride(0), t.stride(1)
    by_row = (T == 1 or st >= H) and (B == 1 or sb >= (T - 1) * st + H)
    by_time = (B == 1 or sb >= H) and (T == 1 or st >= (B - 1) * sb + H)
    if not (by_row or by_time):
        raise ValueError(f"the elements of {what} overlap (strides {t.stride()})")
    return t


def _rows(what: str, t, B: int, H: int, device) -> torch.Tensor:
    if not (isinstance(t, torch.Tensor) and t.device == device and t.dtype == torch.float32 and tuple(t.shape) == (B, H)):
        raise ValueError(f"{what} must be a float32 [{B}, {H}] tensor on {device}")
    return t.contiguous()


def _lengths(lens, B: int, T: int, device) -> Optional[torch.Tensor]:
    if lens is None:
        return None
    if isinstance(lens, torch.Tensor) and lens.is_cuda:
        if tuple(lens.shape) != (B,) or lens.device != device or lens.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"lens must be an int64 or int32 [{B}] tensor on {device}")
        return lens if lens.dtype is torch.int64 and lens.is_contiguous() else lens.to(torch.int64).contiguous()
    host = np.asarray(lens)
    if host.shape != (B,) or host.dtype.kind not in "iu" or (host < 0).any() or (host > T).any():
        raise ValueError(f"lens must be {B} whole numbers from 0 to {T}")
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("lens on the host cannot be captured into a graph (the graph would keep this call's): copy them to the device first")
    # through pinned memory: a copy out of any other waits for all the work in front of it
    pinned = torch.empty(B, dtype=torch.int64, pin_memory=True)
    pinned.numpy()[:] = host
    return pinned.to(device, non_blocking=True)


_NONE = (0, 0, 0)


def _seq(t: Optional[torch.Tensor]):
    return _NONE if t is None else (t.data_ptr(), *t.stride()[:2])


def _ptr(t: Optional[torch.Tensor]):
    return 0 if t is None else t.data_ptr()


def _workspace(ctx: Context, B: int, T: int, H: int) -> Tuple[Optional[torch.Tensor], int]:
    # a tensor of the call's own: a captured call's workspace is its graph's
    n = ctx.lib.t2_gated_scan_ws(B, T, H)
    if n < 0:
        _lib.check(_lib.T2_EINVAL)
    return (torch.empty(n, dtype=torch.uint8, device=ctx.device), n) if n else (None, 0)


def gated_scan(ctx, z, f, o=None, lens=None, state=None, reverse: bool = False, tape: bool = False, out=None):
    """y [B, T, H] and the final state [B, H] (fp32) of the recurrence over z, f (and o) [B, T, H]; with ``tape`` also the ScanTape of
    the backward pass.

    Any batch and time strides (time-major views, slices of a projection, broadcast inputs), contiguous channels.  ``lens`` [B]: row b
    has positions 0 .. lens[b] - 1; the others give y = 0 and do not touch the state.  Host lengths outside [0, T] raise, device
    lengths are taken as the nearest.  ``reverse`` runs every row from its last position to its first.  ``state``: the state in
    front of the first step (fp32 [B, H], default zeros).  ``out`` takes y (a [B, T, H] view; it must not overlap z, f, o or lens; a state that
    lies in it, such as the last row of the chunk before, is copied first)."""
    _sequence("z", z)
    B, T, H = z.shape
    _sequence("f", f, z)
    if o is not None:
        _sequence("o", o, z)
    ctx = _context(ctx, z)
    device = z.device
    if state is not None:
        state = _rows("state", state, B, H, device)
    lens = _lengths(lens, B, T, device)
    y = _output("out", out, z)
    if state is not None and out is not None:
        begin, end = y.data_ptr(), y.data_ptr() + ((B - 1) * y.stride(0) + (T - 1) * y.stride(1) + H) * y.element_size()
        if state.data_ptr() < end and state.data_ptr() + 4 * B * H > begin:
            state = state.clone()
    final = torch.empty_like(state) if state is not None else torch.empty((B, H), dtype=torch.float32, device=device)
    states = torch.empty((B, -(-T // _lib.T2_SCAN_SPAN), H), dtype=torch.float32, device=device) if tape else None
    ws, n = _workspace(ctx, B, T, H)
    args = _lib.T2ScanArgs.from_buffer_copy(_lib.SCAN_ARGS.pack(_DTYPES[z.dtype], B, T, H, 1 if reverse else 0, *_seq(z), *_seq(f), *_seq(o), *_seq(y), _ptr(lens), _ptr(state),
                               final.data_ptr(), _ptr(states), *_NONE, *_NONE, *_NONE, *_NONE, 0, 0, _ptr(ws), n))
    with ctx.ordered():
        _lib.check(ctx.lib.t2_gated_scan(ctx.handle, args))
    return (y, final, ScanTape(z, f, o, lens, bool(reverse), states, torch._C._cuda_getCurrentRawStream(device.index))) if tape else (y, final)


def gated_scan_backward(ctx, tape: ScanTape, dy, dfinal=None):
    """(dz, df, do, dstate): the gradients of the tape's inputs and of the state in front of the first step, for dy [B, T, H] (any
    batch and time strides) and dfinal [B, H] (fp32, the gradient of the final state, default zeros).  ``do`` is None without an
    output gate.  Positions behind a row's length get zeros.  An input that was broadcast gets the gradient of every place it went
    to: sum it over that axis.  A tape serves any number of backward passes."""
    z = tape.z
    B, T, H = z.shape
    _sequence("dy", dy, z)
    ctx = _context(ctx, z)
    device = z.device
    if dfinal is not None:
        dfinal = _rows("dfinal", dfinal, B, H, device)
    dz, df = _output("dz", None, z), _output("df", None, z)
    do = None if tape.o is None else _output("do", None, z)
    dstate = torch.empty_like(dfinal) if dfinal is not None else torch.empty((B, H), dtype=torch.float32, device=device)
    ws, n = _workspace(ctx, B, T, H)
    args = _lib.T2ScanArgs.from_buffer_copy(_lib.SCAN_ARGS.pack(_DTYPES[z.dtype], B, T, H, int(tape.reverse), *_seq(z), *_seq(tape.f), *_seq(tape.o), *_NONE, _ptr(tape.lens), 0, 0,
                               tape.states.data_ptr(), *_seq(dy), *_seq(dz), *_seq(df), *_seq(do), _ptr(dfinal), dstate.data_ptr(), _ptr(ws), n))
    tape._used()
    with ctx.ordered():
        _lib.check(ctx.lib.t2_gated_scan_backward(ctx.handle, args))
    return dz, df, do, dstate


def gated_scan_step(ctx, z, f, o, state, active=None, out=None):
    """One new position for every row: z, f, o (or None) [B, H] -> y [B, H]; ``state`` [B, H] (fp32) is updated in place.  Rows where
    ``active`` (bool [B] on the device) is False keep their state and get y = 0.  ``out`` takes y; it may be z, f or o itself."""
    if not (isinstance(z, torch.Tensor) and z.is_cuda and z.dim() == 2 and z.dtype in _DTYPES and z.numel()):
        raise ValueError("z must be a non-empty [B, H] device tensor of float32, bfloat16 or float16")
    B, H = shape = z.shape
    dtype, at = z.dtype, z.get_device()
    zs, fs, os = _row_stride("z", z, shape, dtype, at), _row_stride("f", f, shape, dtype, at), 0 if o is None else _row_stride("o", o, shape, dtype, at)
    ss = _row_stride("state", state, shape, torch.float32, at)
    if active is not None:
        if not (isinstance(active, torch.Tensor) and active.get_device() == at and active.dtype == torch.bool and active.shape == shape[:1]):
            raise ValueError(f"active must be a bool [{B}] tensor on {z.device}")
        active = active.contiguous()
    ctx = _context(ctx, z)
    if out is None:
        y, ys = torch.empty_like(z, memory_format=torch.contiguous_format), H
    else:
        y, ys = out, _row_stride("out", out, shape, dtype, at)
    with ctx.ordered():
        _lib.check(ctx.lib.t2_gated_scan_step(ctx.handle, _DTYPES[dtype], B, H, z.data_ptr(), zs, f.data_ptr(), fs, 0 if o is None else o.data_ptr(), os,
                                              state.data_ptr(), ss, 0 if active is None else active.data_ptr(), y.data_ptr(), ys))
    return y


def _row_stride(what: str, t, shape, dtype, at: int) -> int:
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == at:
        row, col = t.stride()
        if col == 1 or shape[1] == 1:
            return row
    raise ValueError(f"{what} must be a {dtype} {tuple(shape)} tensor on cuda:{at} with contiguous rows")
