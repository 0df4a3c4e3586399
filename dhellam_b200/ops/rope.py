"""Rotary position embedding.

The reference uses learned absolute positions (dhellam/core/dshb.py:250-255); RoPE is
needed for the Llama family.  Two forms:

* ``rope_apply_`` rotates the Q and K heads of a packed QKV buffer in place, whole heads with pairs ``(i, i + d/2)`` and
  angles from a table (``rope_table``).  Layout of one row of ``qkv``: ``[nq heads x d | nkv heads x d | nkv heads x d]``.
* ``rope_fwd`` / ``rope_bwd`` rotate separate (strided) queries and keys, out of place or in place: pairs in halves or
  interleaved, the whole head or its first part, any position, frequencies from ``rope_frequencies``, which also states
  the ways in which models are stretched to longer contexts than they were first trained on.
"""
from __future__ import annotations

import math
import struct
from ctypes import c_int, c_void_p
from dataclasses import dataclass

import torch

from .. import kernels as K


def rope_table(max_pos: int, d: int, theta: float, device="cpu"):
    """Returns ``(cos, sin)``, each ``[max_pos, d/2]`` fp32."""
    inv = 1.0 / (theta ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float().to(device), ang.sin().float().to(device)


def rope_apply_(qkv, positions, cos, sin, nq: int, nkv: int, d: int, inverse: bool = False, sm_budget: int = 0, stream=None):
    """Rotates the first ``nq + nkv`` heads of every row of ``qkv [T, (nq+2nkv)*d]`` in place.

    ``positions [T]`` int32 gives the sequence position of each row.  ``inverse`` applies
    the transposed rotation, which is the backward of the forward rotation.
    """
    T = qkv.shape[0]
    assert qkv.shape[1] == (nq + 2 * nkv) * d
    if not K.use_native(qkv):
        v = qkv[:, : (nq + nkv) * d].float().view(T, nq + nkv, d)
        c = cos[positions.long()][:, None, :]
        s = sin[positions.long()][:, None, :]
        if inverse:
            s = -s
        x1, x2 = v[..., : d // 2], v[..., d // 2:]
        r = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)
        qkv[:, : (nq + nkv) * d] = r.view(T, -1).to(qkv.dtype)
        return qkv
    fn = K.proto("dh_rope_inplace", [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int,
                                     c_void_p])
    K.check(fn(qkv.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), T, qkv.stride(0), nq + nkv, d,
               1 if inverse else 0, sm_budget, K.stream_ptr(stream)), "dh_rope_inplace")
    return qkv


# ----------------------------------------------------------------------------- separate heads, other layouts, longer contexts
@dataclass(frozen=True)
class RopeScaling:
    """How the frequencies of a model first trained on ``original_max_position`` positions are stretched ``factor`` times.

    * ``linear``: every frequency divided by ``factor`` (positions interpolated);
    * ``ntk``: the base raised so that the slowest pair is divided by ``factor`` and the fastest stays;
    * ``llama3``: pairs that turn at least ``high_freq_factor`` times within the original length stay, pairs that turn at most
      ``low_freq_factor`` times are divided by ``factor``, linear in the number of turns in between;
    * ``yarn``: the same with a ramp over the pair's index between the pairs of ``beta_fast`` and ``beta_slow`` turns, and
      cosines and sines multiplied by ``attention_factor`` (default ``0.1 ln(factor) + 1``)."""
    kind: str = "linear"
    factor: float = 1.0
    original_max_position: int = 8192
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "llama3", "yarn"):
            raise ValueError(f"unknown rotary scaling {self.kind!r}: linear, ntk, llama3 or yarn")
        if not self.factor >= 1.0 or self.original_max_position <= 0:
            raise ValueError("rotary scaling needs a factor of at least 1 and a positive original length")
        if self.kind == "llama3" and not self.high_freq_factor > self.low_freq_factor > 0:
            raise ValueError("llama3 scaling needs high_freq_factor > low_freq_factor > 0")
        if self.kind == "yarn" and not self.beta_fast > self.beta_slow > 0:
            raise ValueError("yarn scaling needs beta_fast > beta_slow > 0")


def rope_frequencies(rotary_dim: int, theta: float, scaling: RopeScaling | None = None, device="cpu"):
    """``(frequencies [rotary_dim / 2] fp64, scale)``: radians per position of every pair, and the factor on cosines and sines."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"the rotated part of a head has an even number of elements, not {rotary_dim}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    freq, scale = float(theta) ** -i, 1.0
    s = scaling
    if s is not None and s.kind == "linear":
        freq = freq / s.factor
    elif s is not None and s.kind == "ntk":
        freq = (float(theta) * s.factor ** (rotary_dim / max(rotary_dim - 2, 1))) ** -i
    elif s is not None and s.kind == "llama3":
        turns = s.original_max_position * freq / (2 * math.pi)
        keep = ((turns - s.low_freq_factor) / (s.high_freq_factor - s.low_freq_factor)).clamp(0.0, 1.0)
        freq = freq * keep + freq / s.factor * (1.0 - keep)
    elif s is not None:
        def index_of(turns):                 # the (fractional) pair that turns so often within the original length
            return rotary_dim * math.log(s.original_max_position / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo = max(math.floor(index_of(s.beta_fast)), 0)
        hi = min(math.ceil(index_of(s.beta_slow)), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        freq = freq / s.factor * ramp + freq * (1.0 - ramp)
        scale = s.attention_factor if s.attention_factor is not None else 0.1 * math.log(s.factor) + 1.0
    return freq.to(device), scale


def _turn_ref(x, positions, freq, interleaved, scale, transposed):
    r = 2 * freq.numel()
    angle = positions.to(torch.float64).unsqueeze(-1) * freq.to(torch.float64)
    cos, sin = (angle.cos() * scale).float().unsqueeze(-2), (angle.sin() * scale).float().unsqueeze(-2)
    if transposed:
        sin = -sin
    y = x.float().clone()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2:r])
    c, d = a * cos - b * sin, b * cos + a * sin
    a.copy_(c), b.copy_(d)
    return y.to(x.dtype)


# The operands of the kernel as one block of 8-byte fields (RopeCall in csrc/rope.cu): ctypes converts argument by argument, which takes
# several microseconds where a small call has 15 in all.
_ROPE_CALL = struct.Struct("=30qd")
_ROPE_ARGS = [c_void_p]
_TYPES = (torch.bfloat16, torch.float32)
_POSITIONS = (torch.int32, torch.int64)


def _fits(x, lead, d, dtype):
    return x.dim() in (3, 4) and x.shape[:-2] == lead and x.shape[-1] == d and x.dtype == dtype and (x.stride(-1) == 1 or d == 1)


def _disjoint(a, b=None):
    """Whether the heads of ``a`` (and of ``b``, of as many rows in the same memory) are all apart: rows of equal strides in which the heads
    of both follow one another, inside, between or around the row dimensions.  Unusual strides that no such nesting has count as overlapping."""
    if a.dim() == 3:                                     # packed rows, the heads of a row within its stride: what a training step has
        (_, heads, d), (row, step, _) = a.shape, a.stride()
        end = step * (heads - 1) + d
        if b is None:
            if step >= d and end <= row:
                return True
        elif step >= d:
            more, (row_b, step_b, _), at = b.shape[1], b.stride(), (b.data_ptr() - a.data_ptr()) // a.element_size()
            if row_b == row and step_b >= d and at >= end and at + step_b * (more - 1) + d <= row:
                return True
    if a.numel() == 0 or (b is not None and b.numel() == 0):
        return True
    rows = sorted((st, n) for st, n in zip(a.stride()[:-2], a.shape[:-2]) if n > 1)
    steps = [(0, a.stride(-2), a.shape[-2])]
    if b is not None:
        size, first = a.element_size(), a.data_ptr()
        spans = [sum(st * (n - 1) for st, n in zip(x.stride(), x.shape)) * size + size for x in (a, b)]
        if first + spans[0] <= b.data_ptr() or b.data_ptr() + spans[1] <= first:
            return True
        if sorted((st, n) for st, n in zip(b.stride()[:-2], b.shape[:-2]) if n > 1) != rows or (b.data_ptr() - first) % size:
            return False
        steps.append(((b.data_ptr() - first) // size, b.stride(-2), b.shape[-2]))
        steps.sort()
    for inner in range(len(rows) + 1):                   # row dimensions inside the heads
        extent, fits = a.shape[-1], True
        for i in range(len(rows) + 1):
            if i == inner:
                if all(n == 1 or st >= extent for _, st, n in steps) and (
                        len(steps) == 1 or steps[0][0] + steps[0][1] * (steps[0][2] - 1) + extent <= steps[1][0]):
                    extent += max(at + st * (n - 1) for at, st, n in steps) - steps[0][0]
                else:                                    # heads of both in turn
                    starts = sorted(at + st * h for at, st, n in steps for h in range(n))
                    fits &= all(y - x >= extent for x, y in zip(starts, starts[1:]))
                    extent += starts[-1] - starts[0]
            if i < len(rows):
                st, n = rows[i]
                fits &= st >= extent
                extent += st * (n - 1)
        if fits:
            return True
    return False


def _check(q, k, positions, freq, out, what):
    lead, d = q.shape[:-2], q.shape[-1] if q.dim() else 0
    if positions.shape != lead or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: one int32 or int64 position for each of {tuple(lead)} rows, got {positions.dtype} {tuple(positions.shape)}")
    if freq.dtype != torch.float64 or freq.dim() != 1 or not 0 < 2 * freq.numel() <= d:
        raise ValueError(f"{what}: fp64 frequencies of at most half of the {d} elements of a head, got {freq.dtype} {tuple(freq.shape)}")
    inputs = (q,) if k is None else (q, k)
    for x in inputs:
        if not _fits(x, lead, d, q.dtype):
            raise ValueError(f"{what}: queries and keys are [rows..., heads, {d}] of one type, with elements side by side")
    if out is None:
        return
    for x, o in zip(inputs, out):
        if o.shape != x.shape or not _fits(o, lead, d, q.dtype) or not _disjoint(o):
            raise ValueError(f"{what}: an output has its input's shape and type, room for every row and head and elements side by side")
        in_place = o.data_ptr() == x.data_ptr() and o.stride() == x.stride()
        if not in_place and any(o.untyped_storage().data_ptr() == y.untyped_storage().data_ptr() for y in inputs):
            raise ValueError(f"{what}: an output is its own input or shares no memory with the inputs")
    if k is not None:
        oq, ok = out
        # an output that is its own input may still share heads with the other one
        for a, b in ((oq, ok),) + (() if ok is k else ((oq, k),)) + (() if oq is q else ((q, ok),)):
            if a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr() and not _disjoint(a, b):
                raise ValueError(f"{what}: an output shares no heads with the other one, nor with its input")


def _strides(x):
    s = x.stride()
    return s[:3] if len(s) == 4 else (s[0], 0, s[1])


def _turn(q, k, positions, freq, interleaved, scale, out, transposed, sm_budget, stream, what):
    if stream is not None:
        operands = (q, k, positions, freq) + (tuple(out) if out is not None else ())
        return K.run_on_stream(stream, operands, lambda: _turn(q, k, positions, freq, interleaved, scale, out, transposed, sm_budget,
                                                               None, what))
    shape, dtype, pairs = q.shape, q.dtype, freq.numel()
    if out is not None or k is None or len(shape) != 3 or not K.use_native(q):
        return _turn_any(q, k, positions, freq, interleaved, scale, out, transposed, sm_budget, what)
    # packed rows on the GPU, outputs of their own: what `_turn_any` checks, asked once
    T, heads, d = shape
    kshape, (sq, hq, cq), (sk, hk, ck) = k.shape, q.stride(), k.stride() if k.dim() == 3 else (0, 0, 0)
    device, pos_type = q.get_device(), positions.dtype
    if not (dtype in _TYPES and k.dtype is dtype and cq == 1 and ck == 1 and kshape[0] == T and kshape[2] == d and positions.shape == (T,)
            and pos_type in _POSITIONS and freq.dtype is torch.float64 and freq.dim() == 1 and 0 < 2 * pairs <= d
            and device == k.get_device() == positions.get_device() == freq.get_device() == torch._C._cuda_getDevice()
            and positions.is_contiguous() and freq.is_contiguous()):
        return _turn_any(q, k, positions, freq, interleaved, scale, out, transposed, sm_budget, what)
    kv = kshape[1]
    oq = torch.empty_like(q, memory_format=torch.contiguous_format)
    ok = torch.empty_like(k, memory_format=torch.contiguous_format)
    call = _ROPE_CALL.pack(q.data_ptr(), oq.data_ptr(), k.data_ptr(), ok.data_ptr(), sq, 0, hq, heads * d, 0, d, sk, 0, hk, kv * d, 0, d, heads,
                           kv, positions.data_ptr(), pos_type is torch.int64, freq.data_ptr(), T, 1, d, 2 * pairs, bool(interleaved),
                           dtype is torch.float32, transposed, sm_budget, torch._C._cuda_getCurrentRawStream(device), scale)
    K.check(K.proto("dh_rope_heads", _ROPE_ARGS)(call), "dh_rope_heads")
    return oq, ok


def _turn_any(q, k, positions, freq, interleaved, scale, out, transposed, sm_budget, what):
    _check(q, k, positions, freq, out, what)
    oq, ok = out if out is not None else (None, None)
    if not K.use_native(q):
        rq = _turn_ref(q, positions, freq, interleaved, scale, transposed)
        rk = _turn_ref(k, positions, freq, interleaved, scale, transposed) if k is not None else None
        return (rq, rk) if out is None else (oq.copy_(rq), ok.copy_(rk) if k is not None else None)
    shape, dtype = q.shape, q.dtype
    if dtype not in _TYPES:
        raise ValueError(f"{what}: the sm_100a kernel rotates bf16 and fp32, not {dtype}")
    K.require_current_device(what, q, k, positions, freq, oq, ok)
    if not positions.is_contiguous() or not freq.is_contiguous():
        raise ValueError(f"{what}: positions and frequencies must be contiguous")
    if oq is None:
        oq = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is None:
        ok, heads_k, keys, key_strides = None, 0, (0, 0), (0, 0, 0, 0, 0, 0)
    else:
        if ok is None:
            ok = torch.empty_like(k, memory_format=torch.contiguous_format)
        heads_k, keys, key_strides = k.shape[-2], (k.data_ptr(), ok.data_ptr()), _strides(k) + _strides(ok)
    call = _ROPE_CALL.pack(q.data_ptr(), oq.data_ptr(), *keys, *_strides(q), *_strides(oq), *key_strides, shape[-2], heads_k,
                           positions.data_ptr(), positions.dtype == torch.int64, freq.data_ptr(), positions.numel(),
                           1 if len(shape) == 3 else shape[1] or 1, shape[-1], 2 * freq.numel(), bool(interleaved), dtype == torch.float32,
                           transposed, sm_budget, K.current_raw_stream(), scale)
    K.check(K.proto("dh_rope_heads", _ROPE_ARGS)(call), "dh_rope_heads")
    return oq, ok


def rope_fwd(q, k, positions, freq, interleaved: bool = False, scale: float = 1.0, out=None, sm_budget: int = 0, stream=None):
    """Rotated queries and keys ``(q', k')``.

    ``q [T, Hq, d]`` and ``k [T, Hk, d]`` (packed rows, as ``pymha_varlen_fwd`` takes them) or ``[S, B, heads, d]`` (as
    ``attn_fwd`` does), bf16 or fp32, any strides with the elements of a head side by side; ``k`` may be ``None``.
    ``positions [T]`` (``[S, B]``) int32 or int64, any value.  ``freq [r / 2]`` fp64 and ``scale`` come from
    ``rope_frequencies``: the first ``r`` elements of every head are rotated, as pairs ``(i, i + r/2)`` or, interleaved,
    ``(2i, 2i + 1)``; the others are copied.  ``out = (q', k')`` names the outputs, which may be the inputs themselves; they share
    no heads with one another, nor one's with the other's input."""
    return _turn(q, k, positions, freq, interleaved, scale, out, False, sm_budget, stream, "rope_fwd")


def rope_bwd(dq, dk, positions, freq, interleaved: bool = False, scale: float = 1.0, out=None, sm_budget: int = 0, stream=None):
    """Gradients of the queries and keys that ``rope_fwd`` took, from those of what it gave: the transposed rotation, same arguments."""
    return _turn(dq, dk, positions, freq, interleaved, scale, out, True, sm_budget, stream, "rope_bwd")
