"""Vocabulary-parallel cross-entropy and loss scaling.

The reference computes the loss with three tensor-parallel all-reduces (max, target
logit, sum of exponentials; dhellam/operators/loss.py:15-98, or Megatron's
``vocab_parallel_cross_entropy`` from dhellam/core/dshb.py:106).  Here every rank reduces
its vocabulary shard to four numbers per token ``(local max, sum exp(logit - local max),
target logit or 0, sum of logits)`` in one pass, the ranks exchange those in ONE all-gather,
and each rank combines them locally.  The backward overwrites the logits buffer with
``(softmax - onehot) * grad`` in place.

Label smoothing follows the reference's definition (loss.py:66-88): with ``s' = s V / (V - 1)``
the loss is ``(1 - s') * ce - s' * mean_v(log p_v)``.  The mean runs over the WHOLE vocabulary
here (``mean_v log p_v = sum_v logit_v / V - lse``, which only needs the sum of the logits as a
fourth statistic); the reference takes it over the local partition only, which makes its loss
depend on the tensor-parallel size.
"""
from __future__ import annotations

import struct
from ctypes import c_float, c_int, c_int64, c_void_p

import torch
import torch.distributed as dist

from .. import kernels as K
from .comm import group_size


def ce_local_stats(logits, labels, vocab_start: int, sm_budget: int = 0, stream=None):
    """``stats [T,4] fp32 = (max, sumexp relative to max, target logit if owned else 0, sum of logits)``."""
    T, Vl = logits.shape
    if not K.use_native(logits):
        lf = logits.float()
        m = lf.max(dim=-1).values
        se = torch.exp(lf - m[:, None]).sum(-1)
        loc = labels.long() - vocab_start
        own = (loc >= 0) & (loc < Vl)
        tgt = torch.where(own, lf.gather(1, loc.clamp(0, Vl - 1)[:, None]).squeeze(1), torch.zeros_like(m))
        return torch.stack([m, se, tgt, lf.sum(-1)], dim=1)
    stats = torch.empty((T, 4), dtype=torch.float32, device=logits.device)
    fn = K.proto("dh_ce_stats", [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int64, c_int, c_int, c_int, c_void_p])
    K.check(fn(logits.data_ptr(), labels.data_ptr(), stats.data_ptr(), T, Vl, logits.stride(0), vocab_start,
               int(logits.dtype == torch.float32), sm_budget, K.stream_ptr(stream)), "dh_ce_stats")
    return stats


def _smoothing(label_smoothing: float, vocab: int) -> float:
    if not label_smoothing:
        return 0.0
    assert 0.0 < label_smoothing < 1.0 and vocab > 1
    return label_smoothing * vocab / (vocab - 1)


def ce_combine_stats(all_stats, label_smoothing: float = 0.0, vocab: int = 0):
    """``all_stats [R,T,4]`` -> ``(loss [T], lse [T])``; ``vocab`` = full vocabulary size (needed
    only with label smoothing)."""
    if K.use_native(all_stats) and K.is_plain(all_stats) and all_stats.dim() == 3 and all_stats.shape[0] > 0 and all_stats.shape[2] == 4 \
            and all_stats.is_contiguous() and all_stats.dtype == torch.float32 and all_stats.data_ptr() % 16 == 0:
        R, T, _ = all_stats.shape
        loss = torch.empty(T, dtype=torch.float32, device=all_stats.device)
        lse = torch.empty_like(loss)
        fn = K.proto("dh_ce_combine", [c_void_p, c_int, c_int, c_float, c_float, c_void_p, c_void_p, c_void_p])
        K.check(fn(all_stats.data_ptr(), R, T, _smoothing(label_smoothing, vocab), float(vocab), loss.data_ptr(), lse.data_ptr(),
                   K.stream_ptr()), "dh_ce_combine")
        return loss, lse
    m = all_stats[..., 0]
    gmax = m.max(dim=0).values
    se = (all_stats[..., 1] * torch.exp(m - gmax[None])).sum(0)
    tgt = all_stats[..., 2].sum(0)
    lse = torch.log(se) + gmax
    loss = lse - tgt
    s = _smoothing(label_smoothing, vocab)
    if s:
        mean_log_p = all_stats[..., 3].sum(0) / vocab - lse
        loss = (1.0 - s) * loss - s * mean_log_p
    return loss, lse


def vocab_parallel_ce_fwd(logits, labels, vocab_start: int = 0, group=None, stream=None, label_smoothing: float = 0.0):
    """Returns ``(loss_per_token [T] fp32, lse [T] fp32)``."""
    stats = ce_local_stats(logits, labels, vocab_start, stream=stream)
    ws = group_size(group)
    if ws > 1:
        T = stats.shape[0]
        flat = torch.empty((ws * T, 4), dtype=stats.dtype, device=stats.device)
        dist.all_gather_into_tensor(flat, stats, group=group)
        gathered = flat.view(ws, T, 4)
    else:
        gathered = stats.unsqueeze(0)
    return ce_combine_stats(gathered, label_smoothing, logits.shape[1] * ws)


def vocab_parallel_ce_bwd_(logits, labels, lse, grad_per_token, vocab_start: int = 0, sm_budget: int = 0, stream=None,
                           label_smoothing: float = 0.0, vocab: int = 0):
    """Overwrites ``logits`` with ``d loss / d logits`` and returns it.  With label smoothing pass
    the full vocabulary size as ``vocab``: the gradient is ``softmax - (1 - s') onehot - s' / V``."""
    T, Vl = logits.shape
    s = _smoothing(label_smoothing, vocab)
    tcoef, ucoef = 1.0 - s, (s / vocab if s else 0.0)
    if not K.use_native(logits):
        p = torch.exp(logits.float() - lse[:, None])
        loc = labels.long() - vocab_start
        own = (loc >= 0) & (loc < Vl)
        rows = torch.nonzero(own).squeeze(1)
        p[rows, loc[rows]] -= tcoef
        if ucoef:
            p -= ucoef
        logits.copy_((p * grad_per_token[:, None]).to(logits.dtype))
        return logits
    fn = K.proto("dh_ce_grad_inplace", [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int64, c_int, c_int, c_float,
                                        c_float, c_int, c_void_p])
    K.check(fn(logits.data_ptr(), labels.data_ptr(), lse.data_ptr(), grad_per_token.data_ptr(), T, Vl, logits.stride(0),
               vocab_start, int(logits.dtype == torch.float32), tcoef, ucoef, sm_budget, K.stream_ptr(stream)), "dh_ce_grad_inplace")
    return logits


# ----------------------------------------------------------------------------- distillation from a teacher's top logits
_TEACHER_TYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
MAX_TEACHER_ENTRIES = 1024
_MIN_TEMPERATURE, _MAX_TEMPERATURE = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def _distill_operands(what, logits, labels, top_ids, top_logits, temperature):
    shape, ids, id_type = logits.shape, top_ids.shape, top_ids.dtype
    if len(shape) == 2 and len(ids) == 2 and ids[0] == shape[0] and top_logits.shape == ids and (id_type is torch.int32 or id_type is torch.int64) \
            and top_logits.dtype in _TEACHER_TYPES and ids[1] <= MAX_TEACHER_ENTRIES and _MIN_TEMPERATURE <= temperature <= _MAX_TEMPERATURE \
            and (labels is None or (labels.dtype is torch.int32 and labels.shape == shape[:1])):
        return
    if logits.dim() != 2 or top_ids.dim() != 2 or top_ids.shape[0] != logits.shape[0] or top_logits.shape != top_ids.shape:
        raise ValueError(f"{what}: logits [T, V], the teacher's ids and logits [T, K], got {tuple(logits.shape)}, {tuple(top_ids.shape)}, "
                         f"{tuple(top_logits.shape)}")
    if top_ids.dtype not in (torch.int32, torch.int64) or top_logits.dtype not in _TEACHER_TYPES or top_ids.shape[1] > MAX_TEACHER_ENTRIES:
        raise ValueError(f"{what}: up to {MAX_TEACHER_ENTRIES} int32 or int64 ids with bf16, fp16 or fp32 logits a row, got "
                         f"{top_ids.shape[1]} of {top_ids.dtype} and {top_logits.dtype}")
    if labels is not None and (labels.shape != logits.shape[:1] or labels.dtype != torch.int32):
        raise ValueError(f"{what}: {logits.shape[0]} int32 labels, got {labels.dtype} {tuple(labels.shape)}")
    if not _MIN_TEMPERATURE <= temperature <= _MAX_TEMPERATURE:
        raise ValueError(f"{what}: the temperature is a positive normal fp32 number, not {temperature}")


def _distill_native(what, logits, labels, top_ids, top_logits, *others):
    """Operands as the kernels of csrc/distill.cu take them."""
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what}: the sm_100a kernel takes bf16 and fp32 logits, not {logits.dtype}")
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError(f"{what}: the logits of a row lie side by side")
    K.require_current_device(what, logits, labels, top_ids, top_logits, *others)
    if labels is not None and not labels.is_contiguous():
        labels = labels.contiguous()
    return labels, top_ids if top_ids.stride(1) == 1 else top_ids.contiguous(), top_logits if top_logits.stride(1) == 1 else top_logits.contiguous()


# The operands of both kernels as one block of 8-byte fields (DistillCall in csrc/distill.cu): ctypes converts argument by argument,
# which takes 2 us where a small call has 12 in all.
_DISTILL_CALL = struct.Struct("=17qd")
_DISTILL_FWD = [c_void_p] * 5
_DISTILL_BWD = [c_void_p] * 5 + [c_int64]


def _distill_call(logits, labels, ids, top, vocab_start, vocab, temperature, sm_budget):
    T, Vl = logits.shape
    return _DISTILL_CALL.pack(logits.data_ptr(), logits.stride()[0], logits.dtype is torch.float32, labels.data_ptr() if labels is not None else 0,
                              ids.data_ptr(), ids.stride()[0], ids.dtype is torch.int64, top.data_ptr(), top.stride()[0],
                              _TEACHER_TYPES[top.dtype], T, Vl, ids.shape[1], vocab_start, vocab, sm_budget,
                              torch._C._cuda_getCurrentRawStream(logits.get_device()), temperature)


def _teacher_ref(top_ids, top_logits, vocab, temperature):
    """``(q [T, K] fp32, tm [T], lv [T])``: the teacher's distribution over a row's entries (0 on padding), its largest logit and the log of
    its sum relative to that (+inf: the row has no entries)."""
    t = torch.where((top_ids >= 0) & (top_ids < vocab), top_logits.float(), float("-inf"))
    if not t.shape[1]:
        return t, t.new_zeros(t.shape[0]), t.new_full(t.shape[:1], float("inf"))
    tm = t.max(1).values
    none = tm == float("-inf")
    tm = torch.where(none, 0.0, tm)
    q = torch.exp((t - tm[:, None]) / temperature)
    total = torch.where(none, float("inf"), q.sum(1))
    return q / total[:, None], tm, torch.log(total)


def _distill_stats_ref(logits, labels, top_ids, top_logits, vocab_start, vocab, temperature):
    """``stats [T, 8]`` and ``(tm, lv)`` of the teacher.  Stats: maximum m, sums of exp(z - m) and exp((z - m) / tau), z_label - m (+inf: the label is not here), sums of q (z_id - m)
    and q over the entries here, sum of q log q (+inf: the row has no entries), 0."""
    Vl = logits.shape[1]
    lf = logits.float()
    m = lf.max(dim=-1).values.clamp_min(torch.finfo(torch.float32).min)
    rel = lf - m[:, None]
    q, tm, lv = _teacher_ref(top_ids, top_logits, vocab, temperature)
    loc = top_ids.long() - vocab_start
    own = (loc >= 0) & (loc < Vl) & (q != 0)
    zero, inf = torch.zeros_like(q), torch.full_like(m, float("inf"))
    dot = torch.where(own, q * rel.gather(1, loc.clamp(0, Vl - 1)), zero).sum(1)
    ent = torch.where(q != 0, q * torch.log(torch.where(q != 0, q, 1.0)), zero).sum(1)
    target = inf
    if labels is not None:
        loc = labels.long() - vocab_start
        inside = (labels >= 0) & (labels < vocab) & (loc >= 0) & (loc < Vl)
        target = torch.where(inside, rel.gather(1, loc.clamp(0, Vl - 1)[:, None]).squeeze(1), inf)
    return torch.stack([m, torch.exp(rel).sum(1), torch.exp(rel / temperature).sum(1), target, dot, torch.where(own, q, zero).sum(1),
                        torch.where(lv == inf, inf, ent), torch.zeros_like(m)], dim=1), (tm, lv)


def _distill_combine_ref(all_stats, teacher, temperature, hard):
    m = all_stats[..., 0].max(dim=0).values
    inf = torch.full_like(m, float("inf"))
    d = all_stats[..., 0] - m
    s1 = (all_stats[..., 1] * torch.exp(d)).sum(0)
    st = (all_stats[..., 2] * torch.exp(d / temperature)).sum(0)
    has, own, ent = all_stats[..., 3] != inf, all_stats[..., 5], all_stats[0, :, 6]
    target = torch.where(has, all_stats[..., 3] + d, 0.0).sum(0)
    dot = torch.where(own != 0, all_stats[..., 4] + own * d, 0.0).sum(0)
    is_hard, is_soft = has.any(0) & (s1 != 0), (ent != inf) & (st != 0)       # a sum of 0: all logits of the row are -inf
    ce = torch.where(is_hard, torch.log(s1) - target, 0.0) if hard else None
    kd = torch.where(is_soft, temperature * (temperature * (ent + torch.log(st)) - dot), 0.0)
    tm, lv = teacher
    saved = torch.stack([m, torch.where(is_hard, 1.0 / s1, 0.0), torch.where(is_soft, 1.0 / st, 0.0), torch.where(is_soft, lv, inf)], dim=1)
    zero = torch.zeros_like(tm)
    return ce, kd, torch.complex(saved, torch.stack([zero, zero, zero, tm], dim=1))


def vocab_parallel_distill_fwd(logits, labels, top_ids, top_logits, temperature: float = 1.0, vocab_start: int = 0, group=None,
                               sm_budget: int = 0, stream=None):
    """Cross entropy and distillation loss per token, ``(ce [T], kd [T], saved [T, 4])``, losses in fp32.

    ``logits [T, V/t]`` are the student's (bf16 or fp32), this rank's shard of the vocabulary from ``vocab_start`` on.  ``top_ids [T, K]``
    and ``top_logits [T, K]`` are the ids and logits of the teacher's best entries, the same on every rank; an id outside the
    vocabulary is padding.  With ``q = softmax(top_logits / temperature)`` over a row's entries and the student's ``p = softmax(logits /
    temperature)`` over the whole vocabulary, ``kd = temperature^2 KL(q || p)`` (with the roundings of KL, some 2^-22 of its terms, as many
    times); rows without entries give 0.  ``ce`` is the cross entropy
    against ``labels [T]`` int32 (0 where the label lies outside the vocabulary), or ``None`` without labels.  A row whose logits are
    all ``-inf`` has neither loss nor gradient.  ``saved`` (pairs of fp32 numbers, as complex64) goes to
    ``vocab_parallel_distill_bwd_``.  The ranks of ``group`` exchange eight numbers a token in one all-gather."""
    if stream is not None:
        return K.run_on_stream(stream, (logits, labels, top_ids, top_logits), lambda: vocab_parallel_distill_fwd(
            logits, labels, top_ids, top_logits, temperature, vocab_start, group, sm_budget))
    what = "vocab_parallel_distill_fwd"
    _distill_operands(what, logits, labels, top_ids, top_logits, temperature)
    T, Vl = logits.shape
    ws = group_size(group)
    vocab = Vl * ws
    if not 0 <= vocab_start <= vocab - Vl:
        raise ValueError(f"{what}: a shard of {Vl} entries from {vocab_start} on does not lie in a vocabulary of {vocab}")
    native = K.use_native(logits)
    if native:
        labels, top_ids, top_logits = _distill_native(what, logits, labels, top_ids, top_logits)
        call = _distill_call(logits, labels, top_ids, top_logits, vocab_start, vocab, temperature, sm_budget)
        fn = K.proto("dh_distill_fwd", _DISTILL_FWD)
        kd = logits.new_empty(T, dtype=torch.float32)
        ce = torch.empty_like(kd) if labels is not None else None
        saved = logits.new_empty((T, 4), dtype=torch.complex64)
        if ws == 1:
            K.check(fn(call, K.ptr(ce), kd.data_ptr(), saved.data_ptr(), 0), what)
            return ce, kd, saved
        stats = logits.new_empty((T, 8), dtype=torch.float32)
        K.check(fn(call, 0, 0, saved.data_ptr(), stats.data_ptr()), what)
    else:
        stats, teacher = _distill_stats_ref(logits, labels, top_ids, top_logits, vocab_start, vocab, temperature)
    every = stats
    if ws > 1:
        every = torch.empty((ws * T, 8), dtype=stats.dtype, device=stats.device)
        dist.all_gather_into_tensor(every, stats, group=group)
    if not native:
        return _distill_combine_ref(every.view(ws, T, 8), teacher, temperature, labels is not None)
    fn = K.proto("dh_distill_combine", [c_void_p, c_int, c_int, c_float, c_void_p, c_void_p, c_void_p, c_void_p])
    K.check(fn(every.data_ptr(), ws, T, temperature, K.ptr(ce), kd.data_ptr(), saved.data_ptr(), K.stream_ptr()), what)
    return ce, kd, saved


def vocab_parallel_distill_bwd_(logits, labels, top_ids, top_logits, saved, g_ce, g_kd, temperature: float = 1.0, vocab_start: int = 0,
                                out=None, sm_budget: int = 0, stream=None):
    """Overwrites ``logits`` (or ``out``, of their shape and type) with ``d loss / d logits`` and returns it, for the gradients ``g_ce [T]``
    and ``g_kd [T]`` (fp32) of what ``vocab_parallel_distill_fwd`` gave; the other arguments as there (``g_ce`` is ``None`` without
    labels).  Rows with neither gradient become zero, whatever their logits."""
    if stream is not None:
        return K.run_on_stream(stream, (logits, labels, top_ids, top_logits, saved, g_ce, g_kd, out), lambda: vocab_parallel_distill_bwd_(
            logits, labels, top_ids, top_logits, saved, g_ce, g_kd, temperature, vocab_start, out, sm_budget))
    what = "vocab_parallel_distill_bwd_"
    _distill_operands(what, logits, labels, top_ids, top_logits, temperature)
    T, Vl = logits.shape
    out = logits if out is None else out
    if out is not logits:
        row, column = out.stride()
        if out.shape != logits.shape or out.dtype != logits.dtype or (row < Vl and T > 1) or (column != 1 and Vl > 1):
            raise ValueError(f"{what}: an output of the logits' shape and type with room for every row, got {out.dtype} {tuple(out.shape)}")
        if out.untyped_storage().data_ptr() == logits.untyped_storage().data_ptr() \
                and (out.data_ptr() != logits.data_ptr() or out.stride() != logits.stride()):
            raise ValueError(f"{what}: the output is the logits themselves or shares no memory with them")
    elif T > 1 and logits.stride(0) < Vl:
        raise ValueError(f"{what}: logits that are overwritten have room for every row")
    if (g_ce is None) != (labels is None):
        raise ValueError(f"{what}: labels and the gradient of their loss go together")
    if g_kd is None or saved is None:
        raise ValueError(f"{what}: the gradient of the distillation loss and the saved statistics are needed")
    for t, shape, dtype in ((g_kd, (T,), torch.float32), (g_ce, (T,), torch.float32), (saved, (T, 4), torch.complex64)):
        if t is not None and (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()):
            raise ValueError(f"{what}: contiguous fp32 gradients [T] and statistics [T, 4] as they were saved, got {t.dtype} {tuple(t.shape)}")
    if saved.data_ptr() % 16:
        raise ValueError(f"{what}: statistics that start on 16 bytes")
    if K.use_native(logits):
        labels, top_ids, top_logits = _distill_native(what, logits, labels, top_ids, top_logits, saved, g_ce, g_kd, out)
        call = _distill_call(logits, labels, top_ids, top_logits, vocab_start, 2 ** 31 - 1, temperature, sm_budget)
        fn = K.proto("dh_distill_bwd", _DISTILL_BWD)
        K.check(fn(call, saved.data_ptr(), K.ptr(g_ce), g_kd.data_ptr(), out.data_ptr(), out.stride(0)), what)
        return out
    tm, (m, inv, inv_t, lv) = saved[:, 3].imag, saved.real.unbind(1)
    rel = logits.float() - m[:, None]
    gk = torch.where(lv != float("inf"), g_kd, 0.0) * temperature
    d = torch.where(gk[:, None] != 0, torch.exp(rel / temperature) * (gk * inv_t)[:, None], 0.0)
    loc = top_ids.long() - vocab_start
    own = (loc >= 0) & (loc < Vl) & (gk[:, None] != 0)
    w = torch.where(own, torch.exp((top_logits.float() - tm[:, None]) / temperature - lv[:, None]) * gk[:, None], 0.0)
    d.scatter_add_(1, loc.clamp(0, Vl - 1), -w)
    if labels is not None:
        loc = labels.long() - vocab_start
        gc = torch.where(inv != 0, g_ce, 0.0)
        d = d + torch.where(gc[:, None] != 0, torch.exp(rel) * (gc * inv)[:, None], 0.0)
        own = (loc >= 0) & (loc < Vl)
        d.scatter_add_(1, loc.clamp(0, Vl - 1)[:, None], torch.where(own, -gc, 0.0)[:, None])
    return out.copy_(d.to(out.dtype))


def mask_scale_loss_fwd(loss_per_token, loss_mask, scale_func=None):
    """Masked mean with an optional loss-scaling hook (``optimizer.scale_loss`` in the
    reference: dhellam/operators/loss.py:131-164).  Returns ``(scaled_loss, sum, count)``."""
    m = loss_mask.reshape(-1).float()
    s = (loss_per_token.reshape(-1).float() * m).sum()
    n = m.sum()
    loss = s / n.clamp_min(1.0)
    return (scale_func(loss) if scale_func is not None else loss), s, n


def mask_scale_loss_bwd(loss_mask, count, grad_scale: float = 1.0):
    """Gradient of the masked mean with respect to each token's loss."""
    return loss_mask.reshape(-1).float() * (grad_scale / count.clamp_min(1.0))


# ----------------------------------------------------------------------------- reference-style wrappers
def cross_entropy_fwd(inputs: dict, label_smoothing: float = 0.0, group=None, vocab_start: int = None):
    """Dictionary protocol of the reference's ``cross_entropy_fwd`` (dhellam/operators/loss.py:15-98):
    ``inputs = {"vocab_parallel_logits": [..., V/t], "target": [...]}``; returns a context with
    ``loss`` (shape of ``target``) and what the backward needs.  The tensor-parallel group and
    rank come from ``adaptor.parallel_state`` unless given."""
    from ..adaptor import parallel_state as TPS
    logits, target = inputs["vocab_parallel_logits"], inputs["target"]
    if group is None:
        try:
            group = TPS.get_tensor_model_parallel_group()
        except RuntimeError:            # no model-parallel state: a single rank holding the whole vocabulary
            group = None
    Vl = logits.shape[-1]
    if vocab_start is None:
        vocab_start = dist.get_rank(group=group) * Vl if group_size(group) > 1 else 0
    l2 = logits.reshape(-1, Vl)
    loss, lse = vocab_parallel_ce_fwd(l2, target.reshape(-1).to(torch.int32), vocab_start, group, label_smoothing=label_smoothing)
    return {"loss": loss.view(target.shape), "lse": lse, "label_smoothing": label_smoothing, "vocab_size": Vl * group_size(group),
            "logits": logits, "target": target, "vocab_start": vocab_start}


def cross_entropy_bwd(context: dict, dout):
    """``d logits`` for ``dout = d L / d loss`` (shape of ``target``); overwrites the logits buffer
    (dhellam/operators/loss.py:100-127)."""
    logits = context["logits"]
    Vl = logits.shape[-1]
    g = vocab_parallel_ce_bwd_(logits.reshape(-1, Vl), context["target"].reshape(-1).to(torch.int32), context["lse"],
                               dout.reshape(-1).float(), context["vocab_start"], label_smoothing=context["label_smoothing"],
                               vocab=context["vocab_size"])
    return g.view(logits.shape)
