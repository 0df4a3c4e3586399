"""Mixture-of-experts primitives: router, dispatch plan, row permutations, combine.

New relative to the reference (it has no MoE ops; see ``models/moe.py``).  The router runs
as one sm_100a kernel on CUDA tensors (csrc/head_optim.cu, ``router_kernel``: logits, softmax, top-k and gate
normalisation in one pass over the token row), and so do the balance loss with the per-expert counts and the gradient of
gates and balance to the router's logits (csrc/balance.cu); the plan and the permutations use index
arithmetic on the device, and the only host read is the per-expert row count that sizes
the expert GEMMs (dropless routing has data-dependent shapes).
"""
from __future__ import annotations

import struct
from ctypes import c_float, c_int, c_int64, c_void_p
from dataclasses import dataclass
from typing import List, NamedTuple, Optional

import torch
import torch.distributed as dist

from .. import kernels as K
from .comm import group_size


# --------------------------------------------------------------------------- router
def router_topk_fwd(x, w, k: int):
    """``x [T,h]``, ``w [E,h]`` -> ``(probs [T,E] fp32, topi [T,k] int64, gates [T,k] fp32)``
    with ``gates`` the selected probabilities renormalised to sum to one."""
    T, h = x.shape
    E = w.shape[0]
    if x.is_cuda and E <= 64 and k <= 8:
        probs = torch.empty((T, E), dtype=torch.float32, device=x.device)
        topi32 = torch.empty((T, k), dtype=torch.int32, device=x.device)
        gates = torch.empty((T, k), dtype=torch.float32, device=x.device)
        fn = K.proto("dh_router_topk", [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p])
        K.check(fn(x.data_ptr(), w.data_ptr(), probs.data_ptr(), topi32.data_ptr(), gates.data_ptr(), T, h, E, k,
                   K.stream_ptr(None)), "dh_router_topk")
        return probs, topi32.long(), gates
    logits = x.float() @ w.float().t()
    probs = torch.softmax(logits, dim=-1)
    topv, topi = probs.topk(k, dim=-1)
    gates = topv / topv.sum(-1, keepdim=True)
    return probs, topi, gates


class Balance(NamedTuple):
    """What the backward of the balance loss needs."""
    coef: torch.Tensor               # [E] fp32: gradient of the loss with respect to a counted token's probabilities
    mask: Optional[torch.Tensor]     # [T] bool / uint8: the counted tokens (None: all)


def _router_operands(what, probs, topi, mask):
    shape, ids, id_type = probs.shape, topi.shape, topi.dtype
    if len(shape) != 2 or len(ids) != 2 or ids[0] != shape[0] or probs.dtype is not torch.float32 \
            or (id_type is not torch.int32 and id_type is not torch.int64) or not ids[1]:
        raise ValueError(f"{what}: fp32 probabilities [T, E] and int32 or int64 choices [T, k], got {probs.dtype} {tuple(probs.shape)} "
                         f"and {topi.dtype} {tuple(topi.shape)}")
    if mask is not None and (mask.shape != shape[:1] or mask.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"{what}: a mask of {shape[0]} bool or uint8 values, got {mask.dtype} {tuple(mask.shape)}")


def _on_kernel(probs, topi, *others):
    """Whether the kernels of csrc/balance.cu take these operands.  Both functions were composed of PyTorch ops before and still are for
    what only those handle: CPU tensors, the library backend, tensors that are differentiated, traced or on another device, more than
    1024 experts or 32 choices, more than 2^30 choices in all."""
    return K.use_native(probs) and 0 < probs.shape[1] <= 1024 and topi.shape[1] <= 32 and topi.numel() <= 1 << 30 and (probs.stride(1) == 1 or probs.shape[1] == 1) \
        and K.are_plain(probs, topi, *others)


# The operands that both kernels share, as one block of 8-byte fields (BalCall in csrc/balance.cu): ctypes converts argument by argument.
_ROUTER_CALL = struct.Struct("=11q")
_SCRATCH = [c_void_p]
_BALANCE_FWD = [c_void_p] * 5
_ROUTER_BWD = [c_void_p, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_float, c_void_p]


def _router_call(probs, topi, mask, sm_budget):
    T, E = probs.shape
    return _ROUTER_CALL.pack(probs.data_ptr(), probs.stride()[0], topi.data_ptr(), topi.stride()[0], topi.dtype is torch.int64,
                             mask.data_ptr() if mask is not None else 0, T, E, topi.shape[1], sm_budget,
                             torch._C._cuda_getCurrentRawStream(probs.get_device()))


def _balance_coef(topi, E, mask):
    """``(counted [T] bool, counts [E] int64, coef [E] fp32)`` of PyTorch ops that ask the host nothing."""
    T, k = topi.shape
    counted = torch.ones(T, dtype=torch.bool, device=topi.device) if mask is None else mask != 0
    n = counted.sum().clamp_min(1)
    # an extra column takes the choices that count for nobody
    used = torch.where((topi >= 0) & (topi < E) & counted[:, None], topi.long(), E).reshape(-1)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=topi.device).index_add_(0, used, torch.ones_like(used))[:E]
    return counted, counts, counts.to(torch.float32) / n / n * (E / max(k, 1))


def balance_loss_fwd(probs, topi, mask=None, sm_budget: int = 0, stream=None):
    """Load-balancing loss ``E * sum_e f_e * P_e`` (fraction of the choices x mean probability) over the counted tokens.

    ``probs [T, E]`` fp32 and ``topi [T, k]`` (int32 or int64) are the router's probabilities and choices, ``mask [T]`` (bool or
    uint8) leaves out padding tokens.  A choice outside ``[0, E)`` counts for no expert.  Returns ``(loss, counts [E] int32,
    balance)``: the loss is 0 where no token is counted, ``balance`` goes to ``router_topk_bwd``."""
    if stream is not None:
        return K.run_on_stream(stream, (probs, topi, mask), lambda: balance_loss_fwd(probs, topi, mask, sm_budget))
    _router_operands("balance_loss_fwd", probs, topi, mask)
    T, E = probs.shape
    k = topi.shape[1]
    if _on_kernel(probs, topi, mask):
        if topi.stride(1) != 1:
            topi = topi.contiguous()
        if mask is not None and not mask.is_contiguous():
            mask = mask.contiguous()
        call = _router_call(probs, topi, mask, sm_budget)
        loss, coef, counts = probs.new_empty(()), probs.new_empty(E), probs.new_empty(E, dtype=torch.int32)
        words = K.proto("dh_balance_scratch", _SCRATCH, c_int64)(call)
        scratch = probs.new_empty(words) if words else None
        K.check(K.proto("dh_balance_fwd", _BALANCE_FWD)(call, K.ptr(scratch), loss.data_ptr(), counts.data_ptr(), coef.data_ptr()), "dh_balance_fwd")
        return loss, counts, Balance(coef, mask)
    counted, counts, coef = _balance_coef(topi, E, mask)
    loss = (coef * torch.where(counted[:, None], probs, torch.zeros_like(probs)).sum(0)).sum()
    return loss, counts.to(torch.int32), Balance(coef, mask)


def aux_loss(probs, topi, E: int):
    """Load-balancing loss ``E * sum_e f_e * P_e`` (fraction routed x mean probability)."""
    frac = torch.zeros(E, dtype=torch.float32, device=probs.device)
    frac.index_add_(0, topi.reshape(-1), torch.ones(topi.numel(), dtype=torch.float32, device=probs.device))
    frac = frac / topi.numel()
    return E * (frac * probs.mean(0)).sum()


def router_topk_bwd(d_gates, probs, topi, gates, E: int, aux_scale: float = 0.0, balance: Optional[Balance] = None, sm_budget: int = 0,
                    stream=None):
    """Gradient with respect to the router logits ``[T,E]`` (fp32): of the gates (``d_gates [T,k]``) and, times ``aux_scale``, of the
    balance loss.  ``balance`` comes from ``balance_loss_fwd``; without it all tokens count.

    A choice outside ``[0, E)`` (a token that was dropped there) has no gate and gets no gradient; without a ``balance`` it is an error on
    the CPU, as of any index.  A row whose chosen probabilities sum to 0 has no finite gradient (NaN or infinities)."""
    if stream is not None:
        operands = (d_gates, probs, topi, gates) + (tuple(balance) if balance is not None else ())
        return K.run_on_stream(stream, operands, lambda: router_topk_bwd(d_gates, probs, topi, gates, E, aux_scale, balance, sm_budget))
    coef, mask = balance if balance is not None else (None, None)
    T, k = topi.shape
    if probs.shape != (T, E) or d_gates.shape != topi.shape or gates.shape != topi.shape:
        raise ValueError(f"router_topk_bwd: gates and their gradient as the choices {tuple(topi.shape)}, as many rows of {E} "
                         f"probabilities, got {tuple(gates.shape)}, {tuple(d_gates.shape)} and {tuple(probs.shape)}")
    if balance is not None:
        _router_operands("router_topk_bwd", probs, topi, mask)
        if coef.shape != (E,):
            raise ValueError(f"router_topk_bwd: a balance of {E} experts, got {tuple(coef.shape)}")
    # fp64 probabilities, a weight in a tensor and the like were taken before there was a kernel, and still are by the ops below
    if k > 0 and probs.dtype is d_gates.dtype is gates.dtype is torch.float32 and topi.dtype in (torch.int32, torch.int64) \
            and isinstance(aux_scale, (int, float)) and _on_kernel(probs, topi, d_gates, gates, mask, coef) \
            and (coef is None or coef.dtype is torch.float32):
        if aux_scale and coef is None:
            coef = balance_loss_fwd(probs, topi, sm_budget=sm_budget)[2].coef
        if mask is not None and not mask.is_contiguous():
            mask = mask.contiguous()
        if coef is not None and not coef.is_contiguous():
            coef = coef.contiguous()
        (gs, gc), (ds, dc) = gates.stride(), d_gates.stride()
        if k > 1 and not (gc == dc == 1 == topi.stride(1)):
            topi, gates, d_gates = topi.contiguous(), gates.contiguous(), d_gates.contiguous()
            gs = ds = k
        out = probs.new_empty((T, E))
        K.check(K.proto("dh_router_bwd", _ROUTER_BWD)(_router_call(probs, topi, mask, sm_budget), gates.data_ptr(), gs, d_gates.data_ptr(), ds,
                                                      coef.data_ptr() if aux_scale else 0, aux_scale, out.data_ptr()), "dh_router_bwd")
        return out
    valid = (topi >= 0) & (topi < E)
    at = (topi if balance is None and not topi.is_cuda else torch.where(valid, topi, torch.zeros_like(topi))).long()
    topv_sum = torch.where(valid, probs.gather(1, at), 0.0).sum(-1, keepdim=True)
    dot = torch.where(valid, d_gates * gates, 0.0).sum(-1, keepdim=True)
    d_topv = torch.where(valid, (d_gates - dot) / topv_sum, 0.0)
    d_probs = torch.zeros_like(probs)
    d_probs.scatter_add_(1, at, d_topv)
    if aux_scale:
        d_aux = aux_scale * (_balance_coef(topi, E, None)[2] if coef is None else coef)[None, :]
        if mask is not None:
            d_aux = torch.where(mask[:, None] != 0, d_aux, torch.zeros_like(d_aux))
        d_probs = d_probs + d_aux
    return probs * (d_probs - (d_probs * probs).sum(-1, keepdim=True))


# --------------------------------------------------------------------------- dispatch plan
@dataclass
class DispatchPlan:
    num_tokens: int
    src_row: torch.Tensor            # [T*k] token index of every dispatched copy, grouped by expert
    src_slot: torch.Tensor           # [T*k] flat (token * k + choice) index of every copy
    send_counts: List[int]           # rows sent to every expert-parallel rank
    recv_counts: List[int]           # rows received from every rank
    recv_sort: Optional[torch.Tensor]  # permutation (src-rank major -> expert major) on the receiver
    expert_rows: List[int]           # rows per local expert after the exchange


def make_plan(topi, E: int, ep: int, group) -> DispatchPlan:
    T, k = topi.shape
    flat = topi.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    src_slot = order
    src_row = torch.div(order, k, rounding_mode="floor")
    counts = torch.bincount(flat, minlength=E)                    # per global expert
    el = E // ep
    if ep == 1:
        c = counts.tolist()
        return DispatchPlan(T, src_row, src_slot, [int(sum(c))], [int(sum(c))], None, [int(v) for v in c])
    send_mat = counts.view(ep, el)                                # [dest rank, local expert]
    recv_mat = torch.empty_like(send_mat)                         # [src rank, local expert]
    dist.all_to_all_single(recv_mat, send_mat.contiguous(), group=group)
    rm = recv_mat.tolist()
    send_counts = [int(v) for v in send_mat.sum(1).tolist()]
    recv_counts = [int(sum(r)) for r in rm]
    # received rows are ordered (src rank, local expert); sort them expert-major
    seg_expert = torch.tensor([e for s in range(ep) for e in range(el)], device=topi.device)
    seg_len = recv_mat.reshape(-1)
    row_expert = torch.repeat_interleave(seg_expert, seg_len)
    recv_sort = torch.sort(row_expert, stable=True).indices
    expert_rows = [int(sum(rm[s][e] for s in range(ep))) for e in range(el)]
    return DispatchPlan(T, src_row, src_slot, send_counts, recv_counts, recv_sort, expert_rows)


# --------------------------------------------------------------------------- row movement
def permute_rows(x, index):
    """``out[i] = x[index[i]]``."""
    return x.index_select(0, index)


def unpermute_rows(x, index):
    """Inverse of ``permute_rows``: ``out[index[i]] = x[i]``."""
    out = torch.empty_like(x)
    out.index_copy_(0, index, x)
    return out


def scatter_add_rows(x, index, n_rows: int):
    """``out[index[i]] += x[i]`` with fp32 accumulation."""
    out = torch.zeros((n_rows, x.shape[1]), dtype=torch.float32, device=x.device)
    out.index_add_(0, index, x.float())
    return out


def combine_rows(yb, plan: DispatchPlan, gates):
    """Weighted un-permute: ``out[token] = sum_k gate[token,k] * y[copy(token,k)]``."""
    g = gates.reshape(-1).index_select(0, plan.src_slot)          # gate of every copy, dispatch order
    out = torch.zeros((plan.num_tokens, yb.shape[1]), dtype=torch.float32, device=yb.device)
    out.index_add_(0, plan.src_row, yb.float() * g[:, None])
    return out.to(yb.dtype)


def combine_rows_bwd(d_out, yb, plan: DispatchPlan, gates):
    """Returns ``(d_yb [T*k,h], d_gates [T,k] fp32)``."""
    g = gates.reshape(-1).index_select(0, plan.src_slot)
    d_rows = d_out.index_select(0, plan.src_row).float()
    d_yb = (d_rows * g[:, None]).to(yb.dtype)
    d_copy = (d_rows * yb.float()).sum(-1)
    d_gates = torch.zeros(gates.numel(), dtype=torch.float32, device=yb.device)
    d_gates.index_copy_(0, plan.src_slot, d_copy)
    return d_yb, d_gates.view_as(gates)
