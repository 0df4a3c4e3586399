"""Synthetic token data of a named shape, and micro-batch construction.

The reference's dataset blob is not part of its repository and its demo run only needs
token ids of the right shape (script/run.sh:60-75); its head block can also fabricate a
batch on the device (``initialize_pre_process_data``, dhellam/core/dshb.py:53-73).  Here
every rank derives its micro-batches from ``(seed, step, micro-batch index, dp rank)``, so
no broadcast over the tensor-parallel group is needed (the reference broadcasts tokens,
labels and masks: megatron.patch:827-910).

Rows are sequence-first (row = s * batch + b).  With context parallelism a rank holds
sequence chunks ``r`` and ``2c-1-r`` of ``2c`` (the load-balanced causal split of
dhellam/core/dstb.py:167-169).
"""
from __future__ import annotations

from typing import List

import torch

from .config import ModelConfig, TrainConfig
from .core.engine import MicroBatch


def cp_chunk_positions(seq: int, cp: int, r: int) -> torch.Tensor:
    """Sequence positions held by context-parallel rank ``r`` (ascending)."""
    if cp == 1:
        return torch.arange(seq, dtype=torch.int32)
    assert seq % (2 * cp) == 0, "sequence must divide by 2 x context-parallel size"
    c = seq // (2 * cp)
    a = torch.arange(r * c, (r + 1) * c, dtype=torch.int32)
    b = torch.arange((2 * cp - 1 - r) * c, (2 * cp - r) * c, dtype=torch.int32)
    return torch.cat([a, b])


def synthetic_tokens(cfg: ModelConfig, batch: int, seed: int) -> torch.Tensor:
    """``[batch, seq+1]`` ids uniform in ``[0, vocab)`` from ``seed`` (CPU generator, so the
    stream is identical on every rank and device)."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, cfg.vocab_size, (batch, cfg.seq_length + 1), generator=g, dtype=torch.int64)


def synthetic_teacher(cfg: ModelConfig, batch: int, k: int, seed: int):
    """``(ids [batch, seq, k] int32, logits [batch, seq, k] fp16)`` of a teacher that knows nothing: entries from ``seed``, falling logits."""
    g = torch.Generator().manual_seed(seed)
    first = torch.randint(0, cfg.vocab_size, (batch, cfg.seq_length, 1), generator=g)
    ids = (first + torch.arange(min(k, cfg.vocab_size)) * 31) % cfg.vocab_size
    logits = 2.0 * torch.randn(ids.shape, generator=g).sort(dim=-1, descending=True).values
    return ids.to(torch.int32), logits.to(torch.float16)


def make_microbatch(cfg: ModelConfig, ps, sample: torch.Tensor, index: int, seed: int, device, pin: bool = False, teacher=None,
                    token_mask=None) -> MicroBatch:
    """Builds this rank's micro-batch from ``sample [B, S+1]`` (tokens; labels are the shift by one) and, for distillation, the teacher's
    ``(ids, logits)``, each ``[B, S, K]``: its best entries for the token that follows each position.  ``token_mask [B, S]`` is 0 on padding,
    which counts neither in the loss nor in the router's balance (synthetic samples and token files have none)."""
    B = sample.shape[0]
    pos = cp_chunk_positions(cfg.seq_length, ps.cp, ps.cp_rank)
    tok = sample[:, :-1][:, pos.long()]          # [B, S_local]
    lab = sample[:, 1:][:, pos.long()]
    tokens = tok.t().contiguous().reshape(-1).to(torch.int32)       # sequence-first rows
    labels = lab.t().contiguous().reshape(-1).to(torch.int32)
    positions = pos[:, None].expand(-1, B).contiguous().reshape(-1)
    T = tokens.numel()
    mask = torch.ones(T, dtype=torch.float32)
    if token_mask is not None:
        if token_mask.shape != (B, cfg.seq_length):
            raise ValueError(f"a token mask of {B} samples of {cfg.seq_length} tokens, got {tuple(token_mask.shape)}")
        token_mask = token_mask[:, pos.long()].t().reshape(-1) != 0
        mask = token_mask.to(torch.float32)
    lo, hi = ps.tp_rank * (T // ps.tp), (ps.tp_rank + 1) * (T // ps.tp)
    dev = torch.device(device)
    host = [tokens, labels, mask, positions]
    if teacher is not None:
        host += [t[:, pos.long()].transpose(0, 1).reshape(T, -1).contiguous() for t in teacher]
    if token_mask is not None:
        host.append(token_mask)
    if dev.type == "cuda":
        if pin:
            host = [t.pin_memory() for t in host]
        host = [t.to(dev, non_blocking=True) for t in host]
    tokens, labels, mask, positions = host[:4]
    teacher_ids, teacher_logits = host[4:6] if teacher is not None else (None, None)
    return MicroBatch(index=index, tokens=tokens, labels=labels, loss_mask=mask, positions=positions, batch=B, seed=seed,
                      positions_local=positions[lo:hi], teacher_ids=teacher_ids, teacher_logits=teacher_logits,
                      token_mask=host[-1] if token_mask is not None else None)


def synthetic_step_batches(cfg: ModelConfig, train: TrainConfig, ps, step: int, device) -> List[MicroBatch]:
    """All micro-batches of one optimizer step for this rank."""
    n = train.num_microbatches(ps.dp)
    out = []
    for i in range(n):
        seed = (train.seed * 1000003 + step * 8191 + ps.dp_rank * 127 + i) & 0x7FFFFFFF
        sample = synthetic_tokens(cfg, train.micro_batch_size, seed)
        teacher = synthetic_teacher(cfg, train.micro_batch_size, train.distill_top_k, seed) if train.distill_alpha else None
        out.append(make_microbatch(cfg, ps, sample, i, seed, device, teacher=teacher))
    return out


# --------------------------------------------------------------------------- real token data
class TokenFileDataset:
    """Samples ``[seq+1]`` windows from a flat file of token ids (``uint16`` / ``int32`` /
    ``int64``, the payload of a Megatron ``.bin`` file or any ``numpy`` memmap-able dump).

    Sample ``i`` of epoch ``e`` starts at a position drawn from a permutation seeded with
    ``(seed, e)``; the file is memory-mapped, nothing is read up front.  This covers what the
    reference gets from Megatron's ``GPTDataset`` for its demo run (script/run.sh:60-75,
    ``--data-path``); document boundaries and blending are not modelled.  ``teacher`` is the ``TeacherTopFile`` of the same tokens."""

    def __init__(self, path: str, seq_length: int, dtype: str = "int32", seed: int = 1234, teacher=None):
        import numpy as np
        self.np = np
        self.tokens = np.memmap(path, dtype=np.dtype(dtype), mode="r")
        self.seq = seq_length
        self.n = (len(self.tokens) - 1) // seq_length
        if self.n <= 0:
            raise ValueError(f"{path}: {len(self.tokens)} tokens are fewer than one sample of {seq_length + 1}")
        self.seed = seed
        self._perm_epoch, self._perm = -1, None
        if teacher is not None and teacher.n not in (len(self.tokens) - 1, len(self.tokens)):      # a wrong k may divide the file too
            raise ValueError(f"{path}: {len(self.tokens)} tokens, but the teacher's entries, {teacher.k} each, of {teacher.n} positions")
        self.teacher = teacher

    def __len__(self):
        return self.n

    def start(self, index: int) -> int:
        """Position of sample ``index`` in the file."""
        epoch, i = divmod(index, self.n)
        if epoch != self._perm_epoch:
            self._perm = self.np.random.default_rng((self.seed, epoch)).permutation(self.n)
            self._perm_epoch = epoch
        return int(self._perm[i]) * self.seq

    def sample(self, index: int) -> torch.Tensor:
        start = self.start(index)
        return torch.from_numpy(self.np.asarray(self.tokens[start:start + self.seq + 1]).astype(self.np.int64))

    def batch(self, first_index: int, batch: int) -> torch.Tensor:
        """``[batch, seq+1]`` of consecutive sample indices."""
        return torch.stack([self.sample(first_index + j) for j in range(batch)])

    def teacher_batch(self, first_index: int, batch: int):
        """``(ids, logits)``, each ``[batch, seq, k]``, of the samples that ``batch`` gives."""
        rows = [self.teacher.rows(self.start(first_index + j), self.seq) for j in range(batch)]
        return torch.stack([i for i, _ in rows]), torch.stack([l for _, l in rows])


class TeacherTopFile:
    """A teacher's best ``k`` entries for the token behind every position of a token file: ``<prefix>.ids`` (int32) and ``<prefix>.logits``
    (float16), each ``[positions, k]`` without a header, memory-mapped.  An id of -1 is padding."""

    def __init__(self, prefix: str, k: int):
        import numpy as np
        self.np, self.k = np, k
        self.ids = np.memmap(prefix + ".ids", dtype=np.int32, mode="r")
        self.logits = np.memmap(prefix + ".logits", dtype=np.float16, mode="r")
        if k <= 0 or len(self.ids) != len(self.logits) or len(self.ids) % k:
            raise ValueError(f"{prefix}: {len(self.ids)} ids and {len(self.logits)} logits are no rows of {k} entries")
        self.n = len(self.ids) // k

    def rows(self, start: int, n: int):
        part = slice(start * self.k, (start + n) * self.k)
        return (torch.from_numpy(self.np.array(self.ids[part])).view(n, self.k), torch.from_numpy(self.np.array(self.logits[part])).view(n, self.k))


def broadcast_batch_on_tp_group(ps, sample, batch: int, seq_plus_one: int, device="cpu") -> torch.Tensor:
    """Hands the ``[batch, seq+1]`` token sample that only the first rank of each
    tensor-parallel group read from disk to the rest of the group (``sample`` is ``None``
    on the others).  Same purpose as the reference's patched ``get_batch_on_this_tp_rank``
    (megatron.patch:827-910), which broadcasts tokens, labels, loss mask and position ids;
    labels, mask and positions are derived on every rank here (``make_microbatch``), so one
    tensor crosses the group instead of four."""
    import torch.distributed as dist
    if ps.tp == 1 or ps.tp_group is None:
        return sample
    dev = torch.device(device)
    if ps.tp_rank == 0:
        buf = sample.to(device=dev, dtype=torch.int64).contiguous()
        assert tuple(buf.shape) == (batch, seq_plus_one)
    else:
        buf = torch.empty((batch, seq_plus_one), dtype=torch.int64, device=dev)
    dist.broadcast(buf, src=ps.tp_ranks[0], group=ps.tp_group)
    return buf


def broadcast_teacher_on_tp_group(ps, teacher, shape, device="cpu"):
    """The same for the teacher's ``(ids, logits)`` of ``shape`` (``None`` on all but the first rank of the group)."""
    import torch.distributed as dist
    if ps.tp == 1 or ps.tp_group is None:
        return teacher
    out = []
    for i, dtype in enumerate((torch.int32, torch.float16)):
        buf = teacher[i].to(device=device, dtype=dtype).contiguous() if ps.tp_rank == 0 else torch.empty(shape, dtype=dtype, device=device)
        assert tuple(buf.shape) == tuple(shape)
        dist.broadcast(buf, src=ps.tp_ranks[0], group=ps.tp_group)
        out.append(buf)
    return tuple(out)


def file_step_batches(ds: TokenFileDataset, cfg: ModelConfig, train: TrainConfig, ps, step: int, device) -> List[MicroBatch]:
    """All micro-batches of one optimizer step for this rank from a token file: data-parallel
    rank ``d`` takes every ``dp``-th micro-batch, the first rank of each tensor-parallel group
    reads and the group receives a broadcast."""
    n = train.num_microbatches(ps.dp)
    B = train.micro_batch_size
    out = []
    dev = torch.device(device)
    bdev = dev if dev.type == "cuda" else torch.device("cpu")
    for i in range(n):
        first = ((step * n + i) * ps.dp + ps.dp_rank) * B
        sample = ds.batch(first, B) if ps.tp_rank == 0 else None
        sample = broadcast_batch_on_tp_group(ps, sample, B, cfg.seq_length + 1, bdev)
        teacher = None
        if train.distill_alpha:
            if ds.teacher is None:
                raise ValueError("distillation (distill_alpha > 0) from a token file needs the teacher's entries of its positions")
            teacher = ds.teacher_batch(first, B) if ps.tp_rank == 0 else None
            teacher = broadcast_teacher_on_tp_group(ps, teacher, (B, cfg.seq_length, ds.teacher.k), bdev)
            teacher = tuple(t.cpu() for t in teacher)
        seed = (train.seed * 1000003 + step * 8191 + ps.dp_rank * 127 + i) & 0x7FFFFFFF
        out.append(make_microbatch(cfg, ps, sample.cpu() if sample.is_cuda else sample, i, seed, device, teacher=teacher))
    return out
