"""Rotary forms, balance loss and distillation together, as an optimizer step of a further-trained model runs them: the engine (one
rank, tensor, context and expert parallel ranks on gloo) against an autograd model of the same mathematics, the data that feeds it, the
command line, and the engine on a GPU against the engine on the CPU."""
import json
import math

import pytest
import torch
import torch.nn.functional as F

import reference_model as RM
from dist_utils import run_ranks

FORMS = dict(rotary_percent=0.5, rotary_interleaved=True, rope_scaling="yarn", rope_scaling_factor=4.0, rope_original_max_position=16)


def _reference_rope(cfg):
    from dhellam_b200.ops.rope import RopeScaling, rope_frequencies
    scaling = None if cfg.rope_scaling == "none" else RopeScaling(cfg.rope_scaling, cfg.rope_scaling_factor, cfg.rope_original_max_position)
    freq, scale = rope_frequencies(cfg.rotary_dim, cfg.rope_theta, scaling)

    def rope(x, pos, theta):
        r = cfg.rotary_dim
        a = pos.double()[:, None] * freq
        c, s = (a.cos() * scale).float()[:, None, None], (a.sin() * scale).float()[:, None, None]
        head, rest = x[..., :r], x[..., r:]
        x1, x2 = (head[..., 0::2], head[..., 1::2]) if cfg.rotary_interleaved else (head[..., : r // 2], head[..., r // 2:])
        y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
        turned = torch.stack([y1, y2], -1).flatten(-2) if cfg.rotary_interleaved else torch.cat([y1, y2], -1)
        return torch.cat([turned, rest], -1)
    return rope


def reference_loss(cfg, layers, head, sample, teacher, alpha, tau, coeff):
    """``(reported loss, loss with the balance term)``."""
    B, S = sample.shape[0], sample.shape[1] - 1
    tok, lab = sample[:, :-1].t().reshape(-1), sample[:, 1:].t().reshape(-1)
    x, aux = head["word_embeddings"][tok], []
    keep, RM._rope = RM._rope, _reference_rope(cfg)
    try:
        for w in layers:
            x = RM.layer_forward(cfg, w, x, B, torch.arange(S), aux)
    finally:
        RM._rope = keep
    y = RM._norm(cfg, x, head["final_ln_weight"], head.get("final_ln_bias"))
    logits = y @ head.get("output_weight", head["word_embeddings"]).t()
    loss = F.cross_entropy(logits, lab)
    if alpha:
        ids, top = (t.transpose(0, 1).reshape(S * B, -1) for t in teacher)
        q = torch.zeros_like(logits).scatter_add(1, ids.long(), torch.softmax(top.float() / tau, 1))
        kd = tau * tau * F.kl_div(F.log_softmax(logits / tau, 1), q, reduction="none").sum(1).mean()
        loss = (1 - alpha) * loss + alpha * kd
    return loss, loss + coeff * torch.stack(aux).sum() if aux and coeff else loss


def _student(rank, world, name, par, n_mb, B, seq, overrides, alpha, tau):
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import make_microbatch, synthetic_teacher, synthetic_tokens
    from dhellam_b200.models.sharding import random_full_head, random_full_layer, shard_head, shard_layer
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    cfg = preset(name, seq_length=seq, **overrides)
    pcfg = ParallelConfig(**par)
    train = TrainConfig(micro_batch_size=B, global_batch_size=B * n_mb * pcfg.dp, dtype="fp32", clip_grad=0.0, distill_alpha=alpha,
                        distill_temperature=tau)
    if world == 1:
        PS.set_state(None)
    tr = Trainer(cfg, pcfg, train, device="cpu")
    ps = tr.ps
    layers = [random_full_layer(cfg, i, 11) for i in range(cfg.num_layers)]
    head = random_full_head(cfg, 11)
    for i, w in enumerate(layers):
        tr.model.load_full_layer_weights(i, w)
    tr.model.load_full_head_weights(head)
    keys = [(d, i) for d in range(pcfg.dp) for i in range(n_mb)]
    samples = {k: synthetic_tokens(cfg, B, 500 + 17 * k[0] + k[1]) for k in keys}
    teachers = {k: synthetic_teacher(cfg, B, 5, 900 + 17 * k[0] + k[1]) for k in keys}
    mine = [(ps.dp_rank, i) for i in range(n_mb)]
    mbs = [make_microbatch(cfg, ps, samples[k], i, 500 + i, "cpu", teacher=teachers[k] if alpha else None) for i, k in enumerate(mine)]
    tr.optimizer.zero_grad()
    losses = tr.engine.run_step(mbs)
    tr.optimizer.reduce_gradients()
    for t in [t for w in layers for t in w.values()] + list(head.values()):
        t.requires_grad_(True)
    total, ref = 0, {}
    for k in keys:
        ref[k], whole = reference_loss(cfg, layers, head, samples[k], teachers[k], alpha, tau, cfg.moe_aux_loss_coeff if cfg.is_moe else 0.0)
        total = total + whole / len(keys)
    total.backward()
    for k, l in zip(mine, losses):
        assert torch.allclose(l, ref[k], rtol=1e-4, atol=1e-5), (k, l, ref[k])
    tol = dict(rtol=5e-3, atol=3e-5)
    for m in tr.model.dctb:
        for which, idx in (("first", m.first_index), ("second", m.second_index)):
            want = shard_layer({n: t.grad for n, t in layers[idx].items()}, cfg, ps.tp, ps.tp_rank, ps.ep, ps.ep_rank)
            for n in m.shapes:
                g = getattr(m, f"{n}_{which}").main_grad
                assert torch.allclose(g, want[n], **tol), (rank, n, idx, float((g - want[n]).abs().max()))
    if tr.model.dchb is not None:
        want = shard_head({n: t.grad for n, t in head.items()}, cfg, ps.tp, ps.tp_rank)
        for n in tr.model.dchb.shapes:
            g = getattr(tr.model.dchb, n).main_grad
            assert torch.allclose(g, want[n], **tol), (rank, n, float((g - want[n]).abs().max()))
    if cfg.is_moe:
        load = tr.expert_load()
        assert load.dtype in (torch.int32, torch.int64)
        assert int(load.sum()) == cfg.num_layers * n_mb * B * seq // pcfg.cp * cfg.moe_top_k


@pytest.mark.parametrize("name,overrides,alpha,tau", [
    ("tiny-llama", FORMS, 0.0, 1.0), ("tiny-llama", {}, 0.6, 2.0), ("tiny-llama", dict(FORMS, rope_scaling="llama3", rotary_interleaved=False), 1.0, 1.5),
    ("tiny-gpt", dict(rotary_percent=0.5, rope_scaling="linear", rope_scaling_factor=2.0), 0.3, 1.0),
    ("tiny-moe", dict(moe_aux_loss_coeff=0.05), 0.0, 1.0), ("tiny-moe", dict(FORMS, moe_aux_loss_coeff=0.05), 0.4, 2.0)])
def test_student_step_matches_autograd(name, overrides, alpha, tau):
    _student(0, 1, name, {}, 2, 2, 32, overrides, alpha, tau)


@pytest.mark.parametrize("name,world,par,overrides", [("tiny-llama", 2, dict(tp=2), FORMS), ("tiny-llama", 2, dict(cp=2), FORMS),
                                                      ("tiny-llama", 2, dict(pp=2), dict(FORMS, num_layers=4))],
                         ids=["tp2", "cp2", "pp2"])
def test_student_step_over_ranks(name, world, par, overrides):
    run_ranks(_student, world, name, par, 2, 2, 32, overrides, 0.6, 2.0)


def test_padding_tokens_do_not_count_in_the_balance():
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import synthetic_step_batches
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    cfg = preset("tiny-moe", seq_length=16, moe_aux_loss_coeff=0.1)
    train = TrainConfig(micro_batch_size=2, global_batch_size=2, dtype="fp32")
    PS.set_state(None)
    tr = Trainer(cfg, ParallelConfig(), train, device="cpu")
    mbs = synthetic_step_batches(cfg, train, tr.ps, 0, "cpu")
    mbs[0].token_mask = torch.arange(32) % 4 != 0
    tr.optimizer.zero_grad()
    tr.engine.run_step(mbs)
    assert int(tr.expert_load().sum()) == cfg.num_layers * 24 * cfg.moe_top_k


def test_configurations_that_are_refused():
    from dhellam_b200.config import ModelConfig, ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import make_microbatch, synthetic_tokens
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    for bad in (dict(rotary_percent=0.0), dict(rotary_percent=0.05), dict(rotary_percent=1.5)):
        with pytest.raises(ValueError):
            ModelConfig(**bad)
    for bad in (dict(distill_alpha=1.5), dict(distill_alpha=-0.1), dict(distill_alpha=0.5, label_smoothing=0.1), dict(distill_temperature=0.0)):
        with pytest.raises(ValueError):
            TrainConfig(**bad)
    with pytest.raises(ValueError):
        PS.set_state(None)
        Trainer(preset("tiny-llama", seq_length=16, rope_scaling="other"), ParallelConfig(), TrainConfig(dtype="fp32"), device="cpu")
    cfg, train = preset("tiny-llama", seq_length=16), TrainConfig(micro_batch_size=1, global_batch_size=1, dtype="fp32", distill_alpha=0.5)
    PS.set_state(None)
    tr = Trainer(cfg, ParallelConfig(), train, device="cpu")
    with pytest.raises(ValueError, match="teacher"):
        tr.train_step([make_microbatch(cfg, tr.ps, synthetic_tokens(cfg, 1, 0), 0, 0, "cpu")])


def _write_teacher(prefix, n, k, vocab):
    import numpy as np
    rng = np.random.default_rng(0)
    rng.integers(0, vocab, (n, k)).astype(np.int32).tofile(prefix + ".ids")
    np.sort(rng.standard_normal((n, k)))[:, ::-1].astype(np.float16).tofile(prefix + ".logits")


def test_teacher_file_lies_beside_the_tokens(tmp_path):
    import numpy as np
    from dhellam_b200.data import TeacherTopFile, TokenFileDataset
    (np.arange(101) % 50).astype(np.int32).tofile(str(tmp_path / "t.bin"))
    _write_teacher(str(tmp_path / "top"), 100, 3, 50)
    top = TeacherTopFile(str(tmp_path / "top"), 3)
    ds = TokenFileDataset(str(tmp_path / "t.bin"), 20, teacher=top)
    ids, logits = ds.teacher_batch(1, 3)
    assert ids.shape == logits.shape == (3, 20, 3) and ids.dtype == torch.int32 and logits.dtype == torch.float16
    raw = np.fromfile(str(tmp_path / "top.ids"), dtype=np.int32).reshape(100, 3)
    for b in range(3):
        start = int(ds.sample(1 + b)[0])              # the tokens count up from 0 to 49, twice
        i = ds.start(1 + b)
        assert i % 50 == start and np.array_equal(ids[b].numpy(), raw[i:i + 20])
    with pytest.raises(ValueError):
        TeacherTopFile(str(tmp_path / "top"), 7)
    _write_teacher(str(tmp_path / "short"), 90, 3, 50)
    with pytest.raises(ValueError):
        TokenFileDataset(str(tmp_path / "t.bin"), 20, teacher=TeacherTopFile(str(tmp_path / "short"), 3))


def _teacher_ranks(rank, world, folder):
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import TeacherTopFile, TokenFileDataset, file_step_batches
    from dhellam_b200.parallel import state as PS
    ps = PS.initialize_model_parallel(ParallelConfig(tp=2))
    cfg = preset("tiny-llama", seq_length=20)
    train = TrainConfig(micro_batch_size=2, global_batch_size=2, dtype="fp32", distill_alpha=0.5)
    ds = TokenFileDataset(folder + "/t.bin", 20, teacher=TeacherTopFile(folder + "/top", 3))
    mb = file_step_batches(ds, cfg, train, ps, 0, "cpu")[0]
    ids, logits = ds.teacher_batch(0, 2)
    assert torch.equal(mb.teacher_ids, ids.transpose(0, 1).reshape(40, 3)) and torch.equal(mb.teacher_logits, logits.transpose(0, 1).reshape(40, 3))


def test_teacher_entries_reach_every_tensor_parallel_rank(tmp_path):
    import numpy as np
    (np.arange(101) % 50).astype(np.int32).tofile(str(tmp_path / "t.bin"))
    _write_teacher(str(tmp_path / "top"), 100, 3, 50)
    run_ranks(_teacher_ranks, 2, str(tmp_path))


def test_command_line_trains_a_student(tmp_path):
    import numpy as np
    from test_train_cli import _run
    (np.arange(4000) % 128).astype(np.int32).tofile(str(tmp_path / "tokens.bin"))
    _write_teacher(str(tmp_path / "top"), 3999, 4, 128)
    out = _run(["--train-iters", "2", "--data-path", str(tmp_path / "tokens.bin"), "--distill-alpha", "0.5", "--distill-temperature", "2.0",
                "--distill-top-k", "4", "--distill-data", str(tmp_path / "top"), "--rotary-percent", "0.5", "--rotary-interleaved",
                "--use-rope-scaling", "--rope-scaling-type", "yarn", "--rope-original-max-position", "16", "--num-experts", "4",
                "--metrics-jsonl", str(tmp_path / "m.jsonl")], str(tmp_path))
    assert "iteration" in out
    recs = [json.loads(l) for l in open(tmp_path / "m.jsonl")]
    assert len(recs) == 2 and all(math.isfinite(r["loss"]) and 1.0 <= r["expert_load_max_over_mean"] <= 4.0 for r in recs)


def test_arguments_reach_the_configuration():
    from dhellam_b200.adaptor.megatron import build_parser, configs_from_args
    def parse(*more):
        return configs_from_args(build_parser().parse_args(["--num-layers", "2", "--bf16", *more]), 1)
    cfg, _, train = parse()
    assert cfg.plain_rope and train.distill_alpha == 0.0
    cfg, _, train = parse("--rotary-percent", "0.25", "--rotary-interleaved", "--use-rope-scaling", "--distill-alpha", "0.3", "--distill-top-k", "9")
    assert (cfg.rotary_dim, cfg.rotary_interleaved, cfg.rope_scaling, cfg.rope_scaling_factor) == (32, True, "llama3", 8.0)
    assert (train.distill_alpha, train.distill_top_k, train.distill_temperature) == (0.3, 9, 1.0)
    cfg, _, _ = parse("--rotary-seq-len-interpolation-factor", "4")
    assert (cfg.rope_scaling, cfg.rope_scaling_factor) == ("linear", 4.0)


def test_a_teachers_entries_of_padding_do_not_matter():
    """Rows that the loss leaves out: NaN and infinities among the teacher's logits there change neither the loss nor a gradient."""
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import synthetic_step_batches
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    cfg = preset("tiny-llama", seq_length=16)
    for alpha in (0.5, 1.0):
        train = TrainConfig(micro_batch_size=2, global_batch_size=2, dtype="fp32", distill_alpha=alpha, distill_temperature=2.0)
        got = []
        for poison in (False, True):
            PS.set_state(None)
            tr = Trainer(cfg, ParallelConfig(), train, device="cpu")
            mbs = synthetic_step_batches(cfg, train, tr.ps, 0, "cpu")
            left_out = torch.arange(32) % 5 == 0
            mbs[0].loss_mask.view(-1)[left_out] = 0
            if poison:
                mbs[0].teacher_logits[left_out] = torch.tensor([math.nan, math.inf] * 8, dtype=torch.float16)
            else:
                mbs[0].teacher_ids[left_out] = -1
            tr.optimizer.zero_grad()
            losses = tr.engine.run_step(mbs)
            got.append((losses[0], tr.model.dchb.word_embeddings.main_grad.clone()))
        assert math.isfinite(float(got[0][0])) and torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_a_teacher_file_of_other_rows_or_without_tokens_is_refused(tmp_path):
    import os
    import subprocess
    import sys
    import numpy as np
    from dhellam_b200.data import TeacherTopFile, TokenFileDataset
    from test_train_cli import ARGS, ROOT
    np.arange(100, dtype=np.int32).tofile(str(tmp_path / "t.bin"))
    _write_teacher(str(tmp_path / "top"), 100, 6, 50)
    with pytest.raises(ValueError, match="200 positions"):          # three entries a row divide the file as well
        TokenFileDataset(str(tmp_path / "t.bin"), 20, teacher=TeacherTopFile(str(tmp_path / "top"), 3))
    p = subprocess.run([sys.executable, os.path.join(ROOT, "train.py")] + ARGS + ["--train-iters", "1", "--distill-alpha", "0.5", "--distill-data",
                       str(tmp_path / "top")], cwd=str(tmp_path), env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)
    assert p.returncode != 0 and "--data-path" in p.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("alpha,tau", [(0.0, 1.0), (0.5, 2.0), (0.7, 1.5)])
@pytest.mark.parametrize("family", ["llama", "moe"])
def test_student_step_on_gpu_matches_the_cpu_engine(family, alpha, tau):
    """bf16 kernels against the fp32 engine with the same weights, data and teacher: within what the plain training step of the same sizes is
    held to (the roundings of the layers in between are the larger part of it), router-side gradients less tightly (near-ties go elsewhere)."""
    from dhellam_b200 import kernels as K
    from dhellam_b200.config import ModelConfig, ParallelConfig, TrainConfig
    from dhellam_b200.data import make_microbatch, synthetic_teacher, synthetic_tokens
    from dhellam_b200.models.sharding import random_full_head, random_full_layer
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    moe = dict(num_experts=4, moe_top_k=2, moe_aux_loss_coeff=0.01, ffn_hidden_size=512) if family == "moe" else dict(ffn_hidden_size=1024)
    cfg = ModelConfig(name="t-student", num_layers=2, hidden_size=512, num_attention_heads=4, num_query_groups=2, head_dim=128, vocab_size=2048,
                      seq_length=256, rope_theta=500000.0, rotary_percent=0.5, rotary_interleaved=True, rope_scaling="yarn",
                      rope_scaling_factor=4.0, rope_original_max_position=64, **moe)
    layers = [random_full_layer(cfg, i, 3) for i in range(cfg.num_layers)]
    head = random_full_head(cfg, 3)
    samples = [synthetic_tokens(cfg, 2, 40 + i) for i in range(2)]
    teachers = [synthetic_teacher(cfg, 2, 16, 70 + i) for i in range(2)]
    results = {}
    for dev, dtype in (("cpu", "fp32"), ("cuda", "bf16")):
        PS.set_state(None)
        train = TrainConfig(micro_batch_size=2, global_batch_size=4, dtype=dtype, clip_grad=0.0, distill_alpha=alpha, distill_temperature=tau)
        tr = Trainer(cfg, ParallelConfig(), train, device=dev)
        for i, w in enumerate(layers):
            tr.model.load_full_layer_weights(i, {k: v.to(dev) for k, v in w.items()})
        tr.model.load_full_head_weights({k: v.to(dev) for k, v in head.items()})
        mbs = [make_microbatch(cfg, tr.ps, s, i, 40 + i, dev, teacher=t if alpha else None) for i, (s, t) in enumerate(zip(samples, teachers))]
        tr.optimizer.zero_grad()
        losses = tr.engine.run_step(mbs)
        if dev == "cuda":
            torch.cuda.synchronize()
            assert K.read_status().code == 0
        if family == "moe":
            assert int(tr.expert_load().sum()) == 2 * 2 * 512 * 2
        results[dev] = ([float(l) for l in losses], {n: p.main_grad.float().cpu().clone() for n, p in tr.model.named_parameters()})
        tr.close()
    for a, b in zip(results["cpu"][0], results["cuda"][0]):
        assert abs(a - b) / abs(a) < 2e-2, (a, b)
    bad = []
    for n, g in results["cpu"][1].items():
        err = ((g - results["cuda"][1][n]).norm() / g.norm().clamp_min(1e-6)).item()
        if err > (0.25 if family == "moe" and ("router" in n or "ln_mlp" in n or "expert" in n) else 8e-2):
            bad.append((n, err))
    assert not bad, bad


def test_options_that_contradict_each_other_are_refused(tmp_path):
    import numpy as np
    import os
    import subprocess
    import sys
    from dhellam_b200.adaptor.megatron import build_parser, configs_from_args
    from test_train_cli import ARGS, ROOT

    def parse(*more):
        return configs_from_args(build_parser().parse_args(["--num-layers", "2", "--bf16", *more]), 1)
    for more in (["--rotary-seq-len-interpolation-factor", "4", "--use-rope-scaling"], ["--distill-data", "teacher"],
                 ["--position-embedding-type", "learned_absolute", "--use-rope-scaling"],
                 ["--position-embedding-type", "learned_absolute", "--rotary-seq-len-interpolation-factor", "2"],
                 ["--position-embedding-type", "learned_absolute", "--rotary-interleaved"],
                 ["--position-embedding-type", "learned_absolute", "--rotary-percent", "0.5"]):
        with pytest.raises(ValueError):
            parse(*more)
    parse("--position-embedding-type", "learned_absolute", "--rotary-base", "10000")      # a number without meaning there, as before
    np.arange(100, dtype=np.int32).tofile(str(tmp_path / "t.bin"))
    _write_teacher(str(tmp_path / "top"), 100, 6, 50)
    p = subprocess.run([sys.executable, os.path.join(ROOT, "train.py")] + ARGS + ["--train-iters", "1", "--data-path", str(tmp_path / "t.bin"),
                       "--distill-top-k", "6", "--distill-data", str(tmp_path / "top")], cwd=str(tmp_path),
                       env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)
    assert p.returncode != 0 and "--distill-alpha" in p.stderr


def test_expert_load_is_kept_by_layer():
    """Each layer has its own experts: counts ``[layers, E]`` against the choices of the layers' routers, over micro-batches and both strands;
    whoever begins a new list of balance losses begins new counts."""
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import synthetic_step_batches
    from dhellam_b200.ops import moe as M
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    cfg = preset("tiny-moe", seq_length=16, moe_aux_loss_coeff=0.1)
    train = TrainConfig(micro_batch_size=2, global_batch_size=6, dtype="fp32")
    PS.set_state(None)
    tr = Trainer(cfg, ParallelConfig(), train, device="cpu")
    assert tr.expert_load() is None
    seen, fwd = [], M.router_topk_fwd
    try:
        M.router_topk_fwd = lambda x, w, k: (lambda r: (seen.append((w.data_ptr(), r[1])), r)[1])(fwd(x, w, k))
        for step in range(2):
            seen.clear()
            tr.optimizer.zero_grad()
            tr.engine.run_step(synthetic_step_batches(cfg, train, tr.ps, step, "cpu"))
            assert len(seen) == 3 * cfg.num_layers
            want = torch.zeros(cfg.num_layers, cfg.num_experts, dtype=torch.int64)
            where = {}
            for j, (first, second) in enumerate(tr.model.blocks):
                where[first.router_weight.data_ptr()], where[second.router_weight.data_ptr()] = j, cfg.num_layers - 1 - j
            for at, topi in seen:
                want[where[at]] += torch.bincount(topi.reshape(-1), minlength=cfg.num_experts)
            load = tr.expert_load()
            assert load.shape == want.shape and torch.equal(load.long(), want)
    finally:
        M.router_topk_fwd = fwd
    tr.env.moe_aux = []
    assert tr.env.moe_counts == [] and tr.expert_load() is None


def _imbalance(rank, world, par):
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import synthetic_step_batches
    from dhellam_b200.trainer import Trainer
    import torch.distributed as dist
    cfg = preset("tiny-moe", seq_length=16, moe_aux_loss_coeff=0.1, num_layers=4)
    pcfg = ParallelConfig(**par)
    tr = Trainer(cfg, pcfg, TrainConfig(micro_batch_size=1, global_batch_size=2 * pcfg.dp, dtype="fp32"), device="cpu")
    train = tr.train
    tr.optimizer.zero_grad()
    tr.engine.run_step(synthetic_step_batches(cfg, train, tr.ps, 0, "cpu"))
    mine = tr.expert_load()
    assert mine.shape == (cfg.num_layers // pcfg.pp, cfg.num_experts)
    every = [torch.empty_like(mine) for _ in range(world)]
    dist.all_gather(every, mine)
    load = (torch.stack(every).sum(0) if pcfg.pp == 1 else torch.cat(every)).double()
    assert math.isclose(tr.expert_imbalance(), float((load.amax(1) / load.mean(1)).max()), rel_tol=1e-12)


@pytest.mark.parametrize("par", [dict(dp=2, ep=2), dict(cp=2), dict(pp=2)], ids=["dp2", "cp2", "pp2"])
def test_expert_imbalance_over_ranks(par):
    run_ranks(_imbalance, 2, par)


def _padded(rank, world, par, dtype):
    """A batch whose samples end in padding, on this rank's share of the sequence, against counting by hand."""
    from dhellam_b200.config import ParallelConfig, TrainConfig, preset
    from dhellam_b200.data import cp_chunk_positions, make_microbatch, synthetic_tokens
    from dhellam_b200.parallel import state as PS
    from dhellam_b200.trainer import Trainer
    cfg = preset("tiny-moe", seq_length=16, moe_aux_loss_coeff=0.1)
    pcfg = ParallelConfig(**par)
    if world == 1:
        PS.set_state(None)
    tr = Trainer(cfg, pcfg, TrainConfig(micro_batch_size=3, global_batch_size=3 * pcfg.dp, dtype="fp32"), device="cpu")
    lengths = torch.tensor([16, 5, 11])
    mask = (torch.arange(16) < lengths[:, None]).to(dtype)
    mb = make_microbatch(cfg, tr.ps, synthetic_tokens(cfg, 3, 0), 0, 0, "cpu", token_mask=mask)
    mine = mask[:, cp_chunk_positions(16, pcfg.cp, tr.ps.cp_rank).long()].t().reshape(-1) != 0
    assert mb.token_mask.dtype == torch.bool and torch.equal(mb.token_mask, mine) and torch.equal(mb.loss_mask.reshape(-1), mine.float())
    tr.optimizer.zero_grad()
    tr.engine.run_step([mb])
    assert int(tr.expert_load().sum()) == cfg.num_layers * int(mine.sum()) * cfg.moe_top_k
    assert make_microbatch(cfg, tr.ps, synthetic_tokens(cfg, 3, 0), 0, 0, "cpu").token_mask is None
    for bad in (mask[:2], mask[:, :8], mask.float().t()):
        with pytest.raises(ValueError):
            make_microbatch(cfg, tr.ps, synthetic_tokens(cfg, 3, 0), 0, 0, "cpu", token_mask=bad)


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int64, torch.float32])
def test_padding_reaches_the_loss_and_the_balance(dtype):
    _padded(0, 1, {}, dtype)


def test_padding_reaches_the_loss_and_the_balance_of_context_parallel_ranks():
    run_ranks(_padded, 2, dict(cp=2), torch.bool)
