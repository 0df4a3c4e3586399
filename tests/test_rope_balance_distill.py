"""Rotary forms, balance loss and distillation on CPU: the reference path against 64 bits, refusals, ranks, gradients by differences."""
import math

import pytest
import torch

import operator_oracles as O
from dhellam_b200.ops import loss as L
from dhellam_b200.ops import moe as M
from dhellam_b200.ops import rope as R


# --------------------------------------------------------------------------- rotary
def test_rope_frequencies_of_every_scaling():
    """Against the definitions written per pair; the ends are exact: fast pairs stay, slow pairs are divided by the factor."""
    r, theta, factor, old = 128, 500000.0, 8.0, 8192
    plain, one = R.rope_frequencies(r, theta)
    assert one == 1.0 and plain.dtype == torch.float64 and torch.allclose(plain, torch.tensor([theta ** (-2 * i / r) for i in range(r // 2)], dtype=torch.float64))
    lin, _ = R.rope_frequencies(r, theta, R.RopeScaling("linear", factor, old))
    assert torch.equal(lin, plain / factor)
    ntk, _ = R.rope_frequencies(r, theta, R.RopeScaling("ntk", factor, old))
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(plain[-1]) / factor, rel_tol=1e-12)
    llama, _ = R.rope_frequencies(r, theta, R.RopeScaling("llama3", factor, old))
    for i in range(r // 2):
        f, wave = float(plain[i]), 2 * math.pi / float(plain[i])
        if wave < old / 4.0:
            want = f
        elif wave > old / 1.0:
            want = f / factor
        else:
            smooth = (old / wave - 1.0) / (4.0 - 1.0)
            want = (1 - smooth) * f / factor + smooth * f
        assert math.isclose(float(llama[i]), want, rel_tol=1e-12), i
    yarn, scale = R.rope_frequencies(r, theta, R.RopeScaling("yarn", factor, old))
    assert math.isclose(scale, 0.1 * math.log(8.0) + 1.0)
    ratio = yarn / plain
    assert float(ratio[0]) == 1.0 and math.isclose(float(ratio[-1]), 1 / factor) and bool((ratio[1:] <= ratio[:-1] + 1e-15).all())
    assert R.rope_frequencies(r, theta, R.RopeScaling("yarn", factor, old, attention_factor=1.25))[1] == 1.25


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,r", [((7, 3, 16), 16), ((5, 2, 2, 10), 6), ((1, 1, 2), 2)])
def test_rope_reference_and_its_backward(shape, r, interleaved):
    torch.manual_seed(0)
    q, k = torch.randn(*shape), torch.randn(*shape[:-2], 1, shape[-1])
    pos = torch.randint(-5, 1000000, shape[:-2])
    freq, _ = R.rope_frequencies(r, 10000.0)
    q2, k2 = R.rope_fwd(q, k, pos, freq, interleaved, scale=1.2)
    for x, y in ((q, q2), (k, k2)):
        want, pair = O.rope(x, pos, freq, interleaved, 1.2)
        assert bool(((y.double() - want).abs() <= O.rope_bound(want, pair, torch.float32)).all())
        assert torch.equal(y[..., r:], x[..., r:])
    # the backward is the transpose: <rope(x), y> = <x, rope_bwd(y)>, and by differences of a linear map
    y = torch.randn(*shape)
    back, _ = R.rope_bwd(y, None, pos, freq, interleaved, scale=1.2)
    assert math.isclose(float((q2.double() * y.double()).sum()), float((q.double() * back.double()).sum()), rel_tol=1e-4, abs_tol=1e-4)
    if not interleaved and r == shape[-1] and len(shape) == 3:
        from dhellam_b200.ops.rope import rope_apply_, rope_table
        pos = torch.arange(shape[0], dtype=torch.int32)
        c, s = rope_table(16, r, 10000.0)
        packed = torch.cat([q, k, k], 1).reshape(shape[0], -1)
        rope_apply_(packed, pos, c, s, shape[1], 1, r)
        q2, k2 = R.rope_fwd(q, k, pos, freq)
        assert torch.allclose(packed[:, : shape[1] * r].view(q.shape), q2, atol=1e-6)


def test_rope_in_place_and_refusals():
    torch.manual_seed(1)
    buf = torch.randn(6, 4, 8)
    q, k = buf[:, :2], buf[:, 2:3]
    pos, (freq, _) = torch.arange(6), R.rope_frequencies(8, 10000.0)
    want = R.rope_fwd(q, k, pos, freq)
    last = buf[:, 3].clone()
    R.rope_fwd(q, k, pos, freq, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(buf[:, 3], last)
    bad = [dict(positions=torch.arange(5)), dict(positions=pos.float()), dict(freq=freq.float()), dict(freq=torch.ones(5, dtype=torch.float64)),
           dict(k=k[:, :, :6]), dict(k=k.double()), dict(q=buf.transpose(1, 2)), dict(out=(q[:5], k)), dict(out=(buf[:, 1:3], buf[:, 3:4])),
           dict(out=(torch.empty(6, 1, 8).expand(6, 2, 8), torch.empty(6, 1, 8))), dict(out=(q, q[:, :1]))]
    for b in bad:
        args = dict(q=q, k=k, positions=pos, freq=freq) | b
        with pytest.raises(ValueError):
            R.rope_fwd(**args)
    for b in (dict(kind="other"), dict(factor=0.5), dict(kind="llama3", factor=2.0, low_freq_factor=4.0), dict(original_max_position=0),
              dict(kind="yarn", factor=2.0, beta_fast=1.0)):
        with pytest.raises(ValueError):
            R.RopeScaling(**b)
    with pytest.raises(ValueError):
        R.rope_frequencies(7, 10000.0)


# --------------------------------------------------------------------------- balance
def router_case(T, E, k, seed=0, device="cpu", masked=True):
    g = torch.Generator().manual_seed(seed)
    probs = torch.softmax(torch.randn(T, E, generator=g) * 2, -1)
    top, ids = probs.topk(k, -1)
    mask = torch.rand(T, generator=g) < 0.7 if masked else None
    d = torch.randn(T, k, generator=g)
    return [None if t is None else t.to(device) for t in (probs, ids, top / top.sum(-1, keepdim=True), d, mask)]


@pytest.mark.parametrize("T,E,k,masked", [(0, 4, 2, False), (1, 1, 1, False), (37, 5, 2, True), (64, 8, 8, True), (9, 3, 1, False)])
def test_balance_reference_against_64_bits(T, E, k, masked):
    probs, ids, gates, dg, mask = router_case(T, E, k, masked=masked)
    loss, counts, bal = M.balance_loss_fwd(probs, ids.to(torch.int32), mask)
    want, wcounts, coef = O.balance(probs, ids, mask)
    assert counts.dtype == torch.int32 and torch.equal(counts, wcounts)
    assert abs(float(loss) - float(want)) <= O.EPS32 * (T + E + 20) * float(want)
    if T and not masked:
        assert torch.allclose(loss, M.aux_loss(probs, ids, E), rtol=1e-5)
    got = M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=bal)
    want, bound = O.router_gradient(dg, probs, ids, gates, 0.3, coef, mask)
    assert bool(((got.double() - want).abs() <= bound).all())


def test_router_gradient_by_differences():
    """Of sum(d * gates(logits)) + w * balance(softmax(logits)) with the choices held, in 64 bits."""
    T, E, k, w = 5, 6, 2, 0.7
    probs, ids, gates, dg, mask = router_case(T, E, k, seed=3)
    logits = probs.double().log()

    def value(l):
        p = torch.softmax(l, -1)
        s = p.gather(1, ids)
        return float((dg.double() * s / s.sum(-1, keepdim=True)).sum() + w * O.balance(p, ids, mask)[0])
    got = M.router_topk_bwd(dg, probs, ids, gates, E, w, balance=M.balance_loss_fwd(probs, ids, mask)[2])
    for t in range(T):
        for e in range(E):
            h = torch.zeros_like(logits)
            h[t, e] = 1e-5
            assert abs((value(logits + h) - value(logits - h)) / 2e-5 - float(got[t, e])) < 1e-5      # fp32 gradient, differences to 1e-9


def test_balance_without_counted_tokens_and_with_choices_out_of_range():
    probs, ids, gates, dg, _ = router_case(6, 4, 2)
    loss, counts, bal = M.balance_loss_fwd(probs, ids, torch.zeros(6, dtype=torch.bool))
    assert float(loss) == 0.0 and int(counts.sum()) == 0 and float(bal.coef.abs().sum()) == 0.0
    ids[0] = torch.tensor([-1, 4])
    ids[1, 1] = -1
    loss, counts, bal = M.balance_loss_fwd(probs, ids)
    assert int(counts.sum()) == 9
    got = M.router_topk_bwd(dg, probs, ids, gates, 4, 0.3, balance=bal)
    want, bound = O.router_gradient(dg, probs, ids, gates, 0.3, O.balance(probs, ids)[2])
    assert bool(((got.double() - want).abs() <= bound).all())
    probs = torch.full_like(probs, float("nan"))
    mask = torch.ones(6, dtype=torch.uint8)
    mask[2] = 0
    clean = torch.softmax(torch.randn(6, 4), -1)
    clean[2] = probs[2]
    assert math.isfinite(float(M.balance_loss_fwd(clean, ids, mask)[0]))


def test_balance_refusals():
    probs, ids, gates, dg, mask = router_case(6, 4, 2)
    bal = M.balance_loss_fwd(probs, ids)[2]
    for bad in (lambda: M.balance_loss_fwd(probs.double(), ids), lambda: M.balance_loss_fwd(probs, ids.float()),
                lambda: M.balance_loss_fwd(probs, ids[:5]), lambda: M.balance_loss_fwd(probs, ids, mask[:5]),
                lambda: M.balance_loss_fwd(probs, ids, mask.float()), lambda: M.balance_loss_fwd(probs, ids[:, :0]),
                lambda: M.router_topk_bwd(dg[:, :1], probs, ids, gates, 4), lambda: M.router_topk_bwd(dg, probs, ids, gates, 5),
                lambda: M.router_topk_bwd(dg, probs, ids, gates[:5], 4),
                lambda: M.router_topk_bwd(dg, probs, ids, gates, 4, 1.0, balance=M.Balance(bal.coef[:3], None))):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------- distillation
def distill_case(T, V, K, seed=0, hard=True, dtype=torch.float32, teacher=torch.float32, scale=3.0):
    """Rows with all entries, with padding, with none; a label twice among the teacher's ids; labels outside the vocabulary."""
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(T, V, generator=g) * scale).to(dtype)
    ids = torch.randint(0, V, (T, K), generator=g, dtype=torch.int32)
    top = (torch.randn(T, K, generator=g) * scale + 5).to(teacher)
    labels = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    for t in range(T):
        if t % 5 == 1 and K > 1:
            ids[t, K // 2:] = torch.tensor([-1, V, V + 7])[t % 3]
        if t % 7 == 2:
            ids[t] = -1
        if t % 4 == 3 and K > 1:
            ids[t, 0] = ids[t, -1] = labels[t]
        if t % 6 == 5:
            labels[t] = (-100, V, V + 5)[t % 3]
    g_ce, g_kd = torch.rand(T, generator=g), torch.rand(T, generator=g)
    for t in range(T):
        if t % 9 == 4:
            g_ce[t] = g_kd[t] = 0.0
    return z, labels if hard else None, ids, top, g_ce if hard else None, g_kd


def check_distill(case, tau, ce, kd, grad, dtype):
    z, labels, ids, top, g_ce, g_kd = case
    want = O.distill(z, labels, ids.cpu(), top.cpu().double(), tau, g_ce, g_kd)
    if labels is not None:
        err = (ce.cpu().double() - want["ce"]).abs()
        assert bool((err <= want["ce_bound"]).all()), float((err / want["ce_bound"].clamp_min(1e-30)).max())
    err = (kd.cpu().double() - want["kd"]).abs()
    assert bool((err <= want["kd_bound"]).all()), float((err / want["kd_bound"].clamp_min(1e-30)).max())
    err = (grad.cpu().double() - want["grad"]).abs()
    bound = want["grad_bound"] * (1 + O.HALF_STEP[dtype]) + O.HALF_STEP[dtype] * want["grad"].abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.7, 3.3])
@pytest.mark.parametrize("T,V,K,hard", [(20, 37, 5, True), (9, 64, 1, False), (1, 1, 1, True), (3, 11, 0, True), (0, 8, 2, True)])
def test_distill_reference_against_64_bits(T, V, K, hard, tau):
    case = z, labels, ids, top, g_ce, g_kd = distill_case(T, V, K, hard=hard)
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, labels, ids, top, tau)
    assert (ce is None) == (not hard) and saved.shape == (T, 4)
    out = torch.empty_like(z)
    grad = L.vocab_parallel_distill_bwd_(z, labels, ids, top, saved, g_ce, g_kd, tau, out=out)
    assert grad is out
    check_distill(case, tau, ce, kd, grad, torch.float32)
    keep = z.clone()
    same = L.vocab_parallel_distill_bwd_(keep, labels, ids, top, saved, g_ce, g_kd, tau)
    assert same is keep and torch.equal(keep, out)


def test_distill_gradient_by_differences():
    T, V, K, tau = 8, 9, 3, 1.7
    z, labels, ids, top, g_ce, g_kd = distill_case(T, V, K, seed=5)
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, labels, ids, top, tau)
    got = L.vocab_parallel_distill_bwd_(z.clone(), labels, ids, top, saved, g_ce, g_kd, tau)

    def value(x):
        r = O.distill(x, labels, ids, top.double(), tau)
        return float((r["ce"] * g_ce.double()).sum() + (r["kd"] * g_kd.double()).sum())
    for t in range(T):
        for v in range(V):
            h = torch.zeros(T, V, dtype=torch.float64)
            h[t, v] = 1e-5
            assert abs((value(z.double() + h) - value(z.double() - h)) / 2e-5 - float(got[t, v])) < 1e-5   # fp32 gradient, differences to 1e-9


def test_distill_equals_cross_entropy_and_vanishes_for_the_students_own_distribution():
    torch.manual_seed(2)
    z, labels = torch.randn(6, 12), torch.randint(0, 12, (6,), dtype=torch.int32)
    ids = torch.arange(12, dtype=torch.int64).expand(6, 12)
    ce, kd, _ = L.vocab_parallel_distill_fwd(z, labels, ids, z.clone(), 2.0)
    assert torch.allclose(ce, L.vocab_parallel_ce_fwd(z, labels)[0], atol=1e-5)
    assert float(kd.abs().max()) < 1e-5


def test_distill_masked_vocabulary_and_infinite_teacher():
    """Entries of -inf in the student (a masked vocabulary) and in the teacher; a chosen entry of -inf costs infinitely much, one
    without weight nothing."""
    z = torch.randn(4, 10)
    z[:, 7:] = float("-inf")
    ids = torch.tensor([[0, 1, 8], [2, 3, 4], [8, 9, 7], [1, 2, 3]], dtype=torch.int32)
    top = torch.tensor([[1.0, 2.0, float("-inf")], [1.0, 0.5, 0.0], [float("-inf")] * 3, [1.0, 2.0, 3.0]])
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, torch.tensor([0, 8, 1, 2], dtype=torch.int32), ids, top)
    assert bool(torch.isfinite(kd).all()) and float(kd[2]) == 0.0 and float(ce[1]) == float("inf")
    grad = L.vocab_parallel_distill_bwd_(z, torch.tensor([0, 8, 1, 2], dtype=torch.int32), ids, top, saved, torch.ones(4), torch.ones(4))
    assert bool(torch.isfinite(grad).all()) and float(grad[3, 7:].abs().max()) == 0.0


def test_distill_refusals():
    z, labels, ids, top, g_ce, g_kd = distill_case(6, 9, 3)
    saved = L.vocab_parallel_distill_fwd(z, labels, ids, top)[2]
    fwd = dict(logits=z, labels=labels, top_ids=ids, top_logits=top)
    for b in (dict(logits=z[0]), dict(labels=labels.long()), dict(labels=labels[:5]), dict(top_ids=ids.float()), dict(top_ids=ids[:5]),
              dict(top_logits=top[:, :2]), dict(top_logits=top.double()), dict(temperature=0.0), dict(temperature=float("inf")),
              dict(temperature=float("nan")), dict(temperature=-1.0), dict(vocab_start=1), dict(vocab_start=-1),
              dict(top_ids=torch.zeros(6, 1025, dtype=torch.int32), top_logits=torch.zeros(6, 1025))):
        with pytest.raises(ValueError):
            L.vocab_parallel_distill_fwd(**(fwd | b))
    wide = torch.zeros(6, 18)
    bwd = fwd | dict(saved=saved, g_ce=g_ce, g_kd=g_kd)
    for b in (dict(g_ce=None), dict(labels=None), dict(g_kd=g_kd.double()), dict(g_kd=g_kd[:5]), dict(saved=saved[:, :3]),
              dict(out=torch.empty(6, 8)), dict(out=torch.empty(6, 9, dtype=torch.bfloat16)), dict(out=torch.empty(1, 9).expand(6, 9)),
              dict(logits=wide[:, :9], out=wide[:, 9:]), dict(temperature=0.0)):
        with pytest.raises(ValueError):
            L.vocab_parallel_distill_bwd_(**(bwd | b))


def _two_shards(rank, world):
    z, labels, ids, top, g_ce, g_kd = distill_case(12, 24, 4, seed=9)
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, labels, ids, top, 1.6)
    whole = L.vocab_parallel_distill_bwd_(z.clone(), labels, ids, top, saved, g_ce, g_kd, 1.6)
    v0 = rank * 12
    import torch.distributed as dist
    shard = z[:, v0:v0 + 12].contiguous()
    ce2, kd2, saved2 = L.vocab_parallel_distill_fwd(shard, labels, ids, top, 1.6, vocab_start=v0, group=dist.group.WORLD)
    assert torch.allclose(ce, ce2, atol=1e-5) and torch.allclose(kd, kd2, atol=1e-5) and torch.allclose(saved, saved2, atol=1e-5)
    grad = L.vocab_parallel_distill_bwd_(shard, labels, ids, top, saved2, g_ce, g_kd, 1.6, vocab_start=v0)
    assert torch.allclose(grad, whole[:, v0:v0 + 12], atol=1e-6)


def test_distill_over_two_vocabulary_shards():
    from dist_utils import run_ranks
    run_ranks(_two_shards, 2)


def test_router_gradient_takes_what_it_took_before():
    """Probabilities in 64 bits, a weight in a tensor, no balance: PyTorch's ops by their types, against the formula."""
    probs, topi, gates, dg = (t.double() if t.is_floating_point() else t for t in router_case(50, 7, 3, 5)[:4])
    topi = topi.long()
    for weight in (0.0, 0.25, torch.tensor(0.25)):
        got = M.router_topk_bwd(dg, probs, topi, gates, 7, weight)
        p = probs.clone()
        d = torch.zeros_like(p).scatter_add(1, topi, (dg - (dg * gates).sum(1, keepdim=True)) / p.gather(1, topi).sum(1, keepdim=True))
        d = d + float(weight) * 7 * torch.bincount(topi.reshape(-1), minlength=7).double() / topi.numel() / 50
        want = p * (d - (d * p).sum(1, keepdim=True))
        # the balance's coefficients are fp32 numbers of three roundings
        assert got.dtype == torch.float64 and float((got - want).abs().max()) <= 1e-12 + 4 * 2.0 ** -24 * 0.25 * 7


def test_questions_about_tensors_need_no_gpu():
    """With the library loaded, where there may be no GPU: a CPU tensor and nothing at all are no operands of a kernel."""
    from ctypes import c_int, c_void_p
    from dhellam_b200 import kernels as K
    K.proto("dh_distill_combine", [c_void_p, c_int])
    assert not K.is_plain(torch.ones(2)) and not K.are_plain(torch.ones(2)) and not K.is_plain(None) and not K.are_plain(None, torch.ones(2))


def test_sizes_beyond_31_bits_of_a_loop_are_refused():
    """By the C functions, before anything is launched (sizes alone: no such tensor is made)."""
    from dhellam_b200 import kernels as K
    from ctypes import c_float, c_int64, c_void_p
    def call(name, types, *args):
        return K.proto(name, types)(*args)
    big = (1 << 30) + 1
    for T, V in ((big, 4), (4, big)):
        c = L._DISTILL_CALL.pack(0, V, 0, 0, 0, 0, 0, 0, 0, 0, T, V, 0, 0, 2 ** 31 - 1, 0, 0, 1.0)
        assert call("dh_distill_fwd", L._DISTILL_FWD, c, 0, 0, 0, 0) != 0
        assert call("dh_distill_bwd", L._DISTILL_BWD, c, 0, 0, 0, 0, V) != 0
    for T, E, k in ((1 << 28, 8, 5), (8, 1025, 2), (8, 4, 33), (8, 0, 1)):
        c = M._ROUTER_CALL.pack(0, E, 0, k, 0, 0, T, E, k, 0, 0)
        assert call("dh_balance_fwd", M._BALANCE_FWD, c, 0, 0, 0, 0) != 0
        assert call("dh_router_bwd", M._ROUTER_BWD, c, 0, k, 0, k, 0, 0.0, 0) != 0
    for heads_q, heads_k in (((1 << 28) + 1, 1), (0, (1 << 28) + 1)):
        c = R._ROPE_CALL.pack(*[0] * 16, heads_q, heads_k, 0, 0, 0, 1, 1, 2, 2, 0, 0, 0, 0, 0, 1.0)
        assert call("dh_rope_heads", R._ROPE_ARGS, c) != 0


def lowest_case(T, V, K, dtype, seed):
    """Rows whose label or whose teacher's entries, one of them up to most, lie on logits of the type's lowest value: losses near the end of
    what fp32 holds."""
    z, labels, ids, top, g_ce, g_kd = distill_case(T, V, K, seed=seed, dtype=dtype, scale=1.0)
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]).to(torch.int32)
    labels = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    low = torch.finfo(dtype).min
    for t in range(T):
        if t % 3 == 0:
            z[t, labels[t]] = low
        if t % 3 == 1:
            z[t, ids[t, -1]] = low
            top[t, -1] = top[t].max() - 2.0
        if t % 3 == 2:
            z[t, ids[t, : K // 5].long()] = low
            top[t] = 4.0
    return z, labels, ids, top, g_ce, g_kd


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.7, 3.3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_losses_near_the_end_of_the_type(dtype, tau):
    """A weight of at most 1/5 on 3.4e38 at a temperature of at most 3.3: the exact losses are fp32 numbers."""
    case = z, labels, ids, top, g_ce, g_kd = lowest_case(9, 400, 50, dtype, 3)
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, labels, ids, top, tau)
    grad = L.vocab_parallel_distill_bwd_(z.clone(), labels, ids, top, saved, g_ce, g_kd, tau)
    assert bool(torch.isfinite(ce).all()) and bool(torch.isfinite(kd).all())
    check_distill(case, tau, ce, kd, grad, dtype)


def far_teacher(T, V, K, dtype, teacher, low, seed):
    """``(case, exact)``: teacher's logits that are all ``low`` (a row whose entries are masked: each has the same weight), or lie a power of two
    above or below steps of a quarter; ``exact`` has them without that (a distribution does not change by it), so that its bounds are those
    of small logits."""
    z, labels, ids, top, g_ce, g_kd = distill_case(T, V, K, seed=seed, dtype=dtype)
    g = torch.Generator().manual_seed(seed)
    if low is None:
        near = torch.randint(0, 8, (T, K), generator=g) / 4
        far = near + (1 << 12) * (2 * torch.randint(0, 2, (T, 1), generator=g) - 1)
    else:
        near, far = torch.zeros(T, K), torch.full((T, K), float(low))
    top = far.to(teacher)
    assert bool((top.double() - top.double().amax(1, keepdim=True) == near.double() - near.double().amax(1, keepdim=True)).all())
    return (z, labels, ids, top, g_ce, g_kd), (z, labels, ids, near, g_ce, g_kd)


FAR_TEACHERS = [(torch.float32, None), (torch.float32, -1e9), (torch.bfloat16, -1e4), (torch.bfloat16, torch.finfo(torch.bfloat16).min),
                (torch.float16, torch.finfo(torch.float16).min), (torch.float32, torch.finfo(torch.float32).min)]


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.5, 1.7])
@pytest.mark.parametrize("teacher,low", FAR_TEACHERS)
def test_distill_teachers_logits_far_from_zero(teacher, low, tau):
    case, exact = far_teacher(12, 60, 16, torch.float32, teacher, low, 7)
    z, labels, ids, top, g_ce, g_kd = case
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, labels, ids, top, tau)
    check_distill(exact, tau, ce, kd, L.vocab_parallel_distill_bwd_(z.clone(), labels, ids, top, saved, g_ce, g_kd, tau), torch.float32)


def test_distill_operands_that_no_vector_load_takes_are_refused():
    """By the C functions, before anything is launched: statistics that do not start on 16 bytes, and temperatures at which an exponent's
    factor leaves fp32."""
    from dhellam_b200 import kernels as K

    def call(tau=1.0, T=4):
        return L._DISTILL_CALL.pack(0, 8, 0, 0, 0, 0, 0, 0, 0, 0, T, 8, 0, 0, 8, 0, 0, tau)

    def refused(why, name, types, *args):
        return K.proto(name, types)(*args) != 0 and why in K.lib().dh_last_error_string().decode()
    none = call(T=0)                      # nothing to launch either way
    for at in (8, 4, 24):
        assert refused("16 bytes", "dh_distill_fwd", L._DISTILL_FWD, none, 0, 0, at, 0)
        assert refused("16 bytes", "dh_distill_fwd", L._DISTILL_FWD, none, 0, 0, 0, at)
        assert refused("16 bytes", "dh_distill_bwd", L._DISTILL_BWD, none, at, 0, 0, 0, 8)
    for tau in (1e-39, 4e-39, 1e-50, 1e39):
        none = call(tau, T=0)
        assert refused("temperature", "dh_distill_fwd", L._DISTILL_FWD, none, 0, 0, 0, 0)
        assert refused("temperature", "dh_distill_bwd", L._DISTILL_BWD, none, 0, 0, 0, 0, 8)
    z, labels, ids, top, g_ce, g_kd = distill_case(6, 9, 3)
    saved = L.vocab_parallel_distill_fwd(z, labels, ids, top)[2]
    flat = torch.zeros(6 * 4 + 1, dtype=saved.dtype)
    odd = flat[1:].view(6, 4).copy_(saved)
    with pytest.raises(ValueError, match="16 bytes"):
        L.vocab_parallel_distill_bwd_(z, labels, ids, top, odd, g_ce, g_kd)
    for tau in (1e-39, 4e-39, 1e39):
        with pytest.raises(ValueError):
            L.vocab_parallel_distill_fwd(z, labels, ids, top, tau)


def test_rope_outputs_that_overlap_are_refused():
    """Outputs that share heads with one another, with themselves or with the other input; layouts in which nothing is shared are taken."""
    buf, pos, (freq, _) = torch.randn(6, 6, 8), torch.arange(6), R.rope_frequencies(8, 10000.0)
    room = torch.zeros(400)
    q, k = torch.randn(6, 3, 8), torch.randn(6, 2, 8)
    bad = [dict(out=(buf[:, :3], buf[:, 2:4])), dict(out=(buf[:, 1:4], buf[:, :2])), dict(q=buf[:, :3], k=buf[:, 2:4], out=(buf[:, :3], buf[:, 2:4])),
           dict(q=buf[:, :3], k=buf[:, 2:4], out=(buf[:, :3], torch.zeros(6, 2, 8))), dict(q=buf[:, 1:4], k=buf[:, :2], out=(torch.zeros(6, 3, 8), buf[:, :2])),
           dict(out=(room.as_strided((6, 3, 8), (24, 4, 1)), k)), dict(out=(room.as_strided((6, 3, 8), (20, 8, 1)), torch.zeros(6, 2, 8))),
           dict(out=(room.as_strided((6, 3, 8), (24, 8, 1)), room.as_strided((6, 2, 8), (24, 8, 1), 100))),
           dict(out=(room.as_strided((6, 3, 8), (40, 8, 1)), room.as_strided((6, 2, 8), (32, 8, 1), 24)))]
    for b in bad:
        with pytest.raises(ValueError):
            R.rope_fwd(**(dict(q=q, k=k, positions=pos, freq=freq) | b))
    want = R.rope_fwd(q, k, pos, freq)
    block = torch.zeros(7, 6, 8)                                             # heads outermost in memory
    wide = torch.zeros(6, 8, 8)
    for out in ((block[:3].transpose(0, 1), block[3:5].transpose(0, 1)), (wide[:, 2:5], wide[:, 5:7]), (wide[:, 4:7], wide[:, 1:3]),
                (wide[:, 0:6:2], wide[:, 1:4:2]), (block[0:6:2].transpose(0, 1), block[1:5:2].transpose(0, 1))):
        got = R.rope_fwd(q, k, pos, freq, out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # sequence-first views of [B, heads, S, d]: queries and keys of every batch beside one another
    store = torch.zeros(2, 5, 3, 8)
    four = store.permute(2, 0, 1, 3)
    q4, k4, p4 = q.view(3, 2, 3, 8), k.view(3, 2, 2, 8), pos.view(3, 2)
    got = R.rope_fwd(q4, k4, p4, freq, out=(four[:, :, :3], four[:, :, 3:]))
    assert torch.equal(got[0].reshape(6, 3, 8), want[0]) and torch.equal(got[1].reshape(6, 2, 8), want[1])
    four.copy_(torch.cat([q4, k4], 2))
    R.rope_fwd(four[:, :, :3], four[:, :, 3:], p4, freq, out=(four[:, :, :3], four[:, :, 3:]))
    assert torch.equal(store.permute(2, 0, 1, 3)[:, :, :3].reshape(6, 3, 8), want[0])


def test_a_corrupted_router_does_not_train_on_in_silence():
    """As before there was a kernel: chosen probabilities that sum to 0 give no finite gradient, and without a balance a choice outside the
    experts is an error of the CPU form."""
    probs, ids, gates, dg, _ = router_case(6, 5, 2)
    bal = M.balance_loss_fwd(probs, ids)[2]
    want = M.router_topk_bwd(dg, probs, ids, gates, 5, 0.3, balance=bal)
    probs[2, ids[2]] = 0.0
    for balance in (None, bal):
        got = M.router_topk_bwd(dg, probs, ids, gates, 5, 0.3, balance=balance)
        assert bool(torch.isnan(got[2]).any()) and torch.equal(got[3:], want[3:]) and torch.equal(got[:2], want[:2])
    for bad in (-1, 5):
        ids[1, 1] = bad
        for choices in (ids, ids.to(torch.int32)):
            with pytest.raises((RuntimeError, IndexError)):
                M.router_topk_bwd(dg, probs, choices, gates, 5)


def test_distill_backward_names_what_is_missing():
    z, labels, ids, top, g_ce, g_kd = distill_case(6, 9, 3)
    saved = L.vocab_parallel_distill_fwd(z, labels, ids, top)[2]
    for s, g in ((None, g_kd), (saved, None)):
        with pytest.raises(ValueError):
            L.vocab_parallel_distill_bwd_(z, labels, ids, top, s, g_ce, g)


def test_distill_calls_without_their_operands_are_refused():
    """By the C functions, before a kernel could write to or read from nothing."""
    from dhellam_b200 import kernels as K

    def refused(why, name, types, *args):
        return K.proto(name, types)(*args) != 0 and why in K.lib().dh_last_error_string().decode()
    bare, labelled = (L._DISTILL_CALL.pack(16, 8, 0, at, 0, 0, 0, 0, 0, 0, 4, 8, 0, 0, 8, 0, 0, 1.0) for at in (0, 16))
    assert refused("no place", "dh_distill_fwd", L._DISTILL_FWD, bare, 0, 16, 0, 0)
    assert refused("no place", "dh_distill_fwd", L._DISTILL_FWD, bare, 0, 0, 0, 16)
    assert refused("no place", "dh_distill_fwd", L._DISTILL_FWD, bare, 0, 0, 16, 0)
    for args in ((bare, 0, 0, 16, 16, 8), (bare, 16, 0, 0, 16, 8), (bare, 16, 0, 16, 0, 8), (labelled, 16, 0, 16, 16, 8)):
        assert refused("no statistics", "dh_distill_bwd", L._DISTILL_BWD, *args)
