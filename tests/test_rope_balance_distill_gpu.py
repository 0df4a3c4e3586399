"""The kernels of csrc/rope.cu, balance.cu and distill.cu against 64 bits (bounds: ``operator_oracles``), on the sizes, types, strides
and masks where they can go wrong, and as a program uses them: in place, on another stream, captured and replayed."""
import math

import pytest
import torch

import operator_oracles as O
from dhellam_b200.ops import loss as L
from dhellam_b200.ops import moe as M
from dhellam_b200.ops import rope as R
from test_rope_balance_distill import FAR_TEACHERS, check_distill, distill_case, far_teacher, lowest_case, router_case

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def replay(fn):
    """``fn()`` captured into a graph after a warm-up, replayed twice; its outputs."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    return out


# --------------------------------------------------------------------------- rotary
def check_rope(q, k, pos, freq, interleaved, scale, **kw):
    for fn, back in ((R.rope_fwd, False), (R.rope_bwd, True)):
        got = fn(q, k, pos, freq, interleaved=interleaved, scale=scale, **kw)
        for x, y in zip((q, k), got):
            if x is None:
                assert y is None
                continue
            want, pair = O.rope(x, pos, freq, interleaved, scale, back)
            err = (y.cpu().double() - want).abs()
            assert y.dtype == x.dtype and bool((err <= O.rope_bound(want, pair, x.dtype)).all()), (fn.__name__, float(err.max()))


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,H,Hk,d,r", [(1, 1, 1, 128, 128), (1, 32, 8, 128, 128), (257, 5, 1, 128, 64), (63, 3, 3, 80, 20), (33, 2, 1, 6, 2),
                                        (40, 4, 2, 96, 38), (2000, 2, 1, 256, 256), (19, 1, 2, 7, 4), (5, 70, 3, 64, 48)])
def test_rope_sizes(T, H, Hk, d, r, dtype, interleaved):
    torch.manual_seed(T + d)
    q, k = torch.randn(T, H, d, device=DEV).to(dtype), torch.randn(T, Hk, d, device=DEV).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), device=DEV, dtype=torch.int32 if T % 2 else torch.int64)
    freq, scale = R.rope_frequencies(r, 500000.0, R.RopeScaling("yarn", 8.0), DEV)
    check_rope(q, k, pos, freq, interleaved, scale)


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_rope_strides_alignment_and_far_positions(dtype, interleaved):
    """Views of a packed projection, of one that starts at an odd element, sequence-first batches, positions beyond 32 bits and below zero."""
    torch.manual_seed(3)
    freq, _ = R.rope_frequencies(32, 10000.0, device=DEV)
    buf = torch.randn(30, 8 * 32 + 3, device=DEV).to(dtype)
    for first in (0, 1, 2):
        heads = buf[:, first:first + 8 * 32].unflatten(1, (8, 32))
        pos = torch.arange(30, device=DEV) - 7 + (1 << 33)
        check_rope(heads[:, :5], heads[:, 5:7], pos, freq, interleaved, 1.0)
    four = torch.randn(6, 5, 4, 40, device=DEV).to(dtype).transpose(0, 1)           # [S, B, heads, d] with the batch outermost in memory
    pos = torch.randint(-1000, 1000, (5, 6), device=DEV)
    check_rope(four[:, :, :3, 4:36], four[:, :, 3:, 4:36], pos, freq, interleaved, 0.9)
    check_rope(four, None, pos, freq, interleaved, 0.9, sm_budget=3)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,H,Hk,d,r", [(700, 5, 1, 96, 38), (1500, 2, 1, 128, 50), (310, 12, 3, 256, 102), (210, 17, 4, 80, 20), (900, 4, 1, 128, 100),
                                        (700, 5, 2, 192, 76), (300, 15, 7, 64, 14), (1500, 2, 1, 256, 254), (4100, 1, 0, 96, 2), (4099, 1, 1, 96, 62),
                                        (260, 100, 3, 16, 6), (2100, 1, 1, 512, 250), (9000, 1, 0, 8, 6)])
def test_rope_halves_of_odd_numbers_of_pairs(T, H, Hk, d, r, dtype):
    """Heads that pass through shared memory: odd halves and halves of 4k + 2, one to four rounds of a warp's lanes, heads that leave a step
    unfilled, queries alone; contiguous, as views of a packed projection, in place, sequence-first, on few SMs."""
    torch.manual_seed(T + r)
    freq, scale = R.rope_frequencies(r, 500000.0, R.RopeScaling("llama3", 8.0), DEV)
    pos = torch.randint(0, 1 << 20, (T,), device=DEV)
    buf = torch.randn(T, H + 2 * Hk + 1, d, device=DEV).to(dtype)
    q, k = buf[:, :H], buf[:, H:H + Hk] if Hk else None
    check_rope(q, k, pos, freq, False, scale)
    check_rope(q.contiguous(), None if k is None else k.contiguous(), pos, freq, False, scale, sm_budget=2)
    want, keep = R.rope_fwd(q, k, pos, freq, scale=scale), buf.clone()
    few = R.rope_fwd(q[5:9], None, pos[5:9], freq, scale=scale)[0]          # a few rows take the other kernel: the same bits
    assert torch.equal(few, want[0][5:9])
    R.rope_fwd(q, k, pos, freq, scale=scale, out=(q, k))
    assert torch.equal(q, want[0]) and (k is None or torch.equal(k, want[1]))
    assert torch.equal(buf[:, H + Hk:], keep[:, H + Hk:]) and torch.equal(buf[:, :H + Hk, r:], keep[:, :H + Hk, r:])
    if T % 10 == 0:
        four = keep.view(10, T // 10, H + 2 * Hk + 1, d).transpose(0, 1)
        got = R.rope_fwd(four[:, :, :H], None, pos.view(10, -1).t().contiguous(), freq, scale=scale)[0]
        assert torch.equal(got.transpose(0, 1).reshape(T, H, d), want[0])


def test_rope_copies_what_it_does_not_turn_bit_by_bit():
    g = torch.Generator().manual_seed(8)
    bits = torch.randint(-32768, 32768, (900, 6, 96), generator=g, dtype=torch.int16).to(DEV)
    x, pos = bits.view(BF), torch.arange(900, device=DEV)
    for r, interleaved in ((38, False), (38, True), (32, False), (20, False), (22, True)):
        q, k = R.rope_fwd(x[:, :5], x[:, 5:], pos, R.rope_frequencies(r, 10000.0, device=DEV)[0], interleaved=interleaved)
        assert torch.equal(torch.cat([q, k], 1).view(torch.int16)[..., r:], bits[..., r:])


def test_rope_in_place_leaves_the_rest_of_the_buffer():
    torch.manual_seed(4)
    buf = torch.randn(50, 10, 64, device=DEV).to(BF)
    freq, scale = R.rope_frequencies(48, 10000.0, device=DEV)
    pos = torch.arange(50, device=DEV)
    q, k = buf[:40, :6], buf[:40, 6:8]
    want = R.rope_fwd(q, k, pos[:40], freq, interleaved=True)
    keep = buf.clone()
    R.rope_fwd(q, k, pos[:40], freq, interleaved=True, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(buf[:, 8:], keep[:, 8:]) and torch.equal(buf[40:], keep[40:]) and torch.equal(buf[:40, :8, 48:], keep[:40, :8, 48:])
    out = torch.full((60, 12, 64), 7.0, device=DEV, dtype=BF)
    R.rope_fwd(keep[:40, :6], keep[:40, 6:8], pos[:40], freq, interleaved=True, out=(out[3:43, 1:7], out[3:43, 7:9]))
    assert torch.equal(out[3:43, 1:7], want[0]) and torch.equal(out[3:43, 7:9], want[1])
    out[3:43, 1:9] = 7.0
    assert bool((out == 7.0).all())
    empty = R.rope_fwd(q[:0], k[:0], pos[:0], freq)
    assert empty[0].shape == (0, 6, 64) and empty[1].shape == (0, 2, 64)


def test_rope_matches_the_table_form_of_whole_heads():
    torch.manual_seed(5)
    T, nq, nkv, d = 77, 4, 2, 128
    qkv = torch.randn(T, (nq + 2 * nkv) * d, device=DEV).to(BF)
    pos = torch.randint(0, 4096, (T,), device=DEV, dtype=torch.int32)
    c, s = R.rope_table(4096, d, 500000.0, DEV)
    heads = qkv.view(T, -1, d)
    q, k = R.rope_fwd(heads[:, :nq], heads[:, nq:nq + nkv], pos, R.rope_frequencies(d, 500000.0, device=DEV)[0])
    R.rope_apply_(qkv, pos, c, s, nq, nkv, d)
    # both round fp32 results that differ in their last bits: one step of bf16 (2^-7 of the value) where they straddle a border
    assert bool(((heads[:, :nq].float() - q.float()).abs() <= 2.0 ** -7 * q.float().abs() + 1e-5).all())
    assert bool(((heads[:, nq:nq + nkv].float() - k.float()).abs() <= 2.0 ** -7 * k.float().abs() + 1e-5).all())


def test_rope_on_another_stream_and_in_a_graph():
    torch.manual_seed(6)
    q, k = torch.randn(300, 4, 64, device=DEV).to(BF), torch.randn(300, 2, 64, device=DEV).to(BF)
    pos, freq = torch.arange(300, device=DEV), R.rope_frequencies(64, 10000.0, device=DEV)[0]
    want = R.rope_fwd(q, k, pos, freq)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = R.rope_fwd(q, k, pos, freq, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = replay(lambda: R.rope_fwd(q, k, pos, freq))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_rope_gpu_refusals():
    q, pos, freq = torch.zeros(4, 2, 8, device=DEV, dtype=BF), torch.arange(4, device=DEV), R.rope_frequencies(8, 1e4, device=DEV)[0]
    for bad in (dict(q=q.half()), dict(positions=pos.cpu()), dict(freq=freq.cpu()), dict(positions=torch.arange(8, device=DEV)[::2]),
                dict(out=(torch.zeros(4, 2, 8, dtype=BF), None))):
        with pytest.raises(ValueError):
            R.rope_fwd(**(dict(q=q, k=None, positions=pos, freq=freq) | bad))


# --------------------------------------------------------------------------- balance
def check_balance(probs, ids, gates, dg, mask, weight=0.3, **kw):
    T, E = probs.shape
    loss, counts, bal = M.balance_loss_fwd(probs, ids, mask, **kw)
    want, wcounts, coef = O.balance(probs, ids, mask)
    assert counts.dtype == torch.int32 and torch.equal(counts.cpu(), wcounts)
    # chains of additions: of tokens within a thread, over threads, over CTAs; then the single operations of the coefficients
    assert abs(float(loss) - float(want)) <= O.EPS32 * (400 + T / 64) * float(want)
    assert bool(((bal.coef.cpu().double() - coef).abs() <= 8 * O.EPS32 * coef).all())
    got = M.router_topk_bwd(dg, probs, ids, gates, E, weight, balance=bal, **kw)
    want, bound = O.router_gradient(dg, probs, ids, gates, weight, coef, mask)
    # the coefficients' own error on top of the oracle's bound
    err = (got.cpu().double() - want).abs()
    assert bool((err <= 2 * bound).all()), float((err / bound).max())
    return loss, counts, got


@pytest.mark.parametrize("masked", [False, True], ids=["all", "padded"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 4, 2), (64, 4, 2), (300, 5, 5), (1000, 61, 4), (2049, 8, 2), (700, 33, 8), (513, 64, 6),
                                   (257, 128, 1), (130, 255, 8), (200, 256, 8), (90, 257, 3), (65, 1000, 8), (70, 1024, 16), (6000, 2, 1)])
def test_balance_sizes(T, E, k, masked):
    probs, ids, gates, dg, mask = router_case(T, E, k, seed=T + E, device=DEV, masked=masked)
    first = check_balance(probs, ids if T % 2 else ids.to(torch.int32), gates, dg, mask)
    again = check_balance(probs, ids if T % 2 else ids.to(torch.int32), gates, dg, mask)
    assert all(torch.equal(a, b) for a, b in zip(first, again))          # sums in a fixed order


def test_balance_many_tokens():
    """Beyond what is counted one by one in Python: against PyTorch in 64 bits."""
    T, E, k = 50001, 96, 6
    probs, ids, gates, dg, mask = router_case(T, E, k, device=DEV)
    loss, counts, bal = M.balance_loss_fwd(probs, ids, mask)
    want = torch.bincount(ids[mask].reshape(-1), minlength=E)
    n = int(mask.sum())
    coef = want.double() * E / (n * float(n) * k)
    assert torch.equal(counts.long(), want)
    assert math.isclose(float(loss), float((coef * probs[mask].double().sum(0)).sum()), rel_tol=O.EPS32 * (400 + T / 64))
    got = M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=bal).double()
    p = probs.double()
    d = 0.3 * coef * mask[:, None].double()
    top = p.gather(1, ids)
    d = d.scatter_add(1, ids, (dg.double() - (dg.double() * gates.double()).sum(1, keepdim=True)) / top.sum(1, keepdim=True))
    want = p * (d - (d * p).sum(1, keepdim=True))
    size = p * (d.abs() + (d.abs() * p).sum(1, keepdim=True)) + p * ((dg.double() * gates.double()).abs().sum(1, keepdim=True) / top.sum(1, keepdim=True))
    assert bool(((got - want).abs() <= O.EPS32 * (E + 2 * k + 30) * size).all())


@pytest.mark.parametrize("T,E,k,masked", [(30000, 61, 4, True), (20011, 90, 8, True), (20011, 134, 3, False), (9000, 135, 3, True), (3000, 1022, 2, True),
                                          (3001, 1023, 2, False), (40000, 30, 2, True), (70001, 3, 2, True)])
def test_balance_of_rows_that_are_no_vectors(T, E, k, masked):
    """Experts that two or no fewer than one float divide, over several clusters and one; NaN where no token is counted; rows with a gap."""
    probs, ids, gates, dg, mask = router_case(T, E, k, device=DEV, masked=masked)
    wide = torch.full((T, E + E % 2 + 2), float("nan"), device=DEV)
    wide[:, :E] = probs
    if masked:
        wide[~mask] = float("nan")
    keep = torch.ones(T, dtype=torch.bool, device=DEV) if mask is None else mask
    want, n = torch.bincount(ids[keep].reshape(-1), minlength=E), int(keep.sum())
    coef = want.double() * E / (n * float(n) * k)
    for p in (wide[:, :E], wide[:, :E].contiguous()):
        loss, counts, bal = M.balance_loss_fwd(p, ids, mask)
        assert torch.equal(counts.long(), want)
        # chains of a thread's rows, of the threads and clusters that hold an expert, and of the experts
        assert math.isclose(float(loss), float((coef * probs[keep].double().sum(0)).sum()), rel_tol=O.EPS32 * (400 + T / 64))
        assert bool(((bal.coef.double() - coef).abs() <= 8 * O.EPS32 * coef).all())
        assert torch.equal(M.balance_loss_fwd(p, ids, mask)[0], loss)


def test_balance_strides_empty_masks_and_masked_values():
    T, E, k = 200, 12, 3
    probs, ids, gates, dg, mask = router_case(T, E, k, device=DEV)
    for first in (0, 1, 4):
        wide = torch.full((T, 20), 9.0, device=DEV)
        wide[:, first:first + E] = probs
        ids2 = torch.stack([ids, -ids], 2)[:, :, 0]                       # neither rows nor choices side by side
        check_balance(wide[:, first:first + E], ids2, gates.t().contiguous().t(), dg.repeat(1, 2)[:, :k], mask.to(torch.uint8) * 3)
        check_balance(wide[:, first:first + E], ids.repeat(1, 2)[:, 1:1 + k], gates, dg, mask)
    none = torch.zeros(T, dtype=torch.bool, device=DEV)
    loss, counts, got = check_balance(probs, ids, gates, dg, none)
    assert float(loss) == 0.0 and int(counts.sum()) == 0
    loss, counts, bal = M.balance_loss_fwd(probs[:0], ids[:0])
    assert float(loss) == 0.0 and int(counts.sum()) == 0 and float(bal.coef.abs().sum()) == 0.0
    assert M.router_topk_bwd(dg[:0], probs[:0], ids[:0], gates[:0], E, 0.3, balance=bal).shape == (0, E)
    dirty = probs.clone()
    dirty[~mask] = float("nan")
    a, b = M.balance_loss_fwd(dirty, ids, mask), M.balance_loss_fwd(probs, ids, mask)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    got = M.router_topk_bwd(dg, dirty, ids, gates, E, 0.3, balance=a[2])
    assert bool(torch.isfinite(got[mask]).all()) and torch.equal(got[mask], M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=b[2])[mask])


def test_balance_choices_out_of_range_twice_and_without_balance():
    T, E, k = 100, 10, 4
    probs, ids, gates, dg, mask = router_case(T, E, k, device=DEV)
    ids[::3, 1] = -1
    ids[::4, 2] = E
    ids[5] = -1
    ids[7, 3] = ids[7, 0]
    check_balance(probs, ids, gates, dg, mask)
    check_balance(probs, ids, gates, dg, mask, weight=0.0)
    plain = M.router_topk_bwd(dg, probs, ids, gates, E)
    want, bound = O.router_gradient(dg, probs, ids, gates, 0.0, torch.zeros(E))
    assert bool(((plain.cpu().double() - want).abs() <= bound).all())
    counted = M.router_topk_bwd(dg, probs, ids, gates, E, 0.3)            # all tokens count
    assert torch.equal(counted, M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=M.balance_loss_fwd(probs, ids)[2]))


def test_router_gradient_with_a_strided_balance():
    T, E, k = 64, 10, 2
    probs, ids, gates, dg, mask = router_case(T, E, k, device=DEV)
    bal = M.balance_loss_fwd(probs, ids, mask)[2]
    want = M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=bal)
    spread = M.Balance(torch.stack([bal.coef] * 2, 1)[:, 0], torch.stack([mask] * 3, 1)[:, 1])
    assert torch.equal(want, M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=spread))


def test_balance_on_another_stream_in_a_graph_and_with_a_budget():
    probs, ids, gates, dg, mask = router_case(3000, 40, 4, device=DEV)

    def step(**kw):
        loss, counts, bal = M.balance_loss_fwd(probs, ids, mask, **kw)
        return loss, counts, M.router_topk_bwd(dg, probs, ids, gates, 40, 0.1, balance=bal, **kw)
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = step(stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a, b) for a, b in zip(want, replay(step)))
    check_balance(probs, ids, gates, dg, mask, sm_budget=5)


def test_balance_of_many_clusters_in_a_graph_and_on_two_streams_at_once():
    """The form whose last kernel is put in place before its predecessor ends, captured; two calls that run side by side."""
    cases = [router_case(9000, 70, 3, seed=s, device=DEV) for s in (1, 2)]

    def step(c, **kw):
        probs, ids, gates, dg, mask = c
        loss, counts, bal = M.balance_loss_fwd(probs, ids, mask, **kw)
        return loss, counts, M.router_topk_bwd(dg, probs, ids, gates, 70, 0.1, balance=bal, **kw)
    want = [step(c) for c in cases]
    assert all(torch.equal(a, b) for a, b in zip(want[0], replay(lambda: step(cases[0]))))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [step(c, stream=s) for c, s in zip(cases, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


def test_router_of_more_experts_than_the_kernel_takes_in_a_graph():
    """PyTorch's ops for 1100 experts ask the host nothing, so they can be captured as before there was a kernel."""
    probs, ids, gates, dg, mask = router_case(60, 1100, 4, device=DEV)
    for balance in (False, True):
        def step():
            bal = M.balance_loss_fwd(probs, ids, mask)[2] if balance else None
            return M.router_topk_bwd(dg, probs, ids, gates, 1100, 0.5, balance=bal)
        want = step()
        assert torch.equal(replay(step), want)
        coef = O.balance(probs.cpu(), ids.cpu(), mask.cpu() if balance else None)[2]
        exact, bound = O.router_gradient(dg.cpu(), probs.cpu(), ids.cpu(), gates.cpu(), 0.5, coef, mask.cpu() if balance else None)
        assert bool(((want.cpu().double() - exact).abs() <= bound).all())


def test_balance_of_differentiated_probabilities_stays_differentiable():
    probs, ids, gates, dg, _ = router_case(20, 6, 2, device=DEV)
    p = probs.clone().requires_grad_(True)
    loss, counts, bal = M.balance_loss_fwd(p, ids)
    loss.backward()
    assert torch.allclose(p.grad, bal.coef.expand(20, 6), rtol=1e-5)


# --------------------------------------------------------------------------- distillation
def on_gpu(case, stride=0, first=0):
    """The case's tensors on the GPU; logits as a view of rows of ``stride`` elements that start at element ``first``."""
    z = case[0]
    if stride:
        wide = torch.full((z.shape[0], stride), 9.0, dtype=z.dtype, device=DEV)
        view = wide[:, first:first + z.shape[1]]
        view.copy_(z)
        z = view
    return (z.to(DEV),) + tuple(None if t is None else t.to(DEV) for t in case[1:])


def run_distill(case, tau, out=None, **kw):
    z, labels, ids, top, g_ce, g_kd = case
    ce, kd, saved = L.vocab_parallel_distill_fwd(z, labels, ids, top, tau, **kw)
    out = torch.empty_like(z) if out is None else out
    return ce, kd, L.vocab_parallel_distill_bwd_(z, labels, ids, top, saved, g_ce, g_kd, tau, out=out, **kw)


@pytest.mark.parametrize("tau", [1.0, 2.0, 4.0, 0.7, 3.3])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,V,K,hard", [(1, 1, 1, True), (1, 40000, 9, True), (20, 37, 5, True), (11, 2048, 8, False), (9, 4099, 33, True),
                                        (40, 1000, 256, True), (5, 16032, 1, True), (6, 777, 0, True), (3, 128256, 64, True)])
def test_distill_sizes(T, V, K, hard, dtype, tau):
    case = distill_case(T, V, K, seed=V, hard=hard, dtype=dtype, teacher=(BF, F32, torch.float16)[T % 3])
    ce, kd, grad = run_distill(on_gpu(case), tau)
    assert (ce is None) == (not hard)
    check_distill(case, tau, ce, kd, grad, dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V,stride,first", [(100, 104, 0), (101, 101, 0), (101, 117, 3), (2050, 2051, 1), (5, 9, 2), (3001, 3016, 8)])
def test_distill_strides_and_alignment(V, stride, first, dtype):
    """Rows that start at any element; what lies beside the rows stays."""
    case = distill_case(13, V, 6, seed=V, dtype=dtype)
    gpu = on_gpu(case, stride, first)
    wide = torch.full((13, stride + 2), 9.0, dtype=dtype, device=DEV)
    out = wide[:, first:first + V]
    ce, kd, grad = run_distill(gpu, 1.5, out=out)
    check_distill(case, 1.5, ce, kd, grad, dtype)
    out.fill_(9.0)
    assert bool((wide == 9.0).all())
    z = gpu[0]
    base = z._base
    keep = grad.clone()
    ce, kd, grad = run_distill(gpu, 1.5, out=z)                           # in place
    check_distill(case, 1.5, ce, kd, grad, dtype)
    z.fill_(9.0)
    assert bool((base == 9.0).all())
    ids64 = (gpu[1], torch.stack([gpu[2].long()] * 2, 2)[:, :, 0], gpu[3].t().contiguous().t()) + gpu[4:]
    ce, kd, grad = run_distill((on_gpu(case, stride, first)[0],) + ids64, 1.5)
    check_distill(case, 1.5, ce, kd, grad, dtype)


@pytest.mark.parametrize("scale", [0.01, 30.0, 3000.0])
@pytest.mark.parametrize("tau", [1.0, 2.0, 1.9])
def test_distill_flat_and_peaked_rows(scale, tau):
    """Logits far above zero, and so far apart that all but one exponential vanish, in rising and in falling order."""
    case = distill_case(8, 5000, 7, seed=1, dtype=F32, scale=scale)
    case[0][0] = case[0][0].sort().values + 5 * scale
    case[0][1] = case[0][1].sort(descending=True).values - 5 * scale
    check_distill(case, tau, *run_distill(on_gpu(case), tau), F32)


def test_distill_infinities_and_nan():
    """A masked vocabulary (-inf and the type's lowest value), infinite teacher's logits, NaN in one row only."""
    for low in (float("-inf"), torch.finfo(F32).min):
        z = torch.randn(6, 3000)
        z[:, 2500:] = low
        z[5, :2900] = low
        ids = torch.tensor([[0, 1, 2600], [2, 3, 4], [2600, 2601, 2602], [1, 2, 3], [5, 5, 5], [2950, 2951, 2960]], dtype=torch.int32)
        top = torch.tensor([[1.0, 2.0, float("-inf")], [1.0, 0.5, 0.0], [float("-inf")] * 3, [1.0, 2.0, 3.0], [0.0, 1.0, 2.0], [1.0, 2.0, 3.0]])
        labels = torch.tensor([0, 7, 1, 2, 5, 2999], dtype=torch.int32)
        if low != float("-inf"):
            labels[1] = 2600
        case = (z, labels, ids, top, torch.rand(6), torch.rand(6))
        for tau in (1.0, 2.0, 1.3):
            ce, kd, grad = run_distill(on_gpu(case), tau)
            assert bool(torch.isfinite(kd).all()) and float(kd[2]) == 0.0 and bool(torch.isfinite(grad).all())
            assert float(grad[3, 2500:].abs().max()) == 0.0
            if low == float("-inf"):
                check_distill(case, tau, ce, kd, grad, F32)
    z = torch.randn(3, 600)
    z[1, 77] = float("nan")
    case = on_gpu((z, torch.zeros(3, dtype=torch.int32), torch.ones(3, 2, dtype=torch.int32), torch.ones(3, 2), torch.ones(3), torch.ones(3)))
    ce, kd, grad = run_distill(case, 2.0)
    assert torch.isnan(ce).tolist() == [False, True, False] and torch.isnan(kd).tolist() == [False, True, False]
    assert bool(torch.isnan(grad[1]).any()) and bool(torch.isfinite(grad[0]).all()) and bool(torch.isfinite(grad[2]).all())
    case[4][1] = case[5][1] = 0.0                                         # a token without loss
    assert float(run_distill(case, 2.0)[2][1].abs().max()) == 0.0


@pytest.mark.parametrize("tau", [1.0, 1.4, 2.0])
def test_distill_rows_of_shards_and_their_combination(tau, monkeypatch):
    """Two ranks' calls one after the other, with the exchange between them replaced by what the two calls send."""
    case = distill_case(17, 4010, 12, seed=4, dtype=BF)
    z, labels, ids, top, g_ce, g_kd = on_gpu(case)
    sent = []
    monkeypatch.setattr(L, "group_size", lambda group: 2)
    monkeypatch.setattr(L.dist, "all_gather_into_tensor", lambda every, stats, group=None: sent.append(stats.clone()))
    for v0 in (0, 2005):
        L.vocab_parallel_distill_fwd(z[:, v0:v0 + 2005], labels, ids, top, tau, vocab_start=v0)
    monkeypatch.setattr(L.dist, "all_gather_into_tensor", lambda every, stats, group=None: every.copy_(torch.cat(sent)))
    ce, kd, saved = L.vocab_parallel_distill_fwd(z[:, :2005], labels, ids, top, tau)
    grad = torch.empty_like(z)
    for v0 in (0, 2005):
        part = slice(v0, v0 + 2005)
        L.vocab_parallel_distill_bwd_(z[:, part], labels, ids, top, saved, g_ce, g_kd, tau, vocab_start=v0, out=grad[:, part])
    check_distill(case, tau, ce, kd, grad, BF)


def test_distill_many_rows_are_the_same_whatever_shares_the_gpu_with_them():
    """More rows than CTAs, fewer SMs, another stream, a graph: bit by bit what a few rows give."""
    case = on_gpu(distill_case(2500, 520, 5, seed=2, dtype=BF))
    want = run_distill(case, 2.5)
    few = tuple(None if t is None else t[1000:1013] for t in case)
    got = run_distill(few, 2.5)
    check = distill_case(2500, 520, 5, seed=2, dtype=BF)
    check_distill(tuple(t[1000:1013] for t in check), 2.5, *got, BF)
    for kw in (dict(sm_budget=7), dict(stream=torch.cuda.Stream())):
        torch.cuda.synchronize()
        got = run_distill(case, 2.5, **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a, b) for a, b in zip(want, replay(lambda: run_distill(case, 2.5))))


@pytest.mark.parametrize("K", [40, 700])
def test_distill_few_rows_in_a_graph_and_on_two_streams_at_once(K):
    """Rows that clusters of CTAs share; more entries than a CTA has threads."""
    cases = [on_gpu(distill_case(7, 50000 + 3 * s, K, seed=s, dtype=BF)) for s in (1, 2)]
    want = [run_distill(c, 1.7) for c in cases]
    check_distill(distill_case(7, 50003, K, seed=1, dtype=BF), 1.7, *want[0], BF)
    assert all(torch.equal(a, b) for a, b in zip(want[0], replay(lambda: run_distill(cases[0], 1.7))))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [run_distill(c, 1.7, stream=s) for c, s in zip(cases, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


def test_distill_all_entries_the_same_id():
    """Every entry of a row, and its label, at one id; ids that share a slot of the table."""
    T, V, K = 6, 70000, 300
    z, labels, ids, top, g_ce, g_kd = distill_case(T, V, K, seed=3, dtype=F32)
    ids[0] = labels[0] = 65
    ids[1] = torch.arange(K) * 227 % V
    ids[2] = (torch.arange(K) % 7) * 4096
    ids[3, ::2] = labels[3] = 12345
    case = (z, labels, ids, top, g_ce, g_kd)
    for tau in (1.0, 2.6):
        check_distill(case, tau, *run_distill(on_gpu(case), tau), F32)


@pytest.mark.parametrize("T,V,K", [(3, 40, k) for k in (1, 31, 32, 33, 63, 127, 500, 1024)] + [(70, 3000, 31), (70, 3000, 127), (30, 3000, 1024),
                                                                                                (1300, 700, 33), (200, 700, 500)])
def test_distill_tables_of_entries(T, V, K):
    """As many entries as a row's places, more entries than the vocabulary has ids (all of them twins), ids that fall on the same place of
    the table, the label among them; few and many rows take CTAs of different sizes."""
    case = z, labels, ids, top, g_ce, g_kd = distill_case(T, V, K, seed=K, scale=2.0)
    ids[0] = torch.arange(K) % V                          # every id, in order
    ids[T // 2] = (torch.arange(K) * 2048) % V            # and multiples of a power of two
    labels[0], labels[T // 2] = 0, 2048 % V
    there = on_gpu(case)
    ce, kd, grad = run_distill(there, 1.7)
    check_distill(case, 1.7, ce, kd, grad, F32)
    for _ in range(3):
        assert torch.equal(run_distill(there, 1.7)[2], grad)


def test_distill_far_rows_of_a_long_batch():
    """Element offsets beyond 32 bits: the last rows of 2^31 + 2^23 logits."""
    T, V = 16450, 131072
    z = torch.zeros(T, V, device=DEV, dtype=BF)
    small = distill_case(6, V, 4, seed=8, dtype=BF)
    z[-6:] = small[0].to(DEV)
    rest = [None if t is None else torch.cat([torch.zeros((T - 6,) + t.shape[1:], dtype=t.dtype), t]).to(DEV) for t in small[1:]]
    ce, kd, grad = run_distill((z, *rest), 2.0, out=z)
    check_distill(small, 2.0, ce[-6:], kd[-6:], grad[-6:], BF)
    assert float(grad[:-6].abs().max()) == 0.0                            # no gradients there


def test_distill_gpu_refusals():
    z, labels, ids, top, g_ce, g_kd = on_gpu(distill_case(4, 64, 3))
    for bad in (dict(logits=z.half()), dict(logits=z.t().contiguous().t()), dict(labels=labels.cpu()), dict(top_ids=ids.cpu())):
        with pytest.raises(ValueError):
            L.vocab_parallel_distill_fwd(**(dict(logits=z, labels=labels, top_ids=ids, top_logits=top) | bad))


def masked_parts(T, V, K, dtype, low, live, seed):
    """``(case, exact)``: rows of which only the columns ``live`` are not ``low``; labels and entries lie there, rows 1, 5, ... have no label.
    ``exact`` has -inf in place of ``low``: from -1e4 on both weigh nothing, in 64 bits either (temperatures up to 4)."""
    a, b = live
    z, labels, ids, top, g_ce, g_kd = distill_case(T, b - a, K, seed=seed, dtype=dtype)
    labels, ids = torch.where((labels >= 0) & (labels < b - a), labels + a, -100), torch.where((ids >= 0) & (ids < b - a), ids + a, -1)
    labels[1::4] = -100
    case, exact = (torch.full((T, V), v, dtype=dtype) for v in (low, float("-inf")))
    case[:, a:b] = exact[:, a:b] = z
    rest = (labels, ids.to(torch.int32), top, g_ce, g_kd)
    return (case, *rest), (exact, *rest)


@pytest.mark.parametrize("low", [-1e4, -1e6, -1e9, "lowest", float("-inf")])
@pytest.mark.parametrize("T,V,dtype", [(3, 3000, F32), (200, 5000, F32), (1, 40000, BF), (3, 40001, F32), (17, 128256, BF)])
def test_distill_masked_parts_of_shared_rows(T, V, dtype, low):
    """Rows that 2 to 8 CTAs share, of which the first eighth, the first half, or all but the last eighth, is masked: the shares of the
    label and of the teacher's entries are far above other shares; no label is no label whatever is masked."""
    low = torch.finfo(dtype).min if low == "lowest" else low
    for part, live in enumerate(((V // 8, V), (V // 2, V), (V - V // 8, V), (V // 3, V // 2))):
        case, exact = masked_parts(T, V, 9, dtype, low, live, seed=V + part)
        for tau in (1.0, 1.5, 2.0, 4.0):
            ce, kd, grad = run_distill(on_gpu(case), tau)
            check_distill(exact, tau, ce, kd, grad, dtype)
            assert float(ce[1::4].abs().sum()) == 0.0


@pytest.mark.parametrize("low", [-1e9, "lowest", float("-inf")])
def test_distill_masked_parts_of_shared_rows_are_what_many_rows_give(low):
    """The same rows held by one CTA each, in a call of many, and as two shards of which one is masked as a whole."""
    low = torch.finfo(F32).min if low == "lowest" else low
    case, exact = masked_parts(4, 6000, 7, F32, low, (3000, 6000), seed=6)
    many = tuple(t.repeat(*([400] + [1] * (t.dim() - 1))) for t in case)
    few, all_rows = run_distill(on_gpu(case), 1.7), run_distill(on_gpu(many), 1.7)
    check_distill(exact, 1.7, *few, F32)
    check_distill(exact, 1.7, *(t[800:804] for t in all_rows), F32)
    z, labels, ids, top, g_ce, g_kd = on_gpu(case)
    stats = []
    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(L, "group_size", lambda group: 2)
        patch.setattr(L.dist, "all_gather_into_tensor", lambda every, mine, group=None: stats.append(mine.clone()))
        for v0 in (0, 3000):
            L.vocab_parallel_distill_fwd(z[:, v0:v0 + 3000], labels, ids, top, 1.7, vocab_start=v0)
        patch.setattr(L.dist, "all_gather_into_tensor", lambda every, mine, group=None: every.copy_(torch.cat(stats)))
        ce, kd, saved = L.vocab_parallel_distill_fwd(z[:, :3000], labels, ids, top, 1.7)
    grad = torch.empty_like(z)
    for v0 in (0, 3000):
        L.vocab_parallel_distill_bwd_(z[:, v0:v0 + 3000], labels, ids, top, saved, g_ce, g_kd, 1.7, vocab_start=v0, out=grad[:, v0:v0 + 3000])
    check_distill(exact, 1.7, ce, kd, grad, F32)


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.7, 3.3])
@pytest.mark.parametrize("T,V,K,dtype", [(9, 400, 50, BF), (9, 400, 50, F32), (6, 40000, 1000, BF), (6, 20001, 700, F32), (700, 900, 40, BF)])
def test_distill_losses_near_the_end_of_the_type(T, V, K, dtype, tau):
    case = lowest_case(T, V, K, dtype, 3)
    ce, kd, grad = run_distill(on_gpu(case), tau)
    assert bool(torch.isfinite(ce).all()) and bool(torch.isfinite(kd).all())
    check_distill(case, tau, ce, kd, grad, dtype)


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.5, 1.7])
@pytest.mark.parametrize("teacher,low", FAR_TEACHERS)
def test_distill_teachers_logits_far_from_zero(teacher, low, tau, monkeypatch):
    """Rows that CTAs share, rows of one CTA, and two shards."""
    for T, V, K in ((6, 30000, 16), (700, 300, 40), (9, 777, 700)):
        case, exact = far_teacher(T, V, K, F32, teacher, low, 7)
        check_distill(exact, tau, *run_distill(on_gpu(case), tau), F32)
    case, exact = far_teacher(8, 4000, 16, F32, teacher, low, 8)
    z, labels, ids, top, g_ce, g_kd = on_gpu(case)
    sent = []
    monkeypatch.setattr(L, "group_size", lambda group: 2)
    monkeypatch.setattr(L.dist, "all_gather_into_tensor", lambda every, stats, group=None: sent.append(stats.clone()))
    for v0 in (0, 2000):
        L.vocab_parallel_distill_fwd(z[:, v0:v0 + 2000], labels, ids, top, tau, vocab_start=v0)
    monkeypatch.setattr(L.dist, "all_gather_into_tensor", lambda every, stats, group=None: every.copy_(torch.cat(sent)))
    grad = torch.empty_like(z)
    for v0 in (0, 2000):                                                  # each rank has what its own call saved
        part = z[:, v0:v0 + 2000]
        ce, kd, saved = L.vocab_parallel_distill_fwd(part, labels, ids, top, tau, vocab_start=v0)
        L.vocab_parallel_distill_bwd_(part, labels, ids, top, saved, g_ce, g_kd, tau, vocab_start=v0, out=grad[:, v0:v0 + 2000])
    check_distill(exact, tau, ce, kd, grad, F32)


def test_router_gradient_of_chosen_probabilities_that_sum_to_zero():
    """No finite gradient in that row, by the kernel and by the PyTorch ops; rows without any choice have the balance's alone."""
    for E in (6, 61, 1100):
        probs, ids, gates, dg, mask = router_case(40, E, 3, device=DEV)
        bal = M.balance_loss_fwd(probs, ids, mask)[2]
        want = M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=bal)
        probs[7, ids[7]] = 0.0
        for weight, balance in ((0.3, bal), (0.0, None)):
            got = M.router_topk_bwd(dg, probs, ids, gates, E, weight, balance=balance)
            assert bool(torch.isnan(got[7]).any()) and bool(torch.isfinite(got[8:]).all()) and bool(torch.isfinite(got[:7]).all())
            assert balance is None or torch.equal(got[8:], want[8:])
        ids[9] = -1
        assert bool(torch.isfinite(M.router_topk_bwd(dg, probs, ids, gates, E, 0.3, balance=bal)[9]).all())


def test_router_gradient_without_a_balance_keeps_its_budget(monkeypatch):
    """The balance that it then counts itself runs on as few SMs."""
    probs, ids, gates, dg, _ = router_case(30, 8, 2, device=DEV)
    seen, fwd = [], M.balance_loss_fwd
    monkeypatch.setattr(M, "balance_loss_fwd", lambda *a, **kw: (seen.append((a, kw)), fwd(*a, **kw))[1])
    M.router_topk_bwd(dg, probs, ids, gates, 8, 0.3, sm_budget=9)
    assert len(seen) == 1 and (seen[0][1].get("sm_budget") or (seen[0][0] + (None,) * 4)[3]) == 9
