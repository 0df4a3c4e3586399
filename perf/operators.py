"""What is measured of the operators that a further-trained (routed, long-context, distilled) model adds to the training step:

* ``rope``      rotary positions of separate queries and keys, forward and backward: pairs in halves or interleaved, a part of
                the head, frequencies scaled for long contexts;
* ``balance``   the router's balance loss with per-expert counts, and the gradient of gates and balance to the router's logits;
* ``distill``   cross entropy and distillation from a teacher's top logits, forward and backward.

Sizes are those of the presets in ``dhellam_b200/config.py`` and of the tests, or generic ones in between.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# --------------------------------------------------------------------------- the cases
def _rope(tokens, heads, kv_heads, head_dim, rotary, interleaved, scaling, base, first, docs=1, dtype="bf16", packed=False):
    return dict(kind="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary, interleaved=interleaved,
                scaling=scaling, base=base, first=first, docs=docs, dtype=dtype, packed=packed)


def _balance(tokens, experts, top_k, padding=0.0, ids="int64"):
    return dict(kind="balance", tokens=tokens, experts=experts, top_k=top_k, padding=padding, ids=ids)


def _distill(tokens, vocab, top, temperature, hard=True, dtype="bf16", pad=0, teacher="bf16", empty=0.0):
    return dict(kind="distill", tokens=tokens, vocab=vocab, top=top, temperature=temperature, hard=hard, dtype=dtype, pad=pad,
                teacher=teacher, empty=empty)


def listed():
    return [
        # one token at a far position: latency only
        dict(name="rope-one-token", **_rope(1, 32, 8, 128, 128, False, "llama3", 500000.0, 130000)),
        # the 8B preset at its sequence length, q and k as they lie in the packed projection, frequencies scaled for long contexts
        dict(name="rope-8b-long", **_rope(65536, 32, 8, 128, 128, False, "llama3", 500000.0, 0, packed=True)),
        # the GPT preset's heads, half of each rotated in interleaved pairs, documents of unequal length packed behind one another
        dict(name="rope-gpt-part", **_rope(3799, 40, 40, 128, 64, True, "none", 10000.0, 0, docs=7)),
        # a small head of which a quarter is rotated, fp32, yarn, sizes that no vector of 16 bytes divides
        dict(name="rope-odd-fp32", **_rope(1531, 12, 3, 80, 20, False, "yarn", 10000.0, 5000, dtype="fp32", packed=True)),
        # the routed test model
        dict(name="balance-small", **_balance(64, 4, 2)),
        # the Mixtral-style preset: one sequence
        dict(name="balance-mixtral", **_balance(16384, 8, 2)),
        # a padded batch, a number of experts that no vector divides
        dict(name="balance-odd", **_balance(5003, 61, 4, padding=0.2, ids="int32")),
        # many small experts over a long packed batch
        dict(name="balance-many", **_balance(65536, 256, 8, padding=0.05, ids="int32")),
        # the smoke run's vocabulary and a few tokens
        dict(name="distill-small", **_distill(32, 2048, 8, 1.0)),
        # few rows of the whole vocabulary (a short sample), both losses at an uneven temperature
        dict(name="distill-few-rows", **_distill(17, 128256, 100, 1.5, empty=0.1)),
        # GPT-sized odd vocabulary without padding: rows that start at any byte, no hard labels
        dict(name="distill-odd-rows", **_distill(2999, 50303, 50, 3.0, hard=False, teacher="fp32")),
        # one sequence of the 8B preset with its vocabulary
        dict(name="distill-8b", **_distill(4096, 128256, 64, 2.0)),
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["rope", "balance", "distill"])
    if kind == "rope":
        while True:
            kv = rng.choice([1, 2, 3, 8, 40])
            d = rng.choice([64, 80, 96, 128, 128, 192, 256])
            case = _rope(_log(rng, 1, 65536), kv * rng.choice([1, 2, 4, 8]), kv, d,
                         2 * max(1, int(d * rng.choice([0.25, 0.4, 0.5, 1.0, 1.0]) / 2)), rng.random() < 0.5,
                         rng.choice(["none", "linear", "ntk", "llama3", "yarn"]), rng.choice([10000.0, 500000.0, 1000000.0]),
                         _log(rng, 1, 1000000) - 1, docs=rng.choice([1, 1, 3, 9]), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                         packed=rng.random() < 0.5)
            if case["heads"] <= 64 and work(case)["bytes"] <= 2.7e9:
                return case
    if kind == "balance":
        experts = _log(rng, 2, 256)
        return _balance(_log(rng, 1, 65536), experts, rng.randint(1, min(8, experts)), padding=rng.choice([0.0, 0.0, 0.1, 0.5]),
                        ids=rng.choice(["int32", "int64"]))
    while True:
        case = _distill(_log(rng, 1, 16384), _log(rng, 500, 160000), _log(rng, 1, 256),
                        rng.choice([1.0, 2.0, 4.0, round(rng.uniform(0.7, 6.0), 2)]), hard=rng.random() < 0.75,
                        dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]), pad=rng.choice([0, 0, 0, 8, 13]),
                        teacher=rng.choice(["bf16", "fp16", "fp32"]), empty=rng.choice([0.0, 0.0, 0.1]))
        if work(case)["bytes"] <= 2.1e9:
            return case


# --------------------------------------------------------------------------- inputs
def _frequencies(rotary, base, scaling):
    """Rotation per position of each pair in 64 bits, and the factor on cosine and sine, for a model first trained at 8192 positions
    and stretched eightfold (llama3, yarn, linear, ntk)."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64) / rotary
    f, factor, old = base ** -i, 8.0, 8192.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        return (base * factor ** (rotary / max(rotary - 2, 1))) ** -i, 1.0
    if scaling == "llama3":
        turns = old * f / (2 * math.pi)                       # turns within the first training length; whole above 4, stretched below 1
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / factor * (1 - keep), 1.0
    if scaling == "yarn":
        def at(turns):
            return rotary * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rotary - 1)
        ramp = ((torch.arange(rotary // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale

    t = case["tokens"]
    if case["kind"] == "rope":
        h, hk, d, dt = case["heads"], case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]

        def heads():
            x = normal(t, h + 2 * hk, d).to(dt)
            q, k = x[:, :h], x[:, h:h + hk]
            return (q, k) if case["packed"] else (q.contiguous(), k.contiguous())
        (q, k), (dq, dk) = heads(), heads()
        # documents of unequal length behind one another, each counted from the case's first position
        cuts = torch.randint(0, t, (case["docs"] - 1,), generator=g, device=DEV)
        at = torch.arange(t, device=DEV)
        starts = torch.zeros(t, dtype=torch.int64, device=DEV).scatter_reduce_(0, cuts, cuts, "amax")
        positions = (at - torch.cummax(starts, 0).values + case["first"]).to(torch.int32)
        freq, factor = _frequencies(case["rotary"], case["base"], case["scaling"])
        return dict(case=case, q=q, k=k, dq=dq, dk=dk, positions=positions, freq=freq.to(DEV), factor=factor)
    if case["kind"] == "balance":
        e, k = case["experts"], case["top_k"]
        logits = normal(t, e) + normal(e)                     # some experts are more popular
        probs = torch.softmax(logits, dim=-1)
        top, ids = probs.topk(k, dim=-1)
        mask = None
        if case["padding"]:
            mask = torch.rand(t, generator=g, device=DEV) >= case["padding"]
        return dict(case=case, probs=probs, ids=ids.to(torch.int32 if case["ids"] == "int32" else torch.int64),
                    gates=top / top.sum(-1, keepdim=True), d_gates=normal(t, k, scale=0.01), mask=mask, weight=0.01)
    v, n = case["vocab"], case["top"]
    dt, tau = TYPES[case["dtype"]], case["temperature"]
    # the teacher's best entries: distinct ids, logits in falling order; some rows hold fewer (id -1 behind the last), some none
    first = torch.randint(0, v, (t, 1), generator=g, device=DEV)
    ids = (first + 7919 * torch.arange(n, device=DEV)) % v
    scores = (12.0 + 2.0 * normal(t, n)).sort(dim=1, descending=True).values
    wide = normal(t, v + case["pad"], scale=1.5)
    wide[:, :v].scatter_add_(1, ids, 0.7 * scores + normal(t, n))
    wide = wide.to(dt)
    held = torch.randint((n + 1) // 2, n + 1, (t, 1), generator=g, device=DEV)
    held = torch.where(torch.rand(t, 1, generator=g, device=DEV) < case["empty"], 0, held)
    ids = torch.where(torch.arange(n, device=DEV) < held, ids, -1).to(torch.int32)
    labels = torch.where(torch.rand(t, generator=g, device=DEV) < 0.5, first[:, 0], torch.randint(0, v, (t,), generator=g, device=DEV))
    counted = (torch.rand(t, generator=g, device=DEV) < 0.9).float()      # prompt tokens carry no loss
    share = counted / counted.sum().clamp_min(1.0)
    teacher = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["teacher"]]
    return dict(case=case, logits=wide[:, :v], ids=ids, scores=scores.to(teacher), labels=labels.to(torch.int32) if case["hard"] else None,
                g_ce=0.4 * share if case["hard"] else None, g_kd=0.6 * share, tau=tau, grad=torch.empty_like(wide)[:, :v])


# --------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "balance": _own_balance, "distill": _own_distill}[kind](state)
    return {"rope": _plain_rope, "balance": _plain_balance, "distill": _plain_distill}[kind](state)


def _own_rope(s):
    from dhellam_b200.ops.rope import rope_bwd, rope_fwd
    form = dict(interleaved=s["case"]["interleaved"], scale=s["factor"])
    q, k = rope_fwd(s["q"], s["k"], s["positions"], s["freq"], **form)
    dq, dk = rope_bwd(s["dq"], s["dk"], s["positions"], s["freq"], **form)
    return dict(q=q, k=k, dq=dq, dk=dk)


def _own_balance(s):
    from dhellam_b200.ops.moe import balance_loss_fwd, router_topk_bwd
    loss, counts, balance = balance_loss_fwd(s["probs"], s["ids"], mask=s["mask"])
    d_logits = router_topk_bwd(s["d_gates"], s["probs"], s["ids"], s["gates"], s["case"]["experts"], s["weight"], balance=balance)
    return dict(loss=loss, counts=counts, d_logits=d_logits)


def _own_distill(s):
    from dhellam_b200.ops.loss import vocab_parallel_distill_bwd_, vocab_parallel_distill_fwd
    given = (s["logits"], s["labels"], s["ids"], s["scores"])
    ce, kd, saved = vocab_parallel_distill_fwd(*given, temperature=s["tau"])
    grad = vocab_parallel_distill_bwd_(*given, saved, s["g_ce"], s["g_kd"], temperature=s["tau"], out=s["grad"])
    return dict(ce=ce, kd=kd, grad=grad)


def _plain_rope(s):
    r, inter = s["case"]["rotary"], s["case"]["interleaved"]
    angle = s["positions"].double()[:, None] * s["freq"]      # far positions need 64 bits
    cos, sin = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]

    def turn(x, sin):
        y = x.float().clone()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if inter else (y[..., :r // 2], y[..., r // 2:r])
        c, d = a * cos - b * sin, b * cos + a * sin
        a.copy_(c), b.copy_(d)
        return y.to(x.dtype)
    return dict(q=turn(s["q"], sin), k=turn(s["k"], sin), dq=turn(s["dq"], -sin), dk=turn(s["dk"], -sin))


def _plain_balance(s):
    p, ids = s["probs"], s["ids"].long()
    (t, e), k = p.shape, ids.shape[1]
    counted = torch.ones(t, device=p.device) if s["mask"] is None else s["mask"].float()
    n = counted.sum().clamp_min(1.0)
    counts = torch.zeros(e, dtype=torch.int32, device=p.device)
    counts.index_add_(0, ids.reshape(-1), counted.to(torch.int32)[:, None].expand(t, k).reshape(-1))
    part = counts.float() / (n * k)
    loss = e * (part * ((p * counted[:, None]).sum(0) / n)).sum()
    top = p.gather(1, ids)
    dp = (s["weight"] * e / n) * counted[:, None] * part
    dp.scatter_add_(1, ids, (s["d_gates"] - (s["d_gates"] * s["gates"]).sum(1, keepdim=True)) / top.sum(1, keepdim=True))
    return dict(loss=loss, counts=counts, d_logits=p * (dp - (dp * p).sum(1, keepdim=True)))


def _plain_distill(s):
    tau, ids = s["tau"], s["ids"].long()
    z = s["logits"].float()
    held = ids >= 0
    some = held.any(1)
    at = ids.clamp_min(0)
    q = (s["scores"].float() / tau).masked_fill(~held, -1e30)
    q = (q - q.amax(1, keepdim=True)).exp() * held
    q = q / q.sum(1, keepdim=True).clamp_min(1e-30)
    top = z.amax(1, keepdim=True)
    z = z - top                                               # every logit against its row's largest
    chosen = z.gather(1, at)
    e = (z / tau).exp()
    total = e.sum(1, keepdim=True)
    log_q = torch.where(q > 0, q, 1.0).log()
    kd = tau * tau * ((q * (log_q - chosen / tau)).sum(1) + total[:, 0].log()) * some
    grad = e * ((s["g_kd"] * some * tau)[:, None] / total)
    grad.scatter_add_(1, at, -(s["g_kd"] * tau)[:, None] * q)
    ce = None
    if s["labels"] is not None:
        lab = s["labels"].long()[:, None]
        target = z.gather(1, lab)[:, 0]
        e = z.exp_()
        total = e.sum(1, keepdim=True)
        ce = total[:, 0].log() - target
        grad += e * (s["g_ce"][:, None] / total)
        grad.scatter_add_(1, lab, -s["g_ce"][:, None])
    return dict(ce=ce, kd=kd, grad=grad.to(s["logits"].dtype))


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    t = case["tokens"]
    if case["kind"] == "rope":
        size = 2 if case["dtype"] == "bf16" else 4
        rows, rotated = t * (case["heads"] + case["kv_heads"]), case["rotary"]
        # q, k, dq, dk read and written, positions
        return dict(bytes=4.0 * size * rows * case["head_dim"] + 4.0 * t, flops=6.0 * rows * rotated)
    if case["kind"] == "balance":
        e, k = case["experts"], case["top_k"]
        ids = 8 if case["ids"] == "int64" else 4
        # probabilities, choices, gates and their gradients, mask read; gradient of the logits, counts, loss written
        return dict(bytes=8.0 * t * e + t * k * (8.0 + ids) + (t if case["padding"] else 0) + 4.0 * e + 4.0, flops=6.0 * t * e)
    v, n, size = case["vocab"], case["top"], 2 if case["dtype"] == "bf16" else 4
    soft = 4 if case["teacher"] == "fp32" else 2
    # logits, the teacher's entries, labels and the tokens' weights read; the gradient and the losses written
    return dict(bytes=2.0 * size * t * v + t * n * (4.0 + soft) + t * (20.0 if case["hard"] else 8.0),
                flops=(12.0 if case["hard"] else 7.0) * t * v)


# --------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "balance": _exact_balance, "distill": _exact_distill}[case["kind"]](case, s)


def _exact_rope(case, s):
    """Pairs as complex numbers, turned by exp(i a)."""
    r = case["rotary"]
    angle = s["positions"].double()[:, None, None] * s["freq"]
    by = torch.polar(torch.full_like(angle, s["factor"]), angle)

    def turn(x, by):
        out = []
        for a in range(0, x.shape[0], 8192):
            y = x[a:a + 8192].double()
            pairs = y[..., :r].unflatten(-1, (-1, 2)) if case["interleaved"] else y[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by[a:a + 8192])
            z = z if case["interleaved"] else z.transpose(-1, -2)
            out.append(torch.cat([z.flatten(-2), y[..., r:]], dim=-1))
        return torch.cat(out)
    return dict(q=turn(s["q"], by), k=turn(s["k"], by), dq=turn(s["dq"], by.conj()), dk=turn(s["dk"], by.conj()))


def _exact_balance(case, s):
    """The gradient by differentiation of both functions of the logits (their softmax is the given probabilities)."""
    e, k = case["experts"], case["top_k"]
    counted = torch.ones(case["tokens"], dtype=torch.bool, device=DEV) if s["mask"] is None else s["mask"]
    chosen = (s["ids"][..., None] == torch.arange(e, device=DEV)).any(1)             # a token's choices are distinct
    counts = (chosen & counted[:, None]).sum(0)
    n = max(int(counted.sum()), 1)
    p0 = s["probs"].double()
    logits = p0.log().requires_grad_(True)
    with torch.enable_grad():
        # the probabilities are rounded: the derivative of exp at the given value, not of a softmax normalised anew
        p = logits.exp()
        p = p - p.detach() + p0
        sel = p.gather(1, s["ids"].long())
        loss = e * (counts.double() / (n * k) * p[counted].sum(0) / n).sum()
        # gates as given: their share in the gradient is stated with them
        d_sel = (s["d_gates"].double() - (s["d_gates"].double() * s["gates"].double()).sum(1, keepdim=True)) / sel.detach().sum(1, keepdim=True)
        (dp,) = torch.autograd.grad(s["weight"] * loss + (d_sel * sel).sum(), logits)
    return dict(loss=loss.detach(), counts=counts.to(torch.int32), d_logits=dp - p0 * dp.sum(1, keepdim=True))


def _exact_distill(case, s):
    """512 rows at a time, the teacher's distribution spread over the whole vocabulary."""
    tau, ce, kd, grad = s["tau"], [], [], []
    for a in range(0, case["tokens"], 512):
        z, ids = s["logits"][a:a + 512].double(), s["ids"][a:a + 512].long()
        held = ids >= 0
        some = held.any(1)
        t = (s["scores"][a:a + 512].double() / tau).masked_fill(~held, float("-inf"))
        q = torch.softmax(t[some], dim=1)
        teacher = torch.zeros_like(z)
        teacher[some] = torch.zeros_like(z[some]).scatter_add_(1, ids[some].clamp_min(0), q)
        log_p = torch.log_softmax(z / tau, dim=1)
        kd.append(tau * tau * (torch.special.xlogy(teacher, teacher) - teacher * log_p).sum(1))
        d = (tau * s["g_kd"][a:a + 512].double())[:, None] * (log_p.exp() * some[:, None] - teacher)
        if s["labels"] is not None:
            lab = s["labels"][a:a + 512].long()[:, None]
            log_p = torch.log_softmax(z, dim=1)
            ce.append(-log_p.gather(1, lab)[:, 0])
            d += s["g_ce"][a:a + 512].double()[:, None] * (log_p.exp() - torch.zeros_like(z).scatter_(1, lab, 1.0))
        grad.append(d)
    return dict(ce=torch.cat(ce) if ce else None, kd=torch.cat(kd), grad=torch.cat(grad))
