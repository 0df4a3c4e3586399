"""Rotary positions, the router's balance and the distillation loss in 64 bits, row by row from their definitions, with the bounds of
the kernels' errors."""
import math

import torch

EPS32 = 2.0 ** -24                       # half a step of fp32, relative
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: EPS32}


# --------------------------------------------------------------------------- rotary
def rope(x, positions, freq, interleaved, scale, transposed=False):
    """``(turned, size)`` of ``x [..., H, d]`` in fp64, pairs as complex numbers; ``size`` is the |x| + |y| of a pair to which
    ``rope_bound`` refers.  An angle in 64 bits is itself rounded: position x frequency (2^-53 of it) here, and there once more, with
    the factor 1 / (2 pi) (2^-53) and the product with it (2^-53) behind it: 4 x 2^-53 of the angle, 5 to be above, which ``size``
    carries in units of the bound's 8e-7 (nothing below a million positions, as much again at 10^9)."""
    x = x.detach().cpu().double()
    freq = freq.cpu().double()
    r = 2 * freq.numel()
    angle = (positions.cpu().double().unsqueeze(-1) * freq).unsqueeze(-2)
    by = torch.polar(torch.full_like(angle, scale), -angle if transposed else angle)
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    else:
        a, b = x[..., : r // 2], x[..., r // 2:r]
    z = torch.complex(a.contiguous(), b.contiguous()) * by
    size = (a.abs() + b.abs()) * abs(scale) * (1 + angle.abs() * 5 * 2.0 ** -53 / 8e-7)
    out, pair = x.clone(), torch.zeros_like(x)
    if interleaved:
        out[..., 0:r:2], out[..., 1:r:2] = z.real, z.imag
        pair[..., 0:r:2] = pair[..., 1:r:2] = size
    else:
        out[..., : r // 2], out[..., r // 2:r] = z.real, z.imag
        pair[..., : r // 2] = pair[..., r // 2:r] = size
    return out, pair


def rope_bound(exact, pair, dtype):
    """The reduced angle in half turns is rounded to 32 bits (2^-25 of a half turn = 9.4e-8 rad), sine and cosine are off by two steps
    (2.4e-7), their product with the scale, two products and a sum by half a step each: below 8e-7 of |x| + |y|.  Then the type's
    rounding.  Elements that are copied have no error."""
    return 8e-7 * pair + HALF_STEP[dtype] * exact.abs() * (1 + 1e-6) * (pair > 0)


# --------------------------------------------------------------------------- balance
def balance(probs, topi, mask=None):
    """``(loss, counts, coef)``, counting choice by choice."""
    p, ids = probs.cpu().double(), topi.cpu().tolist()
    T, E = p.shape
    k = topi.shape[1]
    counted = [True] * T if mask is None else [bool(m) for m in mask.cpu().tolist()]
    n = sum(counted)
    counts = [0] * E
    sums = torch.zeros(E, dtype=torch.float64)
    for t in range(T):
        if not counted[t]:
            continue
        sums += p[t]
        for e in ids[t]:
            if 0 <= e < E:
                counts[e] += 1
    c = torch.tensor(counts, dtype=torch.float64)
    coef = E * c / (n * n * k) if n else torch.zeros(E, dtype=torch.float64)
    return (coef * sums).sum(), torch.tensor(counts, dtype=torch.int32), coef


def router_gradient(d_gates, probs, topi, gates, weight, coef, mask=None):
    """``(gradient of the logits, bound of its error)``."""
    p, dg, g = probs.cpu().double(), d_gates.cpu().double(), gates.cpu().double()
    (T, E), k = p.shape, topi.shape[1]
    out, bound = torch.zeros_like(p), torch.zeros_like(p)
    for t in range(T):
        ids = [(j, e) for j, e in enumerate(topi[t].tolist()) if 0 <= e < E]
        s = sum(float(p[t, e]) for _, e in ids)
        dot = sum(float(dg[t, j] * g[t, j]) for j, _ in ids)
        size = sum(float((dg[t, j] * g[t, j]).abs()) for j, _ in ids)
        d, a = torch.zeros(E, dtype=torch.float64), torch.zeros(E, dtype=torch.float64)
        for j, e in ids:
            if s:
                d[e] += (dg[t, j] - dot) / s
                a[e] += (dg[t, j].abs() + size) / s
        if weight and (mask is None or bool(mask[t])):
            d += weight * coef
            a += abs(weight) * coef
        out[t] = p[t] * (d - (d * p[t]).sum())
        # sums of k products, of k probabilities and of E products, each chain shorter than its number of terms, and ten single operations
        bound[t] = EPS32 * (E + 2 * k + 10) * p[t] * (a + (a * p[t]).sum())
    return out, bound * 1.01 + 1e-40


# --------------------------------------------------------------------------- distillation
def distill(logits, labels, ids, top, tau, g_ce=None, g_kd=None):
    """Dict of ``ce, kd, grad`` in fp64 with ``ce_bound, kd_bound, grad_bound`` (before the gradient's rounding to its type)."""
    z = logits.detach().cpu().double()
    T, V = z.shape
    k = ids.shape[1]
    r = {n: torch.zeros(T, dtype=torch.float64) for n in ("ce", "kd", "ce_bound", "kd_bound")}
    grad, gbound = torch.zeros_like(z), torch.zeros_like(z)
    # sums of exponentials: chains of at most V / 256 + 40 additions, exponentials off by 2 steps, their arguments by 2^-23 of
    # themselves, which weighs most where x exp(-x) is largest (0.37)
    e_sum = EPS32 * (V / 256 + 40) + 8 * EPS32
    for t in range(T):
        m = z[t].max()
        if m == -math.inf:                   # no logit at all: neither loss nor gradient
            gbound[t] = 1e-37
            continue
        lse, lse_t = torch.logsumexp(z[t], 0), torch.logsumexp(z[t] / tau, 0)
        lab = None if labels is None else int(labels[t])
        gc, gk = (0.0 if g_ce is None else float(g_ce[t])), (0.0 if g_kd is None else float(g_kd[t]))
        mag = float(z[t][torch.isfinite(z[t])].abs().max()) if torch.isfinite(z[t]).any() else 0.0
        p, p_t = torch.exp(z[t] - lse), torch.exp(z[t] / tau - lse_t)
        if lab is not None and 0 <= lab < V:
            r["ce"][t] = lse - z[t, lab]
            r["ce_bound"][t] = e_sum + 4 * EPS32 * ((lse - m).abs() + (m - z[t, lab]).abs())
            grad[t] += gc * p
            gbound[t] += abs(gc) * p
            grad[t, lab] -= gc
            gbound[t, lab] += abs(gc)
        held = [(int(ids[t, j]), float(top[t, j])) for j in range(k) if 0 <= int(ids[t, j]) < V]
        held = [(i, s) for i, s in held if s != -math.inf]
        if held:
            w = torch.tensor([s for _, s in held], dtype=torch.float64) / tau
            q = torch.softmax(w, 0)
            lq = torch.log_softmax(w, 0)
            size = 0.0
            for (i, _), qj, lj in zip(held, q.tolist(), lq.tolist()):
                if qj == 0.0:
                    continue
                r["kd"][t] += tau * tau * qj * (lj - (float(z[t, i]) / tau - float(lse_t)))
                size += qj * (abs(lj) + abs(float(z[t, i] - m)) / tau)
                grad[t, i] -= gk * tau * qj
                gbound[t, i] += abs(gk) * tau * qj
            grad[t] += gk * tau * p_t
            gbound[t] += abs(gk) * tau * p_t
            wmax = float(w.abs().max())
            # q itself is off by its exponent's rounding (2^-23 of the logits' size) and its sum's, like the student's
            e_q = EPS32 * (k + 16) + 4 * EPS32 * wmax
            r["kd_bound"][t] = tau * tau * (e_sum + (8 * EPS32 + e_q) * (size + (lse_t - m / tau).abs() + 1))
        # arguments z - lse and z / tau - lse carry three roundings of numbers up to `mag` (and the teacher's of its own), then the sums'
        top_mag = max([abs(s) for _, s in held], default=0.0)
        gbound[t] *= e_sum + EPS32 * (16 + 4 * (mag + 20) * max(1.0, 1.0 / tau) + 4 * (top_mag + 10) / tau)
    return dict(r, grad=grad, grad_bound=gbound + 1e-37)
