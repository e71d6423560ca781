"""Plain 64-bit restatements of the gated linear recurrence (stes_gated_scan_*) and of the distillation loss from a teacher's top
logits (stes_distill*), step by step on the CPU, with running bounds on what fp32 arithmetic may be off by.

The bounds are first-order running error analyses with u = 2^-24 (half a step of fp32): they depend on the inputs and on nothing
that a kernel returns."""
import numpy as np

U = 2.0 ** -24


def _sigmoid(x):
    t = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + t), t / (1 + t))


def gated_scan(pre, h0=None, lengths=None, reverse=False, dh=None, dlast=None, need_grad=False):
    """pre [B,T,2H], h0 [B,H] | [H] | None, dh [B,T,H] | None, dlast [B,H] | None, float64 arrays.
    -> dict of h, last (and dpre, dh0 [B,H]) with `<name>_err`: how far an fp32 evaluation may be off, in any association.

    Error of the states.  A gate is exp2(-|x| log2 e) (argument rounded: |x| u relative; exp2 good to 2 u), 1 + t (u), a reciprocal (2 u)
    and a product (u): under (|x| + 8) u relative, z and a alike.  A state is a sum of terms (product of a's) z c; a term from i steps
    back has met i gates with their errors and at most 3 roundings a step, whatever the association of the time axis, and a
    composition in a tree, in blocks and across workgroups adds fewer than 24 more.  With S the sum of the terms' magnitudes that is
    R_t = a_t (R_{t-1} + (|x| + 12) u S_{t-1}) + (|x| + 12) u z|c|,  S_t = a_t S_{t-1} + z|c|,  bound R_t + 24 u S_t.
    |x| counts as 104 at most: sigmoid(-104) is below half of the least fp32 number, and a gate beyond is 0 or 1 however its argument was
    rounded."""
    pre = np.asarray(pre, np.float64)
    B, T, W = pre.shape
    H = W // 2
    n = np.full(B, T) if lengths is None else np.clip(np.asarray(lengths), 0, T)
    start = np.zeros((B, H)) if h0 is None else np.broadcast_to(np.asarray(h0, np.float64), (B, H)).copy()
    out = {k: np.zeros((B, T, H)) for k in ("h", "h_err")}
    last, last_err = start.copy(), np.zeros((B, H))
    if need_grad:
        out["dpre"], out["dpre_err"] = np.zeros((B, T, W)), np.zeros((B, T, W))
        out["dh0"], out["dh0_err"] = np.zeros((B, H)), np.zeros((B, H))
    for b in range(B):
        order = list(range(n[b]))
        if reverse:
            order.reverse()
        x, S, R = start[b].copy(), np.abs(start[b]), np.zeros(H)
        before, before_err = {}, {}
        for t in order:
            g, c = pre[b, t, :H], pre[b, t, H:]
            z, a = _sigmoid(g), _sigmoid(-g)
            e = (np.minimum(np.abs(g), 104) + 12) * U
            before[t], before_err[t] = x, R + 24 * U * S
            R = a * (R + e * S) + e * z * np.abs(c)
            S = a * S + z * np.abs(c)
            x = a * x + z * c
            out["h"][b, t], out["h_err"][b, t] = x, R + 24 * U * S
        last[b], last_err[b] = x, R + 24 * U * S
        if not need_grad:
            continue
        # carry = a_{s+1} l_{s+1}: the same recurrence the other way round, fed with dh
        carry = np.zeros(H) if dlast is None else np.asarray(dlast, np.float64)[b].copy()
        S, R = np.abs(carry), np.zeros(H)
        for t in reversed(order):
            g, c = pre[b, t, :H], pre[b, t, H:]
            z, a = _sigmoid(g), _sigmoid(-g)
            e = (np.minimum(np.abs(g), 104) + 12) * U
            d = 0.0 if dh is None else np.asarray(dh[b, t], np.float64)
            lam, S = carry + d, S + np.abs(d)
            lam_err = R + 24 * U * S
            diff = c - before[t]
            diff_err = before_err[t] + U * (np.abs(c) + np.abs(before[t]))
            out["dpre"][b, t, :H] = lam * diff * z * a
            out["dpre_err"][b, t, :H] = (lam_err * np.abs(diff) + np.abs(lam) * diff_err) * z * a + np.abs(lam * diff) * z * a * (2 * e + 4 * U)
            out["dpre"][b, t, H:] = lam * z
            out["dpre_err"][b, t, H:] = lam_err * z + np.abs(lam) * z * (e + 2 * U)
            R = a * (R + e * S)
            carry, S = a * lam, a * S
        out["dh0"][b], out["dh0_err"][b] = carry, R + 24 * U * S
    out["last"], out["last_err"] = last, last_err
    return out


def topk_distill(logits, idx, val, tau=1.0, weight=None, denom=None, scale=1.0):
    """logits [M,V], idx [M,k] (below zero: unused), val [M,k], float64 -> dict of loss, dlogits and their fp32 bounds.

    y = (s - max) / tau carries 3 u |y| and its exp2 another (|y| + 2) u; the sum of V such terms in at least 4 strands adds at most
    V / 4 + 16 roundings of its own; so q is good to (4|y| + E + N) u relative with E the q-weighted mean of 4|y| + 2, and p alike
    over k terms.  log q = y - log(sum): its absolute error is the sum of those and 3 u of its parts.  The row sums are added in fp32
    within a workgroup (at most 64 + 16 roundings) and in 64 bits from there on."""
    x = np.asarray(logits, np.float64)
    M, V = x.shape
    idx, val = np.asarray(idx), np.asarray(val, np.float64)
    k = idx.shape[1]
    w = np.ones(M) if weight is None else np.asarray(weight, np.float64)
    denom = float(max(M, 1)) if denom is None else float(denom)
    grad, grad_err = np.zeros((M, V)), np.zeros((M, V))
    total, total_err, total_abs = 0.0, 0.0, 0.0
    for m in range(M):
        at = [j for j in range(k) if idx[m, j] >= 0 and val[m, j] > -np.inf]
        if not at or w[m] == 0:
            continue
        yt = (val[m, at] - val[m, at].max()) / tau
        pe = np.exp(yt)
        pe /= pe.sum()
        e_p = (4 * np.abs(yt) + 4 * (pe * np.abs(yt)).sum() + k + 24) * U
        P, P_err = np.zeros(V), np.zeros(V)
        for j, a in enumerate(at):
            P[idx[m, a]] += pe[j]
            P_err[idx[m, a]] += pe[j] * e_p[j]
        y = (x[m] - x[m].max()) / tau
        with np.errstate(over="ignore", invalid="ignore"):
            q = np.exp(y)
            z = q.sum()
            q /= z
            ay = np.where(q > 0, np.abs(y), 0.0)
            common = 4 * (q * ay).sum() + V / 4 + 24
            e_q = (4 * ay + common) * U
            on = P > 0
            logq = y[on] - np.log(z)
            rel = np.log(P[on]) - logq
            kl = (P[on] * rel).sum()
            kl_err = (P_err[on] * (np.abs(rel) + 1)).sum() + (P[on] * (common + 4 * np.abs(y[on]) + 3 * np.log(z) + 3 * np.abs(np.log(P[on])) + 3 * np.abs(rel))).sum() * U
        f = w[m] * tau / denom * scale
        grad[m] = f * (q - P)
        grad_err[m] = abs(f) * (q * e_q + P_err + 6 * U * (q + P))
        total += w[m] * kl
        total_err += abs(w[m]) * kl_err
        total_abs += abs(w[m] * kl)
    c = tau ** 2 / denom
    return {"loss": total * c, "loss_err": (total_err + 90 * U * total_abs) * c, "dlogits": grad, "dlogits_err": grad_err}
