"""Plain implementations of the operators on rows of logits (pz_process_logits,
pz_distill_*, pz_lm_head_logits_i8), in numpy, from their definitions."""
from __future__ import annotations

import numpy as np

F32 = np.float32


# --------------------------------------------------------------------------
# pz_process_logits
# --------------------------------------------------------------------------
def process_row(x, V, cfg=None, hist=None, bias=None, allowed=None, wide=False):
    """One row: the contract's fp32 steps, or (wide) the same in fp64.
    cfg: (rep, freq, pres); hist: ids; bias: (ids, values); allowed: bools."""
    t = np.float64 if wide else F32
    x = np.array(x, dtype=t)
    with np.errstate(all="ignore"):
        if hist is not None and len(hist) and cfg is not None:
            rep, freq, pres = (t(c) for c in cfg)
            if rep != 1 or freq != 0 or pres != 0:
                for v, c in zip(*np.unique(hist, return_counts=True)):
                    if 0 <= v < V:
                        y = x[v]
                        if rep != 1:
                            y = y / rep if y > 0 else y * rep
                        x[v] = y - (t(c) * freq + pres)
        if bias is not None:
            for v, b in {int(i): b for i, b in zip(*bias)}.items():
                if 0 <= v < V:
                    x[v] = x[v] + t(b)
        if allowed is not None:
            x[~allowed] = -np.inf
    return x


def bf16_round(x):
    """float32 values rounded to bfloat16 (nearest even), as float32."""
    u = np.ascontiguousarray(x, dtype=F32).view(np.uint32)
    r = ((u >> np.uint32(16)) & np.uint32(1)) + np.uint32(0x7FFF)
    with np.errstate(over="ignore"):
        y = ((u + r) & np.uint32(0xFFFF0000)).view(F32)
    return np.where(np.isnan(x), F32(np.nan), y)


def pack_mask(allowed, words):
    """Bools [rows, V] as int32 words [rows, words]; bits past V are set (they
    must not matter)."""
    rows, V = allowed.shape
    bits = np.ones((rows, words * 32), dtype=np.uint8)
    bits[:, :V] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)


# --------------------------------------------------------------------------
# pz_distill_*
# --------------------------------------------------------------------------
def distill_row(x, ids, values, T=1.0, rest=False, weight=1.0):
    """(loss, gradient, bound on the loss's error, bounds on the gradient's)
    of one row in fp64; the bounds are those of the kernels' fp32 steps.

    In units of u = 2^-24: an e = 2^((s - m) c) is off by at most 2u of ex2,
    ln 2 * 3u per unit of its exponent (the difference, c and the product are
    each rounded: 2.1u), a sum of a row by (terms a thread adds + joins + the
    rescalings between them) < 400u, and a listed probability by the exp and
    the division (4u) and its exponent's rounding (2u per unit).  The list's
    own sum is in fp64; loss and gradient are rounded to fp32 once (and the
    factors of the gradient, a handful of times)."""
    u = 2.0 ** -24
    x = np.asarray(x, dtype=np.float64)
    V = x.shape[0]
    zero = (0.0, np.zeros(V), 0.0, np.zeros(V))
    ids, values = np.asarray(ids), np.asarray(values, dtype=np.float64)
    keep = (ids >= 0) & (ids < V)
    ids, values = ids[keep], values[keep]
    if weight == 0 or len(ids) == 0:
        return zero
    with np.errstate(all="ignore"):
        if not rest:
            t = values / T
            if not np.isnan(t).any():
                if t.max() == -np.inf:
                    return zero
                p = np.exp(t - t.max())
                spread = np.where(p > 0, t.max() - t, 0)
            else:
                p, spread = t, t
            p = p / p.sum()
            rho = 0.0
        else:
            p = np.exp(values)
            spread = np.where(p > 0, np.abs(values), 0)
            rho = 0.0 if len(np.unique(ids)) == V else max(0.0, 1.0 - p.sum()) if not np.isnan(p).any() else np.nan
        target, dp = np.zeros(V), np.zeros(V)
        np.add.at(target, ids, p)
        np.add.at(dp, ids, p * (6 + 2 * spread) * u)
        on = np.zeros(V, dtype=bool)
        on[ids] = True
        if np.isnan(x).any() or np.isnan(p).any() or (x == np.inf).any():
            nan = np.full(V, np.nan)
            return np.nan, nan, 0.0, np.zeros(V)
        m = x.max()
        if m == -np.inf:
            return np.inf * weight, np.zeros(V), 0.0, np.zeros(V)
        s = (x - m) / T
        e = np.exp(s)
        S = e.sum()
        log_q = s - np.log(S)
        q = e / S
        mass = p.sum() + rho
        loss = sum(target[v] * (np.log(target[v]) - log_q[v]) for v in np.unique(ids) if target[v] > 0)
        grad = mass * q - target
        # relative error of an e, and of the row's sum
        units = np.where(np.isfinite(s), -s, 0) / np.log(2)
        rel = (4 + 2.1 * units) * u
        rel_S = (400 + 2.1 * float((units * e).sum() / S)) * u
        drho = dp.sum()
        listed = target > 0
        d_loss = (dp[listed] * np.abs(np.log(target[listed]) - log_q[listed])).sum() + mass * rel_S + 8 * u * (
            target[listed] * (np.abs(np.log(target[listed])) + np.abs(s[listed]) + 1)).sum()
        d_grad = mass * q * (rel + rel_S + 8 * u) + dp + target * 4 * u
        if rest and rho != 0:
            s_off = np.where(on, -np.inf, x)
            m_off = s_off.max()
            if m_off == -np.inf:
                loss = np.inf
            else:
                s_off = (s_off - m_off) / T
                e_off = np.exp(s_off)
                S_off = e_off.sum()
                log_r = (m_off - m) / T + np.log(S_off) - np.log(S)
                loss += rho * (np.log(rho) - log_r)
                among = e_off / S_off
                grad -= rho * among
                off_units = np.where(np.isfinite(s_off), -s_off, 0) / np.log(2)
                rel_off = (404 + 2.1 * float((off_units * e_off).sum() / S_off) + 2.1 * off_units) * u
                # 1 - sum p: the sum's own error counts in full
                d_loss += drho * (abs(np.log(rho)) + 1 + abs(log_r)) + rho * (rel_S + 400 * u + 2.1 * u * float(
                    (off_units * e_off).sum() / S_off)) + 8 * u * rho * (abs(np.log(rho)) + abs(log_r) + 1)
                # the pass along the row multiplies e_off by a difference
                far = abs(m_off - m) / T / np.log(2)
                q_off = mass * np.where(on, 0, q)
                d_grad = np.where(on, d_grad, q_off * (rel_off + rel_S + (12 + 2.1 * far) * u)
                                  + rho * among * (rel_off + 8 * u) + drho * among)
                d_grad += q * drho
        scale = weight * T * T
        loss_out = scale * loss
        if abs(loss_out) >= 2.0 ** 128 * (1 - 2.0 ** -25):  # rounds to infinity in fp32
            loss_out = np.sign(loss_out) * np.inf
        d_out = abs(scale) * d_loss + 4 * u * abs(loss_out) if np.isfinite(loss_out) else 0.0
        g = weight * T
        return loss_out, g * grad, d_out, abs(g) * d_grad + 1e-37


def close(got, want, bound, half_step=2.0 ** -24):
    """got is within bound and half a step of its type of want, elementwise;
    infinities and NaN sit in the same places."""
    got, want, bound = (np.asarray(a, dtype=np.float64) for a in (got, want, bound))
    special = ~np.isfinite(want)
    same = np.where(np.isnan(want), np.isnan(got), got == want)
    with np.errstate(all="ignore"):
        near = np.abs(got - want) <= bound * (1 + 2 * half_step) + half_step * np.abs(want)
    return bool(np.all(np.where(special, same, near)))
