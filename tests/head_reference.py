"""Plain 64-bit forms of the model head's operators, on the CPU, and how far
a 32-bit computation of them may be off.

Error bounds: u = 2^-24 is the unit roundoff of 32-bit sums; a result that is
rounded to 16 bits is off by another half unit of its type.  A row's
log-sum-exp has terms 2^(x log2 e - c) whose exponent is rounded once
(|x - m| log2 e u, on terms that fall off as exp(-|x - m|)) and an exp2 good
to 1 ulp; partial sums are a tree over threads of at most a few hundred
sequential terms.  2^-19 covers their relative error; subtracting it from x
rounds twice more, relative to |x - m| and to the log-sum."""

import math

import numpy as np
import torch

U = 2.0 ** -24
HALF_UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
LSE = 2.0 ** -19


def rounding(y, dtype):
    """Half a unit of the type at y."""
    return y.abs() * HALF_UNIT[dtype] + TINY[dtype]


# --- adapter_logits ---------------------------------------------------------

def adapter_logits(x, weight, down, up, adapter, scale):
    """(logits, bound of a 32-bit computation's error)"""
    x, w, down, up, s = (t.double().cpu() for t in (x, weight, down, up, scale))
    y = x @ w.t()
    # n products summed in any order: n u times the sum of their magnitudes
    H = x.shape[1]
    err = (H + 2) * U * (x.abs() @ w.abs().t())
    for t, g in enumerate(adapter.tolist()):
        if g < 0:
            continue
        if g >= down.shape[0]:
            y[t] = math.nan
            continue
        z = s[g] * (down[g] @ x[t])
        zmag = s[g].abs() * (down[g].abs() @ x[t].abs())
        r = up.shape[2]
        y[t] += up[g] @ z
        # z: its own sum, and 22 bits kept of a row's largest
        zerr = (H + 4) * U * zmag + 2.0 ** -21 * (z.abs().max() if r else 0.0)
        err[t] += up[g].abs() @ (zerr + (3 * r + 4) * U * z.abs())
    return y, err


# --- propose ----------------------------------------------------------------

def propose(logits, topk):
    """(ids, logp, bound) of logits [batch, steps, vocab]."""
    x = logits.double().cpu().numpy()
    B, S, V = x.shape
    ids = np.empty((B, S, topk), np.int32)
    lp = np.empty((B, S, topk))
    tol = np.empty((B, S, topk))
    for b in range(B):
        for s in range(S):
            row = x[b, s]
            order = np.where(np.isnan(row), -np.inf, row)
            # (-0 sorts as 0)
            best = np.argsort(-(order + 0.0), kind="stable")[:topk]
            best.sort()
            ids[b, s] = best
            with np.errstate(all="ignore"):
                m = order.max()
                base = 0.0 if m == -np.inf else m
                ls = np.log(np.exp(row - base).sum())
                v = order[best]
                lp[b, s] = np.where((v == -np.inf) & ~np.isnan(ls), -np.inf, (v - base) - ls)
                tol[b, s] = LSE + 2 * U * (np.abs(v - base) + abs(ls))
    return ids, lp, tol


# --- losses -----------------------------------------------------------------

def scores(logits, tokens, lengths):
    """Token log-probabilities [R, C, S] (0 past a key's end), in 64 bits and
    differentiable by the logits."""
    R, S, V = logits.shape
    C = tokens.shape[1]
    ls = torch.log_softmax(logits, -1)
    lp = torch.zeros(R, C, S, dtype=torch.float64)
    rows = []
    for r in range(R):
        valid = torch.arange(S) < lengths[r][:, None]
        at = torch.where(valid, tokens[r].long(), torch.zeros((), dtype=torch.long))
        picked = ls[r][torch.arange(S).expand(C, S), at]
        rows.append(torch.where(valid, picked, torch.zeros_like(picked)))
    return torch.stack(rows) if R else lp


def policy(lp, lengths, old, adv, w, low, high, kl, ref):
    S = lp.shape[2]
    valid = torch.arange(S) < lengths[..., None]
    ratio = torch.exp(lp - old)
    a = adv[..., None]
    each = -torch.minimum(ratio * a, ratio.clamp(1 - low, 1 + high) * a)
    if kl:
        each = each + kl * (torch.expm1(ref - lp) - (ref - lp))
    return torch.where(valid, w[..., None] * each, torch.zeros_like(each)).sum()


def preference(lp, pairs, ref, w, beta, smoothing):
    margin = (lp.sum(-1) - ref).flatten()
    h = beta * (margin[pairs[:, 0].long()] - margin[pairs[:, 1].long()])
    ls = torch.nn.functional.logsigmoid
    return -(w * ((1 - smoothing) * ls(h) + smoothing * ls(-h))).sum()


def gradient_bound(logits, tokens, lengths, g, gerr):
    """Bound of a 32-bit gradient's error: g [R, C, S] the derivatives by the
    token scores, gerr their own error."""
    R, S, V = logits.shape
    C = tokens.shape[1]
    p = torch.softmax(logits, -1)
    valid = torch.arange(S) < lengths[..., None]
    mag = torch.where(valid, g.abs(), torch.zeros_like(g))
    ge = torch.where(valid, gerr, torch.zeros_like(g))
    # sums of up to C terms, a probability good to LSE and a few roundings
    total_err = (ge + (C + 4) * U * mag).sum(1)[..., None]
    err = p * (total_err + (2 * LSE) * mag.sum(1)[..., None])
    at = torch.where(valid, tokens.long(), torch.zeros((), dtype=torch.long)).transpose(1, 2)
    err.scatter_add_(2, at, (ge + (C + 4) * U * mag).transpose(1, 2))
    return err
