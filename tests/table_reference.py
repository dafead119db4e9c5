"""Plain 64-bit forms of the vocabulary table's operators, and how far a
32-bit computation of them may be off.

u = 2^-24 is the unit roundoff of 32-bit sums: n products summed in any order
are off by at most n u times the sum of their magnitudes.  A result that is
rounded to 16 bits is off by another half unit of its type, relative to it; so
are the logits' slopes that the gradients' products take."""

import torch

from head_reference import HALF_UNIT, LSE, TINY, U, rounding  # noqa: F401


def cross_entropy(x, weight, targets, row_weight, smoothing):
    """{name: (value, bound)} of loss, logp, dx, dweight; NaN where the
    definition has none."""
    dtype = x.dtype
    y, r = targets.long(), row_weight.double()
    V, H = weight.shape
    counts = y >= 0
    used = counts & (r != 0)
    xd = torch.where(counts[:, None], x.double(), 0.0)
    w = weight.double()
    l = xd @ w.t()
    le = (H + 2) * U * (xd.abs() @ w.abs().t())
    lse = torch.logsumexp(l, 1, keepdim=True)
    there = counts & (y < V)
    at = torch.where(there, y, torch.zeros_like(y))[:, None]
    picked = torch.where(there[:, None], l.gather(1, at), torch.nan)
    top = l.amax(1, keepdim=True)
    # of the log-sum-exp: the logits' own errors, its terms' and its sum's, and
    # the subtractions of the maximum and of the log-sum
    lsee = le.amax(1, keepdim=True) + LSE + 4 * U * ((picked - top).abs() + (lse - top).abs())
    logp = picked - lse
    logpe = le.gather(1, at) + lsee + U * logp.abs()
    s = smoothing
    mean = l.mean(1, keepdim=True)
    # (a sum of V logits: a lane's few, then tiles in turn, at most 1000 after one another)
    meane = le.mean(1, keepdim=True) + 1000 * U * l.abs().mean(1, keepdim=True)
    each = -(1 - s) * logp + s * (lse - mean)
    eache = (1 - s) * logpe + s * (meane + lsee) + 8 * U * (logp.abs() + lse.abs() + mean.abs())
    rr = torch.where(used, r, 0.0)[:, None]
    terms = torch.where(used[:, None], rr * each, 0.0)
    T = len(y)
    loss = (terms.sum(), (torch.where(used[:, None], rr.abs() * eache, 0.0).sum()
                          + (T + 4) * U * terms.abs().sum()))
    # slopes
    p = torch.exp(l - lse)
    ge = p * (le + lsee + 4 * U * ((l - top).abs() + 1)) + 4 * U * (p + s / V)
    own = torch.zeros_like(p).scatter_(1, at, (1 - s) * there.double()[:, None])
    ge += 4 * U * own
    g = p - own - s / V
    g = torch.where(there[:, None], g, torch.nan)
    # rounded to the type, relative to itself; what lies below float16's range,
    # stored times 2^14 or more, by its least number
    ge = ge + g.abs() * HALF_UNIT[dtype] + TINY[dtype] / (2.0 ** 14 if dtype == torch.float16 else 1.0)
    g, ge = torch.where(used[:, None], g, 0.0), torch.where(used[:, None], ge, 0.0)
    wa, xa = w.abs(), torch.where(used[:, None], xd, 0.0).abs()
    dx = rr * (g @ w)
    dxe = rr.abs() * ((ge @ wa) + (V + 64) * U * (g.abs() @ wa))
    rg = rr * g
    dw = rg.t() @ torch.where(used[:, None], xd, 0.0)
    dwe = (rr.abs() * ge).t() @ xa + (T + 8) * U * (rg.abs().t() @ xa)
    # rows of x are scaled to the largest weight's, by a factor near a power of two
    # that makes the target's slope one of the type's numbers: a state is rounded
    # once more, relative to itself, in the products of its row
    dwe = dwe + HALF_UNIT[dtype] * (rg.abs().t() @ xa)
    if T:
        dwe = dwe + 2 * rr.abs().max() * TINY[dtype] * (g.abs() + ge).sum(0)[:, None]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    logp = torch.where(counts[:, None], logp, zero)[:, 0]
    return dict(loss=loss, logp=(logp, torch.where(counts[:, None], logpe, zero)[:, 0]),
                dx=(dx, dxe + rounding(dx, dtype)), dweight=(dw, dwe + rounding(dw, dtype)))


def pack(weight, group):
    """(codes less 8 [V, H], scales [V, ceil(H / 128) * 128 / group]) in plain
    steps of 32 bits; columns past H are zeros."""
    V, H = weight.shape
    width = (H + 127) // 128 * 128
    w = torch.zeros((V, width), dtype=torch.float32, device=weight.device)
    w[:, :H] = weight.float()
    w = w.view(V, width // group, group)
    odd = ~torch.isfinite(w).all(-1, keepdim=True)
    mag = w.abs()
    first = (mag == mag.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
    scale = (w.gather(-1, first) * -0.125).to(weight.dtype)
    scale = torch.where(odd, torch.nan, scale)
    s = scale.float()
    codes = (w / s).round().clamp(-8, 7)
    codes = torch.where(odd | (s == 0), 0.0, codes)
    return codes.view(V, width)[:, :H].to(torch.int8), scale[..., 0]


def lay_out(codes, scales, group):
    """Codes less 8 and scales as packed_logits takes them, an element at a
    time."""
    V, H = codes.shape
    tiles, chunks = (V + 15) // 16, (H + 127) // 128
    packed = torch.full((tiles, chunks, 64, 4, 8), 8, dtype=torch.int64)
    c = codes.cpu().long() + 8
    v, h = torch.meshgrid(torch.arange(V), torch.arange(H), indexing="ij")
    k = h % 128
    i, q, j = k // 32, k % 32 // 8, k % 8
    packed[v // 16, h // 128, 16 * q + v % 16, i, (j >> 1) + 4 * (j & 1)] = c
    bytes_ = packed[..., ::2] | packed[..., 1::2] << 4
    per = 128 // group
    out = torch.zeros((tiles, chunks, 16, per), dtype=scales.dtype)
    s = scales.cpu()
    v, g = torch.meshgrid(torch.arange(V), torch.arange(chunks * per), indexing="ij")
    out[v // 16, g // per, v % 16, g % per] = s
    return bytes_.to(torch.uint8).reshape(tiles, chunks, 64, 16), out


def packed_logits(x, codes, scales, group):
    """(logits, bound) of codes less 8 [V, H] and scales [V, groups]."""
    V, H = codes.shape
    s = scales.double().repeat_interleave(group, 1)[:, :H]
    w = codes.double() * s
    xd = x.double()
    y = xd @ w.t()
    wa = w.abs()
    err = (H + H // group + 4) * U * (xd.abs() @ wa.t())
    if x.dtype == torch.bfloat16:  # x in float16 over its row's power of two
        big = torch.where(xd.isfinite(), xd, 0.0).abs().amax(1, keepdim=True)
        err = err + big * 2.0 ** -38 * wa.sum(1)
    return y, err


def embed(tokens, table, scale, lengths):
    """Exactly: one 32-bit product, rounded to the type."""
    V = table.shape[0]
    there = valid(tokens, lengths)
    t = torch.where(there, tokens, 0).long()
    y = (table[t.clamp(max=V - 1)].float() * torch.tensor(scale, dtype=torch.float32)).to(table.dtype)
    y = torch.where((t < V)[..., None], y, torch.nan)
    return torch.where(there[..., None], y, 0.0).to(table.dtype)


def valid(tokens, lengths, vocab=None):
    there = tokens >= 0
    if vocab is not None:
        there &= tokens < vocab
    if lengths is not None:
        there &= torch.arange(tokens.shape[-1], device=tokens.device) < lengths[..., None]
    return there


def embed_grad(grad, tokens, vocab, scale, lengths, out=None):
    """(dtable, bound)."""
    there = valid(tokens, lengths, vocab)
    t, g = tokens[there].long(), grad[there].double()
    scale = float(torch.tensor(scale, dtype=torch.float32))
    sums = torch.zeros((vocab, grad.shape[-1]), dtype=torch.float64, device=grad.device)
    mags, n = sums.clone(), torch.zeros(vocab, dtype=torch.float64, device=grad.device)
    sums.index_add_(0, t, g)
    mags.index_add_(0, t, g.abs())
    n.index_add_(0, t, torch.ones_like(t, dtype=torch.float64))
    y = scale * sums
    err = abs(scale) * (n + 2)[:, None] * U * mags
    if out is not None:
        y = y + out.double()
        err = err + 2 * U * y.abs()
    err = err + rounding(y, grad.dtype)
    # rows of other tokens: as they were
    return y, torch.where((n > 0)[:, None], err, 0.0)
