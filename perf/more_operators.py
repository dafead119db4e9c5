"""The operators of a generative retrieval model's vocabulary table, and what
is measured of them: training it on keys without keeping the logits, serving it
in 4 bits, and looking keys' tokens up in it, with the gradient.

  op "xent"        hidden states, table, targets -> loss, the targets' scores,
                   the gradients of both     flashtrie.cross_entropy_loss
  op "packed"      hidden states -> logits by a table of 4-bit weights
                                             flashtrie.packed_logits
  op "embed"       keys' tokens -> their rows of the table, scaled
                                             flashtrie.embed
  op "embed_grad"  the table's gradient from those rows'
                                             flashtrie.embed_grad

Sizes follow the search workloads: vocabularies of 32,768, 262,144 and 2.2M
tokens, 8, 12 or 16 output positions, batches of 1 to 8 requests, K of 10 to
1000.  Hidden states are N(0, 1), logits N(0, 2.5^2).
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIGMA = 2.5


def _ft():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "flash-trie_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flashtrie
    return flashtrie


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one key of one request, as an online update takes it: latency
        dict(name="xent_one_request", op="xent", rows=8, vocab=32768, hidden=512, dtype="bf16",
             smoothing=0.0, table=True),
        # a ragged step: odd numbers of rows and tokens, smoothed targets
        dict(name="xent_ragged", op="xent", rows=777, vocab=50021, hidden=768, dtype="f16",
             smoothing=0.1, table=True),
        # 96 keys of 12 tokens, the table frozen: gradient of the states alone
        dict(name="xent_frozen_table", op="xent", rows=1152, vocab=262144, hidden=1024,
             dtype="bf16", smoothing=0.0, table=False),
        # a training step over 256 keys of 16 tokens
        dict(name="xent_training", op="xent", rows=4096, vocab=262144, hidden=1024, dtype="bf16",
             smoothing=0.1, table=True),
        # one request of 8 positions on the smallest vocabulary: latency
        dict(name="packed_one_request", op="packed", rows=8, vocab=32768, hidden=512, group=32,
             dtype="bf16", out="f32"),
        # seven requests of 12 positions, odd vocabulary
        dict(name="packed_served_batch", op="packed", rows=84, vocab=100003, hidden=1024,
             group=128, dtype="f16", out="f16"),
        # one request of 16 positions on the largest vocabulary
        dict(name="packed_large_vocab", op="packed", rows=16, vocab=2200000, hidden=512, group=64,
             dtype="bf16", out="f32"),
        # ten keys of one request: latency
        dict(name="embed_one_request", op="embed", batch=1, keys=10, steps=8, vocab=32768,
             hidden=512, dtype="f32"),
        # the keys of a batch of beam-1000 searches
        dict(name="embed_beam", op="embed", batch=8, keys=1000, steps=16, vocab=2200000,
             hidden=512, dtype="bf16"),
        # ten keys of one request: latency
        dict(name="embed_grad_one_request", op="embed_grad", batch=1, keys=10, steps=8,
             vocab=32768, hidden=512, dtype="f32"),
        # 128 keys of 13 tokens, odd vocabulary
        dict(name="embed_grad_own_keys", op="embed_grad", batch=128, keys=1, steps=13,
             vocab=100003, hidden=768, dtype="f16"),
        # the keys of a batch of beam-1000 searches: many share their first tokens
        dict(name="embed_grad_beam", op="embed_grad", batch=8, keys=1000, steps=16, vocab=262144,
             hidden=1024, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xent", "packed", "embed", "embed_grad"])
    hidden = 64 * rng.randint(4, 32)
    if op == "xent":  # up to the training step's products
        vocab = _log_uniform(rng, 8192, 2 ** 28 // hidden)
        return dict(op=op, rows=_log_uniform(rng, 1, min(4096, 2 ** 40 // (vocab * hidden))),
                    vocab=vocab, hidden=hidden, dtype=rng.choice(["bf16", "bf16", "f16"]),
                    smoothing=rng.choice([0.0, 0.1]), table=rng.random() < 0.7)
    if op == "packed":  # up to the largest vocabulary's products
        vocab = _log_uniform(rng, 8192, 2200000 * 512 // hidden)
        return dict(op=op, rows=_log_uniform(rng, 1, min(128, 2200000 * 512 * 16 // (vocab * hidden))),
                    vocab=vocab, hidden=hidden, group=rng.choice([32, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]), out=rng.choice(["f32", "same"]))
    dtype = rng.choice(["bf16", "f16", "f32"])
    size = DTYPES[dtype].itemsize
    vocab = _log_uniform(rng, 8192, (2200000 * 512 if op == "embed" else 262144 * 1024) * 2 // (hidden * size))
    steps = rng.randint(1, 16)
    most = (128000 * 512 if op == "embed" else 128000 * 1024) * 2 // (hidden * size * steps)
    if rng.random() < 0.5:
        return dict(op=op, batch=_log_uniform(rng, 1, min(512, most)), keys=1, steps=steps,
                    vocab=vocab, hidden=hidden, dtype=dtype)
    batch = rng.randint(1, 8)
    return dict(op=op, batch=batch, keys=_log_uniform(rng, 2, min(1000, most // batch)),
                steps=steps, vocab=vocab, hidden=hidden, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, dtype, scale, g):
    """N(0, scale^2) of the type, in pieces (the largest is 1.1e9 numbers)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        n = min(1 << 28, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device="cuda", generator=g) * scale
    return out


def _out_dtype(case):
    return DTYPES[case["dtype"] if case["out"] == "same" else case["out"]]


def _prepare_xent(case, g):
    """States that lean to their targets by 0 to 16 of a logit; every 16th row
    or so is padding.  float16 gradients are made at a loss scale."""
    T, V, H, d = case["rows"], case["vocab"], case["hidden"], DTYPES[case["dtype"]]
    weight = _normal((V, H), d, SIGMA / math.sqrt(H), g)
    targets = (torch.rand(T, device="cuda", generator=g) ** 2 * V).long().clamp(max=V - 1)
    lean = torch.rand((T, 1), device="cuda", generator=g) * (16.0 / SIGMA ** 2)
    x = torch.randn((T, H), device="cuda", generator=g) + lean * weight[targets].float()
    padding = torch.rand(T, device="cuda", generator=g) < (1 / 16 if T > 1 else 0.0)
    targets = torch.where(padding, -torch.ones_like(targets), targets)
    scale = 2.0 ** 16 if case["dtype"] == "f16" else 1.0
    w = torch.rand(T, device="cuda", generator=g) + 0.5
    return dict(x=x.to(d), weight=weight, targets=targets.to(torch.int32),
                row_weight=w * (scale / max(1, int((~padding).sum()))),
                smoothing=case["smoothing"], table=case["table"])


def _prepare_packed(case, g):
    """Codes of normal weights and their groups' scales, laid out as
    packed_logits takes them: tiles of 16 tokens by 128 columns, each lane
    16 q + n of 64 holding token n's columns 32 i + 8 q + j, word i, in nibble
    (j >> 1) + 4 (j & 1)."""
    V, H, d = case["vocab"], case["hidden"], DTYPES[case["dtype"]]
    tiles, chunks = (V + 15) // 16, (H + 127) // 128
    packed = torch.empty((tiles, chunks, 64, 16), dtype=torch.uint8, device="cuda")
    for t in range(0, tiles, 1 << 15):
        n = min(1 << 15, tiles - t)
        # tile, token n, chunk, word i, quarter q, column j = 2 low + high
        c = torch.randn((n, 16, chunks, 4, 4, 4, 2), device="cuda", generator=g)
        c = (c * 2.9).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        # tile, chunk, q, n, i, nibble = low + 4 high
        c = c.permute(0, 2, 4, 1, 3, 6, 5).reshape(n, chunks, 64, 16, 2)
        packed[t:t + n] = c[..., 0] | c[..., 1] << 4
    scales = (torch.rand((tiles, chunks, 16, 128 // case["group"]), device="cuda", generator=g) + 0.5)
    scales *= SIGMA / math.sqrt(H) / 2.9
    # of either sign, as the scale of a group whose largest weight is positive is negative
    scales *= 1 - 2 * torch.randint(2, scales.shape, device="cuda", generator=g)
    x = torch.randn((case["rows"], H), device="cuda", generator=g)
    return dict(x=x.to(d), packed=packed, scales=scales.to(d), vocab=V, out_dtype=_out_dtype(case))


def _prepare_tokens(case, g):
    """Keys as a search under a trie returns them: few tokens at the first
    position, more at later ones; lengths from 3 up (some slots without a
    key), tokens past a key's end 0."""
    R, C, S, V = case["batch"], case["keys"], case["steps"], case["vocab"]
    kinds = _kinds(case).to("cuda")
    which = (torch.rand((R, C, S), device="cuda", generator=g) ** 2 * kinds).long()
    # (an odd multiplier spreads the ranks over the vocabulary)
    tokens = (which * 40503 + torch.randint(V, (R, 1, S), device="cuda", generator=g)) % V
    lengths = torch.randint(min(3, S), S + 1, (R, C), device="cuda", generator=g)
    lengths[torch.rand((R, C), device="cuda", generator=g) < 0.03] = 0
    valid = torch.arange(S, device="cuda") < lengths[..., None]
    tokens = torch.where(valid, tokens, torch.zeros_like(tokens))
    return tokens.to(torch.int32), lengths.to(torch.int32)


def _kinds(case):
    return (8.0 * 4.0 ** torch.arange(case["steps"])).clamp(max=case["vocab"])


def _prepare_embed(case, g):
    tokens, lengths = _prepare_tokens(case, g)
    return dict(tokens=tokens, lengths=lengths, scale=math.sqrt(case["hidden"]),
                table=_normal((case["vocab"], case["hidden"]), DTYPES[case["dtype"]],
                              1.0 / math.sqrt(case["hidden"]), g))


def _prepare_embed_grad(case, g):
    tokens, lengths = _prepare_tokens(case, g)
    return dict(tokens=tokens, lengths=lengths, vocab=case["vocab"], scale=math.sqrt(case["hidden"]),
                grad=_normal((*tokens.shape, case["hidden"]), DTYPES[case["dtype"]], 1.0, g))


def prepare(case, seed):
    state = {"xent": _prepare_xent, "packed": _prepare_packed, "embed": _prepare_embed,
             "embed_grad": _prepare_embed_grad}[case["op"]](case, _gen(seed))
    return dict(state, op=case["op"])


# ---------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_xent(s):
    x, w, eps = s["x"].float(), s["weight"].float(), s["smoothing"]
    V = w.shape[0]
    l = x @ w.t()
    counts = s["targets"] >= 0
    at = s["targets"].long().clamp(min=0)[:, None]
    m = l.amax(1, keepdim=True)
    lse = m + (l - m).exp().sum(1, keepdim=True).log()
    picked = l.gather(1, at) - lse
    rw = torch.where(counts, s["row_weight"], 0.0)[:, None]
    loss = -(rw * ((1.0 - eps) * picked + eps * (l.mean(1, keepdim=True) - lse))).sum()
    logp = torch.where(counts[:, None], picked, 0.0)[:, 0]
    g = (l - lse).exp() - eps / V
    g.scatter_add_(1, at, torch.full_like(picked, eps - 1.0))
    g *= rw
    dx = (g @ w).to(s["x"].dtype)
    if not s["table"]:
        return loss, logp, dx
    return loss, logp, dx, (g.t() @ x).to(s["weight"].dtype)


def _codes(packed):
    """[tokens, columns] codes less 8, of every tile's 16 tokens."""
    tiles, chunks = packed.shape[:2]
    c = torch.stack((packed & 15, packed >> 4), -1)
    c = c.view(tiles, chunks, 4, 16, 4, 2, 4).permute(0, 3, 1, 4, 2, 6, 5)
    return c.reshape(tiles * 16, chunks * 128).to(torch.int8) - 8


def _plain_packed(s):
    x, scales = s["x"].float(), s["scales"].float()
    tiles, chunks, _, per = scales.shape
    c = _codes(s["packed"]).float().view(tiles * 16, chunks * per, 128 // per)
    w = c * scales.transpose(1, 2).reshape(tiles * 16, chunks * per, 1)
    w = w.view(tiles * 16, -1)[:s["vocab"], :x.shape[1]]
    return (x @ w.t()).to(s["out_dtype"])


def _valid(s):
    steps = torch.arange(s["tokens"].shape[2], device="cuda")
    return (steps < s["lengths"][..., None]) & (s["tokens"] >= 0)


def _plain_embed(s):
    y = s["table"][s["tokens"].clamp(min=0)].float() * s["scale"]
    return torch.where(_valid(s)[..., None], y, 0.0).to(s["table"].dtype)


def _plain_embed_grad(s):
    g = torch.where(_valid(s)[..., None], s["grad"].float(), 0.0)
    out = torch.zeros((s["vocab"], g.shape[-1]), device="cuda")
    out.index_add_(0, s["tokens"].clamp(min=0).view(-1), g.view(-1, g.shape[-1]))
    return (out * s["scale"]).to(s["grad"].dtype)


def run(state):
    s = state
    if not own:
        return {"xent": _plain_xent, "packed": _plain_packed, "embed": _plain_embed,
                "embed_grad": _plain_embed_grad}[s["op"]](s)
    ft = _ft()
    if s["op"] == "xent":
        out = ft.cross_entropy_loss(s["x"], s["weight"], s["targets"], s["row_weight"],
                                    smoothing=s["smoothing"], weight_grad=s["table"])
        return out if s["table"] else out[:3]
    if s["op"] == "packed":
        return ft.packed_logits(s["x"], s["packed"], s["scales"], s["vocab"],
                                out_dtype=s["out_dtype"])
    if s["op"] == "embed":
        return ft.embed(s["tokens"], s["table"], scale=s["scale"], lengths=s["lengths"])
    return ft.embed_grad(s["grad"], s["tokens"], s["vocab"], scale=s["scale"], lengths=s["lengths"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    V, H, size = case["vocab"], case["hidden"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "xent":  # states and table read, their gradients written
        T, tables = case["rows"], 2 if case["table"] else 1
        return {"bytes": size * (2 * T * H + tables * V * H) + 12 * T,
                "flops": 2 * T * V * H * (1 + tables) + 4 * T * V}
    if case["op"] == "packed":
        T = case["rows"]
        return {"bytes": V * H // 2 + size * (V * H // case["group"] + T * H)
                + _out_dtype(case).itemsize * T * V, "flops": 2 * T * V * H}
    R, C, S = case["batch"], case["keys"], case["steps"]
    n, small = R * C * S, 4 * R * C * (S + 1)
    if case["op"] == "embed":  # different tokens of a request's position: at most its kinds
        rows = R * int(_kinds(case).clamp(max=C).sum())
        return {"bytes": small + size * H * (n + min(rows, V)), "flops": n * H}
    return {"bytes": small + size * H * (n + V), "flops": n * H}


# ---------------------------------------------------------------------------
# 64 bits, from the definitions; gradients by differentiation
# ---------------------------------------------------------------------------

def _exact_xent(s):
    x, w, eps = s["x"].double(), s["weight"].double(), s["smoothing"]
    T, logp = len(x), torch.zeros(len(x), dtype=torch.float64, device="cuda")
    dx, dw, loss = torch.zeros_like(x), torch.zeros_like(w) if s["table"] else None, 0.0
    for i in range(0, T, 256):  # some rows at a time
        rows = i + (s["targets"][i:i + 256] >= 0).nonzero()[:, 0]
        if len(rows) == 0:
            continue
        xr, wr = x[rows].requires_grad_(), w.detach().requires_grad_(s["table"])
        l = torch.log_softmax(xr @ wr.t(), -1)
        picked = l[torch.arange(len(rows), device="cuda"), s["targets"][rows].long()]
        each = -((1 - eps) * picked + eps * l.mean(-1)) if eps else -picked
        part = (s["row_weight"][rows].double() * each).sum()
        grads = torch.autograd.grad(part, [xr, wr] if s["table"] else [xr])
        loss, dx[rows], logp[rows] = loss + part.detach(), grads[0], picked.detach()
        if s["table"]:
            dw += grads[1]
    loss = torch.as_tensor(loss, dtype=torch.float64, device="cuda")
    return (loss, logp, dx, dw) if s["table"] else (loss, logp, dx)


def _exact_packed(s):
    """Word by word and nibble by nibble, a part of the tokens at a time."""
    x, V = s["x"].double(), s["vocab"]
    T, H = x.shape
    tiles, chunks, _, per = s["scales"].shape
    x = torch.cat((x, x.new_zeros((T, chunks * 128 - H))), 1)
    out = torch.empty((T, tiles * 16), dtype=torch.float64, device="cuda")
    j = torch.arange(8, device="cuda")
    shift = 4 * ((j >> 1) + 4 * (j & 1))
    for t in range(0, tiles, 1 << 13):
        words = s["packed"][t:t + (1 << 13)].contiguous().view(torch.int32)
        n = len(words)
        w = torch.empty((n, 16, chunks, 4, 4, 8), dtype=torch.float64, device="cuda")
        for q in range(4):
            part = words[:, :, 16 * q:16 * q + 16]  # tile, chunk, token, word
            w[:, :, :, :, q] = ((part[..., None] >> shift & 15) - 8).transpose(1, 2).double()
        w = w.view(n, 16, chunks, per, 128 // per)
        w = w * s["scales"][t:t + n].double().transpose(1, 2)[..., None]
        out[:, t * 16:(t + n) * 16] = x @ w.reshape(n * 16, -1).t()
    return out[:, :V].contiguous()


def _exact_embed(s):
    steps = torch.arange(s["tokens"].shape[2], device="cuda")
    out = torch.zeros((*s["tokens"].shape, s["table"].shape[1]), dtype=torch.float64, device="cuda")
    there = steps.expand(s["tokens"].shape) < s["lengths"][..., None]
    out[there] = s["table"][s["tokens"][there].long()].double() * s["scale"]
    return out


def _exact_embed_grad(s):
    steps = torch.arange(s["tokens"].shape[2], device="cuda")
    there = steps.expand(s["tokens"].shape) < s["lengths"][..., None]
    table = torch.zeros((s["vocab"], s["grad"].shape[-1]), dtype=torch.float64, device="cuda",
                        requires_grad=True)
    looked_up = table[s["tokens"][there].long()] * s["scale"]
    return torch.autograd.grad(looked_up, table, s["grad"][there].double())[0]


def exact(case, seed):
    s = prepare(case, seed)
    return {"xent": _exact_xent, "packed": _exact_packed, "embed": _exact_embed,
            "embed_grad": _exact_embed_grad}[case["op"]](s)
