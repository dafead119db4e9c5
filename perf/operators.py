"""The operators of a generative retrieval model's head, and what is measured
of them: the vocabulary projection with the adapters of many requests, the
proposals that the trie search takes, and the two losses that train the
model on the keys the search returned.

  op "logits"      hidden states -> logits, each row with its request's
                   low-rank adapter            flashtrie.adapter_logits
  op "propose"     logits -> the K best tokens of each row by ascending id,
                   with log-softmax scores     flashtrie.propose
  op "policy"      clipped policy loss with a KL term over the returned keys,
                   and the logits' gradient    flashtrie.policy_loss
  op "preference"  loss on pairs of returned keys, and the logits' gradient
                                               flashtrie.preference_loss

Sizes follow the search workloads: vocabularies of 32,768, 262,144 and 2.2M
tokens, 8, 12 or 16 output positions, batches of 1 to 8 requests, beams and
K of 10 to 1000.  A row is one (request, position).  Logits are N(0, 2.5^2),
as the workloads' proposals are.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.2, 0.05
BETA, SMOOTHING = 0.1, 0.1
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
        # one request of 8 positions on the smallest vocabulary: latency
        dict(name="logits_one_request", op="logits", requests=1, steps=8, vocab=32768,
             hidden=512, adapters=4, rank=8, dtype="bf16", out="f32", mixed=False),
        # a served batch, one adapter a request, ragged: rows in no order of
        # their adapters, some without one, rank no power of two
        dict(name="logits_served_batch", op="logits", requests=7, steps=12, vocab=262144,
             hidden=1024, adapters=6, rank=12, dtype="bf16", out="bf16", mixed=True),
        # one request of 16 positions on the largest vocabulary
        dict(name="logits_large_vocab", op="logits", requests=1, steps=16, vocab=2200000,
             hidden=512, adapters=2, rank=16, dtype="bf16", out="f32", mixed=False),
        # a training pass over many requests' positions
        dict(name="logits_training", op="logits", requests=256, steps=16, vocab=32768,
             hidden=1024, adapters=16, rank=64, dtype="f16", out="f16", mixed=False),
        # proposals of one request at the smallest beam: latency
        dict(name="propose_one_request", op="propose", requests=1, steps=8, vocab=32768, topk=32,
             dtype="f32", masked=0.0),
        # odd sizes, rows that start at no aligned address, tokens masked
        dict(name="propose_odd", op="propose", requests=3, steps=13, vocab=100003, topk=333,
             dtype="f16", masked=0.4),
        # batch 8 of the 800M-key workload
        dict(name="propose_large_vocab", op="propose", requests=8, steps=16, vocab=2200000,
             topk=1000, dtype="bf16", masked=0.0),
        # ten keys of one request: latency
        dict(name="policy_one_request", op="policy", requests=1, steps=8, vocab=32768, keys=10,
             dtype="f32"),
        # the keys of a batch of beam-1000 searches: a thousand share each row
        dict(name="policy_beam", op="policy", requests=8, steps=16, vocab=262144, keys=1000,
             dtype="bf16"),
        # every key with rows of its own, as a model that reads its own output
        # is trained
        dict(name="policy_own_rows", op="policy", requests=128, steps=16, vocab=32768, keys=1,
             dtype="bf16"),
        # pairs of keys of the same request
        dict(name="preference_beam", op="preference", requests=8, steps=12, vocab=262144, keys=100,
             pairs=400, dtype="bf16"),
        # pairs of keys with rows of their own, odd vocabulary
        dict(name="preference_own_rows", op="preference", requests=64, steps=12, vocab=50021,
             keys=1, pairs=32, dtype="f16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logits", "propose", "policy", "preference"])
    steps = rng.randint(1, 16)
    if op == "logits":
        # weights of 2**21 .. 2**30 bytes; rows such that products stay
        # below the training pass's
        hidden = 64 * rng.randint(4, 32)
        vocab = _log_uniform(rng, 8192, 2200000 * 512 // hidden)
        most = max(1, min(256, 2 ** 37 // (vocab * hidden) // steps))
        requests = _log_uniform(rng, 1, most)
        return dict(op=op, requests=requests, steps=steps, vocab=vocab, hidden=hidden,
                    adapters=rng.randint(1, 8), rank=rng.choice([4, 8, 11, 16, 24, 32, 64])
                    if vocab < 300000 else rng.choice([4, 8, 11, 16]),
                    dtype=rng.choice(["bf16", "bf16", "f16"]), out=rng.choice(["f32", "same"]),
                    mixed=rng.random() < 0.5)
    if op == "propose":
        vocab = _log_uniform(rng, 8192, 2200000)
        requests = rng.randint(1, 8)
        return dict(op=op, requests=requests, steps=steps, vocab=vocab,
                    topk=_log_uniform(rng, 10, 1000), dtype=rng.choice(["bf16", "f16", "f32"])
                    if vocab < 1000000 else rng.choice(["bf16", "f16"]),
                    masked=rng.choice([0.0, 0.0, 0.5]))
    vocab = _log_uniform(rng, 8192, 262144)
    dtype = rng.choice(["bf16", "f16", "f32"]) if vocab < 100000 else rng.choice(["bf16", "f16"])
    own_rows = rng.random() < 0.5
    most = max(2, 2 ** 25 // (vocab * steps))
    if op == "policy":
        return dict(op=op, requests=_log_uniform(rng, 1, min(128, most)) if own_rows
                    else rng.randint(1, min(8, most)), steps=steps, vocab=vocab,
                    keys=1 if own_rows else _log_uniform(rng, 2, 1000), dtype=dtype)
    if own_rows:
        pairs = _log_uniform(rng, 1, min(64, most // 2))
        return dict(op=op, requests=2 * pairs, steps=steps, vocab=vocab, keys=1, pairs=pairs,
                    dtype=dtype)
    keys = _log_uniform(rng, 2, 1000)
    requests = rng.randint(1, min(8, most))
    return dict(op=op, requests=requests, steps=steps, vocab=vocab, keys=keys,
                pairs=requests * rng.randint(1, 4 * keys), dtype=dtype)


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


def _row_adapters(case, g):
    """Each request's adapter: the adapters in turn, every 7th request with
    none; the rows in request order, or in no order."""
    req = torch.arange(case["requests"], device="cuda")
    ad = torch.where(req % 7 == 6, torch.full_like(req, -1), req % case["adapters"])
    rows = ad.repeat_interleave(case["steps"]).to(torch.int32)
    if case["mixed"]:
        rows = rows[torch.randperm(rows.numel(), device="cuda", generator=g)]
    return rows.contiguous()


def _used_adapters(case):
    return len({r % case["adapters"] for r in range(case["requests"]) if r % 7 != 6})


def _prepare_logits(case, g):
    d, T, V, H = DTYPES[case["dtype"]], case["requests"] * case["steps"], case["vocab"], case["hidden"]
    G, r = case["adapters"], case["rank"]
    return dict(x=_normal((T, H), d, 1.0, g), weight=_normal((V, H), d, SIGMA / math.sqrt(H), g),
                down=_normal((G, r, H), d, 1.0 / math.sqrt(H), g),
                up=_normal((G, V, r), d, 0.5 / math.sqrt(r), g),
                adapter=_row_adapters(case, g),
                scale=torch.rand(G, device="cuda", generator=g) * 1.5 + 0.5,
                out_dtype=_out_dtype(case))


def _prepare_propose(case, g):
    R, V = case["requests"] * case["steps"], case["vocab"]
    x = _normal((R, V), DTYPES[case["dtype"]], SIGMA, g)
    if case["masked"] > 0:  # tokens of no key
        x.masked_fill_(torch.rand(V, device="cuda", generator=g) < case["masked"], -math.inf)
    return dict(logits=x.view(case["requests"], case["steps"], V), topk=case["topk"])


def _row_lse(x):
    """log-sum-exp of each row in 64 bits, a row at a time."""
    return torch.stack([torch.logsumexp(r.double(), 0) for r in x.view(-1, x.shape[-1])]
                       ).view(x.shape[:-1])


def _prepare_keys(case, g):
    """Logits, and keys as a search under a trie returns them: few tokens at
    the first position, more at later ones; lengths from 3 up (some slots
    without a key), tokens past a key's end 0."""
    R, S, V, C = case["requests"], case["steps"], case["vocab"], case["keys"]
    x = _normal((R, S, V), DTYPES[case["dtype"]], SIGMA, g)
    kinds = (8.0 * 4.0 ** torch.arange(S, device="cuda")).clamp(max=V).view(1, 1, S)
    which = (torch.rand((R, C, S), device="cuda", generator=g) ** 2 * kinds).long()
    # (an odd multiplier spreads the ranks over the vocabulary)
    tokens = (which * 40503 + torch.randint(V, (R, 1, S), device="cuda", generator=g)) % V
    lengths = torch.randint(min(3, S), S + 1, (R, C), device="cuda", generator=g)
    lengths[torch.rand((R, C), device="cuda", generator=g) < 0.03] = 0
    valid = torch.arange(S, device="cuda") < lengths[..., None]
    tokens = torch.where(valid, tokens, torch.zeros_like(tokens))
    lp = torch.gather(x, 2, tokens.transpose(1, 2)).transpose(1, 2).double()
    lp = torch.where(valid, lp - _row_lse(x)[:, None, :], torch.zeros_like(lp))
    return x, tokens.to(torch.int32), lengths.to(torch.int32), lp, valid


def _noise(shape, scale, g):
    """A model's drift since the keys were scored.  A ratio at a clip's very
    edge has no derivative: none is drawn within 2e-3 of one."""
    d = torch.randn(shape, device="cuda", generator=g) * scale
    for edge in (math.log(1.0 - CLIP_LOW), math.log(1.0 + CLIP_HIGH)):
        d = torch.where((d - edge).abs() < 2e-3, d + 4e-3, d)
    return d


def _prepare_policy(case, g):
    x, tokens, lengths, lp, valid = _prepare_keys(case, g)
    total = max(1, int(lengths.sum()))
    return dict(logits=x, tokens=tokens, lengths=lengths,
                old_logp=torch.where(valid, lp - _noise(lp.shape, 0.15, g), lp).float(),
                ref_logp=torch.where(valid, lp + _noise(lp.shape, 0.3, g), lp).float(),
                advantage=torch.randn(lengths.shape, device="cuda", generator=g),
                weight=torch.full(lengths.shape, 1.0 / total, device="cuda"))


def _prepare_preference(case, g):
    x, tokens, lengths, lp, valid = _prepare_keys(case, g)
    R, C, P = case["requests"], case["keys"], case["pairs"]
    if C == 1:
        pairs = torch.arange(2 * P, device="cuda").view(P, 2)
    else:  # a better and a worse key of the same request
        req = torch.arange(P, device="cuda") % R
        a = torch.randint(C, (P,), device="cuda", generator=g)
        b = (a + torch.randint(1, C, (P,), device="cuda", generator=g)) % C
        pairs = torch.stack([req * C + a, req * C + b], 1)
    ref = lp.sum(-1) + torch.randn((R, C), device="cuda", generator=g)
    return dict(logits=x, tokens=tokens, lengths=lengths, pairs=pairs.to(torch.int32).contiguous(),
                ref_logp=ref.float(), weight=torch.full((P,), 1.0 / P, device="cuda"))


def prepare(case, seed):
    state = {"logits": _prepare_logits, "propose": _prepare_propose, "policy": _prepare_policy,
             "preference": _prepare_preference}[case["op"]](case, _gen(seed))
    return dict(state, op=case["op"])


# ---------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_logits(s):
    x, down, up = s["x"].float(), s["down"].float(), s["up"].float()
    G, r, H = down.shape
    z = (x @ down.reshape(G * r, H).t()).view(-1, G, r)
    hit = s["adapter"][:, None] == torch.arange(G, device=x.device)
    z = z * (hit * s["scale"])[..., None]
    y = x @ s["weight"].float().t()
    y += z.view(-1, G * r) @ up.transpose(1, 2).reshape(G * r, -1)
    return y.to(s["out_dtype"])


def _plain_propose(s):
    x, k = s["logits"].float(), s["topk"]
    m = x.amax(-1, keepdim=True)
    lse = m + (x - m).exp().sum(-1, keepdim=True).log()
    least = x.topk(k).values[..., -1:]
    tie = x == least
    keep = x > least
    # ties: the lowest ids
    keep |= tie & (tie.cumsum(-1) <= k - keep.sum(-1, keepdim=True))
    ids = keep.nonzero()[:, -1].view(*x.shape[:-1], k)
    return ids.to(torch.int32), x.gather(-1, ids) - lse


def _plain_rows(s):
    """Token log-probabilities [R, S, C], the rows' probabilities, and which
    tokens are there."""
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    at = s["tokens"].transpose(1, 2).long()
    steps = torch.arange(x.shape[1], device=x.device)
    valid = steps[:, None] < s["lengths"][:, None, :]
    lp = torch.where(valid, x.gather(2, at) - (m + z.log()), 0.0)
    return lp, e / z, at, valid


def _plain_gradient(s, p, at, g):
    d = -p * g.sum(-1, keepdim=True)
    return d.scatter_add_(2, at, g).to(s["logits"].dtype)


def _plain_policy(s):
    lp, p, at, valid = _plain_rows(s)
    old, ref = s["old_logp"].transpose(1, 2), s["ref_logp"].transpose(1, 2)
    adv, w = s["advantage"][:, None, :], s["weight"][:, None, :]
    ratio = (lp - old).exp()
    clipped = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
    d = ref - lp
    each = -torch.minimum(ratio * adv, clipped * adv) + KL * (d.exp() - d - 1.0)
    loss = torch.where(valid, each * w, 0.0).sum()
    moves = ratio * adv <= clipped * adv
    g = w * (KL * (1.0 - d.exp()) - torch.where(moves, ratio * adv, 0.0))
    g = torch.where(valid, g, 0.0)
    return loss, lp.transpose(1, 2).contiguous(), _plain_gradient(s, p, at, g)


def _plain_preference(s):
    lp, p, at, valid = _plain_rows(s)
    margin = (lp.sum(1) - s["ref_logp"]).reshape(-1)
    a, b = s["pairs"].long().unbind(1)
    h = BETA * (margin[a] - margin[b])
    # softplus(-h) and softplus(h)
    tail = (1.0 + (-h.abs()).exp()).log()
    won, lost = tail - h.clamp(max=0.0), tail + h.clamp(min=0.0)
    loss = (s["weight"] * ((1.0 - SMOOTHING) * won + SMOOTHING * lost)).sum()
    gp = s["weight"] * BETA * (1.0 / (1.0 + (-h).exp()) - (1.0 - SMOOTHING))
    gm = torch.zeros_like(margin).index_add_(0, a, gp).index_add_(0, b, -gp)
    g = torch.where(valid, gm.view(s["ref_logp"].shape)[:, None, :], 0.0)
    return loss, lp.transpose(1, 2).contiguous(), _plain_gradient(s, p, at, g)


def run(state):
    s = state
    if not own:
        return {"logits": _plain_logits, "propose": _plain_propose, "policy": _plain_policy,
                "preference": _plain_preference}[s["op"]](s)
    ft = _ft()
    if s["op"] == "logits":
        return ft.adapter_logits(s["x"], s["weight"], s["down"], s["up"], s["adapter"], s["scale"],
                                 out_dtype=s["out_dtype"])
    if s["op"] == "propose":
        return ft.propose(s["logits"], s["topk"])
    if s["op"] == "policy":
        return ft.policy_loss(s["logits"], s["tokens"], s["lengths"], s["old_logp"],
                              s["advantage"], s["weight"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                              kl_coef=KL, ref_logp=s["ref_logp"])
    return ft.preference_loss(s["logits"], s["tokens"], s["lengths"], s["pairs"], s["ref_logp"],
                              s["weight"], beta=BETA, smoothing=SMOOTHING)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    R, S, V = case["requests"], case["steps"], case["vocab"]
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "logits":
        T, H, r, n = R * S, case["hidden"], case["rank"], _used_adapters(case)
        served = S * sum(q % 7 != 6 for q in range(R))  # rows with an adapter
        return {"bytes": size * (T * H + V * H + n * r * (H + V)) + _out_dtype(case).itemsize * T * V
                + 4 * T, "flops": 2 * T * V * H + 2 * served * r * (H + V)}
    n = R * S * V
    if case["op"] == "propose":
        return {"bytes": size * n + 8 * R * S * case["topk"], "flops": 4 * n}
    C = case["keys"]
    if case["op"] == "policy":  # tokens, old and reference scores in, scores out
        return {"bytes": 2 * size * n + 16 * R * C * S + 12 * R * C, "flops": 7 * n}
    return {"bytes": 2 * size * n + 8 * R * C * S + 8 * R * C + 12 * case["pairs"], "flops": 7 * n}


# ---------------------------------------------------------------------------
# 64 bits, from the definitions; gradients by differentiation
# ---------------------------------------------------------------------------

def _exact_logits(s):
    x = s["x"].double()
    T, V = x.shape[0], s["weight"].shape[0]
    y = torch.empty((T, V), dtype=torch.float64, device="cuda")
    for v in range(0, V, 1 << 17):
        y[:, v:v + (1 << 17)] = x @ s["weight"][v:v + (1 << 17)].double().t()
    for g in range(s["down"].shape[0]):
        rows = (s["adapter"] == g).nonzero()[:, 0]
        if len(rows):
            z = (x[rows] @ s["down"][g].double().t()) * s["scale"][g].double()
            y[rows] += z @ s["up"][g].double().t()
    return y


def _exact_propose(s):
    x = s["logits"].reshape(-1, s["logits"].shape[-1])
    k, ids, lps = s["topk"], [], []
    for row in x:
        first = torch.sort(row.double(), descending=True, stable=True)[1][:k]
        i = first.sort()[0]
        ids.append(i.to(torch.int32))
        lps.append(torch.log_softmax(row.double(), 0)[i])
    shape = (*s["logits"].shape[:-1], k)
    return torch.stack(ids).view(shape), torch.stack(lps).view(shape)


def _exact_loss(s, loss_of):
    """loss_of(token log-probabilities [R, C, S]) -> loss; the logits'
    gradient through a row's log-softmax, a request at a time."""
    R, S, V = s["logits"].shape
    valid = torch.arange(S, device="cuda") < s["lengths"][..., None]
    at = s["tokens"].long()
    lp = torch.stack([torch.log_softmax(s["logits"][r].double(), -1)
                      [torch.arange(S, device="cuda"), at[r]] for r in range(R)])
    lp = torch.where(valid, lp, torch.zeros_like(lp)).requires_grad_()
    loss = loss_of(lp, valid)
    g, = torch.autograd.grad(loss, lp)
    g = torch.where(valid, g, torch.zeros_like(g))
    d = torch.empty((R, S, V), dtype=torch.float64, device="cuda")
    for r in range(R):
        x = s["logits"][r].double().requires_grad_()
        picked = torch.log_softmax(x, -1)[torch.arange(S, device="cuda"), at[r]]
        d[r], = torch.autograd.grad(picked, x, g[r])
    return loss.detach(), lp.detach(), d


def _exact_policy(s):
    old, ref = s["old_logp"].double(), s["ref_logp"].double()
    adv, w = s["advantage"].double()[..., None], s["weight"].double()[..., None]

    def loss_of(lp, valid):
        ratio = torch.exp(lp - old)
        gain = torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
        kl = torch.expm1(ref - lp) - (ref - lp)
        return torch.where(valid, w * (KL * kl - gain), 0.0).sum()

    return _exact_loss(s, loss_of)


def _exact_preference(s):
    a, b = s["pairs"].long().unbind(1)

    def loss_of(lp, valid):
        margin = (lp.sum(-1) - s["ref_logp"].double()).flatten()
        h = BETA * (margin[a] - margin[b])
        logsig = torch.nn.functional.logsigmoid
        return -(s["weight"].double() * ((1 - SMOOTHING) * logsig(h) + SMOOTHING * logsig(-h))).sum()

    return _exact_loss(s, loss_of)


def exact(case, seed):
    s = prepare(case, seed)
    return {"logits": _exact_logits, "propose": _exact_propose, "policy": _exact_policy,
            "preference": _exact_preference}[case["op"]](s)
