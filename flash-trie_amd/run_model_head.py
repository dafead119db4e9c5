#!/usr/bin/env python3
"""A model's head around the trie search: from hidden states to keys, and from
the keys back to the gradient of the head's adapters.

Each round of a small training run on seeded data

1. projects the hidden states of every request and step to the vocabulary,
   each request through its own low-rank adapter (``adapter_logits``);
2. takes the ``--topk-tokens`` best tokens of each row with their
   log-probabilities (``propose``);
3. searches them under the trie (``bs_tbs_gpu``): the keys, with scores;
4. rewards a key by the share of the wanted key's tokens that it has in
   place, and turns the rewards of a request's keys into advantages;
5. weighs the keys by the clipped policy loss with its KL term
   (``policy_loss``), or pairs the best-rewarded key with each other one
   (``preference_loss``), both on the logits that scored them;
6. carries the gradient of the logits to the adapters (plain matrix products)
   and steps them.

With ``--pretrain N`` the head's table is first trained on the wanted keys
themselves, N supervised steps: a step's hidden state is the request's plus the
table's row of the token before it (``embed``), the loss and the gradients of
states and table come without logits (``cross_entropy_loss``), and the lookup's
gradient is added to the table's (``embed_grad``).  With ``--packed GROUP`` a
last search takes its logits from the table in 4 bits (``pack_weight``,
``packed_logits``).

It prints a line per round: the loss, the mean reward of the returned keys,
and of the key that the search ranks first.  Nothing of it is a trained
model: hidden states lean towards a wanted key by ``--signal``.

Example::

    python run_model_head.py --requests 16 --loss preference --rounds 8
"""

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from ft_harness import import_flashtrie  # noqa: E402
from make_example_data import make_keys  # noqa: E402


def parse_args(argv=None):
    p = argparse.ArgumentParser(description=__doc__,
                                formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--num-keys", type=int, default=20000)
    p.add_argument("--key-length", type=int, default=6, help="maximum tokens per key")
    p.add_argument("--vocab-size", type=int, default=8192)
    p.add_argument("--hidden", type=int, default=512)
    p.add_argument("--adapters", type=int, default=3)
    p.add_argument("--rank", type=int, default=16)
    p.add_argument("--dtype", choices=("bfloat16", "float16"), default="bfloat16")
    p.add_argument("--topk-tokens", type=int, default=64)
    p.add_argument("--beam-size", type=int, default=64)
    p.add_argument("--loss", choices=("policy", "preference"), default="policy")
    p.add_argument("--rounds", type=int, default=6, help="searches")
    p.add_argument("--updates", type=int, default=2, help="updates on one search's keys")
    p.add_argument("--lr", type=float, default=2e-3)
    p.add_argument("--kl-coef", type=float, default=0.01)
    p.add_argument("--beta", type=float, default=0.1)
    p.add_argument("--signal", type=float, default=0.35,
                   help="how far the hidden states lean to the wanted key")
    p.add_argument("--pretrain", type=int, default=0, help="supervised steps on the wanted keys")
    p.add_argument("--table-lr", type=float, default=0.5)
    p.add_argument("--packed", type=int, default=0, choices=(0, 32, 64, 128),
                   help="columns to a scale of the table in 4 bits (0: no such search)")
    p.add_argument("--seed", type=int, default=0)
    args = p.parse_args(argv)
    if args.pretrain < 0:
        p.error("--pretrain must be at least 0")
    for name in ("requests", "num_keys", "key_length", "hidden", "adapters", "rank",
                 "topk_tokens", "beam_size", "rounds", "updates"):
        if getattr(args, name) < 1:
            p.error(f"--{name.replace('_', '-')} must be at least 1")
    if args.topk_tokens > args.vocab_size:
        p.error("--topk-tokens must be at most --vocab-size")
    return args


class Head:
    """A shared projection with low-rank adapters, some rows for each."""

    def __init__(self, args, torch, ft):
        g = torch.Generator("cuda").manual_seed(args.seed)
        self.torch, self.ft = torch, ft
        self.dtype = getattr(torch, args.dtype)
        V, H, G, r = args.vocab_size, args.hidden, args.adapters, args.rank

        def normal(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.weight = (normal(V, H) * H ** -0.5).to(self.dtype)
        # the adapters that are trained, in 32 bits; up = 0: no change yet
        self.down = (normal(G, r, H) * H ** -0.5).requires_grad_()
        self.up = torch.zeros(G, V, r, device="cuda", requires_grad=True)
        self.scale = torch.full((G,), 2.0, device="cuda")
        self.optimizer = torch.optim.Adam([self.down, self.up], lr=args.lr)
        self.noise = normal

    def logits(self, x, adapter):
        """float32 logits [rows, vocab] of the adapters as they are now."""
        return self.ft.adapter_logits(
            x, self.weight, self.down.detach().to(self.dtype), self.up.detach().to(self.dtype),
            adapter, self.scale, self.torch.float32)

    def step(self, x, adapter, dlogits):
        """Moves the adapters along the gradient of the logits' loss:
        d up = s dlogits' z, dz = s dlogits up, d down = dz' x, z = down x,
        summed over an adapter's rows."""
        torch = self.torch
        self.down.grad, self.up.grad = torch.zeros_like(self.down), torch.zeros_like(self.up)
        x = x.float()
        with torch.no_grad():
            for g in range(self.down.shape[0]):
                rows = adapter == g
                xs, d = x[rows], dlogits[rows] * self.scale[g]
                self.up.grad[g] = d.t() @ (xs @ self.down[g].t())
                self.down.grad[g] = (d @ self.up[g]).t() @ xs
        self.optimizer.step()


def before(tokens):
    """The tokens one step earlier, -1 (none) in front of a key."""
    out = tokens.roll(1, -1)
    out[..., 0] = -1
    return out.contiguous()


def supervised(ft, x, table, tokens, lengths, scale):
    """(loss, table's gradient) of keys [R, C, S] whose states are x [R, C, S,
    hidden] plus scale times the table's row of the token before; a key's tokens
    share its weight, the keys theirs."""
    R, C, S = tokens.shape
    inputs = before(tokens)
    states = x + ft.embed(inputs, table, scale, lengths)
    there = tokens.new_tensor(range(S)) < lengths[..., None]
    targets = tokens.masked_fill(~there, -1).view(-1)
    share = 1.0 / (lengths.clamp(min=1) * max(1, int((lengths > 0).sum())))
    weight = share.float()[..., None].expand(R, C, S).reshape(-1)
    loss, _, dx, dtable = ft.cross_entropy_loss(states.view(R * C * S, -1), table, targets, weight)
    ft.embed_grad(dx.view(R, C, S, -1), inputs, table.shape[0], scale, lengths, out=dtable)
    return loss, dtable


def pretrain(head, x, wanted, args, log):
    """Steps of plain gradient descent on the table, held in 32 bits."""
    torch, (tok, length) = head.torch, key_arrays([[k] for k in wanted], args.key_length)
    tok, length = torch.from_numpy(tok).cuda(), torch.from_numpy(length).cuda()
    table, losses = head.weight.float(), []
    for n in range(args.pretrain):
        loss, d = supervised(head.ft, x.view(*tok.shape, -1), head.weight, tok, length, 1.0)
        table -= args.table_lr * d.float()
        head.weight = table.to(head.dtype)
        losses.append(loss.item())
        log(f"pretrain {n}: loss {losses[-1]:.5f}")
    return losses


def key_arrays(sents, steps):
    """The search's keys as (tokens [R, C, steps], lengths [R, C]) int32; a
    request with fewer keys than another has keys of no tokens."""
    C = max(1, max(len(s) for s in sents))
    tokens = np.zeros((len(sents), C, steps), dtype=np.int32)
    lengths = np.zeros((len(sents), C), dtype=np.int32)
    for r, keys in enumerate(sents):
        for c, key in enumerate(keys):
            tokens[r, c, :len(key)] = key
            lengths[r, c] = len(key)
    return tokens, lengths


def rewards(tokens, lengths, wanted):
    """Share of the wanted key's tokens in place, over the longer of the two."""
    out = np.zeros(lengths.shape, dtype=np.float32)
    for r, want in enumerate(wanted):
        n = len(want)
        same = (tokens[r, :, :n] == np.asarray(want)) & (np.arange(n) < lengths[r, :, None])
        out[r] = same.sum(1) / np.maximum(lengths[r], n)
    return out


def run(args, log=print):
    """The rounds' lines as dicts."""
    import torch
    ft = import_flashtrie()
    rng = np.random.default_rng(args.seed)
    keys, tokens, offsets = make_keys(rng, args.num_keys, args.key_length, args.vocab_size,
                                      [1.0] * args.key_length)
    trie = ft.Trie()
    trie.build_arrays(tokens, offsets)
    R, S, C = args.requests, args.key_length, args.beam_size
    trie.init_tbs_gpu(R, args.topk_tokens, max_num_outpos=S, max_num_out_beams=C,
                      max_num_out_tokens=C * S, max_num_inter_beams=C * S)

    head = Head(args, torch, ft)
    wanted = [keys[i] for i in rng.integers(0, len(keys), size=R)]
    x = head.noise(R, S, args.hidden)
    for r, want in enumerate(wanted):
        x[r, :len(want)] += args.signal * args.hidden ** 0.5 * head.weight[list(want)].float()
    x = x.reshape(R * S, -1).to(head.dtype)
    adapter = (torch.arange(R, device="cuda", dtype=torch.int32) % args.adapters)
    adapter = adapter.repeat_interleave(S).contiguous()
    base = torch.full_like(adapter, -1)   # the head without its adapters

    def search(logits):
        ids, logp = ft.propose(logits.view(R, S, -1), args.topk_tokens)
        return ft.bs_tbs_gpu(trie, R, [[C] * S] * R, list(ids.cpu().numpy()),
                             list(logp.cpu().numpy()), -1e9, -1e9, 5.0, False)

    lines = []
    if args.pretrain:
        lines.append({"pretrain": pretrain(head, x, wanted, args, log)})
    for n in range(args.rounds):
        logits = head.logits(x, adapter).view(R, S, -1)
        sents, _, search_ms, _ = search(logits)
        tok, length = key_arrays(sents, S)
        reward = rewards(tok, length, wanted)
        found = length > 0
        count = np.maximum(found.sum(1, keepdims=True), 1)
        advantage = np.where(found, reward - (reward * found).sum(1, keepdims=True) / count, 0)
        tok, length = torch.from_numpy(tok).cuda(), torch.from_numpy(length).cuda()
        zeros = torch.zeros(tok.shape, device="cuda")
        adv = torch.from_numpy(advantage.astype(np.float32)).cuda()
        weight = torch.from_numpy((found / count / R).astype(np.float32)).cuda()
        # the tokens' log-probabilities before the updates, and under the base
        _, old, _ = ft.policy_loss(logits, tok, length, zeros, adv, weight, grad=False)
        _, ref, _ = ft.policy_loss(head.logits(x, base).view(R, S, -1), tok, length, zeros, adv,
                                   weight, grad=False)
        pairs, pair_weight = [], []
        for r in range(R):
            a = int(np.argmax(np.where(found[r], reward[r], -1)))
            others = [c for c in range(found.shape[1]) if found[r, c] and reward[r, c] < reward[r, a]]
            pairs += [(r * found.shape[1] + a, r * found.shape[1] + c) for c in others]
            pair_weight += [1 / max(len(others), 1) / R] * len(others)
        pairs = torch.tensor(pairs, dtype=torch.int32).reshape(-1, 2).cuda()
        pair_weight = torch.tensor(pair_weight, dtype=torch.float32).cuda()

        losses = []
        for _ in range(args.updates):
            logits = head.logits(x, adapter).view(R, S, -1)
            if args.loss == "policy":
                loss, _, d = ft.policy_loss(logits, tok, length, old, adv, weight,
                                            kl_coef=args.kl_coef, ref_logp=ref)
            else:
                loss, _, d = ft.preference_loss(logits, tok, length, pairs, ref.sum(2),
                                                pair_weight, beta=args.beta)
            head.step(x, adapter, d.view(R * S, -1))
            losses.append(loss.item())
        line = {"round": n, "losses": losses, "keys": int(found.sum()),
                "mean_reward": float((reward * found).sum() / max(found.sum(), 1)),
                "first_reward": float(reward[:, 0].mean()), "search_ms": search_ms}
        lines.append(line)
        log(f"round {n}: {args.loss} loss {losses[0]:+.5f} -> {losses[-1]:+.5f}  "
            f"keys {line['keys']}  reward: mean {line['mean_reward']:.3f}, "
            f"first {line['first_reward']:.3f}  search {search_ms:.3f} ms")
    if args.packed:
        packed = ft.packed_logits(x, *ft.pack_weight(head.weight, args.packed), args.vocab_size,
                                  torch.float32)
        sents = [search(y)[0] for y in (head.logits(x, base), packed)]
        same = [len({tuple(k) for k in a} & {tuple(k) for k in b}) / max(len(a), 1)
                for a, b in zip(*sents)]
        lines.append({"packed": sum(same) / R, "keys": sum(map(len, sents[1]))})
        log(f"table in 4 bits: {100 * lines[-1]['packed']:.1f}% of the table's own keys")
    return lines


def main(argv=None):
    run(parse_args(argv))
    return 0


if __name__ == "__main__":
    sys.exit(main())
