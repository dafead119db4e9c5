"""flashtrie.policy_loss and flashtrie.preference_loss against plain forms in
64 bits: the loss, the tokens' scores and the logits' gradient (by
differentiating the plain form, and by differences of its loss), within the
bounds of head_reference.py."""

import math

import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = [F32, F16, BF16]


def keys(R, S, V, C, dtype, seed, distinct=None, full=False):
    """Logits and keys; `distinct` tokens a row (few: many keys share one)."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((R, S, V), generator=g) * 2.5).to(dtype)
    tokens = torch.randint(0, min(V, distinct or V), (R, C, S), generator=g)
    tokens = (tokens * 7919 + seed) % V
    lengths = torch.full((R, C), S) if full else torch.randint(0, S + 1, (R, C), generator=g)
    return x, tokens.to(torch.int32), lengths.to(torch.int32), g


def policy_case(R, S, V, C, dtype, seed, **kw):
    x, tokens, lengths, g = keys(R, S, V, C, dtype, seed, **kw)
    lp = ref.scores(x.double(), tokens, lengths)
    d = torch.randn(lp.shape, generator=g) * 0.2
    for edge in (math.log(0.8), math.log(1.3)):  # no derivative there
        d = torch.where((d - edge).abs() < 2e-3, d + 5e-3, d)
    return dict(logits=x, tokens=tokens, lengths=lengths, old_logp=(lp - d).float(),
                ref_logp=(lp + torch.randn(lp.shape, generator=g) * 0.3).float(),
                advantage=torch.randn((R, C), generator=g),
                weight=torch.rand((R, C), generator=g) / max(1, R * C * S))


def check_policy(ft, a, kl=0.05, what=""):
    R, S, V = a["logits"].shape
    C = a["tokens"].shape[1]
    print(what, R, S, V, C, a["logits"].dtype, flush=True)
    gpu = {k: v.cuda() for k, v in a.items()}
    loss, logp, d = ft.policy_loss(**gpu, clip_low=0.2, clip_high=0.3, kl_coef=kl)
    x = a["logits"].double().requires_grad_()
    lp = ref.scores(x, a["tokens"], a["lengths"])
    lp.retain_grad()
    old, rf, adv, w = (a[k].double() for k in ("old_logp", "ref_logp", "advantage", "weight"))
    want = ref.policy(lp, a["lengths"], old, adv, w, 0.2, 0.3, kl, rf)
    want.backward()
    lpd = lp.detach()
    lperr = ref.LSE + 4 * ref.U * (lpd.abs() + 30)
    assert ((logp.double().cpu() - lpd).abs() <= lperr).all(), what
    valid = torch.arange(S) < a["lengths"][..., None]
    assert (logp.cpu()[~valid] == 0).all()
    # a score off by e moves the ratio and exp(ref - lp) by a factor 1 + e
    # and adds e to the KL term; the formulas round a few times more
    ratio, tilt = (lpd - old).exp(), (rf - lpd).exp()
    size = w[..., None].abs() * (adv[..., None].abs() * ratio + kl * (1 + tilt + (rf - lpd).abs()))
    gerr = torch.where(valid, size * (lperr + 16 * ref.U), torch.zeros(()).double())
    terms = torch.where(valid, size, torch.zeros(()).double()).sum()
    tol = gerr.sum() + (R * S * C + 8) * ref.U * terms
    assert abs(loss.item() - want.item()) <= tol, (what, loss.item(), want.item(), tol)
    g = lp.grad
    bound = ref.gradient_bound(a["logits"].double(), a["tokens"], a["lengths"], g, gerr)
    check_gradient(d, x.grad, bound, what)
    return loss, logp, d


def check_gradient(d, want, bound, what):
    got = d.double().cpu()
    tol = bound + ref.rounding(want, d.dtype)
    bad = (got - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), ((got - want).abs() / tol).max())


def preference_case(R, S, V, C, P, dtype, seed, **kw):
    x, tokens, lengths, g = keys(R, S, V, C, dtype, seed, **kw)
    lp = ref.scores(x.double(), tokens, lengths).sum(-1)
    pairs = torch.randint(0, R * C, (P, 2), generator=g)
    return dict(logits=x, tokens=tokens, lengths=lengths, pairs=pairs.to(torch.int32),
                ref_logp=(lp + torch.randn(lp.shape, generator=g) * 3).float(),
                weight=torch.rand(P, generator=g) / max(1, P))


def check_preference(ft, a, beta=0.1, smoothing=0.1, what=""):
    R, S, V = a["logits"].shape
    C, P = a["tokens"].shape[1], a["pairs"].shape[0]
    print(what, R, S, V, C, P, a["logits"].dtype, flush=True)
    gpu = {k: v.cuda() for k, v in a.items()}
    loss, logp, d = ft.preference_loss(**gpu, beta=beta, smoothing=smoothing)
    x = a["logits"].double().requires_grad_()
    lp = ref.scores(x, a["tokens"], a["lengths"])
    lp.retain_grad()
    rf, w = a["ref_logp"].double(), a["weight"].double()
    want = ref.preference(lp, a["pairs"], rf, w, beta, smoothing)
    if P:
        want.backward()
    else:
        x.grad, lp.grad = torch.zeros_like(x), torch.zeros_like(lp)
    lpd = lp.detach()
    lperr = ref.LSE + 4 * ref.U * (lpd.abs() + 30)
    assert ((logp.double().cpu() - lpd).abs() <= lperr).all(), what
    # a margin is off by its scores' errors and the sum's roundings; a
    # sigmoid's slope is at most 1/4
    merr = (lperr.sum(-1) + (S + 2) * ref.U * (lpd.abs().sum(-1) + rf.abs())).flatten()
    pa, pb = a["pairs"].long().unbind(1)
    herr = abs(beta) * (merr[pa] + merr[pb])
    h = beta * ((lpd.sum(-1) - rf).flatten()[pa] - (lpd.sum(-1) - rf).flatten()[pb])
    herr = herr + 4 * ref.U * h.abs()
    tol = (w * (herr + (P + 8) * ref.U * (1 + h.abs()))).sum()
    assert abs(loss.item() - want.item()) <= tol, (what, loss.item(), want.item(), tol)
    per = w * abs(beta) * (herr + 16 * ref.U)
    mag = w * abs(beta)
    kerr = torch.zeros(R * C).double().index_add_(0, pa, per + (P + 4) * ref.U * mag)
    kerr.index_add_(0, pb, per + (P + 4) * ref.U * mag)
    gerr = kerr.view(R, C, 1).expand(R, C, S)
    bound = ref.gradient_bound(a["logits"].double(), a["tokens"], a["lengths"], lp.grad, gerr)
    check_gradient(d, x.grad, bound, what)
    return loss, logp, d


# vectors and spans of the vocabulary, keys across a wave, a workgroup and
# several pairs a thread
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,S,V,C", [(1, 1, 1, 1), (1, 1, 2, 3), (2, 3, 7, 2), (3, 2, 100, 1),
                                     (2, 5, 1001, 63), (2, 3, 8192, 64), (1, 4, 8193, 65),
                                     (2, 2, 33333, 130), (1, 2, 4096, 1024), (1, 2, 5000, 1025),
                                     (1, 1, 20001, 4096), (40, 3, 2050, 1), (2, 17, 300, 5)])
def test_sizes(ft, dtype, R, S, V, C):
    check_policy(ft, policy_case(R, S, V, C, dtype, V + C), what="policy")
    check_preference(ft, preference_case(R, S, V, C, 3 * R * C + 1, dtype, V + C), what="preference")


# all keys of one token, of a few: runs across waves and workgroup turns
@pytest.mark.parametrize("distinct", [1, 2, 5, 70])
@pytest.mark.parametrize("C", [2, 64, 200, 1000, 3000])
def test_shared_tokens(ft, distinct, C):
    check_policy(ft, policy_case(1, 2, 5003, C, F32, distinct, distinct=distinct, full=True),
                 what="policy")
    check_preference(ft, preference_case(1, 2, 5003, C, 500, F32, distinct, distinct=distinct,
                                         full=True), what="preference")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_vocabulary(ft, dtype):
    check_policy(ft, policy_case(1, 2, 2_200_001, 100, dtype, 1), what="policy")
    check_preference(ft, preference_case(2, 2, 262145, 30, 64, dtype, 1), what="preference")


def test_without_kl(ft):
    a = policy_case(2, 4, 501, 6, F32, 2)
    check_policy(ft, a, kl=0.0)
    gpu = {k: v.cuda() for k, v in a.items()}
    ref_logp = gpu.pop("ref_logp")
    x = ft.policy_loss(**gpu)
    y = ft.policy_loss(**gpu, kl_coef=0.0, ref_logp=ref_logp * math.nan)
    assert all(torch.equal(p, q) for p, q in zip(x, y))


@pytest.mark.parametrize("C", [1, 7])
def test_lengths(ft, C):
    """No token at all, one, all of them; out of range: none, all."""
    a = policy_case(6, 4, 300, C, F32, 3, full=True)
    for i, n in enumerate([0, 1, 4, 3, -5, 900]):
        a["lengths"][i] = n
    stop = a["lengths"].clamp(0, 4)
    tokens = a["tokens"].clone()
    for r in range(6):  # past the end: anything
        a["tokens"][r, :, int(stop[r, 0]):] = -1 if r % 2 else 2 ** 31 - 1
    gpu = {k: v.cuda() for k, v in a.items()}
    got = ft.policy_loss(**gpu, kl_coef=0.1)
    want = ft.policy_loss(**{**gpu, "tokens": tokens.cuda(), "lengths": stop.to(torch.int32).cuda()},
                          kl_coef=0.1)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert (got[2][0] == 0).all() and (got[2][4] == 0).all() and (got[2][1, 1:] == 0).all()
    assert (got[1][0] == 0).all() and got[2][2].abs().sum() > 0
    a["lengths"][:] = 0
    loss, logp, d = ft.policy_loss(**{k: v.cuda() for k, v in a.items()}, kl_coef=0.1)
    assert loss == 0 and (logp == 0).all() and (d == 0).all()


def test_unused_rows_are_not_read(ft):
    """NaN and infinities in rows that score no token stay out."""
    for C in (1, 5):
        a = policy_case(2, 4, 900, C, F32, 4, full=True)
        a["lengths"][:] = 2
        want = check_policy(ft, a)
        a["logits"][:, 2] = math.nan
        a["logits"][:, 3] = math.inf
        got = ft.policy_loss(**{k: v.cuda() for k, v in a.items()}, clip_low=0.2, clip_high=0.3,
                             kl_coef=0.05)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_masked_logits(ft):
    """Logits of -infinity and of the type's lowest value beside the tokens."""
    for dtype in DTYPES:
        a = policy_case(2, 3, 700, 4, dtype, 5, distinct=20)
        used = torch.zeros(700, dtype=torch.bool)
        used[a["tokens"].long().flatten()] = True
        a["logits"][..., ~used] = torch.finfo(dtype).min
        lp = ref.scores(a["logits"].double(), a["tokens"], a["lengths"]).float()
        a["old_logp"], a["ref_logp"] = lp + 0.1, lp - 0.2
        check_policy(ft, a, what="lowest")
        a["logits"][..., ~used] = -math.inf
        _, _, d = check_policy(ft, a, what="-inf")
        assert (d[..., (~used).cuda()] == 0).all()


def test_a_masked_token(ft):
    """A token whose own logit is -infinity: its ratio is 0, its KL term
    infinite."""
    a = policy_case(1, 2, 50, 3, F32, 6, full=True)
    a["tokens"][0, :, 0] = torch.tensor([3, 4, 5], dtype=torch.int32)
    a["logits"][0, 0, 3] = -math.inf
    a["old_logp"][0, 0, 0] = -1.0
    gpu = {k: v.cuda() for k, v in a.items()}
    loss, logp, d = ft.policy_loss(**gpu, kl_coef=0.0)
    assert logp[0, 0, 0] == -math.inf and loss.isfinite() and d.isfinite().all()
    loss, _, d = ft.policy_loss(**gpu, kl_coef=0.1)
    assert loss == math.inf and not d[0, 0].isfinite().all() and d[0, 1].isfinite().all()


@pytest.mark.parametrize("C", [1, 6])
@pytest.mark.parametrize("bad", [-1, 200, 2 ** 31 - 1])
def test_tokens_out_of_range(ft, C, bad):
    """Shown as NaN in the key's score and the row's gradient, nowhere else."""
    a = policy_case(2, 3, 200, C, F32, 7, full=True)
    a["tokens"][1, 0, 2] = bad
    loss, logp, d = ft.policy_loss(**{k: v.cuda() for k, v in a.items()}, kl_coef=0.1)
    nan = torch.zeros(2, C, 3, dtype=torch.bool)
    nan[1, 0, 2] = True
    assert loss.isnan() and torch.equal(logp.isnan().cpu(), nan)
    assert d[1, 2].isnan().all() and not d[0].isnan().any() and not d[1, :2].isnan().any()


def test_pairs_out_of_range(ft):
    a = preference_case(3, 2, 100, 2, 4, F32, 8, full=True)
    a["pairs"] = torch.tensor([[0, 1], [6, 2], [-1, 3], [4, 5]], dtype=torch.int32)
    loss, logp, d = ft.preference_loss(**{k: v.cuda() for k, v in a.items()})
    assert loss.isnan() and not logp.isnan().any()
    assert d[1].isnan().all() and not d[0].isnan().any() and not d[2].isnan().any()


@pytest.mark.parametrize("P", [0, 1, 63, 64, 65, 1023, 1025, 5000])
def test_pairs(ft, P):
    check_preference(ft, preference_case(5, 3, 300, 30, P, F32, P, full=True), what="pairs")


def test_pairs_of_one_key(ft):
    """One key in every pair, and pairs of a key with itself."""
    a = preference_case(1, 2, 64, 70, 300, F32, 9, full=True)
    a["pairs"][:, 0] = 5
    a["pairs"][::3, 1] = 5
    check_preference(ft, a)


def test_large_margins(ft):
    for beta in (50.0, -3.0):
        a = preference_case(2, 3, 300, 4, 40, F32, 10, full=True)
        check_preference(ft, a, beta=beta, smoothing=0.0, what="margins")


def test_preference_smoothing_ends(ft):
    for s in (0.0, 0.5, 1.0):
        check_preference(ft, preference_case(2, 3, 100, 4, 9, F32, 11, full=True), smoothing=s)


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_against_differences(ft, which):
    """The gradient along directions against differences of the 64-bit loss."""
    step = 1e-4
    if which == "policy":
        a = policy_case(2, 3, 120, 5, F32, 12, full=True)
        d = ft.policy_loss(**{k: v.cuda() for k, v in a.items()}, clip_low=0.2, clip_high=0.3,
                           kl_coef=0.05)[2].double().cpu()

        def loss(x):
            return ref.policy(ref.scores(x, a["tokens"], a["lengths"]), a["lengths"],
                              a["old_logp"].double(), a["advantage"].double(), a["weight"].double(),
                              0.2, 0.3, 0.05, a["ref_logp"].double())
    else:
        a = preference_case(2, 3, 120, 5, 20, F32, 12, full=True)
        d = ft.preference_loss(**{k: v.cuda() for k, v in a.items()}, beta=0.7,
                               smoothing=0.1)[2].double().cpu()

        def loss(x):
            return ref.preference(ref.scores(x, a["tokens"], a["lengths"]), a["pairs"],
                                  a["ref_logp"].double(), a["weight"].double(), 0.7, 0.1)

    g = torch.Generator().manual_seed(13)
    x = a["logits"].double()
    for _ in range(8):
        v = torch.randn(x.shape, generator=g).double()
        slope = (loss(x + step * v) - loss(x - step * v)) / (2 * step)
        # step^2 times the third derivative along v (of order |v's change of
        # a score|^3, up to 4^3), and 32-bit sums of the gradient
        tol = 64 * step ** 2 + 1e-5 * (d.abs() * v.abs()).sum()
        assert abs((d * v).sum() - slope) <= tol


def test_strides(ft):
    a = policy_case(3, 4, 211, 5, F16, 14)
    gpu = {k: v.cuda() for k, v in a.items()}
    want = ft.policy_loss(**gpu, kl_coef=0.05)
    wide = torch.zeros(4, 3, 260, dtype=F16, device="cuda")
    view = wide.transpose(0, 1)[..., 3:214]
    view.copy_(gpu["logits"])
    tokens = torch.zeros(3, 4, 5, dtype=torch.int32, device="cuda").transpose(1, 2)
    tokens.copy_(gpu["tokens"])
    got = ft.policy_loss(**{**gpu, "logits": view, "tokens": tokens}, kl_coef=0.05)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    one = gpu["logits"][:1].expand(3, 4, 211)  # a request's logits for three
    got = ft.policy_loss(**{**gpu, "logits": one}, kl_coef=0.05)
    want = ft.policy_loss(**{**gpu, "logits": one.contiguous()}, kl_coef=0.05)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_loss_alone_and_repeats(ft):
    a = {k: v.cuda() for k, v in policy_case(4, 6, 9001, 200, BF16, 15, distinct=40).items()}
    b = {k: v.cuda() for k, v in preference_case(4, 6, 9001, 200, 900, BF16, 15,
                                                 distinct=40).items()}
    for fn, q, kw in ((ft.policy_loss, a, dict(kl_coef=0.05)), (ft.preference_loss, b, {})):
        first = fn(**q, **kw)
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(fn(**q, **kw), first))
        loss, logp, d = fn(**q, **kw, grad=False)
        assert d is None and torch.equal(loss, first[0]) and torch.equal(logp, first[1])


def test_empty(ft):
    x = torch.empty(0, 3, 50, device="cuda")
    t = torch.empty(0, 2, 3, dtype=torch.int32, device="cuda")
    n = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    f, f3 = torch.empty(0, 2, device="cuda"), torch.empty(0, 2, 3, device="cuda")
    loss, logp, d = ft.policy_loss(x, t, n, f3, f, f)
    assert loss == 0 and logp.shape == (0, 2, 3) and d.shape == (0, 3, 50)
    pairs = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    assert ft.preference_loss(x, t, n, pairs, f, torch.empty(0, device="cuda"))[0] == 0


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_stream_and_graph(ft, which):
    mk = (lambda s: policy_case(2, 4, 5001, 50, BF16, s)) if which == "policy" else (
        lambda s: preference_case(2, 4, 5001, 50, 99, BF16, s))
    fn = ft.policy_loss if which == "policy" else ft.preference_loss
    kw = dict(kl_coef=0.05) if which == "policy" else {}
    a = {k: v.cuda() for k, v in mk(16).items()}
    want = fn(**a, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fn(**a, **kw)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn(**a, **kw)
    for i in range(4):
        for k, v in mk(30 + i).items():
            a[k].copy_(v)
        graph.replay()
        want = fn(**a, **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i


def test_refusals(ft):
    a = {k: v.cuda() for k, v in policy_case(2, 3, 40, 4, F32, 17).items()}
    for change, exc in [(dict(logits=a["logits"].double()), TypeError),
                        (dict(logits=a["logits"].cpu()), ValueError),
                        (dict(logits=a["logits"][0]), ValueError),
                        (dict(logits=a["logits"].transpose(1, 2)), ValueError),
                        (dict(tokens=a["tokens"].long()), TypeError),
                        (dict(tokens=a["tokens"][:, :, :2]), ValueError),
                        (dict(lengths=a["lengths"][:1]), ValueError),
                        (dict(old_logp=a["old_logp"].half()), TypeError),
                        (dict(advantage=a["advantage"][0]), ValueError),
                        (dict(weight=3.0), TypeError), (dict(ref_logp=None, kl_coef=0.1), ValueError),
                        (dict(clip_low=1.5), ValueError), (dict(clip_high=-0.1), ValueError),
                        (dict(clip_low=math.nan), ValueError), (dict(kl_coef=math.inf), ValueError)]:
        with pytest.raises(exc):
            ft.policy_loss(**{**a, **change})
    b = {k: v.cuda() for k, v in preference_case(2, 3, 40, 4, 5, F32, 18).items()}
    for change, exc in [(dict(pairs=b["pairs"].long()), TypeError),
                        (dict(pairs=b["pairs"][:, :1]), ValueError),
                        (dict(weight=b["weight"][:4]), ValueError),
                        (dict(ref_logp=b["ref_logp"].flatten()), ValueError),
                        (dict(smoothing=1.1), ValueError), (dict(beta=math.nan), ValueError)]:
        with pytest.raises(exc):
            ft.preference_loss(**{**b, **change})
    x = torch.zeros(1, 1, 8, device="cuda")
    t = torch.zeros(1, 4097, 1, dtype=torch.int32, device="cuda")
    z = torch.zeros(1, 4097, device="cuda")
    with pytest.raises(ft.MarisaError, match="4096"):
        ft.policy_loss(x, t, t[..., 0], z[..., None], z, z)


# requests up to the most keys whose slopes are of one size and sign: the
# whole-number sums of the row's table are as large as they get
@pytest.mark.parametrize("distinct", [1, 2])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("C", [1024, 1025, 2047, 2048, 2049, 3000, 4095, 4096])
def test_equal_slopes(ft, C, sign, distinct):
    x, tokens, lengths, _ = keys(2, 1, 5003, C, F32, 19, distinct=distinct, full=True)
    lp = ref.scores(x.double(), tokens, lengths)
    # keys on the policy that made them, one advantage for all
    a = dict(logits=x, tokens=tokens, lengths=lengths, old_logp=lp.float(),
             ref_logp=(lp + 0.3 * sign).float(), advantage=torch.full((2, C), sign),
             weight=torch.full((2, C), 1.0 / (2 * C)))
    check_policy(ft, a, kl=0.0, what="one advantage")
    # the KL term alone
    check_policy(ft, {**a, "advantage": torch.zeros(2, C)}, kl=0.05, what="KL")
    # every key of a request against one of the other
    i = torch.arange(C, dtype=torch.int32)
    pairs = torch.stack([i, i + C] if sign > 0 else [i + C, i], 1)
    check_preference(ft, dict(logits=x, tokens=tokens, lengths=lengths, pairs=pairs,
                              ref_logp=lp.sum(-1).float(), weight=torch.full((C,), 1.0 / C)),
                     what="pairs across requests")


@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
def test_a_masked_token_in_a_pair(ft, smoothing):
    """A pair whose one key holds a token of logit -infinity has h of -+
    infinity: a softplus of it is 0 or infinite, counts only where its share
    of the smoothing is above 0, and the derivative is finite.  Of two such
    keys h is NaN."""
    beta = 0.3
    a = preference_case(1, 2, 50, 4, 2, F32, 20, full=True)
    a["tokens"][0, :, 0] = torch.tensor([3, 4, 5, 6], dtype=torch.int32)
    a["logits"][0, 0, 3] = -math.inf
    w, rf = a["weight"].double(), a["ref_logp"].double()
    lp = ref.scores(a["logits"].double(), a["tokens"], a["lengths"])
    m = lp.sum(-1)[0] - rf[0]
    h = beta * (m[2] - m[3])
    other = w[1] * ((1 - smoothing) * torch.nn.functional.softplus(-h)
                    + smoothing * torch.nn.functional.softplus(h))
    d1 = w[1] * beta * (torch.sigmoid(h) - (1 - smoothing))
    for pair, sig, finite in (((0, 1), 0.0, smoothing == 1.0), ((1, 0), 1.0, smoothing == 0.0)):
        a["pairs"] = torch.tensor([pair, (2, 3)], dtype=torch.int32)
        loss, logp, d = ft.preference_loss(**{k: v.cuda() for k, v in a.items()}, beta=beta,
                                           smoothing=smoothing)
        assert logp[0, 0, 0] == -math.inf and not logp.isnan().any()
        if finite:
            # scores good to LSE and a few units of at most 40, slope at most 1
            assert abs(loss.item() - other) <= w[1] * beta * 4 * (ref.LSE + 200 * ref.U)
        else:
            assert loss == math.inf
        d0 = w[0] * beta * (sig - (1 - smoothing))
        gkey = torch.zeros(4).double()
        gkey[pair[0]] += d0
        gkey[pair[1]] -= d0
        gkey[2] += d1
        gkey[3] -= d1
        g = gkey[None, :, None].expand(1, 4, 2)
        p = torch.softmax(a["logits"].double(), -1)
        want = -p * g.sum(1)[..., None]
        want.scatter_add_(2, a["tokens"].long().transpose(1, 2), g.transpose(1, 2).contiguous())
        gerr = (w.sum() * beta * (4 * beta * (ref.LSE + 200 * ref.U) + 16 * ref.U)).expand(1, 4, 2)
        check_gradient(d, want, ref.gradient_bound(a["logits"].double(), a["tokens"], a["lengths"],
                                                   g, gerr), (pair, smoothing))
    a["tokens"][0, 1, 0] = 3
    a["pairs"] = torch.tensor([(0, 1), (2, 3)], dtype=torch.int32)
    loss, _, d = ft.preference_loss(**{k: v.cuda() for k, v in a.items()}, beta=beta,
                                    smoothing=smoothing)
    assert loss.isnan() and d.isnan().any()


# rows in a workgroup's registers, and in parts
@pytest.mark.parametrize("C", [1, 3, 1100])
@pytest.mark.parametrize("V", [60, 40001])
def test_a_row_of_nothing(ft, C, V):
    """A row whose mask leaves nothing: scores of -infinity, no probability
    anywhere; its gradient is its tokens' own slopes, 0 for the policy loss
    without the KL term (the ratio is 0)."""
    a = policy_case(2, 3, V, C, F32, 21, full=True)
    gpu = {k: v.cuda() for k, v in a.items()}
    whole = ft.policy_loss(**gpu)
    a["logits"][1, 1] = -math.inf
    a["old_logp"][1, :, 1] = -2.0
    gpu = {k: v.cuda() for k, v in a.items()}
    loss, logp, d = ft.policy_loss(**gpu)
    assert loss.isfinite() and (logp[1, :, 1] == -math.inf).all()
    assert (d[1, 1] == 0).all()
    rest = torch.ones(2, 3, dtype=torch.bool)
    rest[1, 1] = False
    assert torch.equal(d[rest.cuda()], whole[2][rest.cuda()])
    # preferred keys of the other request: h is infinite, and the keys of the
    # masked row have slopes of -weight beta smoothing
    i = torch.arange(C, dtype=torch.int32, device="cuda")
    w = torch.full((C,), 1.0 / C, device="cuda")
    loss, logp, d = ft.preference_loss(gpu["logits"], gpu["tokens"], gpu["lengths"],
                                       torch.stack([i, i + C], 1), torch.zeros(2, C, device="cuda"),
                                       w, beta=0.5, smoothing=0.25)
    assert (logp[1, :, 1] == -math.inf).all() and d.isfinite().all()
    want = torch.zeros(V).double()
    want.index_add_(0, a["tokens"][1, :, 1].long(), torch.full((C,), -0.5 * 0.25 / C).double())
    # a pair's slope rounds a few times, up to C of them are summed
    assert ((d[1, 1].double().cpu() - want).abs() <= (C + 8) * ref.U * want.abs()).all()


# rows of a key each: of a workgroup's registers, or in parts, where each
# block decides whether the row's token is in its span
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [4097, 8193, 20001, 32769, 50021, 65537, 131073])
def test_rows_of_a_key_each(ft, dtype, V):
    R, S = 7, 4
    span = 4096 if dtype == F32 else 8192  # logits of a block of the gradient
    at = [0, span - 1, span, 2 * span - 1, 2 * span, V - 1, V - 2, (V - 1) // span * span, V // 2]
    tokens = torch.tensor([t % V for t in at] * 4)[:R * S].view(R, 1, S).to(torch.int32)
    a = policy_case(R, S, V, 1, dtype, V)
    lp = ref.scores(a["logits"].double(), tokens, torch.full((R, 1), S))
    a["tokens"] = tokens
    a["lengths"] = torch.tensor([4, 0, 1, 4, 3, 2, 4], dtype=torch.int32)[:, None]
    a["old_logp"], a["ref_logp"] = (lp - 0.1).float(), (lp + 0.2).float()
    check_policy(ft, a, what="policy")
    b = preference_case(R, S, V, 1, 9, dtype, V)
    b.update(tokens=tokens, lengths=a["lengths"], ref_logp=lp.sum(-1).float() * 0.9)
    check_preference(ft, b, what="preference")
    # no gradient wanted
    gpu = {k: v.cuda() for k, v in a.items()}
    full, alone = (ft.policy_loss(**gpu, kl_coef=0.05, grad=g) for g in (True, False))
    assert torch.equal(full[0], alone[0]) and torch.equal(full[1], alone[1])
