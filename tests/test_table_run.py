"""The vocabulary table's operators together, as run_model_head.py uses them:
looked up, trained, packed, served and searched."""

import math

import pytest
import torch

import run_model_head as M
import table_reference as ref

SMALL = ["--requests", "5", "--num-keys", "2000", "--vocab-size", "1111", "--hidden", "96",
         "--rank", "4", "--topk-tokens", "40", "--beam-size", "20", "--rounds", "1"]


def test_before():
    tokens = torch.tensor([[[5, 6, 7], [8, 0, 0]]], dtype=torch.int32)
    assert M.before(tokens).tolist() == [[[-1, 5, 6], [-1, 8, 0]]]


@pytest.mark.parametrize("bad", [["--pretrain", "-1"], ["--packed", "16"]])
def test_arguments(bad):
    with pytest.raises(SystemExit):
        M.parse_args(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("group", ["32", "128"])
def test_run(ft, dtype, group):
    args = M.parse_args(SMALL + ["--pretrain", "3", "--packed", group, "--dtype", dtype])
    first, line, packed = M.run(args, log=lambda *_: None)
    assert len(first["pretrain"]) == 3 and all(math.isfinite(v) for v in first["pretrain"])
    assert line["keys"] > 5 and packed["keys"] > 5 and 0 <= packed["packed"] <= 1
    again = M.run(args, log=lambda *_: None)
    assert again[0] == first and again[2] == packed


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,S,V,H", [(2, 1, 5, 40, 32), (3, 7, 4, 200, 64), (2, 90, 8, 500, 128)])
def test_tied_gradient(ft, dtype, R, C, S, V, H):
    """The gradient of a table that is read on both sides against autograd on
    the definition, 64 bits."""
    g = torch.Generator().manual_seed(R * C)
    table = (torch.randn(V, H, generator=g) * 2.5 * H ** -0.5).to(dtype)
    x = torch.randn(R, C, S, H, generator=g).to(dtype)
    tokens = torch.randint(0, V, (R, C, S), generator=g, dtype=torch.int32)
    lengths = torch.randint(0, S + 1, (R, C), generator=g, dtype=torch.int32)
    lengths[0, 0] = S
    loss, d = M.supervised(ft, x.cuda(), table.cuda(), tokens.cuda(), lengths.cuda(), 1.5)

    w = table.double().requires_grad_()
    inputs, keys = M.before(tokens), int((lengths > 0).sum())
    there = torch.arange(S) < lengths[..., None]
    looked = torch.where((there & (inputs >= 0))[..., None], 1.5 * w[inputs.clamp(min=0).long()], 0.0)
    # (the lookup's and the state's own roundings are not differentiated)
    states = x + ref.embed(inputs, table, 1.5, lengths)
    smooth = x.double() + looked
    smooth = smooth + (states.double() - smooth).detach()
    lp = torch.log_softmax(smooth @ w.t(), -1).gather(-1, tokens[..., None].long())[..., 0]
    share = 1.0 / (lengths.clamp(min=1) * keys)
    total = -torch.where(there, lp * share[..., None], 0.0).sum()
    total.backward()

    rows = torch.where(there, tokens, -1).view(-1)
    weight = share.float()[..., None].expand(R, C, S).reshape(-1)
    flat = states.view(-1, H)
    want = ref.cross_entropy(flat, table, rows, weight, 0.0)
    assert abs(loss.item() - total.item()) <= want["loss"][1] + 1e-6
    # the loss's part by its own bound; the lookup's: dx by its bound, then the sum
    dx, dxe = want["dx"]
    near = dx.view(R, C, S, H)
    _, part = ref.embed_grad(near.to(dtype), inputs, V, 1.5, lengths, want["dweight"][0].to(dtype))
    spread = torch.zeros(V, H, dtype=torch.float64)
    use = there & (inputs >= 0)
    spread.index_add_(0, inputs[use].long(), 1.5 * dxe.view(R, C, S, H)[use])
    tol = want["dweight"][1] + spread + part + ref.rounding(w.grad, dtype)
    assert ((d.double().cpu() - w.grad).abs() <= tol).all()


@pytest.mark.gpu
def test_calls_side_by_side(ft):
    """Every operator on two streams at once, with memory of its own each, as
    one after the other."""
    g = torch.Generator("cuda").manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def calls(T, V, H, dtype):
        w, x = (normal(V, H) * 2 * H ** -0.5).to(dtype), normal(T, H).to(dtype)
        y = torch.randint(-1, V, (T,), device="cuda", generator=g, dtype=torch.int32)
        r = torch.rand(T, device="cuda", generator=g)
        return lambda: (*ft.cross_entropy_loss(x, w, y, r, smoothing=0.1),
                        ft.packed_logits(x, *ft.pack_weight(w, 64), V), ft.embed(y, w, 2.0),
                        ft.embed_grad(x, y, V, 3.0))

    work = [calls(300, 20000, 256, torch.bfloat16), calls(10, 30000, 512, torch.float16),
            calls(5000, 3000, 64, torch.bfloat16), calls(70, 9000, 1024, torch.float16)]
    want = [c() for c in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(3):
        got = []
        for s, c in zip(streams, work):
            with torch.cuda.stream(s):
                got.append([c() for _ in range(3)])
        torch.cuda.synchronize()
        for w, three in zip(want, got):
            for one in three:
                assert all(torch.equal(p, q) for p, q in zip(one, w))


@pytest.mark.gpu
def test_an_error_of_another_call(ft):
    """An error that an earlier call of the application left with the HIP
    runtime is not taken for a launch's."""
    import ctypes
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    w = torch.randn(5000, 64, device="cuda").bfloat16()
    y = torch.arange(3000, device="cuda", dtype=torch.int32)
    r = torch.ones(3000, device="cuda")
    packed = ft.pack_weight(w)
    calls = [lambda: ft.cross_entropy_loss(w[:3000], w, y, r), lambda: ft.cross_entropy_loss(w[:3], w, y[:3], r[:3]),
             lambda: ft.cross_entropy_loss(w[:30, :50], w[:, :50], y[:30], r[:30]), lambda: ft.pack_weight(w),
             lambda: (ft.packed_logits(w[:40], *packed, 5000),), lambda: (ft.embed(y, w),),
             lambda: (ft.embed_grad(w[:3000], y, 5000),), lambda: (ft.embed_grad(w[:30], y[:30], 5000),)]
    for call in calls:
        want = call()
        assert hip.hipSetDevice(1 << 20) != 0  # no such device
        try:
            got = call()
        finally:
            hip.hipGetLastError()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
