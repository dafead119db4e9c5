"""flashtrie.cross_entropy_loss against its definition in 64 bits, within the
bounds of table_reference.py."""

import ctypes as C
import math
import os

import pytest
import torch

import table_reference as ref
import test_table_args as args

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(T, V, H, dtype, seed, lean=4.0, scale=None):
    g = torch.Generator().manual_seed(seed)
    weight = (torch.randn((V, H), generator=g) * 2.5 * H ** -0.5).to(dtype)
    targets = torch.randint(0, V, (T,), generator=g)
    x = torch.randn((T, H), generator=g) + lean / 6.25 * weight[targets].float()
    targets[torch.rand(T, generator=g) < 0.15] = -1
    if T == 1:
        targets[:] = V // 2
    w = (torch.rand(T, generator=g) + 0.5) * ((2.0 ** 12 if dtype == F16 else 1.0) if scale is None else scale)
    return dict(x=x.to(dtype).cuda(), weight=weight.cuda(), targets=targets.to(torch.int32).cuda(),
                row_weight=(w / max(T, 1)).cuda())


def compare(got, want, what):
    for (name, (w, tol)), y in zip(want.items(), got):
        if y is None:
            continue
        y = y.double()
        assert torch.equal(y.isnan(), w.isnan()), (what, name, int(y.isnan().sum()))
        ok = (y == w) | w.isnan() | ((y - w).abs() <= tol)
        assert ok.all(), (what, name, ((y - w).abs() / tol)[~ok].max().item(), int((~ok).sum()))


def check(ft, a, smoothing, what, **kw):
    print(what, tuple(a["x"].shape), tuple(a["weight"].shape), a["x"].dtype, smoothing, flush=True)
    got = ft.cross_entropy_loss(**a, smoothing=smoothing, **kw)
    loss, logp, dx, dw = got
    assert loss.shape == () and loss.dtype == logp.dtype == F32
    compare(got, ref.cross_entropy(**a, smoothing=smoothing), what)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [1, 2, 15, 17, 63, 64, 65, 130, 256, 257, 300, 520])
def test_rows(ft, dtype, T):
    check(ft, inputs(T, 517, 128, dtype, T), 0.1, "rows")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 127, 128, 129, 255, 256, 257, 513, 1000])
@pytest.mark.parametrize("H", [1, 7, 64, 65, 100, 192, 256, 320])
def test_vocabulary_and_hidden(ft, dtype, V, H):
    check(ft, inputs(20, V, H, dtype, V * H), 0.0 if V & 1 else 0.2, "sizes")


@pytest.mark.parametrize("T,V,H,dtype", [(8, 32768, 512, BF16), (100, 20001, 1024, BF16),
                                         (700, 9001, 768, F16), (1100, 8192, 256, BF16),
                                         (33, 70001, 64, F16), (300, 5000, 2048, BF16)])
def test_working_sizes(ft, T, V, H, dtype):
    check(ft, inputs(T, V, H, dtype, T + V), 0.1, "working")


# one pass over the table for few rows: its tiles of 64, 32 and 16 tokens, hidden
# columns that the waves share unevenly, more tiles than workgroups
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H", [*[(t, h) for t in (1, 9, 16) for h in (64, 448, 512, 576, 960, 1024, 1088, 1600, 2048)],
                                 *[(t, h) for t in (17, 32) for h in (64, 320, 512)], (17, 576), (3, 2112), (33, 64)])
def test_few_rows(ft, dtype, T, H):
    for V in (5, 65, 4113):
        a = inputs(T, V, H, dtype, T + V + H)
        whole = check(ft, a, 0.1, "few")
        some = ft.cross_entropy_loss(**a, smoothing=0.1, weight_grad=False)
        assert all(torch.equal(p, q) for p, q in zip(whole[:3], some[:3]))


@pytest.mark.parametrize("T,V,H", [(10, 70000, 128), (25, 70000, 64)])
def test_few_rows_many_tokens(ft, T, V, H):
    check(ft, inputs(T, V, H, BF16, 1), 0.1, "few")


# tables that are read and written past the caches (more than 128 MB), of few rows
# and more; and just under
@pytest.mark.parametrize("T,V,H,dtype", [(9, 70001, 1024, BF16), (20, 140000, 512, F16), (3, 33001, 2048, BF16),
                                         (70, 66000, 1024, F16), (9, 65536, 1024, BF16), (9, 65537, 1024, BF16)])
def test_large_tables(ft, T, V, H, dtype):
    check(ft, inputs(T, V, H, dtype, V), 0.1, "large")


def call(ft, a, dx, dweight, smoothing=0.1):
    """The C call, for what the Python one does not offer."""
    lib = C.CDLL(os.path.join(args.ROOT, "flash-trie_amd", "libflashtrie_amd.so"))
    (T, H), V = a["x"].shape, a["weight"].shape[0]
    loss, logp = torch.empty((), device="cuda"), torch.empty(T, device="cuda")
    s = args.CrossEntropy(
        device=0, dtype=args.BF16, rows=T, hidden=H, vocab=V, x=a["x"].data_ptr(), x_stride=a["x"].stride(0),
        weight=a["weight"].data_ptr(), weight_stride=a["weight"].stride(0), target=a["targets"].data_ptr(),
        row_weight=a["row_weight"].data_ptr(), smoothing=smoothing, loss=loss.data_ptr(), logp=logp.data_ptr(),
        dx=dx.data_ptr() if dx is not None else None, dx_stride=dx.stride(0) if dx is not None else 0,
        dweight=dweight.data_ptr() if dweight is not None else None,
        dweight_stride=dweight.stride(0) if dweight is not None else 0)
    lib.ft_cross_entropy_loss_workspace.restype = C.c_size_t
    n = lib.ft_cross_entropy_loss_workspace(C.byref(s))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.ft_cross_entropy_loss(C.byref(s), C.c_void_p(ws.data_ptr()), C.c_size_t(n), stream) == 0
    torch.cuda.synchronize()
    return loss, logp


@pytest.mark.parametrize("T,V,H", [(10, 300, 64), (100, 300, 128), (300, 700, 192), (20, 90, 50), (0, 40, 64)])
def test_outputs_of_any_stride(ft, T, V, H):
    """The table's gradient alone; both in rows of wider tensors, whose other
    columns stay as they were."""
    a = inputs(T, V, H, BF16, 17)
    want = ft.cross_entropy_loss(**a, smoothing=0.1)
    for with_dx in (False, True):
        dx = torch.full((max(T, 1), H + 9), 5.0, device="cuda").bfloat16()
        dw = torch.full((V, H + 7), 5.0, device="cuda").bfloat16()
        loss, logp = call(ft, a, dx[:T, 3:3 + H] if with_dx and T else None, dw[:, 1:1 + H])
        assert torch.equal(loss, want[0]) and torch.equal(logp, want[1])
        assert torch.equal(dw[:, 1:1 + H], want[3])
        assert (dw[:, 0] == 5).all() and (dw[:, 1 + H:] == 5).all()
        if with_dx and T:
            assert torch.equal(dx[:, 3:3 + H], want[2])
            assert (dx[:, :3] == 5).all() and (dx[:, 3 + H:] == 5).all()
        else:
            assert (dx == 5).all()


@pytest.mark.parametrize("smoothing", [0.0, 1.0, 0.5])
def test_smoothing(ft, smoothing):
    check(ft, inputs(40, 333, 96, BF16, 3), smoothing, "smoothing")


# tiles of 256, 192, 160 and 224 rows, and operands of any alignment
@pytest.mark.parametrize("T,V,H,dtype", [(20000, 4000, 64, BF16), (1152, 60001, 64, BF16),
                                         (777, 90001, 64, F16), (2016, 40001, 128, BF16),
                                         (6000, 30001, 40, F16)])
def test_pieces(ft, T, V, H, dtype):
    """More tokens than a piece of the vocabulary holds: its size goes with
    the rows."""
    check(ft, inputs(T, V, H, dtype, 4), 0.1, "pieces")


def test_what_is_asked_for(ft):
    a = inputs(70, 1000, 128, BF16, 5)
    whole = ft.cross_entropy_loss(**a)
    some = ft.cross_entropy_loss(**a, weight_grad=False)
    none = ft.cross_entropy_loss(**a, grad=False)
    assert some[3] is None and none[2] is None and none[3] is None
    assert all(torch.equal(p, q) for p, q in zip(whole[:3], some[:3]))
    assert all(torch.equal(p, q) for p, q in zip(whole[:2], none[:2]))


def test_by_differences(ft):
    """The gradients against differences of the loss along a direction, in 64
    bits by the definition."""
    a = inputs(33, 200, 64, BF16, 6)
    _, _, dx, dw = ft.cross_entropy_loss(**a, smoothing=0.1)
    g = torch.Generator("cuda").manual_seed(1)
    n = lambda t: torch.randn(t.shape, device="cuda", generator=g, dtype=torch.float64)  # noqa: E731
    vx, vw = n(dx), n(dw)
    y, used = a["targets"].long(), a["targets"] >= 0

    def loss(e):
        l = torch.log_softmax((a["x"].double() + e * vx) @ (a["weight"].double() + e * vw).t(), 1)
        each = -0.9 * l.gather(1, y.clamp(min=0)[:, None])[:, 0] - 0.1 * l.mean(1)
        return (a["row_weight"].double() * each)[used].sum()

    slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
    got = (dx.double() * vx).sum() + (dw.double() * vw).sum()
    want = ref.cross_entropy(**a, smoothing=0.1)
    tol = (want["dx"][1] * vx.abs()).sum() + (want["dweight"][1] * vw.abs()).sum()
    # (a difference over 2e-4 is off by its third derivative's 1e-8)
    assert (got - slope).abs() <= tol + 1e-6 * slope.abs() + 1e-6


def test_padding(ft):
    """Rows without a target, or of weight 0, hold anything and count nothing;
    nor do they reach others."""
    a = inputs(40, 300, 64, BF16, 7)
    a["targets"][:5] = -1
    a["row_weight"][5:8] = 0.0
    a["targets"][5:8] = 7
    clean = ft.cross_entropy_loss(**a)
    a["x"][0], a["x"][1], a["x"][2], a["x"][6] = math.nan, math.inf, -math.inf, math.nan
    a["row_weight"][0] = math.nan
    loss, logp, dx, dw = ft.cross_entropy_loss(**a)
    assert not logp[:5].any() and not dx[:8].any() and logp[6].isnan()
    assert torch.equal(loss, clean[0]) and torch.equal(dw, clean[3]) and torch.equal(dx, clean[2])
    keep = torch.arange(40, device="cuda") != 6
    assert torch.equal(logp[keep], clean[1][keep])


def test_nothing_counts(ft):
    a = inputs(40, 300, 64, F16, 8)
    a["targets"][:] = -3
    for out in ft.cross_entropy_loss(**a, smoothing=0.1):
        assert not out.any()


def test_target_out_of_range(ft):
    a = inputs(20, 300, 64, BF16, 9)
    a["targets"][3] = 300
    a["targets"][4] = 2 ** 31 - 1
    loss, logp, dx, dw = ft.cross_entropy_loss(**a)
    assert loss.isnan() and logp[3:5].isnan().all() and dx[3:5].isnan().all() and dw.isnan().all()
    keep = [i for i in range(20) if i not in (3, 4)]
    assert not logp[keep].isnan().any() and not dx[keep].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_odd_values(ft, dtype):
    a = inputs(20, 300, 64, dtype, 10)
    a["targets"][:] = 5
    a["x"][2, 3] = math.nan
    a["x"][4] = 0.0
    loss, logp, dx, dw = ft.cross_entropy_loss(**a)
    assert loss.isnan() and logp[2].isnan() and dx[2].isnan().all() and dw.isnan().all()
    assert abs(logp[4].item() + math.log(300)) < 1e-5
    keep = [i for i in range(20) if i != 2]
    assert not logp[keep].isnan().any() and not dx[keep].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weights_far_apart(ft, dtype):
    """Each row's gradient is as good as its own weight's; of either sign."""
    a = inputs(64, 400, 128, dtype, 11, scale=1.0)
    a["row_weight"] *= 2.0 ** torch.linspace(-10, 10, 64, device="cuda")
    a["row_weight"][::3] *= -1
    check(ft, a, 0.1, "weights")


def test_sure_rows(ft):
    """Logits far from each other: most probabilities are 0."""
    a = inputs(40, 500, 64, BF16, 12, lean=60.0)
    a["x"] *= 4
    check(ft, a, 0.0, "sure")


def test_strides(ft):
    a = inputs(50, 700, 128, BF16, 13)
    want = ft.cross_entropy_loss(**a, smoothing=0.1)

    def wider(t, left, right):
        w = torch.full((t.shape[0], t.shape[1] + left + right), math.nan, dtype=t.dtype, device="cuda")
        w[:, left:left + t.shape[1]] = t
        return w[:, left:left + t.shape[1]]

    for left, right in ((8, 8), (1, 0), (3, 4)):
        b = dict(a, x=wider(a["x"], left, right), weight=wider(a["weight"], left, right))
        check(ft, b, 0.1, f"strides {left} {right}")
    twice = a["x"][:25].repeat_interleave(2, 0)
    b = dict(a, x=a["x"][:25, None].expand(25, 2, 128).reshape(50, 128))
    assert torch.equal(b["x"], twice)
    check(ft, dict(a, x=a["x"][:1].expand(50, 128)), 0.1, "one state for all")
    check(ft, dict(a, targets=a["targets"].repeat_interleave(2)[::2]), 0.1, "targets apart")
    assert all(torch.equal(p, q) for p, q in zip(want, ft.cross_entropy_loss(**a, smoothing=0.1)))


def test_empty(ft):
    w = torch.randn(100, 64, device="cuda").bfloat16()
    x = w[:0]
    loss, logp, dx, dw = ft.cross_entropy_loss(x, w, torch.empty(0, dtype=torch.int32, device="cuda"),
                                               torch.empty(0, device="cuda"))
    assert loss == 0 and logp.shape == (0,) and dx.shape == (0, 64)
    assert dw.shape == (100, 64) and not dw.any()


def test_stream_and_graph(ft):
    """On another stream; recorded, and replayed on new inputs; two recorded
    calls side by side."""
    a = inputs(300, 3000, 256, BF16, 14)
    want = ft.cross_entropy_loss(**a, smoothing=0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ft.cross_entropy_loss(**a, smoothing=0.1)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    static, other = {k: v.clone() for k, v in a.items()}, inputs(20, 500, 64, F16, 15)
    want_other = ft.cross_entropy_loss(**other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ft.cross_entropy_loss(**static, smoothing=0.1)
        out_other = ft.cross_entropy_loss(**other)
    for i in range(4):
        for k, v in inputs(300, 3000, 256, BF16, 20 + i).items():
            static[k].copy_(v)
        graph.replay()
        want = ft.cross_entropy_loss(**static, smoothing=0.1)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), i
        assert all(torch.equal(p, q) for p, q in zip(out_other, want_other)), i


def test_refusals(ft):
    a = inputs(10, 50, 64, BF16, 16)
    for change, exc in [(dict(x=a["x"].float()), TypeError), (dict(x=a["x"].half()), TypeError),
                        (dict(x=a["x"][0]), ValueError), (dict(x=a["x"].cpu()), ValueError),
                        (dict(x=a["x"][:, :32]), ValueError),
                        (dict(x=a["x"].t()), ValueError), (dict(weight=a["weight"].t()), ValueError),
                        (dict(targets=a["targets"].long()), TypeError),
                        (dict(targets=a["targets"][:9]), ValueError),
                        (dict(row_weight=a["row_weight"].double()), TypeError),
                        (dict(row_weight=a["row_weight"][:9]), ValueError),
                        (dict(x=a["x"].float(), weight=a["weight"].float()), TypeError)]:
        with pytest.raises(exc):
            ft.cross_entropy_loss(**dict(a, **change))
    for s in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="smoothing"):
            ft.cross_entropy_loss(**a, smoothing=s)
    with pytest.raises(ValueError, match="at least 1"):
        ft.cross_entropy_loss(a["x"], a["weight"][:0], a["targets"], a["row_weight"])
