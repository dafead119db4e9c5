"""flashtrie.pack_weight and packed_logits against plain forms: codes, scales
and layout exactly, logits within the bounds of table_reference.py."""

import math

import pytest
import torch

import table_reference as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def table(V, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((V, H), generator=g) * 2.5 * H ** -0.5).to(dtype).cuda()


def states(T, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, H), generator=g).to(dtype).cuda()


def check(ft, x, weight, group, out_dtype, what, out=None):
    print(what, tuple(x.shape), tuple(weight.shape), group, x.dtype, out_dtype, flush=True)
    packed, scales = ft.pack_weight(weight, group)
    codes, s = ref.pack(weight, group)
    y = ft.packed_logits(x, packed, scales, weight.shape[0], out_dtype, out)
    assert y.dtype == out_dtype and y.shape == (x.shape[0], weight.shape[0])
    want, err = ref.packed_logits(x, codes, s, group)
    got = y.double()
    tol = err + ref.rounding(want, out_dtype)
    assert torch.equal(got.isnan(), want.isnan()), what
    ok = (got == want) | want.isnan() | ((got - want).abs() <= tol)
    assert ok.all(), (what, ((got - want).abs() / tol)[~ok].max().item())
    return y


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("V,H", [(1, 1), (15, 31), (16, 128), (17, 129), (50, 100), (100, 384), (33, 513)])
def test_pack(ft, dtype, group, V, H):
    w = table(V, H, dtype, V + H)
    packed, scales = ft.pack_weight(w, group)
    want, want_scales = ref.lay_out(*ref.pack(w, group), group)
    assert torch.equal(packed.cpu(), want) and torch.equal(scales.cpu(), want_scales)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_pack_odd_values(ft, dtype):
    w = table(20, 256, dtype, 1)
    w[0] = 0.0
    w[1, 5], w[2, 6], w[3, 100] = math.nan, math.inf, -math.inf
    w[4, :32] = 1.0                      # equals: the first
    w[5, 3], w[5, 9] = 7.0, -7.0         # of either sign: the first
    w[6, 9], w[6, 3] = 7.0, -7.0
    w[7] = torch.finfo(dtype).smallest_normal
    w[8] = torch.finfo(dtype).smallest_normal / 64
    w[9] = torch.finfo(dtype).max
    w[10, ::2] = -0.0
    for group in (32, 64, 128):
        packed, scales = ft.pack_weight(w, group)
        want, want_scales = ref.lay_out(*ref.pack(w, group), group)
        assert torch.equal(packed.cpu(), want)
        assert torch.equal(scales.cpu().isnan(), want_scales.isnan())
        assert torch.equal(scales.cpu().nan_to_num(3.0), want_scales.nan_to_num(3.0))


def test_pack_error(ft):
    """A weight is off by at most half a step, or by a whole one at the end
    that has no code."""
    w = table(500, 256, F16, 2)
    codes, s = ref.pack(w, 32)
    back = codes.double() * s.double().repeat_interleave(32, 1)
    step = s.double().abs().repeat_interleave(32, 1)
    assert ((back - w.double()).abs() <= step * (1 + 2.0 ** -6)).all()


def test_pack_strides(ft):
    w = table(70, 300, BF16, 3)
    a, b = ft.pack_weight(w[::2, 1:200], 64), ft.pack_weight(w[::2, 1:200].contiguous(), 64)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [1, 2, 8, 15, 16, 17, 32, 33, 48, 50, 64, 65, 84, 96, 97, 128, 130, 300])
def test_rows(ft, dtype, T):
    for group in (32, 64, 128):
        for out in (F32, dtype):
            check(ft, states(T, 256, dtype, T), table(517, 256, dtype, 5), group, out, "rows")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("V", [1, 15, 16, 17, 31, 33, 63, 255, 257, 1000])
@pytest.mark.parametrize("H", [1, 7, 31, 32, 33, 100, 128, 129, 500, 1024])
def test_vocabulary_and_hidden(ft, dtype, V, H):
    check(ft, states(5, H, dtype, V), table(V, H, dtype, H), 32 << V % 3, F32, "sizes")


@pytest.mark.parametrize("T,V,H,group,dtype,out", [
    (8, 32768, 512, 32, BF16, F32), (84, 20003, 1024, 128, F16, F16), (16, 300001, 512, 64, BF16, F32),
    (1, 100003, 1024, 64, F16, F32), (40, 5001, 2048, 32, BF16, BF16), (9, 3001, 4096, 64, BF16, F32),
    (20, 3001, 5000, 128, F16, F32), (70, 1001, 9000, 32, BF16, F32)])
def test_working_sizes(ft, T, V, H, group, dtype, out):
    check(ft, states(T, H, dtype, T), table(V, H, dtype, V), group, out, "working")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_range(ft, dtype):
    """Rows of any size, each with its own."""
    w = table(100, 128, dtype, 6)
    x = states(12, 128, dtype, 7).double()
    top = 38 if dtype == BF16 else 4
    x = (x * 10.0 ** torch.linspace(-top, top - 1, 12, device="cuda", dtype=torch.float64)[:, None]).to(dtype)
    x[3] = 0.0
    x[5, ::2] *= 2.0 ** -20
    check(ft, x, w, 32, F32, "range")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_odd_values(ft, dtype):
    """A NaN or infinity stays in its row, or in its token."""
    w, x = table(100, 256, dtype, 8), states(20, 256, dtype, 9)
    clean = check(ft, x, w, 64, F32, "clean")
    x[3, 7], x[4, 100] = math.nan, math.inf
    w[11, 30], w[50, 200] = math.nan, -math.inf
    y = ft.packed_logits(x, *ft.pack_weight(w, 64), 100, F32)
    assert y[3].isnan().all() and y[:, 11].isnan().all() and y[:, 50].isnan().all()
    assert not y[4].isfinite().any()
    rows = [i for i in range(20) if i not in (3, 4)]
    tokens = [i for i in range(100) if i not in (11, 50)]
    assert torch.equal(y[rows][:, tokens], clean[rows][:, tokens])


def test_columns_past_the_table(ft):
    """Codes and scales past the columns are not looked at."""
    w, x = table(40, 72, BF16, 10), states(5, 72, BF16, 11)
    packed, scales = ft.pack_weight(w, 32)
    want = ft.packed_logits(x, packed, scales, 40, F32)
    scales[:, :, :, 3] = math.nan
    packed.view(torch.int32)[..., 3] = -1
    assert torch.equal(want, ft.packed_logits(x, packed, scales, 40, F32))


def test_rows_that_are_not_its_own(ft):
    big = torch.full((30, 700), 7.0, device="cuda")
    x, w = states(10, 128, F16, 12), table(501, 128, F16, 13)
    check(ft, x, w, 32, F32, "out", out=big[5:25:2, 3:504])
    keep = torch.ones(30, 700, dtype=torch.bool, device="cuda")
    keep[5:25:2, 3:504] = False
    assert (big[keep] == 7.0).all()
    wide = states(20, 300, F16, 14)
    check(ft, wide[::2, 5:133], w, 32, F16, "x of any stride")
    check(ft, wide[:1, :128].expand(10, 128), w, 32, F16, "one row for all")


def test_far_into_memory(ft):
    """A table of more than 2^32 codes, and logits past 2^31."""
    V, H, T = 1 << 23, 640, 300
    packed = torch.full((V // 16, 5, 64, 16), 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.ones((V // 16, 5, 16, 1), dtype=BF16, device="cuda")
    packed[-1, -1, 16 * 3 + 15, 15] = 0x98  # the last column of the last token: code 9
    x = torch.zeros((T, H), dtype=BF16, device="cuda")
    x[-1, -1] = 3.0
    y = ft.packed_logits(x, packed, scales, V)
    assert y[-1, -1] == 3.0
    y[-1, -1] = 0.0
    assert not y.any()


def test_empty(ft):
    w = table(50, 128, F16, 15)
    y = ft.packed_logits(w[:0], *ft.pack_weight(w), 50)
    assert y.shape == (0, 50) and y.dtype == F16


def test_stream_and_graph(ft):
    w, x = table(3000, 512, BF16, 16), states(20, 512, BF16, 17)
    packed, scales = ft.pack_weight(w)
    want = ft.packed_logits(x, packed, scales, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ft.packed_logits(x, *ft.pack_weight(w), 3000)
    s.synchronize()
    assert torch.equal(got, want)
    static, static_w = x.clone(), w.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p2 = ft.pack_weight(static_w)
        out = ft.packed_logits(static, *p2, 3000)
    for i in range(4):
        static.copy_(states(20, 512, BF16, 20 + i))
        static_w.copy_(table(3000, 512, BF16, 30 + i))
        graph.replay()
        want = ft.packed_logits(static, *ft.pack_weight(static_w), 3000)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_out_and_autograd(ft):
    x, w = states(4, 128, F16, 18), table(50, 128, F16, 19)
    p = ft.pack_weight(w)
    out = torch.zeros(4, 50, device="cuda")
    version = out._version
    assert ft.packed_logits(x, *p, 50, out=out) is out and out._version > version
    with pytest.raises(ValueError, match="gradient"):
        ft.packed_logits(x, *p, 50, out=torch.zeros(4, 50, device="cuda", requires_grad=True))


def test_refusals(ft):
    x, w = states(4, 128, F16, 20), table(50, 128, F16, 21)
    p, s = ft.pack_weight(w)
    for args, exc in [((x.float(), p, s, 50), TypeError), ((x.bfloat16(), p, s, 50), TypeError),
                      ((x[:, :64], p, s, 50), None), ((x, p, s, 49), None),
                      ((x, p, s, 48), ValueError), ((x, p, s, 65), ValueError), ((x, p, s, 0), ValueError),
                      ((torch.cat((x, x), 1), p, s, 50), ValueError), ((x, p.int(), s, 50), TypeError),
                      ((x, p[..., :8], s, 50), ValueError), ((x, p, s[..., :3], 50), ValueError),
                      ((x.cpu(), p, s, 50), ValueError), ((x, p, s, 50, torch.bfloat16), TypeError),
                      ((x.t(), p, s, 50), ValueError)]:
        if exc is None:
            ft.packed_logits(*args)
            continue
        with pytest.raises(exc):
            ft.packed_logits(*args)
    for bad, exc in [((w, 16), ValueError), ((w, 0), ValueError), ((w.float(), 32), TypeError),
                     ((w[0], 32), ValueError), ((w.t(), 32), ValueError), ((w.cpu(), 32), ValueError)]:
        with pytest.raises(exc):
            ft.pack_weight(*bad)
