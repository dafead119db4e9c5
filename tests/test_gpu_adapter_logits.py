"""flashtrie.adapter_logits against a plain form in 64 bits, within the
bounds of head_reference.py."""

import math

import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(T, V, H, G, r, dtype, seed, adapter=None):
    g = torch.Generator().manual_seed(seed)

    def n(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()

    if adapter is None:
        adapter = torch.randint(-1, max(1, G), (T,), generator=g)
        if G == 0:
            adapter.fill_(-1)
    return dict(x=n(T, H), weight=n(V, H, scale=H ** -0.5), down=n(G, r, H, scale=H ** -0.5),
                up=n(G, V, r), adapter=adapter.to(torch.int32).cuda(),
                scale=(torch.rand(G, generator=g) * 2 - 0.5).cuda())


def check(ft, a, out_dtype, what, out=None):
    print(what, tuple(a["x"].shape), tuple(a["weight"].shape), tuple(a["up"].shape), out_dtype,
          flush=True)
    y = ft.adapter_logits(**a, out_dtype=out_dtype, out=out)
    assert y.dtype == out_dtype and y.shape == (a["x"].shape[0], a["weight"].shape[0])
    want, err = ref.adapter_logits(**a)
    got = y.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), what
    tol = err + ref.rounding(want, out_dtype)
    ok = (got - want).abs() <= tol
    assert (ok | want.isnan()).all(), (what, ((got - want).abs() / tol)[~want.isnan()].max())
    return y


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 130, 300])
def test_rows(ft, dtype, T):
    a = inputs(T, 517, 136, 5, 12, dtype, T)
    for out in (F32, dtype):
        check(ft, a, out, "rows")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("V", [1, 3, 16, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("H", [1, 7, 8, 31, 33, 64, 65, 100, 500, 1024])
def test_vocabulary_and_hidden(ft, dtype, V, H):
    check(ft, inputs(20, V, H, 3, 8, dtype, V * H), F32, "sizes")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("r", [1, 2, 4, 8, 11, 16, 31, 32, 33, 64, 100, 256])
@pytest.mark.parametrize("T", [5, 70])
def test_ranks(ft, dtype, r, T):
    check(ft, inputs(T, 200, 72, 4, r, dtype, r), F32, "rank")


@pytest.mark.parametrize("T,V,H,G,r", [(8, 32768, 512, 4, 8), (84, 20011, 1024, 6, 12),
                                       (16, 40000, 512, 2, 16), (600, 4099, 256, 16, 64),
                                       (1024, 2048, 320, 40, 16)])
@pytest.mark.parametrize("out", ["f32", "same"])
def test_working_sizes(ft, T, V, H, G, r, out):
    a = inputs(T, V, H, G, r, BF16, T)
    check(ft, a, F32 if out == "f32" else BF16, "working size")


@pytest.mark.parametrize("case", ["none", "all", "last", "each_its_own", "outside", "many"])
def test_adapters(ft, case):
    T, G = 100, 100
    adapter = {"none": torch.full((T,), -1), "all": torch.full((T,), 3),
               "last": torch.full((T,), G - 1), "each_its_own": torch.arange(T).flip(0),
               "outside": torch.tensor([-(2 ** 31), -7, -1, 0, G - 1, G, 2 ** 31 - 1] * 14 + [1, 2]),
               "many": torch.arange(T) % 7}[case]
    check(ft, inputs(T, 150, 40, G, 4, BF16, 1, adapter), F32, case)


def test_more_adapters_than_are_sorted(ft):
    adapter = torch.tensor([9000, 3, 9000, -1, 8999, 3, 0, 9001] * 5)
    check(ft, inputs(40, 24, 16, 9001, 2, F16, 2, adapter), F32, "9001 adapters")


def test_no_adapters(ft):
    a = inputs(9, 130, 64, 0, 1, BF16, 3)
    check(ft, a, BF16, "none at all")
    a["adapter"][4] = 0  # out of range
    assert ft.adapter_logits(**a)[4].isnan().all()


def test_values_of_others_stay_out(ft):
    """NaN and infinities of an adapter reach the rows that have it, no other
    row; a row's own infinities stay in it."""
    a = inputs(40, 140, 64, 3, 8, BF16, 4, torch.arange(40) % 3)
    clean = ft.adapter_logits(**a)
    a["up"][1] = math.nan
    a["down"][1] = math.inf
    y = ft.adapter_logits(**a)
    rows = torch.arange(40) % 3 == 1
    assert y[rows.cuda()].isnan().all()
    assert torch.equal(y[~rows.cuda()], clean[~rows.cuda()])
    a = inputs(40, 140, 64, 3, 8, BF16, 4, torch.arange(40) % 3)
    a["x"][7, 5] = math.nan
    y = ft.adapter_logits(**a)
    others = torch.arange(40) != 7
    assert y[7].isnan().all() and torch.equal(y[others.cuda()], clean[others.cuda()])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_range(ft, dtype):
    """An intermediate beyond a 16-bit type's range, and far below it."""
    for f in (3e4, 1e-4):
        a = inputs(20, 100, 64, 2, 8, dtype, 5)
        a["x"] = (a["x"].float() * 30).to(dtype)
        a["scale"] = a["scale"] * f
        a["up"] = (a["up"].float() * 1e-2).to(dtype)
        check(ft, a, F32, f"scale {f}")


def test_strides(ft):
    g = torch.Generator().manual_seed(6)

    def n(*shape):
        return torch.randn(shape, generator=g).to(F16).cuda()

    T, V, H, G, r = 30, 301, 50, 3, 6
    a = dict(x=n(T, H + 13)[:, 3:3 + H], weight=n(2 * V, H + 1)[::2, 1:],
             down=n(r, G, H + 5).transpose(0, 1)[..., 5:], up=n(G, V + 2, r + 3)[:, 1:1 + V, 2:2 + r],
             adapter=torch.randint(-1, G, (2 * T,), generator=g).to(torch.int32).cuda()[::2],
             scale=torch.rand(G, generator=g).cuda())
    check(ft, a, F32, "strided")
    a["x"] = a["x"][:1].expand(T, H)  # one row for all
    check(ft, a, F16, "a broadcast row")
    big = torch.full((T, V + 9), 7.0, device="cuda")
    y = check(ft, a, F32, "into a slice", out=big[:, 4:4 + V])
    assert y.data_ptr() == big[:, 4:].data_ptr()
    assert (big[:, :4] == 7).all() and (big[:, 4 + V:] == 7).all()


def test_repeats(ft):
    a = inputs(150, 900, 256, 9, 16, BF16, 7)
    y = ft.adapter_logits(**a, out_dtype=F32)
    for _ in range(3):
        assert torch.equal(ft.adapter_logits(**a, out_dtype=F32), y)


def test_empty(ft):
    a = inputs(0, 64, 32, 2, 4, BF16, 8)
    assert ft.adapter_logits(**a).shape == (0, 64)


def test_stream_and_graph(ft):
    a = inputs(24, 700, 128, 3, 8, BF16, 9)
    want = ft.adapter_logits(**a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ft.adapter_logits(**a)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ft.adapter_logits(**a)
    for i in range(4):
        b = inputs(24, 700, 128, 3, 8, BF16, 20 + i)
        for k in a:
            a[k].copy_(b[k])
        graph.replay()
        want = ft.adapter_logits(**a)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_refusals(ft):
    a = inputs(4, 20, 16, 2, 4, BF16, 10)
    y = torch.empty(4, 20, device="cuda")
    for change, exc in [(dict(x=a["x"].float()), TypeError), (dict(weight=a["weight"].half()), TypeError),
                        (dict(x=a["x"].cpu()), ValueError), (dict(x=a["x"][0]), ValueError),
                        (dict(weight=a["weight"][:, :8]), ValueError),
                        (dict(down=a["down"][..., :8]), ValueError),
                        (dict(up=a["up"][:1]), ValueError), (dict(up=a["up"][:, :5]), ValueError),
                        (dict(adapter=a["adapter"].long()), TypeError),
                        (dict(adapter=a["adapter"][:3]), ValueError),
                        (dict(scale=a["scale"].double()), TypeError),
                        (dict(scale=a["scale"][:1]), ValueError),
                        (dict(out_dtype=F16), TypeError), (dict(out=y[:, :19]), ValueError),
                        (dict(out=y, out_dtype=BF16), TypeError),
                        (dict(out=y.t().contiguous().t()), ValueError),
                        (dict(out=y[:1].expand(4, 20)), ValueError),
                        (dict(weight=a["weight"].t().contiguous().t()), ValueError)]:
        with pytest.raises(exc):
            ft.adapter_logits(**{**a, **change})
    big = inputs(4, 20, 16, 1, 257, BF16, 11)
    with pytest.raises(ft.MarisaError, match="256"):
        ft.adapter_logits(**big)


def test_rows_that_overlap_past_32_bits(ft):
    """Rows a little apart of hidden columns that reach further: the last
    rows start below 2^32 bytes and end above.  Whole numbers: sums are
    exact."""
    stride, H, V = 65472, 131072, 256
    T = (2 ** 31 - 1) // stride
    assert (T - 1) * stride + 64 < 2 ** 31 < (T - 1) * stride + H
    g = torch.Generator("cuda").manual_seed(8)

    def whole(n):
        return torch.randint(-1, 2, (n,), device="cuda", generator=g, dtype=torch.int8).to(BF16)

    x = whole((T - 1) * stride + H).as_strided((T, H), (stride, 1))
    w = whole(V * H).view(V, H)
    y = ft.adapter_logits(x, w, w[None, :8], w[None, :, :8],
                          torch.full((T,), -1, dtype=torch.int32, device="cuda"),
                          torch.ones(1, device="cuda"), F32)
    for t in (0, T // 2, T - 3, T - 2, T - 1):
        assert torch.equal(y[t].cpu(), w.float().cpu() @ x[t].float().cpu()), t


def test_out_and_autograd(ft):
    """A tensor written through out= has changed for autograd too; one that
    requires a gradient is refused there, as torch's own out= are."""
    a = inputs(4, 20, 16, 2, 4, BF16, 13)
    out = torch.ones(4, 20, device="cuda")
    leaf = torch.ones(4, 20, device="cuda", requires_grad=True)
    product = (leaf * out).sum()  # keeps `out` for its gradient
    ft.adapter_logits(**a, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with pytest.raises(ValueError, match="requires a gradient"):
        ft.adapter_logits(**a, out=leaf)
    with torch.no_grad():
        assert torch.equal(ft.adapter_logits(**a, out=leaf), ft.adapter_logits(**a, out_dtype=F32))


@pytest.mark.parametrize("T,V,H,G,r", [(8, 32768, 512, 4, 8), (84, 20011, 1024, 6, 12),
                                       (16, 40000, 512, 2, 16), (600, 4099, 256, 16, 64),
                                       (1024, 2048, 320, 40, 16)])
@pytest.mark.parametrize("out", ["f32", "same"])
def test_working_sizes_f16(ft, T, V, H, G, r, out):
    a = inputs(T, V, H, G, r, F16, T)
    check(ft, a, F32 if out == "f32" else F16, "working size")


# few rows of a vocabulary past the tiles of 64 tokens
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,V,H,r", [(1, 49153, 512, 8), (16, 49153, 512, 11), (1, 50001, 64, 8),
                                     (16, 50001, 1000, 16), (9, 65537, 192, 64)])
def test_few_rows_large_vocabulary(ft, dtype, T, V, H, r):
    check(ft, inputs(T, V, H, 3, r, dtype, T + V), F32, "few rows")


# one row tile of three stages, from one step of 64 columns to sixteen
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [97, 112, 128])
@pytest.mark.parametrize("H", [64, 128, 192, 256, 1000])
@pytest.mark.parametrize("r", [8, 11, 40])
def test_128_rows(ft, dtype, T, H, r):
    check(ft, inputs(T, 777, H, 4, r, dtype, T + H), F32, "128 rows")


# the tiles of 256 rows by 256 tokens: steps odd and even, the vocabulary's
# last tile on the one before it, ranks of whole vectors and not
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [129, 300, 600])
@pytest.mark.parametrize("V", [256, 257, 4099])
@pytest.mark.parametrize("H,r", [(64, 8), (64, 11), (128, 11), (128, 64), (192, 8), (256, 40)])
def test_large_tiles(ft, dtype, T, V, H, r):
    a = inputs(T, V, H, 5, r, dtype, T + V + H)
    check(ft, a, F32, "large tiles")
    check(ft, a, dtype, "large tiles")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("r", [8, 11])
def test_large_tiles_adapters(ft, dtype, r):
    """Adapters out of range, and one of NaN and infinities, stay in their
    rows."""
    T, V, H = 290, 600, 128
    adapter = torch.arange(T) % 5 - 1
    adapter[[0, 77, 255, 256, 289]] = torch.tensor([4, 2 ** 31 - 1, 9, 4, 5])
    a = inputs(T, V, H, 4, r, dtype, 14, adapter)
    clean = check(ft, a, F32, "out of range")
    a["up"][1] = math.nan
    a["down"][2] = math.inf
    y = ft.adapter_logits(**a, out_dtype=F32)
    sick = ((adapter == 1) | (adapter == 2)).cuda()
    assert y[sick].isnan().all()
    assert torch.equal(y[~sick].nan_to_num(7.0), clean[~sick].nan_to_num(7.0))
