"""flashtrie.embed exactly and embed_grad within the bounds of
table_reference.py."""

import ctypes as C
import math
import os

import pytest
import torch

import table_reference as ref
import test_table_args as args

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = [F32, F16, BF16]


def normal(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def keys(shape, V, seed, kinds=None):
    """Tokens as keys have them (few at their first positions), some padding
    and some out of range; lengths of which some are 0 or too long."""
    g = torch.Generator().manual_seed(seed)
    kinds = V if kinds is None else kinds
    t = torch.randint(0, kinds, shape, generator=g) * 40503 % V
    t[torch.rand(shape, generator=g) < 0.05] = -1
    n = torch.randint(-1, shape[-1] + 2, shape[:-1], generator=g)
    return t.to(torch.int32).cuda(), n.to(torch.int32).cuda()


def check(ft, grad, tokens, vocab, scale, lengths, what, out=None):
    print(what, tuple(grad.shape), vocab, grad.dtype, flush=True)
    want, tol = ref.embed_grad(grad, tokens, vocab, scale, lengths, out)
    got = ft.embed_grad(grad, tokens, vocab, scale, lengths, out)
    assert got.dtype == grad.dtype and got.shape == (vocab, grad.shape[-1])
    ok = (got.double() - want).abs() <= tol
    assert ok.all(), (what, ((got.double() - want).abs() / tol)[~ok].max().item(), int((~ok).sum()))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [1, 3, 8, 9, 64, 100, 255, 256, 257, 512, 513, 1024, 2050])
@pytest.mark.parametrize("shape", [(1,), (7,), (3, 5), (2, 9, 4)])
def test_embed(ft, dtype, H, shape):
    w = normal((50, H), dtype, H)
    tokens, lengths = keys(shape, 50, H)
    for n in (None, lengths) if len(shape) > 1 else (None,):
        for scale in (1.0, 5.3, -0.25):
            y = ft.embed(tokens, w, scale, n)
            assert y.dtype == dtype and torch.equal(y, ref.embed(tokens, w, scale, n))


def test_embed_odd_tokens(ft):
    w = normal((50, 100), BF16, 1)
    w[7] = math.nan
    tokens = torch.tensor([[7, -1, 50, 49, 0], [-2 ** 31, 2 ** 31 - 1, 7, 3, 3]], dtype=torch.int32).cuda()
    y = ft.embed(tokens, w, math.inf)
    assert y[0, 2].isnan().all() and y[1, 1].isnan().all() and y[0, 0].isnan().all()
    assert not y[0, 1].any() and not y[1, 0].any()
    y = ft.embed(tokens, w, 2.0, torch.tensor([2, 0], dtype=torch.int32).cuda())
    assert y[0, 0].isnan().all() and not y[0, 1:].any() and not y[1].any()


def test_embed_strides(ft):
    wide = normal((60, 300), F16, 2)
    tokens, n = keys((4, 6, 5), 30, 3)
    for w in (wide[::2, 3:104], wide[:30, :256], wide[:1].expand(30, 300)):
        assert torch.equal(ft.embed(tokens, w, 3.0, n), ref.embed(tokens, w, 3.0, n))
    assert torch.equal(ft.embed(tokens.transpose(0, 1), wide), ft.embed(tokens.transpose(0, 1).contiguous(), wide))


def test_embed_far_into_memory(ft):
    w = torch.empty((1 << 23, 520), dtype=BF16, device="cuda")  # past 2^32 elements
    w[-1], w[0], w[1 << 22] = 3.0, 1.0, 2.0
    tokens = torch.tensor([0, 1 << 22, (1 << 23) - 1], dtype=torch.int32).cuda()
    assert ft.embed(tokens, w)[:, 519].tolist() == [1.0, 2.0, 3.0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [1, 5, 8, 64, 100, 512, 520, 1030])
@pytest.mark.parametrize("shape,V,kinds", [((1,), 1, 1), ((9,), 300, 300), ((40, 6), 90, 5),
                                           ((3, 50, 4), 700, 700), ((2, 300, 4), 1000, 3)])
def test_grad_sizes(ft, dtype, H, shape, V, kinds):
    tokens, lengths = keys(shape, V, H + V, kinds)
    g = normal((*shape, H), dtype, H)
    check(ft, g, tokens, V, 1.0, None, "sizes")
    if len(shape) > 1:
        check(ft, g, tokens, V, 3.7, lengths, "lengths")


# around the sizes that one workgroup sorts, and that take longer runs
@pytest.mark.parametrize("n", [7, 8, 9, 64, 1023, 1025, 2047, 2048, 2049, 4097, 16383, 16384, 16385,
                               70001, 140000])
@pytest.mark.parametrize("kinds", [1, 3, 40, 5000])
def test_grad_counts(ft, n, kinds):
    tokens, _ = keys((n,), 5003, n + kinds, kinds)
    check(ft, normal((n, 24), F32, n), tokens, 5003, 0.5, None, "counts")


@pytest.mark.parametrize("V", [1, 2, 255, 511, 512, 513, 65536, 262143, 262144, 300000, 2200001, 1 << 24])
@pytest.mark.parametrize("n", [500, 5000])
def test_grad_vocabularies(ft, V, n):
    """Every number of digits and passes."""
    tokens, _ = keys((n,), V, V % 1000 + n)
    tokens[0], tokens[1], tokens[-1] = V - 1, 0, V - 1
    check(ft, normal((n, 8), BF16, n), tokens, V, 2.0, None, "vocabularies")


@pytest.mark.parametrize("dtype", DTYPES)
def test_grad_working_sizes(ft, dtype):
    for shape, V, H in [((8, 100, 12), 32768, 512), ((128, 1, 13), 50021, 768), ((2, 1000, 16), 262144, 256)]:
        tokens, lengths = keys(shape, V, 5, 3000)
        check(ft, normal((*shape, H), dtype, 6), tokens, V, math.sqrt(H), lengths, "working")


def test_grad_of_one_token(ft):
    """A token at every position, and one at each end of a run."""
    tokens = torch.full((20000,), 3, dtype=torch.int32, device="cuda")
    g = normal((20000, 33), F32, 7)
    check(ft, g, tokens, 5, 1.0, None, "one token")
    tokens = (torch.arange(20000, device="cuda") // 32).to(torch.int32)
    check(ft, g, tokens, 700, 1.0, None, "a run each")
    tokens = ((torch.arange(20000, device="cuda") + 1) // 32).to(torch.int32)
    check(ft, g, tokens, 700, 1.0, None, "across runs")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [100, 5000])
def test_grad_added(ft, dtype, n):
    """Onto what is there; rows of other tokens and what lies beside are left
    alone, NaN among them."""
    big = normal((130, 80), dtype, 8)
    tokens, _ = keys((n,), 50, 9, 20)
    out = big[3:103:2, 5:75]
    there = ref.valid(tokens, None, 50)
    absent = [v for v in range(50) if not (tokens[there] == v).any()]
    out[absent[0]] = math.nan
    before, g = big.clone(), normal((n, 70), dtype, 10)
    want, tol = ref.embed_grad(g, tokens, 50, 0.3, None, out)
    version = out._version
    assert ft.embed_grad(g, tokens, 50, 0.3, out=out) is out and out._version > version
    ok = (out.double() - want).abs() <= tol
    ok[absent] = True
    assert ok.all()
    mask = torch.ones_like(big, dtype=torch.bool)
    rows = [v for v in range(50) if v not in absent]
    mask[3:103:2, 5:75][rows] = False
    same = (big == before) | (big.isnan() & before.isnan())
    assert same[mask].all()


def test_grad_padding_is_not_read(ft):
    tokens, lengths = keys((30, 8), 100, 11)
    tokens[0, 0], tokens[1, 0], lengths[:2] = 100, 2 ** 31 - 1, 8
    g = normal((30, 8, 64), BF16, 12)
    want = ft.embed_grad(g, tokens, 100, 1.0, lengths)
    g[~ref.valid(tokens, lengths, 100)] = math.nan
    assert torch.equal(want, ft.embed_grad(g, tokens, 100, 1.0, lengths))


def test_grad_nan_stays_in_its_token(ft):
    tokens = torch.tensor([1, 2, 3, 2, 1], dtype=torch.int32).cuda()
    g = normal((5, 40), F32, 13)
    g[1, 3], g[4, 5] = math.nan, math.inf
    y = ft.embed_grad(g, tokens, 6)
    assert y[2, 3].isnan() and y[1, 5] == math.inf and int((~y.isfinite()).sum()) == 2


def test_grad_strides(ft):
    wide = normal((12, 10, 6, 200), F16, 14)
    tokens, n = keys((6, 10, 6), 40, 15)
    want = ft.embed_grad(wide[::2, :, :, 7:108].contiguous(), tokens, 40, 1.5, n)
    assert torch.equal(want, ft.embed_grad(wide[::2, :, :, 7:108], tokens, 40, 1.5, n))
    flat = wide.view(-1, 200)[:360, :101]
    assert torch.equal(ft.embed_grad(flat, tokens.view(-1), 40), ft.embed_grad(flat.contiguous(), tokens.view(-1), 40))
    one = wide[0, 0, 0, :50].expand(6, 10, 6, 50)
    check(ft, one, tokens, 40, 1.0, None, "one row for all")


@pytest.mark.parametrize("n", [0, 50, 5000])
@pytest.mark.parametrize("H", [40, 41])
def test_grad_in_wider_rows(ft, n, H):
    """The C call with a gradient in rows of a wider tensor, whose other columns
    stay as they were."""
    lib = C.CDLL(os.path.join(args.ROOT, "flash-trie_amd", "libflashtrie_amd.so"))
    V, big = 300, torch.full((300, 60), 5.0, dtype=F16, device="cuda")
    tokens, _ = keys((n,), V, 25, 40)
    g = normal((n, H), F16, 26)
    s = args.EmbedGrad(device=0, dtype=args.F16, groups=1, steps=n, hidden=H, vocab=V, tokens=tokens.data_ptr(),
                       grad=g.data_ptr(), grad_stride=H, scale=2.0, dtable=big.data_ptr() + 6, dtable_stride=60)
    lib.ft_embed_grad_workspace.restype = C.c_size_t
    size = lib.ft_embed_grad_workspace(C.byref(s))
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.ft_embed_grad(C.byref(s), C.c_void_p(ws.data_ptr()), C.c_size_t(size), stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(big[:, 3:3 + H], ft.embed_grad(g, tokens, V, 2.0))
    assert (big[:, :3] == 5).all() and (big[:, 3 + H:] == 5).all()


def test_grad_repeats(ft):
    tokens, n = keys((8, 500, 8), 3000, 16, 30)
    g = normal((8, 500, 8, 256), BF16, 17)
    want = ft.embed_grad(g, tokens, 3000, 1.0, n)
    for _ in range(3):
        assert torch.equal(want, ft.embed_grad(g, tokens, 3000, 1.0, n))


def test_grad_far_into_memory(ft):
    """A gradient of more than 2^32 elements: its zeros, and its last row."""
    V = (1 << 24) - 3
    g = torch.ones((3, 264), dtype=F16, device="cuda")
    tokens = torch.tensor([V - 1, 5, V - 1], dtype=torch.int32).cuda()
    torch.full((V, 264), math.nan, dtype=F16, device="cuda")  # (what the allocator hands out next)
    y = ft.embed_grad(g, tokens, V)
    assert (y[V - 1] == 2).all() and (y[5] == 1).all()
    y[V - 1], y[5] = 0, 0
    for part in y.split(1 << 22):
        assert not part.any()


def test_empty(ft):
    w = normal((50, 64), F32, 18)
    for shape in [(0,), (0, 4), (3, 0), (2, 0, 4)]:
        t = torch.empty(shape, dtype=torch.int32, device="cuda")
        y = ft.embed(t, w)
        assert y.shape == (*shape, 64)
        g = ft.embed_grad(y, t, 50)
        assert g.shape == (50, 64) and not g.any()
        out = w.clone()
        assert torch.equal(ft.embed_grad(y, t, 50, out=out), w)


def test_stream_and_graph(ft):
    """On another stream; recorded with the lookup, replayed on new keys, two
    calls of one recording side by side."""
    V, shape = 4000, (4, 300, 8)
    w = normal((V, 128), BF16, 19)
    tokens, n = keys(shape, V, 20, 50)
    g = normal((*shape, 128), BF16, 21)
    want = ft.embed(tokens, w, 2.0, n), ft.embed_grad(g, tokens, V, 2.0, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ft.embed(tokens, w, 2.0, n), ft.embed_grad(g, tokens, V, 2.0, n)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    st, sn, few = tokens.clone(), n.clone(), tokens[0, :, 0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ft.embed(st, w, 2.0, sn)
        d = ft.embed_grad(y, st, V, 2.0, sn)
        d2 = ft.embed_grad(y[0, :, 0], few, V)
    for i in range(4):
        t, m = keys(shape, V, 30 + i, 50)
        st.copy_(t), sn.copy_(m), few.copy_(t[0, :, 0])
        graph.replay()
        ey = ft.embed(st, w, 2.0, sn)
        want = ey, ft.embed_grad(ey, st, V, 2.0, sn), ft.embed_grad(ey[0, :, 0], few, V)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip((y, d, d2), want)), i


def test_refusals(ft):
    w, t = normal((50, 64), F32, 22), torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    n = torch.zeros(3, dtype=torch.int32, device="cuda")
    for args, exc in [((t.long(), w), TypeError), ((t.cpu(), w), ValueError), ((t, w[0]), ValueError),
                      ((t, w.double()), TypeError), ((t, w.t()), ValueError), ((t, w, 1.0, n[:2]), ValueError),
                      ((t, w, 1.0, n.long()), TypeError), ((t[0], w, 1.0, n[:1]), ValueError),
                      ((t[None, None], w), ValueError), ((t[0, 0], w), ValueError), ((3, w), TypeError),
                      ((t, w[:0]), ValueError)]:
        with pytest.raises(exc):
            ft.embed(*args)
    g = normal((3, 4, 64), F32, 23)
    out = normal((50, 64), F32, 24)
    for args, exc in [((g, t.long(), 50), TypeError), ((g[0], t, 50), ValueError), ((g[:2], t, 50), ValueError),
                      ((g.double(), t, 50), TypeError), ((g, t, 0), ValueError), ((g, t, -1), ValueError),
                      ((g, t, 50, 1.0, n[:2]), ValueError), ((g, t, 49, 1.0, n, out), ValueError),
                      ((g, t, 50, 1.0, n, out.half()), TypeError), ((g, t, 50, 1.0, n, out[:, :63]), ValueError),
                      ((g, t, 50, 1.0, n, out[:1].expand(50, 64)), ValueError),
                      ((g.transpose(1, 2), t, 50), ValueError), ((g.cpu(), t, 50), ValueError)]:
        with pytest.raises(exc):
            ft.embed_grad(*args)
    with pytest.raises(ValueError, match="gradient"):
        ft.embed_grad(g, t, 50, out=out.clone().requires_grad_())
    with pytest.raises(ft.MarisaError, match="2\\^24"):
        ft.embed_grad(g[..., :1], t, (1 << 24) + 1)
