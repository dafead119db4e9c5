"""flashtrie.propose against a plain form in 64 bits: ids exactly (ties to
the lowest id), scores within the bounds of head_reference.py."""

import math

import numpy as np
import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(ft, logits, topk, what):
    print(what, tuple(logits.shape), topk, logits.dtype, flush=True)
    ids, lp = ft.propose(logits, topk)
    assert ids.dtype == torch.int32 and lp.dtype == torch.float32
    wid, wlp, tol = ref.propose(logits, topk)
    got = ids.cpu().numpy()
    assert got.shape == wid.shape and np.array_equal(got, wid), what
    glp = lp.double().cpu().numpy()
    assert np.array_equal(np.isnan(glp), np.isnan(wlp)), what
    same = (glp == wlp) | np.isnan(wlp)
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(glp - wlp) <= tol)).all(), (what, np.nanmax(np.abs(glp - wlp) - tol))
    return ids, lp


def normal(shape, dtype, seed=0, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).to(dtype).cuda()


# vector and group edges, a group per proposal or more, one workgroup of
# groups and several keys a thread
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,K", [(1, 1), (2, 1), (7, 7), (8, 3), (9, 9), (63, 5), (64, 64), (65, 10),
                                 (255, 4), (256, 4), (257, 4), (500, 400), (1000, 1000), (2049, 63),
                                 (4097, 1024), (8191, 32), (32768, 100), (50021, 333),
                                 (140001, 1000), (262147, 4096)])
def test_sizes(ft, dtype, V, K):
    check(ft, normal((2, 3, V), dtype, V), K, "random")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_vocabulary(ft, dtype):
    check(ft, normal((1, 2, 2_200_001), dtype, 1), 1000, "large")


@pytest.mark.parametrize("rows", [(1, 1), (1, 16), (64, 9)])
def test_rows(ft, rows):
    check(ft, normal((*rows, 3001), torch.bfloat16, 2), 17, "rows")


# rows in order, of one value or of few: more candidates than are held at once
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [1, 1000, 4096])
@pytest.mark.parametrize("V", [33000, 300001])
def test_ties_and_order(ft, dtype, V, K):
    g = torch.Generator().manual_seed(V + K)
    up = torch.arange(V, dtype=torch.float32) * 1e-3
    rows = [up, up.flip(0), torch.full((V,), -1.5), torch.randint(0, 2, (V,), generator=g).float(),
            torch.zeros(V), torch.randint(0, 300, (V,), generator=g).float()]
    rows[4][::2] = -0.0  # equal to 0: the lowest ids of either sign
    check(ft, torch.stack(rows)[None].to(dtype).cuda(), K, "ties")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,K", [(40, 12), (5003, 200), (70001, 64)])
def test_masks(ft, dtype, V, K):
    x = normal((1, 9, V), dtype, 3)
    lowest = torch.finfo(dtype).min
    x[0, 0, :] = -math.inf                    # nothing left
    x[0, 1, K - 3:] = -math.inf               # fewer than K left
    x[0, 2, 5:] = lowest                      # masked by the lowest value
    x[0, 3, 1::2] = -math.inf
    x[0, 4, 7] = math.nan                     # the row's scores are NaN
    x[0, 5, 11] = math.inf
    x[0, 6, :] = math.nan
    x[0, 7, :] = lowest
    x[0, 8, :-1] = -math.inf
    check(ft, x, K, "masks")


@pytest.mark.parametrize("shift", [-3e4, 1e4, 6e4])
def test_far_from_zero(ft, shift):
    x = normal((1, 4, 9001), torch.float32, 4) + shift
    check(ft, x, 50, "shifted")


def test_strides(ft):
    big = normal((4, 6, 5010), torch.float16, 5)
    check(ft, big[1:3, ::2, 3:5004], 77, "inner rows at odd addresses")
    check(ft, big[:1, :, 1:4002].expand(3, 6, 4001), 20, "one request for three")
    check(ft, big.transpose(0, 1)[..., :700], 20, "steps before requests")


def test_empty(ft):
    for shape in [(0, 3, 50), (2, 0, 50)]:
        ids, lp = ft.propose(torch.empty(shape, device="cuda"), 5)
        assert ids.shape == lp.shape == (*shape[:2], 5)


def test_stream_and_graph(ft):
    """On another stream, then recorded: every replay on new logits against
    the eager call, with other work between the replays."""
    x = normal((2, 4, 40003), torch.bfloat16, 6)
    want = ft.propose(x, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ft.propose(x, 64)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ft.propose(static, 64)
    for i in range(4):
        static.copy_(normal(x.shape, torch.bfloat16, 10 + i))
        graph.replay()
        want = ft.propose(static, 64)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals(ft):
    x = torch.zeros(1, 2, 100, device="cuda")
    for bad, exc in [(x[0], ValueError), (x.cpu(), ValueError), (x.int(), TypeError),
                     (x.transpose(1, 2), ValueError), (x.double(), TypeError)]:
        with pytest.raises(exc):
            ft.propose(bad, 2)
    for k in (0, -1, 101):
        with pytest.raises(ValueError, match="topk"):
            ft.propose(x, k)
    with pytest.raises(ft.MarisaError, match="4096"):
        ft.propose(torch.zeros(1, 1, 5000, device="cuda"), 4097)
    with pytest.raises(ft.MarisaError, match="2\\^24"):
        ft.propose(torch.zeros(1, 1, (1 << 24) + 1, device="cuda", dtype=torch.float16), 4)
