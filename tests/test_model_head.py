"""The example that runs the model head's operators around the trie search
(flash-trie_amd/run_model_head.py)."""

import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch  # noqa: F401  (before flashtrie: one HIP runtime)

import run_model_head as M


def test_key_arrays():
    tok, length = M.key_arrays([[[5, 6], [7]], [], [[1, 2, 3]]], 3)
    assert tok.dtype == length.dtype == np.int32
    assert tok.tolist() == [[[5, 6, 0], [7, 0, 0]], [[0] * 3] * 2, [[1, 2, 3], [0] * 3]]
    assert length.tolist() == [[2, 1], [0, 0], [3, 0]]
    tok, length = M.key_arrays([[], []], 2)
    assert tok.shape == (2, 1, 2) and not length.any()


def test_rewards():
    tok, length = M.key_arrays([[[5, 6, 7], [5, 9], [5, 6, 7, 8], [0]]], 4)
    r = M.rewards(tok, length, [(5, 6, 7)])
    assert r[0] == pytest.approx([1, 1 / 3, 3 / 4, 0])
    # a padding zero is no token, wanted or not
    assert M.rewards(tok, length, [(5, 9, 0)])[0, 1] == pytest.approx(2 / 3)


@pytest.mark.parametrize("bad", [["--rank", "0"], ["--topk-tokens", "20", "--vocab-size", "10"],
                                 ["--loss", "other"]])
def test_arguments(bad, capsys):
    with pytest.raises(SystemExit):
        M.parse_args(bad)


@pytest.mark.parametrize("order,error,text", [
    ("torch, flashtrie", "ValueError", "must be on the GPU"),
    ("flashtrie, torch", "MarisaError", "import torch first")])
def test_import_order(ft, order, error, text):
    """torch and the module share a HIP runtime when torch comes first; the
    other order is refused before anything is launched."""
    code = (f"import {order}\n"
            "try:\n    flashtrie.propose(torch.zeros(1, 1, 4), 2)\n"
            "except Exception as e:\n    print(type(e).__name__, e)\n")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                         cwd=os.path.dirname(M.__file__), check=True).stdout
    assert out.startswith(error) and text in out, out


@pytest.mark.gpu
@pytest.mark.parametrize("loss,dtype", [("policy", "bfloat16"), ("preference", "float16")])
def test_rounds(ft, loss, dtype):
    """An update lowers the loss that it follows, on the same keys."""
    args = M.parse_args(["--requests", "6", "--num-keys", "3000", "--vocab-size", "1111",
                         "--hidden", "96", "--rank", "5", "--rounds", "8", "--loss", loss,
                         "--dtype", dtype, "--lr", "1e-2"])
    lines = M.run(args, log=lambda *_: None)
    assert len(lines) == 8
    for x in lines:
        assert x["keys"] > 6 and all(math.isfinite(v) for v in x["losses"])
        assert x["losses"][1] < x["losses"][0]
    if loss == "preference":
        # no adapter's change yet: every margin is zero
        assert lines[0]["losses"][0] == pytest.approx(math.log(2), rel=1e-5)


@pytest.mark.gpu
def test_adapter_gradients(ft):
    """The adapters' gradients against autograd on the plain form, 64 bits."""
    args = M.parse_args(["--vocab-size", "77", "--hidden", "40", "--adapters", "3", "--rank", "6",
                         "--topk-tokens", "5"])
    head = M.Head(args, torch, ft)
    with torch.no_grad():
        head.up.copy_(head.noise(*head.up.shape))
    x = head.noise(13, 40).to(head.dtype)
    adapter = torch.tensor([0, 2, -1, 0, 2, 2, 0, -1, 0, 0, 2, 2, 0], dtype=torch.int32)
    d = head.noise(13, 77)
    down, up = (t.detach().double().cpu().requires_grad_() for t in (head.down, head.up))
    plain, scale = x.double().cpu(), head.scale.double().cpu()

    def total(down, up, x, d):
        return sum((scale[g] * (up[g] @ (down[g] @ x[t])) * d[t]).sum()
                   for t, g in enumerate(adapter.tolist()) if g >= 0)

    total(down, up, plain, d.double().cpu()).backward()
    want = [down.grad, up.grad]
    mags = [t.detach().abs().requires_grad_() for t in (down, up)]
    total(*mags, plain.abs(), d.double().cpu().abs()).backward()
    head.step(x, adapter.cuda(), d)
    for got, w, m in zip((head.down.grad, head.up.grad), want, mags):
        # two sums of at most 77 products each, the scale and the result's rounding
        assert ((got.double().cpu() - w).abs() <= 2 * 80 * 2.0 ** -24 * m.grad).all()
    assert not head.down.grad[1].any() and not head.up.grad[1].any()


@pytest.mark.gpu
def test_same_seed_same_rounds(ft):
    args = M.parse_args(["--requests", "3", "--num-keys", "500", "--vocab-size", "300",
                         "--hidden", "64", "--rounds", "2"])
    runs = [M.run(args, log=lambda *_: None) for _ in range(2)]
    assert runs[0][0]["losses"][0] == runs[1][0]["losses"][0]
    assert [x["keys"] for x in runs[0]] == [x["keys"] for x in runs[1]]


@pytest.mark.gpu
def test_an_error_of_another_call(ft):
    """An error that an earlier call of the application left with the HIP
    runtime is not taken for a launch's."""
    import ctypes
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    x = torch.randn(2, 3, 50000, device="cuda")
    h = torch.randn(20, 64, device="cuda").bfloat16()
    none = torch.full((20,), -1, dtype=torch.int32, device="cuda")
    tok = torch.zeros(2, 4, 3, dtype=torch.int32, device="cuda")
    one, old = torch.ones(2, 4, device="cuda"), torch.zeros(2, 4, 3, device="cuda")
    length = torch.full((2, 4), 3, dtype=torch.int32, device="cuda")
    pairs = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    calls = [lambda: ft.propose(x, 5), lambda: ft.propose(x[..., :100], 5),
             lambda: (ft.adapter_logits(h, h, h[None, :4], h[None, :, :4], none, one[0, :1]),),
             lambda: ft.policy_loss(x, tok, length, old, one, one),
             lambda: ft.preference_loss(x, tok, length, pairs, one, one[0, :1])]
    for call in calls:
        want = call()
        assert hip.hipSetDevice(1 << 20) != 0  # no such device
        try:
            got = call()
        finally:
            hip.hipGetLastError()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
