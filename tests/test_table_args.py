"""The C ABI of the vocabulary table's operators (include/flashtrie_amd.h)
without a GPU: the argument structs' layout, what is refused and with which
code, workspace sizes, the kernels' resources.  Nothing here reaches a launch:
a valid call ends at the device."""

import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import yaml

import build as ftbuild  # flash-trie_amd/build.py
from test_lds_copies_codegen import unwaited
from test_operator_args import (ANY, BF16, E_ARG, E_LIMIT, F, F16, F32, HEADER, I32, I64, P, ROOT,
                                U32, U64, change, struct)

CrossEntropy = struct(
    "ft_cross_entropy_loss_args", ("device", I32), ("dtype", I32), ("rows", U64), ("hidden", U32),
    ("vocab", U32), ("x", P), ("x_stride", I64), ("weight", P), ("weight_stride", I64),
    ("target", P), ("row_weight", P), ("smoothing", F), ("loss", P), ("logp", P), ("dx", P),
    ("dx_stride", I64), ("dweight", P), ("dweight_stride", I64))
Pack = struct("ft_pack_weight_args", ("device", I32), ("dtype", I32), ("hidden", U32),
              ("vocab", U32), ("group", U32), ("weight", P), ("weight_stride", I64), ("packed", P),
              ("scales", P))
Packed = struct("ft_packed_logits_args", ("device", I32), ("dtype", I32), ("out_dtype", I32),
                ("rows", U64), ("hidden", U32), ("vocab", U32), ("group", U32), ("x", P),
                ("x_stride", I64), ("packed", P), ("scales", P), ("out", P), ("out_stride", I64))
Embed = struct("ft_embed_args", ("device", I32), ("dtype", I32), ("groups", U64), ("steps", U64),
               ("hidden", U32), ("vocab", U32), ("tokens", P), ("lengths", P), ("table", P),
               ("table_stride", I64), ("scale", F), ("out", P))
EmbedGrad = struct("ft_embed_grad_args", ("device", I32), ("dtype", I32), ("groups", U64),
                   ("steps", U64), ("hidden", U32), ("vocab", U32), ("tokens", P), ("lengths", P),
                   ("grad", P), ("grad_stride", I64), ("scale", F), ("add", I32), ("dtable", P),
                   ("dtable_stride", I64))


def cross_entropy(**kw):
    return change(CrossEntropy(
        device=0, dtype=BF16, rows=70, hidden=64, vocab=1000, x=ANY, x_stride=64, weight=ANY,
        weight_stride=64, target=ANY, row_weight=ANY, loss=ANY, logp=ANY, dx=ANY, dx_stride=64,
        dweight=ANY, dweight_stride=64), kw)


def pack(**kw):
    return change(Pack(device=0, dtype=F16, hidden=64, vocab=100, group=32, weight=ANY,
                       weight_stride=64, packed=ANY, scales=ANY), kw)


def packed(**kw):
    return change(Packed(device=0, dtype=F16, out_dtype=F32, rows=4, hidden=64, vocab=100,
                         group=32, x=ANY, x_stride=64, packed=ANY, scales=ANY, out=ANY,
                         out_stride=100), kw)


def embed(**kw):
    return change(Embed(device=0, dtype=F32, groups=3, steps=4, hidden=64, vocab=100, tokens=ANY,
                        lengths=ANY, table=ANY, table_stride=64, scale=1.0, out=ANY), kw)


def embed_grad(**kw):
    return change(EmbedGrad(device=0, dtype=F32, groups=3, steps=4, hidden=64, vocab=100,
                            tokens=ANY, lengths=ANY, grad=ANY, grad_stride=64, scale=1.0,
                            dtable=ANY, dtable_stride=64), kw)


CALLS = {"cross_entropy_loss": cross_entropy, "pack_weight": pack, "packed_logits": packed,
         "embed": embed, "embed_grad": embed_grad}


@pytest.fixture(scope="module")
def lib(ft):
    lib = C.CDLL(os.path.join(ROOT, "flash-trie_amd", "libflashtrie_amd.so"))
    lib.ft_last_error.restype = C.c_char_p
    for n in CALLS:
        getattr(lib, f"ft_{n}_workspace").restype = C.c_size_t
        getattr(lib, f"ft_{n}").argtypes = [P, P, C.c_size_t, P]
    return lib


def need_of(lib, name, a):
    return getattr(lib, f"ft_{name}_workspace")(C.byref(a))


def call(lib, name, a, workspace=ANY, size=1 << 62):
    rc = getattr(lib, f"ft_{name}")(C.byref(a), workspace, size, None)
    return rc, need_of(lib, name, a), lib.ft_last_error().decode()


def test_layouts(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    structs = [CrossEntropy, Pack, Packed, Embed, EmbedGrad]
    lines = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{HEADER}"', "int main(void) {"]
    for s in structs:
        lines.append(f'printf("%zu\\n", sizeof({s.__name__}));')
        lines += [f'printf("%zu\\n", offsetof({s.__name__}, {n}));' for n, _ in s._fields_]
    src = tmp_path / "l.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-o", tmp_path / "l", src], check=True)
    got = subprocess.run([tmp_path / "l"], check=True, capture_output=True, text=True).stdout
    want = []
    for s in structs:
        want += [C.sizeof(s)] + [getattr(s, n).offset for n, _ in s._fields_]
    assert [int(x) for x in got.split()] == want


REFUSED = [
    *[("cross_entropy_loss", kw, code, text) for kw, code, text in [
        (dict(dtype=F32), E_ARG, "float16 or bfloat16"),
        (dict(dtype=7), E_ARG, "float16 or bfloat16"),
        (dict(smoothing=-0.1), E_ARG, "smoothing"),
        (dict(smoothing=1.5), E_ARG, "smoothing"),
        (dict(smoothing=float("nan")), E_ARG, "smoothing"),
        (dict(rows=(1 << 22) + 1), E_LIMIT, "rows"),
        (dict(rows=(1 << 64) - 1), E_LIMIT, "rows"),
        (dict(rows=1 << 22, vocab=1 << 24), E_LIMIT, "rows"),
        (dict(dx_stride=63), E_ARG, "overlap"),
        (dict(dx_stride=-64), E_ARG, "overlap"),
        (dict(dweight_stride=63), E_ARG, "overlap"),
        *[({n: None}, E_ARG, "null pointer")
          for n in ("x", "weight", "target", "row_weight", "loss", "logp")]]],
    *[(c, kw, code, text) for c in ("pack_weight", "packed_logits") for kw, code, text in [
        (dict(dtype=F32), E_ARG, "float16 or bfloat16"),
        (dict(group=0), E_ARG, "group"),
        (dict(group=16), E_ARG, "group"),
        (dict(group=256), E_ARG, "group"),
        (dict(packed=ANY + 8), E_ARG, "aligned"),
        (dict(scales=ANY + 2), E_ARG, "aligned"),
        (dict(vocab=1 << 24, hidden=1 << 16, out_stride=1 << 24) if c == "packed_logits" else
         dict(vocab=1 << 24, hidden=1 << 16), E_LIMIT, "too large"),
        (dict(packed=None), E_ARG, "null pointer"),
        (dict(scales=None), E_ARG, "null pointer")]],
    ("pack_weight", dict(weight=None), E_ARG, "null pointer"),
    ("packed_logits", dict(out_dtype=BF16), E_ARG, "x's type"),
    ("packed_logits", dict(rows=(1 << 22) + 1), E_LIMIT, "rows"),
    ("packed_logits", dict(out_stride=99), E_ARG, "overlap"),
    ("packed_logits", dict(x=None), E_ARG, "null pointer"),
    ("packed_logits", dict(out=None), E_ARG, "null pointer"),
    *[(c, kw, code, text) for c in ("embed", "embed_grad") for kw, code, text in [
        (dict(dtype=3), E_ARG, "float32, float16 or bfloat16"),
        (dict(groups=1 << 62, steps=4), E_LIMIT, "tokens"),
        (dict(groups=1 << 33, steps=1 << 33), E_LIMIT, "tokens"),
        (dict(groups=(1 << 27) + 1, steps=1), E_LIMIT, "tokens"),
        (dict(groups=1 << 27, steps=1, hidden=1 << 16), E_LIMIT, "tokens"),
        (dict(tokens=None), E_ARG, "null pointer")]],
    ("embed", dict(table=None), E_ARG, "null pointer"),
    ("embed", dict(out=None), E_ARG, "null pointer"),
    ("embed_grad", dict(grad=None), E_ARG, "null pointer"),
    ("embed_grad", dict(dtable=None), E_ARG, "null pointer"),
    ("embed_grad", dict(dtable_stride=63), E_ARG, "overlap"),
    ("embed_grad", dict(dtable_stride=0), E_ARG, "overlap"),
    *[(c, kw, code, text) for c in CALLS for kw, code, text in [
        (dict(hidden=0), E_ARG, "at least 1"),
        (dict(vocab=0), E_ARG, "at least 1"),
        (dict(vocab=(1 << 24) + 1), E_LIMIT, "2^24"),
        (dict(hidden=(1 << 16) + 1), E_LIMIT, "2^16")]],
]


@pytest.mark.parametrize("name,kw,code,text", REFUSED)
def test_refused(lib, name, kw, code, text):
    rc, need, message = call(lib, name, CALLS[name](**kw))
    assert (rc, need) == (code, 0)
    assert message.startswith(f"ft_{name}: ") and text in message


@pytest.mark.parametrize("name", CALLS)
def test_null_arguments(lib, name):
    assert getattr(lib, f"ft_{name}_workspace")(None) == 0
    assert getattr(lib, f"ft_{name}")(None, None, 0, None) == E_ARG
    assert b"null arguments" in lib.ft_last_error()


@pytest.mark.parametrize("name", ["cross_entropy_loss", "packed_logits", "embed_grad"])
def test_workspace(lib, name):
    # (packed_logits: of more columns than a workgroup's LDS holds)
    a = CALLS[name](**(dict(hidden=5000) if name == "packed_logits" else {}))
    rc, need, message = call(lib, name, a, workspace=None)
    assert need > 0 and rc == E_ARG and "workspace" in message
    rc, _, message = call(lib, name, a, workspace=ANY + 16)
    assert rc == E_ARG and "256-byte aligned" in message
    rc, _, message = call(lib, name, a, size=need - 1)
    assert rc == E_LIMIT and "too small" in message


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("device", [-1, 64, 1000])
def test_devices(lib, name, device):
    rc, _, message = call(lib, name, CALLS[name](device=device))
    assert rc < 0 and rc not in (E_ARG, E_LIMIT) and "device" in message


def test_no_logits_are_kept(lib):
    """4096 rows by 262,144 tokens take 4 GB as float32 logits."""
    a = dict(rows=4096, vocab=262144, hidden=1024, x_stride=1024, weight_stride=1024,
             dx_stride=1024, dweight_stride=1024)
    assert need_of(lib, "cross_entropy_loss", cross_entropy(**a)) < 400 << 20
    no_table = need_of(lib, "cross_entropy_loss", cross_entropy(**a, dweight=None))
    alone = need_of(lib, "cross_entropy_loss", cross_entropy(**a, dweight=None, dx=None))
    assert alone < no_table < 400 << 20 and alone < 200 << 20


def test_workspaces_of_the_largest(lib):
    """Sizes near the limits do not wrap round."""
    big = need_of(lib, "cross_entropy_loss",
                  cross_entropy(rows=1 << 22, vocab=16384, hidden=4096, x_stride=4096,
                                weight_stride=4096, dx_stride=4096, dweight_stride=4096))
    assert big > (1 << 22) * 4096 * 6
    assert need_of(lib, "packed_logits", packed(rows=1 << 22, hidden=8192)) >= (1 << 22) * 8192 * 2
    n = need_of(lib, "embed_grad", embed_grad(groups=1 << 24, steps=8, hidden=256, grad_stride=256, dtable_stride=256))
    assert n >= (1 << 27) * 16 + 2 * (1 << 22) * 256 * 4


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    if not (os.path.exists(ftbuild.HIPCC) or shutil.which("hipcc")):
        pytest.skip("no hipcc")
    found = {}
    for name in ("cross_entropy", "packed_logits", "embed"):
        out = tmp_path_factory.mktemp("k") / "k.s"
        subprocess.run([ftbuild.HIPCC] + ftbuild.HIP_FLAGS +
                       ["-x", "hip", "--offload-device-only", "-S", "-o", str(out),
                        os.path.join(ftbuild.CSRC, name + ".hip")],
                       check=True, capture_output=True, text=True)
        found[name] = out.read_text()
    return found


@pytest.mark.parametrize("name", ["cross_entropy", "packed_logits", "embed"])
def test_kernel_resources(listings, name):
    """No scratch memory, which the runtime would allocate at a launch: a call
    allocates nothing."""
    meta = re.search(r"\.amdgpu_metadata\n(.*?)\n\s*\.end_amdgpu_metadata", listings[name], re.S).group(1)
    kernels = yaml.safe_load(meta)["amdhsa.kernels"]
    assert len(kernels) > 5
    for k in kernels:
        assert not k.get(".uses_dynamic_stack", False), k[".name"]
        assert k[".group_segment_fixed_size"] <= 160 * 1024, k[".name"]
        assert k[".vgpr_spill_count"] == k[".private_segment_fixed_size"] == 0, k[".name"]


@pytest.mark.parametrize("name", ["cross_entropy", "packed_logits", "embed"])
def test_copies_are_waited_for(listings, name):
    """A copy from memory straight to LDS counts as a load of its wave: between
    it and the next barrier stands a wait for loads."""
    for kernel, (_, bare) in unwaited(listings[name]).items():
        assert bare == 0, kernel
