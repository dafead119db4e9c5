"""The model head's C ABI (include/flashtrie_amd.h) without a GPU: the
argument structs' layout, what is refused and with which code, workspace
sizes.  Nothing here reaches a launch: a valid call ends at the device."""

import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import yaml

import build as ftbuild  # flash-trie_amd/build.py

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "flashtrie_amd.h")
F32, F16, BF16 = 0, 1, 2
E_ARG, E_LIMIT = -1, -4
P, I32, U32, I64, U64, F = C.c_void_p, C.c_int, C.c_uint32, C.c_int64, C.c_uint64, C.c_float


def struct(name, *fields):
    return type(name, (C.Structure,), {"_fields_": list(fields)})


Logits = struct("ft_adapter_logits_args", ("device", I32), ("dtype", I32), ("out_dtype", I32),
                ("rows", U64), ("hidden", U32), ("vocab", U32), ("adapters", U32), ("rank", U32),
                ("x", P), ("x_stride", I64), ("weight", P), ("weight_stride", I64), ("down", P),
                ("down_stride", I64 * 2), ("up", P), ("up_stride", I64 * 2), ("adapter", P),
                ("scale", P), ("out", P), ("out_stride", I64))
Propose = struct("ft_propose_args", ("device", I32), ("dtype", I32), ("batch", U64),
                 ("steps", U64), ("vocab", U32), ("topk", U32), ("logits", P),
                 ("stride", I64 * 2), ("ids", P), ("logp", P))
Keys = struct("ft_keys", ("device", I32), ("dtype", I32), ("batch", U64), ("steps", U64),
              ("vocab", U32), ("keys", U32), ("logits", P), ("stride", I64 * 2), ("tokens", P),
              ("lengths", P), ("logp", P), ("loss", P), ("dlogits", P), ("dstride", I64 * 2))
Policy = struct("ft_policy_loss_args", ("k", Keys), ("old_logp", P), ("ref_logp", P),
                ("advantage", P), ("weight", P), ("clip_low", F), ("clip_high", F),
                ("kl_coef", F))
Preference = struct("ft_preference_loss_args", ("k", Keys), ("pairs", U64), ("pair", P),
                    ("ref_logp", P), ("weight", P), ("beta", F), ("smoothing", F))
ANY = 1 << 20   # stands for device memory; refused calls do not look at it


def logits(**kw):
    a = Logits(device=0, dtype=BF16, out_dtype=F32, rows=4, hidden=64, vocab=100, adapters=2,
               rank=8, x=ANY, x_stride=64, weight=ANY, weight_stride=64, down=ANY, up=ANY,
               adapter=ANY, scale=ANY, out=ANY, out_stride=100)
    a.down_stride[:] = [8 * 64, 64]
    a.up_stride[:] = [100 * 8, 8]
    return change(a, kw)


def propose(**kw):
    a = Propose(device=0, dtype=F32, batch=2, steps=3, vocab=100, topk=5, logits=ANY, ids=ANY,
                logp=ANY)
    a.stride[:] = [300, 100]
    return change(a, kw)


def keys(a, kw):
    a.k = Keys(device=0, dtype=F32, batch=2, steps=3, vocab=100, keys=4, logits=ANY, tokens=ANY,
               lengths=ANY, logp=ANY, loss=ANY, dlogits=ANY)
    a.k.stride[:] = a.k.dstride[:] = [300, 100]
    change(a.k, {n: v for n, v in kw.items() if hasattr(a.k, n)})
    return change(a, {n: v for n, v in kw.items() if not hasattr(a.k, n)})


def policy(**kw):
    return keys(Policy(old_logp=ANY, ref_logp=ANY, advantage=ANY, weight=ANY, clip_low=0.2,
                       clip_high=0.2, kl_coef=0.1), kw)


def preference(**kw):
    return keys(Preference(pairs=3, pair=ANY, ref_logp=ANY, weight=ANY, beta=0.1), kw)


def change(a, kw):
    for n, v in kw.items():
        if isinstance(v, list):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


@pytest.fixture(scope="module")
def lib(ft):
    lib = C.CDLL(os.path.join(ROOT, "flash-trie_amd", "libflashtrie_amd.so"))
    lib.ft_last_error.restype = C.c_char_p
    for n in ("adapter_logits", "propose", "policy_loss", "preference_loss"):
        getattr(lib, f"ft_{n}_workspace").restype = C.c_size_t
        getattr(lib, f"ft_{n}").argtypes = [P, P, C.c_size_t, P]
    return lib


CALLS = {"adapter_logits": logits, "propose": propose, "policy_loss": policy,
         "preference_loss": preference}


def call(lib, name, a, workspace=ANY, size=1 << 62):
    need = getattr(lib, f"ft_{name}_workspace")(C.byref(a))
    rc = getattr(lib, f"ft_{name}")(C.byref(a), workspace, size, None)
    return rc, need, lib.ft_last_error().decode()


def test_layouts(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    structs = [Logits, Propose, Keys, Policy, Preference]
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
    ("adapter_logits", dict(dtype=F32), E_ARG, "float16 or bfloat16"),
    ("adapter_logits", dict(dtype=9), E_ARG, "float16 or bfloat16"),
    ("adapter_logits", dict(out_dtype=F16), E_ARG, "inputs' type"),
    ("adapter_logits", dict(hidden=0), E_ARG, "at least 1"),
    ("adapter_logits", dict(vocab=0), E_ARG, "at least 1"),
    ("adapter_logits", dict(rank=0), E_ARG, "rank must be at least 1"),
    ("adapter_logits", dict(rank=257), E_LIMIT, "256"),
    ("adapter_logits", dict(vocab=(1 << 24) + 1), E_LIMIT, "2^24"),
    ("adapter_logits", dict(hidden=(1 << 24) + 1), E_LIMIT, "2^24"),
    ("adapter_logits", dict(adapters=(1 << 31) - 1), E_LIMIT, ""),
    ("adapter_logits", dict(rows=1 << 40), E_LIMIT, "rows"),
    ("adapter_logits", dict(rows=(1 << 64) - 1), E_LIMIT, "rows"),
    ("adapter_logits", dict(rows=1 << 20, vocab=1 << 24, out_stride=1 << 24), E_LIMIT, "rows"),
    ("adapter_logits", dict(out_stride=99), E_ARG, "overlap"),
    ("adapter_logits", dict(out_stride=-100), E_ARG, "overlap"),
    *[("adapter_logits", {n: None}, E_ARG, "null pointer")
      for n in ("x", "weight", "down", "up", "adapter", "scale", "out")],
    ("propose", dict(dtype=-1), E_ARG, "float32, float16 or bfloat16"),
    ("propose", dict(topk=0), E_ARG, "topk"),
    ("propose", dict(topk=101), E_ARG, "topk"),
    ("propose", dict(vocab=0, topk=0), E_ARG, "topk"),
    ("propose", dict(vocab=5000, topk=4097), E_LIMIT, "4096"),
    ("propose", dict(vocab=(1 << 24) + 1), E_LIMIT, "2^24"),
    ("propose", dict(batch=1 << 40), E_LIMIT, "rows"),
    ("propose", dict(batch=1 << 33, steps=1 << 33), E_LIMIT, "rows"),
    *[("propose", {n: None}, E_ARG, "null pointer") for n in ("logits", "ids", "logp")],
    *[(c, kw, code, text) for c in ("policy_loss", "preference_loss") for kw, code, text in [
        (dict(dtype=3), E_ARG, "float32, float16 or bfloat16"),
        (dict(vocab=0), E_ARG, "at least 1"),
        (dict(steps=0), E_ARG, "at least 1"),
        (dict(keys=0), E_ARG, "at least 1"),
        (dict(keys=4097), E_LIMIT, "4096"),
        (dict(vocab=(1 << 24) + 1), E_LIMIT, "2^24"),
        (dict(batch=1 << 62), E_LIMIT, "rows"),
        (dict(batch=1 << 18, keys=4096), E_LIMIT, "rows"),
        (dict(dstride=[300, 99]), E_ARG, "overlap"),
        (dict(dstride=[299, 100]), E_ARG, "overlap"),
        *[({n: None}, E_ARG, "null pointer")
          for n in ("logits", "tokens", "lengths", "logp", "loss", "weight")]]],
    ("policy_loss", dict(clip_low=-0.1), E_ARG, "clip_low"),
    ("policy_loss", dict(clip_low=1.1), E_ARG, "clip_low"),
    ("policy_loss", dict(clip_low=float("nan")), E_ARG, "clip_low"),
    ("policy_loss", dict(clip_high=-0.1), E_ARG, "clip_high"),
    ("policy_loss", dict(clip_high=float("inf")), E_ARG, "clip_high"),
    ("policy_loss", dict(kl_coef=float("nan")), E_ARG, "kl_coef"),
    ("policy_loss", dict(ref_logp=None), E_ARG, "ref_logp"),
    *[("policy_loss", {n: None}, E_ARG, "null pointer") for n in ("old_logp", "advantage")],
    ("preference_loss", dict(beta=float("inf")), E_ARG, "beta"),
    ("preference_loss", dict(smoothing=-0.1), E_ARG, "smoothing"),
    ("preference_loss", dict(smoothing=float("nan")), E_ARG, "smoothing"),
    ("preference_loss", dict(batch=0), E_ARG, "pairs of no keys"),
    ("preference_loss", dict(pairs=1 << 40), E_LIMIT, "pairs"),
    *[("preference_loss", {n: None}, E_ARG, "null pointer") for n in ("pair", "ref_logp")],
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


# a call of each operator that needs a workspace
NEEDS = {"adapter_logits": {}, "propose": dict(vocab=300000, stride=[900000, 300000]),
         "policy_loss": {}, "preference_loss": {}}


@pytest.mark.parametrize("name", CALLS)
def test_workspace(lib, name):
    a = CALLS[name](**NEEDS[name])
    rc, need, message = call(lib, name, a, workspace=None)
    assert need > 0 and rc == E_ARG and "workspace" in message
    rc, _, message = call(lib, name, a, workspace=ANY + 16)
    assert rc == E_ARG and "256-byte aligned" in message
    rc, _, message = call(lib, name, a, size=need - 1)
    assert rc == E_LIMIT and "too small" in message


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("device", [-1, 64, 1000])
def test_devices(lib, name, device):
    a = CALLS[name]()
    (a.k if hasattr(a, "k") else a).device = device
    rc, _, message = call(lib, name, a)
    assert rc < 0 and rc not in (E_ARG, E_LIMIT) and "device" in message


def test_workspaces_grow_with_the_work(lib):
    """Per-row parts only: no copy of the logits or the weight."""
    size = lambda a, n: getattr(lib, f"ft_{n}_workspace")(C.byref(a))  # noqa: E731
    few, many = (size(policy(batch=b), "policy_loss") for b in (2, 2000))
    assert few < many < 2000 * 3 * 100 * 4 + few
    rank = [size(logits(rows=1000, rank=r), "adapter_logits") for r in (8, 256)]
    assert rank[0] < rank[1] < 1000 * 256 * 8 + (1 << 20)


@pytest.fixture(scope="module")
def resources(tmp_path_factory):
    """{kernel: its metadata} of the operators' kernels, as hipcc makes them
    for gfx950."""
    if not (os.path.exists(ftbuild.HIPCC) or shutil.which("hipcc")):
        pytest.skip("no hipcc")
    found = {}
    for name in ("adapter_logits", "propose", "key_loss"):
        out = tmp_path_factory.mktemp("k") / "k.s"
        subprocess.run([ftbuild.HIPCC] + ftbuild.HIP_FLAGS +
                       ["-x", "hip", "--offload-device-only", "-S", "-o", str(out),
                        os.path.join(ftbuild.CSRC, name + ".hip")],
                       check=True, capture_output=True, text=True)
        meta = re.search(r"\.amdgpu_metadata\n(.*?)\n\s*\.end_amdgpu_metadata",
                         out.read_text(), re.S).group(1)
        for k in yaml.safe_load(meta)["amdhsa.kernels"]:
            found[k[".name"]] = k
    return found


def test_kernel_resources(resources):
    """No scratch memory, which the runtime would allocate at a launch: a call
    allocates nothing."""
    assert len(resources) > 10
    for name, k in resources.items():
        assert not k.get(".uses_dynamic_stack", False), name
        assert k[".group_segment_fixed_size"] <= 160 * 1024, name
        assert k[".vgpr_spill_count"] == k[".private_segment_fixed_size"] == 0, name


# the most that the launches' thread counts (32 bits) allow, and one more
@pytest.mark.parametrize("name,most,more,text", [
    ("adapter_logits", dict(rows=(1 << 26) - 16), dict(rows=(1 << 26) - 15), "rows"),
    # 2^17 tiles of tokens by fewer than 2^5 of 256 rows
    ("adapter_logits", dict(rows=31 * 256, vocab=1 << 24, out_stride=1 << 24),
     dict(rows=31 * 256 + 1, vocab=1 << 24, out_stride=1 << 24), "rows"),
    # 2^14 tiles of 64 rows by fewer than 2^10 of 128 tokens
    ("adapter_logits", dict(rows=1 << 20, vocab=1023 * 128, out_stride=1023 * 128),
     dict(rows=1 << 20, vocab=1023 * 128 + 1, out_stride=1 << 17), "rows"),
    ("preference_loss", dict(batch=65535, steps=1, keys=4096),
     dict(batch=65536, steps=1, keys=4096), "keys"),
    *[(n, dict(batch=4095, steps=1, vocab=1 << 24, stride=[1 << 24] * 2, dstride=[1 << 24] * 2),
       dict(batch=4096, steps=1, vocab=1 << 24, stride=[1 << 24] * 2, dstride=[1 << 24] * 2), "rows")
      for n in ("policy_loss", "preference_loss")],
])
def test_launch_limits(lib, name, most, more, text):
    need = getattr(lib, f"ft_{name}_workspace")(C.byref(CALLS[name](**most)))
    assert need > 0
    rc, need, message = call(lib, name, CALLS[name](**more))
    assert (rc, need) == (E_LIMIT, 0) and text in message
    if name == "policy_loss":  # without the gradient there is no such launch
        a = CALLS[name](**more, dlogits=None)
        assert getattr(lib, f"ft_{name}_workspace")(C.byref(a)) > 0


def test_too_many_adapters(lib):
    rc, need, message = call(lib, "adapter_logits", logits(adapters=(1 << 31) - 1))
    assert (rc, need) == (E_LIMIT, 0) and message.endswith("too many adapters")
