"""adapter_logits copies operands from memory straight to LDS, where other
waves read them.  Such a copy counts as a load of its wave (vmcnt), which a
barrier does not wait for by itself: the wave that copied has to wait before
the barrier past which the copies are read.  This checks the instructions that
hipcc makes for gfx950 (CPU only: it cross-compiles): between a copy and the
next barrier stands a wait for loads."""

import os
import re
import shutil
import subprocess

import pytest

import build as ftbuild  # flash-trie_amd/build.py

COPY = re.compile(r"global_load_lds_|buffer_load_\w+ .*\blds\b")


def unwaited(listing):
    """(barriers behind copies, those of them without a wait for loads
    between) of each kernel of an assembly listing."""
    found, name = {}, None
    for line in listing.splitlines():
        m = re.match(r"(_Z\w+):", line)
        if m:
            name, copied, waited = m.group(1), False, False
            found[name] = [0, 0]
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            op = line.strip()
            if COPY.match(op):
                copied, waited = True, False
            elif op.startswith("s_waitcnt") and "vmcnt(" in op:
                waited = True
            elif op.startswith("s_barrier"):
                found[name][0] += copied
                found[name][1] += copied and not waited
                copied = waited = False
    return found


def test_the_check():
    copy, wait = "\tglobal_load_lds_dwordx4 v[0:1], off", "\ts_waitcnt vmcnt(0) lgkmcnt(0)"
    for lines, want in [([copy, wait, "\ts_barrier"], [1, 0]), ([copy, "\ts_barrier"], [1, 1]),
                        ([copy, "\ts_waitcnt lgkmcnt(0)", "\ts_barrier"], [1, 1]),
                        ([wait, copy, "\ts_barrier", "\ts_barrier"], [1, 1]),
                        (["\tbuffer_load_dwordx4 v3, s[4:7], s9 offen lds", wait, copy,
                          "\ts_barrier"], [1, 1]),
                        (["\tbuffer_load_dwordx4 v[0:3], v4, s[4:7], 0 offen", "\ts_barrier"], [0, 0])]:
        assert unwaited("\n".join(["_Zk:"] + lines + [".Lfunc_end0:"])) == {"_Zk": want}


def test_copies_are_waited_for(tmp_path):
    if not (os.path.exists(ftbuild.HIPCC) or shutil.which("hipcc")):
        pytest.skip("no hipcc")
    out = tmp_path / "k.s"
    subprocess.run([ftbuild.HIPCC] + ftbuild.HIP_FLAGS +
                   ["-x", "hip", "--offload-device-only", "-S", "-o", str(out),
                    os.path.join(ftbuild.CSRC, "adapter_logits.hip")],
                   check=True, capture_output=True, text=True)
    kernels = unwaited(out.read_text())
    copying = {k: v for k, v in kernels.items() if v[0]}
    assert any("logits_tile" in k for k in copying) and any("logits_staged" in k for k in copying)
    for name, (_, bare) in copying.items():
        assert bare == 0, name
