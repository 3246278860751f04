"""The wait states of loads into LDS, in the built library's own code (no GPU).

The loads of ``lucid_amd/csrc/lq_dma.h`` are inline asm, which the compiler's hazard pass does not
see, so the asm keeps the distances itself.  In wait states (an instruction is one, ``s_nop n`` is
n + 1) a load into LDS needs
  * 1 after a scalar write of M0, which holds its LDS address;
  * 5 after a vector instruction's write of a scalar register that it reads."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "lucid_amd", "_lib", "liblucid_amd.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

_SCALARS = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b")


def _scalars(text: str) -> set[int]:
    found: set[int] = set()
    for lo, hi, one in _SCALARS.findall(text):
        found |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return found


def _is_lds_load(text: str) -> bool:
    op = text.split(None, 1)[0]
    return "_load_lds_" in op or (op.startswith("buffer_load") and text.endswith(" lds"))


def _states(text: str) -> int:
    return int(text.split()[1], 0) + 1 if text.startswith("s_nop") else 1


def violations(lines):
    """(function, load, what) of every load into LDS that is too near to what it depends on."""
    fn, recent = "", []
    for line in lines:
        if not line.startswith("\t"):
            if line.endswith(">:"):
                fn, recent = line, []
            continue
        text = line.split("//", 1)[0].strip()
        if not text:
            continue
        if _is_lds_load(text):
            need, distance = _scalars(text), 0
            for earlier in reversed(recent):
                if distance >= 5:
                    break
                dst = earlier.split(",", 1)[0]
                if distance < 1 and earlier.startswith("s_") and re.search(r"\bm0$", dst):
                    yield fn, text, f"M0 written {distance} wait states before by {earlier}"
                if earlier.startswith("v_") and _scalars(dst) & need:
                    yield fn, text, f"scalars written {distance} wait states before by {earlier}"
                distance += _states(earlier)
        recent = recent[-7:] + [text]


def test_the_check_sees_what_it_is_for():
    """Its own rules, on listings written for it."""
    def of(*code):
        return [what for _, _, what in violations(["<f>:"] + ["\t" + c for c in code])]

    load = "buffer_load_dwordx4 v1, s[4:7], s9 offen lds"
    copy = "global_load_lds_dwordx4 v[2:3], off nt"
    for use in (load, copy):
        assert of("s_mov_b32 m0, s3", use) and of("s_add_i32 m0, s3, 16", use)
        assert not of("s_mov_b32 m0, s3", "s_nop 0", use) and not of("s_mov_b32 s8, m0", use)
    assert of("v_readfirstlane_b32 s6, v0", "s_nop 3", load) and not of("v_readfirstlane_b32 s6, v0", "s_nop 4", load)
    assert not of("v_readfirstlane_b32 s8, v0", load)
    assert not of("s_mov_b32 m0, s3", "buffer_load_dwordx4 v[0:3], v1, s[4:7], 0 offen")


@pytest.mark.skipif(shutil.which(OBJDUMP) is None or not os.path.exists(LIB), reason="needs the built library and ROCm")
def test_loads_into_lds_keep_their_distance(tmp_path):
    lib = shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    objects = sorted(p for p in tmp_path.iterdir() if p.name.endswith("gfx950"))
    assert objects
    bad, loads = [], 0
    for obj in objects:
        with subprocess.Popen([OBJDUMP, "-d", str(obj)], stdout=subprocess.PIPE, text=True) as p:
            lines = []
            for line in p.stdout:
                lines.append(line.rstrip("\n"))
                loads += "_load_lds_" in line or " lds " in line
            bad += violations(lines)
        assert p.returncode == 0
    assert loads > 1000  # the copies are found at all
    assert not bad, f"{len(bad)} of {loads}: " + "; ".join(f"{fn} {load}: {what}" for fn, load, what in bad[:3])
