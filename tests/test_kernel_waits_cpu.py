"""Wait states that hand-written instructions need, in the built code objects.

A direct global -> LDS load takes its LDS address from m0 and may take its base
from scalar registers.  One wait state has to lie between a scalar write of m0
and the load, and five between a vector instruction's write of a scalar
register and a memory instruction that reads it.  The compiler sees to that in
its own code, not within inline code and not before it, so the listing of every
kernel is looked over: each instruction is one wait state, s_nop n is n + 1."""

import os
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
KERNELS = ROOT / "tensor-ash_amd" / "lib" / "kernels"
LLVM = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm" / "bin"


def listing(code_object, tmp_path):
    elf = tmp_path / (code_object.stem + ".elf")
    subprocess.run([str(LLVM / "clang-offload-bundler"), "--unbundle", "--type=o", f"--input={code_object}",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--output={elf}"], check=True, capture_output=True)
    return subprocess.run([str(LLVM / "llvm-objdump"), "-d", "--no-show-raw-insn", str(elf)], check=True,
                          capture_output=True, text=True).stdout


def registers(operand):
    """The scalar registers of "s5", "s[4:7]" or "vcc"; none for others."""
    if operand == "vcc":
        return {"vcc"}
    m = re.fullmatch(r"s(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    return set(range(int(m[1] or m[2]), int(m[1] or m[3]) + 1))


def faults(text):
    """(direct loads, those that come too early with what they wait for)."""
    loads, found, before, kernel = 0, [], [], ""
    for line in text.splitlines():
        m = re.match(r"^[0-9a-f]+ <(.*)>:", line)
        if m:
            kernel, before = m[1], []
            continue
        ins = line.split("//")[0].strip()
        if not ins:
            continue
        name, *operands = re.split(r"[ ,]+", ins)
        if re.match(r"(global|buffer|scratch)_load_lds_", name) or (name.startswith("buffer_load") and "lds" in operands):
            loads += 1
            reads = set().union(*(registers(o) for o in operands))
            waits = 0
            for earlier in reversed(before[-6:]):
                what, *of = re.split(r"[ ,]+", earlier)
                if waits < 1 and what.startswith("s_") and of[:1] == ["m0"]:
                    found.append((kernel, ins, earlier))
                written = of[:2] if "_co_" in what or "div_scale" in what else of[:1]
                if waits < 5 and what.startswith("v_") and set().union(*map(registers, written)) & reads:
                    found.append((kernel, ins, earlier))
                waits += int(of[0], 0) + 1 if what == "s_nop" else 1
        before.append(ins)
    return loads, found


@pytest.mark.parametrize("lines,bad", [
    (["s_mov_b32 m0, s4", "global_load_lds_dwordx4 v1, s[2:3]"], 1),
    (["s_mov_b32 m0, s4", "s_nop 0", "global_load_lds_dwordx4 v1, s[2:3]"], 0),
    (["s_mov_b32 m0, s4", "v_add_u32_e32 v2, v3, v4", "global_load_lds_dwordx4 v[2:3], off"], 0),
    (["v_readfirstlane_b32 s3, v7", "s_mov_b32 m0, s4", "s_nop 2", "global_load_lds_dwordx4 v1, s[2:3]"], 1),
    (["v_readfirstlane_b32 s3, v7", "s_mov_b32 m0, s4", "s_nop 3", "global_load_lds_dwordx4 v1, s[2:3]"], 0),
    (["v_readfirstlane_b32 s9, v7", "s_mov_b32 m0, s9", "s_nop 0", "global_load_lds_dwordx4 v1, s[2:3]"], 0)])
def test_the_rule(lines, bad):
    loads, found = faults("0000000000001000 <kernel>:\n" + "\n".join("\t" + x for x in lines))
    assert loads == 1 and len(found) == bad


@pytest.mark.parametrize("name,least", [("attention", 100), ("gemm_f16", 100), ("gemm_f16w3", 20), ("gemm_f32", 100),
                                        ("gemm_f32x6", 20), ("tree_attention", 100)])
def test_direct_loads_wait(name, least, tmp_path):
    loads, found = faults(listing(KERNELS / f"{name}.hsaco", tmp_path))
    assert loads >= least and not found, (loads, len(found), found[:4])


def test_no_other_kernel_loads_into_lds(tmp_path):
    """A code object that begins to has to be named above."""
    seen = {f.stem for f in KERNELS.glob("*.hsaco") if faults(listing(f, tmp_path))[0]}
    assert seen == {"attention", "gemm_f16", "gemm_f16w3", "gemm_f32", "gemm_f32x6", "tree_attention"}
