"""Wait states that the hardware does not check and that the compiler does not
add around inline assembly, looked for in the built kernels' instructions:

  * one between a scalar write of M0 and a load that goes straight into LDS
  * five between a vector instruction's write of a scalar register and a memory
    instruction that takes its address from it

An instruction counts as one, s_nop N as N + 1."""
import glob
import os
import re
import shutil
import subprocess

import pytest

import glint_word2vec_amd

PKG = os.path.dirname(glint_word2vec_amd.__file__)
LLVM = "/opt/rocm/llvm/bin"


def _tool(name):
    path = os.path.join(LLVM, name)
    return path if os.path.exists(path) else shutil.which(name)


TOOLS = {n: _tool(n) for n in ("llvm-objcopy", "clang-offload-bundler",
                               "llvm-objdump")}


def _instructions(library, tmp_path):
    """The library's gfx950 instructions, one list for each function."""
    bundle, code = str(tmp_path / "bundle"), str(tmp_path / "code")
    subprocess.check_call([TOOLS["llvm-objcopy"], "--dump-section",
                           f".hip_fatbin={bundle}", library,
                           str(tmp_path / "rest")])
    subprocess.check_call([
        TOOLS["clang-offload-bundler"], "--unbundle", "--type=o",
        "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={bundle}",
        f"--output={code}"])
    text = subprocess.check_output(
        [TOOLS["llvm-objdump"], "-d", "--no-show-raw-insn",
         "--no-leading-addr", code], text=True)
    functions = []
    for line in text.splitlines():
        if re.match(r"^<[^>]+>:$|^[0-9a-f]+ <", line):
            functions.append([])
        elif functions and line[:1] in " \t":
            line = line.split("//")[0].strip()
            if line:
                functions[-1].append(line)
    return functions


def _registers(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m[1])} if m else set()


def _parts(line):
    name, _, rest = line.partition(" ")
    return name, [o.strip().split(" ")[0] for o in rest.split(",")]


def _written(name, operands):
    """Scalar registers that a vector instruction writes."""
    if not name.startswith("v_"):
        return set()
    out = _registers(operands[0])
    if "_co_" in name or name.startswith("v_div_scale"):
        out |= _registers(operands[1])
    return out


def _waits(name, operands):
    return int(operands[0], 0) + 1 if name == "s_nop" else 1


def _faults(lines):
    found = []
    parts = [_parts(line) for line in lines]
    for i, (name, operands) in enumerate(parts):
        if not name.startswith(("global_", "buffer_", "flat_", "scratch_")):
            continue
        to_lds = "_lds_" in name or " lds" in lines[i]
        reads = set().union(*map(_registers, operands))
        waited = 0
        for before, args in reversed(parts[max(0, i - 5):i]):
            if waited < 1 and to_lds and before.startswith("s_") \
                    and args[0] == "m0":
                found.append(("M0", lines[i]))
            if waited < 5 and reads & _written(before, args):
                found.append(("address", lines[i]))
            waited += _waits(before, args)
    return found


def test_what_is_looked_for():
    load = "global_load_lds_dwordx4 v1, s[2:3]"
    m0, base = "s_mov_b32 m0, s5", "v_readfirstlane_b32 s3, v9"
    for lines, kinds in (
            ([m0, load], {"M0"}), ([m0, "s_nop 0", load], set()),
            ([m0, "s_mov_b64 s[8:9], s[2:3]", load], set()),
            ([base, m0, "s_nop 2", load], {"address"}),
            ([base, m0, "s_nop 3", load], set()),
            ([base, "s_nop 4", load], set()), ([base, load], {"address"}),
            ([base, m0, "s_mov_b64 s[8:9], s[2:3]",
              "global_load_lds_dwordx4 v1, s[8:9]"], set()),
            (["v_cmp_eq_u32_e64 s[2:3], v1, v2",
              "global_load_dword v1, v2, s[2:3]"], {"address"}),
            (["v_add_co_u32_e64 v1, s[2:3], v1, v2",
              "buffer_load_dword v1, v2, s[0:3], 0 offen"], {"address"}),
            (["v_mov_b32_e32 v2, s3", load], set())):
        assert {k for k, _ in _faults(lines)} == kinds, lines


@pytest.mark.skipif(not all(TOOLS.values()), reason="no LLVM tools")
@pytest.mark.parametrize("name", ["_hip_native", "_vocab_native"])
def test_no_wait_state_is_missing(name, tmp_path):
    built = glob.glob(os.path.join(PKG, name + "*.so"))
    if not built:
        pytest.skip("not built")
    functions = _instructions(built[0], tmp_path)
    assert sum(map(len, functions)) > 10_000
    loads = sum("_lds_" in line.split(" ")[0] for f in functions for line in f)
    assert loads > 100 or name != "_vocab_native"
    found = [f for lines in functions for f in _faults(lines)]
    assert not found, f"{len(found)}, such as {found[:3]}"
