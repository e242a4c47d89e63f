"""Statements of inline assembly keep the hardware's rules by themselves: the compiler does not look into them."""
import glob
import os
import re
import shutil
import subprocess

from h2o4gpu_amd.build import HIPCC

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "h2o4gpu_amd", "csrc")
STATEMENT = re.compile(r"asm volatile\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)((?::[^;]*)?)\);")


def statements():
    for name in sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        for m in STATEMENT.finditer(open(name).read()):
            text = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
            lines = [line.strip() for line in re.split(r"\\n|;", text.replace("\\t", " ")) if line.strip()]
            clobbers = re.findall(r'"([^"]+)"', m.group(2).split(":")[3]) if m.group(2).count(":") >= 3 else []
            yield os.path.basename(name), lines, clobbers


def test_they_are_found():
    assert any("buffer_load" in line for _, lines, _ in statements() for line in lines)


def test_a_written_m0_is_named():
    for name, lines, clobbers in statements():
        if any(re.match(r"s_\w+ m0,", line) for line in lines):
            assert "m0" in clobbers, (name, lines)


# ---- what the compiler made of them

LOAD = re.compile(r"^\s+buffer_load_\w+ v\d+, s\[(\d+):(\d+)\], .*\blds\b")


def scalars(operand):
    m = re.match(r"s\[(\d+):(\d+)\]$|s(\d+)$", operand)
    return set() if not m else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def too_near(listing):
    """Loads to LDS that read a scalar register less than five states after a vector instruction wrote it. An instruction
    is one state, s_nop n is n + 1."""
    found, lines = [], [line.split("//")[0] for line in listing]
    for i, line in enumerate(lines):
        m = LOAD.match(line)
        if not m:
            continue
        reads, states = set(range(int(m[1]), int(m[2]) + 1)), 0
        for before in reversed(lines[max(0, i - 8):i]):
            words = before.split(None, 1)
            if states >= 5 or not words or words[0].endswith(":"):
                break
            operands = [o.strip() for o in words[1].split(",")] if len(words) > 1 else []
            if words[0].startswith("v_") and any(scalars(o) & reads for o in operands[:2 if "_co_" in words[0] or "mad_u64" in words[0] else 1]):
                found.append((before.strip(), line.strip()))
            states += int(operands[0]) + 1 if words[0] == "s_nop" else 1
    return found


def test_what_is_too_near_is_found():
    load = "\tbuffer_load_dwordx4 v6, s[16:19], 0 offen lds   // 0001: E05D1000"
    near = "\tv_readfirstlane_b32 s18, v3", "\ts_mov_b32 m0, s71", "\ts_nop 2"
    assert len(too_near(near + (load,))) == 1
    assert not too_near(near + ("\ts_nop 0", load)) and not too_near(("\tv_readfirstlane_b32 s20, v3", load))
    assert len(too_near(("\tv_mad_u64_u32 v[2:3], s[16:17], v4, s42, v[6:7]", load))) == 1
    assert not too_near(("\tv_mov_b32_e32 v2, s17", load))


def test_built_loads_wait_for_scalar_registers(hip, tmp_path):
    tool = os.path.join(os.path.dirname(os.path.dirname(HIPCC)), "llvm", "bin", "llvm-objdump")
    shutil.copy(hip.LIB_PATH, tmp_path / "lib.so")
    subprocess.check_call([tool, "--offloading", "lib.so"], cwd=tmp_path, stdout=subprocess.DEVNULL)
    loads = 0
    for part in sorted(tmp_path.glob("*gfx950")):
        listing = subprocess.run([tool, "-d", "--no-show-raw-insn", str(part)], check=True, capture_output=True,
                                 text=True).stdout.splitlines()
        loads += sum(bool(LOAD.match(line)) for line in listing)
        assert not too_near(listing)
    assert loads > 0
