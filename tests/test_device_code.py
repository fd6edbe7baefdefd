"""The gfx950 code in the built device library holds no instruction that
would change the rounding the kernels promise (disassembled here, no GPU).

* v_fma_mix{lo,hi}_f16 / v_mad_mix{lo,hi}_f16 round an FP32 multiply-add
  straight to FP16 once. The kernels round like the reference CPU kernels:
  the FP32 result first, then to FP16. The compiler forms these from
  f2h(fmaf(...)) unless the value is kept opaque, and the difference shows
  only on rare inputs, so it is checked on the code itself.
* Packed FP32 arithmetic (v_pk_fma_f32, v_pk_mul_f32, v_pk_add_f32) is
  disabled for all device code by the build flags; none may appear.

The library's .hip_fatbin section is a sequence of offload bundles (one per
HIP source); each one's gfx950 code object is unbundled and disassembled.
"""

import pathlib
import re
import subprocess

import pytest

import mlvc_hip

LLVM = pathlib.Path("/opt/rocm/llvm/bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
FORBIDDEN = re.compile(r"\b(v_(?:fma|mad)_mix(?:lo|hi)_f16|v_pk_(?:fma|mul|add)_f32)\b")

pytestmark = pytest.mark.skipif(not (LLVM / "llvm-objdump").exists(), reason="ROCm LLVM tools not available")


@pytest.fixture(scope="module")
def disassembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("isa")
    fatbin = out / "fatbin.bin"
    subprocess.run(["objcopy", f"--dump-section=.hip_fatbin={fatbin}", str(mlvc_hip.DEVICE_LIB), str(out / "lib.so")],
                   check=True, capture_output=True)
    data = fatbin.read_bytes()
    starts = [m.start() for m in re.finditer(re.escape(MAGIC), data)]
    assert starts, "no offload bundle in the device library"
    texts = []
    for k, st in enumerate(starts):
        end = starts[k + 1] if k + 1 < len(starts) else len(data)
        b, co = out / f"b{k}.bin", out / f"c{k}.o"
        b.write_bytes(data[st:end])
        subprocess.run([str(LLVM / "clang-offload-bundler"), "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                        f"--input={b}", f"--output={co}", "--unbundle"], check=True, capture_output=True)
        texts.append(subprocess.run([str(LLVM / "llvm-objdump"), "-d", str(co)], check=True, capture_output=True,
                                    text=True).stdout)
    return texts


def test_device_library_holds_gfx950_kernels(disassembly):
    assert sum(t.count("v_mfma") for t in disassembly) > 1000  # the conv kernels
    assert all("elf64-amdgpu" in t for t in disassembly)


def test_no_single_rounding_mix_or_packed_fp32(disassembly):
    bad = set()
    for text in disassembly:
        kernel = None
        for line in text.splitlines():
            if line.endswith(">:"):
                kernel = line.split("<", 1)[-1][:-2]
            m = FORBIDDEN.search(line)
            if m:
                bad.add((kernel, m.group(1)))
    assert not bad, sorted(bad)[:20]


# Wait states the hardware asks for before a buffer load and does not insert itself; the compiler inserts
# them for its own instructions and cannot see into assembly. Scalar write of m0 before a load to LDS: 1;
# vector write of a scalar register (a lane's value made uniform) before a load that reads it: 5.
BUFFER_LOAD = re.compile(r"^buffer_load_\S+ (.*)$")
SCALARS = re.compile(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])")


def _scalars(text):
    """Numbers of the scalar registers that a piece of assembly names."""
    found = set()
    for one, first, last in SCALARS.findall(text):
        found.update(range(int(first or one), int(last or one) + 1))
    return found


def _missing_waits(text):
    """(kernel, load, write before it) of every load that comes too soon after a write of what it reads."""
    bad, kernel, before = [], None, []  # before: (instruction, wait states it stands for), latest last
    for line in text.splitlines():
        if line.endswith(">:"):
            kernel, before = line.split("<", 1)[-1][:-2], []
            continue
        code = line.split("//")[0].strip()
        if not line.startswith("\t") or not code:
            continue
        load = BUFFER_LOAD.match(code)
        if load:
            to_lds, reads, waited = code.endswith(" lds"), _scalars(load[1]), 0
            for instruction, states in reversed(before):
                name, _, operands = instruction.partition(" ")
                target = operands.split(",")[0].strip()
                if waited < 1 and to_lds and name.startswith("s_") and target == "m0":
                    bad.append((kernel, code, instruction))
                if waited < 5 and name.startswith("v_") and reads & _scalars(target):
                    bad.append((kernel, code, instruction))
                waited += states
                if waited >= 5:
                    break
        nop = re.match(r"s_nop (\d+)$", code)
        before = before[-5:] + [(code, int(nop[1]) + 1 if nop else 1)]
    return bad


def test_wait_states_are_counted():
    code = "0 <k>:\n\ts_mov_b32 m0, s1 // 0\n\t%sbuffer_load_dwordx4 v1, s[4:7], 0 offen lds // 1\n"
    assert _missing_waits(code % "") and not _missing_waits(code % "s_nop 0\n\t")
    code = "0 <k>:\n\tv_readfirstlane_b32 s6, v2\n\ts_nop %d\n\tbuffer_load_dwordx4 v1, v2, s[4:7], 0 offen\n"
    assert _missing_waits(code % 3) and not _missing_waits(code % 4)


def test_loads_wait_for_their_scalar_operands(disassembly):
    assert any(" lds\n" in t or " lds " in t for t in disassembly)
    bad = [b for text in disassembly for b in _missing_waits(text)]
    assert not bad, (len(bad), bad[:5])
