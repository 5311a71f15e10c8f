"""The machine code hipcc made of the kernels, read and executed without a GPU."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

from mallie_amd import build as b  # noqa: E402

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# the forms of gfx950's packed FP32 (two floats in a register pair); v_pk_*_f16 and the like are other instructions
PACKED_F32 = re.compile(r"\bv_pk_(?:add|mul|fma)_f32\b|\bv_pk_mov_b32\b")


def device_code(lib, tmp):
    """The disassembly of every code object in a library built here."""
    copy = os.path.join(tmp, "lib.so")  # llvm-objdump writes the code objects beside its input
    shutil.copy(lib, copy)
    subprocess.run([OBJDUMP, "--offloading", copy], check=True, capture_output=True)
    objs = sorted(f for f in os.listdir(tmp) if f.startswith("lib.so.") and "gfx950" in f)
    return [subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", os.path.join(tmp, f)], check=True, capture_output=True, text=True).stdout for f in objs]


@pytest.mark.parametrize("lib", [b.LIB, b.LIB_OCC, b.LIB_LITERAL], ids=os.path.basename)
def test_no_kernel_holds_packed_fp32(lib, tmp_path):
    """Some forms of packed FP32 have given wrong results on the MI355X now and then, without an error.  The compiler makes them of
    ordinary float code by itself, so only the flag that takes the feature away keeps them out."""
    if not os.path.isfile(lib) or not os.path.isfile(OBJDUMP):
        pytest.skip("needs the built library and ROCm's llvm-objdump")
    texts = device_code(lib, str(tmp_path))
    assert len(texts) >= 8 and any("v_fma_f64" in t for t in texts), "the disassembly was not read"
    found = [m for t in texts for m in PACKED_F32.findall(t)]
    assert not found, "%d of %s" % (len(found), sorted(set(found)))


def test_every_compile_line_takes_packed_fp32_away():
    """Tools that look at the kernels' code, or build a kernel of their own, compile it as the library is compiled."""
    assert " ".join(b.KERNEL_FLAGS).endswith("-Xclang -target-feature -Xclang -packed-fp32-ops") and b.FLAGS[:len(b.KERNEL_FLAGS)] == b.KERNEL_FLAGS
    bad = []
    for top in ("tools", "profiles", "mallie_amd"):
        for d, _, files in os.walk(os.path.join(ROOT, top)):
            for f in files:
                if f.endswith((".py", ".sh", ".hip", ".hpp")):
                    with open(os.path.join(d, f)) as fh:
                        bad += ["%s:%d" % (os.path.relpath(os.path.join(d, f), ROOT), i) for i, l in enumerate(fh, 1)
                                if "--offload-arch=gfx950" in l and "-packed-fp32-ops" not in l]
    assert not bad, bad


def test_the_kernels_as_the_library_compiles_them_match_the_oracle(tmp_path):
    """The gfx950 instruction streams of the library's own flags, executed by the tests' interpreter: frames, records and counters equal
    the oracle's."""
    if not os.path.isfile(os.path.join(ROOT, "tests", "emu", "build_emu.py")) or not os.path.isfile("/opt/rocm/bin/hipcc"):
        pytest.skip("needs tests/emu and hipcc")
    sys.path.insert(0, os.path.join(ROOT, "tests", "emu"))
    import build_emu
    lib = build_emu.build()
    dumps = [str(tmp_path / s) for s in ("mgpu_render_sm.s", "mgpu_kernels.s", "mgpu_render_w5.s", "mgpu_trace_sm.s")]
    procs = [subprocess.Popen([b.hipcc()] + b.KERNEL_FLAGS + ["-S", "--cuda-device-only", os.path.join(b.CSRC, os.path.basename(d)[:-2] + ".hip"), "-o", d],
                              stderr=subprocess.DEVNULL) for d in dumps]
    assert [p.wait() for p in procs] == [0] * len(procs)
    assert not any(PACKED_F32.search(open(d).read()) for d in dumps)
    env = {k: v for k, v in os.environ.items() if not k.startswith("MGPU_")}
    env.update(MALLIE_MGPU_LIB=lib, MALLIE_ALLOW_EMULATOR="1", MALLIE_NO_TORCH="1", MGPU_EMU_ISA=":".join(dumps))
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.join(ROOT, "tests", "emu", "cases_emu.py"), "-q", "-x", "-p", "no:cacheprovider",
                        "-k", "render_kernels or five_wave or batched_trace or gfx950"], env=env, capture_output=True, text=True, cwd=ROOT, timeout=1500)
    assert r.returncode == 0 and " passed" in r.stdout and "skipped" not in r.stdout.splitlines()[-1], r.stdout[-4000:] + r.stderr[-2000:]
