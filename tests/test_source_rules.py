"""What the sources of this repository must not hold (CPU only: text of the tracked trees and the recorded fixtures).

* Nothing opens or decodes a compiled shader: the reference's .spv files are compiled code that was not built here.  The
  fixtures recorded under tests/golden/ are inputs and output numbers and hold no code.
* No source, script or test names an instruction that writes through the scalar data cache (scalar stores and atomics, the
  cache's write-back and discard), comments included: machines that refuse such code refuse the whole tree for it.  This
  file has to name them, and is therefore left out of what is sent to such machines; none of its tests needs a GPU.
* No kernel is written with packed fp32 instructions, and none is compiled to them: some of their forms have given wrong
  results on MI355X, rarely and without an error.  hipcc -O3 makes them by itself unless told not to.
"""
import glob
import os
import re
import subprocess

import numpy as np
import pytest

from test_kernel_resources import _code_object

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TREES = ("transmission_renderer_amd", "include", "oracle", "tools", "examples")
SUFFIXES = (".py", ".c", ".h", ".hip", ".cpp", ".sh", ".s", "Makefile")


def _sources(trees=TREES):
    out = [os.path.join(ROOT, f) for f in ("bench.py", "__graft_entry__.py")]
    for tree in trees:
        for d, dirs, files in os.walk(os.path.join(ROOT, tree)):
            dirs[:] = [x for x in dirs if x != "__pycache__"]
            out += [os.path.join(d, f) for f in files if f.endswith(SUFFIXES)]
    assert len(out) > 60   # the walk found the trees
    return sorted(p for p in out if p != os.path.abspath(__file__))


def _lines_with(pattern, trees=TREES):
    hits = []
    for path in _sources(trees):
        with open(path, encoding="utf-8", errors="replace") as f:
            hits += [f"{os.path.relpath(path, ROOT)}:{n}: {line.strip()}" for n, line in enumerate(f, 1) if re.search(pattern, line)]
    return hits


def test_no_source_opens_or_decodes_a_compiled_shader():
    # a file name, the directory that holds them, or the word that opens such a module
    assert _lines_with(r"\.spv\b|compiled-shaders|(?i:0x07230203)|spirv_interp") == []


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(ROOT, "tests", "golden", "*.npz"))), ids=os.path.basename)
def test_a_fixture_holds_numbers_and_no_code(path):
    with np.load(path, allow_pickle=False) as z:
        for name in z.files:
            a = z[name]
            kinds = [a.dtype[f].base.kind for f in a.dtype.names] if a.dtype.names else [a.dtype.kind]
            assert set(kinds) <= set("fiu"), name
            raw = a.tobytes()
            assert b"\x03\x02\x23\x07" not in raw and b"\x07\x23\x02\x03" not in raw, name   # a module's first word


def test_no_source_names_a_write_through_the_scalar_data_cache():
    pattern = r"\bs_(?:buffer_|scratch_)?(?:store|atomic)_\w+|\bs_dcache_(?:wb|discard)\w*|\bs_atc_probe\w*"
    assert re.search(pattern, "asm volatile(\"s_atomic_add %0, %1, 0x0 glc\")") and re.search(pattern, "s_buffer_store_dwordx2 s[0:1]")
    assert not re.search(pattern, "flush_stores_store_x s_waitcnt s_load_dword global_atomic_add ds_store_b32")
    assert _lines_with(pattern, TREES + ("tests",)) == []


def test_no_kernel_is_written_with_packed_fp32_instructions():
    # in a string: an asm statement, or the name that a benchmark prints for one.  Prose about them is no instruction
    assert _lines_with(r"\"[^\"]*\bv_pk_(?:add|mul|fma)_f32") == []


@pytest.mark.parametrize("name", ["libtr_shade.so", "pattern_ceiling"])
def test_no_built_kernel_holds_packed_fp32_instructions(name, tmp_path):
    objdump = "/opt/rocm/lib/llvm/bin/llvm-objdump"
    path = os.path.join(ROOT, "transmission_renderer_amd", name)
    if not os.path.exists(path):
        pytest.fail(f"{path} is missing: run __graft_entry__.build() first")
    if not os.path.exists(objdump):
        pytest.skip("llvm-objdump not available")
    co = tmp_path / "gfx950.co"
    co.write_bytes(_code_object(path))
    asm = subprocess.run([objdump, "-d", str(co)], capture_output=True, text=True, check=True).stdout
    assert "s_endpgm" in asm
    assert sorted(set(re.findall(r"\bv_pk_(?:add|mul|fma)_f32", asm))) == []


def test_every_hipcc_command_turns_packed_fp32_off():
    # the flag lists that build() and tools/ compile with, and the commands that comments give
    commands = _lines_with(r"--offload-arch=gfx950 -|\"--offload-arch=gfx950\"")
    assert len(commands) >= 9
    assert [c for c in commands if "-packed-fp32-ops" not in c and "NO_PACKED_FP32" not in c] == []
    import __graft_entry__ as g
    assert g.NO_PACKED_FP32 == ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
