"""No GPU code of this tree writes through the scalar data cache: no scalar stores, no scalar memory atomics, no write-back or discard of
that cache, neither as a source nor as text that a tool inserts into assembly.  Kernels write through vector memory only.  (Checked on the
text of the sources, comments included; runs on the CPU and reads files only.)"""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# s_store_*, s_buffer_store_*, s_scratch_store_*, s_atomic_*, s_buffer_atomic_*, s_dcache_wb*, s_dcache_discard*, and the builtins of the write-back;
# at the start of a word, or behind the escaped tab or newline of a quoted assembly line
SCALAR_WRITE = re.compile(r"(?:(?<![A-Za-z0-9_])|(?<=\\[tn]))s_(?:(?:buffer_|scratch_)?(?:store|atomic)|dcache_(?:wb|discard))|builtin_amdgcn_s_dcache_(?:wb|discard)", re.I)
SOURCE = re.compile(r"(?:\.(?:hip|cu|cpp|cc|c|hpp|h|s|asm|inc|ll|sed|py|sh|txt|mk)|/Makefile)$", re.I)
# CPU tests that only name the instructions: this one, and the unit test of a rewriter that is no longer in the tree
NAMES_ONLY = {"tests/test_scalar_cache_rule.py", "tests/test_host.py"}


def sources():
    """Every source, script and build file of the checkout: not records (profiles/), build products or folders of tools (a leading . or _)."""
    for top, dirs, files in os.walk(ROOT):
        rel = os.path.relpath(top, ROOT)
        dirs[:] = [d for d in dirs if d[0] not in "._" and d not in ("build", "build_exp", "gpurun_out") and os.path.join(rel, d) != "./profiles"]
        for f in files:
            name = os.path.normpath(os.path.join(rel, f))
            if SOURCE.search("/" + name):
                yield name


def test_no_source_writes_through_the_scalar_data_cache():
    seen, bad = 0, []
    for name in sources():
        seen += 1
        if name in NAMES_ONLY:
            continue
        with open(os.path.join(ROOT, name), errors="replace") as f:
            bad += [f"{name}:{i}: {line.strip()[:100]}" for i, line in enumerate(f, 1) if SCALAR_WRITE.search(line)]
    assert seen > 50 and os.path.normpath("rayhs_amd/csrc/trace_kernel.hip") in set(sources())   # the walk reaches the kernels
    assert not bad, "\n".join(bad)


def test_files_that_only_name_the_instructions_are_cpu_tests():
    for name in NAMES_ONLY:
        assert name.startswith("tests/") and name.endswith(".py")
        assert not re.search(r"^\s*@?(?:pytestmark\s*=\s*)?pytest\.mark\.gpu", open(os.path.join(ROOT, name)).read(), re.M), name


@pytest.mark.parametrize("text, writes", [
    ("s_store_dword s0, s[2:3], 0x0", True), ("s_buffer_store_dwordx2 s[0:1], s[4:7], s8", True), ("s_scratch_store_dword s0, s[2:3], 0", True),
    ("\ts_atomic_add s5, s[2:3], 0x10", True), ("\"s_buffer_atomic_or s1, s[4:7], 0\"", True), ("s_dcache_wb", True), (r'asm volatile("s_waitcnt lgkmcnt(0)\n\ts_dcache_wb");', True), (r'f"\ts_atomic_add s1, s[2:3], 0"', True), ("s_dcache_wb_vol", True),
    ("s_dcache_discard s[2:3], 0x0", True), ("__builtin_amdgcn_s_dcache_wb();", True), ("S_STORE_DWORD s0, s[2:3], 0", True),
    ("s_load_dwordx16 s[0:15], s[2:3], 0x0", False), ("s_buffer_load_dword s0, s[4:7], 0", False), ("s_dcache_inv", False),
    ("ws_store(ws, slot, v); cx_store3(cx, CX_V, v); ds_store_b32 v0, v1", False), ("global_atomic_add v[0:1], v2, off", False)])
def test_the_pattern_tells_scalar_cache_writes_from_other_memory_instructions(text, writes):
    assert bool(SCALAR_WRITE.search(text)) is writes
