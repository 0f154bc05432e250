"""What no GPU source of this tree may hold, checked on its text (CPU only: no GPU, no build).

Scalar data cache: GPU code here never WRITES through it (scalar stores, scalar atomics, that cache's write-back and discard).  The
survivors, the one place that ever did, leave through coalesced vector stores."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SKIP = {".git", "__pycache__", ".pytest_cache", "gpurun_out", "_work", "build", "profiles", "node_modules"}
SOURCES = (".c", ".cc", ".cpp", ".h", ".hpp", ".hip", ".cu", ".cl", ".s", ".S", ".asm", ".ll", ".py", ".sh", ".cmake", ".mk")

# mnemonics and builtins, put together from parts: this file is itself one of the texts that are searched
_S = "s" + "_"
SCALAR_CACHE_WRITE = re.compile(r"\b%s(?:buffer_|scratch_)?(?:store|atomic)_\w+|%s(?:wb|discard)" % (_S, _S + "dcache_"))


def source_files():
    for d, dirs, files in os.walk(ROOT):
        dirs[:] = [x for x in dirs if x not in SKIP]
        for f in files:
            if f.endswith(SOURCES) or f in ("Makefile", "CMakeLists.txt"):
                yield os.path.join(d, f)


def hits(rx):
    out = []
    for p in source_files():
        with open(p, errors="replace") as fh:
            for k, line in enumerate(fh, 1):
                if rx.search(line):
                    out.append("%s:%d: %s" % (os.path.relpath(p, ROOT), k, line.strip()[:100]))
    return out


def test_the_search_sees_the_sources():
    names = {os.path.relpath(p, ROOT) for p in source_files()}
    assert {"gr-ieee80211_amd/csrc/c8p_engine.hip", "gr-ieee80211_amd/csrc/c8p_viterbi_lean.h", "gr-ieee80211_amd/csrc/Makefile",
            "tools/gen_lean_asm.py", "tools/probe_issue.hip"} <= names


def test_pattern_knows_the_instructions():
    for x in ("store_dword", "store_dwordx4", "buffer_store_dwordx2", "scratch_store_dword", "atomic_add", "buffer_atomic_swap_x2",
              "dcache_wb", "dcache_wb_vol", "dcache_discard_x2"):
        assert SCALAR_CACHE_WRITE.search('"' + _S + x + ' s[20:21]"'), x
    for x in ("global_store_dword v0, v1, s[2:3]", "buffer_store_dword", "ds_write_b32", _S + "load_dwordx4", _S + "dcache_inv", "global_atomic_add"):
        assert not SCALAR_CACHE_WRITE.search(x), x


def test_no_source_writes_through_the_scalar_data_cache():
    assert hits(SCALAR_CACHE_WRITE) == []
