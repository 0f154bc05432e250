"""What no GPU source of this tree may hold, checked on its text (CPU only: no GPU, no build).

Scalar data cache: GPU code here never WRITES through it (scalar stores, scalar atomics, that cache's write-back and discard).  The
survivors, the one place that ever did, leave through coalesced vector stores.

Packed FP32: no instruction that works on a register pair of floats, written by hand or formed by the compiler (some of their forms have
given wrong results on this hardware, now and then and without an error): the text of the sources, every line that calls hipcc, and the
assembly of the library's two builds (cross-compiled here with the Makefile's own command lines).

Loads in inline asm: a statement waits for its own loads.  The compiler takes a statement's outputs as written when it ends, and gives
their registers to other values: a load still in flight would then overwrite one of those, an address among them."""
import os
import re
import shlex
import subprocess

import pytest

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


PACKED_FP32 = re.compile(r"\bv_pk_(?:add|mul|fma)_" + "f32")


def test_no_source_holds_a_packed_fp32_instruction():
    assert hits(PACKED_FP32) == []


def test_every_hipcc_line_switches_packed_fp32_off():
    """a file that gives hipcc its --offload-arch gives it the feature switch too, as often"""
    seen, bad = [], []
    arch, off = re.compile(r"--offload-arch="), re.compile(r"-Xclang -target-feature -Xclang -packed-fp32-ops")
    for p in source_files():
        if os.path.abspath(p) == os.path.abspath(__file__):
            continue
        text = open(p, errors="replace").read()
        n = len([m for m in arch.finditer(text)])
        if n:
            seen.append(os.path.relpath(p, ROOT))
            if len(off.findall(text)) != n:
                bad.append(os.path.relpath(p, ROOT))
    assert {"gr-ieee80211_amd/csrc/Makefile", "gnuradio/CMakeLists.txt", "tools/hipflags.sh"} <= set(seen)
    assert bad == []


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """{library: device assembly}, built with the command lines that make would run for the libraries"""
    csrc = os.path.join(ROOT, "gr-ieee80211_amd", "csrc")
    tmp, running, out = tmp_path_factory.mktemp("asm"), {}, {}
    for lib in ("../libc8p_rx.so", "../libc8p_rx_exp.so"):
        line = subprocess.run(["make", "-s", "-n", "-B", "-C", csrc, lib], capture_output=True, text=True, timeout=60)
        assert line.returncode == 0, line.stderr
        cmd = shlex.split(line.stdout.strip().splitlines()[-1])
        assert cmd[cmd.index("-o") + 1] == lib and "-shared" in cmd, cmd
        dst = str(tmp / (os.path.basename(lib) + ".s"))
        cmd[cmd.index("-o") + 1] = dst
        cmd[cmd.index("-shared")] = "-S"
        running[lib] = (subprocess.Popen(cmd + ["--cuda-device-only"], cwd=csrc, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True), dst)
    for lib, (p, dst) in running.items():
        err = p.communicate(timeout=900)[1]
        assert p.returncode == 0, err[-2000:]
        out[lib] = open(dst).read()
    return out


def test_the_built_kernels_hold_no_packed_fp32_and_no_scalar_cache_write(assembly):
    for lib, text in assembly.items():
        assert "k_rx_1ss_lds" in text and "v_fma_f32" in text, lib
        assert PACKED_FP32.search(text) is None, (lib, PACKED_FP32.search(text).group(0))
        assert SCALAR_CACHE_WRITE.search(text) is None, (lib, SCALAR_CACHE_WRITE.search(text).group(0))


# an asm statement, or one of the probes' macros that make one of their text argument
ASM = re.compile(r"\b(?:asm|__asm__)\b(?:\s+(?:volatile|__volatile__))?\s*\(|\bPROBE(?:_HARD)?\s*\(")
LOAD = re.compile(r"\b(?:s_load|s_buffer_load|ds_read|ds_load|ds_bpermute|ds_permute|ds_swizzle|global_load|flat_load|buffer_load|scratch_load)\w*")
LGKM0, VM0 = re.compile(r"s_waitcnt[^\n]*\blgkmcnt\(0\)"), re.compile(r"s_waitcnt[^\n]*\bvmcnt\(0\)")


def asm_texts(src):
    """the instruction text of every asm statement: its string literals up to the first ':' outside a literal"""
    for m in ASM.finditer(src):
        k, depth, text = m.end(), 1, []
        while k < len(src) and depth:
            if src[k] == '"':
                lit = re.compile(r'"((?:[^"\\]|\\.)*)"', re.S).match(src, k)
                text.append(lit.group(1))
                k = lit.end()
                continue
            if src[k] == ":":
                break
            depth += {"(": 1, ")": -1}.get(src[k], 0)
            k += 1
        yield src.count("\n", 0, m.start()) + 1, "".join(text).replace("\\n", "\n").replace("\\t", " ")


def unwaited(text):
    """the last load of a statement that no full wait of its counter follows, or None (exact counts may stand between)"""
    for kind, wait in ((r"^(?:s_|ds_)", LGKM0), (r"^(?!s_|ds_)", VM0)):
        loads = [m for m in LOAD.finditer(text) if re.match(kind, m.group(0))]
        if loads and not wait.search(text, loads[-1].end()):
            return loads[-1].group(0)
    return None


def test_statement_reader():
    t = dict(asm_texts('asm volatile("s_load_dword %0, %1, 0x0\\n\\t" "s_waitcnt lgkmcnt(0)" : "=s"(a) : "s"(p));\n asm("ds_read_b32 %0, %1" : "=v"(a) : "v"(p));'))
    assert list(t) == [1, 2] and unwaited(t[1]) is None and unwaited(t[2]) == "ds_read_b32"
    assert unwaited("global_load_dword v0, v1, s[0:1]\ns_waitcnt lgkmcnt(0)") == "global_load_dword"
    assert unwaited("ds_read_b32 v0, v1\ns_waitcnt lgkmcnt(0)\nds_read_b32 v2, v1\ns_waitcnt lgkmcnt(1)") == "ds_read_b32"


def test_asm_statements_wait_for_their_own_loads():
    n, bad = 0, []
    for p in source_files():
        if p.endswith((".h", ".hip", ".cc", ".cpp", ".c")):
            for line, text in asm_texts(open(p, errors="replace").read()):
                n += bool(LOAD.search(text))
                if unwaited(text):
                    bad.append("%s:%d: %s" % (os.path.relpath(p, ROOT), line, unwaited(text)))
    assert n >= 20 and bad == []                     # (the generated block loops and the probes' exchange bodies)


REG = re.compile(r"\b([vs])(?:(\d+)\b|\[(\d+):(\d+)\])")


def named_registers(text):
    out = set()
    for m in REG.finditer(re.sub(r"%\[\w+\]", "", text)):
        lo, hi = (m.group(2), m.group(2)) if m.group(2) else (m.group(3), m.group(4))
        out |= {m.group(1) + str(k) for k in range(int(lo), int(hi) + 1)}
    return out


def test_registers_an_asm_statement_names_are_declared():
    """a register named in the text (not an operand) is bound to an operand or a clobber: the compiler counts the registers of a kernel,
    and keeps live values out of them, by the declarations alone"""
    csrc = os.path.join(ROOT, "gr-ieee80211_amd", "csrc")
    n = 0
    for f in sorted(os.listdir(csrc)):
        if not f.endswith((".h", ".hip")):
            continue
        src = open(os.path.join(csrc, f)).read()
        for line, text in asm_texts(src):
            named = named_registers(text)
            if named:
                start = sum(len(x) + 1 for x in src.split("\n")[:line - 1])
                decl = src[start:src.index(";\n", src.index(" : ", start))]
                declared = set(re.findall(r'"([vs]\d+)"', decl)) | set(re.findall(r'\{([vs]\d+)\}', decl))
                assert named <= declared, (f, line, sorted(named - declared))
                n += 1
    assert n >= 16
    probe = open(os.path.join(ROOT, "tools", "probe_issue.hip")).read()
    hard = set(re.findall(r'"([vs]\d+)"', re.search(r"#define HARD (.*)", probe).group(1)))
    plain = set(re.findall(r'"([vs]\d+)"', re.search(r"asm volatile\(BODY : OPS : INS : (.*?)\)", probe).group(1)))
    cand = re.search(r'#define CAND "(.*)"', probe).group(1)
    assert named_registers(cand) <= hard
    for m in re.finditer(r"^PROBE(_HARD)?\((\w+),", probe, re.M):
        text = probe[m.end():probe.index("\nPROBE", m.end()) if "\nPROBE" in probe[m.end():] else probe.index("\nstruct Probe", m.end())]
        text = re.sub(r"//.*", "", text)
        text = re.sub(r"^#define (?:.*\\\n)*.*$", "", text, flags=re.M)
        named = named_registers("".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text, re.S)).replace("\\n", "\n").replace("\\t", " "))
        assert named <= (hard if m.group(1) else plain), (m.group(2), sorted(named))


PRIORITY = re.compile("StreamCreateWith" + "Priority|StreamPriority" + "Range|STREAM_" + r"PRIORITY|is_high_priority_" + r"stream\s*=\s*True|Stream\([^)]*\bpriority\s*=")


def test_every_stream_has_the_default_priority():
    """work on streams of different priorities has hung this hardware for good: no source asks for one, and no environment switch can"""
    assert PRIORITY.search("torch.cuda.Stream" + "(device=0, priority=-1)") and not PRIORITY.search("torch.cuda.Stream(device=0)")
    assert hits(PRIORITY) == []


def test_the_library_cannot_make_a_stream_of_another_priority():
    lib = os.path.join(ROOT, "gr-ieee80211_amd", "libc8p_rx.so")
    if not os.path.exists(lib):
        pytest.skip("libc8p_rx.so is not built")
    import shutil
    if shutil.which("nm") is None:
        pytest.skip("no nm")
    names = subprocess.run(["nm", "-D", "--undefined-only", lib], capture_output=True, text=True, check=True).stdout
    assert "hipStreamCreateWithFlags" in names and PRIORITY.search(names) is None


def test_build_compiles_on_every_call(monkeypatch):
    """__graft_entry__.build() is the check that the sources compile: it must not be satisfied by libraries that are there already"""
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, *a, **k: calls.append(cmd))
    if os.path.exists(os.path.join(ROOT, "gr-ieee80211_amd", "libc8p_rx.so")):
        entry.build()
    else:
        pytest.skip("libc8p_rx.so is not built")
    assert len(calls) >= 4 and all(c[0] == "make" and "-B" in c for c in calls), calls
