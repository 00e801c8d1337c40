"""What the native sources must not hold, read from their text: instructions that have proved unsafe on the hardware, in probes that
nothing builds and in comments as much as in kernels.  The patterns are spelt so that this file does not match them."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FOLDERS = ("crispresso2_amd", "include", "oracle", "tests", "tools")
SUFFIXES = (".hip", ".h", ".hpp", ".c", ".cc", ".cpp", ".s", ".S", ".py", ".sh", ".mk")
NAMES = ("Makefile", "CMakeLists.txt")
SKIPPED = ("__pycache__", "lib", "_ref", "golden", "build")          # built files and recorded data


def sources():
    found = [os.path.join(ROOT, n) for n in os.listdir(ROOT)]
    for folder in FOLDERS:
        for d, subs, names in os.walk(os.path.join(ROOT, folder)):
            subs[:] = [x for x in subs if x not in SKIPPED]
            found += [os.path.join(d, n) for n in names]
    return sorted(f for f in found if os.path.isfile(f) and (f.endswith(SUFFIXES) or os.path.basename(f) in NAMES))


def lines_with(pattern):
    rx = re.compile(pattern)
    out = []
    for f in sources():
        with open(f, encoding="utf-8", errors="replace") as fh:
            out += ["%s:%d: %s" % (os.path.relpath(f, ROOT), k, m.group(0)) for k, line in enumerate(fh, 1) for m in [rx.search(line)] if m]
    return out


def test_the_walk_reaches_every_kind_of_source():
    got = {os.path.relpath(f, ROOT) for f in sources()}
    assert {"bench.py", "crispresso2_amd/csrc/Makefile", "crispresso2_amd/csrc/c2_k_align.hip", "crispresso2_amd/csrc/c2_fastq.cpp",
            "include/crispresso2_amd.h", "oracle/c2_oracle.c", "tests/emu/emu_harness.cpp", "tools/build_variant.sh"} <= got


def test_nothing_writes_through_the_scalar_data_cache():
    """Scalar stores, scalar atomics, and the scalar data cache's write-back and discard: data is written by vector stores."""
    assert lines_with(r"\bs_(?:[a-z0-9]+_)*(?:store|atomic|dcache)(?:_[a-z0-9]+)*") == []


def test_no_source_writes_packed_fp32_arithmetic():
    """The two-wide float add, multiply and multiply-add: some of their forms give wrong results now and then, without an error."""
    assert lines_with(r"\bv_pk_(?:add|mul|fma)_f32") == []


PACKED_FP32_OFF = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def test_every_unit_is_compiled_with_packed_fp32_off():
    """The compiler makes packed FP32 from ordinary float code by itself unless it is told not to: every compile line of the library,
    of the A/B builds, and the build line of each probe."""
    out = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "crispresso2_amd", "csrc"), "HIPCC=hipcc"],
                         check=True, capture_output=True, text=True).stdout
    compiles = [x for x in out.splitlines() if x.startswith("hipcc") and " -c " in x]
    units = [re.search(r" -c (\S+) -o \.\./lib/obj/(\S+)\.o$", x).groups() for x in compiles]
    assert len(units) == 6 and all(src in (obj + ".hip", obj + ".cpp") for src, obj in units)
    assert all(PACKED_FP32_OFF in x for x in compiles)
    lines = []
    for f in sources():
        if f.endswith((".sh", ".hip")):
            with open(f, encoding="utf-8") as fh:
                lines += [x for x in fh if "hipcc " in x and "--offload-arch" in x and ".hip" in x]
    assert lines and all(PACKED_FP32_OFF in x for x in lines)


def test_build_compiles_also_where_a_library_is_there(monkeypatch):
    """File times cannot say whether a built library belongs to the sources beside it (a copied tree, a changed compiler or variable):
    build() asks make for every unit."""
    import __graft_entry__ as entry

    class Stop(Exception):
        pass

    asked = []

    def check_call(cmd, *a, **k):
        asked.append(cmd)
        raise Stop
    monkeypatch.setattr(entry.subprocess, "check_call", check_call)
    try:
        entry.build()
    except Stop:
        pass
    assert len(asked) == 1 and asked[0][0] == "make"
    out = subprocess.run(asked[0] + ["-n"], check=True, capture_output=True, text=True).stdout
    assert len([x for x in out.splitlines() if " -c " in x]) == 6
