"""CPU: what the build files build, and which libraries a process maps."""
import os
import subprocess
import sys

import pytest

from transformer_vae_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def planned(*goals):
    """The commands that make would run for a tree without anything built (nothing is run)."""
    return subprocess.run(["make", "-n", "-B", "-C", _lib.CSRC, *goals], capture_output=True, text=True, check=True).stdout


def test_the_library_is_built_without_torch():
    # the C interface's users have neither torch's headers nor, perhaps, a Python
    plan = planned()
    assert "libtvae_hip.so" in plan and "host.cpp" not in plan and "python" not in plan
    plan = planned("all", "host")
    assert "libtvae_hip.so" in plan and "host.cpp" in plan


def test_the_nodes_call_the_library_that_was_loaded(tmp_path):
    """Where another build of the library is put in the default's place, the autograd nodes follow, and no second copy is mapped."""
    other = tmp_path / "libtvae_other.so"
    other.write_bytes(open(_lib.LIB_PATH, "rb").read())
    code = (f"from transformer_vae_amd import _lib; _lib.LIB_PATH = {str(other)!r}; _lib.host(); "
            "print({l.split()[-1] for l in open('/proc/self/maps') if 'libtvae' in l})")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=True, cwd=ROOT).stdout
    assert eval(out) == {str(other)}


def test_a_library_without_the_operators_is_named():
    code = ("import ctypes; from transformer_vae_amd import _lib; h = _lib.host(); "
            "import pytest\nwith pytest.raises(RuntimeError, match='tvae_last_error'): h.bind(ctypes.CDLL('libc.so.6')._handle)")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)


def test_the_nodes_follow_torch(tmp_path):
    """Built again where torch or Python have changed since, with the C++ ABI that torch was built with."""
    import torch
    pkg = tmp_path / "transformer_vae_amd"
    for d in (pkg / "csrc", tmp_path / "include"):
        d.mkdir(parents=True)
    for f in ("Makefile", "host.cpp"):
        (pkg / "csrc" / f).write_bytes(open(os.path.join(_lib.CSRC, f), "rb").read())
    (tmp_path / "include" / "tvae_hip.h").write_bytes(open(_lib.HEADER, "rb").read())
    (tmp_path / "bin").mkdir()
    cxx = tmp_path / "bin" / "cxx"
    cxx.write_text('#!/bin/sh\necho "$@" >> ' + str(tmp_path / "ran") + '\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"\n')
    cxx.chmod(0o755)
    make = lambda: subprocess.run(["make", "-C", str(pkg / "csrc"), "host", f"CXX={cxx}", f"PYTHON={sys.executable}"], check=True, capture_output=True)
    runs = lambda: (tmp_path / "ran").read_text().splitlines()
    make(), make()
    assert len(runs()) == 1
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}" in runs()[0]
    (stamp,) = [p for p in (pkg / "csrc").iterdir() if torch.__version__ in p.read_text(errors="replace")]
    stamp.write_text(stamp.read_text().replace(torch.__version__, "1.0"))
    make(), make()
    assert len(runs()) == 2


def test_other_flags_build_everything_again():
    # objects of a tree from before a flag was set must not stay (that no packed fp32 instructions are used is one of them)
    plan = subprocess.run(["make", "-n", "-W", "Makefile", "-C", _lib.CSRC], capture_output=True, text=True, check=True).stdout
    sources = [f for f in os.listdir(_lib.CSRC) if f.endswith(".hip")]
    lines = plan.splitlines()
    for f in sources:
        (line,) = [l for l in lines if f"-c {f}" in l]
        assert "-packed-fp32-ops" in line


def test_variants_hold_every_source_built_as_the_library_is(tmp_path):
    """tools/build_variant.sh: a variant that lacks a source lacks its entry points, and the package cannot load it."""
    pkg = tmp_path / "transformer_vae_amd"
    (pkg / "csrc").mkdir(parents=True)
    (tmp_path / "tools").mkdir()
    (tmp_path / "tools" / "build_variant.sh").write_bytes(open(os.path.join(ROOT, "tools", "build_variant.sh"), "rb").read())
    sources = sorted(f[:-4] for f in os.listdir(_lib.CSRC) if f.endswith(".hip"))
    (pkg / "csrc" / "Makefile").write_bytes(open(os.path.join(_lib.CSRC, "Makefile"), "rb").read())
    for f in sources:
        (pkg / "csrc" / (f + ".hip")).write_text("TVAE_SPLITS\n" if f == "mmd_q32" else "")
        (pkg / "csrc" / (f + ".o")).write_text(f)
    for f in ("tvae_common.h", "mmd_common.h", "mmd_q32.h", "norm_common.h", "norm_rows.h"):
        (pkg / "csrc" / f).write_text("")
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "tvae_hip.h").write_text("")
    hipcc = tmp_path / "hipcc"
    hipcc.write_text('#!/bin/sh\necho "$@" >> ' + str(tmp_path / "ran") + '\nwhile [ "$1" != -o ]; do shift; done\necho variant > "$2"\n')
    hipcc.chmod(0o755)
    subprocess.run(["bash", str(tmp_path / "tools" / "build_variant.sh"), "x", "-DTVAE_SPLITS=3"], check=True, capture_output=True,
                   env={**os.environ, "HIPCC": str(hipcc)})
    compiled, linked = (tmp_path / "ran").read_text().splitlines()
    assert "-c mmd_q32.hip" in compiled and "-DTVAE_SPLITS=3" in compiled and "-packed-fp32-ops" in compiled and "-fno-slp-vectorize" in compiled
    assert {os.path.basename(w)[:-2] for w in linked.split() if w.endswith(".o")} == set(sources)
    assert (pkg / "variants" / "libtvae_x.so").exists()
