"""The host checks of kvmem_hip_slot_map, kvmem_hip_qkv_rows and
kvmem_hip_attention, without a GPU: tests/operator_refusals.cpp is linked with
the library and makes calls that must all be refused, with a message, before
any HIP call; the argument structs of the Python view have the header's sizes."""
from __future__ import annotations

import os
import subprocess

import pytest

from conftest import PKG_DIR, ROOT, load_pkg

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", f"-I{ROOT / 'include'}", f"-I{PKG_DIR / 'csrc'}"]


def build(tmp, src):
    load_pkg()
    exe = tmp / "refusals"
    cmd = [HIPCC, *FLAGS, str(src), "-x", "none", str(PKG_DIR / "libkvmem_hip.so"), f"-Wl,-rpath,{PKG_DIR}", "-o",
           str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return exe


def test_every_bad_call_is_refused(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc is not installed")
    r = subprocess.run([str(build(tmp_path, ROOT / "tests" / "operator_refusals.cpp"))], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0 and "all refused" in r.stdout, r.stdout + r.stderr


def test_argument_structs_match_the_header(tmp_path):
    kv = load_pkg()
    src = tmp_path / "sizes.cpp"
    src.write_text('#include "kvmem_internal.hpp"\n#include <cstdio>\nint main() { std::printf("%zu %zu %zu %zu %zu %zu", '
                   "sizeof(kvmem_hip_slot_map_args), sizeof(kvmem_hip_qkv_args), sizeof(kvmem_hip_attn_args), "
                   "offsetof(kvmem_hip_slot_map_args, n_missing), offsetof(kvmem_hip_qkv_args, xf), "
                   "offsetof(kvmem_hip_attn_args, workspace)); }\n")
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc is not installed")
    out = subprocess.run([str(build(tmp_path, src))], capture_output=True, text=True, timeout=120).stdout
    C = kv.C
    assert [int(x) for x in out.split()] == [C.sizeof(kv.SlotMapArgs), C.sizeof(kv.QkvArgs), C.sizeof(kv.AttnArgs),
                                             kv.SlotMapArgs.n_missing.offset, kv.QkvArgs.xf.offset,
                                             kv.AttnArgs.workspace.offset]
