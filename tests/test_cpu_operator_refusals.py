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
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc is not installed")
    structs = {"kvmem_hip_slot_map_args": kv.SlotMapArgs, "kvmem_hip_qkv_args": kv.QkvArgs,
               "kvmem_hip_attn_args": kv.AttnArgs}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'std::printf("%zu\\n", sizeof({name}));')
        want.append(kv.C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'std::printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "sizes.cpp"
    src.write_text("#include <cstddef>\n#include <cstdio>\n#include \"kvmem_hip.h\"\nint main() {\n" + "\n".join(lines)
                   + "\n}\n")
    out = subprocess.run([str(build(tmp_path, src))], capture_output=True, text=True, timeout=120).stdout
    assert [int(x) for x in out.split()] == want
