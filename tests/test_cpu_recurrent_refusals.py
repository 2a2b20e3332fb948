"""The host checks of kvmem_hip_conv_rows, kvmem_hip_linear_attention and
kvmem_hip_verify_draft, without a GPU (tests/recurrent_refusals.cpp); the argument
structs of the Python view have the header's sizes and offsets."""
from __future__ import annotations

import os
import subprocess

import pytest

from conftest import ROOT, load_pkg
from test_cpu_operator_refusals import HIPCC, build

needs_hipcc = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is not installed")


@needs_hipcc
def test_every_bad_call_is_refused(tmp_path):
    r = subprocess.run([str(build(tmp_path, ROOT / "tests" / "recurrent_refusals.cpp"))], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0 and "all refused" in r.stdout, r.stdout + r.stderr


@needs_hipcc
def test_argument_structs_match_the_header(tmp_path):
    kv = load_pkg()
    lines, want = [], []
    for name, cls in {"kvmem_hip_conv_args": kv.ConvArgs, "kvmem_hip_linear_args": kv.LinearArgs,
                      "kvmem_hip_verify_args": kv.VerifyArgs}.items():
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
