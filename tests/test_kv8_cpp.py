"""The 8-bit KV cache through the C++ host side (include/infr_hip.hpp, tests/cpp/kv8.cpp), and its structs as the binding
notes write them in Rust."""
import ctypes
import os
import re
import subprocess

import pytest

from infr_amd import backend as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CPP = os.path.join(ROOT, "tests", "cpp")
EXE = os.path.join(CPP, "_build", "kv8")


def exe():
    if not os.path.exists(EXE):
        from oracle import oracle  # noqa: F401  (builds the library the other program links)
        B.load_library()
        subprocess.run(["make", "-C", CPP], check=True, capture_output=True)
    return EXE


def test_without_a_device_it_refuses_to_run():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    r = subprocess.run([exe()], capture_output=True, text=True)
    assert r.returncode == 99 and "no usable gfx950 device" in r.stdout


@pytest.mark.gpu
def test_prompt_single_tokens_and_an_eviction():
    r = subprocess.run([exe()], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout[-3000:] + r.stderr[-1000:]


def test_the_rust_mirror_of_the_parameters_matches_the_c_header(tmp_path):
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    body = re.search(r"pub struct HipKv8 \{([^}]*)\}", text).group(1)
    rust = [tuple(x.strip() for x in f.split(":")) for f in body.split(",") if f.strip()]
    kinds = {"u32": ctypes.c_uint32, "i32": ctypes.c_int, "f32": ctypes.c_float}
    assert [(n, kinds[t]) for n, t in rust] == [(n, t) for n, t in B._Kv8Params._fields_]
    src = tmp_path / "p.c"
    lines = "".join(f'printf("%zu\\n", offsetof(infr_hip_kv8_params_t, {n}));' for n, _ in rust)
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "infr_hip.h"\n'
                   f'int main(void) {{ {lines} printf("%zu\\n", sizeof(infr_hip_kv8_params_t)); return 0; }}')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "p"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(B._Kv8Params, n).offset for n, _ in rust] + [ctypes.sizeof(B._Kv8Params)]
