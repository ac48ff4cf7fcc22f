"""A host shim over the rules that choose a microscaled product's kernel (csrc/q4d_mx.h).  Compiled from the text below
when first asked for; it holds no device code and launches nothing."""

import ctypes
import subprocess
import tempfile
from functools import lru_cache
from pathlib import Path

from llm_accelerator_amd import _lib

ROOT = Path(__file__).resolve().parents[1]
ROCM = Path("/opt/rocm")
SOURCE = r"""
#include "q4d_mx.h"
using namespace q4d;
static void give(const MxForm& f, int* out) { out[0] = f.path; out[1] = f.mt; out[2] = f.nt; out[3] = f.waves; }
extern "C" {
void shim_mx_form(int M, int N, int K, int kind, int* out) { give(mx_form(M, N, K, (MxKind)kind), out); }
void shim_mx_score_form(int M, int N, int K, int* out) { give(mx_score_form(M, N, K), out); }
}
"""
PATHS = ("rows", "head", "tiles")


@lru_cache(maxsize=None)
def load() -> ctypes.CDLL:
    _lib.load()
    with tempfile.TemporaryDirectory() as d:
        src, so = Path(d) / "shim.cpp", Path(d) / "shim.so"
        src.write_text(SOURCE)
        subprocess.run([str(ROCM / "llvm/bin/clang++"), "-shared", "-fPIC", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROOT / 'llm_accelerator_amd' / 'csrc'}", f"-I{ROCM / 'include'}", str(src),
                        str(_lib.LIB_PATH), "-o", str(so)], check=True)
        lib = ctypes.CDLL(str(so))
    i, p = ctypes.c_int, ctypes.c_void_p
    lib.shim_mx_form.argtypes, lib.shim_mx_form.restype = [i, i, i, i, p], None
    lib.shim_mx_score_form.argtypes, lib.shim_mx_score_form.restype = [i, i, i, p], None
    return lib


def form(m: int, n: int, k: int, codes: bool) -> tuple:
    """(path, blocks' rows of x, of weights, waves), the rows in units of 16 (tiles: 32 and 128)."""
    out = (ctypes.c_int * 4)()
    load().shim_mx_form(m, n, k, 0 if codes else 2, out)
    return (PATHS[out[0]], *out[1:])


def score_form(m: int, n: int, k: int) -> tuple:
    out = (ctypes.c_int * 4)()
    load().shim_mx_score_form(m, n, k, out)
    return (PATHS[out[0]], *out[1:])
