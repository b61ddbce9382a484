"""In-tree build of the CUDA library (``python -m triton_op_b200.build``).

nvcc turns the sources in ``csrc/`` into ``lib/libpa_decode_sm100.so`` for sm_100a, one object each
(side by side, and only what is older than its sources), and the host compiler turns ``csrc/pa_calls.cpp``
into ``lib/pa_calls.so``, the ordinary calls' way from torch tensors to that library.  nvcc
cross-compiles, so this also runs on a machine without a GPU.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libpa_decode_sm100.so")
CALLS_PATH = os.path.join(LIB_DIR, "pa_calls.so")
CALLS_SOURCE = "pa_calls.cpp"
_COMMON = ["pa_common.cuh", "pa_params.cuh", "pa_host.h", os.path.join("..", "..", "include", "pa_decode_sm100.h")]
# source -> headers it includes
SOURCES = {
    "pa_decode_sm100.cu": _COMMON + [
        "pa_partition_fp8.cuh", "pa_partition_bf16.cuh", "pa_partition_tc.cuh", "pa_tcgen05.cuh", "pa_reduce.cuh",
        "pa_cache_write.cuh", "pa_exchange.cuh", "pa_stream_probe.cuh"],
    CALLS_SOURCE: ["pa_places.h", os.path.join("..", "..", "include", "pa_decode_sm100.h")],
    "pa_blocks_sm100.cu": _COMMON + ["pa_places.h", "pa_block_score.cuh", "pa_block_select.cuh", "pa_cache_append.cuh", "pa_tcgen05.cuh"],
}

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: cannot build the sm_100a library")
    return exe


def _calls_command() -> list:
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    flags = [f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + sysconfig.get_paths()["include"]]
    for path in include:
        flags += ["-isystem", path]
    libs = ["-L" + os.path.join(root, "lib")] + ["-l" + n for n in ("c10", "c10_cuda", "torch_cpu", "torch_cuda", "torch", "torch_python")]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden"] + flags + ["-o", CALLS_PATH, os.path.join(CSRC, CALLS_SOURCE)] + libs


def _object(source: str) -> str:
    if source == CALLS_SOURCE:
        return CALLS_PATH
    return os.path.join(LIB_DIR, os.path.splitext(source)[0] + ".o")


def _stale(target: str, source: str) -> bool:
    if not os.path.exists(target):
        return True
    built = os.path.getmtime(target)
    return any(os.path.getmtime(os.path.join(CSRC, d)) > built for d in [source] + SOURCES[source])


def needs_build() -> bool:
    return any(_stale(CALLS_PATH if s == CALLS_SOURCE else LIB_PATH, s) for s in SOURCES)


def build(force: bool = False, verbose: bool = False, trace: bool = False) -> str:
    """Compile the library if it is missing or older than its sources; returns its path.
    ``trace`` adds the instantiations that stamp SM clocks into ``PaDecodeParams.trace`` (tuning aid)."""
    if not force and not needs_build():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    flags = NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + (["-DPA_TRACE_BUILD"] if trace else [])
    jobs = {s: subprocess.Popen(_calls_command() if s == CALLS_SOURCE else
                                [_nvcc()] + flags + ["-c", "-o", _object(s), os.path.join(CSRC, s)],
                                stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
            for s in SOURCES if force or _stale(_object(s), s)}
    logs = {s: (job.communicate()[0], job.returncode) for s, job in jobs.items()}
    for s, (text, code) in logs.items():
        if code != 0:
            if os.path.exists(_object(s)):
                os.remove(_object(s))
            raise RuntimeError(f"the compiler failed on {s}:\n{text}")
        if verbose:
            sys.stderr.write(text)
    proc = subprocess.run([_nvcc()] + NVCC_FLAGS + ["-shared", "-o", LIB_PATH] + [_object(s) for s in SOURCES if s != CALLS_SOURCE],
                          capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv or "--trace" in sys.argv, verbose="-v" in sys.argv, trace="--trace" in sys.argv))
