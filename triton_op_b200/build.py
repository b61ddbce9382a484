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


CALLS_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden"]


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
    return ["g++"] + CALLS_FLAGS + flags + ["-o", CALLS_PATH, os.path.join(CSRC, CALLS_SOURCE)] + libs


def _object(source: str) -> str:
    if source == CALLS_SOURCE:
        return CALLS_PATH
    return os.path.join(LIB_DIR, os.path.splitext(source)[0] + ".o")


def _how(source: str, trace: bool = False) -> str:
    """What a product depends on besides its sources' times; kept beside it.  (No paths: a built tree may be moved.)"""
    if source != CALLS_SOURCE:
        return " ".join(_cuda_flags(trace))
    import sysconfig
    try:
        import torch
    except ImportError:
        return ""
    return " ".join(CALLS_FLAGS + [torch.__version__, str(torch._C._GLIBCXX_USE_CXX11_ABI), str(sysconfig.get_config_var("SOABI"))])


def _cuda_flags(trace: bool) -> list:
    return NVCC_FLAGS + (["-DPA_TRACE_BUILD"] if trace else [])


def _built_so(source: str, trace: bool) -> bool:
    """The product was built the way it would be built now."""
    try:
        with open(_object(source) + ".how") as f:
            return f.read() == _how(source, trace)
    except OSError:
        return False


def _note(source: str, trace: bool) -> None:
    with open(_object(source) + ".how", "w") as f:
        f.write(_how(source, trace))


def _older(target: str, source: str) -> bool:
    if not os.path.exists(target):
        return True
    built = os.path.getmtime(target)
    return any(os.path.getmtime(os.path.join(CSRC, d)) > built for d in [source] + SOURCES[source])


def needs_build(trace: bool = False) -> bool:
    return any(_older(CALLS_PATH if s == CALLS_SOURCE else LIB_PATH, s) or not _built_so(s, trace) for s in SOURCES)


def build(force: bool = False, verbose: bool = False, trace: bool = False) -> str:
    """Compile what is missing, older than its sources or built in another way (other flags; for the host
    calls, another torch or Python); returns the CUDA library's path.
    ``trace`` adds the instantiations that stamp SM clocks into ``PaDecodeParams.trace`` (tuning aid).
    The CUDA library needs neither torch nor its headers: it is there even where the host calls fail to compile,
    which is raised at the end."""
    if not force and not needs_build(trace):
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    cuda = [s for s in SOURCES if s != CALLS_SOURCE]
    todo = [s for s in SOURCES if force or _older(_object(s), s) or not _built_so(s, trace)]
    jobs, logs = {}, {}
    for s in todo:
        if os.path.exists(_object(s) + ".how"):
            os.remove(_object(s) + ".how")       # until it is built and linked
        try:
            command = (_calls_command() if s == CALLS_SOURCE else
                       [_nvcc()] + _cuda_flags(trace) + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", _object(s), os.path.join(CSRC, s)])
            jobs[s] = subprocess.Popen(command, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        except (OSError, ImportError) as e:      # no such compiler, no torch
            logs[s] = (str(e), -1)
    logs.update({s: (job.communicate()[0], job.returncode) for s, job in jobs.items()})
    failed = [s for s in todo if logs[s][1] != 0]
    for s in todo:
        if s in failed and os.path.exists(_object(s)):
            os.remove(_object(s))
        elif verbose:
            sys.stderr.write(logs[s][0])
    if not any(s in cuda for s in failed):
        proc = subprocess.run([_nvcc()] + NVCC_FLAGS + ["-shared", "-o", LIB_PATH] + [_object(s) for s in cuda], capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
        for s in todo:
            if s not in failed:
                _note(s, trace)
    if failed:
        raise RuntimeError("\n".join(f"the compiler failed on {s}:\n{logs[s][0]}" for s in failed))
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv or "--trace" in sys.argv, verbose="-v" in sys.argv, trace="--trace" in sys.argv))
