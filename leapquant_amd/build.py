"""Builds liblq.so (the HIP kernels + C ABI of include/lq.h) in-tree for gfx950, liblq_seq.so (the operators on whole
sequences, include/lq_seq.h) with lq_seq_call.so (their calls from Python), liblq_attn.so (the operators of softmax-attention
layers, include/lq_attn.h) with lq_attn_call.so, and liblq_probe.so (a streaming-read probe that bench.py times as the memory
system's ceiling; not part of the API).

    python -m leapquant_amd.build          # -> leapquant_amd/_build/liblq.so, liblq_seq.so, lq_seq_call.so, liblq_attn.so, ..

hipcc cross-compiles without a GPU.  Every HIP file gets `-Xclang -target-feature -Xclang -packed-fp32-ops` (no
packed FP32 instructions in the device code).
"""
import concurrent.futures
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "_build")
LIB = os.path.join(OUT, "liblq.so")
SOURCES = ("lq_step.hip", "lq_step_bf16.hip", "lq_flush.hip", "lq_dequant.hip", "lq_dense.hip", "lq_noalloc.hip")
SEQ_LIB = os.path.join(OUT, "liblq_seq.so")
SEQ_SOURCES = ("lq_seq_conv.hip", "lq_seq_norm.hip", "lq_seq_steps.hip", "lq_seq_delta.hip")
SEQ_CALL = os.path.join(OUT, "lq_seq_call.so")
ATTN_LIB = os.path.join(OUT, "liblq_attn.so")
ATTN_SOURCES = ("lq_attn_rope.hip", "lq_attn_core.hip")
ATTN_CALL = os.path.join(OUT, "lq_attn_call.so")
PROBE_LIB = os.path.join(OUT, "liblq_probe.so")
PROBE_SOURCES = ("lq_probe.hip",)
ARCH = os.environ.get("LQ_OFFLOAD_ARCH", "gfx950")


def hipcc():
    for p in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if p and (os.path.sep not in p or os.path.exists(p)):
            return p
    raise RuntimeError("hipcc not found")


def _compile_one(cc, flags, s, verbose):
    src = os.path.join(CSRC, s)
    obj = os.path.join(OUT, s.replace(".hip", ".o"))
    cmd = [cc] + flags + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("hipcc failed on %s:\n%s" % (s, r.stderr))
    if verbose:
        err = "\n".join(x for x in r.stderr.splitlines() if "packed-fp32-ops" not in x)
        if err.strip():
            print(err)
    return obj


def _compile_link(cc, flags, sources, lib, verbose):
    # one hipcc process per source file, run side by side (each is single-threaded)
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(len(sources), os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile_one(cc, flags, s, verbose), sources))
    tmp = lib + ".tmp"
    cmd = [cc, "--offload-arch=%s" % ARCH, "-shared", "-fPIC", "-o", tmp] + objs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n%s" % r.stderr)
    os.replace(tmp, lib)


def _build_call(lib, call):
    """The Python extension in front of a library: host C++ on torch's tensors, found beside the library it calls."""
    import torch
    t = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(hipcc())) if os.path.sep in hipcc() else "/opt/rocm"
    tmp = call + ".tmp"
    name = os.path.splitext(os.path.basename(call))[0]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           '-DLQ_TORCH_VERSION="%s"' % torch.__version__,
           os.path.join(CSRC, name + ".cpp"), "-o", tmp]
    cmd += ["-isystem" + d for d in (os.path.join(t, "include"), os.path.join(t, "include", "torch", "csrc", "api", "include"),
                                     os.path.join(rocm, "include"), sysconfig.get_paths()["include"])]
    cmd += ["-L" + os.path.join(t, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10_hip", "-lc10", "-L" + OUT,
            "-l" + os.path.basename(lib)[3:-3], "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("building %s.so failed:\n%s" % (name, r.stderr))
    os.replace(tmp, call)


def build(verbose=False):
    os.makedirs(OUT, exist_ok=True)
    cc = hipcc()
    # -amdgpu-atomic-optimizer-strategy=None: every atomic of the library is issued by one lane, so the optimizer's
    # wave-wide rewrite buys nothing, and its result broadcast (a readfirstlane right after the atomic) makes the wave
    # wait for the atomic's return at once -- the flush's schedule take would then hold wave 0 for its round trip
    flags = ["--offload-arch=%s" % ARCH, "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-Wno-inline-asm",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-mllvm", "-amdgpu-atomic-optimizer-strategy=None"]
    _compile_link(cc, flags, SOURCES, LIB, verbose)
    _compile_link(cc, flags, SEQ_SOURCES, SEQ_LIB, verbose)
    _build_call(SEQ_LIB, SEQ_CALL)
    _compile_link(cc, flags, ATTN_SOURCES, ATTN_LIB, verbose)
    _build_call(ATTN_LIB, ATTN_CALL)
    _compile_link(cc, flags, PROBE_SOURCES, PROBE_LIB, verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
