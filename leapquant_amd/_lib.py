"""ctypes binding of liblq.so (include/lq.h) and liblq_seq.so (include/lq_seq.h).  The product path has no fallback: if a
library is missing or a call fails, this raises."""
import ctypes
import importlib.machinery
import importlib.util
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_build", "liblq.so")
SEQ_LIB_PATH = os.path.join(_HERE, "_build", "liblq_seq.so")
SEQ_CALL_PATH = os.path.join(_HERE, "_build", "lq_seq_call.so")
ABI_VERSION = 6
SEQ_ABI_VERSION = 1
SCHED_INTS = 512           # include/lq.h: LQ_SCHED_INTS

c_void_p, c_int, c_float, c_ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong


class LqState(ctypes.Structure):
    _fields_ = [("ssm", c_void_p), ("slot_stride", c_ll), ("Kbuf", c_void_p), ("Ubuf", c_void_p),
                ("Wbuf", c_void_p), ("Pbuf", c_void_p), ("Gbuf", c_void_p), ("hcnt", c_void_p),
                ("NS", c_int), ("HV", c_int), ("H", c_int), ("K", c_int), ("V", c_int), ("L", c_int), ("R", c_int),
                ("ctl", c_void_p), ("qmax", c_float), ("sched", c_void_p)]


class LqStepIO(ctypes.Structure):
    _fields_ = [("mixed", c_void_p), ("a", c_void_p), ("b", c_void_p), ("A_log", c_void_p), ("dt_bias", c_void_p),
                ("idx", c_void_p), ("out", c_void_p), ("N", c_int), ("scale", c_float), ("gate_bf16", c_int)]


class LqConv(ctypes.Structure):
    _fields_ = [("state", c_void_p), ("weight", c_void_p), ("bias", c_void_p), ("slot_stride", c_ll),
                ("ch_stride", c_ll), ("tap_stride", c_ll), ("W", c_int), ("silu", c_int), ("NS", c_int)]


class LqSeqs(ctypes.Structure):
    _fields_ = [("loc", c_void_p), ("idx", c_void_p), ("src", c_void_p), ("N", c_int), ("T", c_int)]


class LqDelta(ctypes.Structure):
    _fields_ = [("S", c_void_p), ("slot_stride", c_ll)] + [(n, c_int) for n in ("NS", "HV", "H", "K", "V")] + \
               [(n, c_void_p) for n in ("mixed", "a", "b", "A_log", "dt_bias", "out")] + \
               [(n, c_ll) for n in ("mixed_ld", "a_ld", "b_ld")] + \
               [("scale", c_float), ("gate_bf16", c_int), ("kda", c_int), ("glb", c_float)]


class LqNorm(ctypes.Structure):
    _fields_ = [(n, c_void_p) for n in ("x", "z", "weight", "res", "out")] + \
               [(n, c_ll) for n in ("x_ld", "x_hd", "z_ld", "z_hd", "o_ld", "o_hd")] + \
               [(n, c_int) for n in ("rows", "heads", "D")] + [(n, c_float) for n in ("eps", "scale", "offset")] + \
               [("act", c_int), ("weight_bf16", c_int)]


# exported symbol -> (restype, argtypes); must match include/lq.h
SIGNATURES = {
    "lq_abi_version": (c_int, []),
    "lq_gdn_step": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), c_void_p]),
    "lq_gdn_step_conv": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), ctypes.POINTER(LqConv), c_void_p]),
    "lq_kda_step": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), c_float, c_void_p]),
    "lq_kda_decode": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), c_float, c_void_p, c_void_p]),
    "lq_gdn_decode": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), ctypes.POINTER(LqConv), c_void_p,
                              c_void_p]),
    "lq_gdn_decode_deferred": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), ctypes.POINTER(LqConv),
                                       c_void_p, c_void_p]),
    "lq_flush": (c_int, [ctypes.POINTER(LqState), c_void_p, c_void_p, c_int, c_int, c_float, c_void_p]),
    "lq_quantize": (c_int, [ctypes.POINTER(LqState), c_void_p, c_void_p, c_int, c_float, c_void_p]),
    "lq_dequant": (c_int, [ctypes.POINTER(LqState), c_void_p, c_int, c_float, c_void_p]),
    "lq_kda_dequant": (c_int, [ctypes.POINTER(LqState), c_void_p, c_int, c_float, c_void_p]),
    "lq_kda_checkpoint": (c_int, [ctypes.POINTER(LqState), c_void_p, c_void_p, c_int, c_float, c_void_p]),
    "lq_lowrank": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p]),
    "lq_conv_update": (c_int, [ctypes.POINTER(LqConv), c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]),
    "lq_dense_step": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, ctypes.POINTER(LqStepIO),
                              c_void_p]),
    "lq_decode_noalloc": (c_int, [ctypes.POINTER(LqState), ctypes.POINTER(LqStepIO), c_void_p, c_int, c_float,
                                  c_void_p]),
}

# the same of include/lq_seq.h; the structures go as addresses, so that a caller may hand over their bytes (PACK_*), which a
# call from Python builds in a quarter of a structure's time
SEQ_SIGNATURES = {
    "lq_seq_abi_version": (c_int, []),
    "lq_delta_steps": (c_int, [c_void_p, c_void_p, c_void_p]),
    "lq_delta_prefill": (c_int, [c_void_p, c_void_p, c_void_p, c_ll, c_void_p]),
    "lq_delta_workspace": (c_ll, [c_void_p, c_void_p]),
    "lq_delta_check": (c_int, [c_void_p, c_void_p, c_int]),
    "lq_conv_seq": (c_int, [c_void_p, c_void_p, c_void_p, c_ll, c_void_p, c_int, c_void_p]),
    "lq_gated_norm": (c_int, [c_void_p, c_void_p]),
    "lq_add_norm": (c_int, [c_void_p, c_void_p]),
}
_SEQS, _DELTA, _NORM = struct.Struct("@3P2i0P"), struct.Struct("@Pq5i6P3qf2if0P"), struct.Struct("@5P6q3i3f2i0P")
for _layout, _type in ((_SEQS, LqSeqs), (_DELTA, LqDelta), (_NORM, LqNorm)):
    assert _layout.size == ctypes.sizeof(_type)
pack_seqs, pack_delta, pack_norm = _SEQS.pack, _DELTA.pack, _NORM.pack

_LIB = [None]
_SEQ_LIB = [None]


def _load(path, signatures, abi, version):
    if not os.path.exists(path):
        raise RuntimeError("%s is missing (%s): build it with `python -m leapquant_amd.build`"
                           % (os.path.basename(path), path))
    L = ctypes.CDLL(path)
    v = getattr(L, abi)() if hasattr(L, abi) else None
    if v != version:
        raise RuntimeError("%s ABI %s, expected %d: rebuild it" % (os.path.basename(path), v, version))
    for name, (res, args) in signatures.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    return L


def lib():
    """The loaded liblq.so (raises if it has not been built)."""
    if _LIB[0] is None:
        _LIB[0] = _load(LIB_PATH, SIGNATURES, "lq_abi_version", ABI_VERSION)
    return _LIB[0]


def seq_lib():
    """The loaded liblq_seq.so (raises if it has not been built)."""
    if _SEQ_LIB[0] is None:
        _SEQ_LIB[0] = _load(SEQ_LIB_PATH, SEQ_SIGNATURES, "lq_seq_abi_version", SEQ_ABI_VERSION)
    return _SEQ_LIB[0]


_SEQ_CALL = [None]


def seq_call():
    """The loaded lq_seq_call.so, a Python extension (raises if it has not been built, or for other structures than those of
    this binding, or against another torch)."""
    if _SEQ_CALL[0] is None:
        import torch
        seq_lib()                        # the library behind it, of the same version
        if not os.path.exists(SEQ_CALL_PATH):
            raise RuntimeError("%s is missing: build it with python -m leapquant_amd.build" % SEQ_CALL_PATH)
        loader = importlib.machinery.ExtensionFileLoader("lq_seq_call", SEQ_CALL_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("lq_seq_call", SEQ_CALL_PATH, loader=loader))
        loader.exec_module(module)
        built = getattr(module, "ABI", None), getattr(module, "TORCH", None)
        if built != (SEQ_ABI_VERSION, torch.__version__):
            raise RuntimeError("lq_seq_call.so: ABI %s with torch %s, expected %d with %s: rebuild it"
                               % (built + (SEQ_ABI_VERSION, torch.__version__)))
        _SEQ_CALL[0] = module
    return _SEQ_CALL[0]


_ERR = {-1: "bad argument (unsupported shape / size / pointer)", -2: "HIP launch error",
        -3: "more (row, head) pairs than the static due list of lq_decode_noalloc holds (N * HV <= 65536)"}


def check(rc, what):
    if rc != 0:
        raise RuntimeError("%s failed: %s (status %d)" % (what, _ERR.get(rc, "unknown"), rc))
