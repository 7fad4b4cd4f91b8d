"""ctypes binding of liblq.so (include/lq.h), liblq_seq.so (include/lq_seq.h) and liblq_attn.so (include/lq_attn.h).  The product path has no fallback: if a
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
ATTN_LIB_PATH = os.path.join(_HERE, "_build", "liblq_attn.so")
ATTN_CALL_PATH = os.path.join(_HERE, "_build", "lq_attn_call.so")
ABI_VERSION = 6
SEQ_ABI_VERSION = 1
ATTN_ABI_VERSION = 1
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


class LqPages(ctypes.Structure):
    _fields_ = [(n, c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + \
               [(n, c_ll) for n in ("page_ld", "row_ld", "head_ld", "s_page_ld", "s_row_ld", "s_head_ld")] + \
               [(n, c_int) for n in ("NP", "page", "HK", "D", "int8")]


class LqBatch(ctypes.Structure):
    _fields_ = [("loc", c_void_p), ("lens", c_void_p), ("table", c_void_p), ("table_ld", c_ll), ("width", c_int), ("N", c_int),
                ("T", c_int)]


class LqRows(ctypes.Structure):
    _fields_ = [("p", c_void_p), ("ld", c_ll), ("hd", c_ll)]


class LqRope(ctypes.Structure):
    _fields_ = [(n, LqRows) for n in ("q", "k", "v", "out")] + [(n, c_void_p) for n in ("q_weight", "k_weight", "inv_freq")] + \
               [(n, c_int) for n in ("HQ", "rot", "weight_bf16", "freq64", "interleaved")] + [("eps", c_float), ("offset", c_float)]


class LqAttention(ctypes.Structure):
    _fields_ = [(n, LqRows) for n in ("q", "gate", "out")] + [("HQ", c_int), ("window", c_int), ("scale", c_float)]


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
# the same of include/lq_attn.h
ATTN_SIGNATURES = {
    "lq_attn_abi_version": (c_int, []),
    "lq_rope_norm": (c_int, [ctypes.POINTER(LqRope), ctypes.POINTER(LqPages), ctypes.POINTER(LqBatch), c_void_p]),
    "lq_attend": (c_int, [ctypes.POINTER(LqAttention), ctypes.POINTER(LqPages), ctypes.POINTER(LqBatch), c_int, c_void_p, c_ll,
                          c_void_p]),
    "lq_attend_workspace": (c_ll, [ctypes.POINTER(LqAttention), ctypes.POINTER(LqPages), ctypes.POINTER(LqBatch), c_int]),
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
_ATTN_LIB = [None]
_ATTN_CALL = [None]


def _extension(name, path, version):
    """A Python extension in front of one of the libraries (raises if it has not been built, or for other structures than
    those of this binding, or against another torch)."""
    import torch
    if not os.path.exists(path):
        raise RuntimeError("%s is missing: build it with python -m leapquant_amd.build" % path)
    loader = importlib.machinery.ExtensionFileLoader(name, path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location(name, path, loader=loader))
    loader.exec_module(module)
    built = getattr(module, "ABI", None), getattr(module, "TORCH", None)
    if built != (version, torch.__version__):
        raise RuntimeError("%s.so: ABI %s with torch %s, expected %d with %s: rebuild it" % ((name,) + built + (version, torch.__version__)))
    return module


def seq_call():
    """The loaded lq_seq_call.so."""
    if _SEQ_CALL[0] is None:
        seq_lib()                        # the library behind it, of the same version
        _SEQ_CALL[0] = _extension("lq_seq_call", SEQ_CALL_PATH, SEQ_ABI_VERSION)
    return _SEQ_CALL[0]


def attn_lib():
    """The loaded liblq_attn.so (raises if it has not been built)."""
    if _ATTN_LIB[0] is None:
        _ATTN_LIB[0] = _load(ATTN_LIB_PATH, ATTN_SIGNATURES, "lq_attn_abi_version", ATTN_ABI_VERSION)
    return _ATTN_LIB[0]


def attn_call():
    """The loaded lq_attn_call.so."""
    if _ATTN_CALL[0] is None:
        attn_lib()                       # the library behind it, of the same version
        _ATTN_CALL[0] = _extension("lq_attn_call", ATTN_CALL_PATH, ATTN_ABI_VERSION)
    return _ATTN_CALL[0]


_ERR = {-1: "bad argument (unsupported shape / size / pointer)", -2: "HIP launch error",
        -3: "more (row, head) pairs than the static due list of lq_decode_noalloc holds (N * HV <= 65536)"}


def check(rc, what):
    if rc != 0:
        raise RuntimeError("%s failed: %s (status %d)" % (what, _ERR.get(rc, "unknown"), rc))
