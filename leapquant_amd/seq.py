"""Operators that take whole sequences through a linear-attention layer (HIP, include/lq_seq.h), beside the one-token decode
of `kernels` and `state`:

  conv_prefill     the depthwise causal conv1d over a ragged batch of prompts, its taps in the conv cache's slots
  delta_prefill    the gated delta rule of Gated DeltaNet over a ragged batch, in chunks on the matrix cores
  delta_steps      the same recurrence token by token (GDN, and KDA with its gate a key channel): single and drafted tokens
  gated_norm       the norm of the block's output times its gate
  add_norm         the residual add and the norm before the next block

A ragged batch is given by `loc` [N + 1] (sequence n holds the packed tokens loc[n] .. loc[n + 1] - 1), `idx` [N], the slots
that take the sequences' last states, and `src` [N], the slots they start from (None: idx, in place).  A src outside the
cache's slots 1 .. NS - 1 (0, -1) starts from zero; an idx outside them makes a padding sequence: outputs zero, no slot written.
As in the decode calls slot 0 is padding.  The caller keeps the slots that one sequence of a call writes apart from those
that another reads or writes.  Calls launch on the current stream of their tensors' device, never synchronise and can be
captured in a graph; they work forward only (no autograd).
"""
import ctypes

import torch

from . import _lib
from .kernels import GDN_DIMS, _raw_stream, conv_struct

_ACT = {"silu": 0, "sigmoid": 1}
_F32, _BF16, _I32 = torch.float32, torch.bfloat16, torch.int32
_KDA_DIMS = ((128, 128),)
_NOT_PLAIN = 1           # lq_seq_call: arguments to be converted or refused below; nothing was launched


def _on(dev, **tensors):
    """Every tensor on GPU `dev` (a device index; -1: the host)."""
    for name, t in tensors.items():
        if t is not None and t.get_device() != dev:
            raise ValueError("%s is on %s, expected %s" % (name, t.device, "cuda:%d" % dev if dev >= 0 else "cpu"))
    if dev < 0:
        raise ValueError("liblq takes GPU tensors only, got cpu tensors")


def _index(t, n, name):
    """An int32 index tensor of n elements; other integer types are converted."""
    if t.shape != (n,):
        raise ValueError("%s: 1-D with %d elements expected, got shape %s" % (name, n, tuple(t.shape)))
    if t.dtype is _I32 and t.is_contiguous():
        return t
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype is torch.bool:
        raise TypeError("%s: integers expected, got %s" % (name, t.dtype))
    return t.to(_I32).contiguous()


def _batch(idx, loc, src, T):
    """lq_seqs' bytes, and the index tensors that have to live until the launch."""
    N = idx.shape[0] if idx.dim() else -1
    idx, loc = _index(idx, N, "idx"), _index(loc, N + 1, "loc")
    if src is None:
        return _lib.pack_seqs(loc.data_ptr(), idx.data_ptr(), 0, N, T), (idx, loc)
    src = _index(src, N, "src")
    return _lib.pack_seqs(loc.data_ptr(), idx.data_ptr(), src.data_ptr(), N, T), (idx, loc, src)


def _rows(t, T, C, name, align):
    """Row stride of a bf16 [T, C] with packed rows; its start and stride are multiples of `align` elements."""
    if t.dtype is not _BF16:
        raise TypeError("%s: dtype %s, expected torch.bfloat16" % (name, t.dtype))
    if t.shape != (T, C):
        raise ValueError("%s: shape %s, expected (%d, %d)" % (name, tuple(t.shape), T, C))
    ld, one = t.stride()
    if T < 2:
        ld = -(-C // align) * align              # a single row has no stride of its own
    if (one != 1 and C > 1) or ld < C or ld % align or t.data_ptr() % (2 * align):
        raise ValueError("%s: packed rows expected, with their start and stride aligned to %d bytes (strides %s)"
                         % (name, 2 * align, t.stride()))
    return ld


def _param(t, n, name):
    """A gate parameter of n values in fp32 or bf16 as the kernels read it; other float types are converted."""
    if t.numel() != n:
        raise ValueError("%s: %d elements expected, got shape %s" % (name, n, tuple(t.shape)))
    if t.dtype is not _F32 and t.dtype is not _BF16:
        t = t.detach().float()
    return t if t.is_contiguous() else t.detach().contiguous()


def _delta(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src, scale, kda, glb, chunks=False):
    """Bytes of lq_delta and lq_seqs, and the tensors that have to live until the launch."""
    if S.dtype is not _F32 or S.dim() != 4:
        raise TypeError("S: fp32 [NS, HV, V, K] expected, got %s %s" % (S.dtype, tuple(S.shape)))
    NS, HV, V, K = S.shape
    if (K, V) not in (_KDA_DIMS if kda else GDN_DIMS):
        raise ValueError("head dims (K, V) in %s, got (%d, %d)" % (_KDA_DIMS if kda else GDN_DIMS, K, V))
    if H <= 0 or HV % H:
        raise ValueError("H = %d key heads do not divide HV = %d value heads" % (H, HV))
    SS, *packed = S.stride()
    if NS < 2:
        SS = HV * V * K
    if packed != [V * K, K, 1] or S.data_ptr() % 16 or SS % 4 or SS < HV * V * K:
        raise ValueError("S: packed [HV, V, K] slots expected, 16-byte aligned with a stride divisible by 4 (strides %s)"
                         % (S.stride(),))
    if mixed.dim() != 2:
        raise ValueError("mixed: [T, 2HK + HV V] expected, got shape %s" % (tuple(mixed.shape),))
    T, KA = mixed.shape[0], K if kda else 1
    mixed_ld = _rows(mixed, T, 2 * H * K + HV * V, "mixed", 8)
    if kda and a.dim() == 3:
        if a.shape[1:] != (HV, K) or a.stride()[1:] != (K, 1):
            raise ValueError("a: packed [T, HV, K] rows expected, got shape %s strides %s" % (tuple(a.shape), a.stride()))
        a = a.flatten(1)
    a_ld, b_ld = _rows(a, T, HV * KA, "a", 4 if kda else 1), _rows(b, T, HV, "b", 1)
    if out.dtype is not _BF16 or out.shape != (T, HV, V) or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out: contiguous 16-byte aligned bf16 [T, HV, V] expected")
    if chunks and (T * HV > 1 << 30 or mixed_ld > 1 << 24):
        raise ValueError("at most 2^30 tokens times value heads and rows of 2^24 elements in a call, got %d and %d"
                         % (T * HV, mixed_ld))
    A_log, dt_bias = _param(A_log, HV, "A_log"), _param(dt_bias, HV * KA, "dt_bias")
    seqs, live = _batch(idx, loc, src, T)
    _on(S.get_device(), mixed=mixed, a=a, b=b, A_log=A_log, dt_bias=dt_bias, idx=idx, loc=loc, out=out, src=src)
    d = _lib.pack_delta(S.data_ptr(), SS, NS, HV, H, K, V, mixed.data_ptr(), a.data_ptr(), b.data_ptr(), A_log.data_ptr(),
                        dt_bias.data_ptr(), out.data_ptr(), mixed_ld, a_ld, b_ld, K ** -0.5 if scale is None else scale,
                        (A_log.dtype is _BF16) + 2 * (dt_bias.dtype is _BF16), kda, glb)
    return d, seqs, (live, a, A_log, dt_bias)


def _rule(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src, scale, kda, glb, chunks, before=None):
    """The gated delta rule in chunks or token by token.  `before`, a callable, is called when nothing is left that refuses
    the call (arguments checked, workspace taken), right before the launch."""
    name = "lq_delta_prefill" if chunks else "lq_delta_steps"
    rc = _lib.seq_call().delta(S, mixed, a, b, A_log, dt_bias, idx, loc, out, src, H, scale, kda, glb, chunks, before)
    if rc != _NOT_PLAIN:
        return _lib.check(rc, name)
    d, seqs, live = _delta(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src, scale, kda, glb, chunks=chunks)
    L = _lib.seq_lib()
    with torch.cuda.device(S.get_device()):
        _lib.check(L.lq_delta_check(d, seqs, chunks), name)
        n = L.lq_delta_workspace(d, seqs) if chunks else 0
        work = torch.empty(n, dtype=torch.uint8, device=S.device) if n > 0 else None
        if before is not None:
            before()
        if chunks:
            _lib.check(L.lq_delta_prefill(d, seqs, work.data_ptr() if n > 0 else None, n, _raw_stream(S)), name)
        else:
            _lib.check(L.lq_delta_steps(d, seqs, _raw_stream(S)), name)


def delta_prefill(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src=None, scale=None):
    """The gated delta rule of Gated DeltaNet over the prompts of a ragged batch, in chunks on the matrix cores.

    S: fp32 state cache [NS, HV, V, K] (the fp32 states of the slots src are read, those of idx written).  mixed: bf16
    [T, 2HK + HV V] after the conv, q | k | v; a, b: bf16 [T, HV] raw gates.  The three may be column ranges of wider rows.
    A_log, dt_bias: [HV].  out: bf16 [T, HV, V].  scale: of the queries, K^-1/2 by default.  Gates, norms and state as the
    decode step's, with beta = sigmoid(b) not rounded.  A NaN or infinity in a token reaches all tokens of its chunk of 32."""
    _rule(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src, scale, False, 0.0, True)


def delta_steps(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src=None, scale=None, kda=False, gate_lower_bound=0.0):
    """The gated delta rule token by token: for single tokens, drafted tokens and short prompts.  Arguments as
    `delta_prefill`; kda: Kimi Delta Attention, with a [T, HV, K] and dt_bias [HV * K] and, where gate_lower_bound is not
    0, its bounded gate gate_lower_bound * sigmoid(exp(A_log) (a + dt_bias))."""
    if gate_lower_bound and not kda:
        raise ValueError("gate_lower_bound: KDA only")
    _rule(S, mixed, a, b, A_log, dt_bias, idx, loc, out, H, src, scale, bool(kda), gate_lower_bound, False)


def conv_prefill(x, conv_state, weight, bias, idx, loc, out, src=None, silu=True):
    """The depthwise causal conv1d of width 4 over a ragged batch: out [T, C] (bf16) from the packed tokens x [T, C] (bf16,
    possibly a column range of wider rows), out_t = act(sum_j w_j x_{t-3+j} + bias).  conv_state [NS, C, 3] (any strides): the
    inputs before a sequence's first token come from its slot src, its last three are left in slot idx.  out may not overlap x."""
    rc = _lib.seq_call().conv(x, conv_state, weight, bias, idx, loc, out, src, bool(silu))
    if rc != _NOT_PLAIN:
        return _lib.check(rc, "lq_conv_seq")
    if x.dim() != 2:
        raise ValueError("x: [T, C] expected, got shape %s" % (tuple(x.shape),))
    T, C = x.shape
    ld = _rows(x, T, C, "x", 1)
    if weight.shape[0] != C:
        raise ValueError("weight: [%d, 4] expected, got shape %s" % (C, tuple(weight.shape)))
    if out.dtype is not _BF16 or out.shape != (T, C) or not out.is_contiguous():
        raise ValueError("out: contiguous bf16 [T, C] expected")
    seqs, live = _batch(idx, loc, src, T)
    cv = conv_struct(conv_state, weight, bias, silu)
    _on(x.get_device(), conv_state=conv_state, weight=weight, bias=bias, idx=idx, loc=loc, out=out, src=src)
    with torch.cuda.device(x.get_device()):
        _lib.check(_lib.seq_lib().lq_conv_seq(ctypes.byref(cv), seqs, x.data_ptr(), ld, out.data_ptr(), C, _raw_stream(x)),
                   "lq_conv_seq")


def _norm(x, z, weight, out, res, eps, scale, offset, act):
    """lq_norm's bytes."""
    shape = x.shape
    nd = len(shape)
    D = shape[-1] if nd else 0
    if x.dtype is not _BF16 or not 1 <= nd <= 3 or not 1 <= D <= 16384:
        raise ValueError("x: bf16 [rows, D] or [rows, heads, D] with D <= 16384 expected, got %s %s" % (x.dtype, tuple(shape)))
    sx, sz, so = x.stride(), z.stride(), out.stride()
    for name, t in (("z", z), ("out", out)):
        if t.dtype is not _BF16 or t.shape != shape:
            raise ValueError("%s: bf16 %s expected, got %s %s" % (name, tuple(shape), t.dtype, tuple(t.shape)))
    if D > 1 and not sx[-1] == sz[-1] == so[-1] == 1:
        raise ValueError("packed elements expected in the last dimension (strides %s, %s, %s)" % (sx, sz, so))
    if any(n > 1 and s < D for n, s in zip(shape[:-1], so)):
        raise ValueError("out: rows that overlap each other (strides %s)" % (so,))
    if res is not None and (res.dtype is not _BF16 or res.shape != shape or res.stride() != so):
        raise ValueError("res: bf16 %s laid out as out expected, got %s %s strides %s"
                         % (tuple(shape), res.dtype, tuple(res.shape), res.stride()))
    if weight.shape != (D,) or (weight.dtype is not _BF16 and weight.dtype is not _F32) or not weight.is_contiguous():
        raise ValueError("weight: contiguous fp32 or bf16 [%d] expected" % D)
    _on(x.get_device(), z=z, weight=weight, out=out, res=res)
    if nd == 3:
        rows, heads = shape[0], shape[1]
        lds = sx[0], sx[1], sz[0], sz[1], so[0], so[1]
        if not heads:
            rows = heads = 0
    else:
        rows, heads = shape[0] if nd == 2 else 1, 1
        lds = (sx[0], 0, sz[0], 0, so[0], 0) if nd == 2 else (0,) * 6
    return _lib.pack_norm(x.data_ptr(), z.data_ptr(), weight.data_ptr(), res.data_ptr() if res is not None else 0,
                          out.data_ptr(), *lds, rows, heads or 1, D, eps, scale, offset, act, weight.dtype is _BF16)


def gated_norm(x, z, weight, out, eps=1e-6, gate="silu", offset=0.0):
    """The norm after a block times its gate: out = x rsqrt(mean(x^2) + eps) (offset + weight) act(z) over the last
    dimension, act SiLU or sigmoid.  x, z, out: bf16 [rows, D] or [rows, heads, D], any row and head strides; weight fp32 or
    bf16 [D]; offset 1 for weights stored around zero.  out may be x."""
    if gate not in _ACT:
        raise ValueError("gate: 'silu' or 'sigmoid' expected, got %r" % (gate,))
    rc = _lib.seq_call().norm(x, z, weight, out, None, eps, 0.0, offset, _ACT[gate], False)
    if rc != _NOT_PLAIN:
        return _lib.check(rc, "lq_gated_norm")
    n = _norm(x, z, weight, out, None, eps, 0.0, offset, _ACT[gate])
    with torch.cuda.device(x.get_device()):
        _lib.check(_lib.seq_lib().lq_gated_norm(n, _raw_stream(x)), "lq_gated_norm")


def add_norm(x, y, weight, res, out, eps=1e-6, scale=1.0, offset=0.0):
    """The residual add and the norm before the next block: res = x + scale y, out = res rsqrt(mean(res^2) + eps)
    (offset + weight), of the sum before it is rounded to bf16.  Shapes as `gated_norm`; res and out are laid out alike; res
    may be x or y (in place)."""
    rc = _lib.seq_call().norm(x, y, weight, out, res, eps, scale, offset, 0, True)
    if rc != _NOT_PLAIN:
        return _lib.check(rc, "lq_add_norm")
    n = _norm(x, y, weight, out, res, eps, scale, offset, 0)
    with torch.cuda.device(x.get_device()):
        _lib.check(_lib.seq_lib().lq_add_norm(n, _raw_stream(x)), "lq_add_norm")
