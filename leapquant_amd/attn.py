"""Operators that take sequences through a softmax-attention layer with a paged cache (HIP, include/lq_attn.h): the layers
that hybrid stacks have between the linear-attention ones, which `seq`, `kernels` and `state` take.

  rope_norm        the norms of each head's queries and keys and their rotation by position; keys and values into the pages
  attend           the attention of a batch's new tokens over the pages: single and drafted tokens, prompts and pieces of them

A layer's cache is `Pages(k, v)`: [pages, page, heads, D] each in bf16 (D 64, 128 or 256, a page a multiple of 16 tokens, any strides
of the first three dimensions, the same for both), or `Pages(k, v, k_scale, v_scale)` in 8 bits: int8 codes whose values are code *
scale, with fp32 scales [pages, page, heads], one a token and head.

A ragged batch is given by `loc` [N + 1] (sequence n holds the packed new tokens loc[n] .. loc[n + 1] - 1), `lens` [N], the cached
tokens of each sequence with the new ones, which are the last of them, and `table` [N, width]: token t of sequence n is at t %
page in page table[n, t // page].  New tokens before a sequence's position 0 (all of them where lens is 0: padding) have outputs of
zero, whatever their inputs hold, and write nothing; rows that no sequence holds are left as they are.  A table entry outside
the cache is not written; it reads page 0.  The three are int32; other integer types are converted in each call, far values held to
int32's range.  Calls launch on the current stream of their tensors' device, never synchronise and can be captured in a graph;
they work forward only (no autograd).
"""
import typing

import torch

from . import _lib


class Pages(typing.NamedTuple):
    """A layer's cache of keys and values, in bf16 or in 8 bits with scales."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: typing.Optional[torch.Tensor] = None
    v_scale: typing.Optional[torch.Tensor] = None


def rope_norm(q, k, v, q_weight, k_weight, inv_freq, pages, table, loc, lens, out, eps=1e-6, offset=0.0, interleaved=False):
    """Before the attention: x rsqrt(mean(x^2) + eps) (offset + weight) over each head of q and k, then its first rot = 2 len(inv_freq)
    elements turned by the token's position times inv_freq, in pairs (i, i + rot / 2), or (2i, 2i + 1) where interleaved.  q goes to
    out (which may be q), k and v to their places in the pages, each rounded once.

    q, out: bf16 [T, HQ, D]; k, v: bf16 [T, HK, D]; any token and head strides divisible by 16 bytes.  Weights fp32 or bf16 [D]; offset
    1 for weights stored around zero.  inv_freq: fp32 or fp64, a multiple of 8 elements (none: no rotation); angles are formed in
    64 bits.  Pages in 8 bits take code = rint(x / scale) with scale = max|x| / 127 of a token's head: NaN where the head holds one, 0
    where max|x| <= 1e-30, with codes of 0 for these and for infinite ones.  Two new tokens of a call do not share a place in the pages."""
    _lib.attn_call().rope_norm(q, k, v, q_weight, k_weight, inv_freq, pages, table, loc, lens, out, eps, offset, interleaved)


def attend(q, pages, table, loc, lens, out, scale=None, window=0, gate=None, longest=None):
    """out = softmax(scale q k^T) v over the cached tokens at and before each new token's position, the last `window` of them
    where window is not 0, times sigmoid(gate) where a gate is given.  The new tokens' keys and values are in the pages already.

    q, out, gate: bf16 [T, HQ, D], any token and head strides divisible by 16 bytes; out may be q.  HQ is a multiple of the pages'
    heads; head h reads head h // (HQ / HK).  scale: positive (below 2^127), D^-1/2 by default.  longest: new tokens of the longest
    sequence where the host knows them (a host integer, which decides on speed only; decode batches without it take up to 1.6 times as
    long).  A table no wider than the batch needs saves short contexts a launch.  What a token does not see, infinities and NaN
    among it, does not reach its output."""
    _lib.attn_call().attend(q, pages, table, loc, lens, out, scale, window, gate, longest)
