"""Serving operators: a key/value cache in pages, held in 8 bits, what writes it, what reads it, and attention over packed prompts.

The reference generates through a contiguous bf16 cache and one library attention call
(models/flashmhf/modeling_mhffnmoe.py:556-592) with all sequences of a batch padded to one length.  Here sequences of different
lengths share a pool of pages; lengths and page numbers live on the device, so that a captured generation step follows them.

    pages = KVPages.empty(num_pages, n_kv, page_size, head_dim, device)      # one layer
    q, k_rot = paged_append(pages, k, v, cos, sin, lengths, table, q=q, cu_seqlens=cu, rotated_keys=True)   # prompts
    o = prompt_attention(q, k_rot, v, cu)
    lengths += cu[1:] - cu[:-1]
    q, _ = paged_append(pages, k, v, cos, sin, lengths, table, q=q)          # one token a sequence
    o = paged_attention(q, pages, lengths + 1, table)

All of them are for serving: bf16 CUDA tensors, no gradients (NotImplementedError for a tensor that wants one).  What only the
device knows, such as a page number that the pool does not have, is left out there and reported by ``check_device_status()``.
What a call writes in place (pages, scales, ``out``) has a new version for autograd."""
from typing import NamedTuple

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 96, 128)


class KVPages(NamedTuple):
    """One layer's pool of pages: codes ``k``, ``v`` float8_e4m3fn [num_pages, n_kv, page_size, head_dim] (a page contiguous) and
    scales ``k_scale``, ``v_scale`` fp32 [num_pages, n_kv], powers of two; a key is code * scale."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_pages, n_kv, page_size, head_dim, device="cuda"):
        """A pool whose contents are undefined until they are appended (a page's first rows set its scale)."""
        codes = [torch.empty(num_pages, n_kv, page_size, head_dim, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        scales = [torch.ones(num_pages, n_kv, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    def values(self):
        """(keys, values) that the codes stand for, bf16 [num_pages, n_kv, page_size, head_dim]; exact."""
        return tuple((c.float() * s[:, :, None, None]).bfloat16() for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))


def paged_append(pages, k, v, cos, sin, lengths, page_table, q=None, cu_seqlens=None, rotated_keys=False):
    """Rotate the queries and keys of new tokens and put keys and values into the pages; returns (rotated q, rotated k).

    k, v [T, n_kv, head_dim], q [T, n_q, head_dim] or None, bf16 (views of one projection are read in place); cos, sin fp32
    [positions, head_dim/2]; ``lengths`` int32 [B]: what each sequence held before the call (negative: no sequence, its rows are
    left out); ``page_table`` int32 [B, max_pages].  ``cu_seqlens`` int32 [B+1]: the rows of each sequence; None: one token a
    sequence.  ``rotated_keys``: also return the rotated keys in bf16.  What is not asked for comes back as None.

    The rotation is done in fp32 as the halves of a head, x1 c - x2 s and x2 c + x1 s.  The scale of a page and head is the
    smallest power of two (at least 2^-60) under which the largest new value is at most 448, and at least the page's scale where
    the page held rows of the sequence already; those are rescaled when it grows, which is exact but for codes that become
    subnormal.  NaN and infinities are held as NaN and do not count for the scale.  ``pages`` is changed in place;
    ``lengths`` is not.  A page that is written must belong to one sequence of the call."""
    return _lib.native().paged_append(pages.k, pages.v, pages.k_scale, pages.v_scale, k, v, cos, sin, lengths, page_table, q, cu_seqlens,
                                      rotated_keys)


def paged_attention(q, pages, lengths, page_table, scale=None, out=None, return_lse=False):
    """Attention of the newest tokens of each sequence over its pages: o like q, bf16.

    q [B, n_q, head_dim] (one token a sequence) or [B, n_new, n_q, head_dim] with n_new up to 16, rotated and already appended;
    ``lengths`` int32 [B]: positions in the cache, those of the new tokens included (new token i sees the first
    lengths - (n_new - 1 - i)); n_q a multiple of n_kv.  ``scale`` defaults to head_dim ** -0.5.  A row that sees nothing gives
    zeros.  ``scale`` and its product with log2(e) are finite in fp32.  ``out``: like q, its last dimension contiguous and the others in steps of 16 bytes; it may be q itself.  ``return_lse``: also the natural logarithm of the sum of exponentials, fp32, q's shape without the last dimension
    (-inf for a row that sees nothing): what parts of a longer attention are merged with.  Rows of a page behind a sequence's length are
    never used, whatever they hold; a value of a later new token that is not a finite number also reaches the new tokens before it.
    Maxima, sums and outputs are held in fp32; a weight is rounded to fp16 before it meets the values (by 2^-11 of itself, or 2^-24 of the row's
    largest), and a query by 2^-39 of its row's largest.  The cache is read once for each eight query rows of a key/value head."""
    o, lse = _lib.native().paged_attention(q, pages.k, pages.v, pages.k_scale, pages.v_scale, lengths, page_table, scale, out, return_lse)
    return (o, lse) if return_lse else o


def prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, causal=True, scale=None, out=None, return_lse=False):
    """Attention over packed sequences: q [T, n_q, head_dim], k, v [T_k, n_kv, head_dim], bf16; o like q.

    Rows cu_seqlens[b] .. cu_seqlens[b+1]-1 of q belong to sequence b, and those of ``cu_seqlens_k`` (default: the same) of k and
    v; int32 [B+1] on the device.  Causal: the last row sees all keys of its sequence, each row before it one less; a row that
    sees nothing gives zeros.  Rows of no sequence are left as they are (in a new output: undefined).  ``out`` as for ``paged_attention``; it must
    not lie over k or v.  ``return_lse`` as for
    ``paged_attention``, [T, n_q].  Sequences do not touch each other, whatever their neighbours hold; within a sequence the mask gives
    weights of zero, so that a value which is not a finite number also reaches up to 127 rows before its own.  Maxima, sums and outputs are held in
    fp32; a weight is rounded to bf16 before it meets the values (by 2^-8 of itself at most), the sum of weights is of unrounded ones."""
    o, lse = _lib.native().prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k, causal, scale, out, return_lse)
    return (o, lse) if return_lse else o
