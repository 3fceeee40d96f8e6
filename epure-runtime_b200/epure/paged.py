"""A paged key-value cache shared by several sequences, quantised as it is written, and the attention of one new
token a sequence over it (include/epq_paged.h).

The reference decodes one sequence through the Hugging Face model's own dense cache.  Here the keys and values of
all sequences live in pools of pages; a page table maps token ``t`` of sequence ``s`` to slot ``t % page_size`` of
page ``table[s, t // page_size]``.  A pool holds the activations' type, int8 or 8-bit floats (e4m3) with one
float32 scale a token and head.

``KVPages`` names the tensors of one layer; ``write``, ``read`` and ``attend`` are the operators on it.
``PagedKVCache`` owns the pools of all layers and hands pages out.  The operators have no gradient: with grad mode
on they refuse tensors that require one."""
from typing import NamedTuple, Optional

import torch

from . import _native

FORMATS = {"same": None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


class KVPages(NamedTuple):
    """One layer's cache: pools ``k``, ``v`` [pages, kv_heads, page_size, head_dim], the int32 page ``table``
    [seqs, max_pages] and, for 8-bit pools, float32 scales [pages, kv_heads, page_size]."""
    k: torch.Tensor
    v: torch.Tensor
    table: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None


def write(pages, k, v, seq, pos, q=None, q_out=None, cos=None, sin=None, interleaved=False, qk_norm=False, eps=1e-6):
    """Writes rows ``k``, ``v`` [m, kv_heads, head_dim] as tokens ``pos`` (int64 [m]) of sequences ``seq`` (int32
    [m]), quantised where the pool is 8-bit.

    ``qk_norm`` first normalises every head of q and k (RMSNorm, weight 1); with tables ``cos``, ``sin``
    (epure.rotary) q and k are rotated by ``pos``.  Returns q so treated (``q_out``, a new tensor, or q itself
    given as q_out), or None without q.  A row with a negative position is padding.  No two rows may name the
    same token."""
    return (_native.tensor_calls or _native.load_tensor_calls()).write(*pages, k, v, seq, pos, q, q_out, cos, sin,
                                                                       interleaved, qk_norm, eps)


def read(pages, seq, pos, dtype=None):
    """``(k, v)`` [m, kv_heads, head_dim] of cached tokens, in ``dtype`` (default: the pool's own type, bfloat16
    for 8-bit pools)."""
    return (_native.tensor_calls or _native.load_tensor_calls()).read(*pages, seq, pos, dtype)


def attend(pages, q, lengths, seq=None, scale=None, window=0, out=None, return_lse=False):
    """Attention of one new token a sequence: q [batch, heads, head_dim] over the first ``lengths`` (int64 [batch])
    tokens of sequences ``seq`` (int32 [batch], default 0..batch-1), the last ``window`` of them where window > 0;
    ``scale`` defaults to head_dim ** -0.5.  Query head h reads key head h // (heads / kv_heads).  A length of 0
    gives zeros.  Returns out, or ``(out, lse)`` with the float32 log-sum-exp [batch, heads] of the scores
    (-inf for an empty row), with which results over disjoint sets of tokens can be joined."""
    return (_native.tensor_calls or _native.load_tensor_calls()).attend(*pages, q, lengths, seq, scale, window, out,
                                                                        return_lse)


class PagedKVCache:
    """The pools of every layer over one page table, and which pages are free.

    ``format``: "same" (the activations' ``dtype``; a float32 cache can be written and read, but not attended
    over), "int8" or "fp8".  Pages are handed out by ``reserve(seq,
    tokens)`` and given back by ``release(seq)``; both change the table on the device in the current stream's
    order, so a captured step sees them at its next replay."""

    def __init__(self, layers, pages, page_size, kv_heads, head_dim, seqs, max_tokens, format="same",
                 dtype=torch.bfloat16, device="cuda"):
        if format not in FORMATS:
            raise ValueError(f"epure: format must be one of {tuple(FORMATS)} (got {format!r})")
        if min(layers, pages, page_size, kv_heads, seqs, max_tokens) < 1:
            raise ValueError("epure: layers, pages, page_size, kv_heads, seqs and max_tokens must be positive")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"epure: head_dim must be a multiple of 16 up to 256 (got {head_dim})")
        self.device = torch.device(device)
        self.page_size, self.seqs, self.format, self.dtype = page_size, seqs, format, dtype
        self.max_tokens = max_tokens
        store = FORMATS[format] or dtype
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=store, device=self.device)
        self.v = torch.zeros(shape, dtype=store, device=self.device)
        scales = format != "same"
        self.k_scale = torch.zeros(shape[:4], device=self.device) if scales else None
        self.v_scale = torch.zeros(shape[:4], device=self.device) if scales else None
        self.table = torch.full((seqs, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=self.device)
        self._free = list(range(pages - 1, -1, -1))
        self._held = [[] for _ in range(seqs)]

    def layer(self, i):
        """Layer ``i``'s ``KVPages``."""
        s = self.k_scale is not None
        return KVPages(self.k[i], self.v[i], self.table, self.k_scale[i] if s else None,
                       self.v_scale[i] if s else None)

    def free_pages(self):
        return len(self._free)

    def _check(self, seq):
        if not 0 <= seq < self.seqs:
            raise IndexError(f"epure: sequence {seq} of a cache of {self.seqs}")

    def reserve(self, seq, tokens):
        """Makes room for the first ``tokens`` tokens of sequence ``seq``."""
        self._check(seq)
        if tokens > self.max_tokens:
            raise ValueError(f"epure: {tokens} tokens; this cache holds max_tokens={self.max_tokens} a sequence")
        held = self._held[seq]
        more = -(-tokens // self.page_size) - len(held)
        if more <= 0:
            return
        if more > len(self._free):
            raise RuntimeError(f"epure: the cache is full ({len(self._free)} pages free, {more} needed)")
        got = self._free[:-more - 1:-1]
        first = len(held)
        self.table[seq, first:first + more] = torch.tensor(got, dtype=torch.int32).to(self.device)
        held += got                                    # behind the copy: where it raises, no page is lost
        del self._free[-more:]

    def release(self, seq):
        """Gives sequence ``seq``'s pages back."""
        self._check(seq)
        self._free += reversed(self._held[seq])
        self._held[seq] = []
        self.table[seq].fill_(-1)
