"""A paged key-value cache shared by several sequences, quantised as it is written, and the attention of one new
token a row over it (include/epq_paged.h): over all of a row's tokens, over those of selected blocks, and for rows
that share a prefix, which is then read once for all of them.

The reference decodes one sequence through the Hugging Face model's own dense cache.  Here the keys and values of
all sequences live in pools of pages; a page table maps token ``t`` of sequence ``s`` to slot ``t % page_size`` of
page ``table[s, t // page_size]``.  A pool holds the activations' type, int8 or 8-bit floats (e4m3) with one
float32 scale a token and head.

``KVPages`` names the tensors of one layer; ``write``, ``read``, ``attend``, ``attend_shared``, ``summarise`` and
``select`` are the operators on it.  ``PagedKVCache`` owns the pools of all layers and hands pages out.  The operators have no gradient: with grad mode
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


def attend(pages, q, lengths, seq=None, scale=None, window=0, out=None, return_lse=False, blocks=None):
    """Attention of one new token a sequence: q [batch, heads, head_dim] over the first ``lengths`` (int64 [batch])
    tokens of sequences ``seq`` (int32 [batch], default 0..batch-1), the last ``window`` of them where window > 0;
    ``scale`` defaults to head_dim ** -0.5.  Query head h reads key head h // (heads / kv_heads).  A length of 0
    gives zeros.  Returns out, or ``(out, lse)`` with the float32 log-sum-exp [batch, heads] of the scores
    (-inf for an empty row), with which results over disjoint sets of tokens can be joined.

    ``blocks`` (int32 [batch, kv_heads, count], as ``select`` returns it) attends over the tokens of the listed pages
    of a row's sequence alone, those below its length: page ``j`` holds tokens ``j * page_size`` on.  A list names
    each page at most once and -1 for none; its first ``ceil(length / page_size)`` entries are looked at."""
    return (_native.tensor_calls or _native.load_tensor_calls()).attend(*pages, q, lengths, seq, scale, window, out,
                                                                        return_lse, blocks)


def attend_shared(pages, q, lengths, starts, prefix, seq=None, scale=None, out=None, return_lse=False,
                  always=False):
    """``attend`` where rows share their first tokens, which are read once for all of them.

    Rows ``starts[g] .. starts[g + 1) - 1`` (int32 [groups + 1], ascending) have the same first ``prefix[g]`` (int64
    [groups]) tokens: either their page tables name the same pages there (``PagedKVCache.share``), or they are rows of
    one sequence (drafted tokens, a prompt's chunk) with lengths of their own.  The shared tokens are
    read through the table of one of the rows.  A row shorter than its group's prefix attends over its own length, rows in no
    group share nothing.  Groups for which reading row by row is reckoned to be faster (few rows, short prefixes) are
    read that way, unless ``always``.

    Nothing is shared, with ``always`` either, in pages whose size is no multiple of 8, by 8-bit heads above 128, and with
    more than 128 query heads a key head.  Rows are taken together in tiles of a group's consecutive rows, as far as the shortest
    row of a tile that is not empty: put rows that are much shorter than their prefix into no group.  Where a batch could
    share and then does not, the call takes about 10 us longer than ``attend``."""
    return (_native.tensor_calls or _native.load_tensor_calls()).attend_shared(*pages, q, lengths, starts, prefix, seq,
                                                                               scale, out, return_lse, always)


def summarise(pages, bounds, lengths, seq=None, first=None):
    """Brings ``bounds`` [pages, kv_heads, 2, head_dim] (of the pool's 16-bit type, bfloat16 for 8-bit pools) up to date:
    the least and the largest of every value of the keys of each page that holds one of the new tokens ``first[b] ..
    lengths[b] - 1`` (int64 [batch]; first None: from 0) of sequence ``seq[b]``, over the page's tokens below
    ``lengths[b]``.  After a decode step ``first = lengths - 1``.  Rows with a page in common must agree about its
    tokens."""
    (_native.tensor_calls or _native.load_tensor_calls()).bounds(*pages, bounds, lengths, seq, first)


def select(pages, bounds, q, lengths, count, seq=None, sinks=1, recent=1):
    """The ``count`` blocks (pages) of each row and key head to attend over, int32 [batch, kv_heads, count] in ascending
    order, -1 behind the last: the first ``sinks``, the last ``recent`` and those of the others in which a query head of
    the key head may find the largest score, ``sum_d max(q_d lo_d, q_d hi_d)`` by their ``bounds`` (ties to the lowest
    block; 8-bit caches have theirs rounded to bfloat16, so a token's score may pass its block's there).  q [batch, heads, head_dim] is what ``attend`` will be given."""
    return (_native.tensor_calls or _native.load_tensor_calls()).select(*pages, bounds, q, lengths, count, seq, sinks,
                                                                        recent)


class PagedKVCache:
    """The pools of every layer over one page table, and which pages are free.

    ``format``: "same" (the activations' ``dtype``; a float32 cache can be written and read, but not attended
    over), "int8" or "fp8".  Pages are handed out by ``reserve(seq,
    tokens)`` and given back by ``release(seq)``; both change the table on the device in the current stream's
    order, so a captured step sees them at its next replay.  ``share(seq, source, tokens)`` lets a sequence begin with
    another's pages.  ``bounds=True`` holds room for ``summarise`` (``bounds[layer]``)."""

    def __init__(self, layers, pages, page_size, kv_heads, head_dim, seqs, max_tokens, format="same",
                 dtype=torch.bfloat16, device="cuda", bounds=False):
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
        self.bounds = torch.zeros(layers, pages, kv_heads, 2, head_dim, dtype=torch.bfloat16 if scales else dtype,
                                  device=self.device) if bounds else None
        self.table = torch.full((seqs, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=self.device)
        self._free = list(range(pages - 1, -1, -1))
        self._held = [[] for _ in range(seqs)]
        self._users = [0] * pages                      # sequences that hold a page

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
        for p in got:
            self._users[p] = 1

    def share(self, seq, source, tokens):
        """Lets the empty sequence ``seq`` begin with the whole pages of the first ``tokens`` tokens of sequence
        ``source``; returns how many tokens these are (a multiple of the page size).  They are not copied: neither
        sequence may write them any more.  The others are ``seq``'s own to reserve and write."""
        self._check(seq)
        self._check(source)
        if self._held[seq]:
            raise ValueError(f"epure: sequence {seq} has pages; release it first")
        if tokens < 0 or tokens > len(self._held[source]) * self.page_size:
            raise ValueError(f"epure: {tokens} tokens of sequence {source}, which has room for "
                             f"{len(self._held[source]) * self.page_size}")
        whole = tokens // self.page_size
        if whole:
            self.table[seq, :whole] = self.table[source, :whole]
            self._held[seq] = self._held[source][:whole]
            for p in self._held[seq]:
                self._users[p] += 1
        return whole * self.page_size

    def release(self, seq):
        """Gives sequence ``seq``'s pages back; one that others share stays theirs."""
        self._check(seq)
        for p in reversed(self._held[seq]):
            self._users[p] -= 1
            if not self._users[p]:
                self._free.append(p)
        self._held[seq] = []
        self.table[seq].fill_(-1)
