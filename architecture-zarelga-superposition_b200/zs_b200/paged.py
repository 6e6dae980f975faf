"""Paged key-value cache of a model that answers: storing new tokens, attention over the
pages, and the cache's page bookkeeping, on the kernels of libzs.so.

The reference answers by running the whole sequence again for every token
(inference.py:25-73).  Here each layer's keys and values stay in pages
[num_pages, Hkv, page, hd] that sequences hold by number:

* paged_append            QK zero-centred RMSNorm + partial RoPE of new tokens, stored in their pages
* paged_prompt_attention  causal GQA attention of packed new tokens (a prompt, or the next part
                          of one after a prefix that is in the cache already)
* paged_decode_attention  the same for one new token per sequence, split over the cache's length
* PagedKVCache            the pages of all layers and their tables: extend, fork, free, compact

All run on the current stream of the tensors' device, never wait for the host and
can be captured in a CUDA graph (outputs and workspaces come from torch's allocator, so each
captured graph has its own).  They have no gradient and refuse inputs that ask for one.

Tables are int32 CUDA tensors: block_table [num_seqs, max_pages], seq_lens [num_seqs] (tokens in
the cache, this call's new ones included), cu_seqlens [num_seqs + 1] (packed rows of each
sequence's new tokens, which lie at its last positions).  A page id out of range, or a position
beyond the table, is skipped and recorded in the device error word (ZS_DEVERR_INDEX).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib as Z
from .build import binding_abi

PAGE_SIZES = (16, 32, 64, 128)
_DTYPES = (torch.bfloat16, torch.float16)
_BINDING = None


def _binding():
    """The compiled binding (csrc/zs_paged_py.cpp): it checks the tensors, allocates outputs and
    workspaces and calls the C ABI, in a tenth of the host time that the same takes here."""
    global _BINDING
    if _BINDING is None:
        Z.lib()   # the library it is linked against, with the package's own error when it is missing
        try:
            from . import _paged
        except ImportError as e:
            raise Z.ZsError(f"the paged operators' binding cannot be loaded ({e}): build it with "
                            "__graft_entry__.build()") from e
        if _paged.abi != binding_abi():
            _fail(f"the paged operators' binding was built for another Python or torch ({_paged.abi}, not "
                  f"{binding_abi()}): build it with __graft_entry__.build()")
        _BINDING = _paged
    return _BINDING


def _fail(msg):
    raise Z.ZsError(msg)


def paged_append(qkvg, k_pages, v_pages, block_table, seq_lens, *, n_heads, cu_seqlens=None, q_weight=None,
                 k_weight=None, eps=1e-6, cos=None, sin=None):
    """q [T, n_heads, hd] of packed new tokens, their keys and values stored in their pages.

    qkvg [T, W] (the pages' dtype): n_heads query heads, Hkv key heads and Hkv value heads of a
    token in one row (columns after them are not read).  q and k: per-head zero-centred RMSNorm
    (q_weight, k_weight f32 [hd]; None: no norm), then the first `rot` pairs (i, i + hd/2) turned
    by cos/sin f32 [positions, rot] at the token's position (None: no rotation); f32 arithmetic,
    one rounding.  cu_seqlens None: row s is sequence s's one new token.  A row outside every
    sequence, or at a negative position (an empty slot), gets a zero q and stores nothing."""
    Z.INSTR.launches += 1
    return (_BINDING or _binding()).append(qkvg, k_pages, v_pages, block_table, seq_lens, n_heads, cu_seqlens, q_weight,
                                           k_weight, eps, cos, sin)


def paged_prompt_attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, *, window=None, k_sink=None,
                           gate=None, scale=None, return_lse=False):
    """o [T, H, hd] (with return_lse also the f32 log-sum-exp [T, H]) of packed new tokens q
    [T, H, hd]: softmax attention over the keys at or before each token's position in its own
    sequence (the last `window` of them), key head h // (H // Hkv), scale 1/sqrt(hd) by default.
    k_sink [H, hd]: one more logit q . k_sink per head whose value is zero.  gate [T, H] (q's dtype;
    a strided view will do): o is multiplied by sigmoid(gate).  Rows that see no key, and rows
    outside every sequence, are zero.  At most 128 query heads share a key head.  A value that is NaN or
    infinite reaches no other sequence, but may reach earlier rows of its own (zero times it)."""
    if cu_seqlens is None:
        _fail("cu_seqlens is required")
    Z.INSTR.launches += 2
    return (_BINDING or _binding()).attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, window, k_sink,
                                              gate, scale, return_lse)


def paged_decode_attention(q, k_pages, v_pages, block_table, seq_lens, *, window=None, k_sink=None, gate=None,
                           scale=None, return_lse=False):
    """paged_prompt_attention for one new token per sequence: row s of q [num_seqs, H, hd] is the
    last token of sequence s.  The keys of a sequence are split over thread blocks and joined in a
    fixed order.  seq_lens[s] == 0 marks an empty slot: its row is zero."""
    Z.INSTR.launches += 2
    return (_BINDING or _binding()).attention(q, k_pages, v_pages, block_table, seq_lens, None, window, k_sink, gate,
                                              scale, return_lse)


class PagedKVCache:
    """The pages of all layers and the tables that say who holds them, on one device.

    kv [n_layers, 2, num_pages, n_kv_heads, page_size, head_dim] (keys, values); a slot is a row of
    block_table [max_seqs, max_pages_per_seq] (-1: no page) with its length in seq_lens;
    ref_count [num_pages] counts the rows that hold a page.  The three tables are views of one
    int32 tensor `meta`, so a copy of it is a snapshot of the bookkeeping.  The tensors may be written but
    not replaced.

    Requests are int32 CUDA tensors (a list or int is uploaded); they are served in order and take
    the lowest-numbered free pages.  Nothing here waits for the host: a request that cannot be
    served changes nothing and is recorded in the device error word, which check() reads."""

    def __init__(self, n_layers, n_kv_heads, head_dim, *, num_pages, page_size=64, max_seqs, max_pages_per_seq,
                 dtype=torch.bfloat16, device="cuda"):
        device = torch.device(device)
        if device.type != "cuda":
            _fail(f"the cache lives on a CUDA device (got {device})")
        if dtype not in _DTYPES or page_size not in PAGE_SIZES or head_dim not in (64, 128):
            _fail(f"the cache holds bf16 or f16 pages of {PAGE_SIZES} tokens of head_dim 64 or 128 (got {dtype}, "
                  f"{page_size}, {head_dim})")
        if (min(n_layers, n_kv_heads, num_pages, max_seqs, max_pages_per_seq) < 1 or num_pages > 2_000_000
                or max_pages_per_seq * page_size > (1 << 31) - 256):
            _fail("n_layers, n_kv_heads, num_pages (at most 2000000), max_seqs and max_pages_per_seq (at most "
                  "2^31 - 256 tokens) must be positive")
        self.kv = torch.zeros(n_layers, 2, num_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device)
        cells = max_seqs * max_pages_per_seq
        self.meta = torch.empty(cells + max_seqs + num_pages, dtype=torch.int32, device=device)
        self.block_table = self.meta[:cells].view(max_seqs, max_pages_per_seq)
        self.seq_lens = self.meta[cells:cells + max_seqs]
        self.ref_count = self.meta[cells + max_seqs:]
        self.reset()
        self._c = Z.KvCache(self.kv.data_ptr(), self.block_table.data_ptr(), self.seq_lens.data_ptr(),
                            self.ref_count.data_ptr(), num_pages, n_layers, n_kv_heads, page_size, head_dim, max_seqs,
                            max_pages_per_seq)

    @property
    def page_size(self):
        return self.kv.size(4)

    def layer(self, i):
        """(k_pages, v_pages) of layer i, views of kv."""
        return self.kv[i, 0], self.kv[i, 1]

    def reset(self):
        """Every slot empty, every page free."""
        self.block_table.fill_(-1)
        self.seq_lens.zero_()
        self.ref_count.zero_()

    def check(self):
        """Wait for the device and raise if a request was refused or an index was out of range
        since the error word was last cleared; clears it."""
        err = Z.device_error(self.kv.device)
        if err:
            Z.clear_device_error(self.kv.device)
            what = [n for b, n in ((0x10, "a slot, page or position out of range, or a slot named twice"),
                                   (0x40, "no free page, or a slot without room")) if err & b]
            raise Z.ZsError(f"paged cache: {'; '.join(what) or 'device error'} (device error word {err:#x})")

    def _list(self, x):
        if torch.is_tensor(x):
            return x
        return torch.tensor([x] if isinstance(x, int) else list(x), dtype=torch.int32, device=self.kv.device)

    def _call(self, op, launches, x=None, y=None):
        if x is not None:
            x = self._list(x)
        if y is not None:
            y = self._list(y)
        Z.INSTR.launches += launches
        (_BINDING or _binding()).pages(op, ctypes.addressof(self._c), self.kv, self.block_table, self.seq_lens,
                                       self.ref_count, x, y)

    def extend(self, slots, n_tokens):
        """Slot slots[i] grows by n_tokens[i] >= 0 tokens, with pages for them; what they hold is
        up to the caller (paged_append).  A slot named twice grows by its first request only.  A refused
        slot has not grown, and tokens stored at its last positions would replace those that it holds:
        compare seq_lens with a copy from before the call, or check(), before storing."""
        self._call(0, 1, slots, n_tokens)

    def fork(self, src, dst):
        """Slot dst[i] becomes a copy of slot src[i] as it was before the call (beam search:
        fork(parents, slots)); what dst[i] held is let go.  Whole pages are shared; the filled
        rows of a last partial page are copied into a page of dst[i]'s own, which has to be free
        before the call (a pool with a page to spare for every slot always has one)."""
        self._call(1, 2, src, dst)

    def free(self, slots):
        """Slots become empty; pages that no slot holds any more are free."""
        self._call(2, 1, slots)

    def compact(self):
        """The pages in use become pages 0 .. U-1 (the k-th free page below U takes the k-th used
        page from U on), so everything held lies in one run at the start of the pool."""
        self._call(3, 2)

    def copy_pages(self, src, dst):
        """Page dst[i] = page src[i], every layer's keys and values; the tables stay.  A page that
        is written must not also be read by the call."""
        self._call(4, 2, src, dst)
