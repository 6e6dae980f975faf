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
import math

import torch

from . import _lib as Z

PAGE_SIZES = (16, 32, 64, 128)
_DTYPES = (torch.bfloat16, torch.float16)


def _refuse(cond, msg):
    if cond:
        raise Z.ZsError(msg)


def _no_grad(*tensors):
    _refuse(torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors),
            "the paged operators have no gradient: call them under torch.no_grad() or on detached tensors")


def _same_device(first, *tensors):
    Z.require_cuda(first, *tensors)
    for t in tensors:
        _refuse(t is not None and t.device != first.device,
                f"all tensors must be on one device (got {first.device} and {t.device if t is not None else None})")


def _pages(k_pages, v_pages):
    """(num_pages, Hkv, page, hd, page stride) of a layer's pages."""
    _refuse(k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype,
            f"k_pages and v_pages must be [num_pages, Hkv, page, hd] of one shape and dtype (got "
            f"{tuple(k_pages.shape)} {k_pages.dtype}, {tuple(v_pages.shape)} {v_pages.dtype})")
    P, Hkv, page, hd = k_pages.shape
    _refuse(k_pages.dtype not in _DTYPES, f"the cache holds bf16 or f16 (got {k_pages.dtype})")
    _refuse(page not in PAGE_SIZES or hd not in (64, 128) or P < 1 or Hkv < 1,
            f"pages hold {PAGE_SIZES} tokens of head_dim 64 or 128 (got {tuple(k_pages.shape)})")
    strides = (page * hd, hd, 1)
    for t in (k_pages, v_pages):
        _refuse(t.stride()[1:] != strides or t.stride(0) % 8 or (P > 1 and t.stride(0) < Hkv * page * hd),
                f"pages must be packed in their last three dimensions (got strides {t.stride()})")
    _refuse(P > 1 and k_pages.stride(0) != v_pages.stride(0), "k_pages and v_pages must have one page stride")
    return P, Hkv, page, hd, max(k_pages.stride(0), Hkv * page * hd)


def _tables(block_table, seq_lens, cu_seqlens):
    _refuse(block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.size(1) < 1
            or (block_table.size(1) > 1 and block_table.stride(1) != 1)
            or (block_table.size(0) > 1 and block_table.stride(0) < block_table.size(1)),
            f"block_table must be int32 [num_seqs, max_pages], rows packed (got {block_table.dtype} "
            f"{tuple(block_table.shape)}, strides {block_table.stride()})")
    n = block_table.size(0)
    for name, t, want in (("seq_lens", seq_lens, n), ("cu_seqlens", cu_seqlens, n + 1)):
        _refuse(t is not None and (t.dim() != 1 or t.dtype != torch.int32 or t.numel() != want or not t.is_contiguous()),
                f"{name} must be a contiguous int32 [{want}] (got {t.dtype if t is not None else None} "
                f"{tuple(t.shape) if t is not None else None})")
    return n, max(block_table.stride(0), block_table.size(1))


def paged_append(qkvg, k_pages, v_pages, block_table, seq_lens, *, n_heads, cu_seqlens=None, q_weight=None,
                 k_weight=None, eps=1e-6, cos=None, sin=None):
    """q [T, n_heads, hd] of packed new tokens, their keys and values stored in their pages.

    qkvg [T, W] (the pages' dtype): n_heads query heads, Hkv key heads and Hkv value heads of a
    token in one row (columns after them are not read).  q and k: per-head zero-centred RMSNorm
    (q_weight, k_weight f32 [hd]; None: no norm), then the first `rot` pairs (i, i + hd/2) turned
    by cos/sin f32 [positions, rot] at the token's position (None: no rotation); f32 arithmetic,
    one rounding.  cu_seqlens None: row s is sequence s's one new token.  A row outside every
    sequence, or at a negative position (an empty slot), gets a zero q and stores nothing."""
    _same_device(k_pages, v_pages, qkvg, block_table, seq_lens, cu_seqlens, q_weight, k_weight, cos, sin)
    _no_grad(qkvg, k_pages, v_pages, q_weight, k_weight)
    P, Hkv, page, hd, stride = _pages(k_pages, v_pages)
    H = int(n_heads)
    n, bt_ld = _tables(block_table, seq_lens, cu_seqlens)
    _refuse(qkvg.dim() != 2 or qkvg.dtype != k_pages.dtype or qkvg.size(1) < (H + 2 * Hkv) * hd or H < 1 or H % Hkv,
            f"qkvg must be {k_pages.dtype} [T, >= (H + 2 Hkv) hd] with H % Hkv == 0 (got {qkvg.dtype} "
            f"{tuple(qkvg.shape)}, H={H}, Hkv={Hkv}, hd={hd})")
    T = qkvg.size(0)
    _refuse(cu_seqlens is None and T != n, f"without cu_seqlens each sequence has one row (got {T} rows, {n} sequences)")
    _refuse((q_weight is None) != (k_weight is None), "q_weight and k_weight come together")
    if q_weight is not None:
        for w in (q_weight, k_weight):
            _refuse(w.dtype != torch.float32 or w.shape != (hd,), f"norm weights must be f32 [{hd}]")
        q_weight, k_weight = _aligned(q_weight), _aligned(k_weight)
    _refuse((cos is None) != (sin is None), "cos and sin come together")
    rot, rows, table_ld = 0, 0, 0
    if cos is not None:
        for t in (cos, sin):
            _refuse(t.dim() != 2 or t.dtype != torch.float32 or t.shape != cos.shape or t.size(1) > hd // 2
                    or t.size(0) < 1, f"cos and sin must be f32 [positions, rot <= {hd // 2}] of one shape")
        if (cos.stride(1) != 1 or sin.stride(1) != 1 or cos.stride(0) != sin.stride(0)
                or cos.stride(0) < cos.size(1)):
            cos, sin = cos.contiguous(), sin.contiguous()
        rows, rot = cos.shape
        table_ld = max(cos.stride(0), rot)
    q = torch.empty(T, H, hd, dtype=qkvg.dtype, device=qkvg.device)
    if T == 0 or n == 0:
        return q.zero_()
    if qkvg.stride(1) != 1 or qkvg.stride(0) % 8 or qkvg.data_ptr() % 16 or (T > 1 and qkvg.stride(0) < qkvg.size(1)):
        qkvg = qkvg[:, :(H + 2 * Hkv) * hd].contiguous()
        qkvg = qkvg.clone() if qkvg.data_ptr() % 16 else qkvg
    Z.count(1)
    Z.check(Z.lib().zs_paged_append(
        qkvg.data_ptr(), max(qkvg.stride(0), (H + 2 * Hkv) * hd), Z.ptr(q_weight), Z.ptr(k_weight), float(eps),
        Z.ptr(cos) if rot else None, Z.ptr(sin) if rot else None, table_ld, rows, rot, k_pages.data_ptr(),
        v_pages.data_ptr(), stride, P, block_table.data_ptr(), bt_ld, block_table.size(1), seq_lens.data_ptr(),
        Z.ptr(cu_seqlens), n, T, H, Hkv, hd, page, q.data_ptr(), Z.dtype_code(q.dtype), Z.stream_of(q)),
        "zs_paged_append")
    return q


def _aligned(t):
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _attention_inputs(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, window, k_sink, gate, scale):
    _same_device(k_pages, v_pages, q, block_table, seq_lens, cu_seqlens, k_sink, gate)
    _no_grad(q, k_pages, v_pages, k_sink, gate)
    P, Hkv, page, hd, stride = _pages(k_pages, v_pages)
    n, bt_ld = _tables(block_table, seq_lens, cu_seqlens)
    _refuse(q.dim() != 3 or q.dtype != k_pages.dtype or q.size(2) != hd or q.size(1) < 1 or q.size(1) % Hkv,
            f"q must be {k_pages.dtype} [T, H, {hd}] with H % Hkv == 0 (got {q.dtype} {tuple(q.shape)}, Hkv={Hkv})")
    T, H, _ = q.shape
    _refuse(cu_seqlens is None and T != n, f"q has one row per sequence (got {T} rows, {n} sequences)")
    w = 0 if window is None else int(window)
    _refuse(window is not None and (w <= 0 or w >= 1 << 31), f"window must be None or positive (got {window!r})")
    if k_sink is not None:
        _refuse(k_sink.shape != (H, hd), f"k_sink must be [{H}, {hd}] (got {tuple(k_sink.shape)})")
        k_sink = k_sink.contiguous()
        Z.dtype_code(k_sink.dtype)
    ldg = 0
    if gate is not None:
        _refuse(gate.shape != (T, H) or gate.dtype != q.dtype,
                f"gate must be {q.dtype} [{T}, {H}] (got {gate.dtype} {tuple(gate.shape)})")
        if (H > 1 and gate.stride(1) != 1) or (T > 1 and gate.stride(0) < H):
            gate = gate.contiguous()
        ldg = max(gate.stride(0), H)
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if (q.stride(2) != 1 or (H > 1 and q.stride(1) != hd) or q.stride(0) % 8 or q.data_ptr() % 16
            or (T > 1 and q.stride(0) < H * hd)):
        q = q.contiguous()
        q = q.clone() if q.data_ptr() % 16 else q
    head = (q.data_ptr(), max(q.stride(0), H * hd), k_pages.data_ptr(), v_pages.data_ptr(), stride, P,
            block_table.data_ptr(), bt_ld, block_table.size(1), seq_lens.data_ptr())
    o = torch.empty(T, H, hd, dtype=q.dtype, device=q.device)
    tail = (H, Hkv, hd, page, w, scale, Z.ptr(k_sink), Z.dtype_code(k_sink.dtype) if k_sink is not None else 0,
            Z.ptr(gate), ldg, o.data_ptr())
    return n, head, tail, o, (q, k_sink, gate)


def _lse_of(return_lse, o):
    return torch.empty(o.shape[:2], dtype=torch.float32, device=o.device) if return_lse else None


def paged_prompt_attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, *, window=None, k_sink=None,
                           gate=None, scale=None, return_lse=False):
    """o [T, H, hd] (with return_lse also the f32 log-sum-exp [T, H]) of packed new tokens q
    [T, H, hd]: softmax attention over the keys at or before each token's position in its own
    sequence (the last `window` of them), key head h // (H // Hkv), scale 1/sqrt(hd) by default.
    k_sink [H, hd]: one more logit q . k_sink per head whose value is zero.  gate [T, H] (q's dtype;
    a strided view will do): o is multiplied by sigmoid(gate).  Rows that see no key, and rows
    outside every sequence, are zero."""
    n, head, tail, o, keep = _attention_inputs(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, window, k_sink,
                                               gate, scale)
    _refuse(cu_seqlens is None, "cu_seqlens is required")
    lse = _lse_of(return_lse, o)
    if o.size(0) == 0 or n == 0:
        o.zero_()
        return (o, lse.fill_(-math.inf)) if return_lse else o
    Z.count(1)
    Z.check(Z.lib().zs_paged_prompt_attention(*head, cu_seqlens.data_ptr(), n, o.size(0), *tail, Z.ptr(lse),
                                              Z.dtype_code(o.dtype), Z.stream_of(o)), "zs_paged_prompt_attention")
    return (o, lse) if return_lse else o


def paged_decode_attention(q, k_pages, v_pages, block_table, seq_lens, *, window=None, k_sink=None, gate=None,
                           scale=None, return_lse=False):
    """paged_prompt_attention for one new token per sequence: row s of q [num_seqs, H, hd] is the
    last token of sequence s.  The keys of a sequence are split over thread blocks and joined in a
    fixed order.  seq_lens[s] == 0 marks an empty slot: its row is zero."""
    n, head, tail, o, keep = _attention_inputs(q, k_pages, v_pages, block_table, seq_lens, None, window, k_sink, gate,
                                               scale)
    lse = _lse_of(return_lse, o)
    if n:
        L = Z.lib()
        ws = torch.empty(int(L.zs_paged_decode_workspace(n, o.size(1), k_pages.size(1), o.size(2))),
                         dtype=torch.uint8, device=o.device)
        Z.count(1)
        Z.check(L.zs_paged_decode_attention(*head, n, *tail, Z.ptr(lse), Z.dtype_code(o.dtype), ws.data_ptr(),
                                            ws.numel(), Z.stream_of(o)), "zs_paged_decode_attention")
    return (o, lse) if return_lse else o


class PagedKVCache:
    """The pages of all layers and the tables that say who holds them, on one device.

    kv [n_layers, 2, num_pages, n_kv_heads, page_size, head_dim] (keys, values); a slot is a row of
    block_table [max_seqs, max_pages_per_seq] (-1: no page) with its length in seq_lens;
    ref_count [num_pages] counts the rows that hold a page.  The three tables are views of one
    int32 tensor `meta`, so a copy of it is a snapshot of the bookkeeping.

    Requests are int32 CUDA tensors (a list or int is uploaded); they are served in order and take
    the lowest-numbered free pages.  Nothing here waits for the host: a request that cannot be
    served changes nothing and is recorded in the device error word, which check() reads."""

    def __init__(self, n_layers, n_kv_heads, head_dim, *, num_pages, page_size=64, max_seqs, max_pages_per_seq,
                 dtype=torch.bfloat16, device="cuda"):
        device = torch.device(device)
        _refuse(device.type != "cuda", f"the cache lives on a CUDA device (got {device})")
        _refuse(dtype not in _DTYPES or page_size not in PAGE_SIZES or head_dim not in (64, 128),
                f"the cache holds bf16 or f16 pages of {PAGE_SIZES} tokens of head_dim 64 or 128 (got {dtype}, "
                f"{page_size}, {head_dim})")
        _refuse(min(n_layers, n_kv_heads, num_pages, max_seqs, max_pages_per_seq) < 1 or num_pages > 2_000_000
                or max_pages_per_seq * page_size >= 1 << 31,
                "n_layers, n_kv_heads, num_pages (at most 2000000), max_seqs and max_pages_per_seq must be positive")
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

    def _requests(self, *lists):
        out = []
        for x in lists:
            if isinstance(x, int):
                x = [x]
            if not torch.is_tensor(x):
                x = torch.tensor(list(x), dtype=torch.int32, device=self.kv.device)
            _refuse(x.dtype != torch.int32 or x.dim() != 1 or not x.is_contiguous() or x.device != self.kv.device,
                    f"requests are contiguous int32 [n] tensors on {self.kv.device} (got {x.dtype} {tuple(x.shape)} "
                    f"on {x.device})")
            out.append(x)
        _refuse(len({x.numel() for x in out}) != 1, "request lists must have one length")
        return out

    def _workspace(self, n):
        return torch.empty(int(Z.lib().zs_kv_workspace(ctypes.byref(self._c), n)), dtype=torch.uint8,
                           device=self.kv.device)

    def _call(self, name, launches, *lists):
        n = lists[0].numel() if lists else 0
        if lists and n == 0:
            return
        ws = self._workspace(n)
        Z.count(launches)
        args = [x.data_ptr() for x in lists] + ([n] if lists else [])
        Z.check(getattr(Z.lib(), name)(ctypes.byref(self._c), *args, ws.data_ptr(), ws.numel(),
                                       Z.stream_of(self.kv)), name)

    def extend(self, slots, n_tokens):
        """Slot slots[i] grows by n_tokens[i] >= 0 tokens, with pages for them; what they hold is
        up to the caller (paged_append).  A slot named twice grows by its first request only."""
        self._call("zs_kv_extend", 1, *self._requests(slots, n_tokens))

    def fork(self, src, dst):
        """Slot dst[i] becomes a copy of slot src[i] as it was before the call (beam search:
        fork(parents, slots)); what dst[i] held is let go.  Whole pages are shared; the filled
        rows of a last partial page are copied into a page of dst[i]'s own."""
        self._call("zs_kv_fork", 4, *self._requests(src, dst))

    def free(self, slots):
        """Slots become empty; pages that no slot holds any more are free."""
        (s,) = self._requests(slots)
        if s.numel():
            Z.count(1)
            Z.check(Z.lib().zs_kv_free(ctypes.byref(self._c), s.data_ptr(), s.numel(), Z.stream_of(self.kv)),
                    "zs_kv_free")

    def compact(self):
        """The pages in use become pages 0 .. U-1 (the k-th free page below U takes the k-th used
        page from U on), so everything held lies in one run at the start of the pool."""
        self._call("zs_kv_compact", 3)

    def copy_pages(self, src, dst):
        """Page dst[i] = page src[i], every layer's keys and values; the tables stay.  A page that
        is written must not also be read by the call."""
        self._call("zs_kv_copy_pages", 2, *self._requests(src, dst))
