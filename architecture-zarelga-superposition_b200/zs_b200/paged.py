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
import functools
import math

import torch

from . import _lib as Z

PAGE_SIZES = (16, 32, 64, 128)
_DTYPES = {torch.bfloat16: Z.ZS_BF16, torch.float16: Z.ZS_F16}


def _fail(msg):
    raise Z.ZsError(msg)


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail("the paged operators have no gradient: call them under torch.no_grad() or on detached tensors")


def _same_device(first, *tensors):
    """Index of the CUDA device that holds all the tensors."""
    dev = first.get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            Z.require_cuda(t)
            _fail(f"all tensors must be on one device (got {first.device} and {t.device})")
    if dev < 0:
        Z.require_cuda(first)
    return dev


# One decode step is a few microseconds of kernel time per call, so the checks below read each
# tensor's shape and strides once and build their messages only when they refuse.

def _pages(k_pages, v_pages):
    """(num_pages, Hkv, page, hd, page stride, dtype) of a layer's pages."""
    shape, dtype = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != dtype:
        _fail(f"k_pages and v_pages must be [num_pages, Hkv, page, hd] of one shape and dtype (got "
              f"{tuple(shape)} {dtype}, {tuple(v_pages.shape)} {v_pages.dtype})")
    P, Hkv, page, hd = shape
    if dtype not in _DTYPES or page not in PAGE_SIZES or hd not in (64, 128) or P < 1 or Hkv < 1:
        _fail(f"the cache holds bf16 or f16 pages of {PAGE_SIZES} tokens of head_dim 64 or 128 (got {dtype} "
              f"{tuple(shape)})")
    ks, vs = k_pages.stride(), v_pages.stride()
    run = page * hd
    if P == 1:
        ks, vs = (Hkv * run,) + ks[1:], (Hkv * run,) + vs[1:]
    if ks != vs or ks[0] % 8 or ks[0] < Hkv * run or ks[3] != 1 or ks[2] != hd or (ks[1] != run and Hkv > 1):
        _fail("k_pages and v_pages must be packed in their last three dimensions, with one page stride that is a "
              f"multiple of 8 (got strides {k_pages.stride()}, {v_pages.stride()})")
    return P, Hkv, page, hd, ks[0], dtype


def _int32_list(name, t, want):
    if t.dtype != torch.int32 or t.shape != (want,) or not t.is_contiguous():
        _fail(f"{name} must be a contiguous int32 [{want}] (got {t.dtype} {tuple(t.shape)})")


def _tables(block_table, seq_lens, cu_seqlens):
    """(num_seqs, max_pages, row stride) of the block table."""
    shape = block_table.shape
    if len(shape) != 2 or block_table.dtype != torch.int32 or shape[1] < 1:
        _fail(f"block_table must be int32 [num_seqs, max_pages] (got {block_table.dtype} {tuple(shape)})")
    n, m = shape
    ld, inner = block_table.stride()
    if (inner != 1 and m > 1) or (ld < m and n > 1):
        _fail(f"block_table rows must be packed and apart (got strides {block_table.stride()})")
    _int32_list("seq_lens", seq_lens, n)
    if cu_seqlens is not None:
        _int32_list("cu_seqlens", cu_seqlens, n + 1)
    return n, m, max(ld, m)


def _aligned(t):
    if t.stride(0) != 1:
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def paged_append(qkvg, k_pages, v_pages, block_table, seq_lens, *, n_heads, cu_seqlens=None, q_weight=None,
                 k_weight=None, eps=1e-6, cos=None, sin=None):
    """q [T, n_heads, hd] of packed new tokens, their keys and values stored in their pages.

    qkvg [T, W] (the pages' dtype): n_heads query heads, Hkv key heads and Hkv value heads of a
    token in one row (columns after them are not read).  q and k: per-head zero-centred RMSNorm
    (q_weight, k_weight f32 [hd]; None: no norm), then the first `rot` pairs (i, i + hd/2) turned
    by cos/sin f32 [positions, rot] at the token's position (None: no rotation); f32 arithmetic,
    one rounding.  cu_seqlens None: row s is sequence s's one new token.  A row outside every
    sequence, or at a negative position (an empty slot), gets a zero q and stores nothing."""
    dev = _same_device(k_pages, v_pages, qkvg, block_table, seq_lens, cu_seqlens, q_weight, k_weight, cos, sin)
    _no_grad(qkvg, k_pages, v_pages, q_weight, k_weight)
    P, Hkv, page, hd, stride, dtype = _pages(k_pages, v_pages)
    n, m, bt_ld = _tables(block_table, seq_lens, cu_seqlens)
    H = int(n_heads)
    width = (H + 2 * Hkv) * hd
    shape = qkvg.shape
    if len(shape) != 2 or qkvg.dtype != dtype or shape[1] < width or H < 1 or H % Hkv:
        _fail(f"qkvg must be {dtype} [T, >= (H + 2 Hkv) hd] with H % Hkv == 0 (got {qkvg.dtype} {tuple(shape)}, "
              f"H={H}, Hkv={Hkv}, hd={hd})")
    T = shape[0]
    if cu_seqlens is None and T != n:
        _fail(f"without cu_seqlens each sequence has one row (got {T} rows, {n} sequences)")
    if (q_weight is None) != (k_weight is None):
        _fail("q_weight and k_weight come together")
    if q_weight is not None:
        for w in (q_weight, k_weight):
            if w.dtype != torch.float32 or w.shape != (hd,):
                _fail(f"norm weights must be f32 [{hd}] (got {w.dtype} {tuple(w.shape)})")
        q_weight, k_weight = _aligned(q_weight), _aligned(k_weight)
    if (cos is None) != (sin is None):
        _fail("cos and sin come together")
    rot = rows = table_ld = 0
    if cos is not None:
        shape = cos.shape
        if (len(shape) != 2 or sin.shape != shape or cos.dtype != torch.float32 or sin.dtype != torch.float32
                or shape[1] > hd // 2 or shape[0] < 1):
            _fail(f"cos and sin must be f32 [positions, rot <= {hd // 2}] of one shape (got {cos.dtype} "
                  f"{tuple(shape)}, {sin.dtype} {tuple(sin.shape)})")
        rows, rot = shape
        st = cos.stride()
        if sin.stride() != st or st[1] != 1 or st[0] < rot:
            cos, sin = cos.contiguous(), sin.contiguous()
            st = (rot, 1)
        table_ld = st[0]
    q = qkvg.new_empty((T, H, hd))
    if T == 0 or n == 0:
        return q.zero_()
    ld, inner = qkvg.stride()
    x = qkvg.data_ptr()
    if inner != 1 or ld % 8 or x % 16 or (T > 1 and ld < width):
        qkvg = qkvg[:, :width].clone(memory_format=torch.contiguous_format)
        x, ld = qkvg.data_ptr(), width
    Z.count(1)
    rc = Z.lib().zs_paged_append(
        x, max(ld, width), Z.ptr(q_weight), Z.ptr(k_weight), eps, cos.data_ptr() if rot else None,
        sin.data_ptr() if rot else None, table_ld, rows, rot, k_pages.data_ptr(), v_pages.data_ptr(), stride, P,
        block_table.data_ptr(), bt_ld, m, seq_lens.data_ptr(), Z.ptr(cu_seqlens), n, T, H, Hkv, hd, page,
        q.data_ptr(), _DTYPES[dtype], torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        Z.check(rc, "zs_paged_append")
    return q


@functools.lru_cache(maxsize=64)
def _decode_workspace(H, Hkv, hd):
    return Z.lib().zs_paged_decode_workspace(1, H, Hkv, hd)   # the same for any number of sequences


@functools.lru_cache(maxsize=256)
def _prompt_workspace(*sizes):
    return Z.lib().zs_paged_prompt_workspace(*sizes)


def _attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, window, k_sink, gate, scale, return_lse, decode):
    dev = _same_device(k_pages, v_pages, q, block_table, seq_lens, cu_seqlens, k_sink, gate)
    _no_grad(q, k_pages, v_pages, k_sink, gate)
    P, Hkv, page, hd, stride, dtype = _pages(k_pages, v_pages)
    n, m, bt_ld = _tables(block_table, seq_lens, cu_seqlens)
    shape = q.shape
    if len(shape) != 3 or q.dtype != dtype or shape[2] != hd or shape[1] < 1 or shape[1] % Hkv:
        _fail(f"q must be {dtype} [T, H, {hd}] with H % Hkv == 0 (got {q.dtype} {tuple(shape)}, Hkv={Hkv})")
    T, H, _ = shape
    if decode:
        if T != n:
            _fail(f"q has one row per sequence (got {T} rows, {n} sequences)")
    elif H // Hkv > 128:
        _fail(f"at most 128 query heads share a key head (got H={H}, Hkv={Hkv})")
    w = 0
    if window is not None:
        w = int(window)
        if w <= 0 or w >= 1 << 31:
            _fail(f"window must be None or positive (got {window!r})")
    if k_sink is not None:
        if k_sink.shape != (H, hd) or not k_sink.is_floating_point():
            _fail(f"k_sink must be a floating-point [{H}, {hd}] (got {k_sink.dtype} {tuple(k_sink.shape)})")
        if k_sink.dtype != torch.float32 or not k_sink.is_contiguous() or k_sink.data_ptr() % 16:
            k_sink = k_sink.to(torch.float32, copy=True, memory_format=torch.contiguous_format)
    ldg = 0
    if gate is not None:
        if gate.shape != (T, H) or gate.dtype != dtype:
            _fail(f"gate must be {dtype} [{T}, {H}] (got {gate.dtype} {tuple(gate.shape)})")
        ldg, inner = gate.stride()
        if (inner != 1 and H > 1) or (ldg < H and T > 1):
            gate = gate.contiguous()
            ldg = H
        ldg = max(ldg, H)
    o = q.new_empty((T, H, hd))
    lse = torch.empty((T, H), dtype=torch.float32, device=q.device) if return_lse else None
    if T == 0 or n == 0:
        o.zero_()
        return (o, lse.fill_(-math.inf)) if return_lse else o
    ldq, head, inner = q.stride()
    x = q.data_ptr()
    if inner != 1 or (head != hd and H > 1) or ldq % 8 or x % 16 or (T > 1 and ldq < H * hd):
        q = q.clone(memory_format=torch.contiguous_format)
        x, ldq = q.data_ptr(), H * hd
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    elif not scale >= 0.0:
        _fail(f"scale must not be negative (got {scale!r})")
    L = Z.lib()
    args = (x, max(ldq, H * hd), k_pages.data_ptr(), v_pages.data_ptr(), stride, P, block_table.data_ptr(), bt_ld, m,
            seq_lens.data_ptr())
    more = (H, Hkv, hd, page, w, scale, Z.ptr(k_sink), Z.ptr(gate), ldg, o.data_ptr(), Z.ptr(lse),
            _DTYPES[dtype])
    stream = torch._C._cuda_getCurrentRawStream(dev)
    Z.count(2)
    if decode:
        size = _decode_workspace(H, Hkv, hd)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        rc = L.zs_paged_decode_attention(*args, n, *more, ws.data_ptr(), size, stream)
    else:
        size = _prompt_workspace(T, n, H, Hkv, hd, m, page, w)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        rc = L.zs_paged_prompt_attention(*args, cu_seqlens.data_ptr(), n, T, *more, ws.data_ptr(), size, stream)
    if rc:
        Z.check(rc, "zs_paged_decode_attention" if decode else "zs_paged_prompt_attention")
    return (o, lse) if return_lse else o


def paged_prompt_attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, *, window=None, k_sink=None,
                           gate=None, scale=None, return_lse=False):
    """o [T, H, hd] (with return_lse also the f32 log-sum-exp [T, H]) of packed new tokens q
    [T, H, hd]: softmax attention over the keys at or before each token's position in its own
    sequence (the last `window` of them), key head h // (H // Hkv), scale 1/sqrt(hd) by default.
    k_sink [H, hd]: one more logit q . k_sink per head whose value is zero.  gate [T, H] (q's dtype;
    a strided view will do): o is multiplied by sigmoid(gate).  Rows that see no key, and rows
    outside every sequence, are zero."""
    return _attention(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, window, k_sink, gate, scale, return_lse,
                      False)


def paged_decode_attention(q, k_pages, v_pages, block_table, seq_lens, *, window=None, k_sink=None, gate=None,
                           scale=None, return_lse=False):
    """paged_prompt_attention for one new token per sequence: row s of q [num_seqs, H, hd] is the
    last token of sequence s.  The keys of a sequence are split over thread blocks and joined in a
    fixed order.  seq_lens[s] == 0 marks an empty slot: its row is zero."""
    return _attention(q, k_pages, v_pages, block_table, seq_lens, None, window, k_sink, gate, scale, return_lse, True)


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
        if device.type != "cuda":
            _fail(f"the cache lives on a CUDA device (got {device})")
        if dtype not in _DTYPES or page_size not in PAGE_SIZES or head_dim not in (64, 128):
            _fail(f"the cache holds bf16 or f16 pages of {PAGE_SIZES} tokens of head_dim 64 or 128 (got {dtype}, "
                  f"{page_size}, {head_dim})")
        if (min(n_layers, n_kv_heads, num_pages, max_seqs, max_pages_per_seq) < 1 or num_pages > 2_000_000
                or max_pages_per_seq * page_size > (1 << 31) - 256):
            _fail("n_layers, n_kv_heads, num_pages (at most 2000000), max_seqs and max_pages_per_seq must be positive")
        self.kv = torch.zeros(n_layers, 2, num_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device)
        cells = max_seqs * max_pages_per_seq
        self.meta = torch.empty(cells + max_seqs + num_pages, dtype=torch.int32, device=device)
        self.block_table = self.meta[:cells].view(max_seqs, max_pages_per_seq)
        self.seq_lens = self.meta[cells:cells + max_seqs]
        self.ref_count = self.meta[cells + max_seqs:]
        self.reset()
        self._dev = self.kv.get_device()
        self._c = ctypes.pointer(Z.KvCache(
            self.kv.data_ptr(), self.block_table.data_ptr(), self.seq_lens.data_ptr(), self.ref_count.data_ptr(),
            num_pages, n_layers, n_kv_heads, page_size, head_dim, max_seqs, max_pages_per_seq))

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

    def _requests(self, lists):
        out = []
        for x in lists:
            if not torch.is_tensor(x):
                x = torch.tensor([x] if isinstance(x, int) else list(x), dtype=torch.int32, device=self.kv.device)
            if x.dtype != torch.int32 or x.dim() != 1 or not x.is_contiguous() or x.get_device() != self._dev:
                _fail(f"requests are contiguous int32 [n] tensors on {self.kv.device} (got {x.dtype} "
                      f"{tuple(x.shape)} on {x.device})")
            out.append(x)
        if len(out) > 1 and out[0].shape != out[1].shape:
            _fail("request lists must have one length")
        return out

    def _call(self, name, launches, *lists):
        lists = self._requests(lists)
        n = lists[0].size(0) if lists else 0
        if lists and n == 0:
            return
        L = Z.lib()
        size = L.zs_kv_workspace(self._c, n)
        ws = torch.empty(size, dtype=torch.uint8, device=self.kv.device)
        args = [x.data_ptr() for x in lists]
        if lists:
            args.append(n)
        Z.count(launches)
        rc = getattr(L, name)(self._c, *args, ws.data_ptr(), size, torch._C._cuda_getCurrentRawStream(self._dev))
        if rc:
            Z.check(rc, name)

    def extend(self, slots, n_tokens):
        """Slot slots[i] grows by n_tokens[i] >= 0 tokens, with pages for them; what they hold is
        up to the caller (paged_append).  A slot named twice grows by its first request only."""
        self._call("zs_kv_extend", 1, slots, n_tokens)

    def fork(self, src, dst):
        """Slot dst[i] becomes a copy of slot src[i] as it was before the call (beam search:
        fork(parents, slots)); what dst[i] held is let go.  Whole pages are shared; the filled
        rows of a last partial page are copied into a page of dst[i]'s own."""
        self._call("zs_kv_fork", 2, src, dst)

    def free(self, slots):
        """Slots become empty; pages that no slot holds any more are free."""
        (s,) = self._requests([slots])
        if s.numel():
            Z.count(1)
            Z.check(Z.lib().zs_kv_free(self._c, s.data_ptr(), s.numel(), Z.stream_of(self.kv)), "zs_kv_free")

    def compact(self):
        """The pages in use become pages 0 .. U-1 (the k-th free page below U takes the k-th used
        page from U on), so everything held lies in one run at the start of the pool."""
        self._call("zs_kv_compact", 2)

    def copy_pages(self, src, dst):
        """Page dst[i] = page src[i], every layer's keys and values; the tables stay.  A page that
        is written must not also be read by the call."""
        self._call("zs_kv_copy_pages", 2, src, dst)
