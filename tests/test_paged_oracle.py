"""The paged restatements against the contiguous attention oracle, and the refusals that the C entry
points make before they touch the device."""
import ctypes

import numpy as np
import pytest

from oracle import attention as A
from oracle import paged as O


@pytest.mark.parametrize("window,sink", [(0, False), (5, True), (40, False)])
def test_attention_over_pages_is_attention(window, sink):
    r = np.random.default_rng(0)
    S, H, Hkv, hd, page = 37, 4, 2, 64, 16
    q, k, v = r.normal(size=(1, S, H, hd)), r.normal(size=(1, S, Hkv, hd)), r.normal(size=(1, S, Hkv, hd))
    ks = r.normal(size=(H, hd)) if sink else None
    ref, _ = A.attention_forward(q, k, v, window=window, k_sink=ks)
    table = [[4, 1, 6]]
    kp, vp = (np.full((8, Hkv, page, hd), np.nan) for _ in range(2))
    for p in range(S):
        kp[table[0][p // page], :, p % page] = k[0, p]
        vp[table[0][p // page], :, p % page] = v[0, p]
    for n in (S, 9, 1):                 # a whole prompt, its last part after a prefix, one token
        o, lse, spread, _ = O.attention(q[0, S - n:], kp, vp, table, [S], [0, n], window=window, k_sink=ks)
        np.testing.assert_allclose(o, np.asarray(ref, dtype=np.float64)[0, S - n:], rtol=1e-5, atol=1e-5)
        assert np.isfinite(lse).all() and (spread >= np.abs(o) - 1e-12).all()


def test_cache_conserves_pages():
    r = np.random.default_rng(1)
    c = O.Cache(r.normal(size=(1, 2, 30, 1, 16, 64)), 5, 8)
    for _ in range(300):
        a, b = ([int(x) for x in r.integers(0, 5, 3)] for _ in range(2))
        r.choice([lambda: c.extend(a, [int(x) for x in r.integers(0, 40, 3)]), lambda: c.fork(a, b),
                  lambda: c.free(a[:1]), c.compact])()
        held = [p for row in c.table for p in row if p >= 0]
        assert [held.count(p) for p in range(30)] == c.ref
        assert [sum(p >= 0 for p in row) for row in c.table] == [-(-n // 16) for n in c.lens]


def _attn_args(**kw):
    # numbers in place of pointers: a refused call reads none of them
    a = dict(q=1 << 20, ldq=512, k=1 << 21, v=1 << 22, stride=2 * 16 * 64, pages=4, table=1 << 23, bt_ld=3, max_pages=3,
             lens=1 << 24, cu=1 << 25, n=2, tokens=5, H=8, Hkv=2, hd=64, page=16, window=0, scale=0.1, sink=None,
             gate=None, ldg=0, o=1 << 26, lse=None, dtype=1)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(o=None), 1), (dict(table=None), 1), (dict(cu=None), 1), (dict(dtype=0), 3),
    (dict(hd=96), 2), (dict(page=48), 2), (dict(H=7), 2), (dict(n=0), 2), (dict(tokens=0), 2), (dict(pages=0), 2),
    (dict(bt_ld=2), 2), (dict(window=-1), 2), (dict(scale=-0.1), 1), (dict(ldq=504), 2), (dict(stride=64), 7), (dict(stride=2 * 16 * 64 + 4), 7),
    (dict(q=(1 << 20) + 2), 4), (dict(k=(1 << 21) + 8), 4), (dict(ldq=516), 4), (dict(sink=(1 << 27) + 4), 4),
    (dict(gate=1 << 27, ldg=7), 2), (dict(max_pages=1 << 28, bt_ld=1 << 28), 2)])
def test_entry_points_refuse_before_the_device(kw, code):
    from zs_b200 import _lib, build

    build.build()
    L = _lib.lib()
    args = _attn_args(**kw)
    assert L.zs_paged_prompt_attention(*args, 1 << 28, 1 << 40, None) == code
    if "cu" not in kw and "tokens" not in kw:
        d = args[:10] + [args[11]] + args[13:]
        assert L.zs_paged_decode_attention(*d, 1 << 28, 1 << 40, None) == code
    if not kw.keys() & {"o", "window", "scale", "sink", "gate", "ldq", "cu", "q"}:
        a = dict(zip(("q", "ldq", "k", "v", "stride", "pages", "table", "bt_ld", "max_pages", "lens", "cu", "n",
                      "tokens", "H", "Hkv", "hd", "page"), args))
        assert L.zs_paged_append(a["q"], 2048, None, None, 1e-6, None, None, 0, 0, 0, a["k"], a["v"], a["stride"],
                                 a["pages"], a["table"], a["bt_ld"], a["max_pages"], a["lens"], a["cu"], a["n"],
                                 a["tokens"], a["H"], a["Hkv"], a["hd"], a["page"], 1 << 26, args[-1], None) == code


def test_attention_refuses_a_missing_workspace():
    from zs_b200 import _lib

    L = _lib.lib()
    args = _attn_args()
    d = args[:10] + [args[11]] + args[13:]
    assert L.zs_paged_decode_attention(*d, None, 1 << 40, None) == 6
    assert L.zs_paged_decode_attention(*d, 1 << 28, 0, None) == 6
    assert L.zs_paged_prompt_attention(*args, None, 1 << 40, None) == 6
    assert L.zs_paged_prompt_workspace(5, 2, 8, 2, 64, 3, 16, 0) > 0


@pytest.mark.parametrize("kw,code", [(dict(kv=None), 1), (dict(num_pages=0), 2), (dict(num_pages=2000001), 2),
                                     (dict(page_size=20), 2), (dict(head_dim=32), 2), (dict(max_pages=0), 2),
                                     (dict(kv=(1 << 20) + 4), 4), ({}, 6)])
def test_bookkeeping_refuses_before_the_device(kw, code):
    from zs_b200 import _lib

    L = _lib.lib()
    f = dict(kv=1 << 20, block_table=1 << 21, seq_lens=1 << 22, ref_count=1 << 23, num_pages=8, n_layers=1,
             n_kv_heads=1, page_size=16, head_dim=64, max_seqs=2, max_pages=4)
    f.update(kw)
    c = ctypes.byref(_lib.KvCache(*f.values()))
    assert L.zs_kv_extend(c, 1 << 24, 1 << 25, 2, None, 0, None) == code
    assert L.zs_kv_fork(c, 1 << 24, 1 << 25, 2, 1 << 26, 0, None) == code
    assert L.zs_kv_compact(c, 1 << 26, 0, None) == code
    assert L.zs_kv_copy_pages(c, 1 << 24, 1 << 25, 2, 1 << 26, 0, None) == code
    if code != 6:
        assert L.zs_kv_free(c, 1 << 24, 2, None) == code


def test_operators_refuse_cpu_tensors():
    import torch

    from zs_b200 import ZsError, paged

    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ZsError):
        paged.paged_decode_attention(q, k, k, t, n)
    with pytest.raises(ZsError):
        paged.paged_prompt_attention(q, k, k, t, n, torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(ZsError):
        paged.paged_append(torch.zeros(1, 192, dtype=torch.bfloat16), k, k, t, n, n_heads=1)
    with pytest.raises(ZsError):
        paged.PagedKVCache(1, 1, 64, num_pages=2, max_seqs=1, max_pages_per_seq=1, device="cpu")
