"""The paged key-value cache on the GPU against the float64 restatements of oracle/paged.py.

Tolerances.  With u = finfo(dtype).eps / 2 (half a step, relative), an output o = sum_k w_k v_k / sum_k w_k is
off by: its own rounding, u |o|; the weights' rounding to dtype for the products, u sum w|v| / sum w =
u * spread; the error of a logit, which moves a weight and the denominator by a relative 2 dS each way,
dS <= 2 (hd + 8) 2^-24 * (largest sum |q_i k_i| scale) for f32 sums of hd exact products (and the factor log2 e);
and the f32 softmax arithmetic (exp2 within 2^-21, sums of positive terms, joins of partial sums), 2^-14 of
spread in all.  Products of second order are covered by a factor 1.01.  Values below the smallest normal number
(f16) are off by at most its step, 2^-24."""
import math

import numpy as np
import pytest
import torch

from oracle import paged as O

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _world(lens, new, *, H, Hkv, hd, page, dtype, window=None, sink=None, gate=False, gain=1.0, seed=0, strided=False,
           poison=True, extra_rows=0):
    """A cache with sequences of the given lengths whose last new[s] tokens are the queries.  Everything
    that no query may see is NaN; the table past a sequence's pages holds numbers that are no page."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    M, P = max(1, max(need)) + 2, sum(need) + 3
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed + 1))
    pool = torch.randn(P, 2, Hkv, page, hd, device="cuda", generator=g).to(dtype)
    k, v = (pool[:, 0], pool[:, 1]) if strided else (pool[:, 0].contiguous(), pool[:, 1].contiguous())
    table = torch.full((len(lens), M), -123456, dtype=torch.int32)
    if poison:
        dead = torch.ones(P, page, dtype=torch.bool)
    at = 0
    for s, n in enumerate(lens):
        ids = order[at:at + need[s]]
        at += need[s]
        table[s, :need[s]] = ids.int()
        if poison:
            lo = max(0, n - new[s] - window + 1) if window else 0
            for p in range(lo, n):
                dead[ids[p // page], p % page] = False
    if poison:
        where = dead[:, None, :, None].expand(P, Hkv, page, hd).cuda()
        k.masked_fill_(where, float("nan"))
        v.masked_fill_(where, float("nan"))
    T = sum(new) + extra_rows
    width = H * hd + (16 if strided else 0)
    q = (torch.randn(T, width, device="cuda", generator=g) * gain).to(dtype)[:, :H * hd].view(T, H, hd) if not strided \
        else (torch.randn(T, width, device="cuda", generator=g) * gain).to(dtype).as_strided((T, H, hd), (width, hd, 1))
    ks = (torch.randn(H, hd, device="cuda", generator=g) * 0.5).to(sink) if sink is not None else None
    gt = torch.randn(T, H + 5, device="cuda", generator=g).to(dtype)[:, 3:3 + H] if gate else None
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    return dict(q=q, k=k, v=v, table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), cu=cu,
                window=window, ks=ks, gate=gt)


def _check(w, o, lse, scale=None):
    from zs_b200 import _lib as Z

    torch.cuda.synchronize()
    assert Z.device_error() == 0
    q = w["q"]
    hd = q.size(2)
    ro, rl, spread, ds = O.attention(_np(q), _np(w["k"]), _np(w["v"]), w["table"].cpu().numpy(), w["lens"].tolist(),
                                     w["cu"].tolist(), window=w["window"] or 0, k_sink=_np(w["ks"]),
                                     gate=_np(w["gate"]), scale=scale)
    u = U[q.dtype]
    dS = 2 * (hd + 8) * 2.0 ** -24 * ds
    tol = 1.01 * (u * np.abs(ro) + spread * (u + 2 * dS[..., None] + 2.0 ** -14)) + 2.0 ** -24
    err = np.abs(_np(o) - ro)
    assert np.isfinite(_np(o)).all()
    assert (err <= tol).all(), (err / tol).max()
    if lse is not None:
        got, none = _np(lse), np.isneginf(rl)
        assert np.isneginf(got[none]).all()
        assert (np.abs(got[~none] - rl[~none]) <= dS[~none] + 2.0 ** -14 + 2.0 ** -22 * np.abs(rl[~none])).all()


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 400, 1023]

# H, Hkv, hd, page, dtype, window, sink, gate, gain
ATTN = [
    (12, 4, 128, 64, torch.bfloat16, None, torch.float32, True, 1.0),
    (16, 4, 128, 64, torch.bfloat16, None, None, False, 1.0),
    (4, 4, 64, 16, torch.bfloat16, None, None, True, 1.0),
    (5, 1, 64, 32, torch.float16, 70, None, True, 1.0),
    (14, 2, 128, 128, torch.float16, None, torch.float16, False, 1.0),
    (32, 1, 128, 16, torch.bfloat16, 1, None, False, 1.0),
    (48, 2, 64, 64, torch.bfloat16, 129, torch.bfloat16, True, 1.0),
    (8, 1, 128, 32, torch.float16, None, None, False, 6.0),
    (6, 2, 128, 64, torch.bfloat16, 5, torch.float32, False, 6.0),
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("strided", [False, True])
def test_decode_matches_oracle(case, strided):
    from zs_b200 import paged

    H, Hkv, hd, page, dtype, window, sink, gate, gain = case
    w = _world(LENS, [1] * len(LENS), H=H, Hkv=Hkv, hd=hd, page=page, dtype=dtype, window=window, sink=sink, gate=gate,
               gain=gain, strided=strided, seed=H + hd)
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], window=window, k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True)
    _check(w, o, lse)
    again = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], window=window, k_sink=w["ks"],
                                         gate=w["gate"])
    assert torch.equal(o, again)                       # the joins have a fixed order


@pytest.mark.parametrize("lens", [[5000], [1], [0], [0, 0, 0], [4096, 0, 1], [3001, 2999], [20000]])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_few_sequences_split_over_their_length(lens, hd):
    from zs_b200 import paged

    w = _world(lens, [1] * len(lens), H=8, Hkv=2, hd=hd, page=64, dtype=torch.bfloat16, sink=torch.float32, seed=7)
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], k_sink=w["ks"],
                                          return_lse=True)
    _check(w, o, lse)


def test_decode_many_sequences():
    from zs_b200 import paged

    r = np.random.default_rng(0)
    lens = [int(x) for x in r.integers(0, 200, 700)]
    w = _world(lens, [1] * len(lens), H=2, Hkv=1, hd=64, page=16, dtype=torch.bfloat16, gate=True, seed=3)
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], gate=w["gate"],
                                          return_lse=True)
    _check(w, o, lse)


NEW = [0, 1, 2, 10, 3, 17, 60, 1, 65, 100, 128, 120, 257, 700]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("strided", [False, True])
def test_prompt_matches_oracle(case, strided):
    from zs_b200 import paged

    H, Hkv, hd, page, dtype, window, sink, gate, gain = case
    w = _world(LENS, NEW, H=H, Hkv=Hkv, hd=hd, page=page, dtype=dtype, window=window, sink=sink, gate=gate, gain=gain,
               strided=strided, seed=H + hd)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], window=window,
                                          k_sink=w["ks"], gate=w["gate"], return_lse=True, scale=0.11)
    _check(w, o, lse, scale=0.11)


@pytest.mark.parametrize("lens,new", [([1], [1]), ([37], [37]), ([600], [600]), ([3000], [4]), ([2500], [300]),
                                      ([5], [9]), ([0], [3]), ([130, 0, 1], [129, 0, 1])])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_few_sequences(lens, new, hd):
    """Among them sequences shorter than their new tokens: the first ones are padding."""
    from zs_b200 import paged

    w = _world(lens, new, H=3, Hkv=1, hd=hd, page=64, dtype=torch.bfloat16, seed=5)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], return_lse=True)
    _check(w, o, lse)


@pytest.mark.parametrize("H,Hkv,hd", [(128, 1, 64), (100, 1, 128), (66, 2, 64), (17, 1, 128)])
def test_large_groups(H, Hkv, hd):
    """Few tokens a tile, several blocks of query heads in a decode step, sinks in many columns."""
    from zs_b200 import paged

    lens, new = [1, 40, 300], [1, 7, 9]
    w = _world(lens, new, H=H, Hkv=Hkv, hd=hd, page=16, dtype=torch.bfloat16, sink=torch.float32, gate=True, seed=H)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True)
    _check(w, o, lse)
    w = _world(lens, [1] * 3, H=H, Hkv=Hkv, hd=hd, page=16, dtype=torch.bfloat16, sink=torch.float32, gate=True, seed=H)
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True)
    _check(w, o, lse)


@pytest.mark.parametrize("lens,new", [([5], [9]), ([0, 3], [30, 200]), ([130], [400])])
def test_prompt_before_the_first_position(lens, new):
    """Tokens at negative positions (more new tokens than the sequence is long): zero rows, whose
    log-sum-exp is the sink's logit."""
    from zs_b200 import paged

    w = _world(lens, new, H=6, Hkv=2, hd=64, page=16, dtype=torch.float16, sink=torch.float32, gate=True)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True)
    _check(w, o, lse)


def test_prompt_rows_of_no_sequence_are_zero():
    from zs_b200 import paged

    w = _world([70, 33], [70, 20], H=4, Hkv=2, hd=64, page=16, dtype=torch.bfloat16, sink=torch.float32, gate=True,
               extra_rows=300)
    w["q"][90:] = float("nan")
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True)
    assert (o[90:] == 0).all() and torch.isneginf(lse[90:]).all()
    for n in ("q", "gate"):
        w[n] = w[n][:90]
    _check(w, o[:90], lse[:90])


def test_decode_equals_the_last_row_of_a_prompt():
    from zs_b200 import paged

    w = _world([100, 257], [100, 257], H=12, Hkv=4, hd=128, page=32, dtype=torch.bfloat16)
    full = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"])
    last = (w["cu"][1:] - 1).long()
    one = paged.paged_decode_attention(w["q"][last], w["k"], w["v"], w["table"], w["lens"])
    w1 = dict(w, q=w["q"][last], cu=torch.arange(3, dtype=torch.int32, device="cuda"))
    _check(w1, one, None)
    _check(w1, full[last], None)


def test_pages_far_apart_pass_32_bits():
    """A pool of more than 2^32 bytes whose last pages are in use."""
    from zs_b200 import paged

    P, Hkv, page, hd = 70000, 4, 64, 128           # 70000 * 64 KiB = 4.6 GB each of keys and values
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.empty(P, Hkv, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ids = [P - 1, 3, P - 2, 40000]
    for p in ids:
        k[p] = torch.randn(Hkv, page, hd, device="cuda", generator=g).bfloat16()
        v[p] = torch.randn(Hkv, page, hd, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([250], dtype=torch.int32, device="cuda")
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    q = torch.randn(250, 4, hd, device="cuda", generator=g).bfloat16()
    cu = torch.tensor([0, 250], dtype=torch.int32, device="cuda")
    o, lse = paged.paged_prompt_attention(q, k, v, table, lens, cu, return_lse=True)
    one = paged.paged_decode_attention(q[-1:], k, v, table, lens)
    sub = torch.tensor(ids, device="cuda")
    w = dict(q=q, k=k[sub], v=v[sub], table=torch.tensor([[0, 1, 2, 3]]), lens=lens, cu=cu, window=None, ks=None,
             gate=None)
    _check(w, o, lse)
    _check(dict(w, q=q[-1:], cu=torch.tensor([0, 1])), one, None)
    x = torch.randn(250, 3 * 4 * hd, device="cuda", generator=g).bfloat16()
    paged.paged_append(x, k, v, table, lens, n_heads=4, cu_seqlens=cu)
    assert torch.equal(v[P - 1].transpose(0, 1), x[:64, 8 * hd:].view(64, 4, hd))


@pytest.mark.parametrize("page", [16, 128])
def test_bad_pages_read_as_zeros_and_are_recorded(page):
    """Page numbers out of range never reach memory: such keys are zeros (logit 0, value 0)."""
    from zs_b200 import _lib as Z
    from zs_b200 import paged

    w = _world([300, 40], [300, 40], H=4, Hkv=2, hd=64, page=page, dtype=torch.bfloat16, poison=False)
    zero = w["k"].size(0) - 1                       # a page that nobody holds
    while zero in w["table"][0].tolist() or zero in w["table"][1].tolist():
        zero -= 1
    w["k"][zero] = 0
    w["v"][zero] = 0
    good, bad = w["table"].clone(), w["table"].clone()
    for j, p in ((0, -1), (300 // page, w["k"].size(0)), (1, 2 ** 31 - 1)):
        good[0, j], bad[0, j] = zero, p
    args = (w["q"], w["k"], w["v"])
    Z.clear_device_error()
    ref = paged.paged_prompt_attention(*args, good, w["lens"], w["cu"])
    ref1 = paged.paged_decode_attention(w["q"][-2:], w["k"], w["v"], good, w["lens"])
    assert Z.device_error() == 0
    got = paged.paged_prompt_attention(*args, bad, w["lens"], w["cu"])
    assert Z.device_error() == 0x10
    Z.clear_device_error()
    got1 = paged.paged_decode_attention(w["q"][-2:], w["k"], w["v"], bad, w["lens"])
    assert Z.device_error() == 0x10
    Z.clear_device_error()
    assert torch.equal(got, ref) and torch.equal(got1, ref1)
    k0, v0 = w["k"].clone(), w["v"].clone()
    x = torch.randn(340, 8 * 64, device="cuda").bfloat16()
    q = paged.paged_append(x, w["k"], w["v"], bad, w["lens"], n_heads=4, cu_seqlens=w["cu"])
    assert Z.device_error() == 0x10
    Z.clear_device_error()
    paged.paged_append(x, k0, v0, good, w["lens"], n_heads=4, cu_seqlens=w["cu"])
    k0[zero], v0[zero] = 0, 0
    assert torch.equal(w["k"], k0) and torch.equal(w["v"], v0)
    lost = torch.zeros(340, dtype=torch.bool, device="cuda")
    for j in (0, 1, 300 // page):
        lost[j * page:min(300, (j + 1) * page)] = True
    assert (q[lost] == 0).all() and torch.equal(q[~lost].flatten(1), x[~lost][:, :256])


def test_lengths_beyond_the_table_are_cut_and_recorded():
    from zs_b200 import _lib as Z
    from zs_b200 import paged

    w = _world([128], [4], H=2, Hkv=1, hd=64, page=16, dtype=torch.bfloat16, poison=False)
    table = w["table"][:, :8].contiguous()
    over = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    Z.clear_device_error()
    paged.paged_decode_attention(w["q"][:1], w["k"], w["v"], table, over)
    assert Z.device_error() == 0x10
    Z.clear_device_error()
    paged.paged_prompt_attention(w["q"], w["k"], w["v"], table, over, w["cu"])
    assert Z.device_error() == 0x10
    Z.clear_device_error()
    under = torch.tensor([-5], dtype=torch.int32, device="cuda")
    assert (paged.paged_decode_attention(w["q"][:1], w["k"], w["v"], table, under) == 0).all()
    assert (paged.paged_prompt_attention(w["q"], w["k"], w["v"], table, under, w["cu"]) == 0).all()
    assert Z.device_error() == 0


# ------------------------------------------------------------------------------------ append

# H, Hkv, hd, page, dtype, norm, rot
APPEND = [
    (12, 4, 128, 64, torch.bfloat16, True, 8),
    (4, 4, 64, 16, torch.float16, True, 32),
    (5, 1, 64, 32, torch.bfloat16, False, 12),
    (16, 2, 128, 128, torch.float16, True, 0),
    (3, 3, 128, 16, torch.bfloat16, False, 0),
    (7, 1, 128, 64, torch.bfloat16, True, 61),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("decode", [False, True])
def test_append_matches_oracle(case, decode):
    from zs_b200 import _lib as Z
    from zs_b200 import paged

    H, Hkv, hd, page, dtype, norm, rot = case
    new = [1] * len(LENS) if decode else NEW
    w = _world(LENS, new, H=H, Hkv=Hkv, hd=hd, page=page, dtype=dtype, poison=False, seed=11, strided=True)
    T = sum(new)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(T, (H + 2 * Hkv) * hd + 24, device="cuda", generator=g).to(dtype)
    wq, wk = (torch.randn(hd, device="cuda", generator=g) * 0.3 for _ in range(2)) if norm else (None, None)
    cos = sin = None
    if rot:
        ang = torch.rand(1100, rot, device="cuda", generator=g) * 6.3
        cos, sin = ang.cos(), ang.sin()
    k0, v0 = w["k"].clone(), w["v"].clone()
    q = paged.paged_append(x, w["k"], w["v"], w["table"], w["lens"], n_heads=H, q_weight=wq, k_weight=wk, cos=cos,
                           sin=sin, cu_seqlens=None if decode else w["cu"])
    assert Z.device_error() == 0
    rq, rk, rv, (qs, ks) = O.append(_np(x), _np(k0), _np(v0), w["table"].cpu().numpy(), w["lens"].tolist(),
                                    w["cu"].tolist(), n_heads=H, q_weight=_np(wq), k_weight=_np(wk), cos=_np(cos),
                                    sin=_np(sin))
    # one rounding, and f32 arithmetic on |a| + |b|: a sum of hd squares (its relative error halves
    # in the root), the root, three products, two of the rotation: (hd / 2 + 8) 2^-24
    for got, ref, size in ((q, rq, qs), (w["k"], rk, ks)):
        assert (np.abs(_np(got) - ref) <= 1.01 * U[dtype] * np.abs(ref) + (hd / 2 + 8) * 2.0 ** -24 * size
                + 2.0 ** -24).all()
    assert np.array_equal(_np(w["v"]), rv)
    # what is neither a new token's key nor value keeps its bits
    same = torch.from_numpy(rk == _np(k0)).cuda()
    assert torch.equal(w["k"][same], k0[same])


def test_append_leaves_rows_behind_the_last_sequence_and_empty_slots():
    from zs_b200 import _lib as Z
    from zs_b200 import paged

    w = _world([20, 9], [5, 9], H=2, Hkv=2, hd=64, page=16, dtype=torch.bfloat16, poison=False, extra_rows=40)
    k0, v0 = w["k"].clone(), w["v"].clone()
    x = torch.randn(54, 6 * 64, device="cuda").bfloat16()
    x[14:] = float("nan")
    q = paged.paged_append(x, w["k"], w["v"], w["table"], w["lens"], n_heads=2, cu_seqlens=w["cu"])
    assert (q[14:] == 0).all()
    changed = (w["v"] != v0).any(3).any(1).sum().item()
    assert changed == 14
    empty = torch.zeros(2, dtype=torch.int32, device="cuda")
    w["k"].copy_(k0), w["v"].copy_(v0)
    q = paged.paged_append(x[:2], w["k"], w["v"], w["table"], empty, n_heads=2)
    assert (q == 0).all() and torch.equal(w["k"], k0) and torch.equal(w["v"], v0)
    assert Z.device_error() == 0
    # a position past the rotation table is refused
    cos = torch.ones(10, 4, device="cuda")
    q = paged.paged_append(x[:14], w["k"], w["v"], w["table"], w["lens"], n_heads=2, cu_seqlens=w["cu"], cos=cos,
                           sin=cos)
    assert Z.device_error() == 0x10
    Z.clear_device_error()
    assert (q[:5] == 0).all() and (q[5:] != 0).any(2).all()


# ------------------------------------------------------------------------------ bookkeeping

def _cache(P=40, page=16, slots=6, M=9, L=2, Hkv=3, hd=64, seed=0, dtype=torch.bfloat16):
    from zs_b200 import paged

    c = paged.PagedKVCache(L, Hkv, hd, num_pages=P, page_size=page, max_seqs=slots, max_pages_per_seq=M, dtype=dtype)
    c.kv.copy_(torch.randn(c.kv.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
    return c, O.Cache(c.kv.float().cpu().numpy(), slots, M)


def _same(c, ref, refused=0):
    from zs_b200 import _lib as Z

    assert c.meta.tolist() == ref.meta()
    assert np.array_equal(c.kv.float().cpu().numpy(), ref.kv)
    assert (Z.device_error() != 0) == (ref.refused != refused)
    Z.clear_device_error()


@pytest.mark.parametrize("page,dtype", [(16, torch.bfloat16), (32, torch.float16), (64, torch.bfloat16),
                                        (128, torch.bfloat16)])
def test_bookkeeping_matches_oracle_over_a_long_run(page, dtype):
    """Random requests of every kind, among them slots out of range, named twice and pools that run out."""
    c, ref = _cache(page=page, dtype=dtype, seed=page)
    r = np.random.default_rng(page)
    for step in range(120):
        before = ref.refused
        op = r.choice(["extend", "extend", "fork", "free", "compact", "copy"])
        n = int(r.integers(1, 8))
        slots = [int(x) for x in r.integers(-1 if r.random() < 0.1 else 0, 7 if r.random() < 0.1 else 6, n)]
        if r.random() < 0.6:
            slots = list(dict.fromkeys(slots))
        n = len(slots)
        if op == "extend":
            t = [int(x) for x in r.integers(-1 if r.random() < 0.1 else 0, int(r.choice([2, page, 4 * page])) + 1, n)]
            c.extend(slots, t), ref.extend(slots, t)
        elif op == "fork":
            src = [int(x) for x in r.integers(0, 6, n)]
            c.fork(src, slots), ref.fork(src, slots)
        elif op == "free":
            c.free(slots[:2]), ref.free(slots[:2])
        elif op == "compact":
            c.compact(), ref.compact()
        else:
            a, b = ([int(x) for x in r.integers(0, 41 if r.random() < 0.1 else 40, n)] for _ in range(2))
            c.copy_pages(a, b), ref.copy_pages(a, b)
        _same(c, ref, before)


def test_large_tables():
    """More requests than a block has threads, more pages than it looks at in one pass."""
    c, ref = _cache(P=20000, page=16, slots=2100, M=8, L=1, Hkv=1)
    r = np.random.default_rng(5)
    slots = [int(x) for x in r.permutation(2100)]
    t = [int(x) for x in r.integers(0, 8 * 16 + 1, 2100)]
    c.extend(slots, t), ref.extend(slots, t)
    _same(c, ref)
    c.free(slots[::2]), ref.free(slots[::2])
    src = [int(x) for x in r.integers(0, 2100, 1500)]
    c.fork(src, slots[:1500]), ref.fork(src, slots[:1500])
    _same(c, ref)
    c.compact(), ref.compact()
    _same(c, ref)
    c.compact(), ref.compact()          # nothing to do
    _same(c, ref)


@pytest.mark.parametrize("n,M", [(1024, 4), (1024, 12), (1025, 4), (1025, 12), (300, 40), (1, 9000)])
def test_many_requests(n, M):
    """On both sides of a block's threads, of the cells that it rewrites itself and of the pages that it lists."""
    S = 1100 if M < 100 else 8
    c, ref = _cache(P=16000, page=16, slots=S, M=M, L=1, Hkv=1)
    r = np.random.default_rng(n + M)
    slots = [int(x) for x in r.permutation(S)[:n]]
    for most in (16, 30, min(M, 20) * 16 - 46):
        t = [int(x) for x in r.integers(0, most + 1, n)]
        c.extend(slots, t), ref.extend(slots, t)
        _same(c, ref)
    src, dst = (slots if n > 1 else slots * 2), [int(x) for x in r.permutation(S)[:max(n, 2)]]
    c.fork(src, dst), ref.fork(src, dst)
    _same(c, ref)
    c.fork(dst, src[:1] + dst[1:]), ref.fork(dst, src[:1] + dst[1:])
    _same(c, ref)


def test_lengths_below_zero_are_refused():
    """A table that is not the cache's own: nothing is written before a row of the table."""
    from zs_b200 import _lib as Z

    c, _ = _cache()
    c.extend([0, 1], [20, 20])
    c.seq_lens[1] = -1000
    before = c.meta.clone()
    c.extend([1], [5])
    assert torch.equal(c.meta, before) and Z.device_error() == 0x10
    Z.clear_device_error()
    c.fork([1], [2])
    assert torch.equal(c.meta, before) and Z.device_error() == 0x10
    Z.clear_device_error()
    c.extend([0, 1], [30, 1])
    assert c.seq_lens.tolist()[:2] == [50, -1000] and c.block_table[0, :4].min() >= 0
    assert (c.block_table[1:] == before[:54].view(6, 9)[1:]).all()
    Z.clear_device_error()


def test_beam_permutation_and_check():
    from zs_b200 import ZsError

    c, ref = _cache()
    c.extend([0, 1, 2], [40, 33, 48]), ref.extend([0, 1, 2], [40, 33, 48])
    c.fork([1, 2, 0, 0], [0, 1, 2, 3]), ref.fork([1, 2, 0, 0], [0, 1, 2, 3])
    _same(c, ref)
    c.check()
    c.extend([0], [10 ** 6])
    with pytest.raises(ZsError, match="without room"):
        c.check()
    c.check()
    with pytest.raises(ZsError):
        c.extend([0, 1], [3])
    c.free([])
    c.reset()
    assert c.meta[:-40].tolist() == [-1] * 54 + [0] * 6 and c.ref_count.sum().item() == 0


# ----------------------------------------------------------------------- refusals and streams

def test_refusals():
    from zs_b200 import ZsError, paged

    w = _world([30, 20], [3, 2], H=4, Hkv=2, hd=64, page=16, dtype=torch.bfloat16)

    def call(f=paged.paged_prompt_attention, **kw):
        a = dict(w, **kw)
        extra = {k: a[k] for k in ("window", "k_sink", "gate", "scale") if k in kw}
        if f is paged.paged_prompt_attention:
            return f(a["q"], a["k"], a["v"], a["table"], a["lens"], a["cu"], **extra)
        return f(a["q"][:2], a["k"], a["v"], a["table"], a["lens"], **extra)

    call()
    call(paged.paged_decode_attention)
    bad = [dict(q=w["q"].half()), dict(q=w["q"][:, :3]), dict(q=w["q"].cpu()), dict(k=w["k"].float(), v=w["v"].float()),
           dict(k=w["k"][:, :, :8], v=w["v"][:, :, :8]), dict(k=w["k"].transpose(1, 2)), dict(v=w["v"][:, :1]),
           dict(table=w["table"].long()), dict(table=w["table"][0]), dict(lens=w["lens"].long()),
           dict(scale=-1.0), dict(scale=float("nan")), dict(lens=w["lens"][:1]), dict(cu=w["cu"][:2]), dict(cu=w["cu"].long()), dict(window=0), dict(window=-3),
           dict(k_sink=torch.zeros(3, 64, device="cuda")), dict(gate=torch.zeros(5, 4, device="cuda")),
           dict(gate=torch.zeros(4, 4, device="cuda", dtype=torch.bfloat16)),
           dict(q=w["q"].clone().requires_grad_(True)), dict(table=w["table"][:1].expand(2, -1))]
    for kw in bad:
        with pytest.raises(ZsError):
            call(**kw)
    with pytest.raises(ZsError):
        paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"])
    x = torch.zeros(5, 8 * 64, dtype=torch.bfloat16, device="cuda")
    t = torch.ones(64, 8, device="cuda")

    def app(x=x, cu=w["cu"], **kw):
        return paged.paged_append(x, w["k"], w["v"], w["table"], w["lens"], **dict(dict(n_heads=4, cu_seqlens=cu), **kw))

    app()
    for kw in (dict(x=x[:, :500]), dict(x=x.float()), dict(cu=None), dict(n_heads=3), dict(n_heads=0),
               dict(q_weight=torch.zeros(64, device="cuda")), dict(cos=t), dict(cos=t, sin=t[:3]),
               dict(cos=t.double(), sin=t.double()), dict(cos=t.repeat(1, 5), sin=t.repeat(1, 5)),
               dict(x=x.clone().requires_grad_(True))):
        with pytest.raises(ZsError):
            app(**kw)
    for kw in (dict(page_size=8), dict(page_size=48), dict(num_pages=0), dict(max_seqs=0), dict(dtype=torch.float32),
               dict(num_pages=2_000_001), dict(device="cpu")):
        with pytest.raises(ZsError):
            paged.PagedKVCache(1, 1, kw.pop("hd", 64), **dict(dict(num_pages=2, max_seqs=1, max_pages_per_seq=1), **kw))


def test_empty_calls():
    from zs_b200 import paged

    w = _world([30], [3], H=4, Hkv=2, hd=64, page=16, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    none = (w["table"][:0], torch.zeros(0, **i32), torch.zeros(1, **i32))
    assert paged.paged_decode_attention(w["q"][:0], w["k"], w["v"], *none[:2]).shape == (0, 4, 64)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], *none, return_lse=True)
    assert (o == 0).all() and torch.isneginf(lse).all()
    assert paged.paged_append(torch.zeros(0, 512, dtype=torch.bfloat16, device="cuda"), w["k"], w["v"], *none[:2],
                              n_heads=4).shape == (0, 4, 64)


def test_graphs_share_nothing_and_replay():
    """Two captured decode steps replayed at the same time on two streams, and a capture whose tables
    change between replays."""
    from zs_b200 import paged

    ws = [_world([900, 30, 2000], [1] * 3, H=8, Hkv=2, hd=128, page=64, dtype=torch.bfloat16, seed=s) for s in (1, 2)]

    def call(w):
        return paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"])

    want = [call(w) for w in ws]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for w in ws:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(w))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in ws]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, r in zip(outs, want):
        assert torch.equal(o, r)
    w = ws[0]
    w["lens"].copy_(torch.tensor([64, 0, 1999], dtype=torch.int32))
    graphs[0].replay()
    _check(w, outs[0], None)


def test_bookkeeping_and_append_in_a_graph():
    from zs_b200 import paged

    c, ref = _cache(P=30, page=16, slots=3, M=9, L=1, Hkv=2)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    one = torch.ones(3, dtype=torch.int32, device="cuda")
    x = torch.randn(3, 6 * 64, device="cuda").bfloat16()
    c.extend(slots, one)
    ref.extend([0, 1, 2], [1, 1, 1])
    k, v = c.layer(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.extend(slots, one)
        q = paged.paged_append(x, k, v, c.block_table, c.seq_lens, n_heads=2)
        o = paged.paged_decode_attention(q, k, v, c.block_table, c.seq_lens)
    for _ in range(40):
        g.replay()
        ref.extend([0, 1, 2], [1, 1, 1])
    torch.cuda.synchronize()
    assert c.meta.tolist() == ref.meta()
    assert torch.isfinite(o).all()
    for s in range(3):
        for p in range(1, 41):
            assert torch.equal(v[ref.table[s][p // 16], :, p % 16].flatten(), x[s, 256:])


def test_prompt_and_page_moves_in_graphs():
    """A prompt, a fork, a compaction and a copy recorded and replayed, two prompts at once."""
    from zs_b200 import paged

    ws = [_world([700, 90], [500, 90], H=8, Hkv=2, hd=128, page=32, dtype=torch.bfloat16, seed=s) for s in (3, 4)]

    def call(w):
        return paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"])

    want = [call(w) for w in ws]
    graphs, outs = [], []
    for w in ws:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(w))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in ws]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, r in zip(outs, want):
        assert torch.equal(o, r)

    c, ref = _cache(P=40, page=16, slots=6, M=9)
    c.extend([0, 1, 2, 3], [40, 33, 48, 100]), ref.extend([0, 1, 2, 3], [40, 33, 48, 100])
    i32 = dict(dtype=torch.int32, device="cuda")
    src, dst, one = (torch.tensor(x, **i32) for x in ([1, 0, 3], [0, 4, 5], [2, 1]))
    a, b = torch.tensor([0, 3], **i32), torch.tensor([39, 38], **i32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.fork(src, dst)
        c.free(one)
        c.compact()
        c.copy_pages(a, b)
    for _ in range(3):
        g.replay()
        ref.fork([1, 0, 3], [0, 4, 5]), ref.free([2, 1]), ref.compact(), ref.copy_pages([0, 3], [39, 38])
        c.extend([1, 2], [20, 5]), ref.extend([1, 2], [20, 5])
    _same(c, ref)


def test_work_behind_a_call_sees_its_results():
    """Nothing to join (one tile a sequence): what follows in the stream still waits for the call."""
    from zs_b200 import paged

    w = _world([60] * 600, [1] * 600, H=16, Hkv=16, hd=128, page=64, dtype=torch.bfloat16, poison=False)
    table = w["table"].contiguous()
    want = paged.paged_decode_attention(w["q"], w["k"], w["v"], table, w["lens"]).clone()
    torch.cuda.synchronize()
    for _ in range(20):
        got = paged.paged_decode_attention(w["q"], w["k"], w["v"], table, w["lens"])
        copy = got.clone()
        got.zero_()
        assert torch.equal(copy, want)
        assert (got == 0).all()


def test_another_stream():
    from zs_b200 import paged

    w = _world([500, 77], [1, 1], H=8, Hkv=2, hd=64, page=16, dtype=torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"])
        p = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"])
    torch.cuda.current_stream().wait_stream(s)
    _check(w, o, None)
    _check(w, p, None)
