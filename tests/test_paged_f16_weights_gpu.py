"""f16 paged attention where one key takes nearly all the weight and has little value, so that the result comes from
many keys of tiny weights.

Bound.  As in test_paged_gpu.py, and one term more: f16 rounds a weight below its smallest normal number by up to
2^-25.  The kernels keep the largest weight of a key tile (at most 128 keys) at 2^7 or more of that unit, so the keys of
a tile lose at most 128 * 2^-25 / 2^7 = 2^-25 of the tile's largest weight, and all tiles together at most 2^-25 of the
sum of weights, times the largest value."""
import math

import numpy as np
import pytest
import torch

from oracle import paged as O
from test_paged_gpu import U, _np

pytestmark = pytest.mark.gpu

SCALE = math.log(2.0)          # a logit of x weighs 2^x


def _world(n, where, logit, top_value, hd, H=3, page=64, spread=False, seed=0):
    """n keys of logit 0 (spread: 0 to -3) and value near 1, but those at `where`: `logit` and top_value."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    M = -(-n // page)
    x = torch.zeros(n, 2, hd, device="cuda")
    if spread:
        x[:, 0, 0] = -3 * torch.rand(n, device="cuda", generator=g)
    x[:, 1] = 1 - 0.25 * torch.rand(n, hd, device="cuda", generator=g)
    x[where, 0, 0] = logit
    x[where, 1] = top_value
    pool = torch.zeros(M * page, 2, hd, device="cuda")
    pool[:n] = x
    pages = pool.half().view(M, page, 2, hd).permute(2, 0, 1, 3).unsqueeze(2).contiguous()
    q = torch.zeros(5, H, hd, device="cuda", dtype=torch.float16)
    q[:, :, 0] = 1
    table = torch.arange(M, dtype=torch.int32, device="cuda").view(1, M)
    return q, pages[0], pages[1], table, torch.tensor([n], dtype=torch.int32, device="cuda")


def _compare(q, k, v, table, lens, cu, o, lse):
    hd = q.size(2)
    ro, rl, spread, ds = O.attention(_np(q), _np(k), _np(v), table.cpu().numpy(), lens.tolist(), cu, scale=SCALE)
    dS = 2 * (hd + 8) * 2.0 ** -24 * ds
    u = U[torch.float16]
    vmax = v.abs().max().item()
    tol = 1.01 * (u * np.abs(ro) + spread * (u + 2 * dS[..., None] + 2.0 ** -14)) + 2.0 ** -24 + 2.0 ** -25 * vmax
    err = np.abs(_np(o) - ro)
    assert np.isfinite(_np(o)).all() and (err <= tol).all(), (err / tol).max()
    assert (np.abs(_np(lse) - rl) <= dS + 2.0 ** -14 + 2.0 ** -22 * np.abs(rl)).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("logit,n,spread", [(26, 32768, False), (24.625, 32768, False), (24.625, 20000, True),
                                            (20.5, 5000, True), (16.3, 700, True), (30, 32768, True), (60, 9000, True)])
@pytest.mark.parametrize("where", ["first", "last", "middle", "many"])
def test_small_weights_are_kept(hd, logit, n, spread, where):
    from zs_b200 import paged

    at = {"first": [0], "last": [n - 6], "middle": [n // 2], "many": list(range(3, n - 6, 500))}[where]
    q, k, v, table, lens = _world(n, at, logit, 0.0, hd, spread=spread)
    cu = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    o, lse = paged.paged_prompt_attention(q, k, v, table, lens, cu, scale=SCALE, return_lse=True)
    _compare(q, k, v, table, lens, [0, 5], o, lse)
    o, lse = paged.paged_decode_attention(q[:1], k, v, table, lens, scale=SCALE, return_lse=True)
    _compare(q[:1], k, v, table, lens, [0, 1], o, lse)


@pytest.mark.parametrize("hd", [64, 128])
def test_rising_and_falling_logits(hd):
    """Logits that climb, fall and jump by more than f16's range from tile to tile, values of both signs and sizes."""
    from zs_b200 import paged

    n = 3000
    q, k, v, table, lens = _world(n, [0], 0.0, 1.0, hd)
    g = torch.Generator(device="cuda").manual_seed(4)
    t = torch.arange(n, device="cuda", dtype=torch.float32)
    for wave in (t / 20, -t / 20, 40 * torch.sin(t / 90), 25 * ((t // 130) % 3 - 1), 100 * torch.sin(t)):
        flat_k, flat_v = torch.zeros(table.size(1) * 64, hd, device="cuda"), torch.zeros(table.size(1) * 64, hd, device="cuda")
        flat_k[:n, 0] = wave
        flat_v[:n] = torch.randn(n, hd, device="cuda", generator=g)
        k.copy_(flat_k.view(-1, 1, 64, hd)), v.copy_(flat_v.view(-1, 1, 64, hd))
        cu = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
        o, lse = paged.paged_prompt_attention(q, k, v, table, lens, cu, scale=SCALE, return_lse=True)
        _compare(q, k, v, table, lens, [0, 5], o, lse)
        o, lse = paged.paged_decode_attention(q[:1], k, v, table, lens, scale=SCALE, return_lse=True)
        _compare(q[:1], k, v, table, lens, [0, 1], o, lse)
