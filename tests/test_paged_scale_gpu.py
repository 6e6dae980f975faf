"""Paged attention with a softmax scale of zero, or one so small that f32 holds it as zero or as a subnormal:
every visible key weighs the same.  Inputs and bounds as in test_paged_gpu.py (a logit's error is proportional to
the scale, so it vanishes here)."""
import pytest
import torch

from test_paged_gpu import LENS, NEW, _check, _world

pytestmark = pytest.mark.gpu

# lens, new, H, Hkv, hd, page, dtype, window, sink, gate
CASES = [
    (LENS, NEW, 12, 4, 128, 64, torch.bfloat16, None, torch.float32, True),
    (LENS, NEW, 5, 1, 64, 32, torch.float16, 70, None, True),
    ([3000], [4], 8, 2, 64, 64, torch.bfloat16, None, None, False),
    ([2500, 0, 40], [300, 0, 40], 4, 4, 128, 16, torch.float16, None, torch.float32, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x-{'-'.join(str(x).replace('torch.', '') for x in c[2:])}")
@pytest.mark.parametrize("scale", [0.0, 1e-300, 1e-45, 1e-39])
def test_a_scale_of_nothing_gives_the_mean(case, scale):
    from zs_b200 import paged

    lens, new, H, Hkv, hd, page, dtype, window, sink, gate = case
    kw = dict(H=H, Hkv=Hkv, hd=hd, page=page, dtype=dtype, window=window, sink=sink, gate=gate, seed=hd)
    w = _world(lens, new, **kw)
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], window=window,
                                          k_sink=w["ks"], gate=w["gate"], return_lse=True, scale=scale)
    _check(w, o, lse, scale=scale)
    w = _world(lens, [1] * len(lens), **kw)
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], window=window,
                                          k_sink=w["ks"], gate=w["gate"], return_lse=True, scale=scale)
    _check(w, o, lse, scale=scale)
