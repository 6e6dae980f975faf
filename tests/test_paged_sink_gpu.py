"""The key sink is f32 whatever the type of the queries: values that f16 does not hold, large and small ones.  Bounds as
in test_paged_gpu.py."""
import pytest
import torch

from test_paged_gpu import LENS, NEW, _check, _world

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hkv,hd", [(6, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("q_gain,sink_gain", [(2.0 ** -9, 2.0 ** 9), (2.0 ** -12, 2.0 ** 18), (2.0 ** -5, 2.0 ** 17),
                                              (2.0 ** 9, 2.0 ** -22), (2.0 ** 9, 2.0 ** -30), (1.0, 0.0)])
def test_sinks_beyond_f16(H, Hkv, hd, q_gain, sink_gain):
    """Queries times sink stays moderate, the sink itself does not; one head's sink is ordinary, one is zero."""
    from zs_b200 import paged

    w = _world(LENS, NEW, H=H, Hkv=Hkv, hd=hd, page=64, dtype=torch.float16, sink=torch.float32, gate=True, gain=q_gain)
    w["ks"] *= sink_gain
    w["ks"][1] /= sink_gain if sink_gain else 1.0
    w["ks"][2] = 0
    # one element far above the others
    w["ks"][3, 5] *= 2.0 ** 8
    scale = 0.05
    o, lse = paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True, scale=scale)
    _check(w, o, lse, scale=scale)
    w["q"], w["gate"] = w["q"][:len(LENS)].contiguous(), w["gate"][:len(LENS)].contiguous()
    w["cu"] = torch.arange(len(LENS) + 1, dtype=torch.int32, device="cuda")
    o, lse = paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], k_sink=w["ks"],
                                          gate=w["gate"], return_lse=True, scale=scale)
    _check(w, o, lse, scale=scale)
