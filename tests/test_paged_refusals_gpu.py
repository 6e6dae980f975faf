"""Inputs that carry a tangent: the paged operators have no derivative in either direction."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from test_paged_gpu import _world

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["q", "k", "ks", "gate"])
def test_tangents_are_refused(which):
    from zs_b200 import ZsError, paged

    w = _world([20, 9], [1, 1], H=2, Hkv=2, hd=64, page=16, dtype=torch.bfloat16, sink=torch.float32, gate=True,
               poison=False)

    def both():
        kw = dict(k_sink=w["ks"], gate=w["gate"])
        paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], w["cu"], **kw)
        paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"], **kw)

    both()
    with fwAD.dual_level():
        w[which] = fwAD.make_dual(w[which], torch.ones_like(w[which]))
        for no_grad in (False, True):
            with torch.set_grad_enabled(not no_grad):
                for call in (lambda: paged.paged_prompt_attention(w["q"], w["k"], w["v"], w["table"], w["lens"],
                                                                  w["cu"], k_sink=w["ks"], gate=w["gate"]),
                             lambda: paged.paged_decode_attention(w["q"], w["k"], w["v"], w["table"], w["lens"],
                                                                  k_sink=w["ks"], gate=w["gate"])):
                    with pytest.raises(ZsError, match="derivative|gradient"):
                        call()
        if which == "k":
            x = torch.randn(2, 6 * 64, device="cuda").bfloat16()
            with pytest.raises(ZsError, match="derivative|gradient"):
                paged.paged_append(x, w["k"], w["v"], w["table"], w["lens"], n_heads=2)
