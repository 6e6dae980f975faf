"""What the paged operators refuse beside wrong types and sizes: inputs that carry a tangent (they have no derivative
in either direction), and a cache whose tensors were replaced (its bookkeeping would go on in the old memory)."""
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


@pytest.mark.parametrize("name", ["kv", "block_table", "seq_lens", "ref_count"])
@pytest.mark.parametrize("how", ["replaced", "moved"])
def test_a_cache_whose_tensors_were_replaced_is_refused(name, how):
    from zs_b200 import ZsError, paged

    c = paged.PagedKVCache(1, 1, 64, num_pages=8, page_size=16, max_seqs=2, max_pages_per_seq=4)
    c.extend([0], [20])
    old = getattr(c, name)
    was = old.clone()
    if how == "replaced":
        setattr(c, name, old.clone())
    else:
        old.data = old.data.clone()
    for call in (lambda: c.extend([0], [1]), lambda: c.fork([0], [1]), lambda: c.free([0]), lambda: c.compact(),
                 lambda: c.copy_pages([0], [5])):
        with pytest.raises(ZsError, match="instead of replacing"):
            call()
    assert torch.equal(getattr(c, name), was)
