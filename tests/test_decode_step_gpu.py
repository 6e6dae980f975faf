"""DecodeStep: what a recorded step leaves alone, and when it is recorded again."""
import pytest
import torch

from test_generate_gpu import _model

pytestmark = pytest.mark.gpu


def _prefill(m, c, slots, ids):
    n = torch.tensor([len(x) for x in ids], dtype=torch.int32, device="cuda")
    cu = torch.cat([n.new_zeros(1), n.cumsum(0).int()])
    c.extend(slots, n)
    at = torch.tensor(slots, device="cuda")
    return m.forward_paged(torch.cat(ids).cuda(), c, c.block_table[at], c.seq_lens[at], cu)


def _seq(c, slot):
    """Keys and values of a slot's tokens, all layers."""
    n, page = int(c.seq_lens[slot]), c.page_size
    ids = c.block_table[slot, :-(-n // page)].long()
    x = c.kv[:, :, ids].transpose(2, 3)                       # [L, 2, Hkv, pages, page, hd]
    return x.reshape(*x.shape[:3], -1, x.size(-1))[..., :n, :].clone()


@pytest.mark.parametrize("length", [32, 37])
def test_a_slot_that_does_not_grow_keeps_its_tokens(length):
    """Of two slots forked at a page's end (or inside a page) one is idle while the other goes on: both keep
    what they hold, and the idle one goes on later as if it had not waited."""
    from zs_b200.generate import DecodeStep

    cfg, m = _model()
    ids = torch.randint(0, cfg.vocab_size, (length,), generator=torch.Generator().manual_seed(2))

    def run(idle_first):
        c = m.new_cache(2, 96, page_size=16, num_pages=14)
        _prefill(m, c, [0], [ids])
        c.fork([0], [1])
        step = DecodeStep(m, c)
        out = []
        for k in range(4):
            step.active.copy_(torch.tensor([1, 0 if idle_first else 1]))
            step.tokens.copy_(torch.tensor([5 + k, 900 - k]))
            was = _seq(c, 1)
            out.append(step()[0].clone())
            if idle_first:
                assert torch.equal(_seq(c, 1), was)
        if idle_first:
            assert int(c.seq_lens[1]) == length
            later = []
            for k in range(4):
                step.active.copy_(torch.tensor([0, 1]))
                step.tokens.copy_(torch.tensor([0, 900 - k]))
                was = _seq(c, 0)
                later.append(step()[1].clone())
                assert torch.equal(_seq(c, 0), was)
        c.check()
        return out, _seq(c, 0), _seq(c, 1)

    a, a0, a1 = run(False)
    b, b0, b1 = run(True)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert torch.equal(a0, b0) and torch.equal(a1, b1)


def test_a_step_that_finds_no_page_changes_no_token():
    from zs_b200 import ZsError
    from zs_b200.generate import DecodeStep

    cfg, m = _model(layers=2, windows=(None, 40))
    g = torch.Generator().manual_seed(5)
    ids = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (16, 20)]
    c = m.new_cache(2, 32, page_size=16, num_pages=3)
    _prefill(m, c, [0, 1], ids)                              # three pages, slot 0 at its page's end
    step = DecodeStep(m, c)
    step.active.fill_(1)
    step.tokens.copy_(torch.tensor([7, 8]))
    for k in range(3):                                       # the first one runs, the others are replays
        was = _seq(c, 0)
        step()
        assert int(c.seq_lens[0]) == 16 and int(c.seq_lens[1]) == 21 + k
        assert torch.equal(_seq(c, 0), was)
        with pytest.raises(ZsError, match="no free page"):
            c.check()
