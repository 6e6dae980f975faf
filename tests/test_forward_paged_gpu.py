"""MoELM.forward_paged and new_cache at their edges."""
import pytest
import torch

from _util import rel_err
from test_generate_gpu import TOL, _logits, _model

pytestmark = pytest.mark.gpu


def test_a_sequence_without_new_tokens_gets_no_other_ones_logits():
    cfg, m = _model()
    g = torch.Generator(device="cuda").manual_seed(1)
    seqs = [torch.randint(0, cfg.vocab_size, (n,), device="cuda", generator=g) for n in (30, 21, 40, 18)]
    c = m.new_cache(4, 128, page_size=16)
    slots = torch.arange(4, dtype=torch.int32, device="cuda")

    def run(parts):
        n = torch.tensor([p.numel() for p in parts], dtype=torch.int32, device="cuda")
        cu = torch.cat([n.new_zeros(1), n.cumsum(0).int()])
        c.extend(slots, n)
        return m.forward_paged(torch.cat(parts), c, c.block_table, c.seq_lens, cu)

    none = seqs[0][:0]
    run([none, seqs[1], none, seqs[3]])
    was = c.kv.clone()
    got = run([seqs[0], none, seqs[2], none])
    for i in (0, 2):
        assert rel_err(got[i], _logits(m, seqs[i])[-1]) < TOL
    assert (got[1] == 0).all() and (got[3] == 0).all()
    for s in (1, 3):                                         # and their tokens stay
        ids = c.block_table[s, :2].long()
        assert torch.equal(c.kv[:, :, ids], was[:, :, ids])
    got = run([none, none, none, none])
    assert got.shape == (4, cfg.vocab_size) and (got == 0).all()
    c.check()


def test_rows_beyond_the_tokens_are_not_read():
    """cu_seqlens that count more rows than there are: no row outside the call's is asked for."""
    from zs_b200 import _lib as Z

    cfg, m = _model(layers=1, windows=(None,))
    c = m.new_cache(2, 64, page_size=16)
    c.extend([0, 1], [8, 50])
    ids = torch.randint(0, cfg.vocab_size, (20,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    cu = torch.tensor([0, 8, 58], dtype=torch.int32, device="cuda")
    got = m.forward_paged(ids, c, c.block_table, c.seq_lens, cu)
    assert rel_err(got[0], _logits(m, ids[:8])[-1]) < TOL
    assert torch.isfinite(got).all() and Z.device_error() == 0


def test_a_default_cache_forks_between_full_slots():
    """Every slot holds as many tokens as it may, none shares a page: each takes over another one's sequence."""
    cfg, m = _model(layers=1, windows=(None,))
    c = m.new_cache(3, 40, page_size=16)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    c.extend(slots, torch.tensor([40, 39, 33], dtype=torch.int32, device="cuda"))
    c.kv.copy_(torch.randn(c.kv.shape, device="cuda"))

    def held(s):
        n = int(c.seq_lens[s])
        x = c.kv[:, :, c.block_table[s, :-(-n // 16)].long()].transpose(2, 3)
        return x.reshape(*x.shape[:3], -1, x.size(-1))[..., :n, :].clone()

    was = [held(s) for s in range(3)]
    for _ in range(5):                                       # the pages let go serve the next fork
        c.fork([1, 2, 0], [0, 1, 2])
        c.check()
        was = [was[1], was[2], was[0]]
        for s in range(3):
            assert torch.equal(held(s), was[s])


def test_packed_prompts_through_sparse_routing():
    """Two of eight experts a token.  A rounding may swap two experts of nearly one score, so sequences are compared
    whose routing is the same in both paths; short ones, so that most are."""
    from test_decode_step_gpu import _sparse_model

    cfg, m = _sparse_model()
    g = torch.Generator().manual_seed(7)
    seqs = [torch.randint(0, cfg.vocab_size, (1 + i % 6,), generator=g).cuda() for i in range(60)]
    n = torch.tensor([s.numel() for s in seqs], dtype=torch.int32, device="cuda")
    cu = torch.cat([n.new_zeros(1), n.cumsum(0).int()])
    c = m.new_cache(len(seqs), 32, page_size=16)
    chosen = []
    hooks = [b.mlp.register_forward_hook(lambda _m, _a, out: chosen.append(out[1][0].sort(-1)[0])) for b in m.layers]
    c.extend(torch.arange(len(seqs), dtype=torch.int32, device="cuda"), n)
    got = m.forward_paged(torch.cat(seqs), c, c.block_table, c.seq_lens, cu)
    for h in hooks:
        h.remove()
    assert len(torch.stack(chosen).unique()) == 8            # every expert has tokens
    alike = 0
    for i, s in enumerate(seqs):
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            want, routing = m(s.view(1, -1))
        rows = slice(int(cu[i]), int(cu[i + 1]))
        if all(torch.equal(a[rows], b[0].sort(-1)[0]) for a, b in zip(chosen, routing)):
            alike += 1
            assert rel_err(got[i], want[0, -1].float()) < TOL
    assert alike >= len(seqs) // 2
    c.check()
