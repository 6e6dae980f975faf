"""DecodeStep: what a recorded step leaves alone, and when it is recorded again."""
import pytest
import torch
import torch.nn as nn

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


def _sparse_model():
    """Two of eight routed experts a token."""
    from modeling.model_config import ModelConfig
    from zs_b200.lm import MoELM

    cfg = ModelConfig(vocab_size=1024, embed_size=256, hidden_size=256, transformer_depth=3, intermediate_size=256,
                      n_experts=9, n_shared_experts=1, n_experts_per_token=2, n_attention_heads=4,
                      n_key_value_heads=2, attention_window_pattern=(None, 40, None), max_position_embeddings=512,
                      sequence_length=512, pos_rope_dims=32, attention_sink=True, use_qk_norm=True)
    torch.manual_seed(0)
    return cfg, MoELM(cfg).cuda()


def _other_linear(m, cfg):
    new = nn.Linear(cfg.hidden_size, cfg.vocab_size, bias=False, device="cuda")
    m.output_layer = new


def _other_block(m, cfg):
    _, n = _sparse_model()
    n.layers[1].self_attn.q_proj.weight.data.mul_(-1)
    m.layers[1] = n.layers[1]


def _other_gate_bias(m, cfg):
    b = m.layers[0].mlp.gate.expert_biases
    m.layers[0].mlp.gate.expert_biases = torch.arange(b.numel(), device="cuda", dtype=b.dtype)


def _other_rotation(m, cfg):
    att = m.layers[2].self_attn
    att.pos_cos_cache, att.pos_sin_cache = att.pos_sin_cache.clone(), att.pos_cos_cache.clone()


def _sink_removed(m, cfg):
    m.layers[0].self_attn.k_sink = None


def _fewer_layers(m, cfg):
    del m.layers[2]


def _other_tokens(m, cfg, step):
    step.tokens = step.tokens + 100


def _back_at_the_old_address(m, cfg):
    w = m.output_layer.weight
    w.data = w.data * 2
    w.data = w.data * 3                                      # may lie where the first one lay


CHANGES = [_other_linear, _other_block, _other_gate_bias, _other_rotation, _sink_removed, _fewer_layers,
           _other_tokens, _back_at_the_old_address]


@pytest.mark.parametrize("change", CHANGES, ids=lambda f: f.__name__[1:])
def test_a_recorded_step_follows_its_modules_and_buffers(change):
    from zs_b200.generate import DecodeStep

    cfg, m = _sparse_model()
    c = m.new_cache(2, 64, page_size=16)
    step = DecodeStep(m, c)
    step.active.fill_(1)
    step.tokens.copy_(torch.tensor([3, 9]))
    for _ in range(3):
        step()
    recorded = step.graph
    step()
    assert step.graph is recorded
    meta, kv = c.meta.clone(), c.kv.clone()
    old = step().clone()
    c.meta.copy_(meta)
    c.kv.copy_(kv)
    with torch.no_grad():
        change(m, cfg, *([step] if change is _other_tokens else []))
    changed = False
    for k in range(3):                                       # recorded anew, then replayed
        got = step().clone()
        assert step.graph is not recorded
        c.meta.copy_(meta)
        c.kv.copy_(kv)
        c.extend(step.slots, step.active)
        want = m.forward_paged(step.tokens, c, c.block_table, c.seq_lens)
        assert torch.equal(got, want)
        changed |= not torch.equal(got, old)
        meta, kv = c.meta.clone(), c.kv.clone()
    assert changed
    c.check()


def test_a_step_is_recorded_on_a_stream_of_its_device(monkeypatch):
    """Not on the stream that torch keeps for captures, which may be another device's."""
    from zs_b200.generate import DecodeStep

    given, real = [], torch.cuda.graph

    class Graph(real):
        def __init__(self, graph, **kw):
            given.append((torch.cuda.current_device(), kw.get("stream")))
            super().__init__(graph, **kw)

    monkeypatch.setattr(torch.cuda, "graph", Graph)
    cfg, m = _model(layers=1, windows=(None,))
    step = DecodeStep(m, m.new_cache(1, 32, page_size=16))
    step.active.fill_(1)
    step(), step()
    ((device, stream),) = given
    assert stream is not None and stream.device.index == device == step.cache.kv.device.index
