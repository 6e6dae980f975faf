"""Continuing prompts with a trained MoELM from a paged key-value cache.

The reference's inference.py:25-73 runs the whole sequence again for every new
token.  Here the prompts run once, packed, and every further step runs one token
per sequence: the step's kernels are recorded into one CUDA graph and replayed,
since the launches would cost more than the work.
"""
from __future__ import annotations

import itertools
import math
import operator

import torch

from . import _lib as Z
from .dense import one_group_routing


def sharded(model):
    """Whether the model's experts are sharded over ranks."""
    from scattermoe.expert_parallel import ExpertParallelGLUMLP

    return any(isinstance(m, ExpertParallelGLUMLP) for m in model.modules())


def _refuse_sharded(model):
    if sharded(model):
        raise Z.ZsError("a decode step cannot be recorded with experts sharded over ranks (their exchange reads its "
                        "sizes on the host): call forward_paged for every step, on all ranks alike")


class DecodeStep:
    """One decode step of all slots of a cache as a CUDA graph: the slots grow by `active` (0 or 1)
    tokens, `tokens` go in, `logits` come out.  A slot that does not grow (inactive, or refused for want
    of a page or of room) keeps what it holds and may go on later; its row of the logits means nothing.

    The recorded kernels read the weights' bf16 shadows, the parameters and the buffers where they lay at the
    recording.  The package's optimizer writes those in place; after any other change (of a weight by a
    torch operation or load_state_dict; another tensor, parameter, buffer or module in the place of one;
    another `model`, `cache`, `slots`, `active` or `tokens`) the step is recorded again.  Changes that no
    tensor or module shows (a flag, a hook) need `graph = None`.  Experts sharded over ranks
    (shard_experts) are refused."""

    def __init__(self, model, cache):
        _refuse_sharded(model)
        dev = cache.kv.device
        n = cache.seq_lens.numel()
        self.model, self.cache = model, cache
        self.slots = torch.arange(n, dtype=torch.int32, device=dev)
        self.active = torch.zeros(n, dtype=torch.int32, device=dev)
        self.tokens = torch.zeros(n, dtype=torch.long, device=dev)
        self.logits = None
        self.graph = None

    def _run(self):
        c = self.cache
        before = c.seq_lens.clone()
        c.extend(self.slots, self.active)
        # a slot that did not grow has no new token: with a length of zero nothing is stored for it (its
        # last position holds a token, maybe on a page that it shares) and nothing is read
        lens = c.seq_lens * (c.seq_lens > before)
        return self.model.forward_paged(self.tokens, c, c.block_table, lens)

    @staticmethod
    def _place(t):
        """Where a kernel reads tensor t, and the change by torch that its shadow is in step with."""
        sh = getattr(t, "_zs_sh", None)
        return t.data_ptr(), None if sh is None else (sh.data_ptr(), t._version)

    def _own(self):
        c = self.cache
        return self.model, c, c.kv, c.block_table, c.seq_lens, self.slots, self.active, self.tokens

    def _remember(self):
        """What the recorded kernels depend on: this object's inputs and every module's modules, parameters and
        buffers by identity, every tensor by its place.  The tensors' memory is held, so an address stands for it."""
        self._inputs = self._own()
        dicts = [d for m in self.model.modules() for d in (m._modules, m._parameters, m._buffers)]
        values = [v for d in dicts for v in d.values()]
        tensors = [v for v in values if torch.is_tensor(v)]
        self._read = dicts, [len(d) for d in dicts], values, tensors, [self._place(t) for t in tensors]
        self._memory = [(t.detach(), getattr(t, "_zs_sh", None)) for t in tensors]

    def _current(self):
        # 0.15 ms of host time for 16 layers (357 modules), beside 2.3 ms of kernels for 64 slots
        dicts, lens, values, tensors, places = self._read
        return (all(map(operator.is_, self._own(), self._inputs)) and list(map(len, dicts)) == lens
                and all(map(operator.is_, itertools.chain.from_iterable(d.values() for d in dicts), values))
                and list(map(self._place, tensors)) == places)

    def __call__(self):
        if self.graph is not None and self._current():
            self.graph.replay()
            self.logits = self._static
            return self.logits
        _refuse_sharded(self.model)
        # a step outside the recording first (a real one): it makes or refreshes every lazily
        # made buffer, then the next ones are recorded
        self.logits = self._run()
        # tensors that other code may drop while the graph still reads them
        self._held = one_group_routing(self.tokens.numel(), self.tokens.device)
        with torch.cuda.device(self.tokens.device):
            torch.cuda.current_stream().synchronize()
            graph = torch.cuda.CUDAGraph()
            # a stream of this device: torch's own one for captures lies on the device of the process's first capture,
            # and nothing that runs on another device is recorded there
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                static = self._run()
        self._remember()
        self.graph, self._static = graph, static
        return self.logits


def sample(logits, temperature=0.0, generator=None):
    """Token ids [n]: the largest logit (the lowest id of equals), or with a temperature a draw from
    softmax(logits / temperature).  A row without a finite largest logit gets any id: torch.multinomial
    ends the process's GPU context where a probability is no number."""
    if math.isnan(temperature):
        raise Z.ZsError(f"temperature must be a number (got {temperature})")
    if temperature <= 0.0:
        return logits.argmax(-1)
    x = logits.float()
    # the quotients stay numbers at both ends of f32: of the distance to the largest logit, which is zero for
    # itself, under a small temperature; of the logits, which are finite or -inf, under a large one
    x = (x - x.amax(-1, keepdim=True)) / max(temperature, 1e-38) if temperature < 1e-3 else x / min(temperature, 1e38)
    p = torch.softmax(x, -1)
    p = p.masked_fill(p.isnan(), 1.0)
    return torch.multinomial(p, 1, generator=generator).squeeze(-1)


@torch.no_grad()
def generate(model, prompts, max_new_tokens, *, temperature=0.0, eos_token_id=None, page_size=64, generator=None):
    """Continuations (a list of lists of ids) of prompts (a list of non-empty id sequences).  Greedy
    by default; a sequence ends after eos_token_id (which is part of it) or max_new_tokens ids.  Refuses a
    model whose experts are sharded over ranks (see DecodeStep)."""
    _refuse_sharded(model)
    prompts = [torch.as_tensor(p, dtype=torch.long).reshape(-1).cpu() for p in prompts]
    if not prompts or min(p.numel() for p in prompts) < 1:
        raise Z.ZsError("generate needs prompts of at least one token")
    ids = torch.cat(prompts)
    if int(ids.min()) < 0 or int(ids.max()) >= model.embedding.weight.size(0):
        raise Z.ZsError(f"token ids must lie in [0, {model.embedding.weight.size(0)}) (got {int(ids.min())} to "
                        f"{int(ids.max())})")
    if max_new_tokens < 1:
        return [[] for _ in prompts]
    dev = model.embedding.weight.device
    lens = [p.numel() for p in prompts]
    longest = max(lens) + max_new_tokens
    if longest > model.config.max_position_embeddings:
        raise Z.ZsError(f"{longest} positions exceed the model's {model.config.max_position_embeddings}")
    cache = model.new_cache(len(prompts), longest, page_size=page_size, num_pages=len(prompts) * -(-longest // page_size))
    step = DecodeStep(model, cache)
    n_new = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.zeros(len(prompts) + 1, dtype=torch.int32, device=dev)
    cu[1:] = n_new.cumsum(0)
    cache.extend(step.slots, n_new)
    logits = model.forward_paged(ids.to(dev), cache, cache.block_table, cache.seq_lens, cu)
    out = torch.full((len(prompts), max_new_tokens), -1, dtype=torch.long, device=dev)
    step.active.fill_(1)
    for i in range(max_new_tokens):
        tok = sample(logits, temperature, generator)
        out[:, i] = torch.where(step.active.bool(), tok, -1)
        if eos_token_id is not None:
            step.active.mul_((tok != eos_token_id).int())
            # ask the device now and then only: the answer costs a wait
            if i % 16 == 15 and not bool(step.active.any()):
                break
        if i + 1 < max_new_tokens:
            step.tokens.copy_(tok)
            logits = step()
    cache.check()
    return [[t for t in row if t >= 0] for row in out.tolist()]
