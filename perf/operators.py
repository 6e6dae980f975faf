"""Cases of the paged key-value cache operators (zs_b200.paged): what each call gets, its
plain form in elementary torch operations, its 64-bit value, and the work it cannot do without.

Four operators serve a trained model from a cache of fixed-size pages:

  append   per-head q/k zero-centred RMSNorm + partial RoPE of new tokens' projections,
           k and v stored in their sequences' pages
  prompt   causal grouped-head attention of packed new tokens over the pages
  decode   the same for one new token per sequence
  fork / compact   page bookkeeping: sequences that share pages, and a pool without holes

`own` chooses between the plain form (False) and the package's calls (True).
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ----------------------------------------------------------------------------------- cases

def _lens(case):
    """(new tokens, tokens in the cache after the call) of each sequence."""
    r = random.Random(case["lens"])
    new, total = [], []
    for _ in range(case["seqs"]):
        n = 1 if case["op"] == "decode" else r.randint(case["new_lo"], case["new_hi"])
        new.append(n)
        t = r.randint(case["len_lo"], case["len_hi"])
        total.append(t if case["op"] == "decode" else max(n, t))       # a decode slot may be empty
    return new, total


def listed():
    return [
        # a single conversation that has just begun: nothing but latency
        dict(name="decode_one_short", op="decode", seqs=1, len_lo=300, len_hi=300, H=12, Hkv=4, hd=128, page=64,
             window=0, sink=True, gate=True, dtype="bf16", lens=1),
        # a batch of conversations of very different ages, the 12-head model with sink and gate
        dict(name="decode_ragged_batch", op="decode", seqs=32, len_lo=1, len_hi=4096, H=12, Hkv=4, hd=128, page=64,
             window=0, sink=True, gate=True, dtype="bf16", lens=2),
        # a sliding-window layer in half precision, heads of 64, small pages
        dict(name="decode_window_f16", op="decode", seqs=129, len_lo=100, len_hi=8191, H=16, Hkv=4, hd=64, page=16,
             window=512, sink=False, gate=True, dtype="f16", lens=3),
        # long documents at full batch, the 16-head model
        dict(name="decode_long_batch", op="decode", seqs=64, len_lo=30000, len_hi=32768, H=16, Hkv=4, hd=128, page=64,
             window=0, sink=False, gate=True, dtype="bf16", lens=4),
        # one short question
        dict(name="prompt_one_short", op="prompt", seqs=1, new_lo=37, new_hi=37, len_lo=37, len_hi=37, H=12, Hkv=4,
             hd=128, page=64, window=0, sink=True, gate=True, dtype="bf16", lens=5),
        # a packed batch of prompts of different lengths
        dict(name="prompt_packed", op="prompt", seqs=9, new_lo=5, new_hi=4096, len_lo=1, len_hi=1, H=12, Hkv=4,
             hd=128, page=64, window=0, sink=True, gate=True, dtype="bf16", lens=6),
        # the next questions of long conversations: short chunks over long prefixes, windowed, half precision
        dict(name="prompt_after_prefix", op="prompt", seqs=6, new_lo=20, new_hi=700, len_lo=9000, len_hi=16384, H=8,
             Hkv=1, hd=64, page=32, window=4096, sink=False, gate=False, dtype="f16", lens=7),
        # one long document
        dict(name="prompt_one_long", op="prompt", seqs=1, new_lo=32768, new_hi=32768, len_lo=32768, len_hi=32768,
             H=16, Hkv=4, hd=128, page=64, window=0, sink=False, gate=True, dtype="bf16", lens=8),
        # one token of each of 64 running sequences
        dict(name="append_decode_step", op="append", seqs=64, new_lo=1, new_hi=1, len_lo=1, len_hi=8192, H=12, Hkv=4,
             hd=128, page=64, rot=8, norm=True, dtype="bf16", lens=9),
        # a packed batch of prompts
        dict(name="append_prompts", op="append", seqs=11, new_lo=100, new_hi=4096, len_lo=1, len_hi=4096, H=16, Hkv=4,
             hd=128, page=64, rot=8, norm=True, dtype="bf16", lens=10),
        # beam search: the best beams of each of four questions are continued by others
        dict(name="fork_beams", op="fork", seqs=32, len_lo=500, len_hi=2000, layers=16, Hkv=4, hd=128, page=64,
             dtype="bf16", lens=11),
        # a pool with holes left by finished conversations
        dict(name="compact_pool", op="compact", seqs=48, len_lo=100, len_hi=4096, layers=8, Hkv=4, hd=128, page=64,
             dtype="bf16", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "append", "fork", "compact"])
    H, Hkv = rng.choice([(12, 4), (16, 4), (4, 4), (8, 1), (8, 8), (32, 4), (5, 1), (14, 2)])
    c = dict(op=op, Hkv=Hkv, hd=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
             dtype=rng.choice(["bf16", "bf16", "f16"]), lens=rng.randrange(1 << 30))
    if op in ("fork", "compact"):
        hi = _log(rng, 40, 3000)
        return dict(c, seqs=_log(rng, 2, 48), len_lo=rng.randint(0, hi), len_hi=hi, layers=rng.randint(1, 8),
                    Hkv=min(Hkv, 4))
    c.update(H=H)
    if op == "append":
        hi = _log(rng, 1, 3000)
        seqs = max(1, min(_log(rng, 1, 200), 30000 // hi))
        return dict(c, seqs=seqs, new_lo=rng.randint(1, hi), new_hi=hi, len_lo=1, len_hi=rng.randint(1, 8192),
                    rot=rng.choice([0, 8, c["hd"] // 2, 12]), norm=rng.random() < 0.8)
    c.update(window=rng.choice([0, 0, _log(rng, 1, 4000)]), sink=rng.random() < 0.5, gate=rng.random() < 0.7)
    if op == "decode":
        hi = _log(rng, 1, 60000)
        seqs = max(1, min(_log(rng, 1, 300), 1_000_000 // (hi * max(1, Hkv // 4))))
        return dict(c, seqs=seqs, len_lo=rng.randint(0, hi), len_hi=hi)
    hi = _log(rng, 1, 8000)
    seqs = max(1, min(_log(rng, 1, 40), 16000 // hi))
    return dict(c, seqs=seqs, new_lo=rng.randint(1, hi), new_hi=hi, len_lo=1, len_hi=_log(rng, 1, 16000))


def _visible(new, total, window):
    """Query-key pairs of one sequence."""
    if not window or window >= total:
        return sum(range(total - new + 1, total + 1))
    lo, hi = total - new + 1, total            # keys seen without the window, first and last query
    full = max(0, hi - max(lo, window) + 1)    # queries that see a whole window
    part = new - full
    return full * window + part * (lo + lo + part - 1) // 2


def work(case):
    es = 2
    if case["op"] in ("fork", "compact"):
        row = case["layers"] * 2 * case["Hkv"] * case["hd"] * es      # one token's keys and values
        t = _tables(case)
        rows = sum(n for _, _, n in t["moves"])
        return {"bytes": 2 * rows * row + 8 * len(t["moves"]) + 4 * len(t["meta"]), "flops": 0}
    new, total = _lens(case)
    T = sum(new)
    if case["op"] == "append":
        heads = case["H"] + 2 * case["Hkv"]
        return {"bytes": 2 * T * heads * case["hd"] * es + T * 2 * case["rot"] * 4,
                "flops": T * (case["H"] + case["Hkv"]) * case["hd"] * 8}
    win = case["window"]
    keys = sum(t if not win else min(t, win + n - 1) for n, t in zip(new, total))
    pairs = sum(_visible(n, t, win) for n, t in zip(new, total) if t)
    b = 2 * keys * case["Hkv"] * case["hd"] * es + 2 * T * case["H"] * case["hd"] * es
    b += T * case["H"] * es * bool(case["gate"]) + 4 * sum(-(-t // case["page"]) for t in total)
    return {"bytes": b, "flops": 4 * case["H"] * case["hd"] * pairs}


# ------------------------------------------------------------------------------- page tables

def _tables(case):
    """The cache's tables before a fork or a compaction, and the page rows that it has to move.

    meta is the int32 concatenation of the block table [slots, pages a slot may hold], the
    lengths [slots] and the reference counts [pages]."""
    r = random.Random(case["lens"])
    ps, n = case["page"], case["seqs"]
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(n)]
    need = [-(-t // ps) for t in lens]
    M = max(1, -(-case["len_hi"] // ps))
    slots = n + 3 if case["op"] == "fork" else n
    P = sum(need) + 2 * slots + 5 if case["op"] == "fork" else sum(need) + 5
    order = list(range(P))
    r.shuffle(order)                           # pages as they lie after many sequences came and went
    table, ref, at = [[-1] * M for _ in range(slots)], [0] * P, 0
    for s in range(n):
        for j in range(need[s]):
            table[s][j] = order[at]
            ref[order[at]] += 1
            at += 1
    lens += [0] * (slots - n)
    out = {"ps": ps, "M": M, "P": P, "slots": slots}
    if case["op"] == "fork":
        # groups of up to 8 beams: each slot is continued from a slot of its group
        src = [min(n - 1, (s // 8) * 8 + r.randrange(min(8, n - (s // 8) * 8))) for s in range(n)]
        out.update(src=src, dst=list(range(n)))
        moves, free = [], [p for p in range(P) if ref[p] == 0]
        for s, d in zip(out["src"], out["dst"]):
            if s != d and lens[s] % ps:
                moves.append((table[s][lens[s] // ps], free.pop(0), lens[s] % ps))
        out["moves"] = moves
    else:
        # every third sequence has ended
        for s in range(0, n, 3):
            for j in range(need[s]):
                ref[table[s][j]] -= 1
            table[s], lens[s] = [-1] * M, 0
        used = [p for p in range(P) if ref[p]]
        holes = [p for p in range(len(used)) if not ref[p]]
        out["moves"] = [(a, b, ps) for a, b in zip([p for p in used if p >= len(used)], holes)]
    out["meta"] = [x for row in table for x in row] + lens + ref
    return out


# ------------------------------------------------------------------------------------ inputs

def _package():
    p = str(ROOT / "architecture-zarelga-superposition_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    from zs_b200 import paged

    return paged


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(dtype)

    ps, Hkv, hd = case["page"], case["Hkv"], case["hd"]
    st = {"case": case}
    if case["op"] in ("fork", "compact"):
        t = _tables(case)
        st.update(t=t, meta0=torch.tensor(t["meta"], dtype=torch.int32, device="cuda"))
        shape = (case["layers"], 2, t["P"], Hkv, ps, hd)
        if own:
            cache = _package().PagedKVCache(case["layers"], Hkv, hd, num_pages=t["P"], page_size=ps,
                                            max_seqs=t["slots"], max_pages_per_seq=t["M"], dtype=dt, device="cuda")
            st.update(cache=cache, kv=cache.kv, meta=cache.meta)
        else:
            st.update(kv=torch.empty(shape, dtype=dt, device="cuda"), meta=torch.empty_like(st["meta0"]))
        for layer in range(shape[0]):
            st["kv"][layer].copy_(randn(*shape[1:]))
        st["meta"].copy_(st["meta0"])
        if case["op"] == "fork":
            st["src"] = torch.tensor(t["src"], dtype=torch.int32, device="cuda")
            st["dst"] = torch.tensor(t["dst"], dtype=torch.int32, device="cuda")
        return st

    new, total = _lens(case)
    B, T, H = case["seqs"], sum(new), case["H"]
    need = [-(-n // ps) for n in total]
    M, P = max(1, max(need)), sum(need) + 7
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed))
    table = torch.full((B, M), -1, dtype=torch.int32)
    at = 0
    for s in range(B):
        table[s, :need[s]] = order[at:at + need[s]].to(torch.int32)
        at += need[s]
    cu = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32)
    st.update(new=new, total=total, table=table.cuda(), lens=torch.tensor(total, dtype=torch.int32, device="cuda"),
              cu=cu.cuda(), scale=1.0 / math.sqrt(hd))
    # the projections' rows: q heads, k heads, v heads, gate logits, zero padding to a multiple of 16
    W = (H + 2 * Hkv) * hd + H
    W += -W % 16
    if case["op"] == "append":
        st["qkvg"] = randn(T, W)
        st["wq"], st["wk"] = (randn(hd, dtype=torch.float32, scale=0.1) for _ in range(2))
        if not case["norm"]:
            st["wq"] = st["wk"] = None
        st["k"], st["v"] = (torch.zeros(P, Hkv, ps, hd, dtype=dt, device="cuda") for _ in range(2))
        st["cos"] = st["sin"] = None
        if case["rot"]:
            inv = 10000.0 ** (-torch.arange(case["rot"], dtype=torch.float64, device="cuda") / case["rot"])
            ang = torch.outer(torch.arange(max(total), dtype=torch.float64, device="cuda"), inv)
            st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        return st
    st["k"], st["v"] = randn(P, Hkv, ps, hd), randn(P, Hkv, ps, hd)
    st["q"] = randn(T, H, hd)
    st["sink"] = randn(H, hd, dtype=torch.float32, scale=0.3) if case["sink"] else None
    st["gate"] = randn(T, W)[:, (H + 2 * Hkv) * hd:][:, :H] if case["gate"] else None
    return st


# ------------------------------------------------------------------------------------- calls

def run(st):
    op = st["case"]["op"]
    if op in ("fork", "compact"):
        st["meta"].copy_(st["meta0"])          # a pass starts from the tables as they were
        return (_run_own_pages if own else {"fork": _plain_fork, "compact": _plain_compact}[op])(st)
    if own:
        return _run_own(st)
    return _plain_append(st) if op == "append" else _plain_attention(st)


def _run_own(st):
    paged, c = _package(), st["case"]
    if c["op"] == "append":
        q = paged.paged_append(st["qkvg"], st["k"], st["v"], st["table"], st["lens"], n_heads=c["H"],
                               cu_seqlens=st["cu"], q_weight=st["wq"], k_weight=st["wk"], eps=1e-6, cos=st["cos"],
                               sin=st["sin"])
        return {"q": q, "k": st["k"], "v": st["v"]}
    kw = dict(window=c["window"] or None, k_sink=st["sink"], gate=st["gate"])
    if c["op"] == "decode":
        return paged.paged_decode_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], **kw)
    return paged.paged_prompt_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["cu"], **kw)


def _run_own_pages(st):
    cache = st["cache"]
    if st["case"]["op"] == "fork":
        cache.fork(st["src"], st["dst"])
    else:
        cache.compact()
    return {"kv": st["kv"], "meta": st["meta"]}


# -------------------------------------------------------------------------------- plain forms

def _plain_append(st):
    c = st["case"]
    H, Hkv, hd, ps, rot = c["H"], c["Hkv"], c["hd"], c["page"], c["rot"]
    T = st["qkvg"].size(0)
    x = st["qkvg"].float()
    q = x[:, :H * hd].view(T, H, hd)
    k = x[:, H * hd:(H + Hkv) * hd].view(T, Hkv, hd)
    v = x[:, (H + Hkv) * hd:(H + 2 * Hkv) * hd].view(T, Hkv, hd)
    tok = torch.arange(T, device="cuda")
    seq = torch.searchsorted(st["cu"][1:].long(), tok, right=True)
    pos = tok - st["cu"].long()[seq + 1] + st["lens"].long()[seq]

    def norm_rope(t, w):
        if w is not None:
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + w)
        if rot:
            cos, sin = st["cos"][pos].unsqueeze(1), st["sin"][pos].unsqueeze(1)
            half = hd // 2
            a, b = t[..., :rot], t[..., half:half + rot]
            t = torch.cat([a * cos - b * sin, t[..., rot:half], b * cos + a * sin, t[..., half + rot:]], -1)
        return t

    q, k = norm_rope(q, st["wq"]), norm_rope(k, st["wk"])
    dt = st["k"].dtype
    page, off = st["table"][seq, pos // ps].long(), pos % ps
    st["k"][page, :, off] = k.to(dt)
    st["v"][page, :, off] = v.to(dt)
    return {"q": q.to(dt), "k": st["k"], "v": st["v"]}


def _plain_attention(st):
    c = st["case"]
    H, Hkv, hd, ps, win = c["H"], c["Hkv"], c["hd"], c["page"], c["window"]
    G = H // Hkv
    out = torch.empty_like(st["q"])
    at = 0
    for s, (n, total) in enumerate(zip(st["new"], st["total"])):
        rows = slice(at, at + n)
        at += n
        first = max(0, total - n - win + 1) // ps if win else 0        # the first page that any query sees
        pages = st["table"][s, first:-(-total // ps)].long()
        m = pages.numel() * ps
        K = st["k"][pages].transpose(0, 1).reshape(Hkv, m, hd)[:, :total - first * ps].float()
        V = st["v"][pages].transpose(0, 1).reshape(Hkv, m, hd)[:, :total - first * ps].float()
        kpos = torch.arange(first * ps, first * ps + K.size(1), device="cuda")
        step = max(1, min(n, (1 << 28) // max(1, H * K.size(1))))
        for i in range(0, n, step):
            q = st["q"][rows][i:i + step].float()                       # [t, H, hd]
            t = q.size(0)
            qpos = torch.arange(total - n + i, total - n + i + t, device="cuda")
            keys = max(0, min(K.size(1), total - n + i + t - first * ps))   # none after the last query's own
            qg = q.view(t, Hkv, G, hd).permute(1, 2, 0, 3).reshape(Hkv, G * t, hd)
            S = (qg @ K[:, :keys].transpose(1, 2)).view(Hkv, G, t, keys) * st["scale"]
            dead = kpos[:keys] > qpos[:, None]
            if win:
                dead |= qpos[:, None] - kpos[:keys] >= win
            S = S.masked_fill_(dead, float("-inf"))
            if st["sink"] is not None:
                z = (q * st["sink"].float()).sum(-1).view(t, Hkv, G).permute(1, 2, 0).unsqueeze(-1) * st["scale"]
            else:
                z = torch.full((Hkv, G, t, 1), float("-inf"), device="cuda")
            top = torch.maximum(S.amax(-1, keepdim=True), z) if keys else z
            top = torch.where(top == float("-inf"), torch.zeros_like(top), top)     # a row that sees nothing
            S = S.sub_(top).exp_()
            den = S.sum(-1, keepdim=True) + (z - top).exp()
            o = (S.view(Hkv, G * t, keys) @ V[:, :keys]).view(Hkv, G, t, hd)
            o = o / torch.where(den > 0, den, torch.ones_like(den))
            o = o.permute(2, 0, 1, 3).reshape(t, H, hd)
            if st["gate"] is not None:
                o = o * torch.sigmoid(st["gate"][rows][i:i + step].float()).unsqueeze(-1)
            out[rows][i:i + step] = o.to(out.dtype)
    return out


def _split(st):
    t = st["t"]
    a, b = t["slots"] * t["M"], t["slots"] * t["M"] + t["slots"]
    m = st["meta"]
    return m[:a].view(t["slots"], t["M"]), m[a:b], m[b:]


def _plain_fork(st):
    """dst[i] becomes a copy of src[i]: whole pages shared, the last partial page copied into the
    lowest free page, in the order of i; all sources as they were before the call."""
    table, lens, ref = _split(st)
    ps = st["t"]["ps"]
    src, dst = st["src"].long(), st["dst"].long()
    M, P = table.size(1), ref.numel()
    changed = src != dst
    L = lens[src].long()
    full, tail = L // ps, L % ps
    rows = table[src].clone()
    col = torch.arange(M, device="cuda")
    fresh = changed & (tail > 0)
    free_rank = torch.cumsum((ref == 0).int(), 0) - 1
    by_rank = torch.full((P + 1,), P, dtype=torch.long, device="cuda")
    by_rank.scatter_(0, torch.where(ref == 0, free_rank.long(), P), torch.arange(P, device="cuda"))
    got = by_rank[(torch.cumsum(fresh.int(), 0) - 1).clamp_min(0).long()].int()
    old_tail = rows.gather(1, full.clamp_max(M - 1)[:, None]).squeeze(1).long()
    is_tail = fresh[:, None] & (col == full[:, None])
    rows = torch.where(is_tail, got[:, None], rows)
    # the partial pages' filled rows, every layer's keys and values: the other copies write a
    # page's own rows over it
    to = torch.where(fresh, got.long(), 0)
    frm = torch.where(fresh, old_tail, 0)
    keep = (torch.arange(ps, device="cuda") < tail[:, None]) & fresh[:, None]
    kv = st["kv"]
    sel = keep.nonzero()
    i, r = sel[:, 0], sel[:, 1]
    kv[:, :, to[i], :, r] = kv[:, :, frm[i], :, r]
    # counts: the old rows let go, the new rows held
    one = torch.ones((), dtype=torch.int32, device="cuda")
    old = table[dst]
    hit = torch.zeros(P + 1, dtype=torch.int32, device="cuda")
    hit.index_put_((torch.where((old >= 0) & changed[:, None], old, P).long().flatten(),), -one, accumulate=True)
    hit.index_put_((torch.where((rows >= 0) & changed[:, None], rows, P).long().flatten(),), one, accumulate=True)
    ref += hit[:P]
    table[dst] = rows
    lens[dst] = L.int()
    return {"kv": kv, "meta": st["meta"]}


def _plain_compact(st):
    """The pages in use become pages 0 .. U-1: the k-th hole below U takes the k-th used page from U on."""
    table, _, ref = _split(st)
    P = ref.numel()
    ids = torch.arange(P, device="cuda")
    used = ref > 0
    U = used.sum()
    frm = (used & (ids >= U)).nonzero().squeeze(1)
    to = (~used & (ids < U)).nonzero().squeeze(1)
    kv = st["kv"]
    kv[:, :, to] = kv[:, :, frm]
    name = ids.int()
    name[frm] = to.int()
    ref[to] = ref[frm]
    ref[frm] = 0
    table.copy_(torch.where(table >= 0, name[table.clamp_min(0).long()], table))
    return {"kv": kv, "meta": st["meta"]}


# -------------------------------------------------------------------------- values in 64 bits

def exact(case, seed):
    global own
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    if case["op"] in ("fork", "compact"):
        kv = st["kv"].double()
        for a, b, rows in st["t"]["moves"]:
            kv[:, :, b, :, :rows] = kv[:, :, a, :, :rows]
        return {"kv": kv, "meta": None}
    if case["op"] == "append":
        return _exact_append(st)
    return _exact_attention(st)


def _exact_append(st):
    c = st["case"]
    H, Hkv, hd, ps, rot = c["H"], c["Hkv"], c["hd"], c["page"], c["rot"]
    x = st["qkvg"].double()
    k, v = st["k"].double(), st["v"].double()
    table = st["table"].tolist()
    out_q, at = [], 0
    for s, (n, total) in enumerate(zip(st["new"], st["total"])):
        xs = x[at:at + n].clone()
        at += n
        heads = xs[:, :(H + 2 * Hkv) * hd].reshape(n, H + 2 * Hkv, hd)
        if st["wq"] is not None:
            for lo, hi, w in ((0, H, st["wq"]), (H, H + Hkv, st["wk"])):
                part = heads[:, lo:hi]
                rms = ((part * part).sum(-1, keepdim=True) / hd + 1e-6).sqrt()
                heads[:, lo:hi] = part / rms * (w.double() + 1.0)
        if rot:
            z = torch.complex(heads[:, :H + Hkv, :rot].contiguous(),
                              heads[:, :H + Hkv, hd // 2:hd // 2 + rot].contiguous())
            turn = torch.complex(st["cos"][total - n:total].double(), st["sin"][total - n:total].double())
            z = z * turn[:, None]
            heads[:, :H + Hkv, :rot] = z.real
            heads[:, :H + Hkv, hd // 2:hd // 2 + rot] = z.imag
        out_q.append(heads[:, :H])
        pos = total - n
        while pos < total:                     # page by page
            end = min(total, (pos // ps + 1) * ps)
            p, i = table[s][pos // ps], pos - (total - n)
            rows = slice(pos % ps, pos % ps + end - pos)
            k[p, :, rows] = heads[i:i + end - pos, H:H + Hkv].transpose(0, 1)
            v[p, :, rows] = heads[i:i + end - pos, H + Hkv:].transpose(0, 1)
            pos = end
    return {"q": torch.cat(out_q), "k": k, "v": v}


def _exact_attention(st):
    c = st["case"]
    H, Hkv, hd, ps, win = c["H"], c["Hkv"], c["hd"], c["page"], c["window"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    table, at = st["table"].tolist(), 0
    for s, (n, total) in enumerate(zip(st["new"], st["total"])):
        if total == 0:
            at += n
            continue
        pages = torch.tensor(table[s][:-(-total // ps)], device="cuda")
        for h in range(H):
            K = st["k"][pages, h // (H // Hkv)].reshape(-1, hd)[:total].double()
            V = st["v"][pages, h // (H // Hkv)].reshape(-1, hd)[:total].double()
            for i in range(0, n, 4096):
                t = min(4096, n - i)
                q = st["q"][at + i:at + i + t, h].double()
                end = total - n + i + t
                logit = q @ K[:end].T * st["scale"]
                ahead = torch.arange(end, device="cuda") - torch.arange(end - t, end, device="cuda")[:, None]
                ok = ahead <= 0
                if win:
                    ok &= ahead > -win
                logit = torch.where(ok, logit, float("-inf"))
                lse = torch.logsumexp(logit, 1)
                if st["sink"] is not None:
                    lse = torch.logaddexp(lse, q @ st["sink"][h].double() * st["scale"])
                o = torch.exp(logit - lse[:, None]) @ V[:end]
                if st["gate"] is not None:
                    o = o / (1.0 + torch.exp(-st["gate"][at + i:at + i + t, h].double()))[:, None]
                out[at + i:at + i + t, h] = o
        at += n
    return out
