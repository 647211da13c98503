"""Performance cases of the decoding operators: attention through a sliding window with sinks (over plain rows and over
a paged cache), the pages of that cache, and beam search's selection with the reordering of states.

A case is a dict of plain values.  ``prepare`` makes its inputs from a seed, ``run`` makes one pass: with ``own`` false
in elementary torch operations, with ``own`` true through this package.  ``exact`` computes the same in 64 bits, one
sequence at a time, and ``work`` says what a pass cannot do without.
"""
import math
import random

import torch

own = False


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # Moonshine's encoder on one 10 s utterance: a narrow window with a little look-ahead, fused q|k|v rows.
        dict(name="window_utterance", op="window", dtype="bf16", seqs=1, tokens=501, past=0, q_heads=10, kv_heads=10, dim=64,
             left=16, right=4, sinks=0, fused=True),
        # The same encoder on a bucket of segments of unlike lengths, activations in 32 bits.
        dict(name="window_segments_f32", op="window", dtype="f32", seqs=32, tokens=1501, past=0, q_heads=10, kv_heads=10, dim=64,
             left=64, right=16, sinks=4, fused=False),
        # A long causal prompt whose window covers a quarter of it; shared key heads.
        dict(name="window_long", op="window", dtype="bf16", seqs=1, tokens=16384, past=0, q_heads=16, kv_heads=4, dim=128,
             left=4095, right=0, sinks=4, fused=False),
        # One decoder token of Moonshine, one utterance: latency.
        dict(name="cache_token", op="cache", dtype="bf16", seqs=1, tokens=1, context=201, q_heads=10, kv_heads=10, dim=64,
             page=16, left=-1, right=0, sinks=0),
        # A serving batch of single tokens over long contexts with shared key heads.
        dict(name="cache_batch", op="cache", dtype="bf16", seqs=64, tokens=1, context=8192, q_heads=32, kv_heads=8, dim=128,
             page=16, left=-1, right=0, sinks=0),
        # Prompts processed in chunks over what the cache holds already, through a window.
        dict(name="cache_chunk", op="cache", dtype="bf16", seqs=4, tokens=515, context=16000, q_heads=16, kv_heads=4, dim=128,
             page=32, left=2047, right=0, sinks=4),
        # Streaming decoders in 32 bits: each sees its last 1024 tokens and the first four.
        dict(name="cache_window_f32", op="cache", dtype="f32", seqs=16, tokens=1, context=5000, q_heads=10, kv_heads=10, dim=64,
             page=16, left=1023, right=0, sinks=4),
        # One step of a beam search over eight utterances: the beams take their parents' pages and append a token.
        dict(name="pages_beam_step", op="step", dtype="bf16", items=8, beams=8, context=200, tokens=1, layers=14, kv_heads=10,
             dim=64, page=16),
        # Prompts of a batch enter the cache.
        dict(name="pages_prompts", op="append", dtype="bf16", seqs=32, tokens=1001, layers=14, kv_heads=10, dim=64, page=16),
        # A pool whose sequences ended at random is put together again.
        dict(name="pages_compact", op="compact", dtype="bf16", pages=3001, live=0.5, slots=64, layers=14, kv_heads=10, dim=64,
             page=16),
        # One utterance's beams over Moonshine's vocabulary: latency.
        dict(name="beam_utterance", op="beam", dtype="bf16", items=1, beams=4, vocab=32768, states=2, width=640),
        # A batch of beams, with the recurrent states of the beams that survive.
        dict(name="beam_batch", op="beam", dtype="f32", items=64, beams=8, vocab=32768, states=4, width=640),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["window", "window", "cache", "cache", "step", "append", "compact", "beam", "beam"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 10])
    group = rng.choice([1, 1, 2, 4, 8])
    if op == "window":
        seqs = _log(rng, 1, 48)
        tokens = _log(rng, 3, max(4, min(12000, 30000 // seqs)))
        if kv * group > 16:
            group = 1
        if dtype == "f32":  # no more than the largest listed case costs
            tokens = min(tokens, 4001)
        right = rng.choice([0, 0, 3, 16, -1]) if tokens < 3000 else 0
        left = rng.choice([_log(rng, 4, 4096), _log(rng, 4, 300), -1 if tokens < 5000 else 2000])
        return dict(op=op, dtype=dtype, seqs=seqs, tokens=tokens, past=rng.choice([0, 0, _log(rng, 1, 500)]), q_heads=kv * group,
                    kv_heads=kv, dim=dim, left=left, right=right, sinks=rng.choice([0, 1, 4, 17]), fused=rng.random() < 0.5)
    if op == "cache":
        seqs = _log(rng, 1, 64)
        tokens = rng.choice([1, 1, 1, 2, 5, _log(rng, 8, 400)])
        context = tokens + _log(rng, 1, max(2, min(40000, 400000 // (seqs * kv))))
        return dict(op=op, dtype=dtype, seqs=seqs, tokens=tokens, context=context, q_heads=kv * group, kv_heads=kv, dim=dim,
                    page=rng.choice([8, 16, 32, 64, 128]), left=rng.choice([-1, _log(rng, 8, 4096)]), right=0,
                    sinks=rng.choice([0, 1, 4, 20]))
    layers, page = _log(rng, 1, 16), rng.choice([8, 16, 32, 64])
    if op == "step":
        return dict(op=op, dtype=dtype, items=_log(rng, 1, 24), beams=rng.choice([1, 2, 4, 5, 8]), context=_log(rng, 2, 700),
                    tokens=rng.choice([1, 1, 2, 19]), layers=layers, kv_heads=kv, dim=dim, page=page)
    if op == "append":
        seqs = _log(rng, 1, 32)
        return dict(op=op, dtype=dtype, seqs=seqs, tokens=_log(rng, 1, 500), layers=layers, kv_heads=kv, dim=dim, page=page)
    if op == "compact":
        each = layers * 2 * kv * page * dim * (2 if dtype == "bf16" else 4)
        return dict(op=op, dtype=dtype, pages=_log(rng, 5, max(6, min(9000, int(1.5e9) // each))), live=rng.choice([0.1, 0.5, 0.9]),
                    slots=_log(rng, 1, 100), layers=layers, kv_heads=kv, dim=dim, page=page)
    beams = rng.choice([1, 2, 4, 5, 8, 16, 32])
    items = _log(rng, 1, 64)
    vocab = max(beams + 1, min(_log(rng, 40, 200000), 16000000 // (items * beams)))
    return dict(op="beam", dtype=dtype, items=items, beams=beams, vocab=vocab, states=rng.choice([1, 2, 4]),
                width=rng.choice([7, 320, 640, 1024]))


# ----------------------------------------------------------------------------------------------------------- lengths
def _key(case):
    return ",".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name")


def _lengths(case, count, most, least=1):
    """Ragged lengths: the first is the longest, the others between a quarter of it and it.  They go by the case alone."""
    rng = random.Random(_key(case))
    return [most] + [rng.randint(max(least, most // 4), most) for _ in range(count - 1)]


def _offsets(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


def _visible(n_q, n_k, left, right, sinks):
    """Pairs of a query and a key that it sees; query i stands at position n_k - n_q + i."""
    p = torch.arange(n_k - n_q, n_k, dtype=torch.int64)
    hi = p.clamp(max=n_k - 1) if right < 0 else (p + right).clamp(max=n_k - 1)
    hi = torch.full_like(p, n_k - 1) if right < 0 else hi
    lo = torch.zeros_like(p) if left < 0 else (p - left).clamp(min=0)
    inside = (hi - lo + 1).clamp(min=0)
    first = torch.minimum(lo, hi + 1).clamp(min=0, max=sinks)
    return int((inside + first).sum())


def _touched(n_q, n_k, left, right, sinks):
    """Keys that any query of the sequence sees."""
    if left < 0:
        return n_k
    lo = max(0, n_k - n_q - left)
    return n_k - lo + min(lo, sinks)


# ------------------------------------------------------------------------------------------------------------- inputs
def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _normal(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, device="cuda", dtype=dtype)
    return x.normal_(0.0, scale, generator=g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(case, g, pages):
    shape = (case["layers"] if "layers" in case else 1, pages, case["kv_heads"], case["page"], case["dim"])
    return _normal(g, shape, _type(case)), _normal(g, shape, _type(case))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"window": _prepare_window, "cache": _prepare_cache, "step": _prepare_step, "append": _prepare_append,
            "compact": _prepare_compact, "beam": _prepare_beam}[case["op"]](case, g)


def _prepare_window(c, g):
    lens = _lengths(c, c["seqs"], c["tokens"])
    n_q, n_k = sum(lens), sum(lens) + c["past"] * len(lens)
    hq, hk, d, dt = c["q_heads"], c["kv_heads"], c["dim"], _type(c)
    if c["fused"] and not c["past"]:
        rows = _normal(g, (n_q, (hq + 2 * hk) * d), dt)
        q, k, v = (t.unflatten(1, (-1, d)) for t in rows.split([hq * d, hk * d, hk * d], 1))
    else:
        q, k, v = _normal(g, (n_q, hq, d), dt), _normal(g, (n_k, hk, d), dt), _normal(g, (n_k, hk, d), dt)
    return dict(case=c, q=q, k=k, v=v, q_offsets=_ints(_offsets(lens)), k_offsets=_ints(_offsets([n + c["past"] for n in lens])))


def _paged(c, g, lens, extra):
    """Sequences of `lens` tokens on pages in random order; `extra` free pages."""
    P = c["page"]
    need = [-(-n // P) for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need) + 2), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(table.shape[1], device="cuda")
    n = torch.tensor(need, device="cuda")
    at = n.cumsum(0) - n
    mine = col < n[:, None]
    table = torch.where(mine, order[(at[:, None] + col).clamp(max=total - 1)], table)
    refs = torch.zeros(total, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table.clamp(min=0).flatten(), mine.flatten().to(torch.int32))
    return total, table.contiguous(), _ints(lens), refs


def _prepare_cache(c, g):
    ctx = _lengths(c, c["seqs"], c["context"], c["tokens"])
    news = [min(n, x) for n, x in zip(_lengths(dict(c, of="q"), c["seqs"], c["tokens"]), ctx)]
    pages, table, lens, refs = _paged(c, g, ctx, 3)
    k, v = _pool(c, g, pages)
    q = _normal(g, (sum(news), c["q_heads"], c["dim"]), _type(c))
    return dict(case=c, k=k, v=v, table=table, lens=lens, refs=refs, q=q, offsets=_ints(_offsets(news)))


def _prepare_step(c, g):
    """Slots [0, n) hold the beams' parents, slots [n, 2 n) take the beams."""
    n, P, m = c["items"] * c["beams"], c["page"], c["context"]
    width = -(-(m + c["tokens"]) // P) + 1
    prompt = (m // 2) // P  # the beams of an utterance share the pages of its first half
    own_pages = -(-m // P) - prompt
    pages = c["items"] * prompt + n * own_pages + n * (width - prompt) + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((2 * n, width), -1, dtype=torch.int32, device="cuda")
    shared = order[:c["items"] * prompt].view(c["items"], 1, prompt).expand(-1, c["beams"], -1).reshape(n, prompt)
    table[:n, :prompt] = shared
    table[:n, prompt:prompt + own_pages] = order[c["items"] * prompt:][:n * own_pages].view(n, own_pages)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table.clamp(min=0).flatten(), (table >= 0).flatten().to(torch.int32))
    lens = torch.cat([torch.full((n,), m, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)]).cuda()
    k, v = _pool(c, g, pages)
    new = (c["layers"], n * c["tokens"], c["kv_heads"], c["dim"])
    parent = torch.randint(0, c["beams"], (c["items"], c["beams"]), generator=g, device="cuda")
    parent = (parent + torch.arange(c["items"], device="cuda")[:, None] * c["beams"]).flatten().to(torch.int32)
    return dict(case=c, k=k, v=v, table=table, lens=lens, refs=refs, parent=parent, first=n, n=n,
                offsets=_ints([c["tokens"] * i for i in range(n + 1)]), k_new=_normal(g, new, _type(c)), v_new=_normal(g, new, _type(c)))


def _prepare_append(c, g):
    counts = _lengths(c, c["seqs"], c["tokens"])
    P = c["page"]
    pages = sum(-(-n // P) for n in counts) + 7
    table = torch.full((c["seqs"], -(-c["tokens"] // P) + 1), -1, dtype=torch.int32, device="cuda")
    k, v = _pool(c, g, pages)
    new = (c["layers"], sum(counts), c["kv_heads"], c["dim"])
    return dict(case=c, k=k, v=v, table=table, lens=torch.zeros(c["seqs"], dtype=torch.int32, device="cuda"),
                refs=torch.zeros(pages, dtype=torch.int32, device="cuda"), parent=torch.full((c["seqs"],), -1, dtype=torch.int32, device="cuda"),
                first=0, n=c["seqs"], offsets=_ints(_offsets(counts)), k_new=_normal(g, new, _type(c)), v_new=_normal(g, new, _type(c)))


def _prepare_compact(c, g):
    pages, slots = c["pages"], c["slots"]
    live = max(1, int(pages * c["live"]))
    width = -(-live // slots) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(slots * width, device="cuda").view(slots, width)
    share = -(-live // slots)
    at = at // width * share + at % width
    mine = (torch.arange(width, device="cuda") < share) & (at < live)
    table = torch.where(mine, order[at.clamp(max=live - 1)], -1).to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table.clamp(min=0).flatten(), mine.flatten().to(torch.int32))
    lens = (mine.sum(1) * c["page"]).to(torch.int32)
    k, v = _pool(c, g, pages)
    return dict(case=c, k=k, v=v, table=table.contiguous(), lens=lens, refs=refs, table0=table.clone(), refs0=refs.clone())


def _prepare_beam(c, g):
    b, w, n = c["items"], c["beams"], c["vocab"]
    logits = _normal(g, (b, w, n), _type(c), 2.5)
    banned = torch.randint(0, n, (max(1, n // 100),), generator=g, device="cuda")
    logits[:, :, banned] = -math.inf  # tokens that the decoder never writes
    logits[:, :, 0].clamp_(min=0.0)
    scores = torch.empty((b, w), device="cuda").uniform_(-30.0, -0.1, generator=g).sort(1, descending=True).values
    finished = torch.rand((b, w), generator=g, device="cuda") < 0.1
    states = [_normal(g, (b * w, c["width"]), torch.float32) for _ in range(c["states"])]
    return dict(case=c, logits=logits, scores=scores, finished=finished, eos=2, states=states)


# ----------------------------------------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    if c["op"] == "window":
        return _plain_window(state, c)
    if c["op"] == "cache":
        return _plain_cache(state, c)
    if c["op"] == "beam":
        return _plain_beam(state)
    if c["op"] == "compact":
        state["table"].copy_(state["table0"])
        state["refs"].copy_(state["refs0"])
        _plain_compact(state)
    else:
        _plain_fork(state)
        _plain_reserve(state, c)
        _plain_write(state, c)
    return {n: state[n] for n in ("k", "v", "table", "lens", "refs")}


def _own(s, c):
    if c["op"] == "window":
        from nspeech_b200.attention import window_attention
        return window_attention(s["q"], s["k"], s["v"], left=c["left"], right=c["right"], sinks=c["sinks"],
                                q_offsets=s["q_offsets"], k_offsets=s["k_offsets"])
    if c["op"] == "beam":
        from nspeech_b200.beam import beam_reorder, beam_select
        scores, parents, tokens, finished = beam_select(s["logits"], s["scores"], s["finished"], eos=s["eos"])
        states = beam_reorder(s["states"], parents)
        return dict(scores=scores, parents=parents, tokens=tokens, finished=finished, states=states)
    if "cache" not in s:
        from nspeech_b200.cache import PagedCache
        s["cache"] = PagedCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    cache = s["cache"]
    if c["op"] == "cache":
        return cache.attention(s["q"], layer=0, offsets=s["offsets"], left=c["left"], right=c["right"], sinks=c["sinks"])
    if c["op"] == "compact":
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
        cache.compact()
    else:
        cache.fork(s["parent"], first=s["first"])
        cache.reserve(s["offsets"], first=s["first"])
        cache.write(s["k_new"], s["v_new"], s["offsets"], first=s["first"])
    return {n: s[n] for n in ("k", "v", "table", "lens", "refs")}


# -------------------------------------------------------------------------------------------------------- plain forms
def _spread(offsets, most):
    """Rows of each sequence, padded to `most`: their indexes, and which are there."""
    off = offsets.long()
    at = off[:-1, None] + torch.arange(most, device=off.device)
    there = at < off[1:, None]
    return torch.where(there, at, 0), there


def _plain_attention(q, k, v, n_q, n_k, left, right, sinks, there=None):
    """q [b, i, h, d], k and v [b, j, kv, d], all padded; n_q and n_k [b].  Masked softmax in 32 bits."""
    b, i, h, d = q.shape
    j, kv = k.shape[1], k.shape[2]
    q = q.float().view(b, i, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    q = (q * (d ** -0.5)).reshape(b, kv, h // kv * i, d)
    s = torch.matmul(q, k.float().permute(0, 2, 3, 1)).view(b, kv, h // kv, i, j)
    p = (n_k - n_q)[:, None, None] + torch.arange(i, device=q.device)[:, None]
    key = torch.arange(j, device=q.device)
    seen = (key < n_k[:, None, None]) & (p < n_k[:, None, None])
    if there is not None:
        seen = seen & there[:, None, :]
    if right >= 0:
        seen = seen & (key <= p + right)
    if left >= 0:
        seen = seen & ((key >= p - left) | (key < sinks))
    seen = seen[:, None, None]
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, kv, h // kv * i, j), v.float().permute(0, 2, 1, 3)).view(b, kv, h // kv, i, d)
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, i, h, d)


def _packed(o, offsets, rows):
    off = offsets.long()
    r = torch.arange(rows, device=o.device)
    b = torch.searchsorted(off, r, right=True) - 1
    return o[b, r - off[b]]


def _plain_window(s, c):
    qi, _ = _spread(s["q_offsets"], c["tokens"])
    ki, _ = _spread(s["k_offsets"], c["tokens"] + c["past"])
    n_q, n_k = s["q_offsets"].diff().long(), s["k_offsets"].diff().long()
    o = _plain_attention(s["q"][qi], s["k"][ki], s["v"][ki], n_q, n_k, c["left"], c["right"], c["sinks"])
    return _packed(o, s["q_offsets"], s["q"].shape[0]).to(s["q"].dtype)


def _plain_cache(s, c):
    qi, _ = _spread(s["offsets"], c["tokens"])
    page = s["table"].clamp(min=0).long()
    k = s["k"][0][page].permute(0, 1, 3, 2, 4).flatten(1, 2)
    v = s["v"][0][page].permute(0, 1, 3, 2, 4).flatten(1, 2)
    there = (s["table"] >= 0).repeat_interleave(c["page"], 1)
    o = _plain_attention(s["q"][qi], k, v, s["offsets"].diff().long(), s["lens"].long(), c["left"], c["right"], c["sinks"], there)
    return _packed(o, s["offsets"], s["q"].shape[0]).to(s["q"].dtype)


def _count(refs, pages, sign):
    """One more (or less) reference to each of `pages`, -1 being none."""
    pages = pages.flatten()
    refs.index_add_(0, pages.clamp(min=0), (pages >= 0).to(torch.int32), alpha=sign)


def _plain_fork(s):
    """Slots [first, first + n) become what the slots `parent` were; -1 frees."""
    at, src = slice(s["first"], s["first"] + s["n"]), s["parent"].long()
    old, old_len = s["table"][at], s["lens"]
    new = torch.where((src >= 0)[:, None], s["table"][src.clamp(min=0)], -1)
    new_len = torch.where(src >= 0, old_len[src.clamp(min=0)], 0)
    _count(s["refs"], new, 1)
    _count(s["refs"], old, -1)
    s["table"][at], s["lens"][at] = new, new_len


def _plain_reserve(s, c):
    """Room for the new tokens: the lowest free pages in the slots' order.  A last page that another slot holds too is
    copied first, but for the last of its holders where all of them append."""
    P, refs = c["page"], s["refs"]
    at, add = slice(s["first"], s["first"] + s["n"]), s["offsets"].diff().long()
    table, old = s["table"][at], s["lens"][at].long()
    new = old + add
    tail_at = (old - 1).clamp(min=0) // P
    part = (old % P != 0) & (add > 0)
    tail = torch.where(part, table.gather(1, tail_at[:, None])[:, 0].long(), -1)
    same = (tail[:, None] == tail) & part[:, None] & part
    held = refs[tail.clamp(min=0)]
    last = ~same.triu(1).any(1)
    copied = part & (held > 1) & ~((held == same.sum(1)) & last)
    have, want = -(-old // P), -(-new // P)
    need = want - have + copied
    begin = need.cumsum(0) - need
    ids = torch.arange(refs.numel(), device=refs.device)
    free = torch.where(refs == 0, ids, refs.numel()).sort().values
    col = torch.arange(table.shape[1], device=refs.device)
    swap = copied[:, None] & (col == tail_at[:, None])
    fresh = (col >= have[:, None]) & (col < want[:, None])
    rank = begin[:, None] + torch.where(swap, 0, copied[:, None] + col - have[:, None])
    page = free[rank.clamp(0, refs.numel() - 1)]
    taken = torch.where(swap | fresh, page, -1)
    _count(refs, taken, 1)
    _count(refs, torch.where(copied, tail, -1), -1)
    s["table"][at] = torch.where(taken >= 0, taken.to(torch.int32), table)
    s["lens"][at] = new.to(torch.int32)
    which = copied.nonzero()[:, 0]
    src, dst = tail[which], page.gather(1, tail_at[:, None])[:, 0][which]
    kept = (torch.arange(P, device=refs.device) < (old % P)[which][:, None])[None, :, None, :, None]
    for pool in (s["k"], s["v"]):
        pool[:, dst] = torch.where(kept, pool[:, src], pool[:, dst])


def _plain_write(s, c):
    off, n = s["offsets"].long(), s["k_new"].shape[1]
    r = torch.arange(n, device=off.device)
    b = torch.searchsorted(off, r, right=True) - 1
    pos = s["lens"][s["first"] + b].long() - (off[b + 1] - r)
    page = s["table"][s["first"] + b, pos // c["page"]].long()
    for pool, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        pool[:, page, :, pos % c["page"]] = new.transpose(0, 1)


def _plain_compact(s):
    """The live pages above the count of live ones go into the free ones below it, each in order."""
    refs = s["refs"]
    ids = torch.arange(refs.numel(), device=refs.device)
    live = refs > 0
    count = live.sum()
    moves = live & (ids >= count)
    holes = torch.where(~live & (ids < count), ids, refs.numel()).sort().values
    to = torch.where(moves, holes[(moves.cumsum(0) - 1).clamp(min=0)], ids)
    src = moves.nonzero()[:, 0]
    for pool in (s["k"], s["v"]):
        pool[:, to[src]] = pool[:, src]
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].to(torch.int32), -1))
    old = refs.clone()
    refs[src] = 0
    refs[to[src]] = old[src]


def _plain_beam(s):
    """The best of all beams' continuations by log probability; a finished beam only goes on as it is."""
    x, b = s["logits"].double(), s["logits"].shape[0]
    w, n = x.shape[1], x.shape[2]
    x = torch.where(x.isnan() | (x == math.inf), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    total = (x - torch.where(top == -math.inf, 0.0, top)).exp().sum(-1, keepdim=True).log() + top
    gain = torch.where(x == -math.inf, x, x - total)
    score = s["scores"].double()[..., None] + gain
    done = s["finished"][..., None]
    token = torch.arange(n, device=x.device)
    score = torch.where(done, s["scores"].double()[..., None], score)
    score = torch.where(score.isnan(), -math.inf, score)
    low = torch.finfo(torch.float64).min
    key = torch.where(done & (token != s["eos"]), -math.inf, score.clamp(min=low)).view(b, w * n)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :w]
    beam, token = order // n, order % n
    row = (beam + torch.arange(b, device=x.device)[:, None] * w).to(torch.int32)
    finished = s["finished"].gather(1, beam) | (token == s["eos"])
    states = [t[row.flatten().long()] for t in s["states"]]
    return dict(scores=score.view(b, w * n).gather(1, order).float(), parents=row, tokens=token.to(torch.int32), finished=finished,
                states=states)


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(q, k, v, left, right, sinks):
    """One sequence: q [i, h, d], k and v [j, kv, d]; a block of queries at a time against the keys that it can see."""
    (n, h, d), (m, kv, _) = q.shape, k.shape
    out = torch.zeros((n, h, d), dtype=torch.float64, device=q.device)
    for lo in range(0, n, 512):
        hi = min(n, lo + 512)
        p = torch.arange(lo, hi, device=q.device) + (m - n)
        begin = 0 if left < 0 else max(0, int(m - n + lo) - left)
        end = m if right < 0 else min(m, m - n + hi + right)
        pick = torch.tensor(sorted(set(range(min(sinks, max(end, 0)))) | set(range(begin, max(end, begin)))), device=q.device, dtype=torch.long)
        if not pick.numel():
            continue
        see = torch.ones((hi - lo, pick.numel()), dtype=torch.bool, device=q.device)
        if right >= 0:
            see &= pick <= p[:, None] + right
        if left >= 0:
            see &= (pick >= p[:, None] - left) | (pick < sinks)
        kk, vv = k[pick].double(), v[pick].double()
        for head in range(h):
            t = (q[lo:hi, head].double() @ kk[:, head * kv // h].T) / math.sqrt(d)
            t = torch.where(see, t, -math.inf)
            e = torch.exp(t - t.amax(1, keepdim=True).clamp(min=-1e300)) * see
            z = e.sum(1, keepdim=True)
            out[lo:hi, head] = torch.where(z > 0, e @ vv[:, head * kv // h] / z.clamp(min=1e-300), 0.0)
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "window":
        qo, ko = s["q_offsets"].tolist(), s["k_offsets"].tolist()
        return torch.cat([_exact_rows(s["q"][a:b], s["k"][x:y], s["v"][x:y], c["left"], c["right"], c["sinks"])
                          for a, b, x, y in zip(qo, qo[1:], ko, ko[1:])])
    if c["op"] == "cache":
        got, off, lens = [], s["offsets"].tolist(), s["lens"].tolist()
        for i, n in enumerate(lens):
            pages = s["table"][i, :-(-n // c["page"])].long()
            k, v = (t[0, pages].transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])[:n] for t in (s["k"], s["v"]))
            got.append(_exact_rows(s["q"][off[i]:off[i + 1]], k, v, c["left"], c["right"], c["sinks"]))
        return torch.cat(got)
    if c["op"] == "beam":
        return _exact_beam(s)
    return dict(_exact_pages(s, c), table=None, lens=None, refs=None)


def _exact_beam(s):
    scores = torch.empty(s["scores"].shape, dtype=torch.float64)
    states = [torch.empty(t.shape, dtype=torch.float64) for t in s["states"]]
    w = scores.shape[1]
    for b in range(scores.shape[0]):
        found = []
        for k in range(w):
            base = float(s["scores"][b, k])
            if bool(s["finished"][b, k]):
                found.append((-base, k, s["eos"]))
                continue
            x = s["logits"][b, k].double().nan_to_num(nan=-math.inf, posinf=-math.inf, neginf=-math.inf)
            x = x - torch.logsumexp(x, 0)
            best = torch.sort(x, dim=0, descending=True, stable=True)
            found += [(-(base + g), k, t) for g, t in zip(best.values[:w].tolist(), best.indices[:w].tolist())]
        for r, (score, k, _) in enumerate(sorted(found)[:w]):
            scores[b, r] = -score
            for t, u in zip(states, s["states"]):
                t[b * w + r] = u[b * w + k].double()
    return dict(scores=scores, parents=None, tokens=None, finished=None, states=states)


def _exact_pages(s, c):
    """The pools after the pass, with the pages' bookkeeping in lists, one slot after the other."""
    P = c["page"]
    k, v = s["k"].double(), s["v"].double()
    table, refs, lens = s["table"].tolist(), s["refs"].tolist(), s["lens"].tolist()
    if c["op"] == "compact":
        live = sum(r > 0 for r in refs)
        holes = [i for i in range(live) if not refs[i]]
        high = [i for i in range(live, len(refs)) if refs[i]]
        for t in (k, v):
            t[:, holes] = t[:, high]
        return dict(k=k, v=v)
    first, n, off = s["first"], s["n"], s["offsets"].tolist()
    for i, p in enumerate(s["parent"].tolist()):  # the slots that take are not among those that give
        table[first + i] = list(table[p]) if p >= 0 else [-1] * len(table[first + i])
        lens[first + i] = lens[p] if p >= 0 else 0
        for page in table[first + i]:
            if page >= 0:
                refs[page] += 1
    free = iter([i for i, r in enumerate(refs) if not r])
    for i in range(n):
        row, old, add = table[first + i], lens[first + i], off[i + 1] - off[i]
        if add and old % P and refs[row[old // P]] > 1:  # the parents keep theirs, so every shared last page is copied
            src, dst = row[old // P], next(free)
            refs[src] -= 1
            row[old // P], refs[dst] = dst, 1
            for t in (k, v):
                t[:, dst, :, :old % P] = t[:, src, :, :old % P]
        for col in range(-(-old // P), -(-(old + add) // P)):
            row[col] = next(free)
            refs[row[col]] = 1
        lens[first + i] = old + add
        pos = torch.arange(old, old + add)
        page = torch.tensor(row)[pos // P].cuda()
        for t, new in ((k, s["k_new"]), (v, s["v_new"])):
            t[:, page, :, (pos % P).cuda()] = new[:, off[i]:off[i + 1]].transpose(0, 1).double()
    return dict(k=k, v=v)


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "window":
        lens = _lengths(c, c["seqs"], c["tokens"])
        pairs = sum(_visible(n, n + c["past"], c["left"], c["right"], c["sinks"]) for n in lens)
        keys = sum(_touched(n, n + c["past"], c["left"], c["right"], c["sinks"]) for n in lens)
        return {"bytes": size * c["dim"] * (2 * sum(lens) * c["q_heads"] + 2 * keys * c["kv_heads"]),
                "flops": 4 * c["dim"] * c["q_heads"] * pairs}
    if c["op"] == "cache":
        ctx = _lengths(c, c["seqs"], c["context"], c["tokens"])
        news = [min(n, x) for n, x in zip(_lengths(dict(c, of="q"), c["seqs"], c["tokens"]), ctx)]
        pairs = sum(_visible(n, m, c["left"], c["right"], c["sinks"]) for n, m in zip(news, ctx))
        keys = sum(_touched(n, m, c["left"], c["right"], c["sinks"]) for n, m in zip(news, ctx))
        return {"bytes": size * c["dim"] * (2 * sum(news) * c["q_heads"] + 2 * keys * c["kv_heads"]) + 4 * keys // c["page"],
                "flops": 4 * c["dim"] * c["q_heads"] * pairs}
    if c["op"] == "beam":
        rows = c["items"] * c["beams"]
        return {"bytes": rows * (c["vocab"] * size + 8 * c["states"] * c["width"] + 18), "flops": 3 * rows * c["vocab"]}
    token = 2 * c["layers"] * c["kv_heads"] * c["dim"] * size  # a token's keys and values in all layers
    if c["op"] == "step":
        n = c["items"] * c["beams"]
        row = -(-c["context"] // c["page"])
        return {"bytes": 2 * n * token * (c["tokens"] + c["context"] % c["page"]) + 12 * n * row, "flops": 0}
    if c["op"] == "append":
        counts = _lengths(c, c["seqs"], c["tokens"])
        return {"bytes": 2 * token * sum(counts) + 8 * sum(-(-n // c["page"]) for n in counts), "flops": 0}
    live = max(1, int(c["pages"] * c["live"]))
    moved = live * (c["pages"] - live) / c["pages"]  # as many live pages lie above their count, on the mean
    return {"bytes": 2 * moved * token * c["page"] + 8 * c["pages"] + 8 * live, "flops": 0}
