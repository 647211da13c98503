"""Edges of the decoding operators' contracts: what unseen rows, masked queries, full-size pools and directly following
launches do, against plain implementations in 64 bits (tolerances as in test_decode_ops_gpu.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_decode_ops_gpu import DT, attention64, beam64, check_rows, make_cache, nq, offsets  # noqa: E402, F401


def unseen_keys(n_q, n_k, left, sinks):
    """[a, b): the keys after the sinks that lie before the first query's window."""
    return min(sinks, n_k), max(0, n_k - n_q - left)


GAPS = [(200, 300, 50, 4), (300, 400, 20, 70), (150, 390, 5, 130), (400, 460, 59, 0), (129, 257, 0, 1), (150, 600, 100, 4), (40, 160, 9, 30)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (6, 2, 128), (2, 1, 40)])
@pytest.mark.parametrize("n_q,n_k,left,sinks", GAPS)
def test_keys_between_the_sinks_and_the_window_may_hold_anything(dt, hq, hk, d, n_q, n_k, left, sinks):
    """Of a sequence with more keys than queries, the keys that no query sees: their values change nothing."""
    from nspeech_b200.attention import window_attention
    a, b = unseen_keys(n_q, n_k, left, sinks)
    assert b == 0 or a < b
    g = torch.Generator().manual_seed(n_q + d)
    q, k, v = (torch.randn((n, h, d), generator=g).to(DT[dt]) for n, h in ((n_q, hq), (n_k, hk), (n_k, hk)))
    want = attention64(q, k, v, left, 0, sinks)
    for bad in (float("nan"), float("inf")):
        k[a:b], v[a:b] = bad, bad
        check_rows(window_attention(q.cuda(), k.cuda(), v.cuda(), left, 0, sinks), *want)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("page", [8, 64, 256])
@pytest.mark.parametrize("left,sinks", [(50, 4), (20, 70), (5, 130)])
def test_cached_tokens_between_the_sinks_and_the_window_may_hold_anything(dt, page, left, sinks):
    lens, news = [300, 390, 700], [200, 150, 180]
    cache, rows = make_cache(dt, lens, page, 2, 64, seed=page)
    for i, (m, n) in enumerate(zip(lens, news)):
        for j in range(*unseen_keys(n, m, left, sinks)):
            at = int(cache.table[i, j // page]), slice(None), j % page
            cache.k[1][at], cache.v[1][at] = float("nan"), float("nan")
    q = torch.randn((sum(news), 4, 64), generator=torch.Generator().manual_seed(left)).to(DT[dt])
    got = cache.attention(q.cuda(), 1, offsets(news), left=left, sinks=sinks)
    at = np.concatenate([[0], np.cumsum(news)])
    for i, (a, b) in enumerate(zip(at, at[1:])):
        check_rows(got[a:b], *attention64(q[a:b], rows[i][0][1], rows[i][1][1], left, 0, sinks))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n_q,n_k,hq,hk,d", [(1, 5, 2, 2, 64), (1, 3000, 2, 2, 64), (1, 3000, 4, 1, 128), (4, 900, 2, 2, 64), (9, 3000, 2, 1, 64),
                                             (40, 3000, 2, 2, 128), (300, 300, 4, 2, 64), (140, 5000, 2, 2, 64)])
def test_a_query_that_is_not_a_number_gives_none(dt, n_q, n_k, hq, hk, d):
    """Its softmax has no value, whatever form runs and however the keys are split; other rows are as they would be."""
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(n_q + n_k)
    q, k, v = (torch.randn((n, h, d), generator=g).to(DT[dt]) for n, h in ((n_q, hq), (n_k, hk), (n_k, hk)))
    want, tol = attention64(q, k, v, -1, 0, 0)
    row = n_q // 2
    q[row, 1, 3] = float("nan")
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), -1, 0).cpu()
    assert bool(torch.isnan(got[row, 1]).all())
    got[row, 1], want[row, 1] = 0, 0
    check_rows(got, want, tol)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[6, 40, 9], [3000, 5, 700]])
def test_a_cached_token_s_query_that_is_not_a_number_gives_none(dt, lens):
    cache, rows = make_cache(dt, lens, 16, 2, 64)
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(2)).to(DT[dt])
    q[0, 2, 5] = float("nan")
    got = cache.attention(q.cuda(), 0).cpu()
    assert bool(torch.isnan(got[0, 2]).all())
    for i in range(3):
        want, tol = attention64(q[i:i + 1].nan_to_num(0.0), rows[i][0][0], rows[i][1][0], -1, 0, 0)
        keep = torch.ones((1, 4), dtype=torch.bool)
        keep[0, 2] = i > 0
        check_rows(got[i:i + 1][keep], want[keep], tol[keep])


@pytest.mark.parametrize("pages,slots,longest", [(1 << 20, 4096, 2048), (400001, 37, 2048), (140003, 4096, 100)])
def test_the_largest_pools_and_calls(pages, slots, longest):
    """Pools and calls at the sizes that the header allows: room, forks and a compaction against numpy."""
    from nspeech_b200.cache import PagedCache
    cols = longest // 8 + 2
    cache = PagedCache.create(1, pages, 8, 1, 8, slots, cols)
    rng = np.random.default_rng(pages)
    counts = rng.integers(0, longest, slots)
    counts[0] = longest
    cache.reserve(offsets(counts))
    cache.check()
    need = -(-counts // 8)
    want = np.full((slots, cols), -1)
    want[np.arange(cols) < need[:, None]] = np.arange(need.sum())
    assert np.array_equal(cache.table.cpu().numpy(), want) and np.array_equal(cache.lens.cpu().numpy(), counts)
    cache.k[0, :, 0, 0, 0] = (torch.arange(pages, device="cuda") % 251).bfloat16()  # marks that move with their pages
    src = rng.integers(-1, slots, slots).astype(np.int32)
    src[: slots // 2] = -1
    cache.fork(torch.from_numpy(src).cuda())
    cache.check()
    want = np.where(src[:, None] >= 0, want[src], -1)
    refs = np.bincount(want[want >= 0], minlength=pages)
    assert np.array_equal(cache.table.cpu().numpy(), want) and np.array_equal(cache.refs.cpu().numpy(), refs)
    marks = np.where(want >= 0, want % 251, 0)
    cache.compact()
    cache.check()
    live = int((refs > 0).sum())
    assert int(cache.live) == live
    to = np.arange(pages)
    to[live + np.flatnonzero(refs[live:])] = np.flatnonzero(refs[:live] == 0)
    want = np.where(want >= 0, to[want], -1)
    assert np.array_equal(cache.table.cpu().numpy(), want)
    pos = torch.from_numpy(np.where(want >= 0, want, 0)).cuda().long()
    got = cache.k[0, :, 0, 0, 0][pos].float().cpu().numpy()
    assert np.array_equal(np.where(want >= 0, got, 0), marks)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("beams", [1, 8, 32])
@pytest.mark.parametrize("last", [5, 40, 700])
def test_beam_select_after_rounds_of_equal_values(dt, beams, last):
    """Rounds with more equal best values than are listed, each followed by one with a few better values at places of
    other lanes: what a round lists is that round's logits."""
    from nspeech_b200.beam import beam_select
    rng, rounds = np.random.default_rng(last), 9
    items = max(40, 320 // beams)  # several rounds a CTA
    x = np.zeros((items, beams, rounds * 8192 + last), np.float32)
    for r in range(rounds):
        x[:, :, r * 8192:] = r / 2  # all of a round equal, above the one before
        at = r * 8192 + rng.integers(0, 8192, 11)
        if r % 2:
            x[:, :, at] = r / 2 + 0.25 + np.arange(11) / 64
    x += rng.integers(0, 2, (items, 1, 1))
    lt = torch.from_numpy(x).to(DT[dt])
    scores = np.arange(items * beams, dtype=np.float32).reshape(items, beams) * -0.0101  # no ties across beams: 0.6464 k is 0.01 off any integer
    got = [t.cpu() for t in beam_select(lt.cuda(), torch.from_numpy(scores).cuda())]
    for i in range(0, items, 13):
        want = beam64(lt[i].float().numpy(), scores[i], np.zeros(beams, bool), -1)
        assert got[1][i].tolist() == [i * beams + b for _, b, _ in want]
        assert got[2][i].tolist() == [t for _, _, t in want]


class Layers:
    """Layers of attention between Q8_0-path projections (weights kept at bf16 precision, f32 activations)."""

    def __init__(self, layers=3, heads=2, kv=1, dim=64, width=128):
        from nspeech_b200.fast_matmul import QWeight
        g = torch.Generator().manual_seed(23)
        self.heads, self.kv, self.dim, self.width, self.layers = heads, kv, dim, width, layers
        sizes = {"qkv": ((heads + 2 * kv) * dim, width), "o": (width, heads * dim)}
        self.w = [{n: (torch.randn(s, generator=g) * s[1] ** -0.5).bfloat16().float() for n, s in sizes.items()} for _ in range(layers)]
        self.q = [{n: QWeight.from_f32(t.numpy()) for n, t in w.items()} for w in self.w]

    def step(self, cache, x):
        """One token a slot: a projection's keys and values go straight into the cache, a layer after the other."""
        n = x.shape[0]
        cache.reserve(1, 0, n)
        for i, q in enumerate(self.q):
            qkv = q["qkv"].linear(x).view(n, -1, self.dim)
            q1, k, v = qkv.split([self.heads, self.kv, self.kv], 1)
            cache.write(k, v, 1, 0, n, layer=i)
            a = cache.attention(q1, i, n=n)
            x = q["o"].linear(a.reshape(n, -1)) + x
        return x

    def run64(self, xs):
        """The last token's output after the tokens xs [t, width] of one sequence."""
        x = xs.double()
        for w in self.w:
            q, k, v = (x @ w["qkv"].double().T).view(len(x), -1, self.dim).split([self.heads, self.kv, self.kv], 1)
            a = attention64(q, k, v, -1, 0, 0)[0]
            x = a.reshape(len(x), -1) @ w["o"].double().T + x
        return x[-1]


@pytest.mark.parametrize("slots", [1, 6])
def test_layers_write_what_the_projection_before_has_just_made(slots):
    """Projection, write and attention follow one another directly in every layer, eagerly and in a replayed graph, over
    buffers that hold the step before's values."""
    from nspeech_b200.cache import PagedCache
    net, steps = Layers(), 12
    xs = torch.randn((slots, steps, net.width), generator=torch.Generator().manual_seed(slots))
    want = torch.stack([torch.stack([net.run64(xs[i, :t + 1]) for t in range(steps)]) for i in range(slots)])
    # six projections of f32 activations as bf16 hi + lo planes, each 2^-16 of a sum of absolute terms below 8; gains below 2
    def close(y, t):
        assert bool(((y.double().cpu() - want[:, t]).abs() < 2e-3).all()), t

    def begin():
        return PagedCache.create(net.layers, 4 * slots, 8, net.kv, net.dim, slots, 4, torch.float32)

    cache = begin()
    for t in range(steps):
        close(net.step(cache, xs[:, t].contiguous().cuda()), t)
    cache.check()
    cache, x = begin(), torch.zeros((slots, net.width), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        net.step(begin(), x)  # this stream's workspaces
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = net.step(cache, x)
    for t in range(steps):
        x.copy_(xs[:, t])
        graph.replay()
        close(y, t)
    cache.check()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_greedy_decoding_over_padded_rows(dt):
    from nspeech_b200.beam import beam_select
    g = torch.Generator().manual_seed(12)
    padded = torch.randn((5, 1032), generator=g).to(DT[dt]).cuda()
    last = torch.randn((5, 3, 1001), generator=g).to(DT[dt]).cuda()
    scores = -torch.rand((5, 1), generator=g).cuda()
    for logits in (padded[:, :1000].unsqueeze(1), last[:, -1:]):
        want = beam_select(logits.contiguous(), scores)
        assert all(torch.equal(a, b) for a, b in zip(beam_select(logits, scores), want))
        assert torch.equal(want[2][:, 0].long(), logits[:, 0].float().argmax(1))


def test_states_that_stand_for_other_values_and_outputs_that_autograd_has_saved():
    from nspeech_b200.attention import window_attention
    from nspeech_b200.beam import beam_reorder, beam_select
    from nspeech_b200.fast_matmul import MatMulError
    parents = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    state = torch.randn((2, 3), device="cuda")
    for bad, word in ((torch._neg_view(state), "negated"), (torch.randn((2, 3), dtype=torch.cfloat, device="cuda").conj(), "conjugated"),
                      (state.clone().requires_grad_(), "gradient")):
        with pytest.raises(MatMulError, match=word):
            beam_reorder([bad], parents)
    q, w = torch.randn((8, 2, 64), device="cuda"), torch.ones((), device="cuda", requires_grad=True)
    kept = torch.randn((2, 3), device="cuda")
    scores, logits = torch.zeros((1, 2), device="cuda"), torch.randn((1, 2, 9), device="cuda")
    rest = [t.clone() for t in beam_select(logits, scores)[1:]]
    for out, write in ((torch.empty_like(q), lambda t: window_attention(q, q, q, out=t)), (kept, lambda t: beam_reorder([state], parents, out=[t])),
                       (scores, lambda t: beam_select(logits, scores.clone(), out=(t, *rest)))):
        loss = (out * w).sum()  # saves out
        write(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # nothing is tracked there
        out = torch.empty_like(q)
        assert torch.equal(window_attention(q, q, q, out=out), window_attention(q, q, q))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,m,hq,hk,d", [(1, 3000, 4, 2, 64), (5, 90, 2, 2, 64), (300, 300, 8, 2, 64), (1000, 1000, 3, 3, 128), (130, 4000, 2, 1, 40)])
def test_attention_in_place_of_its_queries(dt, n, m, hq, hk, d):
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(n + d)
    q, k, v = (torch.randn((r, h, d), generator=g).to(DT[dt]).cuda() for r, h in ((n, hq), (m, hk), (m, hk)))
    want = window_attention(q, k, v, 200, 0, 3)
    assert torch.equal(window_attention(q, k, v, 200, 0, 3, out=q), want)


def test_beam_reorder_leaves_its_parents_alone():
    from nspeech_b200.beam import beam_reorder
    from nspeech_b200.fast_matmul import MatMulError
    parents = torch.tensor([2, 0, 0, 1], dtype=torch.int32, device="cuda")
    state = torch.arange(8, device="cuda").view(4, 2)
    with pytest.raises(MatMulError, match="parents"):
        beam_reorder([state, parents], parents, out=[state, parents])
    many = [state.clone() for _ in range(17)]
    with pytest.raises(MatMulError, match="parents"):
        beam_reorder(many + [parents], parents, out=many + [parents])
    assert all(torch.equal(t, state) for t in many) and parents.tolist() == [2, 0, 0, 1]
    got = beam_reorder([state, parents], parents)  # they may be read as a state
    assert got[1].tolist() == [0, 2, 2, 0] and torch.equal(got[0], state[parents.long()])
