"""Window attention, the paged cache and beam search against plain implementations in 64 bits.

Tolerances come from the arithmetic.  A score is a sum of head_dim products in f32, (d + 2) roundings of 2^-24 of the
sum of absolute products; exp2 adds 2^-21 at most; the softmax sums up to n terms in f32.  A relative change of e of
every weight moves the output by at most 2 e sum p |v|.  bf16 rounds each weight (2^-8 of it) and the output (2^-8).
"""
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def nq():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nspeech_b200 import lib
    lib.init(0)
    return lib


DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def visible(n_q, n_k, left, right, sinks):
    p = torch.arange(n_q)[:, None] + (n_k - n_q)
    j = torch.arange(n_k)[None, :]
    see = torch.ones((n_q, n_k), dtype=torch.bool)
    if right >= 0:
        see &= j <= p + right
    if left >= 0:
        see &= (j >= p - left) | (j < sinks)
    return see


def attention64(q, k, v, left, right, sinks, scale=None, there=None):
    """(output, tolerance) of one sequence; q [n, h, d], k and v [m, kv, d] on the CPU; there [m]: keys that exist."""
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    (n, h, d), (m, kv, _) = q.shape, k.shape
    scale = d ** -0.5 if scale is None else scale
    see = visible(n, m, left, right, sinks)
    if there is not None:
        see &= there
    out, tol = torch.zeros(n, h, d, dtype=torch.float64), torch.zeros(n, h, d, dtype=torch.float64)
    if m == 0 or n == 0:
        return out, tol
    for x in range(h):
        kk, vv = k[:, x // (h // kv)], v[:, x // (h // kv)]
        s = torch.where(see, (q[:, x] @ kk.T) * scale, -torch.inf)
        top = s.amax(1, keepdim=True)
        e = torch.exp(s - torch.where(top == -torch.inf, 0.0, top)) * see
        z = e.sum(1, keepdim=True)
        w = torch.where(z > 0, e / z.clamp(min=1e-300), 0.0)
        out[:, x] = w @ torch.where(see.any(0)[:, None], vv, 0.0)
        mass = w @ torch.where(see.any(0)[:, None], vv.abs(), 0.0)
        work = ((q[:, x].abs() @ kk.abs().T) * abs(scale) * see).amax(1, keepdim=True)
        err = (d + 2) * 2.0 ** -24 * work + 2.0 ** -21 + (m + 8) * 2.0 ** -24
        tol[:, x] = 2 * err * mass + (2.0 ** -8 * (mass + out[:, x].abs()) if dt == torch.bfloat16 else 2.0 ** -24 * out[:, x].abs())
    return out, tol + 1e-30


def check_rows(got, want, tol):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.double()).all()
    assert bool((off <= tol).all()), f"off by {float((off / tol.clamp(min=1e-30)).max()):.3f} of the tolerance"


def offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


# lengths: none, one, around the tiles of 32 and 64, several tiles; windows: causal, full, one key, narrow, wide; rows that see nothing
WINDOWS = [(-1, 0, 0), (-1, -1, 0), (0, 0, 0), (16, 4, 0), (7, 0, 1), (63, 0, 4), (100, 33, 70), (-1, 5, 3), (5, -1, 2)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (6, 2, 128), (5, 1, 40), (3, 3, 36), (2, 1, 7)])
def test_window_attention(dt, left, right, sinks, hq, hk, d):
    from nspeech_b200.attention import window_attention
    lens = [0, 1, 65, 31, 200, 0, 64, 129]
    g = torch.Generator().manual_seed(left * 7 + d)
    q, k, v = (torch.randn((sum(lens), h, d), generator=g).to(DT[dt]) for h in (hq, hk, hk))
    off = offsets(lens)
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), left, right, sinks, q_offsets=off, k_offsets=off)
    at = np.concatenate([[0], np.cumsum(lens)])
    for a, b in zip(at, at[1:]):
        check_rows(got[a:b], *attention64(q[a:b], k[a:b], v[a:b], left, right, sinks))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n_q,n_k", [(1, 1), (1, 700), (3, 2000), (9, 1000), (20, 5), (70, 64), (40, 3000), (130, 3500)])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (300, 0, 4), (1000, 2, 130)])
def test_few_queries_over_many_keys(dt, n_q, n_k, left, right, sinks):
    """The split over the keys, with its join; queries before the first key see nothing."""
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(n_q * 31 + n_k)
    q, k, v = (torch.randn((n, h, 64), generator=g).to(DT[dt]) for n, h in ((n_q, 6), (n_k, 2), (n_k, 2)))
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), left, right, sinks)
    check_rows(got, *attention64(q, k, v, left, right, sinks))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,d,hq,hk", [(1000, 64, 2, 2), (700, 128, 4, 1), (333, 20, 1, 1)])
@pytest.mark.parametrize("left,right,sinks", WINDOWS + [(250, 0, 4), (300, 200, 65)])
def test_every_key_counts_once(dt, n, d, hq, hk, left, right, sinks):
    """Equal scores make the output the share of visible keys in each residue class: exact up to the output's rounding."""
    from nspeech_b200.attention import window_attention
    q, k = torch.zeros((n, hq, d)), torch.randn((n, hk, d), generator=torch.Generator().manual_seed(1))
    v = (torch.arange(n)[:, None, None] % d == torch.arange(d)).expand(n, hk, d).float()
    got = window_attention(q.to(DT[dt]).cuda(), k.to(DT[dt]).cuda(), v.to(DT[dt]).cuda(), left, right, sinks).double().cpu()
    see = visible(n, n, left, right, sinks).double()
    want = (see @ v[:, 0].double() / see.sum(1, keepdim=True).clamp(min=1))[:, None].expand(n, hq, d)
    # 1 / n in f32 and the product: two roundings, then the output's
    assert bool(((got - want).abs() <= want * (2.0 ** -8 if dt == "bf16" else 0) + want * 2.0 ** -22).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strides_padding_and_rows_left_alone(dt):
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(3)
    b, t, h, d = 5, 90, 3, 24
    lens = [90, 0, 1, 64, 77]
    rows = torch.randn((b * t, 3 * h * d + 5), generator=g).to(DT[dt])  # rows on no 16-byte boundary
    rows[90:180] = float("nan")  # padding may hold anything
    rows[181:270] = float("inf")
    dev = rows.cuda()
    q, k, v = (dev[:, 1 + i * h * d:1 + (i + 1) * h * d].unflatten(1, (h, d)) for i in range(3))
    out = torch.full((b * t + 4, h, d + 8), -7.0, dtype=DT[dt], device="cuda")[:b * t, :, :d]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    window_attention(q, k, v, 20, 6, 2, q_lens=n, k_lens=n, out=out)
    for i, m in enumerate(lens):
        a = i * t
        check_rows(out[a:a + m], *attention64(*(x[a:a + m].cpu() for x in (q, k, v)), 20, 6, 2))
        assert bool((out[a + m:a + t] == -7).all())
    # offsets that end before the rows do, and head-major rows [h, n, d]
    off = offsets([10, 33])
    for x in (q, k, v):
        x.nan_to_num_(0.0, 0.0, 0.0)
    major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    out = torch.full((b * t, h, d), -7.0, dtype=DT[dt], device="cuda")
    window_attention(*major, 8, 0, q_offsets=off, k_offsets=off, out=out)
    check_rows(out[:10], *attention64(*(x[:10].cpu() for x in major), 8, 0, 0))
    check_rows(out[10:43], *attention64(*(x[10:43].cpu() for x in major), 8, 0, 0))
    assert bool((out[43:] == -7).all())


@pytest.mark.parametrize("n,hq,hk,d,left,right,sinks", [(1500, 4, 1, 128, -1, 0, 0), (1100, 3, 3, 64, 200, 0, 4), (700, 7, 1, 96, 500, 40, 130),
                                                       (2100, 2, 1, 40, 1000, 0, 300), (900, 2, 2, 128, 3, 700, 1)])
def test_long_prompts_in_bf16(n, hq, hk, d, left, right, sinks):
    """Many row tiles and key tiles; sinks that reach into the window's tiles; peaked softmax."""
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn((n, h, d), generator=g).bfloat16() for h in (hq, hk, hk))
    for factor in (1.0, 30.0):
        got = window_attention((q * factor).cuda(), k.cuda(), v.cuda(), left, right, sinks)
        check_rows(got, *attention64(q * factor, k, v, left, right, sinks))


def test_negative_and_zero_scale():
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(6)
    for dt in ("f32", "bf16"):
        q, k, v = (torch.randn((150, 2, 64), generator=g).to(DT[dt]) for _ in range(3))
        for scale in (-0.2, 0.0):
            got = window_attention(q.cuda(), k.cuda(), v.cuda(), 40, 0, 2, scale=scale)
            check_rows(got, *attention64(q, k, v, 40, 0, 2, scale))


@pytest.mark.parametrize("page", [8, 256, 1024])
@pytest.mark.parametrize("left,sinks", [(-1, 0), (700, 4), (100, 200)])
def test_prompt_chunks_over_the_cache(page, left, sinks):
    """Many queries over many pages, some of them given back; pages larger than a key tile."""
    lens, news = [2500, 300, 1300], [300, 300, 77]
    cache, rows = make_cache("bf16", lens, page, 2, 64, seed=page)
    q = torch.randn((sum(news), 4, 64), generator=torch.Generator().manual_seed(left + 2)).bfloat16()
    got = cache.attention(q.cuda(), 1, offsets(news), left=left, sinks=sinks)
    at = np.concatenate([[0], np.cumsum(news)])
    for i, (a, b) in enumerate(zip(at, at[1:])):
        check_rows(got[a:b], *attention64(q[a:b], rows[i][0][1], rows[i][1][1], left, 0, sinks))
    cache.trim(600, 9)
    cache.check()
    got = cache.attention(q.cuda(), 1, offsets(news), left=left, sinks=sinks)
    for i, (a, b) in enumerate(zip(at, at[1:])):
        there = (cache.table[i] >= 0).repeat_interleave(page)[:lens[i]].cpu()
        check_rows(got[a:b], *attention64(q[a:b], rows[i][0][1], rows[i][1][1], left, 0, sinks, there=there))


def test_scale_and_no_rows():
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn((50, 2, 64), generator=g) for _ in range(3))
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), scale=0.5)
    check_rows(got, *attention64(q, k, v, -1, -1, 0, 0.5))
    none = window_attention(q[:0].cuda(), k.cuda(), v.cuda())
    assert none.shape == (0, 2, 64)
    assert bool((window_attention(q.cuda(), k[:0].cuda(), v[:0].cuda()) == 0).all())


# --------------------------------------------------------------------------------------------------------- the cache
def make_cache(dt, lens, page, heads, dim, layers=2, extra=5, seed=0, slack=3):
    """A cache whose slots hold `lens` tokens on shuffled pages; free pages and the pages' ends hold NaN."""
    from nspeech_b200.cache import PagedCache
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1]) + slack), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    k, v = (torch.full((layers, pages, heads, page, dim), float("nan")) for _ in range(2))
    rows = []
    for i, n in enumerate(lens):
        kk, vv = (torch.randn((layers, n, heads, dim), generator=g).to(DT[dt]) for _ in range(2))
        rows.append((kk, vv))
        for c in range(need[i]):
            pg = order.pop()
            table[i, c], refs[pg] = pg, 1
            m = min(page, n - c * page)
            k[:, pg, :, :m] = kk[:, c * page:c * page + m].transpose(1, 2).float()
            v[:, pg, :, :m] = vv[:, c * page:c * page + m].transpose(1, 2).float()
    cache = PagedCache(k.to(DT[dt]).cuda(), v.to(DT[dt]).cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), refs.cuda())
    return cache, rows


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("page,hq,hk,d", [(8, 4, 4, 64), (16, 12, 3, 128), (64, 2, 2, 20), (128, 8, 1, 128)])
@pytest.mark.parametrize("left,sinks", [(-1, 0), (40, 0), (100, 9), (0, 1)])
@pytest.mark.parametrize("tokens", [1, 2, 37])
def test_cache_attention(dt, page, hq, hk, d, left, sinks, tokens):
    lens = [300, 1, 0, 64, 129, 2000]
    news = [min(n, tokens) for n in lens]
    cache, rows = make_cache(dt, lens, page, hk, d, seed=page + d)
    q = torch.randn((sum(news) + 3, hq, d), generator=torch.Generator().manual_seed(tokens)).to(DT[dt])
    out = torch.full(q.shape, -7.0, dtype=DT[dt], device="cuda")
    cache.attention(q.cuda(), 1, offsets(news), left=left, sinks=sinks, out=out)
    at = np.concatenate([[0], np.cumsum(news)])
    for i, (a, b) in enumerate(zip(at, at[1:])):
        check_rows(out[a:b], *attention64(q[a:b], rows[i][0][1], rows[i][1][1], left, 0, sinks))
    assert bool((out[at[-1]:] == -7).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_cache_attention_of_single_tokens_over_some_slots(dt):
    """No offsets: one token for each of slots [2, 5); cross attention (right = -1) sees every token."""
    lens = [5, 9, 33, 500, 64, 7]
    cache, rows = make_cache(dt, lens, 16, 2, 64)
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(1)).to(DT[dt])
    got = cache.attention(q.cuda(), 0, first=2, n=3, right=-1)
    for i in range(3):
        check_rows(got[i:i + 1], *attention64(q[i:i + 1], rows[2 + i][0][0], rows[2 + i][1][0], -1, -1, 0))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_trim_and_attention_without_the_trimmed_pages(dt):
    lens = [500, 17, 64, 200]
    cache, rows = make_cache(dt, lens, 16, 2, 64)
    live = int((cache.refs > 0).sum())
    cache.trim(window=50, sinks=4)
    cache.check()
    for i, n in enumerate(lens):
        for c in range(-(-n // 16)):
            gone = c >= 1 and (c + 1) * 16 <= n - 50
            assert (int(cache.table[i, c]) == -1) == gone
    freed = live - int((cache.refs > 0).sum())
    assert freed == sum(max(0, (n - 50) // 16 - 1) if n > 50 else 0 for n in lens)
    # new tokens after the trim see exactly their window
    cache.reserve(1)
    new = torch.randn((4, 2, 64), generator=torch.Generator().manual_seed(8)).to(DT[dt])
    for layer in range(2):
        cache.write(new.cuda(), new.cuda(), 1, layer=layer)
    q = torch.randn((4, 2, 64), generator=torch.Generator().manual_seed(9)).to(DT[dt])
    got = cache.attention(q.cuda(), 1, left=50, sinks=4)
    wide = cache.attention(q.cuda(), 1)  # no window: the trimmed keys are not seen either
    cache.check()
    for i, n in enumerate(lens):
        k, v = (torch.cat([r[1], new[i:i + 1]]) for r in rows[i])
        check_rows(got[i:i + 1], *attention64(q[i:i + 1], k, v, 50, 0, 4))
        there = torch.tensor([j < 16 or (j // 16 + 1) * 16 > n - 50 or n <= 50 for j in range(n + 1)])
        check_rows(wide[i:i + 1], *attention64(q[i:i + 1], k, v, -1, 0, 0, there=there))


class Model:
    """The cache's rules in lists, one slot after the other; each token is a number."""

    def __init__(self, slots, pages, page, max_pages):
        self.table = [[-1] * max_pages for _ in range(slots)]
        self.lens, self.refs, self.page = [0] * slots, [0] * pages, page
        self.data = [[None] * page for _ in range(pages)]

    def fork(self, first, src):
        old = [list(r) for r in self.table], list(self.lens)
        for i, s in enumerate(src):
            for pg in self.table[first + i]:
                self.refs[pg] -= pg >= 0
            self.table[first + i] = list(old[0][s]) if s >= 0 else [-1] * len(self.table[0])
            self.lens[first + i] = old[1][s] if s >= 0 else 0
            for pg in self.table[first + i]:
                self.refs[pg] += pg >= 0

    def reserve(self, first, counts):
        P, n = self.page, len(counts)
        grow = [i for i in range(n) if counts[i] and self.lens[first + i] % P]
        tail = {i: self.table[first + i][self.lens[first + i] // P] for i in grow}
        held = dict(enumerate(self.refs))
        copied = set()
        for i in grow:
            holders = [j for j in grow if tail[j] == tail[i]]
            if held[tail[i]] > 1 and not (len(holders) == held[tail[i]] and i == holders[-1]):
                copied.add(i)
        need = [-(-(self.lens[first + i] + c) // P) - -(-self.lens[first + i] // P) + (i in copied) for i, c in enumerate(counts)]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if sum(need) > len(free):
            return 1
        if any(self.lens[first + i] + c > P * len(self.table[0]) for i, c in enumerate(counts)):
            return 2
        free = iter(free)
        before = [list(d) for d in self.data]
        for i, c in enumerate(counts):
            row, old = self.table[first + i], self.lens[first + i]
            if i in copied:
                new = next(free)
                self.data[new][:old % P] = before[row[old // P]][:old % P]
                self.refs[row[old // P]] -= 1
                row[old // P], self.refs[new] = new, 1
            for col in range(-(-old // P), -(-(old + c) // P)):
                row[col] = next(free)
                self.refs[row[col]] = 1
            self.lens[first + i] = old + c
        return 0

    def write(self, first, counts, tokens):
        it = iter(tokens)
        for i, c in enumerate(counts):
            for pos in range(self.lens[first + i] - c, self.lens[first + i]):
                self.data[self.table[first + i][pos // self.page]][pos % self.page] = next(it)

    def trim(self, first, n, sinks, window):
        P = self.page
        for i in range(first, first + n):
            for col in range(-(-sinks // P), max(0, self.lens[i] - window) // P):
                pg = self.table[i][col]
                if pg >= 0:
                    self.refs[pg] -= 1
                    self.table[i][col] = -1

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        up = [p for p in range(live, len(self.refs)) if self.refs[p]]
        to = dict(zip(up, (p for p in range(live) if not self.refs[p])))
        for a, b in to.items():
            self.data[b], self.refs[b], self.refs[a] = list(self.data[a]), self.refs[a], 0
        self.table = [[to.get(p, p) for p in r] for r in self.table]
        return live


def same_as(cache, m, layers):
    assert cache.table.tolist() == m.table
    assert cache.lens.tolist() == m.lens
    assert cache.refs.tolist() == m.refs
    held = [p for p, r in enumerate(m.refs) if r]
    k, v = cache.k.cpu().float(), cache.v.cpu().float()
    for p in held:
        for r, t in enumerate(m.data[p]):
            if t is not None and any(p in row and r + row.index(p) * m.page < n for row, n in zip(m.table, m.lens)):
                for la in range(layers):
                    assert bool((k[la, p, :, r] == t + la * 100).all() and (v[la, p, :, r] == -t - la * 100).all())


@pytest.mark.parametrize("dt,dim,heads", [("f32", 64, 2), ("bf16", 40, 3), ("bf16", 5, 1)])
@pytest.mark.parametrize("page,pages,seed", [(8, 61, 0), (16, 40, 1), (8, 200, 2)])
def test_page_calls_follow_the_rules(nq, dt, dim, heads, page, pages, seed):
    """A long random run of all calls: bookkeeping and every token equal to the model's after each."""
    from nspeech_b200.cache import PagedCache
    rng = np.random.default_rng(seed)
    slots, max_pages, layers = 12, 9, 2
    cache = PagedCache.create(layers, pages, page, heads, dim, slots, max_pages, DT[dt])
    m = Model(slots, pages, page, max_pages)
    token, refused = 0, 0
    for step in range(120):
        first = int(rng.integers(0, slots))
        n = int(rng.integers(1, slots - first + 1))
        kind = rng.choice(["grow", "grow", "grow", "fork", "fork", "free", "trim", "compact"])
        if kind == "grow":
            counts = [int(c) for c in rng.choice([0, 1, 1, 2, page, page + 3, 25], n)]
            got = m.reserve(first, counts)
            off = offsets(counts)
            cache.reserve(off, first)
            new = [float(token + i) % 97 for i in range(sum(counts))]
            token += len(new)
            t = torch.tensor(new, device="cuda").view(-1, 1, 1) + torch.arange(layers, device="cuda").view(-1, 1, 1, 1) * 100
            t = t.expand(layers, len(new), heads, dim).to(DT[dt]).contiguous()
            cache.write(t, -t, off, first)
            if got:
                refused += 1
                with pytest.raises(nq.NqError) as e:
                    cache.check()
                assert e.value.code == nq.NQ_ERR_CACHE
            else:
                m.write(first, counts, new)
        elif kind == "fork":
            src = [int(s) for s in rng.integers(-1 if rng.random() < 0.2 else 0, slots, n)]
            m.fork(first, src)
            cache.fork(torch.tensor(src, dtype=torch.int32, device="cuda"), first)
        elif kind == "free":
            m.fork(first, [-1] * n)
            cache.free(first, n)
        elif kind == "trim":
            sinks, window = int(rng.integers(0, 10)), int(rng.integers(0, 30))
            m.trim(first, n, sinks, window)
            cache.trim(window, sinks, first, n)
        else:
            live = m.compact()
            cache.compact()
            assert int(cache.live) == live
        cache.check()
        same_as(cache, m, layers)
    assert refused or pages == 200


def test_cache_refuses_without_changing_anything(nq):
    from nspeech_b200.cache import PagedCache
    cache = PagedCache.create(1, 6, 8, 1, 8, 4, 3)
    cache.reserve(9, 0, 2)  # four pages
    cache.check()
    before = [t.clone() for t in (cache.table, cache.lens, cache.refs)]

    def refused(bit, call):
        call()
        cache.reserve(1, 0, 1)  # does nothing before the status is read
        cache.free()
        cache.compact()
        cache.trim(0)
        with pytest.raises(nq.NqError) as e:
            cache.check()
        assert e.value.code == nq.NQ_ERR_CACHE and hex(bit) in str(e.value)
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.table, cache.lens, cache.refs)))
        cache.check()

    refused(nq.NQ_CACHE_OUT_OF_PAGES, lambda: cache.reserve(9, 2, 2))
    refused(nq.NQ_CACHE_SLOT_FULL, lambda: cache.reserve(16, 0, 1))
    refused(nq.NQ_CACHE_SLOT_FULL, lambda: cache.reserve(1 << 30, 0, 4))
    bad = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    refused(nq.NQ_CACHE_BAD_INDEX, lambda: cache.fork(bad, 1))
    refused(nq.NQ_CACHE_BAD_INDEX, lambda: cache.fork(bad - 2, 1))
    row = torch.ones((1, 1, 8), dtype=torch.bfloat16, device="cuda")
    refused(nq.NQ_CACHE_BAD_INDEX, lambda: cache.write(row, row, 1, 3, 1))  # slot 3 has no tokens
    cache.fork(torch.tensor([0], dtype=torch.int32, device="cuda"), 3)
    before = [t.clone() for t in (cache.table, cache.lens, cache.refs)]
    held = cache.k.clone()
    refused(nq.NQ_CACHE_SHARED_PAGE, lambda: cache.write(row, row, 1, 3, 1))
    assert torch.equal(held, cache.k)


def test_large_pool_and_many_slots():
    """Pages and slots past one block's reach: 70,000 pages, 3000 slots, against the model's rules in bulk."""
    from nspeech_b200.cache import PagedCache
    slots, pages = 3000, 70001
    cache = PagedCache.create(1, pages, 8, 1, 8, slots, 40)
    rng = np.random.default_rng(5)
    counts = rng.integers(0, 300, slots)
    cache.reserve(offsets(counts))
    cache.check()
    need = -(-counts // 8)
    at = np.concatenate([[0], np.cumsum(need)])
    want = np.full((slots, 40), -1)
    for i in range(slots):
        want[i, :need[i]] = np.arange(at[i], at[i + 1])
    assert np.array_equal(cache.table.cpu().numpy(), want)
    src = rng.integers(-1, slots, slots).astype(np.int32)
    cache.fork(torch.from_numpy(src).cuda())
    cache.check()
    want = np.where(src[:, None] >= 0, want[src], -1)
    refs = np.bincount(want[want >= 0], minlength=pages)
    assert np.array_equal(cache.table.cpu().numpy(), want)
    assert np.array_equal(cache.refs.cpu().numpy(), refs)
    cache.compact()
    cache.check()
    live = int((refs > 0).sum())
    assert int(cache.live) == live
    to = np.arange(pages)
    to[live + np.flatnonzero(refs[live:])] = np.flatnonzero(refs[:live] == 0)
    assert np.array_equal(cache.table.cpu().numpy(), np.where(want >= 0, to[want], -1))
    assert int((cache.refs[:live] > 0).sum()) == live and int(cache.refs[live:].sum()) == 0


# -------------------------------------------------------------------------------------------------------------- beams
def beam64(logits, scores, finished, eos):
    """[(score, beam, token)] best first: by score, then beam, then (within a beam) logit and token."""
    found = []
    for b in range(logits.shape[0]):
        base = scores[b] if not np.isnan(scores[b]) else -np.inf
        if finished[b]:
            found.append((base, b, eos))
            continue
        x = np.where(np.isnan(logits[b]) | (logits[b] == np.inf), -np.inf, logits[b]).astype(np.float64)
        top = x.max()
        lse = top + np.log(np.exp(x - top).sum()) if top > -np.inf else 0.0
        order = np.argsort(-x, kind="stable")[:logits.shape[0]]
        found += [(base + (x[t] - lse) if x[t] > -np.inf else -np.inf, b, int(t)) for t in order]
    return sorted(found, key=lambda c: (-c[0], c[1]))[:logits.shape[0]]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("items,beams,vocab", [(1, 1, 1), (1, 4, 3), (3, 4, 32768), (2, 32, 4097), (5, 7, 1000), (2, 32, 33),
                                              (1, 5, 200003), (9, 2, 8192), (40, 8, 5000)])
def test_beam_select(dt, items, beams, vocab):
    from nspeech_b200.beam import beam_select
    rng = np.random.default_rng(vocab + beams)
    logits = torch.from_numpy(rng.standard_normal((items, beams, vocab)).astype(np.float32) * 3).to(DT[dt])
    scores = torch.from_numpy(-rng.random((items, beams)).astype(np.float32) * 8)
    finished = torch.from_numpy(rng.random((items, beams)) < 0.2)
    eos = min(vocab - 1, 2)
    got = [t.cpu() for t in beam_select(logits.cuda(), scores.cuda(), finished.cuda(), eos)]
    for i in range(items):
        want = beam64(logits[i].float().numpy(), scores[i].numpy(), finished[i].numpy(), eos)
        assert got[1][i].tolist() == [i * beams + b for _, b, _ in want]
        assert got[2][i].tolist() == [t for _, _, t in want]
        assert got[3][i].tolist() == [bool(finished[i, b]) or t == eos for _, b, t in want]
        # the row's sum: terms of 2^-23 in f32, summed 16 at a time; then one rounding
        s = np.array([w[0] for w in want])
        assert np.all(np.abs(got[0][i].numpy() - s) <= np.abs(s) * 2.0 ** -24 + 2.0 ** -19)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("beams", [1, 3, 32])
@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "banned", "few", "odd", "first step", "all finished", "zeros"])
def test_beam_select_ties_and_masks(dt, beams, kind):
    from nspeech_b200.beam import beam_select
    vocab, eos = 9001, 5
    rng = np.random.default_rng(7)
    x = np.zeros((1, beams, vocab), np.float32)
    scores, finished = np.zeros((1, beams), np.float32), np.zeros((1, beams), bool)
    if kind in ("ascending", "descending"):
        x[:] = np.arange(vocab) * (1 / 64 if kind == "ascending" else -1 / 64)
    elif kind == "banned":
        x[:] = -np.inf
    elif kind == "few":
        x[:] = rng.choice([-np.inf, torch.finfo(torch.bfloat16).min], x.shape)
        x[0, :, 77] = 1.0
    elif kind == "odd":
        x[:] = rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0], x.shape)
    elif kind == "first step":
        x[:] = rng.integers(-3, 3, (1, 1, vocab))
        scores[:, 1:] = -np.inf
    elif kind == "all finished":
        finished[:] = True
        scores[:] = -rng.integers(0, 3, scores.shape)
    elif kind == "zeros":
        x[:] = rng.choice([0.0, -0.0], x.shape)
    lt = torch.from_numpy(x).to(DT[dt])
    got = [t.cpu() for t in beam_select(lt.cuda(), torch.from_numpy(scores).cuda(), torch.from_numpy(finished).cuda(), eos)]
    want = beam64(lt[0].float().numpy(), scores[0], finished[0], eos)
    assert got[1][0].tolist() == [b for _, b, _ in want]
    assert got[2][0].tolist() == [t for _, _, t in want]
    s = np.array([w[0] for w in want])
    same = np.isinf(s) & (got[0][0].numpy() == s)
    with np.errstate(invalid="ignore"):
        assert np.all(same | (np.abs(got[0][0].numpy() - s) <= np.abs(s) * 2.0 ** -24 + 2.0 ** -19))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("beams", [1, 2, 8, 32])
def test_beam_select_over_many_rounds(dt, beams):
    """Rows of several rounds a CTA where the best come early, late, scattered or in runs of equal values."""
    from nspeech_b200.beam import beam_select
    vocab, rng = 150001, np.random.default_rng(3)
    rows = [np.linspace(5, -5, vocab), np.linspace(-5, 5, vocab), np.sin(np.arange(vocab) * 0.37) * 6, np.repeat(rng.standard_normal(151), 1000)[:vocab],
            np.where(np.arange(vocab) % 4096 == 5, 3.0, -1.0), np.where(np.arange(vocab) > 140000, 0.5, 0.25), rng.standard_normal(vocab) * 4]
    x = np.stack([rows[(b * 5 + i) % len(rows)] for i in range(3) for b in range(beams)]).reshape(3, beams, vocab).astype(np.float32)
    x[:, :, 70000:90000:7] = -np.inf
    lt = torch.from_numpy(x).to(DT[dt])
    scores = -np.arange(3 * beams, dtype=np.float32).reshape(3, beams) / 64
    got = [t.cpu() for t in beam_select(lt.cuda(), torch.from_numpy(scores).cuda())]
    for i in range(3):
        want = beam64(lt[i].float().numpy(), scores[i], np.zeros(beams, bool), -1)
        assert got[1][i].tolist() == [i * beams + b for _, b, _ in want]
        assert got[2][i].tolist() == [t for _, _, t in want]


def test_beam_select_strided_rows_and_outputs_in_place():
    from nspeech_b200.beam import beam_select
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn((3, 4, 1003), generator=g, device="cuda")
    logits = wide[:, :, 2:1002]  # rows 1003 apart, on no 16-byte boundary
    scores = -torch.rand((3, 4), generator=g, device="cuda")
    finished = torch.zeros((3, 4), dtype=torch.bool, device="cuda")
    finished[1, 2] = True
    want = beam_select(logits.contiguous(), scores, finished, 1)
    got = beam_select(logits, scores, finished, 1, out=(scores, torch.empty_like(want[1]), torch.empty_like(want[2]), finished))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("rows", [1, 4, 65, 2500])
def test_beam_reorder(rows):
    from nspeech_b200.beam import beam_reorder
    g = torch.Generator(device="cuda").manual_seed(rows)
    parents = torch.randint(0, rows, (rows,), generator=g, device="cuda", dtype=torch.int32)
    for shapes, dtype in ([((640,), (2, 320), (1,)), torch.float32], [((7,), (3, 5)), torch.bfloat16], [((13,),), torch.uint8],
                          [((), (9,)), torch.int64], [((4100,),) * 18, torch.bfloat16]):
        states = [torch.randint(0, 100, (rows, *s), generator=g, device="cuda").to(dtype) for s in shapes]
        want = [t[parents.long()] for t in states]
        assert all(torch.equal(a, b) for a, b in zip(beam_reorder(states, parents), want))
        beam_reorder(states, parents, out=states)
        assert all(torch.equal(a, b) for a, b in zip(states, want))
    state = torch.arange(rows, device="cuda")
    assert torch.equal(beam_reorder([state], parents * 0 - 1)[0], state)  # out of range: the row stays


def test_beam_reorder_of_columns_and_of_the_same_state_twice():
    from nspeech_b200.beam import beam_reorder
    from nspeech_b200.fast_matmul import MatMulError
    from nspeech_b200.lib import NqError
    parents = torch.tensor([2, 0, 0, 1], dtype=torch.int32, device="cuda")
    whole = torch.arange(4 * 96, device="cuda").view(4, 96)
    want = whole[parents.long()]
    twice = beam_reorder([whole, whole], parents)  # read twice, written once each
    assert torch.equal(twice[0], want) and torch.equal(twice[1], want)
    columns = [whole[:, :32], whole[:, 32:40], whole[:, 40:]]
    beam_reorder(columns, parents, out=columns)
    assert torch.equal(whole, want)
    with pytest.raises(NqError, match="overlap"):
        beam_reorder([whole, whole], parents, out=[whole, whole])
    many = [whole.clone() for _ in range(17)] + [whole]
    with pytest.raises(MatMulError, match="overlap"):
        beam_reorder(many, parents, out=many[:17] + [many[0]])
    assert torch.equal(whole, want)


# ------------------------------------------------------------------------------------------------ a decoder, end to end
class Decoder:
    """One attention layer, an output projection and a lm_head on Q8_0-path weights (kept at bf16 precision, f32
    activations), embeddings by token and position."""

    def __init__(self, vocab=199, heads=2, kv=1, dim=32, width=64):
        from nspeech_b200.fast_matmul import QWeight
        g = torch.Generator().manual_seed(11)
        self.heads, self.kv, self.dim, self.width = heads, kv, dim, width
        mats = {"qkv": ((heads + 2 * kv) * dim, width, 0.3), "o": (width, heads * dim, 0.3), "head": (vocab, width, 0.5)}
        self.w = {n: (torch.randn((a, b), generator=g) * s).to(torch.bfloat16).float() for n, (a, b, s) in mats.items()}
        self.q = {n: QWeight.from_f32(t.numpy()) for n, t in self.w.items()}
        self.embed = torch.randn((vocab, width), generator=g)
        self.place = torch.randn((64, width), generator=g) * 0.5
        self.embed_dev, self.place_dev = self.embed.cuda(), self.place.cuda()

    def step(self, cache, tokens, pos, n, left, sinks):
        x = self.embed_dev[tokens] + self.place_dev[pos]
        qkv = self.q["qkv"].linear(x).view(n, -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv, self.kv], 1)
        cache.reserve(1, 0, n)
        cache.write(k, v, 1, 0, n)
        a = cache.attention(q, 0, first=0, n=n, left=left, sinks=sinks)
        y = self.q["o"].linear(a.reshape(n, -1)) + x
        return self.q["head"].linear(y)

    def log_probs64(self, history, left, sinks):
        """Log probabilities after a history of tokens, recomputed from its start."""
        w = {n: t.double() for n, t in self.w.items()}
        x = self.embed.double()[history] + self.place.double()[:len(history)]
        q, k, v = (x @ w["qkv"].T).view(len(history), -1, self.dim).split([self.heads, self.kv, self.kv], 1)
        a, _ = attention64(q[-1:], k, v, left, 0, sinks)
        y = a.reshape(1, -1) @ w["o"].T + x[-1:]
        return torch.log_softmax(y @ w["head"].T, 1)[0]


def test_beam_search_over_the_cache_and_its_graph():
    """Two utterances of four beams: at every step the chosen candidates' scores, recomputed in 64 bits from each beam's
    history of tokens alone, are the best there are; and a captured step replayed gives the eager run's results."""
    from nspeech_b200.beam import beam_reorder, beam_select
    from nspeech_b200.cache import PagedCache
    items, beams, steps, left, sinks, eos = 2, 4, 21, 9, 2, 0
    n, dec = items * beams, Decoder()

    def begin():
        cache = PagedCache.create(1, 40, 8, dec.kv, dec.dim, n, 5, torch.float32)
        s = dict(tokens=torch.tensor([3] * beams + [17] * beams, device="cuda"), pos=torch.zeros(1, dtype=torch.long, device="cuda"),
                 scores=torch.tensor([[0.0] + [-float("inf")] * (beams - 1)] * items, device="cuda"),
                 finished=torch.zeros((items, beams), dtype=torch.bool, device="cuda"),
                 history=torch.zeros((n, steps + 1), dtype=torch.int32, device="cuda"), parents=None)
        s["history"][:, 0] = s["tokens"]
        return cache, s

    def one(cache, s):
        logits = dec.step(cache, s["tokens"], s["pos"], n, left, sinks).view(items, beams, -1)
        scores, parents, tokens, finished = beam_select(logits, s["scores"], s["finished"], eos)
        cache.fork(parents.view(-1))
        cache.trim(left, sinks)
        beam_reorder([s["history"]], parents, out=[s["history"]])
        s["pos"] += 1
        s["history"].scatter_(1, s["pos"].expand(n, 1), tokens.view(n, 1))
        s["tokens"].copy_(tokens.view(-1))
        s["scores"].copy_(scores)
        s["finished"].copy_(finished)
        return parents

    cache, s = begin()
    trail = []
    for t in range(steps):
        old = s["scores"].cpu().double(), s["finished"].cpu(), s["history"][:, :t + 1].cpu().long()
        one(cache, s)
        trail.append((s["scores"].clone(), s["history"].clone()))
        new = s["scores"].cpu().double()
        for i in range(items):
            every = []
            for b in range(beams):
                if old[1][i, b]:
                    every.append(old[0][i, b].view(1))
                elif old[0][i, b] > -np.inf:
                    every.append(old[0][i, b] + dec.log_probs64(old[2][i * beams + b], left, sinks))
            best = torch.cat(every).sort(descending=True).values[:beams]
            # f32 activations through two projections of bf16 hi + lo planes: 2^-16 of terms of about 10 in sum
            assert bool(((new[i] - best).abs() < 2e-3).all())
    cache.check()
    # the same from a captured step
    graph_cache, g = begin()
    one(graph_cache, g)
    first = {k: g[k].clone() for k in ("tokens", "pos", "scores", "finished", "history")}
    keep = [x.clone() for x in (graph_cache.k, graph_cache.v, graph_cache.table, graph_cache.lens, graph_cache.refs, graph_cache.state)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(graph_cache, g)  # this stream's workspaces
    torch.cuda.synchronize()
    for k, x in first.items():
        g[k].copy_(x)
    for x, y in zip((graph_cache.k, graph_cache.v, graph_cache.table, graph_cache.lens, graph_cache.refs, graph_cache.state), keep):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one(graph_cache, g)
    for t in range(1, steps):
        graph.replay()
        assert torch.equal(g["scores"], trail[t][0]) and torch.equal(g["history"], trail[t][1])
    graph_cache.check()
    assert torch.equal(cache.table, graph_cache.table) and torch.equal(cache.refs, graph_cache.refs)


def test_scales_below_the_normal_numbers():
    from nspeech_b200.attention import window_attention
    g = torch.Generator().manual_seed(8)
    for dt in ("f32", "bf16"):
        q, k, v = (torch.randn((150, 2, 64), generator=g).to(DT[dt]) for _ in range(3))
        got = window_attention(q.cuda(), k.cuda(), v.cuda(), 40, 0, 2, scale=1e-40)
        check_rows(got, *attention64(q, k, v, 40, 0, 2, 1e-40))


def test_the_first_call_of_a_process_may_be_captured():
    program = """
import torch
from nspeech_b200.attention import window_attention
from nspeech_b200.beam import beam_select
torch.manual_seed(0)
q, x = torch.randn(300, 4, 64, device="cuda").bfloat16(), torch.randn(2, 3, 1000, device="cuda")
scores = torch.zeros(2, 3, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a, b = window_attention(q, q, q, 20, 0), beam_select(x, scores)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(a, window_attention(q, q, q, 20, 0))
assert all(torch.equal(s, t) for s, t in zip(b, beam_select(x, scores)))
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=300)
    assert "captured" in r.stdout, r.stderr[-2000:]


def test_calls_on_another_stream():
    from nspeech_b200.attention import window_attention
    from nspeech_b200.beam import beam_select
    side = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((n, 2, 64), generator=g, device="cuda", dtype=torch.bfloat16) for n in (2, 4000, 4000))
    logits, scores = torch.randn((4, 4, 30000), generator=g, device="cuda"), torch.zeros((4, 4), device="cuda")
    want = window_attention(q, k, v, right=0), beam_select(logits, scores)
    torch.cuda.synchronize()
    for _ in range(20):
        got = window_attention(q, k, v, right=0, stream=side), beam_select(logits, scores, stream=side)
        torch.empty(1 << 20, device="cuda").fill_(1.0)  # would take a workspace that was given back too early
    side.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
