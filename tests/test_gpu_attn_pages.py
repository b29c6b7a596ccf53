"""attn_pages on the GPU against its definition (pages_ref.attend), within a bound
derived from its sums, and the paged cache's operators together as a server uses
them."""
import math
import random

import numpy as np
import pytest
import torch

import pages_ref as P

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def pool(pages, page, kv, hd, seed, scale=0.02):
    """K and V of blocks with codes of all sizes; the last page's scales are NaN."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for by in (scale, 0.5 * scale):
        codes = (40 * torch.randn(pages, kv, page, hd, generator=g)).round().clamp(-127, 127).to(torch.int8)
        d = by * (0.5 + torch.rand(pages, kv, generator=g))
        d[-1] = float("nan")
        out.append(P.Pool(codes, d))
    return out


def cache_of(gpu, ref):
    k, v = ref
    return gpu.PagedCache(torch.from_numpy(k.codes).cuda(), torch.from_numpy(v.codes).cuda().transpose(2, 3).contiguous(),
                          torch.from_numpy(k.scale).cuda(), torch.from_numpy(v.scale).cuda())


def hide(table, length, count, page, window, sinks, pages, seed):
    """The table with entries that no query needs replaced: pages of the pool whose
    scales are NaN, and numbers outside it."""
    rng = random.Random(seed)
    table = table.clone()
    for b in range(table.shape[0]):
        ln = min(max(length[b], 0), table.shape[1] * page)
        first = ln - min(max(count[b], 0), ln)
        for i in range(table.shape[1]):
            lo, hi = i * page, (i + 1) * page
            if lo >= ln or (window and hi <= first - window + 1 and lo >= sinks) or count[b] <= 0:
                table[b, i] = rng.choice([pages - 1, -1, pages, 2 ** 31 - 1, -2 ** 31])
    return table


def agree(got, y, bound):
    live = ~torch.isnan(bound)
    assert (got[~live] == 9.25).all()
    assert torch.equal(torch.isnan(got[live]), torch.isnan(y[live]))
    ok = live & ~torch.isnan(y)
    err = (got[ok] - y[ok]).abs()
    assert (err <= bound[ok]).all(), (float((err / bound[ok].clamp_min(1e-300)).max()), float(err.max()))


def check(gpu, ref, q, table, length, count=None, window=0, sinks=0, scale=None):
    n, t, heads, hd = q.shape
    page, pages = ref[0].page, len(ref[0].codes)
    cnt = [t] * n if count is None else count
    scale = hd ** -0.5 if scale is None else scale
    y, bound = P.attend(q, *ref, table, length, cnt, scale, window, sinks)
    out = torch.full(q.shape, 9.25, device="cuda")
    cache = cache_of(gpu, ref)
    shown = hide(table, length, [min(max(c, 0), t) for c in cnt], page, window, sinks, pages, n * t)
    gpu.attn_pages(q.cuda(), cache, shown.cuda(), ints(*length), None if count is None else ints(*count), scale=scale,
                   window=window, sinks=sinks, out=out)
    agree(out.cpu().double(), y, bound)
    return out


def tables(n, most, pages, seed):
    """Pages of the pool but the last, in any order; some stand in two tables."""
    g = torch.Generator().manual_seed(seed)
    every = torch.cat([torch.randperm(pages - 1, generator=g) for _ in range(-(-n * most // (pages - 1)))])
    return every[:n * most].view(n, most).to(I32)


@pytest.mark.parametrize("heads,kv,hd", [(16, 8, 128), (4, 4, 64), (7, 1, 80), (16, 1, 96), (12, 3, 16), (2, 1, 256), (6, 2, 208), (5, 5, 192),
                                         (3, 1, 48), (4, 2, 112)])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_decoding(gpu, page, heads, kv, hd):
    length = [1, 0, page, page + 1, 64, 65, 700, 15, 3 * page - 1, 300]
    n, most = len(length), -(-700 // page) + 1
    ref = pool(n * most // 2 + 2, page, kv, hd, hd)
    q = torch.randn(n, 1, heads, hd, generator=torch.Generator().manual_seed(1)) * 1.5
    table = tables(n, most, len(ref[0].codes), 2)
    check(gpu, ref, q, table, length)
    check(gpu, ref, q, table, length, window=37, sinks=4)


@pytest.mark.parametrize("page,t,heads,kv,hd", [(16, 2, 16, 8, 128), (64, 5, 6, 2, 64), (32, 16, 3, 3, 80), (128, 3, 10, 2, 128), (16, 7, 2, 1, 256)])
def test_a_few_positions(gpu, page, t, heads, kv, hd):
    length = [t, t - 1, 1, 333, 64 + t, 0, 129, 257]
    count = [t, t, 1, t - 1, t, t, 0, -3]
    n, most = len(length), -(-333 // page)
    ref = pool(n * most + 1, page, kv, hd, hd)
    q = torch.randn(n, t, heads, hd, generator=torch.Generator().manual_seed(1)) * 1.5
    table = tables(n, most, len(ref[0].codes), 2)
    check(gpu, ref, q, table, length, count)
    check(gpu, ref, q, table, [333, 90, 64, 65, 128, 63, 200, 127], window=1, sinks=0)
    check(gpu, ref, q, table, [333, 90, 64, 65, 128, 63, 200, 127], count, window=70, sinks=66)


@pytest.mark.parametrize("page,t,heads,kv,hd", [(16, 17, 4, 4, 64), (64, 100, 16, 8, 128), (32, 130, 7, 1, 80), (128, 257, 3, 3, 96), (256, 64, 2, 1, 256),
                                                (16, 300, 2, 2, 16), (64, 70, 6, 2, 208), (32, 90, 5, 5, 48), (64, 65, 4, 1, 144), (16, 33, 6, 3, 176),
                                                (64, 200, 2, 1, 112)])
def test_prompts(gpu, page, t, heads, kv, hd):
    length = [t, t + 1, t + 150, t - 1, 1, 0, t + 64]
    count = [t, t - 3, t, t, 1, 5, 0]
    n, most = len(length), -(-(t + 150) // page)
    ref = pool(n * most + 1, page, kv, hd, hd)
    q = torch.randn(n, t, heads, hd, generator=torch.Generator().manual_seed(1)) * 1.5
    table = tables(n, most, len(ref[0].codes), 2)
    check(gpu, ref, q, table, length)
    check(gpu, ref, q, table, length, count)
    check(gpu, ref, q, table, length, count, window=50, sinks=3)


@pytest.mark.parametrize("heads,kv,hd", [(40, 2, 64), (33, 1, 128), (64, 2, 80), (17, 1, 256)])
def test_one_position_of_many_query_heads(gpu, heads, kv, hd):
    """More than sixteen query heads of a kv head: decoding by the kernel for prompts."""
    page, length = 32, [1, 0, 700, 64, 333]
    ref = pool(60, page, kv, hd, hd)
    table = tables(5, 22, 60, 2)
    q = torch.randn(5, 1, heads, hd, generator=torch.Generator().manual_seed(1)) * 1.5
    check(gpu, ref, q, table, length)
    check(gpu, ref, q, table, length, window=50, sinks=3)


def test_long_caches(gpu):
    """Streams whose parts are joined: more than a chunk a wave, and parts of heads
    that begin and end inside a workgroup's stretch."""
    page, heads, kv, hd = 32, 4, 2, 64
    length = [9000, 1, 5000, 64, 8191]
    ref = pool(600, page, kv, hd, 3)
    table = tables(5, 282, 600, 2)
    q = torch.randn(5, 1, heads, hd, generator=torch.Generator().manual_seed(1))
    check(gpu, ref, q, table, length)
    for length in ([9000], [4097]):
        check(gpu, ref, q[:1], table[:1], length)
    check(gpu, ref, q[:1], table[:1], [9000], window=2000, sinks=100)
    q = torch.randn(1, 40, heads, hd, generator=torch.Generator().manual_seed(1))
    check(gpu, ref, q, table[:1], [9000])


@pytest.mark.parametrize("t", [1, 40])
def test_blocks_and_pages_that_are_not_there(gpu, t):
    """A query that sees a row of such a block is NaN, of that kv head; no other is."""
    page, heads, kv, hd, most = 16, 4, 2, 64, 12
    ref = pool(40, page, kv, hd, 5)
    ref[0].scale[3, 1], ref[1].scale[4, 0], ref[1].scale[5, 1] = np.nan, np.inf, -1.0
    table = torch.tensor([[0, 1, 2, 6, 7, 8, 9, 10, 11, 12, 13, 14], [0, 3, 2, 6, 7, 8, 9, 10, 11, 12, 13, 14],
                          [0, 1, 2, 6, 7, 8, 9, 10, 4, 12, 13, 14], [0, 1, 2, 6, 7, 8, 9, 10, 11, 12, 13, 5],
                          [0, 1, 2, -1, 7, 8, 9, 10, 11, 12, 13, 14], [0, 1, 2, 6, 7, 8, 9, 10, 11, 12, 40, 14]], dtype=I32)
    q = torch.randn(6, t, heads, hd, generator=torch.Generator().manual_seed(1))
    for window, sinks in ((0, 0), (20, 0), (20, 50), (140, 0)):
        check(gpu, ref, q, table, [190, 190, 190, 170, 190, 175], window=window, sinks=sinks)
    q[0, 0, 1, 3], q[1, t - 1, 2, 5], q[2, 0, 0, 0] = float("inf"), float("nan"), float("-inf")
    check(gpu, ref, q, table, [190, 30, 100, 0, 17, 60])


@pytest.mark.parametrize("t", [1, 40])
def test_blocks_of_all_sizes(gpu, t):
    """Scales from 1e-30 to 1e30 beside each other, zero and denormal ones: what a
    block has does not cost others their bits, least of all one that is not seen."""
    page, heads, kv, hd = 16, 4, 2, 64
    ref = pool(26, page, kv, hd, 5)
    g = torch.Generator().manual_seed(8)
    q = torch.randn(3, t, heads, hd, generator=g)
    table = tables(3, 8, 26, 2)
    for side in (0, 1):
        keep = ref[side].scale.copy()
        for pattern in ([1e-30, 1.0, 1e30], [0.0, 1e-3], [1e-42, 1e-38], [1e30, 1e36], [0.0], [-0.0, 1e-20, 1e10]):
            if side == 0:  # (scores stay within f32's range)
                pattern = [min(x, 1e4) for x in pattern]
            for i in range(25):
                ref[side].scale[i] = pattern[i % len(pattern)]
            check(gpu, ref, q, table, [128, 100, 50])
            check(gpu, ref, q, table, [128, 127, 70], window=30, sinks=2)
        ref[side].scale[:] = keep


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("of", [0.0, 1.0])
def test_small_values_of_split_heads(gpu, t, of):
    """V's scales far below 1 over rows of like scores, whose weights' sum is large: the
    result is an ordinary number, also where parts of the rows are joined."""
    page, heads, kv, hd = 32, 4, 2, 64
    ref = pool(300, page, kv, hd, 5)
    table = tables(3, 282, 300, 2)
    q = of * torch.randn(3, t, heads, hd, generator=torch.Generator().manual_seed(8))
    keep = ref[1].scale.copy()
    for by in (1e-20, 1e-26, 1e-28, 1e-30, 1e-33):
        ref[1].scale[:] = keep * np.float32(by)
        check(gpu, ref, q, table, [9000, 700, 4100])
        check(gpu, ref, q[:1], table[:1], [9000], window=3000, sinks=70)


@pytest.mark.parametrize("t", [1, 40])
def test_queries_of_all_sizes(gpu, t):
    """Zero queries, tiny ones, ones with a value far above the others, and scores past 2^23."""
    page, heads, kv, hd = 32, 4, 2, 128
    ref = pool(26, page, kv, hd, 5)
    table = tables(2, 8, 26, 2)
    g = torch.Generator().manual_seed(8)
    for by in (0.0, 1e-30, 1e-42, 1e3, 1e6, 1e9):
        q = torch.randn(2, t, heads, hd, generator=g) * by
        check(gpu, ref, q, table, [256, 100])
    q = torch.randn(2, t, heads, hd, generator=g)
    q[..., 7] *= 1e5
    for side in (0, 1):
        ref[side].codes[..., 7] = 0
    check(gpu, ref, q, table, [256, 100])
    check(gpu, ref, q, table, [256, 100], scale=-0.3)


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("length,window", [(300, 0), (9000, 0), (9000, 2500)])
@pytest.mark.parametrize("power", [5, 13, 14, 15, 16])
def test_large_scores_are_exact(gpu, t, length, window, power):
    """Scores of 2^12 to 2^23 whose softmax is known: with a scale of ln 2 they are q.k
    in powers of two, here whole numbers below 2^24 and so exact in f32, weights powers
    of two. What is left: the pieces of weight times scale (2^-22 of itself, 2^-38 of the
    largest), the sum over the rows, and 32 half steps of factors and joins. Some rows
    have the largest code, a few steps apart by a second value; the others are at least
    2^power below."""
    page, heads, kv, hd, sinks = 32, 4, 2, 64, 40
    g = torch.Generator().manual_seed(power)
    ref = pool(300, page, kv, hd, 5)
    codes = torch.zeros(300, kv, page, hd, dtype=torch.int8)
    codes[..., 0] = torch.where(torch.rand(300, kv, page, generator=g) < 0.02, 127, torch.randint(-127, 127, (300, kv, page), generator=g)).to(torch.int8)
    codes[..., 1] = torch.randint(0, 6, (300, kv, page), generator=g)
    codes[..., 2:] = torch.randint(-127, 128, (300, kv, page, hd - 2), generator=g)     # (against zeros in q)
    ref[0].codes[:], ref[0].scale[:] = codes.numpy(), 1.0
    table = tables(1, 282, 300, 2)
    q = torch.zeros(1, t, heads, hd)
    q[..., 0], q[..., 1] = 2.0 ** power, 1.0
    got = gpu.attn_pages(q.cuda(), cache_of(gpu, ref), table.cuda(), ints(length), scale=math.log(2), window=window, sinks=sinks).cpu().double()
    k, v = (half.rows(table[0], length).double().transpose(0, 1) for half in ref)       # (kv, rows, hd)
    d = torch.from_numpy(ref[1].scale)[table[0].long()].double().repeat_interleave(page, 0)[:length].T
    s = k[..., 0] * 2.0 ** power + k[..., 1]
    j = torch.arange(length)
    for i in range(t):
        at = length - t + i
        seen = (j <= at) & ((j > at - window) | (j < sinks)) if window else j <= at
        w = torch.exp2((s - s[:, seen].max(1, keepdim=True).values).masked_fill(~seen, -math.inf))
        w = w / w.sum(1, keepdim=True)
        y, size = (torch.bmm(w[:, None], x)[:, 0].repeat_interleave(heads // kv, 0) for x in (v, v.abs()))
        lost = 2.0 ** -38 * (w * d).amax(1) * 127 * length
        bound = (2.0 ** -22 + (length + 32) * P.EPS) * size + lost.repeat_interleave(heads // kv)[:, None]
        err = (got[0, i] - y).abs()
        assert (err <= bound).all(), (i, float((err / bound).max()))


def test_one_large_weight_beside_many_small_ones(gpu):
    """A first row that takes nearly all the weight and is nothing in V: the result is
    made of the others' weights, 2^-30 of the largest each."""
    page, heads, kv, hd = 64, 2, 2, 64
    for t, by in ((1, 160.0), (40, 160.0)):
        ref = pool(34, page, kv, hd, 5)
        ref[0].codes[:] = 0
        ref[0].codes[0, :, 0, 0] = 127
        ref[0].scale[:] = 1.0 / 127
        ref[1].codes[0, :, 0] = 0
        q = torch.zeros(1, t, heads, hd)
        q[..., 0] = by
        table = torch.arange(32, dtype=I32)[None]
        check(gpu, ref, q, table, [2000])


def test_strided_tensors(gpu):
    """q cut from a fused projection, a y of head-major rows, a pool whose K and V lie
    side by side, tables within wider ones."""
    page, heads, kv, hd, n, pages = 32, 4, 2, 48, 2, 9
    for t in (1, 30):
        ref = pool(pages, page, kv, hd, 5)
        both = torch.full((pages, 2, kv + 1, page * hd), 77, dtype=torch.int8, device="cuda")
        k, v = both[:, 0, :kv].unflatten(-1, (page, hd)), both[:, 1, :kv].unflatten(-1, (hd, page))
        k.copy_(torch.from_numpy(ref[0].codes))
        v.copy_(torch.from_numpy(ref[1].codes).transpose(2, 3))
        scales = torch.zeros(pages, 3 * kv, device="cuda")
        ks, vs = scales[:, :kv], scales[:, 2 * kv:]
        ks.copy_(torch.from_numpy(ref[0].scale))
        vs.copy_(torch.from_numpy(ref[1].scale))
        table = tables(n, 4, pages, 2)
        wide = torch.full((n, 9), -1, dtype=I32, device="cuda")
        wide[:, 3:7] = table.cuda()
        fused = torch.randn(n, t, 3, heads, hd, generator=torch.Generator().manual_seed(1)).cuda()
        q = fused[:, :, 1]
        out = torch.full((n, heads, t, hd), 9.25, device="cuda").transpose(1, 2)
        gpu.attn_pages(q, gpu.PagedCache(k, v, ks, vs), wide[:, 3:7], ints(100, 77), out=out)
        agree(out.cpu().double(), *P.attend(q.cpu(), *ref, table, [100, 77], [t, t], hd ** -0.5))


def test_a_pool_past_4_gb(gpu):
    page, kv, hd, pages = 256, 8, 256, 8300                       # 512 KB of K a page
    few = pool(6, page, kv, hd, 5)
    cache = gpu.PagedCache(torch.zeros(pages, kv, page, hd, dtype=torch.int8, device="cuda"),
                           torch.zeros(pages, kv, hd, page, dtype=torch.int8, device="cuda"),
                           torch.zeros(pages, kv, device="cuda"), torch.zeros(pages, kv, device="cuda"))
    where = [8299, 4096, 8192, 1, 5000]
    for i, at in enumerate(where):
        cache.k[at], cache.v[at] = torch.from_numpy(few[0].codes[i]).cuda(), torch.from_numpy(few[1].codes[i]).cuda().transpose(1, 2)
        cache.k_scale[at], cache.v_scale[at] = torch.from_numpy(few[0].scale[i]).cuda(), torch.from_numpy(few[1].scale[i]).cuda()
    for t in (1, 20):
        q = torch.randn(1, t, 8, hd, generator=torch.Generator().manual_seed(1))
        out = torch.full(q.shape, 9.25, device="cuda")
        gpu.attn_pages(q.cuda(), cache, ints(*where)[None], ints(1200), out=out)
        agree(out.cpu().double(), *P.attend(q, *few, torch.arange(5, dtype=I32)[None], [1200], [t], hd ** -0.5))


def test_every_run_gives_the_same_bits(gpu):
    page, heads, kv, hd = 64, 16, 8, 128
    ref = pool(60, page, kv, hd, 5)
    cache = cache_of(gpu, ref)
    q = torch.randn(1, 1, heads, hd, device="cuda")
    table = tables(1, 20, 60, 2).cuda()
    first = gpu.attn_pages(q, cache, table, ints(1000))
    for _ in range(5):
        assert torch.equal(gpu.attn_pages(q, cache, table, ints(1000)), first)


def serve(gpu, S, n, steps, seed, act):
    """Requests that arrive with prompts, grow by a token a step and end, over pages
    that are given back and taken again: act(lengths, counts, k, v, q) makes a step."""
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    lengths = [0] * n
    for _ in range(steps):
        counts = []
        for b in range(n):
            kind = rng.random()
            if lengths[b] == 0 or kind < 0.1:
                new = rng.choice([0, rng.randrange(1, S["t"] + 1)])
                lengths[b] = 0
            else:
                new = 1 if lengths[b] < S["cap"] else 0
            lengths[b] += new
            counts.append(new)
        k, v = (torch.randn(n, S["t"], S["kv"], S["hd"], generator=g) for _ in range(2))
        q = torch.randn(n, S["t"], S["heads"], S["hd"], generator=g)
        act(list(lengths), counts, k, v, q)


SERVER = dict(t=37, cap=120, kv=2, hd=64, heads=4)


@pytest.mark.parametrize("captured", [False, True])
def test_serving(gpu, captured):
    """kv_pages, kv_store_pages, attn_pages and kv_load_pages step by step, eagerly
    and as one captured graph that serves every step."""
    S, n, page, pages = SERVER, 5, 16, 30
    most = -(-S["cap"] // page)
    tabs = P.Pages(n, most, pages)
    side = pool(pages + 1, page, S["kv"], S["hd"], 4)
    cache = cache_of(gpu, side)
    dev = dict(table=tabs.table().cuda(), held=tabs.held().cuda(), free=tabs.free().cuda(), left=tabs.left().cuda(),
               length=ints(*[0] * n), before=ints(*[0] * n), count=ints(*[0] * n), status=ints(0),
               k=torch.zeros(n, S["t"], S["kv"], S["hd"], device="cuda"), v=torch.zeros(n, S["t"], S["kv"], S["hd"], device="cuda"),
               q=torch.zeros(n, S["t"], S["heads"], S["hd"], device="cuda"), y=torch.zeros(n, S["t"], S["heads"], S["hd"], device="cuda"),
               slots=torch.zeros(n, S["cap"], dtype=I32, device="cuda"),
               rows=[torch.zeros(n, S["cap"], S["kv"], S["hd"], device="cuda") for _ in range(2)])
    need = gpu.attn_pages_work(dev["q"], cache, dev["table"])
    work = torch.empty(need, device="cuda") if need else None
    def step():
        # (requests that begin again give their old pages back first)
        gpu.kv_pages(dev["before"], page, dev["held"], dev["free"], dev["left"], dev["table"], dev["status"])
        gpu.kv_pages(dev["length"], page, dev["held"], dev["free"], dev["left"], dev["table"], dev["status"])
        gpu.kv_store_pages(dev["k"], dev["v"], cache, dev["table"], dev["length"], dev["count"], dev["status"])
        gpu.attn_pages(dev["q"], cache, dev["table"], dev["length"], dev["count"], out=dev["y"], work=work)
        gpu.kv_slots(dev["table"], dev["length"], page, S["cap"], dev["length"], out=dev["slots"])
        gpu.kv_load_pages(cache, dev["slots"], dev["rows"][0], dev["rows"][1])

    graph = None
    if captured:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()                                              # (nothing yet: all lengths are 0)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()

    def act(lengths, counts, k, v, q):
        before = [0 if c == x else x - c for x, c in zip(lengths, counts)]
        assert tabs.fit(before, page) and tabs.fit(lengths, page)
        for name, x in (("k", k), ("v", v), ("q", q)):
            dev[name].copy_(x)
        for name, x in (("before", before), ("length", lengths), ("count", counts)):
            dev[name].copy_(ints(*x))
        dev["y"].fill_(9.25)
        graph.replay() if captured else step()
        table = tabs.table()
        assert int(dev["status"]) == 0
        assert torch.equal(dev["table"].cpu(), table) and torch.equal(dev["held"].cpu(), tabs.held())
        for b in range(n):
            for half, x in zip(side, (k, v)):
                half.store(x[b, :counts[b]], table[b], lengths[b] - counts[b])
            for half, got in zip(side, dev["rows"]):
                assert torch.equal(got[b, :lengths[b]].cpu(), half.rows(table[b], lengths[b]))
        agree(dev["y"].cpu().double(), *P.attend(q, *side, table, lengths, counts, S["hd"] ** -0.5))

    serve(gpu, S, n, 25, 11, act)


@pytest.mark.parametrize("t", [1, 40])
def test_a_captured_call_of_split_heads_serves_all_lengths(gpu, t):
    """Lengths, counts and tables change between replays: heads that were whole are split
    and the other way round, over the workspace that the last replay left."""
    page, heads, kv, hd, n = 32, 4, 2, 64, 3
    ref = pool(300, page, kv, hd, 5)
    cache = cache_of(gpu, ref)
    table = tables(n, 282, 300, 2)
    q = torch.zeros(n, t, heads, hd, device="cuda")
    dev, length, count = table.cuda(), ints(*[0] * n), ints(*[0] * n)
    out = torch.zeros(q.shape, device="cuda")
    work = torch.full((gpu.attn_pages_work(q, cache, dev),), float("nan"), device="cuda")
    assert work.numel() > 0

    def call():
        gpu.attn_pages(q, cache, dev, length, count, out=out, work=work)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i, (ln, c) in enumerate([([9000, 1, 300], [t, 1, t]), ([64, 5000, 64], [t, 0, t]), ([0, 0, 9024], [1, 0, 1]), ([9000, 9000, 9000], [t, t, t])]):
        x = torch.randn(q.shape, generator=torch.Generator().manual_seed(i))
        q.copy_(x), length.copy_(ints(*ln)), count.copy_(ints(*c)), dev.copy_(table.roll(i, 1))
        out.fill_(9.25)
        graph.replay()
        got = out.cpu()
        agree(got.double(), *P.attend(x, *ref, table.roll(i, 1), ln, c, hd ** -0.5))
        out.fill_(9.25)
        call()
        assert torch.equal(out.cpu(), got)


def test_another_stream_than_the_current_tensors_were_made_on(gpu):
    page, heads, kv, hd = 32, 4, 2, 64
    ref = pool(26, page, kv, hd, 5)
    cache = cache_of(gpu, ref)
    table = tables(3, 8, 26, 2)
    streams = [torch.cuda.Stream() for _ in range(3)]
    q = [torch.randn(3, t, heads, hd, generator=torch.Generator().manual_seed(t)) for t in (1, 5, 60)]
    out = []
    for s, x in zip(streams, q):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out.append(gpu.attn_pages(x.cuda(), cache, table.cuda(), ints(200, 256, 77)))
    torch.cuda.synchronize()
    for x, y in zip(q, out):
        agree(y.cpu().double(), *P.attend(x, *ref, table, [200, 256, 77], [x.shape[1]] * 3, hd ** -0.5))
