"""kv_pages, kv_slots, kv_store_pages and kv_load_pages on the GPU against their
definitions (pages_ref.py): pages, slots, codes, scales and values exactly."""
import random

import numpy as np
import pytest
import torch

import pages_ref as P

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def bits(x):
    return x.contiguous().view(torch.uint8)


# ---------------------------------------------------------------------------
# kv_pages, kv_slots
# ---------------------------------------------------------------------------


class Device:
    def __init__(self, ref, wide=0):
        n, most = len(ref.rows), ref.most
        self.table = torch.full((n, most + wide), -1, dtype=I32, device="cuda")[:, :most]  # (rows further apart than long)
        self.table.copy_(ref.table())
        self.held, self.free, self.left = ref.held().cuda(), ref.free().cuda(), ref.left().cuda()

    def same(self, ref):
        assert torch.equal(self.table.cpu(), ref.table()) and torch.equal(self.held.cpu(), ref.held())
        assert torch.equal(self.left.cpu(), ref.left())
        k = len(ref.stack)
        assert torch.equal(self.free.cpu()[:k], ref.free()[:k])


@pytest.mark.parametrize("n,most,page,pages", [(1, 1, 16, 1), (1, 40, 16, 40), (5, 7, 32, 20), (64, 9, 16, 300), (1024, 4, 64, 2500),
                                               (1025, 70, 16, 30000), (3000, 30, 128, 60000), (5000, 3, 256, 9000), (2, 65536, 16, 131072)])
def test_tables_follow_lengths(gpu, n, most, page, pages):
    rng = random.Random(n * most)
    order = list(range(pages))
    rng.shuffle(order)
    ref = P.Pages(n, most, pages, order)
    dev = Device(ref, wide=3)
    lengths = [0] * n
    for step in range(6):
        before = list(lengths)
        for b in range(n):
            kind = rng.random()
            if kind < 0.2:
                lengths[b] = 0
            elif kind < 0.5:
                lengths[b] = rng.randrange(0, most * page + 1)
            elif kind < 0.9:
                lengths[b] = min(lengths[b] + 1, most * page)
        while not ref.fit(lengths, page):  # (too few pages: one that is refused, then fewer rows)
            status = ints(0)
            gpu.kv_pages(ints(*lengths), page, dev.held, dev.free, dev.left, dev.table, status)
            assert int(status) == 1
            dev.same(ref)
            lengths = [x // 2 for x in lengths]
        status = ints(0)
        gpu.kv_pages(ints(*lengths), page, dev.held, dev.free, dev.left, dev.table, status)
        assert int(status) == 0
        dev.same(ref)
        if step == 3:  # back, and as it was
            table, free = dev.table.clone(), dev.free.clone()
            if ref.fit(before, page):
                gpu.kv_pages(ints(*before), page, dev.held, dev.free, dev.left, dev.table)
                dev.same(ref)
                assert ref.fit(lengths, page)
                gpu.kv_pages(ints(*lengths), page, dev.held, dev.free, dev.left, dev.table)
                dev.same(ref)
                assert torch.equal(dev.table, table) and torch.equal(dev.free[:len(ref.stack)], free[:len(ref.stack)])


@pytest.mark.parametrize("most", [8, 40000])
def test_a_step_that_cannot_be_made_changes_nothing(gpu, most):
    ref = P.Pages(3, most, 12)
    assert ref.fit([100, 17, 0], 16)
    for lengths, held, left in (((-1, 17, 0), None, None), ((100, 17, most * 16 + 1), None, None), ((100, 2 ** 31 - 1, 0), None, None),
                                ((128, 64, 16), None, None), ((0, 0, 0), (7, most + 1, 0), None), ((0, 0, 0), (7, -1, 0), None),
                                ((0, 0, 0), None, 4), ((0, 0, 0), None, -1), ((0, 0, 0), None, 2 ** 31 - 1)):
        dev = Device(ref)
        if held is not None:
            dev.held = ints(*held)
        if left is not None:
            dev.left = ints(left)
        before = [x.clone() for x in (dev.table, dev.held, dev.free, dev.left)]
        status = ints(0)
        gpu.kv_pages(ints(*lengths), 16, dev.held, dev.free, dev.left, dev.table, status)
        assert int(status) == 1, (lengths, held, left)
        for x, y in zip((dev.table, dev.held, dev.free, dev.left), before):
            assert torch.equal(x, y), (lengths, held, left)


def test_slots(gpu):
    rng = random.Random(5)
    for n, most, page, t in ((1, 1, 16, 1), (7, 5, 32, 300), (65, 3, 16, 29), (3, 40, 128, 513)):
        table = torch.tensor([[rng.randrange(-1, 1000) for _ in range(most)] for _ in range(n)], dtype=I32)
        length = [rng.randrange(-3, most * page + 5) for _ in range(n)]
        count = [rng.randrange(-2, t + 3) for _ in range(n)]
        for c in (count, [t] * n):
            out = torch.full((n, t), 9, dtype=I32, device="cuda")
            got = gpu.kv_slots(table.cuda(), ints(*length), page, t, ints(*c) if c is count else None, out=out)
            assert torch.equal(got.cpu(), P.slots(table, length, c, page, t))
    far = torch.tensor([[2 ** 31 // 16 - 1, 2 ** 31 // 16, 2 ** 31 - 1]], dtype=I32)      # the last slot, and past it
    assert gpu.kv_slots(far.cuda(), ints(48), 16, 48).cpu().tolist()[0] == list(range(2 ** 31 - 16, 2 ** 31)) + [-1] * 32


# ---------------------------------------------------------------------------
# kv_store_pages, kv_load_pages
# ---------------------------------------------------------------------------


def pools(pages, page, kv, hd, seed, scale=0.02):
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(-127, 128, (pages, kv, page, hd), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [scale * torch.rand(pages, kv, generator=g) for _ in range(2)]
    return [P.Pool(c, s) for c, s in zip(codes, scales)]


def cache_of(gpu, ref):
    k, v = ref
    return gpu.PagedCache(torch.from_numpy(k.codes).cuda(), torch.from_numpy(v.codes).cuda().transpose(2, 3).contiguous(),
                          torch.from_numpy(k.scale).cuda(), torch.from_numpy(v.scale).cuda())


def same(cache, ref):
    k, v = ref
    assert torch.equal(bits(cache.k_scale.cpu()), bits(torch.from_numpy(k.scale)))
    assert torch.equal(bits(cache.v_scale.cpu()), bits(torch.from_numpy(v.scale)))
    assert torch.equal(cache.k.cpu(), torch.from_numpy(k.codes))
    assert torch.equal(cache.v.cpu().transpose(2, 3), torch.from_numpy(v.codes))


def edge_rows(shape, seed):
    """Rows of ordinary values, of one value, zeros, of either sign's extreme, tiny
    (denormal scales) and huge ones, and halves between codes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    f = x.reshape(-1, shape[-1])
    for i in range(f.shape[0]):
        kind = i % 11
        if kind == 1:
            f[i] = 0.0
        elif kind == 2:
            f[i] = -0.75
        elif kind == 3:
            f[i, 0] = -5.0
        elif kind == 5 and i % 3 == 0:
            f[i] *= 1e-41
        elif kind == 7 and i % 5 == 0:
            f[i] *= 3e4
        elif kind == 8:
            f[i] = torch.arange(shape[-1]).remainder(17) * 0.5 - 4.0
    return x


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv,hd,t", [(8, 128, 1), (2, 64, 5), (3, 80, 77), (1, 256, 300), (5, 16, 130), (4, 96, 261)])
def test_store_and_load_are_exact(gpu, page, kv, hd, t):
    n, most = 3, (t + 2 * page - 1) // page + 1
    pages = n * most + 2
    ref = pools(pages, page, kv, hd, 1)
    cache = cache_of(gpu, ref)
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(pages, generator=g)[:n * most].view(n, most).to(I32)
    count = [t, max(t // 2, 1), 0]
    start = [page - 1, 0, 3]
    x = [edge_rows((n, t, kv, hd), s) for s in (3, 4)]
    length = [s + c for s, c in zip(start, count)]
    status = ints(0)
    gpu.kv_store_pages(x[0].cuda(), x[1].cuda(), cache, table.cuda(), ints(*length), ints(*count), status)
    for side, xs in zip(ref, x):
        for b in range(n):
            side.store(xs[b, :count[b]], table[b], start[b])
    same(cache, ref)
    assert int(status) == 0
    slots = gpu.kv_slots(table.cuda(), ints(*length), page, t, ints(*length))
    out = [torch.full((n, t, kv, hd), 7.5, device="cuda") for _ in range(2)]
    gpu.kv_load_pages(cache, slots, out[0], out[1])
    for side, got in zip(ref, out):
        for b in range(n):
            c = min(length[b], t)
            want = side.rows(table[b], length[b])[length[b] - c:]
            assert torch.equal(bits(got[b, :c].cpu()), bits(want)) and (got[b, c:] == 7.5).all()


def test_rows_one_by_one_grow_a_block(gpu):
    """The codes in front follow the scale, token by token over two pages."""
    page, kv, hd = 16, 2, 64
    ref = pools(3, page, kv, hd, 1)
    cache = cache_of(gpu, ref)
    table = torch.tensor([[2, 0]], dtype=I32)
    g = torch.Generator().manual_seed(9)
    for r in range(20):
        x = [torch.randn(1, 1, kv, hd, generator=g) * (1.0 + r % 7) for _ in range(2)]
        gpu.kv_store_pages(x[0].cuda(), x[1].cuda(), cache, table.cuda(), ints(r + 1))
        for side, xs in zip(ref, x):
            side.store(xs[0], table[0], r)
        same(cache, ref)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_block_with_an_infinity_or_nan_is_nan_until_it_begins_again(gpu, value):
    page, kv, hd = 16, 2, 32
    ref = pools(2, page, kv, hd, 1)
    cache = cache_of(gpu, ref)
    table = torch.tensor([[1, 0]], dtype=I32)

    def put(x, start):
        gpu.kv_store_pages(x[None].cuda(), x[None].cuda(), cache, table.cuda(), ints(start + len(x)))
        for side in ref:
            side.store(x, table[0], start)
        same(cache, ref)
        slots = gpu.kv_slots(table.cuda(), ints(start + len(x)), page, start + len(x))
        got = gpu.kv_load_pages(cache, slots)[0].cpu()[0]
        return torch.isnan(got).all(-1), torch.isnan(got).any(-1)

    x = torch.randn(5, kv, hd)
    put(x, 0)
    bad = x.clone()
    bad[2, 1, 7] = value
    every, some = put(bad, 5)
    assert every[:, 1].all() and not some[:, 0].any()
    every, some = put(x, 10)                                   # its scale stays NaN behind such rows
    assert every[:, 1].all() and not some[:, 0].any()
    every, some = put(torch.randn(20, kv, hd), 0)
    assert not some.any()


def test_scales_that_no_block_has(gpu):
    """Not finite or negative: NaN, to loads and to rows stored behind."""
    page, kv, hd = 32, 5, 48
    ref = pools(2, page, kv, hd, 1)
    for side in ref:
        side.scale[1] = [-1.0, np.inf, np.nan, -np.inf, 0.5]
    cache = cache_of(gpu, ref)
    table = torch.tensor([[1]], dtype=I32)
    slots = gpu.kv_slots(table.cuda(), ints(3), page, 3)
    for got, side in zip(gpu.kv_load_pages(cache, slots), ref):
        assert torch.equal(torch.isnan(got.cpu()[0]).all(0).all(-1), torch.tensor([True, True, True, True, False]))
        assert torch.equal(got.cpu()[0, :, 4], side.rows(table[0], 3)[:, 4])
    x = torch.randn(1, 2, kv, hd)
    gpu.kv_store_pages(x.cuda(), x.cuda(), cache, table.cuda(), ints(5))
    for side in ref:
        side.store(x[0], table[0], 3)
    same(cache, ref)


def test_rows_that_do_not_fit_are_not_written(gpu):
    page, kv, hd, t = 16, 2, 32, 20
    ref = pools(9, page, kv, hd, 1)
    cache = cache_of(gpu, ref)
    #                     fits     bad page  bad, unused  past table  count     count    length   idle     low
    table = torch.tensor([[0, 1], [2, 9], [3, 9], [4, 5], [6, 7], [6, 7], [6, 7], [-1, -1], [-5, 8]], dtype=I32)
    length = [20, 20, 12, 33, 32, 32, 3, 2 ** 31 - 1, 20]
    count = [20, 10, 12, 20, 21, -1, 4, 0, 1]
    x = torch.randn(9, t, kv, hd)
    for rows, flag in (([0], 0), ([1], 1), ([2], 0), ([3], 1), ([4], 1), ([5], 1), ([6], 1), ([7], 0), ([8], 0)):
        status = ints(0)
        gpu.kv_store_pages(x[rows].cuda(), x[rows].cuda(), cache, table[rows].cuda(), ints(*[length[r] for r in rows]),
                           ints(*[count[r] for r in rows]), status)
        assert int(status) == flag, rows
        if flag == 0 and count[rows[0]] > 0:
            for side in ref:
                side.store(x[rows[0], :count[rows[0]]], table[rows[0]], length[rows[0]] - count[rows[0]])
        same(cache, ref)
    status = ints(0)
    gpu.kv_store_pages(x.cuda(), x.cuda(), cache, table.cuda(), ints(*length), ints(*count), status)
    assert int(status) == 1
    for b in (0, 2, 8):
        for side in ref:
            side.store(x[b, :count[b]], table[b], length[b] - count[b])
    same(cache, ref)


def test_loads_by_any_slots(gpu):
    page, kv, hd = 32, 3, 80
    ref = pools(6, page, kv, hd, 1)
    cache = cache_of(gpu, ref)
    rng = random.Random(3)
    slot = [[rng.choice([-1, -2, 6 * page, 2 ** 31 - 1, -2 ** 31, rng.randrange(6 * page), rng.randrange(6 * page)]) for _ in range(131)]
            for _ in range(2)]
    slots = torch.full((2, 140), 3, dtype=I32, device="cuda")[:, 4:135]
    slots.copy_(torch.tensor(slot, dtype=I32))
    out = [torch.full((2, 131, kv, hd), 7.5, device="cuda") for _ in range(2)]
    gpu.kv_load_pages(cache, slots, out[0], out[1])
    for got, side in zip(out, ref):
        v = side.values().transpose(1, 2).reshape(6 * page, kv, hd)
        for b in range(2):
            for t, s in enumerate(slot[b]):
                want = torch.full((kv, hd), 7.5) if s == -1 else v[s] if 0 <= s < 6 * page else torch.full((kv, hd), float("nan"))
                assert torch.equal(bits(got[b, t].cpu()), bits(want)) or (torch.isnan(want).all() and torch.isnan(got[b, t]).all())


def test_pools_and_rows_at_strides(gpu):
    """K and V of a page side by side in one buffer with room behind the heads,
    head-major rows, tables that are part of wider ones."""
    pages, page, kv, hd, n, t = 7, 32, 3, 48, 2, 40
    ref = pools(pages, page, kv, hd, 1)
    both = torch.full((pages, 2, kv + 1, page * hd), 77, dtype=torch.int8, device="cuda")
    k = both[:, 0, :kv].unflatten(-1, (page, hd))
    v = both[:, 1, :kv].unflatten(-1, (hd, page))
    scales = torch.full((pages, 3 * kv), 5.0, device="cuda")
    k.copy_(torch.from_numpy(ref[0].codes))
    v.copy_(torch.from_numpy(ref[1].codes).transpose(2, 3))
    ks, vs = scales[:, :kv], scales[:, 2 * kv:]
    ks.copy_(torch.from_numpy(ref[0].scale))
    vs.copy_(torch.from_numpy(ref[1].scale))
    cache = gpu.PagedCache(k, v, ks, vs)
    table = torch.full((n, 5), 1000, dtype=I32, device="cuda")[:, 1:4]
    table.copy_(torch.tensor([[6, 1, 2], [0, 5, 3]]))
    x = torch.randn(2, n, kv, t, hd)
    xd = x.cuda().transpose(2, 3)
    gpu.kv_store_pages(xd[0], xd[1], cache, table, ints(47, 40))
    for side, xs in zip(ref, x):
        for b, start in enumerate((7, 0)):
            side.store(xs[b].transpose(0, 1).contiguous(), table.cpu()[b], start)
    same(cache, ref)
    assert (both[:, :, kv] == 77).all() and (scales[:, kv:2 * kv] == 5.0).all()
    out = torch.full((2, n, kv, t, hd), 7.5, device="cuda").transpose(2, 3)
    gpu.kv_load_pages(cache, gpu.kv_slots(table, ints(47, 40), page, t), out[0], out[1])
    for got, side in zip(out, ref):
        for b, length in enumerate((47, 40)):
            assert torch.equal(got[b].cpu(), side.rows(table.cpu()[b], length)[length - t:])


def test_a_block_past_2_to_31_bytes(gpu):
    """Pages whose bytes lie past 2^31 and 2^32 of the pool."""
    page, kv, hd = 256, 8, 256                                   # 512 KB of K a page
    pages = 8300
    cache = gpu.PagedCache(torch.zeros(pages, kv, page, hd, dtype=torch.int8, device="cuda"),
                           torch.zeros(pages, kv, hd, page, dtype=torch.int8, device="cuda"),
                           torch.zeros(pages, kv, device="cuda"), torch.zeros(pages, kv, device="cuda"))
    table = torch.tensor([[8299, 4097, 3]], dtype=I32, device="cuda")
    x = torch.randn(1, 600, kv, hd)
    gpu.kv_store_pages(x.cuda(), x.cuda(), cache, table, ints(600))
    ref = P.Pool(torch.zeros(3, kv, page, hd, dtype=torch.int8), torch.zeros(3, kv))
    ref.store(x[0], [0, 1, 2], 0)
    for i, at in enumerate((8299, 4097, 3)):
        assert torch.equal(cache.k[at].cpu(), torch.from_numpy(ref.codes[i]))
        assert torch.equal(cache.v[at].cpu().transpose(1, 2), torch.from_numpy(ref.codes[i]))
    assert int(cache.k.view(torch.uint8).view(pages, -1)[:3].count_nonzero()) == 0
    got = gpu.kv_load_pages(cache, gpu.kv_slots(table, ints(600), page, 600))
    want = ref.rows([0, 1, 2], 600)
    assert torch.equal(got[0][0].cpu(), want) and torch.equal(got[1][0].cpu(), want)
