"""kv_store, kv_load and attn_kv on the GPU against their definitions
(kv_ref.py): codes and values exactly, the attention within a bound derived from
its sums."""
import numpy as np
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu
I32 = torch.int32
JUNK = {"f32": float("nan"), "f16": float("nan"), "bf16": float("nan"), "q8_0": 0x7e, "q4_0": 0x7e}  # 0x7e7e: NaN


def ints(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def junk(shape, kind, hd):
    """A cache whose every value reads as NaN."""
    if kind in R.FLOAT:
        return torch.full((*shape, hd), float("nan"), dtype=R.FLOAT[kind], device="cuda")
    return torch.full((*shape, hd // R.BLOCK * R.UNIT[kind]), 0x7e, dtype=torch.uint8, device="cuda")


def bits(x):
    return x.contiguous().view(torch.uint8)


# ---------------------------------------------------------------------------
# kv_store, kv_load
# ---------------------------------------------------------------------------


def edge_values(shape, seed):
    """Rows of ordinary values, of one value, of zeros, ties of the largest
    magnitude with either sign first, tiny and huge blocks, halves between codes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    f = x.reshape(-1, shape[-1])
    for i in range(f.shape[0]):
        kind = i % 9
        if kind == 1:
            f[i] = 0.0
        elif kind == 2:
            f[i] = -0.75
        elif kind == 3:
            f[i, 3], f[i, 17] = 5.0, -5.0
        elif kind == 4:
            f[i, 3], f[i, 17] = -5.0, 5.0
        elif kind == 5:
            f[i] *= 1e-7
        elif kind == 6:
            f[i] *= 1e-41
        elif kind == 7:
            f[i] *= 3e4
        elif kind == 8:
            f[i] = torch.arange(shape[-1]).remainder(17) * 0.5 - 4.0
    return x


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("n,t,kv,hd", [(1, 1, 8, 128), (3, 5, 2, 96), (2, 33, 1, 64), (1, 7, 3, 256), (2, 9, 2, 32)])
def test_store_and_load_are_exact(gpu, kind, n, t, kv, hd):
    if kind in R.FLOAT and hd == 96:
        hd = 91
    cap = t + 6
    k, v = edge_values((n, t, kv, hd), 1), edge_values((n, t, kv, hd), 2)
    slot = ints(*[(3 * b) % 7 for b in range(n)])
    caches = [junk((n, cap, kv), kind, hd) for _ in range(2)]
    want = [c.cpu().clone() for c in caches]
    for c, x in zip(want, (k, v)):
        for b in range(n):
            c[b, int(slot[b]):int(slot[b]) + t] = R.pack(x[b], kind)
    h = [R.handle(gpu, c, kind, hd) for c in caches]
    status = ints(0)
    gpu.kv_store(k.cuda(), v.cuda(), h[0], h[1], slot, status=status)
    for c, w in zip(caches, want):
        assert torch.equal(bits(c.cpu()), bits(w))
    assert int(status) == 0
    got = gpu.kv_load(h[0], h[1], slot, t)
    for x, w in zip(got, want):
        for b in range(n):
            ref = R.values(w[b, int(slot[b]):int(slot[b]) + t], kind)
            assert torch.equal(bits(x[b].cpu()), bits(ref))


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
def test_a_block_with_an_infinity_or_nan_reads_back_as_nan(gpu, kind):
    x = torch.randn(1, 4, 1, 64)
    x[0, 1, 0, 5], x[0, 2, 0, 40], x[0, 3, 0, 63] = float("inf"), float("-inf"), float("nan")
    c = [junk((1, 4, 1), kind, 64) for _ in range(2)]
    h = [R.handle(gpu, a, kind, 64) for a in c]
    gpu.kv_store(x.cuda(), x.cuda(), h[0], h[1], ints(0))
    got = gpu.kv_load(h[0], h[1], ints(0), 4)[0].cpu().view(4, 2, 32)
    bad = torch.tensor([[0, 0], [1, 0], [0, 1], [0, 1]], dtype=torch.bool)
    assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
    assert torch.equal(bits(c[0].cpu()[0]), bits(R.pack(x[0], kind)))


@pytest.mark.parametrize("kind", ["q4_0", "bf16", "f32"])
def test_counts_and_rows_that_do_not_fit(gpu, kind):
    """Rows past count stay; a sequence that does not fit is not written at all
    and sets the status; a load outside the cache gives NaN rows."""
    n, t, cap, kv, hd = 7, 5, 9, 2, 64
    k = torch.randn(n, t, kv, hd)
    caches = [junk((n, cap, kv), kind, hd) for _ in range(2)]
    before = caches[0].cpu().clone()
    h = [R.handle(gpu, c, kind, hd) for c in caches]
    #              fits  full  idle  high     low      count    count
    slot = ints(4, 4, -1, 5, -1, 0, 0)
    count = ints(2, 5, 0, 5, 3, 6, -1)
    status = ints(0)
    gpu.kv_store(k.cuda(), k.cuda(), h[0], h[1], slot, count, status)
    want = before.clone()
    want[0, 4:6] = R.pack(k[0, :2], kind)
    want[1, 4:9] = R.pack(k[1], kind)
    for c in caches:
        assert torch.equal(bits(c.cpu()), bits(want))
    assert int(status) == 1
    status.zero_()
    gpu.kv_store(k[:3].cuda(), k[:3].cuda(), R.handle(gpu, caches[0][:3], kind, hd),
                 R.handle(gpu, caches[1][:3], kind, hd), slot[:3].contiguous(), count[:3].contiguous(), status)
    assert int(status) == 0
    out = [torch.full((n, t, kv, hd), 7.5, device="cuda") for _ in range(2)]
    gpu.kv_load(h[0], h[1], ints(4, 7, 0, -2, 2 ** 31 - 1, -2 ** 31, 3), t, ints(2, 5, 0, 5, 5, 1, 9), out[0], out[1])
    got = out[0].cpu()
    vals = R.values(want, kind)
    assert torch.equal(got[0, :2], vals[0, 4:6]) and (got[0, 2:] == 7.5).all()
    assert torch.equal(got[1, :2], vals[1, 7:9]) and torch.isnan(got[1, 2:]).all()
    assert (got[2] == 7.5).all() and torch.isnan(got[3:5]).all()
    assert torch.isnan(got[5, :1]).all() and (got[5, 1:] == 7.5).all()
    assert torch.isnan(got[6]).all()                # (junk; the count is cut to 5)


@pytest.mark.parametrize("kind", R.TYPES)
def test_store_and_load_of_strided_tensors(gpu, kind):
    """Head-major caches, k and v interleaved in one buffer, k and v cut from a
    fused projection, and sequences further apart than their rows."""
    n, t, cap, kv, hd = 2, 5, 8, 3, 64
    width = hd if kind in R.FLOAT else hd // 32 * R.UNIT[kind]
    fused = torch.randn(n, t, 5, kv, hd).cuda()
    k, v = fused[:, :, 1], fused[:, :, 4]
    both = junk((n + 1, kv, cap, 2), kind, hd)
    kc, vc = (both[:n, :, :, i, :width].transpose(1, 2) for i in range(2))
    h = [R.handle(gpu, c, kind, hd) for c in (kc, vc)]
    slot = ints(3, 0)
    gpu.kv_store(k, v, h[0], h[1], slot)
    for c, x in ((kc, k), (vc, v)):
        for b in range(n):
            assert torch.equal(bits(c[b, int(slot[b]):int(slot[b]) + t].cpu()), bits(R.pack(x[b].cpu().contiguous(), kind)))
    assert torch.equal(bits(both[n]), bits(junk((kv, cap, 2), kind, hd)))
    got = gpu.kv_load(h[0], h[1], slot, t)
    for x, c in zip(got, (kc, vc)):
        for b in range(n):
            assert torch.equal(x[b].cpu(), R.values(c[b, int(slot[b]):int(slot[b]) + t].cpu().contiguous(), kind))


# ---------------------------------------------------------------------------
# attn_kv
# ---------------------------------------------------------------------------


def check(gpu, kind, q, k, v, length, count=None, window=0, sinks=0, scale=None, make=None, lengths_given=True):
    """One call against the definition; rows no query sees hold NaN."""
    n, t, heads, hd = q.shape
    cap = k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    cnt = [t] * n if count is None else count
    caches = []
    for x in (k, v):
        c = R.pack(x, kind)
        ref = R.values(c, kind)
        caches.append((c, ref))
    y, bound = R.attend(q, caches[0][1], caches[1][1], [min(max(x, 0), cap) for x in length],
                        [min(max(x, 0), t) for x in cnt], scale, window, sinks)
    dev = []
    for c, _ in caches:
        c = c.clone()
        for b in range(n):
            ln = min(max(length[b], 0), cap)
            first = ln - min(max(cnt[b], 0), t)
            c[b, ln:] = junk((1,), kind, hd)[0].cpu()
            if window:
                c[b, min(sinks, ln):max(min(sinks, ln), first - window + 1)] = junk((1,), kind, hd)[0].cpu()
        dev.append((make or (lambda z: z))(c.cuda()))
    out = torch.full(q.shape, 9.25, device="cuda")
    h = [R.handle(gpu, c, kind, hd) for c in dev]
    gpu.attn_kv(q.cuda(), h[0], h[1], ints(*length) if lengths_given else None, None if count is None else ints(*count),
                scale=scale, window=window, sinks=sinks, out=out)
    got = out.cpu().double()
    none = torch.isnan(y)
    assert (got[none] == 9.25).all()
    err = (got - y)[~none].abs()
    assert (err <= bound[~none]).all(), (float((err / bound[~none].clamp_min(1e-300)).max()), float(err.max()))
    return out


def rand(n, t, heads, kv, hd, cap, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    return 1.5 * r(n, t, heads, hd), r(n, cap, kv, hd), 0.5 * r(n, cap, kv, hd)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("t,kv,g,hd,cap", [(1, 8, 2, 128, 38), (1, 8, 2, 128, 700), (1, 1, 1, 64, 1), (1, 2, 16, 64, 333),
                                           (2, 4, 4, 96, 129), (5, 2, 7, 128, 190), (17, 2, 1, 64, 65),
                                           (40, 2, 2, 128, 200), (130, 1, 2, 64, 131), (3, 2, 2, 256, 77)])
def test_attention(gpu, kind, t, kv, g, hd, cap):
    q, k, v = rand(1, t, kv * g, kv, hd, cap, 3)
    check(gpu, kind, q, k, v, [cap])


@pytest.mark.parametrize("kind,hd", [("f32", 1), ("f32", 37), ("f16", 40), ("f16", 75), ("bf16", 80), ("bf16", 254),
                                     ("f16", 33), ("f32", 200), ("q8_0", 32), ("q4_0", 32), ("q4_0", 160), ("q8_0", 224)])
@pytest.mark.parametrize("t", [1, 21])
def test_head_dims(gpu, kind, hd, t):
    q, k, v = rand(2, t, 6, 3, hd, 90, 4)
    check(gpu, kind, q, k, v, [90, 57])


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f16", "bf16", "f32"])
@pytest.mark.parametrize("t,count", [(1, None), (1, [1, 0, 1, 1, 1, 0]), (6, [6, 0, 3, 6, 1, 2]), (70, [70, 0, 33, 70, 1, 2])])
def test_ragged_batches(gpu, kind, t, count):
    """Lengths of zero, one, and past the capacity; more positions than rows;
    queries that are padding."""
    q, k, v = rand(6, t, 4, 2, 64, 150, 5)
    check(gpu, kind, q, k, v, [150, 0, 71, 1, 900, 0], count)


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f16", "bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 0), (33, 70), (299, 4), (300, 4), (5000, 9000)])
@pytest.mark.parametrize("t", [1, 4, 90])
def test_window_and_sinks(gpu, kind, window, sinks, t):
    q, k, v = rand(2, t, 4, 2, 64, 300, 6)
    check(gpu, kind, q, k, v, [300, 171], window=window, sinks=sinks)


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f16", "bf16", "f32"])
@pytest.mark.parametrize("t", [1, 3, 50])
def test_strides(gpu, kind, t):
    """Head-major caches, and rows of a wider buffer, both off the usual
    alignment; q cut from a fused projection; y strided."""
    n, kv, g, hd, cap = 2, 2, 2, 64, 70
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 7)
    width = hd if kind in R.FLOAT else hd // 32 * R.UNIT[kind]

    def head_major(c):
        return c.transpose(1, 2).contiguous().transpose(1, 2)

    def wider(c):
        big = torch.zeros(n, cap + 1, kv, width + 7 if kind in R.FLOAT else width + 14, dtype=c.dtype, device="cuda")
        s = big[:, 1:, :, 5 if kind in R.FLOAT else 10:][..., :width]
        s.copy_(c)
        return s

    base = check(gpu, kind, q, k, v, [cap, 41])
    for make in (head_major, wider):
        check(gpu, kind, q, k, v, [cap, 41], make=make)
    fused = torch.randn(n, t, 3, kv * g, hd, device="cuda")
    fused[:, :, 1] = q.cuda()
    out = torch.zeros(n, kv * g, t, hd, device="cuda").transpose(1, 2)
    c = [R.handle(gpu, R.pack(x, kind).cuda(), kind, hd) for x in (k, v)]
    gpu.attn_kv(fused[:, :, 1], c[0], c[1], ints(cap, 41), out=out)
    assert torch.equal(out, base)


def test_without_length_every_row_is_filled(gpu):
    q, k, v = rand(2, 3, 4, 2, 64, 50, 8)
    check(gpu, "q4_0", q, k, v, [50, 50], lengths_given=False)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 6.0])
@pytest.mark.parametrize("t", [1, 40])
def test_scales(gpu, scale, t):
    """Zero (a mean), negative, and one that leaves single rows all the weight."""
    q, k, v = rand(1, t, 4, 2, 64, 100, 9)
    for kind in ("q4_0", "f16", "f32"):
        check(gpu, kind, q, k, v, [100], scale=scale)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("t", [1, 40])
def test_magnitudes(gpu, kind, t):
    """Small and large q, k and v, within F16's range where the cache is F16."""
    q, k, v = rand(1, t, 4, 2, 64, 100, 10)
    for a, b, c in ((1e-4, 1e3, 1e-4), (3e3, 1e-3, 2e3), (1.0, 1e-3, 1e-3)):
        check(gpu, kind, q * a, k * b, v * c, [100])


@pytest.mark.parametrize("kind", ["q4_0", "f16", "f32"])
def test_long_offsets(gpu, kind):
    """Rows and sequences more than 2^32 bytes apart."""
    kv, hd, cap, n = 1, 64, 70, 2
    q, k, v = rand(n, 1, 2, kv, hd, cap, 11)
    width = hd if kind in R.FLOAT else hd // 32 * R.UNIT[kind]
    size = R.pack(k, kind).element_size()
    row, seq = (80 << 20) // size, (6 << 30) // size          # cap rows cover 5.5 GB
    pool = torch.empty(seq + cap * row, dtype=R.pack(k, kind).dtype, device="cuda")
    make = [0]

    def far(c):
        s = pool.as_strided((n, cap, kv, width), (seq, row, width, 1), 1024 * make[0])
        make[0] += 1
        s.copy_(c)
        return s

    check(gpu, kind, q, k, v, [cap, 33], make=far)


def test_same_bits_each_time_and_on_any_stream(gpu):
    q, k, v = rand(3, 1, 16, 8, 128, 1500, 12)
    c = [gpu.Q4Tensor(R.pack(x, "q4_0").cuda(), 128) for x in (k, v)]
    q, length = q.cuda(), ints(1500, 700, 3)
    first = gpu.attn_kv(q, c[0], c[1], length)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        assert torch.equal(gpu.attn_kv(q, c[0], c[1], length), first)
        with torch.cuda.stream(s):
            other = gpu.attn_kv(q, c[0], c[1], length)
        s.synchronize()
        assert torch.equal(other, first)


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_decoding_step_captured_and_replayed(gpu, kind, window, sinks):
    """A prompt, then one captured step (kv_store and attn_kv, the slots and
    lengths advanced on the device) replayed token after token: each replay is the
    eager call on the same cache, and the definition."""
    n, heads, kv, hd, cap, prompt = 3, 4, 2, 64, 160, [70, 1, 101]
    g = torch.Generator().manual_seed(13)
    r = lambda *s: torch.randn(s, generator=g)
    caches = [junk((n, cap, kv), kind, hd) for _ in range(2)]
    h = [R.handle(gpu, c, kind, hd) for c in caches]
    pk, pv = r(n, 101, kv, hd).cuda(), r(n, 101, kv, hd).cuda()
    count = ints(*prompt)
    gpu.kv_store(pk, pv, h[0], h[1], ints(0, 0, 0), count)
    pq = r(n, 101, heads, hd)
    y = torch.full(pq.shape, 9.25, device="cuda")
    gpu.attn_kv(pq.cuda(), h[0], h[1], count, count, window=window, sinks=sinks, out=y)
    vals = [R.values(c.cpu(), kind) for c in caches]
    ref, bound = R.attend(pq, vals[0], vals[1], prompt, prompt, hd ** -0.5, window, sinks)
    real = ~torch.isnan(ref)
    assert ((y.cpu().double() - ref)[real].abs() <= bound[real]).all() and (y.cpu()[~real] == 9.25).all()

    q, k, v = (torch.zeros(n, 1, x, hd, device="cuda") for x in (heads, kv, kv))
    slot, length, status = count.clone(), count + 1, ints(0)
    out = torch.zeros(n, 1, heads, hd, device="cuda")

    def step():
        gpu.kv_store(k, v, h[0], h[1], slot, None, status)
        gpu.attn_kv(q, h[0], h[1], length, window=window, sinks=sinks, out=out)
        slot.add_(1)
        length.add_(1)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    keep = [x.clone() for x in (slot, length)] + [c.clone() for c in caches]
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x, y0 in zip((slot, length, *caches), keep):
        x.copy_(y0)
    for token in range(6):
        for x in (q, k, v):
            x.copy_(r(*x.shape))
        graph.replay()
        eager = gpu.attn_kv(q, h[0], h[1], length - 1, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        lens = [p + token + 1 for p in prompt]
        vals = [R.values(c.cpu(), kind) for c in caches]
        ref, bound = R.attend(q.cpu(), vals[0], vals[1], lens, [1] * n, hd ** -0.5, window, sinks)
        assert ((out.cpu().double() - ref).abs() <= bound).all()
        for b in range(n):
            assert torch.equal(bits(caches[0][b, lens[b] - 1].cpu()), bits(R.pack(k[b, 0].cpu(), kind)))
    assert int(status) == 0


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("window", [0, 50])
def test_blocks_whose_values_are_out_of_f16s_range(gpu, kind, t, window):
    """K and V blocks with d of thousands, and among them ordinary and tiny ones,
    first and last in the cache."""
    q, k, v = rand(2, t, 4, 2, 64, 300, 14)
    k = k * 1e4
    v[:, 100:120] *= 1e5
    v[:, 120:130] *= 1e-4
    v[:, 200:, 1] *= 3e3
    check(gpu, kind, q * 1e-4, k, v, [300, 131], window=window, sinks=3)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("hd", [96, 64])
@pytest.mark.parametrize("t,kv,g", [(1, 12, 1), (1, 2, 16), (5, 8, 2), (3, 3, 5), (33, 2, 2)])
def test_head_layouts(gpu, kind, hd, t, kv, g):
    """Groups of heads that do and do not fill the matrix unit's columns."""
    q, k, v = rand(2, t, kv * g, kv, hd, 85, 15)
    check(gpu, kind, q, k, v, [85, 40])


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("t,hd", [(1, 64), (3, 64), (40, 64), (6, 160)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite_is_its_own_rows_queries_alone(gpu, kind, t, hd, bad):
    """An infinity or NaN in k of one head and v of another, at rows that some of
    the queries see, and in one query: NaN there, every other result as ever."""
    n, kv, g, cap = 1, 4, 2, 100
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 16)
    row, late = cap - t // 2 - 1, cap - 1
    caches = [R.pack(x, kind) for x in (k, v)]
    y, bound = R.attend(q, R.values(caches[0], kind), R.values(caches[1], kind), [cap], [t], hd ** -0.5, window=60, sinks=2)
    k, v = k.clone(), v.clone()
    k[0, row, 0, 5] = float("nan")
    v[0, row, 1, 7] = bad
    v[0, late, 3, hd - 1] = bad
    v[0, 30, 2] = bad                     # behind the window of all queries, or of the later ones
    k[0, 30, 2] = bad
    q = q.clone()
    q[0, 0, 4] = float("nan")             # the first query of kv head 2's first head
    nan = torch.zeros(t, kv * g, dtype=torch.bool)
    p = torch.arange(cap - t, cap)
    nan[p >= row, 0:4] = True
    nan[p >= late, 6:8] = True
    nan[30 > p - 60, 4:6] = True
    nan[0, 4] = True
    c = [R.handle(gpu, R.pack(x, kind).cuda(), kind, hd) for x in (k, v)]
    got = gpu.attn_kv(q.cuda(), c[0], c[1], ints(cap), window=60, sinks=2).cpu().double()
    assert torch.isnan(got[0][nan]).any(-1).all()
    assert ((got - y).abs()[0][~nan] <= bound[0][~nan]).all()


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f16"])
@pytest.mark.parametrize("t,row", [(1, 12 << 20), (1, 20 << 20), (1, 40 << 20), (40, 12 << 20), (40, 20 << 20)])
def test_rows_megabytes_apart(gpu, kind, t, row):
    """Row strides on either side of what the kernels take at 32-bit offsets."""
    kv, hd, cap = 2, 64, 70
    q, k, v = rand(1, t, 4, kv, hd, cap, 17)
    width = hd if kind in R.FLOAT else hd // 32 * R.UNIT[kind]
    size = R.pack(k, kind).element_size()
    pool = torch.empty((cap * row + (1 << 20)) // size, dtype=R.pack(k, kind).dtype, device="cuda")
    make = [0]

    def far(c):
        s = pool.as_strided((1, cap, kv, width), (0, row // size, width, 1), 4096 * make[0])
        make[0] += 1
        s.copy_(c)
        return s

    check(gpu, kind, q, k, v, [cap], make=far)


@pytest.mark.parametrize("kind", ["q4_0", "q8_0"])
@pytest.mark.parametrize("t", [1, 3])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
def test_long_caches_at_odd_addresses(gpu, kind, t, window, sinks):
    """Few queries over long caches that no 4-byte read is aligned in."""
    n, kv, g, hd, cap = 2, 8, 2, 64, 4000
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 18)

    def odd(c):
        pool = torch.empty(c.numel() + 2, dtype=torch.uint8, device="cuda")
        s = pool[2:].view(c.shape)
        s.copy_(c)
        return s

    check(gpu, kind, q, k, v, [cap, 1999], window=window, sinks=sinks, make=odd)


@pytest.mark.parametrize("kind", ["q4_0", "f16"])
@pytest.mark.parametrize("t", [1, 33])
def test_rows_megabytes_apart_in_parts(gpu, kind, t):
    """As above, with enough of them that the keys of a query are split."""
    kv, g, hd, cap, row = 8, 2, 64, 150, 40 << 20
    q, k, v = rand(1, t, kv * g, kv, hd, cap, 19)
    size = R.pack(k, kind).element_size()
    width = hd if kind in R.FLOAT else hd // 32 * R.UNIT[kind]
    pool = torch.empty(cap * row // size, dtype=R.pack(k, kind).dtype, device="cuda")
    make = [0]

    def far(c):
        s = pool.as_strided((1, cap, kv, width), (0, row // size, width, 1), 4096 * make[0])
        make[0] += 1
        s.copy_(c)
        return s

    check(gpu, kind, q, k, v, [cap], make=far)


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "f16"])
@pytest.mark.parametrize("t", [1, 3])
def test_more_sequences_than_a_wave_has_lanes(gpu, kind, t):
    n, kv, g, hd, cap = 150, 4, 2, 32, 300
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 20)
    length = [(37 * b * b + 11 * b) % (cap + 1) for b in range(n)]
    count = [min(b % (t + 2), t, length[b]) for b in range(n)]
    check(gpu, kind, q, k, v, length, count)
    check(gpu, kind, q, k, v, length, [0] * (n - 1) + [min(t, length[-1])])


@pytest.mark.parametrize("kind", ["q4_0", "f16"])
@pytest.mark.parametrize("n,t,kv,g,cap", [(2, 700, 4, 2, 900),      # keys split, rows of one part and of several
                                          (1, 380, 100, 1, 380),    # rows in two
                                          (1, 500, 100, 1, 530),    # whole rows, all at once
                                          (1, 700, 100, 1, 700)])   # and more than that
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 70)])
def test_prompts_of_many_tiles(gpu, kind, n, t, kv, g, cap, window, sinks):
    hd = 32
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 21)
    length = [cap, 400][:n]
    check(gpu, kind, q, k, v, length, [min(t, x) - 3 * b for b, x in enumerate(length)], window, sinks)


@pytest.mark.parametrize("kind", ["q4_0", "q8_0", "bf16", "f32"])
@pytest.mark.parametrize("t", [1, 5, 40])
def test_sequences_that_share_a_cache(gpu, kind, t):
    """One cache's rows at a sequence stride of zero, several queries' continuations."""
    n, kv, g, hd, cap = 3, 4, 2, 64, 900
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 22)
    k, v = (x[:1].expand(n, -1, -1, -1).contiguous() for x in (k, v))
    check(gpu, kind, q, k, v, [cap] * n, [t, 1, 0], make=lambda c: c[:1].contiguous().expand(n, -1, -1, -1))
    c = R.pack(k[:1], kind).cuda()
    h = R.handle(gpu, c.expand(n, -1, -1, -1), kind, hd)
    x, y = gpu.kv_load(h, h, ints(0, 7, 300), t)
    for b, slot in enumerate((0, 7, 300)):
        want = R.values(c[0, slot:slot + t].cpu().contiguous(), kind)
        assert torch.equal(x[b].cpu(), want) and torch.equal(y[b].cpu(), want)


@pytest.mark.parametrize("kind,hd", [(k, hd) for k in R.TYPES for hd in (160, 192, 224, 256)] +
                         [("f32", 129), ("f16", 130), ("bf16", 250), ("f16", 131)])
@pytest.mark.parametrize("t,cap", [(1, 300), (90, 200), (300, 700)])
def test_long_heads(gpu, kind, hd, t, cap):
    n, kv, g = 2, 2, 3
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 23)
    check(gpu, kind, q, k, v, [cap, 100], [t, min(t, 60)])
    check(gpu, kind, q, k, v, [cap, 100], [t, min(t, 60)], window=50, sinks=3)
