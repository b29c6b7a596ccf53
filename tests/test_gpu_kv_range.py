"""attn_kv over values of very different sizes on the GPU: what one row holds is
not to change what the others come to. The bound is kv_ref.attend_by_row's."""
import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rand(n, t, heads, kv, hd, cap, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    return 1.5 * r(n, t, heads, hd), r(n, cap, kv, hd), 0.5 * r(n, cap, kv, hd)


def run(gpu, kind, q, k, v, length, count=None, window=0, sinks=0, scale=None):
    """One call against the definition, over the values that the cache holds."""
    n, t, heads, hd = q.shape
    scale = hd ** -0.5 if scale is None else scale
    cache = [R.pack(x, kind) for x in (k, v)]
    y, bound = R.attend_by_row(q, *(R.values(c, kind) for c in cache), kind, length, count or [t] * n, scale, window, sinks)
    h = [R.handle(gpu, c.cuda(), kind, hd) for c in cache]
    got = gpu.attn_kv(q.cuda(), h[0], h[1], ints(*length), None if count is None else ints(*count), scale=scale,
                      window=window, sinks=sinks).cpu().double()
    real = ~torch.isnan(y)
    err = (got - y).abs()[real]
    assert (err <= bound[real]).all(), float((err / bound[real].clamp_min(1e-300)).max())  # (false for a NaN too)
    return got


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("t,hd,cap", [(1, 64, 1), (1, 128, 70), (40, 64, 40), (40, 128, 200), (300, 64, 300), (5, 160, 90)])
@pytest.mark.parametrize("small", [0.0, 1e-20, 1e-30])
def test_queries_and_keys_of_zero_and_next_to_it(gpu, kind, t, hd, cap, small):
    """All weights alike: the mean of V, whatever rows are hidden. All of q and K
    at once, a part of each, and only the keys of one tile."""
    q, k, v = rand(2, t, 4, 2, hd, cap, 31)
    run(gpu, kind, q * small, k * small, v, [cap, (cap + 1) // 2])
    part = torch.rand(q.shape[:3], generator=torch.Generator().manual_seed(32)) < 0.5
    qs = torch.where(part[..., None], q * small, q)
    ks = k.clone()
    ks[:, :64] *= small
    ks[:, 64::3] *= small
    run(gpu, kind, qs, ks, v, [cap, (cap + 1) // 2])
    run(gpu, kind, q * small, k * small, v * small, [cap, (cap + 1) // 2], window=30, sinks=2)
    run(gpu, kind, q * small, k * small, v, [0, cap])


def cases(*shapes, kinds=R.TYPES):
    """Shapes for all types."""
    return [(k, *x) for k in kinds for x in shapes]


LARGE = {"f32": 1e12, "bf16": 1e12, "f16": 1e4, "q8_0": 1.5e6, "q4_0": 1e5}  # (finite as the cache holds them: d up to 53000)


@pytest.mark.parametrize("kind,t,hd,cap", cases((40, 64, 200), (130, 128, 130), (3, 128, 300), (5, 160, 90), (64, 32, 64)))
@pytest.mark.parametrize("window", [0, 20])
def test_a_large_key_does_not_touch_the_queries_that_do_not_see_it(gpu, kind, t, hd, cap, window):
    """Ahead of the first queries and, with the window, behind the last."""
    q, k, v = rand(1, t, 4, 2, hd, cap, 33)
    for row in (cap - t, cap - t // 2, cap - 1):
        x = k.clone()
        x[0, row] *= LARGE[kind]
        run(gpu, kind, q, x, v, [cap], window=window, sinks=1)


@pytest.mark.parametrize("kind,t,hd,cap", cases((1, 64, 100), (1, 128, 700), (40, 64, 200), (130, 128, 130), (5, 160, 90)))
def test_a_large_key_of_no_weight(gpu, kind, t, hd, cap):
    """Its scores are far below the others'; it moves no other row's weight."""
    q, k, v = rand(1, t, 4, 2, hd, cap, 34)
    q = q.abs() + 0.5
    for row in (0, cap - t, cap // 3):
        x = k.clone()
        x[0, row] = -LARGE[kind]
        run(gpu, kind, q, x, v, [cap])


@pytest.mark.parametrize("kind,t,hd,cap", cases((40, 64, 200), (130, 128, 130), (3, 128, 300), (5, 160, 90), (300, 32, 300)))
@pytest.mark.parametrize("window", [0, 20])
def test_a_large_value_does_not_touch_the_queries_that_do_not_see_it(gpu, kind, t, hd, cap, window):
    q, k, v = rand(1, t, 4, 2, hd, cap, 35)
    for row in (cap - t, cap - t // 2, cap - 1):
        x = v.clone()
        x[0, row] *= LARGE[kind]
        run(gpu, kind, q, k, x, [cap], window=window, sinks=1)


@pytest.mark.parametrize("kind,t,hd,cap", cases((1, 64, 100), (1, 128, 700), (40, 64, 200), (130, 128, 130), (5, 160, 90)))
def test_a_large_value_of_no_weight(gpu, kind, t, hd, cap):
    q, k, v = rand(1, t, 4, 2, hd, cap, 36)
    q = q.abs() + 0.5
    for row in (0, cap - t, cap // 3):
        x, z = k.clone(), v.clone()
        x[0, row] = -1e4
        z[0, row] *= LARGE[kind]
        run(gpu, kind, q, x, z, [cap])


@pytest.mark.parametrize("kind,t,kv,g,hd", cases((1, 8, 2, 128), (1, 8, 1, 64), (2, 4, 2, 64), (40, 4, 2, 64)))
def test_heads_of_different_sizes(gpu, kind, t, kv, g, hd):
    """A head whose values are large beside heads of ordinary and small ones."""
    q, k, v = rand(2, t, kv * g, kv, hd, 150, 37)
    v[:, :, 1] *= LARGE[kind] / 20
    v[:, :, 0] *= 0.06
    v[:, 70:, 2] *= LARGE[kind] / 20
    run(gpu, kind, q, k, v, [150, 90])
    k[:, :, 1], q[:, :, g:2 * g] = k[:, :, 1] * LARGE[kind] / 20, q[:, :, g:2 * g] * 1e-5
    k[:, :, 0] *= 1e-3
    run(gpu, kind, q, k, v, [150, 90])


@pytest.mark.parametrize("kind,t,hd", cases((1, 128), (1, 64), (3, 160), (40, 128), (40, 64), kinds=["q8_0", "q4_0"]))
def test_blocks_of_different_sizes(gpu, kind, t, hd):
    """One block of a row large, the next one small: both exact."""
    q, k, v = rand(1, t, 4, 2, hd, 150, 38)
    v[..., :32] *= LARGE[kind] / 10
    v[..., 32:64] *= 0.05
    v[:, 60:90] *= 1e-3
    run(gpu, kind, q, k, v, [150])
    q[..., :32] *= 1e-6
    k[..., :32] *= LARGE[kind] / 10
    k[..., 32:64] *= 0.05
    run(gpu, kind, q, k, v, [150])


@pytest.mark.parametrize("kind,t,hd", cases((1, 64), (40, 64), (130, 128), (7, 200), kinds=["f32", "bf16"]))
def test_rows_of_all_sizes(gpu, kind, t, hd):
    """Rows of V from 1e-30 to 1e30 and of K from 1e-12 to 1e3, in any order."""
    q, k, v = rand(2, t, 4, 2, hd, 200, 39)
    g = torch.Generator().manual_seed(40)
    up = lambda lo, hi: 10.0 ** (lo + (hi - lo) * torch.rand((2, 200, 2, 1), generator=g))
    run(gpu, kind, q, k, v * up(-30, 30), [200, 131])
    run(gpu, kind, q, k * up(-12, 0), v * up(-30, 30), [200, 131], window=30, sinks=4)
    run(gpu, kind, q, k * up(-12, 3), v * up(-3, 3), [200, 131])


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("t,hd,cap", [(1, 64, 100), (1, 128, 700), (3, 160, 90), (40, 64, 150), (130, 128, 130)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 22, 2.0 ** 24, 3.0 * 2 ** 24, 2.0 ** 26, 2.0 ** 30, 2.0 ** 40])
def test_scores_past_whole_numbers(gpu, kind, t, hd, cap, sign, size):
    """Scores so large that f32 holds no units of them: the row of the largest has
    all the weight. Its score is twice the others' (half, where they are below
    zero), so that the others' weights are below e^-1000: what is left is that
    row's own values, off by the weight's and the sum's half steps (8) and, where
    V is two F16 pieces, by 2^-23 of themselves and 2^-30 of the row's largest."""
    q, k, v = rand(1, t, 4, 2, hd, cap, 41)
    k = 1.0 + k.abs().clamp(max=1.0)
    star = cap - t // 2 - 1
    k[0, star] = 4.0 if sign > 0 else 0.5
    q = torch.full(q.shape, sign * size / hd ** 0.5)
    cache = [R.pack(x, kind) for x in (k, v)]
    h = [R.handle(gpu, c.cuda(), kind, hd) for c in cache]
    got = gpu.attn_kv(q.cuda(), h[0], h[1], ints(cap)).cpu()
    assert torch.isfinite(got).all()
    want = R.values(cache[1], kind)[0, star].double().repeat_interleave(2, 0)
    bound = (8 * R.EPS + 2.0 ** -23) * want.abs() + 2.0 ** -30 * want.abs().amax(-1, keepdim=True)
    for i in range(star - (cap - t), t):
        assert ((got[0, i].double() - want).abs() <= bound).all(), i


@pytest.mark.parametrize("kind,hd", [(k, 64) for k in R.TYPES] + [("f16", 75), ("bf16", 33), ("q8_0", 160), ("f32", 200)])
@pytest.mark.parametrize("t", [1, 3, 40])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("score", [1.0, -1.0])
def test_an_infinite_key_is_nan_for_those_that_see_it(gpu, kind, hd, t, sign, score):
    """Whatever the sign of its score; a block's d becomes infinite where a value is
    past what F16's d holds. Queries that do not see it, and other heads, are as ever."""
    n, kv, g, cap = 1, 4, 2, 100
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 42)
    row = cap - t // 2 - 1
    cache = [R.pack(x, kind) for x in (k, v)]
    y, bound = R.attend_by_row(q.abs() * sign * score, *(R.values(c, kind) for c in cache), kind, [cap], [t], hd ** -0.5,
                               window=60, sinks=2)
    k = k.clone()
    k[0, row, 1] = sign * 1e30 if kind in ("q8_0", "q4_0") else k[0, row, 1]
    k[0, row, 1, 5] = sign * (1e30 if kind in ("q8_0", "q4_0") else float("inf"))
    k[0, 20, 2, 7] = sign * (1e30 if kind in ("q8_0", "q4_0") else float("inf"))  # behind the window
    q = q.abs() * sign * score
    h = [R.handle(gpu, R.pack(x, kind).cuda(), kind, hd) for x in (k, v)]
    got = gpu.attn_kv(q.cuda(), h[0], h[1], ints(cap), window=60, sinks=2).cpu().double()
    nan = torch.zeros(t, kv * g, dtype=torch.bool)
    p = torch.arange(cap - t, cap)
    nan[p >= row, g:2 * g] = True
    nan[20 > p - 60, 2 * g:3 * g] = True
    assert torch.isnan(got[0][nan]).all()
    assert ((got - y).abs()[0][~nan] <= bound[0][~nan]).all()


@pytest.mark.parametrize("kind,hd", [(k, 64) for k in R.TYPES] + [("f16", 75), ("q8_0", 160)])
@pytest.mark.parametrize("t", [1, 3, 40])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("zeros", [False, True])
def test_a_query_that_is_not_finite(gpu, kind, hd, t, value, zeros):
    """NaN for that query and head, whatever the keys' signs, zero among them or not."""
    n, kv, g, cap = 1, 4, 2, 100
    q, k, v = rand(n, t, kv * g, kv, hd, cap, 43)
    k = k.abs() + 0.5
    if zeros:
        k[0, ::3] = 0.0
    cache = [R.pack(x, kind) for x in (k, v)]
    y, bound = R.attend_by_row(q, *(R.values(c, kind) for c in cache), kind, [cap], [t], hd ** -0.5)
    q = q.clone()
    nan = torch.zeros(t, kv * g, dtype=torch.bool)
    for i, head in ((0, 1), (t - 1, 6)):
        q[0, i, head, 3] = value
        nan[i, head] = True
    h = [R.handle(gpu, c.cuda(), kind, hd) for c in cache]
    got = gpu.attn_kv(q.cuda(), h[0], h[1], ints(cap)).cpu().double()
    assert torch.isnan(got[0][nan]).all()
    assert ((got - y).abs()[0][~nan] <= bound[0][~nan]).all()


@pytest.mark.parametrize("kind,t,hd", cases((1, 64), (40, 64), (130, 128), (3, 160)))
@pytest.mark.parametrize("window", [0, 70])
def test_rows_of_all_sizes_beside_what_is_not_finite(gpu, kind, t, hd, window):
    """Rows of many sizes, among them some with a NaN that no query, or only the
    later ones, see, and a channel far above the others."""
    q, k, v = rand(2, t, 4, 2, hd, 200, 44)
    q[..., 7] *= 1e-3
    g = torch.Generator().manual_seed(45)
    wide = {"f32": 6.0, "bf16": 6.0, "f16": 2.0, "q8_0": 2.0, "q4_0": 2.0}[kind]
    up = lambda: 10.0 ** (wide * (2 * torch.rand((2, 200, 2, 1), generator=g) - 1))
    v = v * up()
    v[..., 5] *= 50.0
    k = k * up().clamp(max=3.0)
    k[..., 7] *= 50.0
    length = [200, 131]
    cache = [R.pack(x, kind) for x in (k, v)]
    y, bound = R.attend_by_row(q, *(R.values(c, kind) for c in cache), kind, length, [t, t], hd ** -0.5, window, 2)
    nan = torch.zeros(2, t, 4, dtype=torch.bool)
    for b in range(2):
        p = torch.arange(length[b] - t, length[b])
        for row, head, which in ((length[b] - 1, 0, 0), (length[b] - 1 - t // 2, 1, 1), (40, 0, 1)):
            (k, v)[which][b, row, head, 3] = float("nan")
            seen = (row <= p) & ((row > p - window) if window else (row >= 0))
            nan[b, seen, 2 * head:2 * head + 2] = True
    h = [R.handle(gpu, R.pack(x, kind).cuda(), kind, hd) for x in (k, v)]
    got = gpu.attn_kv(q.cuda(), h[0], h[1], ints(*length), window=window, sinks=2).cpu().double()
    real = ~torch.isnan(y).any(-1)
    assert torch.isnan(got[nan & real]).all()
    fine = real & ~nan
    err = (got - y).abs()[fine]
    assert (err <= bound[fine]).all(), float((err / bound[fine].clamp_min(1e-300)).max())


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("t,cap", [(1, 700), (70, 300)])
def test_captured_over_zeros_and_replayed(gpu, kind, t, cap):
    """A call captured while its inputs are zeros, replayed over ordinary values,
    over rows of very different sizes and over zeros again: the eager call's
    results each time, and the definition's."""
    n, heads, kv, hd = 2, 4, 2, 64
    q, k, v = rand(n, t, heads, kv, hd, cap, 46)
    g = torch.Generator().manual_seed(47)
    up = 10.0 ** (8 * torch.rand((n, cap, kv, 1), generator=g) - 4) if kind in ("f32", "bf16") else torch.ones(n, cap, kv, 1)
    up[:, ::9] *= 1.0 if kind == "f16" else 1e5
    zero = [R.pack(torch.zeros_like(x), kind).cuda() for x in (k, v)]
    cache = [x.clone() for x in zero]
    h = [R.handle(gpu, c, kind, hd) for c in cache]
    length, qd = ints(cap, cap - 33), torch.zeros(q.shape, device="cuda")
    out = torch.zeros(q.shape, device="cuda")
    call = lambda: gpu.attn_kv(qd, h[0], h[1], length, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    assert (out == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for a, b, c in ((q, k, v), (q, k * up.clamp(max=10.0), v * up), (0 * q, 0 * k, v), (q, k, v * up), (0 * q, 0 * k, 0 * v)):
        qd.copy_(a)
        host = [R.pack(x, kind) for x in (b, c)]
        for x, y in zip(cache, host):
            x.copy_(y)
        graph.replay()
        eager = gpu.attn_kv(qd, h[0], h[1], length)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        y, bound = R.attend_by_row(a, *(R.values(x, kind) for x in host), kind, [cap, cap - 33], [t, t], hd ** -0.5)
        assert ((out.cpu().double() - y).abs() <= bound).all()
