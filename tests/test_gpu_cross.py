"""attn_cross on the GPU against its definition, within the bound of
kv_ref.attend_by_row: a query that sees all rows is the newest position over a
cache of them."""
import math

import pytest
import torch

import kv_ref as R

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def attend(q, k, v, kind, length, count, scale):
    """(y, bound): the positions of a kv head as so many heads of one position."""
    n, t, heads, hd = q.shape
    kv = k.shape[2]
    many = q.reshape(n, t, kv, heads // kv, hd).transpose(1, 2).reshape(n, 1, -1, hd)
    back = [x.reshape(n, kv, t, heads // kv, hd).transpose(1, 2).reshape(n, t, heads, hd)
            for x in R.attend_by_row(many, k, v, kind, length, [1] * n, scale)]
    for b in range(n):
        back[0][b, count[b]:] = float("nan")
    return back


def states(kind, n, rows, kv, hd, seed):
    """K and V as a cache holds them, and their values."""
    g = torch.Generator().manual_seed(seed)
    packed = [R.pack(torch.randn(n, rows, kv, hd, generator=g) * by, kind) for by in (1.0, 0.5)]
    return packed, [R.values(c, kind) for c in packed]


def junk(c, kind, length):
    """The cache with every row past a sequence's length reading as NaN."""
    c = c.clone()
    for b, ln in enumerate(length):
        c[b, max(ln, 0):] = float("nan") if kind in R.FLOAT else 0x7e
    return c


def check(gpu, kind, heads, kv, hd, t, rows, length, count=None, scale=None, make=lambda x: x, lengths_given=True, q=None):
    n = len(length)
    q = torch.randn(n, t, heads, hd, generator=torch.Generator().manual_seed(t)) * 1.5 if q is None else q
    packed, values = states(kind, n, rows, kv, hd, rows)
    clamped = [min(max(x, 0), rows) for x in length]
    cnt = [t] * n if count is None else [min(max(x, 0), t) for x in count]
    y, bound = attend(q, *values, kind, clamped, cnt, hd ** -0.5 if scale is None else scale)
    k, v = (R.handle(gpu, make(junk(c, kind, clamped).cuda()), kind, hd) for c in packed)
    out = torch.full(q.shape, 9.25, device="cuda")
    gpu.attn_cross(q.cuda(), k, v, ints(*length) if lengths_given else None, None if count is None else ints(*count),
                   scale=scale, out=out)
    got = out.cpu().double()
    none = torch.isnan(y)
    assert (got[none] == 9.25).all()
    err = (got - y)[~none].abs()
    assert (err <= bound[~none]).all(), (float((err / bound[~none].clamp_min(1e-300)).max()), float(err.max()))


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("heads,kv,hd,t,rows", [(16, 16, 64, 1, 300), (12, 12, 64, 130, 130), (16, 8, 128, 1, 1000), (4, 2, 128, 200, 77),
                                                (7, 1, 96, 5, 260), (3, 3, 32, 17, 1), (2, 1, 256, 33, 150), (8, 2, 160, 2, 65)])
def test_all_queries_see_all_rows(gpu, kind, heads, kv, hd, t, rows):
    length = [rows, rows - 1, 1, 0, max(1, rows // 2), -4, rows + 7]
    check(gpu, kind, heads, kv, hd, t, rows, length)
    check(gpu, kind, heads, kv, hd, t, rows, length, [t, 1, t, t, t - 1, 0, t + 3])
    check(gpu, kind, heads, kv, hd, t, rows, [rows] * 2, lengths_given=False, scale=-0.3)


@pytest.mark.parametrize("kind", sorted(R.FLOAT))
@pytest.mark.parametrize("hd", [1, 7, 40, 80, 91])
def test_heads_of_odd_length(gpu, kind, hd):
    check(gpu, kind, 6, 3, hd, 1, 90, [90, 33])
    check(gpu, kind, 6, 3, hd, 70, 90, [90, 33])


@pytest.mark.parametrize("kind", R.TYPES)
def test_one_position_of_many_query_heads(gpu, kind):
    check(gpu, kind, 40, 2, 64, 1, 700, [700, 0, 1, 65])
    check(gpu, kind, 17, 1, 256, 1, 90, [90, 33])


@pytest.mark.parametrize("kind", ["f16", "f32", "q8_0"])
@pytest.mark.parametrize("t", [1, 30])
def test_a_captured_call_of_split_heads_serves_all_lengths(gpu, kind, t):
    """Lengths and counts change between replays, over the workspace that the last left."""
    n, rows, heads, kv, hd = 3, 9000, 4, 2, 64
    packed, values = states(kind, n, rows, kv, hd, 5)
    k, v = (R.handle(gpu, c.cuda(), kind, hd) for c in packed)
    q, out = (torch.zeros(n, t, heads, hd, device="cuda") for _ in range(2))
    length, count = ints(*[0] * n), ints(*[0] * n)
    work = torch.full((gpu.attn_cross_work(q, k),), float("nan"), device="cuda")
    assert work.numel() > 0

    def call():
        gpu.attn_cross(q, k, v, length, count, out=out, work=work)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i, (ln, c) in enumerate([([9000, 1, 300], [t, 1, t]), ([64, 5000, 64], [t, 0, t]), ([0, 0, 9000], [1, 0, 1])]):
        x = torch.randn(q.shape, generator=torch.Generator().manual_seed(i))
        q.copy_(x), length.copy_(ints(*ln)), count.copy_(ints(*c))
        out.fill_(9.25)
        graph.replay()
        got = out.cpu()
        y, bound = attend(x, *values, kind, ln, c, hd ** -0.5)
        live = ~torch.isnan(y)
        assert (got[~live] == 9.25).all() and ((got.double() - y)[live].abs() <= bound[live]).all()
        out.fill_(9.25)
        call()
        assert torch.equal(out.cpu(), got)


@pytest.mark.parametrize("kind", R.TYPES)
def test_long_states(gpu, kind):
    """Queries whose parts are joined."""
    check(gpu, kind, 2, 1, 64, 1, 9000, [9000, 4500])
    check(gpu, kind, 2, 1, 64, 40, 5000, [5000])
    check(gpu, kind, 4, 4, 64, 600, 700, [700, 650])


@pytest.mark.parametrize("kind,hd,length", [("f16", 64, [131072 + 37]), ("bf16", 64, [200000, 5]), ("f16", 40, [140000, 0, 1]),
                                            ("f32", 64, [120000]), ("bf16", 128, [70000, 64]), ("f16", 256, [50000, 16])])
def test_one_head_for_every_workgroup(gpu, kind, hd, length):
    """One kv head whose rows are shared out over all workgroups that the chip holds,
    up to 1024 parts of one result. Scores are all 0 and values whole numbers, so that
    weights are 1 and sums exact, whatever their order: what is left is 1/l and its
    product, half a step each."""
    n, rows = len(length), max(length)
    v = ((torch.arange(rows)[:, None] * 7 + torch.arange(hd) * 3) % 13 - 5).float()
    v[rows - rows // 4:] += 3.0                                            # (no part is like another)
    k = torch.zeros(n, rows, 1, hd, dtype=R.FLOAT[kind], device="cuda")
    vs = v[None, :, None].expand(n, -1, -1, -1).to(R.FLOAT[kind]).cuda()
    q = torch.randn(n, 1, 2, hd, generator=torch.Generator().manual_seed(1)).cuda()
    want = torch.stack([v[:ln].double().mean(0) if ln else torch.zeros(hd).double() for ln in length])[:, None, None]
    for _ in range(2):
        got = gpu.attn_cross(q, k, vs, ints(*length)).cpu().double()
        assert ((got - want).abs() <= 2 * 2.0 ** -24 * 1.001 * want.abs()).all(), float((got - want).abs().max())


@pytest.mark.parametrize("kind", ["f32", "bf16", "q8_0"])
@pytest.mark.parametrize("t", [1, 60])
def test_what_is_not_finite(gpu, kind, t):
    """An infinity or NaN in a row of K or V, or a query: NaN, to its own head only."""
    n, rows, heads, kv, hd = 2, 100, 4, 2, 64
    packed, _ = states(kind, n, rows, kv, hd, 3)
    q = torch.randn(n, t, heads, hd)
    want = torch.zeros(n, t, heads, dtype=torch.bool)
    for side, (b, row, h) in zip(packed, ((0, 17, 1), (1, 99, 0))):
        if kind in R.FLOAT:
            side[b, row, h, 5] = float("inf")
        else:
            side[b, row, h, :2] = torch.tensor([0, 0x7e], dtype=torch.uint8)
        want[b, :, h * 2:h * 2 + 2] = True
    q[0, t - 1, 0, 3], q[1, 0, 3, 0] = float("nan"), float("-inf")
    want[0, t - 1, 0] = want[1, 0, 3] = True
    k, v = (R.handle(gpu, c.cuda(), kind, hd) for c in packed)
    got = gpu.attn_cross(q.cuda(), k, v).cpu()
    assert torch.equal(torch.isnan(got).all(-1), want) and torch.equal(torch.isnan(got).any(-1), want)
    got = gpu.attn_cross(q.cuda(), k, v, ints(17, 99)).cpu()      # (they are past the rows now)
    own = torch.zeros_like(want)
    own[0, t - 1, 0] = own[1, 0, 3] = True
    assert torch.equal(torch.isnan(got).any(-1), own)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t", [1, 40])
def test_states_of_all_sizes(gpu, kind, t):
    """Rows of very different sizes beside each other, zeros, and queries of all
    sizes: a row errs by its own values alone."""
    n, rows, heads, kv, hd = 2, 90, 4, 2, 64
    g = torch.Generator().manual_seed(t)
    big = 1e4 if kind == "f16" else 1e30
    for sizes, of_q in (([1.0, 1e-6, 0.0], 1.0), ([1e-3, 10.0], 100.0), ([1.0], 1e-20), ([1.0], 0.0)):
        k = torch.randn(n, rows, kv, hd, generator=g) * torch.tensor(sizes).repeat(rows)[:rows, None, None]
        v = torch.randn(n, rows, kv, hd, generator=g) * torch.tensor([1.0, 1.0 / big, big, 0.0]).repeat(rows)[:rows, None, None]
        packed = [R.pack(x, kind) for x in (k, v)]
        q = torch.randn(n, t, heads, hd, generator=g) * of_q
        y, bound = attend(q, *(R.values(c, kind) for c in packed), kind, [rows, 33], [t] * n, hd ** -0.5)
        got = gpu.attn_cross(q.cuda(), *(c.cuda() for c in packed), ints(rows, 33)).cpu().double()
        err = (got - y).abs()
        assert (err <= bound).all(), (sizes, of_q, float((err / bound.clamp_min(1e-300)).max()))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,rows", [(1, 300), (1, 9000), (40, 300), (40, 9000)])
@pytest.mark.parametrize("power", [5, 13, 16])
def test_large_scores_are_exact(gpu, kind, t, rows, power):
    """Scores of 2^12 to 2^23 whose softmax is known: with a scale of ln 2 they are q.k
    in powers of two, here whole numbers below 2^24 and so exact in f32, weights powers
    of two. What is left: the pieces of weights and, f32, of V (2^-22 of themselves, or
    2^-39 of the largest, f32's of the largest times its row's size), the sum over the
    rows, and 32 half steps of factors and joins."""
    heads, kv, hd = 4, 2, 64
    g = torch.Generator().manual_seed(power)
    k = torch.zeros(1, rows, kv, hd)
    k[..., 0] = torch.where(torch.rand(1, rows, kv, generator=g) < 0.02, 127, torch.randint(-127, 127, (1, rows, kv), generator=g))
    k[..., 1] = torch.randint(0, 6, (1, rows, kv), generator=g)
    v = R.pack(torch.randn(1, rows, kv, hd, generator=g), kind)
    q = torch.zeros(1, t, heads, hd)
    q[..., 0], q[..., 1] = 2.0 ** power, 1.0
    got = gpu.attn_cross(q.cuda(), R.pack(k, kind).cuda(), v.cuda(), scale=math.log(2)).cpu().double()
    s = (k[0, :, :, 0].double() * 2.0 ** power + k[0, :, :, 1].double()).T                  # (kv, rows)
    x = R.values(v, kind)[0].double().transpose(0, 1)
    w = torch.exp2(s - s.amax(1, keepdim=True))
    w = w / w.sum(1, keepdim=True)
    y, size, sums = (torch.bmm(a[:, None], b)[:, 0] for a, b in ((w, x), (w, x.abs()), (torch.ones_like(w), x.abs())))
    top = x.abs().amax(2)
    bound = (2.0 ** -22 + (rows + 32) * R.EPS) * size + 2.0 ** -39 * w.amax(1)[:, None] * sums
    if kind == "f32":
        bound = bound + (2.0 ** -25 * (w * top).sum(1) + rows * 2.0 ** -24 * (w * top).amax(1))[:, None]
    y, bound = (a.repeat_interleave(heads // kv, 0) for a in (y, bound))
    err = (got[0] - y).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "q4_0"])
def test_layouts(gpu, kind):
    """Head-major states, queries cut from a fused projection, and one sequence of
    states for all queries by a stride of 0."""
    heads, kv, hd, rows = 6, 2, 64, 70
    for t in (1, 50):
        check(gpu, kind, heads, kv, hd, t, rows, [70, 30], make=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2))
        fused = torch.randn(2, t, 3, heads, hd)
        check(gpu, kind, heads, kv, hd, t, rows, [70, 30], q=fused[:, :, 1])
        packed, values = states(kind, 1, rows, kv, hd, 9)
        k, v = (R.handle(gpu, c.cuda().expand(5, -1, -1, -1), kind, hd) for c in packed)
        q = torch.randn(5, t, heads, hd)
        y, bound = attend(q, *(x.expand(5, -1, -1, -1) for x in values), kind, [70, 1, 69, 0, 33], [t] * 5, hd ** -0.5)
        got = gpu.attn_cross(q.cuda(), k, v, ints(70, 1, 69, 0, 33)).cpu().double()
        assert ((got - y).abs() <= bound).all()


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [40, 3000])
def test_v_of_another_layout_than_k(gpu, kind, rows):
    """V's rows start where the kernel for few queries does not read them (an odd
    element of 16 bits; f32: heads of another length in the row), K's where it does."""
    heads, kv, hd = 4, 2, 64
    packed, values = states(kind, 2, rows, kv, hd, 9)
    k = packed[0].cuda()
    wide = torch.zeros(2, rows, kv, hd + 3, dtype=R.FLOAT[kind], device="cuda")
    v = wide[..., 1:hd + 1]
    v.copy_(packed[1])
    for t in (1, 3):
        q = torch.randn(2, t, heads, hd, generator=torch.Generator().manual_seed(t))
        y, bound = attend(q, *values, kind, [rows, rows // 2], [t, t], hd ** -0.5)
        for a, b in ((k, v), (k, packed[1].cuda())):
            got = gpu.attn_cross(q.cuda(), a, b, ints(rows, rows // 2)).cpu().double()
            assert ((got - y).abs() <= bound).all()


def test_a_decoder_layer_and_its_encoder_together(gpu):
    """An encoder's layer that looks both ways over its own q, k and v, the states
    stored in a cache by kv_store, and a decoder's tokens against them, beside the
    decoder's own attention; eagerly, and as one captured graph over new inputs."""
    n, rows, t, heads, hd, cap = 3, 50, 1, 4, 64, 20
    z = lambda *s: torch.zeros(*s, device="cuda")
    s = dict(q=z(n, rows, heads, hd), k=z(n, rows, heads, hd), v=z(n, rows, heads, hd), enc=z(n, rows, heads, hd), y=z(n, t, heads, hd),
             x=z(n, t, heads, hd), own=z(n, t, heads, hd), length=ints(*[0] * n), at=ints(*[0] * n), filled=ints(*[1] * n), zero=ints(*[0] * n))
    states_ = [z(n, rows, heads, hd).half() for _ in range(2)]
    cache = [z(n, cap, heads, hd).half() for _ in range(2)]
    work = [torch.empty(max(1, w), device="cuda") for w in (gpu.attn_cross_work(s["q"], s["k"]), gpu.attn_cross_work(s["x"], states_[0]),
                                                           gpu.attn_kv_work(s["x"], cache[0]))]

    def step():
        gpu.attn_cross(s["q"], s["k"], s["v"], s["length"], s["length"], out=s["enc"], work=work[0])
        gpu.kv_store(s["enc"], s["enc"], states_[0], states_[1], s["zero"], s["length"])
        gpu.kv_store(s["x"], s["x"], cache[0], cache[1], s["at"])
        gpu.attn_kv(s["x"], cache[0], cache[1], s["filled"], out=s["own"], work=work[2])
        gpu.attn_cross(s["own"], states_[0], states_[1], s["length"], out=s["y"], work=work[1])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator().manual_seed(4)
    for i in range(6):
        length = [[50, 3, 17], [1, 0, 49], [33, 33, 33]][i % 3]
        for name in ("q", "k", "v", "x"):
            s[name].copy_(torch.randn(s[name].shape, generator=g))
        s["length"].copy_(ints(*length)), s["at"].copy_(ints(i, i, i)), s["filled"].copy_(ints(i + 1, i + 1, i + 1))
        results = []
        for run in (step, graph.replay):
            s["enc"].fill_(9.25)
            run()
            results.append([s[name].cpu() for name in ("enc", "own", "y")])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        enc, own, y = results[0]
        q, k, v = (s[name].cpu() for name in ("q", "k", "v"))
        want, bound = attend(q, k, v, "f32", length, length, hd ** -0.5)
        live = ~torch.isnan(want)
        assert (enc[~live] == 9.25).all() and ((enc.double() - want)[live].abs() <= bound[live]).all()
        held = [enc.half().float(), enc.half().float()]
        want, bound = attend(own, *held, "f16", length, [t] * n, hd ** -0.5)
        assert ((y.double() - want).abs() <= bound).all()
