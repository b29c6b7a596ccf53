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
