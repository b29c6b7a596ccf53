// Causal attention over a KV cache (shp_attn_kv): one pass over the rows that
// a tile of queries sees, with the running maximum and sum of the softmax.
//
//   s_j = scale * q.k_j      m = max s_j      l = sum e^(s_j - m)
//   y   = sum e^(s_j - m) v_j / l
//
// The rows r = t*G + g of a kv head are its G query heads at the positions t,
// so a tile of them reads each cache row once. Scores are kept transposed,
// S^T = K Q^T: a lane then holds scores of one query, and they are the second
// operand of O^T = V^T P^T as they stand, with the keys in the order that the
// first product left them in.
#include <climits>
#include <cmath>

#include "shp_kv.hpp"

namespace shp {
namespace {

struct AttnArgs {
    const char *    q;
    const char *    k;
    const char *    v;
    char *          y;
    const int32_t * length;  // or null: cap
    const int32_t * count;   // or null: T
    float *         work;    // partials of nsplit > 1: [rows][nsplit][hd], then m and l [rows][nsplit][2]
    int64_t         qh, qt, qn, kh, kt, kn, vh, vt, vn, yh, yt, yn;
    float           scale;  // times log2 e
    int32_t         window;  // 0: none
    int32_t         sinks;
    int32_t         T;
    int32_t         G;  // query heads of a kv head
    int32_t         KV;
    int32_t         N;
    int32_t         hd;
    int32_t         cap;
    int32_t         nsplit;
    int32_t         tiles;  // of rows
    FastDiv         fG;
    FastDiv         fsplit;
};

// The key tiles, KT rows each, that a tile of queries at positions p0..p1
// reads: [0, first) and then from second on; `n` in all.
struct KeyTiles {
    int32_t first;
    int32_t second;
    int32_t n;
};

template <int KT> __device__ __forceinline__ KeyTiles key_tiles(const AttnArgs & a, int32_t p0, int32_t p1) {
    KeyTiles s{ 0, 0, 0 };
    if (p1 < 0) {
        return s;
    }
    const int32_t last = p1 / KT;
    if (a.window > 0) {
        const int32_t lo = max(p0 - a.window + 1, 0);
        s.second         = lo / KT;
        s.first          = min((min(a.sinks, p1 + 1) + KT - 1) / KT, s.second);
    }
    s.n = s.first + last - s.second + 1;
    return s;
}

__device__ __forceinline__ int32_t key_tile(const KeyTiles & s, int32_t i) {
    return i < s.first ? i : s.second + i - s.first;
}

// Whether a query at p sees row j.
__device__ __forceinline__ bool sees(const AttnArgs & a, int32_t p, int32_t j) {
    return j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
}

// Whether a query of positions p0..p1 sees row j.
__device__ __forceinline__ bool seen_by(const AttnArgs & a, int32_t p0, int32_t p1, int32_t j) {
    return j <= p1 && (a.window == 0 || j > p0 - a.window || j < a.sinks);
}

// A sequence's filled rows and new positions.
struct SeqLens {
    int32_t length;
    int32_t count;
};

__device__ __forceinline__ SeqLens seq_lens(const AttnArgs & a, int n) {
    SeqLens s{ a.cap, a.T };
    if (a.length != nullptr) {
        s.length = min(max(a.length[n], 0), a.cap);
    }
    if (a.count != nullptr) {
        s.count = min(max(a.count[n], 0), a.T);
    }
    return s;
}

__device__ __forceinline__ float * partial_o(const AttnArgs & a, int64_t row, int split) {
    return a.work + (row * a.nsplit + split) * a.hd;
}

__device__ __forceinline__ float * partial_ml(const AttnArgs & a, int64_t row, int split) {
    const int64_t rows = static_cast<int64_t>(a.N) * a.KV * a.T * a.G;
    return a.work + rows * a.nsplit * a.hd + (row * a.nsplit + split) * 2;
}

// The maximum, or the sum, over the four lanes c, c+16, c+32, c+48.
__device__ __forceinline__ float max_quarters(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float sum_quarters(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// What a row's softmax comes to: 1/l, or 0 where the row sees nothing. A row
// whose scores are all -infinity has no softmax: 0/0.
__device__ __forceinline__ float over(float l, bool sees_any) {
    return l == 0.0f && !sees_any ? 0.0f : 1.0f / l;
}

// ---------------------------------------------------------------------------
// Any type, stride and alignment: a wave takes 16 rows and, of its split, 16
// keys at a time, in F32 matrix instructions (16x16x4) fed value by value.
// ---------------------------------------------------------------------------

template <int KIND, int HD> __global__ __launch_bounds__(64) void k_attn_any(const AttnArgs a) {
    constexpr int KT    = 16;
    const int     lane  = threadIdx.x;
    const int     c     = lane & 15;
    const int     g     = lane >> 4;
    const int     tile  = static_cast<int>(fastdiv(blockIdx.x, a.fsplit));
    const int     split = static_cast<int>(blockIdx.x) - tile * a.nsplit;
    const int     h     = blockIdx.y;
    const int     n     = blockIdx.z;
    const SeqLens len   = seq_lens(a, n);
    const int     r     = tile * 16 + c;
    const int     t     = static_cast<int>(fastdiv(static_cast<uint32_t>(r), a.fG));
    const int     gq    = r - t * a.G;
    const int     t0    = static_cast<int>(fastdiv(static_cast<uint32_t>(tile * 16), a.fG));
    if (t0 >= len.count) {
        return;
    }
    const int     t1    = min(static_cast<int>(fastdiv(static_cast<uint32_t>(tile * 16 + 15), a.fG)), len.count - 1);
    const int32_t base  = len.length - len.count;
    const int32_t p0    = base + t0;
    const int32_t p1    = base + t1;
    const bool    live  = t < len.count;
    const int32_t p     = live ? base + t : -1;
    const int     head  = h * a.G + gq;
    const int     steps = (a.hd + 3) / 4;

    float         qf[HD / 4];
    const float * qr = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
#pragma unroll
    for (int s = 0; s < HD / 4; ++s) {
        const int dim = 4 * s + g;
        qf[s]         = live && dim < a.hd ? qr[dim] * a.scale : 0.0f;
    }
    f32x4 o[HD / 16];
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) {
        o[u] = splat4(0.0f);
    }
    float          m  = -INFINITY;
    float          l  = 0.0f;
    const KeyTiles kt = key_tiles<KT>(a, p0, p1);
    const int      per = (kt.n + a.nsplit - 1) / a.nsplit;
    const int      end = min(kt.n, (split + 1) * per);
    const char *   kb  = a.k + n * a.kn + h * a.kh;
    const char *   vb  = a.v + n * a.vn + h * a.vh;
    for (int i = split * per; i < end; ++i) {
        const int32_t j0  = key_tile(kt, i) * KT;
        const int32_t jr  = j0 + c;
        const char *  kr  = kb + static_cast<int64_t>(jr) * a.kt;
        const bool    has = jr < len.length;
        f32x4         acc = splat4(0.0f);
#pragma unroll
        for (int s = 0; s < HD / 4; ++s) {
            if (s < steps) {
                const int   dim = 4 * s + g;
                const float kv  = has && dim < a.hd ? kv_value<KIND>(kr, dim) : 0.0f;
                acc             = __builtin_amdgcn_mfma_f32_16x16x4f32(kv, qf[s], acc, 0, 0, 0);
            }
        }
        float top = m;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[e] = sees(a, p, j0 + 4 * g + e) ? acc[e] : -INFINITY;
            top    = fmaxf(top, acc[e]);
        }
        top               = max_quarters(top);
        const float ref   = top == -INFINITY ? 0.0f : top;
        const float alpha = exp2f(m - ref);
        m                 = top;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[e] = exp2f(acc[e] - ref);
            l += acc[e];
        }
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) {
            if (16 * u < a.hd) {
                o[u] *= alpha;
                const int dim = 16 * u + c;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int32_t j = j0 + 4 * g + s;
                    const float   x = dim < a.hd && seen_by(a, p0, p1, j) ?
                                          kv_value<KIND>(vb + static_cast<int64_t>(j) * a.vt, dim) : 0.0f;
                    o[u]            = __builtin_amdgcn_mfma_f32_16x16x4f32(x, acc[s], o[u], 0, 0, 0);
                }
            }
        }
    }
    l = sum_quarters(l);
    if (!live) {
        return;
    }
    const int64_t row = ((static_cast<int64_t>(n) * a.KV + h) * a.T + t) * a.G + gq;
    float *       out;
    float         by = 1.0f;
    if (a.nsplit == 1) {
        out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
        by  = over(l, p >= 0);
    } else {
        out = partial_o(a, row, split);
        if (g == 0) {
            float * ml = partial_ml(a, row, split);
            ml[0]      = m;
            ml[1]      = l;
        }
    }
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int dim = 16 * u + 4 * g + e;
            if (dim < a.hd) {
                out[dim] = o[u][e] * by;
            }
        }
    }
}

// The splits of a row joined: a wave a row.
__global__ __launch_bounds__(256) void k_attn_join(const AttnArgs a, int64_t row0) {
    const int64_t rows = static_cast<int64_t>(a.N) * a.KV * a.T * a.G;
    const int64_t row  = row0 + static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    const int     lane = threadIdx.x % kWave;
    if (row >= rows) {
        return;
    }
    const int64_t gq   = row % a.G;
    const int64_t t    = row / a.G % a.T;
    const int64_t h    = row / a.G / a.T % a.KV;
    const int     n    = static_cast<int>(row / a.G / a.T / a.KV);
    const SeqLens len  = seq_lens(a, n);
    if (t >= len.count) {
        return;
    }
    float top = -INFINITY;
    for (int s = lane; s < a.nsplit; s += kWave) {
        top = fmaxf(top, partial_ml(a, row, s)[0]);
    }
    top             = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float       l   = 0.0f;
    for (int s = lane; s < a.nsplit; s += kWave) {
        const float * ml = partial_ml(a, row, s);
        l += ml[1] * exp2f(ml[0] - ref);
    }
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        l += __shfl_xor(l, off);
    }
    const float by  = over(l, len.length - len.count + t >= 0);
    float *     out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + (h * a.G + gq) * a.yh);
    for (int dim = lane; dim < a.hd; dim += kWave) {
        float v = 0.0f;
        for (int s = 0; s < a.nsplit; ++s) {
            const float * ml = partial_ml(a, row, s);
            if (ml[1] != 0.0f) {
                v += partial_o(a, row, s)[dim] * exp2f(ml[0] - ref);
            }
        }
        out[dim] = v * by;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// How many splits of the key axis give the chip work: a few waves for each of
// its 256 CUs, of at least 64 keys each.
int32_t plan_splits(int64_t tiles, int64_t keys) {
    const int64_t want = (2048 + tiles - 1) / tiles;
    const int64_t most = (keys + 63) / 64;
    const int64_t n    = want < most ? want : most;
    return static_cast<int32_t>(n < 1 ? 1 : n > 128 ? 128 : n);
}

// Positions and windows are int32, and so are their sums and differences.
constexpr int64_t kAttnMaxKeys = int64_t{ 1 } << 30;

struct AttnPlan {
    int32_t window;
    int32_t sinks;
    int32_t tiles;
    int32_t nsplit;
};

shp_status_t plan_attn(const shp_tensor * q, const shp_tensor * k_cache, int32_t window, int32_t sinks, AttnPlan & p) {
    if (!well_formed(q) || !kv_well_formed(k_cache) || q->ne[0] != k_cache->ne[0] || q->ne[1] % k_cache->ne[1] != 0 ||
        q->ne[3] != k_cache->ne[3] || window < 0 || sinks < 0) {
        return SHP_ERR_INVALID_ARG;
    }
    if (q->type != SHP_TYPE_F32 || q->ne[0] > kKvMaxDim || q->ne[1] > kKvMaxSeqs || q->ne[3] > kKvMaxSeqs ||
        q->ne[2] > kKvMaxRows / q->ne[1] || k_cache->ne[2] > kAttnMaxKeys || !kv_addressable(*q) ||
        !kv_addressable(*k_cache)) {
        return SHP_ERR_UNSUPPORTED;
    }
    const int64_t cap  = k_cache->ne[2];
    const int64_t T    = q->ne[2];
    const int64_t rows = q->ne[1] / k_cache->ne[1] * T;
    p.window           = window >= cap ? 0 : window;  // every row is within it
    p.sinks            = static_cast<int32_t>(sinks < cap ? sinks : cap);
    int64_t keys       = cap;
    if (p.window > 0 && p.window + p.sinks + T < keys) {
        keys = p.window + p.sinks + T;
    }
    p.tiles  = static_cast<int32_t>((rows + 15) / 16);
    p.nsplit = plan_splits(p.tiles * k_cache->ne[1] * q->ne[3], keys);
    return SHP_OK;
}

int64_t plan_floats(const AttnPlan & p, const shp_tensor & q) {
    return p.nsplit == 1 ? 0 : q.ne[1] * q.ne[2] * q.ne[3] * p.nsplit * (q.ne[0] + 2);
}

template <int KIND> shp_status_t launch_any(const AttnArgs & a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.tiles) * static_cast<unsigned>(a.nsplit), static_cast<unsigned>(a.KV),
                    static_cast<unsigned>(a.N));
    if (a.hd <= 64) {
        hipLaunchKernelGGL((k_attn_any<KIND, 64>), grid, dim3(64), 0, stream, a);
    } else if (a.hd <= 128) {
        hipLaunchKernelGGL((k_attn_any<KIND, 128>), grid, dim3(64), 0, stream, a);
    } else {
        hipLaunchKernelGGL((k_attn_any<KIND, 256>), grid, dim3(64), 0, stream, a);
    }
    return launch_status();
}

shp_status_t launch_join(const AttnArgs & a, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.N) * a.KV * a.T * a.G;
    return in_launches((rows + 3) / 4, 256, [&](int64_t first, dim3 grid) {
        hipLaunchKernelGGL(k_attn_join, grid, dim3(256), 0, stream, a, first * 4);
    });
}

}  // namespace
}  // namespace shp

using namespace shp;

extern "C" shp_status_t shp_attn_kv_work(const shp_tensor * q,
                                         const shp_tensor * k_cache,
                                         int32_t            window,
                                         int32_t            sinks,
                                         int64_t *          floats) {
    AttnPlan p{};
    if (floats == nullptr) {
        return SHP_ERR_INVALID_ARG;
    }
    const shp_status_t st = plan_attn(q, k_cache, window, sinks, p);
    if (st == SHP_OK) {
        *floats = plan_floats(p, *q);
    }
    return st;
}

extern "C" shp_status_t shp_attn_kv(const shp_tensor * q,
                                    const shp_tensor * k_cache,
                                    const shp_tensor * v_cache,
                                    const shp_tensor * length,
                                    const shp_tensor * count,
                                    float              scale,
                                    int32_t            window,
                                    int32_t            sinks,
                                    shp_tensor *       work,
                                    shp_tensor *       y,
                                    shp_stream_t       stream) {
    AttnPlan     p{};
    shp_status_t st = kv_check_caches(k_cache, v_cache);
    if (st == SHP_OK) {
        st = plan_attn(q, k_cache, window, sinks, p);
    }
    if (st != SHP_OK) {
        return st;
    }
    if (!well_formed(y) || !same_shape(*q, *y) || (length != nullptr && !kv_numbers(length, q->ne[3])) ||
        (count != nullptr && !kv_numbers(count, q->ne[3])) || !(fabsf(scale) < INFINITY)) {
        return SHP_ERR_INVALID_ARG;
    }
    const int64_t floats = plan_floats(p, *q);
    if (floats > 0 && (!well_formed(work) || work->type != SHP_TYPE_F32 || !contiguous(*work) || nelements(*work) < floats)) {
        return SHP_ERR_INVALID_ARG;
    }
    if (y->type != SHP_TYPE_F32 || !kv_aligned(*q) || !kv_aligned(*y) || !kv_addressable(*y) || !kv_rows_apart(*y) ||
        (length != nullptr && !i32_aligned(*length)) || (count != nullptr && !i32_aligned(*count)) ||
        (floats > 0 && !rows_aligned(*work, 16))) {
        return SHP_ERR_UNSUPPORTED;
    }
    const shp_tensor * others[6] = { q, k_cache, v_cache, length, count, floats > 0 ? work : nullptr };
    for (const shp_tensor * t : others) {
        if (t != nullptr && (kv_overlap(*y, *t) || (floats > 0 && t != work && kv_overlap(*work, *t)))) {
            return SHP_ERR_UNSUPPORTED;
        }
    }
    if (dry_run()) {
        return SHP_OK;
    }
    auto nb = [](const shp_tensor & t, int d) { return static_cast<int64_t>(t.ne[d] > 1 ? t.nb[d] : 0); };
    AttnArgs a{};
    a.q      = static_cast<const char *>(q->data);
    a.k      = static_cast<const char *>(k_cache->data);
    a.v      = static_cast<const char *>(v_cache->data);
    a.y      = static_cast<char *>(y->data);
    a.length = length != nullptr ? static_cast<const int32_t *>(length->data) : nullptr;
    a.count  = count != nullptr ? static_cast<const int32_t *>(count->data) : nullptr;
    a.work   = floats > 0 ? static_cast<float *>(work->data) : nullptr;
    a.qh = nb(*q, 1), a.qt = nb(*q, 2), a.qn = nb(*q, 3);
    a.kh = nb(*k_cache, 1), a.kt = nb(*k_cache, 2), a.kn = nb(*k_cache, 3);
    a.vh = nb(*v_cache, 1), a.vt = nb(*v_cache, 2), a.vn = nb(*v_cache, 3);
    a.yh = nb(*y, 1), a.yt = nb(*y, 2), a.yn = nb(*y, 3);
    a.scale  = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);  // exp(x) = exp2(x log2 e)
    a.window = p.window;
    a.sinks  = p.sinks;
    a.T      = static_cast<int32_t>(q->ne[2]);
    a.KV     = static_cast<int32_t>(k_cache->ne[1]);
    a.G      = static_cast<int32_t>(q->ne[1] / k_cache->ne[1]);
    a.N      = static_cast<int32_t>(q->ne[3]);
    a.hd     = static_cast<int32_t>(q->ne[0]);
    a.cap    = static_cast<int32_t>(k_cache->ne[2]);
    a.nsplit = p.nsplit;
    a.tiles  = p.tiles;
    a.fG     = make_fastdiv(static_cast<uint32_t>(a.G));
    a.fsplit = make_fastdiv(static_cast<uint32_t>(a.nsplit));
    const hipStream_t s = as_stream(stream);
    switch (kv_kind(k_cache->type)) {
        case kKvF32:
            st = launch_any<kKvF32>(a, s);
            break;
        case kKvF16:
            st = launch_any<kKvF16>(a, s);
            break;
        case kKvBF16:
            st = launch_any<kKvBF16>(a, s);
            break;
        case kKvQ8:
            st = launch_any<kKvQ8>(a, s);
            break;
        default:
            st = launch_any<kKvQ4>(a, s);
            break;
    }
    return st == SHP_OK && a.nsplit > 1 ? launch_join(a, s) : st;
}
