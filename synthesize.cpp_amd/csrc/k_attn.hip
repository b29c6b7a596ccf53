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
#include "shp_attn.hpp"

namespace shp {
namespace {

// ---------------------------------------------------------------------------
// Any type, stride and alignment, for what the other kernels do not take (rows
// 16 MB and more apart, 16-bit rows of an odd length): a wave takes 16 rows and,
// of its split, 16 keys at a time, in F32 matrix instructions (16x16x4) fed value
// by value. Bound by those loads (2048 positions of 8 heads of 256 values over 4:
// 1.8 to 2.8 ms, MI355X).
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
    const int32_t base  = first_position(a, len);
    const int32_t p0    = position(a, base, t0);
    const int32_t p1    = position(a, base, t1);
    const bool    live  = t < len.count;
    const int32_t p     = live ? position(a, base, t) : -1;
    const int     head  = h * a.G + gq;
    const int     steps = (a.hd + 3) / 4;

    // An infinity in q or in a row of K is NaN to every query that sees the row,
    // also where its score would be -infinity.
    auto          or_nan = [](float x) { return fabsf(x) < INFINITY ? x : NAN; };
    float         qf[HD / 4];
    const float * qr = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
#pragma unroll
    for (int s = 0; s < HD / 4; ++s) {
        const int dim = 4 * s + g;
        qf[s]         = live && dim < a.hd ? or_nan(qr[dim]) * a.scale : 0.0f;
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
                const float kv  = has && dim < a.hd ? or_nan(kv_value<KIND>(kr, dim)) : 0.0f;
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
                    float         x = dim < a.hd && seen_by(a, p0, p1, j) ?
                                          kv_value<KIND>(vb + static_cast<int64_t>(j) * a.vt, dim) : 0.0f;
                    const uint64_t bad = __ballot(!(fabsf(x) < INFINITY));
                    if (bad != 0) {  // NaN for the queries that see it, and no others
                        x = fabsf(x) < INFINITY ? x : 0.0f;
#pragma unroll
                        for (int quarter = 0; quarter < 4; ++quarter) {
                            if ((bad >> (16 * quarter) & 0xffffu) != 0 && sees(a, p, j0 + 4 * quarter + s)) {
                                l = NAN;
                            }
                        }
                    }
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

// Parts of a row's result; one has been written to y.
__device__ __forceinline__ int parts_of(const AttnArgs & a, const SeqLens & len, const RowOf & r) {
    return a.per == 0 ? a.nsplit : wide_parts(a, len, (r.t * a.G + r.gq) / kWideRows);
}

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join(const AttnArgs a, int64_t row0) {
    const int64_t row = row0 + blockIdx.x;
    const RowOf   r   = row_of(a, row);
    const SeqLens len = seq_lens(a, r.n);
    if (r.t >= len.count) {
        return;
    }
    const int parts = parts_of(a, len, r);
    if (parts <= 1) {
        return;
    }
    join_parts<HD>(parts, a.hd, [&](int s) { return partial_ml(a, row, s); }, [&](int s) { return partial_o(a, row, s); },
                   out_of(a, r), position(a, first_position(a, len), r.t) >= 0);
}

// Many rows of a few parts: HD/4 lanes a row, each the row's weights for itself
// (16336 rows of four parts, MI355X: 9.7 us, 26 a workgroup a row).
constexpr int kFewParts = 8;

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join_rows(const AttnArgs a, int64_t row0) {
    constexpr int ROWS = kJoinThreads * 4 / HD;
    const int64_t row  = row0 + static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / (HD / 4);
    const int     dim  = threadIdx.x % (HD / 4) * 4;
    if (row >= static_cast<int64_t>(a.N) * a.KV * a.T * a.G || dim >= a.hd) {
        return;
    }
    const RowOf   r   = row_of(a, row);
    const SeqLens len = seq_lens(a, r.n);
    if (r.t >= len.count) {
        return;
    }
    const int parts = parts_of(a, len, r);
    if (parts <= 1) {
        return;
    }
    float m[kFewParts], l[kFewParts];
    f32x4 o[kFewParts];
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < kFewParts; ++s) {
        const int     p  = min(s, parts - 1);
        const float * ml = partial_ml(a, row, p);
        m[s]             = ml[0];
        l[s]             = s < parts ? ml[1] : 0.0f;
        o[s]             = s < parts ? *reinterpret_cast<const f32x4 *>(partial_o(a, row, p) + dim) : splat4(0.0f);
        top              = fmaxf(top, m[s]);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    float       sum = 0.0f;
    f32x4       v   = splat4(0.0f);
#pragma unroll
    for (int s = 0; s < kFewParts; ++s) {
        if (l[s] != 0.0f) {  // (no key, and nothing that counts in o)
            const float w = __builtin_amdgcn_exp2f(m[s] - ref);
            sum += w * l[s];
            v += o[s] * w;
        }
    }
    const float by  = over(sum, position(a, first_position(a, len), r.t) >= 0);
    float *     out = out_of(a, r) + dim;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (dim + e < a.hd) {
            out[e] = v[e] * by;
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// How many splits of the key axis give the chip work: `want` workgroups or
// waves in all, each with at least one of its `units`.
int32_t plan_splits(int64_t tiles, int64_t units, int64_t want) {
    int64_t n = (want + tiles - 1) / tiles;
    n         = n < units ? n : units;
    return static_cast<int32_t>(n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n);
}

// Positions and windows are int32, and so are their sums and differences.
constexpr int64_t kAttnMaxKeys = int64_t{ 1 } << 30;

// Whether k_attn_wide takes a cache: 64 rows lie at 32-bit offsets, and a row
// ends with a whole dword (the last that its descriptor lets through).
bool wide_takes(const shp_tensor & c) {
    return (c.ne[2] == 1 || c.nb[2] < (size_t{ 1 } << 24)) &&
           (kv_blocks(kv_kind(c.type)) || kv_bytes_of_row(c) % 4 == 0);
}

constexpr int64_t kWideSpan    = 2;    // key tiles at least: 300 positions take 20.9 us, with 3 23.4
constexpr int64_t kWhole       = 4;    // chunks a wave of a group of k_attn_few that is not split
constexpr int64_t kShortGroups = 256;  // its groups where a short cache is shared out by heads, at most
constexpr int64_t kFewGroups   = 256;  // parts of one of its groups that have one chunk a wave

// Workgroups of k_attn_wide that the chip holds.
int64_t wide_groups(int64_t hd) {
    return hd <= 4 * kKvBlock ? 512 : 256;
}

}  // namespace

// `rows` query rows of each of `pairs` (kv head, sequence), of T positions, over
// `keys` of `cap` rows, for a chip that holds `chip` workgroups.
void plan_spans(int64_t rows, int64_t T, int64_t cap, int64_t keys, int64_t pairs, int64_t chip, bool causal, AttnPlan & p) {
    // Splits of equally many key tiles for all rows, however many a row has,
    // as short as lets the chip hold all of them at once: 2048 positions of
    // 16 heads take 81 us, and 99 with every row in thirds (Q4_0, 8 kv heads,
    // MI355X). Where the row tiles alone are more than half of what it holds,
    // long rows are halved (2560 positions: 123 us, whole rows 169), and from
    // three quarters on all are left whole (3584 positions: 234 us, halves 264).
    const int64_t tiles = (rows + kWideRows - 1) / kWideRows;
    const int64_t most  = (keys + kTileKeys - 1) / kTileKeys + (p.window > 0 ? 2 : 0);
    int64_t       span  = (most + kMaxSplits - 1) / kMaxSplits;
    span                = span > kWideSpan ? span : kWideSpan;
    // Where all rows have all keys, whole rows from 3/8 of the chip on, or halves of long
    // ones while both are on it (4 x 510 queries over as many rows, 12 heads of 64, F16:
    // 22.0 us, halves 31.0; 2 x 1000 over 1500, 16 heads of 128 over 8, F32: halves 117, whole
    // 147, F16 78 and 75), and below that a workgroup for each CU (2 x 100 over 1500, F16:
    // 27.7 in sixths, 33 in twelfths). These three shapes are all that both sides were
    // measured at.
    const int64_t held = causal ? chip : chip / 2;
    if (!causal && tiles * pairs >= chip * 3 / 8) {
        span = tiles * pairs * 2 <= chip && most > 16 ? (most + 1) / 2 : most;
    } else if (tiles * pairs > chip * 3 / 4) {
        span = most;
    } else if (tiles * pairs > chip / 2) {
        span = span > (most + 1) / 2 ? span : (most + 1) / 2;
    } else {
        auto fits = [&](int64_t of) {
            int64_t groups = 0;
            for (int64_t t = 0; t < tiles && groups <= held; ++t) {
                // of a whole cache, and within a window all alike
                const int64_t end = causal ? cap - T + ((t + 1) * kWideRows * T + rows - 1) / rows : cap;
                const int64_t n   = ((end < cap ? end : cap) + kTileKeys - 1) / kTileKeys;
                groups += ((n < most ? n : most) + of - 1) / of * pairs;
            }
            return groups <= held;
        };
        for (int64_t upto = most; span < upto;) {  // the shortest that fits
            const int64_t mid = (span + upto) / 2;
            if (fits(mid)) {
                upto = mid;
            } else {
                span = mid + 1;
            }
        }
    }
    p.span   = static_cast<int32_t>(span < most ? span : most);
    p.nsplit = static_cast<int32_t>((most + p.span - 1) / p.span);
}

namespace {

shp_status_t plan_attn(const shp_tensor * q, const shp_tensor * k_cache, int32_t window, int32_t sinks, bool causal, AttnPlan & p) {
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
    const int64_t kv = k_cache->ne[1];
    const int64_t tiles16 = (rows + 15) / 16;
    p.few            = rows <= 16 && kv_blocks(kv_kind(k_cache->type));
    p.hgs            = 0;
    p.cross          = !causal && rows <= 16 && cross_few_takes(*k_cache);
    if (p.cross) {
        plan_cross_few(kv_kind(k_cache->type), q->ne[0], cap, kv * q->ne[3], p);
        p.few             = p.cross;
        const int64_t fit = p.wgs * 2 * kCols / (q->ne[1] * q->ne[2] * q->ne[3]);
        p.nsplit          = p.parts ? plan_splits(tiles16 * kv * q->ne[3], fit, 2048) : 1;
    } else if (p.few) {
        while ((rows << (p.hgs + 1)) <= 16 && kv % (int64_t{ 2 } << p.hgs) == 0 &&
               k_cache->nb[1] == kv_bytes_of_row(*k_cache)) {
            ++p.hgs;
        }
        const int waves  = few_waves(k_cache->ne[0]);
        auto      groups = [&] { return (kv >> p.hgs) * q->ne[3]; };
        auto      chunks = [&] { return ((keys << p.hgs) + kChunk - 1) / kChunk + (p.window > 0 ? 2 : 0); };
        // A short cache is shared out by heads, so that no group has more than a
        // chunk for each wave, rather than by keys (38 rows of 8 heads, MI355X:
        // 11.3 to 7.1 us a call).
        while (p.hgs > 0 && chunks() > waves && groups() * 2 <= kShortGroups && chunks() <= kWhole * waves << p.hgs &&
               (kv_bytes_of_row(*k_cache) << (p.hgs - 1)) % 16 == 0) {
            --p.hgs;
        }
        // up to kWhole chunks a wave a group is not split: that many take less than a second launch
        const int64_t deep  = chunks() <= kWhole * waves ? (chunks() + waves - 1) / waves : 1;
        const int64_t units = (chunks() + waves * deep - 1) / (waves * deep) * groups();
        p.per               = static_cast<int32_t>(waves * deep);
        p.few               = units < INT32_MAX;
        p.parts             = units > groups();
        p.groups            = static_cast<int32_t>(groups());
        // A chunk a wave, while a group has no more parts for its join than one of
        // a CU; past that two chunks (4000 rows of 12 heads of 64 values: 12.9 us,
        // 15.5 with two chunks; 8191 rows of 8 heads of 128: 17.3 us, 21.5 with one
        // chunk, 19.2 with three).
        const int64_t want = units > kFewGroups * groups() ? (units + 1) / 2 : units;
        const int64_t most = few_resident(kv_kind(k_cache->type), k_cache->ne[0]);
        p.wgs              = static_cast<int32_t>(want < most ? want : most);
        // where the caches' strides are not that kernel's: as many splits as its workspace holds
        const int64_t fit = p.wgs * 2 * kCols / (q->ne[1] * q->ne[2] * q->ne[3]);
        p.nsplit          = p.parts ? plan_splits(tiles16 * kv * q->ne[3], fit, 2048) : 1;
    }
    p.wide = !p.few && wide_takes(*k_cache);
    if (p.wide) {
        plan_spans(rows, T, cap, keys, kv * q->ne[3], wide_groups(q->ne[0]), causal, p);
    } else if (!p.few) {
        p.nsplit = plan_splits(tiles16 * kv * q->ne[3], (keys + 63) / 64, 2048);
    }
    return SHP_OK;
}

}  // namespace

int64_t plan_floats(const AttnPlan & p, const shp_tensor & q) {
    const int64_t row = (q.ne[0] + 3) / 4 * 4 + 2;
    if (p.few) {
        return !p.parts ? 0 : static_cast<int64_t>(p.wgs) * 2 * kCols * row + 2 * static_cast<int64_t>(p.groups);
    }
    return p.nsplit == 1 ? 0 : q.ne[1] * q.ne[2] * q.ne[3] * p.nsplit * row;
}

namespace {

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

}  // namespace

shp_status_t launch_join(const AttnArgs & a, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.N) * a.KV * a.T * a.G;
    auto          go   = [&](auto kernel) {
        return in_launches(rows, kJoinThreads, [&](int64_t first, dim3 grid) {
            hipLaunchKernelGGL(kernel, grid, dim3(kJoinThreads), 0, stream, a, first);
        });
    };
    if (a.nsplit <= kFewParts) {
        auto rows_a_block = [&](auto kernel, int each) {
            return in_launches((rows + each - 1) / each, kJoinThreads, [&](int64_t first, dim3 grid) {
                hipLaunchKernelGGL(kernel, grid, dim3(kJoinThreads), 0, stream, a, first * each);
            });
        };
        return a.hd <= 64  ? rows_a_block(k_attn_join_rows<64>, 16) :
               a.hd <= 128 ? rows_a_block(k_attn_join_rows<128>, 8) :
                             rows_a_block(k_attn_join_rows<256>, 4);
    }
    return a.hd <= 64 ? go(k_attn_join<64>) : a.hd <= 128 ? go(k_attn_join<128>) : go(k_attn_join<256>);
}

// The checks that shp_attn_kv, shp_attn_cross and shp_attn_pages share once a call is planned, and
// the arguments but for the cache's; `read`: what y and work may not overlap, beside q.
shp_status_t attn_args(const shp_tensor *         q,
                       const shp_tensor *         length,
                       const shp_tensor *         count,
                       float                      scale,
                       const AttnPlan &           p,
                       const shp_tensor * const * read,
                       int                        n_read,
                       const shp_tensor *         work,
                       const shp_tensor *         y,
                       AttnArgs &                 a) {
    // exp(x) = exp2(x log2 e)
    const float scale2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
    if (!well_formed(y) || !same_shape(*q, *y) || (length != nullptr && !kv_numbers(length, q->ne[3])) ||
        (count != nullptr && !kv_numbers(count, q->ne[3])) || !(fabsf(scale2) < INFINITY)) {
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
    for (int i = -2; i < n_read; ++i) {
        const shp_tensor * t = i == -2 ? q : i == -1 ? (floats > 0 ? work : nullptr) : read[i];
        if (t != nullptr && (kv_overlap(*y, *t) || (floats > 0 && t != work && kv_overlap(*work, *t)))) {
            return SHP_ERR_UNSUPPORTED;
        }
    }
    auto nb  = [](const shp_tensor & t, int d) { return static_cast<int64_t>(t.ne[d] > 1 ? t.nb[d] : 0); };
    a.q      = static_cast<const char *>(q->data);
    a.y      = static_cast<char *>(y->data);
    a.length = length != nullptr ? static_cast<const int32_t *>(length->data) : nullptr;
    a.count  = count != nullptr ? static_cast<const int32_t *>(count->data) : nullptr;
    a.work   = floats > 0 ? static_cast<float *>(work->data) : nullptr;
    a.qh = nb(*q, 1), a.qt = nb(*q, 2), a.qn = nb(*q, 3);
    a.yh = nb(*y, 1), a.yt = nb(*y, 2), a.yn = nb(*y, 3);
    a.scale  = scale2;
    a.window = p.window;
    a.sinks  = p.sinks;
    a.apart  = -1;
    a.T      = static_cast<int32_t>(q->ne[2]);
    a.N      = static_cast<int32_t>(q->ne[3]);
    a.hd     = static_cast<int32_t>(q->ne[0]);
    a.hd4    = (a.hd + 3) / 4 * 4;
    a.nsplit = p.nsplit;
    a.fsplit = make_fastdiv(static_cast<uint32_t>(a.nsplit > 0 ? a.nsplit : 1));
    return SHP_OK;
}

// Tiles of `rows` rows for a chip that holds `chip` workgroups, `per` key tiles a split.
void wide_args(int32_t per, int32_t rows, int64_t chip, AttnArgs & a) {
    a.tiles              = static_cast<int32_t>((static_cast<int64_t>(a.T) * a.G + rows - 1) / rows);
    a.per                = per;
    a.fper               = make_fastdiv(static_cast<uint32_t>(a.per));
    const int64_t groups = static_cast<int64_t>(a.tiles) * a.KV;
    // with all of them on the chip, two to a CU, a long row tile's neighbour is a
    // short one (4096 positions: 274 us, with the longest first throughout 287)
    const bool twos = a.nsplit == 1 && a.N == 1 && groups > chip / 2 && groups <= chip;
    a.half          = twos ? static_cast<int32_t>((chip / 2 + a.KV - 1) / a.KV) : a.tiles;
}

namespace {

shp_status_t attn_work(const shp_tensor * q, const shp_tensor * k_cache, int32_t window, int32_t sinks, bool causal, int64_t * floats) {
    AttnPlan p{};
    if (floats == nullptr) {
        return SHP_ERR_INVALID_ARG;
    }
    const shp_status_t st = plan_attn(q, k_cache, window, sinks, causal, p);
    if (st == SHP_OK) {
        *floats = plan_floats(p, *q);
    }
    return st;
}

shp_status_t attn(const shp_tensor * q,
                  const shp_tensor * k_cache,
                  const shp_tensor * v_cache,
                  const shp_tensor * length,
                  const shp_tensor * count,
                  float              scale,
                  int32_t            window,
                  int32_t            sinks,
                  bool               causal,
                  shp_tensor *       work,
                  shp_tensor *       y,
                  shp_stream_t       stream) {
    AttnPlan     p{};
    shp_status_t st = kv_check_caches(k_cache, v_cache);
    if (st == SHP_OK) {
        st = plan_attn(q, k_cache, window, sinks, causal, p);
    }
    if (st != SHP_OK) {
        return st;
    }
    AttnArgs           a{};
    const shp_tensor * read[4] = { k_cache, v_cache, length, count };
    st                         = attn_args(q, length, count, scale, p, read, 4, work, y, a);
    if (st != SHP_OK || dry_run()) {
        return st;
    }
    a.apart = causal ? -1 : 0;
    auto nb = [](const shp_tensor & t, int d) { return static_cast<int64_t>(t.ne[d] > 1 ? t.nb[d] : 0); };
    a.k     = static_cast<const char *>(k_cache->data);
    a.v     = static_cast<const char *>(v_cache->data);
    a.kh = nb(*k_cache, 1), a.kt = nb(*k_cache, 2), a.kn = nb(*k_cache, 3);
    a.vh = nb(*v_cache, 1), a.vt = nb(*v_cache, 2), a.vn = nb(*v_cache, 3);
    a.KV    = static_cast<int32_t>(k_cache->ne[1]);
    a.G     = static_cast<int32_t>(q->ne[1] / k_cache->ne[1]);
    a.cap   = static_cast<int32_t>(k_cache->ne[2]);
    a.tiles = static_cast<int32_t>((static_cast<int64_t>(a.T) * a.G + 15) / 16);
    a.fG    = make_fastdiv(static_cast<uint32_t>(a.G));
    a.fKV   = make_fastdiv(static_cast<uint32_t>(a.KV));
    const hipStream_t s     = as_stream(stream);
    const int         kind  = kv_kind(k_cache->type);
    int32_t           run   = 0;
    if (p.cross && cross_few_takes(*v_cache)) {
        return launch_cross_few(kind, a, p, s);
    }
    const int piece = p.few && !p.cross ? few_piece(*k_cache, *v_cache, p.hgs, run) : 0;
    if (piece > 0) {
        return launch_attn_few(kind, a, p, piece, run, s);
    }
    if (wide_takes(*k_cache) && wide_takes(*v_cache)) {
        int32_t per = p.span;
        if (!p.wide) {  // in place of k_attn_few: splits as its workspace has room for
            const int64_t most = (a.cap + kTileKeys - 1) / kTileKeys + 2;
            per                = static_cast<int32_t>((most + a.nsplit - 1) / a.nsplit);
        }
        wide_args(per, kWideRows, wide_groups(a.hd), a);
        st = launch_attn_wide(kind, a, s);
        return st == SHP_OK && a.nsplit > 1 ? launch_join(a, s) : st;
    }
    switch (kind) {
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

}  // namespace
}  // namespace shp

using namespace shp;

extern "C" shp_status_t shp_attn_kv_work(const shp_tensor * q,
                                         const shp_tensor * k_cache,
                                         int32_t            window,
                                         int32_t            sinks,
                                         int64_t *          floats) {
    return attn_work(q, k_cache, window, sinks, true, floats);
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
    return attn(q, k_cache, v_cache, length, count, scale, window, sinks, true, work, y, stream);
}

extern "C" shp_status_t shp_attn_cross_work(const shp_tensor * q, const shp_tensor * k, int64_t * floats) {
    return attn_work(q, k, 0, 0, false, floats);
}

extern "C" shp_status_t shp_attn_cross(const shp_tensor * q,
                                       const shp_tensor * k,
                                       const shp_tensor * v,
                                       const shp_tensor * length,
                                       const shp_tensor * count,
                                       float              scale,
                                       shp_tensor *       work,
                                       shp_tensor *       y,
                                       shp_stream_t       stream) {
    return attn(q, k, v, length, count, scale, 0, 0, false, work, y, stream);
}
