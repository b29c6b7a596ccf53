// Causal attention over a paged cache in 8 bits (shp_attn_pages). As in k_attn.hip
// scores are kept transposed, S^T = K Q^T, then O^T = V^T P^T, and the rows r = t*G +
// g of a kv head are its G query heads at the positions t.
//
// A block's codes are exact as F16, so K and V are one piece each; q and the weights
// are two. A block's scale is one number for sixteen rows and more: K's goes into the
// scores, V's into the weights,
//   s_j = (q.c_j) d_k     w_j = 2^(s_j - m) d_v 2^(14 - x)     l = sum 2^(s_j - m)
// where m is the query's largest score so far and x what the largest of 2^(s_j - m)
// d_v needs: with e the exponent of d_v, x = max(s_j - m + e), so that w_j stays
// below 2^15, and its pieces lose at most 2^-39 of the largest. m and x are of each query's own: what one
// does not see has no part in it. A sum that has a weight of NaN is NaN.
//
// Tokens are put into a score matrix in an order of their own: the result of S^T
// leaves a lane with rows 4 g + e (of 16; 8 q + 4 g + e of 32) of every tile, and
// the second product wants eight or sixteen tokens that follow each other in
// V's columns. So row 4 a + b of tile t is token 16 a + 4 t + b (few), and row 8 q +
// 4 g + b token 16 g + 4 q + b (many): a lane then holds the scores of sixteen
// tokens that follow each other, in one block, and V's columns are operands as they lie.
#include "shp_attn.hpp"
#include "shp_pages.hpp"

namespace shp {
namespace {

struct PagesArgs {
    FewArgs f;
    Pool    pool;
    Tables  tables;
};

// Eight codes as an operand: with their top bits turned they are code + 128, which
// under the exponent bytes of 1024 is 1152 + code.
__device__ __forceinline__ f16x8 operand(const Magic & m, uint32_t w0, uint32_t w1) {
    constexpr uint32_t kLow = 0x05010500u, kHigh = 0x05030502u;  // bytes 0 and 1, or 2 and 3, each below the exponent's
    auto               two  = [&](uint32_t w, uint32_t which) { return as_f16x2(__builtin_amdgcn_perm(m.e1024, w, which)) - splat2(1152.0f); };
    const uint32_t     a    = w0 ^ 0x80808080u;
    const uint32_t     b    = w1 ^ 0x80808080u;
    return join8(two(a, kLow), two(a, kHigh), two(b, kLow), two(b, kHigh));
}

// split2() in fewer instructions: the rest by a mixed multiply-add, which is exact as well.
__device__ __forceinline__ void split_weights(float a, float b, f16x2 & hi, f16x2 & lo) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    hi = __builtin_convertvector((f32x2{ a, b }), f16x2);
    lo = __builtin_convertvector((f32x2{ __builtin_fmaf(static_cast<float>(hi[0]), -1.0f, a), __builtin_fmaf(static_cast<float>(hi[1]), -1.0f, b) }), f16x2);
}

// A page's number, or what it is to be read as: 0 for one outside the pool.
struct PageId {
    int32_t id;
    bool    in;
};

__device__ __forceinline__ PageId page_id(const PagesArgs & p, int32_t entry) {
    const bool in = static_cast<uint32_t>(entry) < static_cast<uint32_t>(p.pool.pages);
    return PageId{ in ? entry : 0, in };
}

__device__ __forceinline__ int32_t entry_of(const PagesArgs & p, const int32_t * table, int32_t row) {
    return table[min(row >> p.pool.shift, p.tables.most - 1)];
}

// A block's scale as it is read. (What it counts as is formed where it is used: that waits
// for the load.)
__device__ __forceinline__ float scale_at(const PoolSide & s, const PageId & page, int h) {
    return s.scale[page.id * s.sp + h];
}

__device__ __forceinline__ float scale_of(float read, bool in) {
    return in ? block_scale(read) : NAN;
}

// d_k times what brings q back, within what is a normal number: with sums of
// products below 2^29 nothing is lost at the lower end, and at the upper one 0
// times it stays 0. A NaN stays one.
__device__ __forceinline__ float score_scale(float d, float by) {
    const float f = d * by;
    return f < 0x1p-126f ? 0x1p-126f : f > 0x1.fffffep127f ? 0x1.fffffep127f : f;
}

constexpr float kTopWeight = 14.0f;    // weights reach 2^14 and stay below 2^15
constexpr float kLeastX    = -100.0f;  // of scales of 2^-100 and less

// 2^(s - m) to w: d_v 2^(14 - x). A group of tokens that is not seen counts for
// nothing whatever its scale is.
__device__ __forceinline__ float weight_scale(float d, float x, bool any) {
    const float f = d * __builtin_amdgcn_exp2f(kTopWeight - x);
    return !any ? 0.0f : f > 0x1.fffffep127f ? 0x1.fffffep127f : f;
}

// A partial result's weights are times 2^-k, so that with values up to f32's largest
// neither it nor the sum over all parts passes that: its largest score is m + k
// then, which is exact enough while m is below 2^22 (from there on k is 0). A sum is
// brought back by 2^(x - 14) after that, or after 1/l: their product, of two numbers far
// below 1, may itself be next to nothing or 0 where the result is neither.
__device__ __forceinline__ float part_shift(float m, float l) {
    return fabsf(m) < 0x1p22f ? static_cast<float>(exponent_of(l) + 12) : 0.0f;
}

// ---------------------------------------------------------------------------
// Few queries (decoding): at most 16 columns, the queries of one kv head. A wave
// takes 64 tokens at a time and reads them from the pool straight into the operands'
// registers, 16 bytes a lane, K's of the next 64 ahead of the exponentials and V's
// ahead of the next scores. 64 streams of 512 to 8192 rows (16 heads of 128 values over 8,
// MI355X) take 115 us, 5.0 TB/s; 38 rows 8.0 us, in which the length, the
// table, the codes, two products and the waves' join follow each other.
// ---------------------------------------------------------------------------

constexpr int kPageChunk  = 64;
constexpr int kPageWaves  = 4;

// hd is HD, or (FULL false) some less: then dimensions past it are read from
// the row's first ones, against zeros in q.
template <int HD, bool FULL>
__global__ __launch_bounds__(64 * kPageWaves, HD <= 128 ? 2 : 1) void k_attn_pages_few(const PagesArgs p) {
    constexpr int KS    = HD / 64;
    constexpr int TILES = HD / 16;
    extern __shared__ __align__(16) char lds[];
    const FewArgs &  f     = p.f;
    const AttnArgs & a     = f.a;
    const int        wave  = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int        lane  = threadIdx.x % kWave;
    const int        c     = lane & 15;
    const int        g     = lane >> 4;
    const int        wg    = blockIdx.x;
    const int        hd    = FULL ? HD : a.hd;
    const int        page  = 1 << p.pool.shift;
    const Line       line  = few_line(f, wg, lane);
    const int32_t    last  = line.end;
    int32_t          unit  = line.begin;
    const Magic      magic;

    // this lane's query; its row of K in a tile of 16
    const int  t    = static_cast<int>(fastdiv(static_cast<uint32_t>(c), a.fG));
    const int  gq   = c - t * a.G;
    const int  krow = 16 * (c >> 2);
    if (unit >= last) {
        return;
    }
    Place   at    = line.at;
    int     n     = at.n;
    int     h     = f.groups == 1 ? 0 : (unit - at.before) / at.units;
    int32_t begin = at.before + h * at.units;
    for (;;) {
        const int     u0  = unit - begin;
        const int     u1  = min(last - begin, at.units);
        const SeqLens len = seq_lens(a, n);
        if (a.work != nullptr && u0 == 0 && threadIdx.x == 0) {
            few_span(f, n * f.groups + h)[0] = wg;
            few_span(f, n * f.groups + h)[1] = few_owner(f, line.total, begin + at.units - 1);
        }
        const KeyTiles  kt    = few_tiles(f, len);
        const int32_t   base  = len.length - len.count;
        const int32_t   p1    = len.length - 1;
        const bool      live  = c < f.cols && t < len.count;
        const int32_t   pos   = live ? base + t : -1;
        const int       head  = h * a.G + gq;
        const int32_t * table = table_of(p.tables, n);
        const PoolSide & ks   = p.pool.side[0];
        const PoolSide & vs   = p.pool.side[1];
        const char *    kb    = ks.codes + h * ks.ch;
        const char *    vb    = vs.codes + h * vs.ch;

        f32x4 o[TILES];
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            o[u] = splat4(0.0f);
        }
        float m = -INFINITY;
        float x = kLeastX;
        float l = 0.0f;

        const int end = min(kt.n, u1 * f.per);
        int       i   = u0 * f.per + wave;

        // the entries of the tables for K's rows and V's columns, the codes and the
        // scales of a chunk
        int32_t ke = 0, ve = 0;
        u32x4   kr[4][KS];
        u32x4   vr[TILES];
        float   dk = 0.0f, dv = 0.0f;
        bool    in = true;  // (of K's and V's scales: one block)
        auto    first_of = [&](int32_t tile) { return key_tile(kt, tile) * kPageChunk; };
        auto    entries  = [&](int32_t tile) {
            const int32_t j0 = first_of(tile);
            ke               = entry_of(p, table, j0 + krow);
            ve               = entry_of(p, table, j0 + 16 * g);
        };
        auto fetch_k = [&](int32_t tile) {
            const int32_t j0   = first_of(tile);
            const PageId  id   = page_id(p, ke);
            const char *  from = kb + id.id * ks.cp + (((j0 + krow) & (page - 1)) + (c & 3)) * hd;
            const PageId  own  = page_id(p, ve);
            dk                 = scale_at(ks, own, h);
            in                 = own.in;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int dim = 64 * s + 16 * g;
                    kr[x][s]      = *reinterpret_cast<const u32x4 *>(from + 4 * x * hd + (FULL || dim < hd ? dim : 0));
                }
            }
        };
        auto fetch_v = [&](int32_t tile) {
            const int32_t j0   = first_of(tile);
            const PageId  id   = page_id(p, ve);
            const char *  from = vb + id.id * vs.cp + ((j0 + 16 * g) & (page - 1)) + c * page;
            dv                 = scale_at(vs, id, h);
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                if (FULL || 16 * u < hd) {
                    vr[u] = *reinterpret_cast<const u32x4 *>(from + 16 * u * page);
                }
            }
        };
        if (i < end) {
            entries(i);
            fetch_k(i);
            fetch_v(i);
            if (i + kPageWaves < end) {
                entries(i + kPageWaves);
            }
        }

        // the queries' operands: the largest value of each scaled to [2^13, 2^14)
        f16x8 qh[2 * KS], ql[2 * KS];
        float qscale;
        {
            const float * qr = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
            float         q[2 * KS][8];
            float         top = 0.0f;
#pragma unroll
            for (int s = 0; s < 2 * KS; ++s) {
                const int   dim = 64 * (s / 2) + 16 * g + 8 * (s % 2);
                const bool  has = live && (FULL || dim < hd);
                const f32x4 x0  = has ? ld4u(qr + dim) : splat4(0.0f);
                const f32x4 x1  = has ? ld4u(qr + dim + 4) : splat4(0.0f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    q[s][e] = (e < 4 ? x0[e] : x1[e - 4]) * a.scale;
                    top     = fmaxf(top, fabsf(q[s][e]));
                }
            }
            top            = max_quarters(top);
            const int   ex = exponent_of(top) - 13;
            const float to = pow2(-ex);
            qscale         = pow2(ex);
#pragma unroll
            for (int s = 0; s < 2 * KS; ++s) {
                f16x2 hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    split2(q[s][2 * e] * to, q[s][2 * e + 1] * to, hi[e], lo[e]);
                }
                qh[s] = join8(hi[0], hi[1], hi[2], hi[3]);
                ql[s] = join8(lo[0], lo[1], lo[2], lo[3]);
            }
        }

        // a chunk, and (MORE) the next one's codes on their way
        auto chunk = [&](auto more) {
            constexpr bool MORE = decltype(more)::value;
            const int32_t  j0   = first_of(i);
            f32x4          sc[4] = { splat4(0.0f), splat4(0.0f), splat4(0.0f), splat4(0.0f) };
#pragma unroll
            for (int s = 0; s < 2 * KS; ++s) {
                f16x8 k[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    k[x] = operand(magic, kr[x][s / 2][2 * (s % 2)], kr[x][s / 2][2 * (s % 2) + 1]);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    sc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[x], qh[s], sc[x], 0, 0, 0);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    sc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[x], ql[s], sc[x], 0, 0, 0);
                }
            }
            const float by = score_scale(scale_of(dk, in), qscale);
            const float d  = scale_of(dv, in);
            if constexpr (MORE) {
                fetch_k(i + kPageWaves);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                sc[x] *= by;  // (rounded as the largest is: what is subtracted from it leaves no score above 0)
            }
            const bool all = j0 + kPageChunk - 1 <= base && (a.window == 0 || j0 > p1 - a.window || j0 + kPageChunk <= a.sinks);
            if (!all) {
                int g16 = 16 * g;
                asm volatile("" : "+v"(g16));  // (the rows' keys are not to wait in registers for this)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[x][e] = sees(a, pos, j0 + g16 + 4 * x + e) ? sc[x][e] : -INFINITY;
                    }
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    top = fmaxf(top, sc[x][e]);
                }
            }
            const bool any = top != -INFINITY;
            const float most = fmaxf(m, max_quarters(top));
            const float ref  = most == -INFINITY ? 0.0f : most;
            const float down = m - ref;  // -infinity before the first
            const float need = max_quarters(top - ref + static_cast<float>(exponent_of(d)));
            const float now  = fmaxf(fmaxf(x + down, need), kLeastX);
            if (__any(down != 0.0f || now != x)) {
                l *= __builtin_amdgcn_exp2f(down);
                const float turn = __builtin_amdgcn_exp2f(down + x - now);
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    o[u] *= turn;
                }
            }
            m = most;
            x = now;
            const float wf = weight_scale(d, x, any);
            f16x2       ph[8], pl[8];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(sc[y][e] - ref);
                    l += w[e];
                    w[e] *= wf;
                }
                split_weights(w[0], w[1], ph[2 * y], pl[2 * y]);
                split_weights(w[2], w[3], ph[2 * y + 1], pl[2 * y + 1]);
            }
            constexpr int kAtOnce = 4;  // tiles of V whose products take turns
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const f16x8 bh = join8(ph[4 * half], ph[4 * half + 1], ph[4 * half + 2], ph[4 * half + 3]);
                const f16x8 bl = join8(pl[4 * half], pl[4 * half + 1], pl[4 * half + 2], pl[4 * half + 3]);
#pragma unroll
                for (int u = 0; u < TILES; u += kAtOnce) {
                    if (FULL || 16 * u < hd) {
                        f16x8 v[kAtOnce];
#pragma unroll
                        for (int k = 0; k < kAtOnce; ++k) {
                            v[k] = operand(magic, vr[u + k][2 * half], vr[u + k][2 * half + 1]);
                        }
#pragma unroll
                        for (int k = 0; k < kAtOnce; ++k) {
                            o[u + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], bh, o[u + k], 0, 0, 0);
                        }
#pragma unroll
                        for (int k = 0; k < kAtOnce; ++k) {
                            o[u + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[k], bl, o[u + k], 0, 0, 0);
                        }
                    }
                }
            }
            if constexpr (MORE) {
                fetch_v(i + kPageWaves);
            }
        };
        for (; i + kPageWaves < end; i += kPageWaves) {
            chunk(std::true_type{});
            if (i + 2 * kPageWaves < end) {
                entries(i + 2 * kPageWaves);
            }
        }
        if (i < end) {
            chunk(std::false_type{});
        }
        l = sum_quarters(l);

        // the waves' results joined in LDS: [wave][tile][lane], then m, l and x of a column
        f32x4 * of = reinterpret_cast<f32x4 *>(lds);
        f32x4 * ml = of + kPageWaves * TILES * kWave;
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            of[(wave * TILES + u) * kWave + lane] = o[u];
        }
        if (g == 0) {
            ml[wave * 16 + c] = f32x4{ m, l, x, 0.0f };
        }
        __syncthreads();
        float top = -INFINITY;
        f32x4 of_wave[kPageWaves];
#pragma unroll
        for (int w = 0; w < kPageWaves; ++w) {
            of_wave[w] = ml[w * 16 + c];
            top        = fmaxf(top, of_wave[w][0]);
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        float       part[kPageWaves];
        l = 0.0f;
        x = kLeastX;
#pragma unroll
        for (int w = 0; w < kPageWaves; ++w) {
            part[w] = of_wave[w][0] - ref + of_wave[w][2];
            x       = fmaxf(x, part[w]);
            l += of_wave[w][1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(of_wave[w][0] - ref) * of_wave[w][1];
        }
#pragma unroll
        for (int w = 0; w < kPageWaves; ++w) {
            part[w] = __builtin_amdgcn_exp2f(part[w] - x);
        }
        if (live) {
            float *     out;
            float       by;
            const float by_x = __builtin_amdgcn_exp2f(x - kTopWeight);
            if (u0 == 0 && u1 == at.units) {
                out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
                by  = over(l, pos >= 0);
            } else {
                const int   which = u0 == 0 ? 1 : 0;
                const float k     = part_shift(ref, l);
                out               = few_o(f, wg, which, c);
                by                = __builtin_amdgcn_exp2f(-k);
                if (wave == 0 && g == 0) {
                    float * pml = few_ml(f, wg, which, c);
                    pml[0]      = top + k;
                    pml[1]      = l * by;
                }
            }
#pragma unroll
            for (int u = wave; u < TILES; u += kPageWaves) {
                if (FULL || 16 * u < hd) {
                    f32x4 v = splat4(0.0f);
#pragma unroll
                    for (int w = 0; w < kPageWaves; ++w) {
                        v += of[(w * TILES + u) * kWave + lane] * part[w];
                    }
                    *reinterpret_cast<f32x4u *>(out + 16 * u + 4 * g) = v * by * by_x;
                }
            }
        }
        unit = begin + u1;
        if (unit >= last) {
            return;
        }
        __syncthreads();  // the next group's results go where these were
        begin = unit;
        if (++h == f.groups) {
            h = 0;
            do {
                at.units = few_units(f, ++n);
            } while (at.units == 0);
        }
    }
}

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join_pages(const FewArgs f, int64_t row0) {
    join_few<HD>(f, row0 + blockIdx.x);
}

// ---------------------------------------------------------------------------
// Many queries (prompts): a workgroup of four waves, in KG groups side by side. A wave
// has 32 rows, and a group 64 tokens at a time, every KG-th tile of them, which it brings
// into LDS as F16 operands, K by row and V by column, both as the pool has them: the next
// tile while this one's scores are formed, so that a tile takes one barrier, and the one
// after that is on its way in registers. Matrix instructions 32x32x16. With KG 1 a
// workgroup has 128 rows, which share a tile; with 2 it has 64, and its groups' results are
// joined in LDS.
// 8192 positions of 16 heads of 128 over 8 take 528 to 541 us (MI355X): two products at
// 1.02 to 1.04 PFLOP/s, where a large F16 product reaches 1.32. Two barriers a tile, with the tile brought into LDS between them: 575;
// scales made ready as they are read, which waits for them: 15 us of 526. A lone
// workgroup's tile takes 2.0 us, of which the matrix units work 0.9: 1021 positions 31.4 us.
// ---------------------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWideBlock = 256;
constexpr int kWaves     = kWideBlock / kWave;
constexpr int kVStride   = kTileKeys * 2 + 16;  // bytes of a column of V in LDS, off the banks' period

constexpr int key_stride(int nb) {
    return nb * kKvBlock * 2 + 16;
}

// LDS of a group's tile; of two tiles of each, or of the results of all groups but the first.
constexpr int tile_lds(int nb) {
    return kTileKeys * key_stride(nb) + nb * kKvBlock * kVStride;
}

constexpr int wide_lds(int nb, int kg) {
    const int tiles = kg * 2 * tile_lds(nb);
    const int join  = (kWaves - kWaves / kg) * kWave * (nb * 64 + 16);
    return tiles > join ? tiles : join;
}

// The value that lane K of each four has.
template <int K> __device__ __forceinline__ int32_t quad(int32_t v) {
    return static_cast<int32_t>(dpp_u32<K * 0x55>(static_cast<uint32_t>(v)));
}

// hd is 32 NB, or (FULL false) 16 less.
template <int NB, int KG, bool FULL>
__global__ __launch_bounds__(kWideBlock, NB <= 4 && KG == 1 ? 2 : 1) void k_attn_pages_wide(const PagesArgs p) {
    constexpr int HD      = NB * kKvBlock;
    constexpr int KSTRIDE = key_stride(NB);
    constexpr int ROWS    = 32 * kWaves / KG;     // of the workgroup
    constexpr int GROUP   = kWideBlock / KG;      // threads of a group
    extern __shared__ __align__(16) char lds[];
    const AttnArgs & a = p.f.a;

    const int     tid   = threadIdx.x % GROUP;
    const int     kg    = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / GROUP);
    const int     wave  = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int     lane  = tid % kWave;
    char * const  mem   = lds + kg * 2 * tile_lds(NB);  // of the group: two tiles in turn
    const int     c     = lane & 31;
    const int     g     = lane >> 5;
    const int     part0 = static_cast<int>(fastdiv(blockIdx.x, a.fKV));
    const int     h     = static_cast<int>(blockIdx.x) - part0 * a.KV;
    const int     back  = static_cast<int>(fastdiv(static_cast<uint32_t>(part0), a.fsplit));
    const int     tile  = back < a.half ? a.tiles - 1 - back : back - a.half;
    const int     split = part0 - back * a.nsplit;
    const int     n     = blockIdx.y;
    const SeqLens len   = seq_lens(a, n);
    auto          t_of  = [&](int r) { return static_cast<int>(fastdiv(static_cast<uint32_t>(r), a.fG)); };
    const int     t0    = t_of(tile * ROWS);
    if (t0 >= len.count) {
        return;
    }
    const Magic   magic;
    const int32_t base = len.length - len.count;
    const int32_t p0   = base + t0;
    const int32_t p1   = base + min(t_of(tile * ROWS + ROWS - 1), len.count - 1);
    // this wave's positions, and this lane's query
    const int     r0   = tile * ROWS + wave * 32;
    const int32_t w0   = base + t_of(r0);
    const int32_t w1   = t_of(r0) < len.count ? base + min(t_of(r0 + 31), len.count - 1) : -1;
    const int     r    = r0 + c;
    const int     t    = t_of(r);
    const int     gq   = r - t * a.G;
    const bool    live = t < len.count;
    const int32_t pos  = live ? base + t : -1;
    const int     head = h * a.G + gq;

    const KeyTiles kt  = key_tiles<kTileKeys>(a, p0, p1);
    const int      beg = split * a.per;
    const int      end = __builtin_amdgcn_readfirstlane(min(kt.n, beg + a.per));
    if (split > 0 && beg >= kt.n) {
        return;
    }
    const int dest = __builtin_amdgcn_readfirstlane(kt.n <= a.per ? -1 : split);

    // Of a tile, thread id of its group takes 16 bytes of K's row id / (HD/16), z times
    // GROUP threads on, and of V's column id / 4 the sixteen tokens id % 4.
    constexpr int    ALL    = kTileKeys * (HD / 16);
    constexpr int    CHUNKS = (ALL + GROUP - 1) / GROUP;  // of each, a thread
    auto             mine   = [&](int z) { return ALL % GROUP == 0 || tid + GROUP * z < ALL; };
    const int        hd     = FULL ? HD : a.hd;
    const int        page   = 1 << p.pool.shift;
    const PoolSide & ks     = p.pool.side[0];
    const PoolSide & vs     = p.pool.side[1];
    const char *     kb     = ks.codes + h * ks.ch;
    const char *     vb     = vs.codes + h * vs.ch;
    const int32_t *  table  = table_of(p.tables, n);
    auto             row_k  = [&](int z) { return (tid + GROUP * z) / (HD / 16); };
    auto             dim_of = [&](int z) { return (tid + GROUP * z) % (HD / 16) * 16; };

    // The table's entries for a tile's four times sixteen rows, in the lanes k and k + 4 j,
    // which read the scales too.
    int32_t entry = 0;
    u32x4   kr[CHUNKS], vr[CHUNKS];
    float   dk = 0.0f, dv = 0.0f;
    bool    in = true;
    auto    at      = [&](int i) { return __builtin_amdgcn_readfirstlane(key_tile(kt, min(i, end - 1)) * kTileKeys); };
    auto    entries = [&](int i) { entry = entry_of(p, table, at(i) + lane % 4 * 16); };
    auto    fetch   = [&](int i) {
        const int32_t j0    = at(i);
        const PageId  id    = page_id(p, entry);
        const int32_t of[4] = { quad<0>(id.id), quad<1>(id.id), quad<2>(id.id), quad<3>(id.id) };
#pragma unroll
        for (int z = 0; z < CHUNKS; ++z) {
            const int     row  = row_k(z);
            const int32_t low  = row & 16 ? of[1] : of[0];
            const int32_t high = row & 16 ? of[3] : of[2];
            const char *  from = kb + (row & 32 ? high : low) * ks.cp + ((j0 + row) & (page - 1)) * hd + dim_of(z);
            if (FULL && ALL % GROUP == 0) {
                kr[z] = *reinterpret_cast<const u32x4 *>(from);
            } else {
                kr[z] = u32x4{};
                if (mine(z) && dim_of(z) < hd) {
                    kr[z] = *reinterpret_cast<const u32x4 *>(from);
                }
            }
        }
        const char * from = vb + id.id * vs.cp + ((j0 + tid % 4 * 16) & (page - 1));
#pragma unroll
        for (int z = 0; z < CHUNKS; ++z) {
            const int dim = tid / 4 + GROUP / 4 * z;
            if (FULL && ALL % GROUP == 0) {
                vr[z] = *reinterpret_cast<const u32x4 *>(from + dim * page);
            } else {
                vr[z] = u32x4{};
                if (mine(z) && dim < hd) {
                    vr[z] = *reinterpret_cast<const u32x4 *>(from + dim * page);
                }
            }
        }
        dk = scale_at(ks, id, h);
        dv = scale_at(vs, id, h);
        in = id.in;
    };
    // part of a tile's 4 CHUNKS into LDS: half an id's sixteen codes of K, then of V
    auto stage_part = [&](char * kl, int part) {
        const int z = part / 2 % CHUNKS, half = part % 2;
        if (!mine(z)) {
            return;
        }
        if (part < 2 * CHUNKS) {
            const int row = row_k(z);
            const int in  = (row & 32) + 8 * (row >> 2 & 3) + 4 * (row >> 4 & 1) + (row & 3);
            reinterpret_cast<f16x8 *>(kl + in * KSTRIDE + 2 * dim_of(z))[half] = operand(magic, kr[z][2 * half], kr[z][2 * half + 1]);
        } else {
            char * vl = kl + kTileKeys * KSTRIDE;
            reinterpret_cast<f16x8 *>(vl + (tid / 4 + GROUP / 4 * z) * kVStride + tid % 4 * 32)[half] =
                operand(magic, vr[z][2 * half], vr[z][2 * half + 1]);
        }
    };
    // (past its last tile a group reads that again, and nothing of it counts)
    if (beg < end) {
        entries(beg + kg);
        fetch(beg + kg);
        entries(beg + kg + KG);
    }

    // the query's operands; the largest of its values scaled to [2^13, 2^14)
    f16x8 qh[2 * NB], ql[2 * NB];
    float qscale;
    {
        const float * qr = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
        float         q[2 * NB][8];
        float         top = 0.0f;
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            const int   at  = 16 * s + 8 * g;
            const bool  has = live && at < hd;
            const f32x4 x0  = has ? ld4u(qr + at) : splat4(0.0f);
            const f32x4 x1  = has ? ld4u(qr + at + 4) : splat4(0.0f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[s][e] = (e < 4 ? x0[e] : x1[e - 4]) * a.scale;
                top     = fmaxf(top, fabsf(q[s][e]));
            }
        }
        const Pair both = swap32(top);
        top             = fmaxf(both.a, both.b);
        const int   ex  = exponent_of(top) - 13;
        const float to  = pow2(-ex);
        qscale          = pow2(ex);
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            f16x2 hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                split2(q[s][2 * e] * to, q[s][2 * e + 1] * to, hi[e], lo[e]);
            }
            qh[s] = join8(hi[0], hi[1], hi[2], hi[3]);
            ql[s] = join8(lo[0], lo[1], lo[2], lo[3]);
        }
    }

    f32x16 o[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
        o[u] = f32x16{};
    }
    float m = -INFINITY;
    float x = kLeastX;
    float l = 0.0f;
    auto  max_halves = [](float v) {
        const Pair both = swap32(v);
        return fmaxf(both.a, both.b);
    };

    // (group 2 y + g of a tile)
    auto of_group = [&](float v, int y) {
        const float one   = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 2 * y));
        const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 2 * y + 1));
        return g == 0 ? one : other;
    };
    float kscale[2], vscale[2];
    if (beg < end) {
#pragma unroll
        for (int part = 0; part < 4 * CHUNKS; ++part) {
            stage_part(mem, part);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            kscale[y] = score_scale(of_group(scale_of(dk, in), y), qscale);
            vscale[y] = of_group(scale_of(dv, in), y);
        }
        fetch(beg + kg + KG);
        entries(beg + kg + 2 * KG);
    }
    char * kl = mem;
    for (int first = beg; first < end; first += KG) {
        const int     i  = first + kg;
        const int32_t j0 = at(i);
        char * const  vl = kl + kTileKeys * KSTRIDE;
        __syncthreads();  // this tile is in LDS, and the one before is used up
        // scores of token 32 y + 16 g + e, and under their products the next tile on its
        // way into LDS and the one after that into registers
        __builtin_amdgcn_s_setprio(1);
        char * const other = kl == mem ? mem + tile_lds(NB) : mem;
        f32x16       sc[2] = { f32x16{}, f32x16{} };
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            f16x8 k[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                k[y] = *reinterpret_cast<const f16x8 *>(kl + (32 * y + c) * KSTRIDE + 32 * s + 16 * g);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                sc[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[y], qh[s], sc[y], 0, 0, 0);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                sc[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[y], ql[s], sc[y], 0, 0, 0);
            }
#pragma unroll
            for (int part = 4 * CHUNKS * s / (2 * NB); part < 4 * CHUNKS * (s + 1) / (2 * NB); ++part) {
                stage_part(other, part);
            }
        }
        kl = other;
        const float by_now[2] = { kscale[0], kscale[1] }, d_now[2] = { vscale[0], vscale[1] };
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            kscale[y] = score_scale(of_group(scale_of(dk, in), y), qscale);
            vscale[y] = of_group(scale_of(dv, in), y);
        }
        fetch(i + 2 * KG);
        entries(i + 3 * KG);
        __builtin_amdgcn_s_setprio(0);
        if (i >= end || j0 > w1) {
            continue;  // none of it is seen by this wave's queries
        }
        const bool all = j0 + kTileKeys - 1 <= w0 && (a.window == 0 || j0 > w1 - a.window || j0 + kTileKeys <= a.sinks);
        if (!all) {
            int g16 = 16 * g;
            asm volatile("" : "+v"(g16));
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[y][e] = sees(a, pos, j0 + 32 * y + e + g16) ? sc[y][e] : -INFINITY;
                }
            }
        }
        float top[2], times[2];
        bool  any[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            top[y] = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                top[y] = fmaxf(top[y], sc[y][e]);
            }
            any[y]   = top[y] != -INFINITY;
            times[y] = any[y] ? by_now[y] : 1.0f;  // (a scale of tokens that are not seen may be NaN)
            top[y] *= times[y];
        }
        const float most = fmaxf(m, max_halves(fmaxf(top[0], top[1])));
        const float ref  = most == -INFINITY ? 0.0f : most;
        const float down = m - ref;
        // A score is rounded with the difference from the largest, which leaves it above 0
        // by half a step of the largest score at most: 1/16 here. From there on it is
        // rounded before.
        if (__any(fabsf(ref) >= 0x1p20f)) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                sc[y] *= times[y];
                times[y] = 1.0f;
            }
        }
        const float need = max_halves(fmaxf(top[0] - ref + static_cast<float>(exponent_of(d_now[0])),
                                            top[1] - ref + static_cast<float>(exponent_of(d_now[1]))));
        const float now  = fmaxf(fmaxf(x + down, need), kLeastX);
        if (__any(down != 0.0f || now != x)) {
            l *= __builtin_amdgcn_exp2f(down);
            const float turn = __builtin_amdgcn_exp2f(down + x - now);
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                o[u] *= turn;
            }
        }
        m = most;
        x = now;
        const float wf[2] = { weight_scale(d_now[0], x, any[0]), weight_scale(d_now[1], x, any[1]) };
        // weights of the sixteen tokens 32 y + 16 s + 8 g + .. (part 2 y + s of four)
        f16x8 ph[2], pl[2];
        auto  weigh = [&](int part) {
            const int y = part / 2, s = part % 2;
            f16x2     hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    w[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[y][8 * s + 2 * e + k], times[y], -ref));
                    l += w[k];
                    w[k] *= wf[y];
                }
                split_weights(w[0], w[1], hi[e], lo[e]);
            }
            ph[part % 2] = join8(hi[0], hi[1], hi[2], hi[3]);
            pl[part % 2] = join8(lo[0], lo[1], lo[2], lo[3]);
        };
        weigh(0);
#pragma unroll
        for (int part = 0; part < 4; ++part) {
            f16x8 v[NB];
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                v[u] = *reinterpret_cast<const f16x8 *>(vl + (32 * u + c) * kVStride + 64 * (part / 2) + 32 * g + 16 * (part % 2));
            }
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[u], ph[part % 2], o[u], 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[u], pl[part % 2], o[u], 0, 0, 0);
            }
            if (part < 3) {
                weigh(part + 1);
            }
        }
    }
    const Pair sum = swap32(l);
    l              = sum.a + sum.b;
    if constexpr (KG > 1) {
        // the first group takes the others' results from LDS: [group and wave][tile, four
        // elements][lane], and m, l and x of a lane
        constexpr int WAVES = kWaves / KG;
        f32x4 *       of    = reinterpret_cast<f32x4 *>(lds);
        f32x4 *       mlx   = of + (kWaves - WAVES) * NB * 4 * kWave;
        auto          slot  = [&](int group) { return (group - 1) * WAVES + wave; };
        __syncthreads();
        if (kg > 0) {
#pragma unroll
            for (int u = 0; u < NB; ++u) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    of[((slot(kg) * NB + u) * 4 + e) * kWave + lane] = f32x4{ o[u][4 * e], o[u][4 * e + 1], o[u][4 * e + 2], o[u][4 * e + 3] };
                }
            }
            mlx[slot(kg) * kWave + lane] = f32x4{ m, l, x, 0.0f };
        }
        __syncthreads();
        if (kg > 0) {
            return;
        }
#pragma unroll
        for (int group = 1; group < KG; ++group) {
            const f32x4 its  = mlx[slot(group) * kWave + lane];
            const float most = fmaxf(m, its[0]);
            const float ref  = most == -INFINITY ? 0.0f : most;
            const float xa = m - ref + x, xb = its[0] - ref + its[2];
            l   = l * __builtin_amdgcn_exp2f(m - ref) + its[1] * __builtin_amdgcn_exp2f(its[0] - ref);
            m   = most;
            x   = fmaxf(fmaxf(xa, xb), kLeastX);
            const float ta = __builtin_amdgcn_exp2f(xa - x), tb = __builtin_amdgcn_exp2f(xb - x);
#pragma unroll
            for (int u = 0; u < NB; ++u) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x4 v = of[((slot(group) * NB + u) * 4 + e) * kWave + lane];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        o[u][4 * e + k] = o[u][4 * e + k] * ta + v[k] * tb;
                    }
                }
            }
        }
    }
    if (!live) {
        return;
    }
    const int64_t row  = ((static_cast<int64_t>(n) * a.KV + h) * a.T + t) * a.G + gq;
    const float   by_x = __builtin_amdgcn_exp2f(x - kTopWeight);
    float *       out;
    float         by;
    if (dest < 0) {
        out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
        by  = over(l, pos >= 0);
    } else {
        const float k = part_shift(m, l);
        out           = partial_o(a, row, dest);
        by            = __builtin_amdgcn_exp2f(-k);
        if (g == 0) {
            float * ml = partial_ml(a, row, dest);
            ml[0]      = m + k;
            ml[1]      = l * by;
        }
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int dim = 32 * u + 2 * e + 4 * g;
            if (dim < hd) {
                *reinterpret_cast<f32x4u *>(out + dim) =
                    f32x4{ o[u][e] * by * by_x, o[u][e + 1] * by * by_x, o[u][e + 2] * by * by_x, o[u][e + 3] * by * by_x };
            }
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Workgroups that the chip's 256 CUs hold.
constexpr int64_t resident(int64_t hd) {
    return hd <= 128 ? 512 : 256;
}
static_assert(resident(0) <= kMaxParts && resident(kKvMaxDim) <= kMaxParts);  // one head may have all of them

constexpr int64_t kWhole     = 4;    // chunks a wave of a head that is not split
constexpr int64_t kMostParts = 256;  // parts of a head that have one chunk a wave

shp_status_t plan_pages(const shp_tensor * q, const shp_tensor * k, const shp_tensor * table, int32_t window, int32_t sinks,
                        AttnPlan & p) {
    if (!well_formed(q) || !codes_formed(k) || q->ne[0] != k->ne[0] || q->ne[1] % k->ne[2] != 0 || window < 0 || sinks < 0) {
        return SHP_ERR_INVALID_ARG;
    }
    if (page_shift(k->ne[1]) < 0) {
        return SHP_ERR_UNSUPPORTED;
    }
    Tables             tables{};
    const shp_status_t st = check_table(table, q->ne[3], k->ne[1], tables);
    if (st != SHP_OK) {
        return st;
    }
    if (q->type != SHP_TYPE_F32 || q->ne[0] > kKvMaxDim || q->ne[0] % 16 != 0 || q->ne[1] > kKvMaxSeqs || q->ne[3] > kKvMaxSeqs ||
        q->ne[2] > kKvMaxRows / q->ne[1] || !kv_addressable(*q)) {
        return SHP_ERR_UNSUPPORTED;
    }
    const int64_t cap  = tables.cap;
    const int64_t T    = q->ne[2];
    const int64_t kv   = k->ne[2];
    const int64_t rows = q->ne[1] / kv * T;
    p.window           = window >= cap ? 0 : window;
    p.sinks            = static_cast<int32_t>(sinks < cap ? sinks : cap);
    int64_t keys       = cap;
    if (p.window > 0 && int64_t{ p.window } + p.sinks + T < keys) {
        keys = int64_t{ p.window } + p.sinks + T;
    }
    const int64_t chip = resident(q->ne[0]);
    p.few              = rows <= kCols;
    if (p.few) {
        p.groups             = static_cast<int32_t>(kv * q->ne[3]);
        const int64_t chunks = (keys + kPageChunk - 1) / kPageChunk + (p.window > 0 ? 2 : 0);
        const int64_t deep   = chunks <= kWhole * kPageWaves ? (chunks + kPageWaves - 1) / kPageWaves : 1;
        const int64_t units  = (chunks + kPageWaves * deep - 1) / (kPageWaves * deep) * p.groups;
        if (units >= INT32_MAX) {
            return SHP_ERR_UNSUPPORTED;
        }
        p.per              = static_cast<int32_t>(kPageWaves * deep);
        p.parts            = units > p.groups;
        const int64_t want = units > kMostParts * p.groups ? (units + 1) / 2 : units;
        p.wgs              = static_cast<int32_t>(want < chip ? want : chip);
    } else {
        plan_spans(rows, T, cap, keys, kv * q->ne[3], chip, true, p);
        // Two groups of a workgroup rather than splits, whose results go through memory
        // and a second launch, while a head has few tiles for the rows that there are:
        // 512 positions take 20.2 us, 22.2 in splits (16 heads of 128 over 8, MI355X), 1021
        // 32.8, 37.1; but 128 over 768 rows 24.8, 19.9, and 20 over 512 19.0, 14.6. The rule
        // comes from these four. 256 are those that the chip holds at once, one a CU, with
        // heads of 96 and 128 values; of shorter ones it holds 512, which was not measured.
        // Heads of an odd multiple of 16 have no form of this kind, and are split (1000
        // positions of 80: 30.7 us, of 96: 26.8).
        const int64_t most   = (keys + kTileKeys - 1) / kTileKeys + (p.window > 0 ? 2 : 0);
        const int64_t groups = (rows + kWideRows / 2 - 1) / (kWideRows / 2) * kv * q->ne[3];
        p.groups             = 1;
        if (q->ne[0] % kKvBlock == 0 && q->ne[0] <= 4 * kKvBlock && groups <= 256 && most > 1 && most <= 5 + groups / 20) {
            p.groups = 2;
            p.span   = static_cast<int32_t>(most);
            p.nsplit = 1;
        }
    }
    return SHP_OK;
}

template <int HD, bool FULL> shp_status_t launch_few_as(const PagesArgs & p, hipStream_t stream) {
    constexpr int lds = kPageWaves * (HD / 16 * kWave + 16) * 16;
    hipLaunchKernelGGL((k_attn_pages_few<HD, FULL>), dim3(static_cast<unsigned>(p.f.wgs)), dim3(64 * kPageWaves), lds, stream, p);
    const shp_status_t st = launch_status();
    if (st != SHP_OK || p.f.a.work == nullptr) {
        return st;  // no head was split
    }
    constexpr int JOIN = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;
    const int64_t rows = static_cast<int64_t>(p.f.a.N) * p.f.a.KV * p.f.a.T * p.f.a.G;
    return in_launches(rows, kJoinThreads, [&](int64_t first, dim3 grid) {
        hipLaunchKernelGGL(k_attn_join_pages<JOIN>, grid, dim3(kJoinThreads), 0, stream, p.f, first);
    });
}

template <int HD> shp_status_t launch_few(const PagesArgs & p, hipStream_t stream) {
    return p.f.a.hd == HD ? launch_few_as<HD, true>(p, stream) : launch_few_as<HD, false>(p, stream);
}

template <int NB, int KG, bool FULL> shp_status_t launch_wide_as(const PagesArgs & p, hipStream_t stream) {
    const AttnArgs & a = p.f.a;
    const dim3       grid(static_cast<unsigned>(a.KV) * static_cast<unsigned>(a.tiles) * static_cast<unsigned>(a.nsplit),
                          static_cast<unsigned>(a.N));
    hipLaunchKernelGGL((k_attn_pages_wide<NB, KG, FULL>), grid, dim3(kWideBlock), wide_lds(NB, KG), stream, p);
    return launch_status();
}

template <int NB> shp_status_t launch_wide(const PagesArgs & p, int kg, hipStream_t stream) {
    if (p.f.a.hd < NB * kKvBlock) {
        return launch_wide_as<NB, 1, false>(p, stream);
    }
    if constexpr (NB <= 4) {
        if (kg == 2) {
            return launch_wide_as<NB, 2, true>(p, stream);
        }
    }
    return launch_wide_as<NB, 1, true>(p, stream);
}

}  // namespace
}  // namespace shp

using namespace shp;

extern "C" shp_status_t shp_attn_pages_work(const shp_tensor * q,
                                            const shp_tensor * k_pages,
                                            const shp_tensor * table,
                                            int32_t            window,
                                            int32_t            sinks,
                                            int64_t *          floats) {
    AttnPlan p{};
    if (floats == nullptr) {
        return SHP_ERR_INVALID_ARG;
    }
    const shp_status_t st = plan_pages(q, k_pages, table, window, sinks, p);
    if (st == SHP_OK) {
        *floats = plan_floats(p, *q);
    }
    return st;
}

extern "C" shp_status_t shp_attn_pages(const shp_tensor * q,
                                       const shp_tensor * k_pages,
                                       const shp_tensor * v_pages,
                                       const shp_tensor * k_scale,
                                       const shp_tensor * v_scale,
                                       const shp_tensor * table,
                                       const shp_tensor * length,
                                       const shp_tensor * count,
                                       float              scale,
                                       int32_t            window,
                                       int32_t            sinks,
                                       shp_tensor *       work,
                                       shp_tensor *       y,
                                       shp_stream_t       stream) {
    AttnPlan     plan{};
    PagesArgs    p{};
    shp_status_t st = check_pool(k_pages, v_pages, k_scale, v_scale, p.pool);
    st              = st == SHP_OK ? plan_pages(q, k_pages, table, window, sinks, plan) : st;
    if (st != SHP_OK) {
        return st;
    }
    const shp_tensor   kr = codes_as_rows(*k_pages), vr = codes_as_rows(*v_pages);
    const shp_tensor * read[7] = { &kr, &vr, k_scale, v_scale, table, length, count };
    st                         = attn_args(q, length, count, scale, plan, read, 7, work, y, p.f.a);
    if (st != SHP_OK) {
        return st;
    }
    if (length == nullptr) {
        return SHP_ERR_INVALID_ARG;
    }
    if (dry_run()) {
        return SHP_OK;
    }
    st           = check_table(table, q->ne[3], k_pages->ne[1], p.tables);
    AttnArgs & a = p.f.a;
    a.KV         = static_cast<int32_t>(k_pages->ne[2]);
    a.G          = static_cast<int32_t>(q->ne[1] / k_pages->ne[2]);
    a.cap        = p.tables.cap;
    a.fG         = make_fastdiv(static_cast<uint32_t>(a.G));
    a.fKV        = make_fastdiv(static_cast<uint32_t>(a.KV));
    const hipStream_t s = as_stream(stream);
    if (plan.few) {
        FewArgs & f = p.f;
        f.shift     = 6;
        f.groups    = a.KV;
        f.wgs       = plan.wgs;
        f.fwgs      = make_fastdiv(static_cast<uint32_t>(plan.wgs));
        f.per       = plan.per;
        f.fper      = make_fastdiv(static_cast<uint32_t>(plan.per));
        f.cols      = a.T * a.G;
        return a.hd <= 64  ? launch_few<64>(p, s) :
               a.hd <= 128 ? launch_few<128>(p, s) :
               a.hd <= 192 ? launch_few<192>(p, s) :
                             launch_few<256>(p, s);
    }
    wide_args(plan.span, kWideRows / plan.groups, resident(a.hd), a);
    switch ((a.hd + kKvBlock - 1) / kKvBlock) {
        case 1:
            st = launch_wide<1>(p, plan.groups, s);
            break;
        case 2:
            st = launch_wide<2>(p, plan.groups, s);
            break;
        case 3:
            st = launch_wide<3>(p, plan.groups, s);
            break;
        case 4:
            st = launch_wide<4>(p, plan.groups, s);
            break;
        case 5:
            st = launch_wide<5>(p, plan.groups, s);
            break;
        case 6:
            st = launch_wide<6>(p, plan.groups, s);
            break;
        case 7:
            st = launch_wide<7>(p, plan.groups, s);
            break;
        default:
            st = launch_wide<8>(p, plan.groups, s);
            break;
    }
    return st == SHP_OK && a.nsplit > 1 ? launch_join(a, s) : st;
}
