// shp_attn_cross for few queries over plain states (a decoder's token).
//
// At most 16 columns, the queries of one kv head, against chunks of 16 or 32 rows
// that a wave reads straight into the operands' registers, 16 bytes a lane, the next
// K ahead of the exponentials and the next V ahead of the next scores:
//   S^T = K Q^T  F16 and BF16 as they lie, q in two F16 or three BF16 pieces; F32
//                in F32 products (16x16x4);
//   O^T = V^T P^T in F32 products, whose operands are single values: a lane that
//                has read dimensions VE c and on of the row that its own score is
//                of holds the element of VE tiles, so V needs no turning, and
//                weights and values are exact. 4096 cycles of a SIMD for 64 rows of 128
//                values, 32 KB of F16: the chip could take 19 TB/s.
// Bound by the bytes of long states and by latency: 16 sequences of 300 to 1500 rows (16
// heads of 64, MI355X) take 18 to 19.5 us over F16, 3.1 TB/s, 19 over BF16 and 30 over F32
// (3.9 TB/s), in one launch; in stretches, as longer ones are, F16 takes 22, of which 4 are
// the join. Heads of 40 F16 or BF16 values take 26: their form spills registers.
// Every query sees every row, so rows past a sequence's are read as its last one, and
// count for nothing.
#include "shp_attn.hpp"

namespace shp {
namespace {

constexpr int kSplitWaves = 4;  // of a workgroup whose heads are split

// Rows of a chunk: 32, or 16 where that many would take more than 32 registers of a lane for K.
constexpr int cross_rows(int kind, int hd) {
    return 8192 / (hd * kv_unit_bytes(kind)) >= 32 ? 32 : 16;
}

// Waves that a SIMD holds by their registers.
constexpr int cross_occupancy(int kind, int hd) {
    return hd == 64 && kind != kKvF32 ? 4 : hd == 64 ? 3 : hd == 128 ? 2 : 1;
}

constexpr int cross_shift(int kind, int hd) {
    return cross_rows(kind, hd) == 32 ? 5 : 4;
}

typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// a and b: BF16 rounded, as a pair of bits, and what that leaves of them.
__device__ __forceinline__ f16x2 take_b16(float & a, float & b) {
    typedef float  f32x2 __attribute__((ext_vector_type(2)));
    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{ a, b }), b16x2));
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return as_f16x2(w);
}

// Waves of a workgroup that has a whole head: as many as a CU holds, within 16.
constexpr int cross_waves(int kind, int hd) {
    return cross_occupancy(kind, hd) == 4 ? 16 : hd <= 128 ? 8 : 4;
}

// 16 bytes at any 4-byte boundary.
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

// Value i of the 16 bytes w.
template <int KIND> __device__ __forceinline__ float value_of(const u32x4 & w, int i) {
    if constexpr (KIND == kKvF32) {
        return __uint_as_float(w[i]);
    } else {
        const uint32_t h = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
        return KIND == kKvF16 ? f16_bits_to_f32(h) : i & 1 ? __uint_as_float(w[i / 2] & 0xffff0000u) : __uint_as_float(w[i / 2] << 16);
    }
}

// The larger of a magnitude's bits and those of the values in w, in whose order
// infinity is the first that is not finite.
template <int KIND> constexpr uint32_t kInfinite = KIND == kKvF32 ? 0x7f800000u : KIND == kKvF16 ? 0x7c00u : 0x7f80u;

template <int KIND> __device__ __forceinline__ uint32_t larger(uint32_t most, uint32_t w) {
    return KIND == kKvF32 ? max(most, w & 0x7fffffffu) : max(most, max(w & 0x7fffu, w >> 16 & 0x7fffu));
}

// hd is HD, or (FULL false) less, a multiple of HD/16 and of 16 bytes: then what lies
// past it is read from the row's start, against zeros in q and into results that
// are not written.
template <int KIND, int HD, bool FULL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, cross_occupancy(KIND, HD)) void k_cross_few(const FewArgs f) {
    constexpr int  SIZE  = kv_unit_bytes(KIND);
    constexpr int  PER   = 16 / SIZE;          // values of 16 bytes
    constexpr int  ROWS  = cross_rows(KIND, HD);
    constexpr int  TT    = ROWS / 16;          // tiles of rows
    constexpr int  TILES = HD / 16;            // of dimensions, and a lane's of V
    constexpr int  KP    = HD * SIZE / 64;     // K's pieces of a row in a lane: values 4 PER p + PER g and on
    constexpr int  VB    = TILES * SIZE;       // V's bytes of a row in a lane
    constexpr int  VP    = VB < 16 ? 1 : VB / 16;
    constexpr bool F32   = KIND == kKvF32;
    constexpr int  QP    = KIND == kKvF16 ? 2 : 3;  // pieces of q
    extern __shared__ __align__(16) char lds[];
    const AttnArgs & a    = f.a;
    const int        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int        lane = threadIdx.x % kWave;
    const int        c    = lane & 15;
    const int        g    = lane >> 4;
    const int        wg   = blockIdx.x;
    const int        hd   = FULL ? HD : a.hd;
    const Line       line = few_line(f, wg, lane);
    const int32_t    last = line.end;
    int32_t          unit = line.begin;
    const int        t    = static_cast<int>(fastdiv(static_cast<uint32_t>(c), a.fG));
    const int        gq   = c - t * a.G;
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
        const int32_t rows = len.length;
        const int     all  = (rows + ROWS - 1) / ROWS;
        const bool    live = c < f.cols && t < len.count;
        const int     head = h * a.G + gq;
        const char *  kb   = a.k + n * a.kn + h * a.kh;
        const char *  vb   = a.v + n * a.vn + h * a.vh;

        f32x4 o[TILES];
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            o[u] = splat4(0.0f);
        }
        float m = -INFINITY;
        float l = 0.0f;

        const int end = min(all, u1 * f.per);
        int       i   = u0 * f.per + wave;

        u32x4 kr[TT][KP];
        u32x4 vr[TT][4][VP];
        auto  fetch_k = [&](int chunk) {
#pragma unroll
            for (int y = 0; y < TT; ++y) {
                const int32_t row  = min(chunk * ROWS + 16 * y + c, rows - 1);
                const char *  from = kb + row * a.kt;
#pragma unroll
                for (int p = 0; p < KP; ++p) {
                    const int dim = 4 * PER * p + PER * g;
                    kr[y][p]      = *reinterpret_cast<const u32x4_at4 *>(from + (FULL || dim < hd ? dim : 0) * SIZE);
                }
            }
        };
        auto fetch_v = [&](int chunk) {
            const int dim = FULL || TILES * c < hd ? TILES * c : 0;
#pragma unroll
            for (int y = 0; y < TT; ++y) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t row  = min(chunk * ROWS + 16 * y + 4 * g + e, rows - 1);
                    const char *  from = vb + row * a.vt + dim * SIZE;
                    if constexpr (VB == 8) {
                        typedef uint32_t u32x2_at4 __attribute__((ext_vector_type(2), aligned(4)));
                        const u32x2_at4  w = *reinterpret_cast<const u32x2_at4 *>(from);
                        vr[y][e][0][0]     = w[0];
                        vr[y][e][0][1]     = w[1];
                    } else {
#pragma unroll
                        for (int p = 0; p < VP; ++p) {
                            vr[y][e][p] = *reinterpret_cast<const u32x4_at4 *>(from + 16 * p);
                        }
                    }
                }
            }
        };
        if (i < end) {
            fetch_k(i);
            fetch_v(i);
        }

        // the queries' operands: element e of piece p is value 4 PER p + PER g + e.
        // Over F16 the largest value of each is scaled to [2^13, 2^14).
        float qf[F32 ? KP : 1][PER];
        f16x8 qp[F32 ? 1 : KP][QP];
        float qscale = 1.0f;
        {
            const float * qr = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
            float         q[KP][PER];
            float         top = 0.0f;
#pragma unroll
            for (int p = 0; p < KP; ++p) {
                const int  dim = 4 * PER * p + PER * g;
                const bool has = live && (FULL || dim < hd);
#pragma unroll
                for (int k = 0; k < PER / 4; ++k) {
                    const f32x4 x = has ? ld4u(qr + dim + 4 * k) : splat4(0.0f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        q[p][4 * k + e] = x[e] * a.scale;
                        top             = fmaxf(top, fabsf(q[p][4 * k + e]));
                    }
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int p = 0; p < KP; ++p) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        qf[p][e] = q[p][e];
                    }
                }
            } else {
                float to = 1.0f;
                if constexpr (KIND == kKvF16) {
                    top          = max_quarters(top);
                    const int ex = exponent_of(top) - 13;
                    to           = pow2(-ex);
                    qscale       = pow2(ex);
                }
#pragma unroll
                for (int p = 0; p < KP; ++p) {
                    f16x2 piece[QP][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x0 = q[p][2 * e] * to, x1 = q[p][2 * e + 1] * to;
                        if constexpr (KIND == kKvF16) {
                            split2(x0, x1, piece[0][e], piece[1][e]);
                        } else {
#pragma unroll
                            for (int k = 0; k < QP; ++k) {
                                piece[k][e] = take_b16(x0, x1);
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < QP; ++k) {
                        qp[p][k] = join8(piece[k][0], piece[k][1], piece[k][2], piece[k][3]);
                    }
                }
            }
        }

        // a chunk, and (MORE) the next one's rows on their way
        auto chunk = [&](auto more) {
            constexpr bool MORE = decltype(more)::value;
            f32x4          sc[TT];
#pragma unroll
            for (int y = 0; y < TT; ++y) {
                sc[y] = splat4(0.0f);
            }
#pragma unroll
            for (int p = 0; p < KP; ++p) {
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
#pragma unroll
                        for (int y = 0; y < TT; ++y) {
                            sc[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(value_of<KIND>(kr[y][p], e), qf[p][e], sc[y], 0, 0, 0);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < QP; ++k) {
#pragma unroll
                        for (int y = 0; y < TT; ++y) {
                            if constexpr (KIND == kKvF16) {
                                sc[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, kr[y][p]), qp[p][k], sc[y], 0, 0, 0);
                            } else {
                                sc[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, kr[y][p]),
                                                                                __builtin_bit_cast(b16x8, qp[p][k]), sc[y], 0, 0, 0);
                            }
                        }
                    }
                }
            }
            const int32_t j0  = i * ROWS;
            float         top = -INFINITY, low = INFINITY;
#pragma unroll
            for (int y = 0; y < TT; ++y) {
                sc[y] *= qscale;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    low = fminf(low, sc[y][e]);
                }
            }
            // A score of -infinity may be that of finite values, which counts for
            // nothing, or of an infinity in K, which makes the query NaN. (+infinity
            // and NaN do that by themselves.)
            if (__any(low == -INFINITY)) {
#pragma unroll
                for (int y = 0; y < TT; ++y) {
                    uint32_t most = 0;
#pragma unroll
                    for (int p = 0; p < KP; ++p) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            most = larger<KIND>(most, kr[y][p][e]);
                        }
                    }
                    uint64_t of = __ballot(most >= kInfinite<KIND>);
                    of |= of >> 32;
                    of |= of >> 16;  // bit r: row r of the tile
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[y][e] = of >> (4 * g + e) & 1u ? NAN : sc[y][e];
                    }
                }
            }
            if constexpr (MORE) {
                fetch_k(i + WAVES);
            } else if (j0 + ROWS > rows) {
#pragma unroll
                for (int y = 0; y < TT; ++y) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[y][e] = j0 + 16 * y + 4 * g + e < rows ? sc[y][e] : -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < TT; ++y) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    top = fmaxf(top, sc[y][e]);
                }
            }
            const float most = fmaxf(m, max_quarters(top));
            const float ref  = most == -INFINITY ? 0.0f : most;
            if (__any(m != ref)) {
                const float turn = __builtin_amdgcn_exp2f(m - ref);
                l *= turn;
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    o[u] *= turn;
                }
            }
            m = most;
#pragma unroll
            for (int y = 0; y < TT; ++y) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[y][e] = __builtin_amdgcn_exp2f(sc[y][e] - ref);
                    l += sc[y][e];
                }
            }
#pragma unroll
            for (int y = 0; y < TT; ++y) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int u = 0; u < TILES; ++u) {
                        o[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(value_of<KIND>(vr[y][e][u / PER], u % PER), sc[y][e], o[u], 0, 0, 0);
                    }
                }
            }
            if constexpr (MORE) {
                fetch_v(i + WAVES);
            }
        };
        for (; i + WAVES < end; i += WAVES) {
            chunk(std::true_type{});
        }
        if (i < end) {
            chunk(std::false_type{});
        }
        // (an infinity or NaN in V, or a sum past f32)
        uint32_t largest = 0;
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                largest = larger<kKvF32>(largest, __float_as_uint(o[u][e]));
            }
        }
        l = sum_quarters(largest >= kInfinite<kKvF32> ? NAN : l);

        // the waves' results joined in LDS: [wave][tile][lane], then m and l of a column
        f32x4 * of = reinterpret_cast<f32x4 *>(lds);
        float * ml = reinterpret_cast<float *>(of + WAVES * TILES * kWave);
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            of[(wave * TILES + u) * kWave + lane] = o[u];
        }
        if (g == 0) {
            ml[(wave * 16 + c) * 2]     = m;
            ml[(wave * 16 + c) * 2 + 1] = l;
        }
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            top = fmaxf(top, ml[(w * 16 + c) * 2]);
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        float       part[WAVES];
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float wl = ml[(w * 16 + c) * 2 + 1];
            part[w]        = wl == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[(w * 16 + c) * 2] - ref);
            l += part[w] * wl;
        }
        if (live) {
            float * out;
            float   by = 1.0f;
            if (u0 == 0 && u1 == at.units) {
                out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
                by  = over(l, rows > 0);
            } else {
                const int which = u0 == 0 ? 1 : 0;
                out             = few_o(f, wg, which, c);
                if (wave == 0 && g == 0) {
                    float * pml = few_ml(f, wg, which, c);
                    pml[0]      = top;
                    pml[1]      = l;
                }
            }
            // element e of tile u in quarter g is value TILES (4 g + e) + u: the first
            // waves take an e and four tiles each
            for (int from = wave; from < TILES; from += WAVES) {
                const int e = from % 4, u0 = from / 4 * 4;
                f32x4     v = splat4(0.0f);
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        v[u] += reinterpret_cast<const float *>(of + (w * TILES + u0 + u) * kWave + lane)[e] * part[w];
                    }
                }
                const int dim = TILES * (4 * g + e) + u0;
                if (FULL || dim < hd) {
                    *reinterpret_cast<f32x4u *>(out + dim) = v * by;
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

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_cross_join(const FewArgs f, int64_t row0) {
    join_few<HD>(f, row0 + blockIdx.x);
}

template <int KIND, int HD, bool FULL> shp_status_t launch_as(FewArgs & f, int waves, hipStream_t stream) {
    const int lds = waves * (HD / 16 * kWave * 16 + 16 * 2 * 4);
    auto      go  = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(f.wgs)), dim3(static_cast<unsigned>(64 * waves)), lds, stream, f);
        return launch_status();
    };
    if (f.a.work == nullptr && waves > kSplitWaves) {
        return go(k_cross_few<KIND, HD, FULL, cross_waves(KIND, HD)>);
    }
    const shp_status_t st = go(k_cross_few<KIND, HD, FULL, kSplitWaves>);
    if (st != SHP_OK || f.a.work == nullptr) {
        return st;  // no head was split
    }
    const int64_t rows = static_cast<int64_t>(f.a.N) * f.a.KV * f.a.T * f.a.G;
    return in_launches(rows, kJoinThreads, [&](int64_t first, dim3 grid) {
        hipLaunchKernelGGL(k_cross_join<HD>, grid, dim3(kJoinThreads), 0, stream, f, first);
    });
}

template <int KIND> shp_status_t launch(FewArgs & f, int waves, hipStream_t stream) {
    switch (cross_few_dims(f.a.hd)) {
        case 64:
            return f.a.hd == 64 ? launch_as<KIND, 64, true>(f, waves, stream) : launch_as<KIND, 64, false>(f, waves, stream);
        case 128:
            return f.a.hd == 128 ? launch_as<KIND, 128, true>(f, waves, stream) : launch_as<KIND, 128, false>(f, waves, stream);
        default:
            return f.a.hd == 256 ? launch_as<KIND, 256, true>(f, waves, stream) : launch_as<KIND, 256, false>(f, waves, stream);
    }
}

}  // namespace

// A head is whole while its chunks are at most kDeep a wave: what more of them would take
// is less than a second launch.
constexpr int64_t kDeep = 6;

// Workgroups of `waves` that the chip's 256 CUs hold. A head that is split may have all of
// those of kSplitWaves.
constexpr int cross_resident(int kind, int hd, int waves) {
    return 256 * 4 * cross_occupancy(kind, hd) / waves;
}

static_assert(cross_resident(kKvF16, 64, kSplitWaves) <= kMaxParts && cross_resident(kKvF32, 64, kSplitWaves) <= kMaxParts &&
              cross_resident(kKvF16, 128, kSplitWaves) <= kMaxParts && cross_resident(kKvF16, 256, kSplitWaves) <= kMaxParts);

void plan_cross_few(int kind, int64_t hd, int64_t rows, int64_t groups, AttnPlan & p) {
    const int     dims   = static_cast<int>(cross_few_dims(hd));
    const int     most   = cross_waves(kind, dims);
    const int64_t chunk  = cross_rows(kind, dims);
    const int64_t chunks = (rows + chunk - 1) / chunk;
    p.parts              = chunks > kDeep * most;
    p.waves              = !p.parts && chunks > kSplitWaves ? most : kSplitWaves;
    const int64_t deep   = p.parts ? 1 : (chunks + p.waves - 1) / p.waves;
    const int64_t units  = (chunks + p.waves * deep - 1) / (p.waves * deep) * groups;
    const int64_t held   = cross_resident(kind, dims, p.waves);
    p.cross              = units < INT32_MAX;
    p.per                = static_cast<int32_t>(p.waves * deep);
    p.groups             = static_cast<int32_t>(groups);
    p.wgs                = static_cast<int32_t>(units < held ? units : held);
}

bool cross_few_takes(const shp_tensor & c) {
    const int kind = kv_kind(c.type);
    return !kv_blocks(kind) && kv_bytes_of_row(c) % 16 == 0 && c.ne[0] % (cross_few_dims(c.ne[0]) / 16) == 0 && rows_aligned(c, 4);
}

shp_status_t launch_cross_few(int kind, const AttnArgs & a, const AttnPlan & p, hipStream_t stream) {
    FewArgs f{};
    f.a      = a;
    f.shift  = cross_shift(kind, static_cast<int>(cross_few_dims(a.hd)));
    f.groups = a.KV;
    f.wgs    = p.wgs;
    f.fwgs   = make_fastdiv(static_cast<uint32_t>(p.wgs));
    f.per    = p.per;
    f.fper   = make_fastdiv(static_cast<uint32_t>(p.per));
    f.cols   = a.T * a.G;
    switch (kind) {
        case kKvF32:
            return launch<kKvF32>(f, p.waves, stream);
        case kKvF16:
            return launch<kKvF16>(f, p.waves, stream);
        default:
            return launch<kKvBF16>(f, p.waves, stream);
    }
}

}  // namespace shp
