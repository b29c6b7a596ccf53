// shp_attn_kv for few queries over a cache in blocks (decoding).
#include "shp_attn.hpp"

namespace shp {
namespace {

// ---------------------------------------------------------------------------
// Few queries (decoding): at most 16 columns, which are the queries of HG
// neighbouring kv heads. A chunk is 32 cache rows in the order in which they
// lie in memory, HG heads of 32/HG keys, so that a wave reads whole lines
// whatever head_dim is: its score matrix is 32 rows x 16 queries, of which a
// row's own head's columns count and the others are masked (the matrix
// instruction has 16 columns in any case).
//
// A wave keeps a chunk's bytes as they are in its own part of LDS, the next
// chunk's on their way in registers, and forms the operands from them:
//   S^T = K Q^T: codes as F16, exact, against q in two F16 pieces (22 bits and
//         more: q = 2^e (hi + lo)), each block's sum times its d in F32;
//   O^T = V^T P^T: code * d as two F16 pieces, exact (at most 8 + 11 bits),
//         against P in two; lo x lo, below 2^-22 of the product, is left out.
//         Where a d of V is above 256, d is two parts (see kBigD), one after
//         the other.
// P is held times 2^15, so that its pieces keep their bits where it is small:
// a weight is off by at most 2^-40 of the largest, or 2^-22 of itself.
// 64 streams of 512 to 8192 rows (Q4_0, 16 heads of 128 values over 8, MI355X)
// take 93 to 106 us, 3.0 to 3.5 TB/s. Vector instructions, most of them forming
// operands, are 480 a chunk of 4.6 KB: 62 us of issue on every SIMD. Matrix
// instructions are 20 % of the time and LDS 35 %; what overlaps of these, and what
// the rest waits for, has not been measured. One stream of 8191 rows takes 17 us,
// 7 of them the join.
// ---------------------------------------------------------------------------

// Dwords at two-byte boundaries of LDS. A wave's read of them as they are takes
// 65 cycles of the LDS unit on this chip, an aligned one 3.2, so each is put
// together from the two aligned dwords that it lies in. `lo` and `hi` are the
// same address a dword apart, kept from being joined into one 8-byte read (35
// to 65 cycles at a 4-byte boundary).
struct LdsWords {
    const char * lo;
    const char * hi;
    uint32_t     shift;  // 0 or 2 bytes

    __device__ explicit LdsWords(const char * base, int at) {
        lo    = base + (at & ~3);
        int d = 4;
        asm("" : "+v"(d));
        hi    = lo + d;
        shift = static_cast<uint32_t>(at) & 2u;
    }

    // The dword `off` bytes on, a multiple of 4.
    __device__ uint32_t at(int off) const {
        return __builtin_amdgcn_alignbyte(*reinterpret_cast<const uint32_t *>(hi + off),
                                          *reinterpret_cast<const uint32_t *>(lo + off), shift);
    }
};

// One cache's chunk on its way to LDS: a lane's pieces of 16 or 4 bytes.
template <int BYTES, int P> struct Staged;

template <int P> struct Staged<16, P> {
    u32x4 piece[P];

    __device__ void load(int i, const Rsrc & r, int off) { piece[i] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0); }

    __device__ void keep(int i, char * lds, int at) const { reinterpret_cast<u32x4 *>(lds)[at] = piece[i]; }
};

template <int P> struct Staged<4, P> {
    uint32_t piece[P];

    __device__ void load(int i, const Rsrc & r, int off) { piece[i] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0); }

    __device__ void keep(int i, char * lds, int at) const { reinterpret_cast<uint32_t *>(lds)[at] = piece[i]; }
};

// LDS of a workgroup ahead of its waves' parts: the queries' operands and maxima.
__host__ __device__ constexpr int few_shared(int nb, int waves) {
    return 2 * nb * kWave * 16 + waves * kWave * 4;
}

// KIND Q4 or Q8, NB blocks a row (NB 8: at most 8), read in pieces of BYTES;
// RUNS: a key's rows are apart from the next key's.
template <int KIND, int NB, int BYTES, bool RUNS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, few_occupancy(KIND, NB * kKvBlock)) void k_attn_few(const FewArgs f) {
    using C                 = Codes<KIND>;
    constexpr int    UNIT   = kv_unit_bytes(KIND);
    constexpr int    SLOTS  = (NB * C::kWords + 15) / 16;
    constexpr int    TILES  = SLOTS * C::kTiles;
    constexpr int    kAtOnce = 2;  // tiles of V whose products take turns: no wait for the one before (a call 3% shorter; 4: 1%)
    constexpr int    P      = (kChunk * NB * UNIT / BYTES + kWave - 1) / kWave;
    extern __shared__ char lds[];
    const AttnArgs & a    = f.a;
    const int        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int        lane = threadIdx.x % kWave;
    const int        c    = lane & 15;
    const int        g    = lane >> 4;
    const int        wg   = blockIdx.x;
    const int        keys = kChunk >> f.hgs;
    const int        mask = (1 << f.hgs) - 1;
    const int        nb   = NB <= 4 ? NB : f.nb;
    const int        rb   = nb * UNIT;
    const Line       line = few_line(f, wg, lane);
    const int32_t    last = line.end;
    int32_t          unit = line.begin;

    const Magic      magic;

    // this lane's query, the same in every group
    const int hc = static_cast<int>(fastdiv(static_cast<uint32_t>(c), f.fcols));
    const int r  = c - hc * f.cols;
    const int t  = static_cast<int>(fastdiv(static_cast<uint32_t>(r), a.fG));
    // the least upper bound of a score of row 4 g + e (and 16 more): none where
    // the row is of this query's head
    float own[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        own[e] = ((4 * g + e) & mask) == hc ? INFINITY : -INFINITY;
    }
    f16x8 *    qop  = reinterpret_cast<f16x8 *>(lds);
    float *    qmax = reinterpret_cast<float *>(qop + 2 * NB * kWave);
    char *     kl   = lds + few_shared(NB, WAVES) + wave * f.wave_lds;
    char *     vl = kl + kChunk * rb;
    float *    kd = reinterpret_cast<float *>(vl + kChunk * rb);
    _Float16 * vd = reinterpret_cast<_Float16 *>(kd + NB * kChunk);

    // where this lane's pieces lie, from a chunk's first byte: one run, or runs a key apart
    int32_t krel[RUNS ? P : 1], vrel[RUNS ? P : 1];
#pragma unroll
    for (int i = 0; i < (RUNS ? P : 1); ++i) {
        const int pc  = lane + i * kWave;
        const int key = RUNS ? static_cast<int>(fastdiv(static_cast<uint32_t>(pc), f.frun)) : 0;
        const int off = BYTES * (pc - key * f.run);
        krel[i]       = key * static_cast<int32_t>(RUNS ? a.kt : 0) + off;
        vrel[i]       = key * static_cast<int32_t>(RUNS ? a.vt : 0) + off;
    }
    // This lane's K words, those of its quarter in row c, and V words, word
    // c + 16 s of the rows 4 g and on; a second start, two bytes on, for the
    // blocks and rows that are an odd multiple of two bytes further.
    const LdsWords k0(kl, c * rb + 2 + 4 * C::kStep * g);
    const LdsWords k1(kl, c * rb + 4 + 4 * C::kStep * g);
    int            vblock[SLOTS];
    int            vword[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int w = min(c + 16 * s, nb * C::kWords - 1);
        vword[s]    = 4 * g * rb + C::word_offset(w);
        vblock[s]   = w / C::kWords;
    }


    if (unit >= last) {
        return;
    }
    Place   at    = line.at;
    int     n     = at.n;
    int     hg    = f.groups == 1 ? 0 : (unit - at.before) / at.units;
    int32_t begin = at.before + hg * at.units;  // the group's first unit
    for (;;) {
        const int     u0     = unit - begin;
        const int     u1     = min(last - begin, at.units);
        const int     h0     = hg << f.hgs;
        const SeqLens  len   = seq_lens(a, n);
        if (a.work != nullptr && u0 == 0 && threadIdx.x == 0) {
            few_span(f, n * f.groups + hg)[0] = wg;
            few_span(f, n * f.groups + hg)[1] = few_owner(f, line.total, begin + at.units - 1);
        }
        const KeyTiles kt    = few_tiles(f, len);
        const int32_t base   = first_position(a, len);
        const int32_t p1     = len.length - 1;
        const int     head   = (h0 + hc) * a.G + r - t * a.G;
        const bool    live   = hc <= mask && t < len.count;
        const int32_t p      = live ? position(a, base, t) : -1;

        const char * kb = a.k + n * a.kn + h0 * a.kh;
        const char * vb = a.v + n * a.vn + h0 * a.vh;

        f32x4 o[TILES];
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            o[u] = splat4(0.0f);
        }
        float less = INFINITY;  // weights are 2^(score + less)
        float l    = 0.0f;

        // the chunks of these units, one a wave
        const int end = min(kt.n, u1 * f.per);
        int       i   = u0 * f.per + wave;

        Staged<BYTES, P> ks, vs;
        auto             fetch = [&](int32_t tile) {
            const int32_t j0 = key_tile(kt, tile) << (5 - f.hgs);
            const Rsrc    kr = rows_from(kb + static_cast<int64_t>(j0) * a.kt, static_cast<int64_t>(a.cap - j0 - 1) * a.kt + (rb << f.hgs));
            const Rsrc    vr = rows_from(vb + static_cast<int64_t>(j0) * a.vt, static_cast<int64_t>(a.cap - j0 - 1) * a.vt + (rb << f.hgs));
#pragma unroll
            for (int x = 0; x < P; ++x) {
                ks.load(x, kr, RUNS ? krel[x] : krel[0] + x * kWave * BYTES);
                vs.load(x, vr, RUNS ? vrel[x] : krel[0] + x * kWave * BYTES);
            }
        };
        if (i < end) {
            fetch(i);
        }
        // The queries' operands, the same for every wave: in LDS, each wave's blocks
        // formed by it. A query is scaled by a power of two that brings its largest
        // value to [2^13, 2^14), so that both pieces of all that counts are normal.
        float qscale;
        {
            constexpr int MINE = (NB + WAVES - 1) / WAVES;
            const float * qr   = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
            float         q[MINE][8];
            float         top = 0.0f;
#pragma unroll
            for (int k = 0; k < MINE; ++k) {
                const int   b   = wave + k * WAVES;
                const bool  has = live && b < nb;
                const f32x4 x0  = has ? ld4u(qr + 32 * b + C::kFirst * g) : splat4(0.0f);
                const f32x4 x1  = has ? ld4u(qr + 32 * b + C::kFirst * g + C::kSecond) : splat4(0.0f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    q[k][e] = (e < 4 ? x0[C::order(e)] : x1[C::order(e - 4)]) * a.scale;
                    top     = fmaxf(top, fabsf(q[k][e]));
                }
            }
            qmax[wave * kWave + lane] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                top = fmaxf(top, qmax[w * kWave + lane]);
            }
            top = max_quarters(top);
            const int ex   = exponent_of(top) - 13;
            const float to = pow2(-ex);
            qscale         = pow2(ex);
#pragma unroll
            for (int k = 0; k < MINE; ++k) {
                const int b = wave + k * WAVES;
                f16x2     h[4], l[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    split2(q[k][2 * e] * to, q[k][2 * e + 1] * to, h[e], l[e]);
                }
                if (b < nb) {
                    qop[(2 * b) * kWave + lane]     = join8(h[0], h[1], h[2], h[3]);
                    qop[(2 * b + 1) * kWave + lane] = join8(l[0], l[1], l[2], l[3]);
                }
            }
            __syncthreads();
        }

        for (; i < end; i += WAVES) {
            const int32_t j0 = key_tile(kt, i) << (5 - f.hgs);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int x = 0; x < P; ++x) {
                const int pc = lane + x * kWave;
                if (pc < f.pieces) {
                    ks.keep(x, kl, pc);
                    vs.keep(x, vl, pc);
                }
            }
            if (i + WAVES < end) {
                fetch(i + WAVES);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            // d of the 32 rows: K's as F32, V's as they are; a row that no query of
            // the call sees has d = 0
            bool large;
            {
                const int    row  = lane & 31;
                const bool   isk  = lane < 32;
                const char * from = (isk ? kl : vl) + row * rb;
                const bool   keep = seen_by(a, base, p1, j0 + (row >> f.hgs));
                uint16_t     d[NB];
                uint32_t     most = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    d[b] = b < nb && keep ? *reinterpret_cast<const uint16_t *>(from + b * UNIT) : 0;
                    most = max(most, d[b] & 0x7fffu);
                }
                // a row of K or V that holds an infinity or NaN counts for nothing in the products ...
                const uint64_t not_finite = __ballot(most >= kInfD);
                if (not_finite != 0) {
                    uint32_t bad = static_cast<uint32_t>(not_finite | not_finite >> 32);
                    if (most >= kInfD) {
                        most = 0;
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            d[b] = 0;
                        }
                    }
                    // ... make the result of a query that sees one NaN, and no other's
                    for (; bad != 0; bad &= bad - 1) {
                        const int x = __ffs(static_cast<int>(bad)) - 1;
                        if ((x & mask) == hc && sees(a, p, j0 + (x >> f.hgs))) {
                            l = NAN;
                        }
                    }
                }
                large = __any(!isk && most > kBigD);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (b < nb) {
                        if (isk) {
                            kd[b * kChunk + row] = f16_bits_to_f32(d[b]);
                        } else {
                            vd[b * kChunk + row] = __builtin_bit_cast(_Float16, d[b]);
                        }
                    }
                }
                if (large && !isk) {
                    // d = 2^8 first + rest, both exact and values of either within F16's range
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        if (b < nb) {
                            const float    v     = f16_bits_to_f32(d[b]);
                            const _Float16 first = static_cast<_Float16>(v * (1.0f / kLargeBy));
                            vd[(NB + b) * kChunk + row] = first;
                            vd[b * kChunk + row]        = static_cast<_Float16>(v - static_cast<float>(first) * kLargeBy);
                        }
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();

            // scores: rows 16 mt + 4 g + e of the chunk against query c
            f32x4 sc[2] = { splat4(0.0f), splat4(0.0f) };
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b < nb) {
                    const f16x8 qh = qop[(2 * b) * kWave + lane];
                    const f16x8 ql = qop[(2 * b + 1) * kWave + lane];
                    f16x8 k[2];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        uint32_t w[C::kStep];
#pragma unroll
                        for (int i = 0; i < C::kStep; ++i) {
                            const int off = 16 * mt * rb + b * UNIT + 4 * i;
                            w[i]          = b % 2 == 0 ? k0.at(off) : k1.at(off - 2);
                        }
                        k[mt] = C::k_codes(magic, w);
                    }
                    f32x4 x[2];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        x[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[mt], qh, splat4(0.0f), 0, 0, 0);
                    }
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        x[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[mt], ql, x[mt], 0, 0, 0);
                    }
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const f32x4 d = *reinterpret_cast<const f32x4 *>(kd + b * kChunk + 16 * mt + 4 * g);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            sc[mt][e] = __builtin_fmaf(d[e], x[mt][e], sc[mt][e]);
                        }
                    }
                }
            }
            const bool all = j0 + keys - 1 <= base && (a.window == 0 || j0 > p1 - a.window || j0 + keys <= a.sinks);
            float      top = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (a NaN, of a query that is not finite, becomes +infinity, and the weights NaN)
                    sc[mt][e] = fminf(sc[mt][e] * qscale, own[e]);
                }
            }
            if (!all) {  // keys that some queries do not see
                int g4 = 4 * g;
                asm volatile("" : "+v"(g4));  // (the rows' keys are not to wait in registers for this)
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[mt][e] = sees(a, p, j0 + ((16 * mt + g4 + e) >> f.hgs)) ? sc[mt][e] : -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    top = fmaxf(top, sc[mt][e]);
                }
            }
            top             = max_quarters(top);
            const float now = fminf(less, shift_for(top, kPShift));
            if (__any(now < less)) {
                const float alpha = shift_change(less, now);
                l *= alpha;
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    o[u] *= alpha;
                }
            }
            less            = now;
            const float add = shift_added(less);
            f16x2 ph[4], pl[4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(sc[mt][e] + add);
                    l += w[e];
                }
                split2(w[0], w[1], ph[2 * mt], pl[2 * mt]);
                split2(w[2], w[3], ph[2 * mt + 1], pl[2 * mt + 1]);
            }
            const f16x8 bh = join8(ph[0], ph[1], ph[2], ph[3]);
            const f16x8 bl = join8(pl[0], pl[1], pl[2], pl[3]);

            // operand element e of quarter g is row 4 g + e, then 16 + 4 g + e - 4
            auto turn = [&](float by) {
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    o[u] *= by;
                }
            };
            auto products = [&](const _Float16 * ds) {
#pragma unroll
                for (int s = 0; s < SLOTS; ++s) {
                    uint32_t w[8];
                    f16x2    d[4];
                    const f16x4 d0 = *reinterpret_cast<const f16x4 *>(ds + vblock[s] * kChunk + 4 * g);
                    const f16x4 d1 = *reinterpret_cast<const f16x4 *>(ds + vblock[s] * kChunk + 16 + 4 * g);
                    d[0] = f16x2{ d0[0], d0[1] }, d[1] = f16x2{ d0[2], d0[3] };
                    d[2] = f16x2{ d1[0], d1[1] }, d[3] = f16x2{ d1[2], d1[3] };
                    const LdsWords v0(vl, vword[s]);
                    const LdsWords v1(vl, vword[s] + 2);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int off = ((e < 4 ? 0 : 12) + e) * rb;
                        w[e]          = nb % 2 == 0 || e % 2 == 0 ? v0.at(off) : v1.at(off - 2);
                    }
                    // kAtOnce tiles at a time, so that their products need not wait for each other
                    auto tiles = [&](auto uc) {
                        constexpr int U = kAtOnce * decltype(uc)::value;
                        f16x8         ah[kAtOnce], al[kAtOnce];
                        auto          pieces = [&](auto vc) {
                            constexpr int V = decltype(vc)::value;
                            f16x2         hi[4], lo[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const f16x2 code = C::template v_codes<U + V>(magic, w[2 * e], w[2 * e + 1]);
                                hi[e]            = code * d[e];
                                lo[e]            = __builtin_elementwise_fma(code, d[e], -hi[e]);
                            }
                            ah[V] = join8(hi[0], hi[1], hi[2], hi[3]);
                            al[V] = join8(lo[0], lo[1], lo[2], lo[3]);
                        };
                        for_each(std::make_integer_sequence<int, kAtOnce>{}, pieces);
                        f32x4 * x = o + s * C::kTiles + U;
#pragma unroll
                        for (int v = 0; v < kAtOnce; ++v) {
                            x[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[v], bh, x[v], 0, 0, 0);
                        }
#pragma unroll
                        for (int v = 0; v < kAtOnce; ++v) {
                            x[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[v], bl, x[v], 0, 0, 0);
                        }
#pragma unroll
                        for (int v = 0; v < kAtOnce; ++v) {
                            x[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[v], bh, x[v], 0, 0, 0);
                        }
                    };
                    for_each(std::make_integer_sequence<int, C::kTiles / kAtOnce>{}, tiles);
                }
            };
            if (large) {
                turn(1.0f / kLargeBy);
                products(vd + NB * kChunk);
                turn(kLargeBy);
            }
            products(vd);
        }
        l = sum_quarters(l);

        // the waves' results joined in LDS: [wave][value][lane], then -less and l of a column
        __syncthreads();
        float * of = reinterpret_cast<float *>(lds);
        float * ml = of + WAVES * TILES * 4 * kWave;
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                of[((wave * TILES + u) * 4 + e) * kWave + lane] = o[u][e];
            }
        }
        if (g == 0) {
            ml[(wave * 16 + c) * 2]     = -less;
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
            part[w] = __builtin_amdgcn_exp2f(ml[(w * 16 + c) * 2] - ref);
            l += part[w] * ml[(w * 16 + c) * 2 + 1];
        }
        if (live) {
            float * out;
            float   by = 1.0f;
            if (u0 == 0 && u1 == at.units) {
                out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
                by  = over(l, p >= 0);
            } else {
                const int which = u0 == 0 ? 1 : 0;
                out             = few_o(f, wg, which, c);
                if (wave == 0 && g == 0) {
                    float * pml = few_ml(f, wg, which, c);
                    pml[0]      = top;
                    pml[1]      = l;
                }
            }
            // four values of a column a thread, so that a row is written in runs of 64 bytes
            for (int dim = threadIdx.x / 16 * 4; dim < a.hd; dim += 16 * WAVES) {
                f32x4 v = splat4(0.0f);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = C::v_place(dim + k);
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) {
                        v[k] += part[w] * of[w * TILES * 4 * kWave + at + c];
                    }
                }
                *reinterpret_cast<f32x4u *>(out + dim) = v * by;
            }
        }
        unit = begin + u1;
        if (unit >= last) {
            return;
        }
        __syncthreads();  // the next group's chunks go where the results were
        begin = unit;
        if (++hg == f.groups) {
            hg = 0;
            do {
                at.units = few_units(f, ++n);
            } while (at.units == 0);
        }
    }
}

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join_few(const FewArgs f, int64_t row0) {
    join_few<HD>(f, row0 + blockIdx.x);
}

// Whether the rows of HG heads lie one after the other, keys evenly apart and
// 16- or 4-byte pieces of them aligned. `together`: all keys are one run.
bool few_layout(const shp_tensor & c, int hgs, int piece, bool & together) {
    const size_t rb  = kv_bytes_of_row(c);
    const size_t run = rb << hgs;
    const size_t p   = static_cast<size_t>(piece);
    if ((hgs > 0 && c.nb[1] != rb) || reinterpret_cast<uintptr_t>(c.data) % p != 0 || (c.ne[3] > 1 && c.nb[3] % p != 0) ||
        ((c.ne[1] >> hgs) > 1 && (c.nb[1] << hgs) % p != 0)) {
        return false;
    }
    together = c.ne[2] == 1 || c.nb[2] == run;
    // a descriptor's last bytes are read by the dword
    return (run + (together ? static_cast<size_t>(c.ne[2] - 1) * run : size_t{ 0 })) % 4 == 0;
}

bool few_runs(const shp_tensor & c, int hgs, int piece) {
    const size_t p = static_cast<size_t>(piece);
    return (kv_bytes_of_row(c) << hgs) % p == 0 && c.nb[2] % p == 0 && c.nb[2] < (size_t{ 1 } << 25);  // 32 keys within a descriptor's 2^30 bytes
}

template <int KIND, int NB, int BYTES, bool RUNS, int WAVES> shp_status_t launch_few_as(FewArgs & f, hipStream_t stream) {
    using C             = Codes<KIND>;
    constexpr int TILES = (NB * C::kWords + 15) / 16 * C::kTiles;
    const int     rb    = f.nb * kv_unit_bytes(KIND);
    f.wave_lds          = 2 * kChunk * rb + NB * kChunk * 8;
    const int join      = WAVES * (TILES * 4 * kWave + 32) * 4;
    const int stage     = few_shared(NB, WAVES) + f.wave_lds * WAVES;
    const int lds       = stage > join ? stage : join;
    hipLaunchKernelGGL((k_attn_few<KIND, NB, BYTES, RUNS, WAVES>), dim3(static_cast<unsigned>(f.wgs)), dim3(64 * WAVES), lds, stream, f);
    const shp_status_t st = launch_status();
    if (st != SHP_OK || f.a.work == nullptr) {
        return st;  // no group was split
    }
    constexpr int HD   = NB <= 2 ? 64 : NB <= 4 ? 128 : 256;
    const int64_t rows = static_cast<int64_t>(f.a.N) * f.a.KV * f.a.T * f.a.G;
    return in_launches(rows, kJoinThreads, [&](int64_t first, dim3 grid) {
        hipLaunchKernelGGL((k_attn_join_few<HD>), grid, dim3(kJoinThreads), 0, stream, f, first);
    });
}

template <int KIND> shp_status_t launch_few(const AttnArgs & a, const AttnPlan & p, int piece, int32_t run, hipStream_t stream) {
    FewArgs f{};
    f.a      = a;
    f.hgs    = p.hgs;
    f.shift  = 5 - p.hgs;
    f.groups = a.KV >> p.hgs;
    f.wgs    = p.wgs;
    f.fwgs   = make_fastdiv(static_cast<uint32_t>(p.wgs));
    f.per    = p.per;
    f.fper   = make_fastdiv(static_cast<uint32_t>(p.per));
    f.cols   = a.T * a.G;
    f.nb     = a.hd / kKvBlock;
    f.pieces = kChunk * f.nb * kv_unit_bytes(KIND) / piece;
    f.run    = run;
    f.frun   = make_fastdiv(static_cast<uint32_t>(run > 0 ? run : 1));
    f.fcols  = make_fastdiv(static_cast<uint32_t>(f.cols));
    auto go = [&](auto nb, auto waves) {
        constexpr int NB = decltype(nb)::value, WAVES = decltype(waves)::value;
        if constexpr (NB <= 4) {
            if (piece == 4) {
                return launch_few_as<KIND, NB, 4, true, WAVES>(f, stream);
            }
        }
        return run > 0 ? launch_few_as<KIND, NB, 16, true, WAVES>(f, stream) : launch_few_as<KIND, NB, 16, false, WAVES>(f, stream);
    };
    using Four = std::integral_constant<int, 4>;
    switch (f.nb) {
        case 1:
            return go(std::integral_constant<int, 1>{}, Four{});
        case 2:
            return go(std::integral_constant<int, 2>{}, Four{});
        case 3:
            return go(std::integral_constant<int, 3>{}, Four{});
        case 4:
            return go(Four{}, Four{});
        default:
            return go(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    }
}

}  // namespace

// The piece size in which k_attn_few can read both caches, or 0; `run` as in FewArgs.
int few_piece(const shp_tensor & k, const shp_tensor & v, int hgs, int32_t & run) {
    for (int piece : { 16, 4 }) {
        if (piece == 4 && k.ne[0] > 4 * kKvBlock) {
            break;  // a lane would hold 36 to 68 pieces
        }
        bool kt = false, vt = false;
        if (!few_layout(k, hgs, piece, kt) || !few_layout(v, hgs, piece, vt)) {
            continue;
        }
        if (kt && vt && piece == 16) {
            run = 0;
            return piece;
        }
        if (few_runs(k, hgs, piece) && few_runs(v, hgs, piece)) {
            run = static_cast<int32_t>((kv_bytes_of_row(k) << hgs) / static_cast<size_t>(piece));
            return piece;
        }
    }
    return 0;
}

shp_status_t launch_attn_few(int kind, const AttnArgs & a, const AttnPlan & p, int piece, int32_t run, hipStream_t stream) {
    return kind == kKvQ4 ? launch_few<kKvQ4>(a, p, piece, run, stream) : launch_few<kKvQ8>(a, p, piece, run, stream);
}

}  // namespace shp
