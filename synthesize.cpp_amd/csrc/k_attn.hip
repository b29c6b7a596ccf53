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
#include <utility>

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
// P is held times 2^15, so that its pieces keep their bits where it is small:
// a weight is off by at most 2^-40 of the largest, or 2^-23 of itself.
// ---------------------------------------------------------------------------

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int   kChunk   = 32;     // cache rows of a chunk
constexpr float kPShift  = 15.0f;  // P times 2^15, at most half of F16's range
constexpr int   kMaxWaves = 4;     // of a workgroup

__device__ __forceinline__ f16x2 as_f16x2(uint32_t v) {
    return __builtin_bit_cast(f16x2, v);
}

__device__ __forceinline__ f16x2 splat2(float v) {
    return f16x2{ static_cast<_Float16>(v), static_cast<_Float16>(v) };
}

__device__ __forceinline__ f16x8 join8(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return f16x8{ a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1] };
}

// v = hi + lo: F16 rounded, and what that left.
__device__ __forceinline__ void split2(float a, float b, f16x2 & hi, f16x2 & lo) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    hi = __builtin_convertvector((f32x2{ a, b }), f16x2);
    lo = __builtin_convertvector((f32x2{ a - static_cast<float>(hi[0]), b - static_cast<float>(hi[1]) }), f16x2);
}

// How a cache type's bytes become matrix operands.
//   kWords   dwords of codes in 32 values
//   kTiles   values of a dword: each is the row of another 16-row tile of V^T
//   element  value index within 32 of operand element e of quarter g
//   k_codes  operand of the 32 values at `block`, quarter g
//   v_codes  from a dword of two keys: their values u as F16, without d
//   v_index  value index within 32 of value u of dword w
template <int KIND> struct Codes;

template <> struct Codes<kKvQ4> {
    static constexpr int kWords = 4;
    static constexpr int kTiles = 8;

    __device__ static constexpr int element(int g, int e) {
        return 4 * g + (e >= 4 ? 16 : 0) + (e & 1) * 2 + ((e >> 1) & 1);
    }

    // n in a mantissa's low bits: 0x6400 | n is 1024 + n, 0x5400 | n << 4 is 64 + n
    __device__ static f16x2 low(uint32_t w) { return as_f16x2((w & 0x000f000fu) | 0x64006400u) - splat2(1032.0f); }

    __device__ static f16x2 high(uint32_t w) { return as_f16x2((w & 0x00f000f0u) | 0x54005400u) - splat2(72.0f); }

    __device__ static f16x8 k_codes(const char * block, int g) {
        const uint32_t w = *reinterpret_cast<const u32_at2 *>(block + 2 + 4 * g);
        return join8(low(w), low(w >> 8), high(w), high(w >> 8));
    }

    __device__ static int word_offset(int w) { return (w >> 2) * 18 + 2 + 4 * (w & 3); }

    template <int U> __device__ static f16x2 v_codes(uint32_t w0, uint32_t w1) {
        constexpr uint32_t kSel = 0x0c040c00u + (U >> 1) * 0x00010001u;  // byte U/2 of w0 and of w1
        const uint32_t     x    = __builtin_amdgcn_perm(w1, w0, kSel);
        return U & 1 ? high(x) : low(x);
    }

    __device__ static int v_index(int w, int u) { return 32 * (w >> 2) + 4 * (w & 3) + (u >> 1) + 16 * (u & 1); }
};

template <> struct Codes<kKvQ8> {
    static constexpr int kWords = 8;
    static constexpr int kTiles = 4;

    __device__ static constexpr int element(int g, int e) { return 8 * g + e; }

    // q + 128 in a mantissa's low bits
    __device__ static f16x2 biased(uint32_t x) { return as_f16x2(x | 0x64006400u) - splat2(1152.0f); }

    __device__ static f16x8 k_codes(const char * block, int g) {
        const uint32_t w0 = *reinterpret_cast<const u32_at2 *>(block + 2 + 8 * g) ^ 0x80808080u;
        const uint32_t w1 = *reinterpret_cast<const u32_at2 *>(block + 6 + 8 * g) ^ 0x80808080u;
        return join8(biased(__builtin_amdgcn_perm(0, w0, 0x0c010c00u)), biased(__builtin_amdgcn_perm(0, w0, 0x0c030c02u)),
                     biased(__builtin_amdgcn_perm(0, w1, 0x0c010c00u)), biased(__builtin_amdgcn_perm(0, w1, 0x0c030c02u)));
    }

    __device__ static int word_offset(int w) { return (w >> 3) * 34 + 2 + 4 * (w & 7); }

    template <int U> __device__ static f16x2 v_codes(uint32_t w0, uint32_t w1) {
        return biased(__builtin_amdgcn_perm(w1 ^ 0x80808080u, w0 ^ 0x80808080u, 0x0c040c00u + U * 0x00010001u));
    }

    __device__ static int v_index(int w, int u) { return 4 * w + u; }
};

struct FewArgs {
    AttnArgs a;
    int32_t  hgs;      // log2 of HG
    int32_t  cols;     // queries of a kv head: T x G
    int32_t  nb;       // 32-value blocks of a row
    int32_t  pieces;   // of a chunk
    int32_t  run;      // pieces of a key's HG rows where keys are apart, 0 where a chunk is one run
    FastDiv  frun;
    FastDiv  fcols;
    int32_t  wave_lds;
};

template <class Go, int... U> __device__ __forceinline__ void for_each(std::integer_sequence<int, U...>, const Go & go) {
    (go(std::integral_constant<int, U>{}), ...);
}

// A piece of 16 or 4 bytes of a chunk as one load.
template <int BYTES> struct PieceOf {
    typedef u32x4 T;
};

template <> struct PieceOf<4> {
    typedef uint32_t T;
};

// One cache's chunk on its way to LDS: P pieces a lane.
template <int BYTES, int P> struct Staged {
    typename PieceOf<BYTES>::T piece[P];
};

// The pieces of the chunk at key j0, as this lane takes them. Where the chunk
// goes past the cache's end the bytes there are zero, and the piece that the
// end falls in is read in two-byte steps.
template <int BYTES, int P>
__device__ __forceinline__ void fetch(const FewArgs & f, const char * base, int64_t kt, const int32_t (&rel)[P], int lane,
                                      int32_t j0, int32_t keys, int row_bytes, Staged<BYTES, P> & s) {
    typedef typename PieceOf<BYTES>::T T;
    const char * at   = base + static_cast<int64_t>(j0) * kt;
    const int    left = f.a.cap - j0;
    if (left >= keys) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (lane + i * kWave < f.pieces) {
                s.piece[i] = *to_global(reinterpret_cast<const T *>(at + rel[i]));
            }
        }
        return;
    }
    const int bytes = (left << f.hgs) * row_bytes;  // of one run
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int p = lane + i * kWave;
        if (p < f.pieces) {
            const char * src  = at + rel[i];
            const int    have = f.run > 0 ? (static_cast<int>(fastdiv(static_cast<uint32_t>(p), f.frun)) < left ? BYTES : 0)
                                          : min(max(bytes - BYTES * p, 0), BYTES);
            if (have == BYTES) {
                s.piece[i] = *to_global(reinterpret_cast<const T *>(src));
            } else {
                uint32_t v[BYTES / 4] = {};
#pragma unroll
                for (int h = 0; h < BYTES / 2; ++h) {
                    if (2 * h < have) {
                        v[h / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(src)[h]) << (16 * (h & 1));
                    }
                }
                s.piece[i] = __builtin_bit_cast(T, v);
            }
        }
    }
}

// KIND Q4 or Q8, at most NB blocks a row, read in pieces of BYTES.
template <int KIND, int NB, int BYTES, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_attn_few(const FewArgs f) {
    using C                 = Codes<KIND>;
    constexpr int    UNIT   = kv_unit_bytes(KIND);
    constexpr int    SLOTS  = (NB * C::kWords + 15) / 16;
    constexpr int    TILES  = SLOTS * C::kTiles;
    constexpr int    P      = (kChunk * NB * UNIT / BYTES + kWave - 1) / kWave;
    extern __shared__ char lds[];
    const AttnArgs & a    = f.a;
    const int        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int        lane = threadIdx.x % kWave;
    const int        c    = lane & 15;
    const int        g    = lane >> 4;
    const int        split = blockIdx.x;
    const int        h0    = static_cast<int>(blockIdx.y) << f.hgs;
    const int        n     = blockIdx.z;
    const SeqLens    len   = seq_lens(a, n);
    if (len.count == 0) {
        return;
    }
    const int     keys = kChunk >> f.hgs;
    const int     mask = (1 << f.hgs) - 1;
    const int     rb   = f.nb * UNIT;
    const int32_t base = len.length - len.count;
    const int32_t p1   = len.length - 1;

    // this lane's query
    const int  hc   = static_cast<int>(fastdiv(static_cast<uint32_t>(c), f.fcols));
    const int  r    = c - hc * f.cols;
    const int  t    = static_cast<int>(fastdiv(static_cast<uint32_t>(r), a.fG));
    const int  head = (h0 + hc) * a.G + r - t * a.G;
    const bool live = hc <= mask && t < len.count;
    const int32_t p = live ? base + t : -1;

    f16x8 qh[NB], ql[NB];
    float qscale;
    {
        const float * qr  = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
        float         q[NB][8];
        float         top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[b][e] = live && b < f.nb ? qr[32 * b + C::element(g, e)] * a.scale : 0.0f;
                top     = fmaxf(top, fabsf(q[b][e]));
            }
        }
        top = max_quarters(top);
        // the largest of the row in [2^13, 2^14)
        const int ex    = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 127) - 13;
        const float to  = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        qscale          = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f16x2 h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                split2(q[b][2 * e] * to, q[b][2 * e + 1] * to, h[e], l[e]);
            }
            qh[b] = join8(h[0], h[1], h[2], h[3]);
            ql[b] = join8(l[0], l[1], l[2], l[3]);
        }
    }

    char *     kl = lds + wave * f.wave_lds;
    char *     vl = kl + kChunk * rb;
    float *    kd = reinterpret_cast<float *>(vl + kChunk * rb);
    _Float16 * vd = reinterpret_cast<_Float16 *>(kd + NB * kChunk);

    int32_t krel[P], vrel[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int pc  = lane + i * kWave;
        const int key = f.run > 0 ? static_cast<int>(fastdiv(static_cast<uint32_t>(pc), f.frun)) : 0;
        const int off = BYTES * (pc - key * f.run);
        krel[i]       = key * static_cast<int32_t>(f.run > 0 ? a.kt : 0) + off;
        vrel[i]       = key * static_cast<int32_t>(f.run > 0 ? a.vt : 0) + off;
    }
    const char * kb = a.k + n * a.kn + h0 * a.kh;
    const char * vb = a.v + n * a.vn + h0 * a.vh;

    // this lane's V words: word c + 16 s of each row
    int vword[SLOTS], vblock[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int w = min(c + 16 * s, f.nb * C::kWords - 1);
        vword[s]    = C::word_offset(w);
        vblock[s]   = w / C::kWords;
    }

    f32x4 o[TILES];
#pragma unroll
    for (int u = 0; u < TILES; ++u) {
        o[u] = splat4(0.0f);
    }
    float m = -INFINITY;
    float l = 0.0f;

    // the chunks of this split, every WAVES-th from `wave` on
    KeyTiles kt{ 0, 0, 0 };
    if (p1 >= 0) {
        const int32_t last = p1 >> (5 - f.hgs);
        if (a.window > 0) {
            kt.second = max(base - a.window + 1, 0) >> (5 - f.hgs);
            kt.first  = min((min(a.sinks, p1 + 1) + keys - 1) >> (5 - f.hgs), kt.second);
        }
        kt.n = kt.first + last - kt.second + 1;
    }
    const int per = (kt.n + a.nsplit - 1) / a.nsplit;
    const int end = min(kt.n, (split + 1) * per);
    int       i   = split * per + wave;

    Staged<BYTES, P> ks, vs;
    if (i < end) {
        const int32_t j0 = key_tile(kt, i) << (5 - f.hgs);
        fetch<BYTES, P>(f, kb, a.kt, krel, lane, j0, keys, rb, ks);
        fetch<BYTES, P>(f, vb, a.vt, vrel, lane, j0, keys, rb, vs);
    }
    for (; i < end; i += WAVES) {
        const int32_t j0 = key_tile(kt, i) << (5 - f.hgs);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int x = 0; x < P; ++x) {
            const int pc = lane + x * kWave;
            if (pc < f.pieces) {
                reinterpret_cast<typename PieceOf<BYTES>::T *>(kl)[pc] = ks.piece[x];
                reinterpret_cast<typename PieceOf<BYTES>::T *>(vl)[pc] = vs.piece[x];
            }
        }
        if (i + WAVES < end) {
            const int32_t jn = key_tile(kt, i + WAVES) << (5 - f.hgs);
            fetch<BYTES, P>(f, kb, a.kt, krel, lane, jn, keys, rb, ks);
            fetch<BYTES, P>(f, vb, a.vt, vrel, lane, jn, keys, rb, vs);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // d of the 32 rows: K's as F32, V's as they are; a V row that no query
        // of the call sees has d = 0
        {
            const int          row  = lane & 31;
            const bool         isk  = lane < 32;
            const char *       from = (isk ? kl : vl) + row * rb;
            const bool         keep = isk || seen_by(a, base, p1, j0 + (row >> f.hgs));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b < f.nb) {
                    const uint16_t d = *reinterpret_cast<const uint16_t *>(from + b * UNIT);
                    if (isk) {
                        kd[b * kChunk + row] = f16_bits_to_f32(d);
                    } else {
                        vd[b * kChunk + row] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(keep ? d : 0));
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();

        // scores: rows 16 mt + 4 g + e of the chunk against query c
        f32x4 sc[2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            sc[mt] = splat4(0.0f);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b < f.nb) {
                    const f16x8 k = C::k_codes(kl + (16 * mt + c) * rb + b * UNIT, g);
                    f32x4       x = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[b], splat4(0.0f), 0, 0, 0);
                    x             = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[b], x, 0, 0, 0);
                    const f32x4 d = *reinterpret_cast<const f32x4 *>(kd + b * kChunk + 16 * mt + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[mt][e] = __builtin_fmaf(d[e], x[e], sc[mt][e]);
                    }
                }
            }
        }
        float top = m;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int  row = 16 * mt + 4 * g + e;
                const bool see = (row & mask) == hc && sees(a, p, j0 + (row >> f.hgs));
                sc[mt][e]      = see ? sc[mt][e] * qscale : -INFINITY;
                top            = fmaxf(top, sc[mt][e]);
            }
        }
        top             = max_quarters(top);
        const float ref = top == -INFINITY ? 0.0f : top;
        if (__any(top > m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - ref);
            l *= alpha;
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                o[u] *= alpha;
            }
        }
        m = top;
        f16x2 ph[4], pl[4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = __builtin_amdgcn_exp2f(sc[mt][e] - (ref - kPShift));
                l += w[e];
            }
            split2(w[0], w[1], ph[2 * mt], pl[2 * mt]);
            split2(w[2], w[3], ph[2 * mt + 1], pl[2 * mt + 1]);
        }
        const f16x8 bh = join8(ph[0], ph[1], ph[2], ph[3]);
        const f16x8 bl = join8(pl[0], pl[1], pl[2], pl[3]);

        // operand element e of quarter g is row 4 g + e, then 16 + 4 g + e - 4
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            uint32_t w[8];
            f16x2    d[4];
            const f16x4 d0 = *reinterpret_cast<const f16x4 *>(vd + vblock[s] * kChunk + 4 * g);
            const f16x4 d1 = *reinterpret_cast<const f16x4 *>(vd + vblock[s] * kChunk + 16 + 4 * g);
            d[0] = f16x2{ d0[0], d0[1] }, d[1] = f16x2{ d0[2], d0[3] };
            d[2] = f16x2{ d1[0], d1[1] }, d[3] = f16x2{ d1[2], d1[3] };
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = (e < 4 ? 0 : 12) + 4 * g + e;
                w[e]          = *reinterpret_cast<const u32_at2 *>(vl + row * rb + vword[s]);
            }
            auto tile = [&](auto uc) {
                constexpr int U = decltype(uc)::value;
                f16x2         hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 code = C::template v_codes<U>(w[2 * e], w[2 * e + 1]);
                    hi[e]            = code * d[e];
                    lo[e]            = __builtin_elementwise_fma(code, d[e], -hi[e]);
                }
                const f16x8 ah = join8(hi[0], hi[1], hi[2], hi[3]);
                const f16x8 al = join8(lo[0], lo[1], lo[2], lo[3]);
                f32x4 &     x  = o[s * C::kTiles + U];
                x              = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, x, 0, 0, 0);
                x              = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, x, 0, 0, 0);
                x              = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, x, 0, 0, 0);
            };
            for_each(std::make_integer_sequence<int, C::kTiles>{}, tile);
        }
    }
    l = sum_quarters(l);

    // the waves' results joined in LDS: [wave][value][lane], then m and l of a column
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
        part[w] = __builtin_amdgcn_exp2f(ml[(w * 16 + c) * 2] - ref);
        l += part[w] * ml[(w * 16 + c) * 2 + 1];
    }
    if (!live) {
        return;
    }
    const int64_t row = ((static_cast<int64_t>(n) * a.KV + h0 + hc) * a.T + t) * a.G + r - t * a.G;
    float *       out;
    float         by = 1.0f;
    if (a.nsplit == 1) {
        out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
        by  = over(l, p >= 0);
    } else {
        out = partial_o(a, row, split);
        if (wave == 0 && g == 0) {
            float * pml = partial_ml(a, row, split);
            pml[0]      = top;
            pml[1]      = l;
        }
    }
    for (int u = wave; u < TILES; u += WAVES) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                v += part[w] * of[((w * TILES + u) * 4 + e) * kWave + lane];
            }
            const int word = 16 * (u / C::kTiles) + 4 * g + e;
            if (word < f.nb * C::kWords) {
                out[C::v_index(word, u % C::kTiles)] = v * by;
            }
        }
    }
}

// The splits of a row joined: a workgroup a row, whose threads take HD values
// of 256/HD of the splits each.
constexpr int kJoinThreads = 256;
constexpr int kMaxSplits   = 512;

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join(const AttnArgs a, int64_t row0) {
    constexpr int GROUPS = kJoinThreads / HD;
    __shared__ float weight[kMaxSplits];
    __shared__ float lane_max[kJoinThreads / kWave], lane_sum[kJoinThreads / kWave];
    __shared__ float sums[kJoinThreads];
    const int64_t row = row0 + blockIdx.x;
    const int     tid = threadIdx.x;
    const int64_t gq  = row % a.G;
    const int64_t t   = row / a.G % a.T;
    const int64_t h   = row / a.G / a.T % a.KV;
    const int     n   = static_cast<int>(row / a.G / a.T / a.KV);
    const SeqLens len = seq_lens(a, n);
    if (t >= len.count) {
        return;
    }
    const float * ml  = partial_ml(a, row, 0);
    float         top = -INFINITY;
    for (int s = tid; s < a.nsplit; s += kJoinThreads) {
        top = fmaxf(top, ml[2 * s]);
    }
    top = wave_max(top);
    if (tid % kWave == 0) {
        lane_max[tid / kWave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / kWave; ++w) {
        top = fmaxf(top, lane_max[w]);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    float       l   = 0.0f;
    for (int s = tid; s < a.nsplit; s += kJoinThreads) {
        const float w = ml[2 * s + 1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[2 * s] - ref);
        weight[s]     = w;
        l += w * ml[2 * s + 1];
    }
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        l += __shfl_xor(l, off);
    }
    if (tid % kWave == 0) {
        lane_sum[tid / kWave] = l;
    }
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / kWave; ++w) {
        l += lane_sum[w];
    }
    const int     dim   = tid % HD;
    const int     group = tid / HD;
    const float * o     = partial_o(a, row, 0) + dim;
    float         v     = 0.0f;
    if (dim < a.hd) {
#pragma unroll 8
        for (int s = group; s < a.nsplit; s += GROUPS) {
            const float w = weight[s];  // 0: no key, and nothing that counts in o
            v += w != 0.0f ? o[static_cast<int64_t>(s) * a.hd] * w : 0.0f;
        }
    }
    sums[tid] = v;
    __syncthreads();
    if (group == 0 && dim < a.hd) {
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) {
            v += sums[k * HD + dim];
        }
        float * out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + (h * a.G + gq) * a.yh);
        out[dim]    = v * over(l, len.length - len.count + t >= 0);
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

struct AttnPlan {
    bool    few;
    int32_t hgs;
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
    const int64_t kv = k_cache->ne[1];
    p.tiles          = static_cast<int32_t>((rows + 15) / 16);
    p.few            = rows <= 16 && kv_blocks(kv_kind(k_cache->type));
    p.hgs            = 0;
    if (p.few) {
        while ((rows << (p.hgs + 1)) <= 16 && kv % (int64_t{ 2 } << p.hgs) == 0 &&
               k_cache->nb[1] == kv_bytes_of_row(*k_cache)) {
            ++p.hgs;
        }
        const int64_t chunks = ((keys << p.hgs) + kChunk - 1) / kChunk;
        p.nsplit             = plan_splits((kv >> p.hgs) * q->ne[3], (chunks + kMaxWaves - 1) / kMaxWaves, 1024);
    } else {
        p.nsplit = plan_splits(p.tiles * kv * q->ne[3], (keys + 63) / 64, 2048);
    }
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
    auto          go   = [&](auto kernel) {
        return in_launches(rows, kJoinThreads, [&](int64_t first, dim3 grid) {
            hipLaunchKernelGGL(kernel, grid, dim3(kJoinThreads), 0, stream, a, first);
        });
    };
    return a.hd <= 64 ? go(k_attn_join<64>) : a.hd <= 128 ? go(k_attn_join<128>) : go(k_attn_join<256>);
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
    return true;
}

bool few_runs(const shp_tensor & c, int hgs, int piece) {
    const size_t p = static_cast<size_t>(piece);
    return (kv_bytes_of_row(c) << hgs) % p == 0 && c.nb[2] % p == 0 && c.nb[2] < (size_t{ 1 } << 26);
}

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
        if (kt && vt) {
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

template <int KIND, int NB, int BYTES, int WAVES> shp_status_t launch_few_as(FewArgs & f, hipStream_t stream) {
    using C             = Codes<KIND>;
    constexpr int TILES = (NB * C::kWords + 15) / 16 * C::kTiles;
    const int     rb    = f.nb * kv_unit_bytes(KIND);
    f.wave_lds          = 2 * kChunk * rb + NB * kChunk * 6;
    const int join      = WAVES * (TILES * 4 * kWave + 32) * 4;
    const int lds       = f.wave_lds * WAVES > join ? f.wave_lds * WAVES : join;
    const dim3 grid(static_cast<unsigned>(f.a.nsplit), static_cast<unsigned>(f.a.KV >> f.hgs), static_cast<unsigned>(f.a.N));
    hipLaunchKernelGGL((k_attn_few<KIND, NB, BYTES, WAVES>), grid, dim3(64 * WAVES), lds, stream, f);
    return launch_status();
}

template <int KIND> shp_status_t launch_few(const AttnArgs & a, int hgs, int piece, int32_t run, hipStream_t stream) {
    FewArgs f{};
    f.a      = a;
    f.hgs    = hgs;
    f.cols   = a.T * a.G;
    f.nb     = a.hd / kKvBlock;
    f.pieces = kChunk * f.nb * kv_unit_bytes(KIND) / piece;
    f.run    = run;
    f.frun   = make_fastdiv(static_cast<uint32_t>(run > 0 ? run : 1));
    f.fcols  = make_fastdiv(static_cast<uint32_t>(f.cols));
    if (f.nb <= 4) {
        return piece == 16 ? launch_few_as<KIND, 4, 16, 4>(f, stream) : launch_few_as<KIND, 4, 4, 4>(f, stream);
    }
    return launch_few_as<KIND, 8, 16, 2>(f, stream);
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
    const hipStream_t s     = as_stream(stream);
    const int         kind  = kv_kind(k_cache->type);
    int32_t           run   = 0;
    const int         piece = p.few ? few_piece(*k_cache, *v_cache, p.hgs, run) : 0;
    if (piece > 0) {
        st = kind == kKvQ4 ? launch_few<kKvQ4>(a, p.hgs, piece, run, s) : launch_few<kKvQ8>(a, p.hgs, piece, run, s);
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
