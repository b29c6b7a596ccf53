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
    float *         work;    // partials of nsplit > 1: [rows][nsplit][hd4], then m and l [rows][nsplit][2]
    int64_t         qh, qt, qn, kh, kt, kn, vh, vt, vn, yh, yt, yn;
    float           scale;  // times log2 e
    int32_t         window;  // 0: none
    int32_t         sinks;
    int32_t         T;
    int32_t         G;  // query heads of a kv head
    int32_t         KV;
    int32_t         N;
    int32_t         hd;
    int32_t         hd4;  // hd up to a multiple of 4: a partial row's length
    int32_t         cap;
    int32_t         nsplit;
    int32_t         tiles;  // of rows
    FastDiv         fG;
    FastDiv         fsplit;
    FastDiv         fKV;
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
    return a.work + (row * a.nsplit + split) * a.hd4;
}

__device__ __forceinline__ float * partial_ml(const AttnArgs & a, int64_t row, int split) {
    const int64_t rows = static_cast<int64_t>(a.N) * a.KV * a.T * a.G;
    return a.work + rows * a.nsplit * a.hd4 + (row * a.nsplit + split) * 2;
}

// The maximum, or the sum, over the four lanes c, c+16, c+32, c+48, in each of
// them: lanes change places with those 16, then 32 away, without LDS.
struct Pair {
    float a, b;
};

__device__ __forceinline__ Pair swap16(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return Pair{ __uint_as_float(r[0]), __uint_as_float(r[1]) };
#else
    return Pair{ v, v };
#endif
}

__device__ __forceinline__ Pair swap32(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return Pair{ __uint_as_float(r[0]), __uint_as_float(r[1]) };
#else
    return Pair{ v, v };
#endif
}

__device__ __forceinline__ float max_quarters(float v) {
    const Pair p = swap16(v);
    const Pair q = swap32(fmaxf(p.a, p.b));
    return fmaxf(q.a, q.b);
}

__device__ __forceinline__ float sum_quarters(float v) {
    const Pair p = swap16(v);
    const Pair q = swap32(p.a + p.b);
    return q.a + q.b;
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

// Exponents that turn an integer in a mantissa's low bits into an F16. Held in
// vector registers once a kernel, behind the compiler's back: (w & mask) | bits
// is then one v_and_or_b32, which takes at most one scalar or literal operand.
struct Magic {
    uint32_t e1024;  // 0x6400 | n is 1024 + n
    uint32_t e64;    // 0x5400 | n << 4 is 64 + n

    __device__ Magic() : e1024(0x64006400u), e64(0x54005400u) {
#if defined(__HIP_DEVICE_COMPILE__)
        asm("" : "+v"(e1024), "+v"(e64));
#endif
    }
};

// How a cache type's bytes become matrix operands.
//   kWords   dwords of codes in 32 values
//   kTiles   values of a dword: each is the row of another 16-row tile of V^T
//   quarter g's eight operand elements are the values kFirst g + order(0..3)
//   and kSecond more
//   kStep    dwords of codes in a quarter's operand
//   k_codes  that operand
//   v_codes  from a dword of two keys: their values u as F16, without d
//   v_index  value index within 32 of value u of dword w
template <int KIND> struct Codes;

template <> struct Codes<kKvQ4> {
    static constexpr int kWords = 4;
    static constexpr int kStep  = 1;
    static constexpr int kTiles = 8;

    static constexpr int kFirst  = 4;
    static constexpr int kSecond = 16;

    __device__ static constexpr int order(int e) { return (e & 1) * 2 + (e >> 1); }

    __device__ static f16x2 low(const Magic & m, uint32_t w) { return as_f16x2((w & 0x000f000fu) | m.e1024) - splat2(1032.0f); }

    __device__ static f16x2 high(const Magic & m, uint32_t w) { return as_f16x2((w & 0x00f000f0u) | m.e64) - splat2(72.0f); }

    __device__ static f16x8 k_codes(const Magic & m, const uint32_t (&w)[1]) {
        return join8(low(m, w[0]), low(m, w[0] >> 8), high(m, w[0]), high(m, w[0] >> 8));
    }

    __device__ static int word_offset(int w) { return (w >> 2) * 18 + 2 + 4 * (w & 3); }

    template <int U> __device__ static f16x2 v_codes(const Magic & m, uint32_t w0, uint32_t w1) {
        constexpr uint32_t kSel = 0x0c040c00u + (U >> 1) * 0x00010001u;  // byte U/2 of w0 and of w1
        const uint32_t     x    = __builtin_amdgcn_perm(w1, w0, kSel);
        return U & 1 ? high(m, x) : low(m, x);
    }

    __device__ static int v_index(int w, int u) { return 32 * (w >> 2) + 4 * (w & 3) + (u >> 1) + 16 * (u & 1); }
};

template <> struct Codes<kKvQ8> {
    static constexpr int kWords = 8;
    static constexpr int kStep  = 2;
    static constexpr int kTiles = 4;

    static constexpr int kFirst  = 8;
    static constexpr int kSecond = 4;

    __device__ static constexpr int order(int e) { return e; }

    // from q + 128
    __device__ static f16x2 biased(const Magic & m, uint32_t x) { return as_f16x2(x | m.e1024) - splat2(1152.0f); }

    __device__ static f16x8 k_codes(const Magic & m, const uint32_t (&w)[2]) {
        const uint32_t a = w[0] ^ 0x80808080u;
        const uint32_t b = w[1] ^ 0x80808080u;
        return join8(biased(m, __builtin_amdgcn_perm(0, a, 0x0c010c00u)), biased(m, __builtin_amdgcn_perm(0, a, 0x0c030c02u)),
                     biased(m, __builtin_amdgcn_perm(0, b, 0x0c010c00u)), biased(m, __builtin_amdgcn_perm(0, b, 0x0c030c02u)));
    }

    __device__ static int word_offset(int w) { return (w >> 3) * 34 + 2 + 4 * (w & 7); }

    template <int U> __device__ static f16x2 v_codes(const Magic & m, uint32_t w0, uint32_t w1) {
        return biased(m, __builtin_amdgcn_perm(w1 ^ 0x80808080u, w0 ^ 0x80808080u, 0x0c040c00u + U * 0x00010001u));
    }

    __device__ static int v_index(int w, int u) { return 4 * w + u; }
};

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
    int32_t  groups;   // of HG heads
    int32_t  wgs;      // workgroups that share the work
    FastDiv  fwgs;
    int32_t  per;      // chunks of a unit
    FastDiv  fper;
};

// How the work is dealt out. A sequence's chunks make units of one chunk or a
// few for each of a workgroup's waves; sequence after sequence, head group after head
// group, the units of the call stand in one line, of which every workgroup
// takes an equal stretch. So lengths may differ as they like (64 streams of 512
// to 8192 rows, MI355X: XX us, YY with an equal number of workgroups for each
// sequence). A stretch that ends inside a group leaves a partial result; a
// workgroup has two at most, of the group that it begins in and did not begin
// (0), and of the one that it began and did not end (1).
constexpr int kCols = 16;

__device__ __forceinline__ float * few_o(const FewArgs & f, int wg, int which, int col) {
    return f.a.work + (static_cast<int64_t>(wg * 2 + which) * kCols + col) * f.a.hd4;
}

__device__ __forceinline__ float * few_ml(const FewArgs & f, int wg, int which, int col) {
    return f.a.work + static_cast<int64_t>(f.wgs) * 2 * kCols * f.a.hd4 + ((wg * 2 + which) * kCols + col) * 2;
}

// A sequence's key chunks; `len` as seq_lens gives it.
__device__ __forceinline__ KeyTiles few_tiles(const FewArgs & f, const SeqLens & len) {
    const AttnArgs & a     = f.a;
    const int        shift = 5 - f.hgs;
    const int32_t    base  = len.length - len.count;
    const int32_t    p1    = len.length - 1;
    KeyTiles         kt{ 0, 0, 0 };
    if (p1 >= 0) {
        if (a.window > 0) {
            kt.second = max(base - a.window + 1, 0) >> shift;
            kt.first  = min((min(a.sinks, p1 + 1) + (1 << shift) - 1) >> shift, kt.second);
        }
        kt.n = kt.first + (p1 >> shift) - kt.second + 1;
    }
    return kt;
}

// Units of sequence n and head group: at least one where it has a query, which
// then writes its zeros.
__device__ __forceinline__ int few_units(const FewArgs & f, int n) {
    const SeqLens len = seq_lens(f.a, n);
    return len.count == 0 ? 0 : max(static_cast<int>(fastdiv(static_cast<uint32_t>(few_tiles(f, len).n + f.per - 1), f.fper)), 1);
}

// The line's length, and the place of sequence n in it (units of one head
// group), for a whole wave: 64 sequences at a time, a sum over lanes.
struct Line {
    int32_t before;
    int32_t total;
};

__device__ __forceinline__ Line few_line(const FewArgs & f, int n, int lane) {
    if (f.a.N == 1) {
        return Line{ 0, few_units(f, 0) };
    }
    Line s{ 0, 0 };
    for (int first = 0; first < f.a.N; first += kWave) {
        const int i     = first + lane;
        int       units = i < f.a.N ? few_units(f, i) : 0;
        int       below = i < n ? units : 0;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) {
            units += __shfl_xor(units, off);
            below += __shfl_xor(below, off);
        }
        s.total += __builtin_amdgcn_readfirstlane(units);
        s.before += __builtin_amdgcn_readfirstlane(below);
    }
    return s;
}

// The sequence that unit u of the line falls in.
struct Place {
    int32_t n;
    int32_t units;   // of one head group of it
    int32_t before;  // of all head groups of the sequences before it
};

__device__ __forceinline__ Place few_find(const FewArgs & f, int32_t u, int lane) {
    if (f.a.N == 1) {
        return Place{ 0, few_units(f, 0), 0 };
    }
    int32_t before = 0;
    for (int first = 0; first < f.a.N; first += kWave) {
        const int i     = first + lane;
        const int units = i < f.a.N ? few_units(f, i) : 0;
        int       sum   = units;
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) {
            const int v = __shfl_up(sum, off);
            sum += lane >= off ? v : 0;
        }
        const uint64_t past = __ballot(before + sum * f.groups > u);
        if (past != 0) {
            const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int k = __builtin_amdgcn_readlane(units, l);
            return Place{ first + l, k, before + (__builtin_amdgcn_readlane(sum, l) - k) * f.groups };
        }
        before += __builtin_amdgcn_readlane(sum, kWave - 1) * f.groups;
    }
    return Place{ 0, 1, u };  // (u lies in the line)
}

// Where workgroup wg's stretch of `total` units begins, and whose unit u is.
__device__ __forceinline__ int32_t few_start(const FewArgs & f, int32_t total, int32_t wg) {
    const int32_t each = static_cast<int32_t>(fastdiv(static_cast<uint32_t>(total), f.fwgs));
    return each * wg + min(wg, total - each * f.wgs);
}

__device__ __forceinline__ int32_t few_owner(const FewArgs & f, int32_t total, int32_t u) {
    const int32_t each = static_cast<int32_t>(fastdiv(static_cast<uint32_t>(total), f.fwgs));
    const int32_t more = total - each * f.wgs;  // workgroups with one more
    return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each;
}

template <class Go, int... U> __device__ __forceinline__ void for_each(std::integer_sequence<int, U...>, const Go & go) {
    (go(std::integral_constant<int, U>{}), ...);
}

// One cache's chunk on its way to LDS: a lane's pieces of 16 or 4 bytes, read
// through a buffer descriptor that ends with the cache's rows, so that what is
// behind them reads as zero without a test in the kernel.
typedef __amdgpu_buffer_rsrc_t Rsrc;

__device__ __forceinline__ Rsrc rows_from(const char * at, int64_t bytes) {
    constexpr int kRaw32 = 0x00027000;  // 32-bit data, no swizzle
    const int64_t most   = int64_t{ 1 } << 30;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(at), 0, static_cast<int>(bytes < most ? bytes : most), kRaw32);
}

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
__global__ __launch_bounds__(64 * WAVES, NB <= 4 ? 2 : 1) void k_attn_few(const FewArgs f) {
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
    const int        wg   = blockIdx.x;
    const int        keys = kChunk >> f.hgs;
    const int        mask = (1 << f.hgs) - 1;
    const int        nb   = NB <= 4 ? NB : f.nb;
    const int        rb   = nb * UNIT;
    const int32_t    total = few_line(f, 0, lane).total * f.groups;
    const int32_t    last  = few_start(f, total, wg + 1);
    int32_t          unit  = few_start(f, total, wg);

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
    Place   at    = few_find(f, unit, lane);
    int     n     = at.n;
    int     hg    = f.groups == 1 ? 0 : (unit - at.before) / at.units;
    int32_t begin = at.before + hg * at.units;  // the group's first unit
    for (;;) {
    const int     u0     = unit - begin;
    const int     u1     = min(last - begin, at.units);
    const int     h0     = hg << f.hgs;
    const SeqLens  len   = seq_lens(a, n);
    const KeyTiles kt    = few_tiles(f, len);
    const int32_t base   = len.length - len.count;
    const int32_t p1     = len.length - 1;
    const int     head   = (h0 + hc) * a.G + r - t * a.G;
    const bool    live   = hc <= mask && t < len.count;
    const int32_t p      = live ? base + t : -1;

    const char * kb = a.k + n * a.kn + h0 * a.kh;
    const char * vb = a.v + n * a.vn + h0 * a.vh;

    f32x4 o[TILES];
#pragma unroll
    for (int u = 0; u < TILES; ++u) {
        o[u] = splat4(0.0f);
    }
    float m = -INFINITY;
    float l = 0.0f;

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
        const int ex   = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 127) - 13;
        const float to = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        qscale         = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
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
        // d of the 32 rows: K's as F32, V's as they are; a V row that no query
        // of the call sees has d = 0
        {
            const int          row  = lane & 31;
            const bool         isk  = lane < 32;
            const char *       from = (isk ? kl : vl) + row * rb;
            const bool         keep = isk || seen_by(a, base, p1, j0 + (row >> f.hgs));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b < nb) {
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
        f32x4 sc[2] = { splat4(0.0f), splat4(0.0f) };
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b < nb) {
                const f16x8 qh = qop[(2 * b) * kWave + lane];
                const f16x8 ql = qop[(2 * b + 1) * kWave + lane];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    uint32_t w[C::kStep];
#pragma unroll
                    for (int i = 0; i < C::kStep; ++i) {
                        const int off = 16 * mt * rb + b * UNIT + 4 * i;
                        w[i]          = b % 2 == 0 ? k0.at(off) : k1.at(off - 2);
                    }
                    const f16x8 k = C::k_codes(magic, w);
                    f32x4       x = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh, splat4(0.0f), 0, 0, 0);
                    x             = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql, x, 0, 0, 0);
                    const f32x4 d = *reinterpret_cast<const f32x4 *>(kd + b * kChunk + 16 * mt + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[mt][e] = __builtin_fmaf(d[e], x[e], sc[mt][e]);
                    }
                }
            }
        }
        const bool all = j0 + keys - 1 <= base && (a.window == 0 || j0 > p1 - a.window || j0 + keys <= a.sinks);
        float      top = m;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (a NaN of its own head becomes +infinity, and the weights NaN)
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
            const LdsWords v0(vl, vword[s]);
            const LdsWords v1(vl, vword[s] + 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int off = ((e < 4 ? 0 : 12) + e) * rb;
                w[e]          = nb % 2 == 0 || e % 2 == 0 ? v0.at(off) : v1.at(off - 2);
            }
            auto tile = [&](auto uc) {
                constexpr int U = decltype(uc)::value;
                f16x2         hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 code = C::template v_codes<U>(magic, w[2 * e], w[2 * e + 1]);
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
    for (int u = wave; u < TILES; u += WAVES) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                v += part[w] * of[((w * TILES + u) * 4 + e) * kWave + lane];
            }
            const int word = 16 * (u / C::kTiles) + 4 * g + e;
            if (word < nb * C::kWords) {
                out[C::v_index(word, u % C::kTiles)] = v * by;
            }
        }
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

// ---------------------------------------------------------------------------
// Many queries (prompts): a workgroup takes 128 rows, 32 a wave, and 64 keys at
// a time, whose K and V it brings into LDS once, as matrix operands: K by row,
// V by column with the keys in the order in which the scores stand in
// registers. A block's code * d is exact as two F16 pieces; q and P are two
// pieces as well, and each product is hi hi + hi lo + lo hi (a 16-bit cache has
// no second piece). Matrix instructions 32x32x16: S^T = K Q^T has a query in
// each lane, O^T = V^T P^T too.
// ---------------------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileKeys  = 64;
constexpr int kWideRows  = 128;
constexpr int kWideBlock = 256;
constexpr int kVStride   = kTileKeys * 2 + 16;  // bytes of a column of V in LDS, off the banks' period

// A thread's part of a tile on its way to LDS: 32 values of a row of K, and of
// V the four values u = 0..3 of each of eight keys, those that lie next to each
// other in an operand: 16 s + 4 h + 0..3 and 8 more, group 2 s + h. In column
// `dim` of V the groups stand in the order group ^ (dim >> kTurn & 3): sixteen
// lanes that write a group of sixteen columns then meet every bank once (four
// times four without it: a third of the LDS unit's time).
template <int KIND> struct Part;

template <> struct Part<kKvQ4> {
    static constexpr bool kTwo  = true;
    static constexpr int  kTurn = 5;
    uint32_t              k[4];
    uint32_t              v[8];
    uint16_t              kd;
    uint16_t              vd[8];

    // the block `at` bytes into the tile
    __device__ void load_k(const Rsrc & r, int at) {
        kd = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k[i] = __builtin_amdgcn_raw_buffer_load_b32(r, at + 2 + 4 * i, 0, 0);
        }
    }

    // key e's word, `at` bytes into its row that is `row` bytes into the tile, and its d at `block`
    __device__ void load_v(int e, const Rsrc & r, int at, int block, int row) {
        v[e]  = __builtin_amdgcn_raw_buffer_load_b32(r, at, row, 0);
        vd[e] = __builtin_amdgcn_raw_buffer_load_b16(r, block, row, 0);
    }

    // item: word `item % words` and half item / words of its nibbles
    __device__ static int block_at(int item, int words) { return ((item % words) >> 2) * 18; }

    __device__ static int word_at(int item, int words) { return block_at(item, words) + 2 + 4 * (item & 3); }

    __device__ static int items(int nb) { return 8 * nb; }

    __device__ static int words(int nb) { return 4 * nb; }

    // value u of `item`
    __device__ static int index(int item, int words, int u) {
        const int w = item % words;
        return 32 * (w >> 2) + 4 * (w & 3) + u + (item >= words ? 16 : 0);
    }

    __device__ f16x8 k_codes(const Magic & m, int j) const {
        const uint32_t w[1] = { k[j] };
        return Codes<kKvQ4>::k_codes(m, w);
    }

    template <int U> __device__ f16x2 v_codes(const Magic & m, int e, int item, int words) const {
        const uint32_t shift = item >= words ? 4u : 0u;
        return Codes<kKvQ4>::v_codes<2 * U>(m, v[e] >> shift, v[e + 1] >> shift);
    }
};

template <> struct Part<kKvQ8> {
    static constexpr bool kTwo  = true;
    static constexpr int  kTurn = 4;
    uint32_t              k[8];
    uint32_t              v[8];
    uint16_t              kd;
    uint16_t              vd[8];

    __device__ void load_k(const Rsrc & r, int at) {
        kd = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k[i] = __builtin_amdgcn_raw_buffer_load_b32(r, at + 2 + 4 * i, 0, 0);
        }
    }

    __device__ void load_v(int e, const Rsrc & r, int at, int block, int row) {
        v[e]  = __builtin_amdgcn_raw_buffer_load_b32(r, at, row, 0);
        vd[e] = __builtin_amdgcn_raw_buffer_load_b16(r, block, row, 0);
    }

    __device__ static int block_at(int item, int) { return (item >> 3) * 34; }

    __device__ static int word_at(int item, int) { return block_at(item, 0) + 2 + 4 * (item & 7); }

    __device__ static int items(int nb) { return 8 * nb; }

    __device__ static int words(int nb) { return 8 * nb; }

    __device__ static int index(int item, int, int u) { return 4 * item + u; }

    __device__ f16x8 k_codes(const Magic & m, int j) const {
        const uint32_t w[2] = { k[2 * j], k[2 * j + 1] };
        return Codes<kKvQ8>::k_codes(m, w);
    }

    template <int U> __device__ f16x2 v_codes(const Magic & m, int e, int, int) const {
        return Codes<kKvQ8>::v_codes<U>(m, v[e], v[e + 1]);
    }
};

template <int KIND, int NB> constexpr int wide_lds() {
    constexpr int HD = NB * kKvBlock;
    return (kTileKeys * (HD * 2 + 16) + HD * kVStride) * (Part<KIND>::kTwo ? 2 : 1);
}

template <int KIND, int NB> __global__ __launch_bounds__(kWideBlock, 2) void k_attn_wide(const AttnArgs a) {
    using PartT             = Part<KIND>;
    using C                 = Codes<KIND>;
    constexpr int  HD       = NB * kKvBlock;
    constexpr int  UNIT     = kv_unit_bytes(KIND);
    constexpr int  KSTRIDE  = HD * 2 + 16;
    constexpr bool TWO      = PartT::kTwo;
    extern __shared__ char lds[];
    char * const   kh   = lds;
    char * const   kl   = kh + kTileKeys * KSTRIDE;  // (of two pieces)
    char * const   vh   = kl + (TWO ? kTileKeys * KSTRIDE : 0);
    char * const   vl   = vh + HD * kVStride;

    const int     tid   = threadIdx.x;
    const int     wave  = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int     lane  = tid % kWave;
    const int     c     = lane & 31;
    const int     g     = lane >> 5;
    // a kv head's workgroups share an XCD where there are eight heads; the longest rows first
    const int     part0 = static_cast<int>(fastdiv(blockIdx.x, a.fKV));
    const int     h     = static_cast<int>(blockIdx.x) - part0 * a.KV;
    const int     back  = static_cast<int>(fastdiv(static_cast<uint32_t>(part0), a.fsplit));
    const int     tile  = a.tiles - 1 - back;
    const int     split = part0 - back * a.nsplit;
    const int     n     = blockIdx.y;
    const SeqLens len   = seq_lens(a, n);
    auto          t_of  = [&](int r) { return static_cast<int>(fastdiv(static_cast<uint32_t>(r), a.fG)); };
    const int     t0    = t_of(tile * kWideRows);
    if (t0 >= len.count) {
        return;
    }
    const Magic   magic;
    const int32_t base = len.length - len.count;
    const int32_t p0   = base + t0;
    const int32_t p1   = base + min(t_of(tile * kWideRows + kWideRows - 1), len.count - 1);
    // this wave's positions, and this lane's query
    const int     r0   = tile * kWideRows + wave * 32;
    const int32_t w0   = base + t_of(r0);
    const int32_t w1   = base + min(t_of(r0 + 31), len.count - 1);
    const int     r    = r0 + c;
    const int     t    = t_of(r);
    const int     gq   = r - t * a.G;
    const bool    live = t < len.count;
    const int32_t p    = live ? base + t : -1;
    const int     head = h * a.G + gq;

    const KeyTiles kt  = key_tiles<kTileKeys>(a, p0, p1);
    const int      per = static_cast<int>(fastdiv(static_cast<uint32_t>(kt.n + a.nsplit - 1), a.fsplit));
    const int      end = min(kt.n, (split + 1) * per);
    const int      beg = split * per;

    // K: row tid / NB, block tid % NB; V: item tid % items of group tid / items
    const int    items  = PartT::items(NB);
    const int    words  = PartT::words(NB);
    const bool   mine   = tid < kTileKeys * NB;
    const int    krow   = tid / NB;
    const int    kblk   = tid % NB;
    const int    vgroup = tid / items;
    const int    vitem  = tid % items;
    const int    vkey   = 16 * (vgroup >> 1) + 4 * (vgroup & 1);
    const char * kb     = a.k + n * a.kn + h * a.kh;
    const char * vb     = a.v + n * a.vn + h * a.vh;
    const int    kstep  = static_cast<int>(a.kt);
    const int    vstep  = static_cast<int>(a.vt);
    const int    kat    = krow * kstep + kblk * UNIT;
    const int    vat0   = vkey * vstep + PartT::word_at(vitem, words);
    const int    vat1   = vkey * vstep + PartT::block_at(vitem, words);
    PartT        part;
    // (rows past the last that a query sees read as zero)
    auto fetch = [&](int i) {
        const int32_t j0 = key_tile(kt, i) * kTileKeys;
        const Rsrc    kr = rows_from(kb + j0 * a.kt, (p1 - j0) * a.kt + UNIT * NB);
        const Rsrc    vr = rows_from(vb + j0 * a.vt, (p1 - j0) * a.vt + UNIT * NB);
        if (mine) {
            part.load_k(kr, kat);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part.load_v(e, vr, vat0, vat1, (e < 4 ? e : e + 4) * vstep);
            }
        }
    };
    if (beg < end) {
        fetch(beg);
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
            const float * at = qr + 32 * (s / 2) + C::kFirst * (2 * (s % 2) + g);
            const f32x4   x0 = live ? ld4u(at) : splat4(0.0f);
            const f32x4   x1 = live ? ld4u(at + C::kSecond) : splat4(0.0f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[s][e] = (e < 4 ? x0[C::order(e)] : x1[C::order(e - 4)]) * a.scale;
                top     = fmaxf(top, fabsf(q[s][e]));
            }
        }
        const Pair both = swap32(top);
        top             = fmaxf(both.a, both.b);
        const int ex    = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 127) - 13;
        const float to  = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        qscale          = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
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

    // group `even` + g of column 32 u + c
    auto vat = [&](int u, int even) {
        const int turn = (32 * u >> PartT::kTurn & 3) ^ (PartT::kTurn == 4 ? c >> 4 : 0);
        return (32 * u + c) * kVStride + ((even + g) ^ turn) * 16;
    };
    f32x16 o[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
        o[u] = f32x16{};
    }
    float m = -INFINITY;
    float l = 0.0f;

    for (int i = beg; i < end; ++i) {
        const int32_t j0 = key_tile(kt, i) * kTileKeys;
        __syncthreads();  // the tile before is used up
        if (mine) {
            const bool  edge = j0 + kTileKeys - 1 > p0 || (a.window > 0 && j0 <= p1 - a.window && j0 + kTileKeys > a.sinks);
            const f16x2 dk   = as_f16x2(part.kd * 0x10001u);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x8 code = part.k_codes(magic, j);
                f16x2       hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 x = { code[2 * e], code[2 * e + 1] };
                    hi[e]         = x * dk;
                    lo[e]         = __builtin_elementwise_fma(x, dk, -hi[e]);
                }
                const int at = krow * KSTRIDE + kblk * 64 + 16 * j;
                *reinterpret_cast<f16x8 *>(kh + at) = join8(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<f16x8 *>(kl + at) = join8(lo[0], lo[1], lo[2], lo[3]);
            }
            f16x2 dv[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                uint32_t d = part.vd[e] | static_cast<uint32_t>(part.vd[e + 1]) << 16;
                if (edge) {  // rows that no query of the tile sees count for nothing, whatever they hold
                    const int32_t j = j0 + vkey + (e < 4 ? e : e + 4);
                    d &= (seen_by(a, p0, p1, j) ? 0x0000ffffu : 0u) | (seen_by(a, p0, p1, j + 1) ? 0xffff0000u : 0u);
                }
                dv[e / 2] = as_f16x2(d);
            }
            auto column = [&](auto uc) {
                constexpr int U = decltype(uc)::value;
                f16x2         hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f16x2 x = part.template v_codes<U>(magic, 2 * e, vitem, words);
                    hi[e]         = x * dv[e];
                    lo[e]         = __builtin_elementwise_fma(x, dv[e], -hi[e]);
                }
                const int dim = PartT::index(vitem, words, U);
                const int at  = dim * kVStride + (vgroup ^ (dim >> PartT::kTurn & 3)) * 16;
                *reinterpret_cast<f16x8 *>(vh + at) = join8(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<f16x8 *>(vl + at) = join8(lo[0], lo[1], lo[2], lo[3]);
            };
            for_each(std::make_integer_sequence<int, 4>{}, column);
        }
        if (i + 1 < end) {
            fetch(i + 1);
        }
        __syncthreads();
        if (j0 > w1) {
            continue;  // none of it is seen by this wave's queries
        }

        // scores of key 32 x + 8 (i / 4) + 4 g + i % 4
        // (ahead of the waves that are at their exponentials: 8192 positions 860
        // to 790 us)
        __builtin_amdgcn_s_setprio(1);
        f32x16 sc[2] = { f32x16{}, f32x16{} };
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            f16x8 hi[2], lo[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int at = (32 * x + c) * KSTRIDE + 32 * s + 16 * g;
                hi[x]        = *reinterpret_cast<const f16x8 *>(kh + at);
                if constexpr (TWO) {
                    lo[x] = *reinterpret_cast<const f16x8 *>(kl + at);
                }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                sc[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi[x], qh[s], sc[x], 0, 0, 0);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                sc[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi[x], ql[s], sc[x], 0, 0, 0);
            }
            if constexpr (TWO) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    sc[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo[x], qh[s], sc[x], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        const bool all = j0 + kTileKeys - 1 <= w0 && (a.window == 0 || j0 > w1 - a.window || j0 + kTileKeys <= a.sinks);
        if (!all) {
            int g4 = 4 * g;
            asm volatile("" : "+v"(g4));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[x][e] = sees(a, p, j0 + 32 * x + 8 * (e / 4) + e % 4 + g4) ? sc[x][e] : -INFINITY;
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                top = fmaxf(top, sc[x][e]);
            }
        }
        const Pair both = swap32(top);
        top             = fmaxf(m, fmaxf(both.a, both.b) * qscale);
        const float ref = top == -INFINITY ? 0.0f : top;
        if (__any(top > m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - ref);
            l *= alpha;
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                o[u] *= alpha;
            }
        }
        m = top;
        const float less = kPShift - ref;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                f16x2 hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][8 * s + 2 * e], qscale, less));
                    const float a1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][8 * s + 2 * e + 1], qscale, less));
                    l += a0 + a1;
                    split2(a0, a1, hi[e], lo[e]);
                }
                const f16x8 ph = join8(hi[0], hi[1], hi[2], hi[3]);
                const f16x8 pl = join8(lo[0], lo[1], lo[2], lo[3]);
                f16x8 vv[NB];
#pragma unroll
                for (int u = 0; u < NB; ++u) {
                    vv[u] = *reinterpret_cast<const f16x8 *>(vh + vat(u, 4 * x + 2 * s));
                }
#pragma unroll
                for (int u = 0; u < NB; ++u) {
                    o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[u], ph, o[u], 0, 0, 0);
                }
#pragma unroll
                for (int u = 0; u < NB; ++u) {
                    o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[u], pl, o[u], 0, 0, 0);
                }
                if constexpr (TWO) {
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        vv[u] = *reinterpret_cast<const f16x8 *>(vl + vat(u, 4 * x + 2 * s));
                    }
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[u], ph, o[u], 0, 0, 0);
                    }
                }
            }
        }
    }
    const Pair sum = swap32(l);
    l              = sum.a + sum.b;
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
    for (int u = 0; u < NB; ++u) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const f32x4 v                                            = { o[u][e] * by, o[u][e + 1] * by, o[u][e + 2] * by, o[u][e + 3] * by };
            *reinterpret_cast<f32x4u *>(out + 32 * u + 2 * e + 4 * g) = v;
        }
    }
}

// The parts of a row joined: a workgroup a row, whose threads take four values
// of every 1024/HD-th part each.
constexpr int kJoinThreads = 256;
constexpr int kMaxSplits   = 512;

// `parts` partial results of a row into out: ml(s) points to part s's m and l,
// o(s) to its values. Left alone where the row has fewer than two parts.
template <int HD, class ML, class O>
__device__ __forceinline__ void join_parts(int parts, int hd, const ML & ml, const O & o, float * out, bool sees_any) {
    constexpr int    GROUPS = kJoinThreads * 4 / HD;
    __shared__ float weight[kMaxSplits];
    __shared__ float lane_max[kJoinThreads / kWave], lane_sum[kJoinThreads / kWave];
    __shared__ f32x4 sums[kJoinThreads];
    const int        tid = threadIdx.x;
    float            top = -INFINITY;
    for (int s = tid; s < parts; s += kJoinThreads) {
        top = fmaxf(top, ml(s)[0]);
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
    for (int s = tid; s < parts; s += kJoinThreads) {
        const float w = ml(s)[1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml(s)[0] - ref);
        weight[s]     = w;
        l += w * ml(s)[1];
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
    const int dim   = tid % (HD / 4) * 4;
    const int group = tid / (HD / 4);
    f32x4     v     = splat4(0.0f);
    if (dim < hd) {
#pragma unroll 8
        for (int s = group; s < parts; s += GROUPS) {
            // weight 0: no key, and nothing that counts in o
            const float w = weight[s];
            const f32x4 x = *reinterpret_cast<const f32x4 *>(o(s) + dim);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] += w != 0.0f ? x[e] * w : 0.0f;
            }
        }
    }
    sums[tid] = v;
    __syncthreads();
    if (group == 0) {
        for (int k = 1; k < GROUPS; ++k) {
            v += sums[k * (HD / 4) + tid];
        }
        const float by = over(l, sees_any);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (dim + e < hd) {
                out[dim + e] = v[e] * by;
            }
        }
    }
}

// A row of a call: sequence, kv head, position and query head of it.
struct RowOf {
    int32_t n, h, t, gq;
};

__device__ __forceinline__ RowOf row_of(const AttnArgs & a, int64_t row) {
    const int64_t rt = row / a.G;
    const int64_t rh = rt / a.T;
    return RowOf{ static_cast<int32_t>(rh / a.KV), static_cast<int32_t>(rh % a.KV), static_cast<int32_t>(rt % a.T),
                  static_cast<int32_t>(row % a.G) };
}

__device__ __forceinline__ float * out_of(const AttnArgs & a, const RowOf & r) {
    return reinterpret_cast<float *>(a.y + r.n * a.yn + r.t * a.yt + (static_cast<int64_t>(r.h) * a.G + r.gq) * a.yh);
}

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join(const AttnArgs a, int64_t row0) {
    const int64_t row = row0 + blockIdx.x;
    const RowOf   r   = row_of(a, row);
    const SeqLens len = seq_lens(a, r.n);
    if (r.t >= len.count) {
        return;
    }
    join_parts<HD>(a.nsplit, a.hd, [&](int s) { return partial_ml(a, row, s); }, [&](int s) { return partial_o(a, row, s); },
                   out_of(a, r), len.length - len.count + r.t >= 0);
}

template <int HD> __global__ __launch_bounds__(kJoinThreads) void k_attn_join_few(const FewArgs f, int64_t row0) {
    const AttnArgs & a   = f.a;
    const RowOf      r   = row_of(a, row0 + blockIdx.x);
    const SeqLens    len = seq_lens(a, r.n);
    if (r.t >= len.count) {
        return;
    }
    const Line    line  = few_line(f, r.n, threadIdx.x % kWave);
    const int32_t total = line.total * f.groups;
    const int32_t units = few_units(f, r.n);
    const int32_t begin = line.before * f.groups + (r.h >> f.hgs) * units;
    const int32_t w0    = few_owner(f, total, begin);
    const int32_t w1    = few_owner(f, total, begin + units - 1);
    if (w0 == w1) {
        return;  // whole already
    }
    const int col = (r.h & ((1 << f.hgs) - 1)) * f.cols + r.t * a.G + r.gq;
    join_parts<HD>(w1 - w0 + 1, a.hd, [&](int s) { return few_ml(f, w0 + s, s == 0, col); },
                   [&](int s) { return few_o(f, w0 + s, s == 0, col); }, out_of(a, r), len.length - len.count + r.t >= 0);
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

// 64 rows at 32-bit offsets.
constexpr size_t kWideStride = size_t{ 1 } << 24;

struct AttnPlan {
    bool    few;
    bool    wide;
    int32_t hgs;
    int32_t wgs;
    int32_t per;
    bool    parts;
    int32_t window;
    int32_t sinks;
    int32_t tiles;
    int32_t nsplit;
};

constexpr int64_t kWhole = 4;

// Waves of a workgroup of k_attn_few: two where a row is long.
constexpr int few_waves(int64_t hd) {
    return hd <= 4 * kKvBlock ? 4 : 2;
}

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
        const int     waves  = few_waves(k_cache->ne[0]);
        const int64_t groups = (kv >> p.hgs) * q->ne[3];
        const int64_t chunks = ((keys << p.hgs) + kChunk - 1) / kChunk + (p.window > 0 ? 2 : 0);
        // up to kWhole chunks a wave a group is not split: that many take less than a second launch
        const int64_t deep  = chunks <= kWhole * waves ? (chunks + waves - 1) / waves : 1;
        const int64_t units = (chunks + waves * deep - 1) / (waves * deep) * groups;
        p.per               = static_cast<int32_t>(waves * deep);
        p.few               = units < INT32_MAX;
        p.wgs               = static_cast<int32_t>(units < kMaxSplits ? units : kMaxSplits);
        p.parts             = units > groups && p.wgs > 1;
        // where the caches' strides are not that kernel's: as many splits as its workspace holds
        const int64_t most = p.wgs * 2 * kCols / (q->ne[1] * q->ne[2] * q->ne[3]);
        p.nsplit           = p.parts ? plan_splits(p.tiles * kv * q->ne[3], most, 2048) : 1;
    }
    p.wide = !p.few && rows > 16 && k_cache->nb[2] < kWideStride && kv_blocks(kv_kind(k_cache->type)) && k_cache->ne[0] <= 4 * kKvBlock;
    if (p.wide) {
        p.tiles  = static_cast<int32_t>((rows + kWideRows - 1) / kWideRows);
        p.nsplit = plan_splits(p.tiles * kv * q->ne[3], (keys + 4 * kTileKeys - 1) / (4 * kTileKeys), 512);
    } else if (!p.few) {
        p.nsplit = plan_splits(p.tiles * kv * q->ne[3], (keys + 63) / 64, 2048);
    }
    return SHP_OK;
}

int64_t plan_floats(const AttnPlan & p, const shp_tensor & q) {
    const int64_t row = (q.ne[0] + 3) / 4 * 4 + 2;
    if (p.few) {
        return !p.parts ? 0 : static_cast<int64_t>(p.wgs) * 2 * kCols * row;
    }
    return p.nsplit == 1 ? 0 : q.ne[1] * q.ne[2] * q.ne[3] * p.nsplit * row;
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

template <int KIND, int NB> shp_status_t launch_wide_as(const AttnArgs & a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.KV) * static_cast<unsigned>(a.tiles) * static_cast<unsigned>(a.nsplit),
                    static_cast<unsigned>(a.N));
    hipLaunchKernelGGL((k_attn_wide<KIND, NB>), grid, dim3(kWideBlock), (wide_lds<KIND, NB>()), stream, a);
    return launch_status();
}

template <int KIND> shp_status_t launch_wide(const AttnArgs & a, hipStream_t stream) {
    switch ((a.hd + kKvBlock - 1) / kKvBlock) {
        case 1:
            return launch_wide_as<KIND, 1>(a, stream);
        case 2:
            return launch_wide_as<KIND, 2>(a, stream);
        case 3:
            return launch_wide_as<KIND, 3>(a, stream);
        default:
            return launch_wide_as<KIND, 4>(a, stream);
    }
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
    // a descriptor's last bytes are read by the dword
    return (run + (together ? static_cast<size_t>(c.ne[2] - 1) * run : size_t{ 0 })) % 4 == 0;
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

template <int KIND, int NB, int BYTES, bool RUNS, int WAVES> shp_status_t launch_few_as(FewArgs & f, hipStream_t stream) {
    using C             = Codes<KIND>;
    constexpr int TILES = (NB * C::kWords + 15) / 16 * C::kTiles;
    const int     rb    = f.nb * kv_unit_bytes(KIND);
    f.wave_lds          = 2 * kChunk * rb + NB * kChunk * 6;
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
    a.hd4    = (a.hd + 3) / 4 * 4;
    a.cap    = static_cast<int32_t>(k_cache->ne[2]);
    a.nsplit = p.nsplit;
    a.tiles  = p.tiles;
    a.fG     = make_fastdiv(static_cast<uint32_t>(a.G));
    a.fsplit = make_fastdiv(static_cast<uint32_t>(a.nsplit));
    a.fKV    = make_fastdiv(static_cast<uint32_t>(a.KV));
    const hipStream_t s     = as_stream(stream);
    const int         kind  = kv_kind(k_cache->type);
    int32_t           run   = 0;
    const int         piece = p.few ? few_piece(*k_cache, *v_cache, p.hgs, run) : 0;
    if (piece > 0) {
        return kind == kKvQ4 ? launch_few<kKvQ4>(a, p, piece, run, s) : launch_few<kKvQ8>(a, p, piece, run, s);
    }
    if (p.wide && v_cache->nb[2] >= kWideStride) {
        p.wide  = false;  // the splits stay as the workspace has them
        a.tiles = static_cast<int32_t>((static_cast<int64_t>(a.T) * a.G + 15) / 16);
    }
    if (p.wide) {
        st = kind == kKvQ4 ? launch_wide<kKvQ4>(a, s) : launch_wide<kKvQ8>(a, s);
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
