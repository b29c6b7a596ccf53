// What the attention's kernels share (k_attn.hip, k_attn_few.hip,
// k_attn_wide.hip): the arguments, which keys a query sees, partial results
// and their join, and matrix operands from a cache's bytes.
#pragma once

#include <climits>
#include <cmath>
#include <utility>

#include "shp_kv.hpp"

namespace shp {

constexpr int kChunk    = 32;   // cache rows of a chunk of k_attn_few
constexpr int kCols     = 16;   // queries of its workgroups
constexpr int kTileKeys = 64;   // of k_attn_wide
constexpr int kWideRows = 128;  // of its workgroups

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
    int32_t         apart;  // -1: queries stand one row apart; 0: all at the last row, so that all see every row
    int32_t         T;
    int32_t         G;  // query heads of a kv head
    int32_t         KV;
    int32_t         N;
    int32_t         hd;
    int32_t         hd4;  // hd up to a multiple of 4: a partial row's length
    int32_t         cap;
    int32_t         nsplit;
    int32_t         per;  // key tiles of a split of k_attn_wide; 0: k_attn_any, whose rows all have nsplit
    int32_t         tiles;  // of rows
    int32_t         half;   // k_attn_wide: the row tiles that come first, longest first; the others follow shortest first
    FastDiv         fG;
    FastDiv         fsplit;
    FastDiv         fKV;
    FastDiv         fper;
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

// A sequence's filled rows and new positions.
struct SeqLens {
    int32_t length;
    int32_t count;
};

// The row at which query 0 of a sequence stands, and query t for that.
__device__ __forceinline__ int32_t first_position(const AttnArgs & a, const SeqLens & len) {
    return len.length - 1 - ((len.count - 1) & a.apart);
}

__device__ __forceinline__ int32_t position(const AttnArgs & a, int32_t first, int32_t t) {
    return first + (t & a.apart);
}

// Splits of the keys of a row tile of k_attn_wide. One or none: its rows are
// written to y directly.
__device__ __forceinline__ int32_t wide_parts(const AttnArgs & a, const SeqLens & len, int32_t tile) {
    const int32_t t0 = static_cast<int32_t>(fastdiv(static_cast<uint32_t>(tile * kWideRows), a.fG));
    const int32_t t1 = static_cast<int32_t>(fastdiv(static_cast<uint32_t>(tile * kWideRows + kWideRows - 1), a.fG));
    const int32_t p  = first_position(a, len);
    const int32_t n  = key_tiles<kTileKeys>(a, position(a, p, t0), position(a, p, min(t1, len.count - 1))).n;
    return static_cast<int32_t>(fastdiv(static_cast<uint32_t>(n + a.per - 1), a.fper));
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

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kPShift  = 15.0f;  // P times 2^15, at most half of F16's range

// Weights are 2^(score + less), less the least of shift_for() of the scores so far:
// 2^shift for the largest score. From 2^23 on a score holds no more than whole
// numbers, and score + shift would be rounded up to a weight past F16's range; there
// the largest weight is 1 (the others are 1 or next to nothing). What less was
// rounded to is what all weights of a row have in common; it stands for -max in
// a partial result.
__device__ __forceinline__ float shift_for(float top, float shift) {
    return (fabsf(top) < 0x1p23f ? shift : 0.0f) - top;
}

// What weights under `less` become under `now`, at most that; nothing seen: infinity.
__device__ __forceinline__ float shift_change(float less, float now) {
    return now < less ? __builtin_amdgcn_exp2f(now - less) : 1.0f;
}

__device__ __forceinline__ float shift_added(float less) {
    return less == INFINITY ? 0.0f : less;
}

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

// 2^e, e in [-126, 127].
__device__ __forceinline__ float pow2(int e) {
    return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// The exponent of a magnitude, within what pow2() can undo.
__device__ __forceinline__ int exponent_of(float top) {
    return min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 127);
}

// A block's code * d, |code| <= 128, is within F16's range for d up to 256. Beside
// a larger one its values are v = 2^8 hi + lo: hi is 2^-8 v rounded, 2^15 at most,
// and lo the rest, exact: v has 18 bits and whole multiples of 2^-24, of which hi
// takes 11, or those down to 2^-16.
constexpr uint32_t kBigD    = 0x5c00;
constexpr uint32_t kInfD    = 0x7c00;
constexpr float    kLargeBy = 256.0f;

__device__ __forceinline__ void large_pieces(f16x2 code, f16x2 d, f16x2 & hi, f16x2 & lo) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float v = static_cast<float>(code[i]) * static_cast<float>(d[i]);
        hi[i]         = static_cast<_Float16>(v * (1.0f / kLargeBy));
        lo[i]         = static_cast<_Float16>(v - static_cast<float>(hi[i]) * kLargeBy);
    }
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
//   v_place  where value `dim` of O^T is found
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

    // Where value `dim` stands among a wave's results [tile][element][lane]: in
    // tile 16-word slot * kTiles + u, row w % 16 = 4 g + e, lanes 16 g and on.
    __device__ static int v_place(int dim) {
        const int w = 4 * (dim >> 5) + ((dim & 15) >> 2);
        const int u = 2 * (dim & 3) + ((dim >> 4) & 1);
        return (((w >> 4) * kTiles + u) * 4 + (w & 3)) * kWave + 16 * ((w >> 2) & 3);
    }
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

    __device__ static int v_place(int dim) {
        const int w = dim >> 2;
        return (((w >> 4) * kTiles + (dim & 3)) * 4 + (w & 3)) * kWave + 16 * ((w >> 2) & 3);
    }
};

template <class Go, int... U> __device__ __forceinline__ void for_each(std::integer_sequence<int, U...>, const Go & go) {
    (go(std::integral_constant<int, U>{}), ...);
}

// Cache rows are read through a buffer descriptor that ends with them, so that
// what is behind reads as zero without a test in the kernel.
typedef __amdgpu_buffer_rsrc_t Rsrc;

__device__ __forceinline__ Rsrc rows_from(const char * at, int64_t bytes) {
    constexpr int kRaw32 = 0x00027000;  // 32-bit data, no swizzle
    const int64_t most   = int64_t{ 1 } << 30;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(at), 0, static_cast<int>(bytes < most ? bytes : most), kRaw32);
}

// The parts of a row joined: a workgroup a row, whose threads take four values
// of every 1024/HD-th part each.
constexpr int kJoinThreads = 256;
constexpr int kMaxSplits   = 768;   // splits of a row tile's keys
constexpr int kMaxParts    = 1024;  // of one row: those splits, or the workgroups that share a line of units
static_assert(kMaxSplits <= kMaxParts);

// `parts` partial results of a row, kMaxParts at most, into out: ml(s) points to part
// s's m and l, o(s) to its values. Left alone where the row has fewer than two parts.
template <int HD, class ML, class O>
__device__ __forceinline__ void join_parts(int parts, int hd, const ML & ml, const O & o, float * out, bool sees_any) {
    constexpr int    GROUPS = kJoinThreads * 4 / HD;
    __shared__ float weight[kMaxParts];
    __shared__ float lane_max[kJoinThreads / kWave], lane_sum[kJoinThreads / kWave];
    __shared__ f32x4 sums[kJoinThreads];
    const int        tid   = threadIdx.x;
    const int        dim   = tid % (HD / 4) * 4;
    const int        group = tid / (HD / 4);
    // this thread's first values on their way while the weights are formed (one
    // stream of 8191 rows, 256 parts of each row: 1.4 us less than two ahead)
    constexpr int kAhead = 8;
    f32x4         first[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int s = group + k * GROUPS;
        first[k]    = dim < hd && s < parts ? *reinterpret_cast<const f32x4 *>(o(s) + dim) : splat4(0.0f);
    }
    float top = -INFINITY;
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
    f32x4 v   = splat4(0.0f);
    auto  add = [&](int s, const f32x4 & x) {
        const float w = weight[s];  // 0: no key, and nothing that counts in o
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += w != 0.0f ? x[e] * w : 0.0f;
        }
    };
    if (dim < hd) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (group + k * GROUPS < parts) {
                add(group + k * GROUPS, first[k]);
            }
        }
#pragma unroll 8
        for (int s = group + kAhead * GROUPS; s < parts; s += GROUPS) {
            add(s, *reinterpret_cast<const f32x4 *>(o(s) + dim));
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

// ---------------------------------------------------------------------------
// Few queries: what k_attn_few.hip and k_attn_pages.hip share.
// ---------------------------------------------------------------------------

struct FewArgs {
    AttnArgs a;
    int32_t  hgs;      // log2 of HG
    int32_t  shift;    // log2 of the keys of a chunk
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
// to 8192 rows, MI355X: 113 us, 169 with an equal number of workgroups for each
// sequence). A stretch that ends inside a group leaves a partial result; a
// workgroup has two at most, of the group that it begins in and did not begin
// (0), and of the one that it began and did not end (1).
__device__ __forceinline__ float * few_o(const FewArgs & f, int wg, int which, int col) {
    return f.a.work + (static_cast<int64_t>(wg * 2 + which) * kCols + col) * f.a.hd4;
}

__device__ __forceinline__ float * few_ml(const FewArgs & f, int wg, int which, int col) {
    return f.a.work + static_cast<int64_t>(f.wgs) * 2 * kCols * f.a.hd4 + ((wg * 2 + which) * kCols + col) * 2;
}

// The first and last workgroup of a head group.
__device__ __forceinline__ int32_t * few_span(const FewArgs & f, int64_t group) {
    return reinterpret_cast<int32_t *>(few_ml(f, f.wgs, 0, 0)) + 2 * group;
}

// A sequence's key chunks; `len` as seq_lens gives it.
__device__ __forceinline__ KeyTiles few_tiles(const FewArgs & f, const SeqLens & len) {
    const AttnArgs & a     = f.a;
    const int        shift = f.shift;
    const int32_t    base  = first_position(a, len);
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

// The sequence that a unit of the line falls in.
struct Place {
    int32_t n;
    int32_t units;   // of one head group of it
    int32_t before;  // of all head groups of the sequences before it
};

// The line's units of all head groups, and where workgroup wg's stretch begins
// in it, for a whole wave: 64 sequences at a time, a sum over lanes.
struct Line {
    int32_t total;
    int32_t begin;
    int32_t end;
    Place   at;  // of begin, if the stretch is not empty
};

__device__ __forceinline__ int32_t few_start(const FewArgs & f, int32_t total, int32_t wg);

__device__ __forceinline__ Line few_line(const FewArgs & f, int wg, int lane) {
    Line s{};
    if (f.a.N == 1) {
        const int units = few_units(f, 0);
        s.total         = units * f.groups;
        s.at            = Place{ 0, units, 0 };
    } else {
        auto units_of = [&](int first) { return first + lane < f.a.N ? few_units(f, first + lane) : 0; };
        int  units    = units_of(0);
        int  sum      = sum_up_to(units);
        s.total       = __builtin_amdgcn_readlane(sum, kWave - 1);
        for (int first = kWave; first < f.a.N; first += kWave) {
            s.total += __builtin_amdgcn_readlane(sum_up_to(units_of(first)), kWave - 1);
        }
        s.total *= f.groups;
        const int32_t unit   = few_start(f, s.total, wg);
        int32_t       before = 0;
        for (int first = 0; first < f.a.N; first += kWave) {
            if (first > 0) {
                units = units_of(first);
                sum   = sum_up_to(units);
            }
            const uint64_t past = __ballot(before + sum * f.groups > unit);
            if (past != 0) {
                const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
                const int k = __builtin_amdgcn_readlane(units, l);
                s.at        = Place{ first + l, k, before + (__builtin_amdgcn_readlane(sum, l) - k) * f.groups };
                break;
            }
            before += __builtin_amdgcn_readlane(sum, kWave - 1) * f.groups;
        }
    }
    s.begin = few_start(f, s.total, wg);
    s.end   = few_start(f, s.total, wg + 1);
    return s;
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

// One row's parts, by a workgroup.
template <int HD> __device__ __forceinline__ void join_few(const FewArgs & f, int64_t row) {
    const AttnArgs & a   = f.a;
    const RowOf      r   = row_of(a, row);
    const SeqLens    len = seq_lens(a, r.n);
    if (r.t >= len.count) {
        return;
    }
    const int32_t * span = few_span(f, static_cast<int64_t>(r.n) * f.groups + (r.h >> f.hgs));
    const int32_t   w0   = span[0];
    const int32_t   w1   = span[1];
    if (w0 == w1) {
        return;  // whole already
    }
    const int col = (r.h & ((1 << f.hgs) - 1)) * f.cols + r.t * a.G + r.gq;
    join_parts<HD>(w1 - w0 + 1, a.hd, [&](int s) { return few_ml(f, w0 + s, s == 0, col); },
                   [&](int s) { return few_o(f, w0 + s, s == 0, col); }, out_of(a, r), position(a, first_position(a, len), r.t) >= 0);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

struct AttnPlan {
    bool    few;
    bool    cross;  // by k_cross_few
    bool    wide;
    int32_t hgs;
    int32_t groups;  // of heads, all sequences'
    int32_t wgs;
    int32_t per;
    int32_t waves;  // of a workgroup of k_cross_few
    bool    parts;
    int32_t window;
    int32_t sinks;
    int32_t nsplit;
    int32_t span;  // key tiles of a split of k_attn_wide
};

// Waves of a workgroup of k_attn_few: two where a row is long; those that each
// of a CU's four SIMDs holds, by the registers they take; and the workgroups
// that the chip's 256 CUs hold.
constexpr int few_waves(int64_t hd) {
    return hd <= 4 * kKvBlock ? 4 : 2;
}

constexpr int few_occupancy(int kind, int64_t hd) {
    return hd > 4 * kKvBlock ? 1 : kind == kKvQ4 || hd <= 2 * kKvBlock ? 3 : 2;
}

constexpr int few_resident(int kind, int64_t hd) {
    return 256 * 4 * few_occupancy(kind, hd) / few_waves(hd);
}

// (one head group may have all of them)
static_assert(few_resident(kKvQ4, 2 * kKvBlock) <= kMaxParts && few_resident(kKvQ4, 4 * kKvBlock) <= kMaxParts &&
              few_resident(kKvQ4, 8 * kKvBlock) <= kMaxParts);

// k_attn_few.hip: block caches and at most 16 queries of a kv head. The piece
// size in which it can read both caches, or 0; and its launches, join included.
int          few_piece(const shp_tensor & k, const shp_tensor & v, int hgs, int32_t & run);
shp_status_t launch_attn_few(int kind, const AttnArgs & a, const AttnPlan & p, int piece, int32_t run, hipStream_t stream);

// k_attn.hip: splits of a prompt's keys, the workspace of a plan, what all calls check
// and pass on, and the launch that joins the splits of k_attn_wide and k_attn_pages_wide.
void         plan_spans(int64_t rows, int64_t T, int64_t cap, int64_t keys, int64_t pairs, int64_t chip, bool causal,
                        AttnPlan & p);
int64_t      plan_floats(const AttnPlan & p, const shp_tensor & q);
shp_status_t attn_args(const shp_tensor * q, const shp_tensor * length, const shp_tensor * count, float scale, const AttnPlan & p,
                       const shp_tensor * const * read, int n_read, const shp_tensor * work, const shp_tensor * y, AttnArgs & a);
void         wide_args(int32_t per, int32_t rows, int64_t chip, AttnArgs & a);
shp_status_t launch_join(const AttnArgs & a, hipStream_t stream);

// k_cross.hip: plain states of any length, and at most 16 queries of a kv head. The
// head lengths that it is built for, its plan for `rows` rows, whether it reads c.
constexpr int64_t cross_few_dims(int64_t hd) {
    return hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
}

void         plan_cross_few(int kind, int64_t hd, int64_t rows, int64_t groups, AttnPlan & p);
bool         cross_few_takes(const shp_tensor & c);
shp_status_t launch_cross_few(int kind, const AttnArgs & a, const AttnPlan & p, hipStream_t stream);

// k_attn_wide.hip.
shp_status_t launch_attn_wide(int kind, const AttnArgs & a, hipStream_t stream);

}  // namespace shp
