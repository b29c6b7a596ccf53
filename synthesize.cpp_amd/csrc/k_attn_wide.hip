// shp_attn_kv for many queries (prompts).
#include "shp_attn.hpp"

namespace shp {
namespace {

// ---------------------------------------------------------------------------
// Many queries (prompts): a workgroup takes 128 rows, 32 a wave, and 64 keys at
// a time, whose K and V it brings into LDS once, as matrix operands: K by row,
// V by column with the keys in the order in which the scores stand in
// registers. A block's code * d is exact as two F16 pieces, and an F32 value is two
// as well; so are q and P, and each product is hi hi + hi lo + lo hi (an F16 cache
// has no second piece). A BF16 cache is BF16 operands as it is, of any size, and q
// and P are three BF16 pieces, all 24 bits of them. Matrix instructions 32x32x16:
// S^T = K Q^T has a query in each lane, O^T = V^T P^T too.
// Bound by the matrix units: 8192 positions of 16 heads of 128 values over 8 kv
// heads take 700 to 745 us (Q4_0, MI355X), three products at 1.11 to 1.18 PFLOP/s,
// where a large F16 product reaches 1.12, at the clock that such work leaves the
// chip. (K's codes could do with one piece and d by key, as in k_attn_few: two
// products and a half in all.) A prompt that does not fill the chip is bound by the longest row: 1021
// positions 40 us, 10 of them the second launch that joins its splits. 4096
// positions: F16 180 us, BF16 226, Q4_0 250, Q8_0 282, F32 380 to 400, whose
// registers spill. 128 rows and 64 keys are what the registers (O^T, q, a tile under
// way: 256) and two workgroups' LDS hold; heads of more than 128 values have one
// workgroup a CU, with 512 (2048 positions of 8 heads of 256 over 4, Q4_0: 118 us).
// ---------------------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWideBlock = 256;
constexpr int kWaves     = kWideBlock / kWave;
constexpr int kVStride   = kTileKeys * 2 + 16;  // bytes of a column of V in LDS, off the banks' period

// A thread's part of a tile on its way to LDS: 32 values of a row of K, and of
// V the four values u = 0..3 of each of eight keys, those that lie next to each
// other in an operand: 16 s + 4 h + 0..3 and 8 more, group 2 s + h. In column
// `dim` of V the groups stand in the order group ^ (dim >> kTurn & 3): sixteen
// lanes that write a group of sixteen columns then meet every bank once (four
// times four without it: a third of the LDS unit's time).
// F32's pieces are of the values times a power of two (see by_size). A block's are
// of the values themselves, but in a tile where a d is above kBigD, and values may
// be out of F16's range: there the first piece is 2^-8 of its value, and the second
// what 2^8 times that leaves, which is exact as well (18 bits are 11 and 7, whatever
// the sizes: a block of small values beside one of large is as exact as alone).
//   load_k, load_v  from the cache, through descriptors of the tile
//   keep_k, keep_v  or zeros in place of K's row, of V's of key e
//   top_k, top_v    bits that bound the magnitudes, kInf and more where one is
//                   infinite or NaN
//   k_pieces        operand j of the row's four, times `by` (F32), of a large tile
//   v_column        value U of the eight keys, likewise
template <int KIND> struct Part;

// Codes and d.
template <int KIND, int WORDS> struct BlockPart {
    static constexpr bool kTwo = true;
    uint32_t              k[WORDS];
    uint32_t              v[8];
    // (dwords: halves are put into pairs, for which a wave waits as soon as it has
    // asked for them; 8192 positions 780 to 736 us)
    uint32_t              kd;
    uint32_t              vd[8];

    // the block `at` bytes into the tile
    __device__ void load_k(const Rsrc & r, int at) {
        kd = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            k[i] = __builtin_amdgcn_raw_buffer_load_b32(r, at + 2 + 4 * i, 0, 0);
        }
    }

    // key e's word `at` bytes into its row, which is `row` bytes into the tile, and its d at `block`
    __device__ void load_v(int e, const Rsrc & r, int at, int block, int row) {
        v[e]  = __builtin_amdgcn_raw_buffer_load_b32(r, at, row, 0);
        vd[e] = __builtin_amdgcn_raw_buffer_load_b16(r, block, row, 0);
    }

    __device__ void keep_k(bool yes) { kd = yes ? kd : 0; }

    __device__ void keep_v(int e, bool yes) { vd[e] = yes ? vd[e] : 0; }

    static constexpr uint32_t kInf = kInfD;

    __device__ uint32_t top_k() const { return kd & 0x7fffu; }

    __device__ uint32_t top_v(int e) const { return vd[e] & 0x7fffu; }

    __device__ static float magnitude(uint32_t bits) { return f16_bits_to_f32(bits); }

    template <bool LARGE> __device__ static void exact(f16x2 code, f16x2 d, f16x2 & hi, f16x2 & lo) {
        if constexpr (LARGE) {
            large_pieces(code, d, hi, lo);
        } else {
            hi = code * d;
            lo = __builtin_elementwise_fma(code, d, -hi);
        }
    }

    template <bool LARGE> __device__ void k_pieces(const Magic & m, float, int j, f16x8 & hi, f16x8 & lo) const {
        constexpr int STEP = WORDS / 4;
        uint32_t      w[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
            w[i] = k[STEP * j + i];
        }
        const f16x8 code = Codes<KIND>::k_codes(m, w);
        f16x2       h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            exact<LARGE>(f16x2{ code[2 * e], code[2 * e + 1] }, as_f16x2(kd * 0x10001u), h[e], l[e]);
        }
        hi = join8(h[0], h[1], h[2], h[3]);
        lo = join8(l[0], l[1], l[2], l[3]);
    }

    template <int U, bool LARGE> __device__ void v_pieces(const Magic & m, int shift, f16x8 & hi, f16x8 & lo) const {
        f16x2 h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            exact<LARGE>(Codes<KIND>::template v_codes<U>(m, v[2 * e] >> shift, v[2 * e + 1] >> shift),
                         as_f16x2(vd[2 * e] | vd[2 * e + 1] << 16), h[e], l[e]);
        }
        hi = join8(h[0], h[1], h[2], h[3]);
        lo = join8(l[0], l[1], l[2], l[3]);
    }
};

// V's items are a dword's four low or four high nibbles: item `words` + w.
template <> struct Part<kKvQ4> : BlockPart<kKvQ4, 4> {
    static constexpr int kTurn = 5;

    __device__ static int words(int nb) { return 4 * nb; }

    __device__ static int block_at(int item, int words) { return ((item % words) >> 2) * 18; }

    __device__ static int word_at(int item, int words) { return block_at(item, words) + 2 + 4 * (item & 3); }

    __device__ static int index(int item, int words, int u) {
        const int w = item % words;
        return 32 * (w >> 2) + 4 * (w & 3) + u + (item >= words ? 16 : 0);
    }

    template <int U, bool LARGE>
    __device__ void v_column(const Magic & m, float, int item, int words, f16x8 & hi, f16x8 & lo) const {
        v_pieces<2 * U, LARGE>(m, item >= words ? 4 : 0, hi, lo);
    }
};

template <> struct Part<kKvQ8> : BlockPart<kKvQ8, 8> {
    static constexpr int kTurn = 4;

    __device__ static int words(int nb) { return 8 * nb; }

    __device__ static int block_at(int item, int) { return (item >> 3) * 34; }

    __device__ static int word_at(int item, int) { return block_at(item, 0) + 2 + 4 * (item & 7); }

    __device__ static int index(int item, int, int u) { return 4 * item + u; }

    template <int U, bool LARGE> __device__ void v_column(const Magic & m, float, int, int, f16x8 & hi, f16x8 & lo) const {
        v_pieces<U, LARGE>(m, 0, hi, lo);
    }
};

// Plain values, four next to each other a key of V.
template <int KIND> struct PlainPart {
    static constexpr bool  kTwo    = KIND == kKvF32;
    static constexpr int   kTurn   = 4;
    static constexpr int   kSize   = kv_unit_bytes(KIND);
    static constexpr int   kFour   = kSize;  // dwords of four values
    uint32_t               k[8 * kFour];
    uint32_t               v[8][kFour];

    __device__ void load_k(const Rsrc & r, int at) {
#pragma unroll
        for (int i = 0; i < 2 * kFour; ++i) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * i, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                k[4 * i + e] = x[e];
            }
        }
    }

    // What a row has only `ks` values of K's 32 and `vs` of V's four (what was
    // read behind them is the next row's, or zero).
    __device__ void cut(int ks, int vs) {
#pragma unroll
        for (int i = 0; i < 8 * kFour; ++i) {
            k[i] = within(k[i], i, ks);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int i = 0; i < kFour; ++i) {
                v[e][i] = within(v[e][i], i, vs);
            }
        }
    }

    __device__ static uint32_t within(uint32_t w, int i, int values) {
        if constexpr (kSize == 4) {
            return i < values ? w : 0;
        } else {
            return 2 * i + 1 < values ? w : 2 * i < values ? w & 0xffffu : 0;
        }
    }

    __device__ void load_v(int e, const Rsrc & r, int at, int, int row) {
        if constexpr (kFour == 4) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, at, row, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[e][i] = x[i];
            }
        } else {
            const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, at, row, 0);
            v[e][0]      = x[0];
            v[e][1]      = x[1];
        }
    }

    __device__ void keep_k(bool yes) {
#pragma unroll
        for (int i = 0; i < 8 * kFour; ++i) {
            k[i] = yes ? k[i] : 0;
        }
    }

    __device__ void keep_v(int e, bool yes) {
#pragma unroll
        for (int i = 0; i < kFour; ++i) {
            v[e][i] = yes ? v[e][i] : 0;
        }
    }

    // Magnitudes as their bits, in whose order a NaN is the largest.
    static constexpr uint32_t kInf = KIND == kKvF32 ? 0x7f800000u : KIND == kKvF16 ? 0x7c00u : 0x7f80u;

    __device__ static uint32_t top_of(uint32_t m, uint32_t w) {
        if constexpr (kSize == 4) {
            return max(m, w & 0x7fffffffu);
        } else {
            return max(m, max(w & 0x7fffu, w >> 16 & 0x7fffu));
        }
    }

    __device__ uint32_t top_k() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8 * kFour; ++i) {
            m = top_of(m, k[i]);
        }
        return m;
    }

    __device__ uint32_t top_v(int e) const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kFour; ++i) {
            m = top_of(m, v[e][i]);
        }
        return m;
    }

    __device__ static float magnitude(uint32_t bits) {
        return KIND == kKvF32 ? __uint_as_float(bits) : KIND == kKvF16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
    }

    __device__ static int words(int nb) { return 8 * nb; }

    __device__ static int block_at(int, int) { return 0; }

    __device__ static int word_at(int item, int) { return item * 4 * kSize; }

    __device__ static int index(int item, int, int u) { return 4 * item + u; }

    template <bool> __device__ void k_pieces(const Magic &, float by, int j, f16x8 & hi, f16x8 & lo) const {
        f16x2 h[4], l[4] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (kTwo) {
                split2(__uint_as_float(k[8 * j + 2 * e]) * by, __uint_as_float(k[8 * j + 2 * e + 1]) * by, h[e], l[e]);
            } else {
                h[e] = as_f16x2(k[4 * j + e]);  // (BF16's bits, of two values)
            }
        }
        hi = join8(h[0], h[1], h[2], h[3]);
        lo = join8(l[0], l[1], l[2], l[3]);
    }

    template <int U, bool> __device__ void v_column(const Magic &, float by, int, int, f16x8 & hi, f16x8 & lo) const {
        f16x2 h[4], l[4] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (kTwo) {
                split2(__uint_as_float(v[2 * e][U]) * by, __uint_as_float(v[2 * e + 1][U]) * by, h[e], l[e]);
            } else {
                constexpr uint32_t kSel = U % 2 == 0 ? 0x05040100u : 0x07060302u;
                h[e]                    = as_f16x2(__builtin_amdgcn_perm(v[2 * e + 1][U / 2], v[2 * e][U / 2], kSel));
            }
        }
        hi = join8(h[0], h[1], h[2], h[3]);
        lo = join8(l[0], l[1], l[2], l[3]);
    }
};

template <> struct Part<kKvF16> : PlainPart<kKvF16> {};

template <> struct Part<kKvBF16> : PlainPart<kKvBF16> {};

template <> struct Part<kKvF32> : PlainPart<kKvF32> {};

// Bytes of 32 values of a row, and the order of K's in an operand of eight:
// kFirst g + order(0..3), then kSecond more.
template <int KIND> struct KOrder {
    static constexpr int kFirst = 8, kSecond = 4;

    __device__ static constexpr int order(int e) { return e; }
};

template <> struct KOrder<kKvQ4> : Codes<kKvQ4> {};

// F32, whose values may be of any size. One power of two for the K and one for the
// V of a tile cost a value up to 2^-39 of the tile's largest, so they are used
// where no row is much smaller than that: a tile is even where every 32 values of
// K and four of V that are not all zero have one of 2^-14 of the tile's largest and
// more. A tile that is not is taken in several passes, each over rows of about one
// size as if the others were hidden: those down to 2^-(2 kAlike) of the largest that
// are left, or, where none is that in K and V, 2^kAlike times smaller and larger
// than the first. So a value is off by 2^-25 of its own row's largest at most,
// a half step, whatever the others are; a row that a query does not see has no
// other part in its result.
// V's sizes differ from pass to pass: weights are held times 2^(E - X + 15), 2^E
// being that of the pass and 2^X, which is the query's own, what the largest so
// far of weight times 2^E needs. So P loses 2^-39 of the largest weight where one
// size is all that the query sees, and else 2^-39 of the largest of weight times
// 2^E, whose row may be 2^14 smaller than 2^E.
// (4096 positions of 16 heads over 8, MI355X: 377 us, 365 with one power of two in
// any case. A channel thirty times the others leaves all tiles even, one of V a
// thousand times them takes 1.25 times as long, rows from 1e-8 to 1e8 5.7 times.)
constexpr bool by_size(int kind) {
    return kind == kKvF32;
}

constexpr float kEven  = 0x1p-13f;  // of the largest that a wave holds, and waves within a factor of 2
constexpr int   kAlike = 6;
constexpr int   kVTop  = 13;       // the largest value of V comes to 2^13 and more
constexpr int   kMinX  = -99;      // of values of 2^-100 and less

// Three pieces of q and P. The third of q is in LDS: 2 NB operands a lane.
constexpr bool in_three(int kind) {
    return kind == kKvBF16;
}

template <int KIND, int NB> constexpr int wide_lds() {
    constexpr int HD = NB * kKvBlock;
    return (kTileKeys * (HD * 2 + 16) + HD * kVStride) * (Part<KIND>::kTwo ? 2 : 1) + 24 * kWaves +
           (by_size(KIND) ? 2 * 4 * kTileKeys : 0) + (in_three(KIND) ? 2 * NB * kWideBlock * 16 : 0);
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

template <int KIND> __device__ __forceinline__ f32x16 product(const f16x8 & a, const f16x8 & b, const f32x16 & c) {
    if constexpr (in_three(KIND)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
}

template <int KIND, int NB> __global__ __launch_bounds__(kWideBlock, NB <= 4 ? 2 : 1) void k_attn_wide(const AttnArgs a) {
    using PartT             = Part<KIND>;
    using C                 = KOrder<KIND>;
    constexpr int  HD       = NB * kKvBlock;
    constexpr int  UNIT     = kv_unit_bytes(KIND) * (kv_blocks(KIND) ? 1 : kKvBlock);
    constexpr int  KSTRIDE  = HD * 2 + 16;
    constexpr bool TWO      = PartT::kTwo;
    constexpr bool SIZES    = by_size(KIND);
    constexpr bool THREE    = in_three(KIND);
    extern __shared__ char lds[];
    char * const   kh   = lds;
    char * const   kl   = kh + kTileKeys * KSTRIDE;  // (of two pieces)
    char * const   vh   = kl + (TWO ? kTileKeys * KSTRIDE : 0);
    char * const   vl   = vh + HD * kVStride;
    float * const  tops = reinterpret_cast<float *>(vl + (TWO ? HD * kVStride : 0));  // SIZES: each wave's largest of K, of V, and whether some are far below; blocks: whether a d is large
    uint64_t *     bads = reinterpret_cast<uint64_t *>(tops + 4 * kWaves);            // a wave's keys that are not finite in K or V
    uint32_t *     rmax = reinterpret_cast<uint32_t *>(bads + kWaves);                // SIZES: the largest of each row of K, then V
    f16x8 *        q3   = reinterpret_cast<f16x8 *>(bads + kWaves) + threadIdx.x;     // THREE: the third pieces of a lane's query

    const int     tid   = threadIdx.x;
    const int     wave  = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int     lane  = tid % kWave;
    const int     c     = lane & 31;
    const int     g     = lane >> 5;
    // a kv head's workgroups share an XCD where there are eight heads; the longest rows first
    const int     part0 = static_cast<int>(fastdiv(blockIdx.x, a.fKV));
    const int     h     = static_cast<int>(blockIdx.x) - part0 * a.KV;
    const int     back  = static_cast<int>(fastdiv(static_cast<uint32_t>(part0), a.fsplit));
    const int     tile  = back < a.half ? a.tiles - 1 - back : back - a.half;
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
    const int32_t w1   = t_of(r0) < len.count ? base + min(t_of(r0 + 31), len.count - 1) : -1;
    const int     r    = r0 + c;
    const int     t    = t_of(r);
    const int     gq   = r - t * a.G;
    const bool    live = t < len.count;
    const int32_t p    = live ? base + t : -1;
    const int     head = h * a.G + gq;

    const KeyTiles kt  = key_tiles<kTileKeys>(a, p0, p1);
    const int      beg = split * a.per;
    const int      end = min(kt.n, beg + a.per);
    if (split > 0 && beg >= kt.n) {
        return;
    }
    // where the results go: y, or a split's rows (in a scalar register: held in
    // a vector one through the loop it costs 6%)
    const int      dest = __builtin_amdgcn_readfirstlane(kt.n <= a.per ? -1 : split);

    // Part z of a thread is number id = tid + 256 z. K: row id / NB, block id % NB;
    // V: item id % items of group id / items, keys key_v and on.
    // Indexes that begin with tid_again() are not formed ahead of the loop and held
    // through it: those of what only some tiles need, and, with tid_each(), all of
    // them where registers are short (F32: 16 sequences of 4096 rows take 166 us, 211
    // without; heads of 256 values: F16 91, 98; but F16 at 128: 199, 191).
    auto tid_again = [] {
        int id = threadIdx.x;
        asm volatile("" : "+v"(id));
        return id;
    };
    auto tid_each = [&] {
        if constexpr (SIZES || NB > 4) {
            return tid_again();
        } else {
            return tid;
        }
    };
    auto row_k = [](int id, int z) { return (id + kWideBlock * z) / NB; };
    auto key_v = [](int id, int z) {
        const int group = (id + kWideBlock * z) / (8 * NB);
        return 16 * (group >> 1) + 4 * (group & 1);
    };
    constexpr int PARTS = (kTileKeys * NB + kWideBlock - 1) / kWideBlock;
    const int     items = 8 * NB;
    const int     words = PartT::words(NB);
    const int     kstep = static_cast<int>(a.kt);
    const int     vstep = static_cast<int>(a.vt);
    bool          mine[PARTS];
#pragma unroll
    for (int z = 0; z < PARTS; ++z) {
        mine[z] = tid + kWideBlock * z < kTileKeys * NB;
    }
    const char * kb = a.k + n * a.kn + h * a.kh;
    const char * vb = a.v + n * a.vn + h * a.vh;
    const int    rb = static_cast<int>(kv_row_bytes(KIND, a.hd));
    PartT        part[PARTS];
    // (rows past the last that a query sees read as zero)
    auto fetch = [&](int i) {
        const int32_t j0 = key_tile(kt, i) * kTileKeys;
        const Rsrc    kr = rows_from(kb + j0 * a.kt, (p1 - j0) * a.kt + rb);
        const Rsrc    vr = rows_from(vb + j0 * a.vt, (p1 - j0) * a.vt + rb);
        const int     id = tid_each();
#pragma unroll
        for (int z = 0; z < PARTS; ++z) {
            if (mine[z]) {
                const int item = (id + kWideBlock * z) % items;
                const int key  = key_v(id, z) * vstep;
                part[z].load_k(kr, row_k(id, z) * kstep + (id + kWideBlock * z) % NB * UNIT);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    part[z].load_v(e, vr, key + PartT::word_at(item, words), key + PartT::block_at(item, words), (e < 4 ? e : e + 4) * vstep);
                }
            }
        }
    };
    if (beg < end) {
        fetch(beg);
    }

    auto values = [&](const float * row, int at, bool has) {
        f32x4 x = splat4(0.0f);
        if (has && (kv_blocks(KIND) || at + 4 <= a.hd)) {
            x = ld4u(row + at);
        } else if (has) {
            for (int e = 0; at + e < a.hd; ++e) {
                x[e] = row[at + e];
            }
        }
        return x;
    };
    // the query's operands; the largest of its values scaled to [2^13, 2^14)
    f16x8 qh[2 * NB], ql[2 * NB];
    int   qexp;
    {
        const float * qr = reinterpret_cast<const float *>(a.q + n * a.qn + t * a.qt + head * a.qh);
        float         q[2 * NB][8];
        float         top = 0.0f;
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            const int     at = 32 * (s / 2) + C::kFirst * (2 * (s % 2) + g);
            const f32x4   x0 = values(qr, at, live);
            const f32x4   x1 = values(qr, at + C::kSecond, live);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[s][e] = (e < 4 ? x0[C::order(e)] : x1[C::order(e - 4)]) * a.scale;
                top     = fmaxf(top, fabsf(q[s][e]));
            }
        }
        if constexpr (THREE) {
            qexp = 0;
#pragma unroll
            for (int s = 0; s < 2 * NB; ++s) {
                f16x2 hi[4], mid[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e]  = take_b16(q[s][2 * e], q[s][2 * e + 1]);
                    mid[e] = take_b16(q[s][2 * e], q[s][2 * e + 1]);
                    lo[e]  = take_b16(q[s][2 * e], q[s][2 * e + 1]);
                }
                qh[s]              = join8(hi[0], hi[1], hi[2], hi[3]);
                ql[s]              = join8(mid[0], mid[1], mid[2], mid[3]);
                q3[s * kWideBlock] = join8(lo[0], lo[1], lo[2], lo[3]);
            }
        } else {
            const Pair both = swap32(top);
            top             = fmaxf(both.a, both.b);
            qexp            = exponent_of(top) - 13;
            const float to  = pow2(-qexp);
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
    }

    // group `even` + g of column 32 u + c
    auto vat = [&](int lane_of, int u, int even) {
        const int turn = (32 * u >> PartT::kTurn & 3) ^ (PartT::kTurn == 4 ? lane_of >> 4 & 1 : 0);
        return (32 * u + (lane_of & 31)) * kVStride + ((even + (lane_of >> 5)) ^ turn) * 16;
    };
    f32x16 o[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
        o[u] = f32x16{};
    }
    float less = INFINITY;  // weights are 2^(score + less)
    float l    = 0.0f;
    int   X    = kMinX;  // SIZES: o is times 2^(15 + kVTop - X)

    constexpr uint64_t kEvery = ~uint64_t{ 0 };
    uint64_t           left   = kEvery;  // SIZES: the tile's keys that no pass has had,
    uint64_t           pass   = kEvery;  // those of this one,
    bool               alike  = false;   // and whether they are known to be of one size
    bool               again  = false;   // blocks: the second pass over a large tile, of V's second pieces

    for (int i = beg; i < end;) {
        const int32_t j0 = key_tile(kt, i) * kTileKeys;
        float    kby = 1.0f, vby = 1.0f;
        int      kexp   = 0;
        bool     large  = false;   // blocks: a d is
        const bool second = again;
        int      vsize  = 0;       // SIZES: the exponent of V's largest
        const uint64_t member = pass;
        // go(whether the tile is large): what that changes is apart, so that the others' code is as without it
        auto if_large = [&](const auto & go) {
            if constexpr (kv_blocks(KIND)) {
                if (large) {
                    go(std::true_type{});
                    return;
                }
            }
            go(std::false_type{});
        };
        bool     ready  = true;
        const bool edge = j0 + kTileKeys - 1 > p0 || (a.window > 0 && j0 <= p1 - a.window && j0 + kTileKeys > a.sinks);
#pragma unroll
        for (int z = 0; z < PARTS; ++z) {
            if (mine[z]) {
                if (edge) {  // rows that no query of the tile sees count for nothing, whatever they hold
                    const int id = tid_again();
                    part[z].keep_k(seen_by(a, p0, p1, j0 + row_k(id, z)));
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        part[z].keep_v(e, seen_by(a, p0, p1, j0 + key_v(id, z) + (e < 4 ? e : e + 4)));
                    }
                }
                if constexpr (!kv_blocks(KIND)) {
                    if (a.hd < HD) {
                        const int id = tid_again() + kWideBlock * z;
                        part[z].cut(a.hd - kKvBlock * (id % NB), a.hd - 4 * (id % items));
                    }
                }
            }
        }
        {
            if (SIZES && pass != kEvery) {  // the others as if hidden
                const int id = tid_again();
#pragma unroll
                for (int z = 0; z < PARTS; ++z) {
                    if (mine[z]) {
                        part[z].keep_k(pass >> row_k(id, z) & 1);
                        const uint32_t from = static_cast<uint32_t>(pass >> key_v(id, z));
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            part[z].keep_v(e, from >> (e < 4 ? e : e + 4) & 1);
                        }
                    }
                }
            }
            uint32_t tk = 0, tv = 0;
            uint32_t lk = ~0u, lv = ~0u;  // the least that is not 0, less 1
            uint64_t bad = 0;             // keys
            auto     note = [&](uint32_t x, uint32_t & most, uint32_t & least) {
                most  = max(most, x);
                least = min(least, x - 1u);
            };
#pragma unroll
            for (int z = 0; z < PARTS; ++z) {
                if (mine[z]) {
                    note(part[z].top_k(), tk, lk);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        note(part[z].top_v(e), tv, lv);
                    }
                }
            }
            if (__any(max(tk, tv) >= PartT::kInf)) {
                // a value that is not finite makes its key a bad one; in V it counts
                // for nothing in the products (in K it is its key's scores' alone)
                tk = tv = 0;
                lk = lv = ~0u;
#pragma unroll
                for (int z = 0; z < PARTS; ++z) {
                    if (mine[z]) {
                        const int  id = tid_again();
                        const bool it = part[z].top_k() >= PartT::kInf;
                        bad |= static_cast<uint64_t>(it) << row_k(id, z);
                        note(it ? 0 : part[z].top_k(), tk, lk);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const bool is = part[z].top_v(e) >= PartT::kInf;
                            bad |= static_cast<uint64_t>(is) << (key_v(id, z) + (e < 4 ? e : e + 4));
                            part[z].keep_v(e, !is);
                            note(part[z].top_v(e), tv, lv);
                        }
                    }
                }
#pragma unroll
                for (int off = 1; off < kWave; off *= 2) {
                    bad |= __shfl_xor(static_cast<unsigned long long>(bad), off);
                }
            }
            if constexpr (SIZES) {
                const float fk  = wave_max(PartT::magnitude(tk));
                const float fv  = wave_max(PartT::magnitude(tv));
                const bool  odd = (lk != ~0u && PartT::magnitude(lk + 1u) < fk * kEven) ||
                                 (lv != ~0u && PartT::magnitude(lv + 1u) < fv * kEven);
                const float none = __any(odd) ? 1.0f : 0.0f;
                if (lane < 3) {
                    tops[lane * kWaves + wave] = lane == 0 ? fk : lane == 1 ? fv : none;
                }
            } else if constexpr (kv_blocks(KIND)) {
                const float is = __any(max(tk, tv) > kBigD) ? 1.0f : 0.0f;
                if (lane == 0) {
                    tops[wave] = is;
                }
            }
            if (lane == 0) {
                bads[wave] = bad;
            }
        }
        __syncthreads();  // the tile before is used up
        const uint64_t every = bads[0] | bads[1] | bads[2] | bads[3];
        uint64_t       none  = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(every >> 32)));
        none                 = none << 32 | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(every)));
        if constexpr (SIZES) {
            auto waves = [&](int which) { return *reinterpret_cast<const f32x4 *>(tops + which * kWaves); };
            auto most  = [](const f32x4 & t) { return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])); };
            auto apart = [](const f32x4 & t, float top) {
                bool is = false;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    is = is || (t[w] != 0.0f && t[w] < 0.5f * top);
                }
                return is;
            };
            const f32x4 k4 = waves(0), v4 = waves(1);
            const float kt = most(k4);
            const float vt = most(v4);
            if (!alike && __builtin_amdgcn_readfirstlane(apart(k4, kt) || apart(v4, vt) || most(waves(2)) != 0.0f)) {
                if (tid < 2 * kTileKeys) {
                    rmax[tid] = 0;
                }
                __syncthreads();
                auto at_least = [&](int row, uint32_t top) {
                    __hip_atomic_fetch_max(rmax + row, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                };
                const int id = tid_again();
#pragma unroll
                for (int z = 0; z < PARTS; ++z) {
                    if (mine[z]) {
                        at_least(row_k(id, z), part[z].top_k());
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            at_least(kTileKeys + key_v(id, z) + (e < 4 ? e : e + 4), part[z].top_v(e));
                        }
                    }
                }
                __syncthreads();
                // a lane a key; zeros are of any size
                const float    k1   = PartT::magnitude(rmax[lane]);
                const float    v1   = PartT::magnitude(rmax[kTileKeys + lane]);
                const bool     here = left >> lane & 1;
                const int      ke   = exponent_of(k1);
                const int      ve   = exponent_of(v1);
                const uint64_t some = __ballot(here && (k1 != 0.0f || v1 != 0.0f));
                auto           rows = [&](int k0, int k2, int v0, int v2) {
                    return __ballot(here && (k1 == 0.0f || (ke >= k0 && ke <= k2)) && (v1 == 0.0f || (ve >= v0 && ve <= v2)));
                };
                pass = rows(exponent_of(wave_max(here ? k1 : 0.0f)) - 2 * kAlike, INT_MAX,
                            exponent_of(wave_max(here ? v1 : 0.0f)) - 2 * kAlike, INT_MAX);
                if (some != 0 && (pass & some) == 0) {  // no row is of the largest in K and V
                    const int one = __ffsll(static_cast<unsigned long long>(some)) - 1;
                    const int k0  = __builtin_amdgcn_readlane(ke, one), v0 = __builtin_amdgcn_readlane(ve, one);
                    pass          = rows(k0 - kAlike, k0 + kAlike, v0 - kAlike, v0 + kAlike);
                }
                alike = true;
                ready = pass == left;
            }
            kexp  = __builtin_amdgcn_readfirstlane(exponent_of(kt)) - 13;
            vsize = __builtin_amdgcn_readfirstlane(exponent_of(vt));
            kby   = pow2(-kexp);
            vby   = pow2(kVTop - vsize);
        } else if constexpr (kv_blocks(KIND)) {
            const f32x4 t = *reinterpret_cast<const f32x4 *>(tops);
            large         = __builtin_amdgcn_readfirstlane(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) != 0.0f);
        }
        auto stage = [&](auto larger) {
            constexpr bool LARGE  = decltype(larger)::value;
            const int      staged = tid_each();
#pragma unroll
            for (int z = 0; z < PARTS; ++z) {
                if (mine[z]) {
                    const int id   = staged + kWideBlock * z;
                    const int item = id % items;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f16x8 hi, lo;
                        part[z].template k_pieces<LARGE>(magic, kby, j, hi, lo);
                        const int at = id / NB * KSTRIDE + id % NB * 64 + 16 * j;
                        *reinterpret_cast<f16x8 *>(kh + at) = hi;
                        if constexpr (TWO) {
                            *reinterpret_cast<f16x8 *>(kl + at) = lo;
                        }
                    }
                    auto column = [&](auto uc) {
                        constexpr int U = decltype(uc)::value;
                        f16x8         hi, lo;
                        part[z].template v_column<U, LARGE>(magic, vby, item, words, hi, lo);
                        if constexpr (LARGE) {
                            hi = second ? lo : hi;
                            lo = f16x8{};
                        }
                        const int dim = PartT::index(item, words, U);
                        const int at  = dim * kVStride + (id / items ^ (dim >> PartT::kTurn & 3)) * 16;
                        *reinterpret_cast<f16x8 *>(vh + at) = hi;
                        if constexpr (TWO) {
                            *reinterpret_cast<f16x8 *>(vl + at) = lo;
                        }
                    };
                    for_each(std::make_integer_sequence<int, 4>{}, column);
                }
            }
        };
        if_large(stage);
        if constexpr (SIZES) {
            const uint64_t rest = ready ? left & ~pass : left;
            i += rest == 0;
            left  = rest == 0 ? kEvery : rest;
            pass  = ready ? left : pass;
            alike = !ready;
        } else if constexpr (kv_blocks(KIND)) {
            again = large && !second;
            i += !again;
        } else {
            ++i;
        }
        if (i < end) {
            fetch(i);
        }
        __syncthreads();
        if (!ready || j0 > w1) {
            continue;  // to be had again in part, or none of it is seen by this wave's queries
        }
        if (none != 0) {  // ... but it makes the result of a query that sees it NaN, and no other's
            for (; none != 0; none &= none - 1) {
                if (sees(a, p, j0 + __ffsll(static_cast<unsigned long long>(none)) - 1)) {
                    l = NAN;
                }
            }
        }
        // scores of key 32 x + 8 (i / 4) + 4 g + i % 4
        // (ahead of the waves that are at their exponentials: 8192 positions 860
        // to 790 us)
        __builtin_amdgcn_s_setprio(1);
        f32x16 sc[2] = { f32x16{}, f32x16{} };
        auto keys_at = [&](const char * from, int x, int s) {
            return *reinterpret_cast<const f16x8 *>(from + (32 * x + c) * KSTRIDE + 32 * s + 16 * g);
        };
        auto score = [&](auto larger) {
            constexpr bool LARGE = decltype(larger)::value;
#pragma unroll
            for (int s = 0; s < 2 * NB; ++s) {
                f16x8 hi[2], lo[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    hi[x] = keys_at(kh, x, s);
                    if constexpr (TWO && !LARGE) {
                        lo[x] = keys_at(kl, x, s);
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    sc[x] = product<KIND>(hi[x], qh[s], sc[x]);
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    sc[x] = product<KIND>(hi[x], ql[s], sc[x]);
                }
                if constexpr (THREE) {
                    const f16x8 third = q3[s * kWideBlock];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        sc[x] = product<KIND>(hi[x], third, sc[x]);
                    }
                }
                if constexpr (TWO && !LARGE) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        sc[x] = product<KIND>(lo[x], qh[s], sc[x]);
                    }
                }
            }
            if constexpr (LARGE) {
                sc[0] *= kLargeBy;
                sc[1] *= kLargeBy;
#pragma unroll
                for (int s = 0; s < 2 * NB; ++s) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const f16x8 lo = keys_at(kl, x, s);
                        sc[x]          = product<KIND>(lo, qh[s], sc[x]);
                        sc[x]          = product<KIND>(lo, ql[s], sc[x]);
                    }
                }
            }
        };
        if_large(score);
        __builtin_amdgcn_s_setprio(0);
        // (within what is a normal number: a zero query's and zero keys' exponents
        // add up to -226, and 0 times a hidden key's -infinity is NaN)
        const float qs = pow2(min(max(qexp + kexp, -126), 127));
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
        if (SIZES && member != kEvery) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t in = static_cast<uint32_t>(member >> (32 * x)) >> (4 * g);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[x][e] = in >> (8 * (e / 4) + e % 4) & 1u ? sc[x][e] : -INFINITY;
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
        const Pair  both = swap32(top);
        const float here = fmaxf(both.a, both.b) * qs;
        const float now  = fminf(less, shift_for(here, SIZES || THREE ? 0.0f : kPShift));
        int         need = X;
        if constexpr (SIZES) {
            // what this pass's largest weighted row needs, or those before it, whose
            // weights have gone down
            const int down = static_cast<int>(fminf(floorf(less - now), 1000.0f));
            need           = vsize + 1 + static_cast<int>(fmaxf(floorf(here + now), -1000.0f));
            need           = max(max(need, X - down), kMinX);
        }
        auto turn = [&](float by) {
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                o[u] *= by;
            }
        };
        if (__any(now < less || need != X)) {
            const float alpha = shift_change(less, now);
            const float by    = SIZES ? __builtin_ldexpf(alpha, X - need) : alpha;
            l *= alpha;
            turn(by);
        }
        less              = now;
        X                 = need;
        const float add   = shift_added(less);
        const int   times = vsize + 15 - X;
        auto        held  = [&](float score) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score, qs, add));
            l += w;
            return SIZES ? __builtin_ldexpf(w, times) : w;
        };
        // a large tile: V's first pieces, 2^-8 of their values, in the first pass, what
        // they leave in the second, which has been counted in l already
        if (kv_blocks(KIND) && large && !second) {
            turn(1.0f / kLargeBy);
        }
        const float before = l;
        auto        weigh  = [&] {
            const int from = tid_each() % kWave;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    f16x2 hi[4], lo[4], third[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float a0 = held(sc[x][8 * s + 2 * e]);
                        float a1 = held(sc[x][8 * s + 2 * e + 1]);
                        if constexpr (THREE) {
                            hi[e]    = take_b16(a0, a1);
                            lo[e]    = take_b16(a0, a1);
                            third[e] = take_b16(a0, a1);
                        } else {
                            split2(a0, a1, hi[e], lo[e]);
                        }
                    }
                    const f16x8 ph = join8(hi[0], hi[1], hi[2], hi[3]);
                    const f16x8 pl = join8(lo[0], lo[1], lo[2], lo[3]);
                    f16x8 vv[NB];
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        vv[u] = *reinterpret_cast<const f16x8 *>(vh + vat(from, u, 4 * x + 2 * s));
                    }
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        o[u] = product<KIND>(vv[u], ph, o[u]);
                    }
#pragma unroll
                    for (int u = 0; u < NB; ++u) {
                        o[u] = product<KIND>(vv[u], pl, o[u]);
                    }
                    if constexpr (THREE) {
                        const f16x8 p3 = join8(third[0], third[1], third[2], third[3]);
#pragma unroll
                        for (int u = 0; u < NB; ++u) {
                            o[u] = product<KIND>(vv[u], p3, o[u]);
                        }
                    }
                    if constexpr (TWO) {
#pragma unroll
                        for (int u = 0; u < NB; ++u) {
                            vv[u] = *reinterpret_cast<const f16x8 *>(vl + vat(from, u, 4 * x + 2 * s));
                        }
#pragma unroll
                        for (int u = 0; u < NB; ++u) {
                            o[u] = product<KIND>(vv[u], ph, o[u]);
                        }
                    }
                }
            }
        };
        weigh();
        if (kv_blocks(KIND) && large) {
            if (second) {
                l = before;
            } else {
                turn(kLargeBy);
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
    if (dest < 0) {
        out = reinterpret_cast<float *>(a.y + n * a.yn + t * a.yt + head * a.yh);
        by *= over(l, p >= 0);
    } else {
        out = partial_o(a, row, dest);
        if (g == 0) {
            float * ml = partial_ml(a, row, dest);
            ml[0]      = -less;
            ml[1]      = l;
        }
    }
    if constexpr (SIZES) {
#pragma unroll
        for (int u = 0; u < NB; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[u][e] = __builtin_ldexpf(o[u][e] * by, X - 15 - kVTop);
            }
        }
        by = 1.0f;
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int   dim = 32 * u + 2 * e + 4 * g;
            const f32x4 v   = { o[u][e] * by, o[u][e + 1] * by, o[u][e + 2] * by, o[u][e + 3] * by };
            if (kv_blocks(KIND) || dim + 4 <= a.hd) {
                *reinterpret_cast<f32x4u *>(out + dim) = v;
            } else {
                for (int k = 0; dim + k < a.hd; ++k) {
                    out[dim + k] = v[k];
                }
            }
        }
    }
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
        case 4:
            return launch_wide_as<KIND, 4>(a, stream);
        case 5:
            return launch_wide_as<KIND, 5>(a, stream);
        case 6:
            return launch_wide_as<KIND, 6>(a, stream);
        case 7:
            return launch_wide_as<KIND, 7>(a, stream);
        default:
            return launch_wide_as<KIND, 8>(a, stream);
    }
}

}  // namespace

shp_status_t launch_attn_wide(int kind, const AttnArgs & a, hipStream_t stream) {
    switch (kind) {
        case kKvF32:
            return launch_wide<kKvF32>(a, stream);
        case kKvF16:
            return launch_wide<kKvF16>(a, stream);
        case kKvBF16:
            return launch_wide<kKvBF16>(a, stream);
        case kKvQ8:
            return launch_wide<kKvQ8>(a, stream);
        default:
            return launch_wide<kKvQ4>(a, stream);
    }
}

}  // namespace shp
