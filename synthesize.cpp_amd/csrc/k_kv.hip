// The KV cache's rows, written and read back: shp_kv_store and shp_kv_load.
//
// Eight lanes take a block of 32 values, a float4 each, so a wave reads (or,
// loading, writes) 1 KB of F32 at a time; a block's largest magnitude is three
// DPP steps away. Both directions are bound by the F32 side's bytes: 16
// sequences of 8192 rows of 8 heads of 128 values load in 234 us, 5.2 TB/s (a
// large copy: 5.0), and 8192 rows are stored and read back in 35 us (MI355X).
#include <cmath>

#include "shp_kv.hpp"

namespace shp {
namespace {

// k or v: the F32 side and the cache side, byte strides of head, row, sequence.
struct KvSide {
    char *  x;
    char *  c;
    int64_t xh, xt, xn;
    int64_t ch, ct, cn;
};

struct KvArgs {
    KvSide          side[2];
    const int32_t * slot;
    const int32_t * count;   // or null
    int32_t *       status;  // or null
    int32_t         hd;
    int32_t         T;
    int32_t         cap;
    uint32_t        total;  // 32-value pieces of a sequence: T x heads x ceil(hd/32)
    FastDiv         fpieces;  // ceil(hd/32)
    FastDiv         fheads;
};

constexpr int kKvThreads = 256;
constexpr int kKvPieces  = kKvThreads / 8;  // of a workgroup

constexpr int kDppShl4 = 0x104;  // row_shl:4: lane i of each 16 reads lane i + 4

// The largest of eight neighbouring lanes' values, in each of them.
__device__ __forceinline__ float max8(float v) {
    v = fmaxf(v, dpp_f32<kDppQuadXor1>(v));
    v = fmaxf(v, dpp_f32<kDppQuadXor2>(v));
    return fmaxf(v, dpp_f32<kDppHalfMirror>(v));
}

// Of a wave's per-lane truth, the eight bits of this lane's group.
__device__ __forceinline__ uint32_t ballot8(bool v) {
    return static_cast<uint32_t>(__ballot(v) >> (threadIdx.x & 56u)) & 0xffu;
}

// 1/d as the formats' quantisers use it.
__device__ __forceinline__ float inverse_scale(float d) {
    return fabsf(d) >= 0x1p-126f ? 1.0f / d : 0.0f;
}

__device__ __forceinline__ uint16_t f16_bits(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

// Rounded to nearest even; a NaN stays one.
__device__ __forceinline__ uint16_t bf16_bits(float v) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) {
        return static_cast<uint16_t>((u >> 16) | 0x40u);
    }
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

// The values 4j..4j+3 of a block, lane j of its eight, as the block's bytes.
template <int KIND> __device__ __forceinline__ void store_block(char * block, int j, const float (&x)[4]) {
    constexpr uint16_t kNaN16 = 0x7e00;
    float              top    = 0.0f;
    bool               finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top    = fmaxf(top, fabsf(x[i]));
        finite = finite && fabsf(x[i]) < INFINITY;  // false for a NaN
    }
    const float mine = top;
    top              = max8(top);
    const bool bad   = ballot8(!finite) != 0;
    if constexpr (KIND == kKvQ8) {
        const float d  = top / 127.0f;
        const float id = inverse_scale(d);
        uint32_t    w  = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = roundf(x[i] * id);  // half away from zero
            w |= (static_cast<uint32_t>(static_cast<int>(bad ? 0.0f : v)) & 0xffu) << (8 * i);
        }
        *reinterpret_cast<u32_at2 *>(block + 2 + 4 * j) = w;
        if (j == 0) {
            *reinterpret_cast<uint16_t *>(block) = bad ? kNaN16 : f16_bits(d);
        }
    } else {
        // the sign of the first value of the largest magnitude
        bool negative = false;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            negative = fabsf(x[i]) == top ? x[i] < 0.0f : negative;
        }
        const uint32_t have  = ballot8(mine == top);
        const uint32_t signs = ballot8(negative);
        const bool     neg   = (signs >> (__ffs(static_cast<int>(have | 0x100u)) - 1)) & 1u;
        const float    d     = (neg ? -top : top) * -0.125f;
        const float    id    = inverse_scale(d);
        uint32_t       w     = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = fminf(x[i] * id + 8.5f, 15.0f);
            w |= (bad ? 8u : static_cast<uint32_t>(static_cast<int>(v))) << (8 * i);
        }
        const uint32_t high = dpp_u32<kDppShl4>(w);
        if (j < 4) {
            *reinterpret_cast<u32_at2 *>(block + 2 + 4 * j) = w | (high << 4);
        }
        if (j == 0) {
            *reinterpret_cast<uint16_t *>(block) = bad ? kNaN16 : f16_bits(d);
        }
    }
}

template <int KIND> __global__ __launch_bounds__(kKvThreads) void k_kv_store(const KvArgs a) {
    const int     n     = blockIdx.y;
    const KvSide  s     = a.side[blockIdx.z];
    const int32_t count = a.count != nullptr ? a.count[n] : a.T;
    const int32_t slot  = a.slot[n];
    if (count < 0 || count > a.T || (count > 0 && (slot < 0 || slot > a.cap - count))) {
        if (a.status != nullptr && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
            *a.status = 1;
        }
        return;
    }
    const uint32_t p = blockIdx.x * kKvPieces + threadIdx.x / 8;
    if (p >= a.total) {
        return;
    }
    const int      j  = threadIdx.x % 8;
    const uint32_t r  = fastdiv(p, a.fpieces);
    const uint32_t b  = p - r * a.fpieces.d;
    const uint32_t t  = fastdiv(r, a.fheads);
    const uint32_t h  = r - t * a.fheads.d;
    if (static_cast<int32_t>(t) >= count) {
        return;
    }
    const int     e = static_cast<int>(b) * kKvBlock + 4 * j;
    const float * x = reinterpret_cast<const float *>(s.x + n * s.xn + t * s.xt + h * s.xh) + e;
    char *        c = s.c + n * s.cn + (static_cast<int64_t>(slot) + t) * s.ct + h * s.ch;
    float         v[4];
    if (e + 4 <= a.hd) {
        const f32x4 w = ld_stream4u(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = w[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = e + i < a.hd ? x[i] : 0.0f;
        }
    }
    if constexpr (kv_blocks(KIND)) {
        store_block<KIND>(c + static_cast<int64_t>(b) * kv_unit_bytes(KIND), j, v);
    } else if constexpr (KIND == kKvF32) {
        float * o = reinterpret_cast<float *>(c) + e;
        if (e + 4 <= a.hd) {
            *reinterpret_cast<f32x4u *>(o) = f32x4{ v[0], v[1], v[2], v[3] };
        } else {
            for (int i = 0; e + i < a.hd; ++i) {
                o[i] = v[i];
            }
        }
    } else {
        uint64_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w |= static_cast<uint64_t>(KIND == kKvF16 ? f16_bits(v[i]) : bf16_bits(v[i])) << (16 * i);
        }
        uint16_t * o = reinterpret_cast<uint16_t *>(c) + e;
        if (e + 4 <= a.hd) {
            *reinterpret_cast<u64_at2 *>(o) = w;
        } else {
            for (int i = 0; e + i < a.hd; ++i) {
                o[i] = static_cast<uint16_t>(w >> (16 * i));
            }
        }
    }
}

template <int KIND> __global__ __launch_bounds__(kKvThreads) void k_kv_load(const KvArgs a) {
    const int      n     = blockIdx.y;
    const KvSide   s     = a.side[blockIdx.z];
    const int32_t  count = a.count != nullptr ? min(a.count[n], a.T) : a.T;
    const int32_t  slot  = a.slot[n];
    const uint32_t p     = blockIdx.x * kKvPieces + threadIdx.x / 8;
    if (p >= a.total) {
        return;
    }
    const int      j = threadIdx.x % 8;
    const uint32_t r = fastdiv(p, a.fpieces);
    const uint32_t b = p - r * a.fpieces.d;
    const uint32_t t = fastdiv(r, a.fheads);
    const uint32_t h = r - t * a.fheads.d;
    if (static_cast<int32_t>(t) >= count) {
        return;
    }
    const int     e   = static_cast<int>(b) * kKvBlock + 4 * j;
    float *       x   = reinterpret_cast<float *>(s.x + n * s.xn + t * s.xt + h * s.xh) + e;
    const int64_t row = static_cast<int64_t>(slot) + t;
    const char *  c   = s.c + n * s.cn + row * s.ct + h * s.ch;
    f32x4         v   = splat4(__uint_as_float(0x7fc00000u));
    if (row >= 0 && row < a.cap) {
        if constexpr (kv_blocks(KIND)) {
            const char *   block = c + static_cast<int64_t>(b) * kv_unit_bytes(KIND);
            const float    d     = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(block));
            const int      word  = KIND == kKvQ8 ? j : j & 3;
            const uint32_t w     = *reinterpret_cast<const u32_at2 *>(block + 2 + 4 * word);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q = KIND == kKvQ8 ? static_cast<int8_t>(w >> (8 * i)) :
                                              static_cast<int>((w >> (8 * i + (j < 4 ? 0 : 4))) & 15u) - 8;
                v[i]        = static_cast<float>(q) * d;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = e + i < a.hd ? kv_value<KIND>(c, e + i) : 0.0f;
            }
        }
    }
    if (e + 4 <= a.hd) {
        st_stream4u(x, v);
    } else {
        for (int i = 0; e + i < a.hd; ++i) {
            x[i] = v[i];
        }
    }
}

KvSide side_of(const shp_tensor & x, const shp_tensor & c) {
    auto nb = [](const shp_tensor & t, int d) { return static_cast<int64_t>(t.ne[d] > 1 ? t.nb[d] : 0); };
    return KvSide{ static_cast<char *>(x.data), static_cast<char *>(c.data), nb(x, 1), nb(x, 2), nb(x, 3),
                   nb(c, 1),                    nb(c, 2),                    nb(c, 3) };
}

// The checks of both directions, and the arguments. k and v are the F32 side.
shp_status_t kv_args(const shp_tensor * k,
                     const shp_tensor * v,
                     const shp_tensor * k_cache,
                     const shp_tensor * v_cache,
                     const shp_tensor * slot,
                     const shp_tensor * count,
                     bool               store,
                     KvArgs &           a) {
    const shp_status_t st = kv_check_caches(k_cache, v_cache);
    if (st != SHP_OK) {
        return st;
    }
    if (!well_formed(k) || !well_formed(v) || !same_shape(*k, *v) || k->ne[0] != k_cache->ne[0] ||
        k->ne[1] != k_cache->ne[1] || k->ne[3] != k_cache->ne[3] || !kv_numbers(slot, k->ne[3]) ||
        (count != nullptr && !kv_numbers(count, k->ne[3]))) {
        return SHP_ERR_INVALID_ARG;
    }
    if (k->type != SHP_TYPE_F32 || v->type != SHP_TYPE_F32 || !kv_aligned(*k) || !kv_aligned(*v) || !kv_addressable(*k) ||
        !kv_addressable(*v) || !i32_aligned(*slot) || (count != nullptr && !i32_aligned(*count))) {
        return SHP_ERR_UNSUPPORTED;
    }
    const int64_t pieces = (k->ne[0] + kKvBlock - 1) / kKvBlock;
    if (k->ne[1] > kKvMaxRows / pieces || k->ne[2] > kKvMaxRows / (k->ne[1] * pieces)) {
        return SHP_ERR_UNSUPPORTED;
    }
    const shp_tensor * written[2] = { store ? k_cache : k, store ? v_cache : v };
    const shp_tensor * read[4]    = { store ? k : k_cache, store ? v : v_cache, slot, count };
    for (int i = 0; i < 2; ++i) {
        if (!kv_rows_apart(*written[i]) || (i == 0 && kv_overlap(*written[0], *written[1]))) {
            return SHP_ERR_UNSUPPORTED;
        }
        for (const shp_tensor * r : read) {
            if (r != nullptr && kv_overlap(*written[i], *r)) {
                return SHP_ERR_UNSUPPORTED;
            }
        }
    }
    a.side[0] = side_of(*k, *k_cache);
    a.side[1] = side_of(*v, *v_cache);
    a.slot    = static_cast<const int32_t *>(slot->data);
    a.count   = count != nullptr ? static_cast<const int32_t *>(count->data) : nullptr;
    a.hd      = static_cast<int32_t>(k->ne[0]);
    a.T       = static_cast<int32_t>(k->ne[2]);
    a.cap     = static_cast<int32_t>(k_cache->ne[2]);
    a.total   = static_cast<uint32_t>(k->ne[2] * k->ne[1] * pieces);
    a.fpieces = make_fastdiv(static_cast<uint32_t>(pieces));
    a.fheads  = make_fastdiv(static_cast<uint32_t>(k->ne[1]));
    return SHP_OK;
}

template <class Kernel> shp_status_t kv_launch(Kernel kernel, const KvArgs & a, int64_t seqs, hipStream_t stream) {
    const dim3 grid((a.total + kKvPieces - 1) / kKvPieces, static_cast<unsigned>(seqs), 2);
    hipLaunchKernelGGL(kernel, grid, dim3(kKvThreads), 0, stream, a);
    return launch_status();
}

}  // namespace
}  // namespace shp

using namespace shp;

extern "C" shp_status_t shp_kv_store(const shp_tensor * k,
                                     const shp_tensor * v,
                                     const shp_tensor * slot,
                                     const shp_tensor * count,
                                     shp_tensor *       k_cache,
                                     shp_tensor *       v_cache,
                                     shp_tensor *       status,
                                     shp_stream_t       stream) {
    KvArgs             a{};
    const shp_status_t st = kv_args(k, v, k_cache, v_cache, slot, count, true, a);
    if (st != SHP_OK) {
        return st;
    }
    if (status != nullptr) {
        if (!kv_numbers(status, 1)) {
            return SHP_ERR_INVALID_ARG;
        }
        if (!i32_aligned(*status)) {
            return SHP_ERR_UNSUPPORTED;
        }
        for (const shp_tensor * t : { k, v, slot, count, static_cast<const shp_tensor *>(k_cache),
                                      static_cast<const shp_tensor *>(v_cache) }) {
            if (t != nullptr && kv_overlap(*t, *status)) {
                return SHP_ERR_UNSUPPORTED;
            }
        }
        a.status = static_cast<int32_t *>(status->data);
    }
    if (dry_run()) {
        return SHP_OK;
    }
    const hipStream_t s = as_stream(stream);
    switch (kv_kind(k_cache->type)) {
        case kKvF32:
            return kv_launch(k_kv_store<kKvF32>, a, k->ne[3], s);
        case kKvF16:
            return kv_launch(k_kv_store<kKvF16>, a, k->ne[3], s);
        case kKvBF16:
            return kv_launch(k_kv_store<kKvBF16>, a, k->ne[3], s);
        case kKvQ8:
            return kv_launch(k_kv_store<kKvQ8>, a, k->ne[3], s);
        default:
            return kv_launch(k_kv_store<kKvQ4>, a, k->ne[3], s);
    }
}

extern "C" shp_status_t shp_kv_load(const shp_tensor * k_cache,
                                    const shp_tensor * v_cache,
                                    const shp_tensor * slot,
                                    const shp_tensor * count,
                                    shp_tensor *       k,
                                    shp_tensor *       v,
                                    shp_stream_t       stream) {
    KvArgs             a{};
    const shp_status_t st = kv_args(k, v, k_cache, v_cache, slot, count, false, a);
    if (st != SHP_OK || dry_run()) {
        return st;
    }
    const hipStream_t s = as_stream(stream);
    switch (kv_kind(k_cache->type)) {
        case kKvF32:
            return kv_launch(k_kv_load<kKvF32>, a, k->ne[3], s);
        case kKvF16:
            return kv_launch(k_kv_load<kKvF16>, a, k->ne[3], s);
        case kKvBF16:
            return kv_launch(k_kv_load<kKvBF16>, a, k->ne[3], s);
        case kKvQ8:
            return kv_launch(k_kv_load<kKvQ8>, a, k->ne[3], s);
        default:
            return kv_launch(k_kv_load<kKvQ4>, a, k->ne[3], s);
    }
}
