// What the KV cache's kernels share (k_kv.hip, k_attn.hip): the cache types,
// their rows, and the checks of a cache's descriptor.
#pragma once

#include "shp_internal.hpp"

namespace shp {

// Cache types as template arguments.
enum KvKind { kKvF32 = 0, kKvF16 = 1, kKvBF16 = 2, kKvQ8 = 3, kKvQ4 = 4 };

constexpr int    kKvBlock   = 32;  // values of a block
constexpr size_t kQ4Bytes   = 18;  // {f16 d; uint8 q[16]}
constexpr int    kKvMaxDim  = 256;
constexpr int    kKvMaxSeqs = 65535;  // a grid dimension

// Rows of a call's own tensors in one sequence (32-value pieces in the store
// and the load): a launch of eight threads for each stays below 2^32 threads.
constexpr int64_t kKvMaxRows = int64_t{ 1 } << 28;

inline int kv_kind(int32_t type) {
    switch (type) {
        case SHP_TYPE_F32:
            return kKvF32;
        case SHP_TYPE_F16:
            return kKvF16;
        case SHP_TYPE_BF16:
            return kKvBF16;
        case SHP_TYPE_Q8_0:
            return kKvQ8;
        case SHP_TYPE_Q4_0:
            return kKvQ4;
        default:
            return -1;
    }
}

// Bytes of a block of 32 values, or of one value.
__host__ __device__ constexpr int kv_unit_bytes(int kind) {
    return kind == kKvQ8 ? static_cast<int>(kQ8Bytes) : kind == kKvQ4 ? static_cast<int>(kQ4Bytes) : kind == kKvF32 ? 4 : 2;
}

__host__ __device__ constexpr bool kv_blocks(int kind) {
    return kind == kKvQ8 || kind == kKvQ4;
}

__host__ __device__ constexpr int64_t kv_row_bytes(int kind, int64_t ne0) {
    return (kv_blocks(kind) ? ne0 / kKvBlock : ne0) * kv_unit_bytes(kind);
}

// Two- and four-byte loads and stores at a two-byte boundary: block rows have
// no larger one in general.
typedef uint32_t u32_at2 __attribute__((aligned(2)));
typedef uint64_t u64_at2 __attribute__((aligned(2)));

// One value of a cache row, for the forms that take a row value by value.
template <int KIND> __device__ __forceinline__ float kv_value(const char * row, int i) {
    if constexpr (KIND == kKvF32) {
        return reinterpret_cast<const float *>(row)[i];
    } else if constexpr (KIND == kKvF16) {
        return f16_bits_to_f32(reinterpret_cast<const uint16_t *>(row)[i]);
    } else if constexpr (KIND == kKvBF16) {
        return bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(row)[i]);
    } else {
        const char * block = row + (i / kKvBlock) * kv_unit_bytes(KIND);
        const float  d     = f16_bits_to_f32(*reinterpret_cast<const uint16_t *>(block));
        const int    j     = i % kKvBlock;
        if constexpr (KIND == kKvQ8) {
            return static_cast<float>(static_cast<int8_t>(block[2 + j])) * d;
        } else {
            const int byte = static_cast<uint8_t>(block[2 + (j & 15)]);
            return static_cast<float>((j < 16 ? byte & 15 : byte >> 4) - 8) * d;
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// well_formed() with the cache's types.
inline bool kv_well_formed(const shp_tensor * t) {
    if (t == nullptr || t->data == nullptr || t->reserved != 0) {
        return false;
    }
    for (int d = 0; d < 4; ++d) {
        if (t->ne[d] <= 0) {
            return false;
        }
    }
    const int kind = kv_kind(t->type);
    return kind >= 0 && t->nb[0] == static_cast<size_t>(kv_unit_bytes(kind)) &&
           (!kv_blocks(kind) || t->ne[0] % kKvBlock == 0);
}

// Every row starts at a multiple of its element's size (2 for block types).
inline bool kv_aligned(const shp_tensor & t) {
    return rows_aligned(t, t.type == SHP_TYPE_F32 ? 4 : 2);
}

// Bytes of one row of a cache, or of a tensor of the framework's plain types.
inline size_t kv_bytes_of_row(const shp_tensor & t) {
    return kv_kind(t.type) >= 0 ? static_cast<size_t>(kv_row_bytes(kv_kind(t.type), t.ne[0])) : row_bytes(t.type, t.ne[0]);
}

// [lo, hi) of the bytes that t's rows lie in.
inline void kv_span(const shp_tensor & t, uintptr_t & lo, uintptr_t & hi) {
    size_t end = kv_bytes_of_row(t);
    for (int d = 1; d < 4; ++d) {
        end += static_cast<size_t>(t.ne[d] - 1) * t.nb[d];
    }
    lo = reinterpret_cast<uintptr_t>(t.data);
    hi = lo + end;
}

// No two rows of t share a byte: taken by size, each stride is at least what
// the dimensions below it cover.
inline bool kv_rows_apart(const shp_tensor & t) {
    size_t covered = kv_bytes_of_row(t);
    bool   used[4] = { true, t.ne[1] == 1, t.ne[2] == 1, t.ne[3] == 1 };
    for (int pass = 0; pass < 3; ++pass) {
        int next = -1;
        for (int d = 1; d < 4; ++d) {
            if (!used[d] && (next < 0 || t.nb[d] < t.nb[next])) {
                next = d;
            }
        }
        if (next < 0) {
            break;
        }
        if (t.nb[next] < covered) {
            return false;
        }
        used[next] = true;
        covered += static_cast<size_t>(t.ne[next] - 1) * t.nb[next];
    }
    return true;
}

// A byte offset inside t fits 63 bits with room for sums: extents and strides
// that could wrap are refused before any product of them is formed.
inline bool kv_addressable(const shp_tensor & t) {
    for (int d = 1; d < 4; ++d) {
        if (t.ne[d] > int64_t{ 1 } << 31 || t.nb[d] > size_t{ 1 } << 46 ||
            (t.ne[d] > 1 && static_cast<uint64_t>(t.ne[d] - 1) > (uint64_t{ 1 } << 60) / (t.nb[d] > 0 ? t.nb[d] : 1))) {
            return false;
        }
    }
    return t.ne[0] <= int64_t{ 1 } << 31;
}

// Whether two tensors of a call share bytes: that of their spans, except that
// tensors whose rows interleave in one allocation (a k and a v cache in one
// buffer, side by side in each position) share none where their strides are
// the same and their rows fall in different parts of the innermost stride.
inline bool kv_overlap(const shp_tensor & a, const shp_tensor & b) {
    uintptr_t alo, ahi, blo, bhi;
    kv_span(a, alo, ahi);
    kv_span(b, blo, bhi);
    if (!(alo < bhi && blo < ahi)) {
        return false;
    }
    for (int d = 1; d < 4; ++d) {
        if (a.ne[d] > 1 && b.ne[d] > 1) {
            const size_t nb = a.nb[d];
            if (nb == 0 || nb != b.nb[d]) {
                continue;
            }
            // a and b inside one period of this dimension: all smaller strides
            // stay within it, all larger ones are whole periods
            size_t aw = kv_bytes_of_row(a);
            size_t bw = kv_bytes_of_row(b);
            bool   ok = true;
            for (int e = 1; e < 4; ++e) {
                if (e == d) {
                    continue;
                }
                for (const auto * t : { &a, &b }) {
                    if (t->ne[e] == 1) {
                        continue;
                    }
                    if (t->nb[e] < nb) {
                        (t == &a ? aw : bw) += static_cast<size_t>(t->ne[e] - 1) * t->nb[e];
                    } else if (t->nb[e] % nb != 0) {
                        ok = false;
                    }
                }
            }
            const size_t off = (blo >= alo ? blo - alo : nb - (alo - blo) % nb) % nb;  // b's start in a's period
            if (ok && off >= aw && off + bw <= nb) {
                return false;
            }
        }
    }
    return true;
}

// An I32 [n] of per-sequence numbers.
inline bool kv_numbers(const shp_tensor * t, int64_t n) {
    return well_formed(t) && t->type == SHP_TYPE_I32 && t->ne[0] == n && nrows(*t) == 1;
}

// Checks that shp_kv_store, shp_kv_load and shp_attn_kv share: a pair of caches
// of one shape and one type.
inline shp_status_t kv_check_caches(const shp_tensor * k_cache, const shp_tensor * v_cache) {
    if (!kv_well_formed(k_cache) || !kv_well_formed(v_cache) || !same_shape(*k_cache, *v_cache)) {
        return SHP_ERR_INVALID_ARG;
    }
    if (k_cache->type != v_cache->type || !kv_aligned(*k_cache) || !kv_aligned(*v_cache) ||
        k_cache->ne[0] > kKvMaxDim || k_cache->ne[3] > kKvMaxSeqs || k_cache->ne[2] > INT32_MAX ||
        !kv_addressable(*k_cache) || !kv_addressable(*v_cache)) {
        return SHP_ERR_UNSUPPORTED;
    }
    return SHP_OK;
}

}  // namespace shp
