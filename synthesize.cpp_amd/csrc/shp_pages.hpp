// What the paged KV cache's kernels share (k_pages.hip, k_attn_pages.hip): the
// pool as the kernels see it, and the checks of its descriptors.
#pragma once

#include "shp_kv.hpp"

namespace shp {

constexpr int kGroup = 16;  // rows that are in one page whatever its size: a page starts at a multiple of them

// K's or V's half of the pool: strides of page and head in bytes, of a page's scales in floats.
struct PoolSide {
    char *  codes;
    float * scale;
    int64_t cp, ch;
    int64_t sp;
};

struct Pool {
    PoolSide side[2];
    int32_t  pages;
    int32_t  shift;  // log2 of a page's rows
    int32_t  hd;
    int32_t  kv;
};

// The tables, and the rows of a sequence that they have room for.
struct Tables {
    const char * data;
    int64_t      tn;
    int32_t      most;  // pages of a sequence
    int32_t      cap;   // rows
};

__device__ __forceinline__ const int32_t * table_of(const Tables & t, int n) {
    return reinterpret_cast<const int32_t *>(t.data + n * t.tn);
}

// A block's scale as it counts: not finite or negative is NaN (and -0 is 0).
__device__ __forceinline__ float block_scale(float d) {
    return d >= 0.0f && d < INFINITY ? fabsf(d) : NAN;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

inline int page_shift(int64_t page) {
    for (int s = 4; s <= 8; ++s) {
        if (page == int64_t{ 1 } << s) {
            return s;
        }
    }
    return -1;
}

inline bool codes_formed(const shp_tensor * t) {
    if (t == nullptr || t->data == nullptr || t->reserved != 0 || t->type != SHP_TYPE_I8 || t->nb[0] != 1) {
        return false;
    }
    for (int d = 0; d < 4; ++d) {
        if (t->ne[d] <= 0) {
            return false;
        }
    }
    return true;
}

// The tensors' bytes as kv_overlap() wants them: codes as rows of a whole block.
inline shp_tensor codes_as_rows(const shp_tensor & t) {
    shp_tensor r = t;
    r.type       = SHP_TYPE_F32;  // (blocks are whole dwords)
    r.nb[0]      = 4;
    r.ne[0]      = t.ne[0] * t.ne[1] / 4;
    r.ne[1]      = 1;
    r.nb[1]      = static_cast<size_t>(t.ne[0] * t.ne[1]);
    return r;
}

inline shp_status_t check_codes(const shp_tensor * k, const shp_tensor * v) {
    if (!codes_formed(k) || !codes_formed(v) || k->ne[0] != v->ne[1] || k->ne[1] != v->ne[0] || k->ne[2] != v->ne[2] ||
        k->ne[3] != v->ne[3]) {
        return SHP_ERR_INVALID_ARG;
    }
    for (const shp_tensor * t : { k, v }) {
        if (reinterpret_cast<uintptr_t>(t->data) % 16 != 0 || t->nb[1] != static_cast<size_t>(t->ne[0]) ||
            (t->ne[2] > 1 && t->nb[2] % 16 != 0) || (t->ne[3] > 1 && t->nb[3] % 16 != 0) || !kv_addressable(*t)) {
            return SHP_ERR_UNSUPPORTED;
        }
    }
    if (k->ne[0] > kKvMaxDim || k->ne[0] % 16 != 0 || page_shift(k->ne[1]) < 0 || k->ne[2] > kKvMaxSeqs ||
        k->ne[3] > INT32_MAX / k->ne[1]) {
        return SHP_ERR_UNSUPPORTED;
    }
    return SHP_OK;
}

inline shp_status_t check_scale(const shp_tensor * s, const shp_tensor & codes) {
    if (!well_formed(s) || s->ne[0] != codes.ne[2] || s->ne[1] != codes.ne[3] || s->ne[2] != 1 || s->ne[3] != 1) {
        return SHP_ERR_INVALID_ARG;
    }
    return s->type == SHP_TYPE_F32 && kv_aligned(*s) && kv_addressable(*s) ? SHP_OK : SHP_ERR_UNSUPPORTED;
}

inline shp_status_t check_pool(const shp_tensor * k, const shp_tensor * v, const shp_tensor * ks, const shp_tensor * vs, Pool & p) {
    shp_status_t st = check_codes(k, v);
    if (st == SHP_OK) {
        st = check_scale(ks, *k);
    }
    if (st == SHP_OK) {
        st = check_scale(vs, *v);
    }
    if (st != SHP_OK) {
        return st;
    }
    auto side = [](const shp_tensor & c, const shp_tensor & s) {
        auto nb = [](const shp_tensor & t, int d) { return static_cast<int64_t>(t.ne[d] > 1 ? t.nb[d] : 0); };
        return PoolSide{ static_cast<char *>(c.data), static_cast<float *>(s.data), nb(c, 3), nb(c, 2), nb(s, 1) / 4 };
    };
    p.side[0] = side(*k, *ks);
    p.side[1] = side(*v, *vs);
    p.pages   = static_cast<int32_t>(k->ne[3]);
    p.shift   = page_shift(k->ne[1]);
    p.hd      = static_cast<int32_t>(k->ne[0]);
    p.kv      = static_cast<int32_t>(k->ne[2]);
    return SHP_OK;
}

// An I32 [ne0, n] of rows.
inline bool numbers2(const shp_tensor * t, int64_t n) {
    return well_formed(t) && t->type == SHP_TYPE_I32 && t->ne[1] == n && t->ne[2] == 1 && t->ne[3] == 1;
}

inline bool numbers2_usable(const shp_tensor & t) {
    return i32_aligned(t) && kv_addressable(t);
}

// Tables of n sequences, for pages of `page` rows.
inline shp_status_t check_table(const shp_tensor * t, int64_t n, int64_t page, Tables & out) {
    if (!numbers2(t, n)) {
        return SHP_ERR_INVALID_ARG;
    }
    if (!numbers2_usable(*t) || n > kKvMaxSeqs || t->ne[0] > (int64_t{ 1 } << 30) / page) {
        return SHP_ERR_UNSUPPORTED;
    }
    out.data = static_cast<const char *>(t->data);
    out.tn   = n > 1 ? static_cast<int64_t>(t->nb[1]) : 0;
    out.most = static_cast<int32_t>(t->ne[0]);
    out.cap  = static_cast<int32_t>(t->ne[0] * page);
    return SHP_OK;
}

}  // namespace shp
