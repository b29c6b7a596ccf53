// The paged KV cache: tables and slots from lengths (shp_kv_pages, shp_kv_slots),
// and its rows, written and read back (shp_kv_store_pages, shp_kv_load_pages).
#include <cmath>

#include "shp_pages.hpp"

namespace shp {
namespace {

// ---------------------------------------------------------------------------
// Tables. With b_n = max(held_n - need_n, 0) pages to give back and t_n =
// max(need_n - held_n, 0) to take, R and A their sums and i and k numbering the
// pages of all sequences in ascending order,
//   the page of number i goes to  free[left + R - 1 - i],
//   the page of number k is       free[left + R - 1 - k],
// which is a stack's push of every i from the last down and pop of every k from the
// first up: the page taken as number j is the one given back as number j, and past R, or
// left over past A, one of the stack. So every j is moved by itself, and only the
// sums before each sequence follow each other; a page finds its sequence among them
// by bisection. Bound by latency: a step of 64 streams is one kernel of 3.7 us (MI355X), and
// one of 2048 requests that gives back or takes 21 thousand pages two, of 4.8 and 6.8 us.
// ---------------------------------------------------------------------------

constexpr int kStepEach = 4;  // sequences of a thread at a time

struct StepArgs {
    const int32_t * length;
    int32_t *       held;
    int32_t *       free;
    int32_t *       left;
    int32_t *       work;    // k_pages_sums and on: back[N + 1], take[N + 1], {ok, left}
    int32_t *       status;  // or null
    Tables          tables;
    int32_t         N;
    int32_t         pages;
    int32_t         shift;
};

__device__ __forceinline__ int32_t pages_of(const StepArgs & a, int32_t length) {
    return (length >> a.shift) + ((length & ((1 << a.shift) - 1)) != 0 ? 1 : 0);
}

// The sum of a wave's lanes up to and with this one, of numbers below 2^48.
__device__ __forceinline__ int64_t wave_sum_up_to(int64_t v) {
    const int32_t low  = sum_up_to(static_cast<int32_t>(v & 0xffff));
    const int32_t mid  = sum_up_to(static_cast<int32_t>(v >> 16 & 0xffff));
    const int32_t high = sum_up_to(static_cast<int32_t>(v >> 32));
    return low + (static_cast<int64_t>(mid) << 16) + (static_cast<int64_t>(high) << 32);
}

// What kStepEach sequences from n0 on give back, take and need.
struct StepPart {
    int32_t back[kStepEach], take[kStepEach], need[kStepEach];
    int64_t all_back, all_take;
    bool    bad;
};

__device__ __forceinline__ StepPart step_part(const StepArgs & a, int n0) {
    StepPart p{};
    int32_t  lengths[kStepEach], helds[kStepEach];
#pragma unroll
    for (int k = 0; k < kStepEach; ++k) {  // (no branch around the loads: all of them are on their way at once)
        lengths[k] = a.length[min(n0 + k, a.N - 1)];
        helds[k]   = a.held[min(n0 + k, a.N - 1)];
    }
#pragma unroll
    for (int k = 0; k < kStepEach; ++k) {
        const int32_t length = n0 + k < a.N ? lengths[k] : 0;
        const int32_t held   = n0 + k < a.N ? helds[k] : 0;
        const int32_t need   = pages_of(a, max(length, 0));
        p.bad                = p.bad || length < 0 || need > a.tables.most || held < 0 || held > a.tables.most;
        p.back[k]            = max(held, need) - need;  // (of any held and need within the table)
        p.take[k]            = max(held, need) - held;
        p.need[k]            = need;
        p.all_back += p.back[k];
        p.all_take += p.take[k];
    }
    return p;
}

// back and take of the sequences from n0 on, with b and t pages before them (past
// int32 only in a step that is refused).
__device__ __forceinline__ void keep_part(const StepArgs & a, const StepPart & p, int n0, int64_t b, int64_t t, int32_t * back,
                                          int32_t * take, int32_t * need) {
#pragma unroll
    for (int k = 0; k < kStepEach; ++k) {
        if (n0 + k < a.N) {
            back[n0 + k] = static_cast<int32_t>(b);
            take[n0 + k] = static_cast<int32_t>(t);
            if (need != nullptr) {
                need[n0 + k] = p.need[k];
            }
        }
        b += p.back[k];
        t += p.take[k];
    }
}

// One workgroup of THREADS: back[n] and take[n], the pages of the sequences before n, and
// in [N] all of them; need[n], where that is not null, those that n is to have. False where
// the step cannot be made. `left` is the stack's.
template <int THREADS>
__device__ __forceinline__ bool step_sums(const StepArgs & a, int32_t * back, int32_t * take, int32_t * need, int32_t left) {
    constexpr int      WAVES = THREADS / kWave;
    __shared__ int64_t sums[2][WAVES];
    __shared__ int32_t fits;
    const int tid  = threadIdx.x;
    const int wave = tid / kWave;
    auto      can  = [&](int64_t b, int64_t t) { return left >= 0 && left + b <= a.pages && t <= left + b; };
    if (a.N <= kWave * kStepEach) {  // one wave has all of them
        if (wave == 0) {
            const int      n0  = tid * kStepEach;
            const StepPart p   = step_part(a, n0);
            const int64_t  b   = wave_sum_up_to(p.all_back), t = wave_sum_up_to(p.all_take);
            const bool     bad = __any(p.bad);
            keep_part(a, p, n0, b - p.all_back, t - p.all_take, back, take, need);
            if (tid == kWave - 1) {
                back[a.N] = static_cast<int32_t>(b);
                take[a.N] = static_cast<int32_t>(t);
                fits      = !bad && can(b, t);
            }
        }
        __syncthreads();
        return fits != 0;
    }
    int64_t all_b = 0, all_t = 0;
    for (int first = 0; first < a.N; first += THREADS * kStepEach) {
        const int      n0 = first + tid * kStepEach;
        const StepPart p  = step_part(a, n0);
        if (__syncthreads_or(p.bad)) {
            return false;
        }
        int64_t b = wave_sum_up_to(p.all_back), t = wave_sum_up_to(p.all_take);
        if (tid % kWave == kWave - 1) {
            sums[0][wave] = b;
            sums[1][wave] = t;
        }
        __syncthreads();
        b += all_b - p.all_back;
        t += all_t - p.all_take;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            b += w < wave ? sums[0][w] : 0;
            t += w < wave ? sums[1][w] : 0;
            all_b += sums[0][w];
            all_t += sums[1][w];
        }
        keep_part(a, p, n0, b, t, back, take, need);
    }
    if (tid == 0) {
        back[a.N] = static_cast<int32_t>(all_b);
        take[a.N] = static_cast<int32_t>(all_t);
    }
    __syncthreads();
    return can(all_b, all_t);
}

// The sequence that page `i` is of.
__device__ __forceinline__ int sequence_of(const int32_t * sums, int n, int32_t i) {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] <= i) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__device__ __forceinline__ int32_t * table_to(const StepArgs & a, int n) {
    return const_cast<int32_t *>(table_of(a.tables, n));
}

// Page number j of those given back, of those taken, or both.
__device__ __forceinline__ void move_page(const StepArgs & a, const int32_t * back, const int32_t * take, const int32_t * need,
                                          int32_t left, int32_t j) {
    const int32_t all   = back[a.N];
    const bool    from  = j < all;
    const bool    to    = j < take[a.N];
    const int     nb    = from ? sequence_of(back, a.N, j) : 0;
    const int     nt    = to ? sequence_of(take, a.N, j) : 0;
    int32_t *     stack = a.free + (left + all - 1 - j);
    int32_t *     old   = table_to(a, nb) + need[nb] + (j - back[nb]);
    int32_t *     now   = table_to(a, nt) + need[nt] - (take[nt + 1] - j);
    const int32_t page  = *(from ? old : stack);
    *(to ? now : stack) = page;
    if (from) {
        *old = -1;
    }
}

__device__ __forceinline__ void refuse_step(const StepArgs & a) {
    if (threadIdx.x == 0 && a.status != nullptr) {
        *a.status = 1;
    }
}

// The whole step by one workgroup.
template <int THREADS> __global__ __launch_bounds__(THREADS) void k_pages_step(const StepArgs a) {
    extern __shared__ int32_t offsets[];
    int32_t *     back = offsets;
    int32_t *     take = offsets + a.N + 1;
    int32_t *     need = take + a.N + 1;
    const int32_t left = *a.left;
    if (!step_sums<THREADS>(a, back, take, need, left)) {
        refuse_step(a);
        return;
    }
    const int32_t n = max(back[a.N], take[a.N]);
    for (int32_t j = threadIdx.x; j < n; j += THREADS) {
        move_page(a, back, take, need, left, j);
    }
    for (int i = threadIdx.x; i < a.N; i += THREADS) {
        a.held[i] = need[i];
    }
    if (threadIdx.x == 0) {
        *a.left = left + back[a.N] - take[a.N];
    }
}

constexpr int kMoveThreads = 256;

template <int THREADS> __global__ __launch_bounds__(THREADS) void k_pages_sums(const StepArgs a) {
    int32_t *     back  = a.work;
    int32_t *     take  = a.work + a.N + 1;
    int32_t *     state = take + a.N + 1;
    const int32_t left  = *a.left;
    const bool    ok    = step_sums<THREADS>(a, back, take, nullptr, left);
    if (threadIdx.x == 0) {
        state[0] = ok;
        state[1] = left;
    }
    if (!ok) {
        refuse_step(a);
        return;
    }
    // (every thread has read them)
    for (int n = threadIdx.x; n < a.N; n += THREADS) {
        a.held[n] = pages_of(a, a.length[n]);
    }
    if (threadIdx.x == 0) {
        *a.left = left + back[a.N] - take[a.N];
    }
}

// The pages after k_pages_sums; IN_LDS: what a page's place is found by is read once.
template <bool IN_LDS> __global__ __launch_bounds__(kMoveThreads) void k_pages_move(const StepArgs a) {
    extern __shared__ int32_t offsets[];
    const int32_t * back  = a.work;
    const int32_t * take  = a.work + a.N + 1;
    const int32_t * need  = a.held;
    const int32_t * state = take + a.N + 1;
    const int32_t   left  = state[1];
    const int32_t   n     = state[0] == 0 ? 0 : max(back[a.N], take[a.N]);
    if constexpr (IN_LDS) {
        auto keep = [&](int32_t * to, const int32_t * from, int count) {
            constexpr int kAtOnce = 8;
            for (int i = threadIdx.x; i < count; i += kAtOnce * kMoveThreads) {
                int32_t x[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    x[k] = from[min(i + k * kMoveThreads, count - 1)];
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    if (i + k * kMoveThreads < count) {
                        to[i + k * kMoveThreads] = x[k];
                    }
                }
            }
        };
        keep(offsets, back, 2 * (a.N + 1));
        keep(offsets + 2 * (a.N + 1), need, a.N);
        back = offsets;
        take = offsets + a.N + 1;
        need = take + a.N + 1;
        __syncthreads();
    }
    for (int32_t j = static_cast<int32_t>(blockIdx.x * kMoveThreads + threadIdx.x); j < n; j += static_cast<int32_t>(gridDim.x * kMoveThreads)) {
        move_page(a, back, take, need, left, j);
    }
}

struct SlotArgs {
    Tables          tables;
    const int32_t * length;
    const int32_t * count;  // or null
    char *          slots;
    int64_t         sn;
    int32_t         T;
    int32_t         shift;
};

constexpr int kSlotThreads = 256;
constexpr int kSlotEach    = 4;  // slots of a thread, kSlotThreads apart

__global__ __launch_bounds__(kSlotThreads) void k_kv_slots(const SlotArgs a, int32_t first) {
    const int       n      = blockIdx.y;
    const int32_t   count  = a.count != nullptr ? min(max(a.count[n], 0), a.T) : a.T;
    const int64_t   start  = static_cast<int64_t>(a.length[n]) - count;
    const int32_t * table  = table_of(a.tables, n);
    int32_t *       slots  = reinterpret_cast<int32_t *>(a.slots + n * a.sn);
    const int       t0     = (first + static_cast<int>(blockIdx.x)) * kSlotEach * kSlotThreads + static_cast<int>(threadIdx.x);
    int32_t         page[kSlotEach];
#pragma unroll
    for (int k = 0; k < kSlotEach; ++k) {
        const int     t = t0 + k * kSlotThreads;
        const int64_t p = start + t;
        page[k]         = t < count && p >= 0 && p < a.tables.cap ? table[p >> a.shift] : -1;
    }
#pragma unroll
    for (int k = 0; k < kSlotEach; ++k) {
        const int  t  = t0 + k * kSlotThreads;
        const bool in = page[k] >= 0 && page[k] <= INT32_MAX >> a.shift;
        if (t < a.T) {
            slots[t] = in ? (page[k] << a.shift) + static_cast<int32_t>((start + t) & ((1 << a.shift) - 1)) : -1;
        }
    }
}

// ---------------------------------------------------------------------------
// Rows. A workgroup writes one block: its new rows' magnitudes, the scale, the codes
// into LDS in the block's layout, and 16 bytes of the block a thread from there,
// over what the block holds where that stays. 8192 rows of 8 heads of 128 values are stored
// in 21 us (MI355X) and read back in 13.6: 4.7 TB/s of what the two have to move.
// ---------------------------------------------------------------------------

constexpr int kRowThreads = 256;
constexpr int kHeld       = 8;  // float4 of the rows that a thread keeps between its two passes over them

struct RowArgs {
    Pool            pool;
    Tables          tables;  // (the load: slots)
    char *          x[2];
    int64_t         xh[2], xt[2], xn[2];
    const int32_t * length;
    const int32_t * count;   // or null
    int32_t *       status;  // or null
    int32_t         T;
    FastDiv         fkv;
    FastDiv         fquads;  // hd / 4
};

// Bytes from one column of V to the next in LDS: off the banks' period.
__host__ __device__ constexpr int column_bytes(int page) {
    return page + 4;
}

__device__ __forceinline__ uint32_t code_byte(float v, float d) {
    const float c = fminf(fmaxf(rintf(v / d), -127.0f), 127.0f);
    return static_cast<uint32_t>(static_cast<int>(c)) & 0xffu;
}

// Byte b of a word of codes under a scale `by` times as large.
__device__ __forceinline__ uint32_t recode_byte(uint32_t w, int b, float by) {
    const float c = static_cast<float>(static_cast<int8_t>(w >> (8 * b)));
    return (static_cast<uint32_t>(static_cast<int>(rintf(c * by))) & 0xffu) << (8 * b);
}

__device__ __forceinline__ uint32_t recode(uint32_t w, float by) {
    return recode_byte(w, 0, by) | recode_byte(w, 1, by) | recode_byte(w, 2, by) | recode_byte(w, 3, by);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kRowThreads) void k_kv_store_pages(const RowArgs a) {
    extern __shared__ __align__(16) char made[];
    __shared__ uint32_t tops[kRowThreads / kWave];
    const int     tid    = threadIdx.x;
    const int     n      = blockIdx.y;
    const int     side   = blockIdx.z;
    const int32_t count  = a.count != nullptr ? a.count[n] : a.T;
    const int32_t length = a.length[n];
    if (count == 0) {
        return;
    }
    const int       shift = a.pool.shift;
    const int       page  = 1 << shift;
    const int       hd    = a.pool.hd;
    const int32_t * table = table_of(a.tables, n);
    bool            bad   = count < 0 || count > a.T || length < count || length > a.tables.cap;
    const int32_t   start = bad ? 0 : length - count;
    const int32_t   first = start >> shift;
    const int32_t   last  = bad ? -1 : (length - 1) >> shift;
    for (int32_t i = first + tid; i <= last; i += kRowThreads) {
        bad = bad || static_cast<uint32_t>(table[i]) >= static_cast<uint32_t>(a.pool.pages);
    }
    bad                 = __syncthreads_or(bad);
    const int     unit  = static_cast<int>(fastdiv(blockIdx.x, a.fkv));
    const int     h     = static_cast<int>(blockIdx.x) - unit * a.pool.kv;
    if (bad) {
        if (a.status != nullptr && blockIdx.x == 0 && side == 0 && tid == 0) {
            *a.status = 1;
        }
        return;
    }
    const int32_t i = first + unit;
    if (i > last) {
        return;
    }
    const PoolSide & s     = a.pool.side[side];
    const int32_t    id    = table[i];
    char *           block = s.codes + id * s.cp + h * s.ch;
    float *          scale = s.scale + id * s.sp + h;
    const int        r0    = max(start - (i << shift), 0);
    const int        r1    = min(length - (i << shift), page);
    const float      d_old = block_scale(*scale);
    // row r0 + k of the block is row t0 + k of the call
    const int32_t t0    = (i << shift) + r0 - start;
    const char *  x     = a.x[side] + n * a.xn[side] + h * a.xh[side] + t0 * a.xt[side];
    const int     quads = hd / 4;
    const int     items = (r1 - r0) * quads;
    auto          load  = [&](int it) {
        const int row = static_cast<int>(fastdiv(static_cast<uint32_t>(it), a.fquads));
        return ld_stream4u(reinterpret_cast<const float *>(x + row * a.xt[side]) + 4 * (it - row * quads));
    };
    auto bits = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };  // in the order of magnitudes, a NaN the largest
    f32x4    held[kHeld];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int it = tid + k * kRowThreads;
        held[k]      = it < items ? load(it) : splat4(0.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            top = max(top, bits(held[k][e]));
        }
    }
    for (int it = tid + kHeld * kRowThreads; it < items; it += kRowThreads) {
        const f32x4 v = load(it);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            top = max(top, bits(v[e]));
        }
    }
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off)));
    }
    if (tid % kWave == 0) {
        tops[tid / kWave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRowThreads / kWave; ++w) {
        top = max(top, tops[w]);
    }
    const bool  had  = r0 > 0;
    const bool  nan  = top >= 0x7f800000u || (had && !(d_old >= 0.0f));
    const float mine = __uint_as_float(top) * (1.0f / 127.0f);
    const float d    = nan ? NAN : had ? fmaxf(d_old, mine) : mine;
    const bool  grew = !nan && had && d > d_old;
    const float by   = grew ? d_old / d : 1.0f;
    auto        put  = [&](int it, const f32x4 & v) {
        const int row  = static_cast<int>(fastdiv(static_cast<uint32_t>(it), a.fquads));
        const int quad = it - row * quads;
        uint32_t  c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = nan || d == 0.0f ? 0u : code_byte(v[e], d);
        }
        if (side == 0) {
            reinterpret_cast<uint32_t *>(made)[(r0 + row) * quads + quad] = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                made[(4 * quad + e) * column_bytes(page) + r0 + row] = static_cast<char>(c[e]);
            }
        }
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        if (tid + k * kRowThreads < items) {
            put(tid + k * kRowThreads, held[k]);
        }
    }
    for (int it = tid + kHeld * kRowThreads; it < items; it += kRowThreads) {
        put(it, load(it));
    }
    __syncthreads();
    if (tid == 0) {
        *scale = d;
    }
    const int from = grew ? 0 : r0;  // the first row whose codes change
    if (side == 0) {
        u32x4 * out = reinterpret_cast<u32x4 *>(block);
        const int per = hd / 16;
        for (int c = from * per + tid; c < r0 * per; c += kRowThreads) {
            u32x4 w = out[c];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = recode(w[e], by);
            }
            out[c] = w;
        }
        for (int c = r0 * per + tid; c < r1 * per; c += kRowThreads) {
            out[c] = reinterpret_cast<const u32x4 *>(made)[c];
        }
    } else {
        const int g0 = from / kGroup;
        const int ng = (r1 - 1) / kGroup - g0 + 1;
        for (int c = tid; c < hd * ng; c += kRowThreads) {
            const int dim = c / ng;
            const int at  = (g0 + c - dim * ng) * kGroup;  // the first of sixteen rows
            u32x4 *   out = reinterpret_cast<u32x4 *>(block + dim * page + at);
            u32x4     w{};
            const uint32_t * codes = reinterpret_cast<const uint32_t *>(made + dim * column_bytes(page) + at);
            if (at >= r0 && at + kGroup <= r1) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = codes[e];
                }
            } else {
                w = *out;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t now = codes[e];
                    const uint32_t was = recode(w[e], by);
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int      r    = at + 4 * e + b;
                        const uint32_t mask = 0xffu << (8 * b);
                        w[e] = (w[e] & ~mask) | ((r < r0 ? was : r < r1 ? now : w[e]) & mask);
                    }
                }
            }
            *out = w;
        }
    }
}

constexpr int kLoadRows = 64;

// 64 rows of one head: K's as they lie, V's columns turned through LDS.
__global__ __launch_bounds__(kRowThreads) void k_kv_load_pages(const RowArgs a) {
    extern __shared__ __align__(16) char rows[];
    __shared__ int32_t     slot[kLoadRows];
    __shared__ float       scale[kLoadRows];
    const int        tid  = threadIdx.x;
    const int        n    = blockIdx.y;
    const int        side = blockIdx.z;
    const int        tile = static_cast<int>(fastdiv(blockIdx.x, a.fkv));
    const int        h    = static_cast<int>(blockIdx.x) - tile * a.pool.kv;
    const int        hd   = a.pool.hd;
    const int        page = 1 << a.pool.shift;
    const PoolSide & s    = a.pool.side[side];
    if (tid < kLoadRows) {
        const int     t  = tile * kLoadRows + tid;
        const int32_t at = t < a.T ? table_of(a.tables, n)[t] : -1;
        const bool    in = at >= 0 && at >> a.pool.shift < a.pool.pages;
        slot[tid]        = at;
        scale[tid]       = in ? block_scale(s.scale[(at >> a.pool.shift) * s.sp + h]) : NAN;
    }
    __syncthreads();
    auto in_pool = [&](int32_t at) { return at >= 0 && at >> a.pool.shift < a.pool.pages; };
    auto block   = [&](int32_t at) { return s.codes + (at >> a.pool.shift) * s.cp + h * s.ch; };
    const int stride = hd + 4;
    if (side == 1) {
        const int     row = tid % kLoadRows;
        const int32_t at  = slot[row];
        if (in_pool(at)) {
            const char * from = block(at) + (at & (page - 1));
            for (int dim = tid / kLoadRows; dim < hd; dim += kRowThreads / kLoadRows) {
                rows[row * stride + dim] = from[dim * page];
            }
        }
        __syncthreads();
    }
    const int quads = hd / 4;
    char *    x     = a.x[side] + n * a.xn[side] + h * a.xh[side] + static_cast<int64_t>(tile) * kLoadRows * a.xt[side];
    for (int it = tid; it < kLoadRows * quads; it += kRowThreads) {
        const int     row  = static_cast<int>(fastdiv(static_cast<uint32_t>(it), a.fquads));
        const int     quad = it - row * quads;
        const int32_t at   = slot[row];
        if (at == -1) {
            continue;
        }
        uint32_t w = 0;
        if (in_pool(at)) {
            const char * from = side == 0 ? block(at) + (at & (page - 1)) * hd : rows + row * stride;
            w                 = reinterpret_cast<const uint32_t *>(from)[quad];
        }
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = static_cast<float>(static_cast<int8_t>(w >> (8 * e))) * scale[row];
        }
        st_stream4u(reinterpret_cast<float *>(x + row * a.xt[side]) + 4 * quad, v);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// One workgroup makes the step where its sums fit LDS and few table entries can change.
constexpr int64_t kStepSeqs    = 4096;
constexpr int64_t kStepEntries = int64_t{ 1 } << 16;
constexpr int64_t kSmallEntries = 4096;
constexpr int     kMoveGroups  = 128;  // (2048 requests, 10 to 20 thousand pages: 26.1 us the case, with 64 28.2, with 256 26.4)

bool one_group(const shp_tensor & table) {
    return table.ne[1] <= kStepSeqs && table.ne[0] * table.ne[1] <= kStepEntries;
}

int64_t step_ints(const shp_tensor & table) {
    return one_group(table) ? 0 : 2 * (table.ne[1] + 1) + 2;
}

// Whether t, of ne0 I32, is usable.
shp_status_t check_numbers(const shp_tensor * t, int64_t ne0) {
    return !kv_numbers(t, ne0) ? SHP_ERR_INVALID_ARG : i32_aligned(*t) ? SHP_OK : SHP_ERR_UNSUPPORTED;
}

// No two of them share bytes, and no rows of one do.
bool apart(std::initializer_list<const shp_tensor *> written, std::initializer_list<const shp_tensor *> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        if (*w == nullptr) {
            continue;
        }
        if (!kv_rows_apart(**w)) {
            return false;
        }
        for (auto o = w + 1; o != written.end(); ++o) {
            if (*o != nullptr && kv_overlap(**w, **o)) {
                return false;
            }
        }
        for (const shp_tensor * r : read) {
            if (r != nullptr && kv_overlap(**w, *r)) {
                return false;
            }
        }
    }
    return true;
}

// k and v, F32 [hd, kv, T, N], and the strides of both.
shp_status_t check_rows(const shp_tensor * k, const shp_tensor * v, const Pool & p, RowArgs & a) {
    if (!well_formed(k) || !well_formed(v) || !same_shape(*k, *v) || k->ne[0] != p.hd || k->ne[1] != p.kv) {
        return SHP_ERR_INVALID_ARG;
    }
    const int64_t pieces = (k->ne[0] + kKvBlock - 1) / kKvBlock;
    if (k->type != SHP_TYPE_F32 || v->type != SHP_TYPE_F32 || !kv_aligned(*k) || !kv_aligned(*v) || !kv_addressable(*k) ||
        !kv_addressable(*v) || k->ne[3] > kKvMaxSeqs || k->ne[1] > kKvMaxRows / pieces ||
        k->ne[2] > kKvMaxRows / (k->ne[1] * pieces)) {
        return SHP_ERR_UNSUPPORTED;
    }
    auto nb = [](const shp_tensor & t, int d) { return static_cast<int64_t>(t.ne[d] > 1 ? t.nb[d] : 0); };
    int  i  = 0;
    for (const shp_tensor * t : { k, v }) {
        a.x[i]  = static_cast<char *>(t->data);
        a.xh[i] = nb(*t, 1);
        a.xt[i] = nb(*t, 2);
        a.xn[i] = nb(*t, 3);
        ++i;
    }
    a.pool   = p;
    a.T      = static_cast<int32_t>(k->ne[2]);
    a.fkv    = make_fastdiv(static_cast<uint32_t>(p.kv));
    a.fquads = make_fastdiv(static_cast<uint32_t>(p.hd / 4));
    return SHP_OK;
}

}  // namespace
}  // namespace shp

using namespace shp;

extern "C" shp_status_t shp_kv_pages_work(const shp_tensor * table, int64_t * ints) {
    if (ints == nullptr || !well_formed(table)) {
        return SHP_ERR_INVALID_ARG;
    }
    Tables             t{};
    const shp_status_t st = check_table(table, table->ne[1], 1, t);
    if (st == SHP_OK) {
        *ints = step_ints(*table);
    }
    return st;
}

extern "C" shp_status_t shp_kv_pages(const shp_tensor * length,
                                     int32_t            page,
                                     shp_tensor *       held,
                                     shp_tensor *       free_pages,
                                     shp_tensor *       left,
                                     shp_tensor *       table,
                                     shp_tensor *       work,
                                     shp_tensor *       status,
                                     shp_stream_t       stream) {
    if (!well_formed(length) || !well_formed(free_pages)) {
        return SHP_ERR_INVALID_ARG;
    }
    StepArgs      a{};
    const int64_t n = length->ne[0];
    if (page_shift(page) < 0) {
        return SHP_ERR_UNSUPPORTED;
    }
    shp_status_t st = check_table(table, n, page, a.tables);
    for (const shp_tensor * t : { static_cast<const shp_tensor *>(length), static_cast<const shp_tensor *>(held) }) {
        st = st == SHP_OK ? check_numbers(t, n) : st;
    }
    st = st == SHP_OK ? check_numbers(free_pages, free_pages->ne[0]) : st;
    st = st == SHP_OK ? check_numbers(left, 1) : st;
    st = st == SHP_OK && status != nullptr ? check_numbers(status, 1) : st;
    if (st != SHP_OK) {
        return st;
    }
    const int64_t ints = step_ints(*table);
    if (ints > 0 && (!well_formed(work) || work->type != SHP_TYPE_I32 || !contiguous(*work) || nelements(*work) < ints)) {
        return SHP_ERR_INVALID_ARG;
    }
    if (free_pages->ne[0] > INT32_MAX / page || (ints > 0 && !i32_aligned(*work)) ||
        !apart({ held, free_pages, left, table, ints > 0 ? work : nullptr, status }, { length })) {
        return SHP_ERR_UNSUPPORTED;
    }
    if (dry_run()) {
        return SHP_OK;
    }
    a.length = static_cast<const int32_t *>(length->data);
    a.held   = static_cast<int32_t *>(held->data);
    a.free   = static_cast<int32_t *>(free_pages->data);
    a.left   = static_cast<int32_t *>(left->data);
    a.work   = ints > 0 ? static_cast<int32_t *>(work->data) : nullptr;
    a.status = status != nullptr ? static_cast<int32_t *>(status->data) : nullptr;
    a.N      = static_cast<int32_t>(n);
    a.pages  = static_cast<int32_t>(free_pages->ne[0]);
    a.shift  = page_shift(page);
    const hipStream_t s   = as_stream(stream);
    const size_t      lds = static_cast<size_t>(3 * n + 2) * 4;
    if (ints == 0) {
        if (table->ne[0] * n <= kSmallEntries) {
            hipLaunchKernelGGL(k_pages_step<256>, dim3(1), dim3(256), lds, s, a);
        } else {
            hipLaunchKernelGGL(k_pages_step<1024>, dim3(1), dim3(1024), lds, s, a);
        }
        return launch_status();
    }
    if (n <= 512 * kStepEach) {
        hipLaunchKernelGGL(k_pages_sums<512>, dim3(1), dim3(512), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_pages_sums<1024>, dim3(1), dim3(1024), 0, s, a);
    }
    st = launch_status();
    if (st != SHP_OK) {
        return st;
    }
    if (n <= kStepSeqs) {
        hipLaunchKernelGGL(k_pages_move<true>, dim3(kMoveGroups), dim3(kMoveThreads), lds, s, a);
    } else {
        hipLaunchKernelGGL(k_pages_move<false>, dim3(kMoveGroups), dim3(kMoveThreads), 0, s, a);
    }
    return launch_status();
}

extern "C" shp_status_t shp_kv_slots(const shp_tensor * table,
                                     const shp_tensor * length,
                                     const shp_tensor * count,
                                     int32_t            page,
                                     shp_tensor *       slots,
                                     shp_stream_t       stream) {
    if (!well_formed(length)) {
        return SHP_ERR_INVALID_ARG;
    }
    SlotArgs      a{};
    const int64_t n = length->ne[0];
    if (page_shift(page) < 0) {
        return SHP_ERR_UNSUPPORTED;
    }
    shp_status_t st = check_table(table, n, page, a.tables);
    st              = st == SHP_OK ? check_numbers(length, n) : st;
    st              = st == SHP_OK && count != nullptr ? check_numbers(count, n) : st;
    if (st == SHP_OK && !numbers2(slots, n)) {
        st = SHP_ERR_INVALID_ARG;
    }
    if (st != SHP_OK) {
        return st;
    }
    if (!numbers2_usable(*slots) || slots->ne[0] > kKvMaxRows || !apart({ slots }, { table, length, count })) {
        return SHP_ERR_UNSUPPORTED;
    }
    if (dry_run()) {
        return SHP_OK;
    }
    a.length = static_cast<const int32_t *>(length->data);
    a.count  = count != nullptr ? static_cast<const int32_t *>(count->data) : nullptr;
    a.slots  = static_cast<char *>(slots->data);
    a.sn     = n > 1 ? static_cast<int64_t>(slots->nb[1]) : 0;
    a.T      = static_cast<int32_t>(slots->ne[0]);
    a.shift  = page_shift(page);
    const hipStream_t s = as_stream(stream);
    constexpr int64_t kEach = int64_t{ kSlotEach } * kSlotThreads;
    return in_launches((a.T + kEach - 1) / kEach, kSlotThreads, [&](int64_t first, dim3 grid) {
        hipLaunchKernelGGL(k_kv_slots, dim3(grid.x, static_cast<unsigned>(n)), dim3(kSlotThreads), 0, s, a, static_cast<int32_t>(first));
    });
}

extern "C" shp_status_t shp_kv_store_pages(const shp_tensor * k,
                                           const shp_tensor * v,
                                           const shp_tensor * table,
                                           const shp_tensor * length,
                                           const shp_tensor * count,
                                           shp_tensor *       k_pages,
                                           shp_tensor *       v_pages,
                                           shp_tensor *       k_scale,
                                           shp_tensor *       v_scale,
                                           shp_tensor *       status,
                                           shp_stream_t       stream) {
    RowArgs      a{};
    Pool         p{};
    shp_status_t st = check_pool(k_pages, v_pages, k_scale, v_scale, p);
    st              = st == SHP_OK ? check_rows(k, v, p, a) : st;
    if (st != SHP_OK) {
        return st;
    }
    const int64_t n    = k->ne[3];
    const int64_t page = k_pages->ne[1];
    st                 = check_table(table, n, page, a.tables);
    st                 = st == SHP_OK ? check_numbers(length, n) : st;
    st                 = st == SHP_OK && count != nullptr ? check_numbers(count, n) : st;
    st                 = st == SHP_OK && status != nullptr ? check_numbers(status, 1) : st;
    if (st != SHP_OK) {
        return st;
    }
    const shp_tensor kr = codes_as_rows(*k_pages), vr = codes_as_rows(*v_pages);
    const int64_t    units = (k->ne[2] + page - 2) / page + 1;
    if (!apart({ &kr, &vr, k_scale, v_scale, status }, { k, v, table, length, count }) ||
        units > (int64_t{ UINT32_MAX } / kRowThreads) / p.kv) {
        return SHP_ERR_UNSUPPORTED;
    }
    if (dry_run()) {
        return SHP_OK;
    }
    a.length = static_cast<const int32_t *>(length->data);
    a.count  = count != nullptr ? static_cast<const int32_t *>(count->data) : nullptr;
    a.status = status != nullptr ? static_cast<int32_t *>(status->data) : nullptr;
    const dim3   grid(static_cast<unsigned>(units * p.kv), static_cast<unsigned>(n), 2);
    const size_t lds = static_cast<size_t>(p.hd) * static_cast<size_t>(column_bytes(static_cast<int>(page)));
    hipLaunchKernelGGL(k_kv_store_pages, grid, dim3(kRowThreads), lds, as_stream(stream), a);
    return launch_status();
}

extern "C" shp_status_t shp_kv_load_pages(const shp_tensor * k_pages,
                                          const shp_tensor * v_pages,
                                          const shp_tensor * k_scale,
                                          const shp_tensor * v_scale,
                                          const shp_tensor * slots,
                                          shp_tensor *       k,
                                          shp_tensor *       v,
                                          shp_stream_t       stream) {
    RowArgs      a{};
    Pool         p{};
    shp_status_t st = check_pool(k_pages, v_pages, k_scale, v_scale, p);
    st              = st == SHP_OK ? check_rows(k, v, p, a) : st;
    if (st != SHP_OK) {
        return st;
    }
    const int64_t n = k->ne[3];
    if (!numbers2(slots, n) || slots->ne[0] != k->ne[2]) {
        return SHP_ERR_INVALID_ARG;
    }
    const shp_tensor kr = codes_as_rows(*k_pages), vr = codes_as_rows(*v_pages);
    if (!numbers2_usable(*slots) || !apart({ k, v }, { &kr, &vr, k_scale, v_scale, slots })) {
        return SHP_ERR_UNSUPPORTED;
    }
    if (dry_run()) {
        return SHP_OK;
    }
    a.tables.data = static_cast<const char *>(slots->data);
    a.tables.tn   = n > 1 ? static_cast<int64_t>(slots->nb[1]) : 0;
    const int64_t tiles = (k->ne[2] + kLoadRows - 1) / kLoadRows;
    const dim3    grid(static_cast<unsigned>(tiles * p.kv), static_cast<unsigned>(n), 2);
    hipLaunchKernelGGL(k_kv_load_pages, grid, dim3(kRowThreads), kLoadRows * (p.hd + 4), as_stream(stream), a);
    return launch_status();
}
