// ============================================================================
//  attend.hip — attention of new tokens over the paged cache (mars_kv_attend).
//
//  Both products run on MFMA with the queries as columns: S^T = K Q^T, then O^T = V^T P^T.
//  A lane then holds the scores of one query row (its column), the row's statistics are one
//  value per lane, and the accumulator of S^T is, unchanged, the second product's operand
//  P^T: the keys of a step are dealt to the rows of the first product so that a lane's
//  scores are those of 8 consecutive keys, and V^T's fragment of 8 consecutive keys is one
//  16-byte load from the cache (which keeps v with the tokens of an element side by side).
//
//  Rows: the new tokens of a request times the query heads of one kv head, token-major;
//  all read the same keys and values.
//
//  Softmax in base 2 (log2 e is folded into the scale), one pass: each row has a reference
//  m and sums exp2(s - m), fp32. m moves only when a score exceeds it by more than 8 (in a
//  wave of rows together): exp2 stays below 2^8, exact in 16-bit range, and the usual step
//  needs no lane exchange and no rescaling of O.
// ============================================================================
#include "reader.hpp"

#include <algorithm>
#include <cmath>

namespace mars {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0.69314718055994530942f;
// s_waitcnt immediate (gfx9 encoding: vmcnt[3:0] and [15:14], expcnt[6:4], lgkmcnt[11:8]): all loads, or all LDS accesses, done
constexpr int kWaitVm0 = (7 << 4) | (15 << 8);
constexpr int kWaitLgkm0 = 15 | (3 << 14) | (7 << 4);
constexpr float kSlack = 8.0f;       // how far a score may exceed the row's reference

// Every load of this wave is done (LDS ones too), and every other wave got here.
__device__ inline void tile_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Every LDS access of this wave is done, and every other wave got here.
__device__ inline void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 16 (or 4) bytes per lane from global memory straight into LDS: lane l's go to lds + 16 l (4 l) bytes.
__device__ inline void dma16(const void* g, void* lds) { __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0); }
__device__ inline void dma4(const void* g, void* lds) { __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 4, 0, 0); }

template <typename T> struct Vec;
template <> struct Vec<_Float16> {
    using v8 = f16x8;
    using v4 = f16x4;
    static constexpr uint32_t exp_mask = 0x7C00u, one = 0x3C00u;
    __device__ static f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    __device__ static f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Vec<__bf16> {
    using v8 = bf16x8;
    using v4 = bf16x4;
    static constexpr uint32_t exp_mask = 0x7F80u, one = 0x3F80u;
    __device__ static f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ static f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

template <typename V>
__device__ inline V load16(const void* p) {
    return __builtin_bit_cast(V, *static_cast<const u32x4*>(p));
}
// 16 bytes of q, its sign turned where the scale is negative.
template <typename V>
__device__ inline V load_q(const void* p, uint32_t flip) {
    return __builtin_bit_cast(V, *static_cast<const u32x4*>(p) ^ flip);
}

// Of 8 values: nonzero if one of them is an infinity or NaN; the values with those replaced by 0.
template <typename T>
__device__ inline uint32_t exponents_full(u32x4 b) {
    constexpr uint32_t E = Vec<T>::exp_mask, E2 = E | (E << 16), B2 = ((0x8000u - E) << 16) | (0x8000u - E);
    return (((b[0] & E2) + B2) | ((b[1] & E2) + B2) | ((b[2] & E2) + B2) | ((b[3] & E2) + B2)) & 0x80008000u;
}
template <typename T>
__device__ inline u32x4 finite_part(u32x4 b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = b[j] & 0xFFFFu, hi = b[j] >> 16;
        if ((lo & Vec<T>::exp_mask) == Vec<T>::exp_mask) b[j] &= 0xFFFF0000u;
        if ((hi & Vec<T>::exp_mask) == Vec<T>::exp_mask) b[j] &= 0xFFFFu;
    }
    return b;
}

// The table is read with scalar loads (it is constant while the kernel runs): they have a counter of their own, so
// waiting for a page's number does not wait for the tiles in flight.
typedef const __attribute__((address_space(4))) int32_t* TablePtr;
__device__ inline TablePtr table_row(const AttendArgs& a, int request) {
    return (TablePtr)(reinterpret_cast<uintptr_t>(a.table + int64_t(request) * a.max_pages));
}
// The page of uniform key `key`, of a request whose last page is `last`; pages outside the cache count as page 0.
__device__ inline int page_of(const AttendArgs& a, TablePtr table, int key, int last) {
    const int id = table[min(key >> a.page_shift, last)];
    return uint32_t(id) < uint32_t(a.num_pages) ? id : 0;
}

// One unit of a launch's work: a tile of rows of a request under one kv head, over a range of its keys.
struct Item {
    int32_t request, tile, head, split, splits, chunk;
    int32_t part;              // first partial slot of the tile's splits
    int32_t tiles;             // of the request
    bool found;
};

struct SchedLds {
    uint64_t wsum[4];
    Item item;
};

__device__ inline int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor((long long)v, o);
    return v;
}

// Rows of request r that this launch serves, in tiles of `bm`, and its keys.
__device__ inline void request_of(const AttendArgs& a, int r, int bm, int* tiles, int* keys) {
    *tiles = 0;
    *keys = 0;
    if (r >= a.requests) return;
    const int n = max(0, min(a.q_start[r + 1], a.tokens) - max(a.q_start[r], 0));
    const int rows = n * a.group;
    if (rows <= a.rows_lo || rows > a.rows_hi) return;
    *tiles = (rows + bm - 1) / bm;
    *keys = int(min(int64_t(max(a.kv_lens[r], 0)), int64_t(a.max_pages) << a.page_shift));
}

// Workgroup b's item, from the lengths alone: every workgroup of 256 threads sums the launch's work (key steps of 32
// over all tiles), cuts the keys into chunks of work / 2^items_log2, and finds the request that its number falls to. The
// launch has enough workgroups for every item (fewer than 2^31); the last ones may find none.
__device__ Item find_item(const AttendArgs& a, uint32_t b, int bm, int min_chunk, int items_log2, SchedLds& sh) {
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    int tiles0 = 0, keys0 = 0;
    int64_t work = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 256) {
        int tiles, keys;
        request_of(a, r0 + tid, bm, &tiles, &keys);
        if (r0 == 0) { tiles0 = tiles; keys0 = keys; }
        work += int64_t(tiles) * ((keys + 31) >> 5);
    }
    work = wave_sum(work);
    if (lane == 0) sh.wsum[wave] = uint64_t(work);
    if (tid == 0) sh.item.found = false;
    __syncthreads();
    work = int64_t(sh.wsum[0] + sh.wsum[1] + sh.wsum[2] + sh.wsum[3]) * a.kv_heads;
    const int64_t per = (work * 32 + (int64_t(1) << items_log2) - 1) >> items_log2;
    const uint32_t chunk0 = (uint32_t(min(max(per, int64_t(min_chunk)), int64_t(INT32_MAX) - 255)) + 255) & ~255u;
    uint32_t items_before = 0, parts_before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 256) {
        int tiles = tiles0, keys = keys0;
        if (r0) request_of(a, r0 + tid, bm, &tiles, &keys);
        // no more than kMaxSplits chunks a request
        const uint32_t chunk = max(chunk0, (uint32_t(keys) + kMaxSplits * 256 - 1) / (kMaxSplits * 256) * 256);
        const uint32_t splits = max(1u, (uint32_t(keys) + chunk - 1) / chunk);
        const uint32_t items = uint32_t(tiles) * uint32_t(a.kv_heads) * splits, parts = splits > 1 ? items : 0;
        uint32_t xi = items, xp = parts;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t yi = __shfl_up(xi, unsigned(o)), yp = __shfl_up(xp, unsigned(o));
            if (lane >= o) { xi += yi; xp += yp; }
        }
        __syncthreads();
        if (lane == 63) sh.wsum[wave] = (uint64_t(xi) << 32) | xp;
        __syncthreads();
        uint32_t bi = items_before, bp = parts_before;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint64_t s = sh.wsum[w];
            if (w < wave) { bi += uint32_t(s >> 32); bp += uint32_t(s); }
            items_before += uint32_t(s >> 32);
            parts_before += uint32_t(s);
        }
        const uint32_t mine = bi + xi - items;
        if (b >= mine && b - mine < items) {
            const uint32_t local = b - mine, tile_head = local / splits, tile = tile_head / uint32_t(a.kv_heads);
            Item it;
            it.request = r0 + tid;
            it.split = int32_t(local - tile_head * splits);
            it.tile = int32_t(tile);
            it.head = int32_t(tile_head - tile * uint32_t(a.kv_heads));
            it.splits = int32_t(splits);
            it.chunk = int32_t(min(chunk, uint32_t(INT32_MAX / 2)));
            it.part = int32_t(bp + xp - parts + tile_head * splits);
            it.tiles = tiles;
            it.found = true;
            sh.item = it;
        }
        if (b < items_before) break;
    }
    __syncthreads();
    return sh.item;
}

// Partials pass between workgroups of one launch, on any XCD: as relaxed atomics of agent scope, which go through to
// where every XCD sees them, the writers' completed before they count themselves in. (Plain stores and a fence at agent
// scope write back and drop a whole L2 per workgroup: 64 single tokens over 4,096 keys took 497 us so.)
__device__ inline void put_part(float* p, f32x4 v) {
    const u32x4 b = __builtin_bit_cast(u32x4, v);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), uint64_t(b[1]) << 32 | b[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p) + 1, uint64_t(b[3]) << 32 | b[2], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void put_part(float2* p, float2 v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), uint64_t(__float_as_uint(v.y)) << 32 | __float_as_uint(v.x), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline uint64_t get_part(const void* p) {
    return __hip_atomic_load(static_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline f32x4 get_part4(const float* p) {
    const uint64_t lo = get_part(p), hi = get_part(p + 2);
    return __builtin_bit_cast(f32x4, u32x4{uint32_t(lo), uint32_t(lo >> 32), uint32_t(hi), uint32_t(hi >> 32)});
}
__device__ inline float2 get_part2(const float2* p) {
    const uint64_t v = get_part(p);
    return make_float2(__uint_as_float(uint32_t(v)), __uint_as_float(uint32_t(v >> 32)));
}

// Called by every thread of a workgroup that wrote one split's partial: the tile's last workgroup to arrive joins the
// splits. Each sum is taken in the order of the splits by one thread, or, where there are few rows, by up to 8
// threads whose parts are then added in their order: the same bits whoever arrives last.
template <int BM>
struct JoinLds {
    int last;
    float lpart[8][BM];
    __attribute__((aligned(16))) float part[8][128 * 4];     // 256 / ways units each
};
template <typename T, int D, int BM>
__device__ void join_splits(const AttendArgs& a, const Item& it, int row0, int n, JoinLds<BM>& lds) {
    const int tid = int(threadIdx.x);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitVm0);                    // this wave's stores have reached every XCD's view
    __syncthreads();
    if (tid == 0) lds.last = __hip_atomic_fetch_add(&a.arrived[it.part], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(it.splits - 1);
    __syncthreads();
    if (!lds.last) return;
    if (tid == 0) __hip_atomic_store(&a.arrived[it.part], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int valid = min(BM, n * a.group - it.tile * BM), units = valid * (D / 4);
    int ways = 1;                                            // threads per unit of 4 elements
    while (ways < 8 && units * ways * 2 <= 256 && ways < it.splits) ways *= 2;
    const float2* const ml = a.part_ml + int64_t(it.part) * BM;
    const float* const po = a.part_o + int64_t(it.part) * BM * D;
    for (int e0 = 0; e0 < units; e0 += 256 / ways) {
        const int w = tid / (256 / ways), e = e0 + tid % (256 / ways), rr = e / (D / 4), d4 = e % (D / 4);
        f32x4 sum = {0, 0, 0, 0};
        float lsum = 0.0f, top = -kInf;
        if (e < units) {
#pragma unroll 4
            for (int s = 0; s < it.splits; ++s) top = fmaxf(top, get_part2(ml + s * BM + rr).x);
#pragma unroll 4
            for (int s = w; s < it.splits; s += ways) {
                const float2 p = get_part2(ml + s * BM + rr);
                const float f = p.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(p.x - top);
                lsum += f * p.y;
                sum += f * get_part4(po + (int64_t(s) * BM + rr) * D + d4 * 4);
            }
        }
        if (ways > 1) {                                      // units fit one round then
            float* const mine = &lds.part[w][0];
            *reinterpret_cast<f32x4*>(mine + (tid % (256 / ways)) * 4) = sum;
            if (d4 == 0 && e < units) lds.lpart[w][rr] = lsum;
            __syncthreads();
            if (w == 0 && e < units) {
                lsum = 0.0f;
                for (int v = 0; v < ways; ++v) lsum += lds.lpart[v][rr];
                for (int v = 1; v < ways; ++v) sum += *reinterpret_cast<const f32x4*>(&lds.part[v][tid * 4]);
            }
        }
        if (w == 0 && e < units) {
            const int mm = it.tile * BM + rr, ii = mm / a.group, hh = it.head * a.group + mm - ii * a.group;
            const float inv = 1.0f / lsum;
            typename Vec<T>::v4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = top == -kInf ? T(0.0f) : T(sum[j] * inv);
            *reinterpret_cast<typename Vec<T>::v4*>(static_cast<T*>(a.out) + (int64_t(row0) + ii) * a.out_stride + int64_t(hh) * D + d4 * 4) = o;
            if (a.lse && d4 == 0)
                a.lse[(int64_t(row0) + ii) * a.q_heads + hh] = top == -kInf ? -kInf : (top + __builtin_amdgcn_logf(lsum)) * kLn2;
        }
    }
}

// Infinities and NaN among the values. A weight of 0 times one of them is NaN, so where some row of a step does not see
// some key, the products take them as 0, and the workgroup, once its rows are written, adds them to the rows that do see
// them here: every (row, element) looks through the keys [k0, k1). (Rare, and slow.)
template <typename T, int D, int BM>
__device__ void add_not_finite(const AttendArgs& a, const Item& it, int row0, int n, int keys, int prefix, int k0, int k1) {
    const int valid = min(BM, n * a.group - it.tile * BM);
    for (int e = int(threadIdx.x); e < valid * D; e += 256) {
        const int rr = e / D, d = e % D, m = it.tile * BM + rr, i = m / a.group, hq = it.head * a.group + m - i * a.group;
        const int64_t row = int64_t(row0) + i;
        const int end = min(k1, min(max(keys - n + i + 1, prefix), keys));
        float sum = 0.0f;
        for (int k = k0; k < end; ++k) {
            const int id = a.table[int64_t(it.request) * a.max_pages + (k >> a.page_shift)];
            const int64_t page = uint32_t(id) < uint32_t(a.num_pages) ? id : 0;
            const int off = k & ((1 << a.page_shift) - 1);
            if (a.k_eps) {
                const int ek = a.k_eps[(page << a.page_shift) + off], eq = a.q_eps[row];
                if (!(ek < 0 || eq < 0 || ek == eq)) continue;
            }
            const float v = float(static_cast<const T*>(a.v_pages)[page * a.v_stride + ((int64_t(it.head) * D + d) << a.page_shift) + off]);
            if (!(fabsf(v) < kInf)) sum += v;
        }
        if (sum == 0.0f) continue;
        if (it.splits == 1) {
            T* const o = static_cast<T*>(a.out) + row * a.out_stride + int64_t(hq) * D + d;
            *o = T(float(*o) + sum);
        } else {
            float* const o = a.part_o + (int64_t(it.part + it.split) * BM + rr) * D + d;
            const float was = __hip_atomic_load(o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(o, was + sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// ---- few rows: 16 at a time, keys straight from the cache to registers -----------------
// Bound by the cache's bytes. 4 waves take the steps of the chunk in turn (64 keys; 32 for heads of 256), and a wave
// keeps its next step's K and V on the way to registers (16 bytes a lane; whole 128-byte lines, from K rows over the
// elements and from V rows over the step's keys) while it computes this one: 8 waves of a CU have up to 256 KB in
// flight. The waves' sums are joined at the end.
template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void k_attend_few(AttendArgs a) {
    using V = typename Vec<T>::v8;
    constexpr int KC = D / 32, VB = D / 16, NH = D > 128 ? 1 : 2, STEP = 32 * NH;      // NH: halves of 32 keys in a step
    __shared__ union {
        SchedLds sched;
        struct { float ml[4][16][2]; __attribute__((aligned(16))) float ob[2][16][D + 4]; } wave;
        JoinLds<kFewRows> join;
    } lds;
    __shared__ int any_dirty;
    if (threadIdx.x == 0) any_dirty = 0;
    const Item it = find_item(a, blockIdx.x, kFewRows, 256, kFewItemsLog2, lds.sched);
    if (!it.found) return;
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, h = lane >> 4;
    const int r = __builtin_amdgcn_readfirstlane(it.request), head = __builtin_amdgcn_readfirstlane(it.head);
    const int P1 = (1 << a.page_shift) - 1;
    const int row0 = max(a.q_start[r], 0), n = min(a.q_start[r + 1], a.tokens) - row0;
    const int keys = int(min(int64_t(max(a.kv_lens[r], 0)), int64_t(a.max_pages) << a.page_shift));
    const int m = it.tile * kFewRows + col;                 // this lane's row: token i, head of the group
    const bool row_ok = m < n * a.group;
    const int i = row_ok ? m / a.group : 0, hq = head * a.group + (row_ok ? m - i * a.group : 0);
    const int64_t row = int64_t(row0) + i;
    const int prefix = a.prefix ? min(max(a.prefix[r], 0), keys) : 0;
    const int limit = row_ok ? min(max(keys - n + i + 1, prefix), keys) : 0;   // keys [0, limit) may be seen
    const float dec = EXTRA && a.decay ? a.decay[hq] * 1.4426950408889634f : 0.0f;
    const float tq = EXTRA && a.decay ? a.q_times[row] : 0.0f;
    const int eq = EXTRA && a.q_eps ? a.q_eps[row] : -1;

    int lo = row_ok ? limit : INT32_MAX, hi = limit;        // over the rows
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int k0 = __builtin_amdgcn_readfirstlane(it.split * it.chunk), k1 = min(k0 + __builtin_amdgcn_readfirstlane(it.chunk), hi);
    const int steps = k1 > k0 ? (k1 - k0 + STEP - 1) / STEP : 0;

    const TablePtr table = table_row(a, r);
    const int last_page = keys > 0 ? (keys - 1) >> a.page_shift : 0;
    // K: A row `col` of block b holds key 8 (col / 4) + 4 b + col % 4 of 32, so that registers 4 b + j of S hold key 8 h + 4 b + j
    const int kg = col >> 3, kin = 8 * ((col >> 2) & 1) + (col & 3);             // group of 16 keys, key within it (b = 0)
    const T* const kp = static_cast<const T*>(a.k_pages) + ((int64_t(head) << a.page_shift) + kin) * D + h * 8;
    const T* const vp = static_cast<const T*>(a.v_pages) + ((int64_t(head) * D + col) << a.page_shift) + (h & 1) * 8;
    int pages[2 * NH], v_pages[2 * NH];                     // of the step on the way: K's, and (loaded later) V's
    auto find_pages = [&](int s) {
#pragma unroll
        for (int u = 0; u < 2 * NH; ++u) pages[u] = page_of(a, table, k0 + s * STEP + u * 16, last_page);
    };
    V kf[NH][2][KC], vf[NH][VB];
    f32x4 tk[NH][2];
    i32x4 ek[NH][2];
    auto load_k = [&](int s) {
#pragma unroll
        for (int b2 = 0; b2 < NH; ++b2) {
            const int kt = k0 + s * STEP + b2 * 32;
            const int64_t o0 = pages[2 * b2] * a.k_stride + int64_t(kt & P1) * D, o1 = pages[2 * b2 + 1] * a.k_stride + int64_t((kt + 16) & P1) * D;
            const T* const p = kp + (kg ? o1 : o0);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int c = 0; c < KC; ++c) kf[b2][b][c] = load16<V>(p + b * 4 * D + c * 32);
        }
    };
    auto load_v = [&](int s) {
#pragma unroll
        for (int b2 = 0; b2 < NH; ++b2) {
            const int kt = k0 + s * STEP + b2 * 32, a0 = kt & P1, a1 = (kt + 16) & P1;
            const T* const p = vp + (h & 2 ? v_pages[2 * b2 + 1] * a.v_stride + a1 : v_pages[2 * b2] * a.v_stride + a0);
#pragma unroll
            for (int d = 0; d < VB; ++d) vf[b2][d] = load16<V>(p + (int64_t(d) * 16 << a.page_shift));
            const int64_t slot = (int64_t(h & 2 ? v_pages[2 * b2 + 1] : v_pages[2 * b2]) << a.page_shift) + (h & 2 ? a1 : a0) + (h & 1) * 8;
            if (EXTRA && a.k_times) { tk[b2][0] = *reinterpret_cast<const f32x4*>(a.k_times + slot); tk[b2][1] = *reinterpret_cast<const f32x4*>(a.k_times + slot + 4); }
            if (EXTRA && a.k_eps) { ek[b2][0] = *reinterpret_cast<const i32x4*>(a.k_eps + slot); ek[b2][1] = *reinterpret_cast<const i32x4*>(a.k_eps + slot + 4); }
        }
    };

    if (wave < steps) find_pages(wave);
    V q[KC];
    const T* const qp = static_cast<const T*>(a.q) + row * a.q_stride + int64_t(hq) * D + h * 8;
#pragma unroll
    for (int c = 0; c < KC; ++c) q[c] = load_q<V>(qp + c * 32, a.q_flip);
    f32x4 o[VB];
#pragma unroll
    for (int d = 0; d < VB; ++d) o[d] = f32x4{0, 0, 0, 0};
    float mref = 0.0f, mtop = -kInf, l = 0.0f;              // mtop: -inf until the row has seen a key, then mref + kSlack
    bool dirty = false;                                     // a value that is not finite was left out

    auto keep_pages = [&] {
#pragma unroll
        for (int u = 0; u < 2 * NH; ++u) v_pages[u] = pages[u];
    };
    if (wave < steps) {
        load_k(wave);
        keep_pages();
        load_v(wave);
        find_pages(wave + 4);
    }
    for (int s = wave; s < steps; s += 4) {
        const int ks = k0 + s * STEP;
        f32x4 acc[NH][2];
#pragma unroll
        for (int b2 = 0; b2 < NH; ++b2)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                acc[b2][b] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < KC; ++c) acc[b2][b] = Vec<T>::mma(kf[b2][b][c], q[c], acc[b2][b]);
            }
        const bool more = s + 4 < steps;
        if (more) {
            load_k(s + 4);
            keep_pages();
            find_pages(s + 8);
        }
        // x[8 b2 + j]: this lane's key ks + 32 b2 + 8 h + j
        float x[8 * NH];
#pragma unroll
        for (int j = 0; j < 8 * NH; ++j) x[j] = acc[j >> 3][(j >> 2) & 1][j & 3] * a.scale_log2;
        if (EXTRA && a.cap_log2 != 0.0f) {
#pragma unroll
            for (int j = 0; j < 8 * NH; ++j)
                x[j] = a.cap_log2 * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[j])));
        }
        if (EXTRA && a.k_times) {
#pragma unroll
            for (int j = 0; j < 8 * NH; ++j) x[j] -= dec * fmaxf(0.0f, tq - tk[j >> 3][(j >> 2) & 1][j & 3]);
        }
        const bool whole = ks + STEP <= lo && !(EXTRA && a.k_eps);
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8 * NH; ++j) {
                bool in = ks + 32 * (j >> 3) + 8 * h + (j & 7) < limit;
                if (EXTRA && a.k_eps) {
                    const int e = ek[j >> 3][(j >> 2) & 1][j & 3];
                    in = in && (e < 0 || eq < 0 || e == eq);
                }
                x[j] = in ? x[j] : -kInf;
            }
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8 * NH; ++j) top = fmaxf(top, x[j]);
        if (__any(top > mtop)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const bool none = mtop == -kInf;
            const float mnew = none ? top : fmaxf(mref, top);
            if (mnew != -kInf) {
                const float f = none ? 0.0f : __builtin_amdgcn_exp2f(mref - mnew);
                mref = mnew;
                mtop = mnew + kSlack;
                l *= f;
#pragma unroll
                for (int d = 0; d < VB; ++d) o[d] *= f;
            }
        }
        V p[NH];
#pragma unroll
        for (int j = 0; j < 8 * NH; ++j) {
            const float w = __builtin_amdgcn_exp2f(x[j] - mref);
            l += w;
            p[j >> 3][j & 7] = T(w);
        }
        if (!whole) {
            // some row does not see some key: see add_not_finite. Slots past the request's keys hold anything.
            uint32_t odd = 0;
#pragma unroll
            for (int b2 = 0; b2 < NH; ++b2) {
                const int kb = ks + 32 * b2 + 8 * h;
#pragma unroll
                for (int d = 0; d < VB; ++d) {
                    u32x4 b = __builtin_bit_cast(u32x4, vf[b2][d]);
                    if (kb + 8 > keys) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) b[j] &= kb + 2 * j >= keys ? 0u : kb + 2 * j + 1 >= keys ? 0xFFFFu : ~0u;
                    }
                    const uint32_t full = exponents_full<T>(b);
                    odd |= full;
                    if (__any(full != 0)) b = finite_part<T>(b);
                    vf[b2][d] = __builtin_bit_cast(V, b);
                }
            }
            if (__any(odd != 0)) dirty = true;
        }
#pragma unroll
        for (int b2 = 0; b2 < NH; ++b2)
#pragma unroll
            for (int d = 0; d < VB; ++d) o[d] = Vec<T>::mma(vf[b2][d], p[b2], o[d]);
        if (more) load_v(s + 4);
    }

    // join the waves: references first, then sums and O, in wave order
    auto& ml = lds.wave.ml;
    auto& ob = lds.wave.ob;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float mw = mtop == -kInf ? -kInf : mref;
    __syncthreads();                                        // the item has been read
    if (h == 0) ml[wave][col][0] = mw;
    if (dirty && lane == 0) any_dirty = 1;
    __syncthreads();
    float mall = ml[0][col][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) mall = fmaxf(mall, ml[w][col][0]);
    const float f = mw == -kInf ? 0.0f : __builtin_amdgcn_exp2f(mw - mall);
    if (h == 0) ml[wave][col][1] = l * f;
    // o[d][j] is element 16 d + 4 h + j of row `col`
#pragma unroll
    for (int d = 0; d < VB; ++d) o[d] *= f;
    if (wave >= 2) {
#pragma unroll
        for (int d = 0; d < VB; ++d) *reinterpret_cast<f32x4*>(&ob[wave - 2][col][d * 16 + h * 4]) = o[d];
    }
    __syncthreads();
    const float lall = ml[0][col][1] + ml[1][col][1] + ml[2][col][1] + ml[3][col][1];
    if (wave < 2) {
#pragma unroll
        for (int d = 0; d < VB; ++d) o[d] += *reinterpret_cast<const f32x4*>(&ob[wave][col][d * 16 + h * 4]);
    }
    __syncthreads();
    if (wave == 1) {
#pragma unroll
        for (int d = 0; d < VB; ++d) *reinterpret_cast<f32x4*>(&ob[0][col][d * 16 + h * 4]) = o[d];
    }
    __syncthreads();
    const bool joined = it.splits > 1;
    if (wave == 0) {
#pragma unroll
        for (int d = 0; d < VB; ++d) o[d] += *reinterpret_cast<const f32x4*>(&ob[0][col][d * 16 + h * 4]);
        if (row_ok && !joined) {
            const float inv = mall == -kInf ? 0.0f : 1.0f / lall;
            T* const op = static_cast<T*>(a.out) + row * a.out_stride + int64_t(hq) * D + h * 4;
#pragma unroll
            for (int d = 0; d < VB; ++d) {
                typename Vec<T>::v4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = mall == -kInf ? T(0.0f) : T(o[d][j] * inv);
                *reinterpret_cast<typename Vec<T>::v4*>(op + d * 16) = w;
            }
            if (a.lse && h == 0) a.lse[row * a.q_heads + hq] = mall == -kInf ? -kInf : (mall + __builtin_amdgcn_logf(lall)) * kLn2;
        }
        if (row_ok && joined) {
            float* const po = a.part_o + (int64_t(it.part + it.split) * kFewRows + col) * D + h * 4;
#pragma unroll
            for (int d = 0; d < VB; ++d) put_part(po + d * 16, o[d]);
            if (h == 0) put_part(a.part_ml + int64_t(it.part + it.split) * kFewRows + col, make_float2(mall, lall));
        }
    }
    if (any_dirty) {
        __syncthreads();
        add_not_finite<T, D, kFewRows>(a, it, row0, n, keys, prefix, k0, min(k0 + it.chunk, keys));
    }
    if (!joined) return;
    __syncthreads();
    join_splits<T, D, kFewRows>(a, it, row0, n, lds.join);
}

// ---- many rows: 128 at a time, keys staged through LDS ----------------------------------
// Bound by the matrix cores and the softmax's vector work together (32 exp2 per lane and tile of
// 64 keys take as long as the 32 MFMAs). 4 waves of 32 rows each share tiles of 64 keys: K (keys, elements) and
// V (elements, keys) come by global_load_lds_dwordx4 into two buffers, one tile ahead. 16-byte pieces
// of a row are XORed with the row number so that the 16 lanes of a fragment read hit
// the 16 bank groups. The other workgroup of the CU fills the matrix cores while this one's waves
// are in the softmax.
constexpr int kManyKeys = 64;

template <int D>
struct ManyLds {
    u32x4 k[2][kManyKeys * D / 8];
    u32x4 v[2][kManyKeys * D / 8];
    float times[2][kManyKeys];
    int32_t eps[2][kManyKeys];
};

template <typename T, int D, bool EXTRA>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void k_attend_many(AttendArgs a) {
    using V = typename Vec<T>::v8;
    constexpr int KS = D / 16, DB = D / 32, RC = D / 8;      // k-steps of S, blocks of O, 16-byte pieces of a key's row
    __shared__ __attribute__((aligned(16))) union { ManyLds<D> tiles; SchedLds sched; JoinLds<kManyRows> join; } lds;
    ManyLds<D>& sh = lds.tiles;
    const Item it = find_item(a, blockIdx.x, kManyRows, 256, kManyItemsLog2, lds.sched);
    if (!it.found) return;
    __syncthreads();                                         // the item is read before its LDS is used again
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int r = __builtin_amdgcn_readfirstlane(it.request), head = __builtin_amdgcn_readfirstlane(it.head);
    const int P1 = (1 << a.page_shift) - 1;
    const int row0 = max(a.q_start[r], 0), n = min(a.q_start[r + 1], a.tokens) - row0;
    const int keys = int(min(int64_t(max(a.kv_lens[r], 0)), int64_t(a.max_pages) << a.page_shift));
    const int m = it.tile * kManyRows + wave * 32 + col;     // this lane's row: token i, head of the group
    const bool row_ok = m < n * a.group;
    const int i = row_ok ? m / a.group : 0, hq = head * a.group + (row_ok ? m - i * a.group : 0);
    const int64_t row = int64_t(row0) + i;
    const int prefix = a.prefix ? min(max(a.prefix[r], 0), keys) : 0;
    const int limit = row_ok ? min(max(keys - n + i + 1, prefix), keys) : 0;   // keys [0, limit) may be seen
    float dec = 0.0f, tq = 0.0f;
    int eq = -1;
    if constexpr (EXTRA) {
        dec = a.decay ? a.decay[hq] * 1.4426950408889634f : 0.0f;
        tq = a.decay ? a.q_times[row] : 0.0f;
        eq = a.q_eps ? a.q_eps[row] : -1;
    }

    V q[KS];
    const T* const qp = static_cast<const T*>(a.q) + row * a.q_stride + int64_t(hq) * D + h * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = load_q<V>(qp + s * 16, a.q_flip);

    int lo = row_ok ? limit : INT32_MAX, hi = limit;         // over the wave's rows
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    // the workgroup's last row sees the most keys: limits grow with the token
    const int last_i = min((it.tile * kManyRows + kManyRows - 1) / a.group, n - 1);
    const int end = min(max(keys - n + last_i + 1, prefix), keys);
    const int first_limit = min(max(keys - n + it.tile * kManyRows / a.group + 1, prefix), keys);
    const int k0 = it.split * it.chunk, k1 = min(k0 + it.chunk, end);
    const int steps = __builtin_amdgcn_readfirstlane(k1 > k0 ? (k1 - k0 + kManyKeys - 1) / kManyKeys : 0);

    const TablePtr table = table_row(a, r);
    const int last_page = keys > 0 ? (keys - 1) >> a.page_shift : 0;
    // Pieces of 16 bytes in a tile: K's row of a key holds RC of them, V's row of an element the 8 of the tile's 64 keys.
    // Piece c of row w lies at place c ^ swz(w). Load j of a wave fills the 64 places from (4 j + wave) * 64.
    auto kswz = [](int w) { return D == 64 ? (w >> 1) & 7 : w & 15; };
    auto vswz = [](int w) { return (w >> 1) & 7; };
    constexpr int KR = 256 / RC;                             // rows of K per load of the workgroup
    const int krow = tid / RC, kpiece = (tid % RC) ^ kswz(krow), vrow = tid >> 3, vkey = ((tid & 7) ^ vswz(vrow)) * 8;
    static_assert(KR % 16 == 0 || D == 256, "a thread's pieces keep their place in the row");
    const char* const kp = static_cast<const char*>(a.k_pages) + ((int64_t(head) << a.page_shift) * D + krow % 16 * D) * 2;
    const char* const vp = static_cast<const char*>(a.v_pages) + ((int64_t(head) << a.page_shift) * D + (int64_t(vrow) << a.page_shift)) * 2;
    int pages[4];                                            // of the next tile's 4 groups of 16 keys
    auto find_pages = [&](int s) {
#pragma unroll
        for (int u = 0; u < 4; ++u) pages[u] = page_of(a, table, k0 + s * kManyKeys + u * 16, last_page);
    };
    auto stage = [&](int s, int buf) {
        const int kt = k0 + s * kManyKeys;
#pragma unroll
        for (int j = 0; j < RC / 4; ++j) {
            const int u = KR == 32 ? 2 * j + (wave >> 1) : (j * KR) >> 4;      // the wave's rows lie in this group of 16 keys
            const int pg = KR == 32 ? (wave >> 1 ? pages[2 * j + 1] : pages[2 * j]) : pages[(j * KR) >> 4];
            const char* const base = kp + (pg * a.k_stride + int64_t((kt + u * 16) & P1) * D) * 2;
            const int piece = D == 256 ? (tid % RC) ^ kswz(krow + j * KR) : kpiece;
            const int off = (D == 256 ? (j * KR) % 16 * D * 2 : 0) + piece * 16;
            dma16(base + off, &sh.k[buf][j * 256 + wave * 64]);
        }
        const int g = vkey >> 4;
        const int64_t b0 = pages[0] * a.v_stride + ((kt) & P1), b1 = pages[1] * a.v_stride + ((kt + 16) & P1);
        const int64_t b2 = pages[2] * a.v_stride + ((kt + 32) & P1), b3 = pages[3] * a.v_stride + ((kt + 48) & P1);
        const char* const p = vp + ((g & 2 ? (g & 1 ? b3 : b2) : (g & 1 ? b1 : b0)) + (vkey & 15)) * 2;
#pragma unroll
        for (int j = 0; j < RC / 4; ++j)
            dma16(p + (int64_t(j) * 64 << a.page_shift), &sh.v[buf][j * 256 + wave * 64]);
        if constexpr (EXTRA) {
            if (wave == 0) {
                const int e = lane >> 4;
                const int pg = e & 2 ? (e & 1 ? pages[3] : pages[2]) : (e & 1 ? pages[1] : pages[0]);
                const int64_t slot = (int64_t(pg) << a.page_shift) + ((kt + lane) & P1);
                if (a.k_times) dma4(a.k_times + slot, &sh.times[buf][0]);
                if (a.k_eps) dma4(a.k_eps + slot, &sh.eps[buf][0]);
            }
        }
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] = 0.0f;
    float mref = 0.0f, mtop = -kInf, l = 0.0f;               // mtop: -inf until the row has seen a key, then mref + kSlack
    bool dirty = false;                                      // a value that is not finite was left out

    // K's row of lane `col` in a block of 32 keys: reg j of S then holds key 16 (j / 8) + 8 h + j % 8 of the block
    const int ki = (col & 16) + ((col >> 2) & 1) * 8 + ((col >> 3) & 1) * 4 + (col & 3);
    // byte offsets of this lane's fragments in a tile, piece 2 c + h of S's step c and piece 2 t + h of O's: those of
    // c = 0, t = 0, with c or t XORed into the piece bits
    const uint32_t koff = uint32_t(ki * RC + (h ^ kswz(ki))) * 16, voff = uint32_t(col * 8 + (h ^ vswz(col))) * 16;
    const char* const kl = reinterpret_cast<const char*>(&sh.k[0][0]);
    const char* const vl = reinterpret_cast<const char*>(&sh.v[0][0]);
    if (steps > 0) {
        find_pages(0);
        stage(0, 0);
        find_pages(1);
    }
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
        tile_barrier();                                      // the tile is in LDS; nobody reads the other buffer any more
        if (s + 1 < steps) {
            stage(s + 1, buf ^ 1);
            find_pages(s + 2);
        }
        const uint32_t kb = buf * uint32_t(sizeof(sh.k[0])) + koff, vb = buf * uint32_t(sizeof(sh.v[0])) + voff;
        const int kt = k0 + s * kManyKeys;
        if (kt + kManyKeys > first_limit || (EXTRA && a.k_eps)) {
            // some row of the workgroup does not see some key: each thread looks over its pieces of V (see add_not_finite;
            // slots past the request's keys hold anything and become 0)
#pragma unroll
            for (int j = 0; j < RC / 4; ++j) {
                u32x4 b = sh.v[buf][j * 256 + tid];
                const bool past = kt + vkey + 8 > keys;
                if (past) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = kt + vkey + 2 * e;
                        b[e] &= key >= keys ? 0u : key + 1 >= keys ? 0xFFFFu : ~0u;
                    }
                }
                const bool full = exponents_full<T>(b) != 0;
                if (full) b = finite_part<T>(b);
                if (past || full) sh.v[buf][j * 256 + tid] = b;
                dirty |= full;
            }
            lds_barrier();
        }
        if (kt >= hi) continue;                              // the wave's rows end before
        f32x16 x[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[b][j] = 0.0f;
#pragma unroll
            for (int c = 0; c < KS; ++c) x[b] = Vec<T>::mma32(load16<V>(kl + (kb ^ (c * 32)) + b * 32 * RC * 16), q[c], x[b]);
        }
        bool whole = kt + kManyKeys <= lo;
        uint32_t seen = ~0u;                                 // bit 16 b + j
        if constexpr (EXTRA) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) x[b][j] *= a.scale_log2;
            if (a.cap_log2 != 0.0f) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        x[b][j] = a.cap_log2 * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[b][j])));
            }
            if (a.k_times) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        x[b][j] -= dec * fmaxf(0.0f, tq - sh.times[buf][b * 32 + (j >> 3) * 16 + h * 8 + (j & 7)]);
            }
            if (a.k_eps) {
                whole = false;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int e = sh.eps[buf][b * 32 + (j >> 3) * 16 + h * 8 + (j & 7)];
                        if (!(e < 0 || eq < 0 || e == eq)) seen &= ~(1u << (16 * b + j));
                    }
            }
        }
        if (!whole) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const bool in = kt + b * 32 + (j >> 3) * 16 + h * 8 + (j & 7) < limit && ((seen >> (16 * b + j)) & 1u);
                    if (!in) seen &= ~(1u << (16 * b + j));
                    x[b][j] = in ? x[b][j] : -kInf;
                }
        }
        const float c = EXTRA ? 1.0f : a.scale_log2;         // not negative: a negative scale turns q's sign
        float top = x[0][0];
#pragma unroll
        for (int j = 1; j < 16; ++j) top = fmaxf(top, x[0][j]);
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, x[1][j]);
        top *= c;
        if (__any(top > mtop)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            const bool none = mtop == -kInf;
            const float mnew = none ? top : fmaxf(mref, top);
            if (mnew != -kInf) {
                const float f = none ? 0.0f : __builtin_amdgcn_exp2f(mref - mnew);
                mref = mnew;
                mtop = mnew + kSlack;
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= f;
            }
        }
        V p[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float w = __builtin_amdgcn_exp2f(fmaf(x[b][j], c, -mref));
                l += w;
                p[2 * b + (j >> 3)][j & 7] = T(w);
            }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = Vec<T>::mma32(load16<V>(vl + (vb ^ (t * 32)) + d * 32 * 8 * 16), p[t], o[d]);
    }

    l += __shfl_xor(l, 32);
    const bool empty = mtop == -kInf;
    // o[d][j] is element 32 d + 8 (j / 4) + 4 h + j % 4 of row `col`
    if (it.splits == 1 && row_ok) {
        const float inv = empty ? 0.0f : 1.0f / l;
        T* const op = static_cast<T*>(a.out) + row * a.out_stride + int64_t(hq) * D + h * 4;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                typename Vec<T>::v4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = empty ? T(0.0f) : T(o[d][g * 4 + j] * inv);
                *reinterpret_cast<typename Vec<T>::v4*>(op + d * 32 + g * 8) = w;
            }
        if (a.lse && h == 0) a.lse[row * a.q_heads + hq] = empty ? -kInf : (mref + __builtin_amdgcn_logf(l)) * kLn2;
    }
    if (it.splits > 1 && row_ok) {
        const int64_t at = int64_t(it.part + it.split) * kManyRows + wave * 32 + col;
        float* const po = a.part_o + at * D + h * 4;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                put_part(po + d * 32 + g * 8, f32x4{o[d][g * 4], o[d][g * 4 + 1], o[d][g * 4 + 2], o[d][g * 4 + 3]});
        if (h == 0) put_part(a.part_ml + at, make_float2(empty ? -kInf : mref, l));
    }
    __syncthreads();                                         // the LDS of the tiles is free, the rows are written
    if (tid == 0) lds.join.last = 0;
    __syncthreads();
    if (dirty) lds.join.last = 1;
    __syncthreads();
    if (lds.join.last) add_not_finite<T, D, kManyRows>(a, it, row0, n, keys, prefix, k0, min(k0 + it.chunk, keys));
    if (it.splits == 1) return;
    __syncthreads();
    join_splits<T, D, kManyRows>(a, it, row0, n, lds.join);
}

template <typename T, int D, bool EXTRA>
int launch_few(AttendArgs a, hipStream_t s) {
    const int64_t tiles = int64_t(a.tokens) * a.group / kFewRows + std::min(a.requests, a.tokens);
    const int64_t grid = (1 << kFewItemsLog2) + tiles * a.kv_heads;
    MARS_CHECK(grid <= INT32_MAX, MARS_ERR_CAPACITY, "%lld tiles of rows", (long long)grid);
    MARS_LAUNCH((k_attend_few<T, D, EXTRA>), dim3(unsigned(grid)), dim3(256), 0, s, a);
    return MARS_OK;
}

template <typename T, int D, bool EXTRA>
int launch_many(AttendArgs a, hipStream_t s) {
    const int64_t tiles = int64_t(a.tokens) * a.group / kManyRows + std::min(a.requests, a.tokens);
    const int64_t grid = (1 << kManyItemsLog2) + tiles * a.kv_heads;
    MARS_CHECK(grid <= INT32_MAX, MARS_ERR_CAPACITY, "%lld tiles of rows", (long long)grid);
    MARS_LAUNCH((k_attend_many<T, D, EXTRA>), dim3(unsigned(grid)), dim3(256), 0, s, a);
    return MARS_OK;
}

template <typename T, int D>
int launch_dim(AttendArgs a, int32_t max_new, hipStream_t s) {
    // Requests of at most kFewMost rows (new tokens x query heads per kv head) go to k_attend_few, the others to
    // k_attend_many, in a launch of their own each. A bound on the new tokens that rules one of them out saves its launch;
    // a request that breaks the bound is served by the other kernel.
    const int64_t most = std::min<int64_t>(max_new > 0 ? max_new : a.tokens, a.tokens) * a.group;
    const bool few_only = most <= kFewMost, many_only = !few_only && a.requests == 1;
    const bool extra = a.cap_log2 != 0.0f || a.k_times || a.k_eps;
    if (!many_only) {
        AttendArgs f = a;
        f.rows_lo = 0;
        f.rows_hi = few_only ? INT32_MAX : kFewMost;
        if (extra) MARS_TRY((launch_few<T, D, true>(f, s)));
        else MARS_TRY((launch_few<T, D, false>(f, s)));
    }
    if (!few_only) {
        a.rows_lo = many_only ? 0 : kFewMost;
        a.rows_hi = INT32_MAX;
        if (extra) MARS_TRY((launch_many<T, D, true>(a, s)));
        else MARS_TRY((launch_many<T, D, false>(a, s)));
    }
    return MARS_OK;
}

template <typename T>
int launch_typed(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s) {
    switch (r.d.head_dim) {
        case 64: return launch_dim<T, 64>(a, max_new, s);
        case 128: return launch_dim<T, 128>(a, max_new, s);
        default: return launch_dim<T, 256>(a, max_new, s);
    }
}

}  // namespace

int launch_attend(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s) {
    return r.d.dtype == MARS_DTYPE_F16 ? launch_typed<_Float16>(r, a, max_new, s) : launch_typed<__bf16>(r, a, max_new, s);
}

}  // namespace mars
