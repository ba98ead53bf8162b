// ============================================================================
//  reader.hip — the reading path's handle, plan, store and release (mars_reader,
//  mars_kv_*): how the tokens of retrieved memories are laid out in a paged cache.
//  attend.hip holds the attention over it.
// ============================================================================
#include "reader.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <memory>
#include <new>
#include <vector>

namespace mars {
namespace {

// ---- plan -------------------------------------------------------------------------
// One launch, no communication between workgroups: each computes the prefix sums over the
// requests for itself (new tokens, then pages taken; at most 4096 of them, read from L2) and
// then fills its share of the rows: token t's request is found by bisection in LDS, and a
// page handed out in this call is read from the free list by the same arithmetic that writes
// it to the table, so no workgroup waits for another's writes. Launch and latency bound: two
// block scans and a dozen dependent LDS reads (8 requests 4.7 us, 768 requests 7.4 us).
constexpr int kPlanThreads = 512;
constexpr int kPlanTokens = 1024;                        // rows of the step per workgroup
constexpr int kPlanPer = kMaxRequests / kPlanThreads;    // requests per thread, consecutive

// Exclusive prefix of v over the block's threads; *total = the block's sum.
__device__ int64_t block_scan(int64_t v, int64_t* wsum, int64_t* total) {
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, unsigned(o));
        if (lane >= o) x += y;
    }
    __syncthreads();                                     // wsum may still be read from the scan before
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    int64_t before = 0, sum = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        const int64_t s = wsum[w];
        before += w < wave ? s : 0;
        sum += s;
    }
    *total = sum;
    return before + x - v;
}

__global__ __launch_bounds__(kPlanThreads) void k_kv_plan(mars_kv_plan_args a, int page_shift) {
    __shared__ int32_t start[kMaxRequests + 1];          // first row of each request
    __shared__ int32_t fresh[kMaxRequests];              // its first entry's rank among the pages handed out; -1: not served
    __shared__ int32_t cached[kMaxRequests];
    __shared__ int64_t wsum[kPlanThreads / 64];
    const int R = a.num_requests, page = 1 << page_shift, tid = int(threadIdx.x);
    const int per = (R + kPlanThreads - 1) / kPlanThreads;
    const int first = min(tid * per, R), last = min(first + per, R);
    const int64_t free = max(0, min(a.free_count[0], a.free_capacity));

    int32_t n_new[kPlanPer], n_old[kPlanPer];
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = first + i;
        n_new[i] = r < last ? max(a.new_lens[r], 0) : 0;
        n_old[i] = r < last ? max(a.cached_lens[r], 0) : 0;
        sum += n_new[i];
    }
    int64_t total, at = block_scan(sum, wsum, &total);
    int32_t need[kPlanPer];
    bool fits[kPlanPer];
    sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = first + i;
        if (r < last) start[r] = int32_t(min(at, int64_t(INT32_MAX)));
        at += n_new[i];
        const int64_t len = int64_t(n_old[i]) + n_new[i];
        const int64_t pages = (len + page - 1) >> page_shift, have = (int64_t(n_old[i]) + page - 1) >> page_shift;
        fits[i] = pages <= a.max_pages && at <= a.num_tokens && len <= INT32_MAX;
        need[i] = fits[i] ? int32_t(pages - have) : 0;
        sum += need[i];
    }
    if (tid == 0) start[R] = int32_t(min(total, int64_t(INT32_MAX)));
    int64_t all, taken = block_scan(sum, wsum, &all), used = 0;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
        const int r = first + i;
        if (r >= last) continue;
        const bool served = fits[i] && (need[i] == 0 || taken + need[i] <= free);
        fresh[r] = served ? int32_t(min(taken, free)) : -1;
        cached[r] = n_old[i];
        taken += need[i];
        if (served && need[i] > 0) used = taken;
        if (blockIdx.x == 0) {
            a.kv_lens[r] = served ? n_old[i] + n_new[i] : 0;
            if (a.next_lens) a.next_lens[r] = n_old[i] + (served ? n_new[i] : 0);
        }
    }
    if (blockIdx.x == 0) {
        // the last served request that took pages has the largest running count: a maximum, as the prefix grows
#pragma unroll
        for (int o = 32; o; o >>= 1) used = max(used, int64_t(__shfl_xor((long long)used, o)));
        __syncthreads();
        if ((tid & 63) == 0) wsum[tid >> 6] = used;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kPlanThreads / 64; ++w) used = max(used, wsum[w]);
            a.free_count_out[0] = int32_t(free - used);
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int r = tid; r <= R; r += kPlanThreads) a.q_start[r] = start[r];

    // the pages handed out: the requests dealt over the workgroups' threads, 8 to each
    const int eighth = (int(blockIdx.x) * kPlanThreads + tid) >> 3, eighths = int(gridDim.x) * kPlanThreads >> 3;
    for (int r = eighth; r < R; r += eighths) {
        if (fresh[r] < 0) continue;
        const int64_t len = int64_t(cached[r]) + (start[r + 1] - start[r]);
        const int have = int((int64_t(cached[r]) + page - 1) >> page_shift), pages = int((len + page - 1) >> page_shift);
        for (int j = have + (tid & 7); j < pages; j += 8)
            a.block_table[int64_t(r) * a.max_pages + j] = a.free_pages[free - 1 - (fresh[r] + j - have)];
    }
    // slots and positions of this workgroup's rows
    const int t0 = int(blockIdx.x) * kPlanTokens, rows = min(kPlanTokens, a.num_tokens - t0);    // t0 + kPlanTokens may pass 2^31
    for (int i = tid; i < rows; i += kPlanThreads) {
        const int t = t0 + i;
        int64_t slot = -1;
        int32_t pos = 0;
        if (t < start[R]) {
            int lo = 0, hi = R;                          // start[lo] <= t < start[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= t) lo = mid; else hi = mid;
            }
            pos = int32_t(min(int64_t(cached[lo]) + (t - start[lo]), int64_t(INT32_MAX)));
            if (fresh[lo] >= 0) {
                const int have = int((int64_t(cached[lo]) + page - 1) >> page_shift), j = pos >> page_shift;
                const int32_t id = j < have ? a.block_table[int64_t(lo) * a.max_pages + j]
                                            : a.free_pages[free - 1 - (fresh[lo] + j - have)];
                slot = (int64_t(id) << page_shift) + (pos & (page - 1));
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
}

// ---- release ------------------------------------------------------------------------
// One workgroup, since the free list is one line: bound by its own reads and writes where many pages come back at once
// (768 requests of 125 pages 42 us), by latency else (8 of 125 pages 2.6 us).
__global__ __launch_bounds__(kPlanThreads) void k_kv_release(const int32_t* __restrict__ done, int32_t* __restrict__ kv_lens,
                                                             const int32_t* __restrict__ table, int R, int max_pages,
                                                             int32_t* __restrict__ free_pages, int32_t* __restrict__ free_count,
                                                             int free_capacity, int page_shift) {
    __shared__ int32_t rank[kMaxRequests], count[kMaxRequests];
    __shared__ int64_t wsum[kPlanThreads / 64];
    const int tid = int(threadIdx.x), per = (R + kPlanThreads - 1) / kPlanThreads;
    const int first = min(tid * per, R), last = min(first + per, R);
    const int64_t held = max(0, min(free_count[0], free_capacity));
    int64_t sum = 0;
    for (int r = first; r < last; ++r) {
        const int64_t pages = (int64_t(max(kv_lens[r], 0)) + (1 << page_shift) - 1) >> page_shift;
        count[r] = done[r] ? int32_t(min(pages, int64_t(max_pages))) : 0;
        sum += count[r];
    }
    int64_t total, at = block_scan(sum, wsum, &total);
    for (int r = first; r < last; ++r) {
        rank[r] = int32_t(min(held + at, int64_t(INT32_MAX)));
        at += count[r];
        if (done[r]) kv_lens[r] = 0;
    }
    __syncthreads();
    for (int r = tid >> 6; r < R; r += kPlanThreads / 64)
        for (int j = tid & 63; j < count[r]; j += 64)
            if (int64_t(rank[r]) + j < free_capacity) free_pages[rank[r] + j] = table[int64_t(r) * max_pages + j];
    if (tid == 0) free_count[0] = int32_t(min(held + total, int64_t(free_capacity)));
}

// ---- store --------------------------------------------------------------------------
struct StoreArgs {
    mars_kv_store_args s;
    void* k_pages;
    void* v_pages;
    float* times;
    int32_t* eps;
    const uint64_t* freq;
    const int32_t* axis;
    int64_t k_stride, v_stride, slots;                   // page strides (elements); slots the cache has
    int32_t q_heads, kv_heads, head_dim, rope_dim, adjacent, page_shift;
};

// sin and cos of 2 pi * pos * f, f in units of 2^-64 turns per position: whole turns drop out of the 64-bit product
// by themselves, so the phase is exact to pos * 2^-65 turns for every int32 position, and the angle to the rounding of
// its upper 32 bits to fp32. (A product in fp32 is off by 2^-24 of the whole angle: 0.004 rad at position 70,000.)
__device__ inline void turn(int32_t pos, uint64_t f, float* sn, float* cs) {
    const uint64_t phase = uint64_t(int64_t(pos)) * f;
    sincospif(float(int32_t(uint32_t(phase >> 32))) * 0x1p-31f, sn, cs);
}

// Few tokens: a workgroup to each, a pair of values a thread and turn. Latency bound (32 tokens 5.0 us).
constexpr int32_t kStoreFew = 1024;       // see k_kv_store_tile
template <typename T>
__global__ __launch_bounds__(256) void k_kv_store(StoreArgs a) {
    const int t = int(blockIdx.x), half = a.rope_dim / 2, D = a.head_dim;
    __shared__ float sn[128], cs[128];
    for (int i = int(threadIdx.x); i < half; i += 256) {
        turn(a.s.positions[int64_t(a.axis[i]) * a.s.num_tokens + t], a.freq[i], &sn[i], &cs[i]);
        if (a.s.inverse) sn[i] = -sn[i];
    }
    __syncthreads();
    const int64_t slot = a.s.slots ? a.s.slots[t] : -1;
    const bool stored = slot >= 0 && slot < a.slots;
    const int64_t page = stored ? slot >> a.page_shift : 0;
    const int off = stored ? int(slot & ((1 << a.page_shift) - 1)) : 0, P = 1 << a.page_shift;
    const T* const q = static_cast<const T*>(a.s.q);
    const T* const k = static_cast<const T*>(a.s.k);
    const T* const v = static_cast<const T*>(a.s.v);
    const int q_heads = q ? a.q_heads : 0, k_heads = k && stored ? a.kv_heads : 0;
    // a thread reads and writes both elements of a pair, so q_out may be q; pairs past the rotary part are copied
    for (int e = int(threadIdx.x); e < (q_heads + k_heads) * (D / 2); e += 256) {
        const int h = e / (D / 2), j = e % (D / 2);
        const T* const x = h < q_heads ? q + t * a.s.q_stride + h * D : k + t * a.s.k_stride + (h - q_heads) * D;
        T* const to = h < q_heads ? static_cast<T*>(a.s.q_out) + t * a.s.q_out_stride + h * D
                                  : static_cast<T*>(a.k_pages) + page * a.k_stride + (int64_t(h - q_heads) * P + off) * D;
        const bool turns = j < half;
        const int i0 = turns && !a.adjacent ? j : 2 * j, i1 = turns && !a.adjacent ? j + half : 2 * j + 1;
        const float y = float(x[i0]), z = float(x[i1]), c = turns ? cs[j] : 1.0f, s = turns ? sn[j] : 0.0f;
        const T lo = turns ? T(y * c - z * s) : x[i0], hi = turns ? T(y * s + z * c) : x[i1];
        to[i0] = lo;
        to[i1] = hi;
    }
    if (!v || !stored) return;
    for (int e = int(threadIdx.x); e < a.kv_heads * D; e += 256)
        static_cast<T*>(a.v_pages)[page * a.v_stride + int64_t(e) * P + off] = v[t * a.s.v_stride + e];
    if (threadIdx.x == 0 && a.times && a.s.times) a.times[slot] = a.s.times[t];
    if (threadIdx.x == 0 && a.eps && a.s.episodes) a.eps[slot] = a.s.episodes[t];
}

// Many tokens: a workgroup takes kTile of them under one kv head: its k and v, and the group's q heads. The angles of the
// tokens are computed once a workgroup (LDS), q and k move in pieces of 16 bytes, and v, whose pages hold the tokens of an
// element side by side, goes through LDS: where 8 consecutive tokens fill 8 consecutive slots from a multiple of 8 on
// they are written as 16 bytes, and the lanes of a wave fill whole rows of a page; other tokens value by value.
// Bound by the bytes in and out: 4,099 tokens of 32/8 heads of 128, 101 MB, 27 us with all of it in the caches, 36 us from
// and to memory. (A group of 8 has to lie in one workgroup's 64 tokens: where the step's tokens do not begin at a multiple of 8
// slots, 8 of every 64 are written value by value.) Up to kStoreFew tokens k_kv_store has the shorter call, there and here:
//   tokens            512           1,024         1,536         2,048         4,099
//   32/8 of 128       13.3  15.5    15.2  17.2    18.5  18.1    21.7  19.1    65.8  36.3 us
//   8/2 of 256        12.7  15.4    12.7  16.5    12.9  17.0    13.7  17.4    21.6  19.8
//   12/12 of 64       12.7  12.5    12.8  12.3    12.9  12.2    13.0  12.5    20.2  15.2
template <int D>
constexpr int store_tile() { return D == 256 ? 32 : 64; }

template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv_store_tile(StoreArgs a) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    constexpr int kTile = store_tile<D>(), VS = D + 2;
    __shared__ __attribute__((aligned(16))) float2 turns[kTile][D / 2];          // cos, sin
    __shared__ __attribute__((aligned(16))) T vt[kTile][VS];
    __shared__ int64_t slot_of[kTile];
    __shared__ uint8_t lead[kTile];                          // first of 8 written together
    __shared__ uint8_t groups[kTile / 8], singles[kTile];
    __shared__ int counts[2];
    const int t0 = int(blockIdx.x) * kTile, head = int(blockIdx.y), tid = int(threadIdx.x);
    const int nt = min(kTile, a.s.num_tokens - t0), half = a.rope_dim / 2, P = 1 << a.page_shift;
    const T* const q = static_cast<const T*>(a.s.q);
    const T* const k = static_cast<const T*>(a.s.k);
    const T* const v = static_cast<const T*>(a.s.v);
    const int group = q ? a.q_heads / a.kv_heads : 0;

    if (tid < kTile) {
        const int64_t s = k && tid < nt ? a.s.slots[t0 + tid] : -1;
        slot_of[tid] = s >= 0 && s < a.slots ? s : -1;
    }
    // everything the workgroup reads is on the way before the angles are computed: its v, and of q and k the first pieces
    constexpr int VU = kTile * (D / 8) / 256;
    v8 vr[VU];
    if (v) {
#pragma unroll
        for (int u = 0; u < VU; ++u) {
            const int e = tid + u * 256, i = e / (D / 8), c = e % (D / 8);
            if (i < nt) vr[u] = *reinterpret_cast<const v8*>(v + (t0 + i) * a.s.v_stride + head * D + c * 8);
        }
    }
    // q and k: a thread takes two pieces of 8 elements of a head, the partners of each other where they turn (both are read
    // before either is written: q_out may be q), and four such pairs on the way together
    constexpr int U = 4;
    const int heads = group + (k ? 1 : 0), turning = half / 8, pairs = nt * heads * (D / 16);
    v8 y[U], z[U];
    auto first_of = [&](int c) { return c < turning && !a.adjacent ? c * 8 : c * 16; };
    auto second_of = [&](int c) { return c < turning && !a.adjacent ? half + c * 8 : c * 16 + 8; };
    auto read_pairs = [&](int e0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * 256, c = e % (D / 16), ih = e / (D / 16), i = ih / heads, hh = ih % heads;
            if (e >= pairs) break;
            const T* const x = hh < group ? q + (t0 + i) * a.s.q_stride + (head * group + hh) * D : k + (t0 + i) * a.s.k_stride + head * D;
            y[u] = *reinterpret_cast<const v8*>(x + first_of(c));
            z[u] = *reinterpret_cast<const v8*>(x + second_of(c));
        }
    };
    read_pairs(tid);
    for (int e = tid; e < nt * half; e += 256) {
        const int i = e / half, f = e % half;
        float sn, cs;
        turn(a.s.positions[int64_t(a.axis[f]) * a.s.num_tokens + t0 + i], a.freq[f], &sn, &cs);
        turns[i][f] = make_float2(cs, a.s.inverse ? -sn : sn);
    }
    if (v) {
#pragma unroll
        for (int u = 0; u < VU; ++u) {
            const int e = tid + u * 256, i = e / (D / 8), c = e % (D / 8);
            typedef uint32_t u4 __attribute__((ext_vector_type(4)));
            const u4 w = __builtin_bit_cast(u4, vr[u]);
            if (i < nt) {
#pragma unroll
                for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(&vt[i][c * 8])[j] = w[j];
            }
        }
    }
    __syncthreads();
    if (k && tid < kTile) {
        const int64_t s = slot_of[tid];
        bool first = s >= 0 && s % 8 == 0 && tid + 8 <= nt;
        for (int j = 1; j < 8 && first; ++j) first = slot_of[tid + j] == s + j;
        lead[tid] = first;
    }
    __syncthreads();
    if (k && tid < 64) {                                     // one wave: the groups, and the tokens of none
        const bool in = tid < kTile && slot_of[tid] >= 0;
        const int at = in ? int(slot_of[tid] % 8) : 0;
        const bool first = tid < kTile && lead[tid], alone = in && !(tid >= at && lead[tid - at]);
        const uint64_t gs = __ballot(first), ss = __ballot(alone), below = (1ull << tid) - 1;
        if (first) groups[__popcll(gs & below)] = uint8_t(tid);
        if (alone) singles[__popcll(ss & below)] = uint8_t(tid);
        if (tid == 0) { counts[0] = __popcll(gs); counts[1] = __popcll(ss); }
        if (head == 0 && in) {
            if (a.times && a.s.times) a.times[slot_of[tid]] = a.s.times[t0 + tid];
            if (a.eps && a.s.episodes) a.eps[slot_of[tid]] = a.s.episodes[t0 + tid];
        }
    }

    for (int e0 = tid; e0 < pairs; e0 += U * 256) {
        if (e0 != tid) read_pairs(e0);
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int e = e0 + n * 256, c = e % (D / 16), ih = e / (D / 16), i = ih / heads, hh = ih % heads;
            if (e >= pairs) break;
            const bool is_q = hh < group;
            if (!is_q && slot_of[i] < 0) continue;
            T* const to = is_q ? static_cast<T*>(a.s.q_out) + (t0 + i) * a.s.q_out_stride + (head * group + hh) * D
                               : static_cast<T*>(a.k_pages) + (slot_of[i] >> a.page_shift) * a.k_stride + (int64_t(head) * P + (slot_of[i] & (P - 1))) * D;
            v8 u = y[n], w = z[n];
            if (c < turning && !a.adjacent) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 f = turns[i][c * 8 + j];
                    const float yy = float(y[n][j]), zz = float(z[n][j]);
                    u[j] = T(yy * f.x - zz * f.y);
                    w[j] = T(yy * f.y + zz * f.x);
                }
            } else if (c < turning) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 f = turns[i][c * 8 + j];    // pair j of the 16 elements
                    const float yy = float(j < 4 ? y[n][2 * j] : z[n][2 * j - 8]), zz = float(j < 4 ? y[n][2 * j + 1] : z[n][2 * j - 7]);
                    const T lo = T(yy * f.x - zz * f.y), hi = T(yy * f.y + zz * f.x);
                    if (j < 4) { u[2 * j] = lo; u[2 * j + 1] = hi; }
                    else { w[2 * j - 8] = lo; w[2 * j - 7] = hi; }
                }
            }
            *reinterpret_cast<v8*>(to + first_of(c)) = u;
            *reinterpret_cast<v8*>(to + second_of(c)) = w;
        }
    }
    if (!v) return;
    __syncthreads();
    T* const vp = static_cast<T*>(a.v_pages) + int64_t(head) * D * P;
    const int ng = counts[0], ns = counts[1];
    for (int e = tid; e < ng * D; e += 256) {
        const int d = e / ng, i = groups[e % ng];
        v8 x;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = vt[i + j][d];
        *reinterpret_cast<v8*>(vp + (slot_of[i] >> a.page_shift) * a.v_stride + (int64_t(d) << a.page_shift) + (slot_of[i] & (P - 1))) = x;
    }
    for (int e = tid; e < ns * D; e += 256) {
        const int d = e / ns, i = singles[e % ns];
        vp[(slot_of[i] >> a.page_shift) * a.v_stride + (int64_t(d) << a.page_shift) + (slot_of[i] & (P - 1))] = vt[i][d];
    }
}

template <typename T, int D>
int launch_store_tile(const StoreArgs& a, hipStream_t s) {
    const unsigned tiles = unsigned((int64_t(a.s.num_tokens) + store_tile<D>() - 1) / store_tile<D>());
    MARS_LAUNCH((k_kv_store_tile<T, D>), dim3(tiles, unsigned(a.kv_heads)), dim3(256), 0, s, a);
    return MARS_OK;
}
template <typename T>
int launch_store(const StoreArgs& a, hipStream_t s) {
    if (a.s.num_tokens <= kStoreFew) {
        MARS_LAUNCH((k_kv_store<T>), dim3(unsigned(a.s.num_tokens)), dim3(256), 0, s, a);
        return MARS_OK;
    }
    return a.head_dim == 64 ? launch_store_tile<T, 64>(a, s) : a.head_dim == 128 ? launch_store_tile<T, 128>(a, s) : launch_store_tile<T, 256>(a, s);
}

int check_cache(const mars_reader& r, const mars_kv_cache& c) {
    MARS_CHECK(c.k_pages && c.v_pages, MARS_ERR_INVALID, "cache without pages");
    MARS_CHECK(c.num_pages > 0, MARS_ERR_INVALID, "cache of %d pages", c.num_pages);
    const int64_t dense = int64_t(r.d.kv_heads) * r.d.page_size * r.d.head_dim;
    for (const int64_t s : {c.k_page_stride, c.v_page_stride})
        MARS_CHECK(s == 0 || (s >= dense && s % 8 == 0), MARS_ERR_INVALID,
                   "page stride %lld: 0, or a multiple of 8 of at least %lld elements", (long long)s, (long long)dense);
    MARS_CHECK((reinterpret_cast<uintptr_t>(c.k_pages) | reinterpret_cast<uintptr_t>(c.v_pages)) % 16 == 0, MARS_ERR_INVALID,
               "cache pages are not aligned to 16 bytes");
    MARS_CHECK((reinterpret_cast<uintptr_t>(c.times) | reinterpret_cast<uintptr_t>(c.episodes)) % 16 == 0, MARS_ERR_INVALID,
               "cache times or episodes are not aligned to 16 bytes");
    return MARS_OK;
}

int check_rows(const char* what, const void* p, int64_t stride, int64_t width) {
    MARS_CHECK(stride >= width && stride % 8 == 0, MARS_ERR_INVALID, "%s stride %lld: a multiple of 8 of at least %lld elements",
               what, (long long)stride, (long long)width);
    MARS_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0, MARS_ERR_INVALID, "%s is not aligned to 16 bytes", what);
    return MARS_OK;
}

}  // namespace
}  // namespace mars

using namespace mars;

extern "C" {

int mars_reader_create(const mars_reader_desc* d, mars_reader** out) try {
    MARS_CHECK(d && out, MARS_ERR_INVALID, "null argument");
    *out = nullptr;
    MARS_CHECK(d->kv_heads >= 1 && d->q_heads >= d->kv_heads && d->q_heads % d->kv_heads == 0 && d->q_heads <= 4096,
               MARS_ERR_INVALID, "%d query heads over %d kv heads", d->q_heads, d->kv_heads);
    MARS_CHECK(d->q_heads / d->kv_heads <= 64, MARS_ERR_UNSUPPORTED, "%d query heads per kv head (at most 64)",
               d->q_heads / d->kv_heads);
    MARS_CHECK(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, MARS_ERR_UNSUPPORTED,
               "head_dim %d (64, 128 or 256)", d->head_dim);
    MARS_CHECK(d->dtype == MARS_DTYPE_F16 || d->dtype == MARS_DTYPE_BF16, MARS_ERR_UNSUPPORTED, "dtype %d", d->dtype);
    MARS_CHECK(d->page_size >= 16 && d->page_size <= 256 && (d->page_size & (d->page_size - 1)) == 0, MARS_ERR_UNSUPPORTED,
               "page_size %d (16, 32, 64, 128 or 256)", d->page_size);
    MARS_CHECK(d->rope_dim >= 0 && d->rope_dim <= d->head_dim && d->rope_dim % 16 == 0, MARS_ERR_INVALID,
               "rope_dim %d of head_dim %d (a multiple of 16)", d->rope_dim, d->head_dim);
    std::vector<int32_t> axis;
    if (d->rope_dim > 0) {
        MARS_CHECK(d->rope_axes >= 1 && d->rope_axes <= 3, MARS_ERR_INVALID, "%d position axes", d->rope_axes);
        MARS_CHECK(std::isfinite(d->rope_theta) && d->rope_theta > 1.0, MARS_ERR_INVALID, "rope_theta %g", d->rope_theta);
        for (int x = 0; x < d->rope_axes; ++x) {
            MARS_CHECK(d->rope_sections[x] >= 0 && d->rope_sections[x] <= d->rope_dim / 2, MARS_ERR_INVALID,
                       "rope section %d has %d frequencies", x, d->rope_sections[x]);
            axis.insert(axis.end(), size_t(d->rope_sections[x]), x);
        }
        MARS_CHECK(int32_t(axis.size()) == d->rope_dim / 2, MARS_ERR_INVALID, "rope sections hold %zu frequencies, rope_dim %d has %d",
                   axis.size(), d->rope_dim, d->rope_dim / 2);
    }
    auto r = std::make_unique<mars_reader>();
    MARS_TRY(require_device(&r->device));
    r->d = *d;
    while ((1 << r->page_shift) < d->page_size) ++r->page_shift;
    const int rc = [&]() -> int {
        if (d->rope_dim > 0) {
            const int half = d->rope_dim / 2;
            std::vector<uint64_t> f(static_cast<size_t>(half));
            for (int i = 0; i < half; ++i) {
                const long double w = std::pow((long double)(d->rope_theta), -2.0L * i / d->rope_dim) / 6.283185307179586476925286766559L;
                f[size_t(i)] = uint64_t(std::ldexp(w, 64) + 0.5L);
            }
            MARS_TRY(dmalloc(&r->freq, size_t(half)));
            MARS_TRY(dmalloc(&r->axis, size_t(half)));
            MARS_HIP(hipMemcpy(r->freq, f.data(), size_t(half) * sizeof(uint64_t), hipMemcpyHostToDevice));
            MARS_HIP(hipMemcpy(r->axis, axis.data(), size_t(half) * sizeof(int32_t), hipMemcpyHostToDevice));
        }
        r->few_slots = size_t(2) * few_groups(d->head_dim);
        const size_t rows = r->few_slots * kFewRows + (size_t(2) << kManyItemsLog2) * kManyRows;
        MARS_TRY(dmalloc(&r->part_o, rows * size_t(d->head_dim)));
        MARS_TRY(dmalloc(&r->part_ml, rows));
        MARS_TRY(dmalloc(&r->arrived, r->few_slots));
        MARS_HIP(hipMemset(r->arrived, 0, r->few_slots * sizeof(uint32_t)));
        MARS_HIP(hipDeviceSynchronize());
        return MARS_OK;
    }();
    if (rc != MARS_OK) {
        (void)mars_reader_destroy(r.release());
        return rc;
    }
    *out = r.release();
    return MARS_OK;
} catch (const std::bad_alloc&) {
    return set_error(MARS_ERR_NOMEM, "host allocation failed");
}

int mars_reader_destroy(mars_reader* r) {
    if (!r) return MARS_OK;
    (void)use_device(r->device);
    dfree(r->freq); dfree(r->axis); dfree(r->part_o); dfree(r->part_ml); dfree(r->arrived);
    delete r;
    return MARS_OK;
}

int mars_kv_plan(const mars_reader* r, const mars_kv_plan_args* a, void* stream) {
    MARS_CHECK(r && a && a->new_lens && a->cached_lens && a->block_table && a->free_pages && a->free_count && a->q_start &&
               a->kv_lens && a->free_count_out, MARS_ERR_INVALID, "null argument");
    MARS_CHECK(a->num_tokens == 0 || (a->slots && a->positions), MARS_ERR_INVALID, "null argument");
    MARS_CHECK(a->num_requests >= 1 && a->max_pages >= 1 && a->num_tokens >= 0 && a->free_capacity >= 0, MARS_ERR_INVALID,
               "%d requests, %d pages a row, %d tokens, %d free entries", a->num_requests, a->max_pages, a->num_tokens, a->free_capacity);
    MARS_CHECK(a->num_requests <= kMaxRequests, MARS_ERR_CAPACITY, "%d requests (at most %d)", a->num_requests, kMaxRequests);
    MARS_CHECK(a->free_count_out != a->free_count, MARS_ERR_INVALID, "free_count_out is free_count");
    // every workgroup reads the lengths for itself, while the first writes its outputs
    for (const int32_t* const out : {a->kv_lens, a->q_start, a->next_lens})
        MARS_CHECK(!out || (out != a->cached_lens && out != a->new_lens), MARS_ERR_INVALID, "%s is %s",
                   out == a->kv_lens ? "kv_lens" : out == a->q_start ? "q_start" : "next_lens", out == a->cached_lens ? "cached_lens" : "new_lens");
    MARS_CHECK(!a->next_lens || (a->next_lens != a->kv_lens && a->next_lens != a->q_start), MARS_ERR_INVALID, "next_lens is another output");
    MARS_TRY(use_device(r->device));
    const int64_t blocks = std::max<int64_t>(1, (int64_t(a->num_tokens) + kPlanTokens - 1) / kPlanTokens);
    MARS_LAUNCH(k_kv_plan, dim3(unsigned(blocks)), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), *a, r->page_shift);
    return MARS_OK;
}

int mars_kv_release(const mars_reader* r, const int32_t* done, int32_t* kv_lens, const int32_t* block_table, int32_t num_requests,
                    int32_t max_pages, int32_t* free_pages, int32_t* free_count, int32_t free_capacity, void* stream) {
    MARS_CHECK(r && done && kv_lens && block_table && free_pages && free_count, MARS_ERR_INVALID, "null argument");
    MARS_CHECK(num_requests >= 1 && max_pages >= 1 && free_capacity >= 0, MARS_ERR_INVALID,
               "%d requests, %d pages a row, %d free entries", num_requests, max_pages, free_capacity);
    MARS_CHECK(num_requests <= kMaxRequests, MARS_ERR_CAPACITY, "%d requests (at most %d)", num_requests, kMaxRequests);
    MARS_TRY(use_device(r->device));
    MARS_LAUNCH(k_kv_release, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), done, kv_lens, block_table, num_requests,
                max_pages, free_pages, free_count, free_capacity, r->page_shift);
    return MARS_OK;
}

int mars_kv_store(const mars_reader* r, const mars_kv_cache* c, const mars_kv_store_args* s, void* stream) {
    MARS_CHECK(r && s, MARS_ERR_INVALID, "null argument");
    MARS_CHECK(s->num_tokens >= 0, MARS_ERR_INVALID, "%d tokens", s->num_tokens);
    MARS_CHECK(s->q || s->k, MARS_ERR_INVALID, "neither q nor k");
    MARS_CHECK(!s->k == !s->v, MARS_ERR_INVALID, "k and v come together");
    const mars_reader_desc& d = r->d;
    StoreArgs a{};
    a.s = *s;
    if (s->q) {
        MARS_CHECK(s->q_out, MARS_ERR_INVALID, "q without q_out");
        MARS_TRY(check_rows("q", s->q, s->q_stride, int64_t(d.q_heads) * d.head_dim));
        MARS_TRY(check_rows("q_out", s->q_out, s->q_out_stride, int64_t(d.q_heads) * d.head_dim));
        MARS_CHECK(s->q != s->q_out || s->q_stride == s->q_out_stride, MARS_ERR_INVALID, "q_out is q with another stride");
    }
    if (s->k) {
        MARS_CHECK(c && s->slots, MARS_ERR_INVALID, "k and v need a cache and slots");
        MARS_TRY(check_cache(*r, *c));
        MARS_TRY(check_rows("k", s->k, s->k_stride, int64_t(d.kv_heads) * d.head_dim));
        MARS_TRY(check_rows("v", s->v, s->v_stride, int64_t(d.kv_heads) * d.head_dim));
        MARS_CHECK(!s->times || c->times, MARS_ERR_INVALID, "times for a cache without them");
        MARS_CHECK(!s->episodes || c->episodes, MARS_ERR_INVALID, "episodes for a cache without them");
        const int64_t dense = int64_t(d.kv_heads) * d.page_size * d.head_dim;
        a.k_pages = c->k_pages; a.v_pages = c->v_pages; a.times = c->times; a.eps = c->episodes;
        a.k_stride = c->k_page_stride ? c->k_page_stride : dense;
        a.v_stride = c->v_page_stride ? c->v_page_stride : dense;
        a.slots = int64_t(c->num_pages) << r->page_shift;
    }
    MARS_CHECK(d.rope_dim == 0 || s->positions, MARS_ERR_INVALID, "rotary heads need positions");
    if (s->num_tokens == 0) return MARS_OK;
    a.freq = r->freq; a.axis = r->axis;
    a.q_heads = d.q_heads; a.kv_heads = d.kv_heads; a.head_dim = d.head_dim; a.rope_dim = d.rope_dim; a.adjacent = d.rope_adjacent;
    a.page_shift = r->page_shift;
    MARS_TRY(use_device(r->device));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return d.dtype == MARS_DTYPE_F16 ? launch_store<_Float16>(a, st) : launch_store<__bf16>(a, st);
}

int mars_kv_attend(const mars_reader* r, const mars_kv_cache* c, const mars_kv_attend_args* s, void* stream) {
    MARS_CHECK(r && c && s && s->q && s->out && s->q_start && s->kv_lens && s->block_table, MARS_ERR_INVALID, "null argument");
    MARS_CHECK(s->num_requests >= 1 && s->max_pages >= 1 && s->num_tokens >= 0 && s->max_new >= 0, MARS_ERR_INVALID,
               "%d requests, %d pages a row, %d tokens, max_new %d", s->num_requests, s->max_pages, s->num_tokens, s->max_new);
    MARS_CHECK(s->num_requests <= kMaxRequests, MARS_ERR_CAPACITY, "%d requests (at most %d)", s->num_requests, kMaxRequests);
    MARS_TRY(check_cache(*r, *c));
    const mars_reader_desc& d = r->d;
    MARS_CHECK(int64_t(s->max_pages) * d.page_size <= (1 << 30), MARS_ERR_CAPACITY, "%d pages of %d tokens a row", s->max_pages, d.page_size);
    MARS_CHECK(int64_t(s->num_tokens) * d.q_heads <= INT32_MAX, MARS_ERR_CAPACITY, "%d tokens of %d heads", s->num_tokens, d.q_heads);
    MARS_TRY(check_rows("q", s->q, s->q_stride, int64_t(d.q_heads) * d.head_dim));
    MARS_TRY(check_rows("out", s->out, s->out_stride, int64_t(d.q_heads) * d.head_dim));
    MARS_CHECK(!s->decay || (s->q_times && c->times), MARS_ERR_INVALID, "decay needs q_times and the cache's times");
    MARS_CHECK(!s->q_episodes || c->episodes, MARS_ERR_INVALID, "q_episodes needs the cache's episodes");
    MARS_CHECK(std::isfinite(s->cap) && s->cap >= 0.0f, MARS_ERR_INVALID, "cap %g", double(s->cap));
    MARS_CHECK(std::isfinite(s->scale), MARS_ERR_INVALID, "scale %g", double(s->scale));
    if (s->num_tokens == 0) return MARS_OK;
    constexpr double kLog2e = 1.4426950408889634074;
    const double scale = s->scale == 0.0f ? 1.0 / std::sqrt(double(d.head_dim)) : double(s->scale);
    const int64_t dense = int64_t(d.kv_heads) * d.page_size * d.head_dim;
    AttendArgs a{};
    a.q = s->q; a.out = s->out; a.lse = s->lse;
    a.k_pages = c->k_pages; a.v_pages = c->v_pages;
    a.k_times = s->decay ? c->times : nullptr;
    a.k_eps = s->q_episodes ? c->episodes : nullptr;
    a.q_start = s->q_start; a.kv_lens = s->kv_lens; a.table = s->block_table;
    a.decay = s->decay; a.q_times = s->q_times; a.q_eps = s->q_episodes; a.prefix = s->prefix_lens;
    a.part_o = r->part_o; a.part_ml = r->part_ml; a.arrived = r->arrived;
    a.many_o = r->part_o + r->few_slots * kFewRows * size_t(d.head_dim);
    a.many_ml = r->part_ml + r->few_slots * kFewRows;
    a.q_stride = s->q_stride; a.out_stride = s->out_stride;
    a.k_stride = c->k_page_stride ? c->k_page_stride : dense;
    a.v_stride = c->v_page_stride ? c->v_page_stride : dense;
    a.q_flip = scale < 0.0 ? 0x80008000u : 0u;
    // finite: a score of 0 times an infinity would be NaN
    a.scale_log2 = float(std::min(std::fabs(kLog2e * scale), double(FLT_MAX)));
    a.cap_log2 = float(std::min(kLog2e * double(s->cap), double(FLT_MAX)));
    a.cap_rcp = s->cap > 0.0f ? float(std::clamp(1.0 / (kLog2e * double(s->cap)), double(FLT_MIN), double(FLT_MAX))) : 0.0f;
    a.requests = s->num_requests; a.max_pages = s->max_pages; a.tokens = s->num_tokens; a.num_pages = c->num_pages;
    a.q_heads = d.q_heads; a.kv_heads = d.kv_heads; a.group = d.q_heads / d.kv_heads;
    a.page_shift = r->page_shift;
    MARS_TRY(use_device(r->device));
    return launch_attend(*r, a, s->max_new, static_cast<hipStream_t>(stream));
}

}  // extern "C"
