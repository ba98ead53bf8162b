// ============================================================================
//  attend.hpp — attention of new tokens over the paged cache (mars_kv_attend and its forms): the kernels of
//  attend.hip, attend8.hip and attend_shared.hip.
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
//  m and sums exp2(s - m), fp32. m moves only when a score exceeds the one it was taken from by
//  more than 8 (in a wave of rows together), so the usual step needs no lane exchange and no
//  rescaling of O. For fp16 m lies 7 below that score: weights reach 2^15 of the type's 2^16, and
//  those as low as 2^-32 of the largest still count (2^-25 without; it takes no instruction more).
//  bf16 has fp32's range. The weights are rounded to 16 bits for the
//  second product (the matrix cores take no more at that rate); their sum is that of the
//  unrounded ones, fp32 as every other sum. A lane adds a step's weights up before it adds them to
//  the row's sum: one by one, weights below 2^-24 of that sum would be lost however many there are.
//
//  A cache of 8 bits (mars_kv_cache8) holds e4m3 values times a power of two a token and head. K's values become T's on the
//  way to the first product, exactly; V's too in the tiles of many rows, while few rows take them as bf16 and put the key's power of
//  two on its weight. Prefixes that several requests share (mars_kv_shared) are read in a launch of their own, whose
//  sums (O, m and the sum of weights, fp32) the requests' own launch goes on from.
// ============================================================================
#pragma once

#include "reader.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mars {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0.69314718055994530942f;
// s_waitcnt immediate (gfx9 encoding: vmcnt[3:0] and [15:14], expcnt[6:4], lgkmcnt[11:8]): all loads, all LDS accesses, or both, done
constexpr int kWaitVm0 = (7 << 4) | (15 << 8);
constexpr int kWaitVm0Lgkm0 = 7 << 4;
constexpr int kWaitLgkm0 = 15 | (3 << 14) | (7 << 4);
constexpr float kSlack = 8.0f;       // how far a score may exceed the one that the row's reference comes from

// Every load of this wave is done, those into LDS and the reads of LDS too (a product that takes one may come later: the
// buffer it was read from is refilled after this), and every other wave got here.
__device__ inline void tile_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitVm0Lgkm0);
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

// Scores x (base 2) under a cap: cap tanh(y) = x tanh(y) / y, y = x rcp. Up to |y| = 1/2 an odd polynomial (tanh(y) / y fitted
// in y^2 to 1.5e-8 of its value there, 1 at 0), exact to fp32's last bits however small the score beside the cap; beyond it
// cap (1 - 2 / (1 + e^2y)), whose error of 2^-22 cap is no more than 2^-20 of the score there (for scores of a few units it would
// be 6e-6 under a cap of 50, 0.09 under 1e6). k_attend_many looks first whether a wave's tile has a score above half the cap:
// 2 x 4,001 packed tokens 83.5 us where none has, 100 to 107 us where some have, 85.3 us with the second form alone.
__device__ inline float cap_near(float x, float rcp) {
    const float y = x * rcp, z = y * y;
    return x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0.017241491f, -0.053045493f), 0.13325879f), -0.33333144f), 1.0f);
}
__device__ inline float cap_any(float x, float cap, float rcp) {
    const float y = x * rcp;
    const float far = cap * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(2.88539008177792681472f * y)));
    return fabsf(y) < 0.5f ? cap_near(x, rcp) : far;
}

// A pointer the wave holds in SGPRs (the same in every lane), for loads of the form scalar base plus 32-bit offset: the
// compiler does not see what it is made of, or it would add the lane's offset to a part of it ahead of the loop and form
// 64-bit addresses in vector registers.
__device__ inline const char* uniform_ptr(const char* p) {
    uint64_t u = reinterpret_cast<uint64_t>(p);
    u = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(u >> 32)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(u)));
    asm volatile("" : "+s"(u));
    return reinterpret_cast<const char*>(u);
}
__device__ inline uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// 16 (or 4) bytes per lane from global memory straight into LDS: lane l's go to lds + 16 l (4 l) bytes.
__device__ inline void dma16(const void* g, void* lds) { __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0); }
__device__ inline void dma4(const void* g, void* lds) { __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void*)lds, 4, 0, 0); }

template <typename T> struct Vec;
template <> struct Vec<_Float16> {
    using v8 = f16x8;
    using v4 = f16x4;
    using v2 = f16x2;
    static constexpr uint32_t exp_mask = 0x7C00u;
    static constexpr float lift = 7.0f;                      // of the weights: 2^7 where the score is the reference's own
    __device__ static f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    __device__ static f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Vec<__bf16> {
    using v8 = bf16x8;
    using v4 = bf16x4;
    using v2 = bf16x2;
    static constexpr uint32_t exp_mask = 0x7F80u;
    static constexpr float lift = 0.0f;
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

// ---- e4m3 values times powers of two. The conversions are exact: store picks exponents that keep the values within T.
// (gfx950's conversions take the scale's exponent and nothing else of it, 0 for 2^-127 and 255 for NaN; their results are rounded to T.)
// Byte j of a word where a scale's exponent lies.
template <int J>
__device__ inline float scale_at(uint32_t w) { return __uint_as_float(J == 3 ? w >> 1 : w << (23 - 8 * J)); }
__device__ inline void scales16(u32x4 w, float (&s)[16]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s[4 * j] = scale_at<0>(w[j]);
        s[4 * j + 1] = scale_at<1>(w[j]);
        s[4 * j + 2] = scale_at<2>(w[j]);
        s[4 * j + 3] = scale_at<3>(w[j]);
    }
}
// The power of two of exponent byte j of a word, in fp32 (of 0 it is 0, of 255 an infinity).
__device__ inline float power(uint32_t w, int j) { return __uint_as_float((j == 3 ? w >> 1 : w << (23 - 8 * j)) & 0x7F800000u); }
// Two e4m3 values of a word (its upper half if HI) as T, times `scale`.
template <typename T, bool HI>
__device__ inline uint32_t from_e4m3(uint32_t w, float scale) {
    if constexpr (__is_same(T, _Float16)) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
// 8 values of one token: one scale. 8 values of one element: a scale each; the instruction takes one scale for both values of a
// pair, so it runs once with either, and a permutation takes the lower half of the one and the upper half of the other.
template <typename T>
__device__ inline u32x4 token_e4m3(uint32_t w0, uint32_t w1, float s) {
    return u32x4{from_e4m3<T, false>(w0, s), from_e4m3<T, true>(w0, s), from_e4m3<T, false>(w1, s), from_e4m3<T, true>(w1, s)};
}
template <typename T>
__device__ inline u32x4 element_e4m3(uint32_t w0, uint32_t w1, const float* s) {
    auto join = [](uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060100u); };
    return u32x4{join(from_e4m3<T, false>(w0, s[0]), from_e4m3<T, false>(w0, s[1])), join(from_e4m3<T, true>(w0, s[2]), from_e4m3<T, true>(w0, s[3])),
                 join(from_e4m3<T, false>(w1, s[4]), from_e4m3<T, false>(w1, s[5])), join(from_e4m3<T, true>(w1, s[6]), from_e4m3<T, true>(w1, s[7]))};
}
// Of 4 values: nonzero if one of them is NaN (e4m3 has no infinities).
__device__ inline uint32_t nan_e4m3(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
// The first `n` bytes of 16 kept (n may be negative or above 16), the others 0.
__device__ inline u32x4 first_bytes(u32x4 w, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] &= n >= 4 * j + 4 ? ~0u : n <= 4 * j ? 0u : (1u << (8 * (n - 4 * j))) - 1u;
    return w;
}

// What a kernel is compiled for: c8: the cache holds e4m3 values and exponents (mars_kv_cache8); share: it can run as one of
// the two phases of attention with shared prefixes (AttendArgs::phase).
template <bool C8, bool SHARE>
struct Form {
    static constexpr bool c8 = C8, share = SHARE;
};
using Plain = Form<false, false>;
using Shared = Form<false, true>;
using Held8 = Form<true, true>;

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

// The u-th of four values. (Of an array's elements the compiler makes a read from scratch memory at u.)
__device__ inline int pick4(int u, int p0, int p1, int p2, int p3) {
    const int even = u & 2 ? p2 : p0, odd = u & 2 ? p3 : p1;
    return u & 1 ? odd : even;
}

// A piece of a launch's work: a tile of rows of a request under one kv head, over the keys [k0, k1). Where several pieces
// share the tile (splits > 1), each writes a partial: piece 0 to slot0, piece i > 0 to slot1 + (i - 1) * slot_step.
struct Part {
    int32_t request, tile, head;
    int32_t row0, n, keys;     // the request's first row, its new tokens, its keys
    int32_t k0, k1;
    int32_t chunk;             // keys of a piece (k_attend_many)
    int32_t splits, slot, slot0, slot1, slot_step;
    int32_t skip;              // keys that another phase has read: the first piece begins there
    __device__ int slot_of(int i) const { return i == 0 ? slot0 : slot1 + (i - 1) * slot_step; }
};

struct SchedLds {
    int64_t sum[3][4];
    uint64_t wsum[4];
    Part part;
};

__device__ inline int64_t uniform(int64_t v) {
    return int64_t(uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint64_t(v) >> 32)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(v))));
}

// The same part in scalar registers (all threads read one copy).
__device__ inline Part uniform_part(const Part& p) {
    Part q;
    const int32_t* const from = reinterpret_cast<const int32_t*>(&p);
    int32_t* const to = reinterpret_cast<int32_t*>(&q);
#pragma unroll
    for (int i = 0; i < int(sizeof(Part) / 4); ++i) to[i] = __builtin_amdgcn_readfirstlane(from[i]);
    return q;
}

__device__ inline int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor((long long)v, o);
    return v;
}

// Request r, its rows in tiles of `bm`, and its keys; no tiles if the other of the two kernels serves it: requests of up
// to a.few_rows rows are k_attend_few's.
struct Request { int row0, n, tiles, keys, skip, at; };       // at: its row of the table

// Shared prefixes are read in two phases. The first takes each group for a request: all rows of its members over the
// prefix, which all of them see that have it cached, with the pages of the first of those; sums and references go to the state, a row
// and query head each. The second takes the requests again, from behind the prefix on and from that state.
__device__ inline int group_at(const AttendArgs& a, int g) { return min(max(a.group_start[g], 0), a.members); }
// Tokens of group g's prefix: whole pages, no more than a row of the table names.
__device__ inline int shared_of(const AttendArgs& a, int g) {
    return int(min(int64_t(max(a.shared_lens[g], 0)), int64_t(a.max_pages) << a.page_shift)) >> a.page_shift << a.page_shift;
}
// Whether request r has `s` tokens cached, its new ones apart (one that was not served has no keys at all).
__device__ inline bool has_cached(const AttendArgs& a, int r, int s) {
    const int row0 = max(a.q_start[r], 0), n = max(0, min(a.q_start[r + 1], a.tokens) - row0);
    const int64_t keys = min(int64_t(a.kv_lens[r]), int64_t(a.max_pages) << a.page_shift);
    return s <= keys - n;
}
// The first of requests [first, end) that has `s` tokens cached: its row of the table names the prefix, that of one before it need
// not. `end`: none. Four are looked at together, and mostly the first is it.
__device__ inline int holder_of(const AttendArgs& a, int first, int end, int s) {
    constexpr int U = 4;
    for (int m = first; m < end; m += U) {
        bool has[U];
#pragma unroll
        for (int u = 0; u < U; ++u) has[u] = has_cached(a, min(m + u, end - 1), s);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (has[u]) return min(m + u, end - 1);
    }
    return end;
}
// The second phase's skips, by one workgroup of the first: 0 for a request in no group, or that has not the whole prefix cached:
// it reads everything itself. lds: room for the groups' starts.
__device__ inline void find_skips(const AttendArgs& a, int32_t* lds) {
    for (int g = int(threadIdx.x); g <= a.requests; g += 256) lds[g] = a.group_start[g];
    __syncthreads();
    for (int r = int(threadIdx.x); r < a.members; r += 256) {
        int lo = 0, hi = a.requests;                        // the last group that begins at or before r
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (lds[mid] <= r) lo = mid; else hi = mid;
        }
        const int s = lds[lo] <= r && r < lds[lo + 1] ? shared_of(a, lo) : 0;
        a.skips[r] = has_cached(a, r, s) ? s : 0;
    }
}

template <bool FEW, typename F>
__device__ inline Request request_of(const AttendArgs& a, int r) {
    constexpr int bm = FEW ? kFewRows : kManyRows;
    Request q{0, 0, 0, 0, 0, r};
    if (r >= a.requests) return q;
    int start, end, len;
    if (F::share && a.phase == 1) {
        const int first = group_at(a, r), behind = max(group_at(a, r + 1), first);
        start = a.q_start[first];
        end = a.q_start[behind];
        len = shared_of(a, r);
        q.at = min(first, a.members - 1);
        if (len == 0) return q;
        const int holder = holder_of(a, first, behind, len);
        if (holder == behind) return q;                      // every member reads everything itself
        q.at = holder;
    } else {
        start = a.q_start[r];
        end = a.q_start[r + 1];
        len = a.kv_lens[r];
    }
    q.row0 = max(start, 0);
    q.n = max(0, min(end, a.tokens) - q.row0);
    const int rows = q.n * a.group;
    if ((rows <= a.few_rows) != FEW) return q;
    q.tiles = (rows + bm - 1) / bm;
    q.keys = int(min(int64_t(max(len, 0)), int64_t(a.max_pages) << a.page_shift));
    if (F::share && a.phase == 2) q.skip = min(a.skips[r], q.keys);
    return q;
}
// Where the pieces of a phase 1 row's sums lie, if phase 2 joins them (AttendArgs::defer): rows of part_o and part_ml.
__device__ inline int64_t state_row(const AttendArgs& a, int64_t row, int hq) { return row * a.q_heads + hq; }
__device__ inline i32x4 one_piece(const AttendArgs& a, int64_t at) { return i32x4{int32_t(a.state_row0 + at), 0, 0, 1}; }

// Keys [0, limit) that row i of a request's n may see.
template <typename F>
__device__ inline int limit_of(const AttendArgs& a, int keys, int n, int i, int prefix) {
    if (F::share && a.phase == 1) return keys;
    return min(max(keys - n + i + 1, prefix), keys);
}
template <typename F>
__device__ inline int prefix_of(const AttendArgs& a, int request, int keys) {
    return a.prefix && !(F::share && a.phase == 1) ? min(max(a.prefix[request], 0), keys) : 0;
}

// Workgroup b's item of k_attend_many, from the lengths alone: every workgroup of 256 threads sums the launch's tiles
// and work (key steps of 32 over all tiles), cuts the keys into chunks, and finds the request that its number falls to.
// Where there are fewer tiles than three quarters of the workgroups that the CUs hold, chunks of a 2^9-th of all the
// tiles' keys (2 x 511 tokens over 2,500 keys, 256 tiles: 77 us, 104 us whole; in 2^8 or 2^10 chunks 79 and 95 us, and
// 511 tokens over 20,511 keys 208 us, 275 and 238); with more tiles, no chunk has to be smaller than a CU's share of the
// work (768 tiles of causal rows up to 4,001 keys: 112 us whole, 144 us cut once).
// A tile has at most 2 L / C chunks where it has two, and C is at least sum(L) / 2^9 by either rule: 2^10 partial slots.
// The launch has enough workgroups for every item (fewer than 2^31); the last ones may find none. JOIN: the items are
// the blocks of kJoinRows rows of the tiles in several pieces instead, the block's number in Part::slot.
// Rows of a tile that a workgroup of k_attend_join takes: with caches of 8 bits and shared prefixes, where there are few tiles (which
// are in many pieces then), as many as it has threads for (see launch_dim).
template <typename F>
__device__ __host__ inline int join_rows_of(const AttendArgs& a) { return F::share ? a.join_rows : kJoinRows; }
template <bool JOIN, typename F>
struct ManySched {
    const AttendArgs& a;
    SchedLds& sh;
    Request q;                 // this thread's, of the 256 that are looked at: r0 on
    int r0;
    uint32_t chunk0, chunk, splits, each, items, mine, part;
    uint32_t before, end, parts_end;   // items before these 256 and up to their end; partial slots up to there

    // false: no request is k_attend_many's. All threads call it, and find(), together.
    __device__ ManySched(const AttendArgs& args, SchedLds& lds) : a(args), sh(lds) {}
    __device__ bool start() {
        const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
        q = request_of<false, F>(a, tid);
        // the rows of a tile see L - n / 2 keys on average (not less than half of the L keys)
        int64_t full = 0, mean = 0, tiles = 0;
        auto add = [&](const Request& x) {
            const int len = F::share ? x.keys - x.skip : x.keys, cut = F::share && a.phase == 1 ? 0 : x.n / 2;
            full += int64_t(x.tiles) * ((len + 31) >> 5);
            mean += int64_t(x.tiles) * ((max(len - cut, len / 2) + 31) >> 5);
            tiles += x.tiles;
        };
        add(q);
        for (int r = 256; r < a.requests; r += 256) add(request_of<false, F>(a, r + tid));
        full = wave_sum(full);
        mean = wave_sum(mean);
        tiles = wave_sum(tiles);
        if (lane == 0) { sh.sum[0][wave] = full; sh.sum[1][wave] = mean; sh.sum[2][wave] = tiles; }
        __syncthreads();
        int64_t sums[3];
#pragma unroll
        for (int x = 0; x < 3; ++x) sums[x] = (sh.sum[x][0] + sh.sum[x][1] + sh.sum[x][2] + sh.sum[x][3]) * a.kv_heads;
        if (sums[2] == 0) return false;
        constexpr int64_t slots = 1 << kManyItemsLog2;
        const int64_t per = sums[2] < slots * 3 / 4 ? (sums[0] * 32 + slots - 1) / slots : (sums[1] * 64 + slots - 1) / slots;
        chunk0 = (uint32_t(min(max(per, int64_t(kMinChunk)), int64_t(INT32_MAX) - 255)) + 255) & ~255u;
        r0 = 0;
        end = parts_end = 0;
        scan();
        return true;
    }
    // The items of requests r0 .. r0 + 255, whose lengths are in q.
    __device__ void scan() {
        const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6;
        // no more than kMaxSplits chunks a request
        const uint32_t len = uint32_t(F::share ? q.keys - q.skip : q.keys);
        chunk = max(chunk0, (len + kMaxSplits * 256 - 1) / (kMaxSplits * 256) * 256);
        splits = max(1u, (len + chunk - 1) / chunk);
        const uint32_t heads = uint32_t(q.tiles) * uint32_t(a.kv_heads), parts = splits > 1 ? heads * splits : 0;
        each = JOIN ? (splits > 1 ? kManyRows / join_rows_of<F>(a) : 0) : splits;
        items = heads * each;
        uint32_t xi = items, xp = parts;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t yi = __shfl_up(xi, unsigned(o)), yp = __shfl_up(xp, unsigned(o));
            if (lane >= o) { xi += yi; xp += yp; }
        }
        __syncthreads();
        if (lane == 63) sh.wsum[wave] = (uint64_t(xi) << 32) | xp;
        __syncthreads();
        before = end;
        mine = end + xi - items;
        part = parts_end + xp - parts;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint64_t s = sh.wsum[w];
            if (w < wave) { mine += uint32_t(s >> 32); part += uint32_t(s); }
            end += uint32_t(s >> 32);
            parts_end += uint32_t(s);
        }
    }
    // Item b into *out, for calls with rising b; false: there are not so many.
    __device__ bool find(uint32_t b, Part* out) {
        while (b >= end) {
            r0 += 256;
            if (r0 >= a.requests) return false;
            q = request_of<false, F>(a, r0 + int(threadIdx.x));
            scan();
        }
        __syncthreads();                                     // the item before has been read
        if (b >= mine && b - mine < items) {
            const uint32_t local = b - mine, tile_head = local / each, tile = tile_head / uint32_t(a.kv_heads);
            const int32_t split = int32_t(local - tile_head * each), c = int32_t(min(chunk, uint32_t(INT32_MAX / 2)));
            Part& pt = sh.part;
            pt.request = F::share ? q.at : r0 + int(threadIdx.x);
            pt.tile = int32_t(uint32_t(q.tiles) - 1 - tile); // later rows see more keys: first
            pt.head = int32_t(tile_head - tile * uint32_t(a.kv_heads));
            pt.row0 = q.row0;
            pt.n = q.n;
            pt.keys = q.keys;
            pt.chunk = c;
            pt.skip = F::share ? q.skip : 0;
            pt.k0 = pt.skip + split * c;
            pt.k1 = min(q.keys, pt.k0 + c);
            pt.splits = int32_t(splits);
            pt.slot0 = int32_t(part + tile_head * splits);
            pt.slot1 = pt.slot0 + 1;
            pt.slot_step = 1;
            pt.slot = JOIN ? split : pt.slot0 + split;
        }
        __syncthreads();
        *out = uniform_part(sh.part);
        return true;
    }
};

// Partials pass between workgroups of one launch, on any XCD: as relaxed atomics of agent scope, which go through to
// where every XCD sees them, the writers' completed before they count themselves in. (Plain stores and a fence at agent
// scope write back and drop a whole L2 per workgroup: 64 single tokens over 4,096 keys took 497 us so.)
// A wave's stores of such a kind are fast where they fill whole lines, so rows of O are laid out in LDS first.
__device__ inline void put_part(float* p, float2 v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), uint64_t(__float_as_uint(v.y)) << 32 | __float_as_uint(v.x), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
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

// This wave's stores have reached where every XCD sees them. (A workgroup barrier alone does not wait for that: plain
// accesses of one CU meet in its L1, which these pass by.)
__device__ inline void stores_done() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    asm volatile("" ::: "memory");
}

// Joins the pieces of a tile of k_attend_few: the rows' references and weights first (in LDS, 16 threads a row), then 4
// elements a thread, the partials of 16 pieces on the way together.
// Each sum is taken in the order of the pieces by one thread, or by up to 4 threads whose parts are then added in
// their order: the same bits whoever does it.
struct JoinLds {
    int last;
    float scale[kFewRows], lse[kFewRows];
    float2 w[kMaxSplits][kFewRows];                         // (max, sum) of a piece, then its weight
    __attribute__((aligned(16))) float part[4][128 * 4];
    // join_state: a row's pieces, reference and sum; the joined rows, D + 4 floats each, in place of the weights
    i32x4 where[kFewRows];
    float2 ml[kFewRows];
    __device__ float* sum() { return reinterpret_cast<float*>(&w[0][0]); }
};
template <typename T, int D, typename F>
__device__ void join_rows(const AttendArgs& a, const Part& it, JoinLds& lds) {
    const int tid = int(threadIdx.x), splits = it.splits;
    const int rows = min(kFewRows, it.n * a.group - it.tile * kFewRows), units = rows * (D / 4);
    for (int x = tid; x < splits * kFewRows; x += 256)
        if (x % kFewRows < rows) lds.w[x / kFewRows][x % kFewRows] = get_part2(a.part_ml + int64_t(it.slot_of(x / kFewRows)) * kFewRows + x % kFewRows);
    __syncthreads();
    {
        const int rr = tid >> 4, s0 = tid & 15;
        float top = -kInf, sum = 0.0f;
        if (rr < rows)
            for (int s = s0; s < splits; s += 16) top = fmaxf(top, lds.w[s][rr].x);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (rr < rows)
            for (int s = s0; s < splits; s += 16) {
                const float2 p = lds.w[s][rr];
                const float f = p.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(p.x - top);
                sum += f * p.y;
                lds.w[s][rr].x = f;
            }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor(sum, o);
        if (rr < rows && s0 == 0) {
            lds.scale[rr] = top == -kInf ? -kInf : 1.0f / sum;       // -inf: the row sees no key
            lds.lse[rr] = top == -kInf ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
            if (F::share && a.phase == 1)
                a.state_ml[(int64_t(it.row0) + (it.tile * kFewRows + rr) / a.group) * a.q_heads + it.head * a.group + (it.tile * kFewRows + rr) % a.group] =
                    make_float2(top, top == -kInf ? 0.0f : sum);
        }
    }
    __syncthreads();
    int ways = 1;                                            // threads per unit of 4 elements
    while (ways < 4 && units * ways * 2 <= 256 && ways < splits) ways *= 2;
    const int per = 256 / ways, w = tid / per;
    constexpr int U = 16;
    for (int base = 0; base < units; base += per) {
        const int e = base + tid % per, rr = e / (D / 4), d4 = e % (D / 4);
        f32x4 sum = {0, 0, 0, 0};
        if (e < units) {
            const float* const po = a.part_o + rr * D + d4 * 4;
            for (int s = w; s < splits; s += U * ways) {
                f32x4 o[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + u * ways < splits) o[u] = get_part4(po + int64_t(it.slot_of(s + u * ways)) * kFewRows * D);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + u * ways < splits) sum += lds.w[s + u * ways][rr].x * o[u];
            }
        }
        if (ways > 1) {                                      // then every thread has one unit or none
            *reinterpret_cast<f32x4*>(&lds.part[w][(tid % per) * 4]) = sum;
            __syncthreads();
            for (int v = 1; v < ways && w == 0; ++v) sum += *reinterpret_cast<const f32x4*>(&lds.part[v][tid * 4]);
        }
        if (e >= units || w) continue;
        const int mm = it.tile * kFewRows + rr, ii = mm / a.group, hh = it.head * a.group + mm - ii * a.group;
        if (F::share && a.phase == 1) {
            *reinterpret_cast<f32x4*>(a.state_o + ((int64_t(it.row0) + ii) * a.q_heads + hh) * D + d4 * 4) = sum;
            continue;
        }
        const float scale = lds.scale[rr];
        typename Vec<T>::v4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = scale == -kInf ? T(0.0f) : T(sum[j] * scale);
        *reinterpret_cast<typename Vec<T>::v4*>(static_cast<T*>(a.out) + (int64_t(it.row0) + ii) * a.out_stride + int64_t(hh) * D + d4 * 4) = o;
        if (a.lse && d4 == 0) a.lse[(int64_t(it.row0) + ii) * a.q_heads + hh] = lds.lse[rr];
    }
}

// Joins the pieces of the first phase's sums of a tile's rows, as join_rows does: into lds.sum(), the lane's row's (reference, sum of
// weights) returned. All threads call it; the LDS is free again after the next barrier.
template <int D, int U>
__device__ float2 join_state(const AttendArgs& a, const Part& it, JoinLds& lds) {
    const int tid = int(threadIdx.x), rows = min(kFewRows, it.n * a.group - it.tile * kFewRows), units = rows * (D / 4);
    auto row_of = [](i32x4 where, int s) { return int64_t(s == 0 ? where[0] : where[1] + (s - 1) * where[2]); };
    {
        const int rr = tid >> 4, s0 = tid & 15, m = it.tile * kFewRows + rr;
        i32x4 where = {0, 0, 0, 0};
        if (rr < rows) {
            const int64_t at = state_row(a, int64_t(it.row0) + m / a.group, it.head * a.group + m % a.group);
            where = a.defer ? a.state_at[at] : one_piece(a, at);
        }
        float top = -kInf, sum = 0.0f;
        for (int s1 = s0; s1 < where[3]; s1 += 64) {         // four on the way together
            float2 p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u] = s1 + 16 * u < where[3] ? a.part_ml[row_of(where, s1 + 16 * u)] : make_float2(-kInf, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (s1 + 16 * u < where[3]) lds.w[s1 + 16 * u][rr] = p[u];
                top = fmaxf(top, p[u].x);
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
        for (int s = s0; s < where[3]; s += 16) {
            const float2 p = lds.w[s][rr];
            const float f = p.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(p.x - top);
            sum += p.x == -kInf ? 0.0f : f * p.y;
            lds.w[s][rr].x = f;
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor(sum, o);
        if (s0 == 0) {
            lds.where[rr] = where;
            lds.ml[rr] = make_float2(top, sum);
        }
    }
    __syncthreads();
    int ways = 1;                                            // threads per unit of 4 elements
    while (ways < 4 && units * ways * 2 <= 256) ways *= 2;
    const int per = 256 / ways, w = tid / per;
    constexpr int N = (kFewRows * (D / 4) + 255) / 256;     // U: pieces on the way together
    f32x4 sum[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = n * per + tid % per, rr = e / (D / 4), d4 = e % (D / 4);
        sum[n] = f32x4{0, 0, 0, 0};
        if (e >= units) continue;
        const i32x4 where = lds.where[rr];
        for (int s = w; s < where[3]; s += U * ways) {
            f32x4 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * ways < where[3]) o[u] = *reinterpret_cast<const f32x4*>(a.part_o + row_of(where, s + u * ways) * D + d4 * 4);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * ways < where[3]) sum[n] += lds.w[s + u * ways][rr].x * o[u];
        }
    }
    if (ways > 1) {                                          // then every thread has one unit or none
        *reinterpret_cast<f32x4*>(&lds.part[w][(tid % per) * 4]) = sum[0];
        __syncthreads();
        for (int v = 1; v < ways && w == 0; ++v) sum[0] += *reinterpret_cast<const f32x4*>(&lds.part[v][tid * 4]);
    }
    __syncthreads();                                         // the weights are read
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = n * per + tid % per;
        if (e < units && w == 0) *reinterpret_cast<f32x4*>(&lds.sum()[e / (D / 4) * (D + 4) + e % (D / 4) * 4]) = sum[n];
    }
    __syncthreads();
    return lds.ml[tid & 15];
}

// Called by every thread of a workgroup that wrote one piece's partial: the tile's last workgroup to arrive joins them.
template <typename T, int D, typename F>
__device__ void join_last(const AttendArgs& a, const Part& it, JoinLds& lds) {
    stores_done();
    __syncthreads();
    if (threadIdx.x == 0)
        lds.last = __hip_atomic_fetch_add(&a.arrived[it.slot0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(it.splits - 1);
    __syncthreads();
    if (!lds.last) return;
    if (threadIdx.x == 0) __hip_atomic_store(&a.arrived[it.slot0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    join_rows<T, D, F>(a, it, lds);
}

// The steps of `STEP` keys that some row of the workgroup can see by its episode, of a window of kWindow steps: the
// others are neither read nor computed. A key is read if its episode is negative, some row's is, or it lies between the
// least and the greatest of the rows' (exact where the rows ask within one episode, as single tokens do, and where
// episodes follow each other). Entry: the step within the window, kMixed added where rows and keys have to be compared
// one by one.
constexpr int kWindow = 128, kMixed = 1 << 15;
struct StepLds {
    uint16_t flag[kWindow], list[kWindow];
    int count;
    int eq_min[4], eq_max[4];                                // of the waves' rows
};
template <int STEP>
__device__ int list_steps(const AttendArgs& a, int request, int last_page, int k0, int k1, int w0, int steps, int eq_min, int eq_max, StepLds& lds) {
    const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int n = min(kWindow, steps - w0);
    __syncthreads();                                         // the list before is done with
    constexpr int U = 8;                                     // steps whose loads are on the way together
    for (int t0 = wave; t0 < n; t0 += 4 * U) {
        int64_t page[U];
        int e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = min(k0 + (w0 + t0 + 4 * u) * STEP + lane, k1 - 1);
            const int id = a.table[int64_t(request) * a.max_pages + min(key >> a.page_shift, last_page)];
            page[u] = uint32_t(id) < uint32_t(a.num_pages) ? id : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = min(k0 + (w0 + t0 + 4 * u) * STEP + lane, k1 - 1);
            e[u] = a.k_eps[(page[u] << a.page_shift) + (key & ((1 << a.page_shift) - 1))];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t0 + 4 * u;
            const bool in = lane < STEP && k0 + (w0 + t) * STEP + lane < k1;
            const bool any = __any(in && (eq_min < 0 || e[u] < 0 || (e[u] >= eq_min && e[u] <= eq_max)));
            const bool alike = eq_max < 0 || __all(!in || e[u] < 0) || (eq_min == eq_max && __all(!in || e[u] == eq_min));
            if (lane == 0 && t < n) lds.flag[t] = any ? uint16_t(t + (alike ? 0 : kMixed)) : uint16_t(0xFFFF);
        }
    }
    __syncthreads();
    if (wave == 0) {
        int count = 0;
        for (int t0 = 0; t0 < n; t0 += 64) {
            const uint16_t f = t0 + lane < n ? lds.flag[t0 + lane] : uint16_t(0xFFFF);
            const uint64_t on = __ballot(f != 0xFFFF);
            if (f != 0xFFFF) lds.list[count + __popcll(on & ((1ull << lane) - 1))] = f;
            count += __popcll(on);
        }
        if (lane == 0) lds.count = count;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(lds.count);
}

// Infinities and NaN among the values. A weight of 0 times one of them is NaN, so where some row of a step does not see
// some key, the products take them as 0, and the workgroup, once its rows are written, adds them to the rows that do see
// them here: every (row, element) looks through the keys [k0, k1). (Rare, and slow.)
template <typename T, int D, int BM, typename F>
__device__ void add_not_finite(const AttendArgs& a, const Part& it, int prefix) {
    const int row0 = it.row0, n = it.n, keys = it.keys;
    const int valid = min(BM, n * a.group - it.tile * BM);
    for (int e = int(threadIdx.x); e < valid * D; e += 256) {
        const int rr = e / D, d = e % D, m = it.tile * BM + rr, i = m / a.group, hq = it.head * a.group + m - i * a.group;
        const int64_t row = int64_t(row0) + i;
        const int end = min(it.k1, limit_of<F>(a, keys, n, i, prefix));
        float sum = 0.0f;
        for (int k = it.k0; k < end; ++k) {
            const int id = a.table[int64_t(it.request) * a.max_pages + (k >> a.page_shift)];
            const int64_t page = uint32_t(id) < uint32_t(a.num_pages) ? id : 0;
            const int off = k & ((1 << a.page_shift) - 1);
            if (a.k_eps) {
                const int ek = a.k_eps[(page << a.page_shift) + off], eq = a.q_eps[row];
                if (!(ek < 0 || eq < 0 || ek == eq)) continue;
            }
            const int64_t at = page * a.v_stride + ((int64_t(it.head) * D + d) << a.page_shift) + off;
            if constexpr (F::c8) {
                // what the products left out: k_attend_few, which takes values as they are held, NaN; k_attend_many what is not finite as T
                const uint32_t b = static_cast<const uint8_t*>(a.v_pages)[at], e = a.v_scales[((page * a.kv_heads + it.head) << a.page_shift) + off];
                const float v = float(__builtin_bit_cast(typename Vec<T>::v2, from_e4m3<T, false>(b, scale_at<0>(e)))[0]);
                if (BM == kFewRows ? (b & 0x7Fu) == 0x7Fu || e == 255u : !(fabsf(v) < kInf)) sum += v;
            } else {
                const float v = float(static_cast<const T*>(a.v_pages)[at]);
                if (!(fabsf(v) < kInf)) sum += v;
            }
        }
        if (sum == 0.0f) continue;
        if (F::share && a.phase == 1 && it.splits == 1) {
            a.state_o[(row * a.q_heads + hq) * D + d] += sum;
        } else if (it.splits == 1) {
            T* const o = static_cast<T*>(a.out) + row * a.out_stride + int64_t(hq) * D + d;
            *o = T(float(*o) + sum);
        } else {
            float* const o = (BM == kFewRows ? a.part_o : a.many_o) + (int64_t(it.slot) * BM + rr) * D + d;
            if (BM == kFewRows) {
                const float was = __hip_atomic_load(o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(o, was + sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            } else {
                *o += sum;
            }
        }
    }
}

// ---- few rows: 16 at a time, keys straight from the cache to registers -----------------
// Bound by the cache's bytes. A piece's steps go to 4 waves in turn, and a wave keeps its next step's K and V on the way to
// registers (16 bytes a lane: K rows over the elements, V rows over the step's keys) while it computes this one: 8 waves of
// a CU have 128 KB in flight for heads of 128. The waves' sums are joined at the end. bf16, 32/8 heads of 128:
// 64 single tokens over 780 to 7,800 keys (1.15 GB) 215 us, 5.4 TB/s; one over 131,072 (0.54 GB) 110 us.
// Steps of 64 keys spill: 228 and 119 us (first case with cap and decay: 288 and 225 us).
// Of 8 bits a step is 64 keys, the same bytes: the first case (0.58 GB) 122 us, 4.8 TB/s, the other (0.27 GB) 66 us; twice the scores
// and weights a byte: vector units busy 36% of the cycles, and waves wait 41% of their time for data, 35% for an instruction's turn.
template <int D, typename F>
struct FewLds {
    union {
        struct { float ml[4][16][2]; __attribute__((aligned(16))) float ob[2][16][D + 4]; } wave;
        JoinLds join;
        StepLds steps;
    };
    int any_dirty;
    u32x4 q[F::c8 && D == 128 ? D / 32 * 64 : 1];           // see kLean
    u32x4 row[F::c8 && D == 128 ? kFewRows : 1];                     // of a row: decay and time of the query (fp32), limit, episode
};
// Waves a SIMD of the kernels of few rows, as their registers allow.
template <int D, typename F, bool EXTRA>
constexpr int few_waves() { return D > 128 ? 1 : D == 128 ? 2 : F::c8 ? 2 : 3; }
constexpr float kLift8 = -1.0f;     // Vec::lift of k_attend_few over 8 bits
template <typename F>
constexpr int few_step() { return F::c8 ? 64 : 32; }

template <typename T, int D, bool EXTRA, bool CAP, typename F>
__device__ void few_part(const AttendArgs& a, const Part& it, FewLds<D, F>& lds) {
    using V = typename Vec<T>::v8;
    // The second product's type. Of 8 bits it is bfloat16 whatever T is: e4m3 values are exact in it, and a key's power of two goes to its
    // weight, which needs fp32's range. (Converted into T instead, a pair of one element's values takes three instructions for one.)
    using W = std::conditional_t<F::c8, __bf16, T>;
    using VW = typename Vec<W>::v8;
    // A weight takes its key's power of two, up to 2^120: kept to 2^7, so that the product stays in fp32's range (infinity times 0 is NaN).
    constexpr float lift = F::c8 ? kLift8 : Vec<W>::lift;
    // a step's keys; its groups of 16; keys of a lane, in NB blocks of the first product and NT fragments of the second
    constexpr int kStep = few_step<F>(), NG = kStep / 16, NK = kStep / 4, NB = NK / 4, NT = NK / 8, KC = D / 32, VB = D / 16;
    // With times on the way the registers do not suffice for 64 keys a step of heads of 128: there q, which the four waves have in
    // common, and the terms of the rows are read from LDS in every step, and a lane's places in K and V are found anew (64
    // single tokens over 2,000 to 4,000 keys, decayed, 95 us; 108 with 22 values a lane in scratch memory)
    constexpr bool kLean = F::c8 && EXTRA && D == 128;
    int tid = int(threadIdx.x);
    asm volatile("" : "+v"(tid));                          // nothing of a piece is kept in registers for the next
    int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int col = lane & 15, h = lane >> 4;
    const int r = it.request, head = it.head, row0 = it.row0, n = it.n, keys = it.keys, P1 = (1 << a.page_shift) - 1;
    if (tid == 0) lds.any_dirty = 0;                        // read after barriers
    int m = it.tile * kFewRows + col;                       // this lane's row: token i, head of the group
    bool row_ok = m < n * a.group;
    int i = row_ok ? m / a.group : 0, hq = head * a.group + (row_ok ? m - i * a.group : 0);
    int64_t row = int64_t(row0) + i;
    const int prefix = prefix_of<F>(a, r, keys);
    const int limit = row_ok ? limit_of<F>(a, keys, n, i, prefix) : 0;         // keys [0, limit) may be seen
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
    const bool listed = EXTRA && a.k_eps;
    int eq_min = row_ok ? eq : INT32_MAX, eq_max = row_ok ? eq : INT32_MIN;
    if (listed) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            eq_min = min(eq_min, __shfl_xor(eq_min, o));
            eq_max = max(eq_max, __shfl_xor(eq_max, o));
        }
    }
    if constexpr (F::share) {                               // the same in every lane
        eq_min = __builtin_amdgcn_readfirstlane(eq_min);
        eq_max = __builtin_amdgcn_readfirstlane(eq_max);
    }
    const int k0 = it.k0, k1 = min(it.k1, hi);
    const int steps = k1 > k0 ? (k1 - k0 + kStep - 1) / kStep : 0;

    const TablePtr table = table_row(a, r);
    const int last_page = keys > 0 ? (keys - 1) >> a.page_shift : 0;
    // K: A row `col` of block b holds key NK (col / 4) + 4 b + col % 4 of a step, so that registers 4 b + j of S hold key NK h + 4 b + j
    const int kkey = NK * (col >> 2) + (col & 3), kg = kkey >> 4, kin = kkey & 15;            // group of 16 keys, key within it (b = 0)
    int pages[NG], v_pages[NG];                             // of the step on the way: K's, and (loaded later) V's
    auto find_pages = [&](int s) {
#pragma unroll
        for (int u = 0; u < NG; ++u) pages[u] = page_of(a, table, k0 + s * kStep + u * 16, last_page);
    };
    // what a lane has on the way of a step: 16 bytes are 8 elements of a key (keys of an element), or 16 of them in e4m3
    constexpr int KL = F::c8 ? KC / 2 : KC, VL = VB;
    u32x4 kf[NB][KL], vf[VL], kx, vx;                       // kx, vx: exponents of the 16 keys of a lane's group of K, and of V
    f32x4 tk[NB];
    i32x4 ek[NB];
    auto load_k = [&](int s) {
        const int kt = k0 + s * kStep;
        if constexpr (F::c8) {
            const int ln = kLean ? int(here(uint32_t(lane))) : lane, col = ln & 15, h = ln >> 4, kg = col >> 2, kin = col & 3;
            const int pg = pick4(kg, pages[0], pages[1], pages[2], pages[3]), off = (kt + kg * 16) & P1;
            const uint8_t* const p = static_cast<const uint8_t*>(a.k_pages) + pg * a.k_stride + ((int64_t(head) << a.page_shift) + off + kin) * D + h * 16;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int c = 0; c < KL; ++c) kf[b][c] = *reinterpret_cast<const u32x4*>(p + b * 4 * D + c * 64);
            kx = *reinterpret_cast<const u32x4*>(a.k_scales + ((int64_t(pg) * a.kv_heads + head) << a.page_shift) + off);
        } else {
            const T* const kp = static_cast<const T*>(a.k_pages) + ((int64_t(head) << a.page_shift) + kin) * D + h * 8;
            const int64_t o0 = pages[0] * a.k_stride + int64_t(kt & P1) * D, o1 = pages[1] * a.k_stride + int64_t((kt + 16) & P1) * D;
            const T* const p = kp + (kg ? o1 : o0);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int c = 0; c < KL; ++c) kf[b][c] = load16<u32x4>(p + b * 4 * D + c * 32);
        }
    };
    auto load_v = [&](int s) {
        const int kt = k0 + s * kStep;
        int64_t slot;
        if constexpr (F::c8) {
            const int ln = kLean ? int(here(uint32_t(lane))) : lane, col = ln & 15, h = ln >> 4;
            const int pg = pick4(h, v_pages[0], v_pages[1], v_pages[2], v_pages[3]), off = (kt + h * 16) & P1;
            const uint8_t* const p = static_cast<const uint8_t*>(a.v_pages) + pg * a.v_stride + ((int64_t(head) * D + col) << a.page_shift) + off;
#pragma unroll
            for (int d = 0; d < VL; ++d) vf[d] = *reinterpret_cast<const u32x4*>(p + (int64_t(d) * 16 << a.page_shift));
            vx = *reinterpret_cast<const u32x4*>(a.v_scales + ((int64_t(pg) * a.kv_heads + head) << a.page_shift) + off);
            slot = (int64_t(pg) << a.page_shift) + off;
        } else {
            const T* const vp = static_cast<const T*>(a.v_pages) + ((int64_t(head) * D + col) << a.page_shift) + (h & 1) * 8;
            const int a0 = kt & P1, a1 = (kt + 16) & P1;
            const T* const p = vp + (h & 2 ? v_pages[1] * a.v_stride + a1 : v_pages[0] * a.v_stride + a0);
#pragma unroll
            for (int d = 0; d < VL; ++d) vf[d] = load16<u32x4>(p + (int64_t(d) * 16 << a.page_shift));
            slot = (int64_t(h & 2 ? v_pages[1] : v_pages[0]) << a.page_shift) + (h & 2 ? a1 : a0) + (h & 1) * 8;
        }
        if (EXTRA && a.k_times) {
#pragma unroll
            for (int b = 0; b < NB; ++b) tk[b] = *reinterpret_cast<const f32x4*>(a.k_times + slot + 4 * b);
        }
        if (EXTRA && !F::share && a.k_eps) {
#pragma unroll
            for (int b = 0; b < NB; ++b) ek[b] = *reinterpret_cast<const i32x4*>(a.k_eps + slot + 4 * b);
        }
    };
    // the episodes of a step whose rows and keys have to be compared one by one: seldom, and not worth registers for one on the way
    auto load_eps = [&](int ks) {
        const int key = ks + NK * h, id = a.table[int64_t(r) * a.max_pages + min(key >> a.page_shift, last_page)];
        const int64_t slot = (int64_t(uint32_t(id) < uint32_t(a.num_pages) ? id : 0) << a.page_shift) + (key & P1);
#pragma unroll
        for (int b = 0; b < NB; ++b) ek[b] = *reinterpret_cast<const i32x4*>(a.k_eps + slot + 4 * b);
    };

    // q in the order of K's elements: a piece of 16 bytes holds those of two products where the cache is e4m3
    V q[KC];
    const T* const qp = static_cast<const T*>(a.q) + row * a.q_stride + int64_t(hq) * D + h * (F::c8 ? 16 : 8);
#pragma unroll
    for (int c = 0; c < KC; ++c) q[c] = load_q<V>(qp + (F::c8 ? c / 2 * 64 + c % 2 * 8 : c * 32), a.q_flip);
    if constexpr (kLean) {
        if (wave == 0) {
#pragma unroll
            for (int c = 0; c < KC; ++c) lds.q[c * 64 + lane] = __builtin_bit_cast(u32x4, q[c]);
        }
        if (wave == 0 && h == 0) lds.row[col] = u32x4{__float_as_uint(dec), __float_as_uint(tq), uint32_t(limit), uint32_t(eq)};
        __syncthreads();
    }
    f32x4 o[VB];
#pragma unroll
    for (int d = 0; d < VB; ++d) o[d] = f32x4{0, 0, 0, 0};
    float mref = 0.0f, mtop = -kInf, l = 0.0f;              // mtop: -inf until the row has seen a key, then mref + lift + kSlack
    auto keep_pages = [&] {
#pragma unroll
        for (int u = 0; u < NG; ++u) v_pages[u] = pages[u];
    };
    if (F::share && it.skip > 0 && k0 == it.skip) {         // the prefix's sums
        const float2 ml = join_state<D, 8>(a, it, lds.join);
        if (wave == 0 && row_ok && ml.x != -kInf) {
            mref = ml.x;
            mtop = mref + (lift + kSlack);
            l = h == 0 ? ml.y : 0.0f;
#pragma unroll
            for (int d = 0; d < VB; ++d) o[d] = *reinterpret_cast<const f32x4*>(&lds.join.sum()[col * (D + 4) + d * 16 + h * 4]);
        }
    }
    bool dirty = false;                                     // a value that is not finite was left out

    for (int w0 = 0; w0 < steps; w0 += kWindow) {
        const int count = listed ? list_steps<kStep>(a, r, last_page, k0, k1, w0, steps, eq_min, eq_max, lds.steps) : steps;
        auto step_at = [&](int x) { return listed ? w0 + (__builtin_amdgcn_readfirstlane(int(lds.steps.list[x])) & (kWindow - 1)) : x; };
        if (wave < count) {
            find_pages(step_at(wave));
            load_k(step_at(wave));
            keep_pages();
            load_v(step_at(wave));
            if (wave + 4 < count) find_pages(step_at(wave + 4));
        }
        for (int x0 = wave; x0 < count; x0 += 4) {
            const int ks = k0 + step_at(x0) * kStep;
            const bool mixed = listed && (__builtin_amdgcn_readfirstlane(int(lds.steps.list[x0])) & kMixed);
            f32x4 acc[NB];
            if constexpr (kLean) {
                const uint32_t at = here(uint32_t(lane));   // not ahead of the loop
#pragma unroll
                for (int c = 0; c < KC; ++c) q[c] = load16<V>(&lds.q[c * 64 + at]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                acc[b] = f32x4{0, 0, 0, 0};
                float ks8 = 0.0f;
                if constexpr (F::c8) ks8 = scale_at<0>(kx[b] >> (8 * (col & 3)));
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    u32x4 w;
                    if constexpr (F::c8) w = token_e4m3<T>(kf[b][c / 2][c % 2 * 2], kf[b][c / 2][c % 2 * 2 + 1], ks8);
                    else w = kf[b][c];
                    acc[b] = Vec<T>::mma(__builtin_bit_cast(V, w), q[c], acc[b]);
                }
            }
            const bool more = x0 + 4 < count;
            const int next = more ? step_at(x0 + 4) : 0;
            if (more) {
                load_k(next);
                keep_pages();
                if (x0 + 8 < count) find_pages(step_at(x0 + 8));
            }
            // x[j]: this lane's key ks + NK h + j
            float x[NK];
#pragma unroll
            for (int j = 0; j < NK; ++j) x[j] = acc[j >> 2][j & 3] * a.scale_log2;
            if (CAP) {
#pragma unroll
                for (int j = 0; j < NK; ++j) x[j] = cap_any(x[j], a.cap_log2, a.cap_rcp);
            }
            float dec_now = dec, tq_now = tq;
            int limit_now = limit, eq_now = eq;
            if constexpr (kLean) {
                const u32x4 w = lds.row[here(uint32_t(lane)) & 15];
                dec_now = __uint_as_float(w[0]);
                tq_now = __uint_as_float(w[1]);
                limit_now = int(w[2]);
                eq_now = int(w[3]);
            }
            if (EXTRA && a.k_times) {
#pragma unroll
                for (int j = 0; j < NK; ++j) x[j] -= dec_now * fmaxf(0.0f, tq_now - tk[j >> 2][j & 3]);
            }
            const bool whole = ks + kStep <= lo && !mixed;
            if (!whole) {
                if (EXTRA && F::share && mixed) load_eps(ks);
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    bool in = ks + NK * h + j < limit_now;
                    if (mixed) {
                        const int e = ek[j >> 2][j & 3];
                        in = in && (e < 0 || eq_now < 0 || e == eq_now);
                    }
                    x[j] = in ? x[j] : -kInf;
                }
            }
            float top = x[0];
#pragma unroll
            for (int j = 1; j < NK; ++j) top = fmaxf(top, x[j]);
            if (__any(top > mtop)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const bool none = mtop == -kInf;
                const float mnew = none ? top - lift : fmaxf(mref, top - lift);
                if (mnew > -kInf) {                          // not NaN either: the row's sum is then NaN
                    const float f = none ? 0.0f : __builtin_amdgcn_exp2f(mref - mnew);
                    mref = mnew;
                    mtop = mnew + (lift + kSlack);
                    l *= f;
#pragma unroll
                    for (int d = 0; d < VB; ++d) o[d] *= f;
                }
            }
            // the weights as a 16-bit value and a 16-bit rest: the second product costs little where the cache's bytes bound the
            // kernel, and the output's error is that of its own rounding (with one product 1.4 times that, as in k_attend_many).
            // fp16's rests end at 2^-25 as its values do: a weight is off by up to 2^-32 of the row's largest
            VW p[NT], rest[NT];
            float sum = 0.0f;
            auto weigh = [&](int t) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float w = __builtin_amdgcn_exp2f(x[8 * t + j] - mref);
                    sum += w;
                    if constexpr (F::c8) w *= power(vx[2 * t + j / 4], j % 4);
                    p[t][j] = W(w);
                    rest[t][j] = W(w - float(p[t][j]));
                }
            };
            // infinities and NaN: see add_not_finite (in every step: a rest may be 0 or negative). Slots past the request's keys
            // hold anything.
            uint32_t odd = 0;
            const int kb = ks + NK * h;
            if constexpr (F::c8) {
                if (!whole && kb + NK > keys) {
                    vx = first_bytes(vx, keys - kb);
#pragma unroll
                    for (int d = 0; d < VB; ++d) vf[d] = first_bytes(vf[d], keys - kb);
                }
                // exponents of 255 stand for NaN
#pragma unroll
                for (int j = 0; j < 4; ++j) odd |= nan_e4m3(vx[j]) & vx[j];
#pragma unroll
                for (int d = 0; d < VB; ++d) odd |= nan_e4m3(vf[d][0]) | nan_e4m3(vf[d][1]) | nan_e4m3(vf[d][2]) | nan_e4m3(vf[d][3]);
                if (__any(odd != 0)) {
                    dirty = true;
#pragma unroll
                    for (int j = 0; j < 4; ++j) vx[j] &= ~(((nan_e4m3(vx[j]) & vx[j]) >> 7) * 0xFFu);
#pragma unroll
                    for (int d = 0; d < VB; ++d)
#pragma unroll
                        for (int j = 0; j < 4; ++j) vf[d][j] &= ~((nan_e4m3(vf[d][j]) >> 7) * 0xFFu);
                }
                auto add = [&](int d, int t) {
                    const VW w = __builtin_bit_cast(VW, token_e4m3<W>(vf[d][2 * t], vf[d][2 * t + 1], 1.0f));
                    o[d] = Vec<W>::mma(w, rest[t], Vec<W>::mma(w, p[t], o[d]));
                };
                // element by element, so that the registers of V are free for the next step's one after the other (one token over
                // 4,001 keys of 64 requests 93 us, key by key 106); kLean has no registers for all weights at once
                if constexpr (kLean) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        weigh(t);
#pragma unroll
                        for (int d = 0; d < VB; ++d) add(d, t);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < NT; ++t) weigh(t);
#pragma unroll
                    for (int d = 0; d < VB; ++d)
#pragma unroll
                        for (int t = 0; t < NT; ++t) add(d, t);
                }
            } else {
                weigh(0);
#pragma unroll
                for (int d = 0; d < VB; ++d) {
                    u32x4 b = vf[d];
                    if (!whole && kb + 8 > keys) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) b[j] &= kb + 2 * j >= keys ? 0u : kb + 2 * j + 1 >= keys ? 0xFFFFu : ~0u;
                    }
                    const uint32_t full = exponents_full<T>(b);
                    odd |= full;
                    if (__any(full != 0)) b = finite_part<T>(b);
                    vf[d] = b;
                }
                if (__any(odd != 0)) dirty = true;
#pragma unroll
                for (int d = 0; d < VB; ++d) {
                    const VW w = __builtin_bit_cast(VW, vf[d]);
                    o[d] = Vec<W>::mma(w, rest[0], Vec<W>::mma(w, p[0], o[d]));
                }
            }
            l += sum;
            if (more) load_v(next);
        }
        if (!listed) break;
    }

    if constexpr (F::share) {                               // found again, rather than kept in registers that the loop needs
        tid = int(threadIdx.x);
        asm volatile("" : "+v"(tid));
        lane = tid & 63;
        col = lane & 15;
        h = lane >> 4;
        m = it.tile * kFewRows + col;
        row_ok = m < n * a.group;
        i = row_ok ? m / a.group : 0;
        hq = head * a.group + (row_ok ? m - i * a.group : 0);
        row = int64_t(row0) + i;
    }
    // join the waves: references first, then sums and O, in wave order
    auto& ml = lds.wave.ml;
    auto& ob = lds.wave.ob;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float mw = mtop == -kInf && l == 0.0f ? -kInf : mref;   // -inf: the row sees no key; with NaN scores alone its sum is NaN
    __syncthreads();                                        // the list of steps is done with
    if (h == 0) ml[wave][col][0] = mw;
    if (dirty && lane == 0) lds.any_dirty = 1;
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
        if (F::share && a.phase == 1 && row_ok && !joined) {
            const int64_t at = state_row(a, row, hq);
#pragma unroll
            for (int d = 0; d < VB; ++d) *reinterpret_cast<f32x4*>(a.state_o + at * D + d * 16 + h * 4) = o[d];
            if (h == 0) a.state_ml[at] = make_float2(mall, lall);
            if (h == 0) a.state_at[at] = one_piece(a, at);
        } else if (row_ok && !joined) {
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
        if (joined) {
#pragma unroll
            for (int d = 0; d < VB; ++d) *reinterpret_cast<f32x4*>(&ob[0][col][d * 16 + h * 4]) = o[d];
            if (row_ok && h == 0) put_part(a.part_ml + int64_t(it.slot) * kFewRows + col, make_float2(mall, lall));
            if (F::share && a.phase == 1 && a.defer && row_ok && h == 0 && it.slot == it.slot0)
                a.state_at[state_row(a, row, hq)] = i32x4{int32_t(a.many_row0) + it.slot0 * kFewRows + col, int32_t(a.many_row0) + it.slot1 * kFewRows + col,
                                                          it.slot_step * kFewRows, it.splits};
        }
    }
    if (joined) {
        __syncthreads();
        const int valid = min(kFewRows, n * a.group - it.tile * kFewRows);
        float* const po = a.part_o + int64_t(it.slot) * kFewRows * D;
        for (int e = tid; e < valid * (D / 2); e += 256)
            put_part(po + e * 2, *reinterpret_cast<const float2*>(&ob[0][e / (D / 2)][e % (D / 2) * 2]));
    }
    if (lds.any_dirty) {
        stores_done();                                      // of the partials
        __syncthreads();
        add_not_finite<T, D, kFewRows, F>(a, it, prefix);
    }
    if (!joined || (F::share && a.phase == 1 && a.defer)) return;
    __syncthreads();
    join_last<T, D, F>(a, it, lds.join);
}

// The launch's work is one line of steps, request after request, tile after tile, kv head after kv head, and workgroup w
// of G takes the w-th of G equal lengths of it: the bytes of the cache are dealt out evenly whatever the requests'
// lengths, in one round. An end of a length that falls within kFewCut steps of a tile's first or last one moves there
// (short requests are not cut), so a workgroup has at most two pieces that others share: its first and its last.
// Cuts 2, 4, 8 steps from an end: 24 x 5 tokens over up to 3,000 keys 23.3, 22.3, 20.4 us, 4 x 4 over 3,000 29.7, 24.7,
// 25.1 us (with 12 steps of twice the length it was slower again).
constexpr int kFewCut = 8;
// Where there are no more tiles than workgroups, and none of more steps than this, each workgroup takes whole tiles: equal lengths of the
// line would give some of them the ends of two. 64 single tokens over 500 to 1,000 keys (32/8 heads of 128, 8 bits) 27.2 us, 38.4
// without; one over 4,160 (65 steps) 20 and, whole, 44.6. (mars_kv_attend over 16 bits keeps to equal lengths, and its bits.) The bound does not
// look at how many tiles there are, and few long ones leave CUs idle: 1, 4, 16 and 48 requests over 2,304 keys (36 steps) 25.5, 26.0, 28.6
// and 46.1 us; cut, over 16 bits, 16.2, 21.6, 32.0 and 93.5.
constexpr int kFewWhole = 36;
// The same where steps outside the rows' episodes are skipped: equal lengths leave most pieces without any. 48 single tokens that ask within
// 900 of up to 6,001 keys (94 steps) 38 us, 57 cut (16/2 heads 31 and 37). Rows that ask within no episode read all of it, some 0.65 us
// a step: 1, 4, 16 and 48 such requests over 6,912 keys (108 steps) 75, 85, 86 and 158 us; cut, over 16 bits, 24, 32, 91 and 263.
constexpr int kFewWholeListed = 108;
// Steps of a piece of a prefix at least: 2 prefixes of 4,160 tokens for 4 requests each 33.0 us (1: 35.4, 16: 37.0).
constexpr int kFirstSpan = 4;
template <typename F>
struct SpanLds {
    int64_t start[257];        // of 256 requests: steps of the launch before each
    int32_t row0[256], n[256], keys[256];
    int32_t skip[F::share ? 256 : 1], row[F::share ? 256 : 1];     // Request's skip and at
    int64_t total, span;       // F::share: read again after every piece, rather than kept in registers
    int64_t wsum[4];
    int32_t wmost[4];
    int32_t at, most;          // most: steps of the longest tile so far
};
template <typename F>
__device__ inline int steps_of(int keys) { return max(1, (keys + few_step<F>() - 1) / few_step<F>()); }
__device__ inline int units_of(const AttendArgs& a, int n) { return (n * a.group + kFewRows - 1) / kFewRows * a.kv_heads; }

// Requests r0 .. r0 + 255 into the LDS; returns the launch's steps up to their end (base: before them).
// TILES: tiles instead of steps.
template <typename F, bool TILES = false>
__device__ int64_t load_span(const AttendArgs& a, int r0, int64_t base, SpanLds<F>& lds) {
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const Request q = request_of<true, F>(a, r0 + tid);
    const int own = steps_of<F>(F::share ? q.keys - q.skip : q.keys);
    const int64_t work = int64_t(q.tiles) * a.kv_heads * (TILES ? 1 : own);
    int64_t x = work;
    int most = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up((long long)x, unsigned(o));
        if (lane >= o) x += y;
    }
    __syncthreads();                                        // the requests before are done with
    if (lane == 63) { lds.wsum[wave] = x; lds.wmost[wave] = most; }
    __syncthreads();
    int64_t sum = base, mine = base;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) mine += lds.wsum[w];
        sum += lds.wsum[w];
    }
    lds.start[tid] = mine + x - work;
    lds.row0[tid] = q.row0;
    lds.n[tid] = q.tiles ? q.n : 0;
    lds.keys[tid] = q.keys;
    if constexpr (F::share) { lds.skip[tid] = q.skip; lds.row[tid] = q.at; }
    if (tid == 0) {
        lds.start[256] = sum;
        lds.most = max(r0 ? lds.most : 0, max(max(lds.wmost[0], lds.wmost[1]), max(lds.wmost[2], lds.wmost[3])));
    }
    __syncthreads();
    return uniform(sum);
}

template <int D, typename F>
struct FewShared {
    FewLds<D, F> part;
    SpanLds<F> span;
};
template <typename T, int D, bool EXTRA, bool CAP, typename F>
__device__ void few_rows(const AttendArgs& a, int block, int blocks, FewShared<D, F>& shared) {
    FewLds<D, F>& lds = shared.part;
    SpanLds<F>& sp = shared.span;
    const int tid = int(threadIdx.x);
    const int64_t w = block;
    int r0 = 0;
    bool whole = false;
    int next = block;                                       // whole: the tile to take next
    if (F::share && a.whole) {
        int64_t tiles = load_span<F, true>(a, 0, 0, sp);
        for (int r = 256; r < a.requests; r += 256) tiles = load_span<F, true>(a, r, tiles, sp);
        if (tid == 0) sp.total = tiles;
        whole = __builtin_amdgcn_readfirstlane(sp.most) <= (EXTRA && a.k_eps ? kFewWholeListed : kFewWhole);
        __syncthreads();
    }
    auto span_of = [&](int r, int64_t base) { return F::share && whole ? load_span<F, true>(a, r, base, sp) : load_span<F>(a, r, base, sp); };
    int64_t end = F::share && whole && a.requests <= 256 ? 0 : span_of(0, 0), total = end;
    if (!(F::share && whole))
        for (int r = 256; r < a.requests; r += 256) total = span_of(r, total);
    const int most = __builtin_amdgcn_readfirstlane(sp.most);
    if (!(F::share && whole) && a.requests > 256) end = span_of(0, 0);   // back to the first
    // no tile in more than kMaxSplits pieces
    const int64_t span = max(max((total + blocks - 1) / blocks, int64_t(F::share && a.phase == 1 ? kFirstSpan : 1)), int64_t((most + kMaxSplits - 2) / (kMaxSplits - 1))), x0 = w * span, x1 = min(x0 + span, total);
    if (F::share && !whole && tid == 0) { sp.total = total; sp.span = span; }
    int k = 0, steps = 1, unit = 0, s0 = 0;
    if (!(F::share && whole)) {
        if (x0 >= total) return;                            // no steps at all, or none for this workgroup
        while (x0 >= end) {
            r0 += 256;
            end = span_of(r0, end);
        }
        if (x0 >= sp.start[tid] && x0 < sp.start[tid + 1]) sp.at = tid;
        __syncthreads();
        k = __builtin_amdgcn_readfirstlane(sp.at);
        steps = steps_of<F>(__builtin_amdgcn_readfirstlane(F::share ? sp.keys[k] - sp.skip[k] : sp.keys[k]));
        // the first tile and step: ends near a tile's own move to it
        const int64_t local = x0 - uniform(sp.start[k]);
        unit = __builtin_amdgcn_readfirstlane(int(local / steps));
        s0 = __builtin_amdgcn_readfirstlane(int(local - int64_t(unit) * steps));
        if (s0 < min(kFewCut, (steps + 1) / 2)) s0 = 0;
        else if (steps - s0 < kFewCut) { s0 = 0; ++unit; }
    }
    bool first = true;
    for (;;) {
        if (F::share && whole) {
            if (next >= uniform(sp.total)) return;
            for (int64_t e = uniform(sp.start[256]); next >= e;) {
                r0 += 256;
                e = span_of(r0, e);
            }
            __syncthreads();                                // the tile before is done with
            if (next >= sp.start[tid] && next < sp.start[tid + 1]) sp.at = tid;
            __syncthreads();
            k = __builtin_amdgcn_readfirstlane(sp.at);
            unit = __builtin_amdgcn_readfirstlane(int(next - uniform(sp.start[k])));
            next += blocks;
        }
        while (!(F::share && whole) && unit >= units_of(a, __builtin_amdgcn_readfirstlane(sp.n[k]))) {      // on to the next request that has rows
            unit = 0;
            if (r0 + ++k >= a.requests) return;
            if (k < 256) continue;
            r0 += 256;
            end = span_of(r0, F::share ? uniform(sp.start[256]) : end);
            k = 0;
        }
        Part it;
        it.request = F::share ? __builtin_amdgcn_readfirstlane(sp.row[k]) : r0 + k;
        it.skip = F::share ? __builtin_amdgcn_readfirstlane(sp.skip[k]) : 0;
        it.row0 = __builtin_amdgcn_readfirstlane(sp.row0[k]);
        it.n = __builtin_amdgcn_readfirstlane(sp.n[k]);
        it.keys = __builtin_amdgcn_readfirstlane(sp.keys[k]);
        steps = steps_of<F>(it.keys - it.skip);
        // the tile's first step; ours of it
        const int64_t u0 = uniform(sp.start[k]) + int64_t(unit) * steps;
        const int64_t left = !F::share ? x1 - u0 : whole ? int64_t(steps) : min((w + 1) * uniform(sp.span), uniform(sp.total)) - u0;
        const int low = min(kFewCut, (steps + 1) / 2);
        if (left < low) return;
        const int s1 = left >= steps || steps - left < kFewCut ? steps : int(left);
        it.tile = unit / a.kv_heads;
        it.head = unit - it.tile * a.kv_heads;
        it.k0 = it.skip + s0 * few_step<F>();
        it.k1 = min(it.skip + s1 * few_step<F>(), it.keys);
        it.splits = 1;
        it.chunk = 0;
        it.slot = it.slot0 = it.slot1 = it.slot_step = 0;
        if (s0 > 0 || s1 < steps) {
            // the cuts of this tile: ends c span with low <= c span - u0 <= steps - kFewCut. The piece before the first is
            // the last of workgroup c - 1, the one after cut c the first of workgroup c.
            const int64_t length = F::share ? uniform(sp.span) : span;
            const int64_t c0 = (u0 + low + length - 1) / length, c1 = (u0 + steps - kFewCut) / length;
            it.splits = int(c1 - c0) + 2;
            it.slot0 = int(2 * (c0 - 1) + 1);
            it.slot1 = int(2 * c0);
            it.slot_step = 2;
            it.slot = s0 > 0 ? int(2 * w) : it.slot0;
        }
        if (!first) __syncthreads();                        // the LDS of the piece before is done with
        first = false;
        few_part<T, D, EXTRA, CAP, F>(a, uniform_part(it), lds);
        if (F::share && whole) continue;
        if (!F::share && left <= steps) return;             // else the next tile's bounds say so
        s0 = 0;
        ++unit;
    }
}

// How many keys the rows of a tile of k_attend_many see at most: limits grow with the token, so its last row's.
template <typename F>
__device__ inline int tile_end(const AttendArgs& a, const Part& it) {
    const int last = min((it.tile * kManyRows + kManyRows - 1) / a.group, it.n - 1);
    return limit_of<F>(a, it.keys, it.n, last, prefix_of<F>(a, it.request, it.keys));
}
// Sets the tile's pieces to those that its rows see keys of; false if piece `piece` is none of them.
template <typename F>
__device__ inline bool own_pieces(const AttendArgs& a, Part* it, int piece) {
    it->splits = min(it->splits, max(1, (tile_end<F>(a, *it) - (F::share ? it->skip : 0) + it->chunk - 1) / it->chunk));
    return piece < it->splits;
}

// ---- many rows: 128 at a time, keys staged through LDS ----------------------------------
// Bound by the matrix cores and the softmax's vector work together, and by the clock, which falls under that load: heads
// of 128 without extra terms keep the matrix cores busy 48% of the cycles and the vector units 45%, heads of 64 43% and 70%.
// 4 waves of 32 rows each share tiles of 64 keys: K (keys, elements) and V (elements, keys) come straight into two LDS
// buffers, one tile ahead. 16-byte pieces of a row are XORed with the row number so that the 16 lanes of a fragment read hit
// the 16 bank groups (no conflicts counted). The other workgroup of the CU fills the matrix cores while this one's waves are
// in the softmax. 2 x 4,096 tokens over 8,196 keys, bf16, 32/8 heads of 128: 782 to 838 us by the box, 985 to 1,055 TFLOP/s (a product
// of 8,192 cubed reaches 1,168). With cap and decay a score takes twice the vector instructions: 2 x 4,001 tokens of 12 heads of
// 64 within their episodes, vector units busy 72%, matrix cores 11%.
// Of 8 bits the tiles go through registers, where they become T: half as many vector instructions again (bytes to 16 bits 64, their
// addresses and the writes to LDS some 35, beside 207 a wave and tile). 2 x 2,048 tokens over 6,148 keys, heads of 128: 393 to 411
// us by the box (875 to 835 TFLOP/s), 362 to 372 of 16 bits; matrix cores busy 41% and 51%, vector units 53% and 47%. Pieces of 8 bytes,
// whose writes to LDS have no bank conflicts (10% of the cycles here), take more loads: 496 us for 485 (under a profiler), heads of 256
// 631 for 569.
constexpr int kManyKeys = 64;

// Heads of 256 have one wave a SIMD, which nothing covers while it waits for LDS: LDS reads and products stay in the order
// written, and only vector and scalar arithmetic passes (2 x 2,048 tokens over as many cached ones 221 us, 240 us in the
// compiler's order, with cap and decay 280 and 320 us). With two or three waves a SIMD the compiler's order, and its fewer
// registers, are as fast or faster (heads of 64 with every term 92 us, 101 us in this order).
template <int D>
__device__ inline void reads_first() {
    if constexpr (D > 128) __builtin_amdgcn_sched_barrier(0x406);
}

template <int D>
struct ManyLds {
    u32x4 k[2][kManyKeys * D / 8];
    u32x4 v[2][kManyKeys * D / 8];
    float times[2][kManyKeys];
    int32_t eps[2][kManyKeys];
};

template <int D>
struct ManyShared {
    union { ManyLds<D> tiles; SchedLds sched; int any_dirty; };
    StepLds list;
};
template <typename T, int D, bool EXTRA, bool CAP, typename F>
__device__ void many_rows(const AttendArgs& a, int block, ManyShared<D>& lds) {
    using V = typename Vec<T>::v8;
    constexpr int KS = D / 16, DB = D / 32, RC = D / 8;      // k-steps of S, blocks of O, 16-byte pieces of a key's row
    StepLds& list = lds.list;
    ManyLds<D>& sh = lds.tiles;
    Part it;
    {
        ManySched<false, F> sched(a, lds.sched);
        if (!sched.start() || !sched.find(uint32_t(block), &it)) return;
    }
    if (!own_pieces<F>(a, &it, it.slot - it.slot0)) return;
    __syncthreads();                                         // the item is read before its LDS is used again
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int r = it.request, head = it.head;
    const int P1 = (1 << a.page_shift) - 1;
    const int row0 = it.row0, n = it.n, keys = it.keys;
    const int m = it.tile * kManyRows + wave * 32 + col;     // this lane's row: token i, head of the group
    const bool row_ok = m < n * a.group;
    const int i = row_ok ? m / a.group : 0, hq = head * a.group + (row_ok ? m - i * a.group : 0);
    const int64_t row = int64_t(row0) + i;
    const int prefix = prefix_of<F>(a, r, keys);
    const int limit = row_ok ? limit_of<F>(a, keys, n, i, prefix) : 0;         // keys [0, limit) may be seen
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
    const int end = tile_end<F>(a, it);
    const int first_limit = limit_of<F>(a, keys, n, it.tile * kManyRows / a.group, prefix);
    const int k0 = it.k0, k1 = min(it.k1, end);
    const int steps = __builtin_amdgcn_readfirstlane(k1 > k0 ? (k1 - k0 + kManyKeys - 1) / kManyKeys : 0);

    const bool listed = EXTRA && a.k_eps;
    int eq_min = row_ok ? eq : INT32_MAX, eq_max = row_ok ? eq : INT32_MIN;
    if (listed) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            eq_min = min(eq_min, __shfl_xor(eq_min, o));
            eq_max = max(eq_max, __shfl_xor(eq_max, o));
        }
        if (lane == 0) { list.eq_min[wave] = eq_min; list.eq_max[wave] = eq_max; }
        __syncthreads();
        eq_min = min(min(list.eq_min[0], list.eq_min[1]), min(list.eq_min[2], list.eq_min[3]));
        eq_max = max(max(list.eq_max[0], list.eq_max[1]), max(list.eq_max[2], list.eq_max[3]));
    }

    const TablePtr table = table_row(a, r);
    const int last_page = keys > 0 ? (keys - 1) >> a.page_shift : 0;
    // Pieces of 16 bytes in a tile: K's row of a key holds RC of them, V's row of an element the 8 of the tile's 64 keys.
    // Piece c of row w lies at place c ^ swz(w). Load j of a wave fills the 64 places from (4 j + wave) * 64.
    auto kswz = [](int w) { return D == 64 ? (w >> 1) & 7 : w & 15; };
    auto vswz = [](int w) { return (w >> 1) & 7; };
    constexpr int KR = 256 / RC;                             // rows of K per load of the workgroup
    const int krow = tid / RC, kpiece = (tid % RC) ^ kswz(krow), vrow = tid >> 3, vkey = ((tid & 7) ^ vswz(vrow)) * 8;
    static_assert(KR % 16 == 0 || D == 256, "a thread's pieces keep their place in the row");
    // a thread's place in a row of pieces is the same for every load: addresses are a scalar base and a constant offset
    const char* const kp = static_cast<const char*>(a.k_pages) + (int64_t(head) << a.page_shift) * D * 2;
    const char* const vp = static_cast<const char*>(a.v_pages) + (int64_t(head) << a.page_shift) * D * 2;
    const uint32_t k_at = uint32_t(krow % 16 * D * 2 + kpiece * 16);
    const uint32_t k_at2 = D == 256 ? uint32_t((krow + 8) * D * 2 + ((tid % RC) ^ kswz(krow + 8)) * 16) : k_at;     // odd loads
    const uint32_t v_at = uint32_t((vrow << a.page_shift) + vkey) * 2;
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
            const char* const base = uniform_ptr(kp + (pg * a.k_stride + int64_t((kt + u * 16) & P1) * D) * 2);
            dma16(base + here(D == 256 && j % 2 ? k_at2 : k_at), &sh.k[buf][j * 256 + wave * 64]);
        }
        if (a.page_shift >= 6) {                             // the tile lies in one page
#pragma unroll
            for (int j = 0; j < RC / 4; ++j)
                dma16(uniform_ptr(vp + (pages[0] * a.v_stride + (kt & P1)) * 2 + (int64_t(j) * 64 << a.page_shift)) + here(v_at), &sh.v[buf][j * 256 + wave * 64]);
        } else {
            const int g = vkey >> 4;
            const int64_t b0 = pages[0] * a.v_stride + (kt & P1), b1 = pages[1] * a.v_stride + ((kt + 16) & P1);
            const int64_t b2 = pages[2] * a.v_stride + ((kt + 32) & P1), b3 = pages[3] * a.v_stride + ((kt + 48) & P1);
            const char* const p = vp + ((g & 2 ? (g & 1 ? b3 : b2) : (g & 1 ? b1 : b0)) + (vkey & 15)) * 2 + (int64_t(vrow) << a.page_shift) * 2;
#pragma unroll
            for (int j = 0; j < RC / 4; ++j) dma16(p + (int64_t(j) * 64 << a.page_shift), &sh.v[buf][j * 256 + wave * 64]);
        }
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

    // e4m3: a tile comes to registers two tiles ahead, and to LDS as T one tile ahead: what the products then read is what
    // they read of a cache of T. A thread has D / 64 pieces of 16 elements of a key and as many of 16 keys of an element.
    constexpr int RL = F::c8 ? D / 64 : 1, KP = D / 16;
    u32x4 kr[RL], vr[RL], vx;
    uint32_t kx[RL];
    float time_raw = 0.0f;
    int32_t eps_raw = 0;
    // a thread's place in the tile, found anew for every tile where the registers are short (heads of 256 with cap and age 743 us, 794)
    auto thread = [&] { return D == 256 ? int(here(uint32_t(tid))) : tid; };
    auto page4 = [&](int u) { return pick4(u, pages[0], pages[1], pages[2], pages[3]); };
    auto fetch = [&](int s) {
        const int kt = k0 + s * kManyKeys, th = thread();
        // where the tile lies in one page the place is the same for every load: a base and a constant offset
        const int krow8 = th / KP, kpiece8 = th % KP, vrow8 = th >> 2, vgroup8 = th & 3;
        const uint32_t k_at8 = uint32_t(krow8 * D + kpiece8 * 16), kx_at8 = uint32_t(krow8);
        const uint32_t v_at8 = uint32_t((vrow8 << a.page_shift) + vgroup8 * 16), vx_at8 = uint32_t(vgroup8 * 16);
        const char* const kb = static_cast<const char*>(a.k_pages) + (int64_t(head) << a.page_shift) * D;
        const char* const vb = static_cast<const char*>(a.v_pages) + (int64_t(head) << a.page_shift) * D;
        const char* const kxb = reinterpret_cast<const char*>(a.k_scales);
        const char* const vxb = reinterpret_cast<const char*>(a.v_scales);
        if (a.page_shift >= 6) {                             // the tile lies in one page
            const int pg = pages[0], off = kt & P1;
            const int64_t at = ((int64_t(pg) * a.kv_heads + head) << a.page_shift) + off;
            const char* const kt0 = kb + pg * a.k_stride + int64_t(off) * D;
            const char* const vt0 = vb + pg * a.v_stride + off;
#pragma unroll
            for (int j = 0; j < RL; ++j) {
                kr[j] = *reinterpret_cast<const u32x4*>(kt0 + (k_at8 + j * (256 * 16)));
                kx[j] = *reinterpret_cast<const uint8_t*>(kxb + at + (kx_at8 + j * (256 / KP)));
            }
#pragma unroll
            for (int j = 0; j < RL; ++j) {
                vr[j] = *reinterpret_cast<const u32x4*>(vt0 + (int64_t(j) * 64 << a.page_shift) + v_at8);
            }
            vx = *reinterpret_cast<const u32x4*>(vxb + at + vx_at8);
        } else {
#pragma unroll
            for (int j = 0; j < RL; ++j) {
                const int w = krow8 + j * (256 / KP), pg = page4(w >> 4), off = (kt + w) & P1;
                kr[j] = *reinterpret_cast<const u32x4*>(kb + pg * a.k_stride + int64_t(off) * D + kpiece8 * 16);
                kx[j] = *reinterpret_cast<const uint8_t*>(kxb + ((int64_t(pg) * a.kv_heads + head) << a.page_shift) + off);
            }
            const int pg = page4(vgroup8), off = (kt + vgroup8 * 16) & P1;
#pragma unroll
            for (int j = 0; j < RL; ++j) vr[j] = *reinterpret_cast<const u32x4*>(vb + pg * a.v_stride + (int64_t(vrow8 + j * 64) << a.page_shift) + off);
            vx = *reinterpret_cast<const u32x4*>(vxb + ((int64_t(pg) * a.kv_heads + head) << a.page_shift) + off);
        }
        if constexpr (EXTRA) {
            if (wave == 0) {
                const int64_t slot = (int64_t(page4(lane >> 4)) << a.page_shift) + ((kt + lane) & P1);
                if (a.k_times) time_raw = a.k_times[slot];
                if (a.k_eps) eps_raw = a.k_eps[slot];
            }
        }
    };
    bool dirty = false;                                      // a value that is not finite was left out
    // The tile of step s, fetched before, into buffer buf. Where some row of the workgroup does not see some key: see add_not_finite;
    // slots past the request's keys hold anything and become 0.
    auto put_as = [&](auto look, int kt, int buf) {
        const int th = thread(), krow8 = th / KP, kpiece8 = th % KP, vrow8 = th >> 2, vgroup8 = th & 3, left = keys - (kt + vgroup8 * 16);
        if (look && left < 16) {
            vx = first_bytes(vx, left);
#pragma unroll
            for (int j = 0; j < RL; ++j) vr[j] = first_bytes(vr[j], left);
        }
#pragma unroll
        for (int j = 0; j < RL; ++j) {
            const int w = krow8 + j * (256 / KP);
            const float ks = scale_at<0>(kx[j]);
#pragma unroll
            for (int u = 0; u < 2; ++u) sh.k[buf][w * RC + ((2 * kpiece8 + u) ^ kswz(w))] = token_e4m3<T>(kr[j][2 * u], kr[j][2 * u + 1], ks);
        }
        float vs[16];
        scales16(vx, vs);
#pragma unroll
        for (int j = 0; j < RL; ++j) {
            const int w = vrow8 + j * 64;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u32x4 b = element_e4m3<T>(vr[j][2 * u], vr[j][2 * u + 1], vs + 8 * u);
                if constexpr (look) {
                    dirty |= exponents_full<T>(b) != 0;
                    b = finite_part<T>(b);
                }
                sh.v[buf][w * 8 + ((2 * vgroup8 + u) ^ vswz(w))] = b;
            }
        }
        if constexpr (EXTRA) {
            if (wave == 0) {
                sh.times[buf][lane] = time_raw;
                sh.eps[buf][lane] = eps_raw;
            }
        }
    };
    auto put = [&](int s, bool mixed, int buf) {
        const int kt = k0 + s * kManyKeys;
        if (kt + kManyKeys > first_limit || mixed) put_as(std::true_type{}, kt, buf);
        else put_as(std::false_type{}, kt, buf);
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] = 0.0f;
    float mref = 0.0f, mtop = -kInf, l = 0.0f;               // mtop: -inf until the row has seen a key, then mref + lift + kSlack
    if (F::share && it.skip > 0 && k0 == it.skip && row_ok) {        // the prefix's sums
        // Over 8 bits their reference may be k_attend_few's, which weighs in bfloat16 there: taken lower in fp16, so that its weights reach
        // as far down as they do without a prefix.
        constexpr float lower = F::c8 && Vec<T>::lift > 0.0f ? Vec<T>::lift - kLift8 : 0.0f, times = lower > 0.0f ? 256.0f : 1.0f;
        static_assert(lower == 0.0f || lower == 8.0f, "2^lower");
        const int64_t at = row * a.q_heads + hq;
        const float2 ml = a.state_ml[at];
        if (ml.x != -kInf) {
            mref = ml.x - lower;
            mtop = mref + (Vec<T>::lift + kSlack);
            l = h == 0 ? ml.y * times : 0.0f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 w = *reinterpret_cast<const f32x4*>(a.state_o + at * D + d * 32 + g * 8 + h * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[d][g * 4 + j] = w[j] * times;
                }
        }
    }

    // K's row of lane `col` in a block of 32 keys: reg j of S then holds key 16 (j / 8) + 8 h + j % 8 of the block
    const int ki = (col & 16) + ((col >> 2) & 1) * 8 + ((col >> 3) & 1) * 4 + (col & 3);
    // byte offsets of this lane's fragments in a tile, piece 2 c + h of S's step c and piece 2 t + h of O's: those of
    // c = 0, t = 0, with c or t XORed into the piece bits
    const uint32_t koff = uint32_t(ki * RC + (h ^ kswz(ki))) * 16, voff = uint32_t(col * 8 + (h ^ vswz(col))) * 16;
    const char* const kl = reinterpret_cast<const char*>(&sh.k[0][0]);
    const char* const vl = reinterpret_cast<const char*>(&sh.v[0][0]);
    for (int w0 = 0; w0 < steps; w0 += kWindow) {
        const int count = listed ? list_steps<kManyKeys>(a, r, last_page, k0, k1, w0, steps, eq_min, eq_max, list) : steps;
        auto step_at = [&](int x) { return listed ? w0 + (__builtin_amdgcn_readfirstlane(int(list.list[x])) & (kWindow - 1)) : x; };
        auto mixed_at = [&](int x) { return listed && (__builtin_amdgcn_readfirstlane(int(list.list[x])) & kMixed); };
        if (count > 0) {
            find_pages(step_at(0));
            if constexpr (F::c8) {
                fetch(step_at(0));
                put(step_at(0), mixed_at(0), 0);
            } else {
                stage(step_at(0), 0);
            }
            if (count > 1) find_pages(step_at(1));
            if constexpr (F::c8) {
                if (count > 1) fetch(step_at(1));
                if (count > 2) find_pages(step_at(2));
            }
        }
        for (int x0 = 0; x0 < count; ++x0) {
            const int buf = x0 & 1;
            if constexpr (F::c8) lds_barrier();
            else tile_barrier();                                 // the tile is in LDS; nobody reads the other buffer any more
            const int kt = k0 + step_at(x0) * kManyKeys;
            const bool mixed = mixed_at(x0);
            if constexpr (F::c8) {
                if (x0 + 1 < count) put(step_at(x0 + 1), mixed_at(x0 + 1), buf ^ 1);
                if (x0 + 2 < count) fetch(step_at(x0 + 2));
                if (x0 + 3 < count) find_pages(step_at(x0 + 3));
            } else if (x0 + 1 < count) {
                stage(step_at(x0 + 1), buf ^ 1);
                if (x0 + 2 < count) find_pages(step_at(x0 + 2));
            }
            const uint32_t kb = buf * uint32_t(sizeof(sh.k[0])) + koff, vb = buf * uint32_t(sizeof(sh.v[0])) + voff;
            if (!F::c8 && (kt + kManyKeys > first_limit || mixed)) {
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
            // fragments come from LDS ahead of the products that take them, see reads_first
            V kf[2][4], vf[2][DB];
            auto read_k = [&](int g) {
#pragma unroll
                for (int u = 0; u < 4; ++u) kf[g & 1][u] = load16<V>(kl + (kb ^ ((2 * g + (u >> 1)) * 32)) + (u & 1) * 32 * RC * 16);
            };
            auto read_v = [&](int t) {
#pragma unroll
                for (int d = 0; d < DB; ++d) vf[t & 1][d] = load16<V>(vl + (vb ^ (t * 32)) + d * 32 * 8 * 16);
            };
            read_k(0);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) x[b][j] = 0.0f;
#pragma unroll
            for (int g = 0; g < KS / 2; ++g) {
                if (g + 1 < KS / 2) read_k(g + 1);
                else read_v(0);
                reads_first<D>();
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u & 1] = Vec<T>::mma32(kf[g & 1][u], q[2 * g + (u >> 1)], x[u & 1]);
                reads_first<D>();
            }
            const bool whole = kt + kManyKeys <= lo && !mixed;
            if constexpr (EXTRA) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[b][j] *= a.scale_log2;
                if constexpr (CAP) {
                    float most = 0.0f;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int j = 0; j < 16; ++j) most = fmaxf(most, fabsf(x[b][j]));
                    if (__builtin_expect(__any(most * a.cap_rcp >= 0.5f), 0)) {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[b][j] = cap_any(x[b][j], a.cap_log2, a.cap_rcp);
                    } else {
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[b][j] = cap_near(x[b][j], a.cap_rcp);
                    }
                }
                if (a.k_times) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            x[b][j] -= dec * fmaxf(0.0f, tq - sh.times[buf][b * 32 + (j >> 3) * 16 + h * 8 + (j & 7)]);
                }
            }
            if (!whole) {
                // bit j: this lane's row sees key kt + j
                uint64_t seen = limit - kt >= 64 ? ~0ull : limit > kt ? (1ull << (limit - kt)) - 1 : 0ull;
                if (EXTRA && mixed) {
                    // by the tile's few different episodes, each with the keys that have it
                    const int e = sh.eps[buf][lane];
                    uint64_t rest = keys - kt >= 64 ? ~0ull : (1ull << (keys - kt)) - 1, by_episode = 0;
                    while (rest) {
                        const int v = __builtin_amdgcn_readlane(e, __builtin_ctzll(rest));
                        const uint64_t with = __ballot(e == v);
                        by_episode |= v < 0 || eq < 0 || eq == v ? with : 0ull;
                        rest &= ~with;
                    }
                    seen &= by_episode;
                }
                seen >>= 8 * h;                                  // bit 32 b + 16 (j / 8) + j % 8: register j of block b
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint32_t in = uint32_t(__builtin_amdgcn_sbfe(int(seen >> (32 * b)), (j >> 3) * 16 + (j & 7), 1));
                        x[b][j] = __uint_as_float((__float_as_uint(x[b][j]) & in) | (__float_as_uint(-kInf) & ~in));
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
                const float mnew = none ? top - Vec<T>::lift : fmaxf(mref, top - Vec<T>::lift);
                if (mnew > -kInf) {                          // not NaN either: the row's sum is then NaN
                    const float f = none ? 0.0f : __builtin_amdgcn_exp2f(mref - mnew);
                    mref = mnew;
                    mtop = mnew + (Vec<T>::lift + kSlack);
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] *= f;
                }
            }
            V p[4];
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(x[b][j], c, -mref));
                    sum += w;
                    p[2 * b + (j >> 3)][j & 7] = T(w);
                }
            l += sum;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t < 3) read_v(t + 1);
                reads_first<D>();
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = Vec<T>::mma32(vf[t & 1][d], p[t], o[d]);
                reads_first<D>();
            }
        }
        if (!listed) break;
    }

    l += __shfl_xor(l, 32);
    const bool empty = mtop == -kInf && l == 0.0f;           // with NaN scores alone the sum is NaN
    // o[d][j] is element 32 d + 8 (j / 4) + 4 h + j % 4 of row `col`
    if (F::share && a.phase == 1 && it.splits == 1) {
        if (row_ok) {
            const int64_t at = row * a.q_heads + hq;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4*>(a.state_o + at * D + d * 32 + g * 8 + h * 4) = f32x4{o[d][g * 4], o[d][g * 4 + 1], o[d][g * 4 + 2], o[d][g * 4 + 3]};
            if (h == 0) a.state_ml[at] = make_float2(empty ? -kInf : mref, l);
            if (h == 0) a.state_at[at] = one_piece(a, at);
        }
    } else if (it.splits == 1 && row_ok) {
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
        const int64_t at = int64_t(it.slot) * kManyRows + wave * 32 + col;
        float* const po = a.many_o + at * D + h * 4;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(po + d * 32 + g * 8) = f32x4{o[d][g * 4], o[d][g * 4 + 1], o[d][g * 4 + 2], o[d][g * 4 + 3]};
        if (h == 0) a.many_ml[at] = make_float2(empty ? -kInf : mref, l);
        if (F::share && a.phase == 1 && a.defer && h == 0 && it.slot == it.slot0) {
            const int32_t from = int32_t(a.many_row0 + at);
            a.state_at[state_row(a, row, hq)] = i32x4{from, from + kManyRows, kManyRows, it.splits};
        }
    }
    __syncthreads();                                         // the LDS of the tiles is free, the rows are written
    if (tid == 0) lds.any_dirty = 0;
    __syncthreads();
    if (dirty) lds.any_dirty = 1;
    __syncthreads();
    if (lds.any_dirty) add_not_finite<T, D, kManyRows, F>(a, it, prefix);
}

// Joins the pieces that k_attend_many left: their partials come to megabytes, too much for the one workgroup that arrives
// last (2 requests of 64 tokens over 8,000 keys: 114 us so). A thread takes 4 elements of a row and has the references and
// partials of 8 pieces on the way together; the sums are taken in the order of the pieces. Bound by those bytes and, before
// them, by finding the work: 512 pieces of 128 rows of 128 elements, 34 MB just written, 12.9 us; no pieces at all 5.3 us.
// (Twice the workgroups: 15.6 and 8.8 us.)
template <typename T, int D, typename F>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs a) {
    __shared__ SchedLds lds;
    ManySched<true, F> sched(a, lds);
    if (!sched.start()) return;
    Part it;
    for (uint32_t block = blockIdx.x; sched.find(block, &it); block += gridDim.x) {
        const int jr = join_rows_of<F>(a);
        const int r0 = it.slot * jr, rows = min(jr, it.n * a.group - it.tile * kManyRows - r0);
        if (!own_pieces<F>(a, &it, 0) || it.splits == 1) continue;
        const float2* const ml = a.many_ml + int64_t(it.slot0) * kManyRows + r0;
        const float* const po = a.many_o + (int64_t(it.slot0) * kManyRows + r0) * D;
        for (int e = int(threadIdx.x); e < rows * (D / 4); e += 256) {
            const int rr = e / (D / 4), d4 = e % (D / 4);
            constexpr int U = 8;
            float top = -kInf, l = 0.0f;
            f32x4 sum = {0, 0, 0, 0};
            for (int s = 0; s < it.splits; s += U) {
                float2 p[U];
                f32x4 o[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (s + u >= it.splits) break;
                    const int64_t at = int64_t(s + u) * kManyRows + rr;
                    p[u] = ml[at];
                    o[u] = *reinterpret_cast<const f32x4*>(po + at * D + d4 * 4);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (s + u >= it.splits) break;
                    if (p[u].x == -kInf) continue;
                    const float next = fmaxf(top, p[u].x), was = top == -kInf ? 0.0f : __builtin_amdgcn_exp2f(top - next);
                    const float f = __builtin_amdgcn_exp2f(p[u].x - next);
                    l = top == -kInf ? f * p[u].y : l * was + f * p[u].y;
                    sum = top == -kInf ? f * o[u] : sum * was + f * o[u];
                    top = next;
                }
            }
            const int mm = it.tile * kManyRows + r0 + rr, ii = mm / a.group, hh = it.head * a.group + mm - ii * a.group;
            if (F::share && a.phase == 1) {
                const int64_t at = (int64_t(it.row0) + ii) * a.q_heads + hh;
                *reinterpret_cast<f32x4*>(a.state_o + at * D + d4 * 4) = sum;
                if (d4 == 0) a.state_ml[at] = make_float2(top, l);
                continue;
            }
            const float inv = 1.0f / l;
            typename Vec<T>::v4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = top == -kInf ? T(0.0f) : T(sum[j] * inv);
            *reinterpret_cast<typename Vec<T>::v4*>(static_cast<T*>(a.out) + (int64_t(it.row0) + ii) * a.out_stride + int64_t(hh) * D + d4 * 4) = w;
            if (a.lse && d4 == 0)
                a.lse[(int64_t(it.row0) + ii) * a.q_heads + hh] = top == -kInf ? -kInf : (top + __builtin_amdgcn_logf(l)) * kLn2;
        }
    }
}

// ---- the kernels ------------------------------------------------------------------------
template <typename T, int D, bool EXTRA, bool CAP, typename F>
__global__ __launch_bounds__(256, (few_waves<D, F, EXTRA>())) void k_attend_few(AttendArgs a) {
    __shared__ __attribute__((aligned(16))) FewShared<D, F> lds;
    int blocks = int(gridDim.x);
    if (F::share && a.phase == 1 && int(blockIdx.x) == --blocks) {
        static_assert(sizeof(lds) >= (kMaxRequests + 1) * sizeof(int32_t), "room for the starts");
        find_skips(a, reinterpret_cast<int32_t*>(&lds));
        return;
    }
    few_rows<T, D, EXTRA, CAP, F>(a, int(blockIdx.x), blocks, lds);
}

template <typename T, int D, bool EXTRA, bool CAP, typename F>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void k_attend_many(AttendArgs a) {
    __shared__ __attribute__((aligned(16))) ManyShared<D> lds;
    if (F::share && a.phase == 1 && blockIdx.x + 1 == gridDim.x) {
        static_assert(sizeof(lds) >= (kMaxRequests + 1) * sizeof(int32_t), "room for the starts");
        find_skips(a, reinterpret_cast<int32_t*>(&lds));
        return;
    }
    many_rows<T, D, EXTRA, CAP, F>(a, int(blockIdx.x), lds);
}

template <typename T, int D, bool EXTRA, bool CAP, typename F>
int launch_dim(AttendArgs a, int32_t max_new, hipStream_t s) {
    // Requests of at most kFewMost rows (new tokens x query heads per kv head) are k_attend_few's, the others
    // k_attend_many's: 64 requests over 3,000 keys of 16 rows 149 us by the one and 152 by the other, of 20 rows (which few
    // reads the keys twice for) 226 and 154 us, 4 such requests 28.6 and 27.5, 33.6 and 28.0. Where a bound on the new tokens rules one of them out, the other serves every request, also one that
    // breaks the bound. The groups of a first phase, whose rows are known on the device alone, go by their average.
    const int64_t rows = int64_t(a.tokens) * a.group, keys = int64_t(a.max_pages) << a.page_shift;
    const int64_t most = std::min<int64_t>(max_new > 0 ? max_new : a.tokens, a.tokens) * a.group;
    const bool first = F::share && a.phase == 1;
    const bool few_only = first ? rows <= int64_t(kFewMost) * a.requests : F::share && a.phase == 2 ? a.defer != 0 : most <= kFewMost;
    const bool many_only = !few_only && (first || a.requests == 1);
    a.few_rows = few_only ? INT32_MAX : many_only ? -1 : kFewMost;
    // few: one workgroup for each that the CUs hold at a time, fewer where there are not so many steps
    const int64_t few_tiles = few_only ? rows / kFewRows + std::min(a.requests, a.tokens) : std::min(a.requests, a.tokens);
    const int64_t few = std::min<int64_t>(few_tiles * a.kv_heads * ((keys + few_step<F>() - 1) / few_step<F>()), 256 * few_waves<D, F, EXTRA>());
    // no more tiles than workgroups: by the bound on the new tokens, since the rows of each request are not known here
    const int64_t each = (std::min<int64_t>(max_new > 0 ? max_new : a.tokens, a.tokens) * a.group + kFewRows - 1) / kFewRows;
    const int64_t most_tiles = few_only ? std::min<int64_t>(few_tiles, each * std::min(a.requests, a.tokens)) : few_tiles;
    a.whole = !first && most_tiles * a.kv_heads <= 256 * few_waves<D, F, EXTRA>();
    if (!many_only) MARS_LAUNCH((k_attend_few<T, D, EXTRA, CAP, F>), dim3(unsigned(few + first)), dim3(256), 0, s, a);
    if (few_only) return MARS_OK;
    // many: no more than chunks of kMinChunk or more of the tiles' keys, or 2^kManyItemsLog2 chunks and one for each tile
    const int64_t tiles = rows / kManyRows + std::min<int64_t>(a.requests, first ? a.tokens : rows / (kFewMost + 1));
    const int64_t many = std::min(tiles * a.kv_heads * ((keys + kMinChunk - 1) / kMinChunk), (int64_t(1) << kManyItemsLog2) + tiles * a.kv_heads);
    MARS_CHECK(many < INT32_MAX, MARS_ERR_CAPACITY, "%lld tiles of rows", (long long)tiles);
    a.join_rows = tiles * a.kv_heads * (kManyRows / kJoinRows) < 1024 ? 1024 / D : kJoinRows;
    MARS_LAUNCH((k_attend_many<T, D, EXTRA, CAP, F>), dim3(unsigned(many + first)), dim3(256), 0, s, a);
    // no tile is in pieces where a row of the table is one chunk. Rows a workgroup of the join, 16 or 1024 / D: 256 rows under 8 heads over
    // 32,768 keys 17.0 and 12.3 us, two chunks of 511 tokens among 22 single ones 13.4 and 17.8.
    if (keys > kMinChunk && !(first && a.defer)) {
        const int64_t blocks = std::min<int64_t>(tiles * a.kv_heads * (kManyRows / join_rows_of<F>(a)), a.join_rows < kJoinRows ? 2048 : 1024);
        MARS_LAUNCH((k_attend_join<T, D, F>), dim3(unsigned(blocks)), dim3(256), 0, s, a);
    }
    return MARS_OK;
}

// With a.group_start: the groups over their prefixes, then every request from behind them on. Requests of up to shared_few_most() rows
// are then k_attend_few's, which reads their own keys once for every 16 rows, and which joins the pieces of the prefix's sums itself
// as it begins; with more rows three launches take what is one here. 32 requests of 20, 40 and 64 rows behind 6,016 shared keys (32/8
// heads of 128): over some 45 of their own 59, 76, 102 us (67, 88, 109 with three launches), over 675 86, 112, 143 (89, 111, 133), over
// 3,000 187, 267, 329 (184, 214, 235); in 8 bits 74, 92, 123 (92, 115, 140), 88, 118, 152 (110, 135, 158), 148, 192, 242 (190, 219, 239).
template <typename F>
constexpr int shared_few_most() { return F::c8 ? 64 : 48; }
template <typename T, int D, bool EXTRA, bool CAP, typename F>
int launch_phases(AttendArgs a, int32_t max_new, hipStream_t s) {
    if constexpr (F::share) {
        if (a.group_start) {
            const int64_t most = std::min<int64_t>(max_new > 0 ? max_new : a.tokens, a.tokens) * a.group;
            a.defer = most <= shared_few_most<F>();
            AttendArgs first = a;
            first.phase = 1;
            first.part_o = a.many_o;                         // k_attend_few's pieces of the one phase are read while it writes those of the other
            first.part_ml = a.many_ml;
            first.members = a.requests;
            first.requests = a.groups;
            MARS_TRY((launch_dim<T, D, EXTRA, CAP, F>(first, 0, s)));
            a.phase = 2;
        }
    }
    return launch_dim<T, D, EXTRA, CAP, F>(a, max_new, s);
}

// Kernels without extra terms, with times or episodes, and with a cap: its code costs calls without one (two chunks of 511
// tokens among 22 single ones, decayed, 121.7 us without it and 123.9 with it).
template <typename T, int D, typename F>
int launch_terms(const AttendArgs& a, int32_t max_new, hipStream_t s) {
    if (a.cap_rcp != 0.0f) return launch_phases<T, D, true, true, F>(a, max_new, s);
    return a.k_times || a.k_eps ? launch_phases<T, D, true, false, F>(a, max_new, s) : launch_phases<T, D, false, false, F>(a, max_new, s);
}

template <typename F>
int launch_form(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s) {
    const bool f16 = r.d.dtype == MARS_DTYPE_F16;
    switch (r.d.head_dim) {
        case 64: return f16 ? launch_terms<_Float16, 64, F>(a, max_new, s) : launch_terms<__bf16, 64, F>(a, max_new, s);
        case 128: return f16 ? launch_terms<_Float16, 128, F>(a, max_new, s) : launch_terms<__bf16, 128, F>(a, max_new, s);
        default: return f16 ? launch_terms<_Float16, 256, F>(a, max_new, s) : launch_terms<__bf16, 256, F>(a, max_new, s);
    }
}

}  // namespace
}  // namespace mars
