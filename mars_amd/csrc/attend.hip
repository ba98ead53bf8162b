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
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kSlack = 8.0f;       // how far a score may exceed the row's reference

template <typename T> struct Vec;
template <> struct Vec<_Float16> {
    using v8 = f16x8;
    static constexpr uint32_t exp_mask = 0x7C00u, one = 0x3C00u;
    __device__ static f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Vec<__bf16> {
    using v8 = bf16x8;
    static constexpr uint32_t exp_mask = 0x7F80u, one = 0x3F80u;
    __device__ static f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

template <typename V>
__device__ inline V load16(const void* p) {
    return __builtin_bit_cast(V, *static_cast<const u32x4*>(p));
}

// One unit of a launch's work: a tile of rows of a request under one kv head, over a range of its keys.
struct Item {
    int32_t request, tile, head, split, splits, chunk;
    int32_t part;              // first partial slot of the tile's splits
    bool found;
};

struct SchedLds {
    int64_t wsum[4];
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
// over all tiles), cuts the keys into chunks of work / a.items, and finds the request that its number falls to. The
// launch has enough workgroups for every item; the last ones may find none.
__device__ Item find_item(const AttendArgs& a, int b, int bm, int min_chunk, SchedLds& sh) {
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
    if (lane == 0) sh.wsum[wave] = work;
    if (tid == 0) sh.item.found = false;
    __syncthreads();
    work = (sh.wsum[0] + sh.wsum[1] + sh.wsum[2] + sh.wsum[3]) * a.kv_heads;
    const int64_t per = max((work * 32 + a.items - 1) / a.items, int64_t(min_chunk));
    const int64_t chunk0 = (per + 127) & ~int64_t(127);
    int64_t items_before = 0, parts_before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 256) {
        int tiles = tiles0, keys = keys0;
        if (r0) request_of(a, r0 + tid, bm, &tiles, &keys);
        // no more than kMaxSplits chunks a request
        const int64_t chunk = max(chunk0, (int64_t(keys) + kMaxSplits * 128 - 1) / (kMaxSplits * 128) * 128);
        const int64_t splits = max(int64_t(1), (keys + chunk - 1) / chunk);
        const int64_t items = int64_t(tiles) * a.kv_heads * splits;
        const int64_t parts = splits > 1 ? items : 0;
        int64_t xi = items, xp = parts;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t yi = __shfl_up((long long)xi, unsigned(o)), yp = __shfl_up((long long)xp, unsigned(o));
            if (lane >= o) { xi += yi; xp += yp; }
        }
        __syncthreads();
        if (lane == 63) sh.wsum[wave] = (xi << 32) | xp;      // both below 2^31: see the launch
        __syncthreads();
        int64_t bi = items_before, bp = parts_before;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int64_t s = sh.wsum[w];
            if (w < wave) { bi += s >> 32; bp += s & 0xFFFFFFFF; }
            items_before += s >> 32;
            parts_before += s & 0xFFFFFFFF;
        }
        const int64_t mine = bi + xi - items;
        if (b >= mine && b < mine + items) {
            const int64_t local = b - mine, tile_head = local / splits;
            Item it;
            it.request = r0 + tid;
            it.split = int32_t(local - tile_head * splits);
            it.head = int32_t(tile_head % a.kv_heads);
            it.tile = int32_t(tile_head / a.kv_heads);
            it.splits = int32_t(splits);
            it.chunk = int32_t(min(chunk, int64_t(INT32_MAX / 2)));
            it.part = int32_t(bp + xp - parts + tile_head * splits);
            it.found = true;
            sh.item = it;
        }
        if (b < items_before) break;
    }
    __syncthreads();
    return sh.item;
}

// ---- few rows: 16 at a time, keys straight from the cache to registers -----------------
// Bound by the cache's bytes. 4 waves take the 32-key steps of the chunk in turn; a wave reads
// its step's K and V rows into registers (16 bytes a lane) one step ahead, so that 12 waves of
// a CU keep some 100 KB of loads in flight, and the waves' sums are joined at the end.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attend_few(AttendArgs a) {
    using V = typename Vec<T>::v8;
    constexpr int KC = D / 32, VB = D / 16;
    __shared__ SchedLds sched;
    __shared__ float ml[4][16][2];
    __shared__ __attribute__((aligned(16))) float ob[2][16][D + 4];
    __shared__ int arrived_last;
    const Item it = find_item(a, int(blockIdx.x), kFewRows, 128, sched);
    if (!it.found) return;
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, h = lane >> 4;
    const int r = it.request, P1 = (1 << a.page_shift) - 1;
    const int row0 = max(a.q_start[r], 0), n = min(a.q_start[r + 1], a.tokens) - row0;
    const int keys = int(min(int64_t(max(a.kv_lens[r], 0)), int64_t(a.max_pages) << a.page_shift));
    const int m = it.tile * kFewRows + col;                 // this lane's row: token i, head of the group
    const bool row_ok = m < n * a.group;
    const int i = row_ok ? m / a.group : 0, hq = it.head * a.group + (row_ok ? m - i * a.group : 0);
    const int64_t row = int64_t(row0) + i;
    const int prefix = a.prefix ? min(max(a.prefix[r], 0), keys) : 0;
    const int limit = row_ok ? min(max(keys - n + i + 1, prefix), keys) : 0;   // keys [0, limit) may be seen
    const float dec = a.decay ? a.decay[hq] * 1.4426950408889634f : 0.0f;
    const float tq = a.decay ? a.q_times[row] : 0.0f;
    const int eq = a.q_eps ? a.q_eps[row] : -1;

    V q[KC];
    const T* const qp = static_cast<const T*>(a.q) + row * a.q_stride + int64_t(hq) * D + h * 8;
#pragma unroll
    for (int c = 0; c < KC; ++c) q[c] = load16<V>(qp + c * 32);

    int lo = limit, hi = limit;                             // over the wave's rows
    if (!row_ok) lo = INT32_MAX;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    const int k0 = it.split * it.chunk, k1 = min(k0 + it.chunk, hi);
    const int steps = k1 > k0 ? (k1 - k0 + 31) >> 5 : 0;

    const int32_t* const table = a.table + int64_t(r) * a.max_pages;
    const int last_page = keys > 0 ? (keys - 1) >> a.page_shift : 0;
    const int ki = 8 * (col >> 2) + (col & 3);              // key of A row `col`, first block (the second: + 4)
    const T* const kp = static_cast<const T*>(a.k_pages) + (int64_t(it.head) << a.page_shift) * D + h * 8;
    const T* const vp = static_cast<const T*>(a.v_pages) + (int64_t(it.head) << a.page_shift) * D + (int64_t(col) << a.page_shift);
    auto page_at = [&](int key) {
        const int id = table[min(key >> a.page_shift, last_page)];
        return uint32_t(id) < uint32_t(a.num_pages) ? id : 0;
    };
    V kf[2][KC], vf[VB];
    f32x4 tk[2];
    i32x4 ek[2];
    auto load_k = [&](int s) {
        const int key = k0 + s * 32 + ki;
        const T* const p = kp + page_at(key) * a.k_stride + int64_t(key & P1) * D;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < KC; ++c) kf[b][c] = load16<V>(p + b * 4 * D + c * 32);
    };
    auto load_v = [&](int s) {
        const int key = k0 + s * 32 + h * 8, pg = page_at(key);
        const T* const p = vp + pg * a.v_stride + (key & P1);
#pragma unroll
        for (int d = 0; d < VB; ++d) vf[d] = load16<V>(p + (int64_t(d) * 16 << a.page_shift));
        const int64_t slot = (int64_t(pg) << a.page_shift) + (key & P1);
        if (a.k_times) { tk[0] = *reinterpret_cast<const f32x4*>(a.k_times + slot); tk[1] = *reinterpret_cast<const f32x4*>(a.k_times + slot + 4); }
        if (a.k_eps) { ek[0] = *reinterpret_cast<const i32x4*>(a.k_eps + slot); ek[1] = *reinterpret_cast<const i32x4*>(a.k_eps + slot + 4); }
    };

    f32x4 o[VB];
#pragma unroll
    for (int d = 0; d < VB; ++d) o[d] = f32x4{0, 0, 0, 0};
    float mref = 0.0f, mtop = -kInf, l = 0.0f;              // mtop: -inf until the row has seen a key, then mref + kSlack

    if (wave < steps) { load_k(wave); load_v(wave); }
    for (int s = wave; s < steps; s += 4) {
        const int kb = k0 + s * 32 + h * 8;                 // this lane's 8 keys
        f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            acc[0] = Vec<T>::mma(kf[0][c], q[c], acc[0]);
            acc[1] = Vec<T>::mma(kf[1][c], q[c], acc[1]);
        }
        if (s + 4 < steps) load_k(s + 4);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = acc[j >> 2][j & 3] * a.scale_log2;
        if (a.cap_log2 != 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = a.cap_log2 * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[j])));
        }
        if (a.k_times) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] -= dec * fmaxf(0.0f, tq - tk[j >> 2][j & 3]);
        }
        uint32_t seen = 0xFFu;
        const bool whole = k0 + s * 32 + 32 <= lo && !a.k_eps;
        if (!whole) {
            seen = kb >= limit ? 0u : (kb + 8 <= limit ? 0xFFu : (1u << (limit - kb)) - 1u);
            if (a.k_eps) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = ek[j >> 2][j & 3];
                    if (!(e < 0 || eq < 0 || e == eq)) seen &= ~(1u << j);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (seen >> j) & 1u ? x[j] : -kInf;
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
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
        V p;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float w = __builtin_amdgcn_exp2f(x[j] - mref);
            l += w;
            p[j] = T(w);
        }
        if (whole) {
#pragma unroll
            for (int d = 0; d < VB; ++d) o[d] = Vec<T>::mma(vf[d], p, o[d]);
        } else {
            // Keys that some row does not see: a weight of 0 times an infinity or NaN would still be NaN. Such values
            // are taken out of the product and added to the rows that see them, by products of the rows' masks with
            // indicators of +inf, -inf and NaN. Values past the request's keys are nobody's.
            u32x4 sb;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sb[j] = ((seen >> (2 * j)) & 1u ? Vec<T>::one : 0u) | ((seen >> (2 * j + 1)) & 1u ? Vec<T>::one << 16 : 0u);
            const V sv = __builtin_bit_cast(V, sb);
#pragma unroll
            for (int d = 0; d < VB; ++d) {
                u32x4 b = __builtin_bit_cast(u32x4, vf[d]);
                uint32_t odd = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (kb + 2 * j >= keys) b[j] = 0;
                    else if (kb + 2 * j + 1 >= keys) b[j] &= 0xFFFFu;
                    constexpr uint32_t E = Vec<T>::exp_mask;
                    odd |= uint32_t((b[j] & E) == E) | uint32_t((b[j] & (E << 16)) == (E << 16));
                }
                if (__any(odd != 0)) {
                    u32x4 up = {0, 0, 0, 0}, dn = {0, 0, 0, 0}, nan = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int sh = 16 * (j & 1);
                        const uint32_t bits = (b[j >> 1] >> sh) & 0xFFFFu, one = Vec<T>::one << sh;
                        if ((bits & Vec<T>::exp_mask) != Vec<T>::exp_mask) continue;
                        if ((bits & 0x7FFFu) != Vec<T>::exp_mask) nan[j >> 1] |= one;
                        else if (bits & 0x8000u) dn[j >> 1] |= one;
                        else up[j >> 1] |= one;
                        b[j >> 1] &= ~(0xFFFFu << sh);
                    }
                    const f32x4 zero = {0, 0, 0, 0};
                    const f32x4 cu = Vec<T>::mma(__builtin_bit_cast(V, up), sv, zero);
                    const f32x4 cd = Vec<T>::mma(__builtin_bit_cast(V, dn), sv, zero);
                    const f32x4 cn = Vec<T>::mma(__builtin_bit_cast(V, nan), sv, zero);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[d][j] += (cu[j] > 0.0f ? kInf : 0.0f) + (cd[j] > 0.0f ? -kInf : 0.0f) + (cn[j] > 0.0f ? __builtin_nanf("") : 0.0f);
                }
                o[d] = Vec<T>::mma(__builtin_bit_cast(V, b), p, o[d]);
            }
        }
        if (s + 4 < steps) load_v(s + 4);
    }

    // join the waves: references first, then sums and O, in wave order
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float mw = mtop == -kInf ? -kInf : mref;
    if (h == 0) ml[wave][col][0] = mw;
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
            for (int d = 0; d < VB; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) op[d * 16 + j] = mall == -kInf ? T(0.0f) : T(o[d][j] * inv);
            if (a.lse && h == 0) a.lse[row * a.q_heads + hq] = mall == -kInf ? -kInf : (mall + __builtin_amdgcn_logf(lall)) * kLn2;
        }
        if (row_ok && joined) {
            float* const po = a.part_o + (int64_t(it.part + it.split) * kFewRows + col) * D + h * 4;
#pragma unroll
            for (int d = 0; d < VB; ++d) *reinterpret_cast<f32x4*>(po + d * 16) = o[d];
            if (h == 0) a.part_ml[int64_t(it.part + it.split) * kFewRows + col] = make_float2(mall, lall);
        }
    }
    if (!joined) return;
    // the tile's last workgroup to arrive joins the splits, in their order
    __threadfence();
    __syncthreads();
    if (tid == 0) arrived_last = atomicAdd(&a.arrived[it.part], 1u) == uint32_t(it.splits - 1);
    __syncthreads();
    if (!arrived_last) return;
    __threadfence();
    if (tid == 0) a.arrived[it.part] = 0;
    const int valid = min(kFewRows, n * a.group - it.tile * kFewRows);
    for (int e = tid; e < valid * (D / 4); e += 256) {
        const int rr = e / (D / 4), d4 = e % (D / 4);
        float top = -kInf;
        for (int s = 0; s < it.splits; ++s) top = fmaxf(top, a.part_ml[int64_t(it.part + s) * kFewRows + rr].x);
        f32x4 sum = {0, 0, 0, 0};
        float lsum = 0.0f;
        for (int s = 0; s < it.splits; ++s) {
            const float2 p = a.part_ml[int64_t(it.part + s) * kFewRows + rr];
            const float w = p.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(p.x - top);
            lsum += w * p.y;
            sum += w * *reinterpret_cast<const f32x4*>(a.part_o + (int64_t(it.part + s) * kFewRows + rr) * D + d4 * 4);
        }
        const int mm = it.tile * kFewRows + rr, ii = mm / a.group, hh = it.head * a.group + mm - ii * a.group;
        const float inv = 1.0f / lsum;
        T* const op = static_cast<T*>(a.out) + (int64_t(row0) + ii) * a.out_stride + int64_t(hh) * D + d4 * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) op[j] = top == -kInf ? T(0.0f) : T(sum[j] * inv);
        if (a.lse && d4 == 0)
            a.lse[(int64_t(row0) + ii) * a.q_heads + hh] = top == -kInf ? -kInf : (top + __builtin_amdgcn_logf(lsum)) * kLn2;
    }
}

template <typename T, int D>
int launch_few(AttendArgs a, hipStream_t s) {
    const int64_t tiles = int64_t(a.tokens) * a.group / kFewRows + std::min(a.requests, a.tokens);
    const int64_t grid = a.items + tiles * a.kv_heads;
    MARS_CHECK(grid <= INT32_MAX, MARS_ERR_CAPACITY, "%lld tiles of rows", (long long)grid);
    MARS_LAUNCH((k_attend_few<T, D>), dim3(unsigned(grid)), dim3(256), 0, s, a);
    return MARS_OK;
}

template <typename T>
int launch_typed(const mars_reader& r, AttendArgs a, int32_t max_new, hipStream_t s) {
    (void)max_new;
    a.rows_lo = 0;
    a.rows_hi = INT32_MAX;
    a.items = kFewItems;
    switch (r.d.head_dim) {
        case 64: return launch_few<T, 64>(a, s);
        case 128: return launch_few<T, 128>(a, s);
        default: return launch_few<T, 256>(a, s);
    }
}

}  // namespace

int launch_attend(const mars_reader& r, AttendArgs a, int32_t max_new, hipStream_t s) {
    return r.d.dtype == MARS_DTYPE_F16 ? launch_typed<_Float16>(r, a, max_new, s) : launch_typed<__bf16>(r, a, max_new, s);
}

}  // namespace mars
