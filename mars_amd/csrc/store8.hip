// ============================================================================
//  store8.hip — tokens quantised as they are written to a cache of 8 bits
//  (mars_kv_store8), and slots of either cache read back (mars_kv_load, mars_kv_load8).
//
//  A head of a token is D elements x. Its exponent k is the least integer with max |x| <= 448 2^k over the finite x (448 is
//  e4m3's largest value), but at least that of the reader's type: -15 (float16), -117 (bfloat16), so that 2^(k - 9), the least
//  value that can be held, is one of that type's. Held: e4m3(x 2^-k), rounded once to nearest even, and the byte k + 127.
//  Finite elements beyond 61440 (or 240 2^120), the largest held values that the type has too, become that. The scaling is
//  exact, powers of two lose nothing, and one scale a token and head keeps each token's precision whatever its
//  neighbours are: the values keep e4m3's own relative precision of 2^-4 down to 2^-6 units of 2^k, the head's largest being 224 to 448 of
//  them: to 2^-13.8 to 2^-14.8 of it.
// ============================================================================
#include "reader.hpp"

#include <type_traits>

namespace mars {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
constexpr int least_exponent() { return __is_same(T, _Float16) ? -15 : -117; }

// x, or where it is finite and larger than what can be held as a finite T, that.
template <typename T>
__device__ inline float holdable(float x) {
    constexpr float most = __is_same(T, _Float16) ? 61440.0f : 240.0f * 0x1p120f;
    return fabsf(x) < __builtin_inff() ? fminf(fmaxf(x, -most), most) : x;
}
__device__ inline float finite_size(float x) {
    const float m = fabsf(x);
    return m < __builtin_inff() ? m : 0.0f;
}
// The exponent byte for a head whose largest finite size is `top`: 448 = 1.75 2^8.
template <typename T>
__device__ inline uint32_t exponent_for(float top) {
    const uint32_t b = __float_as_uint(top);
    const int k = int(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return uint32_t(max(k, least_exponent<T>()) + 127);
}
// 2^-k of an exponent byte (k + 127 in 10 .. 247).
__device__ inline float inverse_power(uint32_t e) { return __uint_as_float((254u - e) << 23); }
// Two values into half of a word; infinities become NaN. Sizes are at most 448: nothing saturates.
template <bool HI>
__device__ inline uint32_t to_e4m3(uint32_t word, float x, float y, float inv) {
    const float nan = __builtin_nanf("");
    x = fabsf(x) < __builtin_inff() ? x * inv : nan;
    y = fabsf(y) < __builtin_inff() ? y * inv : nan;
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x, y, int(word), HI));
}

// The largest of N neighbouring lanes (from a multiple of N on), in each of them. Up to 16 within a row of lanes: the neighbour, the other
// pair of four, then mirrored halves, whose lanes agree by then.
template <int CTRL>
__device__ inline float max_dpp(float x) {
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true)));
}
template <int N>
__device__ inline float max_over(float x) {
    if constexpr (N > 1) x = max_dpp<0xB1>(x);
    if constexpr (N > 2) x = max_dpp<0x4E>(x);
    if constexpr (N > 4) x = max_dpp<0x141>(x);
    if constexpr (N > 8) x = max_dpp<0x140>(x);
    if constexpr (N > 16) x = fmaxf(x, __shfl_xor(x, 16));
    if constexpr (N > 32) x = fmaxf(x, __shfl_xor(x, 32));
    return x;
}

// Few tokens: a workgroup to each. q as in k_kv_store, a pair a thread and turn; a wave to a head of k or v. Latency bound (32
// tokens 5.8 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv_store8(StoreArgs a) {
    const int t = int(blockIdx.x), half = a.rope_dim / 2, tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    __shared__ float sn[128], cs[128];
    for (int i = tid; i < half; i += 256) {
        turn(a.s.positions[int64_t(a.axis[i]) * a.s.num_tokens + t], a.freq[i], &sn[i], &cs[i]);
        if (a.s.inverse) sn[i] = -sn[i];
    }
    __syncthreads();
    const int64_t slot = a.s.slots ? a.s.slots[t] : -1;
    const bool stored = slot >= 0 && slot < a.slots;
    const T* const q = static_cast<const T*>(a.s.q);
    for (int e = tid; q && e < a.q_heads * (D / 2); e += 256) {          // q_out may be q: a thread reads and writes both of a pair
        const int h = e / (D / 2), j = e % (D / 2);
        const T* const x = q + t * a.s.q_stride + h * D;
        T* const to = static_cast<T*>(a.s.q_out) + t * a.s.q_out_stride + h * D;
        const bool turns = j < half;
        const int i0 = turns && !a.adjacent ? j : 2 * j, i1 = turns && !a.adjacent ? j + half : 2 * j + 1;
        const float y = float(x[i0]), z = float(x[i1]), c = turns ? cs[j] : 1.0f, s = turns ? sn[j] : 0.0f;
        const T lo = turns ? T(y * c - z * s) : x[i0], hi = turns ? T(y * s + z * c) : x[i1];
        to[i0] = lo;
        to[i1] = hi;
    }
    if (!a.s.k || !stored) return;
    const int64_t page = slot >> a.page_shift;
    const int off = int(slot & ((1 << a.page_shift) - 1)), P = 1 << a.page_shift;
    constexpr int N = D / 64;                                // elements of a lane; D / 2 pairs over 64 lanes
    for (int h = wave; h < a.kv_heads; h += 4) {
        const T* const k = static_cast<const T*>(a.s.k) + t * a.s.k_stride + h * D;
        const T* const v = static_cast<const T*>(a.s.v) + t * a.s.v_stride + h * D;
        float w[N];
#pragma unroll
        for (int u = 0; u < N; ++u) w[u] = holdable<T>(float(v[lane + 64 * u]));
        constexpr int NP = (N + 1) / 2;
        float lo[NP], hi[NP], top = 0.0f;
        int i0[NP], i1[NP];
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int j = min(lane + 64 * u, D / 2 - 1);     // heads of 64: half the lanes repeat the last pair
            const bool turns = j < half;
            i0[u] = turns && !a.adjacent ? j : 2 * j;
            i1[u] = turns && !a.adjacent ? j + half : 2 * j + 1;
            const float y = float(k[i0[u]]), z = float(k[i1[u]]);
            lo[u] = holdable<T>(turns ? y * cs[j] - z * sn[j] : y);
            hi[u] = holdable<T>(turns ? y * sn[j] + z * cs[j] : z);
            top = fmaxf(top, fmaxf(finite_size(lo[u]), finite_size(hi[u])));
        }
        const uint32_t ek = exponent_for<T>(max_over<64>(top));
        uint8_t* const kp = static_cast<uint8_t*>(a.k_pages) + page * a.k_stride + (int64_t(h) * P + off) * D;
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const uint32_t b = to_e4m3<false>(0, lo[u], hi[u], inverse_power(ek));
            if (lane + 64 * u >= D / 2) continue;
            kp[i0[u]] = uint8_t(b);
            kp[i1[u]] = uint8_t(b >> 8);
        }
        top = 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u) top = fmaxf(top, finite_size(w[u]));
        const uint32_t ev = exponent_for<T>(max_over<64>(top));
        uint8_t* const vp = static_cast<uint8_t*>(a.v_pages) + page * a.v_stride + int64_t(h) * D * P + off;
#pragma unroll
        for (int u = 0; u < N; ++u) vp[int64_t(lane + 64 * u) * P] = uint8_t(to_e4m3<false>(0, w[u], 0.0f, inverse_power(ev)));
        if (lane == 0) {
            const int64_t at = (page * a.kv_heads + h) * P + off;
            a.k_scales[at] = uint8_t(ek);
            a.v_scales[at] = uint8_t(ev);
        }
    }
    if (tid == 0 && a.times && a.s.times) a.times[slot] = a.s.times[t];
    if (tid == 0 && a.eps && a.s.episodes) a.eps[slot] = a.s.episodes[t];
}

// Many tokens: a workgroup takes kTile of them under one kv head, as k_kv_store_tile does. A head's elements lie with D / 16
// (k, pieces of 16) or D / 8 (v) neighbouring lanes, which find its largest between them; v goes through LDS as bytes, and a
// thread that has 4 elements of 8 tokens turns them with byte permutations into 8 bytes a row of the page. 4,099 tokens, 3 axes:
// 32/8 heads of 128 27 to 29 us (tiles of 64 tokens 30), 8/2 heads of 256 19 us (tiles of 32 24).
template <int D>
constexpr int store8_tile() { return D == 256 ? 16 : D == 128 ? 32 : 64; }

// 4 x 4 bytes: word j of `in` holds 4 elements of token j; word e of the result element e of 4 tokens.
__device__ inline u32x4 turned4(u32x4 in) {
    const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u), d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
    return u32x4{__builtin_amdgcn_perm(c, a, 0x05040100u), __builtin_amdgcn_perm(c, a, 0x07060302u), __builtin_amdgcn_perm(d, b, 0x05040100u),
                 __builtin_amdgcn_perm(d, b, 0x07060302u)};
}

template <typename T, int D>
__global__ __launch_bounds__(256) void k_kv_store8_tile(StoreArgs a) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    constexpr int kTile = store8_tile<D>(), VS = D / 4 + 1;  // words of a token's row of v in LDS
    __shared__ __attribute__((aligned(16))) float2 turns[kTile][D / 2];          // cos, sin
    __shared__ uint32_t vt[kTile][VS];
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
    // everything the workgroup reads is on the way before the angles are computed: its v and k, and of q the first pieces.
    // q and k: two pieces of 8 elements of a head a thread, the partners of each other where they turn (both are read
    // before either is written: q_out may be q)
    constexpr int VU = kTile * (D / 8) / 256, KU = kTile * (D / 16) / 256, U = 4;
    const int turning = half / 8, pairs = nt * group * (D / 16);
    auto first_of = [&](int c) { return c < turning && !a.adjacent ? c * 8 : c * 16; };
    auto second_of = [&](int c) { return c < turning && !a.adjacent ? half + c * 8 : c * 16 + 8; };
    v8 vr[VU], ky[KU], kz[KU], y[U], z[U];
    if (k) {
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int e = tid + u * 256, i = e / (D / 16), c = e % (D / 16);
            if (i >= nt) break;
            const T* const x = k + (t0 + i) * a.s.k_stride + head * D;
            ky[u] = *reinterpret_cast<const v8*>(x + first_of(c));
            kz[u] = *reinterpret_cast<const v8*>(x + second_of(c));
        }
#pragma unroll
        for (int u = 0; u < VU; ++u) {
            const int e = tid + u * 256, i = e / (D / 8), c = e % (D / 8);
            if (i < nt) vr[u] = *reinterpret_cast<const v8*>(v + (t0 + i) * a.s.v_stride + head * D + c * 8);
        }
    }
    auto read_pairs = [&](int e0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * 256, c = e % (D / 16), ih = e / (D / 16), i = ih / group, hh = ih % group;
            if (e >= pairs) break;
            const T* const x = q + (t0 + i) * a.s.q_stride + (head * group + hh) * D;
            y[u] = *reinterpret_cast<const v8*>(x + first_of(c));
            z[u] = *reinterpret_cast<const v8*>(x + second_of(c));
        }
    };
    if (q) read_pairs(tid);
    for (int e = tid; e < nt * half; e += 256) {
        const int i = e / half, f = e % half;
        float sn, cs;
        turn(a.s.positions[int64_t(a.axis[f]) * a.s.num_tokens + t0 + i], a.freq[f], &sn, &cs);
        turns[i][f] = make_float2(cs, a.s.inverse ? -sn : sn);
    }
    __syncthreads();
    // both pieces of a pair turned, in fp32
    auto turned = [&](int i, int c, v8 yy, v8 zz, float (&u)[8], float (&w)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { u[j] = float(yy[j]); w[j] = float(zz[j]); }
        if (c < turning && !a.adjacent) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 f = turns[i][c * 8 + j];
                const float p = u[j], r = w[j];
                u[j] = p * f.x - r * f.y;
                w[j] = p * f.y + r * f.x;
            }
        } else if (c < turning) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = turns[i][c * 8 + j], g = turns[i][c * 8 + 4 + j];          // pairs j and 4 + j of the 16 elements
                const float ya = u[2 * j], yb = u[2 * j + 1], za = w[2 * j], zb = w[2 * j + 1];
                u[2 * j] = ya * f.x - yb * f.y;
                u[2 * j + 1] = ya * f.y + yb * f.x;
                w[2 * j] = za * g.x - zb * g.y;
                w[2 * j + 1] = za * g.y + zb * g.x;
            }
        }
    };
    if (k) {
        auto eight = [](const float (&x)[8], float inv) {
            return u32x2{to_e4m3<true>(to_e4m3<false>(0, x[0], x[1], inv), x[2], x[3], inv), to_e4m3<true>(to_e4m3<false>(0, x[4], x[5], inv), x[6], x[7], inv)};
        };
#pragma unroll
        for (int n = 0; n < VU; ++n) {
            const int e = tid + n * 256, i = e / (D / 8), c = e % (D / 8);
            if (i >= nt) break;                              // a token's lanes go together
            float x[8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = holdable<T>(float(vr[n][j]));
                top = fmaxf(top, finite_size(x[j]));
            }
            const uint32_t ev = exponent_for<T>(max_over<D / 8>(top));
            const u32x2 b = eight(x, inverse_power(ev));
            vt[i][c * 2] = b[0];
            vt[i][c * 2 + 1] = b[1];
            const int64_t s = slot_of[i];
            if (c == 0 && s >= 0) a.v_scales[((s >> a.page_shift) * a.kv_heads + head) * P + (s & (P - 1))] = uint8_t(ev);
        }
#pragma unroll
        for (int n = 0; n < KU; ++n) {
            const int e = tid + n * 256, i = e / (D / 16), c = e % (D / 16);
            if (i >= nt) break;                              // as above
            float u[8], w[8], top = 0.0f;
            turned(i, c, ky[n], kz[n], u, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                u[j] = holdable<T>(u[j]);
                w[j] = holdable<T>(w[j]);
                top = fmaxf(top, fmaxf(finite_size(u[j]), finite_size(w[j])));
            }
            const uint32_t ek = exponent_for<T>(max_over<D / 16>(top));
            if (slot_of[i] < 0) continue;
            const int64_t page = slot_of[i] >> a.page_shift, off = slot_of[i] & (P - 1);
            uint8_t* const to = static_cast<uint8_t*>(a.k_pages) + page * a.k_stride + (int64_t(head) * P + off) * D;
            *reinterpret_cast<u32x2*>(to + first_of(c)) = eight(u, inverse_power(ek));
            *reinterpret_cast<u32x2*>(to + second_of(c)) = eight(w, inverse_power(ek));
            if (c == 0) a.k_scales[(page * a.kv_heads + head) * P + off] = uint8_t(ek);
        }
        if (tid < kTile) {
            const int64_t s = slot_of[tid];
            bool first = s >= 0 && s % 8 == 0 && tid + 8 <= nt;
            for (int j = 1; j < 8 && first; ++j) first = slot_of[tid + j] == s + j;
            lead[tid] = first;
        }
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
            const int e = e0 + n * 256, c = e % (D / 16), ih = e / (D / 16), i = ih / group, hh = ih % group;
            if (e >= pairs) break;
            T* const to = static_cast<T*>(a.s.q_out) + (t0 + i) * a.s.q_out_stride + (head * group + hh) * D;
            v8 lo = y[n], hi = z[n];
            if (c < turning) {
                float u[8], w[8];
                turned(i, c, lo, hi, u, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) { lo[j] = T(u[j]); hi[j] = T(w[j]); }
            }
            *reinterpret_cast<v8*>(to + first_of(c)) = lo;
            *reinterpret_cast<v8*>(to + second_of(c)) = hi;
        }
    }
    if (!v) return;
    __syncthreads();
    uint8_t* const vp = static_cast<uint8_t*>(a.v_pages) + int64_t(head) * D * P;
    const int ng = counts[0], ns = counts[1];
    for (int e = tid; e < ng * (D / 4); e += 256) {
        const int d4 = e / ng, i = groups[e % ng];
        const u32x4 lo = turned4(u32x4{vt[i][d4], vt[i + 1][d4], vt[i + 2][d4], vt[i + 3][d4]});
        const u32x4 hi = turned4(u32x4{vt[i + 4][d4], vt[i + 5][d4], vt[i + 6][d4], vt[i + 7][d4]});
        uint8_t* const to = vp + (slot_of[i] >> a.page_shift) * a.v_stride + (int64_t(d4) * 4 << a.page_shift) + (slot_of[i] & (P - 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x2*>(to + (int64_t(j) << a.page_shift)) = u32x2{lo[j], hi[j]};
    }
    for (int e = tid; e < ns * D; e += 256) {
        const int d = e / ns, i = singles[e % ns];
        vp[(slot_of[i] >> a.page_shift) * a.v_stride + (int64_t(d) << a.page_shift) + (slot_of[i] & (P - 1))] = uint8_t(vt[i][d / 4] >> (8 * (d % 4)));
    }
}

// ---- load ---------------------------------------------------------------------------
// A workgroup takes 64 tokens under one kv head. k's rows lie as the outputs do. Of v, whose pages hold the tokens of an element side by
// side, a run of tokens that lies within 8 slots from a multiple of 8 on is read as one piece an element (8 bytes of e4m3, 16 of
// T: always inside the page, whichever of the 8 are wanted), and goes through LDS to rows. Bound by the bytes: 20,011 tokens of 8 heads
// of 128 in runs of 700, 124 MB, 28 us (4.4 TB/s); 137 tokens of 12 heads of 64 4.7 us.
constexpr int kLoadTile = 64;

template <typename T, int D, bool C8>
__global__ __launch_bounds__(256) void k_kv_load(LoadArgs a) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    constexpr int VS = D + 8;                                // elements of a token's row of v in LDS
    __shared__ __attribute__((aligned(16))) T vt[kLoadTile][VS];
    __shared__ int64_t slot_of[kLoadTile];
    __shared__ uint8_t runs[kLoadTile + 1];                  // the first tokens of the runs, and the end of the last
    __shared__ int count;
    const int t0 = int(blockIdx.x) * kLoadTile, head = int(blockIdx.y), tid = int(threadIdx.x);
    const int nt = min(kLoadTile, a.s.num_tokens - t0), P = 1 << a.page_shift;
    if (tid < 64) {
        int64_t s = tid < nt ? a.s.slots[t0 + tid] : -1;
        if (s >= a.slots) s = -1;
        slot_of[tid] = s;
        const int64_t before = __shfl_up((long long)s, 1u);
        const bool first = tid < nt && (tid == 0 || s < 0 || s % 8 == 0 || s != before + 1);
        const uint64_t on = __ballot(first);
        if (first) runs[__popcll(on & ((1ull << tid) - 1))] = uint8_t(tid);
        if (tid == 0) {
            count = __popcll(on);
            runs[__popcll(on)] = uint8_t(nt);
        }
        if (head == 0 && s >= 0) {
            if (a.s.times) a.s.times[t0 + tid] = a.times[s];
            if (a.s.episodes) a.s.episodes[t0 + tid] = a.eps[s];
        }
    }
    __syncthreads();
    if (!a.s.k) return;
    auto power_of = [](uint32_t e) { return __uint_as_float(e << 23); };         // the conversions read the exponent alone
    auto two = [](uint32_t w, float s, auto hi) {
        if constexpr (__is_same(T, _Float16)) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, decltype(hi)::value));
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, decltype(hi)::value));
    };
    // k: 16 elements a thread and turn of e4m3, 8 of T
    constexpr int E = C8 ? 16 : 8;
    for (int e = tid; e < nt * (D / E); e += 256) {
        const int i = e / (D / E), c = e % (D / E);
        const int64_t s = slot_of[i];
        if (s < 0) continue;
        const int64_t page = s >> a.page_shift, off = s & (P - 1), at = page * a.k_stride + (int64_t(head) * P + off) * D + c * E;
        T* const to = static_cast<T*>(a.s.k) + (t0 + i) * a.s.k_stride + head * D + c * E;
        if constexpr (C8) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.k_pages) + at);
            const float f = power_of(a.k_scales[(page * a.kv_heads + head) * P + off]);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                *reinterpret_cast<u32x4*>(to + 8 * u) = u32x4{two(w[2 * u], f, std::false_type{}), two(w[2 * u], f, std::true_type{}),
                                                              two(w[2 * u + 1], f, std::false_type{}), two(w[2 * u + 1], f, std::true_type{})};
        } else {
            *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.k_pages) + at);
        }
    }
    // v: two elements of a run a thread and turn
    const int n = count;
    for (int e = tid; e < n * (D / 2); e += 256) {
        const int d = e / n * 2, run = e % n, i = runs[run], end = runs[run + 1];
        const int64_t s = slot_of[i];
        if (s < 0) continue;
        const int64_t page = s >> a.page_shift, off = s & (P - 1) & ~int64_t(7), at = page * a.v_stride + ((int64_t(head) * D + d) << a.page_shift) + off;
        const int o = int(s & 7);
        uint32_t x[8];                                       // of 8 tokens, the pair of elements
        if constexpr (C8) {
            const uint8_t* const p = static_cast<const uint8_t*>(a.v_pages) + at;
            const u32x2 lo = *reinterpret_cast<const u32x2*>(p), hi = *reinterpret_cast<const u32x2*>(p + P);
            const u32x2 f = *reinterpret_cast<const u32x2*>(a.v_scales + (page * a.kv_heads + head) * P + off);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pair = ((lo[j / 4] >> (8 * (j % 4))) & 0xFFu) | (((hi[j / 4] >> (8 * (j % 4))) & 0xFFu) << 8);
                x[j] = two(pair, power_of((f[j / 4] >> (8 * (j % 4))) & 0xFFu), std::false_type{});
            }
        } else {
            const T* const p = static_cast<const T*>(a.v_pages) + at;
            const u32x4 lo = *reinterpret_cast<const u32x4*>(p), hi = *reinterpret_cast<const u32x4*>(p + P);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_perm(hi[j / 2], lo[j / 2], j % 2 ? 0x07060302u : 0x05040100u);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= o && i + j - o < end) *reinterpret_cast<uint32_t*>(&vt[i + j - o][d]) = x[j];
    }
    __syncthreads();
    for (int e = tid; e < nt * (D / 8); e += 256) {
        const int i = e / (D / 8), c = e % (D / 8);
        if (slot_of[i] >= 0) *reinterpret_cast<v8*>(static_cast<T*>(a.s.v) + (t0 + i) * a.s.v_stride + head * D + c * 8) = *reinterpret_cast<const v8*>(&vt[i][c * 8]);
    }
}

// Tokens up to which a workgroup takes one of them; twice as many where tiles would not give most CUs a workgroup. us by token and by tile
// (more heads of less: tiles sooner):
//   tokens            1,024         1,100         2,048         4,099
//   32/8 of 128       14.4          -     14.5    -     17.1    -     26.5
//   8/2 of 256        8.8           -     12.9    -     14.2    -     19.4
//   12/12 of 64       8.6           -     10.0    -     11.8    -     18.0
constexpr int32_t kStore8Few = 1024;

template <typename T, int D>
int launch_store_dim(const StoreArgs& a, hipStream_t s) {
    const int64_t tiles = (int64_t(a.s.num_tokens) + store8_tile<D>() - 1) / store8_tile<D>();
    if (a.s.num_tokens <= kStore8Few || (a.s.num_tokens <= 2 * kStore8Few && tiles * a.kv_heads < 192)) {
        MARS_LAUNCH((k_kv_store8<T, D>), dim3(unsigned(a.s.num_tokens)), dim3(256), 0, s, a);
    } else {
        MARS_LAUNCH((k_kv_store8_tile<T, D>), dim3(unsigned(tiles), unsigned(a.kv_heads)), dim3(256), 0, s, a);
    }
    return MARS_OK;
}

template <typename T, int D>
int launch_load_dim(const LoadArgs& a, hipStream_t s) {
    const unsigned tiles = unsigned((int64_t(a.s.num_tokens) + kLoadTile - 1) / kLoadTile);
    if (a.k_scales) MARS_LAUNCH((k_kv_load<T, D, true>), dim3(tiles, unsigned(a.s.k ? a.kv_heads : 1)), dim3(256), 0, s, a);
    else MARS_LAUNCH((k_kv_load<T, D, false>), dim3(tiles, unsigned(a.s.k ? a.kv_heads : 1)), dim3(256), 0, s, a);
    return MARS_OK;
}

}  // namespace

int launch_store8(const mars_reader& r, const StoreArgs& a, hipStream_t s) {
    const bool f16 = r.d.dtype == MARS_DTYPE_F16;
    switch (r.d.head_dim) {
        case 64: return f16 ? launch_store_dim<_Float16, 64>(a, s) : launch_store_dim<__bf16, 64>(a, s);
        case 128: return f16 ? launch_store_dim<_Float16, 128>(a, s) : launch_store_dim<__bf16, 128>(a, s);
        default: return f16 ? launch_store_dim<_Float16, 256>(a, s) : launch_store_dim<__bf16, 256>(a, s);
    }
}

int launch_load(const mars_reader& r, const LoadArgs& a, hipStream_t s) {
    const bool f16 = r.d.dtype == MARS_DTYPE_F16;
    switch (r.d.head_dim) {
        case 64: return f16 ? launch_load_dim<_Float16, 64>(a, s) : launch_load_dim<__bf16, 64>(a, s);
        case 128: return f16 ? launch_load_dim<_Float16, 128>(a, s) : launch_load_dim<__bf16, 128>(a, s);
        default: return f16 ? launch_load_dim<_Float16, 256>(a, s) : launch_load_dim<__bf16, 256>(a, s);
    }
}

}  // namespace mars
