// ============================================================================
//  reader.hpp — shared internals of the reading path (reader.hip: handle, plan,
//  store, release; store8.hip: store into 8 bits, load; attend.hpp: attention).
// ============================================================================
#pragma once

#include "internal.hpp"

namespace mars {
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
}

struct mars_reader {
    mars_reader_desc d{};
    int32_t device = 0;
    int32_t page_shift = 0;
    // Rotary frequencies in 2^-64 turns per position (theta^(-2i/dim) / 2 pi) and the axis of each: rope_dim / 2 entries.
    uint64_t* freq = nullptr;
    int32_t* axis = nullptr;
    // Split attention: partial outputs and their (max, sum), those of k_attend_few (few_slots x 16 rows) before those of
    // k_attend_many, and an arrival counter per tile of k_attend_few, 0 between calls (the last arriver resets its own).
    size_t few_slots = 0;
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    uint32_t* arrived = nullptr;
    // Attention with shared prefixes: behind those the sums of the first phase (kStateRows rows and query heads), where their
    // pieces lie, and every request's skip.
    mars::i32x4* state_at = nullptr;
    int32_t* skips = nullptr;
};

namespace mars {

constexpr int32_t kMaxRequests = MARS_KV_MAX_REQUESTS;

// Workgroups of a k_attend_few launch: as many as 256 CUs hold at a time by their registers (twice as many: 64 ragged
// requests 243 us for 228, one token over 131,072 keys 139 for 121). Two partial slots each.
constexpr int32_t few_groups(int32_t head_dim) { return head_dim == 64 ? 768 : head_dim == 128 ? 512 : 256; }
// k_attend_many cuts the keys of all its tiles into at most about 2^9 chunks; partial slots for twice as many.
constexpr int32_t kFewRows = 16;
constexpr int32_t kFewMost = 16;             // rows of a request that k_attend_few serves best
constexpr int32_t kManyItemsLog2 = 9;
constexpr int32_t kManyRows = 128;
constexpr int32_t kJoinRows = 16;            // of a tile's rows, joined by a workgroup
// Keys of a work item, unless the request has fewer; items are multiples of 256. At least 512: two requests of 56 tokens over
// 1,067 keys (32/8 heads of 64) 27.5 us (22.2), one of 112 tokens over 577 keys among 12 single ones (2/2 of 64) 28.6 us (25.0).
// At least 128, in multiples of 128: two chunks of 511 tokens among 22 single ones (32/8 of 128) 147 us (122).
constexpr int32_t kMinChunk = 256;
constexpr int32_t kMaxSplits = 256;          // pieces of a tile, as many as a join keeps references of in LDS

// Rows times query heads whose sums the first phase of attention with shared prefixes can keep; calls with more read each
// request's own prefix.
constexpr int64_t kStateRows = 1 << 15;
// Nor does a shared prefix pay where all that the tables' rows can name is not more than this: two phases cost some 13 us more than
// one, and pages that several requests read come from the caches at about 9 TB/s. us with groups and without, 32/8 heads of 128 in
// 16 bits (8 bits), one token each: 4 requests over 4,160 shared tokens, 70 MB, 33 and 24 (30 and 26); 16 over 1,000, 74 MB, 28 and 25;
// 8 over 4,160, 140 MB, 35 and 28; 64 over 1,000, 297 MB, 32 and 48 (149 MB: 32 and 29); 16 over 4,160, 280 MB, 31 and 50 (141 MB: 29 and
// 38); 4 over 20,000, 330 MB, 43 and 55 (166 MB: 38 and 40); 64 over 32,768 107 and 937 (91 and 496).
// The host knows the tables' width alone, not what is shared, so the bound errs both ways near it, and a short prefix under wide rows
// pays the two phases: 16 requests that share 64 of some 560 tokens, rows of 2,000 pages, 28 and 23 (22 and 14).
constexpr int64_t kSharedBytes = 128 << 20;

struct AttendArgs {
    const void* q;
    void* out;
    float* lse;
    const void* k_pages;
    const void* v_pages;
    const float* k_times;
    const int32_t* k_eps;
    const int32_t* q_start;
    const int32_t* kv_lens;
    const int32_t* table;
    const float* decay;
    const float* q_times;
    const int32_t* q_eps;
    const int32_t* prefix;
    float* part_o;
    float2* part_ml;
    float* many_o;
    float2* many_ml;
    uint32_t* arrived;
    int64_t q_stride, out_stride, k_stride, v_stride;
    uint32_t q_flip;       // sign bits of a pair of q's elements if the scale is negative
    float scale_log2;      // |scale| * log2(e)
    float cap_log2;        // cap * log2(e); 0: no cap
    int32_t requests, max_pages, tokens, num_pages;
    int32_t q_heads, kv_heads, group;
    int32_t page_shift;
    int32_t few_rows;           // requests of up to so many rows are k_attend_few's
    float cap_rcp;         // 1 / (cap * log2(e)); 0: no cap
    const uint8_t* k_scales;    // a cache of 8 bits: the exponents of its slots
    const uint8_t* v_scales;
    // Shared prefixes (NULL: none): group g is requests group_start[g] .. group_start[g + 1] - 1 of `members`. phase 0: no
    // prefixes; 1: `requests` are the groups; 2: the requests, each behind the skips[r] keys that phase 1 read for it.
    const int32_t* group_start;
    const int32_t* shared_lens;
    int32_t* skips;
    float* state_o;             // sums of phase 1, a row and query head each, and their (reference, sum of weights): behind many_o, many_ml
    float2* state_ml;
    i32x4* state_at;            // with defer, where phase 2 finds a row's pieces: row of part_o of the first, the second, rows between the next, how many
    int64_t many_row0, state_row0;   // rows of part_o before many_o and state_o
    int32_t groups, members, phase, defer;
    int32_t join_rows;          // of a tile, by a workgroup of k_attend_join
    int32_t whole;              // there are no more tiles than workgroups of k_attend_few
};

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
    uint8_t* k_scales;                                   // a cache of 8 bits: the exponents of its slots
    uint8_t* v_scales;
};

// sin and cos of 2 pi * pos * f, f in units of 2^-64 turns per position: whole turns drop out of the 64-bit product
// by themselves, so the phase is exact to pos * 2^-65 turns for every int32 position, and the angle to the rounding of
// its upper 32 bits to fp32. (A product in fp32 is off by 2^-24 of the whole angle: 0.004 rad at position 70,000.)
__device__ inline void turn(int32_t pos, uint64_t f, float* sn, float* cs) {
    const uint64_t phase = uint64_t(int64_t(pos)) * f;
    sincospif(float(int32_t(uint32_t(phase >> 32))) * 0x1p-31f, sn, cs);
}

int launch_store8(const mars_reader& r, const StoreArgs& a, hipStream_t s);

struct LoadArgs {
    mars_kv_load_args s;
    const void* k_pages;
    const void* v_pages;
    const float* times;
    const int32_t* eps;
    const uint8_t* k_scales;    // NULL: a cache of 16 bits
    const uint8_t* v_scales;
    int64_t k_stride, v_stride, slots;                   // page strides (elements); slots the cache has
    int32_t kv_heads, page_shift;
};
int launch_load(const mars_reader& r, const LoadArgs& a, hipStream_t s);

int launch_attend(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s);
int launch_attend8(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s);
int launch_attend_shared(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s);

}  // namespace mars
