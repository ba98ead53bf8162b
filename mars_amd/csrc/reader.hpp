// ============================================================================
//  reader.hpp — shared internals of the reading path (reader.hip: handle, plan,
//  store, release; attend.hip: attention).
// ============================================================================
#pragma once

#include "internal.hpp"

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
};

int launch_attend(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s);

}  // namespace mars
