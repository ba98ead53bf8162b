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
    // Split attention: partial outputs, their (max, sum) and one arrival counter per joined tile.
    // The counters are 0 between calls (the last arriver resets its own).
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    uint32_t* arrived = nullptr;
};

namespace mars {

constexpr int32_t kMaxRequests = MARS_KV_MAX_REQUESTS;

// Keys' work items of a launch: about this many chunks over the cache's length. Partial slots:
// twice as many (a request longer than a chunk of C keys has at most 2 L / C chunks).
constexpr int32_t kFewItemsLog2 = 10;
constexpr int32_t kFewRows = 16;
constexpr int32_t kFewMost = 16;             // rows of a request that k_attend_few serves best
constexpr int32_t kManyItemsLog2 = 9;
constexpr int32_t kManyRows = 128;
constexpr int32_t kMaxSplits = 256;

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
    uint32_t* arrived;
    int64_t q_stride, out_stride, k_stride, v_stride;
    uint32_t q_flip;       // sign bits of a pair of q's elements if the scale is negative
    float scale_log2;      // |scale| * log2(e); with a cap: 2 * log2(e) * scale / cap
    float cap_log2;        // cap * log2(e); 0: no cap
    int32_t requests, max_pages, tokens, num_pages;
    int32_t q_heads, kv_heads, group;
    int32_t page_shift;
    int32_t rows_lo, rows_hi;   // this launch serves requests with rows_lo < rows <= rows_hi (rows = tokens * group)
};

int launch_attend(const mars_reader& r, const AttendArgs& a, int32_t max_new, hipStream_t s);

}  // namespace mars
