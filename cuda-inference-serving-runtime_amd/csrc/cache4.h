// The cache that holds keys and values in 4 bits: how a page lies in memory.
//
// A head's page of P tokens (a power of two from 8 on) is one run of bytes.  A token's key (value) is cut into blocks of 32
// coordinates, the last filled up with zeros; a block is a power of two 2^s and 32 codes: a sign above the number of
// one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Every such number is a bf16 as it is, and the matrix cores' conversions read the codes.
//   keys     [P][DP / 2]                 two coordinates a byte, the first in the low half
//   values   [P / 8][DP / CUT][16][8][CUT / 32]: by eights of tokens, slices of CUT coordinates, sixteenths of a slice, the tokens of an eight
//   scales of the keys [DP / 32][P], of the values the same: s + 127
// What a lane feeds to one matrix instruction (a token's coordinates of the keys, eight tokens of a few coordinates of the
// values) is a run of bytes in both.  4.25 bits a coordinate.
#pragma once
#include "common.h"

#define CACHE4_BIAS 127
#define CACHE4_SITES 64                 // sites whose weights one launch takes
#define CACHE4_NOTHING -1e30f           // a maximum over no keys: finite, so that differences are numbers

__host__ __device__ constexpr int cache4_cut(int dp) { return dp % 128 == 0 ? 128 : dp % 64 == 0 ? 64 : 32; }
__host__ __device__ constexpr int cache4_record(int dp, int page) { return page * (dp + dp / 16); }

// Offsets within a head's page; P = 1 << shift, t a token of the page, d a coordinate (even).
__device__ __forceinline__ int cache4_key_at(int dp, int t, int d) { return t * (dp / 2) + d / 2; }
__device__ __forceinline__ int cache4_value_at(int dp, int shift, int t, int d) {
    const int cut = cache4_cut(dp), w = cut / 16, in = d % cut;
    return ((dp / 2) << shift) + ((((t >> 3) * (dp / cut) + d / cut) * 16 + in / w) * 8 + (t & 7)) * (w / 2) + in % w / 2;
}
__device__ __forceinline__ int cache4_scale_at(int dp, int shift, int t, int block, bool value) {
    return (dp << shift) + (((value ? dp / 32 : 0) + block) << shift) + t;
}

// Calls of the entry points that there is one of for each head size.
struct Attn4Call {
    hipStream_t stream; const void* q; const uint8_t* pages; const int* tables; const int* tasks; void* out; float* stats; float* part_o; float* part_ml;
    long long n_pages;
    int n_tasks, rows_per_task, heads, kv_heads, dim, page, width, window, form, dtype;
    float scale;
};
struct Weights4Call {
    hipStream_t stream; const void* q; const float* stats; const uint8_t* pages; const int* tables; const int* segments; float* weights; float* parts;
    long long n_pages;
    int n_segments, many, span, heads, kv_heads, dim, page, width, window, capacity, n_slots, shares, blocks, dtype;
    float scale;
};
