// What the attention kernels over the paged 8-bit cache share.
#pragma once
#include "kv8.h"

namespace spm {

constexpr int kDecWarps = 4;   // of a CTA
constexpr int kDecStages = 2;
constexpr int kDecPerSm = 3;   // CTAs per SM that the grid is made for
// Tokens of a warp's step.
constexpr int kv8_sub(int head_dim) { return head_dim <= 128 ? 32 : 16; }

struct Kv8Args {
    const int8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    int32_t pages, page, shift, kv_heads, group;
    const void* q;
    int64_t q_token, q_head;
    uint32_t dtype;
    int32_t rows;                              // of q and out
    const int32_t *starts, *lens;
    int32_t requests, most;
    const int32_t* table;
    int32_t width, tile_rows, tiles;           // a tile: tile_rows (query, head of the group) rows
    int32_t unit;                              // tokens
    float scale_log2;
    void* out;
    int64_t o_token, o_head;
    long long* prefix;                         // [requests * tiles + 1] units before a pair
    float* parts;                              // [CTA][2][tile_rows][head_dim + 4]
    int32_t* status;
};

namespace dev {

// A request's cached tokens, within its table row.
__device__ __forceinline__ int kv8_len(const Kv8Args& a, int req) {
    const int len = a.lens[req], cap = a.width << a.shift;
    if (len < 0 || len > cap) flag(a.status, SPM_PAGE_LENGTH);
    return min(max(len, 0), cap);
}

// Keys that the last query of a tile sees (the tile's others see fewer).
__device__ __forceinline__ int kv8_keys(const Kv8Args& a, int nq, int len, int tile) {
    const int last = min(nq, ((tile + 1) * a.tile_rows + a.group - 1) / a.group);
    return max(0, len - nq + last);
}

// Units of keys of pair v = (request, row tile), one at least where the tile
// has rows; 0 for requests whose rows are not what the call says.
__device__ __forceinline__ int kv8_units(const Kv8Args& a, int v) {
    const int req = v / a.tiles, tile = v % a.tiles;
    const int s = a.starts[req], e = a.starts[req + 1];
    if (s < 0 || e < s || e > a.rows || e - s > a.most) {
        flag(a.status, SPM_PAGE_QUERIES);
        return 0;
    }
    if ((long long)tile * a.tile_rows >= (long long)(e - s) * a.group) return 0;
    return max(1, (kv8_keys(a, e - s, kv8_len(a, req), tile) + a.unit - 1) / a.unit);
}

__device__ __forceinline__ float kv8_load(const Kv8Args& a, int64_t i) {
    if (a.dtype == SPM_F32) return static_cast<const float*>(a.q)[i];
    if (a.dtype == SPM_F16) return __half2float(static_cast<const __half*>(a.q)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[i]);
}
__device__ __forceinline__ void kv8_store(const Kv8Args& a, int64_t i, float y) {
    if (a.dtype == SPM_F32) static_cast<float*>(a.out)[i] = y;
    else if (a.dtype == SPM_F16) static_cast<__half*>(a.out)[i] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(y);
}

// acc 2^ref / (sum 2^m); 0 for a row that saw nothing.
__device__ __forceinline__ float kv8_finish(float acc, float ref, float sum, float m) {
    if (sum == 0.f) return 0.f;
    const float y = __fdiv_rn(acc, sum);
    if (ref == -INFINITY) return y;  // every value seen is zero (or NaN)
    // 2^(ref - m) in two steps: it may be past one power's range
    const int e = int(fminf(fmaxf(ref - m, -300.f), 300.f));
    return y * pow2i(e / 2) * pow2i(e - e / 2);
}

}  // namespace dev
}  // namespace spm
