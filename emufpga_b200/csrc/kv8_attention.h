// What the attention kernels over the paged 8-bit cache share.
#pragma once
#include "kv8.h"

namespace spm {

constexpr int kDecWarps = 4;   // of a CTA
constexpr int kDecStages = 2;
// CTAs per SM that the grid is made for: what registers and shared memory hold of row
// tiles of 8 (nt 1) or 16 (nt 2).  Three where two fit leave a second wave (16 requests
// of 3 tokens, 32/8 heads of 128, 3000 to 8000 keys: 99 us instead of 75).
constexpr int kv8_dec_ctas(int head_dim, int nt) { return nt == 2 && head_dim > 64 ? 2 : 3; }
// Tokens of a warp's step.
constexpr int kv8_sub(int head_dim) { return head_dim <= 128 ? 32 : 16; }

// Powers of two by which a weight may lie above 1: a row's accumulator has its reference
// that far under the largest weighted value's.  fp16 holds 2^15 but nothing under 2^-25,
// and the many small weights beside a large one (a first token that takes nearly all
// and has no value to speak of) are the result.
constexpr float kLift = 15.f;

// Rows of a tile of the kernel of many queries; `total`: its form that sums in f32.
constexpr int kv8_prompt_rows(int head_dim, bool total) { return head_dim <= 128 && !total ? 256 : 128; }

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
    bool clear;                                // rows of out that no request has become zero
    bool o_vec;                                // out and its strides are multiples of 16 bytes
    int32_t* prefix;                           // [requests * tiles + 1] units before a pair
    float* parts;                              // [CTA][2][tile_rows][head_dim + 4]
    int32_t* status;
};

// The kernel of many queries (kv8_prompt.cu): a.tile_rows = kv8_prompt_rows(head_dim, total), a.tiles to match.
void launch_kv8_prompt(const Kv8Args& a, int head_dim, bool total, cudaStream_t st);

namespace dev {

// A request's cached tokens, within its table row.
__device__ __forceinline__ int kv8_len(const Kv8Args& a, int len) {
    const int cap = a.width << a.shift;
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
    const int s = a.starts[req], e = a.starts[req + 1], len = a.lens[req];  // (loaded together)
    if (s < 0 || e < s || e > a.rows || e - s > a.most) {
        flag(a.status, SPM_PAGE_QUERIES);
        return 0;
    }
    if ((long long)tile * a.tile_rows >= (long long)(e - s) * a.group) return 0;
    return max(1, (kv8_keys(a, e - s, kv8_len(a, len), tile) + a.unit - 1) / a.unit);
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

// Rows of out that no request has, shared out among the grid's `ctas` CTAs.
template <int HD>
__device__ __forceinline__ void kv8_clear(const Kv8Args& a, long long cta, long long ctas) {
    if (!a.clear) return;
    const int before = min(max(a.starts[0], 0), a.rows), from = min(max(a.starts[a.requests], before), a.rows);
    const int heads = a.kv_heads * a.group, rest = before + a.rows - from;
    for (long long e = cta * blockDim.x + threadIdx.x; e < (long long)rest * heads * HD; e += ctas * blockDim.x) {
        const int row = int(e / (heads * HD)), d = int(e % (heads * HD));
        kv8_store(a, int64_t(row < before ? row : from + row - before) * a.o_token + d / HD * a.o_head + d % HD, 0.f);
    }
}

// Four values of a row, in one piece where out's strides allow it.
__device__ __forceinline__ void kv8_store4(const Kv8Args& a, int64_t i, float4 v) {
    if (!a.o_vec) {
        kv8_store(a, i, v.x);
        kv8_store(a, i + 1, v.y);
        kv8_store(a, i + 2, v.z);
        kv8_store(a, i + 3, v.w);
    } else if (a.dtype == SPM_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + i) = v;
    } else if (a.dtype == SPM_F16) {
        __half2* o = reinterpret_cast<__half2*>(static_cast<__half*>(a.out) + i);
        o[0] = __floats2half2_rn(v.x, v.y);
        o[1] = __floats2half2_rn(v.z, v.w);
    } else {
        __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.out) + i);
        o[0] = __floats2bfloat162_rn(v.x, v.y);
        o[1] = __floats2bfloat162_rn(v.z, v.w);
    }
}

// Sixteen values of a row, in 16-byte pieces where out's strides allow them.
__device__ __forceinline__ void kv8_store16(const Kv8Args& a, int64_t i, const float (&v)[16]) {
    if (a.dtype == SPM_F32) {
        float* o = static_cast<float*>(a.out) + i;
        if (a.o_vec) {
#pragma unroll
            for (int j = 0; j < 4; j++) reinterpret_cast<float4*>(o)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            return;
        }
    } else if (a.o_vec) {
        __align__(16) uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (a.dtype == SPM_F16) {
                const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + i);
        o[0] = make_uint4(w[0], w[1], w[2], w[3]);
        o[1] = make_uint4(w[4], w[5], w[6], w[7]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; j++) kv8_store(a, i + j, v[j]);
}

// Bytes of x (codes + 128) picked by SEL, as two fp16 codes.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t kv8_codes2(uint32_t x) {
    const uint32_t u = __byte_perm(x, 0x64646464u, SEL);
    const __half bias = __ushort_as_half(0x6480);  // 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __halves2half2(bias, bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Two fp16 codes times 2^-11.
__device__ __forceinline__ uint32_t kv8_under(uint32_t x) {
    const __half m = __ushort_as_half(0x1000);  // 2^-11
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&x), __halves2half2(m, m));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t kv8_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float kv8_exp2(float x) {  // to 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(from - to) for integer-valued references, from <= to; 0 where there was none yet.
__device__ __forceinline__ float kv8_step(float from, float to) {
    return from == -INFINITY ? 0.f : pow2i(int(fmaxf(from - to, -126.f)));
}
// The exponent of a scale (a power of two); -inf for 0, NaN for NaN.
__device__ __forceinline__ float kv8_exponent(float s) {
    return s > 0.f ? float((__float_as_int(s) >> 23) - 127) : s == 0.f ? -INFINITY : __int_as_float(0x7fffffff);
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
