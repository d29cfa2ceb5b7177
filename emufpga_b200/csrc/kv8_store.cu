// Storing into the paged 8-bit KV cache (spm_kv8_append) and reading whole
// pages back (spm_kv8_values).
//
// A (page, kv head) has one scale 2^e, the smallest with |x| <= 127 * 2^e over
// the values written.  A power of two rather than amax / 127: x / scale, code *
// scale and the rescaling of rows that are already there when e grows are then
// exact up to the one rounding to an integer, so a page that is filled a token
// at a time, its scale growing on the way, is never more than one step
// (half + quarter + ...) away from its values, and a code is the same whatever
// order sums run in.  It costs less than one of the eight bits.
//
// Bound: bytes (rows in, one byte a value out) for prompts, and each CTA's chain of
// slots, rows, scales and codes; launch latency for a decode tick.  Keys and values
// of 8 x 128 in f32: 8 tokens 3 us, 1024 tokens 7 us (1.5 TB/s), 19 400 bf16 tokens of
// 4 x 128 in 37 prompts 24 us (60 MB, 2.5 TB/s; one launch after another).  Reading
// their pages back as f32 takes 16 us (100 MB, 6.2 TB/s).
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.h"

namespace spm {
namespace {
using namespace dev;

constexpr int kStoreThreads = 256, kStoreWarps = kStoreThreads / 32;
constexpr int kStoreWindow = 64;  // at most: tokens whose runs begin in a CTA's window

struct StoreArgs {
    const void* x[2];         // keys, values
    int64_t token[2], head[2];
    int8_t* codes[2];
    float* scales[2];
    int32_t pages, page, shift, kv_heads, dim;
    const int32_t* slots;
    int32_t tokens, window;
    int32_t* status;
    bool vec;                 // four elements at a time: strides and bases allow it
};

// Sixteen consecutive elements of a row, in their own type.
template <class T>
struct Sixteen {
    static constexpr int W = 4 * sizeof(T);
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* p, bool vec) {
        if (vec) {  // (8 bytes for each four elements)
#pragma unroll
            for (int i = 0; i < W; i += sizeof(T)) {
                if constexpr (sizeof(T) == 4) {
                    const uint4 q = *reinterpret_cast<const uint4*>(p + i);
                    w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
                } else {
                    const uint2 q = *reinterpret_cast<const uint2*>(p + 2 * i);
                    w[i] = q.x, w[i + 1] = q.y;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; i++) {
                if constexpr (sizeof(T) == 4) {
                    w[i] = reinterpret_cast<const uint32_t*>(p)[i];
                } else {
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
                    w[i] = h[0] | uint32_t(h[1]) << 16;
                }
            }
        }
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[j]);
        } else {
            const uint16_t h = uint16_t(j & 1 ? w[j >> 1] >> 16 : w[j >> 1]);
            return to_f32(*reinterpret_cast<const T*>(&h));
        }
    }
};

__device__ __forceinline__ uint32_t code_of(float x, float inv) {
    // rounds half to even; NaN (a value or scale that is not finite) is 0
    return uint32_t(min(max(__float2int_rn(__fmul_rn(x, inv)), -127), 127)) & 0xffu;
}

// The smallest 2^e with amax <= 127 * 2^e, as amax's bits give it: amax =
// m * 2^x with m in [1, 2) lies at or under 127 * 2^(x - 6) iff m <= 127/64.
// 0 for no value but zeros, NaN where a value is not finite.
__device__ __forceinline__ float scale_of(uint32_t amax) {
    if (amax == 0) return 0.f;
    if (amax >= 0x7f800000u) return __int_as_float(0x7fffffff);
    const int x = int(amax >> 23) - 127;  // -127 for subnormals, which the clamp covers
    return pow2i(x - 6 + ((amax & 0x7fffffu) > 0x7e0000u ? 1 : 0));
}

// A CTA for each window of tokens, kv head, keys or values.  A run is the tokens of
// one page that follow one another in the call; a CTA takes the runs that begin
// in its window, whose last may reach up to a page beyond it.
template <class T>
__global__ void __launch_bounds__(kStoreThreads, 4) kv8_append_kernel(const StoreArgs a) {
    __shared__ int32_t slot[kStoreWindow + 256];
    __shared__ int16_t lead[kStoreWindow + 256];   // the first token of a token's run, within the window
    __shared__ uint32_t amax[kStoreWindow];
    __shared__ float inv[kStoreWindow], ratio[kStoreWindow];
    __shared__ int own;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // keys and values of all heads side by side: their rows lie together in memory
    const int kv = blockIdx.x & 1, h = int(blockIdx.x >> 1) % a.kv_heads, w0 = int(blockIdx.x >> 1) / a.kv_heads * a.window;
    const int P = a.page, D = a.dim;
    const int win = min(a.window, a.tokens - w0), span = min(a.tokens - w0, win + P - 1);
    // D / 16 threads to a row, sixteen values each (spare threads idle).  The first rows'
    // values are on their way before anything else is known, and stay in registers.
    const T* x = static_cast<const T*>(kv ? a.x[1] : a.x[0]) + h * (kv ? a.head[1] : a.head[0]);
    const int64_t stride = kv ? a.token[1] : a.token[0];
    const int lanes = D / 16, turns = kStoreThreads / lanes;
    const int mine = tid / lanes, col = 16 * (tid - mine * lanes);
    Sixteen<T> held[2];
#pragma unroll
    for (int u = 0; u < 2; u++)
        if (mine < turns && mine + u * turns < span) held[u].load(x + (w0 + mine + u * turns) * stride + col, a.vec);
    for (int i = tid; i < span; i += kStoreThreads) slot[i] = a.slots[w0 + i];
    if (tid < win) amax[tid] = 0;
    __syncthreads();
    if (warp == 0) {
        int carry = -1, end = span;
        for (int i0 = 0; i0 < end; i0 += 32) {
            const int i = i0 + lane;
            bool first = false;
            if (i < span) {
                const int s = slot[i], before = i ? slot[i - 1] : w0 ? a.slots[w0 - 1] : -2;
                first = s < 0 || before < 0 || s != before + 1 || (s & (P - 1)) == 0;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, first);
            const uint32_t upto = m & (0xffffffffu >> (31 - lane));
            const int l = upto ? i0 + 31 - __clz(upto) : carry;
            if (i < span) lead[i] = int16_t(l);
            // runs that begin behind the window are the next CTAs'
            const uint32_t past = m & (i0 >= win ? 0xffffffffu : i0 + 32 <= win ? 0u : 0xffffffffu << (win - i0));
            if (past) end = i0 + __ffs(past) - 1;
            if (m) carry = i0 + 31 - __clz(m);
        }
        if (lane == 0) own = end;
    }
    __syncthreads();
    const int n = own;
    const uint32_t limit = uint32_t(a.pages) * uint32_t(P);
    int8_t* codes = kv ? a.codes[1] : a.codes[0];
    float* scales = kv ? a.scales[1] : a.scales[0];
    // f(run, slot, sixteen values) for this thread's pieces of the CTA's rows
    auto rows = [&](auto&& f) {
        for (int u = 0, i = mine; i < n && mine < turns; u++, i += turns) {
            const int l = lead[i], s = slot[i];
            if (l < 0) continue;
            if (uint32_t(s) >= limit) {
                if (s != -1) flag(a.status, SPM_PAGE_ID);
                continue;
            }
            if (u == 0) {
                f(l, s, held[0]);
            } else if (u == 1) {
                f(l, s, held[1]);
            } else {  // (a run that goes on behind the window; head_dim over 128)
                Sixteen<T> more;
                more.load(x + (w0 + i) * stride + col, a.vec);
                f(l, s, more);
            }
        }
    };
    rows([&](int l, int, const Sixteen<T>& v) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) m = max(m, __float_as_uint(v.at(j)) & 0x7fffffffu);
        if (m > amax[l]) atomicMax(&amax[l], m);  // (a stale look only costs the atomic)
    });
    __syncthreads();
    if (tid < win) {
        inv[tid] = ratio[tid] = 0.f;
        const int s = slot[tid];
        if (lead[tid] == tid && uint32_t(s) < limit) {
            float* p = scales + size_t(s >> a.shift) * a.kv_heads + h;
            float sc = scale_of(amax[tid]);
            if (s & (P - 1)) {
                const float was = *p;
                if (!(was == was)) sc = was;            // NaN stays
                else if (was > sc) sc = was;
                else if (was > 0.f && sc > was) ratio[tid] = fmaxf(__fdiv_rn(was, sc), pow2i(-126));  // (0: none; any code becomes 0)
            }
            *p = sc;
            inv[tid] = sc > 0.f ? __fdiv_rn(1.f, sc) : 0.f;
        }
    }
    // rows that were there, where the scale has grown (seldom)
    if (__syncthreads_or(tid < win && ratio[tid] != 0.f)) {
        for (int l = 0; l < win; l++) {
            const float q = ratio[l];
            if (q == 0.f) continue;
            const int s = slot[l], rows = s & (P - 1);
            uint32_t* w = reinterpret_cast<uint32_t*>(codes + ((size_t(s >> a.shift) * a.kv_heads + h) * P) * D);
            for (int i = tid; i < rows * D / 4; i += kStoreThreads) {
                const uint32_t c = w[i];
                uint32_t o = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) o |= code_of(float(int8_t(c >> (8 * j))), q) << (8 * j);
                w[i] = o;
            }
        }
    }
    rows([&](int l, int s, const Sixteen<T>& v) {
        const float q = inv[l];
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            // x / scale is exact, at most 127: adding 1.5 * 2^23 rounds it, half to even, to
            // an integer in the low byte; 0 where the scale is 0 or NaN
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; e++) b[e] = __float_as_uint(__fmaf_rn(v.at(j + e), q, 12582912.f));
            const uint32_t lo = __byte_perm(b[0], b[1], 0x0040), hi = __byte_perm(b[2], b[3], 0x0040);
            w[j >> 2] = q == 0.f ? 0 : __byte_perm(lo, hi, 0x5410);
        }
        *reinterpret_cast<uint4*>(codes + ((size_t(s >> a.shift) * a.kv_heads + h) * P + (s & (P - 1))) * D + col) =
            make_uint4(w[0], w[1], w[2], w[3]);
    });
}

struct ValueArgs {
    const int8_t* codes[2];
    const float* scales[2];
    void* out[2];
    const int32_t* ids;
    int32_t n, pages, kv_heads, block;  // block: codes of a (page, head)
    int32_t* status;
};

// Sixteen bytes out for each thread and turn (4 or 8 codes in), so that a warp
// writes whole lines; four turns' loads overlap.
constexpr int kValueTurns = 4;

template <class T>
__global__ void __launch_bounds__(256) kv8_values_kernel(const ValueArgs a) {
    constexpr int V = 16 / sizeof(T);
    // (keys or values by a select: an array in the arguments indexed by the block goes to local memory)
    const int per = a.block / V;  // pieces of a (page, head)
    const bool keys = blockIdx.y == 0;
    const int8_t* const codes = keys ? a.codes[0] : a.codes[1];
    const float* const scales = keys ? a.scales[0] : a.scales[1];
    T* out = static_cast<T*>(keys ? a.out[0] : a.out[1]);
    if (!out) return;
    // this CTA's pieces: one long division for all of them
    const size_t base = size_t(blockIdx.x) * 256 * kValueTurns, ph0 = base / per, total = size_t(a.n) * a.kv_heads * per;
    const uint32_t off = uint32_t(base - ph0 * per) + threadIdx.x;
    uint32_t c[kValueTurns][V / 4];
    float s[kValueTurns];
#pragma unroll
    for (int u = 0; u < kValueTurns; u++) {
        const bool some = base + threadIdx.x + 256 * u < total;
        const uint32_t o = off + 256 * u, skip = o / uint32_t(per), e = (o - skip * per) * V;
        const size_t ph = ph0 + skip;
        size_t at = ph;
        bool known = some;
        if (a.ids && some) {
            const int p = int(ph / a.kv_heads), id = a.ids[p];
            known = uint32_t(id) < uint32_t(a.pages);
            if (!known && e == 0) flag(a.status, SPM_PAGE_ID);
            at = size_t(id) * a.kv_heads + (ph - size_t(p) * a.kv_heads);
        }
        s[u] = known ? __ldg(scales + at) : 0.f;
        const uint32_t* from = reinterpret_cast<const uint32_t*>(codes + at * a.block + e);
#pragma unroll
        for (int j = 0; j < V / 4; j++) c[u][j] = known ? __ldg(from + j) : 0;
    }
#pragma unroll
    for (int u = 0; u < kValueTurns; u++) {
        const size_t i = base + threadIdx.x + 256 * u;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float y = __fmul_rn(float(int8_t(c[u][j >> 2] >> (8 * (j & 3)))), s[u]);
            if constexpr (sizeof(T) == 4) {
                w[j] = __float_as_uint(y);
            } else {
                const T t = from_f32<T>(y);
                const uint32_t b = *reinterpret_cast<const uint16_t*>(&t);
                w[j >> 1] = j & 1 ? w[j >> 1] | b << 16 : b;
            }
        }
        if (i < total) __stcs(reinterpret_cast<uint4*>(out) + i, make_uint4(w[0], w[1], w[2], w[3]));
    }
}

}  // namespace
}  // namespace spm

using namespace spm;

spm_status spm_kv8_append(const spm_kv8* c, uint32_t dtype, const void* k, int64_t k_token, int64_t k_head,
                          const void* v, int64_t v_token, int64_t v_head, int32_t tokens, const int32_t* slots,
                          void* cuda_stream) {
    return guarded([&] {
        kv8_check(c);
        kv8_check_type(dtype);
        if (tokens < 0) fail(SPM_E_ARG, "negative token count");
        if (tokens > INT32_MAX - 65536) fail(SPM_E_ARG, "too many tokens for one call");  // (a window's end fits 32 bits)
        if (tokens == 0) return;
        if (!k || !v || !slots) fail(SPM_E_ARG, "null keys, values or slots");
        DeviceScope scope(c->device);
        const size_t size = dtype == SPM_F32 ? 4 : 2;
        StoreArgs a{};
        a.x[0] = k, a.x[1] = v;
        a.token[0] = k_token, a.token[1] = v_token;
        a.head[0] = k_head, a.head[1] = v_head;
        a.codes[0] = c->k_codes, a.codes[1] = c->v_codes;
        a.scales[0] = c->k_scales, a.scales[1] = c->v_scales;
        a.pages = c->pages, a.page = c->page_tokens, a.shift = __builtin_ctz(unsigned(c->page_tokens));
        a.kv_heads = c->kv_heads, a.dim = c->head_dim;
        a.slots = slots, a.tokens = tokens, a.status = c->status;
        a.vec = !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % (4 * size)) &&
                !((k_token | k_head | v_token | v_head) & 3);
        // windows of a page of prompt tokens, cut down to a warp's token each
        // while that leaves SMs without a CTA (a decode tick)
        a.window = kStoreWindow;
        while (a.window > kStoreWarps && int64_t((tokens + a.window - 1) / a.window) * c->kv_heads * 2 < 2 * device_sms())
            a.window /= 2;
        const int64_t grid = int64_t((tokens + a.window - 1) / a.window) * c->kv_heads * 2;
        if (grid > INT32_MAX) fail(SPM_E_ARG, "too many tokens for one call");
        const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        if (dtype == SPM_F32) kv8_append_kernel<float><<<unsigned(grid), kStoreThreads, 0, st>>>(a);
        else if (dtype == SPM_F16) kv8_append_kernel<__half><<<unsigned(grid), kStoreThreads, 0, st>>>(a);
        else kv8_append_kernel<__nv_bfloat16><<<unsigned(grid), kStoreThreads, 0, st>>>(a);
        CUDA_OK(cudaGetLastError());
    });
}

spm_status spm_kv8_values(const spm_kv8* c, uint32_t dtype, const int32_t* page_ids, int32_t n, void* k_out,
                          void* v_out, void* cuda_stream) {
    return guarded([&] {
        kv8_check(c);
        kv8_check_type(dtype);
        if (n < 0) fail(SPM_E_ARG, "negative page count");
        if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)
            fail(SPM_E_ARG, "outputs must be 16-byte aligned");
        if (n == 0 || (!k_out && !v_out)) return;
        DeviceScope scope(c->device);
        ValueArgs a{};
        a.codes[0] = c->k_codes, a.codes[1] = c->v_codes;
        a.scales[0] = c->k_scales, a.scales[1] = c->v_scales;
        a.out[0] = k_out, a.out[1] = v_out;
        a.ids = page_ids, a.n = n, a.pages = c->pages, a.kv_heads = c->kv_heads;
        a.block = c->page_tokens * c->head_dim;
        a.status = c->status;
        if (!page_ids && n > c->pages) fail(SPM_E_ARG, "the pool has fewer pages");
        const size_t per = size_t(256) * kValueTurns * (dtype == SPM_F32 ? 4 : 8);
        const size_t ctas = (size_t(n) * c->kv_heads * a.block + per - 1) / per;
        if (ctas > INT32_MAX) fail(SPM_E_ARG, "too many pages for one call");
        const dim3 grid(unsigned(ctas), 2);
        const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        if (dtype == SPM_F32) kv8_values_kernel<float><<<grid, 256, 0, st>>>(a);
        else if (dtype == SPM_F16) kv8_values_kernel<__half><<<grid, 256, 0, st>>>(a);
        else kv8_values_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
        CUDA_OK(cudaGetLastError());
    });
}
