// Attention of a prompt's many queries over the paged 8-bit KV cache, on the
// 5th-generation tensor cores (the other half of spm_kv8_attention; the formulas
// and the scaling by powers of two are kv8_attention.cu's).
//
// A CTA owns 128 rows (query x head of the group) of a request and kv head and
// walks the keys in tiles of TN, once:
//   producers (8 warps)  codes from global memory to fp16 (exact) in shared
//                        memory: a token's row of 64 dimensions is 128 bytes in the
//                        128-byte swizzled layout, which is K-major for the keys
//                        (S = Q K^T) and MN-major for the values (O = P V), so both
//                        are written alike and nothing is transposed
//   MMA (1 thread)       S(j + 1) = Q K(j + 1)^T into the other half of two TMEM
//                        buffers while the softmax of S(j) runs, then O += P(j) V(j)
//                        with P from TMEM
//   softmax (4 warps)    a thread owns a row: S from TMEM, scale, mask, the running
//                        references, weights in fp16 back to TMEM
// The references move only where a row's maximum passes them by more than 2^8, so
// that the accumulator is hardly ever read back to be rescaled: weights are then at
// most 2^8, which fp16 holds as exactly as those below 1.
// f32 queries and weights are two fp16 parts (22 bits), twice the products.
//
// What bounds it is the softmax's instructions (16384 exponentials of a 128 x 128
// tile take 1024 cycles of the special function unit alone, its products 1024).
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.h"
#include "kv8_attention.h"
#include "tcgen05.cuh"

namespace spm {
namespace {
using namespace dev;

constexpr int kRows = kv8_prompt_rows;                 // of a tile: the MMA's M
constexpr int kSoftWarps = 4, kFillWarps = 8, kPromptThreads = 32 * (kSoftWarps + kFillWarps + 1);
constexpr int kFillThreads = 32 * kFillWarps;
constexpr float kSlack = 8.f;                          // in powers of two

template <int HD, int NP>
struct PromptShape {
    static constexpr int TN = HD <= 128 ? 128 : 64;    // keys of a tile
    static constexpr int atoms = (HD + 63) / 64;       // 64 dimensions, 128 bytes
    static constexpr int qpart = atoms * kRows * 128;  // bytes of a part of Q
    static constexpr int tile = atoms * TN * 128;      // bytes of a tile of K or V
    static constexpr int stages = NP * qpart + 4 * tile + 4096 <= 227 * 1024 ? 2 : 1;
    // (at least half of an SM's: a second CTA would wait for the first one's TMEM)
    static constexpr int need = NP * qpart + 2 * stages * tile + 1024, smem = need > 120 * 1024 ? need : 120 * 1024;
    static constexpr int s_col = 0, o_col = 2 * TN, p_col = o_col + HD;  // TMEM columns
    static_assert(p_col + NP * TN / 2 <= 512, "TMEM");
};

struct PromptSync {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready, o_done, drained;
    uint32_t tmem;
    volatile int gave_up;
    float qscale[kRows];
    // scales of K and exponents of V's for a tile's blocks of 16 keys; tile j's are
    // overwritten with j + 4, for which P(j) V(j) has to be done
    float ks[4][8], ve[4][8];
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)));
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)));
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The descriptor of an MN-major tile in the 128-byte swizzled layout: 8 rows (k) of
// 64 values (n) to an atom; `next` bytes from 64 values to the next 64, 1024 from 8
// rows to the next 8.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t at, uint32_t next) {
    return uint64_t((at & 0x3FFFFu) >> 4) | (uint64_t(next >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

template <int HD, int NP>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_prompt_kernel(const Kv8Args a) {
    using S = PromptShape<HD, NP>;
    constexpr int TN = S::TN, ST = S::stages;
    extern __shared__ __align__(1024) uint8_t raw[];
    __shared__ PromptSync y;
    const uint32_t qs = (saddr(raw) + 1023u) & ~1023u, ks = qs + NP * S::qpart, vs = ks + ST * S::tile;
    uint8_t* const base = raw + (qs - saddr(raw));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // the last rows see the most keys: they go first
    const int tile = int(gridDim.x) - 1 - int(blockIdx.x), head = blockIdx.y, req = blockIdx.z;
    const int s0 = a.starts[req], e0 = a.starts[req + 1];
    if (s0 < 0 || e0 < s0 || e0 > a.rows || e0 - s0 > a.most) {
        if (tid == 0) flag(a.status, SPM_PAGE_QUERIES);
        return;
    }
    const int nq = e0 - s0, len = kv8_len(a, req), row0 = tile * kRows, rows = min(kRows, nq * a.group - row0);
    if (rows <= 0) return;
    const int keys = kv8_keys(a, nq, len, tile), tiles = (keys + TN - 1) / TN;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&y.k_full[i], kFillThreads);
            mbar_init(&y.k_empty[i], 1);
            mbar_init(&y.v_full[i], kFillThreads);
            mbar_init(&y.v_empty[i], 1);
            mbar_init(&y.s_full[i], 1);
        }
        mbar_init(&y.p_ready, 32 * kSoftWarps);
        mbar_init(&y.o_done, 1);
        mbar_init(&y.drained, 1);
        y.gave_up = 0;
        mbar_fence_init();
    }
    constexpr int kMmaWarp = kSoftWarps + kFillWarps;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&y.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        // ---- Q: rows scaled to 2^10 by a power of two, in fp16 parts ----
        for (int r = warp; r < kRows; r += kSoftWarps + kFillWarps) {
            float x[HD / 32];
            uint32_t big = 0;
            const int qr = row0 + r, qi = qr / a.group, qh = head * a.group + qr % a.group;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                x[i] = r < rows ? kv8_load(a, int64_t(s0 + qi) * a.q_token + qh * a.q_head + lane + 32 * i) : 0.f;
                big = max(big, __float_as_uint(x[i]) & 0x7fffffffu);
            }
            big = __reduce_max_sync(0xffffffffu, big);
            const int up = min(137 - int(big >> 23), 126);
            // (a negative scale is the queries' sign: the largest sum is then the largest score)
            const float mul = a.scale_log2 < 0.f ? -pow2i(up) : pow2i(up);
            if (lane == 0) y.qscale[r] = big < 0x7f800000u ? fabsf(a.scale_log2) * pow2i(-up) : __int_as_float(0x7fffffff);
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                const int d = lane + 32 * i;
                const float v = big < 0x7f800000u ? __fmul_rn(x[i], mul) : 0.f;
                const __half hi = __float2half_rn(v);
                const uint32_t at = uint32_t(d >> 6) * (kRows * 128) + sw128_offset(r, (d & 63) >> 3) + 2 * (d & 7);
                *reinterpret_cast<__half*>(base + at) = hi;
                if (NP == 2) *reinterpret_cast<__half*>(base + S::qpart + at) = __float2half_rn(__fsub_rn(v, __half2float(hi)));
            }
        }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = y.tmem;
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // false once any wait of the CTA has given up
        if (y.gave_up) return false;
        if (mbar_wait(bar, parity)) return true;
        y.gave_up = 1;
        flag(a.status, SPM_PAGE_WAIT);
        return false;
    };

    if (warp >= kSoftWarps && warp < kMmaWarp) {
        // ---- producers: the codes of tile j, converted while those of j + 1 load ----
        constexpr int SEG = HD / 16, N = TN * SEG / kFillThreads;  // 16-byte pieces of a token, and of a thread
        static_assert(TN * SEG % kFillThreads == 0, "whole pieces");
        const int t = tid - 32 * kSoftWarps;
        const int32_t* trow = a.table + size_t(req) * a.width;
        auto page_of = [&](int tok) {
            int p = tok < keys ? __ldg(trow + (tok >> a.shift)) : -1;
            if (tok < keys && uint32_t(p) >= uint32_t(a.pages)) {
                flag(a.status, SPM_PAGE_ID);
                p = a.pages ? 0 : -1;
            }
            return p;
        };
        uint4 c[N];
        auto load = [&](const int8_t* codes, int j) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = t + i * kFillThreads, r = e / SEG, o = e % SEG, tok = j * TN + r;
                const int p = page_of(tok);
                c[i] = make_uint4(0, 0, 0, 0);
                if (p >= 0)
                    c[i] = __ldg(reinterpret_cast<const uint4*>(
                        codes + ((size_t(p) * a.kv_heads + head) * a.page + (tok & (a.page - 1))) * HD + 16 * o));
            }
        };
        auto store = [&](uint8_t* to) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = t + i * kFillThreads, r = e / SEG, o = e % SEG;
                uint32_t h[8];
                const uint32_t w[4] = {c[i].x ^ 0x80808080u, c[i].y ^ 0x80808080u, c[i].z ^ 0x80808080u, c[i].w ^ 0x80808080u};
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    h[2 * q] = kv8_codes2<0x4140>(w[q]);
                    h[2 * q + 1] = kv8_codes2<0x4342>(w[q]);
                }
                // dimensions 16 o ..: two chunks of 8 in the row's atom
                uint8_t* atom = to + (o >> 2) * (TN * 128);
                *reinterpret_cast<uint4*>(atom + sw128_offset(r, 2 * (o & 3))) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(atom + sw128_offset(r, 2 * (o & 3) + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
            }
        };
        if (tiles) load(a.k_codes, 0);
        for (int j = 0; j < tiles; j++) {
            const int st = j % ST;
            const uint32_t again = uint32_t(j / ST - 1) & 1u;
            if (j >= ST && !wait(&y.k_empty[st], again)) break;
            store(base + NP * S::qpart + st * S::tile);
            load(a.v_codes, j);
            if (t < TN / 16) {
                const int p = page_of(j * TN + 16 * t);
                y.ks[j & 3][t] = p >= 0 ? __ldg(a.k_scales + size_t(p) * a.kv_heads + head) : 0.f;
                y.ve[j & 3][t] = p >= 0 ? kv8_exponent(__ldg(a.v_scales + size_t(p) * a.kv_heads + head)) : -INFINITY;
            }
            fence_proxy_async();
            mbar_arrive(&y.k_full[st]);
            if (j >= ST && !wait(&y.v_empty[st], again)) break;
            store(base + NP * S::qpart + (ST + st) * S::tile);
            if (j + 1 < tiles) load(a.k_codes, j + 1);
            fence_proxy_async();
            mbar_arrive(&y.v_full[st]);
        }
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            constexpr uint32_t f32_out = 1u << 4, m = uint32_t(kRows >> 4) << 24;
            constexpr uint32_t id_s = f32_out | m | uint32_t(TN >> 3) << 17;
            constexpr uint32_t id_o = f32_out | m | uint32_t(HD >> 3) << 17 | 1u << 16;  // V is MN-major
            auto scores = [&](int j) {
                if (!wait(&y.k_full[j % ST], uint32_t(j / ST) & 1u)) return false;
                tc_fence_after();
                const uint32_t k = ks + uint32_t(j % ST) * S::tile, d = tmem + S::s_col + uint32_t(j & 1) * TN;
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++)
                        umma_f16(d, sw128_desc(qs + uint32_t(p) * S::qpart + (kk >> 2) * (kRows * 128) + 32u * (kk & 3)),
                                 sw128_desc(k + (kk >> 2) * (TN * 128) + 32u * (kk & 3)), id_s, p != NP - 1 || kk != 0);
                umma_commit(&y.k_empty[j % ST]);
                umma_commit(&y.s_full[j & 1]);
                return true;
            };
            bool ok = tiles == 0 || scores(0);
            for (int j = 0; ok && j < tiles; j++) {
                // (S(j + 1) takes the buffer of S(j - 1), which the softmax had read when P(j - 1) was ready)
                if (j + 1 < tiles && !scores(j + 1)) break;
                if (!wait(&y.v_full[j % ST], uint32_t(j / ST) & 1u)) break;
                if (!wait(&y.p_ready, uint32_t(j) & 1u)) break;
                tc_fence_after();
                const uint32_t v = vs + uint32_t(j % ST) * S::tile;
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                    for (int kk = 0; kk < TN / 16; kk++)
                        umma_f16_ts(tmem + S::o_col, tmem + S::p_col + uint32_t(p) * (TN / 2) + 8u * kk,
                                    sw128_mn_desc(v + 2048u * kk, TN * 128), id_o, j != 0 || p != NP - 1 || kk != 0);
                umma_commit(&y.v_empty[j % ST]);
                umma_commit(&y.o_done);
            }
            umma_commit(&y.drained);  // TMEM is given back when every product has ended
            mbar_wait(&y.drained, 0);
        }
        __syncwarp();
    } else {
        // ---- softmax: thread = row = TMEM lane ----
        const int r = tid;
        const uint32_t lanes = uint32_t(32 * warp) << 16;
        const float qscale = y.qscale[r];
        const int limit = r < rows ? len - nq + (row0 + r) / a.group + 1 : 0;  // keys that the row sees
        float m = -INFINITY, ref = -INFINITY, sum = 0.f;
        bool ok = true;
        for (int j = 0; j < tiles; j++) {
            ok = wait(&y.s_full[j & 1], uint32_t(j >> 1) & 1u);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t s = tmem + lanes + S::s_col + uint32_t(j & 1) * TN;
            const int t0 = j * TN;
            const bool hidden = __any_sync(0xffffffffu, t0 + TN > limit);
            // the row's maximum, and the largest exponent that a weighted value can have
            float top = -INFINITY, reach = -INFINITY;
#pragma unroll
            for (int b = 0; b < TN / 16; b++) {
                float v[16], big = -INFINITY;
                tmem_ld16(s + 16 * b, v);
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (!hidden || t0 + 16 * b + e < limit) big = fmaxf(big, v[e]);
                const float f = qscale * y.ks[j & 3][b];  // not negative, or NaN
                big = big == -INFINITY ? big : f != f ? 0.f : ceilf(big * f);
                top = fmaxf(top, big);
                reach = fmaxf(reach, big + y.ve[j & 3][b]);
            }
            const float m_new = top > m + kSlack || m == -INFINITY ? top : m;
            const float r_new = reach > ref + kSlack || ref == -INFINITY ? reach : ref;
            sum *= kv8_step(m, m_new);
            const float down = kv8_step(ref, r_new);
            m = m_new;
            // P and O are the last product's until it is done
            if (j) {
                ok = wait(&y.o_done, uint32_t(j - 1) & 1u);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (__any_sync(0xffffffffu, r_new != ref)) {
#pragma unroll 1
                    for (int d = 0; d < HD; d += 16) {
                        float v[16];
                        tmem_ld16(tmem + lanes + S::o_col + d, v);
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] *= r_new != ref ? down : 1.f;
                        tmem_st16(tmem + lanes + S::o_col + d, v);
                    }
                }
            }
            ref = r_new;
            const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int b = 0; b < TN / 16; b++) {
                float v[16];
                tmem_ld16(s + 16 * b, v);
                const float f = qscale * y.ks[j & 3][b], ve = y.ve[j & 3][b];
                const float w = ve != ve ? ve : ve == -INFINITY || ref == -INFINITY ? 0.f
                                : pow2i(int(fminf(fmaxf(m0 + ve - ref, -126.f), 126.f)));
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    float p[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const bool seen = !hidden || t0 + 16 * b + e + h < limit;
                        const float x = kv8_exp2(fmaf(v[e + h], f, -m0));
                        sum += seen ? x : 0.f;
                        p[h] = seen ? x * w : 0.f;
                    }
                    hi[e / 2] = kv8_half2(p[0], p[1]);
                    if (NP == 2) {
                        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&hi[e / 2]));
                        lo[e / 2] = kv8_half2(p[0] - q.x, p[1] - q.y);
                    }
                }
                tmem_st8(tmem + lanes + S::p_col + 8 * b, hi);
                if (NP == 2) tmem_st8(tmem + lanes + S::p_col + TN / 2 + 8 * b, lo);
            }
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&y.p_ready);
        }
        if (ok && tiles) ok = wait(&y.o_done, uint32_t(tiles - 1) & 1u);
        tc_fence_after();
        if (__all_sync(0xffffffffu, ok)) {
            const int qr = row0 + r, qi = qr / a.group, qh = head * a.group + qr % a.group;
            const int64_t at = int64_t(s0 + qi) * a.o_token + qh * a.o_head;
#pragma unroll 1
            for (int d = 0; d < HD; d += 16) {
                float v[16];
                if (tiles) {
                    tmem_ld16(tmem + lanes + S::o_col + d, v);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] = 0.f;
                }
                if (r < rows) {
#pragma unroll
                    for (int e = 0; e < 16; e++) v[e] = kv8_finish(v[e], ref, sum, m);
                    kv8_store16(a, at + d, v);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

template <int HD, int NP>
void launch(const Kv8Args& a, cudaStream_t st) {
    constexpr int smem = PromptShape<HD, NP>::smem;
    static_assert(smem + int(sizeof(PromptSync)) <= 227 * 1024, "a CTA's shared memory");
    static unsigned long long done = 0;
    allow_smem(kv8_prompt_kernel<HD, NP>, smem, done);
    const dim3 grid(unsigned(a.tiles), unsigned(a.kv_heads), unsigned(a.requests));
    kv8_prompt_kernel<HD, NP><<<grid, kPromptThreads, smem, st>>>(a);
    CUDA_OK(cudaGetLastError());
}

template <int HD>
void launch_parts(const Kv8Args& a, cudaStream_t st) {
    a.dtype == SPM_F32 ? launch<HD, 2>(a, st) : launch<HD, 1>(a, st);
}

}  // namespace

void launch_kv8_prompt(const Kv8Args& a, int head_dim, cudaStream_t st) {
    switch (head_dim) {
        case 64: launch_parts<64>(a, st); break;
        case 96: launch_parts<96>(a, st); break;
        case 128: launch_parts<128>(a, st); break;
        case 192: launch_parts<192>(a, st); break;
        default: launch_parts<256>(a, st); break;
    }
}

}  // namespace spm
