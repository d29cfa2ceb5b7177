// Attention over the paged 8-bit KV cache (spm_kv8_attention), for decode ticks
// and few queries per request.
//
// Per query row and kv head:  s_j = c 2^(e_j) (q . K_j),  c = scale log2(e),
// out = sum_j 2^(s_j - m) 2^(f_j) V_j / sum_j 2^(s_j - m), with K_j, V_j the int8
// codes and 2^(e_j), 2^(f_j) the scales of key j's page.  One pass with running
// references, all integers, so that every rescaling is a power of two and exact:
// m = ceil(max s) for the sum, and r = max(ceil(max s in a page's 16 rows) + f) - 15
// for the accumulator, which then holds sum_j 2^(s_j + f_j - r) V_j with every
// weight at most 2^15: it fits fp16 whatever the pages' scales are.
//
// Products on the tensor cores (mma.sync).  The 16 rows of an mma are cached tokens
// (or, for the values, head dimensions) and its 8 columns are query rows (tokens x
// heads of the group), so that one pass over the codes serves every query of a kv
// head.
//   Scores: int8 x int8 (m16n8k32).  The codes go in as they lie; a query row is
//   fixed point to its largest value, 23 bits in three signed 8-bit digits (two, 15
//   bits, would gain 2% of a long decode).  Sums are exact in int32.
//   Values: fp16 x fp16 (m16n8k16), fp32 sums.  The codes are exact in fp16: byte
//   permutes make 0x6400 | (code + 128) = 1024 + 128 + code and a subtraction of 1152
//   the code.  Weights are fp16.  For bf16 results one part: 11 bits for weights down
//   to 2^-29 of the row's largest, a bit less for each power of two below.  f16 results
//   take a second part for what is left (one alone would add as much as their own
//   rounding, 1.4 times the error; it takes 5% of a long decode), f32 results hold that
//   part 2^11 up and give it the codes 2^-11 down (both exact): 22 bits down to the
//   same 2^-29, 11 at 2^-40.
//   ldmatrix transposes pairs of bytes: the even and odd dimensions of a 16-byte
//   column become rows g and g + 8.
//
// What bounds it is the cache's bytes (64 requests of 1000 to 16384 keys, 8 kv heads of
// 128: 1.16 GB in 205 us and 9 to join the parts, 5.4 TB/s together, in a short run of
// calls; 235 to 248 in a long one; f16 225 and f32 237 in a short one), nearly as much
// the issue of its products; for a few requests the latency of one unit (8 requests of
// 1200 keys: 11 us).  Each warp streams its own 32 tokens (16 where
// head_dim is over 128) at a time through a ring in shared memory (16-byte asynchronous copies, no barrier
// among warps).  Work is cut into units of four such steps of a (row tile, kv head),
// and every CTA takes an equal run of the units of all requests, so that ragged
// lengths load all SMs alike; where a run ends inside a (row tile, kv head) its
// partial goes to the workspace and kv8_combine_kernel adds the parts in order.
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.h"
#include "kv8_attention.h"

namespace spm {
namespace {
using namespace dev;

constexpr int kDecThreads = 32 * kDecWarps;

// Units of a CTA's run.
__device__ __forceinline__ int kv8_share(int total, int ctas) { return (total + ctas - 1) / ctas; }

__device__ __forceinline__ void ldsm4(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float2 half2_floats(uint32_t b) { return __half22float2(*reinterpret_cast<const __half2*>(&b)); }
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(saddr(dst)), "l"(src) : "memory");
}
// A weight's fp16 parts: one, two, or two of which the second is held 2^11 up.
enum class Weights { kOne, kTwo, kTwoApart };

template <int HD, int NT>
struct DecSmem {
    static constexpr int sub = kv8_sub(HD);
    // a token's codes: the eight rows that an ldmatrix reads lie on distinct banks,
    // by an exclusive or of the 16-byte chunk with the row where a row fills whole
    // bank sweeps, else by 16 bytes between the rows
    static constexpr bool swizzled = HD == 64 || HD % 128 == 0;
    static constexpr int row = swizzled ? HD : HD + 16;
    static __device__ __forceinline__ int at(int r, int chunk) {
        if (HD == 64) return r * row + ((chunk ^ ((r >> 1) & 3)) << 4);
        if (HD % 128 == 0) return r * row + ((chunk ^ (r & 7)) << 4);
        return r * row + (chunk << 4);
    }
    static constexpr int digits = 3;                          // of a query value
    static constexpr int stage = 2 * sub * row + 16;          // keys, values, then 2 + 2 scales
    static constexpr int q = 0;                               // [digits][NT][HD / 32][32 lanes][8]
    static constexpr int qbytes = digits * NT * HD * 8;
    static constexpr int qscale = q + qbytes;                 // [8 NT] floats
    static constexpr int ring = (qscale + 8 * NT * 4 + 15) & ~15;
    static constexpr int state = HD + 4;                      // a row's accumulator, then m, r, l
    static constexpr int ring_bytes = kDecWarps * kDecStages * stage;
    static constexpr int state_bytes = kDecWarps * 8 * NT * state * 4;
    static constexpr int total = ring + (ring_bytes > state_bytes ? ring_bytes : state_bytes);
};

template <int HD, int NT, Weights WT>
__global__ void __launch_bounds__(kDecThreads, kv8_dec_ctas(HD, NT)) kv8_decode_kernel(const Kv8Args a) {
    using L = DecSmem<HD, NT>;
    constexpr int NP = WT == Weights::kOne ? 1 : 2;
    constexpr bool apart = WT == Weights::kTwoApart;
    constexpr float up = apart ? 2048.f : 1.f;
    constexpr int NR = 8 * NT, KB = HD / 32, SUB = L::sub, NB = SUB / 16, UNIT = kDecWarps * SUB, PL = L::digits;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ int wsum[kDecWarps], found[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int V = a.requests * a.tiles;  // (request, row tile) pairs
    kv8_clear<HD>(a, blockIdx.x, gridDim.x);
    pdl_trigger();  // (kv8_combine_kernel's CTAs may come and wait: all of this grid's are resident)

    // ---- this CTA's run of units ----
    auto block_scan = [&](int x, int& before) {  // exclusive sum over threads, and the total
        int v = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += n;
        }
        __syncthreads();
        if (lane == 31) wsum[warp] = v;
        __syncthreads();
        before = v - x;
        int total = 0;
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) {
            if (w < warp) before += wsum[w];
            total += wsum[w];
        }
        return total;
    };
    // (request, row tile) pairs by the thread; one look at the lengths is enough for up
    // to as many pairs as threads
    auto units_of = [&](int v) { return v < V ? kv8_units(a, v) * a.kv_heads : 0; };
    int total = 0, mine = 0, before = 0;
    for (int v0 = 0; v0 < V; v0 += kDecThreads) {
        mine = units_of(v0 + tid);
        const int sum = block_scan(mine, before);
        if (blockIdx.x == 0 && v0 + tid < V) a.prefix[v0 + tid] = total + before;
        total += sum;
    }
    if (blockIdx.x == 0 && tid == 0) a.prefix[V] = total;
    const int share = kv8_share(total, gridDim.x);
    const int begin = min(total, share * int(blockIdx.x)), end = min(total, begin + share);
    if (begin >= end) return;
    for (int v0 = 0, run = 0; v0 < V && run <= begin; v0 += kDecThreads) {
        int sum = total;
        if (V > kDecThreads) {
            mine = units_of(v0 + tid);
            sum = block_scan(mine, before);
        }
        if (run + before <= begin && begin < run + before + mine) found[0] = v0 + tid, found[1] = run + before;
        run += sum;
    }
    __syncthreads();
    int v = found[0], base = found[1], u = begin;  // base: the first unit of pair v

    const int lrow = (lane & 7) + 8 * ((lane >> 3) & 1), lchunk = lane >> 4;  // this lane's ldmatrix row
    uint8_t* ring = sm + L::ring + warp * kDecStages * L::stage;
    float* qscale = reinterpret_cast<float*>(sm + L::qscale);
    for (int piece = 0; u < end; piece++) {
        int nu = kv8_units(a, v);
        while (u >= base + nu * a.kv_heads) {
            base += nu * a.kv_heads;
            v++;
            nu = kv8_units(a, v);
        }
        const int req = v / a.tiles, tile = v % a.tiles;
        const int head = (u - base) / nu, unit0 = (u - base) - head * nu;
        const int units = min(nu - unit0, end - u);
        const int s0 = a.starts[req], nq = a.starts[req + 1] - s0, len = kv8_len(a, a.lens[req]);
        const int row0 = tile * NR, rows = min(NR, nq * a.group - row0);
        const int keys = kv8_keys(a, nq, len, tile);
        const int k0 = unit0 * UNIT, k1 = min(keys, (unit0 + units) * UNIT);
        u += units;
        __syncthreads();  // the ring and the queries of the piece before are done with

        // ---- tokens k0 .. k1 - 1, SUB at a time in turn among the warps ----
        const int steps = max(0, (k1 - k0 - SUB * warp + UNIT - 1) / UNIT);
        const int32_t* trow = a.table + size_t(req) * a.width;
        auto page_of = [&](int j) {  // lanes 0, 1: the pages of step j's blocks of 16 tokens
            const int tok = k0 + SUB * (warp + kDecWarps * j) + 16 * (lane & (NB - 1));
            int p = 0;
            if (j < steps && tok < k1) {
                p = __ldg(trow + (tok >> a.shift));
                if (uint32_t(p) >= uint32_t(a.pages)) {
                    flag(a.status, SPM_PAGE_ID);
                    p = a.pages ? 0 : -1;
                }
            }
            return p;
        };
        auto issue = [&](int j, int mine) {
            if (j < steps) {
                uint8_t* st = ring + (j % kDecStages) * L::stage;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const int tok = k0 + SUB * (warp + kDecWarps * j) + 16 * b;
                    const int p = __shfl_sync(0xffffffffu, mine, b);
                    if (tok >= k1 || p < 0) continue;
                    const size_t at = size_t(p) * a.kv_heads + head;
                    const size_t from = (at * a.page + (tok & (a.page - 1))) * HD;
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        const int c = lane + 32 * i, r = c / (HD / 16), o = c % (HD / 16);
                        cp_async16(st + L::at(16 * b + r, o), a.k_codes + from + 16 * c);
                        cp_async16(st + SUB * L::row + L::at(16 * b + r, o), a.v_codes + from + 16 * c);
                    }
                    if (lane == 0) cp_async4(st + 2 * SUB * L::row + 4 * b, a.k_scales + at);
                    if (lane == 1) cp_async4(st + 2 * SUB * L::row + 8 + 4 * b, a.v_scales + at);
                }
            }
            cp_async_commit();
        };
        // this warp's queries, on their way with the first page numbers
        constexpr int QR = NR / kDecWarps;
        float x[QR][HD / 32];
#pragma unroll
        for (int y = 0; y < QR; y++) {
            const int r = warp + kDecWarps * y, qr = row0 + r, qi = qr / a.group, qh = head * a.group + qr % a.group;
#pragma unroll
            for (int i = 0; i < HD / 32; i++)
                x[y][i] = r < rows ? kv8_load(a, int64_t(s0 + qi) * a.q_token + qh * a.q_head + lane + 32 * i) : 0.f;
        }
        int ahead = page_of(0);
#pragma unroll
        for (int j = 0; j < kDecStages - 1; j++) {
            const int next = page_of(j + 1);
            issue(j, ahead);
            ahead = next;
        }

        // ---- the queries in fixed point, as B operands ----
#pragma unroll
        for (int y = 0; y < QR; y++) {
            const int r = warp + kDecWarps * y;
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) big = max(big, __float_as_uint(x[y][i]) & 0x7fffffffu);
            big = __reduce_max_sync(0xffffffffu, big);
            // the largest to 2^22 .. 2^23, a bit less where its top digit would pass 127 (three
            // digits hold 127 * 65793), or as far up as a power of two reaches
            const int up = min(22 + 127 - int(big >> 23) - ((big & 0x7fffffu) > 0x7efe00u), 126);
            const float mul = pow2i(up);
            if (lane == 0) qscale[r] = big < 0x7f800000u ? a.scale_log2 * pow2i(-up) : __int_as_float(0x7fffffff);
            int8_t* dst = reinterpret_cast<int8_t*>(sm + L::q) + (r >> 3) * HD * 8;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                // dimension 32 i + lane: half, then group t of four within it
                int v = __float2int_rn(__fmul_rn(x[y][i], mul));
                const int at = (i * 32 + (r & 7) * 4 + ((lane >> 2) & 3)) * 8 + ((lane >> 4) << 2) + (lane & 3);
#pragma unroll
                for (int p = 0; p < PL; p++) {
                    const int8_t digit = int8_t(v);
                    dst[p * NT * HD * 8 + at] = digit;
                    v = (v - digit) >> 8;
                }
            }
        }
        __syncthreads();

        float o[HD / 16][NT][4], m_run[NT][2], r_run[NT][2], l_run[NT][2], qs[NT][2];
        int limit[NT][2];  // keys that the lane's columns see
        const int clear = min(k1, len - nq + row0 / a.group + 1);  // every row sees the keys before it
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                m_run[n][c] = r_run[n][c] = -INFINITY;
                l_run[n][c] = 0.f;
                const int r = 8 * n + 2 * t + c;
                qs[n][c] = qscale[r];
                limit[n][c] = r < rows ? len - nq + (row0 + r) / a.group + 1 : 0;
#pragma unroll
                for (int d = 0; d < HD / 16; d++) o[d][n][c] = o[d][n][c + 2] = 0.f;
            }
        for (int j = 0; j < steps; j++) {
            const int next = page_of(j + kDecStages);
            issue(j + kDecStages - 1, ahead);
            ahead = next;
            cp_async_wait<kDecStages - 1>();
            __syncwarp();
            const uint8_t* st = ring + (j % kDecStages) * L::stage;
            const uint32_t kb = saddr(st), vb = kb + SUB * L::row;
            const float* scales = reinterpret_cast<const float*>(st + 2 * SUB * L::row);
            const int tok0 = k0 + SUB * (warp + kDecWarps * j);
            float s[NB][NT][4];
            {
                int sum[PL][NB][NT][4];
#pragma unroll
                for (int p = 0; p < PL; p++)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int n = 0; n < NT; n++) sum[p][b][n][0] = sum[p][b][n][1] = sum[p][b][n][2] = sum[p][b][n][3] = 0;
#pragma unroll
                for (int d = 0; d < KB; d++) {
                    uint2 q[PL][NT];
#pragma unroll
                    for (int p = 0; p < PL; p++)
#pragma unroll
                        for (int n = 0; n < NT; n++)
                            q[p][n] = *reinterpret_cast<const uint2*>(sm + L::q + (((p * NT + n) * KB + d) * 32 + lane) * 8);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t x[4];
                        ldsm4(x, kb + b * 16 * L::row + L::at(lrow, lchunk + 2 * d));
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int p = 0; p < PL; p++) mma_s8(sum[p][b][n], x, q[p][n].x, q[p][n].y);
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float ks = scales[b];
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float f = float(sum[0][b][n][e] + (sum[1][b][n][e] << 8));
                            if (PL == 3) f = fmaf(float(sum[PL - 1][b][n][e]), 65536.f, f);
                            s[b][n][e] = f * (ks * qs[n][e & 1]);
                        }
                }
            }
            // ---- softmax: s[b][n][0, 1] token 16 b + g, columns 2t, 2t + 1; [2, 3] token + 8 ----
            if (tok0 + SUB > clear) {  // some key of the step is hidden from some query, or past the end
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (tok0 + 16 * b + g + 8 * (e >> 1) >= min(limit[n][e & 1], k1)) s[b][n][e] = -INFINITY;
            }
            uint32_t w[NB][NT][NP][2];  // weights as B operands
            float ve[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) ve[b] = tok0 + 16 * b < k1 ? kv8_exponent(scales[2 + b]) : -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float top[NB][2];
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int c = 0; c < 2; c++) top[b][c] = fmaxf(s[b][n][c], s[b][n][c + 2]);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int c = 0; c < 2; c++) top[b][c] = fmaxf(top[b][c], __shfl_xor_sync(0xffffffffu, top[b][c], x));
                float down[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float m = m_run[n][c], r = r_run[n][c];
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float t0 = ceilf(top[b][c]);
                        m = fmaxf(m, t0);
                        r = fmaxf(r, t0 + ve[b] - kLift);
                    }
                    l_run[n][c] *= kv8_step(m_run[n][c], m);
                    down[c] = kv8_step(r_run[n][c], r);
                    m_run[n][c] = m;
                    r_run[n][c] = r;
                    const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        // 2^(m + f - r), at least 0 where the page's values are all zero
                        const float f = ve[b] != ve[b] ? ve[b]
                                        : ve[b] == -INFINITY || r == -INFINITY ? 0.f
                                        : pow2i(int(fminf(fmaxf(m0 + ve[b] - r, -126.f), 126.f)));
#pragma unroll
                        for (int e = c; e < 4; e += 2) {
                            const float p = kv8_exp2(s[b][n][e] - m0);
                            l_run[n][c] += p;
                            // (a masked key adds nothing even to a page of NaN)
                            s[b][n][e] = s[b][n][e] == -INFINITY ? 0.f : p * f;
                        }
                    }
                }
                if (__any_sync(0xffffffffu, down[0] != 1.f || down[1] != 1.f)) {
#pragma unroll
                    for (int d = 0; d < HD / 16; d++) {
                        o[d][n][0] *= down[0];
                        o[d][n][1] *= down[1];
                        o[d][n][2] *= down[0];
                        o[d][n][3] *= down[1];
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t hi = kv8_half2(s[b][n][2 * e], s[b][n][2 * e + 1]);
                        w[b][n][0][e] = transposed(hi);
                        if (NP == 2) {
                            const float2 h = half2_floats(hi);
                            w[b][n][NP - 1][e] = transposed(
                                kv8_half2((s[b][n][2 * e] - h.x) * up, (s[b][n][2 * e + 1] - h.y) * up));
                        }
                    }
            }
            // ---- values: a step's products in an accumulator of their own, added to the
            // running ones in f32 (the tensor cores truncate, which over many steps is a bias) ----
#pragma unroll
            for (int d = 0; d < KB; d++) {
                uint32_t x[NB][4];
#pragma unroll
                for (int b = 0; b < NB; b++) ldsm4t(x[b], vb + b * 16 * L::row + L::at(lrow, lchunk + 2 * d));
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float y[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; n++) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
#pragma unroll
                    for (int b = 0; b < NB; b++) {  // (behind the last token: weights of 0 for whatever codes)
                        const uint32_t lo = x[b][2 * e] ^ 0x80808080u, hi = x[b][2 * e + 1] ^ 0x80808080u;
                        const uint32_t a0 = kv8_codes2<0x4240>(lo), a1 = kv8_codes2<0x4341>(lo), a2 = kv8_codes2<0x4240>(hi),
                                       a3 = kv8_codes2<0x4341>(hi);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            const uint32_t* low = w[b][n][NP - 1];
                            if (apart) mma_f16(y[n], kv8_under(a0), kv8_under(a1), kv8_under(a2), kv8_under(a3), low[0], low[1]);
                            else if (NP == 2) mma_f16(y[n], a0, a1, a2, a3, low[0], low[1]);
                            mma_f16(y[n], a0, a1, a2, a3, w[b][n][0][0], w[b][n][0][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) o[2 * d + e][n][c] += y[n][c];
                }
            }
            __syncwarp();
        }
        cp_async_wait<0>();
        __syncthreads();
        // ---- the warps' states through shared memory, added in warp order ----
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l_run[n][c] += __shfl_xor_sync(0xffffffffu, l_run[n][c], x);
                float* st = reinterpret_cast<float*>(sm + L::ring) + (warp * NR + 8 * n + 2 * t + c) * L::state;
#pragma unroll
                for (int d = 0; d < HD / 16; d++) {
                    st[16 * d + 2 * g] = o[d][n][c];
                    st[16 * d + 2 * g + 1] = o[d][n][c + 2];
                }
                if (g == 0) {
                    st[HD] = m_run[n][c];
                    st[HD + 1] = r_run[n][c];
                    st[HD + 2] = l_run[n][c];
                }
            }
        __syncthreads();
        const bool whole = units == nu;
        // the run's first piece may be a pair's tail or middle, its last one a pair's head
        float* part = a.parts + size_t(2 * blockIdx.x + (piece ? 1 : 0)) * NR * (HD + 4);
        for (int e = tid; e < rows * (HD / 4); e += kDecThreads) {
            const int r = e / (HD / 4), d = e % (HD / 4) * 4;
            const float* st = reinterpret_cast<const float*>(sm + L::ring) + r * L::state;
            float m = -INFINITY, ref = -INFINITY;
#pragma unroll
            for (int x = 0; x < kDecWarps; x++) {
                m = fmaxf(m, st[x * NR * L::state + HD]);
                ref = fmaxf(ref, st[x * NR * L::state + HD + 1]);
            }
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < kDecWarps; x++) {
                const float* sx = st + x * NR * L::state;
                sum = fmaf(sx[HD + 2], kv8_step(sx[HD], m), sum);
                const float down = kv8_step(sx[HD + 1], ref);
                const float4 y = *reinterpret_cast<const float4*>(sx + d);
                acc = make_float4(fmaf(y.x, down, acc.x), fmaf(y.y, down, acc.y), fmaf(y.z, down, acc.z), fmaf(y.w, down, acc.w));
            }
            if (whole) {
                const int qr = row0 + r, qi = qr / a.group, qh = head * a.group + qr % a.group;
                kv8_store4(a, int64_t(s0 + qi) * a.o_token + qh * a.o_head + d,
                           make_float4(kv8_finish(acc.x, ref, sum, m), kv8_finish(acc.y, ref, sum, m),
                                       kv8_finish(acc.z, ref, sum, m), kv8_finish(acc.w, ref, sum, m)));
            } else {
                *reinterpret_cast<float4*>(part + r * (HD + 4) + d) = acc;
                if (d == 0) *reinterpret_cast<float4*>(part + r * (HD + 4) + HD) = make_float4(m, ref, sum, 0.f);
            }
        }
    }
}

// Adds the parts of every (row tile, kv head) that the runs cut, in the order of
// the runs: the part of run c is its second where the pair begins in it after
// another, else its first.  One CTA of head_dim threads for each row; every warp
// forms the parts' factors for itself, a part to a lane, so that nothing waits but
// for the parts themselves.
__global__ void __launch_bounds__(256) kv8_combine_kernel(const Kv8Args a, int grid, int hd) {
    const int v = blockIdx.x, head = blockIdx.y, r = blockIdx.z, V = a.requests * a.tiles, NR = a.tile_rows;
    const int tid = threadIdx.x, lane = tid & 31, W = hd + 4;
    const int req = v / a.tiles, row = (v - req * a.tiles) * NR + r, s0 = a.starts[req], nq = a.starts[req + 1] - s0;
    pdl_wait();
    const int p0 = a.prefix[v], p1 = a.prefix[v + 1], total = a.prefix[V];
    const int nu = (p1 - p0) / a.kv_heads;
    if (nu == 0 || row >= nq * a.group) return;
    const int share = kv8_share(total, grid), u0 = p0 + head * nu, u1 = u0 + nu;
    const int c0 = u0 / share, c1 = (u1 - 1) / share;
    if (c0 == c1) return;  // one run held all of it and wrote the result
    auto part = [&](int c) { return a.parts + (size_t(2 * c + (u0 > share * c ? 1 : 0)) * NR + r) * W; };
    // (m, reference, sum) of a part
    auto state = [&](int c) { return c <= c1 ? *reinterpret_cast<const float4*>(part(c) + hd) : make_float4(-INFINITY, -INFINITY, 0.f, 0.f); };
    constexpr int U = 8;  // parts on their way at a time
    float x[U];
    auto fetch = [&](int c) {
#pragma unroll
        for (int i = 0; i < U; i++) x[i] = c + i <= c1 ? part(c + i)[tid] : 0.f;
    };
    const float4 first = state(c0 + lane);
    fetch(c0);
    float m = first.x, ref = first.y;
    for (int c = c0 + 32; c <= c1; c += 32) {
        const float4 s = state(c + lane);
        m = fmaxf(m, s.x);
        ref = fmaxf(ref, s.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    }
    float sum = 0.f, acc = 0.f;
    for (int b = c0; b <= c1; b += 32) {
        const float4 s = b == c0 ? first : state(b + lane);
        sum = fmaf(s.z, kv8_step(s.x, m), sum);
        const float mul = kv8_step(s.y, ref);
        const int n = min(32, c1 + 1 - b);
        for (int c = 0; c < n; c += U) {
            float y[U];
#pragma unroll
            for (int i = 0; i < U; i++) y[i] = x[i];
            fetch(b + c + U);
#pragma unroll
            for (int i = 0; i < U; i++) acc = fmaf(y[i], __shfl_sync(0xffffffffu, mul, c + i), acc);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int qi = row / a.group, qh = head * a.group + row % a.group;
    kv8_store(a, int64_t(s0 + qi) * a.o_token + qh * a.o_head + tid, kv8_finish(acc, ref, sum, m));
}

template <int HD, int NT, Weights WT>
void launch_decode(const Kv8Args& a, int grid, bool join, cudaStream_t st) {
    constexpr int smem = DecSmem<HD, NT>::total;
    static_assert(smem <= 227 * 1024, "a CTA's shared memory");
    static_assert(kv8_dec_ctas(HD, NT) * (smem + 1024) <= 228 * 1024, "the grid is made for this many CTAs on an SM");
    static std::atomic<unsigned long long> done{0};
    allow_smem(kv8_decode_kernel<HD, NT, WT>, smem, done);
    kv8_decode_kernel<HD, NT, WT><<<grid, kDecThreads, smem, st>>>(a);
    CUDA_OK(cudaGetLastError());
    if (!join) return;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(a.requests * a.tiles), unsigned(a.kv_heads), unsigned(std::min(a.tile_rows, a.most * a.group)));
    cfg.blockDim = dim3(HD);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CUDA_OK(cudaLaunchKernelEx(&cfg, kv8_combine_kernel, a, grid, HD));
}

template <int HD, int NT>
void launch_type(const Kv8Args& a, int grid, bool join, cudaStream_t st) {
    if (a.dtype == SPM_F32) launch_decode<HD, NT, Weights::kTwoApart>(a, grid, join, st);
    else if (a.dtype == SPM_F16) launch_decode<HD, NT, Weights::kTwo>(a, grid, join, st);
    else launch_decode<HD, NT, Weights::kOne>(a, grid, join, st);
}

template <int HD>
void launch_dim(const Kv8Args& a, int nt, int grid, bool join, cudaStream_t st) {
    nt == 1 ? launch_type<HD, 1>(a, grid, join, st) : launch_type<HD, 2>(a, grid, join, st);
}

// How a call is cut, from what the host knows of it.
struct Plan {
    bool prompt;  // kv8_prompt.cu's kernel
    bool join;    // a (row tile, kv head) may be cut: kv8_combine_kernel has parts to add
    int nt, tiles, grid;
    uint64_t prefix_bytes, parts_bytes;
};

// Whether a call's kernel of many queries has to add its tiles in f32.  The tensor cores'
// accumulators truncate: a row's sum loses 2^-23.4 of itself at every product of 16 keys,
// 3e-9 a key with weights of one part, 6e-9 with two (measured with values of one sign:
// 2.4e-5 at 4096 keys, 4.3e-4 at 65536).  Never for f32; for 16-bit results up to a tenth
// of their own rounding, by what the table can hold.
bool sums_in_f32(const spm_kv8* c, uint32_t dtype, int width) {
    const int64_t keys = int64_t(width) * c->page_tokens;
    return dtype == SPM_F32 || keys > (dtype == SPM_F16 ? 8192 : 131072);
}

Plan plan_of(const spm_kv8* c, int heads, int requests, int most, int width, bool total) {
    Plan p;
    const int sms = 148;  // of a B200; the grid need not match the device's for the result
    const int group = heads / c->kv_heads;
    const int64_t rows = int64_t(std::max(most, 1)) * group;
    p.nt = rows <= 8 ? 1 : 2;
    p.tiles = int((rows + 8 * p.nt - 1) / (8 * p.nt));
    const int64_t small = int64_t(requests) * c->kv_heads * p.tiles;
    const int tall = kv8_prompt_rows(c->head_dim, total);
    const int64_t large = int64_t(requests) * c->kv_heads * ((rows + tall - 1) / tall) * (total && c->head_dim > 192 ? 2 : 1);
    // A row tile of 16 costs this kernel as much as one of 128 or 256 costs the kernel of
    // many queries, but shares its keys out over all SMs: 300 such tiles for each wave of
    // the other's CTAs is about where they meet (8 kv heads of 128 in bf16, 1024 / 4096 /
    // 8000 keys: 256 tiles 43 / 95 / 162 us here and 47 / 124 / 221 there, 336 tiles 55 /
    // 124 / 208 and 47 / 132 / 241, 640 tiles 79 / 209 / 372 and 46 / 124 / 222; in f32,
    // which sums apart, 256 tiles 46 / 106 / 180 and 38 / 102 / 184, 320 tiles 57 / 130 / 221
    // and 38 / 102 / 184; heads of 256, 4096 keys, 256 tiles 193 and 212, 512 tiles 345 and 212).
    // (More requests than a grid has in z stay here.)
    p.prompt = rows > 16 && requests <= 65535 && small > 300 * ((large + sms - 1) / sms);
    if (p.prompt) {
        p.tiles = int((rows + tall - 1) / tall);
        p.grid = 0;
        p.join = false;
        p.prefix_bytes = p.parts_bytes = 0;
        return p;
    }
    const int64_t pairs = int64_t(requests) * p.tiles;
    if (pairs > INT32_MAX) fail(SPM_E_ARG, "too many requests and queries for one call");
    const int per_sm = kv8_dec_ctas(c->head_dim, p.nt), unit = kDecWarps * kv8_sub(c->head_dim);
    const int64_t units = (int64_t(width) * c->page_tokens + unit - 1) / unit;
    if (std::max<int64_t>(units, 1) * c->kv_heads > (INT32_MAX - 65536) / std::max<int64_t>(pairs, 1))  // (counted in 32 bits)
        fail(SPM_E_ARG, "too many requests, queries and tokens for one call");
    p.grid = int(std::max<int64_t>(1, std::min<int64_t>(int64_t(per_sm) * sms, std::max<int64_t>(units, 1) * pairs * c->kv_heads)));
    p.join = units > 1 && pairs > 0 && most > 0;  // (a table of one unit: every run holds whole ones)
    p.prefix_bytes = (uint64_t(pairs + 1) * 4 + 15) & ~uint64_t(15);
    p.parts_bytes = !p.join ? 0 : uint64_t(p.grid) * 2 * 8 * p.nt * (c->head_dim + 4) * 4;
    return p;
}

void check_attention(const spm_kv8* c, int32_t heads, int32_t requests, int32_t most, int32_t width) {
    kv8_check(c);
    if (heads < 1 || heads % c->kv_heads || heads > INT32_MAX / 256) fail(SPM_E_ARG, "heads must be a multiple of kv_heads");
    if (requests < 0 || most < 0 || width < 0) fail(SPM_E_ARG, "negative size");
    if (int64_t(width) * c->page_tokens > INT32_MAX) fail(SPM_E_ARG, "positions are 32-bit: table_width * page_tokens must fit");
    if (int64_t(most) * (heads / c->kv_heads) > INT32_MAX - 1024) fail(SPM_E_ARG, "too many queries");
    if (c->kv_heads > 65535) fail(SPM_E_ARG, "too many kv heads");
}

}  // namespace
}  // namespace spm

using namespace spm;

spm_status spm_kv8_attention_workspace(const spm_kv8* c, int32_t heads, int32_t requests, int32_t most,
                                       int32_t table_width, uint64_t* bytes) {
    return guarded([&] {
        if (!bytes) fail(SPM_E_ARG, "null output");
        check_attention(c, heads, requests, most, table_width);
        *bytes = 0;
        for (bool total : {false, true}) {  // (the type is the call's)
            const Plan p = plan_of(c, heads, requests, most, table_width, total);
            *bytes = std::max(*bytes, p.prefix_bytes + p.parts_bytes);
        }
    });
}

spm_status spm_kv8_attention(const spm_kv8* c, uint32_t dtype, const void* q, int64_t q_token, int64_t q_head,
                             int32_t heads, int32_t rows, const int32_t* starts, const int32_t* lens,
                             int32_t requests, int32_t most, const int32_t* table, int32_t table_width, float scale,
                             void* out, int64_t out_token, int64_t out_head, int32_t clear_rest,
                             void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
    return guarded([&] {
        check_attention(c, heads, requests, most, table_width);
        kv8_check_type(dtype);
        if (rows < 0) fail(SPM_E_ARG, "negative row count");
        if (rows == 0 || ((requests == 0 || most == 0) && !clear_rest)) return;
        if (!q || !out || !starts || (requests && !lens) || (requests && table_width && !table)) fail(SPM_E_ARG, "null argument");
        const bool total = sums_in_f32(c, dtype, table_width);
        const Plan p = plan_of(c, heads, requests, most, table_width, total);
        if ((p.prefix_bytes && !workspace) || workspace_bytes < p.prefix_bytes + p.parts_bytes)
            fail(SPM_E_ARG, "the workspace is smaller than spm_kv8_attention_workspace says");
        if (reinterpret_cast<uintptr_t>(workspace) & 15) fail(SPM_E_ARG, "the workspace must be 16-byte aligned");
        DeviceScope scope(c->device);
        Kv8Args a{};
        a.k_codes = c->k_codes, a.v_codes = c->v_codes;
        a.k_scales = c->k_scales, a.v_scales = c->v_scales;
        a.pages = c->pages, a.page = c->page_tokens, a.shift = __builtin_ctz(unsigned(c->page_tokens));
        a.kv_heads = c->kv_heads, a.group = heads / c->kv_heads;
        a.q = q, a.q_token = q_token, a.q_head = q_head, a.dtype = dtype, a.rows = rows;
        a.starts = starts, a.lens = lens, a.requests = requests, a.most = most;
        a.table = table, a.width = table_width, a.tile_rows = p.prompt ? kv8_prompt_rows(c->head_dim, total) : 8 * p.nt, a.tiles = p.tiles;
        a.unit = kDecWarps * kv8_sub(c->head_dim);
        a.scale_log2 = float(double(scale) * 1.4426950408889634);
        a.out = out, a.o_token = out_token, a.o_head = out_head;
        a.prefix = static_cast<int32_t*>(workspace);
        a.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.prefix_bytes);
        a.status = c->status;
        a.clear = clear_rest != 0;
        const int64_t size = dtype == SPM_F32 ? 4 : 2;
        a.o_vec = !((reinterpret_cast<uintptr_t>(out) | uintptr_t(out_token * size) | uintptr_t(out_head * size)) & 15);
        const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        if (p.prompt) {
            launch_kv8_prompt(a, c->head_dim, total, st);
            return;
        }
        switch (c->head_dim) {
            case 64: launch_dim<64>(a, p.nt, p.grid, p.join, st); break;
            case 96: launch_dim<96>(a, p.nt, p.grid, p.join, st); break;
            case 128: launch_dim<128>(a, p.nt, p.grid, p.join, st); break;
            case 192: launch_dim<192>(a, p.nt, p.grid, p.join, st); break;
            default: launch_dim<256>(a, p.nt, p.grid, p.join, st); break;
        }
    });
}
