// Attention of a prompt's many queries over the paged 8-bit KV cache, on the
// 5th-generation tensor cores (the other half of spm_kv8_attention; the formulas
// and the scaling by powers of two are kv8_attention.cu's).
//
// A CTA owns G groups of 128 rows (query x head of the group) of a request and kv
// head and walks the keys in tiles of TN, once:
//   producers            codes from global memory to fp16 (exact) in shared
//                        memory: a token's row of 64 dimensions is 128 bytes in the
//                        128-byte swizzled layout, which is K-major for the keys
//                        (S = Q K^T) and MN-major for the values (O = P V), so both
//                        are written alike and nothing is transposed
//   MMA (1 thread)       per group: O += P(j) V(j) with P from TMEM, then, once that
//                        is done (products of other accumulators do not order each
//                        other), the next S = Q K^T over the P just read
//   softmax (8 warps a group)  two threads own a row, half of a tile's keys each: S
//                        from TMEM, scale, mask, the running references, weights in
//                        fp16 back to where S stood
// With two groups the products of one run under the softmax of the other, and both
// share the conversion of the codes.  head_dim over 128 leaves TMEM and shared memory
// for one group, which has two buffers of S instead.  (Two buffers of 64 keys for
// two groups too: 176 us where one of 128 took 135, 32 heads of 128, 1024 queries over
// 4096 keys; a product of 64 columns takes the tensor cores as long as one of 128.)
// The accumulator's reference lies 2^15, what fp16 holds, under the largest weighted
// value and moves with it, so that weights keep 11 bits down to 2^-29 of the row's
// largest and a step of 2^-39 of it under that, in one part or two.  A slack of 2^14
// instead, which hardly ever reads the accumulator back, took 124.7 us where this takes
// 130.8, and lost every weight under 2^-25 of the largest.  The sum is f32: its reference
// has that slack.
// f32 queries are two fp16 parts (22 bits), and so are the weights of f32 and f16
// results: one part, 11 bits, would add as much to an f16 result as its own rounding.
// For a bf16 result, 8 bits, it is enough.  (1024 queries over 4096 keys, 32/8 heads of
// 128: f16 140 us; heads of 64 126 where one part took 107.)
// The tensor cores truncate their accumulators, which over thousands of keys is a bias
// (sums_in_f32 in kv8_attention.cu says how large).  f32 results, and 16-bit ones over long
// tables, therefore take the form with TOTAL: the products of a tile go to an
// accumulator of their own, which the softmax adds to the running one in f32, the
// reference's move with it.  TMEM holds that for one group of 128 rows, and for 128
// dimensions of values where head_dim is 256 (a cluster of two CTAs to a row tile, each
// with the whole scores).  f32 results are then within 5e-7 at every length; the case
// above takes 195 us in f32 where one accumulator took 147 and was off by up to 2.4e-5,
// 512 queries over 8000 keys 185 where it took 264 (twice the CTAs), heads of 256 390
// and 236.
//
// What bounds it is the softmax: the 16384 exponentials of a 128 x 128 tile take
// 1024 cycles of the special function unit, as long as its products, and its other
// instructions as many again: 131 us for the case above, 459 TFLOP/s.  (One thread a
// row, 128 columns: 136 us; S read once for maximum and weights: 144.)
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv8.h"
#include "kv8_attention.h"
#include "tcgen05.cuh"

namespace spm {
namespace {
using namespace dev;

constexpr int kRows = 128;                             // of a group: the MMA's M
constexpr float kSlack = 14.f;                         // of the sum's reference, in powers of two

// NQ, NP: fp16 parts of a query and of a weight.  TOTAL: every tile's products in an
// accumulator of their own, added to the running ones in f32.
template <int HD, int NQ, int NP, bool TOTAL>
struct PromptShape {
    static constexpr int G = kv8_prompt_rows(HD, TOTAL) / kRows;
    // converting warps: as many as leave the softmax its registers (80 of 24 warps, 96 of 20)
    static constexpr int fill = G == 2 ? 7 : 11;
    static constexpr int threads = 32 * (8 * G + fill + 1);
    static constexpr int TN = HD <= 128 ? 128 : 64;    // keys of a tile
    static constexpr int BUF = G == 1 ? 2 : 1;         // buffers of S
    static constexpr int DV = TOTAL && HD > 192 ? 128 : HD;  // value dimensions of a CTA, as many as TMEM holds twice
    static constexpr int atoms = (HD + 63) / 64;       // 64 dimensions, 128 bytes
    static constexpr int qgroup = atoms * kRows * 128; // bytes of a group's part of Q
    static constexpr int qbytes = G * NQ * qgroup;
    static constexpr int ktile = atoms * TN * 128, vtile = (DV + 63) / 64 * TN * 128;  // bytes of a tile of K and of V
    static constexpr int room = (227 * 1024 - 8192 - qbytes) / (ktile + vtile), stages = room > 4 ? 4 : room;
    static_assert(stages >= 1, "a tile of K and one of V");
    // (at least half of an SM's: a second CTA would wait for the first one's TMEM)
    static constexpr int need = qbytes + stages * (ktile + vtile) + 1024, smem = need > 120 * 1024 ? need : 120 * 1024;
    // TMEM columns: the buffers of S of each group, which its P replaces (16 columns
    // of S, 16 keys, hold the 8 columns of their high parts, then of their low ones),
    // the products with V, and the sums of those
    static constexpr int s_col = 0, o_col = BUF * G * TN, t_col = o_col + G * DV;
    static_assert(t_col + (TOTAL ? G * DV : 0) <= 512, "TMEM");
};

struct PromptSync {
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2][2], p_ready[2][2], o_done[2], o_last[2], met[2], drained;
    uint32_t tmem;
    volatile int gave_up;
    float qscale[2 * kRows];
    float reach[2][2][2 * kRows], state[2][2][2 * kRows];  // of a row's halves (state: m, sum)
    // scales of K and exponents of V's for a tile's blocks of 16 keys; tile j's are
    // overwritten with j + 8's, for which P(j) V(j) has to be done (four stages)
    float ks[8][8], ve[8][8], vn[8][8];  // (vn: NaN for a scale that is, else 0)
    int vi[8][8];                        // ve, -10000 for a scale of 0
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
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&r)[N]) {
    static_assert(N == 8 || N == 16, "the forms below");
    if constexpr (N == 8) {
        tmem_st8(at, r);
    } else {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
        tmem_st16(at, v);
    }
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Thirty-two columns of this warp's lanes, without waiting for them.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
// Waits for this thread's loads from TMEM; the registers of `r` are good after it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) asm volatile("" : "+r"(r[i]));
}

// Two f32 at a time.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 floats_of(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// The descriptor of an MN-major tile in the 128-byte swizzled layout: 8 rows (k) of
// 64 values (n) to an atom; `next` bytes from 64 values to the next 64, 1024 from 8
// rows to the next 8.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t at, uint32_t next) {
    return uint64_t((at & 0x3FFFFu) >> 4) | (uint64_t(next >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

typedef std::true_type Yes;
typedef std::false_type No;

template <int HD, int NQ, int NP, bool TOTAL>
__global__ void __launch_bounds__(PromptShape<HD, NQ, NP, TOTAL>::threads, 1) kv8_prompt_kernel(const Kv8Args a) {
    using S = PromptShape<HD, NQ, NP, TOTAL>;
    constexpr int TN = S::TN, ST = S::stages, G = S::G, BUF = S::BUF, DV = S::DV, FT = 32 * S::fill, kSoftWarps = 8 * G;
    extern __shared__ __align__(1024) uint8_t raw[];
    __shared__ PromptSync y;
    const uint32_t qs = (saddr(raw) + 1023u) & ~1023u, ks = qs + S::qbytes, vs = ks + ST * S::ktile;
    uint8_t* const base = raw + (qs - saddr(raw));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    kv8_clear<HD>(a, (blockIdx.z * (long long)gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x,
                  (long long)gridDim.x * gridDim.y * gridDim.z);
    // the last rows see the most keys: they go first; a row tile's CTAs side by side
    constexpr int parts = HD / DV;
    const int tile = int(gridDim.x - 1 - blockIdx.x) / parts, d0 = DV * int(blockIdx.x % parts), head = blockIdx.y, req = blockIdx.z;
    const int s0 = a.starts[req], e0 = a.starts[req + 1];
    if (s0 < 0 || e0 < s0 || e0 > a.rows || e0 - s0 > a.most) {
        if (tid == 0) flag(a.status, SPM_PAGE_QUERIES);
        return;
    }
    const int nq = e0 - s0, len = kv8_len(a, a.lens[req]), row0 = tile * G * kRows, rows = min(G * kRows, nq * a.group - row0);
    const int groups = (rows + kRows - 1) / kRows;  // that have rows
    if (rows <= 0) return;
    const int keys = kv8_keys(a, nq, len, tile), tiles = (keys + TN - 1) / TN;
    if (tid == 0) {
        for (int i = 0; i < 4; i++) {
            mbar_init(&y.k_full[i], FT);
            mbar_init(&y.k_empty[i], 1);
            mbar_init(&y.v_full[i], FT);
            mbar_init(&y.v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&y.s_full[0][i], 1);
            mbar_init(&y.s_full[1][i], 1);
            mbar_init(&y.p_ready[0][i], 2 * kRows);
            mbar_init(&y.p_ready[1][i], 2 * kRows);
            mbar_init(&y.met[i], 2 * kRows);
            mbar_init(&y.o_done[i], 1);
            mbar_init(&y.o_last[i], 1);
        }
        mbar_init(&y.drained, 1);
        y.gave_up = 0;
        mbar_fence_init();
    }
    constexpr int kMmaWarp = kSoftWarps + S::fill;
    // Each role does what it can before the first products, then all meet: a row tile's
    // CTAs too, which read the same queries before either writes its dimensions (out may be q).
    auto together = [&] {
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();
        if constexpr (parts > 1)
            asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
        tc_fence_after();
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // false once any wait of the CTA has given up
        if (y.gave_up) return false;
        if (mbar_wait(bar, parity)) return true;
        y.gave_up = 1;
        flag(a.status, SPM_PAGE_WAIT);
        return false;
    };

    if (warp >= kSoftWarps && warp < kMmaWarp) {
        // ---- producers: codes of tile j converted while those of j + 1 and the page
        // numbers of j + 2 are on their way ----
        // 16-byte pieces of a token, and of a thread (head_dim 96: the last ones of half the threads)
        constexpr int KSEG = HD / 16, VSEG = DV / 16, NK = (TN * KSEG + FT - 1) / FT, NV = (TN * VSEG + FT - 1) / FT;
        const int t = tid - 32 * kSoftWarps;
        const int32_t* trow = a.table + size_t(req) * a.width;
        uint4 k[NK], v[NV];
        int page[NK], vpage[NV];  // (the same where a CTA has all dimensions)
        auto pages_of = [&](int j, auto seg, auto& page) {
            constexpr int SEG = decltype(seg)::value, N = sizeof(page) / sizeof(int);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int tok = j * TN + (t + i * FT) / SEG;
                page[i] = tok < keys && t + i * FT < TN * SEG ? __ldg(trow + (tok >> a.shift)) : -1;
            }
        };
        typedef std::integral_constant<int, KSEG> KSeg;
        typedef std::integral_constant<int, VSEG> VSeg;
        auto find = [&](int j) {
            pages_of(j, KSeg(), page);
            if constexpr (DV != HD) pages_of(j, VSeg(), vpage);
        };
        // -1 for none, and for a page that is not in the pool
        auto known = [&](int p, int tok) {
            if (tok < keys && uint32_t(p) >= uint32_t(a.pages)) {
                flag(a.status, SPM_PAGE_ID);
                return -1;
            }
            return p;
        };
        auto load = [&](const int8_t* codes, int j, auto seg, const auto& page, auto& c) {
            constexpr int SEG = decltype(seg)::value, N = sizeof(page) / sizeof(int), PIECES = TN * SEG;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = t + i * FT, r = e / SEG, o = e % SEG, tok = j * TN + r;
                const int p = PIECES % FT != 0 && e >= PIECES ? -1 : known(page[i], tok);
                c[i] = make_uint4(0, 0, 0, 0);
                if (p >= 0)
                    c[i] = __ldg(reinterpret_cast<const uint4*>(
                        codes + ((size_t(p) * a.kv_heads + head) * a.page + (tok & (a.page - 1))) * HD + 16 * o));
            }
        };
        auto load_k = [&](int j) { load(a.k_codes, j, KSeg(), page, k); };
        auto load_v = [&](int j) {
            if constexpr (DV == HD) load(a.v_codes, j, KSeg(), page, v);
            else load(a.v_codes + d0, j, VSeg(), vpage, v);
        };
        auto store = [&](uint8_t* to, auto seg, const auto& c) {
            constexpr int SEG = decltype(seg)::value, N = sizeof(c) / sizeof(uint4), PIECES = TN * SEG;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = t + i * FT, r = e / SEG, o = e % SEG;
                if (PIECES % FT != 0 && e >= PIECES) break;
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
        // the scales of tile j's blocks, a thread to a block; likewise a tile ahead
        float kscale = 0.f, vscale = 0.f;
        auto scales = [&](int j) {
            const int tok = j * TN + 16 * t;
            kscale = vscale = 0.f;
            if (t >= TN / 16 || tok >= keys) return;
            const int p = known(__ldg(trow + (tok >> a.shift)), tok);
            if (p < 0) return;
            kscale = __ldg(a.k_scales + size_t(p) * a.kv_heads + head);
            vscale = __ldg(a.v_scales + size_t(p) * a.kv_heads + head);
        };
        if (tiles) {
            find(0);
            load_k(0);
            load_v(0);
            scales(0);
            find(1);
        }
        together();
        for (int j = 0; j < tiles; j++) {
            const int st = j % ST;
            const uint32_t again = uint32_t(j / ST - 1) & 1u;
            if (j >= ST && !wait(&y.k_empty[st], again)) break;
            store(base + S::qbytes + st * S::ktile, KSeg(), k);
            if (t < TN / 16) {
                y.ks[j & 7][t] = kscale;
                const float e = kv8_exponent(vscale);
                y.ve[j & 7][t] = e;
                y.vi[j & 7][t] = vscale > 0.f ? int(e) : -10000;
                y.vn[j & 7][t] = e != e ? e : 0.f;
            }
            fence_proxy_async();
            mbar_arrive(&y.k_full[st]);
            load_k(j + 1);
            scales(j + 1);
            if (j >= ST && !wait(&y.v_empty[st], again)) break;
            store(base + S::qbytes + ST * S::ktile + st * S::vtile, VSeg(), v);
            fence_proxy_async();
            mbar_arrive(&y.v_full[st]);
            load_v(j + 1);
            find(j + 2);
        }
    } else if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&y.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        together();
        const uint32_t tmem = y.tmem;
        if (lane == 0) {
            constexpr uint32_t f32_out = 1u << 4, m = uint32_t(kRows >> 4) << 24;
            constexpr uint32_t id_s = f32_out | m | uint32_t(TN >> 3) << 17;
            constexpr uint32_t id_o = f32_out | m | uint32_t(DV >> 3) << 17 | 1u << 16;  // V is MN-major
            auto scores = [&](int g, int j) {
                const uint32_t k = ks + uint32_t(j % ST) * S::ktile, q = qs + uint32_t(g * NQ) * S::qgroup;
#pragma unroll
                for (int p = NQ - 1; p >= 0; p--)
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++)
                        umma_f16(tmem + S::s_col + (BUF * g + j % BUF) * TN,
                                 sw128_desc(q + uint32_t(p) * S::qgroup + (kk >> 2) * (kRows * 128) + 32u * (kk & 3)),
                                 sw128_desc(k + (kk >> 2) * (TN * 128) + 32u * (kk & 3)), id_s, p != NQ - 1 || kk != 0);
                if (g == groups - 1) umma_commit(&y.k_empty[j % ST]);
                umma_commit(&y.s_full[g][j % BUF]);
            };
            auto keys_in = [&](int j) {
                const bool in = wait(&y.k_full[j % ST], uint32_t(j / ST) & 1u);
                tc_fence_after();
                return in;
            };
            bool ok = true;
            for (int j = 0; ok && j < min(BUF, tiles); j++) {
                ok = keys_in(j);
                for (int g = 0; ok && g < groups; g++) scores(g, j);
            }
            for (int j = 0; ok && j < tiles; j++)
                for (int g = 0; g < groups; g++) {
                    if (g == 0) ok = wait(&y.v_full[j % ST], uint32_t(j / ST) & 1u);
                    // (a barrier for each buffer: the softmax may be a tile further already)
                    ok = ok && wait(&y.p_ready[g][j % BUF], uint32_t(j / BUF) & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t v = vs + uint32_t(j % ST) * S::vtile;
#pragma unroll
                    for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                        for (int kk = 0; kk < TN / 16; kk++)
                            umma_f16_ts(tmem + S::o_col + g * DV, tmem + S::s_col + (BUF * g + j % BUF) * TN + 16u * kk + 8u * p,
                                        sw128_mn_desc(v + 2048u * kk, TN * 128), id_o, (!TOTAL && j != 0) || p != NP - 1 || kk != 0);
                    if (g == groups - 1) umma_commit(&y.v_empty[j % ST]);
                    umma_commit(&y.o_done[g]);
                    if (j + 1 == tiles) umma_commit(&y.o_last[g]);
                    if (j + BUF < tiles) {
                        if (g == 0) ok = keys_in(j + BUF);
                        ok = ok && wait(&y.o_done[g], uint32_t(j) & 1u);
                        if (!ok) break;
                        tc_fence_after();
                        scores(g, j + BUF);
                    }
                }
            umma_commit(&y.drained);  // TMEM is given back when every product has ended
            mbar_wait(&y.drained, 0);
        }
        __syncwarp();
    } else {
        // ---- Q: rows scaled to 2^10 by a power of two, in fp16 parts; four rows' loads together, while the first keys and values come ----
        constexpr int AT_ONCE = 4, STEP = kSoftWarps;
        for (int r0 = warp; r0 < groups * kRows; r0 += AT_ONCE * STEP) {
            float x[AT_ONCE][HD / 32];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                const int r = r0 + u * STEP, qr = row0 + r, qi = qr / a.group, qh = head * a.group + qr % a.group;
#pragma unroll
                for (int i = 0; i < HD / 32; i++)
                    x[u][i] = r < rows ? kv8_load(a, int64_t(s0 + qi) * a.q_token + qh * a.q_head + lane + 32 * i) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                const int r = r0 + u * STEP;
                if (r >= groups * kRows) break;
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < HD / 32; i++) big = max(big, __float_as_uint(x[u][i]) & 0x7fffffffu);
                big = __reduce_max_sync(0xffffffffu, big);
                const int up = min(137 - int(big >> 23), 126);
                // (a negative scale is the queries' sign: the largest sum is then the largest score)
                const float mul = a.scale_log2 < 0.f ? -pow2i(up) : pow2i(up);
                if (lane == 0) y.qscale[r] = big < 0x7f800000u ? fabsf(a.scale_log2) * pow2i(-up) : __int_as_float(0x7fffffff);
#pragma unroll
                for (int i = 0; i < HD / 32; i++) {
                    const int d = lane + 32 * i;
                    const float v = big < 0x7f800000u ? __fmul_rn(x[u][i], mul) : 0.f;
                    const __half hi = __float2half_rn(v);
                    const uint32_t at = uint32_t(r / kRows) * (NQ * S::qgroup) + uint32_t(d >> 6) * (kRows * 128) +
                                        sw128_offset(r % kRows, (d & 63) >> 3) + 2 * (d & 7);
                    *reinterpret_cast<__half*>(base + at) = hi;
                    if (NQ == 2) *reinterpret_cast<__half*>(base + S::qgroup + at) = __float2half_rn(__fsub_rn(v, __half2float(hi)));
                }
            }
        }
        together();
        const uint32_t tmem = y.tmem;
        // ---- softmax: two threads to a row, TMEM lane of its group, half of a tile's columns each ----
        const int g = warp >> 3, half = warp >> 2 & 1, r = g * kRows + 32 * (warp & 3) + lane;
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
        const uint32_t s0col = tmem + lanes + S::s_col + uint32_t(BUF * g) * TN, o = tmem + lanes + S::o_col + uint32_t(g) * DV,
                       total = tmem + lanes + S::t_col + uint32_t(g) * DV;
        constexpr int HC = TN / 64;  // of the 32 columns at a time
        const float qscale = y.qscale[r];
        const int limit = r < rows ? len - nq + (row0 + r) / a.group + 1 : 0;  // keys that the row sees
        // m and the sum are this half's, the accumulator's reference is the row's
        float m = -INFINITY, ref = -INFINITY, sum = 0.f, m0 = 0.f;  // m0: m, 0 for none yet
        bool ok = true;
        const int turns = g < groups ? tiles : 0;
        for (int j = 0; j < turns; j++) {
            ok = wait(&y.s_full[g][j % BUF], uint32_t(j / BUF) & 1u);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            const uint32_t s = s0col + uint32_t(j % BUF) * TN;
            tc_fence_after();
            const int t0 = j * TN;
            const bool hidden = __any_sync(0xffffffffu, t0 + TN > limit);
            // f(columns 32 c .. of S, c).  (Fetching the next columns meanwhile costs 32
            // registers more than there are, and more in spills than it saves.)
            auto columns = [&](auto&& f) {
#pragma unroll 1
                for (int c = HC * half; c < HC * half + HC; c++) {
                    uint32_t v[32];
                    tmem_ld32(s + 32 * c, v);
                    tmem_ld_wait(v);
                    f(v, c);
                }
            };
            // the half's maximum, and the largest exponent that a weighted value can have
            float top = -INFINITY, reach = -INFINITY;
            auto maxima = [&](auto masked) {
                columns([&](const uint32_t (&v)[32], int c) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int b = 2 * c + h;
                        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float y = __uint_as_float(v[16 * h + e]);
                            x[e & 3] = fmaxf(x[e & 3], masked && t0 + 16 * b + e >= limit ? -INFINITY : y);
                        }
                        float big = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        const float f = qscale * y.ks[j & 7][b];  // not negative, or NaN
                        big = big == -INFINITY ? big : f != f ? 0.f : ceilf(big * f);
                        top = fmaxf(top, big);
                        reach = fmaxf(reach, big + y.ve[j & 7][b]);
                    }
                });
            };
            hidden ? maxima(Yes()) : maxima(No());
            // both halves' (two buffers: who writes the next one has read this one's before)
            y.reach[j & 1][half][r] = reach;
            mbar_arrive(&y.met[g]);
            if (top > m + kSlack || (m == -INFINITY && top > m)) {
                sum *= kv8_step(m, top);
                m = m0 = top;
            }
            ok = wait(&y.met[g], uint32_t(j) & 1u);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            reach = fmaxf(reach, y.reach[j & 1][half ^ 1][r]);
            // a warp's rows together
            const bool moves = reach > ref + kLift || (ref == -INFINITY && reach > ref);
            if (TOTAL || __any_sync(0xffffffffu, moves)) {
                const float to = reach - kLift;
                const float down = moves ? kv8_step(ref, to) : 1.f;
                if (moves) ref = to;
                if (j) {
                    // O is the products' until P(j - 1) V(j - 1) is done (the one before is,
                    // TOTAL or S(j) waited for it: the parity is that of one phase alone)
                    ok = wait(&y.o_done[g], uint32_t(j - 1) & 1u);
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll 1
                    for (int d = half * (DV / 2); d < (half + 1) * (DV / 2); d += 16) {
                        float x[16];
                        tmem_ld16(o + d, x);
                        if (TOTAL && j > 1) {  // (P(j) V(j) goes over O once all have sent P(j))
                            float y[16];
                            tmem_ld16(total + d, y);
#pragma unroll
                            for (int e = 0; e < 16; e++) x[e] += y[e];
                        }
#pragma unroll
                        for (int e = 0; e < 16; e++) x[e] *= down;
                        tmem_st16((TOTAL ? total : o) + d, x);
                    }
                }
            }
            const int lift = ref == -INFINITY ? -20000 : int(fminf(fmaxf(m0 - ref, -5000.f), 5000.f));
            const uint64_t minus = pair_of(-m0, -m0);
            uint64_t sums[2] = {0, 0};
            auto weights = [&](auto masked) {
                columns([&](const uint32_t (&v)[32], int c) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int b = 2 * c + h;
                        // 2^(m + ve - ref); 2^-126, 0 in fp16, for a page of zeros; NaN for one of NaN
                        const float f = qscale * y.ks[j & 7][b];
                        const float w = pow2i(min(lift + y.vi[j & 7][b], 126)) + y.vn[j & 7][b];
                        const uint64_t ff = pair_of(f, f), ww = pair_of(w, w);
                        uint32_t out[8 * NP];
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 x = floats_of(
                                fma2(pair_of(__uint_as_float(v[16 * h + e]), __uint_as_float(v[16 * h + e + 1])), ff, minus));
                            uint64_t p = pair_of(kv8_exp2(x.x), kv8_exp2(x.y));
                            if (masked) {
                                // (a masked key adds nothing even to a page of NaN)
                                const bool s0 = t0 + 16 * b + e < limit, s1 = t0 + 16 * b + e + 1 < limit;
                                const float2 q = floats_of(p), z = floats_of(mul2(p, ww));
                                sums[h] = add2(sums[h], pair_of(s0 ? q.x : 0.f, s1 ? q.y : 0.f));
                                p = pair_of(s0 ? z.x : 0.f, s1 ? z.y : 0.f);
                            } else {
                                sums[h] = add2(sums[h], p);
                                p = mul2(p, ww);
                            }
                            const float2 z = floats_of(p);
                            out[e / 2] = kv8_half2(z.x, z.y);
                            if (NP == 2) {
                                const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&out[e / 2]));
                                out[8 * (NP - 1) + e / 2] = kv8_half2(z.x - q.x, z.y - q.y);
                            }
                        }
                        tmem_st<8 * NP>(s + 16 * b, out);
                    }
                });
            };
            hidden ? weights(Yes()) : weights(No());
            const float2 s2 = floats_of(add2(sums[0], sums[1]));
            sum += s2.x + s2.y;
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&y.p_ready[g][j % BUF]);
        }
        // (a barrier of its own: o_done may be two phases behind here, and its parity says nothing)
        if (ok && turns) {
            y.state[0][half][r] = m;
            y.state[1][half][r] = sum;
            mbar_arrive(&y.met[g]);
            ok = wait(&y.o_last[g], 0) && wait(&y.met[g], uint32_t(turns) & 1u);
        }
        tc_fence_after();
        if (__all_sync(0xffffffffu, ok) && g < groups) {
            if (turns) {  // (in the order of the halves for both)
                const float ma = y.state[0][0][r], mb = y.state[0][1][r];
                m = fmaxf(ma, mb);
                sum = y.state[1][0][r] * kv8_step(ma, m) + y.state[1][1][r] * kv8_step(mb, m);
            }
            const int qr = row0 + r, qi = qr / a.group, qh = head * a.group + qr % a.group;
            const int64_t at = int64_t(s0 + qi) * a.o_token + qh * a.o_head + d0;
#pragma unroll 1
            for (int d = half * (DV / 2); d < (half + 1) * (DV / 2); d += 16) {
                float v[16];
                if (tiles) {
                    tmem_ld16(o + d, v);
                    if (TOTAL && tiles > 1) {
                        float y[16];
                        tmem_ld16(total + d, y);
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e] += y[e];
                    }
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
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(y.tmem), "r"(512));
    }
}

template <int HD, int NQ, int NP, bool TOTAL>
void launch(const Kv8Args& a, cudaStream_t st) {
    using S = PromptShape<HD, NQ, NP, TOTAL>;
    static_assert(S::smem + int(sizeof(PromptSync)) <= 227 * 1024, "a CTA's shared memory");
    static std::atomic<unsigned long long> done{0};
    allow_smem(kv8_prompt_kernel<HD, NQ, NP, TOTAL>, S::smem, done);
    const dim3 grid(unsigned(a.tiles) * (HD / S::DV), unsigned(a.kv_heads), unsigned(a.requests));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(S::threads);
    cfg.dynamicSmemBytes = S::smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];  // a row tile's CTAs are a cluster
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = HD / S::DV;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = HD > S::DV ? 1 : 0;
    CUDA_OK(cudaLaunchKernelEx(&cfg, kv8_prompt_kernel<HD, NQ, NP, TOTAL>, a));
}

template <int HD>
void launch_parts(const Kv8Args& a, bool total, cudaStream_t st) {
    // a 16-bit query is one part, to 2^-34 of its largest (see above for the weights)
    if (a.dtype == SPM_F32) launch<HD, 2, 2, true>(a, st);
    else if (a.dtype == SPM_F16) total ? launch<HD, 1, 2, true>(a, st) : launch<HD, 1, 2, false>(a, st);
    else total ? launch<HD, 1, 1, true>(a, st) : launch<HD, 1, 1, false>(a, st);
}

}  // namespace

void launch_kv8_prompt(const Kv8Args& a, int head_dim, bool total, cudaStream_t st) {
    switch (head_dim) {
        case 64: launch_parts<64>(a, total, st); break;
        case 96: launch_parts<96>(a, total, st); break;
        case 128: launch_parts<128>(a, total, st); break;
        case 192: launch_parts<192>(a, total, st); break;
        default: launch_parts<256>(a, total, st); break;
    }
}

}  // namespace spm
