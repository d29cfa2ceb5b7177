// Sampling from logits (spm_sample): temperature, top-k, top-p, min-p.
//
// Every filter keeps a prefix of the tokens sorted by (logit descending, index
// ascending), so the three together keep the shortest one, which a threshold
// names: all keys above it and the first `ties` tokens by index that equal it.
//
// Weights exp((x - max) / T) are formed in 64 bits and held as integers in units
// of 2^-44 (a sum of 2^19 fits 64 bits), so sums are exact, independent of their
// order (shared memory atomics included) and the same on every run; a neighbour
// at a border of top-p or u is told apart at 2^-44 of the largest weight.
//
// The row is not sorted.  A histogram over 1024 bins of (max - x) / T, 1/64
// wide up to 12 and 5/64 up to 32, of counts (top-k) or masses (top-p) shows the bin in which the border
// lies; only what lies there (for top-k: there and above) is listed and sorted,
// a few hundred tokens as a rule.  Where a list would be longer than 2048 (long
// runs of equal logits, a large top_k) the border is found by radix selection
// over the logits' ordered 32-bit keys instead.
//
// What bounds it: the logits' bytes for many rows, and the 64-bit exponentials
// where top-k does not spare them; for few rows the chain of dependent passes and
// cluster barriers.  A row is one thread-block cluster whose CTAs keep its
// slices in shared memory, so the logits are read from HBM once and the
// histograms are added through distributed shared memory.  One row of 49152 takes 18 to 21
// us, 8 of 151936 with top-p 39, 128 of 151936 in bf16 86 with top-k (0.45 TB/s) and 160
// with top-p: about 40 and 170 instructions a logit.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.h"

namespace spm {
namespace {
using namespace dev;
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;       // of a CTA
constexpr int kBins = 1024;
constexpr int kSampleClusters = 16;       // CTAs of a row, at most (8: the portable ones, see launch_type)
constexpr int kList = 2048;               // tokens that are sorted, at most
constexpr int kOwn = 1024;                // of a CTA's slice
constexpr int kSampleSlice = 160 * 1024;  // bytes of a slice that shared memory holds
constexpr int kTable = 128;               // of the exponential
typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int32_t vocab, slice;   // slice: logits of a CTA, a multiple of four for each warp
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p, *u;
    int32_t *token, *kept;
    float* prob;
};

// Order-preserving key; 0 for what is never picked (NaN, -inf).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u || b == 0xff800000u) return 0;
    return b & 0x80000000u ? (b == 0x80000000u ? 0x80000000u : ~b) : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct alignas(16) Shared {
    union {
        struct {
            uint32_t low[kBins], high[kBins];  // this CTA's: counts in low, or masses in two words
            u64 total[kBins];                  // the cluster's
            u64 part[kBins];                   // sums of a share of the bins over some of the CTAs
        };
        struct {
            u64 list[kOwn];     // this CTA's border tokens: key, then the index's complement
            u64 sorted[kList];  // the cluster's
        };
    };
    double table[kTable];                 // 2^(j / kTable)
    u64 scan[32];
    u64 need_out, border, seg_mass[kSampleClusters * kSampleThreads / 32];
    uint32_t seg_count[kSampleClusters * kSampleThreads / 32], seg_ties[kSampleClusters * kSampleThreads / 32];
    float top[kSampleClusters];           // each CTA's largest logit
    uint32_t listed;                      // length of this CTA's list
    uint32_t equal;                       // tokens on the border up to the last one kept
    int bin_out;
    u64 pick_before, pick_ties, pick_total, pick_count;
    int pick_seg;
};

struct Row {
    double top, inv, slope;   // the largest logit, 1 / T, -128 log2(e) / T
    float ftop, bins;         // 64 / T: the first bins of a logit's distance from the top
    const double* table;
    __device__ __forceinline__ double below(float x) const { return x == ftop ? 0.0 : top - double(x); }
    __device__ __forceinline__ double weight(float x) const { return x == ftop ? 1.0 : exp(-below(x) * inv); }
    // round(2^(44 - y)), y = (top - x) log2(e) / T: table-driven (P. T. P. Tang,
    // ACM TOMS 15, 1989), 2^z = 2^e * 2^(j/128) * 2^(r/128), j and e integers, the
    // last factor's series to r^4 (|r| <= 1/2: 2e-15 from the whole one).
    // Without branches, so that several overlap; 0 for -inf and NaN.
    __device__ __forceinline__ u64 mass(float x) const {
        constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low bits
        constexpr double c = 0.69314718055994530942 / kTable;
        const double s = fma(top - double(x), slope, 44.0 * kTable), k = s + magic;
        const int n = __double2loint(k);
        const double r = s - (k - magic);
        const double p = fma(r, fma(r, fma(r, fma(r, c * c * c * c / 24, c * c * c / 6), c * c / 2), c), 1.0);
        const double t = p * table[n & (kTable - 1)];  // in [1, 2) or a rounding beside it
        // t 2^(n >> 7), at most 2^44, added to 2^52: its integer is the mantissa
        const double w = __hiloint2double(__double2hiint(t) + ((n & ~(kTable - 1)) << 13), __double2loint(t)) + 4503599627370496.0;
        // (under 2^-46 the weight is 0, and the exponent above soon past a double's; NaN is not above either)
        const u64 m = s > -2.0 * kTable ? __double_as_longlong(w) & 0xfffffffffffffull : 0;
        return x == INFINITY ? 1ull << 44 : m;
    }
    __device__ __forceinline__ float distance(float x) const { return fminf(ftop - x, 3.402823466e38f); }
    // The bin of a candidate's distance from the top; ascending as x descends.
    __device__ __forceinline__ float place(float x) const {
        const float t = x == INFINITY ? 0.f : distance(x) * bins;
        return fminf(fminf(t, fmaf(t, 0.2f, 0.8f * 768.f)), float(kBins - 1));  // (768 bins of 1/64, then five times as wide)
    }
    __device__ __forceinline__ int bin(float x) const { return int(place(x)); }
    __device__ __forceinline__ bool in_bin(float x, int b) const {
        const float p = place(x);
        return p >= float(b) && p < float(b + 1);
    }
    // And the 1024th part of bin b.
    __device__ __forceinline__ int part(float x, int b) const {
        return int(fminf((place(x) - float(b)) * float(kBins), float(kBins - 1)));
    }
};

// Inclusive sum over the block's threads on top of `base`; base becomes the total.
__device__ __forceinline__ u64 block_sums(Shared& s, u64 w, u64& base) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = w;
    __syncthreads();
    u64 t = lane < kSampleThreads / 32 ? s.scan[lane] : 0;  // a sum for each warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += y;
    }
    const u64 before = __shfl_sync(0xffffffffu, t, (warp + 31) & 31);
    w += base + (warp ? before : 0);
    base += __shfl_sync(0xffffffffu, t, 31);
    return w;
}

// From the cluster's totals, bins in the order FIRST (ascending or descending):
// the bin in which the running sum reaches `need` (>= 1), and what is needed
// inside it; -1 where the sum stays below.
template <bool DOWN>
__device__ void select_bin(Shared& s, u64 need, int& bin, u64& left, u64& all) {
    constexpr int PER = kBins / kSampleThreads;
    static_assert(PER >= 1, "a bin for each thread");
    const int tid = threadIdx.x;
    auto at = [&](int i) { return s.total[DOWN ? kBins - 1 - i : i]; };
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) mine += at(tid * PER + j);
    all = 0;
    u64 before = block_sums(s, mine, all) - mine;
    if (tid == 0) s.bin_out = -1;
    __syncthreads();
    if (need == 0) return;  // the sum alone is asked for
    if (before < need && need <= before + mine) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const u64 t = at(tid * PER + j);
            if (before < need && need <= before + t) {
                s.bin_out = DOWN ? kBins - 1 - (tid * PER + j) : tid * PER + j;
                s.need_out = need - before;
            }
            before += t;
        }
    }
    __syncthreads();
    bin = s.bin_out;
    left = s.need_out;
}

// Descending bitonic sort of n <= kList entries, padded with 0: E neighbours to a
// thread, exchanges among them in registers, up to 32 E apart between lanes, and
// the rest through shared memory.
__device__ void sort_descending(u64* v, int n) {
    constexpr int E = kList / kSampleThreads;
    const int tid = threadIdx.x, i = E * tid;
    int size = 32 * E;
    while (size < n) size *= 2;
    const bool idle = i - E * (tid & 31) >= size;  // a warp of padding
    u64 a[E];
#pragma unroll
    for (int e = 0; e < E; e++) a[e] = i + e < n ? v[i + e] : 0;
    for (int k = 2; k <= size; k *= 2) {
        for (int j = k / 2; j >= E; j /= 2) {
            u64 c[E];
            if (j >= 32 * E) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (!idle) v[i + e] = a[e];
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++) c[e] = idle ? 0 : v[(i ^ j) + e];
            } else {
                if (idle) break;
#pragma unroll
                for (int e = 0; e < E; e++) c[e] = __shfl_xor_sync(0xffffffffu, a[e], j / E);
            }
            const bool larger = ((i & j) == 0) == ((i & k) == 0);  // this place takes the larger
#pragma unroll
            for (int e = 0; e < E; e++) a[e] = larger ? max(a[e], c[e]) : min(a[e], c[e]);
        }
#pragma unroll
        for (int j = E / 2; j > 0; j /= 2) {
            if (j >= k) continue;
#pragma unroll
            for (int e = 0; e < E; e++)
                if (!(e & j)) {
                    const bool down = ((i + e) & k) == 0;
                    const u64 lo = min(a[e], a[e + j]), hi = max(a[e], a[e + j]);
                    a[e] = down ? hi : lo;
                    a[e + j] = down ? lo : hi;
                }
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if (!idle) v[i + e] = a[e];
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
    constexpr int W = kSampleThreads / 32;
    extern __shared__ __align__(16) uint8_t raw[];
    Shared& s = *reinterpret_cast<Shared*>(raw);
    T* held = reinterpret_cast<T*>(raw + sizeof(Shared));
    cg::cluster_group cl = cg::this_cluster();
    const int C = int(cl.num_blocks()), rank = int(cl.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const int i0 = min(a.vocab, rank * a.slice), n = min(a.vocab, i0 + a.slice) - i0;
    const bool holds = a.slice * int(sizeof(T)) <= kSampleSlice;
    // four logits of the slice from i on (a multiple of four); -inf behind its end
    auto four = [&](int i, float (&v)[4]) {
        if (holds) {
            load4(held + i, true, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = i + j < n ? to_f32(x[i0 + i + j]) : -INFINITY;
        }
    };
    // f(four logits, the first's place) over the slice, by whole warps; -inf behind the end
    auto quads = [&](auto&& f) {
        for (int i0 = 128 * warp; i0 < n; i0 += 4 * kSampleThreads) {
            float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (i0 + 4 * lane < n) four(i0 + 4 * lane, v);
            f(v, i0 + 4 * lane);
        }
    };
    // f(logit, its place in the slice) for the candidates of this thread
    auto each = [&](auto&& f) {
        for (int i = 4 * tid; i < n; i += 4 * kSampleThreads) {
            float v[4];
            four(i, v);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (v[j] > -INFINITY) f(v[j], i + j);  // (not -inf, not NaN)
        }
    };
    cg::cluster_group::arrival_token started = cl.barrier_arrive();
    // the row's settings, on their way with its logits
    const float temp = a.temperature ? a.temperature[row] : 1.f, want_p = a.top_p ? a.top_p[row] : 1.f,
                want_min = a.min_p ? a.min_p[row] : 0.f, u = a.u[row];
    const int want_k = a.top_k ? a.top_k[row] : 0;

    // ---- the slice into shared memory; the largest logit (NaN is none) ----
    float top = -INFINITY;
    {
        constexpr int V = 16 / sizeof(T);
        const T* from = x + i0;
        const int head = min(n, int((16 - (reinterpret_cast<uintptr_t>(from) & 15)) & 15) / int(sizeof(T)));
        auto take = [&](int i, T v) {
            if (holds) held[i] = v;
            top = fmaxf(top, to_f32(v));
        };
        if (tid < head) take(tid, from[tid]);
        const int whole = (n - head) / V;
        const uint4* wide = reinterpret_cast<const uint4*>(from + head);
#pragma unroll 4
        for (int i = tid; i < whole; i += kSampleThreads) {
            const uint4 q = __ldcs(wide + i);
            const T* e = reinterpret_cast<const T*>(&q);
            if (holds && head == 0) reinterpret_cast<uint4*>(held)[i] = q;
#pragma unroll
            for (int j = 0; j < V; j++) {
                if (head == 0) top = fmaxf(top, to_f32(e[j]));
                else take(head + V * i + j, e[j]);
            }
        }
        const int rest = head + V * whole;
        if (tid < n - rest) take(rest + tid, from[rest + tid]);
        if (holds && tid < 4 && n + tid < a.slice) held[n + tid] = from_f32<T>(-INFINITY);  // the last four's places
    }
    if (tid < kTable) s.table[tid] = exp2(double(tid) / kTable);
    for (int b = tid; b < kBins; b += kSampleThreads) s.low[b] = s.high[b] = 0;
    if (tid == 0) s.listed = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float* tops = reinterpret_cast<float*>(s.scan);
    if (lane == 0) tops[warp] = top;
    cl.barrier_wait(std::move(started));  // every CTA runs
    __syncthreads();
    if (tid < C) {
#pragma unroll 8
        for (int w = 0; w < W; w++) top = fmaxf(top, tops[w]);
        cl.map_shared_rank(s.top, tid)[rank] = top;
    }
    cl.sync();
#pragma unroll 8
    for (int c = 0; c < C; c++) top = fmaxf(top, s.top[c]);
    if (top == -INFINITY) {  // the same for the whole cluster
        if (rank == 0 && tid == 0) {
            a.token[row] = -1;
            if (a.kept) a.kept[row] = 0;
            if (a.prob) a.prob[row] = 0.f;
        }
        return;
    }
    const bool greedy = !(temp > 0.f);
    Row r;
    r.ftop = top;
    r.top = double(r.ftop);
    r.inv = greedy ? 1.0 : 1.0 / double(temp);
    r.slope = r.inv * -1.4426950408889634074 * kTable;
    r.bins = r.ftop == INFINITY ? 1e30f : fminf(float(64.0 * r.inv), 1e30f);
    r.table = s.table;
    int k = greedy ? 0 : want_k;
    if (k <= 0 || k >= a.vocab) k = 0;
    if (greedy) k = 1;
    const float p = greedy ? 1.f : want_p;
    const bool nucleus = p < 1.f;
    const float least = greedy ? 0.f : want_min;
    // weight >= min_p as a distance from the top; off (NaN too) at 0, 1 at most
    const bool floored = least > 0.f;
    const double reach = floored ? -log(fmin(double(least), 1.0)) : 0.0;
    auto keeps = [&](float v) { return !floored || r.below(v) * r.inv <= reach; };

    auto clear = [&]() {
        for (int b = tid; b < kBins; b += kSampleThreads) s.low[b] = s.high[b] = 0;
        __syncthreads();
    };
    // A 64-bit sum of two 32-bit atomics, the second one for a carry or a weight from
    // 2^-12 on: few.
    auto add_low = [&](int b, u64 w) { return uint32_t(w) ? atomicAdd(&s.low[b], uint32_t(w)) : 0u; };
    auto add_high = [&](int b, u64 w, uint32_t old) {
        const uint32_t up = uint32_t(w >> 32) + (old + uint32_t(w) < old);
        if (up) atomicAdd(&s.high[b], up);
    };
    auto add_mass = [&](int b, u64 w) { add_high(b, w, add_low(b, w)); };
    // the CTAs' histograms added into every CTA's total
    auto gather = [&](bool mass) {
        cl.sync();
        const int share = kBins / C, parts = max(1, min(4, kSampleThreads / share)), each = (C + parts - 1) / parts;
        for (int e = tid; e < share * parts; e += kSampleThreads) {
            const int b = rank * share + e % share, q = e / share;
            u64 sum = 0;
#pragma unroll 4
            for (int c = q * each; c < min(C, (q + 1) * each); c++) {
                sum += cl.map_shared_rank(s.low, c)[b];
                if (mass) sum += u64(cl.map_shared_rank(s.high, c)[b]) << 32;
            }
            if (parts == 1) {
                for (int c = 0; c < C; c++) cl.map_shared_rank(s.total, c)[b] = sum;
            } else {
                s.part[e] = sum;
            }
        }
        if (parts > 1) {
            __syncthreads();
            for (int e = tid; e < share * parts; e += kSampleThreads) {
                const int i = e % share, q = e / share;
                u64 sum = 0;
                for (int g = 0; g < parts; g++) sum += s.part[g * share + i];
#pragma unroll 4
                for (int c = q * each; c < min(C, (q + 1) * each); c++)
                    cl.map_shared_rank(s.total, c)[rank * share + i] = sum;
            }
        }
        cl.sync();
    };
    // the lengths of the cluster's lists together; past kList where one is not whole
    auto listed = [&]() {
        const int m = lane < C ? int(*cl.map_shared_rank(&s.listed, lane)) : 0;
        const int sum = int(__reduce_add_sync(0xffffffffu, uint32_t(m)));
        return __any_sync(0xffffffffu, m > kOwn) ? max(sum, kList + 1) : sum;
    };
    // the lists, whole, in this CTA's `sorted`, its warps sharing out the CTAs; their length
    auto collect = [&]() {
        const int m = lane < C ? int(*cl.map_shared_rank(&s.listed, lane)) : 0;
        int to = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, to, o);
            if (lane >= o) to += y;
        }
        const int len = __shfl_sync(0xffffffffu, to, 31), share = max(1, W / C);
        for (int c = warp % C; c < C; c += W) {
            const int at = __shfl_sync(0xffffffffu, to - m, c), n = __shfl_sync(0xffffffffu, m, c);
            const u64* from = cl.map_shared_rank(s.list, c);
            for (int i = warp / C * 32 + lane; i < n; i += 32 * share) s.sorted[at + i] = from[i];
        }
        __syncthreads();
        return len;
    };
    // lists the candidates that `in` takes; listed counts them even where the list is full
    auto list = [&](auto&& in) {
        quads([&](const float (&v)[4], int i) {
            uint32_t take = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) take |= uint32_t(v[j] > -INFINITY && in(v[j])) << j;
            const uint32_t some = __ballot_sync(0xffffffffu, take != 0);
            if (!some) return;
            const int mine = __popc(take);
            int to = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, to, o);
                if (lane >= o) to += y;
            }
            int at = 0;
            if (lane == 31) at = int(atomicAdd(&s.listed, uint32_t(to)));
            at = __shfl_sync(0xffffffffu, at, 31) + to - mine;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (take >> j & 1) {
                    if (at < kOwn) s.list[at] = u64(key_of(v[j])) << 32 | (0xffffffffu - uint32_t(i0 + i + j));
                    at++;
                }
        });
    };

    uint32_t thr = 1;               // kept: keys above thr, and the first `ties` that equal it
    u64 ties = ~0ull;
    bool radix_k = false, radix_p = false;
    if (k) {
        each([&](float v, int) { atomicAdd(&s.low[r.bin(v)], 1u); });
        gather(false);
        int bin = 0;
        u64 left = 0, all = 0;
        select_bin<false>(s, u64(k), bin, left, all);
        if (bin >= 0) {
            const u64 upto = k - left + s.total[bin];  // tokens of this bin and those before
            __syncthreads();                           // (the list lies over the totals)
            bool whole = upto <= u64(kList);
            if (whole) {
                list([&](float v) { return r.place(v) < float(bin + 1); });
                cl.sync();
                whole = listed() <= kList;
                if (!whole) cl.sync();  // the lists' lengths have been read
            }
            if (whole) {
                // all of them sorted: the borders, and the pick among them, in the first CTA
                int len = rank == 0 ? collect() : 0;
                cl.sync();  // the others' lists have been read
                if (rank) return;
                sort_descending(s.sorted, len);
                len = min(len, k);
                auto mass_at = [&](int i) { return i < len ? r.mass(value_of(uint32_t(s.sorted[i] >> 32))) : 0; };
                u64 total = 0;
                for (int c0 = 0; c0 < len; c0 += kSampleThreads) block_sums(s, mass_at(c0 + tid), total);
                const double want = ceil(double(p) * double(total));
                const u64 need = !nucleus ? total : want < 1.0 ? 1 : min(total, __double2ull_rn(want));
                // a prefix, the first one among it: its length is its count
                int kept = 0;
                u64 before = 0;
                for (int c0 = 0; c0 < len && kept == c0; c0 += kSampleThreads) {
                    const int i = c0 + tid;
                    const u64 own = mass_at(i), w = block_sums(s, own, before);
                    const bool in = i < len && (!nucleus || w - own < need) && keeps(value_of(uint32_t(s.sorted[i] >> 32)));
                    kept += __syncthreads_count(in);
                    if (i == kept - 1) s.need_out = w;
                }
                __syncthreads();
                total = s.need_out;
                u64 target = u > 0.f ? __double2ull_rd(fmin(double(u), 1.0) * double(total)) : 0;
                target = min(target, total - 1);
                __syncthreads();
                // by index: complement first, descending
                for (int i = tid; i < kept; i += kSampleThreads) s.sorted[i] = s.sorted[i] << 32 | s.sorted[i] >> 32;
                __syncthreads();
                sort_descending(s.sorted, kept);
                u64 run = 0;
                for (int c0 = 0; c0 < kept; c0 += kSampleThreads) {
                    const int i = c0 + tid;
                    const u64 own = i < kept ? r.mass(value_of(uint32_t(s.sorted[i]))) : 0, w = block_sums(s, own, run);
                    if (i < kept && w - own <= target && target < w) {
                        a.token[row] = int32_t(0xffffffffu - uint32_t(s.sorted[i] >> 32));
                        if (a.kept) a.kept[row] = kept;
                        if (a.prob) a.prob[row] = float(r.weight(value_of(uint32_t(s.sorted[i]))) * 17592186044416.0 / double(total));
                    }
                }
                return;
            }
            radix_k = true;
        }
        radix_p = nucleus;
    } else if (nucleus) {
        // The border lies above every weight under half of (1 - p) / vocab: all of those
        // sum to less than 1 - p of the total.  They need no bins (a register holds their
        // sum, which goes to the last bin).
        const double edge = 0.5 * (1.0 - fmax(double(p), 0.0)) / double(a.vocab) * 17592186044416.0;
        const u64 small = edge < 1.0 ? 0 : u64(edge);
        u64 rest = 0;
        quads([&](const float (&v)[4], int) {
            u64 m[4];
#pragma unroll
            for (int j = 0; j < 4; j++) m[j] = r.mass(v[j]);
            uint32_t old[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (m[j] < small) {
                    rest += m[j];
                    m[j] = 0;
                }
                old[j] = add_low(r.bin(v[j]), m[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) add_high(r.bin(v[j]), m[j], old[j]);
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
        if (lane == 0) add_mass(kBins - 1, rest);
        gather(true);
        int bin = 0, sub = -1, m = 0;
        u64 need = 0, left = 0, sum = 0;
        select_bin<false>(s, 0, bin, left, sum);
        const double want = ceil(double(p) * double(sum));
        need = want < 1.0 ? 1 : min(sum, __double2ull_rn(want));
        select_bin<false>(s, need, bin, left, sum);
        auto inside = [&](float v) { return r.in_bin(v, bin) && (sub < 0 || r.part(v, bin) == sub); };
        // what lies in the border's bin; in its part of the bin where that is too much
        while (true) {
            __syncthreads();  // (the list lies over the totals)
            list(inside);
            cl.sync();
            m = listed();
            if (m <= kList || sub >= 0) break;
            cl.sync();  // the lists' lengths have been read
            if (tid == 0) s.listed = 0;
            clear();
            each([&](float v, int) {
                if (r.in_bin(v, bin)) add_mass(r.part(v, bin), r.mass(v));
            });
            gather(true);
            select_bin<false>(s, left, sub, left, sum);
        }
        if (m <= kList) {
            // the first CTA sorts and tells the others (their SMs' other rows have the slots)
            if (rank == 0) {
                collect();
                sort_descending(s.sorted, m);
                // the first whose running sum reaches what is needed inside the bin
                u64 run = 0;
                if (tid == 0) s.bin_out = m - 1;
                for (int c0 = 0; c0 < m; c0 += kSampleThreads) {
                    const int i = c0 + tid;
                    const u64 own = i < m ? r.mass(value_of(uint32_t(s.sorted[i] >> 32))) : 0, w = block_sums(s, own, run);
                    if (i < m && w - own < left && left <= w) s.bin_out = i;
                }
                __syncthreads();
                const int last = max(0, s.bin_out);
                thr = uint32_t(s.sorted[last] >> 32);
                // its rank among the tokens that equal it (they lie side by side); `listed` stands,
                // other CTAs may still be adding the lengths up
                if (tid == 0) s.equal = 0;
                __syncthreads();
                for (int i = tid; i <= last; i += kSampleThreads)
                    if (uint32_t(s.sorted[i] >> 32) == thr) atomicAdd(&s.equal, 1u);
                __syncthreads();
                if (tid < C) *cl.map_shared_rank(&s.border, tid) = u64(thr) << 32 | s.equal;
            }
            cl.sync();
            thr = uint32_t(s.border >> 32);
            ties = uint32_t(s.border);
        } else {
            cl.sync();  // the lists' lengths have been read
            radix_p = true;
        }
    }
    // ---- radix selection, ten bits at a time from the top, where a list is too long ----
    constexpr int shift[4] = {22, 12, 2, 0};
    constexpr uint32_t above[4] = {0u, 0xffc00000u, 0xfffff000u, 0xfffffffcu};  // bits that earlier levels have fixed
    constexpr uint32_t digits[4] = {1023u, 1023u, 1023u, 3u};
    if (radix_k) {
        u64 need = u64(k), all;
        uint32_t prefix = 0;
        for (int level = 0; level < 4; level++) {
            clear();
            each([&](float v, int) {
                const uint32_t key = key_of(v);
                if ((key & above[level]) == prefix) atomicAdd(&s.low[key >> shift[level] & digits[level]], 1u);
            });
            gather(false);
            int bin;
            select_bin<true>(s, need, bin, need, all);
            prefix |= uint32_t(bin) << shift[level];
        }
        thr = prefix;
        ties = need;
    }
    if (radix_p) {
        u64 need = 0, all;
        uint32_t prefix = 0;
        int bin;
        for (int level = 0; level < 4; level++) {
            clear();
            each([&](float v, int) {
                const uint32_t key = key_of(v);
                if ((key & above[level]) == prefix && (key > thr || (key == thr && ties == ~0ull)))
                    add_mass(key >> shift[level] & digits[level], r.mass(v));
            });
            // top-k's ties, once for the row
            if (rank == 0 && tid == 0 && ties != ~0ull && (thr & above[level]) == prefix)
                add_mass(thr >> shift[level] & digits[level], r.mass(value_of(thr)) * ties);
            gather(true);
            if (level == 0) {
                select_bin<true>(s, 0, bin, need, all);
                const double want = ceil(double(p) * double(all));
                need = want < 1.0 ? 1 : min(all, __double2ull_rn(want));
            }
            select_bin<true>(s, need, bin, need, all);
            prefix |= uint32_t(bin) << shift[level];
        }
        const u64 w = r.mass(value_of(prefix)), m = (need + w - 1) / w;
        if (prefix > thr || (prefix == thr && m < ties)) {
            thr = prefix;
            ties = m;
        }
    }
    // ---- min-p as a threshold of its own: the least logit that keeps() takes ----
    float cut = thr == 1 ? -INFINITY : value_of(thr);  // kept: above it, and `ties` of its equals
    if (floored) {
        // by bisection over the keys, from a few around the rounded border where they hold it
        const float near = fminf(fmaxf(float(r.top - reach * double(temp)), -3.402823466e38f), r.ftop);
        uint32_t no = 0x007fffffu, yes = key_of(r.ftop);  // below every finite key; the top is kept
        const uint32_t mid = key_of(near);
        if (mid > no + 4 && !keeps(value_of(mid - 4))) no = mid - 4;
        if (mid + 4 < yes && keeps(value_of(mid + 4))) yes = mid + 4;
        while (yes - no > 1) {
            const uint32_t k = no + (yes - no) / 2;
            if (keeps(value_of(k))) yes = k;
            else no = k;
        }
        const float v = value_of(yes);
        if (v > cut) {
            cut = v;
            ties = ~0ull;
        }
    }
    // ---- masses, counts and ties of the warps' segments, in index order ----
    const int seg = a.slice / W, j0 = min(n, warp * seg), j1 = min(n, j0 + seg);
    const u64 tie_mass = r.mass(cut);
    u64 mass = 0;
    uint32_t count = 0, tied = 0;
    // what is kept queues up (where the lists were), so that weights are formed 32 at a time
    float* queue = reinterpret_cast<float*>(s.list) + 64 * warp;
    int waiting = 0;
    for (int b = j0; b < j1; b += 128) {
        const int i = b + 4 * lane;
        float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i < j1) four(i, v);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool in = i + j < j1, up = in && v[j] > cut;
            tied += in && v[j] == cut;
            const uint32_t m = __ballot_sync(0xffffffffu, up);
            if (up) queue[waiting + __popc(m & ((1u << lane) - 1))] = v[j];
            waiting += __popc(m);
            count += __popc(m);
            if (waiting >= 32) {
                __syncwarp();
                waiting -= 32;
                mass += r.mass(queue[waiting + lane]);
                __syncwarp();
            }
        }
    }
    __syncwarp();
    if (lane < waiting) mass += r.mass(queue[lane]);
    if (cut == -INFINITY) tied = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    tied = __reduce_add_sync(0xffffffffu, tied);
    if (lane < C) {
        const int to = rank * W + warp;
        cl.map_shared_rank(s.seg_mass, lane)[to] = mass;
        cl.map_shared_rank(s.seg_count, lane)[to] = count;
        cl.map_shared_rank(s.seg_ties, lane)[to] = tied;
    }
    cl.sync();
    // a few segments to each lane of the first warp; ties go to the first by index
    if (warp == 0) {
        const int segs = C * W, w0 = lane * (kSampleClusters * W / 32), w1 = min(segs, w0 + kSampleClusters * W / 32);
        auto inclusive = [&](u64 v) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += y;
            }
            return v;
        };
        u64 t = 0;
        for (int w = w0; w < w1; w++) t += s.seg_ties[w];
        const u64 ties0 = inclusive(t) - t;
        auto taken = [&](u64 before, int w) { return before >= ties ? 0 : min(u64(s.seg_ties[w]), ties - before); };
        u64 m = 0, c = 0, tb = ties0;
        for (int w = w0; w < w1; w++) {
            const u64 k = taken(tb, w);
            m += k * tie_mass + s.seg_mass[w];
            c += k + s.seg_count[w];
            tb += s.seg_ties[w];
        }
        u64 mb = inclusive(m);
        const u64 total = __shfl_sync(0xffffffffu, mb, 31);
        mb -= m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
        // the first token with cumulated mass > target
        u64 target = u > 0.f ? __double2ull_rd(fmin(double(u), 1.0) * double(total)) : 0;
        target = min(target, total - 1);
        if (lane == 0) s.pick_seg = segs;
        __syncwarp();
        tb = ties0;
        for (int w = w0; w < w1 && mb <= target; w++) {
            const u64 here = taken(tb, w) * tie_mass + s.seg_mass[w];
            if (target < mb + here) {
                s.pick_seg = w;
                s.pick_before = target - mb;  // still to pass inside the segment
                s.pick_ties = tb;
                s.pick_total = total;
                s.pick_count = c;
            }
            mb += here;
            tb += s.seg_ties[w];
        }
    }
    __syncthreads();
    if (s.pick_seg / W != rank) return;
    const int from = min(n, s.pick_seg % W * seg), to = min(n, from + seg);
    u64 run = 0, seen = s.pick_ties;
    const u64 target = s.pick_before;
    const bool some = s.seg_ties[s.pick_seg] != 0;
    for (int c0 = from; c0 < to; c0 += kSampleThreads) {
        const int i = c0 + tid;
        const float v = i < to ? to_f32(holds ? held[i] : x[i0 + i]) : 0.f;
        const bool tie = i < to && v == cut && cut > -INFINITY;
        const u64 rank_of = some ? block_sums(s, tie, seen) : 0;  // this one counted
        const u64 own = tie ? (rank_of <= ties ? tie_mass : 0) : i < to && v > cut ? r.mass(v) : 0;
        const u64 w = block_sums(s, own, run);
        if (w - own <= target && target < w) {
            a.token[row] = i0 + i;
            if (a.kept) a.kept[row] = int32_t(s.pick_count);
            if (a.prob) a.prob[row] = float(r.weight(v) * 17592186044416.0 / double(s.pick_total));
        }
        if (run > target) break;
    }
}

cudaLaunchConfig_t sample_config(int rows, int ctas, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(rows) * unsigned(ctas));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = unsigned(ctas);
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

// Whether the current device has room for a cluster of kSampleClusters CTAs with the longest
// slices (asked for once per device: a part of a GPU may have too few SMs side by side).
template <class T>
bool wide_clusters_fit() {
    static std::atomic<int> known[64] = {};  // 1: no, 2: yes
    static std::atomic<unsigned long long> wide{0};
    int d = 0;
    CUDA_OK(cudaGetDevice(&d));
    if (d < 64 && known[d]) return known[d] == 2;
    allow_wide_clusters(sample_kernel<T>, wide);
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = sample_config(1, kSampleClusters, sizeof(Shared) + kSampleSlice, nullptr, &attr);
    int n = 0;
    const bool fits = cudaOccupancyMaxActiveClusters(&n, sample_kernel<T>, &cfg) == cudaSuccess && n > 0;
    if (!fits) cudaGetLastError();
    if (d < 64) known[d] = fits ? 2 : 1;
    return fits;
}

template <class T>
void launch_sample(const SampleArgs& a, int rows, int ctas, size_t smem, cudaStream_t st) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = sample_config(rows, ctas, smem, st, &attr);
    CUDA_OK(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a));
}

template <class T>
void launch_type(SampleArgs a, int rows, cudaStream_t st) {
    // A row's chain of passes and barriers takes as long as 32768 logits of one CTA (20 of
    // 28 us for one row of 151936 on 16 CTAs), and CTAs beyond two an SM (one, where the
    // slices are long) come in waves: the number of CTAs with the least waves x (chain +
    // slice), 2048 logits each at least.  16 (not portable: where the device holds such a
    // cluster, as a whole B200 does) from 65537 logits on while that leaves an SM to each:
    // 8 rows of 151936 take 38 us so where clusters of 8 take 44, of 49152 30 and 25, 16 rows
    // 66 and 48.  (1024 threads instead of 512, one CTA an SM: 32 us instead of 35 for top-p
    // on one row, 66 instead of 38 on eight.)
    static std::atomic<unsigned long long> done{0};
    allow_smem(sample_kernel<T>, sizeof(Shared) + kSampleSlice, done);
    const int sms = device_sms();
    const int per = 4 * 32;  // four for each warp, of 32 at most
    auto slice_of = [&](int ctas) { return ((a.vocab + ctas - 1) / ctas + per - 1) / per * per; };
    auto smem_of = [&](int ctas) {
        const size_t bytes = size_t(slice_of(ctas)) * sizeof(T);
        return sizeof(Shared) + (bytes <= size_t(kSampleSlice) ? bytes : 0);
    };
    int ctas = 1;
    int64_t least = INT64_MAX;
    for (int c = 1; c <= 8 && (c == 1 || a.vocab > 1024 * c); c *= 2) {
        const int64_t at_once = int64_t(sms) * (2 * (smem_of(c) + 1024) <= size_t(228 * 1024) ? 2 : 1);
        const bool held = size_t(slice_of(c)) * sizeof(T) <= size_t(kSampleSlice);  // else read again at half the rate
        const int64_t cost = (int64_t(rows) * c + at_once - 1) / at_once * (32768 + (held ? 1 : 2) * int64_t(slice_of(c)));
        if (cost <= least) least = cost, ctas = c;
    }
    if (a.vocab > 65536 && int64_t(rows) * kSampleClusters <= sms && wide_clusters_fit<T>()) ctas = kSampleClusters;
    a.slice = slice_of(ctas);
    const size_t smem = smem_of(ctas);
    launch_sample<T>(a, rows, ctas, smem, st);
}

}  // namespace
}  // namespace spm

using namespace spm;

spm_status spm_sample(int device, uint32_t dtype, const void* logits, int64_t row_stride, int32_t rows,
                      int32_t vocab, const float* temperature, const int32_t* top_k, const float* top_p,
                      const float* min_p, const float* u, int32_t* token, int32_t* kept, float* prob,
                      void* cuda_stream) {
    return guarded([&] {
        kv8_check_type(dtype);
        if (rows < 0) fail(SPM_E_ARG, "negative row count");
        if (rows > (1 << 24)) fail(SPM_E_ARG, "too many rows for one call");
        if (vocab < 1 || vocab > (1 << 19)) fail(SPM_E_ARG, "vocab is 1 to 2^19");
        if (rows == 0) return;
        if (!logits || !u || !token) fail(SPM_E_ARG, "null logits, u or token");
        DeviceScope scope(device);
        SampleArgs a{logits, row_stride, vocab, 0, temperature, top_k, top_p, min_p, u, token, kept, prob};
        const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        if (dtype == SPM_F32) launch_type<float>(a, rows, st);
        else if (dtype == SPM_F16) launch_type<__half>(a, rows, st);
        else launch_type<__nv_bfloat16>(a, rows, st);
    });
}
