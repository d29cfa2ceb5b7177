// Sampling from logits (spm_sample): temperature, top-k, top-p, min-p.
//
// Every filter keeps a prefix of the tokens sorted by (logit descending, index
// ascending), so the three together keep the shortest one, which a threshold
// names: all keys above it and the first `ties` tokens by index that equal it.
// No sort: the threshold is found by radix selection over the logits' ordered
// 32-bit keys (11, 11 and 10 bits), by counts for top-k and by masses for top-p.
//
// Weights exp((x - max) / T) are formed in 64 bits and held as integers in units
// of 2^-44 (a sum of 2^19 fits 64 bits), so sums are exact, independent of their order (shared memory atomics
// included) and the same on every run; a neighbour at a border of top-p or u is
// told apart at 2^-44 of the largest weight.
//
// A row is one thread-block cluster: each CTA keeps its slice of the row in
// shared memory, so the logits are read from HBM once, and the cluster's
// histograms are added through distributed shared memory.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.h"

namespace spm {
namespace {
using namespace dev;
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048;
constexpr int kSampleClusters = 8;       // CTAs of a row, at most
constexpr int kSampleSlice = 40 * 1024;  // logits of a slice that shared memory holds
typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int32_t vocab, slice;   // slice: logits of a CTA, a multiple of the warps' 32
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

struct Shared {
    uint32_t hist[kBins];                 // counts, or the masses' low 16 bits
    uint32_t mid[kBins], high[kBins];     // masses' next 16 bits, and the rest
    u64 total[kBins];                     // the cluster's
    u64 scan[kSampleWarps];
    u64 need_out;
    int bin_out;
    uint32_t top[kSampleClusters];        // each CTA's largest key
    u64 seg_mass[kSampleClusters * kSampleWarps];
    uint32_t seg_count[kSampleClusters * kSampleWarps], seg_ties[kSampleClusters * kSampleWarps];
};

struct Row {
    double top, inv;      // the largest logit, 1 / T
    bool inf;             // it is +inf
    __device__ __forceinline__ double weight(float x) const {
        if (inf) return x == INFINITY ? 1.0 : 0.0;
        return exp((double(x) - top) * inv);
    }
    __device__ __forceinline__ u64 mass(float x) const { return __double2ull_rn(weight(x) * 17592186044416.0); }
};

// From the cluster's totals, bins descending: the bin in which the running sum
// reaches `need` (>= 1), and what is still needed inside it.
__device__ void select_bin(Shared& s, u64 need, int& bin, u64& left) {
    constexpr int PER = kBins / kSampleThreads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) mine += s.total[kBins - 1 - (tid * PER + j)];
    u64 incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 n = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += n;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = incl;
    __syncthreads();
    u64 before = incl - mine;
    for (int w = 0; w < warp; w++) before += s.scan[w];
    if (before < need && need <= before + mine) {
        for (int j = 0; j < PER; j++) {
            const int b = kBins - 1 - (tid * PER + j);
            if (need <= before + s.total[b]) {
                s.bin_out = b;
                s.need_out = need - before;
                break;
            }
            before += s.total[b];
        }
    }
    __syncthreads();
    bin = s.bin_out;
    left = s.need_out;
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared& s = *reinterpret_cast<Shared*>(raw);
    float* held = reinterpret_cast<float*>(raw + sizeof(Shared));
    cg::cluster_group cl = cg::this_cluster();
    const int C = int(cl.num_blocks()), rank = int(cl.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const int i0 = min(a.vocab, rank * a.slice), n = min(a.vocab, i0 + a.slice) - i0;
    const bool holds = a.slice <= kSampleSlice;
    auto at = [&](int i) { return holds ? held[i] : to_f32(x[i0 + i]); };

    // ---- the slice into shared memory; the largest key ----
    uint32_t top = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
        const float v = to_f32(x[i0 + i]);
        if (holds) held[i] = v;
        top = max(top, key_of(v));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (tid < kSampleClusters) s.top[tid] = 0;
    __syncthreads();
    if (lane == 0) atomicMax(&s.top[rank], top);
    __syncthreads();
    cl.sync();  // (every CTA's array stands)
    if (tid < C && tid != rank) s.top[tid] = cl.map_shared_rank(s.top, tid)[tid];
    cl.sync();
    top = 0;
    for (int c = 0; c < C; c++) top = max(top, s.top[c]);
    if (top == 0) {
        if (rank == 0 && tid == 0) {
            a.token[row] = -1;
            if (a.kept) a.kept[row] = 0;
            if (a.prob) a.prob[row] = 0.f;
        }
        return;
    }
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    Row r;
    r.top = double(value_of(top));
    r.inf = value_of(top) == INFINITY;
    r.inv = greedy ? 1.0 : 1.0 / double(temp);
    int k = greedy ? 1 : a.top_k ? a.top_k[row] : 0;
    if (k <= 0 || k >= a.vocab) k = 0;
    if (greedy) k = 1;
    const float p = !greedy && a.top_p ? a.top_p[row] : 1.f;
    const bool nucleus = p < 1.f;
    const float least = !greedy && a.min_p ? a.min_p[row] : 0.f;
    const float low = least > 1.f ? 1.f : least;  // (NaN compares as off below)

    auto clear = [&](bool mass) {
        for (int b = tid; b < kBins; b += kSampleThreads) {
            s.hist[b] = 0;
            if (mass) s.mid[b] = s.high[b] = 0;
        }
        __syncthreads();
    };
    // the CTAs' histograms added into every CTA's total
    auto gather = [&](bool mass) {
        __syncthreads();
        cl.sync();
        const int share = kBins / C;
        for (int b = rank * share + tid; b < (rank + 1) * share; b += kSampleThreads) {
            u64 sum = 0;
            for (int c = 0; c < C; c++) {
                sum += cl.map_shared_rank(s.hist, c)[b];
                if (mass)
                    sum += (u64(cl.map_shared_rank(s.mid, c)[b]) << 16) + (u64(cl.map_shared_rank(s.high, c)[b]) << 32);
            }
            for (int c = 0; c < C; c++) cl.map_shared_rank(s.total, c)[b] = sum;
        }
        cl.sync();
    };
    auto add_mass = [&](int b, u64 w) {
        atomicAdd(&s.hist[b], uint32_t(w & 0xffffu));
        atomicAdd(&s.mid[b], uint32_t(w >> 16 & 0xffffu));
        atomicAdd(&s.high[b], uint32_t(w >> 32));
    };
    constexpr int shift[3] = {21, 10, 0};
    constexpr uint32_t above[3] = {0u, 0xffe00000u, 0xfffffc00u};  // key bits that earlier levels have fixed

    uint32_t thr = 1;               // kept: keys above thr, and the first `ties` that equal it
    u64 ties = ~0ull;
    if (k) {
        u64 need = u64(k);
        uint32_t prefix = 0;
        bool all = false;           // fewer candidates than k: all are kept
        for (int level = 0; level < 3 && !all; level++) {
            clear(false);
            for (int i = tid; i < n; i += kSampleThreads) {
                const uint32_t key = key_of(at(i));
                if (key && (key & above[level]) == prefix) atomicAdd(&s.hist[key >> shift[level] & (kBins - 1)], 1u);
            }
            gather(false);
            if (level == 0) {
                s.bin_out = -1;
                __syncthreads();
            }
            int bin;
            select_bin(s, need, bin, need);
            if (level == 0 && bin < 0) all = true;
            else prefix |= uint32_t(bin) << shift[level];
        }
        if (!all) {
            thr = prefix;
            ties = need;
        }
    }
    if (nucleus) {
        u64 need = 0;
        uint32_t prefix = 0;
        for (int level = 0; level < 3; level++) {
            clear(true);
            for (int i = tid; i < n; i += kSampleThreads) {
                const float v = at(i);
                const uint32_t key = key_of(v);
                if (key && (key & above[level]) == prefix && (key > thr || (key == thr && ties == ~0ull)))
                    add_mass(key >> shift[level] & (kBins - 1), r.mass(v));
            }
            // top-k's ties, once for the row
            if (rank == 0 && tid == 0 && ties != ~0ull && (thr & above[level]) == prefix) {
                add_mass(thr >> shift[level] & (kBins - 1), r.mass(value_of(thr)) * ties);
            }
            gather(true);
            if (level == 0) {
                u64 sum = 0;
                for (int b = lane; b < kBins; b += 32) sum += s.total[b];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const double want = ceil(double(p) * double(sum));
                need = want < 1.0 ? 1 : min(sum, __double2ull_rn(want));
            }
            int bin;
            select_bin(s, need, bin, need);
            prefix |= uint32_t(bin) << shift[level];
        }
        const u64 w = r.mass(value_of(prefix)), m = (need + w - 1) / w;
        if (prefix > thr || (prefix == thr && m < ties)) {
            thr = prefix;
            ties = m;
        }
    }
    // ---- masses, counts and ties of the warps' segments, in index order ----
    const int seg = a.slice / kSampleWarps, j0 = min(n, warp * seg), j1 = min(n, j0 + seg);
    auto keeps = [&](float v) { return !(low > 0.f) || r.weight(v) >= double(low); };
    const u64 tie_mass = r.mass(value_of(thr));
    const bool tie_kept = keeps(value_of(thr));
    u64 mass = 0;
    uint32_t count = 0, tied = 0;
    for (int i = j0 + lane; i < j1; i += 32) {
        const float v = at(i);
        const uint32_t key = key_of(v);
        if (key > thr && keeps(v)) {
            mass += r.mass(v);
            count++;
        }
        tied += key == thr && tie_kept;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    count = __reduce_add_sync(0xffffffffu, count);
    tied = __reduce_add_sync(0xffffffffu, tied);
    if (lane < C) {
        const int to = rank * kSampleWarps + warp;
        cl.map_shared_rank(s.seg_mass, lane)[to] = mass;
        cl.map_shared_rank(s.seg_count, lane)[to] = count;
        cl.map_shared_rank(s.seg_ties, lane)[to] = tied;
    }
    cl.sync();
    u64 total = 0, before = 0;       // the row's kept mass; that of the segments before this warp's
    u64 ties_before = 0, ties_all = 0, count_all = 0;
    const int me = rank * kSampleWarps + warp;
    for (int w = 0; w < C * kSampleWarps; w++) {
        if (w == me) before = total, ties_before = ties_all;
        const u64 t = s.seg_ties[w], taken = ties_all >= ties ? 0 : min(t, ties - ties_all);
        total += s.seg_mass[w] + taken * tie_mass;
        count_all += s.seg_count[w] + taken;
        ties_all += t;
    }
    const float u = a.u[row];
    // the first token with cumulated mass > target
    u64 target = u > 0.f ? __double2ull_rd(fmin(double(u), 1.0) * double(total)) : 0;
    target = min(target, total - 1);
    u64 run = before, seen = ties_before;
    const u64 mine = s.seg_mass[me] + (seen >= ties ? 0 : min(u64(s.seg_ties[me]), ties - seen)) * tie_mass;
    if (before <= target && target < before + mine) {
        for (int i = j0; i < j1; i += 32) {
            u64 w = 0;
            float v = 0.f;
            uint32_t key = 0;
            if (i + lane < j1) {
                v = at(i + lane);
                key = key_of(v);
            }
            const bool tie = key == thr && tie_kept && key;
            const uint32_t b = __ballot_sync(0xffffffffu, tie);
            if (tie && seen + __popc(b & ((1u << lane) - 1)) < ties) w = tie_mass;
            else if (key > thr && keeps(v)) w = r.mass(v);
            seen += __popc(b);
            u64 incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const uint32_t over = __ballot_sync(0xffffffffu, run + incl > target);
            if (over) {
                if (lane == __ffs(over) - 1) {
                    a.token[row] = i0 + i + lane;
                    if (a.kept) a.kept[row] = int32_t(count_all);
                    if (a.prob) a.prob[row] = float(r.weight(v) * 17592186044416.0 / double(total));
                }
                break;
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
}

template <class T>
void launch_sample(const SampleArgs& a, int rows, int ctas, size_t smem, cudaStream_t st) {
    static unsigned long long done = 0;
    allow_smem(sample_kernel<T>, sizeof(Shared) + kSampleSlice * sizeof(float), done);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(rows) * unsigned(ctas));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(ctas);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CUDA_OK(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a));
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
        // a CTA for every 2048 logits, eight at most
        int ctas = 1;
        while (ctas < kSampleClusters && vocab > 2048 * ctas) ctas *= 2;
        const int per = kSampleThreads;  // 32 for each warp
        a.slice = ((vocab + ctas - 1) / ctas + per - 1) / per * per;
        const size_t smem = sizeof(Shared) + (a.slice <= kSampleSlice ? size_t(a.slice) * sizeof(float) : 0);
        const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
        if (dtype == SPM_F32) launch_sample<float>(a, rows, ctas, smem, st);
        else if (dtype == SPM_F16) launch_sample<__half>(a, rows, ctas, smem, st);
        else launch_sample<__nv_bfloat16>(a, rows, ctas, smem, st);
    });
}
