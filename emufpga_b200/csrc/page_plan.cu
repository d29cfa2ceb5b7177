// Block tables, slot maps and the stack of free pages of one serving tick, on
// the device (spm_page_plan).
//
// With e_r = ceil(ended_r / P) pages back and f_r = ceil((cached_r + fresh_r) / P)
// - ceil(cached_r / P) pages wanted, exclusive sums over the rows give every
// page its place on the stack and every token its row:
//   push i of row r  -> free[count + E_r + i]           (E: sums of e)
//   page j of row r  <- free[count + E - 1 - (F_r + j)] (F: sums of f)
//   token t          -> row r with S_r <= t < S_r+1     (S: sums of fresh)
//
// What bounds it is latency: a few kilobytes and three dependent phases (push,
// pop, slots), so it is ONE launch of one cluster whose CTAs each form the sums
// in their own shared memory and then share out rows and tokens.  8 requests of a
// decode tick take 6 us (one CTA), 1024 with 96 prompts and 50 000 tokens 15 us (eight).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "abi.h"
#include "device.cuh"

namespace spm {
namespace {
using namespace dev;
namespace cg = cooperative_groups;

constexpr int kPlanThreads = 512, kPlanWarps = kPlanThreads / 32;
constexpr int kPlanRequests = 8192;
constexpr int kPlanTokens = INT32_MAX - 65536;  // the last turn's index fits 32 bits

struct PlanArgs {
    const int32_t *cached, *fresh, *ended;
    int32_t requests, page, shift;
    int32_t* table;
    int32_t width;
    int32_t* free_pages;
    int32_t pages;
    const int32_t* count;
    int32_t* left;
    int32_t tokens;
    int32_t *starts, *lens, *positions, *slots, *status;
};

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    return v;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanArgs a) {
    extern __shared__ int32_t sm[];
    __shared__ long long part[3][kPlanWarps];
    __shared__ int bad, shared_pages;
    cg::cluster_group cl = cg::this_cluster();
    const int R = a.requests, P = a.page, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = int(cl.block_rank()), ranks = int(cl.num_blocks());
    int32_t* S = sm;               // [R + 1] tokens before row r
    int32_t* E = S + R + 1;        // pages back before row r
    int32_t* F = E + R + 1;        // pages taken before row r
    int32_t* C = F + R + 1;        // cached
    if (tid == 0) bad = shared_pages = 0;
    __syncthreads();
    const int count = *a.count;
    // a thread's share of the rows, then the exclusive sums over threads
    const int per = (R + kPlanThreads - 1) / kPlanThreads, r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const long long cap = (long long)a.width << a.shift;
    long long s = 0, e = 0, f = 0;
    bool wrong = false, both = false;
    for (int r = r0; r < r1; r++) {
        const long long c = a.cached[r], n = a.fresh[r], d = a.ended ? a.ended[r] : 0;
        C[r] = int32_t(c);
        wrong |= c < 0 || n < 0 || d < 0 || c + n > cap || d > cap;
        both |= c > 0 && d > 0;  // the row's first pages would lie on the stack and in the row
        S[r] = int32_t(n);
        E[r] = int32_t((d + P - 1) >> a.shift);
        F[r] = int32_t(((c + n + P - 1) >> a.shift) - ((c + P - 1) >> a.shift));
        s += n;
        e += E[r];
        f += F[r];
    }
    if (wrong) bad = 1;
    if (both) shared_pages = 1;
    const long long si = warp_scan(s, lane), ei = warp_scan(e, lane), fi = warp_scan(f, lane);
    if (lane == 31) part[0][warp] = si, part[1][warp] = ei, part[2][warp] = fi;
    __syncthreads();
    if (warp < 3) {
        const long long v = lane < kPlanWarps ? part[warp][lane] : 0;
        const long long i = warp_scan(v, lane);
        if (lane < kPlanWarps) part[warp][lane] = i;
    }
    __syncthreads();
    const long long ts = part[0][kPlanWarps - 1], te = part[1][kPlanWarps - 1], tf = part[2][kPlanWarps - 1];
    int code = 0;
    if (bad) code = SPM_PAGE_LENGTH;
    else if (count < 0 || count + te > a.pages) code = SPM_PAGE_STACK;
    else if (tf > count + te) code = SPM_PAGE_FREE;
    else if (ts > a.tokens) code = SPM_PAGE_TOKENS;
    else if (shared_pages) code = SPM_PAGE_SHARED;
    if (code) {
        // nothing moves: no CTA of the cluster writes table or stack
        for (int i = rank * kPlanThreads + tid; i < a.tokens; i += ranks * kPlanThreads) a.positions[i] = a.slots[i] = -1;
        for (int i = rank * kPlanThreads + tid; i <= R; i += ranks * kPlanThreads) {
            a.starts[i] = 0;
            if (i < R) a.lens[i] = 0;
        }
        cl.sync();  // every CTA has read the count
        if (rank == 0 && tid == 0) {
            *a.left = count;
            flag(a.status, code);
        }
        return;
    }
    s = si - s + (warp ? part[0][warp - 1] : 0);
    e = ei - e + (warp ? part[1][warp - 1] : 0);
    f = fi - f + (warp ? part[2][warp - 1] : 0);
    for (int r = r0; r < r1; r++) {
        const int n = S[r], b = E[r], w = F[r];
        S[r] = int32_t(s);
        E[r] = int32_t(e);
        F[r] = int32_t(f);
        if (rank == 0) {
            a.starts[r] = int32_t(s);
            a.lens[r] = C[r] + n;
        }
        s += n;
        e += b;
        f += w;
    }
    if (tid == 0) {
        S[R] = int32_t(ts);
        E[R] = int32_t(te);
        F[R] = int32_t(tf);
        if (rank == 0) a.starts[R] = int32_t(ts);
    }
    __syncthreads();
    // The row of item t in exclusive sums X: X[row] <= t < X[row + 1].
    auto row_of = [&](const int32_t* X, int t) {
        int lo = 0, hi = R;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (X[mid] <= t) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    // Four items to a thread at a time: their searches and then their loads overlap.
    constexpr int U = 4;
    const int step = ranks * kPlanThreads, me = rank * kPlanThreads + tid;
    // pages of ended requests onto the stack
    for (int t0 = me; t0 < te; t0 += U * step) {
        int page[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int t = t0 + u * step;
            if (t >= te) continue;
            const int r = row_of(E, t);
            page[u] = a.table[size_t(r) * a.width + (t - E[r])];
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (t0 + u * step < te) a.free_pages[count + t0 + u * step] = page[u];
    }
    __threadfence();
    cl.sync();  // the whole stack stands, and the rows' old entries have been read
    if (rank == 0 && tid == 0) *a.left = int32_t(count + te - tf);
    for (int t0 = me; t0 < tf; t0 += U * step) {
        int page[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (t0 + u * step < tf) page[u] = __ldcg(a.free_pages + (count + te - 1 - (t0 + u * step)));
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int t = t0 + u * step;
            if (t >= tf) continue;
            const int r = row_of(F, t), old = int((uint32_t(C[r]) + P - 1) >> a.shift);
            a.table[size_t(r) * a.width + old + (t - F[r])] = page[u];
        }
    }
    __threadfence();
    cl.sync();  // the table stands
    // four tokens in a row to a thread: one search finds the first one's request
    for (int t0 = U * me; t0 < a.tokens; t0 += U * step) {
        int pos[U], page[U];
        int r = t0 < ts ? row_of(S, t0) : 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int t = t0 + u;
            pos[u] = -1;
            if (t >= ts) continue;
            while (S[r + 1] <= t) r++;
            pos[u] = C[r] + t - S[r];
            page[u] = __ldcg(a.table + size_t(r) * a.width + (pos[u] >> a.shift));
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int t = t0 + u;
            if (t >= a.tokens) break;
            int slot = -1;
            if (pos[u] >= 0) {
                if (uint32_t(page[u]) < uint32_t(a.pages)) slot = page[u] * P + (pos[u] & (P - 1));
                else flag(a.status, SPM_PAGE_ID);
            }
            a.positions[t] = pos[u];
            a.slots[t] = slot;
        }
    }
}

}  // namespace
}  // namespace spm

using namespace spm;

spm_status spm_page_plan(int device, const int32_t* cached, const int32_t* fresh, const int32_t* ended,
                         int32_t requests, int32_t page_tokens, int32_t* table, int32_t table_width,
                         int32_t* free_pages, int32_t pages, const int32_t* free_count, int32_t* free_left,
                         int32_t tokens, int32_t* starts, int32_t* lens, int32_t* positions, int32_t* slots,
                         int32_t* status, void* cuda_stream) {
    return guarded([&] {
        if (requests < 0 || requests > kPlanRequests) fail(SPM_E_ARG, "a plan takes 0 to 8192 requests");
        if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)))
            fail(SPM_E_ARG, "page_tokens is 16, 32, 64, 128 or 256");
        if (tokens < 0 || pages < 0 || table_width < 0) fail(SPM_E_ARG, "negative size");
        if (tokens > kPlanTokens) fail(SPM_E_ARG, "a plan takes up to 2^31 - 65537 tokens");
        if (int64_t(table_width) * page_tokens > INT32_MAX || int64_t(pages) * page_tokens > INT32_MAX)
            fail(SPM_E_ARG, "positions and slots are 32-bit: table_width and pages times page_tokens must fit");
        if (!free_count || !free_left || !starts) fail(SPM_E_ARG, "null free_count, free_left or starts");
        if (requests && (!cached || !fresh || !lens)) fail(SPM_E_ARG, "null lengths");
        if ((requests && table_width && !table) || (pages && !free_pages)) fail(SPM_E_ARG, "null table or stack");
        if (tokens && (!positions || !slots)) fail(SPM_E_ARG, "null positions or slots");
        DeviceScope scope(device);
        PlanArgs a{cached, fresh, ended, requests, page_tokens, __builtin_ctz(unsigned(page_tokens)), table, table_width,
                   free_pages, pages, free_count, free_left, tokens, starts, lens, positions, slots, status};
        const size_t smem = size_t(4 * requests + 3) * sizeof(int32_t);
        static std::atomic<unsigned long long> done{0};
        allow_smem(page_plan_kernel, size_t(4 * kPlanRequests + 3) * sizeof(int32_t), done);
        // one CTA up to a few rows and tokens for each of its threads, else a cluster of eight
        const unsigned ctas = requests <= 64 && tokens <= 4 * kPlanThreads ? 1 : 8;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(kPlanThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(cuda_stream);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        CUDA_OK(cudaLaunchKernelEx(&cfg, page_plan_kernel, a));
    });
}
