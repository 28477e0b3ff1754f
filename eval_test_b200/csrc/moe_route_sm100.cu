// Router of a mixture-of-experts layer: the top-k choice with its softmax weights, its gradient, and the plan that
// sorts the chosen copies by expert (what eval/nvfp4_grouped_gemm/reference.py:137-201 gets as a host list of group
// sizes is made here on the device).
//
//   route    p_e = exp(l_e - m) / sum,  m = the row's maximum;  the k largest l_e, ties to the lowest index
//   gradient renormalised over the chosen ones:  dl_{e_j} = w_j (dw_j - sum_i w_i dw_i), 0 elsewhere
//            over all experts:                   dl_e = p_e (g_e - sum_j w_j dw_j), g_e = dw_j where e = e_j, else 0
//   plan     stable counting sort: row(i) = first row of expert e + copies of e before i
//
// Entries that are NaN or -inf and whole rows whose mask is 0 are never chosen.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "moe_common.cuh"

namespace nvfp4 {
namespace {

// Order-preserving map of a float (not NaN) to unsigned; 0 is below every value and marks an excluded entry.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // (-0 counts as +0: the two are equal logits)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
// exp(l - m) with the limit for m = +inf: entries equal to the maximum share the weight.
__device__ __forceinline__ float exp_below(float l, float m) { return l == m ? 1.0f : expf(l - m); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct RouteArgs {
    const void* logits;
    long long ld;              // elements between rows
    const uint8_t* mask;       // [T] or null
    float* weights;            // [T][k]
    int* experts;              // [T][k]
    int T, E, k, renormalize;
};

// Keys of one token's row: lane holds the entries lane + 32 * i.
template <int KIND, int NV>
__device__ __forceinline__ void load_keys(const RouteArgs& a, int t, int lane, uint32_t (&key)[NV]) {
    using T = typename ElemOf<KIND>::type;
    const T* row = reinterpret_cast<const T*>(a.logits) + (long long)t * a.ld;
    const bool live = !a.mask || a.mask[t] != 0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int e = i * 32 + lane;
        float v = -INFINITY;
        if (live && e < a.E) v = to_f32(row[e]);
        key[i] = v > -INFINITY ? order_key(v) : 0u;      // (false for NaN)
    }
}

// One warp, one token.  k rounds of: the lane's best key, the warp's best key, the lowest index that has it.
// 16384 tokens, 256 experts, k = 8: the rounds cost more than the 16 MB of logits.
template <int KIND, int NV>
__device__ __forceinline__ void route_token(const RouteArgs& a, int t, int lane) {
    uint32_t key[NV];
    load_keys<KIND, NV>(a, t, lane, key);
    float total = 0.f, mine = 0.f, top = 0.f;
    int chosen = -1;
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) best = max(best, key[i]);
    for (int j = 0; j < a.k; j++) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, best);
        if (j == 0) {
            top = key_value(m);
            if (!a.renormalize) {
#pragma unroll
                for (int i = 0; i < NV; i++)
                    if (key[i]) total += exp_below(key_value(key[i]), top);
                total = warp_sum(total);
            }
        }
        if (m == 0) break;                                // fewer than k entries are left
        uint32_t at = 0xffffffffu;
        if (best == m) {
#pragma unroll
            for (int i = NV - 1; i >= 0; i--)
                if (key[i] == m) at = i * 32 + lane;
        }
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == j) {
            chosen = (int)at;
            mine = exp_below(key_value(m), top);
        }
        if (lane == (int)(at & 31u)) {
            best = 0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (i == (int)(at >> 5)) key[i] = 0;
                best = max(best, key[i]);
            }
        }
    }
    if (a.renormalize) total = warp_sum(mine);
    if (lane < a.k) {
        a.weights[(long long)t * a.k + lane] = chosen >= 0 ? mine / total : 0.f;
        a.experts[(long long)t * a.k + lane] = chosen;
    }
}

template <int KIND, int NV>
__global__ void __launch_bounds__(256) route_kernel(const RouteArgs a) {
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (blockDim.x >> 5);
    for (int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.T; t += warps) route_token<KIND, NV>(a, t, lane);
}

// One warp, one token.  The chosen experts' terms are handed round by shuffles, so every entry is written once.
template <int KIND, int NV>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteArgs a, const float* __restrict__ dw, void* dlogits) {
    using T = typename ElemOf<KIND>::type;
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (blockDim.x >> 5);
    for (int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.T; t += warps) {
        int e = -1;
        float w = 0.f, g = 0.f;
        if (lane < a.k) {
            e = a.experts[(long long)t * a.k + lane];
            if ((unsigned)e < (unsigned)a.E) {
                w = a.weights[(long long)t * a.k + lane];
                g = dw[(long long)t * a.k + lane];
            } else {
                e = -1;
            }
        }
        const float dot = warp_sum(w * g);
        const bool any = __any_sync(0xffffffffu, e >= 0);
        float p[NV], d[NV];
        if (!a.renormalize) {
            uint32_t key[NV], best = 0;
            load_keys<KIND, NV>(a, t, lane, key);
#pragma unroll
            for (int i = 0; i < NV; i++) best = max(best, key[i]);
            const float top = key_value(__reduce_max_sync(0xffffffffu, best));
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                p[i] = key[i] ? exp_below(key_value(key[i]), top) : 0.f;
                total += p[i];
            }
            total = warp_sum(total);
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] = (any && total > 0.f) ? p[i] / total : 0.f;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) d[i] = a.renormalize ? 0.f : -dot;
        const float own = a.renormalize ? w * (g - dot) : g;
        for (int j = 0; j < a.k; j++) {
            const int ej = __shfl_sync(0xffffffffu, e, j);
            const float gj = __shfl_sync(0xffffffffu, own, j);
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (ej == i * 32 + lane) d[i] += gj;
        }
        T* row = reinterpret_cast<T*>(dlogits) + (long long)t * a.E;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int idx = i * 32 + lane;
            if (idx < a.E) row[idx] = from_f32<T>(a.renormalize ? d[i] : (p[i] > 0.f ? p[i] * d[i] : 0.f));
        }
    }
}

// ------------------------------------------------------------------------------------------------ plan
struct PlanArgs {
    const int* experts;        // [T][k]
    int* offsets;              // [E+1] first sorted row of each expert
    int* tiles;                // [E+1] first 128-row tile of each expert
    int* rows;                 // [T][k] sorted row of a copy, -1: none
    int* slots;                // [T][k] the row counted with every expert padded to whole tiles, -1: none
    int* source;               // [T*k] copy of a sorted row, -1 behind the last
    int T, E, k;
};

constexpr int PLAN_WARPS = 32;

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

// The whole sort is ONE cluster: every warp owns a contiguous run of tokens, counts its copies per expert, the counts
// are summed over the warps of a CTA in its shared memory and over the CTAs through distributed shared memory, and a
// second walk over the same copies hands out the rows in order.  No global scratch, no atomics, so the order is that
// of the copies and a graph can replay it beside any other.  KIND >= 0: the warps choose their tokens' experts first
// (few tokens: one launch for router and plan).
template <int KIND, int NV>
__global__ void __launch_bounds__(PLAN_WARPS * 32, 1) plan_kernel(const PlanArgs p, const RouteArgs a) {
    extern __shared__ uint32_t plan_smem[];
    uint32_t* hist = plan_smem;                         // [PLAN_WARPS][E]
    uint32_t* total = hist + PLAN_WARPS * p.E;          // [E] copies of this CTA
    uint32_t* base = total + p.E;                       // [E] first row of this CTA's copies
    int* shift = reinterpret_cast<int*>(base + p.E);    // [E] slot - row of the expert
    __shared__ uint32_t warp_total[2][PLAN_WARPS];
    __shared__ uint32_t live_rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), ctas = cluster_size();
    const int per = (p.T + (int)ctas * PLAN_WARPS - 1) / ((int)ctas * PLAN_WARPS);
    const long long g = (long long)rank * PLAN_WARPS + warp;
    const int t0 = (int)min((long long)p.T, g * per), t1 = (int)min((long long)p.T, (g + 1) * per);
    const int begin = t0 * p.k, end = t1 * p.k;         // (T * k < 2^31: checked by the caller)

    for (int i = threadIdx.x; i < PLAN_WARPS * p.E; i += blockDim.x) hist[i] = 0;
    if constexpr (KIND >= 0) {
        for (int t = t0; t < t1; t++) route_token<KIND, NV>(a, t, lane);
    }
    __syncthreads();
    uint32_t* own = hist + warp * p.E;
    for (int i0 = begin; i0 < end; i0 += 32) {
        const int i = i0 + lane;
        const int e = i < end ? p.experts[i] : -1;
        const bool ok = (unsigned)e < (unsigned)p.E;
        const uint32_t same = __match_any_sync(0xffffffffu, ok ? e : -1);
        if (ok && lane == __ffs(same) - 1) own[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
        uint32_t run = 0;
        for (int w = 0; w < PLAN_WARPS; w++) {
            const uint32_t c = hist[w * p.E + e];
            hist[w * p.E + e] = run;
            run += c;
        }
        total[e] = run;
    }
    cluster_sync_all();
    // thread e: the expert's copies in all CTAs, in the CTAs before this one; then its first row and first tile
    // (MOE_MAX_EXPERTS = threads of the block)
    uint32_t count = 0, before = 0;
    if (threadIdx.x < p.E) {
        const uint32_t addr = smem_u32(total + threadIdx.x);
        for (uint32_t r = 0; r < ctas; r++) {
            const uint32_t c = ld_cluster_u32(mapa_shared(addr, r));
            before += r < rank ? c : 0;
            count += c;
        }
    }
    const uint32_t ntiles = (count + 127) / 128;
    uint32_t rows_to = count, tiles_to = ntiles;        // inclusive sums over the warp's experts
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, rows_to, o), y = __shfl_up_sync(0xffffffffu, tiles_to, o);
        if (lane >= o) { rows_to += x; tiles_to += y; }
    }
    if (lane == 31) { warp_total[0][warp] = rows_to; warp_total[1][warp] = tiles_to; }
    __syncthreads();
    uint32_t row0 = rows_to - count, tile0 = tiles_to - ntiles;
    for (int w = 0; w < warp; w++) { row0 += warp_total[0][w]; tile0 += warp_total[1][w]; }
    if (threadIdx.x < p.E) {
        base[threadIdx.x] = row0 + before;
        shift[threadIdx.x] = (int)(tile0 * 128u) - (int)row0;
        if (rank == 0) { p.offsets[threadIdx.x] = (int)row0; p.tiles[threadIdx.x] = (int)tile0; }
        if (threadIdx.x == p.E - 1) {
            live_rows = row0 + count;
            if (rank == 0) { p.offsets[p.E] = (int)(row0 + count); p.tiles[p.E] = (int)(tile0 + ntiles); }
        }
    }
    // also: no CTA leaves while a peer may still read its counts
    cluster_sync_all();
    for (int i0 = begin; i0 < end; i0 += 32) {
        const int i = i0 + lane;
        const int e = i < end ? p.experts[i] : -1;
        const bool ok = (unsigned)e < (unsigned)p.E;
        const uint32_t same = __match_any_sync(0xffffffffu, ok ? e : -1);
        int row = -1, slot = -1;
        if (ok) {
            row = (int)(base[e] + own[e]) + __popc(same & ((1u << lane) - 1u));
            slot = row + shift[e];
        }
        __syncwarp();
        if (ok && lane == __ffs(same) - 1) own[e] += __popc(same);
        __syncwarp();
        if (i < end) { p.rows[i] = row; p.slots[i] = slot; }
        if (ok) p.source[row] = i;
    }
    const int n = p.T * p.k;
    for (long long i = (long long)live_rows + rank * blockDim.x + threadIdx.x; i < n; i += (long long)ctas * blockDim.x) p.source[i] = -1;
}

template <int KIND, int NV>
int launch_plan(const PlanArgs& p, const RouteArgs& a, int ctas, cudaStream_t st) {
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64) return NVFP4_ERR_UNSUPPORTED;
    constexpr size_t most = (size_t)(PLAN_WARPS + 3) * MOE_MAX_EXPERTS * 4;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(plan_kernel<KIND, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(PLAN_WARPS * 32);
    cfg.dynamicSmemBytes = (size_t)(PLAN_WARPS + 3) * p.E * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, plan_kernel<KIND, NV>, p, a);
    return e == cudaSuccess ? NVFP4_OK : (int)e;
}

// CTAs of the sorting cluster: one for up to 1024 copies, then up to the eight that every device can place.
int plan_ctas(long long copies) {
    int c = 1;
    while (c < 8 && copies > 1024ll * c) c *= 2;
    return c;
}

template <int KIND, int NV>
int launch_route(const RouteArgs& a, const PlanArgs& p, int dev, cudaStream_t st) {
    // up to 256 tokens the sorting cluster chooses the experts itself, a token for each of its warps
    if (a.T <= 256) {
        int c = 1;
        while (c < 8 && a.T > PLAN_WARPS * c) c *= 2;
        return launch_plan<KIND, NV>(p, a, c, st);
    }
    int blocks = (a.T + 7) / 8;
    if (blocks > 8 * sm_count(dev)) blocks = 8 * sm_count(dev);
    route_kernel<KIND, NV><<<blocks, 256, 0, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    return launch_plan<-1, 1>(p, a, plan_ctas((long long)a.T * a.k), st);
}

template <int KIND, int NV>
int launch_backward(const RouteArgs& a, const float* dw, void* dlogits, int dev, cudaStream_t st) {
    int blocks = (a.T + 7) / 8;
    if (blocks > 8 * sm_count(dev)) blocks = 8 * sm_count(dev);
    route_backward_kernel<KIND, NV><<<blocks, 256, 0, st>>>(a, dw, dlogits);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NVFP4_OK : (int)e;
}

// f(KIND, NV) for the element type and the number of entries a lane holds
template <int KIND, typename F>
int by_width(int E, F&& f) {
    if (E <= 32) return f(std::integral_constant<int, KIND>(), std::integral_constant<int, 1>());
    if (E <= 64) return f(std::integral_constant<int, KIND>(), std::integral_constant<int, 2>());
    if (E <= 128) return f(std::integral_constant<int, KIND>(), std::integral_constant<int, 4>());
    if (E <= 256) return f(std::integral_constant<int, KIND>(), std::integral_constant<int, 8>());
    if (E <= 512) return f(std::integral_constant<int, KIND>(), std::integral_constant<int, 16>());
    return f(std::integral_constant<int, KIND>(), std::integral_constant<int, 32>());
}
template <typename F>
int by_kind(int kind, int E, F&& f) {
    if (kind == NVFP4_F32) return by_width<NVFP4_F32>(E, f);
    if (kind == NVFP4_F16) return by_width<NVFP4_F16>(E, f);
    return by_width<NVFP4_BF16>(E, f);
}

int check_route(int kind, long long ld, int T, int E, int k) {
    if (!kind_ok(kind)) return NVFP4_ERR_UNSUPPORTED;
    if (T <= 0 || E <= 0 || k <= 0 || k > E || ld < 0) return NVFP4_ERR_SHAPE;
    if (E > MOE_MAX_EXPERTS || k > MOE_MAX_CHOICES || (long long)T * k >= (1ll << 31)) return NVFP4_ERR_UNSUPPORTED;
    return NVFP4_OK;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_moe_plan(const void* experts, int T, int E, int k, void* offsets, void* tiles, void* rows, void* slots,
                              void* source, void* stream) {
    if (!experts || !offsets || !tiles || !rows || !slots || !source) return NVFP4_ERR_NULL;
    if (T <= 0 || E <= 0 || k <= 0) return NVFP4_ERR_SHAPE;
    // (padded rows are counted in 32 bits: up to 127 more for every expert)
    if (E > MOE_MAX_EXPERTS || (long long)T * k + 128ll * E >= (1ll << 31)) return NVFP4_ERR_UNSUPPORTED;
    const PlanArgs p{(const int*)experts, (int*)offsets, (int*)tiles, (int*)rows, (int*)slots, (int*)source, T, E, k};
    return launch_plan<-1, 1>(p, RouteArgs{}, plan_ctas((long long)T * k), (cudaStream_t)stream);
}

extern "C" int nvfp4_moe_route(const void* logits, int kind, long long ld, const void* mask, int T, int E, int k, int renormalize,
                               void* weights, void* experts, void* offsets, void* tiles, void* rows, void* slots, void* source,
                               void* stream) {
    if (!logits || !weights || !experts || !offsets || !tiles || !rows || !slots || !source) return NVFP4_ERR_NULL;
    int rc = check_route(kind, ld, T, E, k);
    if (rc) return rc;
    if ((long long)T * k + 128ll * E >= (1ll << 31)) return NVFP4_ERR_UNSUPPORTED;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    const RouteArgs a{logits, ld, (const uint8_t*)mask, (float*)weights, (int*)experts, T, E, k, renormalize};
    const PlanArgs p{(const int*)experts, (int*)offsets, (int*)tiles, (int*)rows, (int*)slots, (int*)source, T, E, k};
    return by_kind(kind, E, [&](auto K, auto V) { return launch_route<decltype(K)::value, decltype(V)::value>(a, p, dev, (cudaStream_t)stream); });
}

extern "C" int nvfp4_moe_route_backward(const void* dweights, const void* logits, int kind, long long ld, const void* weights,
                                        const void* experts, int T, int E, int k, int renormalize, void* dlogits, void* stream) {
    if (!dweights || !logits || !weights || !experts || !dlogits) return NVFP4_ERR_NULL;
    int rc = check_route(kind, ld, T, E, k);
    if (rc) return rc;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    const RouteArgs a{logits, ld, nullptr, (float*)const_cast<void*>(weights), (int*)const_cast<void*>(experts), T, E, k, renormalize};
    return by_kind(kind, E, [&](auto K, auto V) {
        return launch_backward<decltype(K)::value, decltype(V)::value>(a, (const float*)dweights, dlogits, dev, (cudaStream_t)stream);
    });
}
