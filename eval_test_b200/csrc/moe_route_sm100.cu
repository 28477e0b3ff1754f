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

#include <type_traits>

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

// Over the G lanes of a token (every lane of the warp calls these).
template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int G> __device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

struct RouteArgs {
    const void* logits;
    long long ld;              // elements between rows
    const uint8_t* mask;       // [T] or null
    float* weights;            // [T][k]
    int* experts;              // [T][k]
    int T, E, k, renormalize;
    int wide;                  // rows start on 16-byte boundaries
};

// How a token's E entries lie in registers: G lanes with NV entries each, in pieces of VW neighbours (16 bytes), piece i
// of lane l starting at entry (i * G + l) * VW.  A token takes a quarter of a warp up to 128 experts: the rounds of the
// choice are bound by instruction issue, and the steps that reduce over lanes then serve four tokens at once (16384
// tokens of 128 experts, k = 4: 9.4 us against 12.1 us with a warp per token and entries 32 apart).
template <int KIND, int G_, int NV_> struct Layout {
    using T = typename ElemOf<KIND>::type;
    static constexpr int G = G_, NV = NV_, VW = 16 / (int)sizeof(T), PER_WARP = 32 / G_;
    // 16-bit logits: the order of a value takes at most 19 bits of its fp32 key, so its index fits below it and one
    // maximum finds both
    static constexpr bool PACKED = KIND != NVFP4_F32;
    static constexpr int MINE = (MOE_MAX_CHOICES + G - 1) / G;     // choices that a lane keeps
    static __device__ __forceinline__ int entry(int i, int in_group) { return ((i / VW) * G + in_group) * VW + i % VW; }
    static __device__ __forceinline__ float value(uint32_t key) { return key_value(PACKED ? ((key & 0x80000000u) ? key & ~1023u : key | 1023u) : key); }
};

template <typename L>
__device__ __forceinline__ void load_keys(const RouteArgs& a, int t, int in_group, uint32_t (&key)[L::NV]) {
    using T = typename L::T;
    const bool live = t < a.T && (!a.mask || a.mask[t] != 0);
    const T* row = reinterpret_cast<const T*>(a.logits) + (long long)(live ? t : 0) * a.ld;
#pragma unroll
    for (int i = 0; i < L::NV; i += L::VW) {
        const int e0 = L::entry(i, in_group);
        Vec<T, L::VW> v;
        const bool whole = a.wide && e0 + L::VW <= a.E;
        if (live && whole) v.load(row + e0);
#pragma unroll
        for (int q = 0; q < L::VW; q++) {
            float x = -INFINITY;
            if (live && whole) x = v.get(q);
            else if (live && e0 + q < a.E) x = to_f32(row[e0 + q]);
            uint32_t k = x > -INFINITY ? order_key(x) : 0u;      // (false for NaN)
            if (L::PACKED && k) k = (k & ~1023u) | (1023u - (uint32_t)(e0 + q));
            key[i + q] = k;
        }
    }
}

// The tokens t of a warp's groups (t differs between groups, all lanes call it).  k rounds of: the lane's best key, the
// group's best, the lowest index that has it; every lane of the group knows the choice, lane j % G keeps it.
template <typename L>
__device__ __forceinline__ void route_token(const RouteArgs& a, int t, int in_group) {
    constexpr int G = L::G, NV = L::NV;
    uint32_t key[NV], best = 0;
    load_keys<L>(a, t, in_group, key);
#pragma unroll
    for (int i = 0; i < NV; i++) best = max(best, key[i]);
    float total = 0.f, top = 0.f, mine[L::MINE];
    int chosen[L::MINE];
#pragma unroll
    for (int z = 0; z < L::MINE; z++) { mine[z] = 0.f; chosen[z] = -1; }
    for (int j = 0; j < a.k; j++) {
        const uint32_t m = group_max<G>(best);                   // 0: no candidate is left
        const float v = L::value(m);
        if (j == 0) {
            top = v;
            if (!a.renormalize) {
#pragma unroll
                for (int i = 0; i < NV; i++) total += key[i] ? exp_below(L::value(key[i]), top) : 0.f;
                total = group_sum<G>(total);
            }
        }
        uint32_t at;
        if (L::PACKED) {
            at = 1023u - (m & 1023u);
            best = 0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                key[i] = key[i] == m ? 0u : key[i];
                best = max(best, key[i]);
            }
        } else {
            // the lowest index that has the key, as the largest of their complements
            uint32_t low = 0;
#pragma unroll
            for (int i = NV - 1; i >= 0; i--)
                if (key[i] == m) low = 1024u - (uint32_t)L::entry(i, in_group);
            at = 1024u - group_max<G>(low);
            best = 0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if ((uint32_t)L::entry(i, in_group) == at) key[i] = 0u;
                best = max(best, key[i]);
            }
        }
        const float p = m ? exp_below(v, top) : 0.f;
        if (a.renormalize) total += p;
        if (in_group == j % G) {
#pragma unroll
            for (int z = 0; z < L::MINE; z++)
                if (z == j / G) { mine[z] = p; chosen[z] = m ? (int)at : -1; }
        }
    }
    if (t < a.T) {
#pragma unroll
        for (int z = 0; z < L::MINE; z++) {
            const int j = z * G + in_group;
            if (j < a.k) {
                a.weights[(long long)t * a.k + j] = chosen[z] >= 0 ? mine[z] / total : 0.f;
                a.experts[(long long)t * a.k + j] = chosen[z];
            }
        }
    }
}

template <typename L>
__global__ void __launch_bounds__(256) route_kernel(const RouteArgs a) {
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (blockDim.x >> 5);
    for (int t = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * L::PER_WARP; t < a.T; t += warps * L::PER_WARP)
        route_token<L>(a, t + lane / L::G, lane % L::G);
}

// G lanes, one token.  The chosen experts' terms are handed round by shuffles, so every entry is written once.
template <typename L>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteArgs a, const float* dw, void* dlogits) {
    using T = typename L::T;
    constexpr int G = L::G, NV = L::NV;
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31, in_group = lane % G;
    const int warps = gridDim.x * (blockDim.x >> 5);
    for (int t0 = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * L::PER_WARP; t0 < a.T; t0 += warps * L::PER_WARP) {
        const int t = t0 + lane / G;
        int e[L::MINE];
        float w[L::MINE], g[L::MINE], dot = 0.f;
        uint32_t any = 0;
#pragma unroll
        for (int z = 0; z < L::MINE; z++) {
            const int j = z * G + in_group;
            e[z] = -1; w[z] = g[z] = 0.f;
            if (t < a.T && j < a.k) {
                const int id = a.experts[(long long)t * a.k + j];
                if ((unsigned)id < (unsigned)a.E) {
                    e[z] = id;
                    w[z] = a.weights[(long long)t * a.k + j];
                    g[z] = dw[(long long)t * a.k + j];
                    any = 1;
                }
            }
            dot += w[z] * g[z];
        }
        dot = group_sum<G>(dot);
        any = group_max<G>(any);
        float p[NV], d[NV];
        if (!a.renormalize) {
            uint32_t key[NV], best = 0;
            load_keys<L>(a, t, in_group, key);
#pragma unroll
            for (int i = 0; i < NV; i++) best = max(best, key[i]);
            best = group_max<G>(best);
            const float top = L::value(best);
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                p[i] = key[i] ? exp_below(L::value(key[i]), top) : 0.f;
                total += p[i];
            }
            total = group_sum<G>(total);
            // (a row without choices, a masked one say, has gradient 0)
            const float scale = any ? 1.0f / total : 0.f;       // (one division for the row, an ulp more in its entries)
#pragma unroll
            for (int i = 0; i < NV; i++) p[i] *= scale;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) d[i] = a.renormalize ? 0.f : -dot;
#pragma unroll
        for (int z = 0; z < L::MINE; z++) {
            const float own = a.renormalize ? w[z] * (g[z] - dot) : g[z];
            for (int j = z * G; j < a.k && j < (z + 1) * G; j++) {
                const int ej = __shfl_sync(0xffffffffu, e[z], j - z * G, G);
                const float gj = __shfl_sync(0xffffffffu, own, j - z * G, G);
#pragma unroll
                for (int i = 0; i < NV; i++)
                    if (ej == L::entry(i, in_group)) d[i] += gj;
            }
        }
        if (t >= a.T) continue;
        T* row = reinterpret_cast<T*>(dlogits) + (long long)t * a.E;
#pragma unroll
        for (int i = 0; i < NV; i += L::VW) {
            const int e0 = L::entry(i, in_group);
            float f[L::VW];
#pragma unroll
            for (int q = 0; q < L::VW; q++) f[q] = a.renormalize ? d[i + q] : (p[i + q] > 0.f ? p[i + q] * d[i + q] : 0.f);
            if (a.E % L::VW == 0) {                               // (dlogits is contiguous and 16-byte aligned)
                Vec<T, L::VW> o;
                o.set(f);
                if (e0 < a.E) o.store(row + e0);
            } else {
#pragma unroll
                for (int q = 0; q < L::VW; q++) {
                    const float one[1] = {f[q]};
                    Vec<T, 1> o;
                    o.set(one);
                    if (e0 + q < a.E) o.store(row + e0 + q);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ plan
struct PlanArgs {
    const int* experts;        // [T][k]
    int* offsets;              // [E+1] first sorted row of each expert
    int* tiles;                // [E+1] first 128-row tile of each expert
    int* wide;                 // [E+1] first 256-row tile of each expert
    int* rows;                 // [T][k] sorted row of a copy, -1: none
    int* slots;                // [T][k] the row counted with every expert padded to whole tiles, -1: none
    int* source;               // [T*k] copy of a sorted row, -1 behind the last
    uint32_t* counts;          // [blocks][E] copies of a block: the spread form only
    int T, E, k;
};

constexpr int PLAN_WARPS = 32;
// Blocks of the spread form: every block sums the counts of all, so the more experts there are, the fewer blocks (131072
// copies: 64 experts 8.6 us with 128 blocks; 256 experts 15.3 us with 128, 12.8 us with 32; 1024 experts 40.5 us with
// 128, 22.8 us with 16).
__host__ __device__ constexpr int plan_blocks(int E) { return E <= 64 ? 128 : E >= 512 ? 16 : 8192 / E; }
constexpr long long PLAN_CLUSTER_MOST = 16384;   // copies that are sorted by one cluster
constexpr int PLAN_AHEAD = 8;      // rounds of 32 copies whose ids a warp has in flight

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

// Lanes whose key equals this lane's, by one vote per bit (match.any took 1900 cycles a round with a warp's 32 lanes at
// 64 experts, the votes take 300).
__device__ __forceinline__ uint32_t same_key(int key, int bits) {
    uint32_t same = 0xffffffffu;
    for (int b = 0; b < bits; b++) {
        const bool one = (key >> b) & 1;
        const uint32_t vote = __ballot_sync(0xffffffffu, one);
        same &= one ? vote : ~vote;
    }
    return same;
}

// Which tokens a block and a warp of it take: contiguous runs, the blocks' of equal length.  A warp takes at least
// `fewest` tokens (a round of 32 copies, or of the router), so that few tokens do not keep many warps.
struct TokenRange { int begin, end; };
__device__ __forceinline__ TokenRange block_tokens(int T, uint32_t blocks, uint32_t block) {
    const int per = (int)((T + (long long)blocks - 1) / blocks);
    return {(int)min((long long)T, (long long)block * per), (int)min((long long)T, (long long)(block + 1) * per)};
}
__device__ __forceinline__ TokenRange warp_tokens(TokenRange b, int fewest, int warp) {
    const int per = max((b.end - b.begin + PLAN_WARPS - 1) / PLAN_WARPS, fewest);
    return {(int)min((long long)b.end, b.begin + (long long)warp * per), (int)min((long long)b.end, b.begin + (long long)(warp + 1) * per)};
}

// Copies per expert of each block of the spread form (any order: they are only counted).
__global__ void __launch_bounds__(PLAN_WARPS * 32) plan_count_kernel(const PlanArgs p) {
    __shared__ uint32_t count[MOE_MAX_EXPERTS];
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) count[e] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch();
    const TokenRange b = block_tokens(p.T, gridDim.x, blockIdx.x);
    const int end = b.end * p.k;
    for (long long i = (long long)b.begin * p.k + threadIdx.x; i < end; i += blockDim.x) {
        const int e = p.experts[i];
        if ((unsigned)e < (unsigned)p.E) atomicAdd(count + e, 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.counts[blockIdx.x * p.E + e] = count[e];
}

// Every warp counts its copies per expert, the counts are summed over the warps of a block in its shared memory and
// over the blocks, and a second walk over the same copies hands out the rows in order.  No atomics decide an order, so
// it is that of the copies, and nothing is left behind between calls.
//   one cluster (SPREAD = false): the blocks exchange their counts through distributed shared memory.  One launch, no
//     scratch; L: the warps choose their tokens' experts first, in that layout (few tokens: router and plan in one);
//   spread: plan_blocks(E) blocks on as many SMs, whose counts plan_count_kernel has left in memory.
// 131072 copies, 64 experts: 23.9 us in a cluster of 8 (what bounds it is the scattered stores and the votes of eight
// SMs), 8.6 us spread over 128 blocks, the counting included; 16384 copies: 6.3 and 7.1 us.
template <typename L, bool SPREAD>
__global__ void __launch_bounds__(PLAN_WARPS * 32, 1) plan_kernel(const PlanArgs p, const RouteArgs a) {
    extern __shared__ uint32_t plan_smem[];
    uint32_t* hist = plan_smem;                         // [PLAN_WARPS][E]
    uint32_t* total = hist + PLAN_WARPS * p.E;          // [E] copies of this block; spread: of all blocks
    uint32_t* base = total + p.E;                       // [E] first row of this block's copies
    int* shift = reinterpret_cast<int*>(base + p.E);    // [E] slot - row of the expert
    __shared__ uint32_t warp_total[3][PLAN_WARPS];
    __shared__ uint32_t live_rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = SPREAD ? blockIdx.x : cluster_ctarank(), ctas = SPREAD ? gridDim.x : cluster_size();
    int fewest = (31 + p.k) / p.k;
    if constexpr (!std::is_void_v<L>) fewest = max(fewest, L::PER_WARP);
    const TokenRange own_tokens = warp_tokens(block_tokens(p.T, ctas, rank), fewest, warp);
    const int begin = own_tokens.begin * p.k, end = own_tokens.end * p.k;    // (T * k <= MOE_MOST: checked by the caller)

    for (int i = threadIdx.x; i < (PLAN_WARPS + 2) * p.E; i += blockDim.x) hist[i] = 0;
    pdl_wait();
    pdl_launch();
    if constexpr (!std::is_void_v<L>) {
        for (int t = own_tokens.begin; t < own_tokens.end; t += L::PER_WARP) {
            const int tg = t + lane / L::G;
            route_token<L>(a, tg < own_tokens.end ? tg : a.T, lane % L::G);
        }
    }
    __syncthreads();
    if (SPREAD) {
        // total: all blocks, base: the blocks before this one; the block's warps take a share of the blocks each
        const int wide = (p.E + 31) / 32 * 32, shares = PLAN_WARPS * 32 / wide;
        const int share = threadIdx.x / wide, e = threadIdx.x - share * wide;
        if (share < shares && e < p.E) {
            uint32_t all = 0, before = 0;
#pragma unroll 8
            for (uint32_t b = share; b < ctas; b += shares) {
                const uint32_t c = p.counts[b * p.E + e];
                all += c;
                before += b < rank ? c : 0;
            }
            atomicAdd(total + e, all);
            atomicAdd(base + e, before);
        }
    }
    uint32_t* own = hist + warp * p.E;
    const int bits = 32 - __clz(p.E);                   // keys 0 .. E
    // (eight loads in flight; a warp with no more copies than that has its ids still in registers for the second walk)
    int ids[PLAN_AHEAD];
    for (int i0 = begin; i0 < end; i0 += 32 * PLAN_AHEAD) {
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) ids[u] = i0 + 32 * u + lane < end ? p.experts[i0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) {
            if (i0 + 32 * u >= end) break;
            const int e = ids[u];
            const bool ok = (unsigned)e < (unsigned)p.E;
            const uint32_t same = same_key(ok ? e : p.E, bits);
            if (ok && lane == __ffs(same) - 1) own[e] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
        uint32_t run = 0;
#pragma unroll 8
        for (int w = 0; w < PLAN_WARPS; w++) {
            const uint32_t c = hist[w * p.E + e];
            hist[w * p.E + e] = run;
            run += c;
        }
        if (!SPREAD) total[e] = run;
    }
    // thread e: the expert's copies in all blocks, in the blocks before this one; then its first row and first tile
    // (MOE_MAX_EXPERTS = threads of the block)
    uint32_t count = 0, before = 0;
    if (SPREAD) {
        if (threadIdx.x < p.E) { count = total[threadIdx.x]; before = base[threadIdx.x]; }
    } else if (ctas == 1) {
        if (threadIdx.x < p.E) count = total[threadIdx.x];
    } else {
        cluster_sync_all();
        if (threadIdx.x < p.E) {
            const uint32_t addr = smem_u32(total + threadIdx.x);
#pragma unroll 8
            for (uint32_t r = 0; r < ctas; r++) {
                const uint32_t c = ld_cluster_u32(mapa_shared(addr, r));
                before += r < rank ? c : 0;
                count += c;
            }
        }
    }
    const uint32_t ntiles = (count + 127) / 128, nwide = (count + 255) / 256;
    uint32_t rows_to = count, tiles_to = ntiles, wide_to = nwide;    // inclusive sums over the warp's experts
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, rows_to, o), y = __shfl_up_sync(0xffffffffu, tiles_to, o),
                       z = __shfl_up_sync(0xffffffffu, wide_to, o);
        if (lane >= o) { rows_to += x; tiles_to += y; wide_to += z; }
    }
    if (lane == 31) { warp_total[0][warp] = rows_to; warp_total[1][warp] = tiles_to; warp_total[2][warp] = wide_to; }
    __syncthreads();
    // (PLAN_WARPS = lanes of a warp: the sums of the warps before this one)
    const bool earlier = lane < warp;
    const uint32_t row0 = rows_to - count + __reduce_add_sync(0xffffffffu, earlier ? warp_total[0][lane] : 0u);
    const uint32_t tile0 = tiles_to - ntiles + __reduce_add_sync(0xffffffffu, earlier ? warp_total[1][lane] : 0u);
    const uint32_t wide0 = wide_to - nwide + __reduce_add_sync(0xffffffffu, earlier ? warp_total[2][lane] : 0u);
    if (threadIdx.x < p.E) {
        base[threadIdx.x] = row0 + before;
        shift[threadIdx.x] = (int)(tile0 * 128u) - (int)row0;
        if (rank == 0) { p.offsets[threadIdx.x] = (int)row0; p.tiles[threadIdx.x] = (int)tile0; p.wide[threadIdx.x] = (int)wide0; }
        if (threadIdx.x == p.E - 1) {
            live_rows = row0 + count;
            if (rank == 0) {
                p.offsets[p.E] = (int)(row0 + count); p.tiles[p.E] = (int)(tile0 + ntiles); p.wide[p.E] = (int)(wide0 + nwide);
            }
        }
    }
    // also: no CTA of a cluster leaves while a peer may still read its counts
    if (SPREAD || ctas == 1) __syncthreads();
    else cluster_sync_all();
    const bool again = end - begin > 32 * PLAN_AHEAD;
    for (int i0 = begin; i0 < end; i0 += 32 * PLAN_AHEAD) {
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++)
            if (again) ids[u] = i0 + 32 * u + lane < end ? p.experts[i0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) {
            if (i0 + 32 * u >= end) break;
            const int i = i0 + 32 * u + lane, e = ids[u];
            const bool ok = (unsigned)e < (unsigned)p.E;
            const uint32_t same = same_key(ok ? e : p.E, bits);
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
    }
    const int n = p.T * p.k;
    for (long long i = (long long)live_rows + rank * blockDim.x + threadIdx.x; i < n; i += (long long)ctas * blockDim.x) p.source[i] = -1;
}

template <typename L, bool SPREAD>
int launch_plan(const PlanArgs& p, const RouteArgs& a, int ctas, cudaStream_t st) {
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64) return NVFP4_ERR_UNSUPPORTED;
    constexpr size_t most = (size_t)(PLAN_WARPS + 3) * MOE_MAX_EXPERTS * 4;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(plan_kernel<L, SPREAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) return (int)e;
        configured[dev] = true;
    }
    return launch_dependent(plan_kernel<L, SPREAD>, ctas, PLAN_WARPS * 32, (size_t)(PLAN_WARPS + 3) * p.E * 4, SPREAD ? 0 : ctas, st, p, a);
}

// The plan of choices that are in memory.  In a cluster: one CTA or the eight that every device can place (64 experts, one
// against eight: 512 copies 3.1 / 3.7 us, 1024 4.0 / 3.7, 8192 12.7 / 5.0).
int plan_choices(const PlanArgs& p, cudaStream_t st) {
    const long long copies = (long long)p.T * p.k;
    if (copies > PLAN_CLUSTER_MOST) {
        int rc = launch_dependent(plan_count_kernel, plan_blocks(p.E), PLAN_WARPS * 32, 0, 0, st, p);
        return rc ? rc : launch_plan<void, true>(p, RouteArgs{}, plan_blocks(p.E), st);
    }
    return launch_plan<void, false>(p, RouteArgs{}, copies <= 512 ? 1 : 8, st);
}

// Blocks of eight warps for `a.T` tokens, at most eight on an SM.
template <typename L>
int token_blocks(const RouteArgs& a, int dev) {
    const int blocks = (a.T + 8 * L::PER_WARP - 1) / (8 * L::PER_WARP);
    return blocks < 8 * sm_count(dev) ? blocks : 8 * sm_count(dev);
}

template <typename L>
int launch_route(const RouteArgs& a, const PlanArgs& p, int dev, cudaStream_t st) {
    // few tokens: the sorting cluster chooses the experts itself (one launch against two: 1 x 128 bf16 6.4 / 6.9 us, 128 x
    // 128 7.3 / 8.5, 512 x 64 7.7 / 8.7; not where a lane holds sixteen unpacked entries, which the 64 registers of its 1024
    // threads do not: 32 x 256 fp32 12.0 / 8.4).  The choice is bound by instruction issue, so the CTAs take four warps'
    // tokens each as long as there are CTAs
    if constexpr (L::PACKED ? L::NV <= 16 : L::NV <= 8) {
        if (a.T <= 512) {
            int c = 1;
            while (c < 8 && a.T > 4 * L::PER_WARP * c) c *= 2;
            return launch_plan<L, false>(p, a, c, st);
        }
    }
    const int rc = launch_dependent(route_kernel<L>, token_blocks<L>(a, dev), 256, 0, 0, st, a);
    return rc ? rc : plan_choices(p, st);
}

// f(layout) for the element type and the number of experts
template <int KIND, typename F>
int by_width(int E, F&& f) {
    if (E <= 64) return f(Layout<KIND, 8, 8>());
    if (E <= 128) return f(Layout<KIND, 8, 16>());
    if (E <= 256) return f(Layout<KIND, 16, 16>());
    if (E <= 512) return f(Layout<KIND, 32, 16>());
    return f(Layout<KIND, 32, 32>());
}
template <typename F>
int by_kind(int kind, int E, F&& f) {
    if (kind == NVFP4_F32) return by_width<NVFP4_F32>(E, f);
    if (kind == NVFP4_F16) return by_width<NVFP4_F16>(E, f);
    return by_width<NVFP4_BF16>(E, f);
}
// Whether every row of the logits starts on a 16-byte boundary.
int rows_wide(const void* logits, int kind, long long ld) { return ((uintptr_t)logits | (unsigned long long)(ld * elem_bytes(kind))) % 16 == 0; }

int check_route(int kind, long long ld, int T, int E, int k) {
    if (!kind_ok(kind)) return NVFP4_ERR_UNSUPPORTED;
    if (T <= 0 || E <= 0 || k <= 0 || k > E || ld < 0) return NVFP4_ERR_SHAPE;
    if (E > MOE_MAX_EXPERTS || k > MOE_MAX_CHOICES || (long long)T * k > MOE_MOST) return NVFP4_ERR_UNSUPPORTED;
    return NVFP4_OK;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" long long nvfp4_moe_plan_scratch(int T, int E, int k) {
    return T > 0 && E > 0 && k > 0 && (long long)T * k > PLAN_CLUSTER_MOST ? 4ll * plan_blocks(E) * E : 0;
}

extern "C" int nvfp4_moe_plan(const void* experts, int T, int E, int k, void* offsets, void* tiles, void* wide_tiles, void* rows,
                              void* slots, void* source, void* scratch, void* stream) {
    if (!experts || !offsets || !tiles || !wide_tiles || !rows || !slots || !source) return NVFP4_ERR_NULL;
    if (T <= 0 || E <= 0 || k <= 0) return NVFP4_ERR_SHAPE;
    if (E > MOE_MAX_EXPERTS || k > MOE_MAX_CHOICES || (long long)T * k > MOE_MOST) return NVFP4_ERR_UNSUPPORTED;
    if (nvfp4_moe_plan_scratch(T, E, k) && !scratch) return NVFP4_ERR_NULL;
    if (!words(experts, offsets, tiles, wide_tiles, rows, slots, source, scratch)) return NVFP4_ERR_ALIGN;
    const PlanArgs p{(const int*)experts, (int*)offsets, (int*)tiles, (int*)wide_tiles, (int*)rows, (int*)slots, (int*)source, (uint32_t*)scratch, T, E, k};
    return plan_choices(p, (cudaStream_t)stream);
}

extern "C" int nvfp4_moe_route(const void* logits, int kind, long long ld, const void* mask, int T, int E, int k, int renormalize,
                               void* weights, void* experts, void* offsets, void* tiles, void* wide_tiles, void* rows, void* slots,
                               void* source, void* scratch, void* stream) {
    if (!logits || !weights || !experts || !offsets || !tiles || !wide_tiles || !rows || !slots || !source) return NVFP4_ERR_NULL;
    int rc = check_route(kind, ld, T, E, k);
    if (rc) return rc;
    if ((uintptr_t)logits % elem_bytes(kind) || !words(weights, experts, offsets, tiles, wide_tiles, rows, slots, source, scratch))
        return NVFP4_ERR_ALIGN;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    const RouteArgs a{logits, ld, (const uint8_t*)mask, (float*)weights, (int*)experts, T, E, k, renormalize,
                      rows_wide(logits, kind, ld)};
    if (nvfp4_moe_plan_scratch(T, E, k) && !scratch) return NVFP4_ERR_NULL;
    const PlanArgs p{(const int*)experts, (int*)offsets, (int*)tiles, (int*)wide_tiles, (int*)rows, (int*)slots, (int*)source, (uint32_t*)scratch, T, E, k};
    return by_kind(kind, E, [&](auto layout) { return launch_route<decltype(layout)>(a, p, dev, (cudaStream_t)stream); });
}

extern "C" int nvfp4_moe_route_backward(const void* dweights, const void* logits, int kind, long long ld, const void* weights,
                                        const void* experts, int T, int E, int k, int renormalize, void* dlogits, void* stream) {
    if (!dweights || !logits || !weights || !experts || !dlogits) return NVFP4_ERR_NULL;
    if ((uintptr_t)dlogits & 15) return NVFP4_ERR_ALIGN;
    int rc = check_route(kind, ld, T, E, k);
    if (rc) return rc;
    if ((uintptr_t)logits % elem_bytes(kind) || !words(dweights, weights, experts)) return NVFP4_ERR_ALIGN;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    const RouteArgs a{logits, ld, nullptr, (float*)const_cast<void*>(weights), (int*)const_cast<void*>(experts), T, E, k, renormalize,
                      rows_wide(logits, kind, ld)};
    return by_kind(kind, E, [&](auto layout) {
        using L = decltype(layout);
        return launch_dependent(route_backward_kernel<L>, token_blocks<L>(a, dev), 256, 0, 0, (cudaStream_t)stream, a,
                                (const float*)dweights, dlogits);
    });
}
