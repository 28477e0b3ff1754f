// Tokens sorted by expert and back: dispatch (plain and quantised to NVFP4), combine with the router's weights, and the
// gradients of both.  Row r of a sorted buffer belongs to copy source[r]; rows[t][j] is the row of token t's choice j.
//
//   dispatch          xs[rows[t][j]] = x[t]                        gradient: combine without weights
//   combine           out[t] = sum_j w_tj * y[rows[t][j]]          (fp32, j ascending, one rounding)
//   combine gradient  dy[rows[t][j]] = w_tj * dout[t],  dw_tj = <dout[t], y[rows[t][j]]>
//
// Everything is organised by token, so a token's row is read once however many experts it goes to (and quantised
// once); the sorted rows are contiguous, so both sides move whole sectors.  With many tokens dispatch, combine and their
// gradients are HBM-bound (16384 x 8 x 4096 bf16: 0.9 to 1.0 of the copy rate); the quantising dispatch is held up by its
// scales (4096 x 8 x 4096: 28 us for 17 us of bytes at 24 % of DRAM throughput, see dispatch_quant_kernel).
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "moe_common.cuh"
#include "quant_block.cuh"

namespace nvfp4 {
namespace {

struct PermuteArgs {
    const int* rows;       // [T][k]
    const int* live;       // offsets + E: number of rows in use
    int T, k;
    int H;                 // elements of a row
};

// Zeros the rows of a sorted buffer behind the last copy, so that sums over the whole buffer are sums over copies.
// `row` in vectors of V; nothing to do unless choices were dropped.
template <typename V>
__device__ __forceinline__ void zero_tail(V* out, long long row, const PermuteArgs& p) {
    const long long first = (long long)*p.live * row, end = (long long)p.T * p.k * row;
    V zero = {};
    for (long long i = first + (long long)blockIdx.x * blockDim.x + threadIdx.x; i < end; i += (long long)gridDim.x * blockDim.x)
        out[i] = zero;
}

// What one warp does at a time: `U * 32` vectors of one token's row.  Lane j holds the row of the token's choice j (-1:
// none) and its weight; both are fetched one piece ahead, so that their latency does not stand in front of the rows'.
// (Fewer than 2^31 pieces: checked by the caller.)
template <int U, bool WEIGHTED>
struct Pieces {
    const int* rows;               // [T][k]
    const float* weights;          // [T][k]
    unsigned k, row_vecs, segs, n, step, i;
    unsigned t, c;                 // this warp's token and this lane's first vector of the piece
    unsigned next_t, next_seg;
    int row, next_row;
    float w, next_w;

    __device__ __forceinline__ Pieces(const PermuteArgs& p, const float* weights_, int row_vecs_)
        : rows(p.rows), weights(weights_), k(p.k), row_vecs(row_vecs_), segs((row_vecs_ + 32 * U - 1) / (32 * U)) {
        n = (unsigned)p.T * segs;
        step = gridDim.x * (blockDim.x >> 5);
        i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
        fetch(i);
        locate();
    }
    __device__ __forceinline__ void fetch(unsigned at) {
        const unsigned lane = threadIdx.x & 31;
        next_t = at / segs;
        next_seg = at - next_t * segs;
        next_row = -1;
        next_w = 0.f;
        if (at < n && lane < k) {
            const size_t copy = (size_t)next_t * k + lane;
            next_row = rows[copy];
            if (WEIGHTED) next_w = weights[copy];
        }
    }
    __device__ __forceinline__ void locate() {
        t = next_t;
        c = next_seg * (32 * U) + (threadIdx.x & 31);
        row = next_row;
        w = next_row >= 0 ? next_w : 0.f;       // (a choice that is not routed may have any weight)
        fetch(i + step);
    }
    __device__ __forceinline__ bool more() const { return i < n; }
    __device__ __forceinline__ void next() { i += step; locate(); }
};

// One load of a token's vector, k stores.
template <int BYTES, int U>
__global__ void __launch_bounds__(256) dispatch_kernel(const uint8_t* x, long long ld, void* xs, int row_vecs, const PermuteArgs p) {
    using V = typename Bits<BYTES>::type;
    pdl_wait();
    pdl_launch();
    V* out = reinterpret_cast<V*>(xs);
    for (Pieces<U, false> w(p, nullptr, row_vecs); w.more(); w.next()) {
        const V* src = reinterpret_cast<const V*>(x + w.t * ld);
        V v[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (w.c + 32 * u < row_vecs) v[u] = src[w.c + 32 * u];
        for (int j = 0; j < p.k; j++) {
            const int row = __shfl_sync(0xffffffffu, w.row, j);
            if (row < 0) continue;
            V* dst = out + (long long)row * row_vecs + w.c;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (w.c + 32 * u < row_vecs) dst[32 * u] = v[u];
        }
    }
    zero_tail(out, row_vecs, p);
}

// KU rows' loads of U vectors each are in flight at a time.  `pitch`: bytes between rows of y, in 64 bits only where it
// has more than 32 (with 64 throughout the gradient keeps two pointers per row in registers: 8192 x 8 x 4002 fp16 297 us
// against 221).  (Loads past L1 are faster
// for few rows, 4096 x 2 x 2048 fp32 14.7 against 19.3 us, 8192 x 4 x 4096 bf16 54.6 / 56.3, and slower for eight, whose
// loads the compiler then cannot place among the sums: 16384 x 8 x 4096 197 / 180.)
template <typename TI, typename TO, int VN, int KU, int U, bool WEIGHTED, typename PITCH>
__global__ void __launch_bounds__(256, U >= 2 && VN > 1 ? 3 : 4) combine_kernel(const TI* y, PITCH pitch, const float* weights, TO* out,
                                                                      int row_vecs, const PermuteArgs p) {
    pdl_wait();
    pdl_launch();
    for (Pieces<U, WEIGHTED> w(p, weights, row_vecs); w.more(); w.next()) {
        float acc[U][VN] = {};
        const char* at = reinterpret_cast<const char*>(y + (size_t)w.c * VN);
        for (int j0 = 0; j0 < p.k; j0 += KU) {
            Vec<TI, VN> v[KU][U] = {};
#pragma unroll
            for (int j = 0; j < KU; j++) {
                const int row = __shfl_sync(0xffffffffu, w.row, j0 + j);     // (-1 from the k-th lane on)
                const TI* src = reinterpret_cast<const TI*>(at + (unsigned long long)(unsigned)row * pitch);
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (row >= 0 && w.c + 32 * u < row_vecs) v[j][u].template load<(KU < 8)>(src + 32 * u * VN);
            }
#pragma unroll
            for (int j = 0; j < KU; j++) {
                const float wj = WEIGHTED ? __shfl_sync(0xffffffffu, w.w, j0 + j) : 1.0f;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int q = 0; q < VN; q++) acc[u][q] = fmaf(wj, v[j][u].get(q), acc[u][q]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (w.c + 32 * u >= row_vecs) break;
            Vec<TO, VN> o;
            o.set(acc[u]);
            o.store(out + (size_t)w.t * p.H + (size_t)(w.c + 32 * u) * VN);
        }
    }
}

// GROUP threads per token (a warp, or a block for long rows): a vector of dout[t] is read once for KU of the token's
// rows; their dot products stay in registers and are summed over the group at the end, in an order that follows from the
// sizes, the types, the alignment of addresses and pitches and the number of SMs (they choose the vectors and the group).
// `pitch`: bytes between rows of y.
template <typename TI, typename TO, int VN, int GROUP, int KU, int U, typename PITCH>
__global__ void __launch_bounds__(256, 3) combine_backward_kernel(const TO* dout, long long ldo, const TI* y, PITCH pitch,
                                                                  const float* weights, TI* dy, float* dw, int row_vecs,
                                                                  const PermuteArgs p) {
    __shared__ float part[8][KU];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_group = threadIdx.x % GROUP;
    constexpr int PER_BLOCK = 256 / GROUP;
    pdl_wait();
    pdl_launch();
    const PITCH out_pitch = (PITCH)p.H * (PITCH)sizeof(TI);
    for (long long t = (long long)blockIdx.x * PER_BLOCK + threadIdx.x / GROUP; t < p.T; t += (long long)gridDim.x * PER_BLOCK) {
        const TO* d = dout + t * ldo;
        for (int j0 = 0; j0 < p.k; j0 += KU) {
            int row[KU];
            float w[KU], acc[KU];
#pragma unroll
            for (int j = 0; j < KU; j++) {
                row[j] = j0 + j < p.k ? p.rows[t * p.k + j0 + j] : -1;
                w[j] = row[j] >= 0 ? weights[t * p.k + j0 + j] : 0.f;
                acc[j] = 0.f;
            }
            for (int c = in_group; c < row_vecs; c += GROUP * U) {
                Vec<TO, VN> dv[U] = {};
                Vec<TI, VN> v[KU][U] = {};
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (c + GROUP * u < row_vecs) dv[u].load(d + (size_t)(c + GROUP * u) * VN);
#pragma unroll
                for (int j = 0; j < KU; j++) {
                    const TI* src = reinterpret_cast<const TI*>(reinterpret_cast<const char*>(y) + (unsigned long long)(unsigned)row[j] * pitch) + (size_t)c * VN;
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (row[j] >= 0 && c + GROUP * u < row_vecs) v[j][u].load(src + GROUP * u * VN);
                }
#pragma unroll
                for (int j = 0; j < KU; j++) {
                    TI* dst = reinterpret_cast<TI*>(reinterpret_cast<char*>(dy) + (unsigned long long)(unsigned)row[j] * out_pitch) + (size_t)c * VN;
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        float f[VN];
#pragma unroll
                        for (int q = 0; q < VN; q++) {
                            const float g = dv[u].get(q);
                            acc[j] = fmaf(g, v[j][u].get(q), acc[j]);
                            f[q] = w[j] * g;
                        }
                        Vec<TI, VN> o;
                        o.set(f);
                        if (row[j] >= 0 && c + GROUP * u < row_vecs) o.store(dst + GROUP * u * VN);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < KU; j++) {
                if (row[j] < 0) acc[j] = 0.f;             // (dout may hold infinities: they met the zeros of no row)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
            }
            if constexpr (GROUP > 32) {
                if (lane == 0) {
#pragma unroll
                    for (int j = 0; j < KU; j++) part[warp][j] = acc[j];
                }
                __syncthreads();
                if (threadIdx.x < KU && j0 + threadIdx.x < p.k) {
                    float s = 0.f;
#pragma unroll
                    for (int q = 0; q < 8; q++) s += part[q][threadIdx.x];
                    dw[t * p.k + j0 + threadIdx.x] = s;
                }
                __syncthreads();
            } else {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < KU; j++)
                    if (lane == j) s = acc[j];
                if (lane < KU && j0 + lane < p.k) dw[t * p.k + j0 + lane] = s;
            }
        }
    }
    zero_tail(reinterpret_cast<typename Bits<VN * sizeof(TI)>::type*>(dy), row_vecs, p);
}

// One thread per 32 elements of a token: quantised once, their codes (16 bytes) stored for each of the token's rows.
// The scale atoms follow the experts' 128-row tiles: slots[t][j] is the row with every expert padded to whole tiles.
// TABLE = false: the scale bytes are stored for each row, too; two neighbouring lanes hold the four k-blocks of one
// 4-byte group of an atom (K % 64 == 0).  TABLE = true: they go to a row of `table` per token, from where
// gather_scales_kernel makes whole atoms: 4-byte stores 512 bytes apart took as long as everything else together
// (16384 tokens x 8 x 4096: 130 us, 90 us with the table).
template <int KIND, bool TABLE>
__global__ void __launch_bounds__(256) dispatch_quant_kernel(const void* x, long long ld, const int* slots, uint8_t* codes,
                                                             uint8_t* scales, const PermuteArgs p) {
    using T = typename ElemOf<KIND>::type;
    pdl_wait();
    pdl_launch();
    const unsigned units = p.H / 32, lane = threadIdx.x & 31;
    const unsigned n = (unsigned)p.T * units, step = gridDim.x * blockDim.x;    // (fewer than 2^31: checked by the caller)
    for (unsigned i = blockIdx.x * blockDim.x + threadIdx.x; i - lane < n; i += step) {
        const bool in = i < n;
        const unsigned t = in ? i / units : 0, c = in ? i - t * units : 0;
        float xs[32];
        constexpr int VN = 16 / (int)sizeof(T);
        const T* src = reinterpret_cast<const T*>(x) + t * ld + (size_t)c * 32;
#pragma unroll
        for (int v = 0; v < 32 / VN; v++) {
            Vec<T, VN> a;
            a.load(src + v * VN);
#pragma unroll
            for (int q = 0; q < VN; q++) xs[v * VN + q] = a.get(q);
        }
        uint4 w;
        uint32_t s = quantize_block16(xs, w.x, w.y);
        s |= quantize_block16(xs + 16, w.z, w.w) << 8;
        if (TABLE) {
            if (in) reinterpret_cast<uint16_t*>(scales)[i] = (uint16_t)s;
        } else {
            s |= __shfl_down_sync(0xffffffffu, s, 1) << 16;   // (n is even: the two lanes of a group are in range together)
        }
        if (!in) continue;
        const int* rows = p.rows + (size_t)t * p.k;
        const int* at = slots + (size_t)t * p.k;
        uint8_t* dst = codes + (size_t)c * 16;
        for (int j0 = 0; j0 < p.k; j0 += 4) {
            int row[4], slot[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                row[j] = j0 + j < p.k ? rows[j0 + j] : -1;
                slot[j] = !TABLE && j0 + j < p.k ? at[j0 + j] : 0;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (row[j] < 0) continue;
                *reinterpret_cast<uint4*>(dst + (long long)row[j] * units * 16) = w;
                if (!TABLE && (lane & 1) == 0) {
                    const long long atom = (long long)(slot[j] >> 7) * (units / 2) + c / 2;
                    *reinterpret_cast<uint32_t*>(scales + atom * 512 + (slot[j] & 31) * 16 + ((slot[j] & 127) >> 5) * 4) = s;
                }
            }
        }
    }
    zero_tail(reinterpret_cast<uint4*>(codes), units, p);
}

// The scale atoms of one 128-row tile from the tokens' scale rows: a warp makes four atoms (256 elements of K) at a time,
// lane i the 16 bytes of the rows i, i + 32, i + 64, i + 96 in each.  Rows that do not exist get zeros.
__global__ void __launch_bounds__(256) gather_scales_kernel(const uint8_t* table, const int* source, const int* offsets,
                                                            const int* tiles, uint8_t* sf_sw, int E, int k, int K) {
    __shared__ int expert;
    pdl_wait();
    pdl_launch();
    const int tile = blockIdx.x;
    if (tile >= tiles[E]) return;
    for (int e = threadIdx.x; e < E; e += blockDim.x)
        if (tiles[e] <= tile && tile < tiles[e + 1]) expert = e;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = offsets[expert] + (tile - tiles[expert]) * 128, end = offsets[expert + 1];
    long long token[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int row = row0 + q * 32 + lane;
        token[q] = row < end ? source[row] / k : -1;
    }
    const int chunks = K / 256;
    for (int c = blockIdx.y * 8 + warp; c < chunks; c += gridDim.y * 8) {
        uint4 w[4];
#pragma unroll
        for (int q = 0; q < 4; q++)
            w[q] = token[q] >= 0 ? reinterpret_cast<const uint4*>(table + token[q] * (K / 16))[c] : make_uint4(0u, 0u, 0u, 0u);
        uint4* dst = reinterpret_cast<uint4*>(sf_sw + ((long long)tile * (K / 64) + c * 4) * 512) + lane;
        dst[0] = make_uint4(w[0].x, w[1].x, w[2].x, w[3].x);
        dst[32] = make_uint4(w[0].y, w[1].y, w[2].y, w[3].y);
        dst[64] = make_uint4(w[0].z, w[1].z, w[2].z, w[3].z);
        dst[96] = make_uint4(w[0].w, w[1].w, w[2].w, w[3].w);
    }
}

// Blocks of a grid-stride launch over n threads: at most eight resident blocks per SM.
int grid_for(long long n, int dev) {
    long long blocks = (n + 255) / 256;
    const long long cap = 8ll * sm_count(dev);
    return (int)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}

int current_device(int* dev) {
    const cudaError_t e = cudaGetDevice(dev);
    if (e != cudaSuccess) return (int)e;
    return *dev < 64 ? NVFP4_OK : NVFP4_ERR_UNSUPPORTED;
}

int check_sizes(int T, int k, int H, long long ld) {
    if (T <= 0 || k <= 0 || H <= 0 || ld < 0) return NVFP4_ERR_SHAPE;
    if (k > MOE_MAX_CHOICES || (long long)T * k > MOE_MOST || H > MOE_MOST) return NVFP4_ERR_UNSUPPORTED;
    return NVFP4_OK;
}

// Largest power of two, at most `most`, that divides every address and pitch.
int common_alignment(int most, std::initializer_list<unsigned long long> values) {
    unsigned long long all = (unsigned long long)most;
    for (unsigned long long v : values) all |= v;
    return (int)(all & (~all + 1));
}

template <typename F>
int by_type(int kind, F&& f) {
    if (kind == NVFP4_F32) return f(float());
    if (kind == NVFP4_F16) return f(__half());
    return f(__nv_bfloat16());
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_moe_dispatch(const void* x, int kind, long long ld, const void* rows, const void* offsets, int T, int E, int k,
                                  int H, void* xs, void* stream) {
    if (!x || !rows || !offsets || !xs) return NVFP4_ERR_NULL;
    if (!kind_ok(kind)) return NVFP4_ERR_UNSUPPORTED;
    int rc = check_sizes(T, k, H, ld);
    if (rc) return rc;
    if (E <= 0) return NVFP4_ERR_SHAPE;
    const int size = elem_bytes(kind);
    const long long row_bytes = (long long)H * size;
    const int vec = common_alignment(16, {(uintptr_t)x, (uintptr_t)xs, (unsigned long long)(ld * size), (unsigned long long)row_bytes});
    if (vec < size || !words(rows, offsets)) return NVFP4_ERR_ALIGN;
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    const PermuteArgs p{(const int*)rows, (const int*)offsets + E, T, k, H};
    const int row_vecs = (int)(row_bytes / vec);
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto bytes, auto u) {
        constexpr int B = decltype(bytes)::value, U = decltype(u)::value;
        const long long warps = (long long)T * ((row_vecs + 32 * U - 1) / (32 * U));
        if (warps >= (1ll << 31)) return (int)NVFP4_ERR_UNSUPPORTED;
        return launch_dependent(dispatch_kernel<B, U>, grid_for(32 * warps, dev), 256, 0, 0, st, (const uint8_t*)x, ld * size, xs, row_vecs, p);
    };
    auto go_bytes = [&](auto bytes) {
        // one vector per lane while that fills the SMs at most once, else four (bf16, one against four: 8 x 8 x 7168 2.0 /
        // 3.5 us, 256 x 8 x 4096 3.8 / 4.1, 16384 x 8 x 4096 220 / 204)
        const bool one = (long long)T * ((row_vecs + 31) / 32) <= 32ll * sm_count(dev);
        return one ? go(bytes, std::integral_constant<int, 1>()) : go(bytes, std::integral_constant<int, 4>());
    };
    switch (vec) {
        case 16: return go_bytes(std::integral_constant<int, 16>());
        case 8: return go_bytes(std::integral_constant<int, 8>());
        case 4: return go_bytes(std::integral_constant<int, 4>());
        default: return go_bytes(std::integral_constant<int, 2>());
    }
}

extern "C" int nvfp4_moe_combine(const void* y, int kind, long long ld, const void* weights, const void* rows, int T, int k, int H,
                                 void* out, int out_kind, void* stream) {
    if (!y || !rows || !out) return NVFP4_ERR_NULL;
    if (!kind_ok(kind) || !kind_ok(out_kind)) return NVFP4_ERR_UNSUPPORTED;
    int rc = check_sizes(T, k, H, ld);
    if (rc) return rc;
    if ((uintptr_t)y % elem_bytes(kind) || (uintptr_t)out % elem_bytes(out_kind) || !words(weights, rows)) return NVFP4_ERR_ALIGN;
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    const bool far = ld * elem_bytes(kind) >= (1ll << 32);       // rows that only a pitch of 64 bits reaches
    const PermuteArgs p{(const int*)rows, nullptr, T, k, H};
    cudaStream_t st = (cudaStream_t)stream;
    return by_type(kind, [&](auto ti) {
        return by_type(out_kind, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            // vectors of 16 input bytes where both sides are aligned to theirs, else 16-bit elements in pairs, else one by one
            constexpr int VN = 16 / sizeof(TI);
            constexpr unsigned long long O = VN * sizeof(TO) < 16 ? VN * sizeof(TO) : 16;
            const bool wide = H % VN == 0 && ld % VN == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)out % O == 0;
            const bool pair = sizeof(TI) == 2 && !wide && !far && H % 2 == 0 && ld % 2 == 0 && (uintptr_t)y % 4 == 0 && (uintptr_t)out % (2 * sizeof(TO)) == 0;
            const int row_vecs = wide ? H / VN : pair ? H / 2 : H;
            auto go = [&](auto vn, auto ku, auto u, auto pitch) {
                using P = decltype(pitch);
                constexpr int N = decltype(vn)::value, KU = decltype(ku)::value, U = decltype(u)::value;
                const long long warps = (long long)T * ((row_vecs + 32 * U - 1) / (32 * U));
                if (warps >= (1ll << 31)) return (int)NVFP4_ERR_UNSUPPORTED;
                const int grid = grid_for(32 * warps, dev);
                return launch_dependent(weights ? combine_kernel<TI, TO, N, KU, U, true, P> : combine_kernel<TI, TO, N, KU, U, false, P>,
                                        grid, 256, 0, 0, st, (const TI*)y, pitch, (const float*)weights, (TO*)out, row_vecs, p);
            };
            using std::integral_constant;
            auto go_width = [&](auto vn) {
                // as many loads in flight for few choices as for eight (bf16, 512 x 2 x 2048: 2.0 us, 3.2 with one vector
                // of eight rows, 128 x 4 x 4096: 1.9 / 2.4; of two rows, fp32 4096 x 2 x 2048 17.3 us with four vectors,
                // 19.0 with two), and more where a vector is one or two elements (8192 x 8 x 4002 fp16, one, two, four
                // vectors of eight rows: 192, 159, 297 us; 4001 wide 332, 275, 314)
                constexpr int N = decltype(vn)::value;
                const unsigned pitch = (unsigned)(ld * sizeof(TI));
                const auto two = integral_constant<int, 2>();
                const auto of_two = integral_constant<int, N == 8 ? 2 : 4>();
                if constexpr (N != 2) {
                    if (far) return go(vn, two, of_two, (unsigned long long)ld * sizeof(TI));
                }
                if (k <= 2) return go(vn, two, of_two, pitch);
                if (k <= 4) return go(vn, integral_constant<int, 4>(), two, pitch);
                return go(vn, integral_constant<int, 8>(), integral_constant<int, N <= 2 ? 2 : 1>(), pitch);
            };
            if constexpr (sizeof(TI) == 2) {
                if (pair) return go_width(integral_constant<int, 2>());
            }
            return wide ? go_width(integral_constant<int, VN>()) : go_width(integral_constant<int, 1>());
        });
    });
}

extern "C" int nvfp4_moe_combine_backward(const void* dout, int out_kind, long long ldo, const void* y, int kind, long long ld,
                                          const void* weights, const void* rows, const void* offsets, int T, int E, int k, int H,
                                          void* dy, void* dweights, void* stream) {
    if (!dout || !y || !weights || !rows || !offsets || !dy || !dweights) return NVFP4_ERR_NULL;
    if (!kind_ok(kind) || !kind_ok(out_kind)) return NVFP4_ERR_UNSUPPORTED;
    int rc = check_sizes(T, k, H, ld);
    if (rc) return rc;
    if (E <= 0 || ldo < 0) return NVFP4_ERR_SHAPE;
    if ((uintptr_t)y % elem_bytes(kind) || (uintptr_t)dy % elem_bytes(kind) || (uintptr_t)dout % elem_bytes(out_kind) ||
        !words(weights, rows, offsets, dweights))
        return NVFP4_ERR_ALIGN;
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    const bool far = ld * elem_bytes(kind) >= (1ll << 32) || (long long)H * elem_bytes(kind) >= (1ll << 32);
    const PermuteArgs p{(const int*)rows, (const int*)offsets + E, T, k, H};
    cudaStream_t st = (cudaStream_t)stream;
    return by_type(kind, [&](auto ti) {
        return by_type(out_kind, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            constexpr int VN = 16 / sizeof(TI);
            constexpr unsigned long long O = VN * sizeof(TO) < 16 ? VN * sizeof(TO) : 16;
            const bool wide = H % VN == 0 && ld % VN == 0 && ldo % VN == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)dy % 16 == 0 &&
                              (uintptr_t)dout % O == 0;
            const bool pair = sizeof(TI) == 2 && !wide && !far && H % 2 == 0 && ld % 2 == 0 && ldo % 2 == 0 && (uintptr_t)y % 4 == 0 &&
                              (uintptr_t)dy % 4 == 0 && (uintptr_t)dout % (2 * sizeof(TO)) == 0;
            const int row_vecs = wide ? H / VN : pair ? H / 2 : H;
            // a warp per token where its lanes take at most four vectors each, and for few choices where there are tokens
            // enough for that (bf16, 4096 wide, a warp against a block: 16384 x 1 65 against 86 us, 8192 x 4 98 / 105; with
            // eight rows in registers a warp's loads no longer cover its stores: 16384 x 8 372 / 351)
            const bool warp = !far && (row_vecs <= 128 || (k <= 4 && T >= 16 * sm_count(dev)));
            const int grid = grid_for((long long)T * (warp ? 32 : 256), dev);
            auto go = [&](auto vn, auto group, auto ku, auto u, auto pitch) {
                return launch_dependent(
                    combine_backward_kernel<TI, TO, decltype(vn)::value, decltype(group)::value, decltype(ku)::value, decltype(u)::value,
                                            decltype(pitch)>,
                    grid, 256, 0, 0, st, (const TO*)dout, ldo, (const TI*)y, pitch, (const float*)weights, (TI*)dy, (float*)dweights,
                    row_vecs, p);
            };
            using std::integral_constant;
            auto go_group = [&](auto vn, auto group) {
                constexpr int N = decltype(vn)::value;
                const unsigned pitch = (unsigned)(ld * sizeof(TI));
                const auto two = integral_constant<int, 2>();
                const auto of_two = integral_constant<int, N <= 2 ? 8 : 2>();
                if constexpr (N != 2 && decltype(group)::value > 32) {
                    if (far) return go(vn, group, two, of_two, (unsigned long long)ld * sizeof(TI));
                }
                if (k <= 2) return go(vn, group, two, of_two, pitch);
                if (k <= 4) return go(vn, group, integral_constant<int, 4>(), integral_constant<int, N <= 2 ? 4 : 2>(), pitch);
                return go(vn, group, integral_constant<int, 8>(), integral_constant<int, N <= 2 ? 2 : 1>(), pitch);
            };
            auto go_width = [&](auto vn) {
                return warp ? go_group(vn, integral_constant<int, 32>()) : go_group(vn, integral_constant<int, 256>());
            };
            if constexpr (sizeof(TI) == 2) {
                if (pair) return go_width(integral_constant<int, 2>());
            }
            return wide ? go_width(integral_constant<int, VN>()) : go_width(integral_constant<int, 1>());
        });
    });
}

extern "C" long long nvfp4_moe_dispatch_scratch(int T, int k, int K) {
    // a second launch pays for many elements (bf16, without and with: 8192 x 2 x 4096 22 against 24.5 us, 8192 x 4 x 4096
    // 32 / 31, 4096 x 6 x 7168 38 / 36, 16384 x 8 x 4096 130 / 90)
    return T > 0 && k > 0 && K > 0 && K % 256 == 0 && (long long)T * k * K >= (160ll << 20) ? (long long)T * (K / 16) : 0;
}

extern "C" int nvfp4_moe_dispatch_nvfp4(const void* x, int kind, long long ld, const void* offsets, const void* tiles,
                                        const void* rows, const void* slots, const void* source, int T, int E, int k, int K,
                                        void* packed, void* sf_sw, void* scratch, void* stream) {
    if (!x || !offsets || !tiles || !rows || !slots || !source || !packed || !sf_sw) return NVFP4_ERR_NULL;
    if (!kind_ok(kind)) return NVFP4_ERR_UNSUPPORTED;
    int rc = check_sizes(T, k, K, ld);
    if (rc) return rc;
    if (E <= 0) return NVFP4_ERR_SHAPE;
    if (K % 64 != 0) return NVFP4_ERR_K_MULTIPLE;
    if ((long long)T * (K / 32) >= (1ll << 31)) return NVFP4_ERR_UNSUPPORTED;
    const bool table = nvfp4_moe_dispatch_scratch(T, k, K) > 0;
    if (table && !scratch) return NVFP4_ERR_NULL;
    if (((uintptr_t)x & 15) || ld * elem_bytes(kind) % 16 || ((uintptr_t)packed & 15) || ((uintptr_t)sf_sw & 15) ||
        (table && ((uintptr_t)scratch & 15)) || !words(offsets, tiles, rows, slots, source))
        return NVFP4_ERR_ALIGN;
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    const PermuteArgs p{(const int*)rows, (const int*)offsets + E, T, k, K};
    const int grid = grid_for((long long)T * (K / 32), dev);
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto with_table) {
        constexpr bool TB = decltype(with_table)::value;
        auto kernel = kind == NVFP4_F32   ? dispatch_quant_kernel<NVFP4_F32, TB>
                      : kind == NVFP4_F16 ? dispatch_quant_kernel<NVFP4_F16, TB>
                                          : dispatch_quant_kernel<NVFP4_BF16, TB>;
        return launch_dependent(kernel, grid, 256, 0, 0, st, x, ld, (const int*)slots, (uint8_t*)packed, (uint8_t*)(TB ? scratch : sf_sw), p);
    };
    if (!table) return go(std::false_type());
    if ((rc = go(std::true_type()))) return rc;
    // blocks for the most tiles that the copies can fill; those without a tile end at once
    const long long copies = (long long)T * k, active = copies < E ? copies : E;
    const dim3 tiles_grid((unsigned)(active + (copies - active) / 128), (K / 256 + 7) / 8 < 4 ? (K / 256 + 7) / 8 : 4);
    return launch_dependent(gather_scales_kernel, tiles_grid, 256, 0, 0, st, (const uint8_t*)scratch, (const int*)source, (const int*)offsets,
                            (const int*)tiles, (uint8_t*)sf_sw, E, k, K);
}
