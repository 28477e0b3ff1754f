// Tokens sorted by expert and back: dispatch (plain and quantised to NVFP4), combine with the router's weights, and the
// gradients of both.  Row r of a sorted buffer belongs to copy source[r]; rows[t][j] is the row of token t's choice j.
//
//   dispatch          xs[rows[t][j]] = x[t]                        gradient: combine without weights
//   combine           out[t] = sum_j w_tj * y[rows[t][j]]          (fp32, j ascending, one rounding)
//   combine gradient  dy[rows[t][j]] = w_tj * dout[t],  dw_tj = <dout[t], y[rows[t][j]]>
//
// Everything is organised by token, so a token's row is read once however many experts it goes to (and quantised
// once); the sorted rows are contiguous, so both sides move whole sectors.  All of it is HBM-bound.
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

template <int BYTES> struct Bits;
template <> struct Bits<16> { using type = uint4; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<2> { using type = uint16_t; };

// One thread per vector of a token's row: one load, k stores.
template <int BYTES>
__global__ void __launch_bounds__(256) dispatch_kernel(const uint8_t* __restrict__ x, long long ld, void* __restrict__ xs,
                                                       int row_vecs, const PermuteArgs p) {
    using V = typename Bits<BYTES>::type;
    const long long n = (long long)p.T * row_vecs, step = (long long)gridDim.x * blockDim.x;
    V* out = reinterpret_cast<V*>(xs);
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const long long t = i / row_vecs;
        const int c = (int)(i - t * row_vecs);
        const V v = __ldg(reinterpret_cast<const V*>(x + t * ld) + c);
        const int* r = p.rows + t * p.k;
        for (int j = 0; j < p.k; j++) {
            const int row = __ldg(r + j);
            if (row >= 0) out[(long long)row * row_vecs + c] = v;
        }
    }
    zero_tail(out, row_vecs, p);
}

// One thread per vector of an output row: up to eight rows' loads in flight.
template <typename TI, typename TO, int VN>
__global__ void __launch_bounds__(256) combine_kernel(const TI* __restrict__ y, long long ld, const float* __restrict__ weights,
                                                      TO* __restrict__ out, int row_vecs, const PermuteArgs p) {
    const long long n = (long long)p.T * row_vecs, step = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const long long t = i / row_vecs;
        const int c = (int)(i - t * row_vecs);
        float acc[VN] = {};
        for (int j0 = 0; j0 < p.k; j0 += 8) {
            int row[8];
            float w[8];
            Vec<TI, VN> v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                row[j] = j0 + j < p.k ? __ldg(p.rows + t * p.k + j0 + j) : -1;
                w[j] = (weights && row[j] >= 0) ? __ldg(weights + t * p.k + j0 + j) : 1.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (row[j] >= 0) v[j] = *reinterpret_cast<const Vec<TI, VN>*>(y + (long long)row[j] * ld + (long long)c * VN);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (row[j] >= 0) {
#pragma unroll
                    for (int q = 0; q < VN; q++) acc[q] = fmaf(w[j], to_f32(v[j].v[q]), acc[q]);
                }
        }
        Vec<TO, VN> o;
#pragma unroll
        for (int q = 0; q < VN; q++) o.v[q] = from_f32<TO>(acc[q]);
        *reinterpret_cast<Vec<TO, VN>*>(out + t * p.H + (long long)c * VN) = o;
    }
}

// GROUP threads per token (a warp for short rows, a block for long ones): a vector of dout[t] is read once for up to
// eight of the token's rows; their dot products stay in registers and are summed over the group at the end, in an
// order that depends on the sizes alone.
template <typename TI, typename TO, int VN, int GROUP>
__global__ void __launch_bounds__(256) combine_backward_kernel(const TO* __restrict__ dout, long long ldo, const TI* __restrict__ y,
                                                               long long ld, const float* __restrict__ weights,
                                                               TI* __restrict__ dy, float* __restrict__ dw, int row_vecs,
                                                               const PermuteArgs p) {
    __shared__ float part[8][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_group = threadIdx.x % GROUP;
    constexpr int PER_BLOCK = 256 / GROUP;
    for (long long t = (long long)blockIdx.x * PER_BLOCK + threadIdx.x / GROUP; t < p.T; t += (long long)gridDim.x * PER_BLOCK) {
        const TO* d = dout + t * ldo;
        for (int j0 = 0; j0 < p.k; j0 += 8) {
            int row[8];
            float w[8], acc[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                row[j] = j0 + j < p.k ? __ldg(p.rows + t * p.k + j0 + j) : -1;
                w[j] = row[j] >= 0 ? __ldg(weights + t * p.k + j0 + j) : 0.f;
                acc[j] = 0.f;
            }
            for (int c = in_group; c < row_vecs; c += GROUP) {
                const Vec<TO, VN> dv = *reinterpret_cast<const Vec<TO, VN>*>(d + (long long)c * VN);
                Vec<TI, VN> v[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (row[j] >= 0) v[j] = *reinterpret_cast<const Vec<TI, VN>*>(y + (long long)row[j] * ld + (long long)c * VN);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (row[j] >= 0) {
                        Vec<TI, VN> o;
#pragma unroll
                        for (int q = 0; q < VN; q++) {
                            const float g = to_f32(dv.v[q]);
                            acc[j] = fmaf(g, to_f32(v[j].v[q]), acc[j]);
                            o.v[q] = from_f32<TI>(w[j] * g);
                        }
                        *reinterpret_cast<Vec<TI, VN>*>(dy + (long long)row[j] * p.H + (long long)c * VN) = o;
                    }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
            }
            if constexpr (GROUP > 32) {
                if (lane == 0) {
#pragma unroll
                    for (int j = 0; j < 8; j++) part[warp][j] = acc[j];
                }
                __syncthreads();
                if (threadIdx.x < 8 && j0 + threadIdx.x < p.k) {
                    float s = 0.f;
#pragma unroll
                    for (int q = 0; q < 8; q++) s += part[q][threadIdx.x];
                    dw[t * p.k + j0 + threadIdx.x] = s;
                }
                __syncthreads();
            } else {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (lane == j) s = acc[j];
                if (lane < 8 && j0 + lane < p.k) dw[t * p.k + j0 + lane] = s;
            }
        }
    }
    zero_tail(reinterpret_cast<Vec<TI, VN>*>(dy), row_vecs, p);
}

// One thread per 16-element block of a token: quantised once, its codes and scale byte stored for each of the token's
// rows.  Four neighbouring lanes hold the four k-blocks of one 4-byte group of a scale atom (K % 64 == 0).  The scale
// atoms follow the experts' 128-row tiles: slots[t][j] is the row with every expert padded to whole tiles.
template <int KIND>
__global__ void __launch_bounds__(256) dispatch_quant_kernel(const void* __restrict__ x, long long ld, const int* __restrict__ slots,
                                                             uint8_t* __restrict__ codes, uint8_t* __restrict__ sf_sw,
                                                             const PermuteArgs p) {
    using T = typename ElemOf<KIND>::type;
    const int kbs = p.H / 16;
    const int lane = threadIdx.x & 31;
    const long long n = (long long)p.T * kbs, step = (long long)gridDim.x * blockDim.x;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i - lane < n; i += step) {
        const bool in = i < n;
        const long long t = in ? i / kbs : 0;
        const int kb = in ? (int)(i - t * kbs) : 0;
        float xs[16];
        constexpr int VN = 16 / (int)sizeof(T);
        const Vec<T, VN>* src = reinterpret_cast<const Vec<T, VN>*>(reinterpret_cast<const T*>(x) + t * ld + (long long)kb * 16);
#pragma unroll
        for (int v = 0; v < 16 / VN; v++) {
            const Vec<T, VN> a = src[v];
#pragma unroll
            for (int q = 0; q < VN; q++) xs[v * VN + q] = to_f32(a.v[q]);
        }
        uint32_t w0, w1;
        const uint32_t s = quantize_block16(xs, w0, w1);
        // (n is a multiple of 4, so the four lanes of a group are in range together)
        uint32_t word = s;
        word |= __shfl_down_sync(0xffffffffu, s, 1) << 8;
        word |= __shfl_down_sync(0xffffffffu, s, 2) << 16;
        word |= __shfl_down_sync(0xffffffffu, s, 3) << 24;
        if (!in) continue;
        for (int j = 0; j < p.k; j++) {
            const int row = __ldg(p.rows + t * p.k + j);
            if (row < 0) continue;
            *reinterpret_cast<uint2*>(codes + ((long long)row * kbs + kb) * 8) = make_uint2(w0, w1);
            if ((lane & 3) == 0) {
                const int slot = __ldg(slots + t * p.k + j);
                const long long atom = (long long)(slot >> 7) * (kbs / 4) + kb / 4;
                *reinterpret_cast<uint32_t*>(sf_sw + atom * 512 + (slot & 31) * 16 + ((slot & 127) >> 5) * 4) = word;
            }
        }
    }
    zero_tail(reinterpret_cast<uint2*>(codes), kbs, p);
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

int launched() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NVFP4_OK : (int)e;
}

int check_sizes(int T, int k, int H, long long ld) {
    if (T <= 0 || k <= 0 || H <= 0 || ld < 0) return NVFP4_ERR_SHAPE;
    if ((long long)T * k >= (1ll << 31)) return NVFP4_ERR_UNSUPPORTED;
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
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    const long long row_bytes = (long long)H * size;
    const int vec = common_alignment(16, {(uintptr_t)x, (uintptr_t)xs, (unsigned long long)(ld * size), (unsigned long long)row_bytes});
    if (vec < size) return NVFP4_ERR_ALIGN;
    const PermuteArgs p{(const int*)rows, (const int*)offsets + E, T, k, H};
    const int row_vecs = (int)(row_bytes / vec);
    const int grid = grid_for((long long)T * row_vecs, dev);
    cudaStream_t st = (cudaStream_t)stream;
    const uint8_t* src = (const uint8_t*)x;
    switch (vec) {
        case 16: dispatch_kernel<16><<<grid, 256, 0, st>>>(src, ld * size, xs, row_vecs, p); break;
        case 8: dispatch_kernel<8><<<grid, 256, 0, st>>>(src, ld * size, xs, row_vecs, p); break;
        case 4: dispatch_kernel<4><<<grid, 256, 0, st>>>(src, ld * size, xs, row_vecs, p); break;
        default: dispatch_kernel<2><<<grid, 256, 0, st>>>(src, ld * size, xs, row_vecs, p); break;
    }
    return launched();
}

extern "C" int nvfp4_moe_combine(const void* y, int kind, long long ld, const void* weights, const void* rows, int T, int k, int H,
                                 void* out, int out_kind, void* stream) {
    if (!y || !rows || !out) return NVFP4_ERR_NULL;
    if (!kind_ok(kind) || !kind_ok(out_kind)) return NVFP4_ERR_UNSUPPORTED;
    int rc = check_sizes(T, k, H, ld);
    if (rc) return rc;
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    if ((uintptr_t)y % elem_bytes(kind) || (uintptr_t)out % elem_bytes(out_kind) || (uintptr_t)weights % 4) return NVFP4_ERR_ALIGN;
    const PermuteArgs p{(const int*)rows, nullptr, T, k, H};
    cudaStream_t st = (cudaStream_t)stream;
    return by_type(kind, [&](auto ti) {
        return by_type(out_kind, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            // vectors of 16 input bytes where both sides are aligned to theirs
            constexpr int VN = 16 / sizeof(TI);
            constexpr unsigned long long O = VN * sizeof(TO) < 16 ? VN * sizeof(TO) : 16;
            const bool wide = H % VN == 0 && ld % VN == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)out % O == 0;
            const int row_vecs = wide ? H / VN : H;
            const int grid = grid_for((long long)T * row_vecs, dev);
            if (wide)
                combine_kernel<TI, TO, VN><<<grid, 256, 0, st>>>((const TI*)y, ld, (const float*)weights, (TO*)out, row_vecs, p);
            else
                combine_kernel<TI, TO, 1><<<grid, 256, 0, st>>>((const TI*)y, ld, (const float*)weights, (TO*)out, row_vecs, p);
            return launched();
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
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    if ((uintptr_t)y % elem_bytes(kind) || (uintptr_t)dy % elem_bytes(kind) || (uintptr_t)dout % elem_bytes(out_kind) ||
        (uintptr_t)weights % 4 || (uintptr_t)dweights % 4)
        return NVFP4_ERR_ALIGN;
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
            const int row_vecs = wide ? H / VN : H;
            // a warp per token while its lanes take at most four vectors each
            const bool warp = row_vecs <= 128;
            const int grid = grid_for((long long)T * (warp ? 32 : 256), dev);
            auto go = [&](auto vn, auto group) {
                combine_backward_kernel<TI, TO, decltype(vn)::value, decltype(group)::value><<<grid, 256, 0, st>>>(
                    (const TO*)dout, ldo, (const TI*)y, ld, (const float*)weights, (TI*)dy, (float*)dweights, row_vecs, p);
            };
            using std::integral_constant;
            if (wide && warp) go(integral_constant<int, VN>(), integral_constant<int, 32>());
            else if (wide) go(integral_constant<int, VN>(), integral_constant<int, 256>());
            else if (warp) go(integral_constant<int, 1>(), integral_constant<int, 32>());
            else go(integral_constant<int, 1>(), integral_constant<int, 256>());
            return launched();
        });
    });
}

extern "C" int nvfp4_moe_dispatch_nvfp4(const void* x, int kind, long long ld, const void* rows, const void* slots,
                                        const void* offsets, int T, int E, int k, int K, void* packed, void* sf_sw, void* stream) {
    if (!x || !rows || !slots || !offsets || !packed || !sf_sw) return NVFP4_ERR_NULL;
    if (!kind_ok(kind)) return NVFP4_ERR_UNSUPPORTED;
    int rc = check_sizes(T, k, K, ld);
    if (rc) return rc;
    if (E <= 0) return NVFP4_ERR_SHAPE;
    if (K % 64 != 0) return NVFP4_ERR_K_MULTIPLE;
    if (((uintptr_t)x & 15) || ld * elem_bytes(kind) % 16 || ((uintptr_t)packed & 7) || ((uintptr_t)sf_sw & 3)) return NVFP4_ERR_ALIGN;
    int dev = 0;
    if ((rc = current_device(&dev))) return rc;
    const PermuteArgs p{(const int*)rows, (const int*)offsets + E, T, k, K};
    const int grid = grid_for((long long)T * (K / 16), dev);
    cudaStream_t st = (cudaStream_t)stream;
    switch (kind) {
        case NVFP4_F32: dispatch_quant_kernel<NVFP4_F32><<<grid, 256, 0, st>>>(x, ld, (const int*)slots, (uint8_t*)packed, (uint8_t*)sf_sw, p); break;
        case NVFP4_F16: dispatch_quant_kernel<NVFP4_F16><<<grid, 256, 0, st>>>(x, ld, (const int*)slots, (uint8_t*)packed, (uint8_t*)sf_sw, p); break;
        default: dispatch_quant_kernel<NVFP4_BF16><<<grid, 256, 0, st>>>(x, ld, (const int*)slots, (uint8_t*)packed, (uint8_t*)sf_sw, p); break;
    }
    return launched();
}
