// The experts' NVFP4 products of tokens sorted by expert, with the group sizes on the device (nvfp4_moe_plan).
//
//   GEMM : C[r] = fp16( alpha_e * (A*sfa)[r] @ (B_e*sfb_e)^T )                    for every row r of expert e
//   DUAL : C[r] = fp16( silu(alpha_e * A[r]@B1_e^T) * (alpha_e * A[r]@B2_e^T) ), or the same quantised to NVFP4
//
// The roles are exchanged against the GEMM kernels: the WEIGHTS are the 128-row operand of the tensor core instruction
// and the tokens its N side, whose width is any multiple of 16.  An expert has any number of tokens, so with the tokens
// as 128-row tiles a layer of about 128 tokens per expert computes half as much again on rows that do not exist, at a
// clock that the board's power limit sets (64 experts, 8192 copies, N = 4096, K = 7168: 215 us that way, 195 us
// this way on a cool board, 253 and 225 us after a second of it; 1.14 GB at the measured copy rate take 175 us).  An expert's rows start anywhere in A: a TMA box may start
// at any row, and what it reads of the next expert's rows is multiplied but not stored.
//
//   * CTA PAIRS (cluster of 2, cta_group::2, as in gemm_pair_kernel): a tile is 256 weight rows x NT tokens of one
//     expert; each CTA keeps its own 128 weight rows and HALF of the tokens, the tensor cores read the other half from
//     the peer.  With one CTA per tile and all its tokens the time grew by 0.26 us for every row per expert (64 experts,
//     N = 4096, K = 7168: 170 us for one row, 203 us for 128, 463 us for 512) whatever the values were: what limits these
//     products is the bytes that an SM takes in, and how many bytes of weights are on their way;
//   * NT = 256 where experts have many tokens, NT = 128 (smaller stages, seven instead of five of them: more weights in
//     flight) where they have few;
//   * DUAL: two passes over K, x into one accumulator and y into the other.  (Both products in one pass leave TMEM for 128
//     tokens only, and the instruction with 128 columns reads its weights from shared memory twice as often as it can:
//     547 us for 512 rows per expert, N = 2048, K = 7168, against 406 us.)  silu(x) waits in registers for y;
//   * persistent pairs; column tile fastest, so that the pairs that run together share an expert's tokens in L2;
//   * warps 0 and 2 = TMA producers of the weights and of the tokens (both CTAs, own rows; every load counts its bytes on
//     the leader's barrier), warp 1 = MMA issuer (leader), warps 4.. = epilogue, NT / 64 warps per TMEM lane quadrant with
//     two chunks of 32 tokens each (eight warps with 128 values of silu(x) each left their exponentials no room to overlap:
//     15 000 cycles per tile, as long as the products of K = 4096); a stage is 256 K elements: 16 KB of weights, 128 bytes
//     per token (in boxes of 128, 64, 32 and 16 rows), scale atoms;
//   * accumulators in TMEM, lane = weight row, column = token; two of them, which with 256 columns each share 96 that the
//     epilogue drains first (512 columns do not hold both and the scales);
//   * epilogue: the accumulator goes to registers at once, which frees it for the next pass but one; the results, rounded
//     to fp16, are turned over in a piece of shared memory that belongs to the warp, 16 tokens x 32 weight rows at a time,
//     and a lane stores 16 of a token's outputs (32 bytes), or quantises them (they are one block).
// Every mbarrier wait is bounded; on expiry the role records a status code and leaves its loop, the CTA still frees its
// tensor memory and exits.  Before that the issuer waits, again with a limit, for the products that it has issued and, where
// it left its loop, for the stages that are still being filled: the epilogue may have given up in front of it, and what they
// read and write belongs to the next CTA afterwards.  The epilogue's named barrier is reached by all of its warps or by none,
// and by all lanes of a warp; the two hardware cluster barriers (after set-up, before exit) are reached by every thread on
// every path.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_common.cuh"
#include "moe_common.cuh"
#include "nvfp4_internal.h"
#include "ptx_sm100.cuh"
#include "quant_block.cuh"

namespace nvfp4 {

// Status word of a device if an earlier call has already created it, else nullptr (defined in common.cu).
int* status_word_if_allocated(int dev);

namespace {

constexpr int XM = 128;                              // weight rows of a CTA and tile
constexpr int X_PITCH = 144;                         // bytes of two tokens' 32 outputs in a turning buffer (128 + bank spread)
constexpr uint32_t X_TURN_BYTES = 8 * X_PITCH;       // of one epilogue warp
__host__ __device__ constexpr int x_epilogue_warps(int nt) { return 4 * (nt / 64); }
constexpr int X_FIRST_EPILOGUE = 4;                 // warps before it: weights producer, MMA issuer, tokens producer, idle
__host__ __device__ constexpr int x_threads(int nt) { return 32 * (X_FIRST_EPILOGUE + x_epilogue_warps(nt)); }

template <int NT>
struct ExpertStage {                                 // one stage of one CTA
    static constexpr uint32_t W = XM * 128, T = NT / 2 * 128, SFW = 2048, SFT = NT / 128 * 2048;
    static constexpr uint32_t BYTES = W + T + SFW + SFT;
    static constexpr int STAGES = NT == 128 ? 7 : 5;
    static constexpr size_t SMEM = STAGES * BYTES + x_epilogue_warps(NT) * X_TURN_BYTES + 1024;   // + the tables, 12 bytes per expert
    static constexpr size_t TABLES = 3 * (MOE_MAX_EXPERTS + 1) * 4;
    static_assert(SMEM + TABLES <= 227 * 1024 - 256, "shared memory");
    static_assert(W % 1024 == 0 && T % 1024 == 0 && BYTES % 1024 == 0, "swizzle atoms");
};

struct ExpertMaps {
    CUtensorMap a[4];            // the sorted tokens in boxes of 128, 64, 32 and 16 rows
    CUtensorMap b, b2;           // the weights [E][N][K], boxes of 128 rows
    CUtensorMap sa, sb, sb2;     // scale atoms, four (one stage of a 128-row block) to a box
};

struct ExpertParams {
    const int* offsets;    // [E+1] first row of each expert
    const int* tiles;      // [E+1] first 128-row token tile of each expert
    const int* wide;       // [E+1] the same for tiles of 256 rows
    const float* alphas;   // [E] or null
    uint8_t* c;            // fp16 [R][N], or packed e2m1 [R][N/2] ...
    uint8_t* sfc;          // ... with scale atoms [tiles][N/64][512]
    int R, E, N, K;
    float alpha;
    int* status;
    unsigned long long budget_ns;
};

// One tile as the roles of one CTA see it.
struct ExpertTile {
    int e;                 // expert
    int w;                 // this CTA's 128-row block of its weights (the second CTA's may not exist)
    int row, n;            // first token row of the tile and how many there are
    int atoms;             // first 128-row tile of the tokens' scales
};

// The experts' tables in shared memory and the expert of the last tile asked for.  A role asks for its tiles in ascending
// order, so it walks on from there: a binary search in global memory stood in front of every tile with 3 000 cycles (the
// products of K = 4096 take 8 200).  Empty experts have no tiles.
struct ExpertTables {
    const int *offsets, *tiles, *first;      // [E+1]; first: the tiles of NT tokens
    int columns, e;

    template <int NT>
    __device__ __forceinline__ ExpertTile locate(int t, uint32_t rank) {
        const int u = t / columns;
        while (first[e + 1] <= u) e++;
        const int m = u - first[e];
        ExpertTile ti;
        ti.e = e;
        ti.w = (t - u * columns) * 2 + (int)rank;
        ti.row = offsets[e] + m * NT;
        ti.n = min(NT, offsets[e + 1] - ti.row);
        ti.atoms = tiles[e] + m * (NT / 128);
        return ti;
    }
};

// A shared-memory descriptor `units` of 16 bytes behind another one (no carry out of the low word: see the assertion).
__device__ __forceinline__ uint64_t desc_at(uint64_t first, uint32_t units) {
    return (first & 0xffffffff00000000ull) | ((uint32_t)first + units);
}

// What one epilogue warp does with the accumulator of one pass: its 32 weight rows (lanes) of the two 32-token chunks
// group and group + NT / 64.  Columns of the chunks [lo, hi) are shared with the other accumulator: they are read first
// and released (ovl_free), then the rest, then the whole accumulator is released (acc_empty; both barriers are the
// leader's).  The next pass cannot start before ovl_free, so read(j, column), which reads one of the two chunks, has to
// be short.
template <int NT, typename F>
__device__ __forceinline__ void drain(uint32_t t_lane, int group, int chunks, int lo, int hi, uint32_t ovl_free, uint32_t acc_empty,
                                      int lane, F&& read) {
    auto take = [&](bool shared) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int c = j * (NT / 64) + group;
            if (c < chunks && (c >= lo && c < hi) == shared) read(j, t_lane + c * 32);
        }
    };
    // the signals say "these columns have been read": no memory is published, so they need no release (see epilogue_tile)
    if (lo < hi) {
        take(true);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(ovl_free);
    }
    take(false);
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty);
}

// 16 tokens x 32 weight rows of fp16, one weight row per lane, through the warp's piece of shared memory into rows of the
// output.  o: two tokens to a register; token0: their place in the tile; n0: the warp's first weight row.
template <bool QOUT>
__device__ __forceinline__ void turn_and_store(const ExpertParams& p, const ExpertTile& ti, int token0, int n0, const uint32_t* o,
                                               uint8_t* turn, int lane, bool block_exists) {
#pragma unroll
    for (int i = 0; i < 8; i++) *reinterpret_cast<uint32_t*>(turn + i * X_PITCH + lane * 4) = o[i];
    __syncwarp();
    const int token = token0 + (lane & 15), half = lane >> 4;    // this lane stores 16 outputs of one token
    const uint4* src = reinterpret_cast<const uint4*>(turn + (lane & 15) / 2 * X_PITCH + half * 64);
    const uint32_t pick = (lane & 1) ? 0x7632u : 0x5410u;        // this token's half of two words
    uint32_t words[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint4 v = src[j];
        words[2 * j] = __byte_perm(v.x, v.y, pick);
        words[2 * j + 1] = __byte_perm(v.z, v.w, pick);
    }
    __syncwarp();                                                // the buffer may be written again
    const bool live = block_exists && token < ti.n;
    const size_t row = (size_t)ti.row + token;
    if (!QOUT) {
        if (live) st_global_256_hint(p.c + (row * p.N + n0 + half * 16) * 2, words, policy_evict_first());
        return;
    }
    float f[16];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&words[j]));
        f[2 * j] = g.x; f[2 * j + 1] = g.y;
    }
    uint32_t w0, w1, s = quantize_block16(f, w0, w1);
    // the token's other 16 outputs are in the lane 16 further on: one 16-byte store of codes, one of two scales
    const uint32_t w2 = __shfl_down_sync(0xffffffffu, w0, 16), w3 = __shfl_down_sync(0xffffffffu, w1, 16);
    s |= __shfl_down_sync(0xffffffffu, s, 16) << 8;
    if (live && half == 0) {
        *reinterpret_cast<uint4*>(p.c + row * (p.N / 2) + n0 / 2) = make_uint4(w0, w1, w2, w3);
        const size_t atom = (size_t)(ti.atoms + token / 128) * (p.N / 64) + n0 / 64;
        *reinterpret_cast<uint16_t*>(p.sfc + atom * 512 + (token % 32) * 16 + (token % 128) / 32 * 4 + (n0 / 16) % 4) = (uint16_t)s;
    }
}

template <bool DUAL, bool QOUT, int NT>
__global__ void __launch_bounds__(x_threads(NT), 1)
expert_kernel(const __grid_constant__ ExpertMaps maps, const ExpertParams p) {
    using Stage = ExpertStage<NT>;
    constexpr int PASSES = DUAL ? 2 : 1, STAGES = Stage::STAGES;
    // TMEM columns of one stage's scales: four K steps of 4 for the weights, of NT / 32 for the tokens
    constexpr uint32_t SF_COLS = 16 + 4 * (NT / 32);
    constexpr uint32_t SF_BASE = TMEM_COLS - 2 * SF_COLS;
    // where two accumulators do not fit beside the scales, the second overlaps the tail of the first
    constexpr uint32_t ACC1_OFF = 2 * NT <= SF_BASE ? NT : SF_BASE - NT;
    constexpr int OVERLAP = (NT - (int)ACC1_OFF) / 32;          // chunks that the two share
    static_assert((NT - ACC1_OFF) % 32 == 0 && ACC1_OFF % 32 == 0, "tensor memory");

    extern __shared__ uint8_t smem_raw[];
    // same layout in both CTAs (remote arrivals and pair-wide commits address barriers by offset)
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 6];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int gave_up;

    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();                    // 0 = leader
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]);
    const uint32_t acc_full0 = smem_u32(&bars[2 * STAGES]);     // [2] accumulator complete, signalled in both CTAs
    const uint32_t acc_empty0 = acc_full0 + 16;                 // [2] accumulator drained, leader's copy used
    const uint32_t ovl_free = acc_full0 + 32;                   // shared columns drained, leader's copy used
    const uint32_t issued_done = acc_full0 + 40;                // every product of the launch is complete, leader's copy used

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full0 + 8 * s, 2);                        // the leader's copy: its producers + both CTAs' bytes
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(acc_full0 + 8 * b, 1);
            mbar_init(acc_empty0 + 8 * b, 2 * x_epilogue_warps(NT));
        }
        mbar_init(ovl_free, 2 * x_epilogue_warps(NT));
        mbar_init(issued_done, 1);
        gave_up = 0;
        fence_mbar_init();
        prefetch_tmap(&maps.a[0]);
        prefetch_tmap(&maps.a[3]);
        prefetch_tmap(&maps.b);
        prefetch_tmap(&maps.sa);
        prefetch_tmap(&maps.sb);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(&tmem_base_slot), TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers exist before anything is sent to them
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    pdl_wait();
    pdl_launch();

    int* tables = reinterpret_cast<int*>(smem_raw + (smem0 - smem_u32(smem_raw)) + STAGES * Stage::BYTES + x_epilogue_warps(NT) * X_TURN_BYTES);
    for (int i = threadIdx.x; i <= p.E; i += blockDim.x) {
        tables[i] = p.offsets[i];
        tables[p.E + 1 + i] = p.tiles[i];
        tables[2 * (p.E + 1) + i] = (NT == 128 ? p.tiles : p.wide)[i];
    }
    __syncthreads();
    ExpertTables where{tables, tables + p.E + 1, tables + 2 * (p.E + 1), (p.N + 2 * XM - 1) / (2 * XM), 0};
    // the tile count comes from the plan; a launch has enough pairs for the most there can be
    const int total_tiles = where.first[p.E] * where.columns, live_rows = where.offsets[p.E];
    const int kiters = p.K / BK, apb = p.K / 64;                // K steps; scale atoms of a 128-row block
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (warp == 0 || warp == 2) {
        // ------------------------------------------------------------------ producers (both CTAs, own rows): warp 0 the
        // weights, warp 2 the tokens (issuing a copy takes a thread about 70 cycles, and a stage has up to ten)
        if (elect_one()) {
            const bool weights = warp == 0;
            uint32_t slot = 0, phase = 1;
            bool alive = true;
            const uint32_t leader_full0 = mapa_shared(full0, 0);
            for (int t = pair; alive && t < total_tiles; t += npairs) {
                const ExpertTile ti = where.locate<NT>(t, rank);
                const int half = ((ti.n + 31) & ~31) / 2;               // a multiple of 16 tokens in each CTA
                const int atoms = (ti.n + 127) / 128;
                const int row0 = ti.row + (int)rank * half;
                const bool block_exists = ti.w < p.N / XM, peer_exists = (ti.w | 1) < p.N / XM;
                const int atom_w = (ti.e * (p.N / XM) + ti.w) * apb, atom_t = ti.atoms * apb;
                // the leader announces the bytes of both CTAs.  Weight rows beyond N (second CTA of the last column) read
                // as zeros; their scale block does not exist and is not fetched
                const uint32_t tx = weights ? 2u * Stage::W + (peer_exists ? 2u : 1u) * Stage::SFW
                                            : 2u * ((uint32_t)half * 128u + (uint32_t)atoms * 2048u);
                for (int pass = 0; alive && pass < PASSES; pass++) {
                    const CUtensorMap *map_w = pass ? &maps.b2 : &maps.b, *map_sw = pass ? &maps.sb2 : &maps.sb;
                    for (int kit = 0; kit < kiters; kit++) {
                        if (!mbar_wait_cluster(empty0 + 8 * slot, phase, p.budget_ns)) {
                            report_status(p.status, DEV_TIMEOUT_PRODUCER);
                            alive = false;
                            break;
                        }
                        const uint32_t full = leader_full0 + 8 * slot;
                        const uint32_t sW = smem0 + slot * Stage::BYTES, sT = sW + Stage::W;
                        const uint32_t sSFW = sT + Stage::T, sSFT = sSFW + Stage::SFW;
                        const int k0 = kit * BK, ka = kit * (BK / 64);
                        if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * slot, tx);
                        if (weights) {
                            tma_load_3d_pair(sW, map_w, k0, ti.w * XM, ti.e, full);
                            if (block_exists) tma_load_2d_pair(sSFW, map_sw, 0, atom_w + ka, full);
                        } else {
                            int r = 0;
#pragma unroll
                            for (int b = 0; b < 4; b++)
                                if (half & (128 >> b)) {
                                    tma_load_3d_pair(sT + r * 128, &maps.a[b], k0, row0 + r, 0, full);
                                    r += 128 >> b;
                                }
                            for (int j = 0; j < atoms; j++) tma_load_2d_pair(sSFT + j * 2048u, &maps.sa, 0, atom_t + j * apb + ka, full);
                        }
                        if (++slot == STAGES) { slot = 0; phase ^= 1; }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ leader: MMA issuer for the pair (one lane)
        if (elect_one() && rank == 0) {
            // One thread issues everything, so what it computes per instruction counts: the descriptors of a stage differ
            // from those of the first one by their address field, the low bits of the low word.
            const uint64_t d_w0 = make_desc_k_sw128(smem0), d_t0 = make_desc_k_sw128(smem0 + Stage::W);
            const uint64_t d_sfw0 = make_desc_sf(smem0 + Stage::W + Stage::T), d_sft0 = make_desc_sf(smem0 + Stage::W + Stage::T + Stage::SFW);
            static_assert(STAGES * Stage::BYTES < (1u << 18), "the address field holds 18 bits");
            uint32_t slot = 0, phase = 0, odd = 0, seq = 0;     // ring slot and its phase, scale region, passes so far
            bool alive = true;
            for (int t = pair; alive && t < total_tiles; t += npairs) {
                const ExpertTile ti = where.locate<NT>(t, rank);
                const bool two_atoms = ti.n > 128;
                const uint32_t idesc = make_idesc_nvfp4(2 * XM, (ti.n + 31) & ~31);
                for (int pass = 0; alive && pass < PASSES; pass++, seq++) {
                    const uint32_t buf = seq & 1;
                    bool ok = mbar_wait_cluster(acc_empty0 + 8 * buf, ((seq >> 1) & 1) ^ 1, p.budget_ns);
                    if (ok && OVERLAP > 0 && seq > 0) ok = mbar_wait_cluster(ovl_free, (seq - 1) & 1, p.budget_ns);
                    if (!ok) {
                        report_status(p.status, DEV_TIMEOUT_MMA_ACC);
                        alive = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t t_acc = tmem_base + buf * ACC1_OFF;
                    for (int kit = 0; kit < kiters; kit++) {
                        if (!mbar_wait_cluster(full0 + 8 * slot, phase, p.budget_ns)) {   // both CTAs' bytes
                            report_status(p.status, DEV_TIMEOUT_CONSUMER);
                            alive = false;
                            break;
                        }
                        tc_fence_after_sync();
                        const uint32_t at = slot * (Stage::BYTES >> 4);
                        const uint32_t t_sfw = tmem_base + SF_BASE + odd * SF_COLS, t_sft = t_sfw + 16;
#pragma unroll
                        for (int ks = 0; ks < 4; ks++) {
                            tc_cp_sf_atom_pair(t_sfw + 4 * ks, desc_at(d_sfw0, at + 32 * ks));
                            tc_cp_sf_atom_pair(t_sft + ks * (NT / 32), desc_at(d_sft0, at + 32 * ks));
                        }
                        if (NT > 128 && two_atoms) {
#pragma unroll
                            for (int ks = 0; ks < 4; ks++) tc_cp_sf_atom_pair(t_sft + ks * (NT / 32) + 4, desc_at(d_sft0, at + 128 + 32 * ks));
                        }
#pragma unroll
                        for (int ks = 0; ks < 4; ks++)
                            tc_mma_nvfp4_pair(t_acc, desc_at(d_w0, at + 2 * ks), desc_at(d_t0, at + 2 * ks), idesc, t_sfw + 4 * ks,
                                              t_sft + ks * (NT / 32), (kit | ks) != 0 ? 1u : 0u);
                        tc_commit_pair(empty0 + 8 * slot, 3);               // frees the stage in both CTAs
                        odd ^= 1;
                        if (++slot == STAGES) { slot = 0; phase ^= 1; }
                    }
                    if (alive) tc_commit_pair(acc_full0 + 8 * buf, 3);      // accumulators complete in both CTAs
                }
            }
            tc_commit_pair(issued_done, 1);
            if (!mbar_wait_cluster(issued_done, 0, p.budget_ns)) report_status(p.status, DEV_TIMEOUT_MMA_ACC);
            // the stages that nothing was issued for, in their order; behind the last one that was filled, one budget
            for (int s = 0; !alive && s < STAGES && mbar_wait_cluster(full0 + 8 * slot, phase, p.budget_ns); s++)
                if (++slot == STAGES) { slot = 0; phase ^= 1; }
        }
    } else if (warp >= X_FIRST_EPILOGUE) {
        // ------------------------------------------------------------------ epilogue warps (both CTAs)
        const int q = warp & 3, group = (warp - X_FIRST_EPILOGUE) >> 2; // TMEM lane quadrant this warp may access; which chunks it takes
        uint8_t* turn = smem_raw + (smem0 - smem_u32(smem_raw)) + STAGES * Stage::BYTES + (warp - X_FIRST_EPILOGUE) * X_TURN_BYTES;
        const uint32_t l_acc_empty0 = mapa_shared(acc_empty0, 0), l_ovl_free = mapa_shared(ovl_free, 0);
        {
            // rows behind the last copy (choices that were dropped): zero, so that sums over the buffer are sums over copies
            const size_t row_bytes = QOUT ? (size_t)p.N / 2 : (size_t)p.N * 2;
            const uint32_t zero[8] = {};
            const size_t end = (size_t)p.R * row_bytes / 32;
            constexpr int THREADS = 32 * x_epilogue_warps(NT);
            for (size_t i = (size_t)live_rows * row_bytes / 32 + (size_t)blockIdx.x * THREADS + threadIdx.x - 32 * X_FIRST_EPILOGUE; i < end;
                 i += (size_t)gridDim.x * THREADS)
                st_global_256(p.c + i * 32, zero);
        }
        uint32_t seq = 0;
        bool alive = true;
        for (int t = pair; alive && t < total_tiles; t += npairs) {
            const ExpertTile ti = where.locate<NT>(t, rank);
            const int chunks = (ti.n + 31) / 32;         // with tokens in them
            const float alpha = p.alphas ? p.alpha * p.alphas[ti.e] : p.alpha;
            const bool block_exists = ti.w < p.N / XM;
            uint32_t held[DUAL ? 2 : 1][32];             // x, then silu(x) until y is there
            uint32_t out[2][16];                         // fp16 results, two tokens to a register
#pragma unroll
            for (int pass = 0; pass < PASSES; pass++, seq++) {
                const uint32_t buf = seq & 1;
                if (!alive) break;
                // one warp waits for the accumulator and the others for that warp (sixteen waiting warps took power from the
                // rest of the board: 1 %).  If it gives up it says in which pass, so that all of them leave at the same barrier
                // (the lanes wait each for itself, and the limit of one may pass just before another sees the accumulator)
                if (warp == X_FIRST_EPILOGUE) {
                    const bool there = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * buf, (seq >> 1) & 1, p.budget_ns));
                    if (!there && lane == 0) {
                        report_status(p.status, DEV_TIMEOUT_EPILOGUE);
                        *(volatile int*)&gave_up = (int)seq + 1;
                    }
                    __syncwarp();
                }
                named_bar_sync(1, 32 * x_epilogue_warps(NT));
                if (*(volatile int*)&gave_up == (int)seq + 1) {
                    alive = false;
                    break;
                }
                tc_fence_after_sync();
                const uint32_t t_lane = tmem_base + buf * ACC1_OFF + ((uint32_t)(q * 32) << 16);
                // the first accumulator shares its last columns, the second its first
                const int lo = buf == 0 ? NT / 32 - OVERLAP : 0, hi = buf == 0 ? NT / 32 : OVERLAP;
                drain<NT>(t_lane, group, chunks, lo, hi, l_ovl_free, l_acc_empty0 + 8 * buf, lane, [&](int j, uint32_t column) {
                    if (DUAL && pass == 0) {
                        tc_ld_32x32(column, held[j]);
                        tc_wait_ld();
                        return;
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t v[16];
                        tc_ld_32x16(column + 16 * h, v);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            float a = alpha * __uint_as_float(v[2 * i]), b = alpha * __uint_as_float(v[2 * i + 1]);
                            if (DUAL) { a = __uint_as_float(held[j][16 * h + 2 * i]) * a; b = __uint_as_float(held[j][16 * h + 2 * i + 1]) * b; }
                            const __half2 r = __floats2half2_rn(a, b);
                            out[j][8 * h + i] = *reinterpret_cast<const uint32_t*>(&r);
                        }
                    }
                });
                if (DUAL && pass == 0) {
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        if (j * (NT / 64) + group < chunks) {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                held[j][i] = __float_as_uint(silu_mul(alpha * __uint_as_float(held[j][i]), 1.0f));
                        }
                }
            }
            if (!alive) break;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int token0 = (j * (NT / 64) + group) * 32 + 16 * h;
                    if (token0 < ti.n) turn_and_store<QOUT>(p, ti, token0, ti.w * XM + q * 32, out[j] + 8 * h, turn, lane, block_exists);
                }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();   // neither CTA frees tensor memory or exits while the other may still touch it
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// The device's status word.  Its first use allocates it, which a capture in global mode forbids the thread that captures:
// the mode is relaxed for that moment (the allocation belongs to no graph).
int* status_word_anywhere(int dev) {
    int* word = status_word_if_allocated(dev);
    if (word) return word;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    word = status_word(dev);
    cudaThreadExchangeStreamCaptureMode(&mode);
    return word;
}

// Tiles of `rows` rows that R copies over E experts can fill at most: every expert that has rows has at most one tile
// that is not full.
long most_tiles(int R, int E, int rows) {
    const int active = R < E ? R : E;
    return active + (long)(R - active) / rows;
}

template <bool DUAL, bool QOUT, int NT>
int launch_experts(const ExpertMaps& maps, const ExpertParams& p, int dev, cudaStream_t stream) {
    auto kernel = expert_kernel<DUAL, QOUT, NT>;
    constexpr size_t most = ExpertStage<NT>::SMEM + ExpertStage<NT>::TABLES;
    const size_t smem = ExpertStage<NT>::SMEM + 12ull * (p.E + 1);
    static int pairs[64] = {};                           // that are resident at once
    if (!pairs[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) return (int)e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * sm_count(dev));
        cfg.blockDim = dim3(x_threads(NT));
        cfg.dynamicSmemBytes = most;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        if (e != cudaSuccess) return (int)e;
        if (n <= 0) return NVFP4_ERR_UNSUPPORTED;
        pairs[dev] = n;
    }
    const long tiles = most_tiles(p.R, p.E, NT) * ((p.N + 2 * XM - 1) / (2 * XM));
    if (tiles >= (1l << 31)) return NVFP4_ERR_UNSUPPORTED;
    return launch_dependent(kernel, 2 * (int)(tiles < pairs[dev] ? tiles : pairs[dev]), x_threads(NT), smem, 2, stream, maps, p);
}

// What the three entry points share.  b2 / sfb2: the second product of the dual GEMM; sfc: the output is quantised.
template <bool DUAL, bool QOUT>
int expert_product(const void* a, const void* sfa_sw, const void* b, const void* sfb_sw, const void* b2, const void* sfb2_sw,
                   const void* offsets, const void* tiles, const void* wide, const void* alphas, void* c, void* sfc, int R, int E,
                   int N, int K, float alpha, void* stream) {
    const void* ptrs[8] = {a, sfa_sw, b, sfb_sw, DUAL ? b2 : b, DUAL ? sfb2_sw : sfb_sw, QOUT ? sfc : c, c};
    for (const void* ptr : ptrs) {
        if (!ptr) return NVFP4_ERR_NULL;
        if ((uintptr_t)ptr & 15) return NVFP4_ERR_ALIGN;
    }
    if (!offsets || !tiles || !wide) return NVFP4_ERR_NULL;
    if (((uintptr_t)c & 31) || (((uintptr_t)offsets | (uintptr_t)tiles | (uintptr_t)wide | (uintptr_t)alphas) & 3)) return NVFP4_ERR_ALIGN;
    if (R <= 0 || E <= 0 || N <= 0 || K <= 0) return NVFP4_ERR_SHAPE;
    if (K % BK != 0) return NVFP4_ERR_K_MULTIPLE;
    if (N % XM != 0) return NVFP4_ERR_N_MULTIPLE;
    if (E > MOE_MAX_EXPERTS) return NVFP4_ERR_UNSUPPORTED;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 64) return NVFP4_ERR_UNSUPPORTED;
    ExpertMaps maps;
    int rc = make_operand_tmap(&maps.b, b, N, K, E, XM);
    for (int i = 0; i < 4 && !rc; i++) rc = make_operand_tmap(&maps.a[i], a, R, K, 1, 128 >> i);
    if (!rc && DUAL) rc = make_operand_tmap(&maps.b2, b2, N, K, E, XM);
    // scale atoms are counted in 32 bits
    const long atoms_a = most_tiles(R, E, 128) * (K / 64), atoms_b = (long)E * (N / XM) * (K / 64);
    if (!rc && (atoms_a >= (1l << 31) || atoms_b >= (1l << 31))) rc = NVFP4_ERR_UNSUPPORTED;
    if (!rc) rc = make_scale_tmap(&maps.sa, sfa_sw, atoms_a);
    if (!rc) rc = make_scale_tmap(&maps.sb, sfb_sw, atoms_b);
    if (!rc && DUAL) rc = make_scale_tmap(&maps.sb2, sfb2_sw, atoms_b);
    if (rc) return rc;
    if (!DUAL) { maps.b2 = maps.b; maps.sb2 = maps.sb; }
    const ExpertParams p{(const int*)offsets, (const int*)tiles, (const int*)wide, (const float*)alphas, (uint8_t*)c, (uint8_t*)sfc,
                         R, E, N, K, alpha, status_word_anywhere(dev), wait_budget_ns()};
    cudaStream_t st = (cudaStream_t)stream;
    // few rows per expert on average (64 experts, K = 7168, experts liked unequally, NT = 128 against 256): 32 rows 161
    // against 169 us, 64: 172 / 175, 96: 188 / 187, 128: 217 / 204; DUAL 32: 159 / 172, 96: 182 / 200, 128: 213 / 208.  The
    // host knows the number of copies only, so choices that are not routed count as rows here
    const bool few = R <= 96ll * E;
    return few ? launch_experts<DUAL, QOUT, 128>(maps, p, dev, st) : launch_experts<DUAL, QOUT, 256>(maps, p, dev, st);
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_moe_gemm(const void* a, const void* sfa_sw, const void* b, const void* sfb_sw, const void* offsets,
                              const void* tiles, const void* wide_tiles, const void* alphas, void* c, int R, int E, int N, int K,
                              float alpha, void* stream) {
    return expert_product<false, false>(a, sfa_sw, b, sfb_sw, nullptr, nullptr, offsets, tiles, wide_tiles, alphas, c, nullptr, R, E, N, K,
                                        alpha, stream);
}
extern "C" int nvfp4_moe_dual_gemm(const void* a, const void* sfa_sw, const void* b1, const void* sfb1_sw, const void* b2,
                                   const void* sfb2_sw, const void* offsets, const void* tiles, const void* wide_tiles,
                                   const void* alphas, void* c, int R, int E, int N, int K, float alpha, void* stream) {
    return expert_product<true, false>(a, sfa_sw, b1, sfb1_sw, b2, sfb2_sw, offsets, tiles, wide_tiles, alphas, c, nullptr, R, E, N, K,
                                       alpha, stream);
}
extern "C" int nvfp4_moe_dual_gemm_nvfp4(const void* a, const void* sfa_sw, const void* b1, const void* sfb1_sw, const void* b2,
                                         const void* sfb2_sw, const void* offsets, const void* tiles, const void* wide_tiles,
                                         const void* alphas, void* c_packed, void* sfc_sw, int R, int E, int N, int K, float alpha,
                                         void* stream) {
    return expert_product<true, true>(a, sfa_sw, b1, sfb1_sw, b2, sfb2_sw, offsets, tiles, wide_tiles, alphas, c_packed, sfc_sw, R, E, N,
                                      K, alpha, stream);
}
