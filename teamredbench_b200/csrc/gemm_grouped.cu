// gemm_grouped.cu -- matrix products grouped by expert, with ragged numbers of rows.
//
//   grouped_gemm   out[r] = a[r] * b[e]                 for the rows r of group e
//   grouped_wgrad  out[e] = a[rows of e]^T * g[rows of e]
//
// Rows are sorted by group; group e owns rows [offsets[e], offsets[e + 1]), and
// offsets live on the device, so no call waits for the host to read them.  The
// launch covers the largest possible number of tiles and every CTA derives the
// real tile list from the offsets.
//
// No counterpart in the reference, whose GEMM takes one matrix per operand
// (src/teamredbench/benchmarks/mfu.py:229-234).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "trb_common.cuh"
#include "trb_groups.cuh"
#include "trb_launch.cuh"

namespace trb {
namespace grouped {

__device__ int g_grouped_error;

constexpr int kEpiWarps = 8;         // two for each quarter of the TMEM lanes
constexpr int kThreads = 64 + 32 * kEpiWarps;  // producer warp, MMA warp, epilogue warps
constexpr int kBK = 64;              // 16-bit elements per 128-byte swizzle row
constexpr int kInstrK = 16;          // K elements per tcgen05.mma
// Two k-blocks a stage: a stage costs the MMA thread about 260 ns whatever it holds (wait, issue, commit), as long as
// the four products of one k-block with 128 rows take.
constexpr int kStages = 3;
constexpr int kBlockBytes = 128 * 128;    // one CTA's 128 rows (or columns) x 128 bytes of one operand: a k-block
constexpr int kOperandStage = 2 * kBlockBytes;
constexpr size_t kRingBytes = (size_t)kStages * 2 * kOperandStage;
constexpr int kNumAcc = 2;
constexpr int kTmemCols = 512;
constexpr int kEpiBytes = 32 * 64;   // a 32 x 32 block of 16-bit results

// F32 <- BF16 x BF16 or F16 x F16 instruction descriptor; bit 15 / 16: A / B is MN-major.
template <int DT>
__host__ __device__ constexpr uint32_t make_idesc(int m, bool a_mn, bool b_mn) {
    constexpr uint32_t fmt = DT == TRB_BFLOAT16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t idesc_n(uint32_t idesc, int n) { return idesc | ((uint32_t)(n >> 3) << 17); }

template <int DT>
__device__ __forceinline__ uint32_t pack2(uint32_t lo, uint32_t hi) {
    if constexpr (DT == TRB_FLOAT16) {
        __half2 h = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
        return *reinterpret_cast<uint32_t*>(&h);
    } else {
        __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
        return *reinterpret_cast<uint32_t*>(&h);
    }
}

// Four 8 x 8 blocks of 16-bit values from registers (the fragment order of an m16n8 product: thread t holds
// row t / 4, columns 2 (t % 4) and + 1) to shared memory, each transposed; thread 8i + j gives the 16-byte
// row that takes column j of block i.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0),
                 "r"(r1), "r"(r2), "r"(r3)
                 : "memory");
}
// The same without transposing: thread 8i + j gives the 16-byte row that takes row j of block i.
__device__ __forceinline__ void stmatrix_x4(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0), "r"(r1),
                 "r"(r2), "r"(r3)
                 : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr)
                 : "memory");
    return v;
}

// ------------------------------------------------------------------ out[r] = a[r] * b[e]
// A CTA pair (tcgen05.mma.cta_group::2, M = 256) computes the transposed tile
//   out^T[256 columns n, R rows r] = b[e]^T[n, k] * a[r, k]^T:
// the 256 TMEM lanes of the pair run along n, the instruction's N side along
// the R <= 256 rows of one group.  N goes in steps of 32, so a group of r rows
// costs ceil(r / 32) * 32 rows of products instead of whole 128- or 256-row
// tiles, and no row of another group ever meets this group's weights.  A group
// of more than 256 rows is cut into equal chunks.  The price is an epilogue
// that transposes, on the tensor-memory fragments in registers (stmatrix).
// Measured: 32768 rows, 8 groups, 4096 x 4096, 850 to 880 us, 1250 to 1290
// TFLOP/s under the power cap; 4109 rows, 16 groups, 2048 x 4096, 70 us in a
// burst at 1965 MHz and 84 sustained at the cap's 1180; 96 rows, 32 groups,
// 2048 x 1408, 36 us, 4.8 TB/s of weights.  Between the two bounds neither the
// weights' bytes nor the tensor pipe run alone: 37 groups of 4096 x 1024 take
// 57 us with 16 rows each and 75 with 256, where both floors are 48 us.
// Asking the next stages' weights into L2 made it slower (in bursts, 96 rows
// 43 us, 4109 rows 85).  Rows past the group's end are loaded and multiplied
// but not stored; each output depends on its own row only, so what stands
// there (the next group's rows, NaN) does not matter. K past the end is zero
// in both operands (the tensor maps are per group).
struct ProductTile {
    int e, row0, rows, n0;
};

constexpr int kTileN = 256;    // columns of a tile (pair)
constexpr int kTileRows = 256; // largest chunk

__device__ __forceinline__ int chunks_of(int rows) { return (rows + kTileRows - 1) / kTileRows; }

// Tile t: groups in order; inside a group, runs of 8 chunks walk the columns
// together (a weight panel is read by the chunks next to each other in time).
__device__ __forceinline__ ProductTile product_tile(int t, int groups, int num_n, const GroupTable& g) {
    const int e = group_of_chunk(t / num_n, groups, g);
    const int local = t - g.chunk0[e] * num_n;
    const int rows = g.rows[e];
    const int chunks = chunks_of(rows);
    const int run = 8 * num_n;
    const int first = local / run * 8;
    const int width = min(8, chunks - first);
    const int in_run = local - first * num_n;
    const int chunk = first + in_run % width;
    const int per = ((rows + chunks - 1) / chunks + 31) & ~31;
    ProductTile p;
    p.e = e;
    p.row0 = g.start[e] + chunk * per;
    p.rows = min(per, rows - chunk * per);
    p.n0 = in_run / width * kTileN;
    return p;
}

constexpr size_t kProductSmem = kRingBytes + 1024 + kEpiWarps * kEpiBytes;

template <int DT, bool KB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX128,
                        const __grid_constant__ CUtensorMap tmX64, const __grid_constant__ CUtensorMap tmX32,
                        const int* offsets,
                        uint16_t* out, int groups, int total_rows, int N, int K) {
    constexpr uint32_t kIdesc = make_idesc<DT>(256, !KB, false);

    extern __shared__ uint8_t smem_raw[];
    __shared__ int group_words[3 * kMaxGroups + 1];
    __shared__ __align__(8) uint64_t full_bar[kStages];   // leader: both CTAs' TMA bytes land here
    __shared__ __align__(8) uint64_t empty_bar[kStages];  // both: MMA finished reading the stage
    __shared__ __align__(8) uint64_t accf_bar[kNumAcc];   // both: accumulator ready for the epilogue
    __shared__ __align__(8) uint64_t acce_bar[kNumAcc];   // leader: both CTAs' epilogues drained it
    __shared__ __align__(8) uint64_t drain_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;

    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sW = smem_base;
    const uint32_t sX = smem_base + kStages * kOperandStage;
    const uint32_t sEpi = smem_base + (uint32_t)kRingBytes;

    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    const int num_n = (N + kTileN - 1) / kTileN;
    const int num_kb = (K + kBK - 1) / kBK;
    const GroupTable table = {group_words, group_words + kMaxGroups, group_words + 2 * kMaxGroups};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int a = 0; a < kNumAcc; ++a) {
            mbar_init(smem_u32(&accf_bar[a]), 1);
            mbar_init(smem_u32(&acce_bar[a]), 2 * kEpiWarps);  // of both CTAs
        }
        mbar_init(smem_u32(&drain_bar), 1);
        abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX128);
        tma_prefetch_desc(&tmX64);
        tma_prefetch_desc(&tmX32);
    }
    if (warp == 0) {
        tmem_alloc_pair(smem_u32(&tmem_slot), kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // barrier inits of both CTAs visible before any cross-CTA signal
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    // Only now that this block has its TMEM: the next grid's blocks take theirs before they wait for this grid.
    grid_launch_dependents();
    grid_dependency_wait();  // offsets, operands and out may belong to the previous grid until here
    groups = load_groups(offsets, groups, total_rows, table, &g_grouped_error);
    if (warp == 0) scan_chunks(groups, kTileRows, table, lane);
    __syncthreads();
    const int num_tiles = table.chunk0[groups] * num_n;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer (both CTAs; completion on the leader's full barriers)
            uint32_t stage = 0, phase = 0;
            uint32_t issued_mask = 0, issued_phase = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
                const ProductTile p = product_tile(tile, groups, num_n, table);
                const int half = ((p.rows + 31) & ~31) >> 1;  // rows this CTA loads
                const int x_row = p.row0 + (int)rank * half;
                // One box a k-block, of 128, 64 or 32 rows: a request costs more than the rows nobody uses (4109 rows:
                // 76 us with up to three boxes of 32 a k-block, 74 with one).
                const CUtensorMap* tmX = half > 64 ? &tmX128 : half > 32 ? &tmX64 : &tmX32;
                const uint32_t x_bytes = (half > 64 ? 128 : half > 32 ? 64 : 32) * 128;
                const int w_col = p.n0 + (int)rank * 128;
                for (int kb = 0; kb < num_kb; kb += 2) {
                    const int blocks = min(2, num_kb - kb);
                    if (!mbar_wait_cluster(smem_u32(&empty_bar[stage]), phase ^ 1u, &abort_flag)) {
                        atomicCAS(&g_grouped_error, 0, kErrProducerWait);
                        abort_flag = 1;
                        ok = false;
                        break;
                    }
                    const uint32_t fb_local = smem_u32(&full_bar[stage]);
                    // Row-major weights come in boxes of 128 k (past K: zeros); the other boxes are one k-block each.
                    const uint32_t w_bytes = KB ? blocks * kBlockBytes : kOperandStage;
                    if (leader) mbar_arrive_expect_tx(fb_local, 2 * (w_bytes + blocks * x_bytes));
                    const uint32_t fb = fb_local & kPeerBitMask;
                    const uint32_t w = sW + stage * kOperandStage, x = sX + stage * kOperandStage;
                    if constexpr (!KB) {
                        tma_load_3d_pair(w, &tmW, fb, w_col, kb * kBK, p.e);
                        tma_load_3d_pair(w + kBlockBytes, &tmW, fb, w_col + 64, kb * kBK, p.e);
                    }
                    for (int i = 0; i < blocks; ++i) {
                        if constexpr (KB) tma_load_3d_pair(w + i * kBlockBytes, &tmW, fb, (kb + i) * kBK, w_col, p.e);
                        tma_load_2d_pair(x + i * kBlockBytes, tmX, fb, (kb + i) * kBK, x_row);
                    }
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (leader)  // every armed phase completes only once both CTAs' bytes have landed
                for (int s = 0; s < kStages; ++s)
                    if (issued_mask & (1u << s))
                        if (!mbar_wait_cluster(smem_u32(&full_bar[s]), (issued_phase >> s) & 1u, nullptr))
                            atomicCAS(&g_grouped_error, 0, kErrDrainWait);
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            // ---------------- MMA issuer: the leader CTA only
            const uint64_t w_desc0 = KB ? make_sdesc(sW, 16, 1024) : make_sdesc(sW, kBlockBytes, 1024);
            const uint64_t x_desc0 = make_sdesc(sX, 16, 1024);
            constexpr int kWStep = KB ? kInstrK * 2 : kInstrK * 128;           // bytes per instruction K step
            constexpr int kWBlock = KB ? kBlockBytes : kBlockBytes / 2;        // and per k-block
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            int t_local = 0;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs, ++t_local) {
                const ProductTile p = product_tile(tile, groups, num_n, table);
                const uint32_t idesc = idesc_n(kIdesc, (p.rows + 31) & ~31);
                const int acc = t_local & 1;
                if (!mbar_wait_cluster(smem_u32(&acce_bar[acc]), ((uint32_t)(t_local >> 1) & 1u) ^ 1u, &abort_flag)) {
                    atomicCAS(&g_grouped_error, 0, kErrMmaWait);
                    abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(acc * kTileRows);
                for (int kb = 0; kb < num_kb; kb += 2) {
                    if (!mbar_wait_cluster(smem_u32(&full_bar[stage]), phase, &abort_flag)) {
                        atomicCAS(&g_grouped_error, 0, kErrMmaWait);
                        abort_flag = 1;
                        ok = false;
                        break;
                    }
                    const uint64_t off = (uint64_t)((stage * kOperandStage) >> 4);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (kb + i >= num_kb) break;
#pragma unroll
                        for (int ks = 0; ks < kBK / kInstrK; ++ks)
                            mma_pair_f16(d_tmem, w_desc0 + off + (uint64_t)((i * kWBlock + ks * kWStep) >> 4),
                                         x_desc0 + off + (uint64_t)((i * kBlockBytes + ks * kInstrK * 2) >> 4), idesc,
                                         (kb != 0 || i != 0 || ks != 0) ? 1u : 0u);
                    }
                    tc_commit_pair_multicast(smem_u32(&empty_bar[stage]), 0x3);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) tc_commit_pair_multicast(smem_u32(&accf_bar[acc]), 0x3);
            }
            tc_commit_pair_multicast(smem_u32(&drain_bar), 0x1);
            if (!mbar_wait_cluster(smem_u32(&drain_bar), 0, nullptr)) atomicCAS(&g_grouped_error, 0, kErrDrainWait);
        }
    } else {
        // ---------------- epilogue (both CTAs): warps 2..9, a TMEM lane quarter (32 columns of out) and every other
        // block of 32 rows each.  TMEM holds out^T, so 32 x 32 blocks go through shared memory transposed (stmatrix
        // .trans) and leave as 64-byte runs of a row, 16 bytes a lane.
        const int q = warp & 3, first_block = (warp - 2) >> 2;
        const uint32_t acce_leader0 = mapa_shared(smem_u32(&acce_bar[0]), 0);
        const uint32_t acce_leader1 = mapa_shared(smem_u32(&acce_bar[1]), 0);
        const uint32_t buf = sEpi + (uint32_t)((warp - 2) * kEpiBytes);
        // block row j is 64 bytes; its 16-byte piece i stands at i ^ ((j >> 1) & 3), free of bank conflicts both ways
        const uint32_t st_row = buf + (uint32_t)((lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) * 16));
        const uint32_t ld_row = buf + (uint32_t)((lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) * 16));
        int t_local = 0;
        for (int tile = pair; tile < num_tiles; tile += num_pairs, ++t_local) {
            const ProductTile p = product_tile(tile, groups, num_n, table);
            const int acc = t_local & 1;
            bool ok = mbar_wait_cluster(smem_u32(&accf_bar[acc]), (uint32_t)(t_local >> 1) & 1u, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0) {
                    atomicCAS(&g_grouped_error, 0, kErrEpilogueWait);
                    abort_flag = 1;
                }
                break;
            }
            tc_fence_after();
            const uint32_t t_tile = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * kTileRows);
            const int col = p.n0 + (int)rank * 128 + q * 32 + (lane & 3) * 8;
            uint16_t* out_lane = out + (size_t)(p.row0 + (lane >> 2)) * N + col;
#pragma unroll 1
            for (int c = first_block; c * 32 < p.rows; c += 2) {
                uint32_t lo[16], hi[16];  // TMEM lanes 0..15 and 16..31 of the quarter, 32 rows of out
                tmem_ld_16x256b_x4(t_tile + (uint32_t)(c * 32), lo);
                tmem_ld_16x256b_x4(t_tile + (16u << 16) + (uint32_t)(c * 32), hi);
                tmem_wait_ld();
                __syncwarp();  // the previous block has been read out of buf
#pragma unroll
                for (int j = 0; j < 4; ++j)  // rows 8j .. 8j + 7; columns in octets 0..3
                    stmatrix_x4_trans(st_row + (uint32_t)(j * 8 * 64), pack2<DT>(lo[4 * j], lo[4 * j + 1]),
                                      pack2<DT>(lo[4 * j + 2], lo[4 * j + 3]), pack2<DT>(hi[4 * j], hi[4 * j + 1]),
                                      pack2<DT>(hi[4 * j + 2], hi[4 * j + 3]));
                __syncwarp();
                if (col < N) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = c * 32 + i * 8;
                        if (row + (lane >> 2) < p.rows)
                            *reinterpret_cast<uint4*>(out_lane + (size_t)row * N) =
                                ld_shared_v4(ld_row + (uint32_t)(i * 8 * 64));
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc ? acce_leader1 : acce_leader0);
        }
    }

    // Teardown: the leader's MMAs read the peer's shared memory and write its
    // TMEM, so neither CTA releases TMEM or exits before both are done.
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------------ few tiles: K split over a cluster
// The same transposed product with single CTAs (128 columns of out x up to 64
// rows) when the tiles are too few to occupy the GPU: the CL CTAs of a cluster
// take a tile's K in CL parts, each streaming its own share of the weights.
// CTA r owns columns [128 r / CL, ...) of the tile: the others send it their
// fp32 parts through distributed shared memory, and it adds them in the order
// of K, so the result does not depend on timing.  One tile a cluster.
constexpr int kSplitThreads = 192;  // producer warp, MMA warp, 4 epilogue warps
constexpr int kSplitN = 128;
// Tiles of up to R = 64 rows, or 16: then two CTAs fit an SM, each with its own ring, and one streams while the other
// starts or ends.
template <int R>
struct SplitCfg {
    static constexpr int kStages = R == 64 ? 3 : 2;
    static constexpr int kX = 2 * R * 128;  // two k-blocks of the rows of a
    static constexpr size_t kSmem = (size_t)kStages * (kOperandStage + kX) + R * kSplitN * 4 + 1024;
    static constexpr int kPerSm = R == 64 ? 1 : 2;
};

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

template <int DT>
__device__ __forceinline__ uint16_t round16(float v) {
    if constexpr (DT == TRB_FLOAT16) return __half_as_ushort(__float2half_rn(v));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

template <int DT, bool KB, int R>
__global__ void __launch_bounds__(kSplitThreads, SplitCfg<R>::kPerSm)
    grouped_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                         const int* offsets, uint16_t* out, int groups, int total_rows,
                         int N, int K, int cl) {
    constexpr uint32_t kIdesc = make_idesc<DT>(128, !KB, false);
    constexpr int kSplitStages = SplitCfg<R>::kStages;
    constexpr int kSplitX = SplitCfg<R>::kX;
    constexpr int kSplitRows = R;
    constexpr int kTmemSplit = R < 32 ? 32 : R;

    extern __shared__ uint8_t smem_raw[];
    __shared__ int group_words[3 * kMaxGroups + 1];
    __shared__ __align__(8) uint64_t full_bar[kSplitStages];
    __shared__ __align__(8) uint64_t empty_bar[kSplitStages];
    __shared__ __align__(8) uint64_t done_bar;  // all products of the tile
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;

    const uint32_t sW = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sX = sW + kSplitStages * kOperandStage;
    const uint32_t receive = sX + kSplitStages * kSplitX;

    const uint32_t rank = cluster_ctarank();
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int num_n = (N + kSplitN - 1) / kSplitN;
    const int num_kb = (K + kBK - 1) / kBK;
    const GroupTable table = {group_words, group_words + kMaxGroups, group_words + 2 * kMaxGroups};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kSplitStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&done_bar), 1);
        abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), kTmemSplit);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    grid_launch_dependents();  // after the allocation, as above
    grid_dependency_wait();
    groups = load_groups(offsets, groups, total_rows, table, &g_grouped_error);
    if (warp == 0) scan_chunks(groups, kSplitRows, table, lane);
    __syncthreads();
    const int tile = blockIdx.x / cl;
    if (tile >= table.chunk0[groups] * num_n) {  // the whole cluster: the grid covers the most tiles there can be
        if (warp == 1) tmem_dealloc(tmem_base, kTmemSplit);
        return;
    }

    const int chunk = tile / num_n;
    const int e = group_of_chunk(chunk, groups, table);
    const int first = (chunk - table.chunk0[e]) * kSplitRows;
    const int row0 = table.start[e] + first;
    const int rows = min(kSplitRows, table.rows[e] - first);
    const int padded = (rows + 15) & ~15;
    const int n0 = (tile - chunk * num_n) * kSplitN;
    const int kb0 = num_kb * (int)rank / cl, kb1 = num_kb * ((int)rank + 1) / cl;

    cluster_arrive();  // peers may not write here before this CTA runs; the wait is before the first such write

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer
            uint32_t stage = 0, phase = 0;
            int issued = 0;
            for (int kb = kb0; kb < kb1; kb += 2) {
                if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, &abort_flag)) {
                    atomicCAS(&g_grouped_error, 0, kErrProducerWait);
                    abort_flag = 1;
                    break;
                }
                const int blocks = min(2, kb1 - kb);
                const uint32_t bar = smem_u32(&full_bar[stage]);
                const uint32_t w = sW + stage * kOperandStage, x = sX + stage * kSplitX;
                mbar_arrive_expect_tx(bar, (KB ? blocks * kBlockBytes : kOperandStage) + blocks * (kSplitX / 2));
                if constexpr (!KB) {  // boxes of 128 k: a second k-block past this CTA's share is not multiplied
                    tma_load_3d(w, &tmW, bar, n0, kb * kBK, e);
                    tma_load_3d(w + kBlockBytes, &tmW, bar, n0 + 64, kb * kBK, e);
                }
                for (int i = 0; i < blocks; ++i) {
                    if constexpr (KB) tma_load_3d(w + i * kBlockBytes, &tmW, bar, (kb + i) * kBK, n0, e);
                    tma_load_2d(x + i * (kSplitX / 2), &tmX, bar, (kb + i) * kBK, row0);
                }
                ++issued;
                if (++stage == kSplitStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            for (int i = min(issued, kSplitStages); i > 0; --i) {  // no copy in flight when this CTA ends
                if (stage == 0) {
                    stage = kSplitStages;
                    phase ^= 1u;
                }
                --stage;
                if (!mbar_wait(smem_u32(&full_bar[stage]), phase, nullptr))
                    atomicCAS(&g_grouped_error, 0, kErrDrainWait);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---------------- MMA issuer
            const uint64_t w_desc0 = KB ? make_sdesc(sW, 16, 1024) : make_sdesc(sW, kBlockBytes, 1024);
            const uint64_t x_desc0 = make_sdesc(sX, 16, 1024);
            constexpr int kWStep = KB ? kInstrK * 2 : kInstrK * 128;
            constexpr int kWBlock = KB ? kBlockBytes : kBlockBytes / 2;
            const uint32_t idesc = idesc_n(kIdesc, padded);
            uint32_t stage = 0, phase = 0;
            for (int kb = kb0; kb < kb1; kb += 2) {
                if (!mbar_wait(smem_u32(&full_bar[stage]), phase, &abort_flag)) {
                    atomicCAS(&g_grouped_error, 0, kErrMmaWait);
                    abort_flag = 1;
                    break;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (kb + i >= kb1) break;
#pragma unroll
                    for (int ks = 0; ks < kBK / kInstrK; ++ks)
                        mma_f16(tmem_base,
                                w_desc0 + (uint64_t)((stage * kOperandStage + i * kWBlock + ks * kWStep) >> 4),
                                x_desc0 + (uint64_t)((stage * kSplitX + i * (kSplitX / 2) + ks * kInstrK * 2) >> 4),
                                idesc, (kb != kb0 || i != 0 || ks != 0) ? 1u : 0u);
                }
                tc_commit(smem_u32(&empty_bar[stage]));
                if (++stage == kSplitStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            tc_commit(smem_u32(&done_bar));
            if (!mbar_wait(smem_u32(&done_bar), 0, nullptr)) atomicCAS(&g_grouped_error, 0, kErrDrainWait);
        }
    }
    __syncwarp();
    cluster_wait();  // every CTA of the cluster runs
    const int own = kSplitN / cl;  // columns this CTA owns
    if (warp >= 2) {
        // ---------------- epilogue: lane = column of out, TMEM column = row
        const int q = warp & 3;
        const int n = q * 32 + lane;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&done_bar), 0, &abort_flag));
        if (!ok && lane == 0) {
            atomicCAS(&g_grouped_error, 0, kErrEpilogueWait);
            abort_flag = 1;
        }
        if (ok) {
            tc_fence_after();
            const uint32_t owner = mapa_shared(receive, (uint32_t)(n / own)) +
                                   (uint32_t)(((int)rank * kSplitRows * own + n % own) * 4);
            for (int c = 0; c < padded; c += 16) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)c, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (c + i < rows) st_cluster_f32(owner + (uint32_t)((c + i) * own * 4), __uint_as_float(v[i]));
            }
            tc_fence_before();
        }
    }
    // The parts have arrived, and no CTA leaves while a peer may still write into it.
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && ok) {
        for (int i = threadIdx.x - 64; i < rows * own; i += 128) {
            const int r = i / own, c = i - r * own;
            float v = 0.0f;
            for (int src = 0; src < cl; ++src) {
                float p;
                asm volatile("ld.shared.f32 %0, [%1];"
                             : "=f"(p)
                             : "r"(receive + (uint32_t)(((src * kSplitRows + r) * own + c) * 4)));
                v += p;
            }
            const int n = n0 + (int)rank * own + c;
            if (n < N) out[(size_t)(row0 + r) * N + n] = round16<DT>(v);
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemSplit);
    }
}

// ------------------------------------------------------------------ out[e] = a^T * g over the rows of e
// A CTA pair computes 256 x 256 of one group's K x N gradient; the products run
// over the group's rows, 128 per stage, both operands MN-major (their rows are
// the contraction).  The last stage of a group reaches into the next group's
// rows (or past the end, where TMA gives zeros): products run over whole
// 16-row steps only as far as the group goes, and the rows between its end and
// the end of that step are overwritten with zeros in both operands first, so
// that nothing of the next group, infinities and NaN included, gets in.  Such
// a stage lands on a barrier of its own CTA; a fixer warp clears the rows and
// then signals the leader's full barrier.
// A group without rows has a gradient of zeros, which the epilogue writes.
// Measured: 32768 rows, 8 groups, 4096 x 4096, 870 to 910 us, 1210 to 1260
// TFLOP/s under the power cap; 8111 rows, 64 groups, 2048 x 1544, 125 us in a
// burst at 1965 MHz and 140 sustained, bound by reading out tiles of two stages
// each, a seventh column of them for 8 columns (1536 columns: 109 us, 1552: 123;
// zeros alone 64 and 71 us for 1536 and 1544).  4 bytes spill at 168 registers.
struct WgradTile {
    int e, row0, rows, m0, n0;
};

__device__ __forceinline__ WgradTile wgrad_tile(int t, int num_m, int num_n, const int* offsets) {
    const int per = num_m * num_n;
    WgradTile w;
    w.e = t / per;
    w.row0 = offsets[w.e];
    w.rows = offsets[w.e + 1] - w.row0;
    const int local = t - w.e * per;
    const int run = 8 * num_m;
    const int first = local / run * 8;
    const int width = min(8, num_n - first);
    const int in_run = local - first * num_m;
    w.n0 = (first + in_run % width) * 256;  // runs of 8 tiles along a row of the gradient
    w.m0 = in_run / width * 256;
    return w;
}

constexpr int kWgradThreads = kThreads + 32;  // and the fixer warp
constexpr int kWgradBox = 8 * 512;               // 8 rows x 256 results of the gradient
constexpr size_t kWgradSmem = kRingBytes + 1024 + kEpiWarps * kWgradBox;
constexpr int kStageRows = 2 * kBK;

template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWgradThreads, 1)
    grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmG,
                         const __grid_constant__ CUtensorMap tmA64, const __grid_constant__ CUtensorMap tmG64,
                         const int* offsets, uint16_t* out, int groups, int total_rows, int N,
                         int K) {
    constexpr uint32_t kIdesc = make_idesc<DT>(256, true, true) | ((uint32_t)(256 >> 3) << 17);
    constexpr uint32_t kBox = kBlockBytes;  // place of a box of 64 columns x up to 128 rows

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kStages];   // leader: the stage is ready in both CTAs
    __shared__ __align__(8) uint64_t part_bar[kStages];   // both: this CTA's bytes of a stage to be fixed have landed
    __shared__ __align__(8) uint64_t empty_bar[kStages];  // both: MMA finished reading the stage
    __shared__ __align__(8) uint64_t accf_bar[kNumAcc];
    __shared__ __align__(8) uint64_t acce_bar[kNumAcc];
    __shared__ __align__(8) uint64_t drain_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    __shared__ volatile int issued;  // stages that this CTA's producer has asked for (may wrap: only changes count)

    const uint32_t sA = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sG = sA + kStages * kOperandStage;
    const uint32_t sEpi = sG + kStages * kOperandStage;

    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    const int num_m = (K + 255) / 256;
    const int num_n = (N + 255) / 256;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 2);  // leader's producer twice, or one fixer per CTA
            mbar_init(smem_u32(&part_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int a = 0; a < kNumAcc; ++a) {
            mbar_init(smem_u32(&accf_bar[a]), 1);
            mbar_init(smem_u32(&acce_bar[a]), 8);  // the four warps that read it, of both CTAs
        }
        mbar_init(smem_u32(&drain_bar), 1);
        abort_flag = 0;
        issued = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmG);
    }
    if (warp == 0) {
        tmem_alloc_pair(smem_u32(&tmem_slot), kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = tmem_slot;
    grid_launch_dependents();  // after the allocation, as above
    grid_dependency_wait();
    groups = check_groups(offsets, groups, total_rows, &g_grouped_error);
    const int num_tiles = groups * num_m * num_n;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer
            uint32_t stage = 0, phase = 0;
            uint32_t issued_mask = 0, issued_phase = 0;
            uint32_t stages_issued = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
                const WgradTile w = wgrad_tile(tile, num_m, num_n, offsets);
                const int a_col = w.m0 + (int)rank * 128, g_col = w.n0 + (int)rank * 128;
                for (int done = 0; done < w.rows; done += kStageRows) {
                    if (!mbar_wait_cluster(smem_u32(&empty_bar[stage]), phase ^ 1u, &abort_flag)) {
                        atomicCAS(&g_grouped_error, 0, kErrProducerWait);
                        abort_flag = 1;
                        ok = false;
                        break;
                    }
                    const int left = w.rows - done;
                    const CUtensorMap* mapA = left > kBK ? &tmA : &tmA64;  // boxes of 128 or 64 rows
                    const CUtensorMap* mapG = left > kBK ? &tmG : &tmG64;
                    const uint32_t bytes = left > kBK ? 4 * kBox : 2 * kBox;  // of this CTA
                    const bool fix = left < kStageRows && left % kInstrK != 0;
                    const uint32_t a = sA + stage * kOperandStage, g = sG + stage * kOperandStage;
                    const int row = w.row0 + done;
                    if (fix) {
                        const uint32_t bar = smem_u32(&part_bar[stage]);
                        mbar_arrive_expect_tx(bar, bytes);
                        tma_load_2d(a, mapA, bar, a_col, row);
                        tma_load_2d(a + kBox, mapA, bar, a_col + 64, row);
                        tma_load_2d(g, mapG, bar, g_col, row);
                        tma_load_2d(g + kBox, mapG, bar, g_col + 64, row);
                    } else {
                        const uint32_t fb_local = smem_u32(&full_bar[stage]);
                        if (leader) {
                            mbar_arrive_expect_tx(fb_local, 2 * bytes);
                            mbar_arrive(fb_local);
                        }
                        const uint32_t fb = fb_local & kPeerBitMask;
                        tma_load_2d_pair(a, mapA, fb, a_col, row);
                        tma_load_2d_pair(a + kBox, mapA, fb, a_col + 64, row);
                        tma_load_2d_pair(g, mapG, fb, g_col, row);
                        tma_load_2d_pair(g + kBox, mapG, fb, g_col + 64, row);
                    }
                    issued = (int)++stages_issued;
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (leader)  // every armed phase completes only once both CTAs' bytes have landed
                for (int s = 0; s < kStages; ++s)
                    if (issued_mask & (1u << s))
                        if (!mbar_wait_cluster(smem_u32(&full_bar[s]), (issued_phase >> s) & 1u, nullptr))
                            atomicCAS(&g_grouped_error, 0, kErrDrainWait);
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            // ---------------- MMA issuer
            const uint64_t a_desc0 = make_sdesc(sA, kBox, 1024);
            const uint64_t g_desc0 = make_sdesc(sG, kBox, 1024);
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            int t_local = 0;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
                const WgradTile w = wgrad_tile(tile, num_m, num_n, offsets);
                if (w.rows == 0) continue;
                const int acc = t_local & 1;
                if (!mbar_wait_cluster(smem_u32(&acce_bar[acc]), ((uint32_t)(t_local >> 1) & 1u) ^ 1u, &abort_flag)) {
                    atomicCAS(&g_grouped_error, 0, kErrMmaWait);
                    abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(acc * 256);
                for (int done = 0; done < w.rows; done += kStageRows) {
                    if (!mbar_wait_cluster(smem_u32(&full_bar[stage]), phase, &abort_flag)) {
                        atomicCAS(&g_grouped_error, 0, kErrMmaWait);
                        abort_flag = 1;
                        ok = false;
                        break;
                    }
                    const uint64_t off = (uint64_t)((stage * kOperandStage) >> 4);
                    const int left = w.rows - done;
#pragma unroll
                    for (int ks = 0; ks < kStageRows / kInstrK; ++ks) {
                        if (ks * kInstrK >= left) break;
                        const uint64_t o = off + (uint64_t)(ks * kInstrK * 128 >> 4);
                        mma_pair_f16(d_tmem, a_desc0 + o, g_desc0 + o, kIdesc, (done != 0 || ks != 0) ? 1u : 0u);
                    }
                    tc_commit_pair_multicast(smem_u32(&empty_bar[stage]), 0x3);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) tc_commit_pair_multicast(smem_u32(&accf_bar[acc]), 0x3);
                ++t_local;
            }
            tc_commit_pair_multicast(smem_u32(&drain_bar), 0x1);
            if (!mbar_wait_cluster(smem_u32(&drain_bar), 0, nullptr)) atomicCAS(&g_grouped_error, 0, kErrDrainWait);
        }
    } else if (warp == kWgradThreads / 32 - 1) {
        // ---------------- fixer (both CTAs): zeros behind a group's last row
        const uint32_t full_leader0 = mapa_shared(smem_u32(&full_bar[0]), 0);
        uint32_t stage = 0, part_phase = 0;  // part_phase: bit s = parity of part_bar[s]'s next use
        bool ok = true;
        for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
            const WgradTile w = wgrad_tile(tile, num_m, num_n, offsets);
            const int stages = (w.rows + kStageRows - 1) / kStageRows;
            const int left = w.rows - (stages - 1) * kStageRows;  // rows of the last stage
            if (stages > 0 && left % kInstrK != 0) {
                const uint32_t s = (stage + (uint32_t)(stages - 1)) % kStages;
                // from the start of the call on, if no tile before had rows to clear
                ok = mbar_wait_progress(smem_u32(&part_bar[s]), (part_phase >> s) & 1u, &abort_flag, &issued);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) {
                    if (lane == 0) {
                        atomicCAS(&g_grouped_error, 0, kErrProducerWait);
                        abort_flag = 1;
                    }
                    break;
                }
                part_phase ^= 1u << s;
                const int pieces = (((left + kInstrK - 1) & ~(kInstrK - 1)) - left) * 8;  // 16-byte pieces per box
                const uint32_t first = sA + s * kOperandStage + (uint32_t)left * 128;
                for (int i = lane; i < pieces; i += 32) {
                    const uint32_t at = first + (uint32_t)i * 16;
                    st_shared_v4(at, 0, 0, 0, 0);
                    st_shared_v4(at + kBox, 0, 0, 0, 0);
                    st_shared_v4(at + (sG - sA), 0, 0, 0, 0);
                    st_shared_v4(at + (sG - sA) + kBox, 0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(full_leader0 + s * 8);
            }
            stage = (stage + (uint32_t)stages) % kStages;
        }
    } else {
        // ---------------- epilogue (both CTAs): warps 2..5 read the first accumulator, warps 6..9 the second, 32
        // rows of the tile each, so that one tile is read out of TMEM while another waits on its stores.  8 x 256
        // results at a time go through shared memory (stmatrix) and leave as whole rows of the tile, 512 bytes a
        // store: where N is not a multiple of 16, rows begin in the middle of a sector and each end of a run writes
        // a part of one (64 zero gradients of 2048 x 1544: 133 us in runs of 128 bytes, 100 in longer ones, 71 with
        // the tiles of a row of the gradient next to each other in time; 64 us for 2048 x 1536).  60 gradients of
        // 127 rows on average, in bursts: 152 us with one group of eight warps, 132 with a group for each
        // accumulator, 129 with whole rows, 126 in that tile order; 133 with the stores moved to sector boundaries,
        // 182 with sixteen warps and runs of 256 bytes.
        const int q = warp & 3, group = (warp - 2) >> 2;
        const uint32_t acce_leader = mapa_shared(smem_u32(&acce_bar[group]), 0);
        const uint32_t t_rows = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(group * 256);
        const uint32_t buf = sEpi + (uint32_t)((warp - 2) * kWgradBox);
        // 16-byte piece i of row r stands at i ^ (r & 7), free of bank conflicts both ways
        const uint32_t st_row = buf + (uint32_t)((lane & 7) * 512);
        int t_local = 0, empty = 0;  // tiles with products, and without
        for (int tile = pair; tile < num_tiles; tile += num_pairs) {
            const WgradTile w = wgrad_tile(tile, num_m, num_n, offsets);
            const bool products = w.rows > 0;
            const int count = products ? t_local++ : empty++;
            if ((count & 1) != group) continue;
            if (products) {
                // for all stages of a tile, or of two
                bool ok = mbar_wait_progress(smem_u32(&accf_bar[group]), (uint32_t)(count >> 1) & 1u, &abort_flag,
                                             &issued);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) {
                    if (lane == 0) {
                        atomicCAS(&g_grouped_error, 0, kErrEpilogueWait);
                        abort_flag = 1;
                    }
                    break;
                }
                tc_fence_after();
            }
            const int row0 = w.m0 + (int)rank * 128 + q * 32;
            const int col = w.n0 + lane * 8;
#pragma unroll
            for (int b = 0; b < 2; ++b) {  // rows 16 b of the 32
                uint32_t packed[8][8];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t r[4][16];
                    if (products) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tmem_ld_16x256b_x4(t_rows + ((uint32_t)(b * 16) << 16) + (uint32_t)(c * 128 + j * 32), r[j]);
                        tmem_wait_ld();
                        if (b == 1 && c == 1) {  // the accumulator is read out: the next tile but one may have it
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_cluster(acce_leader);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            packed[c * 4 + j][i] = products ? pack2<DT>(r[j][2 * i], r[j][2 * i + 1]) : 0;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row_h = row0 + b * 16 + h * 8;
                    if (row_h >= K) continue;  // warp-uniform: outside the gradient
                    __syncwarp();  // the rows before have been read out of buf
#pragma unroll
                    for (int j = 0; j < 8; ++j)  // column octets 4j .. 4j + 3
                        stmatrix_x4(st_row + (uint32_t)(((j * 4 + (lane >> 3)) ^ (lane & 7)) * 16), packed[j][h],
                                    packed[j][2 + h], packed[j][4 + h], packed[j][6 + h]);
                    __syncwarp();
                    uint16_t* dst = out + ((size_t)w.e * K + row_h) * N + col;
                    if (col < N) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (row_h + i < K)
                                *reinterpret_cast<uint4*>(dst + (size_t)i * N) =
                                    ld_shared_v4(buf + (uint32_t)(i * 512 + ((lane ^ i) * 16)));
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ------------------------------------------------------------------ host side
// Checks shared by both products.
static int check(const char* what, int dtype, int groups, int rows, int n, int k, const void* p0, const void* p1,
                 const void* p2, const int* offsets) {
    if (groups <= 0 || rows < 0 || n <= 0 || k <= 0 || offsets == nullptr ||
        (rows > 0 && (p0 == nullptr || p1 == nullptr || p2 == nullptr))) {
        set_error("%s: sizes must be positive (rows may be 0) and pointers non-null", what);
        return TRB_ERR_ARGS;
    }
    if (dtype != TRB_BFLOAT16 && dtype != TRB_FLOAT16) {
        set_error("%s: unsupported dtype %s (bfloat16 and float16)", what, dtype_name(dtype));
        return TRB_SKIPPED;
    }
    if (groups > kMaxGroups) {
        set_error("%s: at most %d groups (got %d)", what, kMaxGroups, groups);
        return TRB_SKIPPED;
    }
    if (std::max({rows, n, k}) > kMaxExtent) {
        set_error("%s: rows, n and k at most %d (rows=%d n=%d k=%d)", what, kMaxExtent, rows, n, k);
        return TRB_SKIPPED;
    }
    if (n % 8 != 0 || k % 8 != 0) {
        set_error("%s: n and k must be multiples of 8 (n=%d k=%d)", what, n, k);
        return TRB_ERR_ALIGN;
    }
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p0) | reinterpret_cast<uintptr_t>(p1) |
                           reinterpret_cast<uintptr_t>(p2);
    if ((bits & 15u) != 0 || (reinterpret_cast<uintptr_t>(offsets) & 3u) != 0) {
        set_error("%s: matrices must be 16-byte aligned and offsets 4-byte aligned", what);
        return TRB_ERR_ALIGN;
    }
    return TRB_OK;
}

static int pairs_for(int64_t tiles, int dev) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(tiles, device_sm_count(dev) / 2));
}

template <int DT, bool KB>
static int launch_product(int groups, int rows, int n, int k, const void* a, const void* b, const int* offsets,
                          void* out, int dev, cudaStream_t stream) {
    static bool attr_set[64] = {};
    CUtensorMap tmW, tmX128, tmX64, tmX32;
    const uint64_t we[3] = {(uint64_t)(KB ? k : n), (uint64_t)(KB ? n : k), (uint64_t)groups};
    const uint32_t wb[3] = {64, 128, 1};  // KB: 64 k x 128 n, else 64 n x 128 k
    const uint64_t xe[2] = {(uint64_t)k, (uint64_t)rows};
    const uint32_t xb128[2] = {64, 128}, xb64[2] = {64, 64}, xb32[2] = {64, 32}, xb16[2] = {64, 16};
    int rc = gemm::encode_tiled(&tmW, b, 2, 3, we, wb, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != TRB_OK) return rc;
    // Tiles of 128 columns, K split over clusters, where that gives every CTA a place at once: 2 rows, 2 of 8 groups,
    // 2048 x 1024, 6.5 us against the pair's 13.0; 60 rows, 16 groups, 1024 x 1408, 14.1 against 15.6.  More tiles than
    // places: the pair (96 rows, 32 groups, 2048 x 1408: 36 us against 40).  Up to 4 rows a group, tiles of 16 rows and
    // two CTAs an SM (2 rows as above: 6.5 against 9.0 us); more rows make more tiles of 16 (40 rows, 8 groups, 4096 x
    // 1024: 16.0 against 13.2 us).  One cluster more than fit at once is a second round of the whole time: 50 rows, K =
    // 4096, 16 tiles take 16.3 us in clusters of 8 and 11.5 of 4, 34 tiles 23.4 of 4 and 17.8 of 2; 3 rows, 72 tiles 22.9
    // of 4 and 18.3 of 2.
    const bool few = rows <= 4 * (int64_t)std::min(groups, rows);
    const int split_rows = few ? 16 : 64;
    const auto split_kernel = few ? grouped_split_kernel<DT, KB, 16> : grouped_split_kernel<DT, KB, 64>;
    const size_t split_smem = few ? SplitCfg<16>::kSmem : SplitCfg<64>::kSmem;
    static bool split_attr_set[2][64] = {};
    const int64_t split_tiles = (int64_t)((n + kSplitN - 1) / kSplitN) * (rows / split_rows + std::min(groups, rows));
    const int num_kb = (k + kBK - 1) / kBK;
    const auto sm_places = [&](int log2_cl) {  // of clusters with one CTA an SM
        static int places[4][64] = {};
        return clusters_at_once(grouped_split_kernel<DT, KB, 64>, kSplitThreads, SplitCfg<64>::kSmem, 1 << log2_cl, dev,
                                places[log2_cl]);
    };
    // With two CTAs an SM the driver still answers for one.  Twice as many clusters fit for certain, and at most as many
    // as clusters half the size with one; on 148 SMs 33 of 8 do (30 and 33), 71 of 4 (66 and 74) and 148 of 2 (148).
    const auto fits = [&](int log2_cl) {
        const int sure = (few ? 2 : 1) * sm_places(log2_cl);
        return split_tiles <= (few && log2_cl > 0 ? (sure + sm_places(log2_cl - 1)) / 2 : sure);
    };
    int log2_cl = 0;
    while (log2_cl < 3 && num_kb >= 4 << log2_cl && fits(log2_cl + 1)) ++log2_cl;
    if (log2_cl > 0 || (few && fits(0))) {
        rc = gemm::encode_tiled(&tmX32, a, 2, 2, xe, few ? xb16 : xb64, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc != TRB_OK) return rc;
        const int cl = 1 << log2_cl;
        return launch_kernel(split_kernel, (int)split_tiles * cl, kSplitThreads, cl, split_smem, dev,
                             split_attr_set[few], stream, tmW, tmX32, offsets, static_cast<uint16_t*>(out), groups, rows, n,
                             k, cl);
    }
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmX128, a, 2, 2, xe, xb128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmX64, a, 2, 2, xe, xb64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmX32, a, 2, 2, xe, xb32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != TRB_OK) return rc;
    const int64_t num_n = (n + kTileN - 1) / kTileN;
    const int64_t tiles = num_n * ((int64_t)rows / kTileRows + std::min(groups, rows));
    if (tiles > INT32_MAX) {
        set_error("trb_grouped_gemm_launch: too many tiles (rows=%d n=%d groups=%d)", rows, n, groups);
        return TRB_SKIPPED;
    }
    return launch_kernel(grouped_gemm_kernel<DT, KB>, 2 * pairs_for(tiles, dev), kThreads, 0, kProductSmem, dev,
                         attr_set, stream, tmW, tmX128, tmX64, tmX32, offsets, static_cast<uint16_t*>(out), groups, rows, n, k);
}

template <int DT>
static int launch_wgrad(int groups, int rows, int n, int k, const void* a, const void* g, const int* offsets,
                        void* out, int dev, cudaStream_t stream) {
    static bool attr_set[64] = {};
    CUtensorMap tmA, tmG, tmA64, tmG64;
    // Without rows no operand is read; the maps then stand on the output, which is there.
    const uint64_t extent_rows = (uint64_t)std::max(rows, 1);
    const uint64_t ae[2] = {(uint64_t)k, extent_rows}, ge[2] = {(uint64_t)n, extent_rows};
    const uint32_t box[2] = {64, kStageRows}, box64[2] = {64, 64};
    const void *pa = rows > 0 ? a : out, *pg = rows > 0 ? g : out;
    int rc = gemm::encode_tiled(&tmA, pa, 2, 2, ae, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmG, pg, 2, 2, ge, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmA64, pa, 2, 2, ae, box64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TRB_OK) rc = gemm::encode_tiled(&tmG64, pg, 2, 2, ge, box64, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != TRB_OK) return rc;
    const int64_t tiles = (int64_t)groups * ((k + 255) / 256) * ((n + 255) / 256);
    if (tiles > INT32_MAX) {
        set_error("trb_grouped_wgrad_launch: too many tiles (groups=%d n=%d k=%d)", groups, n, k);
        return TRB_SKIPPED;
    }
    return launch_kernel(grouped_wgrad_kernel<DT>, 2 * pairs_for(tiles, dev), kWgradThreads, 0, kWgradSmem, dev,
                         attr_set, stream, tmA, tmG, tmA64, tmG64, offsets, static_cast<uint16_t*>(out), groups, rows, n, k);
}

int read_error(bool clear) {
    int v = 0;
    TRB_CUDA(cudaMemcpyFromSymbol(&v, g_grouped_error, sizeof(int)));
    if (clear) {
        const int zero = 0;
        TRB_CUDA(cudaMemcpyToSymbol(g_grouped_error, &zero, sizeof(int)));
    }
    return v;
}

}  // namespace grouped
}  // namespace trb

extern "C" int trb_grouped_gemm_launch(int dtype, int groups, int rows, int n, int k, const void* a, const void* b,
                                       int b_layout, const int32_t* offsets, void* out, void* stream) {
    using namespace trb;
    clear_error();
    int rc = grouped::check("trb_grouped_gemm_launch", dtype, groups, rows, n, k, a, b, out, offsets);
    if (rc != TRB_OK) return rc;
    if (b_layout != TRB_B_ROW_MAJOR && b_layout != TRB_B_K_MAJOR) {
        set_error("trb_grouped_gemm_launch: unknown b_layout %d", b_layout);
        return TRB_ERR_ARGS;
    }
    if (rows == 0) return TRB_OK;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool kb = b_layout == TRB_B_K_MAJOR;
    if (dtype == TRB_BFLOAT16)
        return kb ? grouped::launch_product<TRB_BFLOAT16, true>(groups, rows, n, k, a, b, offsets, out, dev, s)
                  : grouped::launch_product<TRB_BFLOAT16, false>(groups, rows, n, k, a, b, offsets, out, dev, s);
    return kb ? grouped::launch_product<TRB_FLOAT16, true>(groups, rows, n, k, a, b, offsets, out, dev, s)
              : grouped::launch_product<TRB_FLOAT16, false>(groups, rows, n, k, a, b, offsets, out, dev, s);
}

extern "C" int trb_grouped_wgrad_launch(int dtype, int groups, int rows, int n, int k, const void* a, const void* g,
                                        const int32_t* offsets, void* out, void* stream) {
    using namespace trb;
    clear_error();
    const int rc = grouped::check("trb_grouped_wgrad_launch", dtype, groups, rows, n, k, a, g, out, offsets);
    if (rc != TRB_OK) return rc;
    if (out == nullptr) {
        set_error("trb_grouped_wgrad_launch: out is null");
        return TRB_ERR_ARGS;
    }
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == TRB_BFLOAT16
               ? grouped::launch_wgrad<TRB_BFLOAT16>(groups, rows, n, k, a, g, offsets, out, dev, s)
               : grouped::launch_wgrad<TRB_FLOAT16>(groups, rows, n, k, a, g, offsets, out, dev, s);
}
