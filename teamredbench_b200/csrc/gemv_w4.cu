// gemv_w4.cu -- few rows times matrices of 4-bit weights with a scale per group of k.
//
//   out[r, n] = sum over groups g of k:  s[e, n, g] * sum over k in g of x[r, k] * (q[e, n, k] - z[e, n, g])
//
// for the rows r of expert e (one expert: a plain matrix).  q is stored two to
// a byte along k, the low four bits first.
//
// The bytes of q bound it: 1/2 byte per weight, read once for up to 8 (16)
// rows of x.  The products run on mma.sync m16n8k16, 16 outputs x 8 rows of x
// per instruction -- at one row the tensor pipe still does with one
// instruction per 256 weights what would take 256 FMA lanes, and the exact
// products of small whole numbers with 16-bit x accumulate in fp32.  Weights
// become 16-bit floats by bit operations: a 4-bit q ORed into the mantissa of
// 128 is 128 + q exactly, and subtracting 128 + z is exact too, so nothing is
// rounded before the product, and the scale is applied in fp32 to each
// group's sum.
//
// A CTA takes rows of 16 outputs of one group in jobs.  The boxes of a job (16
// outputs x 256 k, 128 bytes of q a row) are one sequence, cut evenly among the
// 16 warps, so a warp works through neighbouring boxes of one or two rows
// whatever k is, with nothing to wait for but its own boxes: they come by TMA
// through a private ring.  What a warp has summed of a row goes to shared
// memory when it leaves the row, and at the job's end the parts of each row are
// added in the order of k.
//
// No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "trb_common.cuh"
#include "trb_groups.cuh"

namespace trb {
namespace w4 {

__device__ int g_w4_error;

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;    // outputs of a box
constexpr int kBoxK = 256;   // k of a box: one 128-byte swizzle row
constexpr int kBlockK = 32;  // k of a block: 16 bytes a row, two products
constexpr uint32_t kBoxBytes = kRows * 128;
constexpr int kMaxDepth = 8;

// Scales a thread holds of a unit (see the kernel) for groups that span gb blocks.
__host__ __device__ constexpr int held_scales(int gb) { return gb <= 2 ? 4 : gb == 4 ? 2 : 1; }
constexpr int kJobRows = 16;  // rows of 16 outputs in a job, at most

struct Shape {
    int groups, rows, n, k;
    int k_groups;       // scales per output
    int group_log2;
    int depth;          // boxes in each warp's ring
    int tokens;         // rows of x taken at once
};

template <int DT>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == TRB_BFLOAT16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
            "%2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
            "%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Pair p of a word of eight q: (q[p], q[p + 4]) as two 16-bit floats.  bf16: 128 + q each.  f16 has mantissa bits
// enough to take q where it stands in the word or its upper half: 1024 + q for even p, 64 + q for odd p.
// One lop3 for the mask and the exponent together (written as & and |, it became two).
__device__ __forceinline__ uint32_t mask_or(uint32_t v, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
    return r;
}
template <int DT>
__device__ __forceinline__ void biased_pairs(uint32_t w, uint32_t (&pair)[4]) {
    if constexpr (DT == TRB_BFLOAT16) {
#pragma unroll
        for (int p = 0; p < 4; ++p) pair[p] = mask_or(w >> (4 * p), 0x000F000Fu, 0x43004300u);
    } else {
        pair[0] = mask_or(w, 0x000F000Fu, 0x64006400u);
        pair[1] = mask_or(w, 0x00F000F0u, 0x54005400u);
        pair[2] = mask_or(w >> 8, 0x000F000Fu, 0x64006400u);
        pair[3] = mask_or(w >> 8, 0x00F000F0u, 0x54005400u);
    }
}
// Byte i of four zero points as two equal 16-bit floats with the same bias, for even and odd pairs.
template <int DT>
__device__ __forceinline__ void biased_zeros(uint32_t bytes, int i, uint32_t& even, uint32_t& odd) {
    const uint32_t twice = 0x4040u + 0x0101u * (uint32_t)i;
    if constexpr (DT == TRB_BFLOAT16) {
        even = odd = __byte_perm(bytes, 0x43u, twice);
    } else {
        even = __byte_perm(bytes, 0x64u, twice);
        odd = __byte_perm(bytes << 4, 0x54u, twice);
    }
}
template <int DT>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    if constexpr (DT == TRB_BFLOAT16) {
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    } else {
        __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<uint32_t*>(&r);
    }
}
template <int DT>
__device__ __forceinline__ float scale_of(uint32_t pair, int i) {  // the lower or upper 16 bits
    if constexpr (DT == TRB_BFLOAT16) return __uint_as_float(i ? pair & 0xFFFF0000u : pair << 16);
    else return __half2float(__ushort_as_half((unsigned short)(i ? pair >> 16 : pair & 0xFFFFu)));
}
template <int DT>
__device__ __forceinline__ uint16_t round16(float v) {
    if constexpr (DT == TRB_BFLOAT16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    else return __half_as_ushort(__float2half_rn(v));
}

// Rows of 16 outputs [row, row + rows) of group e for the rows of x in chunk q, and a warp's share of their boxes:
// boxes [p, p_end) of the job's sequence, the first of them box `box` of row `p_row`.
struct Job {
    int first;  // in the count of all rows of outputs of all chunks
    int rows, row, q, e;
    int p, p_end, p_row, box;
};

// NT * 8 rows of x at once; a group of k spans GB blocks (8: a box or more); Z: zero points given; V: scales and zero
// points may be read kHeld at a time.
template <int DT, int NT, int GB, bool Z, bool V>
__global__ void __launch_bounds__(kThreads, 1)
    gemv_w4_kernel(const __grid_constant__ CUtensorMap tmQ, const uint16_t* __restrict__ x,
                   const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros,
                   const int* __restrict__ offsets, uint16_t* __restrict__ out, const Shape sh) {
    // Scales travel in units: the groups of kUnit boxes of each output, kHeld of them in each of its four threads.
    constexpr int kUnit = GB == 1 ? 2 : 4;
    constexpr int kHeld = held_scales(GB);

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kWarps * kMaxDepth];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int num_box = (sh.k + kBoxK - 1) / kBoxK;
    const int rows_n = (sh.n + kRows - 1) / kRows;

    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t ring = (uint32_t)(warp * sh.depth) * kBoxBytes;             // offsets into smem
    const uint32_t xs = (uint32_t)(kWarps * sh.depth) * kBoxBytes;
    float* red = reinterpret_cast<float*>(smem + xs + (size_t)num_box * 512 * sh.tokens);
    const int part = sh.tokens * kRows;                                        // one warp's sums of a row
    int* words = reinterpret_cast<int*>(red + (kWarps + kJobRows) * part);
    const GroupTable table = {words, words + sh.groups, words + 2 * sh.groups};
    const uint32_t ring_addr = smem_u32(smem) + ring;
    const uint32_t bars = smem_u32(&full_bar[warp * kMaxDepth]);

    if (lane == 0) {
        for (int s = 0; s < sh.depth; ++s) mbar_init(bars + s * 8, 1);
        fence_mbar_init();
        if (warp == 0) tma_prefetch_desc(&tmQ);
    }
    grid_launch_dependents();
    grid_dependency_wait();
    int groups = sh.groups;
    if (offsets != nullptr) {
        groups = load_groups(offsets, sh.groups, sh.rows, table, &g_w4_error);
    } else if (threadIdx.x == 0) {
        table.start[0] = 0;
        table.rows[0] = sh.rows;
    }
    __syncthreads();
    if (warp == 0) scan_chunks(groups, sh.tokens, table, lane);
    __syncthreads();

    // This CTA's share of the rows of outputs, contiguous so that x stays in shared memory.
    const int64_t total = (int64_t)table.chunk0[groups] * rows_n;
    const int end = (int)(total * (blockIdx.x + 1) / gridDim.x);
    auto first_box = [&](int rows, int w) { return rows * num_box * w / kWarps; };
    auto job_at = [&](int first) {
        Job j = {};
        j.first = first;
        if (first >= end) return j;
        j.q = first / rows_n;
        j.row = first - j.q * rows_n;
        j.rows = min(min(end - first, rows_n - j.row), kJobRows);
        j.e = group_of_chunk(j.q, groups, table);
        j.p = first_box(j.rows, warp);
        j.p_end = first_box(j.rows, warp + 1);
        j.p_row = j.p / num_box;
        j.box = j.p - j.p_row * num_box;
        return j;
    };
    auto issue = [&](int box, int row, int e, int slot) {
        if (lane == 0) {
            mbar_arrive_expect_tx(bars + slot * 8, kBoxBytes);
            tma_load_3d(ring_addr + slot * kBoxBytes, &tmQ, bars + slot * 8, box * 128, row * kRows, e);
        }
    };
    // Scales and zero points of the unit that begins at box `box`, for outputs g and g + 8 of row `row`.
    uint32_t sc_next[2][(kHeld + 1) / 2], zr_next[2];
    auto load_unit = [&](int box, int row, int e) {
        const int kg = GB == 1   ? box * 8 + 4 * t
                       : GB == 2 ? (box + t) * 4
                       : GB == 4 ? (box + t) * 2
                                 : ((box + t) * kBoxK) >> sh.group_log2;
        const size_t at0 = ((size_t)e * sh.n + row * kRows + g) * sh.k_groups + kg;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const size_t at = at0 + (size_t)(i * 8 * sh.k_groups);
            const bool in = row * kRows + i * 8 + g < sh.n && kg < sh.k_groups;
            if constexpr (kHeld == 1) {
                sc_next[i][0] = in ? scales[at] : 0;
                if constexpr (Z) zr_next[i] = in ? zeros[at] : 0;
            } else if constexpr (V && kHeld == 4) {  // k_groups is a multiple of kHeld
                const uint2 v = in ? *reinterpret_cast<const uint2*>(scales + at) : make_uint2(0, 0);
                sc_next[i][0] = v.x;
                sc_next[i][1] = v.y;
                if constexpr (Z) zr_next[i] = in ? *reinterpret_cast<const uint32_t*>(zeros + at) : 0;
            } else if constexpr (V) {
                sc_next[i][0] = in ? *reinterpret_cast<const uint32_t*>(scales + at) : 0;
                if constexpr (Z) zr_next[i] = in ? *reinterpret_cast<const uint16_t*>(zeros + at) : 0;
            } else {
                if constexpr (Z) zr_next[i] = 0;
#pragma unroll
                for (int j = 0; j < kHeld; ++j) {
                    const bool in_j = in && kg + j < sh.k_groups;
                    const uint32_t v = (uint32_t)(in_j ? scales[at + j] : 0) << (16 * (j & 1));
                    sc_next[i][j >> 1] = j & 1 ? sc_next[i][j >> 1] | v : v;
                    if constexpr (Z) zr_next[i] |= (uint32_t)(in_j ? zeros[at + j] : 0) << (8 * j);
                }
            }
        }
    };

    int slot = 0, chunk = -1;
    uint32_t phase = 0;
    int tokens = 0, row0 = 0;
    bool failed = false;
    // The place behind the last box requested of the job at hand.
    int a_box = 0, a_row = 0, a_left = 0;
    auto begin = [&](const Job& j) {  // request a job's first boxes (the ring is empty) and scales
        a_box = j.box;
        a_row = j.row + j.p_row;
        a_left = j.p_end - j.p;
        if (a_left == 0) return;
        load_unit(a_box, a_row, j.e);
        for (int s = slot, i = 0; i < sh.depth && a_left > 0; ++i) {
            if (!failed) issue(a_box, a_row, j.e, s);
            if (++s == sh.depth) s = 0;
            --a_left;
            if (++a_box == num_box) {
                a_box = 0;
                ++a_row;
            }
        }
    };

    Job job = job_at((int)(total * blockIdx.x / gridDim.x));
    begin(job);
    while (job.first < end) {
        if (job.q != chunk) {  // other rows of x: in shared memory, [block of 32 k][row][t]: the 8 values of thread t
            chunk = job.q;     // in the order the pairs of a word of q come in
            const int first = (chunk - table.chunk0[job.e]) * sh.tokens;
            row0 = table.start[job.e] + first;
            tokens = min(sh.tokens, table.rows[job.e] - first);
            uint4* x_out = reinterpret_cast<uint4*>(smem + xs);
            for (int c = 0; c < tokens; ++c)
#pragma unroll 2
                for (int j = threadIdx.x; j < num_box * 32; j += kThreads) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (j * 8 < sh.k) v = *reinterpret_cast<const uint4*>(x + (size_t)(row0 + c) * sh.k + j * 8);
                    x_out[((j >> 2) * tokens + c) * 4 + (j & 3)] =
                        make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                   __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
                }
            __syncthreads();
        }
    // Columns of the products past the last row of x are computed from that row and not used.
        const uint32_t x_block = (uint32_t)tokens * 64;
        uint32_t x_lane[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) x_lane[c] = xs + (uint32_t)(min(c * 8 + g, tokens - 1) * 64 + t * 16);

        float sum[NT][4];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[c][i] = 0.0f;
        int box = job.box, row = job.p_row;
        for (int left = job.p_end - job.p; left > 0;) {
            const int boxes = min(min(kUnit, left), num_box - box);
            uint32_t sc[2][(kHeld + 1) / 2], zr[2] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < (kHeld + 1) / 2; ++j) sc[i][j] = sc_next[i][j];
                if constexpr (Z) zr[i] = zr_next[i] & 0x0F0F0F0Fu;
            }
            uint32_t x_at = (uint32_t)(box * 8) * x_block;
            left -= boxes;
            box += boxes;
            const bool row_done = box == num_box;
            if (row_done) box = 0;
            if (left > 0) load_unit(box, job.row + row + row_done, job.e);
            for (int in_unit = 0; in_unit < boxes; ++in_unit) {
                if (!failed && !mbar_wait(bars + slot * 8, (phase >> slot) & 1u, nullptr)) {
                    if (lane == 0) atomicCAS(&g_w4_error, 0, kErrBulkWait);
                    failed = true;  // go on without the weights: the other warps wait at the joins
                    for (int s = 0; s < sh.depth; ++s) mbar_wait(bars + s * 8, (phase >> s) & 1u, nullptr);
                }
                // 16-byte piece b of row g stands at b ^ g (the tensor map's swizzle)
                const uint32_t q_lane = ring + slot * kBoxBytes + (uint32_t)(g * 128 + g * 16 + t * 4);
                float acc[NT][4];
                uint32_t pair[2], even[2], odd[2], zw[2];
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    if (b % GB == 0) {
                        const int src = GB == 1 ? in_unit * 2 + (b >> 2) : in_unit;
                        const int held = GB == 8 ? 0 : (b / GB) % kHeld;
#pragma unroll
                        for (int c = 0; c < NT; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[c][i] = 0.0f;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (held % 2 == 0) pair[i] = __shfl_sync(0xffffffffu, sc[i][held >> 1], src, 4);
                            if constexpr (Z) {
                                if (held == 0) zw[i] = __shfl_sync(0xffffffffu, zr[i], src, 4);
                                biased_zeros<DT>(zw[i], held, even[i], odd[i]);
                            } else {
                                biased_zeros<DT>(8u, 0, even[i], odd[i]);
                            }
                        }
                    }
                    uint4 xv[NT];
#pragma unroll
                    for (int c = 0; c < NT; ++c)
                        xv[c] = *reinterpret_cast<const uint4*>(smem + x_lane[c] + x_at);
                    x_at += x_block;
                    const uint8_t* at = smem + (q_lane ^ (uint32_t)(b * 16));
                    const uint32_t lo = *reinterpret_cast<const uint32_t*>(at);
                    const uint32_t hi = *reinterpret_cast<const uint32_t*>(at + 8 * 128);
                    uint32_t lo_pairs[4], hi_pairs[4];
                    biased_pairs<DT>(lo, lo_pairs);
                    biased_pairs<DT>(hi, hi_pairs);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t a[4] = {sub2<DT>(lo_pairs[2 * h], even[0]), sub2<DT>(hi_pairs[2 * h], even[1]),
                                               sub2<DT>(lo_pairs[2 * h + 1], odd[0]),
                                               sub2<DT>(hi_pairs[2 * h + 1], odd[1])};
#pragma unroll
                        for (int c = 0; c < NT; ++c)
                            mma_16816<DT>(acc[c], a, h ? xv[c].z : xv[c].x, h ? xv[c].w : xv[c].y);
                    }
                    if (b % GB == GB - 1) {
                        const int held = GB == 8 ? 0 : (b / GB) % kHeld;
                        const float s0 = scale_of<DT>(pair[0], held & 1), s1 = scale_of<DT>(pair[1], held & 1);
#pragma unroll
                        for (int c = 0; c < NT; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sum[c][i] = fmaf(i < 2 ? s0 : s1, acc[c][i], sum[c][i]);
                    }
                }
                __syncwarp();  // all threads have read the box
                if (a_left > 0) {
                    if (!failed) issue(a_box, a_row, job.e, slot);
                    --a_left;
                    if (++a_box == num_box) {
                        a_box = 0;
                        ++a_row;
                    }
                }
                phase ^= 1u << slot;
                if (++slot == sh.depth) slot = 0;
            }
            if (row_done || left == 0) {  // this warp is done with the row
                // (warp, row) pairs of a job go up one at a time, so their sums are places of their own
                float* mine = red + (warp + row) * part;
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int token = c * 8 + 2 * t + (i & 1);
                        if (token < tokens) mine[token * kRows + (i >> 1) * 8 + g] = sum[c][i];
                        sum[c][i] = 0.0f;
                    }
                ++row;
            }
        }

        const Job next = job_at(job.first + job.rows);
        begin(next);
        __syncthreads();
        const int boxes = job.rows * num_box;
        for (int i = threadIdx.x; i < job.rows * tokens * kRows; i += kThreads) {
            const int in_row = i % (tokens * kRows), row = i / (tokens * kRows);
            const int token = in_row / kRows, n = (job.row + row) * kRows + in_row % kRows;
            // warp w has box p when boxes * w / 16 <= p < boxes * (w + 1) / 16 (whole quotients)
            const int w0 = (kWarps * (row * num_box + 1) - 1) / boxes, w1 = (kWarps * (row + 1) * num_box - 1) / boxes;
            float v = 0.0f;
            for (int w = w0; w <= w1; ++w)
                if (first_box(job.rows, w) < first_box(job.rows, w + 1)) v += red[(w + row) * part + in_row];
            if (n < sh.n) out[(size_t)(row0 + token) * sh.n + n] = round16<DT>(v);
        }
        __syncthreads();
        job = next;
    }
}

// ------------------------------------------------------------------ host side
template <int DT, int NT, int GB, bool Z, bool V>
static int launch_kernel(const CUtensorMap& tmQ, const void* x, const void* scales, const void* zeros,
                         const int* offsets, void* out, Shape sh, int dev, cudaStream_t stream) {
    static bool attr_set[64] = {};
    constexpr size_t kMaxSmem = 226 * 1024;
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(gemv_w4_kernel<DT, NT, GB, Z, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)kMaxSmem));
        if (dev < 64) attr_set[dev] = true;
    }
    const int num_box = (sh.k + kBoxK - 1) / kBoxK;
    sh.tokens = std::min({sh.rows, NT * 8, 256 / num_box});  // x takes at most 128 KiB
    const size_t fixed = 1024 + (size_t)num_box * 512 * sh.tokens +
                         (size_t)(kWarps + kJobRows) * sh.tokens * kRows * 4 + (size_t)(3 * sh.groups + 1) * 4;
    const size_t slots = (size_t)kWarps * kBoxBytes;  // one box for each warp
    sh.depth = (int)std::min<size_t>(4, (kMaxSmem - fixed) / slots);
    const size_t smem = fixed + sh.depth * slots;
    const int64_t rows_n = (sh.n + kRows - 1) / kRows;
    const int64_t tiles = rows_n * ((int64_t)sh.rows / sh.tokens + std::min(sh.groups, sh.rows));
    if (tiles > INT32_MAX) {
        set_error("trb_gemv_w4_launch: too many outputs (rows=%d n=%d groups=%d)", sh.rows, sh.n, sh.groups);
        return TRB_SKIPPED;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles, device_sm_count(dev)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    TRB_CUDA(cudaLaunchKernelEx(&cfg, gemv_w4_kernel<DT, NT, GB, Z, V>, tmQ, static_cast<const uint16_t*>(x),
                                static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), offsets,
                                static_cast<uint16_t*>(out), sh));
    return TRB_OK;
}

template <int DT, int NT, int GB, bool Z>
static int launch_scales(const CUtensorMap& tmQ, const void* x, const void* scales, const void* zeros,
                         const int* offsets, void* out, const Shape& sh, int dev, cudaStream_t stream) {
    constexpr int kHeld = held_scales(GB);
    const bool vector = kHeld > 1 && sh.k_groups % kHeld == 0 &&
                        reinterpret_cast<uintptr_t>(scales) % (2 * kHeld) == 0 &&
                        reinterpret_cast<uintptr_t>(zeros) % kHeld == 0;
    if constexpr (kHeld > 1)
        if (vector) return launch_kernel<DT, NT, GB, Z, true>(tmQ, x, scales, zeros, offsets, out, sh, dev, stream);
    return launch_kernel<DT, NT, GB, Z, false>(tmQ, x, scales, zeros, offsets, out, sh, dev, stream);
}

template <int DT, int NT, bool Z>
static int launch_group(const void* x, const void* q, const void* scales, const void* zeros, const int* offsets,
                        void* out, const Shape& sh, int dev, cudaStream_t stream) {
    CUtensorMap tmQ;
    const uint64_t extent[3] = {(uint64_t)sh.k / 2, (uint64_t)sh.n, (uint64_t)sh.groups};
    const uint32_t box[3] = {128, kRows, 1};
    const int rc = gemm::encode_tiled(&tmQ, q, 1, 3, extent, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != TRB_OK) return rc;
    switch (sh.group_log2) {
        case 5: return launch_scales<DT, NT, 1, Z>(tmQ, x, scales, zeros, offsets, out, sh, dev, stream);
        case 6: return launch_scales<DT, NT, 2, Z>(tmQ, x, scales, zeros, offsets, out, sh, dev, stream);
        case 7: return launch_scales<DT, NT, 4, Z>(tmQ, x, scales, zeros, offsets, out, sh, dev, stream);
        default: return launch_scales<DT, NT, 8, Z>(tmQ, x, scales, zeros, offsets, out, sh, dev, stream);
    }
}

template <int DT>
static int launch(const void* x, const void* q, const void* scales, const void* zeros, const int* offsets, void* out,
                  const Shape& sh, int dev, cudaStream_t stream) {
    // More than 8 rows a group on average: 16 rows at once read the weights half as often.
    if (sh.rows > 8 * (int64_t)sh.groups)
        return zeros ? launch_group<DT, 2, true>(x, q, scales, zeros, offsets, out, sh, dev, stream)
                     : launch_group<DT, 2, false>(x, q, scales, zeros, offsets, out, sh, dev, stream);
    return zeros ? launch_group<DT, 1, true>(x, q, scales, zeros, offsets, out, sh, dev, stream)
                 : launch_group<DT, 1, false>(x, q, scales, zeros, offsets, out, sh, dev, stream);
}

int read_error(bool clear) {
    int v = 0;
    TRB_CUDA(cudaMemcpyFromSymbol(&v, g_w4_error, sizeof(int)));
    if (clear) {
        const int zero = 0;
        TRB_CUDA(cudaMemcpyToSymbol(g_w4_error, &zero, sizeof(int)));
    }
    return v;
}

}  // namespace w4
}  // namespace trb

extern "C" int trb_gemv_w4_launch(int dtype, int groups, int rows, int n, int k, int group_size, const void* x,
                                  const void* q, const void* scales, const void* zeros, const int32_t* offsets,
                                  void* out, void* stream) {
    using namespace trb;
    clear_error();
    if (groups <= 0 || rows < 0 || n <= 0 || k <= 0 || q == nullptr || scales == nullptr ||
        (rows > 0 && (x == nullptr || out == nullptr)) || (offsets == nullptr && groups != 1)) {
        set_error("trb_gemv_w4_launch: sizes must be positive (rows may be 0), pointers non-null, and several groups "
                  "need offsets");
        return TRB_ERR_ARGS;
    }
    if (dtype != TRB_BFLOAT16 && dtype != TRB_FLOAT16) {
        set_error("trb_gemv_w4_launch: unsupported dtype %s (bfloat16 and float16)", dtype_name(dtype));
        return TRB_SKIPPED;
    }
    if (group_size < 32 || (group_size & (group_size - 1)) != 0 || k % group_size != 0) {
        set_error("trb_gemv_w4_launch: the group size must be a power of two of at least 32 that divides k (group size "
                  "%d, k %d)", group_size, k);
        return TRB_SKIPPED;
    }
    if (k > 65536 || groups > kMaxGroups) {
        set_error("trb_gemv_w4_launch: k at most 65536 and at most %d groups (k=%d groups=%d)", kMaxGroups, k, groups);
        return TRB_SKIPPED;
    }
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(q)) & 15u) != 0 ||
        ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(out)) & 1u) != 0 ||
        (reinterpret_cast<uintptr_t>(offsets) & 3u) != 0) {
        set_error("trb_gemv_w4_launch: x and q must be 16-byte aligned, the others as their elements");
        return TRB_ERR_ALIGN;
    }
    if (rows == 0) return TRB_OK;
    int dev = 0;
    TRB_CUDA(cudaGetDevice(&dev));
    w4::Shape sh = {};
    sh.groups = groups;
    sh.rows = rows;
    sh.n = n;
    sh.k = k;
    sh.k_groups = k / group_size;
    while ((1 << sh.group_log2) < group_size) ++sh.group_log2;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == TRB_BFLOAT16 ? w4::launch<TRB_BFLOAT16>(x, q, scales, zeros, offsets, out, sh, dev, s)
                                 : w4::launch<TRB_FLOAT16>(x, q, scales, zeros, offsets, out, sh, dev, s);
}
