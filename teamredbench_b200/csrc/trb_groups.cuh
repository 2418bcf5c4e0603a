// trb_groups.cuh -- rows sorted by group (expert) with offsets on the device.
#pragma once

#include "trb_common.cuh"

namespace trb {

constexpr int kMaxGroups = 1024;
// Largest rows, n and k.  The kernels round sizes up to whole tiles and stages (a chunk's rows: up to one part in 256
// above them) and step past the end by a stage in 32-bit integers, so sizes near 2^31 would wrap.
constexpr int kMaxExtent = 0x7F000000;

#if defined(__CUDACC__)

// Shared-memory arrays of the groups of one launch.
struct GroupTable {
    int* start;   // first row
    int* rows;
    int* chunk0;  // chunks of the groups before this one; [groups] = all chunks (scan_chunks)
};

// Reads the offsets (all threads of the CTA; ends with a barrier).  Offsets
// that decrease or leave [0, total_rows] set the error word; the call then
// computes nothing (returns 0 groups), so that no offsets, however wrong,
// reach outside the operands.
__device__ __forceinline__ int load_groups(const int* offsets, int groups, int total_rows, const GroupTable& g,
                                           int* error) {
    bool bad = false;
    for (int e = threadIdx.x; e < groups; e += blockDim.x) {
        const int lo = offsets[e], hi = offsets[e + 1];
        bad = bad || lo < 0 || hi < lo || hi > total_rows;
        g.start[e] = lo;
        g.rows[e] = hi - lo;
    }
    if (!__syncthreads_or(bad)) return groups;
    if (threadIdx.x == 0) atomicCAS(error, 0, kErrOffsets);
    return 0;
}

// The check alone.
__device__ __forceinline__ int check_groups(const int* offsets, int groups, int total_rows, int* error) {
    bool bad = false;
    for (int e = threadIdx.x; e < groups; e += blockDim.x)
        bad = bad || offsets[e] < 0 || offsets[e + 1] < offsets[e] || offsets[e + 1] > total_rows;
    if (!__syncthreads_or(bad)) return groups;
    if (threadIdx.x == 0) atomicCAS(error, 0, kErrOffsets);
    return 0;
}

// Exclusive scan of the groups' chunk counts, ceil(rows / chunk_rows) each (one warp).
__device__ __forceinline__ void scan_chunks(int groups, int chunk_rows, const GroupTable& g, int lane) {
    int base = 0;
    for (int e0 = 0; e0 < groups; e0 += 32) {
        const int e = e0 + lane;
        const int c = e < groups ? (g.rows[e] + chunk_rows - 1) / chunk_rows : 0;
        int sum = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (e < groups) g.chunk0[e] = base + sum - c;
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) g.chunk0[groups] = base;
}

// The group of chunk q, 0 <= q < chunk0[groups]: the last one whose chunks begin at or before q.
__device__ __forceinline__ int group_of_chunk(int q, int groups, const GroupTable& g) {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (g.chunk0[mid] <= q) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

#endif  // __CUDACC__

}  // namespace trb
