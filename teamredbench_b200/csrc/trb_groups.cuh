// trb_groups.cuh -- rows sorted by group (expert) with offsets on the device.
#pragma once

#include <initializer_list>

#include "trb_common.cuh"

namespace trb {

constexpr int kMaxGroups = 1024;
// Largest rows, n and k.  The kernels round sizes up to whole tiles and stages (a chunk's rows: up to one part in 256
// above them) and step past the end by a stage in 32-bit integers, so sizes near 2^31 would wrap.
constexpr int kMaxExtent = 0x7F000000;

// Memory that a call reads or writes.
struct Span {
    const void* at;
    uint64_t bytes;
    Span(const void* p, uint64_t size, uint64_t rows, uint64_t width = 1, uint64_t groups = 1) : at(p) {
        const unsigned __int128 all = (unsigned __int128)(size * groups) * rows * width;
        bytes = p == nullptr ? 0 : all > UINT64_MAX ? UINT64_MAX : (uint64_t)all;
    }
};
// CTAs read what others write where the two overlap, in any order, so such a call is refused.
inline int check_apart(const char* what, std::initializer_list<Span> written, std::initializer_list<Span> read) {
    const auto overlap = [](const Span& a, const Span& b) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
        return a.bytes > 0 && b.bytes > 0 && (x <= y ? y - x < a.bytes : x - y < b.bytes);
    };
    for (auto w = written.begin(); w != written.end(); ++w) {
        bool bad = false;
        for (const Span& r : read) bad = bad || overlap(*w, r);
        for (auto other = w + 1; other != written.end(); ++other) bad = bad || overlap(*w, *other);
        if (bad) {
            set_error("%s: results must not overlap operands or each other", what);
            return TRB_ERR_ARGS;
        }
    }
    return TRB_OK;
}

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
