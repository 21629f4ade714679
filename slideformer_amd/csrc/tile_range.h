// slideformer_amd: where a tile's operand is read in memory, as plain arithmetic
// that the kernels and a test on the host share.
//
// An operand is a matrix of `count` rows of `width` 16-bit elements, `stride` bytes
// apart.  A workgroup reads it a step of kDepth k at a time: from the step's corner on,
// each lane at its own offset, through a buffer descriptor whose range ends
// with the matrix.  What lies beyond the range reads as zero.
#ifndef SLIDEFORMER_AMD_TILE_RANGE_H
#define SLIDEFORMER_AMD_TILE_RANGE_H

#include <cstdint>

#ifdef __HIPCC__
#define LA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LA_HOST_DEVICE inline
#endif

namespace tile {

constexpr int kDepth = 32;          // k per step

struct Walk {
    uint64_t at;                    // the next step's corner, in bytes from the matrix's first
    uint64_t left;                  // bytes from there to the matrix's end
    uint64_t stride;                // bytes from step to step
    uint64_t back;                  // and from the last to the first
    uint32_t wanted;                // steps in all
    uint32_t steps;                 // with data to read
    uint32_t k;                     // the next step's place among them

    // The walk begins at step `begin` of `all` and goes round.  A step has data where its
    // corner lies inside the matrix; a tile that starts past the last row (by rows) or column
    // (by columns) has none, and its `left`, which would be below zero, is not read.
    LA_HOST_DEVICE void init(bool by_rows, uint64_t count, uint64_t width, uint64_t row_bytes, uint64_t tile_at,
                             uint64_t k_at, uint32_t all, uint32_t begin)
    {
        const uint64_t from = by_rows ? tile_at * row_bytes + k_at * 2 : k_at * row_bytes + tile_at * 2;
        const uint64_t tiles = by_rows ? count : width, depth = by_rows ? width : count;
        const uint64_t there = tile_at < tiles && k_at < depth ? (depth - k_at + kDepth - 1) / kDepth : 0;
        wanted = all;
        k = begin;
        steps = there < all ? static_cast<uint32_t>(there) : all;
        stride = by_rows ? kDepth * 2 : kDepth * row_bytes;
        back = stride - stride * all;
        at = from + stride * begin;
        left = (count - 1) * row_bytes + width * 2 - from - stride * begin;
    }

    // The descriptor's range for the step that is next, the `turned`-th of the walk.
    LA_HOST_DEVICE uint32_t range(uint32_t turned) const
    {
        const uint32_t low = static_cast<uint32_t>(left), high = static_cast<uint32_t>(left >> 32);
        return turned < wanted && k < steps ? (high ? 0xffffffffu : low) : 0u;
    }

    LA_HOST_DEVICE void turn()
    {
        ++k;
        const uint64_t by = k == wanted ? back : stride;
        k = k == wanted ? 0 : k;
        at += by;
        left -= by;
    }
};

// Bytes from a step's corner to what lane `lane` of wave `wave` reads in its load `n`, 16 of them.
LA_HOST_DEVICE uint32_t load_offset(int side, bool by_rows, uint32_t n, uint32_t wave, uint32_t lane, uint32_t row_bytes)
{
    if (by_rows) return (n * 64 + wave * 16 + lane / 4) * row_bytes + ((lane % 4) ^ (lane / 8 % 4)) * 16;
    const uint32_t lanes = static_cast<uint32_t>(side) / 8;             // to a row
    const uint32_t row = (n * 4 + wave) * (64 / lanes) + lane / lanes;
    const uint32_t f = (row & 3) | (row >> 3 & 1) << 2;
    return row * row_bytes + (((lane % lanes / 2) ^ f) * 2 + lane % 2) * 16;
}

}  // namespace tile

#undef LA_HOST_DEVICE

#endif  // SLIDEFORMER_AMD_TILE_RANGE_H
