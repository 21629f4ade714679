// slideformer_amd: 256 x 256 tiles of a matrix product on the matrix cores
// (gfx950, wave64), 16-bit operands, fp32 sums.
//
// D[o, i] = sum over k of O[o, k] * I[i, k].  `i` is the dimension along which D
// is contiguous in memory ("inner"), `o` the other ("outer").  Each operand lies
// in memory in one of two ways:
//   by rows      row of the tile's dimension, k contiguous;
//   by columns   row of k, the tile's dimension contiguous.
// so no operand is transposed in memory for any of the three products of a linear
// layer with a loss.
//
// A workgroup of 8 waves computes one tile.  Both operands go from memory into
// LDS 64 k at a time without passing registers, two stages in turn.  The LDS
// image is permuted so that no read has bank conflicts; since the loads write
// LDS linearly, the permutation is applied to the addresses that they read:
//   by rows      [256][64]: 16-byte chunk c of row r is at chunk c ^ (r & 7), so 8
//                lanes that read one chunk column of 8 rows hit 8 chunks;
//   by columns   [64][256]: 32-byte segment s of row k is at s ^ (k & 15), so the
//                four rows that a transposing read takes at one s differ in banks.
// Rows and columns beyond a matrix's memory read as zeros through the buffer
// descriptor's range.
#ifndef SLIDEFORMER_AMD_TILE_PRODUCT_H
#define SLIDEFORMER_AMD_TILE_PRODUCT_H

#include "ops_common.h"

namespace tile {

constexpr int kTile = 256;          // both sides of a tile
constexpr int kDepth = 64;          // k per stage
constexpr int kThreads = 512;
constexpr int kStageBytes = kTile * kDepth * 2;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    __device__ static f32x4 run(s16x8 a, s16x8 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};
template <> struct Mfma<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    __device__ static f32x4 run(s16x8 a, s16x8 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};

// An operand in memory: `count` rows of `width` 16-bit elements, `stride` bytes apart.
struct Matrix {
    const void* data;
    uint64_t count, width, stride;
};

// One operand's share of a workgroup's work.  BY_ROWS: see above.
template <bool BY_ROWS> struct Operand {
    const char* at;                 // this stage's corner in memory
    const char* end;                // one past the matrix's last byte
    uint64_t step;                  // bytes from stage to stage
    uint32_t offset[4];             // of this lane's four loads
    uint32_t stage;                 // this wave's place in a stage

    __device__ void init(const Matrix& m, uint64_t tile_at, uint64_t k_at)
    {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
        const char* data = static_cast<const char*>(m.data);
        end = data + (m.count - 1) * m.stride + m.width * 2;
        if constexpr (BY_ROWS) {
            at = data + tile_at * m.stride + k_at * 2;
            step = kDepth * 2;
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n)
                offset[n] = (n * 64 + wave * 8 + lane / 8) * static_cast<uint32_t>(m.stride) +
                            ((lane % 8) ^ (lane / 8)) * 16;
        } else {
            at = data + k_at * m.stride + tile_at * 2;
            step = kDepth * m.stride;
            const uint32_t k = wave * 2 + lane / 32;        // & 15: the rows of one lane's loads are 16 apart
            const uint32_t chunk = (((lane % 32 / 2) ^ k) * 2 + lane % 2) * 16;
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n) offset[n] = (n * 16 + k) * static_cast<uint32_t>(m.stride) + chunk;
        }
        stage = wave * 1024;
    }

    // Loads the next stage into `lds`; returns at once.  Written in assembly,
    // which takes no result in a register: the compiler would wait for every such
    // load before the next read of LDS, the one stage in flight included.  The
    // loop waits itself, once a stage.
    __device__ void load(lds_char* lds)
    {
        const int64_t left = end - at;
        const uint32_t range = left <= 0 ? 0 : left > 0x7ffffff0 ? 0x7ffffff0 : static_cast<uint32_t>(left);
        const uint64_t address = reinterpret_cast<uint64_t>(at);
        const u32x4_t rsrc{static_cast<uint32_t>(address), static_cast<uint32_t>(address >> 32), range, 0x00020000u};
        const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + stage;
#pragma unroll
        for (uint32_t n = 0; n < 4; ++n)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(to + n * 8192), "v"(offset[n]), "s"(rsrc)
                         : "m0");
        at += step;
    }
};

// The 16 x 32 fragment of tile rows `at`.. and k `half` * 32.., as the matrix
// instructions take it: lane l holds row l % 16, k (l / 16) * 8 .. + 7.
template <bool BY_ROWS> struct Fragments {
    uint32_t base;

    __device__ void init(uint32_t tile_at)
    {
        const uint32_t lane = threadIdx.x % 64, row = lane % 16, group = lane / 16;
        if constexpr (BY_ROWS) {
            base = (tile_at + row) * 128 + ((group ^ (row & 7)) * 16);
        } else {
            const uint32_t k = group * 8 + row / 4;
            base = k * 512 + (((tile_at / 16) ^ (k & 15)) * 32) + (row % 4) * 8;
        }
    }

    __device__ s16x8 read(const lds_char* lds, int n, int half) const
    {
        if constexpr (BY_ROWS) {
            return *reinterpret_cast<const lds_s16x8*>(lds + (base ^ (half * 64)) + n * 2048);
        } else {
            // lanes 4j .. 4j+3 of a group of 16 read 16 elements of row j; lane l gets column l of the four rows
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(lds + (base ^ (n * 32)) + half * 16384));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(lds + (base ^ ((n ^ 4) * 32)) + half * 16384 + 2048));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// A wave's part of the tile: 128 inner x 64 outer.  Element [s][t][r] of a lane
// is inner 16 s + (lane / 16) * 4 + r, outer 16 t + lane % 16 of that part.
typedef f32x4 Sums[8][4];

__device__ __forceinline__ uint32_t wave_inner() { return threadIdx.x / 64 % 2 * 128; }
__device__ __forceinline__ uint32_t wave_outer() { return threadIdx.x / 128 * 64; }

template <typename T, bool INNER_ROWS, bool OUTER_ROWS>
__device__ void product(const Matrix& inner, uint64_t inner_at, const Matrix& outer, uint64_t outer_at, uint64_t k_at,
                        uint32_t stages, lds_char* lds, Sums& sums)
{
    Operand<INNER_ROWS> load_inner;
    Operand<OUTER_ROWS> load_outer;
    Fragments<INNER_ROWS> read_inner;
    Fragments<OUTER_ROWS> read_outer;
    load_inner.init(inner, inner_at, k_at);
    load_outer.init(outer, outer_at, k_at);
    read_inner.init(wave_inner());
    read_outer.init(wave_outer());
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t) sums[s][t] = f32x4{0, 0, 0, 0};
    if (stages == 0) return;
    load_inner.load(lds);
    load_outer.load(lds + kStageBytes);
    for (uint32_t stage = 0; stage < stages; ++stage) {
        lds_char* now = lds + (stage & 1) * (2 * kStageBytes);
        // this stage has arrived, and every wave has done with the other half
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (stage + 1 < stages) {
            lds_char* next = lds + (~stage & 1) * (2 * kStageBytes);
            load_inner.load(next);
            load_outer.load(next + kStageBytes);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            s16x8 a[8], b[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) b[t] = read_outer.read(now + kStageBytes, t, half);
#pragma unroll
            for (int s = 0; s < 8; ++s) a[s] = read_inner.read(now, s, half);
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int t = 0; t < 4; ++t) sums[s][t] = Mfma<T>::run(a[s], b[t], sums[s][t]);
        }
    }
}

// The tile that workgroup `id` of a launch computes.  Consecutive workgroups go
// to different XCDs in turn; each XCD takes a run of consecutive tiles, in bands of
// `kBand` outer tiles, so that what runs on it together shares operands in its L2.
constexpr uint32_t kXcds = 8;
constexpr uint32_t kBand = 4;

struct Place {
    uint32_t outer, inner;
    bool valid;
};

__device__ __forceinline__ Place place(uint32_t id, uint32_t outers, uint32_t inners)
{
    const uint32_t total = outers * inners;
    const uint32_t share = (total + kXcds - 1) / kXcds;
    const uint32_t at = id % kXcds * share + id / kXcds;
    Place p{0, 0, id / kXcds < share && at < total};
    if (!p.valid) return p;
    const uint32_t band = at / (kBand * inners);
    const uint32_t size = outers - band * kBand < kBand ? outers - band * kBand : kBand;
    const uint32_t in_band = at - band * kBand * inners;
    p.outer = band * kBand + in_band % size;
    p.inner = in_band / size;
    return p;
}

inline uint64_t places(uint64_t outers, uint64_t inners) { return ceil_div(outers * inners, kXcds) * kXcds; }

}  // namespace tile

#endif  // SLIDEFORMER_AMD_TILE_PRODUCT_H
