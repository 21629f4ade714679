// slideformer_amd: square tiles of a matrix product on the matrix cores (gfx950,
// wave64), 16-bit operands, fp32 sums.
//
// D[o, i] = sum over k of O[o, k] * I[i, k].  `i` is the dimension along which D
// is contiguous in memory ("inner"), `o` the other ("outer").  Each operand lies
// in memory in one of two ways:
//   by rows      row of the tile's dimension, k contiguous;
//   by columns   row of k, the tile's dimension contiguous.
// so no operand is transposed in memory for any of the three products of a linear
// layer with a loss.
//
// A workgroup of 4 waves computes one tile of SIDE x SIDE, a quarter of it per wave.
//   SIDE 256     one wave on each SIMD: 128 x 128 sums in 256 registers.  A step of
//                32 k takes a wave 64 matrix instructions (1024 cycles) and the workgroup
//                64 KB of LDS reads and 32 KB of writes (768 cycles at 128 bytes each), so
//                LDS stays behind the matrix cores; with eight waves of 128 x 64 the reads
//                alone would take as long as the products.
//   SIDE 128     three workgroups on a compute unit, each in the others' pauses: a
//                product with few tiles or few steps is made of starts and ends.  Two,
//                with a step more in LDS, took 1024 x 50257 x 768 369 us instead of 342.
// What a wave multiplies in one step it reads from LDS during the step before,
// instruction by instruction between the products, so that neither waits for the
// other.  Operands go from memory into LDS without passing registers, three or four
// steps ahead.  The LDS image is permuted so that no read has bank conflicts; since the
// loads write LDS linearly, the permutation is applied to the addresses that they read:
//   by rows      [SIDE][32]: 16-byte chunk c of row r is at chunk c ^ (r / 2 % 4), so 8
//                lanes that read one chunk column of 8 rows hit all 128 bytes of banks;
//   by columns   [32][SIDE]: 32-byte segment s of row k is at s ^ f(k), f taking bits 0, 1
//                and 3 of k, so the eight rows that two groups of lanes read at one s by
//                a transposing read differ in banks.
// Rows and columns beyond a matrix's memory read as zeros through the buffer
// descriptor's range.
#ifndef SLIDEFORMER_AMD_TILE_PRODUCT_H
#define SLIDEFORMER_AMD_TILE_PRODUCT_H

#include "ops_common.h"
#include "tile_range.h"

namespace tile {

constexpr int kThreads = 256;
constexpr uint32_t kXcds = 8;       // consecutive workgroups go to different ones in turn

template <int SIDE> struct Sizes {
    static constexpr int kPanelBytes = SIDE * kDepth * 2;   // one operand's share of a step
    static constexpr int kStepBytes = 2 * kPanelBytes;
    static constexpr int kAhead = SIDE == 256 ? 4 : 3;      // steps in LDS
    static constexpr int kLdsBytes = kAhead * kStepBytes;
    static constexpr int kLoads = kPanelBytes / 4096;       // of a lane, for a panel
    static constexpr int kWave = SIDE / 2;                  // side of a wave's quarter
    static constexpr int kParts = kWave / 16;               // its fragments
    static constexpr int kRow = kWave + 4;                  // distance of rows that are handed out
    static constexpr int kHandOutBytes = 4 * 32 * kRow * 4;
    static constexpr int kResident = SIDE == 256 ? 1 : 3;   // workgroups on a compute unit
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;

// c += a b^T.  Written in assembly to keep a sum in its registers: left to itself
// the compiler gives each product a destination of its own, and with all
// accumulation registers in use it then moves sums about, more often than it
// multiplies.  It cannot see that the results of these take a while; settle() waits.
template <typename T> __device__ __forceinline__ void multiply(const s16x8& a, const s16x8& b, f32x4& c);
template <> __device__ __forceinline__ void multiply<__bf16>(const s16x8& a, const s16x8& b, f32x4& c)
{
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <> __device__ __forceinline__ void multiply<_Float16>(const s16x8& a, const s16x8& b, f32x4& c)
{
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// The same where registers are no concern, with the compiler's own waits.
template <typename T> __device__ __forceinline__ f32x4 product_of(const s16x8& a, const s16x8& b, const f32x4& c);
template <> __device__ __forceinline__ f32x4 product_of<__bf16>(const s16x8& a, const s16x8& b, const f32x4& c)
{
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 product_of<_Float16>(const s16x8& a, const s16x8& b, const f32x4& c)
{
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

// An operand in memory: `count` rows of `width` 16-bit elements, `stride` bytes apart.
struct Matrix {
    const void* data;
    uint64_t count, width, stride;
};

// One operand's share of a workgroup's work.  BY_ROWS: see above.
template <int SIDE, bool BY_ROWS> struct Operand {
    static constexpr uint32_t kLoads = Sizes<SIDE>::kLoads;
    Walk walk;                      // in addresses
    uint32_t offset[kLoads];        // of this lane's loads
    u32x4_t rsrc;

    // The product begins at step `begin` and goes round: see Product::run.
    __device__ void init(const Matrix& m, uint64_t tile_at, uint64_t k_at, uint32_t all, uint32_t begin)
    {
        walk.init(BY_ROWS, m.count, m.width, m.stride, tile_at, k_at, all, begin);
        walk.at += reinterpret_cast<uint64_t>(m.data);
#pragma unroll
        for (uint32_t n = 0; n < kLoads; ++n)
            offset[n] = load_offset(SIDE, BY_ROWS, n, threadIdx.x / 64, threadIdx.x % 64, static_cast<uint32_t>(m.stride));
    }

    // Turns to the next step, the `turned`-th; one without data reads zeros.
    __device__ __forceinline__ void turn(uint32_t turned)
    {
        rsrc = u32x4_t{static_cast<uint32_t>(walk.at), static_cast<uint32_t>(walk.at >> 32), walk.range(turned),
                       0x00020000u};
        walk.turn();
    }

    // Load `n` of the step, to this wave's place `lds`; returns at once.  Written in
    // assembly, which takes no result in a register: the compiler would wait for
    // every load in flight before any read of LDS.  The loop waits itself.
    __device__ void load(uint32_t lds, int n) const
    {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(lds + n * 4096), "v"(offset[n]), "s"(rsrc)
                     : "m0");
    }
};

// The 16 x 32 fragment of tile rows `tile_at` + 16 n .., as the matrix instructions
// take it: lane l holds row l % 16, k (l / 16) * 8 .. + 7.
template <int SIDE, bool BY_ROWS> struct Fragments {
    uint32_t base;

    __device__ void init(uint32_t tile_at)
    {
        const uint32_t lane = threadIdx.x % 64, row = lane % 16, group = lane / 16;
        if constexpr (BY_ROWS) {
            base = (tile_at + row) * 64 + (group ^ (row / 2 % 4)) * 16;
        } else {
            const uint32_t k = group * 8 + row / 4;         // and four rows further in the second read
            const uint32_t f = (k & 3) | (k >> 3 & 1) << 2;
            base = k * (SIDE * 2) + ((tile_at / 16) ^ f) * 32 + (row % 4) * 8;
        }
    }

    __device__ s16x8 read(const lds_char* lds, int n) const
    {
        if constexpr (BY_ROWS) {
            return *reinterpret_cast<const lds_s16x8*>(lds + base + n * 1024);
        } else {
            // lanes 4j .. 4j+3 of a group of 16 read 16 elements of row j; lane l gets column l of the four rows
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + (base ^ (n * 32))));
            const s16x4 hi =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds + (base ^ (n * 32)) + 4 * SIDE * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// A wave's quarter of the tile.  Element [s][t][r] of a lane is inner
// 16 s + (lane / 16) * 4 + r, outer 16 t + lane % 16 of that quarter.
template <int SIDE> using Sums = f32x4[Sizes<SIDE>::kParts][Sizes<SIDE>::kParts];
template <int SIDE> using Step = s16x8[2][Sizes<SIDE>::kParts];     // fragments of one step: inner, outer

template <int SIDE> __device__ __forceinline__ uint32_t wave_inner() { return threadIdx.x / 64 % 2 * (SIDE / 2); }
template <int SIDE> __device__ __forceinline__ uint32_t wave_outer() { return threadIdx.x / 128 * (SIDE / 2); }

// Waits until at most `left` loads of this wave are in flight and its reads of
// LDS are done, then for the other waves to come this far.
template <int LEFT> __device__ __forceinline__ void arrive()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(LEFT) : "memory");
}

// Places all sums in accumulation registers, and waits until what wrote them has
// and what reads them may: longer than any matrix instruction or move needs.
template <int PARTS> __device__ __forceinline__ void settle(f32x4 (&sums)[PARTS][PARTS])
{
#pragma unroll
    for (int s = 0; s < PARTS; ++s)
#pragma unroll
        for (int t = 0; t < PARTS; ++t) asm volatile("" : "+a"(sums[s][t]));
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15");
#pragma unroll
    for (int s = 0; s < PARTS; ++s)
#pragma unroll
        for (int t = 0; t < PARTS; ++t) asm volatile("" : "+a"(sums[s][t]));
}

template <typename T, int SIDE, bool INNER_ROWS, bool OUTER_ROWS> struct Product {
    using Z = Sizes<SIDE>;
    Operand<SIDE, INNER_ROWS> load_inner;
    Operand<SIDE, OUTER_ROWS> load_outer;
    Fragments<SIDE, INNER_ROWS> read_inner;
    Fragments<SIDE, OUTER_ROWS> read_outer;
    lds_char* lds;
    uint32_t place;                 // of this wave's loads in a panel

    // One step: multiplies `now`, reads the fragments of the next step into `then`,
    // and loads the step Z::kAhead from here over this one, whose reads are over.
    __device__ __forceinline__ void step(uint32_t at, const Step<SIDE>& now, Step<SIDE>& then, Sums<SIDE>& sums)
    {
        // in groups of four products: reads in the first half, loads in the second
        constexpr int kGroups = Z::kParts * Z::kParts / 4, kHalf = kGroups / 2;
        constexpr int kReads = Z::kParts / kHalf, kLoads = 2 * Z::kLoads / kHalf;
        // the next step's loads have arrived: only those of two steps more are in flight
        arrive<(Z::kAhead - 2) * 2 * Z::kLoads>();
        const lds_char* from = lds + (at + 1) % Z::kAhead * Z::kStepBytes;
        const uint32_t to =
            __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) +
                                           at % Z::kAhead * Z::kStepBytes + place);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (g < kHalf) {
#pragma unroll
                for (int k = 0; k < kReads; ++k) {
                    then[0][g * kReads + k] = read_inner.read(from, g * kReads + k);
                    then[1][g * kReads + k] = read_outer.read(from + Z::kPanelBytes, g * kReads + k);
                }
            }
            if (g == kHalf - 1) load_inner.turn(at + Z::kAhead);
            if (g == kHalf + kHalf / 4) load_outer.turn(at + Z::kAhead);
            if (g >= kHalf) {
#pragma unroll
                for (int k = (g - kHalf) * kLoads; k < (g - kHalf + 1) * kLoads; ++k) {
                    if (k < Z::kLoads) load_inner.load(to, k);
                    else load_outer.load(to + Z::kPanelBytes, k - Z::kLoads);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int s = (g * 4 + k) / Z::kParts, t = (g * 4 + k) % Z::kParts;
                multiply<T>(now[0][s], now[1][t], sums[s][t]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    __device__ __forceinline__ void run(const Matrix& inner, uint64_t inner_at, const Matrix& outer, uint64_t outer_at,
                                        uint64_t k_at, uint32_t steps, char* shared, Sums<SIDE>& sums)
    {
#pragma unroll
        for (int s = 0; s < Z::kParts; ++s)
#pragma unroll
            for (int t = 0; t < Z::kParts; ++t) sums[s][t] = f32x4{0, 0, 0, 0};
        if (steps == 0) return;
        lds = (lds_char*)shared;
        place = threadIdx.x / 64 * 1024;
        // Each XCD begins at an eighth of k of its own: rows a power of two apart would
        // otherwise all be read from the same few memory channels at a time (200 x 128256 x
        // 4096, forward: 327 -> 274 us; where operands come from the caches it makes no
        // difference).  Within an XCD, whose tiles share operands, all go together.
        const uint32_t begin = blockIdx.x % kXcds * steps / kXcds;
        load_inner.init(inner, inner_at, k_at, steps, begin);
        load_outer.init(outer, outer_at, k_at, steps, begin);
        read_inner.init(wave_inner<SIDE>());
        read_outer.init(wave_outer<SIDE>());
#pragma unroll
        for (int ahead = 0; ahead < Z::kAhead; ++ahead) {
            const uint32_t to = __builtin_amdgcn_readfirstlane(
                static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + ahead * Z::kStepBytes + place);
            load_inner.turn(ahead);
            load_outer.turn(ahead);
#pragma unroll
            for (int n = 0; n < Z::kLoads; ++n) load_inner.load(to, n);
#pragma unroll
            for (int n = 0; n < Z::kLoads; ++n) load_outer.load(to + Z::kPanelBytes, n);
        }
        arrive<(Z::kAhead - 1) * 2 * Z::kLoads>();
        Step<SIDE> even, odd;
#pragma unroll
        for (int n = 0; n < Z::kParts; ++n) {
            even[0][n] = read_inner.read(lds, n);
            even[1][n] = read_outer.read(lds + Z::kPanelBytes, n);
        }
        settle(sums);
        for (uint32_t at = 0; at < steps; at += 2) {
            step(at, even, odd, sums);
            step(at + 1, odd, even, sums);
        }
        settle(sums);
        // the loads that read zeros are over, and every wave has done with LDS
        arrive<0>();
    }
};

// sums = the tile at (inner_at, outer_at) over `steps` steps from k_at, an even number.
template <typename T, int SIDE, bool INNER_ROWS, bool OUTER_ROWS>
__device__ __forceinline__ void product(const Matrix& inner, uint64_t inner_at, const Matrix& outer, uint64_t outer_at,
                                        uint64_t k_at, uint32_t steps, char* shared, Sums<SIDE>& sums)
{
    Product<T, SIDE, INNER_ROWS, OUTER_ROWS> p;
    p.run(inner, inner_at, outer, outer_at, k_at, steps, shared, sums);
}

// Hands a wave's quarter of the tile out by rows: emit(outer, inner, v) with eight
// consecutive inner elements, neighbouring lanes along a row, so that what is
// stored from them fills whole lines.  Goes through this wave's part of LDS, 32 rows
// at a time; the row distance, four more than the quarter's side, keeps its accesses
// free of bank conflicts.
template <int SIDE, typename Emit>
__device__ __forceinline__ void by_rows(const Sums<SIDE>& sums, char* shared, const Emit& emit)
{
    using Z = Sizes<SIDE>;
    constexpr uint32_t kLanes = Z::kWave / 8;               // to a row
    const uint32_t lane = threadIdx.x % 64;
    float* mine = reinterpret_cast<float*>(shared) + threadIdx.x / 64 * (32 * Z::kRow);
#pragma unroll
    for (int part = 0; part < Z::kParts / 2; ++part) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < Z::kParts; ++s)
                *reinterpret_cast<f32x4*>(mine + (t * 16 + lane % 16) * Z::kRow + s * 16 + lane / 16 * 4) =
                    sums[s][part * 2 + t];
        // the wave's own stores, seen by its own loads: the hardware keeps them in order
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (uint32_t row = lane / kLanes; row < 32; row += 64 / kLanes) {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(mine + row * Z::kRow + lane % kLanes * 8);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(mine + row * Z::kRow + lane % kLanes * 8 + 4);
            const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            emit(wave_outer<SIDE>() + part * 32 + row, wave_inner<SIDE>() + lane % kLanes * 8, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The tile that workgroup `id` of a launch computes.  Consecutive workgroups go
// to different XCDs in turn; each XCD takes a run of consecutive tiles, in bands of
// `kBand` outer tiles, so that what runs on it together shares operands in its L2.
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
