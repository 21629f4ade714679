// slideformer_amd: what the attention kernels share (gfx950, wave64): where a
// workgroup's sequence lies, tiles of rows on their way from memory into LDS, and
// fragments of them for the matrix cores.
//
// A wave works on 32 rows of one operand, in the columns of v_mfma_f32_32x32x16: lane l
// holds column l % 32.  The result of a first product then is the second operand
// of the next one as it lies in the registers: lane l has of column l % 32 the rows
// 8 (i / 4) + 4 (l / 32) + i % 4 (i = 0 .. 15), and a product over 16 of these rows takes
// eight of them from either half of the lanes, in any order that the first operand is read
// in too.  So scores never go through LDS, and a row's maximum and sum are found within a
// lane and its partner l ^ 32.
//
// A tile in LDS is 64 rows of D elements, 16-byte chunk c of row r at chunk c ^ swizzle(r).
// The 16 lanes that read at a time cover all 64 banks then, both where they read one
// chunk of 16 rows and where they read, transposing, 32 elements of four rows (241 and
// over 173 bytes a cycle and compute unit of 256, measured; with eight different
// chunks instead of sixteen 121).
#ifndef SLIDEFORMER_AMD_ATTENTION_TILE_H
#define SLIDEFORMER_AMD_ATTENTION_TILE_H

#include "memory_overlap.h"
#include "ops_common.h"

namespace att {

constexpr uint32_t kWave = 64;
constexpr uint32_t kTileRows = 64;
constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

template <typename T> __device__ __forceinline__ f32x16 mfma(const s16x8& a, const s16x8& b, const f32x16& c);
template <> __device__ __forceinline__ f32x16 mfma<__bf16>(const s16x8& a, const s16x8& b, const f32x16& c)
{
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma<_Float16>(const s16x8& a, const s16x8& b, const f32x16& c)
{
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zeros()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// Eight of a lane's values, as the second operand of a product over 16 rows.
template <typename T> __device__ __forceinline__ s16x8 rounded(const f32x16& x, int half)
{
    typedef T v8 __attribute__((ext_vector_type(8)));
    v8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[half * 8 + i]);
    return __builtin_bit_cast(s16x8, v);
}

// Exchanges the upper lanes of a and the lower lanes of b: lane l < 32 gets {a of l, a of l + 32}, lane l + 32
// {b of l, b of l + 32}.
struct Halves {
    uint32_t lo, hi;
};
__device__ __forceinline__ Halves halves(uint32_t a, uint32_t b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ float both_max(float x)
{
    const Halves h = halves(__float_as_uint(x), __float_as_uint(x));
    return fmaxf(__uint_as_float(h.lo), __uint_as_float(h.hi));
}
__device__ __forceinline__ float both_sum(float x)
{
    const Halves h = halves(__float_as_uint(x), __float_as_uint(x));
    return __uint_as_float(h.lo) + __uint_as_float(h.hi);
}

// 2^x by the hardware's instruction: what is below 2^-126 is zero, which no sum of
// probabilities up to 1 notices.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// threadIdx.x % kWave, made anew: kept from a kernel's start it takes a register through its loop.
__device__ __forceinline__ uint32_t lane_now() { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x)
{
    return static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 | uniform(static_cast<uint32_t>(x));
}

// The bits of r % 16 in reverse; D = 64 has eight chunks to a row, two rows to all banks.
template <int D> __device__ __forceinline__ uint32_t swizzle(uint32_t r)
{
    const uint32_t f = (r & 1) << 3 | (r & 2) << 1 | (r & 4) >> 1 | (r & 8) >> 3;
    return f % (D / 8);
}

template <int D> struct Tile {
    static constexpr uint32_t kRowBytes = D * 2;
    static constexpr uint32_t kChunks = D / 8;              // of 16 bytes, to a row
    static constexpr uint32_t kBytes = kTileRows * kRowBytes;
};

// Rows of a matrix of 16-bit elements in memory, `stride` bytes apart: `rows` of them from `at` on.
struct Rows {
    uint64_t at;
    int32_t rows;
};

// This lane's share of the loads of ROWS rows by WAVES waves into LDS.  They do not pass
// through registers: 64 lanes write 1024 bytes of LDS in order, and the swizzle is applied to
// the addresses that are read.  What lies beyond the rows, or the last whole chunk
// of a row, reads as zero through the descriptor's range.
template <int D, uint32_t ROWS, uint32_t WAVES> struct Loader {
    static constexpr uint32_t kLoads = ROWS * Tile<D>::kRowBytes / (WAVES * 1024);
    static constexpr uint32_t kRowsOfLoad = 1024 / Tile<D>::kRowBytes;
    static_assert(kLoads * WAVES * 1024 == ROWS * Tile<D>::kRowBytes, "whole loads");
    uint32_t offset[kLoads];
    uint32_t stride, width;         // bytes of a row's distance, of what is read of it

    __device__ __forceinline__ void init(uint32_t wave, uint32_t row_stride, uint32_t dim)
    {
        const uint32_t lane = threadIdx.x % kWave;
        stride = row_stride;
        width = dim * 2;
#pragma unroll
        for (uint32_t n = 0; n < kLoads; ++n) {
            const uint32_t row = (n * WAVES + wave) * kRowsOfLoad + lane / Tile<D>::kChunks;
            const uint32_t chunk = (lane % Tile<D>::kChunks) ^ swizzle<D>(row);
            offset[n] = chunk * 8 < dim ? row * stride + chunk * 16 : 0x80000000u;
        }
    }

    // The descriptor of `count` rows (up to ROWS) from `at` on.
    __device__ __forceinline__ u32x4_t descriptor(uint64_t at, int32_t count) const
    {
        const uint32_t rows = count <= 0 ? 0u : count < static_cast<int32_t>(ROWS) ? static_cast<uint32_t>(count) : ROWS;
        return {uniform(static_cast<uint32_t>(at)), uniform(static_cast<uint32_t>(at >> 32)) & 0xffffu,
                uniform(rows ? (rows - 1) * stride + width : 0u), 0x00020000u};
    }

    // The loads of such rows into `lds`, the place of this wave's first 1024 bytes; returns at once.
    // Written in assembly, which takes no result in a register: the compiler would
    // wait for every load in flight before any read of LDS.  The loops wait themselves.
    // The wait states before the first load are for the descriptor, which vector instructions may have written.
    __device__ __forceinline__ void load(const u32x4_t& rsrc, uint32_t lds) const
    {
        if constexpr (kLoads == 2) {
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                         "s_add_u32 m0, m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
                         :
                         : "s"(uniform(lds)), "v"(offset[0]), "v"(offset[1]), "s"(rsrc), "n"(WAVES * 1024)
                         : "m0", "scc");
        } else {
            static_assert(kLoads % 4 == 0, "four loads at a time");
#pragma unroll
            for (uint32_t n = 0; n < kLoads; n += 4)
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
                             "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\t"
                             "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
                             "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds"
                             :
                             : "s"(uniform(lds + n * WAVES * 1024)), "v"(offset[n]), "v"(offset[n + 1]), "v"(offset[n + 2]),
                               "v"(offset[n + 3]), "s"(rsrc), "n"(WAVES * 1024)
                             : "m0", "scc");
        }
    }

    // Row `first` of `m` on.
    __device__ __forceinline__ void load(const Rows& m, int32_t first, uint32_t lds) const
    {
        const u32x4_t rsrc = descriptor(m.at + static_cast<uint64_t>(first < 0 ? 0 : first) * stride, m.rows - first);
        load(rsrc, lds);
    }
};

// The same of 64 fp32 values, `bytes` of them from `at` on.
__device__ __forceinline__ void load_values(uint64_t at, uint32_t bytes, uint32_t lds)
{
    const u32x4_t rsrc = {uniform(static_cast<uint32_t>(at)), uniform(static_cast<uint32_t>(at >> 32)) & 0xffffu,
                          uniform(bytes), 0x00020000u};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(uniform(lds)), "v"(threadIdx.x % kWave * 4), "s"(rsrc)
                 : "m0");
}

// Waits until at most LEFT loads of this wave are in flight and its reads of LDS are done.
template <int LEFT> __device__ __forceinline__ void arrived()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(LEFT) : "memory");
}
// The same, then for the other waves to come this far.
template <int LEFT> __device__ __forceinline__ void arrive()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(LEFT) : "memory");
}

// First operands from a tile in LDS.
//   rows(k, block)     rows 32 block + l % 32, elements 16 k + 8 (l / 32) .. + 7: a product over D takes D / 16;
//   columns(d, block)  elements 32 d + l % 32 of the rows 16 block + 4 (l / 32) + {0 .. 3, 8 .. 11}: those that lane
//                      l has of 16 rows of a result.
template <int D> struct Fragments {
    uint32_t row_at[D / 16], column_at[D / 32][2];

    __device__ __forceinline__ void init()
    {
        const uint32_t lane = threadIdx.x % kWave, half = lane / 32;
        const uint32_t row = lane % 32;
        const uint32_t row_base = row * Tile<D>::kRowBytes + (half ^ swizzle<D>(row)) * 16;
#pragma unroll
        for (uint32_t k = 0; k < D / 16; ++k) row_at[k] = row_base ^ (k * 32);
        const uint32_t key = 4 * half + lane % 16 / 4;
        const uint32_t chunk = (lane / 16 % 2) * 2 + lane % 4 / 2;
#pragma unroll
        for (uint32_t d = 0; d < D / 32; ++d)
#pragma unroll
            for (uint32_t more = 0; more < 2; ++more)
                column_at[d][more] = (key + 8 * more) * Tile<D>::kRowBytes +
                                     ((chunk + d * 4) ^ swizzle<D>(key + 8 * more)) * 16 + lane % 2 * 8;
    }

    __device__ __forceinline__ s16x8 rows(const lds_char* tile, int k, int block) const
    {
        return *reinterpret_cast<const lds_s16x8*>(tile + row_at[k] + block * (32 * Tile<D>::kRowBytes));
    }

    __device__ __forceinline__ s16x8 columns(const lds_char* tile, int d, int block) const
    {
        const lds_char* at = tile + block * (16 * Tile<D>::kRowBytes);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + column_at[d][0]));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + column_at[d][1]));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// ---------------------------------------------------------------------------
// where things lie
// ---------------------------------------------------------------------------
// Heads of rows in memory; distances in bytes.
struct Heads {
    const char* data;
    uint64_t batch, row, head;
    __device__ __forceinline__ const char* at(uint64_t b, uint64_t r, uint64_t h) const
    {
        return data + b * batch + r * row + h * head;
    }
};

// The sequences of a call.  With `starts` they lie one after the other in `rows` rows,
// without it each has `rows` rows of its own of which `lengths` (or all) are there.
struct Sequences {
    const void *starts, *key_starts, *lengths, *key_lengths;
    int wide;                       // indices of 64 bits
    uint32_t batch, rows, key_rows;
    uint32_t group;                 // query heads that share a key head
    int causal;
    uint32_t window;                // 0: none
};

// An index as the device has it, made to lie in [0, most].
__device__ __forceinline__ uint32_t index_at(const void* p, int wide, uint32_t i, uint32_t most)
{
    int64_t x = wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
    x = x < 0 ? 0 : x;
    return x > most ? most : static_cast<uint32_t>(x);
}

// One workgroup's piece: tile `tile` of sequence `batch`.  Rows that belong to no sequence are
// pieces as well, with `length` rows and no key: they get what a row without keys gets.
struct Piece {
    uint32_t batch;                 // to address by; 0 where the rows are flat
    uint32_t tile;
    uint32_t first, length;         // the sequence's queries among the flat rows
    uint32_t key_first, keys;
    uint32_t stored;                // rows from `first` on that the result has
    uint32_t key_stored;
    bool rest;                      // rows of no sequence
    bool valid;
};

// Piece `id` of those that the sequences' rows (by_keys: keys) make in tiles of `tile_rows`, each row counting
// `times`.  All values are the same in all lanes.
__device__ __forceinline__ Piece locate(const Sequences& s, uint32_t id, bool by_keys, uint32_t times,
                                        uint32_t tile_rows)
{
    Piece p{};
    if (!s.starts) {
        const uint32_t stored = by_keys ? s.key_rows : s.rows;
        const uint32_t tiles = ceil_div(stored * times, tile_rows);
        // tile by tile, not sequence by sequence: causal calls have their long pieces first (8 x 1024 tokens, 12 heads of
        // 64: 26.3 us and not 29.8, gradients 79 and not 91), and often one sequence's pieces on one L2
        p.tile = id / s.batch;
        p.batch = id - p.tile * s.batch;
        p.valid = p.tile < tiles;
        if (!p.valid) return p;
        p.length = s.lengths ? uniform(index_at(s.lengths, s.wide, p.batch, s.rows)) : s.rows;
        p.keys = s.key_lengths ? uniform(index_at(s.key_lengths, s.wide, p.batch, s.key_rows)) : s.key_rows;
        p.stored = s.rows;
        p.key_stored = s.key_rows;
        return p;
    }
    // 64 sequences at a time: how many tiles each has, and where the running sum passes `id`; the last two
    // of all are the rows behind the last sequence and those before the first
    const void* starts = by_keys ? s.key_starts : s.starts;
    const uint32_t most = by_keys ? s.key_rows : s.rows;
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t before = 0;
    for (uint32_t at = 0; at < s.batch + 2; at += kWave) {
        const uint32_t e = at + lane;
        uint32_t begin = 0, end = 0;
        if (e < s.batch + 2) {
            begin = e == s.batch + 1 ? 0 : index_at(starts, s.wide, e, most);
            end = e == s.batch ? most : index_at(starts, s.wide, e == s.batch + 1 ? 0 : e + 1, most);
        }
        const uint32_t length = end > begin ? end - begin : 0;
        const uint32_t tiles = ceil_div(length * times, tile_rows);
        uint32_t sum = tiles;
#pragma unroll
        for (uint32_t d = 1; d < kWave; d <<= 1) {
            const uint32_t other = __shfl_up(sum, d);
            if (lane >= d) sum += other;
        }
        const uint64_t past = __ballot(before + sum > id);
        if (past) {
            const int l = __builtin_ctzll(past);
            const uint32_t found = at + l;
            p.tile = id - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));
            const uint32_t first = __builtin_amdgcn_readlane(begin, l), count = __builtin_amdgcn_readlane(length, l);
            p.valid = true;
            p.rest = found >= s.batch;
            p.first = p.key_first = first;
            p.length = p.stored = p.keys = p.key_stored = count;
            if (p.rest) {
                (by_keys ? p.length : p.keys) = 0;
                return p;
            }
            const void* others = by_keys ? s.starts : s.key_starts;
            const uint32_t others_most = by_keys ? s.rows : s.key_rows;
            const uint32_t other = uniform(index_at(others, s.wide, found, others_most));
            const uint32_t other_end = uniform(index_at(others, s.wide, found + 1, others_most));
            const uint32_t other_count = other_end > other ? other_end - other : 0;
            if (by_keys) {
                p.first = other;
                p.length = p.stored = other_count;
            } else {
                p.key_first = other;
                p.keys = p.key_stored = other_count;
            }
            return p;
        }
        before += __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return p;
}

// How many pieces there may be.
inline uint64_t pieces(const Sequences& s, bool by_keys, uint64_t times, uint64_t tile_rows)
{
    const uint64_t rows = by_keys ? s.key_rows : s.rows;
    if (s.starts) return rows * times / tile_rows + s.batch + 2;
    return s.batch * ceil_div(rows * times, tile_rows);
}

// The keys that query `i` of a sequence sees: [lo, hi), hi <= lo where it sees none.  A causal query sees
// itself and what came before it, the last query the last key; with a window the last `window` of them.
struct Seen {
    int32_t lo, hi;
};
__device__ __forceinline__ Seen seen(const Sequences& s, const Piece& p, uint32_t i)
{
    if (i >= p.length) return {0, 0};
    if (!s.causal) return {0, static_cast<int32_t>(p.keys)};
    const int32_t hi = static_cast<int32_t>(i) + 1 + static_cast<int32_t>(p.keys) - static_cast<int32_t>(p.length);
    const int32_t lo = s.window && hi > static_cast<int32_t>(s.window) ? hi - static_cast<int32_t>(s.window) : 0;
    return {lo, hi};
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Rows as the kernels load them: whole 16-byte chunks at multiples of 16 bytes, a tile within a descriptor's reach.
// What lies otherwise is copied to where it does, dim rounded up to a multiple of eight.
struct PackArgs {
    Heads from;
    char* to;
    uint32_t rows, heads, dim;
    uint64_t chunks;
};

static __global__ __launch_bounds__(256) void pack_kernel(PackArgs a)
{
    const uint32_t to_row = ceil_div(a.dim, 8u);
    for (uint64_t at = blockIdx.x * 256ull + threadIdx.x; at < a.chunks; at += gridDim.x * 256ull) {
        const uint64_t head_row = at / to_row;
        const uint32_t first = static_cast<uint32_t>(at % to_row) * 8;
        const uint64_t row = head_row / a.heads;
        const uint16_t* from =
            reinterpret_cast<const uint16_t*>(a.from.at(row / a.rows, row % a.rows, head_row % a.heads)) + first;
        uint32_t x[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) x[i] = first + i < a.dim ? from[i] : 0u;
        *reinterpret_cast<u32x4_t*>(a.to + at * 16) =
            u32x4_t{x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16};
    }
}

inline bool reachable(const void* p) { return !p || la_ptr::device_accessible(p); }

inline bool there(const la_heads_t& h) { return h.data && reinterpret_cast<uintptr_t>(h.data) % 2 == 0; }

inline bool there_fp32(const la_heads_t& h) { return h.data && reinterpret_cast<uintptr_t>(h.data) % 4 == 0; }

inline uint64_t sets(const la_attention_t& c) { return c.starts ? 1 : c.batch; }
inline uint64_t flat_rows(const la_attention_t& c) { return sets(c) * c.rows; }
inline uint64_t flat_keys(const la_attention_t& c) { return sets(c) * c.key_rows; }

inline bool in_chunks(const la_attention_t& c, const la_heads_t& h, bool queries)
{
    const uint64_t rows = queries ? c.rows : c.key_rows, heads = queries ? c.heads : c.kv_heads;
    return c.dim % 8 == 0 && reinterpret_cast<uintptr_t>(h.data) % 16 == 0 && (rows < 2 || h.row_stride % 8 == 0) &&
           (heads < 2 || h.head_stride % 8 == 0) && (sets(c) < 2 || h.batch_stride % 8 == 0);
}

inline bool as_it_lies(const la_attention_t& c, const la_heads_t& h, bool queries)
{
    return in_chunks(c, h, queries) && h.row_stride < 1u << 24;
}

inline uint64_t packed_bytes(const la_attention_t& c, const la_heads_t& h, bool queries)
{
    if (as_it_lies(c, h, queries)) return 0;
    const uint64_t rows = queries ? flat_rows(c) : flat_keys(c);
    return ceil_div(rows * (queries ? c.heads : c.kv_heads) * ceil_div(c.dim, 8ull) * 16, 256ull) * 256;
}

inline la_memory::Place place_of(const la_attention_t& c, const la_heads_t& h, bool queries)
{
    return {reinterpret_cast<uintptr_t>(h.data), 2 * c.dim,
            {sets(c), queries ? c.rows : c.key_rows, queries ? c.heads : c.kv_heads},
            {2 * h.batch_stride, 2 * h.row_stride, 2 * h.head_stride}};
}

// lse: an fp32 to a head.
inline la_memory::Place place_of_lse(const la_attention_t& c)
{
    return {reinterpret_cast<uintptr_t>(c.lse.data), 4, {sets(c), c.rows, c.heads},
            {4 * c.lse.batch_stride, 4 * c.lse.row_stride, 4 * c.lse.head_stride}};
}

// Whether results share no memory with one another, with `read`, or with the indices: kernels read and write in no order,
// and one what the next reads.  They may lie between one another, as parts of a projection's gradient do.
template <int WRITTEN, int READ>
inline bool results_apart(const la_attention_t& c, const la_memory::Place (&written)[WRITTEN],
                          const la_memory::Place (&read)[READ])
{
    using la_memory::flat;
    using la_memory::Place;
    const uint64_t size = c.index_dtype == LA_I64 ? 8 : 4;
    const Place indices[] = {flat(c.starts, (c.batch + 1) * size), flat(c.key_starts, (c.batch + 1) * size),
                             flat(c.lengths, c.batch * size), flat(c.key_lengths, c.batch * size)};
    for (int k = 0; k < WRITTEN; ++k) {
        for (const Place& p : read)
            if (shared(written[k], p)) return false;
        for (const Place& p : indices)
            if (shared(written[k], p)) return false;
        for (int m = 0; m < k; ++m)
            if (shared(written[k], written[m])) return false;
    }
    return true;
}

inline Heads plain(const la_heads_t& h, uint64_t size = 2)
{
    return {static_cast<const char*>(h.data), h.batch_stride * size, h.row_stride * size, h.head_stride * size};
}

// `h` as the kernels read it; where it has to be copied, to `space`, which moves on.
inline int heads_of(const la_attention_t& c, const la_heads_t& h, bool queries, Heads& got, char*& space, hipStream_t st)
{
    got = plain(h);
    const uint64_t bytes = packed_bytes(c, h, queries);
    if (bytes == 0) return LA_OK;
    const uint64_t rows = queries ? c.rows : c.key_rows, heads = queries ? c.heads : c.kv_heads;
    const uint64_t width = ceil_div(c.dim, 8ull) * 16;
    const PackArgs a{got, space, static_cast<uint32_t>(rows), static_cast<uint32_t>(heads), static_cast<uint32_t>(c.dim),
                     sets(c) * rows * heads * (width / 16)};
    const uint64_t blocks = ceil_div(a.chunks, 256ull);
    got = {space, rows * heads * width, heads * width, width};
    space += bytes;
    return launch(pack_kernel, dim3(static_cast<uint32_t>(blocks < 65536 ? blocks : 65536)), dim3(256), st, a);
}

inline Sequences sequences_of(const la_attention_t& c)
{
    const void* key_starts = c.starts && !c.key_starts ? c.starts : c.key_starts;
    return {c.starts, key_starts, c.lengths, c.key_lengths, c.index_dtype == LA_I64, static_cast<uint32_t>(c.batch),
            static_cast<uint32_t>(c.rows), static_cast<uint32_t>(c.key_rows),
            static_cast<uint32_t>(c.heads / c.kv_heads), c.causal,
            static_cast<uint32_t>(c.window < 1u << 30 ? c.window : 1u << 30)};
}

inline bool indices_reachable(const la_attention_t& c)
{
    return reachable(c.starts) && reachable(c.key_starts) && reachable(c.lengths) && reachable(c.key_lengths);
}

// What does not depend on the pointers to data.
inline int check_call(const la_attention_t* call)
{
    if (!call) return LA_EINVAL;
    const la_attention_t& c = *call;
    if (c.dtype != LA_BF16 && c.dtype != LA_F16) return LA_EDTYPE;
    const bool indices = c.starts || c.key_starts || c.lengths || c.key_lengths;
    if (indices && c.index_dtype != LA_I32 && c.index_dtype != LA_I64) return LA_EDTYPE;
    const uintptr_t size = c.index_dtype == LA_I64 ? 8 : 4;
    for (const void* p : {c.starts, c.key_starts, c.lengths, c.key_lengths})
        if (reinterpret_cast<uintptr_t>(p) % size) return LA_EINVAL;
    if (c.starts ? c.lengths || c.key_lengths : c.key_starts != nullptr) return LA_EINVAL;
    constexpr uint64_t kMost = 1ull << 30;
    if (c.batch > kMost || c.rows > kMost || c.key_rows > kMost || c.heads > kMost || c.heads == 0 || c.kv_heads == 0 ||
        c.heads % c.kv_heads || c.dim == 0 || c.dim > 128 || c.batch == 0)
        return LA_EINVAL;
    // rows of all heads are counted in 32 bits
    if (flat_rows(c) > kMost / c.heads || flat_keys(c) > kMost / c.kv_heads) return LA_EINVAL;
    if (c.starts && !c.key_starts && c.rows != c.key_rows) return LA_EINVAL;
    if ((c.window && !c.causal) || !(c.scale > 0.0f) || !std::isfinite(c.scale)) return LA_EINVAL;
    return LA_OK;
}

}  // namespace att

#endif  // SLIDEFORMER_AMD_ATTENTION_TILE_H
