// slideformer_amd: the gradients of attention (gfx950, wave64).
//
// With P = exp(scale q k - lse), computed again from q, k and the rows' lse, dP = dO V^T and
// delta = sum over elements of dO O, per row: dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q,
// dV = P^T dO.
//
// Two kernels, and no float is added atomically: grad_q_kernel has 32 rows of queries to
// a wave and goes over the keys, grad_kv_kernel 32 keys to a wave and goes over the rows of all
// query heads that share them.  Both compute S and dP, so that there are seven products
// where five would do; the two more cost less than adding dQ in memory from every tile
// of keys would, and results do not depend on an order.
//
// As in the forward pass each product's result is the next one's second operand as it
// lies in the registers: (K Q^T, V dO^T) -> dS^T -> K^T dS^T by queries, and (Q K^T, dO V^T) -> P, dS ->
// (dO^T P, Q^T dS) by keys.
//
// delta is the diagonal of O dO^T, by the matrix instructions that make dP of V and dO, in the
// same order: a row that sees one key has O = V and exactly no dS.
//
// P and dS are rounded to the operands' 16 bits before the last three products, as the matrix cores take them, and
// delta, but for short sequences and windows, is that of the O that was given, itself rounded: bf16 gradients of q and k
// are up to 2.8e-3 off where rounding the exact ones is 1.7e-3 off, fp16 3.5e-4 and 2.1e-4.  A delta from the sums of P dP
// would not have O's rounding, but would be wrong with an lse over more keys than the call has.  Everything else is fp32.
#include "attention_tile.h"

#include <algorithm>

namespace {

using namespace att;

struct GradArgs {
    Heads q, k, v, out, grad_out, lse;
    Heads grad_q, grad_k, grad_v;
    float *less, *delta;            // [heads][flat rows], by grad_q_kernel: minus lse in base 2, and delta
    Sequences seq;
    uint32_t heads, kv_heads, dim, read_dim;
    uint32_t rows_all;              // flat rows
    float scale;
    int q_aligned, k_aligned, v_aligned;
    int keep_rest;
    uint32_t parts, chain;          // of grad_kv_kernel: see Span
    uint32_t pieces;                // of keys
    int neighbours;                 // a piece's parts beside each other, not a part's pieces
    float* partial;                 // [part][flat keys][kv_heads][k's and v's][D]
    uint32_t keys_all;              // flat keys
};

// The rows that see keys [from, to) of a sequence, those of a workgroup in tiles of 64, of each of its query heads.
// Where they are more than `chain` tiles, up to `parts` workgroups share them and add their sums in join_kv_kernel: a
// launch takes as long as its longest chain of tiles.
struct Span {
    Seen rows;
    int32_t tile_from, tiles;       // of one head
    int32_t count;                  // of all heads
    int32_t parts;
};

// Those that see some of keys [from, to): none where the sequence has no such key.
__device__ __forceinline__ Seen rows_of(const Sequences& s, const Piece& p, uint32_t from, uint32_t to)
{
    if (from >= p.keys) return {0, 0};
    Seen r{0, static_cast<int32_t>(p.length)};
    if (!s.causal) return r;
    const int32_t shift = static_cast<int32_t>(p.keys) - static_cast<int32_t>(p.length);
    r.lo = static_cast<int32_t>(from) - shift;
    r.lo = r.lo < 0 ? 0 : r.lo;
    const int32_t last = static_cast<int32_t>(to) - 1 - shift;           // sees key `to` - 1 as its last
    if (s.window && last + static_cast<int64_t>(s.window) < r.hi) r.hi = last + static_cast<int32_t>(s.window);
    return r;
}

template <int D> __device__ __forceinline__ Span span_of(const GradArgs& a, const Piece& p)
{
    const uint32_t first = p.tile * 128, past = first + 128 < p.keys ? first + 128 : p.keys;
    Span s{};
    s.rows = p.rest ? Seen{0, 0} : rows_of(a.seq, p, first, past);
    s.tile_from = s.rows.lo / static_cast<int32_t>(kTileRows);
    const int32_t to = s.rows.hi > 0 ? (s.rows.hi + static_cast<int32_t>(kTileRows) - 1) / static_cast<int32_t>(kTileRows) : 0;
    s.tiles = to > s.tile_from ? to - s.tile_from : 0;
    s.count = s.tiles * static_cast<int32_t>(a.seq.group);
    s.parts = 1;
    if (a.parts > 1 && s.count > static_cast<int32_t>(a.chain)) {
        s.parts = (s.count + static_cast<int32_t>(a.chain) - 1) / static_cast<int32_t>(a.chain);
        s.parts = s.parts < static_cast<int32_t>(a.parts) ? s.parts : static_cast<int32_t>(a.parts);
    }
    return s;
}

// Waits until what wrote these sums has, and what reads them may: longer than any matrix instruction needs.
template <int N> __device__ __forceinline__ void settle(f32x16 (&x)[N])
{
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+a"(x[n]));
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15");
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+a"(x[n]));
}

// dS in the operands' 16 bits.  bfloat16 has fp32's range.  fp16 has not: what a wave rounds is brought near the
// top of its range by a power of two for each column, which shrinks when a larger value comes, and its
// sums with it; P, at most 1, by a fixed one.
template <typename T> struct Range {
    static constexpr float kP = 0.0f;
    __device__ __forceinline__ float factor() const { return 1.0f; }
    template <bool SETTLE, int N> __device__ __forceinline__ void fit(f32x16&, f32x16 (&)[N]) {}
};
template <> struct Range<_Float16> {
    static constexpr float kP = 14.0f;                   // P is held times 2^14
    float up = 0x1p60f;
    __device__ __forceinline__ float factor() const { return up; }
    template <bool SETTLE, int N> __device__ __forceinline__ void fit(f32x16& x, f32x16 (&sums)[N])
    {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, __builtin_fabsf(x[i]));
        if (__any(most * up > 32768.0f)) {
            // to 2^10 .. 2^11: five doublings before it shrinks again
            most = both_max(most);
            int e;
            (void)frexpf(most, &e);
            e = 11 - e;
            e = e < -60 ? -60 : e > 60 ? 60 : e;
            const float now = most * up > 32768.0f && most < INFINITY ? __builtin_ldexpf(1.0f, e) : up;
            const float shrink = now / up;
            up = now;
            if constexpr (SETTLE) settle(sums);
#pragma unroll
            for (int n = 0; n < N; ++n) sums[n] *= shrink;
            if constexpr (SETTLE) settle(sums);
        }
        x *= up;
    }
};

// Of 16 values of rows (or keys) first + 8 (i / 4) + 4 (l / 32) + i % 4, those outside [lo, hi) become zero.
__device__ __forceinline__ void hide(f32x16& x, int32_t first, const Seen& range)
{
    const int32_t half = static_cast<int32_t>(threadIdx.x % kWave / 32) * 4;
    const uint32_t from = static_cast<uint32_t>(range.lo - first - half);
    const uint32_t count = range.hi > range.lo ? static_cast<uint32_t>(range.hi - range.lo) : 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t at = i / 4 * 8 + i % 4;
        x[i] = at - from < count ? x[i] : 0.0f;
    }
}

// This lane's row as an operand: elements 16 k + 8 (l / 32) .. + 7.
template <int D> __device__ __forceinline__ void load_row(s16x8 (&q)[D / 16], const char* row, bool there, uint32_t dim)
{
    const uint32_t half = threadIdx.x % kWave / 32;
#pragma unroll
    for (uint32_t k = 0; k < D / 16; ++k) {
        u32x4_t u = {0, 0, 0, 0};
        if (there && k * 16 + half * 8 < dim) u = *reinterpret_cast<const u32x4_t*>(row + (k * 16 + half * 8) * 2);
        q[k] = __builtin_bit_cast(s16x8, u);
    }
}
// It is there: no load of it is in flight beside those that are counted by hand.
template <int D> __device__ __forceinline__ void have_row(s16x8 (&q)[D / 16])
{
#pragma unroll
    for (uint32_t k = 0; k < D / 16; ++k) asm volatile("" : "+v"(q[k]));
}

template <typename T, int D>
__device__ __forceinline__ f32x16 product(const lds_char* tile, const s16x8 (&x)[D / 16], const Fragments<D>& f, int block)
{
    f32x16 s = zeros();
#pragma unroll
    for (int k = 0; k < D / 16; ++k) s = mfma<T>(f.rows(tile, k, block), x[k], s);
    return s;
}

// A lane's row of 32 of a result [D][32 rows].
template <typename T, int D>
__device__ __forceinline__ void store_row(char* to, const f32x16 (&x)[D / 32], float scale, bool there, uint32_t dim,
                                          bool aligned)
{
    const uint32_t half = threadIdx.x % kWave / 32;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Halves h = halves(__float_as_uint(x[d][j * 8 + i]), __float_as_uint(x[d][j * 8 + 4 + i]));
                v[i] = __uint_as_float(h.lo) * scale;
                v[4 + i] = __uint_as_float(h.hi) * scale;
            }
            const uint32_t at = d * 32 + j * 16 + half * 8;
            T* out = reinterpret_cast<T*>(to) + at;
            if (!there) continue;
            if (aligned && at + 8 <= dim) {
                *reinterpret_cast<u32x4_t*>(out) = Elem<T>::pack(v);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    if (at + i < dim) out[i] = Elem<T>::from_f32(v[i]);
            }
        }
}

// Workgroups whose rows see no more keys than these make delta from P and dP instead, in 32 bits, which takes as long again as
// two of the three products: out is rounded, and where a row sees few keys dP - delta may be much smaller than
// either.  Two tokens, two heads: grads were 0.22 off; windows of two or three keys 0.03.  128 rows in windows of 64
// keys see 191, in three tiles or, where the first begins inside one, four.  What is beyond is at most 2.8e-3 off.
constexpr int32_t kOwnKeys = 192;

// 128 rows to a workgroup, 32 to a wave, tiles of 64 keys as in the forward pass, and two workgroups on a compute unit.
// 8192 tokens in five packed documents of 717 to 3588, 32/8 heads of 128 in bf16: 244 us, 0.95 PFLOP/s of its three
// products (261 in the first twenty launches, while the clock is found); 8 x 1024 tokens, 12 heads of 64, 33 us.  The
// matrix cores are busy 51 and 35 % of the cycles: between a tile's scores and its sums a wave has exponentials, and one
// other wave whose products could go on meanwhile.
template <typename T, int D> __global__ __launch_bounds__(256, 2) void grad_q_kernel(GradArgs a)
{
    constexpr uint32_t kBytes = Tile<D>::kBytes;
    __shared__ __attribute__((aligned(1024))) char shared[4 * kBytes];
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    Piece p = locate(a.seq, blockIdx.x / a.kv_heads, false, a.seq.group, 128);
    if (!p.valid) return;
    p.tile = ceil_div(p.stored * a.seq.group, 128u) - 1 - p.tile;
    const uint32_t wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t group = a.seq.group;
    const uint32_t row = p.tile * 128 + wave * 32 + lane % 32;
    const uint32_t token = row / group, head = kv_head * group + row % group;
    const bool there = token < p.length;
    const Seen mine = seen(a.seq, p, token);
    const uint64_t flat = static_cast<uint64_t>(p.batch) * a.seq.rows + p.first + token;

    const uint32_t last_row = p.length * group;
    const auto range = [&](uint32_t row_from, uint32_t row_to) {
        row_to = row_to < last_row ? row_to : last_row;
        if (row_from >= row_to) return Seen{0, 0};
        return Seen{seen(a.seq, p, row_from / group).lo, seen(a.seq, p, (row_to - 1) / group).hi};
    };
    const Seen all = range(p.tile * 128, p.tile * 128 + 128);
    const uint32_t wave_row = p.tile * 128 + wave * 32;
    const Seen own = range(wave_row, wave_row + 32);
    const bool full = wave_row + 32 <= last_row;
    const Seen common = full ? Seen{seen(a.seq, p, (wave_row + 31) / group).lo, seen(a.seq, p, wave_row / group).hi}
                             : Seen{0, 0};
    int32_t tile = all.lo / static_cast<int32_t>(kTileRows);
    const int32_t end = all.hi > 0 ? (all.hi + static_cast<int32_t>(kTileRows) - 1) / static_cast<int32_t>(kTileRows) : 0;

    // the first tile is on its way while this lane's row is fetched
    const Rows keys{reinterpret_cast<uint64_t>(a.k.at(p.batch, p.key_first, kv_head)), static_cast<int32_t>(p.keys)};
    const Rows values{reinterpret_cast<uint64_t>(a.v.at(p.batch, p.key_first, kv_head)), static_cast<int32_t>(p.keys)};
    Loader<D, kTileRows, 4> load_k, load_v;
    load_k.init(wave, static_cast<uint32_t>(a.k.row), a.read_dim);
    load_v.init(wave, static_cast<uint32_t>(a.v.row), a.read_dim);
    lds_char* lds = (lds_char*)shared;
    const uint32_t place = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + wave * 1024;
    if (tile < end) {
        load_k.load(keys, tile * kTileRows, place);
        load_v.load(values, tile * kTileRows, place + kBytes);
    }
    s16x8 q[D / 16], g[D / 16];
    float delta, lse2;
    {
        s16x8 o[D / 16];
        load_row<D>(g, a.grad_out.at(p.batch, p.first + token, head), there, a.read_dim);
        load_row<D>(o, a.out.at(p.batch, p.first + token, head), there, a.read_dim);
        load_row<D>(q, a.q.at(p.batch, p.first + token, head), there, a.read_dim);
        lse2 = there ? *reinterpret_cast<const float*>(a.lse.at(p.batch, p.first + token, head)) * kLog2E : 0.0f;
        f32x16 x = zeros();
#pragma unroll
        for (int k = 0; k < D / 16; ++k) x = mfma<T>(o[k], g[k], x);
        // column c's own row: element 4 (c / 8) + c % 4 of the half of lanes c / 4 % 2
        const uint32_t c = lane % 32;
        float found = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) found = c / 8 * 4 + c % 4 == static_cast<uint32_t>(i) ? x[i] : found;
        const Halves h = halves(__float_as_uint(found), __float_as_uint(found));
        delta = __uint_as_float(c / 4 % 2 ? h.hi : h.lo);
        have_row<D>(q);
        have_row<D>(g);
        asm volatile("" : "+v"(lse2));
    }
    Fragments<D> f;
    f.init();
    const float factor = a.scale * kLog2E;
    if (tile < end && all.hi - all.lo <= kOwnKeys) {
        // delta from P and dP themselves, in a pass of its own
        float products = 0.0f, sum = 0.0f;
        uint32_t buffer = 0;
        for (int32_t t = tile; t < end; ++t, buffer ^= 2 * kBytes) {
            arrive<0>();
            if (t + 1 < end) {
                load_k.load(keys, (t + 1) * kTileRows, place + (buffer ^ 2 * kBytes));
                load_v.load(values, (t + 1) * kTileRows, place + (buffer ^ 2 * kBytes) + kBytes);
            }
            const int32_t first_key = t * static_cast<int32_t>(kTileRows);
            const lds_char *k = lds + buffer, *v = k + kBytes;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                f32x16 s = product<T, D>(k, q, f, b);
                f32x16 d = product<T, D>(v, g, f, b);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = exp2_of(__builtin_fmaf(s[i], factor, -lse2));
                    d[i] *= s[i];
                }
                hide(s, first_key + b * 32, mine);
                hide(d, first_key + b * 32, mine);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sum += s[i];
                    products += d[i];
                }
            }
        }
        sum = both_sum(sum);
        products = both_sum(products);
        // where keys are missing that lse covers, and where there is one, delta stays that of out
        if (mine.hi - mine.lo > 1 && __builtin_fabsf(sum - 1.0f) < 0x1p-12f) delta = products / sum;
        arrive<0>();                                     // all waves have read the tiles
        load_k.load(keys, tile * kTileRows, place);
        load_v.load(values, tile * kTileRows, place + kBytes);
    }
    if (there && lane < 32) {
        const uint64_t at = static_cast<uint64_t>(head) * a.rows_all + flat;
        a.less[at] = Range<T>::kP - lse2;
        a.delta[at] = delta;
    }

    f32x16 sums[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) sums[d] = zeros();
    Range<T> scaled;
    if (tile < end) {
        uint32_t buffer = 0;
        for (; tile < end; ++tile, buffer ^= 2 * kBytes) {
            arrive<0>();
            if (tile + 1 < end) {
                load_k.load(keys, (tile + 1) * kTileRows, place + (buffer ^ 2 * kBytes));
                load_v.load(values, (tile + 1) * kTileRows, place + (buffer ^ 2 * kBytes) + kBytes);
            }
            const int32_t first_key = tile * static_cast<int32_t>(kTileRows);
            if (first_key >= own.hi || first_key + static_cast<int32_t>(kTileRows) <= own.lo) continue;
            const lds_char *k = lds + buffer, *v = k + kBytes;
            const bool partly = first_key < common.lo || first_key + static_cast<int32_t>(kTileRows) > common.hi;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                f32x16 s = product<T, D>(k, q, f, b);
                f32x16 d = product<T, D>(v, g, f, b);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    d[i] = exp2_of(__builtin_fmaf(s[i], factor, -lse2)) * (d[i] - delta);
                if (partly) hide(d, first_key + b * 32, mine);
                scaled.template fit<false>(d, sums);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const s16x8 ds = rounded<T>(d, half);
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) sums[e] = mfma<T>(f.columns(k, e, b * 2 + half), ds, sums[e]);
                }
            }
        }
    }
    const bool stored = token < (a.keep_rest ? (p.rest ? 0u : p.length) : p.stored);
    store_row<T, D>(const_cast<char*>(a.grad_q.at(p.batch, p.first + token, head)), sums, a.scale / scaled.factor(), stored,
                    a.dim, a.q_aligned);
}

// The products of grad_kv_kernel, in assembly: the sums stay in accumulation registers, and so do a wave's own
// keys and values; left to itself the compiler moves them to and fro.  It adds no wait states
// to these.  Their first operands come from LDS and need none, P and dS are settled before the sums begin, and
// scores are read no sooner than a phase later.
template <typename T> __device__ __forceinline__ void add_product(f32x16& c, const s16x8& a, const s16x8& b);
template <> __device__ __forceinline__ void add_product<__bf16>(f32x16& c, const s16x8& a, const s16x8& b)
{
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <> __device__ __forceinline__ void add_product<_Float16>(f32x16& c, const s16x8& a, const s16x8& b)
{
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <typename T> __device__ __forceinline__ void score(f32x16& c, const s16x8& a, const s16x8& b, bool first);
template <> __device__ __forceinline__ void score<__bf16>(f32x16& c, const s16x8& a, const s16x8& b, bool first)
{
    if (first) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "a"(b));
    else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
}
template <> __device__ __forceinline__ void score<_Float16>(f32x16& c, const s16x8& a, const s16x8& b, bool first)
{
    if (first) asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "a"(b));
    else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b));
}

// One wait for four reads of LDS in place of one for each.
__device__ __forceinline__ void wait_for(const s16x8& a, const s16x8& b, const s16x8& c, const s16x8& d)
{
    asm volatile("" : : "v"(a), "v"(b), "v"(c), "v"(d));
}

template <int N> struct Number {
    static constexpr int value = N;
};

// A wave's 32 keys and what it goes through, 32 rows at a time:
//   products   the scores S and dP of the next rows (2 D / 16 matrix instructions), between which
//   values     P and dS of these rows are made of theirs;
//   sums       dV and dK of these rows (4 D / 32 matrix instructions).
// So the matrix cores have work while exponentials are taken, though a SIMD has one wave.
template <typename T, int D> struct Keys {
    static constexpr uint32_t kBytes = Tile<D>::kBytes;
    static constexpr uint32_t kRowValues = kTileRows * 4;    // bytes of a tile's lse, and of its delta
    static constexpr uint32_t kBuffer = 2 * kBytes + 4 * 2 * kRowValues;     // Q, dO, and a copy of these for each wave
    static constexpr int kSteps = D / 16, kParts = D / 32;
    static constexpr int kEach = 16 / (2 * kSteps);          // values made beside a product
    f32x16 sums_k[kParts], sums_v[kParts];
    s16x8 k[kSteps], v[kSteps];
    Range<T> scaled;
    // Buffers come in two pairs.  What is read of the one in a pair is known beforehand; after a pair the places are
    // moved to the other one, those of the scores, which run ahead, before those of the sums.
    Fragments<D> f;
    const lds_char* values;
    const lds_char* lds;
    uint32_t rows_on, columns_on;   // to the other pair
    float factor;

    struct Scores {
        f32x16 s, d;
    };

    // Of the tile in buffer BUF: fragment m of block B for the scores, S's and dP's in turn,
    template <int BUF, int B> __device__ __forceinline__ s16x8 row_fragment(int m) const
    {
        return f.rows(lds + BUF * kBuffer + m % 2 * kBytes, m / 2, B);
    }
    // and for the sums: dV's, then dK's.
    template <int BUF, int B> __device__ __forceinline__ s16x8 column_fragment(int m) const
    {
        return f.columns(lds + BUF * kBuffer + (m < 2 * kParts ? kBytes : 0), m % kParts, B * 2 + m / kParts % 2);
    }

    // Scores alone, of block 0 of the first tile.
    __device__ __forceinline__ void begin(Scores& x)
    {
#pragma unroll
        for (int m = 0; m < 2 * kSteps; ++m) {
            const s16x8 a = row_fragment<0, 0>(m);
            if (m % 2) score<T>(x.d, a, v[m / 2], m < 2);
            else score<T>(x.s, a, k[m / 2], m < 2);
        }
        asm volatile("s_nop 15\n\ts_nop 15");
    }

    // What a block begins with, read from LDS while the one before ends.
    static constexpr int kAhead = 4;
    struct Begin {
        s16x8 rows[kAhead];
        f32x4 less[4], delta[4];
    };
    template <int BUF, int B> __device__ __forceinline__ void read_values(Begin& x) const
    {
        const lds_char* at = values + BUF * kBuffer + B * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x.less[i] = *reinterpret_cast<const lds_f32x4*>(at + i * 32);
            x.delta[i] = *reinterpret_cast<const lds_f32x4*>(at + kRowValues + i * 32);
        }
    }
    template <int BUF, int B> __device__ __forceinline__ void read_rows(Begin& x) const
    {
#pragma unroll
        for (int m = 0; m < kAhead; ++m) x.rows[m] = row_fragment<BUF, B>(m);
    }

    __device__ __forceinline__ void move_rows()
    {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) f.row_at[k] += rows_on;
        values += static_cast<int32_t>(rows_on);
        rows_on = -rows_on;
    }
    __device__ __forceinline__ void move_columns()
    {
#pragma unroll
        for (int d = 0; d < kParts; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k) f.column_at[d][k] += columns_on;
        columns_on = -columns_on;
    }

    // Block B of the tile in buffer BUF of a pair, whose scores are in `now`; the next block's into `then`.  `between` is called
    // before the sums, beside which `beside` is called 4 * kParts times.
    template <int BUF, int B, typename Between, typename Beside>
    __device__ __forceinline__ void block(Scores& now, Scores& then, Begin& begin, int32_t first_row, const Seen& mine,
                                          bool partly, const Between& between, const Beside& beside)
    {
        constexpr int kNext = B ? 1 - BUF : BUF, kAfter = 1 - BUF;
        s16x8 rows[2 * kSteps], columns[4 * kParts];
#pragma unroll
        for (int m = 0; m < kAhead; ++m) rows[m] = begin.rows[m];
#pragma unroll
        for (int m = 0; m < 2 * kSteps; ++m) {
            // four at a time, so that they are waited for once in four products
            if (m % kAhead == 0)
#pragma unroll
                for (int n = m + kAhead; n < m + 2 * kAhead; ++n) {
                    if (n < 2 * kSteps) rows[n] = row_fragment<kNext, 1 - B>(n);
                    else columns[n - 2 * kSteps] = column_fragment<BUF, B>(n - 2 * kSteps);
                }
            if (m % kAhead == 0) wait_for(rows[m], rows[m + 1], rows[m + 2], rows[m + 3]);
            if (m % 2) score<T>(then.d, rows[m], v[m / 2], m < 2);
            else score<T>(then.s, rows[m], k[m / 2], m < 2);
#pragma unroll
            for (int i = m * kEach; i < (m + 1) * kEach; ++i) {
                now.s[i] = exp2_of(__builtin_fmaf(now.s[i], factor, begin.less[i / 4][i % 4]));
                now.d[i] = now.s[i] * (now.d[i] - begin.delta[i / 4][i % 4]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (partly) {
            hide(now.s, first_row + B * 32, mine);
            hide(now.d, first_row + B * 32, mine);
        }
        scaled.template fit<true>(now.d, sums_k);
        between();
        s16x8 p[2] = {rounded<T>(now.s, 0), rounded<T>(now.s, 1)}, ds[2] = {rounded<T>(now.d, 0), rounded<T>(now.d, 1)};
        asm volatile("s_nop 1" : "+v"(p[0]), "+v"(p[1]), "+v"(ds[0]), "+v"(ds[1]));
#pragma unroll
        for (int m = 0; m < 4 * kParts; ++m) {
            if (m % kAhead == 0 && m + kAhead < 4 * kParts)
#pragma unroll
                for (int n = m + kAhead; n < m + 2 * kAhead; ++n) columns[n] = column_fragment<BUF, B>(n);
            if (m + kAhead == 4 * kParts) {
                read_values<kNext, 1 - B>(begin);
                if (BUF == 1 && B == 0) move_rows();
                read_rows<kAfter, B>(begin);
            }
            if (m % kAhead == 0) wait_for(columns[m], columns[m + 1], columns[m + 2], columns[m + 3]);
            if (m < 2 * kParts) add_product<T>(sums_v[m % kParts], columns[m], p[m / kParts]);
            else add_product<T>(sums_k[m % kParts], columns[m], ds[m / kParts - 2]);
            beside(m);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (BUF == 1 && B == 1) move_columns();
    }
};

// 128 keys to a workgroup, 32 to a wave; all waves go over the same tiles of 64 rows of one query
// head after the other.  Four tiles are in LDS: one whose sums are made, one whose scores are, two on their way.  One wave
// on a SIMD (two of D = 64): both sums and both own operands of 128 keys take 360 registers.
// 8192 tokens in five packed documents of 717 to 3588, 32/8 heads of 128 in bf16: 389 us, 0.79 PFLOP/s of its four
// products (440 in the first twenty launches); 8 x 1024 tokens, 12 heads of 64, 45 us.  The matrix cores are busy 51 and
// 35 % of the cycles, bound by issue (a wave alone issues an instruction in 5.5 cycles, a product takes 32); and compute
// units have work 71 % of the first case's time, for the longest document's first keys are the longest chain.  Two parts
// for each such piece took 10 % longer with the card full, probably since their rows do not come from L2 together.
template <typename T, int D> __global__ __launch_bounds__(256, 1) void grad_kv_kernel(GradArgs a)
{
    using Mine = Keys<T, D>;
    constexpr uint32_t kBytes = Mine::kBytes, kRowValues = Mine::kRowValues, kBuffer = Mine::kBuffer;
    __shared__ __attribute__((aligned(1024))) char shared[4 * kBuffer];
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    const uint32_t id = blockIdx.x / a.kv_heads;
    const Piece p = locate(a.seq, a.neighbours ? id / a.parts : id % a.pieces, true, 1, 128);
    if (!p.valid) return;
    const uint32_t wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t group = a.seq.group;
    const uint32_t key = p.tile * 128 + wave * 32 + lane % 32;
    const bool there = key < p.keys;
    const Span span = span_of<D>(a, p);
    const int32_t part = static_cast<int32_t>(a.neighbours ? id % a.parts : id / a.pieces);
    if (part >= span.parts) return;
    const int32_t tile_from = span.tile_from, tile_to = span.tile_from + span.tiles;
    const int32_t begun = static_cast<int32_t>(static_cast<int64_t>(span.count) * part / span.parts);
    const int32_t count =
        static_cast<int32_t>(static_cast<int64_t>(span.count) * (part + 1) / span.parts) - begun;
    const Seen mine = rows_of(a.seq, p, key, key + 1);
    const uint32_t wave_first = p.tile * 128 + wave * 32;
    const Seen common = wave_first + 32 <= p.keys ? Seen{rows_of(a.seq, p, wave_first + 31, wave_first + 32).lo,
                                                         rows_of(a.seq, p, wave_first, wave_first + 1).hi}
                                                  : Seen{0, 0};

    Mine w;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) w.sums_k[d] = w.sums_v[d] = zeros();
    if (count > 0) {
        w.factor = a.scale * kLog2E;
        Loader<D, kTileRows, 4> load_q, load_g;
        load_q.init(wave, static_cast<uint32_t>(a.q.row), a.read_dim);
        load_g.init(wave, static_cast<uint32_t>(a.grad_out.row), a.read_dim);
        w.lds = (lds_char*)shared;
        const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(w.lds));
        const uint32_t values = 2 * kBytes + wave * 2 * kRowValues;
        w.f.init();
        w.values = w.lds + values + lane / 32 * 16;
        w.rows_on = w.columns_on = 2 * kBuffer;
        // the tile that is loaded next: tiles of a head, then the next head's; past the last nothing
        uint32_t load_head = kv_head * group + begun / span.tiles, load_to = 0;
        int32_t tile = tile_from + begun % span.tiles, load_tile = tile, loads = count, left = 0;
        u32x4_t rsrc_q, rsrc_g;
        uint64_t at_q = 0, at_g = 0, values_at = 0;
        uint32_t values_bytes;
        const uint32_t step_q = kTileRows * load_q.stride, step_g = kTileRows * load_g.stride;
        // In parts, to go between products: where the tile lies, and its loads.
        constexpr int kParts = 4, kLoads = 2 * Loader<D, kTileRows, 4>::kLoads + 2;      // of a wave, for a tile
        const auto aim = [&] {
            const int32_t from = load_tile * static_cast<int32_t>(kTileRows);
            const uint64_t row = static_cast<uint64_t>(p.first) + from;
            left = static_cast<int32_t>(p.length) - from;
            at_q = uniform(reinterpret_cast<uint64_t>(a.q.at(p.batch, row, load_head)));
            at_g = uniform(reinterpret_cast<uint64_t>(a.grad_out.at(p.batch, row, load_head)));
            values_at = (static_cast<uint64_t>(load_head) * a.rows_all + static_cast<uint64_t>(p.batch) * a.seq.rows + row) * 4;
        };
        aim();
        const auto turn = [&] {
            const int32_t rows = loads-- > 0 ? left : 0;
            rsrc_q = load_q.descriptor(at_q, rows);
            rsrc_g = load_g.descriptor(at_g, rows);
            values_bytes = rows <= 0 ? 0u : rows < static_cast<int32_t>(kTileRows) ? rows * 4u : kRowValues;
        };
        const auto advance = [&] {
            at_q += step_q;
            at_g += step_g;
            values_at += kRowValues;
            left -= static_cast<int32_t>(kTileRows);
            if (++load_tile == tile_to) {
                load_tile = tile_from;
                ++load_head;
                aim();
            }
        };
        const auto load_part = [&](int n) {
            if (n == 0) load_q.load(rsrc_q, base + load_to + wave * 1024);
            if (n == 1) load_g.load(rsrc_g, base + load_to + wave * 1024 + kBytes);
            if (n == 2)
                load_values(reinterpret_cast<uint64_t>(a.less) + values_at, values_bytes, base + load_to + values);
            if (n == 3) {
                load_values(reinterpret_cast<uint64_t>(a.delta) + values_at, values_bytes, base + load_to + values + kRowValues);
                load_to = load_to == 3 * kBuffer ? 0 : load_to + kBuffer;
                advance();
            }
        };
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            turn();
#pragma unroll
            for (int k = 0; k < kParts; ++k) load_part(k);
        }
        load_row<D>(w.k, a.k.at(p.batch, p.key_first + key, kv_head), there, a.read_dim);
        load_row<D>(w.v, a.v.at(p.batch, p.key_first + key, kv_head), there, a.read_dim);
#pragma unroll
        for (int m = 0; m < D / 16; ++m) asm volatile("" : "+a"(w.k[m]), "+a"(w.v[m]));
        // the first tile, and these rows, which were asked for later than all three
        arrive<2 * kLoads>();
        typename Mine::Scores even, odd;
        typename Mine::Begin begin;
        w.begin(even);
        w.template read_rows<0, 1>(begin);
        w.template read_values<0, 0>(begin);
        // One tile, in buffer kBuf of a pair.
        const auto step = [&](auto buffer) {
            constexpr int kBuf = decltype(buffer)::value;
            const int32_t first_row = tile * static_cast<int32_t>(kTileRows);
            const bool partly = first_row < common.lo || first_row + static_cast<int32_t>(kTileRows) > common.hi;
            w.template block<kBuf, 0>(
                even, odd, begin, first_row, mine, partly,
                // the next tile is there, and all waves have done with the one before this
                [&] { arrive<kLoads>(); },
                [&](int m) {
                    if (m == 0) turn();
                    if (m > 0 && m <= kParts) load_part(m - 1);
                });
            w.template block<kBuf, 1>(odd, even, begin, first_row, mine, partly, [] {}, [](int) {});
            if (++tile == tile_to) tile = tile_from;
        };
        // where there is an odd number of tiles, one of zeros follows
        for (int32_t t = 0; t < count; t += 2) {
            step(Number<0>{});
            step(Number<1>{});
        }
        // loads into LDS that nobody reads are over before the workgroup is
        arrive<0>();
    }
    settle(w.sums_k);
    settle(w.sums_v);
    constexpr float kShrinkP = Range<T>::kP == 0.0f ? 1.0f : 0x1p-14f;
    const float scale_k = a.scale * kShrinkP / w.scaled.factor();
    if (span.parts > 1) {
        float* to = a.partial + ((static_cast<uint64_t>(part) * a.keys_all + static_cast<uint64_t>(p.batch) * a.seq.key_rows +
                                  p.key_first + key) * a.kv_heads + kv_head) * (2 * D);
        if (!there) return;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float x[4], y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = w.sums_k[d][i + e] * scale_k;
                    y[e] = w.sums_v[d][i + e] * kShrinkP;
                }
                const uint32_t at = d * 32 + i * 2 + lane / 32 * 4;
                *reinterpret_cast<u32x4_t*>(to + at) = Elem<float>::pack(x);
                *reinterpret_cast<u32x4_t*>(to + D + at) = Elem<float>::pack(y);
            }
        return;
    }
    const bool stored = key < (a.keep_rest ? (p.rest ? 0u : p.keys) : p.key_stored);
    store_row<T, D>(const_cast<char*>(a.grad_v.at(p.batch, p.key_first + key, kv_head)), w.sums_v, kShrinkP, stored, a.dim,
                    a.v_aligned);
    store_row<T, D>(const_cast<char*>(a.grad_k.at(p.batch, p.key_first + key, kv_head)), w.sums_k, scale_k, stored, a.dim,
                    a.k_aligned);
}

// The sums of keys whose rows several workgroups shared, in the order of the parts: eight elements to a lane.  A workgroup
// takes 256 / (2 D / 8) of a piece's 128 keys, one round of loads: 5.3 us for 70 pieces of up to three parts, where all 128
// in one workgroup's rounds took 20.
template <typename T, int D> __global__ __launch_bounds__(256) void join_kv_kernel(GradArgs a)
{
    constexpr uint32_t kChunks = 2 * D / 8;              // of a key's two rows
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    const Piece p = locate(a.seq, blockIdx.x / a.kv_heads, true, 1, 128);
    if (!p.valid) return;
    const Span span = span_of<D>(a, p);
    if (span.parts < 2) return;
    const uint32_t key = p.tile * 128 + blockIdx.y * (256 / kChunks) + threadIdx.x / kChunks, e = threadIdx.x % kChunks * 8;
    // beyond a sequence's keys there are no sums; those rows get zeros, if anything
    if (key >= (a.keep_rest ? p.keys : p.key_stored)) return;
    float v[8] = {};
    if (key < p.keys)
#pragma unroll 4
        for (int32_t part = 0; part < span.parts; ++part) {
            const float* from = a.partial + ((static_cast<uint64_t>(part) * a.keys_all +
                                              static_cast<uint64_t>(p.batch) * a.seq.key_rows + p.key_first + key) *
                                                 a.kv_heads + kv_head) * (2 * D) + e;
            float lo[4], hi[4];
            load_vec<float>(from, 0, 8, lo);
            load_vec<float>(from, 1, 8, hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] += lo[i];
                v[4 + i] += hi[i];
            }
        }
    const bool of_v = e >= D;
    const Heads& to = of_v ? a.grad_v : a.grad_k;
    T* out = reinterpret_cast<T*>(const_cast<char*>(to.at(p.batch, p.key_first + key, kv_head)));
    const uint32_t first = e % D;
    if ((of_v ? a.v_aligned : a.k_aligned) && first + 8 <= a.dim) {
        *reinterpret_cast<u32x4_t*>(out + first) = Elem<T>::pack(v);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (first + i < a.dim) out[first + i] = Elem<T>::from_f32(v[i]);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
uint64_t row_values_bytes(const la_attention_t& c) { return ceil_div(flat_rows(c) * c.heads * 4, 256ull) * 256; }

// How the rows of keys are shared out, from what the host knows: sequences of average length, of which one may be as long
// as all are.
struct Parts {
    uint64_t parts = 1, chain = 0, bytes = 0;
    bool neighbours = false;
};

Parts parts_of(const la_attention_t& c)
{
    Parts p;
    const uint64_t rows = c.starts ? ceil_div(c.rows, c.batch) : c.rows;
    const uint64_t keys = c.starts ? ceil_div(c.key_rows, c.batch) : c.key_rows;
    const uint64_t fill = c.dim <= 64 ? 512 : 256;       // workgroups that the card takes at a time
    const uint64_t group = c.heads / c.kv_heads, workgroups = c.batch * c.kv_heads * ceil_div(keys, 128);
    const uint64_t most = c.window ? (128 + c.window) / kTileRows + 2 : ~0ull;          // tiles of a head that see 128 keys
    const uint64_t tiles = std::min(ceil_div(rows, kTileRows), most);
    const uint64_t longest = group * std::min<uint64_t>(ceil_div(c.rows, kTileRows), most);
    if (longest > 8 && workgroups > 0 && workgroups < fill) {
        // Without parts, and with: 16/2 heads of 64, 1 x 1024 tokens 160 and 43 us, of 128 1 x 2048 450 and 126; 16/4 heads
        // of 64, 8 x 1024 130 and 114.  No more parts than the card has room for (32/8 heads of 128, 4 x 512: 72 us, and 90
        // with chains of ten tiles), and none of fewer than six tiles, which take about as long as the join.  Chains of full
        // or windowed sequences are about as long as each other; causal ones are of all lengths up to the longest, and
        // half a part is left over of each.
        const bool alike = !c.causal || most == tiles;
        const uint64_t chain = alike ? ceil_div(group * tiles, fill / workgroups)
                                     : ceil_div(workgroups * group * (tiles / 2 + 1), fill - workgroups / 2);
        // More than four only where the launch is resident at once if all have them: workgroups go to the compute
        // units in turn, and wait behind long ones where others are free (32/8 heads of 128, 1 x 1024: 77 us, and 98 with
        // eight; 16/2 heads 97 and 75).
        const uint64_t most_parts = std::min<uint64_t>(16, std::max<uint64_t>(4, fill / workgroups));
        p.chain = std::max({chain, ceil_div(group * tiles, most_parts), uint64_t{6}});
        p.parts = std::min(most_parts, ceil_div(longest, p.chain));
        // Where not all are resident at once, long chains begin with all parts of the longest: 16/2 heads of 128, 1 x 8192
        // tokens 1108 us, and 1358 with all first parts first; 32/8 heads, 1 x 2048 (chains of 45 tiles) 170 and 199, but
        // 2 x 1024 (24) 110 and 100.
        p.neighbours = workgroups * p.parts > fill && p.chain > 32;
    }
    if (p.parts > 1)
        p.bytes = ceil_div(p.parts * flat_keys(c) * c.kv_heads * 2 * (c.dim <= 64 ? 64 : 128) * sizeof(float), 256ull) * 256;
    return p;
}

template <typename T, int D> int run(const la_attention_t& c, const GradArgs& a, hipStream_t stream)
{
    int rc = LA_OK;
    const uint64_t by_rows = pieces(a.seq, false, a.seq.group, 128) * c.kv_heads;
    const uint64_t by_keys = pieces(a.seq, true, 1, 128) * c.kv_heads;
    if (flat_rows(c) > 0) rc = launch(grad_q_kernel<T, D>, dim3(static_cast<uint32_t>(by_rows)), dim3(256), stream, a);
    if (rc == LA_OK && flat_keys(c) > 0)
        rc = launch(grad_kv_kernel<T, D>, dim3(static_cast<uint32_t>(by_keys * a.parts)), dim3(256), stream, a);
    if (rc == LA_OK && flat_keys(c) > 0 && a.parts > 1)
        rc = launch(join_kv_kernel<T, D>, dim3(static_cast<uint32_t>(by_keys), 128 / (256 / (2 * D / 8))), dim3(256), stream, a);
    return rc;
}

template <typename T> int run(const la_attention_t& c, const GradArgs& a, hipStream_t stream)
{
    return c.dim <= 64 ? run<T, 64>(c, a, stream) : run<T, 128>(c, a, stream);
}

}  // namespace

extern "C" {

uint64_t la_attention_grad_workspace(const la_attention_t* call)
{
    if (check_call(call) != LA_OK) return 0;
    const la_attention_t& c = *call;
    return 2 * row_values_bytes(c) + parts_of(c).bytes + packed_bytes(c, c.q, true) + packed_bytes(c, c.k, false) +
           packed_bytes(c, c.v, false) + packed_bytes(c, c.out, true) + packed_bytes(c, c.grad_out, true);
}

int la_attention_grad(const la_attention_t* call, void* workspace, uint64_t workspace_bytes, la_stream_t stream)
{
    int rc = check_call(call);
    if (rc != LA_OK) return rc;
    const la_attention_t& c = *call;
    const bool rows = flat_rows(c) > 0, keys = flat_keys(c) > 0;
    if ((rows && (!there(c.q) || !there(c.out) || !there(c.grad_out) || !there(c.grad_q) ||
                  !there_fp32(c.lse))) ||
        (keys && (!there(c.k) || !there(c.v) || !there(c.grad_k) || !there(c.grad_v))))
        return LA_EINVAL;
    rc = check_workspace(workspace, workspace_bytes, la_attention_grad_workspace(call), 256);
    if (rc != LA_OK) return rc;
    const Sequences s = sequences_of(c);
    if (pieces(s, false, s.group, 128) * c.kv_heads >> 31 || pieces(s, true, 1, 128) * c.kv_heads >> 31) return LA_EINVAL;
    for (const void* p : {c.q.data, c.k.data, c.v.data, c.out.data, c.grad_out.data, c.grad_q.data, c.grad_k.data,
                          c.grad_v.data, c.lse.data})
        if (!reachable(p)) return LA_EFAULT;
    if (!indices_reachable(c) || !reachable(workspace)) return LA_EFAULT;
    if (!results_apart(c, {place_of(c, c.grad_q, true), place_of(c, c.grad_k, false), place_of(c, c.grad_v, false)},
                       {place_of(c, c.q, true), place_of(c, c.k, false), place_of(c, c.v, false), place_of(c, c.out, true),
                        place_of(c, c.grad_out, true), place_of_lse(c)}))
        return LA_EINVAL;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    GradArgs a{};
    a.lse = plain(c.lse, 4);
    a.less = reinterpret_cast<float*>(ws);
    a.delta = reinterpret_cast<float*>(ws + row_values_bytes(c));
    ws += 2 * row_values_bytes(c);
    const Parts parts = parts_of(c);
    a.parts = static_cast<uint32_t>(parts.parts);
    a.chain = static_cast<uint32_t>(parts.chain);
    a.neighbours = parts.neighbours;
    a.pieces = static_cast<uint32_t>(pieces(s, true, 1, 128));
    a.partial = reinterpret_cast<float*>(ws);
    a.keys_all = static_cast<uint32_t>(flat_keys(c));
    ws += parts.bytes;
    rc = heads_of(c, c.q, true, a.q, ws, st);
    if (rc == LA_OK) rc = heads_of(c, c.k, false, a.k, ws, st);
    if (rc == LA_OK) rc = heads_of(c, c.v, false, a.v, ws, st);
    if (rc == LA_OK) rc = heads_of(c, c.out, true, a.out, ws, st);
    if (rc == LA_OK) rc = heads_of(c, c.grad_out, true, a.grad_out, ws, st);
    if (rc != LA_OK) return rc;
    a.grad_q = plain(c.grad_q);
    a.grad_k = plain(c.grad_k);
    a.grad_v = plain(c.grad_v);
    a.seq = s;
    a.heads = static_cast<uint32_t>(c.heads);
    a.kv_heads = static_cast<uint32_t>(c.kv_heads);
    a.dim = static_cast<uint32_t>(c.dim);
    a.read_dim = ceil_div(a.dim, 8u) * 8;
    a.rows_all = static_cast<uint32_t>(flat_rows(c));
    a.scale = c.scale;
    a.q_aligned = in_chunks(c, c.grad_q, true);
    a.k_aligned = in_chunks(c, c.grad_k, false);
    a.v_aligned = in_chunks(c, c.grad_v, false);
    a.keep_rest = c.keep_rest;
    return c.dtype == LA_BF16 ? run<__bf16>(c, a, st) : run<_Float16>(c, a, st);
}

}  // extern "C"
