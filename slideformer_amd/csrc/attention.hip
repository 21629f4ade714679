// slideformer_amd: softmax attention over packed or padded sequences, with query
// heads that share key heads (gfx950, wave64).
//
// For a query row q of a sequence with keys k_j and values v_j that it sees:
// s_j = scale q k_j, lse = log sum exp s_j, out = sum exp(s_j - lse) v_j.  One pass over the keys
// with the running maximum m, the running sum l of exp(s_j - m), and the running sum of
// exp(s_j - m) v_j, which both shrink by exp(m - m') when the maximum grows to m'.
//
// The query heads of one key head are rows beside each other, (token, head) in the order
// in which they lie in memory: a tile of keys is loaded once for all of them, and a single new
// token with eight query heads is eight rows.
//
// Scores are S^T = K Q^T, so a lane holds scores of one row (see attention_tile.h); their exponentials, rounded
// to the 16 bits that the matrix cores take, are the second operand of out^T += V^T P^T.  That rounding is the one
// before the result's own: half a step for each probability, in no direction, so a row's result is off by less than
// half a step of its largest terms (bf16: 2.2e-3 of all results where the rounding of exact ones is 1.6e-3).  bf16 has
// fp32's range.  fp16 has not: see Held.  The sum l is that of the unrounded values, in fp32 like the maxima and the sums
// of products.
#include "attention_tile.h"

#include <algorithm>

namespace {

using namespace att;

constexpr uint32_t kMostParts = 64;                      // the join has a lane for each

struct ForwardArgs {
    Heads q, k, v, out, lse;
    float* partial;                 // of each part: [part][row][D], then lse in base 2: [part][row]
    Sequences seq;
    uint32_t heads, kv_heads, dim;  // dim: of the result
    uint32_t read_dim;              // of q, k, v: a multiple of 8
    float scale;
    uint32_t parts, part_tiles;     // the keys' tiles are shared out in runs of part_tiles
    uint32_t rows_all;              // flat rows of the result, over all heads
    int aligned;                    // rows of the result may be written 16 bytes at a time
};

// How P is held, relative to a row's reference st.top: times 2^kUp.  Exponentials need the maximum of no tile but a
// row's first: those of later ones add up to less than kMost nearly always, and where they do not, the scores are made
// again and the references raised.  Looking for the maximum of every tile instead is 21 more vector instructions of about
// 165, which bind heads of 64.
template <typename T> struct Held {
    static constexpr bool kLowers = false;
    static constexpr float kUp = 0.0f, kDown = 1.0f, kMost = 4096.0f;
};
// fp16 holds 2^-24 to 65504, and where one key is far above the others, as a text's first token often is, the others are
// below that beside it: 40000 of them, 17.5 lower, gave results up to 49 % off where the first one's value is small.  So
// P is held times 2^9, and where a tile's sum is less than kLeast, the reference is lowered to the tile's maximum, and
// `sum` and `out`, in fp32, raised by as much; so are the wave's other rows whose sum is less than kLow, which would soon
// be next.  A probability is then off by half a step, or by 2^-20 of its tile's sum.  Lowering ends with sums of kLowered
// and more, beside which what is lower still is nothing in fp16 results; it is by 2^kStep at the most, so that sums of
// products stay below 2^(kStep + 50) * 65504.
// 8192 tokens, causal, 32 and 8 heads of 128: 562 us, and 553 with P held times 1 as bf16's; 8 x 1024, 12 heads of 64:
// 28.9 and 27.4; with a first key 17.5 above the others 563 and 29.5.
template <> struct Held<_Float16> {
    static constexpr bool kLowers = true;
    static constexpr float kUp = 9.0f, kDown = 0x1p-9f, kMost = 65024.0f;    // 127 * 2^9; each term is below 65504
    static constexpr float kLeast = 0x1p-5f, kLow = 0x1p5f;                  // 2^-14 and 2^-4 times 2^9
    static constexpr float kLowered = 0x1p50f, kStep = 40.0f;
};

// The running state of 32 rows in a wave: of row l % 32 a lane has the elements 32 d + 8 (i / 4) + 4 (l / 32) + i % 4.
template <int D> struct State {
    f32x16 out[D / 32];             // times 2^Held::kUp
    float top;                      // the score that `sum` and `out` are relative to: -inf until the row's first key
    float sum;                      // over this half's keys, or, where Held::kLowers, all; times 2^Held::kUp
    __device__ __forceinline__ void init(const Seen& row)
    {
#pragma unroll
        for (int d = 0; d < D / 32; ++d) out[d] = zeros();
        top = row.hi > row.lo ? -INFINITY : 0.0f;        // one that sees nothing waits for no key
        sum = 0.0f;
    }
};

template <typename T, int D, int KEYS>
__device__ __forceinline__ void scores(f32x16 (&s)[KEYS / 32], const s16x8 (&q)[D / 16], const lds_char* k,
                                       const Fragments<D>& f)
{
#pragma unroll
    for (int b = 0; b < KEYS / 32; ++b) {
        s[b] = zeros();
#pragma unroll
        for (int e = 0; e < D / 16; ++e) s[b] = mfma<T>(f.rows(k, e, b), q[e], s[b]);
    }
}

// Scores of keys outside the row's [lo, hi) become -inf, whatever they were.
template <int KEYS>
__device__ __forceinline__ void mask(f32x16 (&s)[KEYS / 32], int32_t first_key, const Seen& row)
{
    const int32_t half = static_cast<int32_t>(threadIdx.x % kWave / 32) * 4;
    const uint32_t from = static_cast<uint32_t>(row.lo - first_key - half);
    const uint32_t count = row.hi > row.lo ? static_cast<uint32_t>(row.hi - row.lo) : 0u;
#pragma unroll
    for (int b = 0; b < KEYS / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t key = b * 32 + i / 4 * 8 + i % 4;
            s[b][i] = key - from < count ? s[b][i] : -INFINITY;
        }
}

// P of scores relative to st.top, as it is held, in their place; returns its sum over this half's keys, or all.
template <typename T, int D, int KEYS>
__device__ __forceinline__ float exponentials(const State<D>& st, f32x16 (&s)[KEYS / 32], float factor)
{
    // rows that have seen nothing yet: 0, and exp2(-inf) below
    const float from = st.top == -INFINITY ? 0.0f : __builtin_fmaf(-st.top, factor, Held<T>::kUp);
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < KEYS / 32; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = exp2_of(__builtin_fmaf(s[b][i], factor, from));
#pragma unroll
        for (int i = 0; i < 16; i += 4) sum += (s[b][i] + s[b][i + 1]) + (s[b][i + 2] + s[b][i + 3]);
    }
    return Held<T>::kLowers ? both_sum(sum) : sum;
}

// The sum over all keys, relative to st.top.
template <typename T, int D> __device__ __forceinline__ float sum_of(const State<D>& st)
{
    return Held<T>::kLowers ? st.sum * Held<T>::kDown : both_sum(st.sum);
}

// Moves the rows' references to the maxima of these scores, up in any case, down where `lower` says so, and brings the
// sums to them.
template <typename T, int D, int KEYS>
__device__ __forceinline__ void refer(State<D>& st, const f32x16 (&s)[KEYS / 32], float factor, bool lower)
{
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < KEYS / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = both_max(top);
    if constexpr (Held<T>::kLowers) {
        top = fmaxf(top, lower ? st.top - Held<T>::kStep / factor : st.top);
    } else {
        top = fmaxf(top, st.top);
    }
    const float times = top == st.top ? 1.0f : exp2_of((st.top - top) * factor);
    st.top = top;
    st.sum *= times;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) st.out[d] *= times;
}

// Takes KEYS keys (32 or 64) of a tile in.
template <typename T, int D, int KEYS>
__device__ __forceinline__ void take(State<D>& st, const s16x8 (&q)[D / 16], const lds_char* k, const lds_char* v,
                                     const Fragments<D>& f, float factor, bool partly, int32_t first_key, const Seen& row)
{
    f32x16 s[KEYS / 32];
    scores<T, D, KEYS>(s, q, k, f);
    if (partly) mask<KEYS>(s, first_key, row);
    if (__any(st.top == -INFINITY)) refer<T, D, KEYS>(st, s, factor, false);
    float sum = exponentials<T, D, KEYS>(st, s, factor);
    bool again, lower = false;
    if constexpr (Held<T>::kLowers) {
        // in one comparison what is nearly never so, NaN and 0 (nothing seen) among it
        constexpr uint32_t kFrom = __builtin_bit_cast(uint32_t, Held<T>::kLeast);
        constexpr uint32_t kTo = __builtin_bit_cast(uint32_t, Held<T>::kMost);
        again = __any(__float_as_uint(sum) - kFrom > kTo - kFrom);
        if (again) {
            const bool lowers = sum > 0.0f && st.sum < Held<T>::kLowered;
            lower = lowers && sum < Held<T>::kLow;
            again = __any(sum > Held<T>::kMost || (lowers && sum < Held<T>::kLeast));
        }
    } else {
        again = __any(sum > Held<T>::kMost);
    }
    if (again) {
        scores<T, D, KEYS>(s, q, k, f);
        if (partly) mask<KEYS>(s, first_key, row);
        refer<T, D, KEYS>(st, s, factor, lower);
        sum = exponentials<T, D, KEYS>(st, s, factor);
    }
    st.sum += sum;
#pragma unroll
    for (int b = 0; b < KEYS / 32; ++b)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const s16x8 p = rounded<T>(s[b], half);
#pragma unroll
            for (int d = 0; d < D / 32; ++d) st.out[d] = mfma<T>(f.columns(v, d, b * 2 + half), p, st.out[d]);
        }
}

// Eight elements of a row from either half of the lanes' four: lane l gets elements 16 j + 8 (l / 32) .. + 7 of
// its row, j = 0, 1 of the 32 that `x` has.
__device__ __forceinline__ void neighbours(const f32x16& x, int j, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Halves h = halves(__float_as_uint(x[j * 8 + i]), __float_as_uint(x[j * 8 + 4 + i]));
        v[i] = __uint_as_float(h.lo);
        v[4 + i] = __uint_as_float(h.hi);
    }
}

template <typename T>
__device__ __forceinline__ void store_eight(char* row, uint32_t at, uint32_t dim, bool aligned, const float (&v)[8])
{
    T* to = reinterpret_cast<T*>(row) + at;
    if (aligned && at + 8 <= dim) {
        *reinterpret_cast<u32x4_t*>(to) = Elem<T>::pack(v);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (at + i < dim) to[i] = Elem<T>::from_f32(v[i]);
    }
}

__device__ __forceinline__ void put(const char* to, float x) { *reinterpret_cast<float*>(const_cast<char*>(to)) = x; }

// The wave's 32 rows, rows `first` of the piece on, to the result or to this part's partial one.
template <typename T, int D>
__device__ __forceinline__ void finish(const ForwardArgs& a, const Piece& p, uint32_t kv_head, uint32_t part, uint32_t row,
                                       State<D>& st)
{
    const uint32_t half = lane_now() / 32;
    const uint32_t token = row / a.seq.group, head = kv_head * a.seq.group + row % a.seq.group;
    const float sum = sum_of<T>(st);
    // a row that sees nothing: zeros, and -inf
    const float scale = sum == 0.0f ? 0.0f : Held<T>::kDown / sum;
    const bool there = token < p.stored;
    const uint64_t flat = (static_cast<uint64_t>(p.batch) * a.seq.rows + p.first + token) * a.heads + head;
    if (a.parts > 1) {
        const uint64_t at = static_cast<uint64_t>(part) * a.rows_all + flat;
        float* to = a.partial + at * D;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float v[4] = {st.out[d][i] * scale, st.out[d][i + 1] * scale, st.out[d][i + 2] * scale,
                                    st.out[d][i + 3] * scale};
                if (there) *reinterpret_cast<u32x4_t*>(to + d * 32 + i * 2 + half * 4) = Elem<float>::pack(v);
            }
        if (there && half == 0)
            a.partial[static_cast<uint64_t>(a.parts) * a.rows_all * D + at] =
                sum == 0.0f ? -INFINITY : st.top * a.scale * kLog2E + __builtin_amdgcn_logf(sum);
        return;
    }
    char* to = const_cast<char*>(a.out.at(p.batch, p.first + token, head));
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float v[8];
            neighbours(st.out[d], j, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= scale;
            if (there) store_eight<T>(to, d * 32 + j * 16 + half * 8, a.dim, a.aligned, v);
        }
    if (there && half == 0)
        put(a.lse.at(p.batch, p.first + token, head),
            sum == 0.0f ? -INFINITY : st.top * a.scale + __builtin_amdgcn_logf(sum) * kLn2);
}

// This lane's row as the second operand of the scores: elements 16 k + 8 (l / 32) .. + 7.
template <int D>
__device__ __forceinline__ void load_row(s16x8 (&q)[D / 16], const char* row, bool there, uint32_t dim)
{
    const uint32_t half = threadIdx.x % kWave / 32;
#pragma unroll
    for (uint32_t k = 0; k < D / 16; ++k) {
        u32x4_t u = {0, 0, 0, 0};
        if (there && k * 16 + half * 8 < dim) u = *reinterpret_cast<const u32x4_t*>(row + (k * 16 + half * 8) * 2);
        q[k] = __builtin_bit_cast(s16x8, u);
    }
    // the loads are over before others begin that are counted by hand
#pragma unroll
    for (uint32_t k = 0; k < D / 16; ++k) asm volatile("" : "+v"(q[k]));
}

// 128 rows to a workgroup, 32 to a wave; all waves go over the same tiles of 64 keys, two of which are
// in LDS: one in work, the next on its way.  Two workgroups on a compute unit (four of D = 64), each in the
// other's pauses.  8192 tokens, causal, 32 and 8 heads of 128 in bf16: 511 us, 1.08 PFLOP/s, the matrix cores busy 60 % of
// the cycles (launches settle at that after some twenty; those first ones, while the clock is found, take 522 to 677).
// 8 x 1024 tokens, causal, 12 heads of 64: 28 us, 0.46 PFLOP/s, matrix cores busy 31 %: with half the products for each
// exponential the vector instructions bind, 15 to a product, and the launch is as long as its longest piece.  Two
// variants took fewer cycles and no less time, as the clock sank with them (1.95 GHz in a first launch, 1.6 to 1.7 under
// load): scores of the next tile between the exponentials of this one, and eight waves that take turns at multiplying and
// at exponentials (541 and 530, where this took 525).
template <typename T, int D> __global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attention_kernel(ForwardArgs a)
{
    constexpr uint32_t kBytes = Tile<D>::kBytes;
    __shared__ __attribute__((aligned(1024))) char shared[4 * kBytes];
    const uint32_t kv_head = blockIdx.x % a.kv_heads, part = blockIdx.y;
    Piece p = locate(a.seq, blockIdx.x / a.kv_heads, false, a.seq.group, 128);
    if (!p.valid) return;
    {
        // the last rows of a causal sequence see the most keys: they begin
        const uint32_t tiles = ceil_div(p.stored * a.seq.group, 128u);
        p.tile = tiles - 1 - p.tile;
    }
    const uint32_t wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t group = a.seq.group;
    const uint32_t row = p.tile * 128 + wave * 32 + lane % 32;
    const uint32_t token = row / group;
    const Seen mine = seen(a.seq, p, token);

    // the keys that the workgroup's rows see, and this wave's
    const uint32_t last_row = p.length * group;          // one past
    const auto range = [&](uint32_t row_from, uint32_t row_to) {
        row_to = row_to < last_row ? row_to : last_row;
        if (row_from >= row_to) return Seen{0, 0};
        return Seen{seen(a.seq, p, row_from / group).lo, seen(a.seq, p, (row_to - 1) / group).hi};
    };
    const Seen all = range(p.tile * 128, p.tile * 128 + 128);
    const uint32_t wave_row = p.tile * 128 + wave * 32;
    const Seen own = range(wave_row, wave_row + 32);
    // and those that all of them see
    const bool full = wave_row + 32 <= last_row;
    const Seen common = full ? Seen{seen(a.seq, p, (wave_row + 31) / group).lo, seen(a.seq, p, wave_row / group).hi}
                             : Seen{0, 0};
    int32_t tile = all.lo / static_cast<int32_t>(kTileRows);
    int32_t end = all.hi > 0 ? (all.hi + static_cast<int32_t>(kTileRows) - 1) / static_cast<int32_t>(kTileRows) : 0;
    if (a.parts > 1) {
        const int32_t from = static_cast<int32_t>(part * a.part_tiles), to = from + static_cast<int32_t>(a.part_tiles);
        tile = tile > from ? tile : from;
        end = end < to || part + 1 == a.parts ? end : to;
    }

    State<D> st;
    st.init(mine);
    if (tile < end) {
        const Rows keys{reinterpret_cast<uint64_t>(a.k.at(p.batch, p.key_first, kv_head)), static_cast<int32_t>(p.keys)};
        const Rows values{reinterpret_cast<uint64_t>(a.v.at(p.batch, p.key_first, kv_head)), static_cast<int32_t>(p.keys)};
        Loader<D, kTileRows, 4> load_k, load_v;
        load_k.init(wave, static_cast<uint32_t>(a.k.row), a.read_dim);
        load_v.init(wave, static_cast<uint32_t>(a.v.row), a.read_dim);
        Fragments<D> f;
        f.init();
        lds_char* lds = (lds_char*)shared;
        const uint32_t place = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + wave * 1024;
        const float factor = a.scale * kLog2E;
        load_k.load(keys, tile * kTileRows, place);
        load_v.load(values, tile * kTileRows, place + kBytes);
        s16x8 q[D / 16];
        load_row<D>(q, a.q.at(p.batch, p.first + token, kv_head * group + row % group), token < p.length, a.read_dim);
        uint32_t buffer = 0;
        for (; tile < end; ++tile, buffer ^= 2 * kBytes) {
            arrive<0>();
            if (tile + 1 < end) {
                load_k.load(keys, (tile + 1) * kTileRows, place + (buffer ^ 2 * kBytes));
                load_v.load(values, (tile + 1) * kTileRows, place + (buffer ^ 2 * kBytes) + kBytes);
            }
            const int32_t first_key = tile * static_cast<int32_t>(kTileRows);
            if (first_key < own.hi && first_key + static_cast<int32_t>(kTileRows) > own.lo) {
                const lds_char* k = lds + buffer;
                const bool partly = first_key < common.lo || first_key + static_cast<int32_t>(kTileRows) > common.hi;
                take<T, D, 64>(st, q, k, k + kBytes, f, factor, partly, first_key, mine);
            }
        }
    }
    finish<T, D>(a, p, kv_head, part, wave_row + lane_now() % 32, st);
}

// At most 32 rows to a workgroup (a single new token's heads): its waves take the same rows and different keys, each
// with tiles of its own in LDS and without waiting for the others, and join at the end.  Two waves, so that
// two workgroups or more are on a compute unit and one's start and end are under the other's loads.
// Bound by memory: a wave takes 0.8 us for 32 keys where loads do not bind.  16 rows of 32/8 heads of 128 over caches
// of 8192 filled to 5600 on average, 367 MB: 76 us, 4.8 TB/s; one row over 65536, 268 MB: 43.7 us, 6.1 TB/s.  With five
// tiles in a ring, four of them on their way, one row over 65536 keys of eight heads took 47.9 us instead of 44.4, with
// four waves 46.5.
constexpr uint32_t kFewWaves = 2;

template <typename T, int D> __global__ __launch_bounds__(kFewWaves * 64, 1) void few_rows_kernel(ForwardArgs a)
{
    constexpr uint32_t kKeys = 32, kBytes = Tile<D>::kBytes / 2;
    constexpr uint32_t kOwn = 4 * kBytes;                // a wave's share of LDS: keys and values of two tiles
    __shared__ __attribute__((aligned(1024))) char shared[kFewWaves * kOwn];
    const uint32_t kv_head = blockIdx.x % a.kv_heads, part = blockIdx.y;
    const Piece p = locate(a.seq, blockIdx.x / a.kv_heads, false, a.seq.group, 32);
    if (!p.valid) return;
    const uint32_t wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t group = a.seq.group;
    const uint32_t row = p.tile * 32 + lane % 32;
    const uint32_t token = row / group;
    const Seen mine = seen(a.seq, p, token);

    const uint32_t last_row = p.length * group, row_from = p.tile * 32;
    const uint32_t row_to = row_from + 32 < last_row ? row_from + 32 : last_row;
    Seen all{0, 0}, common{0, 0};
    if (row_from < row_to) {
        const Seen first = seen(a.seq, p, row_from / group), last = seen(a.seq, p, (row_to - 1) / group);
        all = {first.lo, last.hi};
        // those that all of them see: none where rows behind a sequence's are among what is written
        if (row_to == row_from + 32 || row_to == p.stored * group) common = {last.lo, first.hi};
    }
    int32_t tile = all.lo / static_cast<int32_t>(kKeys);
    int32_t end = all.hi > 0 ? (all.hi + static_cast<int32_t>(kKeys) - 1) / static_cast<int32_t>(kKeys) : 0;
    if (a.parts > 1) {
        const int32_t from = static_cast<int32_t>(part * a.part_tiles), to = from + static_cast<int32_t>(a.part_tiles);
        tile = tile > from ? tile : from;
        end = end < to || part + 1 == a.parts ? end : to;
    }

    State<D> st;
    st.init(mine);
    lds_char* lds = (lds_char*)shared;
    if (tile < end) {
        const Rows keys{reinterpret_cast<uint64_t>(a.k.at(p.batch, p.key_first, kv_head)), static_cast<int32_t>(p.keys)};
        const Rows values{reinterpret_cast<uint64_t>(a.v.at(p.batch, p.key_first, kv_head)), static_cast<int32_t>(p.keys)};
        Loader<D, kKeys, 1> load_k, load_v;
        load_k.init(0, static_cast<uint32_t>(a.k.row), a.read_dim);
        load_v.init(0, static_cast<uint32_t>(a.v.row), a.read_dim);
        Fragments<D> f;
        f.init();
        const lds_char* own = lds + wave * kOwn;
        const uint32_t place = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(own));
        const float factor = a.scale * kLog2E;
        // A wave's tiles, from one of them on and round: caches that lie a power of two apart would otherwise all be
        // read from the same few memory channels at a time.
        const int32_t mine_from = tile + static_cast<int32_t>(wave);
        const int32_t count = mine_from < end ? (end - mine_from + static_cast<int32_t>(kFewWaves) - 1) / static_cast<int32_t>(kFewWaves) : 0;
        const uint32_t ids = gridDim.x * gridDim.y, id = blockIdx.x + blockIdx.y * gridDim.x;
        int32_t at = static_cast<int32_t>(static_cast<uint64_t>(id) * static_cast<uint32_t>(count) / ids), load_at = at;
        const auto first_of = [&](int32_t t) {
            return (mine_from + t * static_cast<int32_t>(kFewWaves)) * static_cast<int32_t>(kKeys);
        };
        const auto turn = [&](int32_t& t) { t = t + 1 == count ? 0 : t + 1; };
        const auto load = [&](uint32_t to) {
            load_k.load(keys, first_of(load_at), place + to);
            load_v.load(values, first_of(load_at), place + to + kBytes);
            turn(load_at);
        };
        if (count > 0) load(0);
        s16x8 q[D / 16];
        load_row<D>(q, a.q.at(p.batch, p.first + token, kv_head * group + row % group), token < p.length, a.read_dim);
        uint32_t buffer = 0;
        for (int32_t t = 0; t < count; ++t, buffer ^= 2 * kBytes) {
            // after the last tile the first one is loaded again, and waited for like any other
            load(buffer ^ 2 * kBytes);
            arrived<2 * Loader<D, kKeys, 1>::kLoads>();
            const lds_char* k = own + buffer;
            const int32_t first_key = first_of(at);
            turn(at);
            const bool partly = first_key < common.lo || first_key + static_cast<int32_t>(kKeys) > common.hi;
            take<T, D, 32>(st, q, k, k + kBytes, f, factor, partly, first_key, mine);
            // what was read is read before the next loads write over it
            arrived<2 * Loader<D, kKeys, 1>::kLoads>();
        }
        arrived<0>();
    }
    // the waves' states, each shrunk to the largest of their maxima, added in the order of the waves
    st.sum = sum_of<T>(st);
    __syncthreads();                                     // no tile is read any more
    constexpr uint32_t kRow = D + 4;                     // keeps 32 rows' accesses in different banks
    static_assert(kFewWaves * 32 * (kRow + 2) * 4 <= kFewWaves * kOwn, "the states fit the tiles' place");
    float(*tops)[32] = reinterpret_cast<float(*)[32]>(shared + kFewWaves * 32 * kRow * 4);
    float(*sums)[32] = tops + kFewWaves;
    if (lane < 32) tops[wave][lane] = st.top, sums[wave][lane] = st.sum;
    __syncthreads();
    const uint32_t r = lane % 32;
    float top = tops[0][r];
#pragma unroll
    for (uint32_t w = 1; w < kFewWaves; ++w) top = fmaxf(top, tops[w][r]);
    const float factor = a.scale * kLog2E;
    float sum = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kFewWaves; ++w)
        sum += tops[w][r] == -INFINITY ? sums[w][r] : sums[w][r] * exp2_of((tops[w][r] - top) * factor);
    const float shrink = st.top == -INFINITY ? 1.0f : exp2_of((st.top - top) * factor);
    float* mine_out = reinterpret_cast<float*>(shared) + wave * 32 * kRow;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float v[4] = {st.out[d][i] * shrink, st.out[d][i + 1] * shrink, st.out[d][i + 2] * shrink,
                                st.out[d][i + 3] * shrink};
            *reinterpret_cast<u32x4_t*>(mine_out + r * kRow + d * 32 + i * 2 + lane / 32 * 4) = Elem<float>::pack(v);
        }
    __syncthreads();
    // a row to 2 * kFewWaves lanes; the statistics are those of lane row % 32
    const uint32_t out_row = threadIdx.x / (2 * kFewWaves), at = threadIdx.x % (2 * kFewWaves);
    const uint32_t piece_row = p.tile * 32 + out_row, out_token = piece_row / group;
    const uint32_t head = kv_head * group + piece_row % group;
    // from lanes of rows that may not be there: before any lane leaves
    const float row_sum = __shfl(sum, static_cast<int>(out_row % 32)), row_top = __shfl(top, static_cast<int>(out_row % 32));
    if (out_token >= p.stored) return;
    const float scale = row_sum == 0.0f ? 0.0f : Held<T>::kDown / row_sum;
    const uint64_t flat = (static_cast<uint64_t>(p.batch) * a.seq.rows + p.first + out_token) * a.heads + head;
    char* to = const_cast<char*>(a.out.at(p.batch, p.first + out_token, head));
    float* part_to = a.partial + (static_cast<uint64_t>(part) * a.rows_all + flat) * D;
#pragma unroll
    for (uint32_t e = at * 8; e < D; e += 16 * kFewWaves) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float* from = reinterpret_cast<const float*>(shared) + out_row * kRow + e + i;
            v[i] = from[0];
#pragma unroll
            for (uint32_t w = 1; w < kFewWaves; ++w) v[i] += from[w * 32 * kRow];
            v[i] *= scale;
        }
        if (a.parts > 1) store_vec<float, 8>(part_to, e / 8, D, v);
        else store_eight<T>(to, e, a.dim, a.aligned, v);
    }
    if (at == 0) {
        if (a.parts > 1)
            a.partial[static_cast<uint64_t>(a.parts) * a.rows_all * D + static_cast<uint64_t>(part) * a.rows_all + flat] =
                row_sum == 0.0f ? -INFINITY : row_top * factor + __builtin_amdgcn_logf(row_sum);
        else
            put(a.lse.at(p.batch, p.first + out_token, head),
                row_sum == 0.0f ? -INFINITY : row_top * a.scale + __builtin_amdgcn_logf(row_sum) * kLn2);
    }
}

// The parts' results of one row into one, each by its share exp(lse of the part - lse of all): a wave to a row, eight
// elements to a lane, the lanes beside each other in turn on the parts.  All latency: 4.8 us for 32 rows of 64 parts,
// as for 512 of 4, with the launch before it about 10 us of a step.  Partial results are fp32.
template <typename T, int D> __global__ __launch_bounds__(256) void join_kernel(ForwardArgs a)
{
    constexpr uint32_t kLanes = D / 8, kSide = kWave / kLanes;
    __shared__ float shares[4][kMostParts];
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t flat = blockIdx.x * 4 + uniform(threadIdx.x / kWave);
    if (flat >= a.rows_all) return;
    const float* lses = a.partial + static_cast<uint64_t>(a.parts) * a.rows_all * D + flat;
    const float lse = lane < a.parts ? lses[static_cast<uint64_t>(lane) * a.rows_all] : -INFINITY;
    float top = lse;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float share = lse == -INFINITY ? 0.0f : exp2_of(lse - top);
    const float sum = wave_sum(share);
    shares[threadIdx.x / kWave][lane] = share;
    __builtin_amdgcn_wave_barrier();                     // read by this wave alone, whose accesses stay in order
    float v[8] = {};
#pragma unroll 4
    for (uint32_t part = lane / kLanes; part < a.parts; part += kSide) {
        const float w = shares[threadIdx.x / kWave][part];
        const float* from = a.partial + (static_cast<uint64_t>(part) * a.rows_all + flat) * D;
        float lo[4], hi[4];
        load_vec<float>(from, lane % kLanes * 2, D, lo);
        load_vec<float>(from, lane % kLanes * 2 + 1, D, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __builtin_fmaf(w, lo[i], v[i]);
            v[4 + i] = __builtin_fmaf(w, hi[i], v[4 + i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (uint32_t d = kLanes; d < kWave; d <<= 1) v[i] += __shfl_xor(v[i], static_cast<int>(d));
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
    const uint32_t head = flat % a.heads, row = flat / a.heads;
    char* to = const_cast<char*>(a.out.at(row / a.seq.rows, row % a.seq.rows, head));
    if (lane < kLanes) store_eight<T>(to, lane * 8, a.dim, a.aligned, v);
    if (lane == 0)
        put(a.lse.at(row / a.seq.rows, row % a.seq.rows, head),
            sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint64_t kFill = 512;                          // workgroups that fill the card, two on a compute unit

struct Plan {
    bool few;                                            // rows of a sequence fit a workgroup of few_rows_kernel
    uint64_t parts, part_tiles;
    uint64_t pieces;
    uint32_t padded;                                     // the kernels' D
    uint64_t partial_bytes;
};

Plan plan_of(const la_attention_t& c)
{
    Plan p{};
    const Sequences s = sequences_of(c);
    const uint64_t group = c.heads / c.kv_heads;
    p.padded = c.dim <= 64 ? 64 : 128;
    // Packed queries are of few rows if they are on average; longer ones among them are more pieces.
    const uint64_t rows = s.starts ? ceil_div(c.rows, c.batch) : c.rows;
    p.few = rows * group <= 32;
    p.pieces = pieces(s, false, group, p.few ? 32 : 128);
    const uint64_t tile = p.few ? 32 : kTileRows;
    // Keys are shared out where there are too few pieces to fill the card: in parts of 512 keys and more for two
    // workgroups on a compute unit, in shorter ones for one; what is left then is the start and the join.
    //   One row, 8 heads of 128: 4096 keys 18.5 us in parts of 512 and 12.2 of 128, 16384 keys 20.4 in 32 parts and 21.7
    //   in 64; four rows, 8192 keys, 33.8 in 16 and 36.6 in 8; 256 keys 10.2 in one part and 11.5 in two.
    //   128 rows, 12 heads of 64, 1024 keys: 15.6 us in two parts and 12.7 in four; 512 keys 11.0 in one and 12.4 in two.
    // What the join reads of many rows grows with the workgroups, and a part's own time with its keys, so a part of these
    // has 8 keys for each workgroup too: 12 heads of 64, 4 x 1024 tokens (384 workgroups) take 43 us in two parts and 24
    // in one; 32/8 heads of 128, 128 rows of 8 sequences (256), 41 and 27 against 1024 keys and 317 and 332 against
    // 16384; and one such sequence of 4096 (32) 23 in eight parts and 75 in one.
    const uint64_t keys = s.starts ? ceil_div(c.key_rows, c.batch) : c.key_rows;
    const uint64_t tiles = ceil_div(keys, tile), workgroups = std::max<uint64_t>(1, p.pieces * c.kv_heads);
    const uint64_t joined = p.few ? 0 : 8 * workgroups, least = std::max<uint64_t>(p.few ? 128 : 256, joined);
    const auto fill = [&](uint64_t of) { return p.few ? ceil_div(of, workgroups) : of / workgroups; };
    const uint64_t shorter = std::min(fill(kFill / 2), keys < 3 * least ? 1 : keys / least);
    p.parts = std::min(fill(kFill), std::max(shorter, keys / std::max<uint64_t>(512, joined)));
    p.parts = std::max<uint64_t>(1, std::min<uint64_t>(p.parts, kMostParts));
    p.part_tiles = ceil_div(std::max<uint64_t>(1, tiles), p.parts);
    p.parts = std::max<uint64_t>(1, ceil_div(tiles, p.part_tiles));
    p.partial_bytes = p.parts > 1 ? p.parts * flat_rows(c) * c.heads * (p.padded + 1) * sizeof(float) : 0;
    p.partial_bytes = ceil_div(p.partial_bytes, 256) * 256;
    return p;
}

template <typename T, int D> int run(const Plan& p, const ForwardArgs& a, hipStream_t stream)
{
    const dim3 grid(static_cast<uint32_t>(p.pieces * a.kv_heads), static_cast<uint32_t>(p.parts));
    int rc = p.few ? launch(few_rows_kernel<T, D>, grid, dim3(kFewWaves * 64), stream, a)
                   : launch(attention_kernel<T, D>, grid, dim3(256), stream, a);
    if (rc == LA_OK && p.parts > 1)
        rc = launch(join_kernel<T, D>, dim3(ceil_div(a.rows_all, 4u)), dim3(256), stream, a);
    return rc;
}

template <typename T> int run(const Plan& p, const ForwardArgs& a, hipStream_t stream)
{
    return p.padded == 64 ? run<T, 64>(p, a, stream) : run<T, 128>(p, a, stream);
}

}  // namespace

extern "C" {

uint64_t la_attention_workspace(const la_attention_t* call)
{
    if (check_call(call) != LA_OK || flat_rows(*call) == 0) return 0;
    const Plan p = plan_of(*call);
    return p.partial_bytes + packed_bytes(*call, call->q, true) + packed_bytes(*call, call->k, false) +
           packed_bytes(*call, call->v, false);
}

int la_attention(const la_attention_t* call, void* workspace, uint64_t workspace_bytes, la_stream_t stream)
{
    int rc = check_call(call);
    if (rc != LA_OK) return rc;
    const la_attention_t& c = *call;
    if (flat_rows(c) == 0) return LA_OK;
    if (!there(c.q) || !there(c.out) || !there_fp32(c.lse) ||
        (flat_keys(c) > 0 && (!there(c.k) || !there(c.v))))
        return LA_EINVAL;
    const Plan p = plan_of(c);
    rc = check_workspace(workspace, workspace_bytes, la_attention_workspace(call), 256);
    if (rc != LA_OK) return rc;
    if (p.pieces * c.kv_heads >> 31) return LA_EINVAL;
    if (!reachable(c.q.data) || !reachable(c.k.data) || !reachable(c.v.data) || !reachable(c.out.data) ||
        !reachable(c.lse.data) || !indices_reachable(c) || (la_attention_workspace(call) && !reachable(workspace)))
        return LA_EFAULT;
    if (!results_apart(c, {place_of(c, c.out, true), place_of_lse(c)},
                       {place_of(c, c.q, true), place_of(c, c.k, false), place_of(c, c.v, false)}))
        return LA_EINVAL;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    ForwardArgs a{};
    a.partial = reinterpret_cast<float*>(ws);
    ws += p.partial_bytes;
    rc = heads_of(c, c.q, true, a.q, ws, st);
    if (rc == LA_OK) rc = heads_of(c, c.k, false, a.k, ws, st);
    if (rc == LA_OK) rc = heads_of(c, c.v, false, a.v, ws, st);
    if (rc != LA_OK) return rc;
    a.out = plain(c.out);
    a.lse = plain(c.lse, 4);
    a.seq = sequences_of(c);
    a.heads = static_cast<uint32_t>(c.heads);
    a.kv_heads = static_cast<uint32_t>(c.kv_heads);
    a.dim = static_cast<uint32_t>(c.dim);
    a.read_dim = ceil_div(a.dim, 8u) * 8;
    a.scale = c.scale;
    a.parts = static_cast<uint32_t>(p.parts);
    a.part_tiles = static_cast<uint32_t>(p.part_tiles);
    a.rows_all = static_cast<uint32_t>(flat_rows(c) * c.heads);
    a.aligned = in_chunks(c, c.out, true);
    return c.dtype == LA_BF16 ? run<__bf16>(p, a, st) : run<_Float16>(p, a, st);
}

}  // extern "C"
