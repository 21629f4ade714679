// slideformer_amd: softmax cross entropy of hidden states against a vocabulary
// matrix, with its gradients (gfx950, wave64).  The loss holds one tile of scores at a
// time; with gradients the softmax of a piece of the rows is held, in 16 bits.
//
//   s = X W^T,  loss_i = log(sum_v exp(s_iv)) - s_i,t(i),
//   D_iv = exp(s_iv) / sum_v exp(s_iv) - [v = t(i)],  dX = D W,  dW = D^T X.
//
// Rows without a target take no part: the trained rows' indices are listed on the
// device, X is gathered by them, and every product works on as many rows as
// there are, which only the device knows.  What an ignored row holds (NaN
// too) reaches nothing, and a batch that is half prompt costs half.
//
// A tile of scores is reduced where it is computed: each row's largest score m
// and sum of exp(s - m) over the tile's 256 columns go to `parts`, and are
// joined over the tiles afterwards in a fixed order.  With gradients the tile
// also leaves exp(s - m) in 16 bits for a piece of the rows at a time; one pass
// then turns it into D, since exp(s - lse) = exp(s - m) exp(m - lse) and both are
// known by then.  That keeps the work at three matrix products: cutting the
// vocabulary into pieces instead would save the row pieces' memory (bounded by
// piece_rows here), but each piece's softmax needs every score of the row first,
// so all scores would be computed twice.
//
// D is rounded to the operands' 16 bits, as the matrix cores take it, on top of the
// rounding of exp(s - m): two relative errors of at most 2^-8 (bf16) each, of
// independent sign, in sums over thousands of terms.  fp16 has few exponents: there
// exp(s - m) and D are held times 2^13, so that probabilities down to 2^-27 stay normal
// numbers.  Everything else is fp32.
#include "tile_product.h"

namespace {

using tile::f32x4;

constexpr int kWave = 64;
constexpr int kTile = 256;          // rows and columns are padded to: whole tiles of either side

// What the device finds out: trained rows, and the factor of every gradient.
struct Plan {
    uint32_t rows;
    float factor;
};

struct Part {
    float top, sum;
};

template <typename T> constexpr float kHeld = 1.0f;             // factor in which D is held
template <> constexpr float kHeld<_Float16> = 8192.0f;

// Rows of the piece that starts at `first` and has room for `most`.
__device__ __forceinline__ uint32_t piece_rows(const Plan* plan, uint32_t first, uint32_t most)
{
    const uint32_t rows = plan->rows;
    return rows <= first ? 0 : rows - first < most ? rows - first : most;
}

__device__ __forceinline__ uint32_t round_up(uint32_t x, uint32_t to) { return (x + to - 1) / to * to; }

// ---------------------------------------------------------------------------
// which tiles, how many runs of k
// ---------------------------------------------------------------------------
// About how long a product of `tiles` tiles over `steps` steps of k takes in `splits`
// runs of k, in us.  The chip holds 256 tiles of 256 x 256 at a time, or 768 of
// 128 x 128, so they run in rounds; those of the larger ones end together.  A round
// costs its steps and a start and an end; the partial sums of a split product are
// written and read once more.  The constants are from products of 1000 to 3072
// rows, 20000 to 128256 columns and 768 to 4096 k: of 256, 0.86 us a step and 12 us
// a round; of 128, about 0.9 us (three on a compute unit) and 6.5 us.
__host__ __device__ __forceinline__ float product_us(int side, uint32_t tiles, uint32_t steps, uint32_t splits,
                                                     float partial_bytes)
{
    const float k = static_cast<float>(steps) / static_cast<float>(splits);
    const float all = static_cast<float>(tiles) * static_cast<float>(splits);
    const float join = static_cast<float>(splits) * partial_bytes * (2.0f / 4.0e6f);
    if (side == 256) return ceilf(all / 256.0f) * (0.86f * k + 12.0f) + join;
    return fmaxf(1.0f, all / 768.0f) * (0.9f * k + 6.5f) + join;
}

constexpr uint32_t kMostSplits = 64;

// ---------------------------------------------------------------------------
// the trained rows
// ---------------------------------------------------------------------------
// What the states' gradient needs decided once the rows are known: in how many runs
// of k each piece is taken, whose partial sums have `room` floats.
struct SplitArgs {
    uint32_t* splits;               // [pieces], null without gradients
    uint64_t room;
    uint32_t pieces, most, hidden, steps, side, max_splits;
};

// How many runs of k `rows` rows may take.
__host__ __device__ __forceinline__ uint32_t runs_in(uint64_t room, uint64_t rows, uint64_t hidden, uint32_t max_splits)
{
    const uint64_t fit = rows > 0 ? room / (rows * hidden) : max_splits;
    return fit < max_splits ? static_cast<uint32_t>(fit) : max_splits;
}

// One workgroup (the list is in order, and 8192 targets are one trip: 5 us) lists the rows whose target is not `ignore`, in order.
constexpr uint32_t kListed = 8;                                  // targets per thread and trip

__global__ __launch_bounds__(1024) void list_rows_kernel(const int64_t* targets, uint32_t n, int64_t ignore,
                                                         uint64_t vocab, int mean, const float* grad_scale, float held,
                                                         uint32_t* rows, int32_t* row_targets, Plan* plan,
                                                         SplitArgs split)
{
    __shared__ uint32_t counts[16];
    uint32_t done = 0;
    for (uint32_t base = 0; base < n; base += 1024 * kListed) {
        const uint32_t first = base + threadIdx.x * kListed;
        int64_t t[kListed];
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t k = 0; k < kListed; ++k) {
            t[k] = first + k < n ? targets[first + k] : ignore;
            mine += t[k] != ignore;
        }
        uint32_t upto = mine;                                    // over the wave, this lane's included
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const uint32_t y = __shfl_up(upto, d);
            if (threadIdx.x % kWave >= static_cast<uint32_t>(d)) upto += y;
        }
        __syncthreads();
        if (threadIdx.x % kWave == kWave - 1) counts[threadIdx.x / kWave] = upto;
        __syncthreads();
        uint32_t at = done + upto - mine;
        for (uint32_t w = 0; w < 16; ++w) {
            if (w < threadIdx.x / kWave) at += counts[w];
            done += counts[w];
        }
#pragma unroll
        for (uint32_t k = 0; k < kListed; ++k) {
            if (t[k] == ignore) continue;
            rows[at] = first + k;
            row_targets[at] = static_cast<uint64_t>(t[k]) < vocab ? static_cast<int32_t>(t[k]) : -1;
            ++at;
        }
    }
    if (threadIdx.x == 0) {
        plan->rows = done;
        plan->factor = (grad_scale ? *grad_scale : 1.0f) / (mean && done > 0 ? static_cast<float>(done) : 1.0f) / held;
    }
    if (!split.splits) return;
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (uint32_t p = wave; p < split.pieces; p += 16) {
        const uint32_t first = p * split.most;
        const uint32_t piece = done <= first ? 0 : done - first < split.most ? done - first : split.most;
        const uint32_t tiles = ceil_div(piece, split.side) * ceil_div(split.hidden, split.side);
        float least = lane < runs_in(split.room, piece, split.hidden, split.max_splits)
                          ? product_us(split.side, tiles, split.steps, lane + 1, 4.0f * piece * split.hidden)
                          : 3.0e38f;
        uint32_t best = lane + 1;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const float other = __shfl_xor(least, d);
            const uint32_t its = __shfl_xor(best, d);
            if (other < least || (other == least && its < best)) {
                least = other;
                best = its;
            }
        }
        if (lane == 0) split.splits[p] = best;
    }
}

// Bound by memory and small: 14 us for 4096 x 4096 beside products of milliseconds.
// Workgroup b < rows: row b of the gathered X, zeros after the last trained row and
// after the row's end; the others zero what an ignored row answers.
template <typename T>
__global__ __launch_bounds__(256) void gather_kernel(const T* x, uint64_t x_stride, uint32_t hidden, uint32_t padded,
                                                     const uint32_t* rows, const Plan* plan, T* gathered,
                                                     uint32_t gathered_rows, const int64_t* targets, int64_t ignore,
                                                     float* row_loss, T* grad_x, uint64_t grad_x_stride)
{
    if (blockIdx.x < gathered_rows) {
        const uint32_t row = blockIdx.x, count = plan->rows;
        if (row >= round_up(count, kTile)) return;
        T* to = gathered + static_cast<uint64_t>(row) * padded;
        for (uint32_t vec = threadIdx.x; vec * 8 < padded; vec += 256) {
            float v[8] = {};
            if (row < count) load_vec<T>(x + rows[row] * x_stride, vec, hidden, v);
            store_vec<T, 8>(to, vec, padded, v);
        }
        return;
    }
    const uint32_t row = blockIdx.x - gathered_rows;
    if (targets[row] != ignore) return;
    if (threadIdx.x == 0 && row_loss) row_loss[row] = 0.0f;
    if (!grad_x) return;
    const float zero[8] = {};
    for (uint32_t vec = threadIdx.x; vec * 8 < hidden; vec += 256)
        store_vec<T, 8>(grad_x + row * grad_x_stride, vec, hidden, zero);
}

// A vocabulary matrix whose rows are not whole, aligned stages of k: a padded copy.
// 32003 x 1023: 28 us, 4.7 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* weight, uint64_t stride, uint32_t hidden, uint32_t padded,
                                                  T* to)
{
    const uint64_t row = blockIdx.x;
    for (uint32_t vec = threadIdx.x; vec * 8 < padded; vec += 256) {
        float v[8];
        load_vec<T>(weight + row * stride, vec, hidden, v);
        store_vec<T, 8>(to + row * padded, vec, padded, v);
    }
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------
struct ScoreArgs {
    tile::Matrix weight, x;
    const Plan* plan;
    const int32_t* row_targets;
    Part* parts;                    // [rows of the piece][tiles of the vocabulary]
    float* target_scores;           // [rows of the piece]
    void* held;                     // [rows of the piece][columns], or null
    uint32_t first, most, vocab, columns, tiles, steps;
};

// What the waves that share a tile's rows tell each other: [largest, sum][wave][row of the tile].
template <int WAVES, int ROWS> struct Exchange {
    float at[2][WAVES][ROWS];
};

// Reduces a wave's INNER x OUTER fragments of scores (inner the vocabulary, from
// `inner_at` of vocabulary tile `inner`; outer rows, from `outer_at` of the tile that
// starts at row `first` of the piece): target scores and the tile's part of each row
// are written, and the sums become exp(s - m).  `part` of WAVES shares the rows.
template <int SIDE, int INNER, int OUTER, int WAVES, int ROWS>
__device__ __forceinline__ void reduce_scores(const ScoreArgs& a, uint32_t inner, uint32_t first, uint32_t rows,
                                              uint32_t part, uint32_t inner_at, uint32_t outer_at,
                                              f32x4 (&sums)[INNER][OUTER], Exchange<WAVES, ROWS>& exchange)
{
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t column = inner * SIDE + inner_at + lane / 16 * 4;
    if (inner * SIDE + SIDE > a.vocab)                           // columns past the vocabulary take no part
#pragma unroll
        for (int s = 0; s < INNER; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (column + s * 16 + r >= a.vocab)
#pragma unroll
                    for (int t = 0; t < OUTER; ++t) sums[s][t][r] = -INFINITY;
    float top[OUTER];
#pragma unroll
    for (int t = 0; t < OUTER; ++t) {
        const uint32_t row = outer_at + t * 16 + lane % 16;
        // the target's score, in the one lane that holds it
        const uint32_t target = (first + row < rows ? a.row_targets[a.first + first + row] : -1) - column;
        if (target < INNER * 16 && target % 16 < 4)
#pragma unroll
            for (int s = 0; s < INNER; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (target == s * 16u + r) a.target_scores[first + row] = sums[s][t][r];
        top[t] = -INFINITY;
#pragma unroll
        for (int s = 0; s < INNER; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) top[t] = fmaxf(top[t], sums[s][t][r]);
        top[t] = fmaxf(top[t], __shfl_xor(top[t], 16));
        top[t] = fmaxf(top[t], __shfl_xor(top[t], 32));
        if (lane < 16) exchange.at[0][part][row] = top[t];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < OUTER; ++t) {
        const uint32_t row = outer_at + t * 16 + lane % 16;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top[t] = fmaxf(top[t], exchange.at[0][w][row]);
        // exp(s - m) as a power of 2, one multiply-add before it; a row of -inf gives zeros
        constexpr float kLog2e = 1.44269504088896340736f;
        const float base = top[t] == -INFINITY ? 0.0f : top[t] * -kLog2e;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < INNER; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sums[s][t][r], kLog2e, base));
                sum += e;
                sums[s][t][r] = e;
            }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (lane < 16) exchange.at[1][part][row] = sum;
    }
    __syncthreads();
    if (part == 0 && lane < 16)
#pragma unroll
        for (int t = 0; t < OUTER; ++t) {
            const uint32_t row = outer_at + t * 16 + lane;
            float sum = exchange.at[1][0][row];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += exchange.at[1][w][row];
            a.parts[static_cast<uint64_t>(first + row) * a.tiles + inner] = Part{top[t], sum};
        }
}

// s = X W^T by tiles, reduced where they are: 3072 x 128256 x 4096 in 2.76 ms, 1.17 PFLOP/s
// with the softmax's part and 790 MB of exp(s - m) written; bound by the matrix
// cores at the clock that power leaves (1.9 GHz, 55 % of cycles busy) and a start
// and an end per tile, a sixth of it at k = 4096.
template <typename T, int SIDE>
__global__ __launch_bounds__(tile::kThreads, tile::Sizes<SIDE>::kResident) void scores_kernel(ScoreArgs a)
{
    __shared__ __attribute__((aligned(1024))) char lds[tile::Sizes<SIDE>::kLdsBytes];
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    const tile::Place at = tile::place(blockIdx.x, ceil_div(rows, SIDE), a.tiles);
    if (!at.valid) return;
    tile::Sums<SIDE> sums;
    tile::product<T, SIDE, true, true>(a.weight, at.inner * SIDE, a.x, a.first + at.outer * SIDE, 0, a.steps, lds, sums);

    // after what the tile is handed out through
    auto* exchange = reinterpret_cast<Exchange<2, SIDE>*>(lds + tile::Sizes<SIDE>::kHandOutBytes);
    reduce_scores<SIDE>(a, at.inner, at.outer * SIDE, rows, threadIdx.x / kWave % 2, tile::wave_inner<SIDE>(),
                        tile::wave_outer<SIDE>(), sums, *exchange);
    if (!a.held) return;
    T* held = static_cast<T*>(a.held) + static_cast<uint64_t>(at.outer) * SIDE * a.columns + at.inner * SIDE;
    tile::by_rows<SIDE>(sums, lds, [&](uint32_t outer, uint32_t inner, const float(&v)[8]) {
        float e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = v[k] * kHeld<T>;
        *reinterpret_cast<u32x4_t*>(held + static_cast<uint64_t>(outer) * a.columns + inner) = Elem<T>::pack(e);
    });
}

// The same for at most kFewRows rows: the time is that of reading the vocabulary
// matrix, which goes from memory to registers in the order that the matrix
// instructions take it, 16 * INNER of its rows a wave; the states come from the caches.
// Rows of any alignment and width are read where they lie.  13 rows of 128256 x
// 4096: 207 us (5.1 TB/s), the call 220; of 60001 x 1023, which
// tiles need a padded copy of, the call 71 us and 102.  From 17 rows on tiles are as
// fast or faster (40 rows of 128256 x 4096: 268 us, four fragments of rows here 343).
constexpr uint32_t kFewRows = 16;

template <typename T, int INNER> __global__ __launch_bounds__(256) void few_scores_kernel(ScoreArgs a)
{
    constexpr int SIDE = 64 * INNER;
    __shared__ Exchange<4, kFewRows> exchange;
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    if (rows == 0) return;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t width = a.weight.width, steps = a.steps;
    const T* weight[INNER];
#pragma unroll
    for (uint32_t s = 0; s < INNER; ++s) {
        const uint32_t row = blockIdx.x * SIDE + wave * (16 * INNER) + s * 16 + lane % 16;
        weight[s] = reinterpret_cast<const T*>(static_cast<const char*>(a.weight.data) +
                                               (row < a.vocab ? row : a.vocab - 1) * a.weight.stride);
    }
    const T* x = static_cast<const T*>(a.x.data) + (a.first + lane % 16) * (a.x.stride / 2);
    // workgroups begin at different k: rows a power of two apart would otherwise all
    // be read from the same few memory channels at a time (251 -> 223 us for one row of
    // 128256 x 4096)
    const uint32_t skew = blockIdx.x * 10 % (steps / 2) * 2;
    f32x4 sums[INNER][1] = {};
    u32x4_t w[2][2][INNER], v[2][2];                                 // [buffer][step of the pair]
    const auto load = [&](int b, uint32_t step) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = step + h + skew;
            const uint32_t vec = (at < steps ? at : at - steps) * 4 + lane / 16;
#pragma unroll
            for (int s = 0; s < INNER; ++s) w[b][h][s] = load_raw<T>(weight[s], vec, width);
            v[b][h] = *reinterpret_cast<const u32x4_t*>(x + vec * 8);
        }
    };
    const auto multiply = [&](int b) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < INNER; ++s)
                sums[s][0] = tile::product_of<T>(__builtin_bit_cast(tile::s16x8, w[b][h][s]),
                                                 __builtin_bit_cast(tile::s16x8, v[b][h]), sums[s][0]);
    };
    load(0, 0);
    for (uint32_t step = 0; step < steps; step += 4) {              // steps come in pairs
        if (step + 2 < steps) load(1, step + 2);
        multiply(0);
        if (step + 4 < steps) load(0, step + 4);
        if (step + 2 < steps) multiply(1);
    }
    reduce_scores<SIDE>(a, blockIdx.x, 0, rows, wave, wave * (16 * INNER), 0, sums, exchange);
    if (!a.held) return;
    // the rows after these are written as zeros with D
    T* held = static_cast<T*>(a.held) + static_cast<uint64_t>(lane % 16) * a.columns + blockIdx.x * SIDE +
              wave * (16 * INNER) + lane / 16 * 4;
#pragma unroll
    for (int s = 0; s < INNER; ++s) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        v4 e;
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = static_cast<T>(sums[s][0][r] * kHeld<T>);
        *reinterpret_cast<v4*>(held + s * 16) = e;
    }
}

// ---------------------------------------------------------------------------
// the rows' losses
// ---------------------------------------------------------------------------
// lse of a row from its parts, by the THREADS threads that call it together.
template <int THREADS> __device__ __forceinline__ float row_lse(const Part* parts, uint32_t tiles, float* lds)
{
    const uint32_t thread = threadIdx.x % THREADS, wave = threadIdx.x / kWave;
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t k = thread; k < tiles; k += THREADS) top = fmaxf(top, parts[k].top);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if constexpr (THREADS > kWave) {
        if (threadIdx.x % kWave == 0) lds[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) top = fmaxf(top, lds[w]);
    }
    const float base = top == -INFINITY ? 0.0f : top;
    for (uint32_t k = thread; k < tiles; k += THREADS) sum += parts[k].sum * expf(parts[k].top - base);
    sum = wave_sum(sum);
    if constexpr (THREADS > kWave) {
        if (threadIdx.x % kWave == 0) lds[THREADS / kWave + wave] = sum;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) sum += lds[THREADS / kWave + w];
    }
    return base + logf(sum);
}

__global__ __launch_bounds__(256) void row_loss_kernel(const Part* parts, uint32_t tiles, const Plan* plan,
                                                       uint32_t first, uint32_t most, const uint32_t* rows,
                                                       const int32_t* row_targets, const float* target_scores,
                                                       float* row_loss)
{
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= piece_rows(plan, first, most)) return;
    const float lse = row_lse<kWave>(parts + static_cast<uint64_t>(row) * tiles, tiles, nullptr);
    if (threadIdx.x % kWave == 0)
        row_loss[rows[first + row]] =
            row_targets[first + row] >= 0 ? lse - target_scores[row] : __builtin_nanf("");
}

// The sum of the rows' losses, in 64 bits and a fixed order, by one workgroup.
template <uint32_t THREADS>
__device__ void write_loss(const float* row_loss, const uint32_t* rows, const Plan* plan, int mean, float* loss)
{
    __shared__ double lds[THREADS / kWave];
    const uint32_t count = plan->rows;
    double sum = 0.0;
#pragma unroll 4
    for (uint32_t k = threadIdx.x; k < count; k += THREADS) sum += static_cast<double>(row_loss[rows[k]]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (uint32_t w = 1; w < THREADS / kWave; ++w) sum += lds[w];
    *loss = static_cast<float>(mean && count > 0 ? sum / count : sum);
}

__global__ __launch_bounds__(1024) void loss_kernel(const float* row_loss, const uint32_t* rows, const Plan* plan,
                                                    int mean, float* loss)
{
    write_loss<1024>(row_loss, rows, plan, mean, loss);
}

// ---------------------------------------------------------------------------
// D, in place of exp(s - m)
// ---------------------------------------------------------------------------
// Each workgroup joins its row's parts itself, a few KB out of the caches, rather
// than wait for a launch that does it once.  3072 x 128256: 305 us, 5.2 TB/s, bound by
// memory.
constexpr uint32_t kPerGroup = 4;                                // 16-byte vectors per thread

template <typename T>
__global__ __launch_bounds__(256) void softmax_grad_kernel(ScoreArgs a, const uint32_t* rows, float* row_loss)
{
    __shared__ float lds[8];
    const uint32_t row = blockIdx.y, count = piece_rows(a.plan, a.first, a.most);
    // rows past the last are zeros to the end of its pair of steps, as the matrix's gradient sums over rows; what
    // lies beyond only reaches rows of the states' gradient that are not written
    if (row >= round_up(count, 2 * tile::kDepth)) return;
    const uint32_t side = a.columns / a.tiles;
    const Part* parts = a.parts + static_cast<uint64_t>(row) * a.tiles;
    T* mine = static_cast<T*>(a.held) + static_cast<uint64_t>(row) * a.columns;
    int32_t target = -1;
    float lse = 0.0f;
    if (row < count) {
        target = a.row_targets[a.first + row];
        // a target that is none makes the row NaN
        lse = target >= 0 ? row_lse<256>(parts, a.tiles, lds) : __builtin_nanf("");
        if (blockIdx.x == 0 && threadIdx.x == 0)
            row_loss[rows[a.first + row]] = target >= 0 ? lse - a.target_scores[row] : lse;
    }
#pragma unroll
    for (uint32_t k = 0; k < kPerGroup; ++k) {
        const uint32_t vec = (blockIdx.x * kPerGroup + k) * 256 + threadIdx.x;
        if (vec * 8 >= a.columns) return;
        float d[8] = {};
        if (row < count) {
            load_vec<T>(mine, vec, a.columns, d);
            const float f = expf(parts[vec * 8 / side].top - lse);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                d[e] = d[e] * f - (static_cast<int32_t>(vec * 8 + e) == target ? kHeld<T> : 0.0f);
        }
        store_vec<T, 8>(mine, vec, a.columns, d);
    }
}

// ---------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------
struct GradXArgs {
    tile::Matrix weight, held;
    const Plan* plan;
    const uint32_t* rows;
    float* partial;                 // [splits][trained rows of the piece][hidden]
    const uint32_t* splits;         // runs of k of this piece
    uint32_t first, most, hidden, inners, pairs;               // pairs of steps
};

// D W, W by columns.  3072 x 4096 over k = 128256 in four runs: 2.50 ms, 1.29 PFLOP/s,
// the matrix cores busy 63 % of cycles at 1.9 GHz.
template <typename T, int SIDE>
__global__ __launch_bounds__(tile::kThreads, tile::Sizes<SIDE>::kResident) void grad_x_kernel(GradXArgs a)
{
    __shared__ __attribute__((aligned(1024))) char lds[tile::Sizes<SIDE>::kLdsBytes];
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    const uint32_t outers = ceil_div(rows, SIDE);
    if (outers == 0) return;
    const uint32_t splits = *a.splits;
    const tile::Place at = tile::place(blockIdx.x, outers * splits, a.inners);
    if (!at.valid) return;
    const uint32_t split = at.outer / outers, outer = at.outer % outers;
    const uint32_t from = static_cast<uint64_t>(a.pairs) * split / splits * 2;
    const uint32_t to = static_cast<uint64_t>(a.pairs) * (split + 1) / splits * 2;
    tile::Sums<SIDE> sums;
    tile::product<T, SIDE, false, true>(a.weight, at.inner * SIDE, a.held, outer * SIDE,
                                        static_cast<uint64_t>(from) * tile::kDepth, to - from, lds, sums);
    float* partial = a.partial + (static_cast<uint64_t>(split) * rows + outer * SIDE) * a.hidden;
    tile::by_rows<SIDE>(sums, lds, [&](uint32_t row, uint32_t inner, const float(&v)[8]) {
        if (outer * SIDE + row < rows)
            store_vec<float, 8>(partial + static_cast<uint64_t>(row) * a.hidden, (at.inner * SIDE + inner) / 8,
                                a.hidden, v);
    });
}

// The last workgroup, after the piece's rows, writes the loss where it is known.
template <typename T>
__global__ __launch_bounds__(256) void join_grad_x_kernel(GradXArgs a, T* grad_x, uint64_t grad_x_stride,
                                                          const float* row_loss, int mean, float* loss)
{
    if (blockIdx.x == a.most) {
        write_loss<256>(row_loss, a.rows, a.plan, mean, loss);
        return;
    }
    const uint32_t row = blockIdx.x, rows = piece_rows(a.plan, a.first, a.most);
    if (row >= rows) return;
    const uint32_t splits = *a.splits;
    const float factor = a.plan->factor;
    T* out = grad_x + a.rows[a.first + row] * grad_x_stride;
    for (uint32_t vec = threadIdx.x; vec * 8 < a.hidden; vec += 256) {
        float sum[8] = {};
#pragma unroll 4
        for (uint32_t k = 0; k < splits; ++k) {
            const float* partial = a.partial + (static_cast<uint64_t>(k) * rows + row) * a.hidden;
            float lo[4], hi[4];
            load_vec<float>(partial, vec * 2, a.hidden, lo);
            load_vec<float>(partial, vec * 2 + 1, a.hidden, hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[e] += lo[e];
                sum[4 + e] += hi[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] *= factor;
        store_vec<T, 8>(out, vec, a.hidden, sum);
    }
}

struct GradWeightArgs {
    tile::Matrix x, held;
    const Plan* plan;
    void* grad_weight;
    float* total;                   // [vocab][hidden] where the rows take more than one piece and
                                    // grad_weight cannot hold their sum, being of 16 bits; else null
    uint64_t stride;
    uint32_t first, most, vocab, hidden, inners, outers;
    int accumulate;
};

// D^T X, both by columns.  128256 x 4096 over 3072 rows: 2.85 ms, 1.13 PFLOP/s; k is
// 96 steps, so starts and ends of tiles take an eighth, and 1 GB is written.
template <typename T, typename W, int SIDE>
__global__ __launch_bounds__(tile::kThreads, tile::Sizes<SIDE>::kResident) void grad_weight_kernel(GradWeightArgs a)
{
    __shared__ __attribute__((aligned(1024))) char lds[tile::Sizes<SIDE>::kLdsBytes];
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    if (rows == 0 && a.first > 0) return;
    const tile::Place at = tile::place(blockIdx.x, a.outers, a.inners);
    if (!at.valid) return;
    tile::Sums<SIDE> sums;
    tile::product<T, SIDE, false, false>(a.x, at.inner * SIDE, a.held, at.outer * SIDE, 0,
                                         ceil_div(rows, 2 * tile::kDepth) * 2, lds, sums);
    constexpr bool kHoldsSum = __is_same(W, float);                  // over the pieces, without a buffer beside it
    const bool last = a.first + rows >= a.plan->rows;
    const float factor = a.plan->factor;
    tile::by_rows<SIDE>(sums, lds, [&](uint32_t outer, uint32_t inner, const float(&sum)[8]) {
        const uint32_t row = at.outer * SIDE + outer, vec = (at.inner * SIDE + inner) / 8;
        if (row >= a.vocab) return;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = sum[k];
        if constexpr (!kHoldsSum) {
            float* total = a.total + static_cast<uint64_t>(row) * a.hidden;
            if (a.first > 0)
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k)
                    if (vec * 8 + k < a.hidden) v[k] += total[vec * 8 + k];
            if (!last) {
                store_vec<float, 8>(total, vec, a.hidden, v);
                return;
            }
        }
        W* out = static_cast<W*>(a.grad_weight) + row * a.stride;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= factor;
        if (a.accumulate || (kHoldsSum && a.first > 0))
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (vec * 8 + k < a.hidden) v[k] += Elem<W>::to_f32(out[vec * 8 + k]);
        store_vec<W, 8>(out, vec, a.hidden, v);
    });
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint64_t kMaxRows = 1ull << 22;
constexpr uint64_t kMaxHidden = 1ull << 16;
constexpr uint64_t kMaxVocab = 1ull << 21;          // a tile's rows stay within 32-bit offsets
constexpr uint64_t kForwardRows = 16384;            // rows of a piece without gradients: only `parts` grows with it
constexpr uint64_t kMostRows = 32768;               // and of any piece: a launch's second dimension has 16 bits

constexpr uint64_t kPair = 2 * tile::kDepth;        // k is padded to: a product takes an even number of steps

bool sizes_ok(const la_linear_loss_t& c)
{
    return c.n <= kMaxRows && c.hidden > 0 && c.hidden <= kMaxHidden && c.vocab > 0 && c.vocab <= kMaxVocab &&
           c.weight_stride <= kMaxVocab && c.piece_rows <= kMaxRows;
}

// Whether the products can read the matrix where it lies.
bool reads_in_place(const la_linear_loss_t& c)
{
    return c.hidden % kPair == 0 && c.weight_stride % 8 == 0 && reinterpret_cast<uintptr_t>(c.weight) % 16 == 0;
}

bool copies_weight(const la_linear_loss_t& c) { return !reads_in_place(c) && (c.grads || c.n > kFewRows); }

// The least time of a product of rows x columns in tiles of this side, over the ways to split it.
float least_us(int side, uint64_t rows, uint64_t columns, uint64_t k, uint64_t max_splits)
{
    const uint64_t tiles = ceil_div(rows, side) * ceil_div(columns, side), steps = ceil_div(k, kPair) * 2;
    float least = product_us(side, tiles, steps, 1, max_splits > 1 ? 4.0f * rows * columns : 0.0f);
    for (uint32_t s = 2; s <= max_splits; ++s) {
        const float us = product_us(side, tiles, steps, s, 4.0f * rows * columns);
        if (us < least) least = us;
    }
    return least;
}

int side_of(uint64_t rows, uint64_t columns, uint64_t k, uint64_t max_splits)
{
    return least_us(128, rows, columns, k, max_splits) < least_us(256, rows, columns, k, max_splits) ? 128 : 256;
}

// Sizes and the workspace's parts (offsets in bytes).
struct Layout {
    int score_side, grad_x_side, grad_w_side;
    uint64_t padded, columns, all, piece, pieces, max_splits, room;
    uint64_t plan, splits, rows, row_targets, gathered, weight, parts, target_scores, row_loss, held, partial, total, size;

    Layout(const la_linear_loss_t& c, uint64_t piece_rows)
    {
        padded = ceil_div(c.hidden, kPair) * kPair;
        columns = ceil_div(c.vocab, kTile) * kTile;
        all = c.n > 0 ? ceil_div(c.n, kTile) * kTile : kTile;     // no rows: one empty piece, which clears grad_weight
        piece = ceil_div(piece_rows, kTile) * kTile;
        if (piece == 0 || piece > all) piece = all;
        if (piece > kMostRows) piece = kMostRows;
        pieces = ceil_div(all, piece);
        // As many runs of k as would take the memory of a piece's D, or the 64 MiB of one round of large tiles, if
        // all its rows were trained.  Their partial sums have half of that, of one run at the least: the full
        // rows' tiles fill the chip in few runs, and fewer rows have room for more.
        const uint64_t one = piece * c.hidden, most = piece * columns / 2;
        max_splits = (most > (16u << 20) ? most : 16u << 20) / one;
        if (max_splits > columns / kTile) max_splits = columns / kTile;
        if (max_splits > kMostSplits) max_splits = kMostSplits;
        if (max_splits == 0) max_splits = 1;
        room = most / 2 > (16u << 20) ? most / 2 : 16u << 20;
        if (room > max_splits * one) room = max_splits * one;
        if (room < one) room = one;
        const uint64_t rows_of_piece = c.n < piece ? c.n : piece;
        // few rows: workgroups of 256 of the matrix's rows where they fill the chip, else of 128
        score_side = c.n <= kFewRows ? (columns / kTile >= 256 ? 256 : 128) : side_of(rows_of_piece, c.vocab, c.hidden, 1);
        grad_x_side = side_of(rows_of_piece, c.hidden, c.vocab, runs_in(room, rows_of_piece, c.hidden, max_splits));
        grad_w_side = side_of(c.vocab, c.hidden, rows_of_piece, 1);
        uint64_t at = 0;
        const auto take = [&](uint64_t bytes) {
            const uint64_t here = at;
            at += ceil_div(bytes, 256) * 256;
            return here;
        };
        plan = take(sizeof(Plan));
        splits = take(pieces * 4);
        rows = take(c.n * 4);
        row_targets = take(c.n * 4);
        gathered = take(all * padded * 2);
        weight = !copies_weight(c) ? 0 : take(c.vocab * padded * 2);
        parts = take(piece * (columns / score_side) * sizeof(Part));
        target_scores = take(piece * 4);
        row_loss = c.row_loss ? 0 : take(c.n * 4);
        held = c.grads ? take(piece * columns * 2) : 0;
        partial = c.grads ? take(room * 4) : 0;
        total = c.grads && pieces > 1 && c.grad_weight_dtype != LA_F32 ? take(c.vocab * c.hidden * 4) : 0;
        size = at;
    }
};

// The sum over pieces, where grad_weight cannot hold it, can take more than the pieces
// save: all rows are one piece where that takes no more memory.
Layout layout_of(const la_linear_loss_t& c)
{
    const Layout asked(c, c.grads ? c.piece_rows : kForwardRows);
    if (asked.total == 0 || asked.all > kMostRows) return asked;
    const Layout whole(c, asked.all);
    return whole.size <= asked.size ? whole : asked;
}

template <typename T> int run_scores(const la_linear_loss_t& c, const Layout& l, const ScoreArgs& a, hipStream_t st)
{
    if (c.n <= kFewRows)
        return l.score_side == 256 ? launch(few_scores_kernel<T, 4>, dim3(a.tiles), dim3(256), st, a)
                                   : launch(few_scores_kernel<T, 2>, dim3(a.tiles), dim3(256), st, a);
    const dim3 grid(tile::places(l.piece / l.score_side, a.tiles)), block(tile::kThreads);
    return l.score_side == 128 ? launch(scores_kernel<T, 128>, grid, block, st, a)
                               : launch(scores_kernel<T, 256>, grid, block, st, a);
}

template <typename T, int SIDE>
int run_grad_x(const la_linear_loss_t& c, const Layout& l, GradXArgs a, const float* row_loss, hipStream_t st)
{
    a.inners = ceil_div(a.hidden, SIDE);
    // rows in whole tiles times runs: rows times runs are bounded by the partial sums' room, each run's last tile is partial
    uint64_t outers = l.room / (a.hidden * static_cast<uint64_t>(SIDE)) + l.max_splits;
    if (outers > l.piece / SIDE * l.max_splits) outers = l.piece / SIDE * l.max_splits;
    const int rc =
        launch(grad_x_kernel<T, SIDE>, dim3(tile::places(outers, a.inners)), dim3(tile::kThreads), st, a);
    if (rc != LA_OK) return rc;
    const bool last = a.first + l.piece >= l.all;
    return launch(join_grad_x_kernel<T>, dim3(l.piece + (last && c.loss ? 1 : 0)), dim3(256), st, a,
                  static_cast<T*>(c.grad_x), c.grad_x_stride, row_loss, c.mean, c.loss);
}

template <typename T, typename W, int SIDE> int run_grad_weight(GradWeightArgs a, hipStream_t st)
{
    a.inners = ceil_div(a.hidden, SIDE);
    a.outers = ceil_div(a.vocab, SIDE);
    return launch(grad_weight_kernel<T, W, SIDE>, dim3(tile::places(a.outers, a.inners)), dim3(tile::kThreads), st, a);
}

template <typename T, typename W> int run(const la_linear_loss_t& c, char* ws, hipStream_t st)
{
    const Layout l = layout_of(c);
    Plan* plan = reinterpret_cast<Plan*>(ws + l.plan);
    uint32_t* splits = reinterpret_cast<uint32_t*>(ws + l.splits);
    uint32_t* rows = reinterpret_cast<uint32_t*>(ws + l.rows);
    int32_t* row_targets = reinterpret_cast<int32_t*>(ws + l.row_targets);
    T* gathered = reinterpret_cast<T*>(ws + l.gathered);
    Part* parts = reinterpret_cast<Part*>(ws + l.parts);
    float* target_scores = reinterpret_cast<float*>(ws + l.target_scores);
    float* row_loss = c.row_loss ? c.row_loss : reinterpret_cast<float*>(ws + l.row_loss);
    T* held = c.grads ? reinterpret_cast<T*>(ws + l.held) : nullptr;
    T* grad_x = c.grads ? static_cast<T*>(c.grad_x) : nullptr;

    int rc = launch(list_rows_kernel, dim3(1), dim3(1024), st, c.targets, c.n, c.ignore_index, c.vocab, c.mean,
                    c.grad_scale, kHeld<T>, rows, row_targets, plan,
                    SplitArgs{c.grads ? splits : nullptr, l.room, static_cast<uint32_t>(l.pieces),
                              static_cast<uint32_t>(l.piece), static_cast<uint32_t>(c.hidden),
                              static_cast<uint32_t>(l.columns / tile::kDepth), static_cast<uint32_t>(l.grad_x_side),
                              static_cast<uint32_t>(l.max_splits)});
    if (rc != LA_OK) return rc;
    rc = launch(gather_kernel<T>, dim3(l.all + c.n), dim3(256), st, static_cast<const T*>(c.x), c.x_stride, c.hidden,
                l.padded, rows, plan, gathered, l.all, c.targets, c.ignore_index, row_loss, grad_x, c.grad_x_stride);
    if (rc != LA_OK) return rc;
    tile::Matrix weight{c.weight, c.vocab, c.hidden, c.weight_stride * 2};
    if (copies_weight(c)) {
        T* copy = reinterpret_cast<T*>(ws + l.weight);
        rc = launch(pad_kernel<T>, dim3(c.vocab), dim3(256), st, static_cast<const T*>(c.weight), c.weight_stride,
                    c.hidden, l.padded, copy);
        if (rc != LA_OK) return rc;
        weight = tile::Matrix{copy, c.vocab, l.padded, l.padded * 2};
    }
    const tile::Matrix x{gathered, l.all, l.padded, l.padded * 2};
    const tile::Matrix d{held, l.piece, l.columns, l.columns * 2};
    const uint32_t vocab = c.vocab, hidden = c.hidden, columns = l.columns, tiles = l.columns / l.score_side;

    for (uint64_t p = 0; p < l.pieces; ++p) {
        const uint32_t first = p * l.piece, most = l.piece;
        const ScoreArgs scores{weight, x, plan, row_targets, parts, target_scores, held, first, most, vocab, columns,
                               tiles, static_cast<uint32_t>(l.padded / tile::kDepth)};
        rc = run_scores<T>(c, l, scores, st);
        if (rc != LA_OK) return rc;
        if (!c.grads) {
            rc = launch(row_loss_kernel, dim3(most / 4), dim3(256), st, parts, tiles, plan, first, most, rows,
                        row_targets, target_scores, row_loss);
            if (rc != LA_OK) return rc;
            continue;
        }
        rc = launch(softmax_grad_kernel<T>, dim3(ceil_div(columns, 8 * 256 * kPerGroup), most), dim3(256), st, scores,
                    rows, row_loss);
        if (rc != LA_OK) return rc;
        const GradXArgs gx{weight, d, plan, rows, reinterpret_cast<float*>(ws + l.partial), splits + p, first, most,
                           hidden, 0, static_cast<uint32_t>(columns / kPair)};
        rc = l.grad_x_side == 128 ? run_grad_x<T, 128>(c, l, gx, row_loss, st)
                                  : run_grad_x<T, 256>(c, l, gx, row_loss, st);
        if (rc != LA_OK) return rc;
        const tile::Matrix piece_x{gathered + first * l.padded, l.piece < l.all - first ? l.piece : l.all - first,
                                   l.padded, l.padded * 2};
        const GradWeightArgs gw{piece_x, d, plan, c.grad_weight,
                                l.total ? reinterpret_cast<float*>(ws + l.total) : nullptr, c.grad_weight_stride,
                                first, most, vocab, hidden, 0, 0, c.accumulate};
        rc = l.grad_w_side == 128 ? run_grad_weight<T, W, 128>(gw, st) : run_grad_weight<T, W, 256>(gw, st);
        if (rc != LA_OK) return rc;
    }
    if (!c.loss || c.grads) return LA_OK;
    return launch(loss_kernel, dim3(1), dim3(1024), st, row_loss, rows, plan, c.mean, c.loss);
}

bool reachable(const void* p) { return !p || la_ptr::device_accessible(p); }

}  // namespace

extern "C" {

uint64_t la_linear_loss_workspace(const la_linear_loss_t* call)
{
    return call && sizes_ok(*call) ? layout_of(*call).size : 0;
}

int la_linear_loss(const la_linear_loss_t* call, void* workspace, uint64_t workspace_bytes, la_stream_t stream)
{
    if (!call) return LA_EINVAL;
    const la_linear_loss_t& c = *call;
    if (c.dtype != LA_BF16 && c.dtype != LA_F16) return LA_EDTYPE;
    if (c.grads && c.grad_weight_dtype != c.dtype && c.grad_weight_dtype != LA_F32) return LA_EDTYPE;
    if (!sizes_ok(c)) return LA_EINVAL;
    int rc = check_matrix(c.weight, c.dtype, c.hidden, c.weight_stride);
    if (rc == LA_OK && c.n > 0) rc = check_matrix(c.x, c.dtype, c.hidden, c.x_stride);
    if (rc == LA_OK && c.n > 0) rc = check_matrix(c.targets, LA_I64, 1, 1);
    if (rc == LA_OK && c.loss) rc = check_matrix(c.loss, LA_F32, 1, 1);
    if (rc == LA_OK && c.row_loss) rc = check_matrix(c.row_loss, LA_F32, 1, 1);
    if (rc == LA_OK && c.grads) {
        if (c.n > 0) rc = check_matrix(c.grad_x, c.dtype, c.hidden, c.grad_x_stride);
        if (rc == LA_OK) rc = check_matrix(c.grad_weight, c.grad_weight_dtype, c.hidden, c.grad_weight_stride);
        if (rc == LA_OK && c.grad_scale) rc = check_matrix(c.grad_scale, LA_F32, 1, 1);
    }
    if (rc == LA_OK) rc = check_workspace(workspace, workspace_bytes, layout_of(c).size, 256);
    if (rc != LA_OK) return rc;
    if (!reachable(workspace) || !reachable(c.weight) || (c.n > 0 && (!reachable(c.x) || !reachable(c.targets))) ||
        !reachable(c.loss) || !reachable(c.row_loss) ||
        (c.grads && ((c.n > 0 && !reachable(c.grad_x)) || !reachable(c.grad_weight) || !reachable(c.grad_scale))))
        return LA_EFAULT;
    char* ws = static_cast<char*>(workspace);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool wide = c.grads && c.grad_weight_dtype == LA_F32;
    if (c.dtype == LA_BF16) return wide ? run<__bf16, float>(c, ws, st) : run<__bf16, __bf16>(c, ws, st);
    return wide ? run<_Float16, float>(c, ws, st) : run<_Float16, _Float16>(c, ws, st);
}

}  // extern "C"
