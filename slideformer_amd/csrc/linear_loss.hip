// slideformer_amd: softmax cross entropy of hidden states against a vocabulary
// matrix, with its gradients, without the scores ever being held (gfx950, wave64).
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
using tile::kTile;

constexpr int kWave = 64;

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
// the trained rows
// ---------------------------------------------------------------------------
// One workgroup lists the rows whose target is not `ignore`, in order.
constexpr uint32_t kListed = 8;                                  // targets per thread and trip

__global__ __launch_bounds__(1024) void list_rows_kernel(const int64_t* targets, uint32_t n, int64_t ignore,
                                                         uint64_t vocab, int mean, const float* grad_scale, float held,
                                                         uint32_t* rows, int32_t* row_targets, Plan* plan)
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
}

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
    void* held;                     // [rows of the piece][tiles * 256], or null
    uint32_t first, most, vocab, tiles, steps;
};

template <typename T> __global__ __launch_bounds__(tile::kThreads, 1) void scores_kernel(ScoreArgs a)
{
    __shared__ __attribute__((aligned(1024))) char lds[tile::kLdsBytes];
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    const tile::Place at = tile::place(blockIdx.x, ceil_div(rows, kTile), a.tiles);
    if (!at.valid) return;
    tile::Sums sums;
    tile::product<T, true, true>(a.weight, at.inner * kTile, a.x, a.first + at.outer * kTile, 0, a.steps,
                                 lds, sums);

    // [largest, sum][inner half][row of the tile], after what the tile is handed out through
    float(*exchange)[2][kTile] = reinterpret_cast<float(*)[2][kTile]>(lds + tile::kHandOutBytes);
    const uint32_t lane = threadIdx.x % kWave, half = threadIdx.x / kWave % 2;
    const uint32_t column = at.inner * kTile + tile::wave_inner() + lane / 16 * 4;
    if (at.inner * kTile + kTile > a.vocab)                      // columns past the vocabulary take no part
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (column + s * 16 + r >= a.vocab)
#pragma unroll
                    for (int t = 0; t < 8; ++t) sums[s][t][r] = -INFINITY;
    float top[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const uint32_t row = tile::wave_outer() + t * 16 + lane % 16;
        const uint32_t in_piece = at.outer * kTile + row;
        // the target's score, in the one lane that holds it
        const uint32_t target = (in_piece < rows ? a.row_targets[a.first + in_piece] : -1) - column;
        if (target < 128 && target % 16 < 4)
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (target == s * 16u + r) a.target_scores[in_piece] = sums[s][t][r];
        top[t] = -INFINITY;
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) top[t] = fmaxf(top[t], sums[s][t][r]);
        top[t] = fmaxf(top[t], __shfl_xor(top[t], 16));
        top[t] = fmaxf(top[t], __shfl_xor(top[t], 32));
        if (lane < 16) exchange[0][half][row] = top[t];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const uint32_t row = tile::wave_outer() + t * 16 + lane % 16;
        top[t] = fmaxf(exchange[0][0][row], exchange[0][1][row]);
        // exp(s - m) as a power of 2, one multiply-add before it; a row of -inf gives zeros
        constexpr float kLog2e = 1.44269504088896340736f;
        const float base = top[t] == -INFINITY ? 0.0f : top[t] * -kLog2e;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sums[s][t][r], kLog2e, base));
                sum += e;
                sums[s][t][r] = e;
            }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (lane < 16) exchange[1][half][row] = sum;
    }
    __syncthreads();
    if (half == 0 && lane < 16)
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const uint32_t row = tile::wave_outer() + t * 16 + lane;
            a.parts[static_cast<uint64_t>(at.outer * kTile + row) * a.tiles + at.inner] =
                Part{top[t], exchange[1][0][row] + exchange[1][1][row]};
        }
    if (!a.held) return;
    T* held = static_cast<T*>(a.held) + static_cast<uint64_t>(at.outer) * kTile * a.tiles * kTile + at.inner * kTile;
    tile::by_rows(sums, lds, [&](uint32_t outer, uint32_t inner, const float(&v)[8]) {
        float e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = v[k] * kHeld<T>;
        *reinterpret_cast<u32x4_t*>(held + static_cast<uint64_t>(outer) * a.tiles * kTile + inner) =
            Elem<T>::pack(e);
    });
}

// ---------------------------------------------------------------------------
// the rows' losses
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void row_loss_kernel(const Part* parts, uint32_t tiles, const Plan* plan,
                                                       uint32_t first, uint32_t most, const uint32_t* rows,
                                                       const int32_t* row_targets, const float* target_scores,
                                                       float* lse, float* row_loss)
{
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / kWave, lane = threadIdx.x % kWave;
    if (row >= piece_rows(plan, first, most)) return;
    const Part* mine = parts + static_cast<uint64_t>(row) * tiles;
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t k = lane; k < tiles; k += kWave) top = fmaxf(top, mine[k].top);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float base = top == -INFINITY ? 0.0f : top;
    for (uint32_t k = lane; k < tiles; k += kWave) sum += mine[k].sum * expf(mine[k].top - base);
    sum = wave_sum(sum);
    if (lane != 0) return;
    const float total = base + logf(sum);
    const bool known = row_targets[first + row] >= 0;
    lse[row] = known ? total : __builtin_nanf("");
    row_loss[rows[first + row]] = known ? total - target_scores[row] : __builtin_nanf("");
}

__global__ __launch_bounds__(1024) void loss_kernel(const float* row_loss, const uint32_t* rows, const Plan* plan,
                                                    int mean, float* loss)
{
    __shared__ double lds[16];
    double sum = 0.0;
    for (uint32_t k = threadIdx.x; k < plan->rows; k += 1024) sum += static_cast<double>(row_loss[rows[k]]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) sum += lds[w];
    *loss = static_cast<float>(mean && plan->rows > 0 ? sum / plan->rows : sum);
}

// ---------------------------------------------------------------------------
// D, in place of exp(s - m)
// ---------------------------------------------------------------------------
constexpr uint32_t kPerGroup = 4;                                // 16-byte vectors per thread

template <typename T>
__global__ __launch_bounds__(256) void softmax_grad_kernel(T* held, const Part* parts, const float* lse,
                                                           const int32_t* row_targets, const Plan* plan,
                                                           uint32_t first, uint32_t most, uint32_t tiles)
{
    const uint32_t row = blockIdx.y, rows = piece_rows(plan, first, most);
    if (row >= round_up(rows, kTile)) return;
    const uint32_t width = tiles * kTile;
    T* mine = held + static_cast<uint64_t>(row) * width;
    const int32_t target = row < rows ? row_targets[first + row] : -1;
    const float total = row < rows ? lse[row] : 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kPerGroup; ++k) {
        const uint32_t vec = (blockIdx.x * kPerGroup + k) * 256 + threadIdx.x;
        if (vec * 8 >= width) return;
        float d[8] = {};
        if (row < rows) {
            load_vec<T>(mine, vec, width, d);
            const float top = parts[static_cast<uint64_t>(row) * tiles + vec / (kTile / 8)].top;
            const float f = expf(top - total);
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                d[e] = d[e] * f - (static_cast<int32_t>(vec * 8 + e) == target ? kHeld<T> : 0.0f);
        }
        store_vec<T, 8>(mine, vec, width, d);
    }
}

// ---------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------
struct GradXArgs {
    tile::Matrix weight, held;
    const Plan* plan;
    const uint32_t* rows;
    float* partial;                 // [splits][rows of the piece][hidden]
    uint32_t first, most, hidden, inners, pairs, max_splits;   // pairs of steps
};

// Into how many runs of k a product of `tiles` tiles is split.  A compute unit
// holds one workgroup, so the tiles run in rounds of 256 and the last round may be
// nearly empty; with more, shorter runs it is fuller.  Each run costs a pass over
// its partial sums, counted here as a fiftieth of a round.
__device__ __forceinline__ uint32_t splits_of(uint32_t tiles, uint32_t max_splits)
{
    uint32_t best = 1;
    float least = 3.0e38f;
    for (uint32_t s = 1; s <= max_splits; ++s) {
        const float cost = static_cast<float>((tiles * s + 255) / 256) / static_cast<float>(s) +
                           0.02f * static_cast<float>(s);
        if (cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}

template <typename T> __global__ __launch_bounds__(tile::kThreads, 1) void grad_x_kernel(GradXArgs a)
{
    __shared__ __attribute__((aligned(1024))) char lds[tile::kLdsBytes];
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    const uint32_t outers = ceil_div(rows, kTile);
    if (outers == 0) return;
    const uint32_t splits = splits_of(outers * a.inners, a.max_splits);
    const tile::Place at = tile::place(blockIdx.x, outers * splits, a.inners);
    if (!at.valid) return;
    const uint32_t split = at.outer / outers, outer = at.outer % outers;
    const uint32_t from = static_cast<uint64_t>(a.pairs) * split / splits * 2;
    const uint32_t to = static_cast<uint64_t>(a.pairs) * (split + 1) / splits * 2;
    tile::Sums sums;
    tile::product<T, false, true>(a.weight, at.inner * kTile, a.held, outer * kTile,
                                  static_cast<uint64_t>(from) * tile::kDepth, to - from, lds, sums);
    float* partial = a.partial + (static_cast<uint64_t>(split) * a.most + outer * kTile) * a.hidden;
    tile::by_rows(sums, lds, [&](uint32_t row, uint32_t inner, const float(&v)[8]) {
        if (outer * kTile + row < rows)
            store_vec<float, 8>(partial + static_cast<uint64_t>(row) * a.hidden, (at.inner * kTile + inner) / 8,
                                a.hidden, v);
    });
}

template <typename T>
__global__ __launch_bounds__(256) void join_grad_x_kernel(GradXArgs a, T* grad_x, uint64_t grad_x_stride)
{
    const uint32_t row = blockIdx.x, rows = piece_rows(a.plan, a.first, a.most);
    if (row >= rows) return;
    const uint32_t splits = splits_of(ceil_div(rows, kTile) * a.inners, a.max_splits);
    const float factor = a.plan->factor;
    T* out = grad_x + a.rows[a.first + row] * grad_x_stride;
    for (uint32_t vec = threadIdx.x; vec * 4 < a.hidden; vec += 256) {
        float sum[4] = {};
        for (uint32_t k = 0; k < splits; ++k) {
            float v[4];
            load_vec<float>(a.partial + (static_cast<uint64_t>(k) * a.most + row) * a.hidden, vec, a.hidden, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += v[e];
        }
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (vec * 4 + e < a.hidden) out[vec * 4 + e] = Elem<T>::from_f32(sum[e] * factor);
    }
}

struct GradWeightArgs {
    tile::Matrix x, held;
    const Plan* plan;
    void* grad_weight;
    float* total;                   // [vocab][hidden] where the rows take more than one piece, else null
    uint64_t stride;
    uint32_t first, most, vocab, hidden, inners, outers;
    int accumulate;
};

template <typename T, typename W>
__global__ __launch_bounds__(tile::kThreads, 1) void grad_weight_kernel(GradWeightArgs a)
{
    __shared__ __attribute__((aligned(1024))) char lds[tile::kLdsBytes];
    const uint32_t rows = piece_rows(a.plan, a.first, a.most);
    if (rows == 0 && a.first > 0) return;
    const tile::Place at = tile::place(blockIdx.x, a.outers, a.inners);
    if (!at.valid) return;
    tile::Sums sums;
    tile::product<T, false, false>(a.x, at.inner * kTile, a.held, at.outer * kTile, 0, ceil_div(rows, 2 * tile::kDepth) * 2,
                                   lds, sums);
    const bool last = a.first + rows >= a.plan->rows;
    const float factor = a.plan->factor;
    tile::by_rows(sums, lds, [&](uint32_t outer, uint32_t inner, const float(&sum)[8]) {
        const uint32_t row = at.outer * kTile + outer, vec = (at.inner * kTile + inner) / 8;
        if (row >= a.vocab) return;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = sum[k];
        float* total = a.total + static_cast<uint64_t>(row) * a.hidden;
        if (a.first > 0)
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (vec * 8 + k < a.hidden) v[k] += total[vec * 8 + k];
        if (!last) {
            store_vec<float, 8>(total, vec, a.hidden, v);
            return;
        }
        W* out = static_cast<W*>(a.grad_weight) + row * a.stride;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= factor;
        if (a.accumulate)
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

// Sizes and the workspace's parts (offsets in bytes).
struct Layout {
    uint64_t padded, tiles, inners, all, piece, pieces, max_splits;
    uint64_t plan, rows, row_targets, gathered, weight, parts, target_scores, lse, row_loss, held, partial, total, size;

    explicit Layout(const la_linear_loss_t& c)
    {
        padded = ceil_div(c.hidden, kPair) * kPair;
        tiles = ceil_div(c.vocab, kTile);
        inners = ceil_div(c.hidden, kTile);
        all = c.n > 0 ? ceil_div(c.n, kTile) * kTile : kTile;     // no rows: one empty piece, which clears grad_weight
        piece = ceil_div(c.grads ? c.piece_rows : kForwardRows, kTile) * kTile;
        if (piece > kMostRows) piece = kMostRows;
        if (piece == 0 || piece > all) piece = all;
        pieces = ceil_div(all, piece);
        // enough runs of k for four rounds of workgroups
        const uint64_t grad_x_tiles = piece / kTile * inners;
        max_splits = ceil_div(1024, grad_x_tiles);
        if (max_splits > 64) max_splits = 64;
        if (max_splits > tiles) max_splits = tiles;
        uint64_t at = 0;
        const auto take = [&](uint64_t bytes) {
            const uint64_t here = at;
            at += ceil_div(bytes, 256) * 256;
            return here;
        };
        plan = take(sizeof(Plan));
        rows = take(c.n * 4);
        row_targets = take(c.n * 4);
        gathered = take(all * padded * 2);
        weight = reads_in_place(c) ? 0 : take(c.vocab * padded * 2);
        parts = take(piece * tiles * sizeof(Part));
        target_scores = take(piece * 4);
        lse = take(piece * 4);
        row_loss = c.row_loss ? 0 : take(c.n * 4);
        held = c.grads ? take(piece * tiles * kTile * 2) : 0;
        partial = c.grads ? take(max_splits * piece * c.hidden * 4) : 0;
        total = c.grads && pieces > 1 ? take(c.vocab * c.hidden * 4) : 0;
        size = at;
    }
};

template <typename T, typename W> int run(const la_linear_loss_t& c, char* ws, hipStream_t st)
{
    const Layout l(c);
    Plan* plan = reinterpret_cast<Plan*>(ws + l.plan);
    uint32_t* rows = reinterpret_cast<uint32_t*>(ws + l.rows);
    int32_t* row_targets = reinterpret_cast<int32_t*>(ws + l.row_targets);
    T* gathered = reinterpret_cast<T*>(ws + l.gathered);
    Part* parts = reinterpret_cast<Part*>(ws + l.parts);
    float* target_scores = reinterpret_cast<float*>(ws + l.target_scores);
    float* lse = reinterpret_cast<float*>(ws + l.lse);
    float* row_loss = c.row_loss ? c.row_loss : reinterpret_cast<float*>(ws + l.row_loss);
    T* held = c.grads ? reinterpret_cast<T*>(ws + l.held) : nullptr;
    T* grad_x = c.grads ? static_cast<T*>(c.grad_x) : nullptr;

    int rc = launch(list_rows_kernel, dim3(1), dim3(1024), st, c.targets, c.n, c.ignore_index, c.vocab, c.mean,
                    c.grad_scale, kHeld<T>, rows, row_targets, plan);
    if (rc != LA_OK) return rc;
    rc = launch(gather_kernel<T>, dim3(l.all + c.n), dim3(256), st, static_cast<const T*>(c.x), c.x_stride, c.hidden,
                l.padded, rows, plan, gathered, l.all, c.targets, c.ignore_index, row_loss, grad_x, c.grad_x_stride);
    if (rc != LA_OK) return rc;
    tile::Matrix weight{c.weight, c.vocab, c.hidden, c.weight_stride * 2};
    if (!reads_in_place(c)) {
        T* copy = reinterpret_cast<T*>(ws + l.weight);
        rc = launch(pad_kernel<T>, dim3(c.vocab), dim3(256), st, static_cast<const T*>(c.weight), c.weight_stride,
                    c.hidden, l.padded, copy);
        if (rc != LA_OK) return rc;
        weight = tile::Matrix{copy, c.vocab, l.padded, l.padded * 2};
    }
    const tile::Matrix x{gathered, l.all, l.padded, l.padded * 2};
    const tile::Matrix d{held, l.piece, l.tiles * kTile, l.tiles * kTile * 2};

    for (uint64_t p = 0; p < l.pieces; ++p) {
        const uint32_t first = p * l.piece, most = l.piece;
        const ScoreArgs scores{weight, x, plan, row_targets, parts, target_scores, held, first, most,
                               static_cast<uint32_t>(c.vocab), static_cast<uint32_t>(l.tiles),
                               static_cast<uint32_t>(l.padded / tile::kDepth)};
        rc = launch(scores_kernel<T>, dim3(tile::places(most / kTile, l.tiles)), dim3(tile::kThreads), st, scores);
        if (rc != LA_OK) return rc;
        rc = launch(row_loss_kernel, dim3(most / 4), dim3(256), st, parts, l.tiles, plan, first, most, rows,
                    row_targets, target_scores, lse, row_loss);
        if (rc != LA_OK || !c.grads) {
            if (rc != LA_OK) return rc;
            continue;
        }
        rc = launch(softmax_grad_kernel<T>, dim3(ceil_div(l.tiles * kTile, 8 * 256 * kPerGroup), most), dim3(256), st,
                    held, parts, lse, row_targets, plan, first, most, l.tiles);
        if (rc != LA_OK) return rc;
        const GradXArgs gx{weight, d, plan, rows, reinterpret_cast<float*>(ws + l.partial), first, most,
                           static_cast<uint32_t>(c.hidden), static_cast<uint32_t>(l.inners),
                           static_cast<uint32_t>(l.tiles * (kTile / kPair)),
                           static_cast<uint32_t>(l.max_splits)};
        rc = launch(grad_x_kernel<T>, dim3(tile::places(most / kTile * l.max_splits, l.inners)), dim3(tile::kThreads),
                    st, gx);
        if (rc != LA_OK) return rc;
        rc = launch(join_grad_x_kernel<T>, dim3(most), dim3(256), st, gx, grad_x, c.grad_x_stride);
        if (rc != LA_OK) return rc;
        const tile::Matrix piece_x{gathered + first * l.padded, l.piece < l.all - first ? l.piece : l.all - first,
                                   l.padded, l.padded * 2};
        const GradWeightArgs gw{piece_x, d, plan, c.grad_weight,
                                l.pieces > 1 ? reinterpret_cast<float*>(ws + l.total) : nullptr, c.grad_weight_stride,
                                first, most, static_cast<uint32_t>(c.vocab), static_cast<uint32_t>(c.hidden),
                                static_cast<uint32_t>(l.inners), static_cast<uint32_t>(l.tiles), c.accumulate};
        rc = launch(grad_weight_kernel<T, W>, dim3(tile::places(l.tiles, l.inners)), dim3(tile::kThreads), st, gw);
        if (rc != LA_OK) return rc;
    }
    if (!c.loss) return LA_OK;
    return launch(loss_kernel, dim3(1), dim3(1024), st, row_loss, rows, plan, c.mean, c.loss);
}

bool reachable(const void* p) { return !p || la_ptr::device_accessible(p); }

}  // namespace

extern "C" {

uint64_t la_linear_loss_workspace(const la_linear_loss_t* call)
{
    return call && sizes_ok(*call) ? Layout(*call).size : 0;
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
    if (rc == LA_OK) rc = check_workspace(workspace, workspace_bytes, Layout(c).size, 256);
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
