// slideformer_amd: embedding lookup with scaling, and its gradient by sorted
// tokens (gfx950, wave64).
//
// Lookup: out[i] = scale * W[t_i], a gather of whole rows; it reads and writes
// each row once and is bound by memory.
//
// Gradient: dW[t] = scale * sum over i with t_i = t of dY[i].  The tokens are
// sorted (stably, so equal tokens keep their order), the rows of dY are then
// walked in sorted order in blocks of kBlock positions, and each run of equal
// tokens is summed in fp32 registers and written once.  Nothing is added
// atomically: equal calls give equal bits.  Runs that cross a block's end leave
// fp32 partials, which a second pass adds in the order of the blocks, so a token
// that fills the whole batch is summed by all blocks and not by one wave.
#include "ops_common.h"

namespace {

constexpr int kWave = 64;

template <typename I> __device__ __forceinline__ uint64_t token_at(const I* tokens, uint64_t i)
{
    // a negative token becomes a huge one
    return static_cast<uint64_t>(static_cast<int64_t>(tokens[i]));
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
// A wave takes kLookup 16-byte vectors per lane of one row, all loaded before
// the first is stored.
constexpr int kLookup = 4;

template <typename T, typename I>
__global__ __launch_bounds__(256) void embedding_kernel(const I* tokens, uint64_t n, const T* weight, uint64_t vocab,
                                                        uint32_t hidden, uint64_t weight_stride, float scale, T* out,
                                                        uint64_t out_stride, uint32_t units)
{
    constexpr int E = Elem<T>::kCount;
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    const uint64_t i = unit / units;
    if (i >= n) return;
    const uint32_t first = static_cast<uint32_t>(unit % units) * (kLookup * kWave) + threadIdx.x % kWave;
    const uint64_t t = token_at(tokens, i);
    T* to = out + i * out_stride;
    const uint32_t vecs = (hidden + E - 1) / E;
    float x[kLookup][E];
    if (t < vocab) {
        const T* row = weight + t * weight_stride;
#pragma unroll
        for (int k = 0; k < kLookup; ++k)
            if (first + k * kWave < vecs) load_vec<T>(row, first + k * kWave, hidden, x[k]);
    }
#pragma unroll
    for (int k = 0; k < kLookup; ++k) {
        if (first + k * kWave >= vecs) break;
#pragma unroll
        for (int e = 0; e < E; ++e) x[k][e] = t < vocab ? x[k][e] * scale : __builtin_nanf("");
        store_vec<T, E>(to, first + k * kWave, hidden, x[k]);
    }
}

// ---------------------------------------------------------------------------
// sorting the tokens
// ---------------------------------------------------------------------------
// A chunk of kChunk tokens is sorted by counting, for each, the tokens of the
// chunk that come before it: kChunk compares a token, spread over the whole GPU
// with no data exchanged.  Chunks are then merged by binary search: a token's
// place is its place in its own chunk plus, for each other chunk, the number of
// tokens before it there (equal ones count in earlier chunks only).
constexpr int kChunk = 4096;
constexpr int kRankTokens = 64;           // tokens ranked by one workgroup, four lanes each
constexpr int32_t kNone = INT32_MAX;      // sorts after every token

__device__ __forceinline__ int32_t sort_key(uint64_t t, uint64_t vocab, int64_t padding)
{
    return t < vocab && t != static_cast<uint64_t>(padding) ? static_cast<int32_t>(t) : kNone;
}

template <typename I>
__global__ __launch_bounds__(256) void rank_kernel(const I* tokens, uint32_t n, uint64_t vocab, int64_t padding,
                                                   int32_t* keys, uint32_t* places)
{
    __shared__ __attribute__((aligned(16))) int32_t chunk[kChunk];
    const uint32_t base = blockIdx.x / (kChunk / kRankTokens) * kChunk;
    const uint32_t mine = blockIdx.x % (kChunk / kRankTokens) * kRankTokens + threadIdx.x / 4;
    const uint32_t size = n - base < kChunk ? n - base : kChunk;
    if (mine - threadIdx.x / 4 >= size) return;                    // the whole workgroup
    for (uint32_t k = threadIdx.x; k < kChunk; k += 256)
        chunk[k] = k < size ? sort_key(token_at(tokens, base + k), vocab, padding) : kNone;
    __syncthreads();
    const int32_t key = chunk[mine];
    const uint32_t lane = threadIdx.x % 4;
    uint32_t before = 0;
    for (uint32_t quad = lane; quad * 4 < size; quad += 4) {
        const int4 k = *reinterpret_cast<const int4*>(chunk + quad * 4);
        const int32_t other[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            before += other[e] < key || (other[e] == key && quad * 4 + e < mine);
    }
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    if (lane == 0 && mine < size) {
        keys[base + before] = key;
        places[base + before] = base + mine;
    }
}

__global__ __launch_bounds__(256) void merge_kernel(const int32_t* keys, const uint32_t* places, uint32_t n,
                                                    int32_t* sorted, uint32_t* sorted_places)
{
    // 16 lanes a token, each searching every 16th chunk
    const uint32_t at = blockIdx.x * 16 + threadIdx.x / 16;
    const uint32_t lane = threadIdx.x % 16;
    const uint32_t own = at / kChunk;
    uint32_t before = 0;
    if (at < n) {
        const int32_t key = keys[at];
        for (uint32_t c = lane; c * kChunk < n; c += 16) {
            if (c == own) continue;
            uint32_t lo = c * kChunk, hi = n - lo < kChunk ? n : lo + kChunk;
            const uint32_t start = lo;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                const int32_t k = keys[mid];
                if (k < key || (k == key && c < own)) lo = mid + 1;
                else hi = mid;
            }
            before += lo - start;
        }
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) before += __shfl_xor(before, d);
    if (at < n && lane == 0) {
        const uint32_t to = at % kChunk + before;
        sorted[to] = keys[at];
        sorted_places[to] = places[at];
    }
}

// ---------------------------------------------------------------------------
// sums over runs of equal tokens
// ---------------------------------------------------------------------------
constexpr int kBlock = 16;                // sorted positions walked by one wave

template <typename T>
__global__ __launch_bounds__(256) void clear_kernel(T* weight, uint64_t rows, uint32_t hidden, uint64_t stride,
                                                    uint32_t units)
{
    constexpr int E = Elem<T>::kCount;
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    const uint64_t row = unit / units;
    if (row >= rows) return;
    const uint32_t first = static_cast<uint32_t>(unit % units) * (kLookup * kWave) + threadIdx.x % kWave;
    const float zero[E] = {};
#pragma unroll
    for (int k = 0; k < kLookup; ++k)
        if ((first + k * kWave) * E < hidden) store_vec<T, E>(weight + row * stride, first + k * kWave, hidden, zero);
}

template <typename O, int E>
__device__ __forceinline__ void write_row(O* weight, int32_t key, uint64_t stride, uint32_t vec, uint32_t hidden,
                                          float scale, bool accumulate, const float (&sum)[E])
{
    O* row = weight + static_cast<uint64_t>(key) * stride;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t at = vec * E + e;
        x[e] = sum[e] * scale + (accumulate && at < hidden ? Elem<O>::to_f32(row[at]) : 0.0f);
    }
    store_vec<O, E>(row, vec, hidden, x);
}

// partial[2 * block]: the sum of the run that came in from the block before;
// partial[2 * block + 1]: that of the run that starts here and goes on.
template <typename T, typename O>
__global__ __launch_bounds__(256) void run_sums_kernel(const int32_t* keys, const uint32_t* places, uint32_t n,
                                                       const T* grad, uint64_t grad_stride, uint32_t hidden,
                                                       O* weight, uint64_t weight_stride, float scale, int accumulate,
                                                       float* partial, uint32_t slices)
{
    constexpr int E = Elem<T>::kCount;
    const uint32_t unit = blockIdx.x * 4 + threadIdx.x / kWave;
    const uint32_t block = unit / slices;
    const uint32_t vec = unit % slices * kWave + threadIdx.x % kWave;
    const uint32_t first = block * kBlock;
    if (first >= n || vec * E >= hidden) return;
    const uint32_t last = n - first < kBlock ? n : first + kBlock;
    int32_t key = keys[first];
    bool came_in = first > 0 && keys[first - 1] == key;
    float sum[E] = {};
    for (uint32_t at = first; at < last && key != kNone; ++at) {
        float x[E];
        load_vec<T>(grad + static_cast<uint64_t>(places[at]) * grad_stride, vec, hidden, x);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += x[e];
        const int32_t next = at + 1 < n ? keys[at + 1] : kNone;
        if (next == key && at + 1 < last) continue;
        if (next == key || came_in)
            store_vec<float, E>(partial + (2ull * block + (came_in ? 0 : 1)) * hidden, vec, hidden, sum);
        else
            write_row<O, E>(weight, key, weight_stride, vec, hidden, scale, accumulate, sum);
        key = next;
        came_in = false;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    }
}

template <typename T, typename O>
__global__ __launch_bounds__(256) void join_runs_kernel(const int32_t* keys, uint32_t n, uint32_t hidden, O* weight,
                                                        uint64_t weight_stride, float scale, int accumulate,
                                                        const float* partial, uint32_t slices)
{
    constexpr int E = Elem<T>::kCount;
    const uint32_t unit = blockIdx.x * 4 + threadIdx.x / kWave;
    uint32_t block = unit / slices;
    const uint32_t vec = unit % slices * kWave + threadIdx.x % kWave;
    uint32_t end = (block + 1) * kBlock;                            // the position after this block
    if (end >= n || vec * E >= hidden) return;
    const int32_t key = keys[end - 1];
    if (key == kNone || keys[end] != key) return;                   // nothing goes on
    if (block > 0 && keys[block * kBlock] == key && keys[block * kBlock - 1] == key) return;   // it started earlier
    float sum[E], x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t at = vec * E + e;
        sum[e] = at < hidden ? partial[(2ull * block + 1) * hidden + at] : 0.0f;
    }
    do {
        ++block;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t at = vec * E + e;
            x[e] = at < hidden ? partial[2ull * block * hidden + at] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += x[e];
        end += kBlock;
    } while (end < n && keys[end - 1] == key && keys[end] == key);
    write_row<O, E>(weight, key, weight_stride, vec, hidden, scale, accumulate, sum);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint64_t kMaxTokens = 1ull << 30;
constexpr uint64_t kMaxHidden = 1ull << 24;
constexpr uint64_t kMaxGrid = (1ull << 24) - 1;   // a launch has under 2^32 threads

uint64_t pad(uint64_t bytes) { return ceil_div(bytes, 256) * 256; }

// keys and places of the sorted chunks, of the sorted whole, then the partials
uint64_t grad_workspace(uint64_t n, uint64_t hidden)
{
    return 4 * pad(4 * n) + pad(ceil_div(n, kBlock) * 2 * hidden * 4);
}

template <typename T>
int lookup(int token_dtype, const void* tokens, uint64_t n, const void* weight, uint64_t vocab, uint64_t hidden,
           uint64_t weight_stride, float scale, void* out, uint64_t out_stride, hipStream_t st)
{
    const uint64_t units = ceil_div(hidden, kLookup * kWave * Elem<T>::kCount);
    const uint64_t grid = ceil_div(n * units, 4);
    if (grid > kMaxGrid) return LA_EINVAL;
    if (token_dtype == LA_I32)
        return launch(embedding_kernel<T, int32_t>, dim3(grid), dim3(256), st, static_cast<const int32_t*>(tokens), n,
                      static_cast<const T*>(weight), vocab, hidden, weight_stride, scale, static_cast<T*>(out),
                      out_stride, units);
    return launch(embedding_kernel<T, int64_t>, dim3(grid), dim3(256), st, static_cast<const int64_t*>(tokens), n,
                  static_cast<const T*>(weight), vocab, hidden, weight_stride, scale, static_cast<T*>(out), out_stride,
                  units);
}

struct GradCall {
    int token_dtype;
    const void* tokens;
    uint32_t n;
    const void* grad;
    uint64_t grad_stride;
    void* weight;
    uint64_t vocab;
    uint32_t hidden;
    uint64_t weight_stride;
    float scale;
    int64_t padding;
    int accumulate;
    char* workspace;
    hipStream_t st;
};

template <typename T, typename O> int sum_runs(const GradCall& c, const int32_t* keys, const uint32_t* places)
{
    float* partial = reinterpret_cast<float*>(c.workspace + 4 * pad(4ull * c.n));
    const uint32_t slices = ceil_div(c.hidden, kWave * Elem<T>::kCount);
    const uint64_t blocks = ceil_div(c.n, kBlock);
    const uint64_t grid = ceil_div(blocks * slices, 4);
    if (grid > kMaxGrid) return LA_EINVAL;
    int rc = launch(run_sums_kernel<T, O>, dim3(grid), dim3(256), c.st, keys, places, c.n,
                    static_cast<const T*>(c.grad), c.grad_stride, c.hidden, static_cast<O*>(c.weight), c.weight_stride,
                    c.scale, c.accumulate, partial, slices);
    if (rc != LA_OK || blocks == 1) return rc;
    return launch(join_runs_kernel<T, O>, dim3(grid), dim3(256), c.st, keys, c.n, c.hidden, static_cast<O*>(c.weight),
                  c.weight_stride, c.scale, c.accumulate, partial, slices);
}

template <typename T, typename O> int grad(const GradCall& c)
{
    if (!c.accumulate) {
        const uint64_t units = ceil_div(c.hidden, kLookup * kWave * Elem<O>::kCount);
        const uint64_t grid = ceil_div(c.vocab * units, 4);
        if (grid > kMaxGrid) return LA_EINVAL;
        const int rc = launch(clear_kernel<O>, dim3(grid), dim3(256), c.st, static_cast<O*>(c.weight), c.vocab,
                              c.hidden, c.weight_stride, units);
        if (rc != LA_OK) return rc;
    }
    if (c.n == 0) return LA_OK;
    int32_t* keys = reinterpret_cast<int32_t*>(c.workspace);
    uint32_t* places = reinterpret_cast<uint32_t*>(c.workspace + pad(4ull * c.n));
    const uint32_t chunks = ceil_div(c.n, kChunk);
    const dim3 rank_grid(chunks * (kChunk / kRankTokens));
    int rc = c.token_dtype == LA_I32
                 ? launch(rank_kernel<int32_t>, rank_grid, dim3(256), c.st, static_cast<const int32_t*>(c.tokens), c.n,
                          c.vocab, c.padding, keys, places)
                 : launch(rank_kernel<int64_t>, rank_grid, dim3(256), c.st, static_cast<const int64_t*>(c.tokens), c.n,
                          c.vocab, c.padding, keys, places);
    if (rc != LA_OK) return rc;
    if (chunks > 1) {
        int32_t* sorted = reinterpret_cast<int32_t*>(c.workspace + 2 * pad(4ull * c.n));
        uint32_t* sorted_places = reinterpret_cast<uint32_t*>(c.workspace + 3 * pad(4ull * c.n));
        rc = launch(merge_kernel, dim3(ceil_div(c.n, 16)), dim3(256), c.st, keys, places, c.n, sorted, sorted_places);
        if (rc != LA_OK) return rc;
        keys = sorted;
        places = sorted_places;
    }
    return sum_runs<T, O>(c, keys, places);
}

bool token_types(int dtype) { return dtype == LA_I32 || dtype == LA_I64; }

}  // namespace

extern "C" {

int la_ops_abi_version(void) { return LA_OPS_ABI_VERSION; }

int la_embedding(int token_dtype, const void* tokens, uint64_t n, int dtype, const void* weight, uint64_t vocab,
                 uint64_t hidden, uint64_t weight_stride, float scale, void* out, uint64_t out_stride,
                 la_stream_t stream)
{
    if (!token_types(token_dtype) || !is_float_dtype(dtype)) return LA_EDTYPE;
    if (n == 0 || hidden == 0) return LA_OK;
    if (n > kMaxTokens || hidden > kMaxHidden || vocab > static_cast<uint64_t>(INT32_MAX)) return LA_EINVAL;
    int rc = check_matrix(tokens, token_dtype, 1, 1);
    if (rc == LA_OK && vocab > 0) rc = check_matrix(weight, dtype, hidden, weight_stride);
    if (rc == LA_OK) rc = check_matrix(out, dtype, hidden, out_stride);
    if (rc != LA_OK) return rc;
    if (!la_ptr::device_accessible(tokens) || (vocab > 0 && !la_ptr::device_accessible(weight)) ||
        !la_ptr::device_accessible(out))
        return LA_EFAULT;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == LA_F32)
        return lookup<float>(token_dtype, tokens, n, weight, vocab, hidden, weight_stride, scale, out, out_stride, st);
    if (dtype == LA_BF16)
        return lookup<__bf16>(token_dtype, tokens, n, weight, vocab, hidden, weight_stride, scale, out, out_stride, st);
    return lookup<_Float16>(token_dtype, tokens, n, weight, vocab, hidden, weight_stride, scale, out, out_stride, st);
}

uint64_t la_embedding_grad_workspace(uint64_t n, uint64_t hidden)
{
    return n > kMaxTokens || hidden > kMaxHidden ? 0 : grad_workspace(n, hidden);
}

int la_embedding_grad(int token_dtype, const void* tokens, uint64_t n, int g_dtype, const void* grad_out,
                      uint64_t grad_stride, int out_dtype, void* grad_weight, uint64_t vocab, uint64_t hidden,
                      uint64_t weight_stride, float scale, int64_t padding_idx, int accumulate, void* workspace,
                      uint64_t workspace_bytes, la_stream_t stream)
{
    if (!token_types(token_dtype) || !is_float_dtype(g_dtype) || !is_float_dtype(out_dtype)) return LA_EDTYPE;
    if (out_dtype != g_dtype && out_dtype != LA_F32) return LA_EDTYPE;
    if (vocab == 0 || hidden == 0) return LA_OK;
    if (n > kMaxTokens || hidden > kMaxHidden || vocab > static_cast<uint64_t>(INT32_MAX)) return LA_EINVAL;
    int rc = check_matrix(grad_weight, out_dtype, hidden, weight_stride);
    if (rc == LA_OK && n > 0) rc = check_matrix(tokens, token_dtype, 1, 1);
    if (rc == LA_OK && n > 0) rc = check_matrix(grad_out, g_dtype, hidden, grad_stride);
    if (rc == LA_OK && n > 0) rc = check_workspace(workspace, workspace_bytes, grad_workspace(n, hidden), 16);
    if (rc != LA_OK) return rc;
    if (!la_ptr::device_accessible(grad_weight) ||
        (n > 0 && (!la_ptr::device_accessible(tokens) || !la_ptr::device_accessible(grad_out) ||
                   !la_ptr::device_accessible(workspace))))
        return LA_EFAULT;
    const GradCall c{token_dtype, tokens, static_cast<uint32_t>(n), grad_out, grad_stride, grad_weight, vocab,
                     static_cast<uint32_t>(hidden), weight_stride, scale, padding_idx, accumulate != 0,
                     static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
    if (g_dtype == LA_F32) return grad<float, float>(c);
    if (g_dtype == LA_BF16) return out_dtype == LA_F32 ? grad<__bf16, float>(c) : grad<__bf16, __bf16>(c);
    return out_dtype == LA_F32 ? grad<_Float16, float>(c) : grad<_Float16, _Float16>(c);
}

}  // extern "C"
