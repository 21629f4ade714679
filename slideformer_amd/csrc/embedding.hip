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
// the first is stored.  8192 tokens of 128256 x 4096 bf16: 20.2 us, 6.6 TB/s; one
// token: 2.9 us, a launch and two loads that depend on each other.
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
// chunk that come before it: kChunk compares a token, spread over many workgroups
// with no data exchanged.  Chunks are then merged by binary search: a token's
// place is its place in its own chunk plus, for each other chunk, the number of
// tokens before it there (equal ones count in earlier chunks only).  Two launches
// whatever the vocabulary; with chunks of 1024 they take 8192 tokens 5.6 + 5.0 us, with
// chunks of 4096 the counting alone took 54.
constexpr int kChunk = 1024;
constexpr int kRankLanes = 16;            // that share one token's compares
constexpr int kRankTokens = 256 / kRankLanes;   // ranked by one workgroup
constexpr int kRankGroups = kChunk / kRankTokens;
constexpr uint32_t kNone = 0x7fffffffu;   // sorts after every token

__device__ __forceinline__ uint32_t sort_key(uint64_t t, uint64_t vocab, int64_t padding)
{
    return t < vocab && t != static_cast<uint64_t>(padding) ? static_cast<uint32_t>(t) : kNone;
}

// The workgroups after the first `groups` clear the marks of the tokens that occur.
template <typename I>
__global__ __launch_bounds__(256) void rank_kernel(const I* tokens, uint32_t n, uint64_t vocab, int64_t padding,
                                                   uint32_t* keys, uint32_t* places, uint32_t groups, uint4* marks)
{
    const uint32_t group = blockIdx.x;
    if (group >= groups) {
        const uint64_t at = static_cast<uint64_t>(group - groups) * 256 + threadIdx.x;
        if (at * 16 < vocab) marks[at] = uint4{0, 0, 0, 0};
        return;
    }
    __shared__ __attribute__((aligned(16))) uint32_t chunk[kChunk];
    const uint32_t base = group / kRankGroups * kChunk;
    const uint32_t mine = group % kRankGroups * kRankTokens + threadIdx.x / kRankLanes;
    const uint32_t size = n - base < kChunk ? n - base : kChunk;
    if (group % kRankGroups * kRankTokens >= size) return;          // the whole workgroup
#pragma unroll
    for (uint32_t k = threadIdx.x; k < kChunk; k += 256)
        chunk[k] = k < size ? sort_key(token_at(tokens, base + k), vocab, padding) : kNone;
    __syncthreads();
    const uint32_t key = chunk[mine];
    const uint32_t lane = threadIdx.x % kRankLanes;
    uint32_t before = 0;
#pragma unroll 4
    for (uint32_t quad = lane; quad < kChunk / 4; quad += kRankLanes) {
        const uint4 k = *reinterpret_cast<const uint4*>(chunk + quad * 4);
        const uint32_t other[4] = {k.x, k.y, k.z, k.w};
        // an equal key counts where it stands before
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) before += other[e] < key + (quad * 4 + e < mine);
    }
#pragma unroll
    for (int d = kRankLanes / 2; d > 0; d >>= 1) before += __shfl_xor(before, d);
    if (lane == 0 && mine < size) {
        keys[base + before] = key;
        places[base + before] = base + mine;
    }
}

// 16 lanes a token: the searches of its chunks run beside each other, ten loads
// deep each.  8192 tokens: 5 us, which is their latency.  There are n / 1024 searches a
// token, so a batch of many chunks pays for their square: the whole gradient of 50257 x 256
// takes 47 us for 32768 tokens and 324 for 131072, where torch's index_add takes 69 and 175.
__global__ __launch_bounds__(256) void merge_kernel(const uint32_t* keys, const uint32_t* places, uint32_t n,
                                                    uint32_t* sorted, uint32_t* sorted_places, uint8_t* marks)
{
    // 16 lanes a token, each searching every 16th chunk
    const uint32_t at = blockIdx.x * 16 + threadIdx.x / 16;
    const uint32_t lane = threadIdx.x % 16;
    const uint32_t own = at / kChunk;
    uint32_t before = 0;
    if (at < n) {
        const uint32_t key = keys[at];
        for (uint32_t c = lane; c * kChunk < n; c += 16) {
            if (c == own) continue;
            uint32_t lo = c * kChunk, hi = n - lo < kChunk ? n : lo + kChunk;
            const uint32_t start = lo;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                const uint32_t k = keys[mid];
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
        const uint32_t key = keys[at];
        sorted[to] = key;
        sorted_places[to] = places[at];
        if (marks && key != kNone) marks[key] = 1;
    }
}

// ---------------------------------------------------------------------------
// sums over runs of equal tokens
// ---------------------------------------------------------------------------
// A wave sums kBlock positions, all of whose rows it loads before it stores the
// first sum: a later load would wait for the stores before it too.  Alone, 8192
// tokens 4096 wide take 39 us in blocks of 8, 59 us in blocks of 32 by four trips.
constexpr int kBlock = 8;
constexpr int kJoinWaves = 4;             // that share the blocks of a long run
constexpr int kFlight = 4;                // partials in flight in each

template <typename O, int E>
__device__ __forceinline__ void write_row(O* weight, uint32_t key, uint64_t stride, uint32_t vec, uint32_t hidden,
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

struct SumArgs {
    const uint32_t* keys;
    const uint32_t* places;
    const void* grad;
    void* weight;
    float* partial;
    const uint8_t* marks;           // of the tokens that occur
    uint64_t grad_stride, weight_stride, vocab;
    uint32_t n, hidden, slices, groups;
    float scale;
    int accumulate;
};

// Zeros in a row by one wave.  They are not read here again, and nontemporal stores
// leave the caches to the sums: 241 -> 235 us for 8192 tokens of 128256 x 4096, 47 ->
// 41 us for 4095 of 50257 x 768 in fp32.
template <typename O> __device__ __forceinline__ void clear_row(O* to, uint32_t hidden)
{
    constexpr uint32_t E = Elem<O>::kCount;
    for (uint32_t vec = threadIdx.x % kWave; vec * E < hidden; vec += kWave) {
        if (vec * E + E <= hidden) {
            __builtin_nontemporal_store(u32x4_t{0, 0, 0, 0}, reinterpret_cast<u32x4_any*>(to + vec * E));
        } else {
            const float zero[E] = {};
            store_vec<O, E>(to, vec, hidden, zero);
        }
    }
}

// partial[2 * block]: the sum of the run that came in from the block before;
// partial[2 * block + 1]: that of the run that starts here and goes on.
// The workgroups after the first `groups` clear the rows of tokens that do not occur:
// the sums wait for scattered rows, and the zeros keep memory busy meanwhile.
template <typename T, typename O> __global__ __launch_bounds__(256, 8) void run_sums_kernel(SumArgs a)
{
    if (blockIdx.x >= a.groups) {
        const uint64_t row = __builtin_amdgcn_readfirstlane((blockIdx.x - a.groups) * 4 + threadIdx.x / kWave);
        if (row < a.vocab && !a.marks[row]) clear_row(static_cast<O*>(a.weight) + row * a.weight_stride, a.hidden);
        return;
    }
    const uint32_t* keys = a.keys;
    const uint32_t* places = a.places;
    const T* grad = static_cast<const T*>(a.grad);
    O* weight = static_cast<O*>(a.weight);
    float* partial = a.partial;
    const uint32_t n = a.n, hidden = a.hidden, slices = a.slices;
    constexpr int E = Elem<T>::kCount;
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / kWave);
    const uint32_t block = unit / slices;
    const uint32_t vec = unit % slices * kWave + threadIdx.x % kWave;
    const uint32_t first = block * kBlock;
    if (first >= n || vec * E >= hidden) return;
    uint32_t key = keys[first];
    if (key == kNone) return;                                       // nothing but tokens that are left out
    bool came_in = first > 0 && keys[first - 1] == key;
    uint32_t next[kBlock];
    u32x4_t x[kBlock];                                              // as loaded: half the registers
    float sum[E] = {};
#pragma unroll
    for (uint32_t k = 0; k < kBlock; ++k) {
        const uint32_t at = first + k;
        next[k] = at + 1 < n ? keys[at + 1] : kNone;
        const uint64_t place = at < n ? places[at] : places[first];  // beyond the end: any row, not added
        x[k] = load_raw<T>(grad + place * a.grad_stride, vec, hidden);
    }
#pragma unroll
    for (uint32_t k = 0; k < kBlock; ++k) {
        if (key == kNone) break;
        float row[E];
        Elem<T>::unpack(x[k], row);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += row[e];
        if (next[k] == key && k + 1 < kBlock) continue;
        if (next[k] == key || came_in)
            store_vec<float, E>(partial + (2ull * block + (came_in ? 0 : 1)) * hidden, vec, hidden, sum);
        else
            write_row<O, E>(weight, key, a.weight_stride, vec, hidden, a.scale, a.accumulate, sum);
        key = next[k];
        came_in = false;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    }
}

// A workgroup joins the run that starts in block `unit / slices` and goes on.  Its
// waves take turns of kFlight partials and their sums are added in order.  8192
// tokens of 128256 x 4096 with a most frequent one of 490: 14.3 us, latency; 8192 equal
// tokens of 50257 x 256, 1024 partials one workgroup joins: 168 us for the whole call,
// 26 where tokens differ.
template <typename T, typename O> __global__ __launch_bounds__(256) void join_runs_kernel(SumArgs a)
{
    constexpr int E = Elem<T>::kCount;
    __shared__ float lds[kJoinWaves - 1][E][kWave];
    const uint32_t* keys = a.keys;
    const uint32_t n = a.n, hidden = a.hidden;
    const uint32_t block = blockIdx.x / a.slices, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t vec = blockIdx.x % a.slices * kWave + lane;
    const uint32_t end = (block + 1) * kBlock;                      // the position after this block
    if (end >= n) return;
    const uint32_t key = keys[end - 1];
    if (key == kNone || keys[end] != key) return;                   // nothing goes on
    if (block > 0 && keys[end - kBlock] == key && keys[end - kBlock - 1] == key) return;   // it started earlier
    const auto load = [&](uint64_t which, float(&x)[E]) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            float part[4];
            load_vec<float>(a.partial + which * hidden, (vec * E + e) / 4, hidden, part);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[e + k] = part[k];
        }
    };
    float sum[E] = {};
    if (wave == 0) load(2ull * block + 1, sum);
    // the blocks that begin with the same token, found 64 at a time
    for (uint32_t from = block + 1;; from += kWave) {
        const uint64_t start = static_cast<uint64_t>(from + lane) * kBlock;
        const uint64_t same = __ballot(start < n && keys[start < n ? start : 0] == key);
        const uint32_t count = same == ~0ull ? kWave : __builtin_ctzll(~same);
        for (uint32_t k = wave * kFlight; k < count; k += kJoinWaves * kFlight) {
            float x[kFlight][E];
#pragma unroll
            for (uint32_t f = 0; f < kFlight; ++f)
                if (k + f < count) load(2ull * (from + k + f), x[f]);
#pragma unroll
            for (uint32_t f = 0; f < kFlight; ++f)
                if (k + f < count)
#pragma unroll
                    for (int e = 0; e < E; ++e) sum[e] += x[f][e];
        }
        if (count < kWave) break;
    }
    if (wave > 0)
#pragma unroll
        for (int e = 0; e < E; ++e) lds[wave - 1][e][lane] = sum[e];
    __syncthreads();
    if (wave > 0 || vec * E >= hidden) return;
#pragma unroll
    for (int w = 0; w < kJoinWaves - 1; ++w)
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += lds[w][e][lane];
    write_row<O, E>(static_cast<O*>(a.weight), key, a.weight_stride, vec, hidden, a.scale, a.accumulate, sum);
}

// Up to kFewTokens tokens need no sorting: each wave looks through all of them.  The
// first `groups` workgroups have one for each token and slice of its row, which sums
// all rows of the token's where it is its first occurrence: wave k those among tokens
// 64 k to 64 k + 63, in order, kTogether of them in flight at a time; the waves' sums are
// added in order too.  The other workgroups have a wave for each row of the
// matrix, which clears it where no token is its own.  One launch for four: 7
// tokens of 23587 x 1600 fp32 27 us, sorted 34; 250 of 2000 x 512 5.4 and 13 us; 256 equal
// ones of 1000 x 4096 bf16 10 and 16 us (340 by one wave, a row after the other).
constexpr uint32_t kFewTokens = 256;
constexpr int kTogether = 16;

// Which of the tokens are `row`, as bits; returns whether any is.
template <typename I>
__device__ __forceinline__ bool find(const I* tokens, uint32_t n, uint64_t row, uint64_t (&mine)[kFewTokens / kWave])
{
    uint64_t any = 0;
#pragma unroll
    for (uint32_t k = 0; k < kFewTokens / kWave; ++k) {
        mine[k] = 0;
        if (k * kWave < n) {
            const uint32_t at = k * kWave + threadIdx.x % kWave;
            mine[k] = __ballot(at < n && token_at(tokens, at < n ? at : 0) == row);
        }
        any |= mine[k];
    }
    return any != 0;
}

template <typename T, typename O, typename I>
__global__ __launch_bounds__(256) void few_tokens_kernel(const I* tokens, uint32_t n, int64_t padding, const T* grad,
                                                         uint64_t grad_stride, O* weight, uint64_t vocab,
                                                         uint32_t hidden, uint64_t weight_stride, float scale,
                                                         uint32_t slices, uint32_t groups)
{
    constexpr int E = Elem<T>::kCount;
    uint64_t mine[kFewTokens / kWave];
    if (blockIdx.x >= groups) {
        const uint64_t row = __builtin_amdgcn_readfirstlane((blockIdx.x - groups) * 4 + threadIdx.x / kWave);
        if (row < vocab && (!find(tokens, n, row, mine) || row == static_cast<uint64_t>(padding)))
            clear_row(weight + row * weight_stride, hidden);
        return;
    }
    __shared__ float lds[kFewTokens / kWave][E][kWave];
    const uint32_t own = blockIdx.x / slices, lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t vec = blockIdx.x % slices * kWave + lane;
    const uint64_t row = token_at(tokens, own);
    if (row >= vocab || row == static_cast<uint64_t>(padding)) return;
    find(tokens, n, row, mine);
    uint32_t first = kFewTokens, waves = 0;                         // that have rows of this token
#pragma unroll
    for (uint32_t k = 0; k < kFewTokens / kWave; ++k)
        if (mine[k]) {
            if (first == kFewTokens) first = k * kWave + __builtin_ctzll(mine[k]);
            ++waves;
        }
    if (first != own) return;                                       // the whole workgroup
    uint64_t left = 0;
#pragma unroll
    for (uint32_t k = 0; k < kFewTokens / kWave; ++k)
        if (k == wave) left = mine[k];
    float sum[E] = {};
    while (left) {
        u32x4_t x[kTogether];
        const int count = __builtin_popcountll(left);
#pragma unroll
        for (int f = 0; f < kTogether; ++f)
            if (f < count) {
                x[f] = load_raw<T>(grad + (wave * kWave + __builtin_ctzll(left)) * grad_stride, vec, hidden);
                left &= left - 1;
            }
#pragma unroll
        for (int f = 0; f < kTogether; ++f)
            if (f < count) {
                float g[E];
                Elem<T>::unpack(x[f], g);
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] += g[e];
            }
    }
    if (waves > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) lds[wave][e][lane] = sum[e];
        __syncthreads();
        if (wave == own / kWave)
            for (uint32_t k = wave + 1; k < kFewTokens / kWave; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] += lds[k][e][lane];
    }
    if (wave != own / kWave || vec * E >= hidden) return;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] *= scale;
    store_vec<O, E>(weight + row * weight_stride, vec, hidden, sum);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint64_t kMaxTokens = 1ull << 30;
constexpr uint64_t kMaxHidden = 1ull << 24;
constexpr uint64_t kMaxGrid = (1ull << 24) - 1;   // a launch has under 2^32 threads

uint64_t pad(uint64_t bytes) { return ceil_div(bytes, 256) * 256; }

// Keys and places of the sorted chunks, of the sorted whole, the marks, then the partials.
struct Workspace {
    uint64_t keys, places, sorted, sorted_places, marks, partial, size;

    Workspace(uint64_t n, uint64_t vocab, uint64_t hidden)
    {
        keys = 0;
        places = keys + pad(4 * n);
        sorted = places + pad(4 * n);
        sorted_places = sorted + pad(4 * n);
        marks = sorted_places + pad(4 * n);
        partial = marks + pad(vocab);
        size = partial + pad(ceil_div(n, kBlock) * 2 * hidden * 4);
    }
};

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

template <typename I> int sort(const GradCall& c, const Workspace& w)
{
    uint32_t* keys = reinterpret_cast<uint32_t*>(c.workspace + w.keys);
    uint32_t* places = reinterpret_cast<uint32_t*>(c.workspace + w.places);
    uint8_t* marks = c.accumulate ? nullptr : reinterpret_cast<uint8_t*>(c.workspace + w.marks);
    const uint64_t groups = ceil_div(c.n, kChunk) * kRankGroups;
    const uint64_t clear = marks ? ceil_div(c.vocab, 256 * 16) : 0;
    if (groups + clear == 0) return LA_OK;
    int rc = launch(rank_kernel<I>, dim3(groups + clear), dim3(256), c.st, static_cast<const I*>(c.tokens), c.n,
                    c.vocab, c.padding, keys, places, groups, reinterpret_cast<uint4*>(marks));
    if (rc != LA_OK || c.n == 0) return rc;
    return launch(merge_kernel, dim3(ceil_div(c.n, 16)), dim3(256), c.st, keys, places, c.n,
                  reinterpret_cast<uint32_t*>(c.workspace + w.sorted),
                  reinterpret_cast<uint32_t*>(c.workspace + w.sorted_places), marks);
}

template <typename T, typename O, typename I> int few_tokens(const GradCall& c)
{
    const uint64_t slices = ceil_div(c.hidden, kWave * Elem<T>::kCount);
    const uint64_t groups = c.n * slices, clear = ceil_div(c.vocab, 4);
    if (groups + clear > kMaxGrid) return LA_EINVAL;
    return launch(few_tokens_kernel<T, O, I>, dim3(groups + clear), dim3(256), c.st, static_cast<const I*>(c.tokens),
                  c.n, c.padding, static_cast<const T*>(c.grad), c.grad_stride, static_cast<O*>(c.weight), c.vocab,
                  c.hidden, c.weight_stride, c.scale, slices, groups);
}

template <typename T, typename O> int grad(const GradCall& c)
{
    if (c.n <= kFewTokens && !c.accumulate)
        return c.token_dtype == LA_I32 ? few_tokens<T, O, int32_t>(c) : few_tokens<T, O, int64_t>(c);
    const Workspace w(c.n, c.vocab, c.hidden);
    SumArgs a{};
    a.keys = reinterpret_cast<const uint32_t*>(c.workspace + w.sorted);
    a.places = reinterpret_cast<const uint32_t*>(c.workspace + w.sorted_places);
    a.grad = c.grad;
    a.weight = c.weight;
    a.partial = reinterpret_cast<float*>(c.workspace + w.partial);
    a.marks = reinterpret_cast<const uint8_t*>(c.workspace + w.marks);
    a.grad_stride = c.grad_stride;
    a.weight_stride = c.weight_stride;
    a.vocab = c.vocab;
    a.n = c.n;
    a.hidden = c.hidden;
    a.slices = ceil_div(c.hidden, kWave * Elem<T>::kCount);
    a.scale = c.scale;
    a.accumulate = c.accumulate;
    const uint64_t blocks = ceil_div(c.n, kBlock);
    const uint64_t groups = ceil_div(blocks * a.slices, 4);
    const uint64_t clear = c.accumulate ? 0 : ceil_div(c.vocab, 4);
    a.groups = groups;
    if (blocks * a.slices > kMaxGrid || groups + clear > kMaxGrid) return LA_EINVAL;
    if (groups + clear == 0) return LA_OK;
    int rc = c.token_dtype == LA_I32 ? sort<int32_t>(c, w) : sort<int64_t>(c, w);
    if (rc != LA_OK) return rc;
    rc = launch(run_sums_kernel<T, O>, dim3(groups + clear), dim3(256), c.st, a);
    if (rc != LA_OK || blocks <= 1) return rc;
    return launch(join_runs_kernel<T, O>, dim3(blocks * a.slices), dim3(256), c.st, a);
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

uint64_t la_embedding_grad_workspace(uint64_t n, uint64_t vocab, uint64_t hidden)
{
    const bool fits = n <= kMaxTokens && hidden <= kMaxHidden && vocab <= static_cast<uint64_t>(INT32_MAX);
    return fits ? Workspace(n, vocab, hidden).size : 0;
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
    if (rc == LA_OK) rc = check_workspace(workspace, workspace_bytes, Workspace(n, vocab, hidden).size, 16);
    if (rc != LA_OK) return rc;
    if (!la_ptr::device_accessible(grad_weight) ||
        !la_ptr::device_accessible(workspace) ||
        (n > 0 && (!la_ptr::device_accessible(tokens) || !la_ptr::device_accessible(grad_out))))
        return LA_EFAULT;
    const GradCall c{token_dtype, tokens, static_cast<uint32_t>(n), grad_out, grad_stride, grad_weight, vocab,
                     static_cast<uint32_t>(hidden), weight_stride, scale, padding_idx, accumulate != 0,
                     static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
    if (g_dtype == LA_F32) return grad<float, float>(c);
    if (g_dtype == LA_BF16) return out_dtype == LA_F32 ? grad<__bf16, float>(c) : grad<__bf16, __bf16>(c);
    return out_dtype == LA_F32 ? grad<_Float16, float>(c) : grad<_Float16, _Float16>(c);
}

}  // extern "C"
