// slideformer_amd: the root-mean-square norm of every query and key head and the
// position rotation after it, in one pass, and its gradient (gfx950, wave64).
//
// Forward, per head of a token: r = 1 / sqrt(mean(x^2) + eps), y = x r w, then each pair
// (a, b) of the rotated elements becomes (a cos - b sin, b cos + a sin).
// Gradient: with g the pairs of dy turned back, (a cos + b sin, b cos - a sin), and u = x r,
// dx = r (g w - u mean(g w u)), dw = sum over all heads and tokens of g u.
//
// Bound by memory, or for few tokens by latency.  A head is 256 bytes: eight lanes with
// two 16-byte accesses each in 16-bit types, whose elements are pairs of one another, so a
// head's sum needs three exchanges and the rotation none.  A wave stays on one token,
// whose row of the tables it reads once for all heads it takes.
#include "memory_overlap.h"
#include "ops_common.h"

#include <algorithm>

namespace {

constexpr uint32_t kWave = 64;

struct HeadRows {
    char* data;
    uint64_t row, head;             // distances in bytes
};

struct RotaryArgs {
    HeadRows q, k, q_out, k_out, grad_q, grad_k;
    const void *q_weight, *k_weight;
    const float *cos, *sin;
    const void* at;
    uint64_t positions;
    float* partial;                 // of each workgroup: the sums for its heads' weight, [dim]
    uint32_t n, heads, kv_heads, dim, rotated;
    uint32_t lanes;                 // to a head: a power of two
    uint32_t chunks, kv_chunks;     // waves that share a token's query heads, and its key heads
    uint32_t workers;               // workgroups of a gradient that take query heads; the others take key heads
    int wide;
    float eps, per_dim;
};

// Two of a head's 16-byte vectors, a lane's share of it.
struct Slot {
    uint32_t first[2];              // their first elements
    uint32_t count[2];              // how many of them there are
    uint32_t pair, pairs;           // the pairs that they make up; 0 pairs: elements that are not rotated
};

template <bool INTERLEAVED, uint32_t V> __device__ __forceinline__ Slot slot_of(uint32_t s, uint32_t dim, uint32_t rotated)
{
    const uint32_t pairs = rotated / 2, turning = ceil_div(pairs, V);
    Slot t;
    t.pair = s * V;
    t.pairs = s < turning ? (pairs - s * V < V ? pairs - s * V : V) : 0u;
    if (!INTERLEAVED && s < turning) {
        t.first[0] = s * V;
        t.first[1] = pairs + s * V;
        t.count[0] = t.count[1] = t.pairs;
        return t;
    }
    const uint32_t from = s < turning ? s * 2 * V : rotated + (s - turning) * 2 * V;
    const uint32_t end = s < turning ? rotated : dim;
    const uint32_t left = from < end ? end - from : 0;
    t.first[0] = from;
    t.first[1] = from + V;
    t.count[0] = left < V ? left : V;
    t.count[1] = left <= V ? 0 : left - V < V ? left - V : V;
    return t;
}

inline uint32_t slots(uint32_t dim, uint32_t rotated, uint32_t v)
{
    return ceil_div(rotated / 2, v) + ceil_div(dim - rotated, 2 * v);
}

// WHOLE: every lane of every head has two whole vectors, so that there are no branches between its loads.
template <typename T, bool WHOLE = false> __device__ __forceinline__ u32x4_t load_some(const T* from, uint32_t count)
{
    constexpr uint32_t V = Elem<T>::kCount;
    if (WHOLE || count == V) return *reinterpret_cast<const u32x4_any*>(from);
    T x[V];
#pragma unroll
    for (uint32_t i = 0; i < V; ++i) x[i] = i < count ? from[i] : Elem<T>::from_f32(0.0f);
    return __builtin_bit_cast(u32x4_t, x);
}

// PAST_CACHES: results of a batch that the caches would not hold until they are read.
template <typename T, bool WHOLE, bool PAST_CACHES = false>
__device__ __forceinline__ void store_some(T* to, uint32_t count, const float (&x)[Elem<T>::kCount])
{
    constexpr uint32_t V = Elem<T>::kCount;
    if (WHOLE || count == V) {
        if (PAST_CACHES) __builtin_nontemporal_store(Elem<T>::pack(x), reinterpret_cast<u32x4_any*>(to));
        else *reinterpret_cast<u32x4_any*>(to) = Elem<T>::pack(x);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < V; ++i)
            if (i < count) to[i] = Elem<T>::from_f32(x[i]);
    }
}

// Partners i of a lane's pairs in its two vectors: (0, i), (1, i), or neighbours.
template <bool INTERLEAVED, int V> struct Pair {
    __device__ static constexpr int vec(int i, int side) { return INTERLEAVED ? (2 * i + side) / V : side; }
    __device__ static constexpr int element(int i, int side) { return INTERLEAVED ? (2 * i + side) % V : i; }
};

template <bool INTERLEAVED, int V, bool BACK>
__device__ __forceinline__ void rotate(float (&x)[2][V], const Slot& t, const float (&cos)[V], const float (&sin)[V])
{
    using P = Pair<INTERLEAVED, V>;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float &a = x[P::vec(i, 0)][P::element(i, 0)], &b = x[P::vec(i, 1)][P::element(i, 1)];
        const float s = BACK ? -sin[i] : sin[i];
        const float turned_a = __builtin_fmaf(a, cos[i], -(b * s)), turned_b = __builtin_fmaf(b, cos[i], a * s);
        a = t.pairs ? turned_a : a;
        b = t.pairs ? turned_b : b;
    }
}

// A token's row of both tables, this lane's pairs of it; NaN for a position outside them.
template <int V, bool WHOLE>
__device__ __forceinline__ void angles(const RotaryArgs& a, uint32_t token, const Slot& t, float (&cos)[V], float (&sin)[V])
{
    int64_t at = token;
    if (a.at) at = a.wide ? static_cast<const int64_t*>(a.at)[token] : static_cast<const int32_t*>(a.at)[token];
    const bool good = at >= 0 && static_cast<uint64_t>(at) < a.positions;
    const uint64_t row = (good ? static_cast<uint64_t>(at) : 0) * (a.rotated / 2) + t.pair;
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const uint32_t left = t.pairs > static_cast<uint32_t>(i) ? t.pairs - i : 0, count = left < 4 ? left : 4;
        float c[4] = {}, s[4] = {};
        // where every lane is whole, one whose elements do not turn has no pairs, else as many as elements in a vector
        if (a.positions && (!WHOLE || t.pairs)) {
            Elem<float>::unpack(load_some<float, WHOLE>(a.cos + row + i, count), c);
            Elem<float>::unpack(load_some<float, WHOLE>(a.sin + row + i, count), s);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cos[i + k] = good ? c[k] : NAN;
            sin[i + k] = good ? s[k] : NAN;
        }
    }
}

template <typename T>
__device__ __forceinline__ void weights(const void* weight, const Slot& t, float (&w)[2][Elem<T>::kCount])
{
    constexpr int V = Elem<T>::kCount;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (weight) {
            Elem<T>::unpack(load_some<T>(static_cast<const T*>(weight) + t.first[h], t.count[h]), w[h]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) w[h][i] = 1.0f;
        }
    }
}

template <int CONTROL> __device__ __forceinline__ float moved(float x)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CONTROL, 0xf, 0xf, true));
}

// The sum over a head's lanes, in each of them.  Up to 16 lanes the exchanges are operands of the sums.
__device__ __forceinline__ float head_sum(float x, uint32_t lanes)
{
    if (lanes > 1) x += moved<0xb1>(x);                  // lane ^ 1
    if (lanes > 2) x += moved<0x4e>(x);                  // lane ^ 2
    if (lanes > 4) x += moved<0x141>(x);                 // 7 - lane of eight
    if (lanes > 8) x += moved<0x140>(x);                 // 15 - lane of sixteen
    if (lanes > 16) x += __shfl_xor(x, 16);
    if (lanes > 32) x += __shfl_xor(x, 32);
    return x;
}

template <typename T> __device__ __forceinline__ T* head_at(const HeadRows& r, uint32_t token, uint32_t head)
{
    return reinterpret_cast<T*>(r.data + static_cast<uint64_t>(token) * r.row + static_cast<uint64_t>(head) * r.head);
}

// One wave takes U query heads, or key heads, of a token for each of its groups of lanes, all loads first.
// Bound by memory: 8192 tokens of 32 and 8 heads of 128 in bf16, 172 MB, take 32.6 us, 5.3 TB/s, where a copy of
// 2 GiB reaches 4.9; 37.0 with stores that stay in the caches, 1.5 more with U = 2.  With the attention that reads them next
// the stores past the caches gain for shorter batches and lose a little for longer ones: 1100 tokens in windows of 128
// 24.2 us and 27.0, 2048 28.4 and 29.7, 8192 94 and 95; causal, 2048 tokens 62 and 63, two times 2048 103.5 and 100.1.
template <typename T, bool INTERLEAVED, bool WHOLE, int U> __global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a)
{
    constexpr int V = Elem<T>::kCount;
    const uint32_t lane = threadIdx.x % kWave, groups = kWave / a.lanes;
    uint64_t item = blockIdx.x * 4ull + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const bool query = item < static_cast<uint64_t>(a.n) * a.chunks;
    if (!query) item -= static_cast<uint64_t>(a.n) * a.chunks;
    const uint32_t chunks = query ? a.chunks : a.kv_chunks, heads = query ? a.heads : a.kv_heads;
    if (item >= static_cast<uint64_t>(a.n) * chunks) return;
    const HeadRows from = query ? a.q : a.k, to = query ? a.q_out : a.k_out;
    const void* weight = query ? a.q_weight : a.k_weight;
    const uint32_t token = static_cast<uint32_t>(item / chunks);
    const uint32_t first = static_cast<uint32_t>(item % chunks) * groups * U + lane / a.lanes;
    const Slot t = slot_of<INTERLEAVED, V>(lane % a.lanes, a.dim, a.rotated);
    u32x4_t raw[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t head = first + u * groups;
        const bool there = head < heads;
        const T* x = head_at<T>(from, token, there ? head : 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            raw[u][h] = u32x4_t{0, 0, 0, 0};
            if (there) raw[u][h] = load_some<T, WHOLE>(x + t.first[h], t.count[h]);
        }
    }
    float cos[V], sin[V], w[2][V];
    angles<V, WHOLE>(a, token, t, cos, sin);
    weights<T>(weight, t, w);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t head = first + u * groups;
        float x[2][V];
#pragma unroll
        for (int h = 0; h < 2; ++h) Elem<T>::unpack(raw[u][h], x[h]);
        if (weight) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) sum = __builtin_fmaf(x[1][i], x[1][i], __builtin_fmaf(x[0][i], x[0][i], sum));
            sum = head_sum(sum, a.lanes);
            const float r = 1.0f / sqrtf(__builtin_fmaf(sum, a.per_dim, a.eps));
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < V; ++i) x[h][i] = x[h][i] * r * w[h][i];
        }
        rotate<INTERLEAVED, V, false>(x, t, cos, sin);
        if (head < heads) {
            T* out = head_at<T>(to, token, head);
#pragma unroll
            for (int h = 0; h < 2; ++h) store_some<T, WHOLE, (U > 1)>(out + t.first[h], t.count[h], x[h]);
        }
    }
}

// A wave goes over items like those above and keeps the sums for the weight in registers; a workgroup's are
// added in the order of its waves, the workgroups' by join_kernel.  The next item is on its way while one is
// computed.  8192 tokens of 32 and 8 heads of 128 in bf16, 257 MB: 53 us, 4.8 TB/s, and 5 for the join; four waves
// on a SIMD without the next item on its way took 100, branches between the loads 74.
template <typename T, bool INTERLEAVED, bool WHOLE, int U> __global__ __launch_bounds__(256, 2) void rotary_grad_kernel(RotaryArgs a)
{
    constexpr int V = Elem<T>::kCount;
    __shared__ float sums[4][kWave][2][V];
    const uint32_t lane = threadIdx.x % kWave, groups = kWave / a.lanes;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const bool query = blockIdx.x < a.workers;
    const uint32_t worker = query ? blockIdx.x : blockIdx.x - a.workers;
    const uint32_t workers = query ? a.workers : gridDim.x - a.workers;
    const uint32_t chunks = query ? a.chunks : a.kv_chunks, heads = query ? a.heads : a.kv_heads;
    const HeadRows from_g = query ? a.grad_q : a.grad_k, from_x = query ? a.q : a.k, to = query ? a.q_out : a.k_out;
    const void* weight = query ? a.q_weight : a.k_weight;
    const Slot t = slot_of<INTERLEAVED, V>(lane % a.lanes, a.dim, a.rotated);
    float w[2][V], dw[2][V] = {};
    weights<T>(weight, t, w);
    const uint64_t items = static_cast<uint64_t>(a.n) * chunks, stride = workers * 4ull;
    struct Item {
        u32x4_t g[U][2], x[U][2];
        float cos[V], sin[V];
        uint32_t token, first;
    };
    const auto load = [&](Item& d, uint64_t item) {
        d.token = static_cast<uint32_t>(item / chunks);
        d.first = static_cast<uint32_t>(item % chunks) * groups * U + lane / a.lanes;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t head = d.first + u * groups;
            const bool there = head < heads;
            const T* g = head_at<T>(from_g, d.token, there ? head : 0);
            const T* x = head_at<T>(from_x, d.token, there ? head : 0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                d.g[u][h] = d.x[u][h] = u32x4_t{0, 0, 0, 0};
                if (there) d.g[u][h] = load_some<T, WHOLE>(g + t.first[h], t.count[h]);
                if (there && weight) d.x[u][h] = load_some<T, WHOLE>(x + t.first[h], t.count[h]);
            }
        }
        angles<V, WHOLE>(a, d.token, t, d.cos, d.sin);
    };
    const auto compute = [&](const Item& d) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t head = d.first + u * groups;
            float g[2][V];
#pragma unroll
            for (int h = 0; h < 2; ++h) Elem<T>::unpack(d.g[u][h], g[h]);
            rotate<INTERLEAVED, V, true>(g, t, d.cos, d.sin);
            if (weight) {
                float x[2][V], squares = 0.0f, products = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    Elem<T>::unpack(d.x[u][h], x[h]);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        squares = __builtin_fmaf(x[h][i], x[h][i], squares);
                        products = __builtin_fmaf(g[h][i] * w[h][i], x[h][i], products);
                    }
                }
                squares = head_sum(squares, a.lanes);
                products = head_sum(products, a.lanes);
                // a head that is not there is all zeros, and adds none, whatever eps is
                const float r = head < heads ? 1.0f / sqrtf(__builtin_fmaf(squares, a.per_dim, a.eps)) : 0.0f;
                const float mean = products * r * a.per_dim;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float unit = x[h][i] * r;
                        dw[h][i] = __builtin_fmaf(g[h][i], unit, dw[h][i]);
                        g[h][i] = r * __builtin_fmaf(-unit, mean, g[h][i] * w[h][i]);
                    }
            }
            if (head < heads) {
                T* out = head_at<T>(to, d.token, head);
#pragma unroll
                for (int h = 0; h < 2; ++h) store_some<T, WHOLE>(out + t.first[h], t.count[h], g[h]);
            }
        }
    };
    Item one, other;
    uint64_t item = worker * 4ull + wave;
    if (item < items) load(one, item);
    while (item < items) {
        if (item + stride < items) load(other, item + stride);
        compute(one);
        item += stride;
        if (item >= items) break;
        if (item + stride < items) load(one, item + stride);
        compute(other);
        item += stride;
    }
    if (!weight) return;
    for (uint32_t d = a.lanes; d < kWave; d <<= 1)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < V; ++i) dw[h][i] += __shfl_xor(dw[h][i], static_cast<int>(d));
    if (lane < a.lanes)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < V; ++i) sums[wave][lane][h][i] = dw[h][i];
    __syncthreads();
    if (threadIdx.x >= a.lanes) return;
    float* mine = a.partial + static_cast<uint64_t>(blockIdx.x) * a.dim;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (uint32_t i = 0; i < V; ++i)
            if (i < t.count[h])
                mine[t.first[h] + i] = (sums[0][lane][h][i] + sums[1][lane][h][i]) + (sums[2][lane][h][i] + sums[3][lane][h][i]);
}

struct JoinArgs {
    const float* partial;
    void* weight[2];
    uint32_t first[2], workers[2];  // of the workgroups with query heads, and with key heads
    uint32_t dim;
    int accumulate;
};

// Sixteen waves, 64 neighbouring sums of one weight to a workgroup: each takes a run of the workgroups' partial sums.
template <typename W> __global__ __launch_bounds__(1024) void join_kernel(JoinArgs a)
{
    __shared__ float sums[16][kWave];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t at = blockIdx.x * kWave + lane;
    W* to = static_cast<W*>(blockIdx.y ? a.weight[1] : a.weight[0]);
    if (!to) return;
    const uint32_t workers = blockIdx.y ? a.workers[1] : a.workers[0];
    const float* partial = a.partial + static_cast<uint64_t>(blockIdx.y ? a.first[1] : a.first[0]) * a.dim;
    const uint32_t run = ceil_div(workers, 16u), from = wave * run;
    const uint32_t end = from + run < workers ? from + run : workers;
    float sum = 0.0f;
    if (at < a.dim)
#pragma unroll 16
        for (uint32_t k = from; k < end; ++k) sum += partial[static_cast<uint64_t>(k) * a.dim + at];
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave > 0 || at >= a.dim) return;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += sums[k][lane];
    to[at] = Elem<W>::from_f32(a.accumulate ? sum + Elem<W>::to_f32(to[at]) : sum);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint64_t kMostDim = 256;                       // 64 lanes of eight fp32
constexpr uint64_t kMostWorkers = 512;                   // workgroups with partial sums: two to a compute unit

bool reachable(const void* p) { return !p || la_ptr::device_accessible(p); }

bool bad(const la_heads_t& h, int dtype)
{
    return !h.data || reinterpret_cast<uintptr_t>(h.data) % static_cast<uintptr_t>(dtype_bytes(dtype));
}

bool bad(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(dtype_bytes(dtype)); }

HeadRows rows_of(const la_heads_t& h, int dtype)
{
    const uint64_t size = static_cast<uint64_t>(dtype_bytes(dtype));
    return {static_cast<char*>(const_cast<void*>(h.data)), h.row_stride * size, h.head_stride * size};
}

int check_call(const la_rotary_t* call)
{
    if (!call) return LA_EINVAL;
    const la_rotary_t& c = *call;
    if (!is_float_dtype(c.dtype) || (c.at && c.at_dtype != LA_I32 && c.at_dtype != LA_I64)) return LA_EDTYPE;
    constexpr uint64_t kMost = 1ull << 30;
    if (c.dim == 0 || c.dim > kMostDim || c.rotated > c.dim || c.rotated % 2 || c.n > kMost || c.heads > kMost ||
        c.kv_heads > kMost || (c.n > 0 && c.heads + c.kv_heads > kMost / c.n))
        return LA_EINVAL;
    if (c.n == 0 || c.heads + c.kv_heads == 0) return LA_OK;
    if ((c.heads && bad(c.q_out, c.dtype)) || (c.kv_heads && bad(c.k_out, c.dtype)) || bad(c.q_weight, c.dtype) ||
        bad(c.k_weight, c.dtype) || (c.at && bad(c.at, c.at_dtype)) || bad(c.cos, LA_F32) || bad(c.sin, LA_F32) ||
        (c.rotated && (!c.cos || !c.sin)))
        return LA_EINVAL;
    return LA_OK;
}

int check_reach(const la_rotary_t& c)
{
    const void* all[] = {c.q.data, c.k.data, c.q_out.data, c.k_out.data, c.q_weight, c.k_weight, c.cos, c.sin, c.at};
    for (const void* p : all)
        if (!reachable(p)) return LA_EFAULT;
    return LA_OK;
}

la_memory::Place place_of(const la_rotary_t& c, const la_heads_t& h, uint64_t heads)
{
    const uint64_t size = static_cast<uint64_t>(dtype_bytes(c.dtype));
    return {reinterpret_cast<uintptr_t>(h.data), c.dim * size, {c.n, heads, 1}, {h.row_stride * size, h.head_stride * size, 0}};
}

// Heads are read and written by waves of their own, in no order: a result lies exactly where heads of its own kind are read,
// each read whole before it is written, or where nothing is read; and no two results share memory.  The scales'
// gradients are written after everything is read.
bool results_apart(const la_rotary_t& c, bool grad)
{
    using la_memory::flat;
    using la_memory::Place;
    using la_memory::shared;
    const uint64_t size = static_cast<uint64_t>(dtype_bytes(c.dtype)), table = c.positions * (c.rotated / 2) * sizeof(float);
    const Place outs[] = {place_of(c, c.q_out, c.heads), place_of(c, c.k_out, c.kv_heads)};
    const bool x_read[] = {!grad || c.q_weight, !grad || c.k_weight};
    const Place none{}, heads[] = {x_read[0] ? place_of(c, c.q, c.heads) : none, x_read[1] ? place_of(c, c.k, c.kv_heads) : none,
                                   grad ? place_of(c, c.grad_q, c.heads) : none, grad ? place_of(c, c.grad_k, c.kv_heads) : none};
    const Place others[] = {flat(c.q_weight, c.dim * size), flat(c.k_weight, c.dim * size), flat(c.cos, table), flat(c.sin, table),
                            flat(c.at, c.at ? c.n * static_cast<uint64_t>(dtype_bytes(c.at_dtype)) : 0)};
    for (int out = 0; out < 2; ++out) {
        for (int k = 0; k < 4; ++k)
            if (shared(outs[out], heads[k]) && !(k % 2 == out && same(outs[out], heads[k]))) return false;
        for (const Place& other : others)
            if (shared(outs[out], other)) return false;
    }
    if (shared(outs[0], outs[1])) return false;
    if (!grad) return true;
    const uint64_t bytes = c.dim * static_cast<uint64_t>(dtype_bytes(c.weight_grad_dtype));
    const Place scales[] = {c.q_weight ? flat(c.grad_q_weight, bytes) : none, c.k_weight ? flat(c.grad_k_weight, bytes) : none};
    for (const Place& of : scales)
        if (shared(of, outs[0]) || shared(of, outs[1])) return false;
    return !shared(scales[0], scales[1]);
}

RotaryArgs args_of(const la_rotary_t& c)
{
    RotaryArgs a{};
    a.q = rows_of(c.q, c.dtype);
    a.k = rows_of(c.k, c.dtype);
    a.q_out = rows_of(c.q_out, c.dtype);
    a.k_out = rows_of(c.k_out, c.dtype);
    a.q_weight = c.q_weight;
    a.k_weight = c.k_weight;
    a.cos = c.cos;
    a.sin = c.sin;
    a.at = c.at;
    a.wide = c.at_dtype == LA_I64;
    a.positions = c.positions;
    a.n = static_cast<uint32_t>(c.n);
    a.heads = static_cast<uint32_t>(c.heads);
    a.kv_heads = static_cast<uint32_t>(c.kv_heads);
    a.dim = static_cast<uint32_t>(c.dim);
    a.rotated = static_cast<uint32_t>(c.rotated);
    a.eps = c.eps;
    a.per_dim = 1.0f / static_cast<float>(c.dim);
    a.lanes = 1;
    while (a.lanes < slots(a.dim, a.rotated, 16 / dtype_bytes(c.dtype))) a.lanes *= 2;
    return a;
}

// Heads that a group of lanes takes at a time: up to `most`, as even as the token's query heads allow; one
// where there are too few tokens to fill the card otherwise.
uint32_t heads_at_a_time(RotaryArgs& a, uint32_t most)
{
    const uint32_t groups = kWave / a.lanes, each = std::max(1u, ceil_div(a.heads, groups));
    uint32_t u = ceil_div(each, ceil_div(each, most));
    if (static_cast<uint64_t>(a.n) * each <= 4096) u = 1;
    a.chunks = ceil_div(a.heads, groups * u);
    a.kv_chunks = ceil_div(a.kv_heads, groups * u);
    return u;
}

template <typename T, bool INTERLEAVED, bool WHOLE> int forward(RotaryArgs& a, hipStream_t st)
{
    const uint32_t u = heads_at_a_time(a, 4);
    const dim3 grid(static_cast<uint32_t>(ceil_div(static_cast<uint64_t>(a.n) * (a.chunks + a.kv_chunks), 4ull)));
    switch (u) {
    case 1: return launch(rotary_kernel<T, INTERLEAVED, WHOLE, 1>, grid, dim3(256), st, a);
    case 2: return launch(rotary_kernel<T, INTERLEAVED, WHOLE, 2>, grid, dim3(256), st, a);
    case 3: return launch(rotary_kernel<T, INTERLEAVED, WHOLE, 3>, grid, dim3(256), st, a);
    default: return launch(rotary_kernel<T, INTERLEAVED, WHOLE, 4>, grid, dim3(256), st, a);
    }
}

// Whether all lanes have two whole vectors.
bool whole(const RotaryArgs& a, uint32_t v)
{
    return a.rotated / 2 % v == 0 && (a.dim - a.rotated) % (2 * v) == 0 && slots(a.dim, a.rotated, v) == a.lanes;
}

template <typename T> int forward(RotaryArgs& a, bool interleaved, hipStream_t st)
{
    if (whole(a, Elem<T>::kCount)) return interleaved ? forward<T, true, true>(a, st) : forward<T, false, true>(a, st);
    return interleaved ? forward<T, true, false>(a, st) : forward<T, false, false>(a, st);
}

// Workgroups of a gradient's launch: a.workers for the query heads, those returned for the key heads; in proportion to
// their items, and at least one where there are such heads.
uint32_t share_out(RotaryArgs& a)
{
    const uint64_t q = ceil_div(static_cast<uint64_t>(a.n) * a.chunks, 4ull);
    const uint64_t k = ceil_div(static_cast<uint64_t>(a.n) * a.kv_chunks, 4ull);
    const uint64_t of_k = a.kv_chunks ? kMostWorkers * a.kv_chunks / (a.chunks + a.kv_chunks) : 0;
    const uint64_t most_k = std::max<uint64_t>(1, std::min(of_k, kMostWorkers - 1));
    a.workers = static_cast<uint32_t>(std::min(q, kMostWorkers - most_k));
    return static_cast<uint32_t>(std::min(k, most_k));
}

template <typename T, bool INTERLEAVED, bool WHOLE>
int backward(RotaryArgs& a, uint32_t u, uint32_t kv_workers, hipStream_t st)
{
    const dim3 grid(a.workers + kv_workers);
    return u == 1 ? launch(rotary_grad_kernel<T, INTERLEAVED, WHOLE, 1>, grid, dim3(256), st, a)
                  : launch(rotary_grad_kernel<T, INTERLEAVED, WHOLE, 2>, grid, dim3(256), st, a);
}

template <typename T> int backward(RotaryArgs& a, bool interleaved, uint32_t u, uint32_t kv_workers, hipStream_t st)
{
    if (whole(a, Elem<T>::kCount))
        return interleaved ? backward<T, true, true>(a, u, kv_workers, st) : backward<T, false, true>(a, u, kv_workers, st);
    return interleaved ? backward<T, true, false>(a, u, kv_workers, st) : backward<T, false, false>(a, u, kv_workers, st);
}

}  // namespace

extern "C" {

int la_qk_norm_rotary(const la_rotary_t* call, la_stream_t stream)
{
    int rc = check_call(call);
    if (rc != LA_OK) return rc;
    const la_rotary_t& c = *call;
    if (c.n == 0 || c.heads + c.kv_heads == 0) return LA_OK;
    if ((c.heads && bad(c.q, c.dtype)) || (c.kv_heads && bad(c.k, c.dtype))) return LA_EINVAL;
    rc = check_reach(c);
    if (rc == LA_OK && !results_apart(c, false)) rc = LA_EINVAL;
    if (rc != LA_OK) return rc;
    RotaryArgs a = args_of(c);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (c.dtype == LA_F32) return forward<float>(a, c.interleaved != 0, st);
    return c.dtype == LA_BF16 ? forward<__bf16>(a, c.interleaved != 0, st) : forward<_Float16>(a, c.interleaved != 0, st);
}

uint64_t la_qk_norm_rotary_grad_workspace(const la_rotary_t* call)
{
    if (!call || call->dim > kMostDim || !(call->q_weight || call->k_weight)) return 0;
    return kMostWorkers * call->dim * sizeof(float);
}

int la_qk_norm_rotary_grad(const la_rotary_t* call, void* workspace, uint64_t workspace_bytes, la_stream_t stream)
{
    int rc = check_call(call);
    if (rc != LA_OK) return rc;
    const la_rotary_t& c = *call;
    const bool normed = c.q_weight || c.k_weight;
    if (normed && c.weight_grad_dtype != c.dtype && c.weight_grad_dtype != LA_F32) return LA_EDTYPE;
    if (normed && ((c.q_weight && (!c.grad_q_weight || bad(c.grad_q_weight, c.weight_grad_dtype))) ||
                   (c.k_weight && (!c.grad_k_weight || bad(c.grad_k_weight, c.weight_grad_dtype)))))
        return LA_EINVAL;
    const bool any = c.n > 0 && c.heads + c.kv_heads > 0;
    if (any && ((c.heads && (bad(c.grad_q, c.dtype) || (c.q_weight && bad(c.q, c.dtype)))) ||
                (c.kv_heads && (bad(c.grad_k, c.dtype) || (c.k_weight && bad(c.k, c.dtype))))))
        return LA_EINVAL;
    rc = check_workspace(workspace, workspace_bytes, la_qk_norm_rotary_grad_workspace(call), 16);
    if (rc != LA_OK) return rc;
    if (any) rc = check_reach(c);
    if (rc == LA_OK && (!reachable(c.grad_q_weight) || !reachable(c.grad_k_weight) || (normed && !reachable(workspace)) ||
                        (any && (!reachable(c.grad_q.data) || !reachable(c.grad_k.data)))))
        rc = LA_EFAULT;
    if (rc == LA_OK && !results_apart(c, true)) rc = LA_EINVAL;
    if (rc != LA_OK) return rc;
    RotaryArgs a = args_of(c);
    a.grad_q = rows_of(c.grad_q, c.dtype);
    a.grad_k = rows_of(c.grad_k, c.dtype);
    a.partial = normed ? static_cast<float*>(workspace) : nullptr;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    uint32_t kv_workers = 0;
    if (any) {
        const uint32_t u = heads_at_a_time(a, 2);
        kv_workers = share_out(a);
        const bool interleaved = c.interleaved != 0;
        rc = c.dtype == LA_F32    ? backward<float>(a, interleaved, u, kv_workers, st)
             : c.dtype == LA_BF16 ? backward<__bf16>(a, interleaved, u, kv_workers, st)
                                  : backward<_Float16>(a, interleaved, u, kv_workers, st);
        if (rc != LA_OK) return rc;
    }
    if (!normed) return LA_OK;
    const JoinArgs j{a.partial, {c.q_weight ? c.grad_q_weight : nullptr, c.k_weight ? c.grad_k_weight : nullptr},
                     {0, a.workers}, {a.workers, kv_workers}, a.dim, c.accumulate};
    const dim3 grid(ceil_div(a.dim, kWave), 2);
    return c.weight_grad_dtype == LA_F32    ? launch(join_kernel<float>, grid, dim3(1024), st, j)
           : c.weight_grad_dtype == LA_BF16 ? launch(join_kernel<__bf16>, grid, dim3(1024), st, j)
                                            : launch(join_kernel<_Float16>, grid, dim3(1024), st, j);
}

}  // extern "C"
