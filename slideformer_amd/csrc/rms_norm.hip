// slideformer_amd: the root-mean-square norm with the residual's addition, its
// 8-bit form and its gradient (gfx950, wave64).
//
// Forward, per row: z = x + residual, r = 1 / sqrt(mean(z^2) + eps), y = z r w.
// Gradient: with u = z r and g = dy w, dz = r (g - u mean(g u)) + dz', where dz' is
// the gradient that reaches z past the norm; dw = sum over rows of dy u.
//
// All of it is bound by memory: a row is read once, kept in registers as fp32
// while its sum is formed, and written once.
#include "ops_common.h"

namespace {

constexpr int kWave = 64;

// The sum of x over the THREADS threads that share a row (one wave, or a whole
// workgroup through `lds`).
template <int THREADS> __device__ __forceinline__ float row_sum(float x, float* lds)
{
    x = wave_sum(x);
    if constexpr (THREADS > kWave) {
        __syncthreads();                                    // the previous use of lds is over
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) x += lds[w];
    }
    return x;
}

template <int THREADS> __device__ __forceinline__ uint32_t row_max(uint32_t x, float* lds)
{
    x = wave_max_u32(x);
    if constexpr (THREADS > kWave) {
        __syncthreads();
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = __uint_as_float(x);
        __syncthreads();
        x = 0;
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) {
            const uint32_t y = __float_as_uint(lds[w]);
            x = y > x ? y : x;
        }
    }
    return x;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
struct NormArgs {
    const void* x;
    const void* residual;
    const void* weight;
    void* summed;
    void* out;
    float* scales;
    float* rstd;
    uint64_t n, x_stride, residual_stride, summed_stride, out_stride;
    uint32_t hidden;
    float eps;
};

struct Int8Out {
    static constexpr float kTop = 127.0f;
    template <int E> __device__ static void store(void* row, uint32_t vec, uint32_t hidden, const float (&y)[E])
    {
        int8_t* to = static_cast<int8_t*>(row) + vec * E;
        uint32_t words[E / 4];
#pragma unroll
        for (int w = 0; w < E / 4; ++w) {
            words[w] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float q = fminf(fmaxf(__builtin_rintf(y[4 * w + b]), -127.0f), 127.0f);
                words[w] |= (static_cast<uint32_t>(static_cast<int32_t>(q)) & 0xffu) << (8 * b);
            }
        }
        store_words<E>(to, vec, hidden, words);
    }
    template <int E, typename P>
    __device__ static void store_words(P* to, uint32_t vec, uint32_t hidden, const uint32_t (&words)[E / 4])
    {
        if (vec * E + E <= hidden) {
            typedef uint32_t any __attribute__((aligned(1)));
#pragma unroll
            for (int w = 0; w < E / 4; ++w) reinterpret_cast<any*>(to)[w] = words[w];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (vec * E + e < hidden) to[e] = static_cast<P>(words[e / 4] >> (8 * (e % 4)));
        }
    }
};

// E4M3 without infinities (largest value 448), rounded by the hardware's conversion
struct Fp8Out {
    static constexpr float kTop = 448.0f;
    template <int E> __device__ static void store(void* row, uint32_t vec, uint32_t hidden, const float (&y)[E])
    {
        uint8_t* to = static_cast<uint8_t*>(row) + vec * E;
        uint32_t words[E / 4];
#pragma unroll
        for (int w = 0; w < E / 4; ++w) {
            float c[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) c[b] = fminf(fmaxf(y[4 * w + b], -448.0f), 448.0f);
            int word = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
            word = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], word, true);
            words[w] = static_cast<uint32_t>(word);
        }
        Int8Out::store_words<E>(to, vec, hidden, words);
    }
};

template <typename T> struct SameOut {
    static constexpr float kTop = 0.0f;                     // no scale
    template <int E> __device__ static void store(void* row, uint32_t vec, uint32_t hidden, const float (&y)[E])
    {
        store_vec<T, E>(static_cast<T*>(row), vec, hidden, y);
    }
};

template <typename T>
__device__ __forceinline__ void load_sum(const NormArgs& a, uint64_t row, uint32_t vec, float (&z)[Elem<T>::kCount])
{
    load_vec<T>(static_cast<const T*>(a.x) + row * a.x_stride, vec, a.hidden, z);
    if (a.residual) {
        float r[Elem<T>::kCount];
        load_vec<T>(static_cast<const T*>(a.residual) + row * a.residual_stride, vec, a.hidden, r);
#pragma unroll
        for (int e = 0; e < Elem<T>::kCount; ++e) z[e] += r[e];
    }
}

// The scale of a row whose largest |y| has these bits: 0 for a row of zeros,
// NaN for one with an infinity or NaN (whose bits are above any finite one's).
__device__ __forceinline__ float row_scale(uint32_t top_bits, float steps)
{
    return top_bits >= 0x7f800000u ? __builtin_nanf("") : __uint_as_float(top_bits) / steps;
}

template <typename Out, int E> __device__ __forceinline__ void to_steps(float scale, float (&y)[E])
{
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = scale > 0.0f ? y[e] / scale : 0.0f;
}

// THREADS threads hold a row of at most THREADS * VPT vectors in registers: x, the
// residual and the scales are all on their way before the row is summed, and nothing is
// read twice.  8192 x 4096 bf16: 43.4 us, 6.2 TB/s; one row 2.9 us; 1037 x 5120 to
// int8 15.3 us, four rows a compute unit at once and two reductions long.
template <typename T, typename Out, int THREADS, int VPT>
__global__ __launch_bounds__(256) void norm_kernel(NormArgs a)
{
    constexpr int E = Elem<T>::kCount;
    constexpr int ROWS = 256 / THREADS;
    __shared__ float lds[4];
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * ROWS + threadIdx.x / THREADS;
    if (row >= a.n) return;                                 // whole waves; a workgroup of one row never gets here
    const uint32_t tid = threadIdx.x % THREADS;
    float z[VPT][E];
    float square = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) load_sum<T>(a, row, k * THREADS + tid, z[k]);
    u32x4_t weight[VPT];                                    // on its way while the row is summed
#pragma unroll
    for (int k = 0; k < VPT; ++k)
        weight[k] = load_raw<T>(static_cast<const T*>(a.weight), k * THREADS + tid, a.hidden);
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) square = __builtin_fmaf(z[k][e], z[k][e], square);
    if (a.summed)
#pragma unroll
        for (int k = 0; k < VPT; ++k)
            store_vec<T, E>(static_cast<T*>(a.summed) + row * a.summed_stride, k * THREADS + tid, a.hidden, z[k]);
    const float r = 1.0f / sqrtf(row_sum<THREADS>(square, lds) / static_cast<float>(a.hidden) + a.eps);
    if (a.rstd && tid == 0) a.rstd[row] = r;
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        float w[E];
        Elem<T>::unpack(weight[k], w);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            z[k][e] = z[k][e] * r * w[e];
            if constexpr (Out::kTop > 0.0f) {
                const uint32_t bits = __float_as_uint(z[k][e]) & 0x7fffffffu;
                top = bits > top ? bits : top;
            }
        }
    }
    float scale = 0.0f;
    if constexpr (Out::kTop > 0.0f) {
        scale = row_scale(row_max<THREADS>(top, lds), Out::kTop);
        if (tid == 0) a.scales[row] = scale;
    }
    char* out = static_cast<char*>(a.out) + row * a.out_stride * (Out::kTop > 0.0f ? 1 : sizeof(T));
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        if constexpr (Out::kTop > 0.0f) to_steps<Out, E>(scale, z[k]);
        Out::template store<E>(out, k * THREADS + tid, a.hidden, z[k]);
    }
}

// Rows too long for registers: z is formed again from x and the residual in
// each pass, out of the caches.
template <typename T, typename Out> __global__ __launch_bounds__(256) void long_norm_kernel(NormArgs a)
{
    constexpr int E = Elem<T>::kCount;
    __shared__ float lds[4];
    const uint64_t row = blockIdx.x;
    const uint32_t vecs = ceil_div(a.hidden, static_cast<uint32_t>(E));
    float square = 0.0f;
    for (uint32_t vec = threadIdx.x; vec < vecs; vec += 256) {
        float z[E];
        load_sum<T>(a, row, vec, z);
#pragma unroll
        for (int e = 0; e < E; ++e) square = __builtin_fmaf(z[e], z[e], square);
    }
    const float r = 1.0f / sqrtf(row_sum<256>(square, lds) / static_cast<float>(a.hidden) + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = r;
    const auto normed = [&](uint32_t vec, float (&z)[E]) {
        float w[E];
        load_sum<T>(a, row, vec, z);
        load_vec<T>(static_cast<const T*>(a.weight), vec, a.hidden, w);
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = z[e] * r * w[e];
    };
    float scale = 0.0f;
    if constexpr (Out::kTop > 0.0f) {
        uint32_t top = 0;
        for (uint32_t vec = threadIdx.x; vec < vecs; vec += 256) {
            float y[E];
            normed(vec, y);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t bits = __float_as_uint(y[e]) & 0x7fffffffu;
                top = bits > top ? bits : top;
            }
        }
        scale = row_scale(row_max<256>(top, lds), Out::kTop);
        if (threadIdx.x == 0) a.scales[row] = scale;
    }
    char* out = static_cast<char*>(a.out) + row * a.out_stride * (Out::kTop > 0.0f ? 1 : sizeof(T));
    for (uint32_t vec = threadIdx.x; vec < vecs; vec += 256) {
        float y[E];
        normed(vec, y);
        if (a.summed) {
            float z[E];
            load_sum<T>(a, row, vec, z);
            store_vec<T, E>(static_cast<T*>(a.summed) + row * a.summed_stride, vec, a.hidden, z);
        }
        if constexpr (Out::kTop > 0.0f) to_steps<Out, E>(scale, y);
        Out::template store<E>(out, vec, a.hidden, y);
    }
}

template <typename T, typename Out> int norm_rows(const NormArgs& a, hipStream_t st)
{
    const uint32_t vecs = ceil_div(a.hidden, static_cast<uint32_t>(Elem<T>::kCount));
    // One wave a row up to two vectors per lane, a workgroup beyond.  8192 rows: of 512
    // a wave 8.8 us, a workgroup 14.2; of 1024 12.3 and 14.9, of 1536 (four vectors
    // in a wave) 19.3 and 17.8.
    if (vecs <= 64) return launch(norm_kernel<T, Out, 64, 1>, dim3(ceil_div(a.n, 4)), dim3(256), st, a);
    if (vecs <= 128) return launch(norm_kernel<T, Out, 64, 2>, dim3(ceil_div(a.n, 4)), dim3(256), st, a);
    if (vecs <= 256) return launch(norm_kernel<T, Out, 256, 1>, dim3(a.n), dim3(256), st, a);
    if (vecs <= 512) return launch(norm_kernel<T, Out, 256, 2>, dim3(a.n), dim3(256), st, a);
    if (vecs <= 1024) return launch(norm_kernel<T, Out, 256, 4>, dim3(a.n), dim3(256), st, a);
    if (vecs <= 2048) return launch(norm_kernel<T, Out, 256, 8>, dim3(a.n), dim3(256), st, a);
    return launch(long_norm_kernel<T, Out>, dim3(a.n), dim3(256), st, a);
}

template <typename T> int norm(int out_dtype, const NormArgs& a, hipStream_t st)
{
    if (out_dtype == LA_I8) return norm_rows<T, Int8Out>(a, st);
    if (out_dtype == LA_F8E4M3) return norm_rows<T, Fp8Out>(a, st);
    return norm_rows<T, SameOut<T>>(a, st);
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------
struct NormGradArgs {
    const void* grad_out;
    const void* summed;
    const float* rstd;
    const void* weight;
    const void* grad_summed;
    void* grad_x;
    float* partial;                 // [workers][hidden], null without a weight gradient
    uint64_t n, grad_out_stride, summed_stride, grad_summed_stride, grad_x_stride;
    uint32_t hidden, workers;
};

// A worker (a wave, or a workgroup) takes every `workers`-th row; its share of
// dw stays in registers until its last row.  8192 x 4096 bf16: 46.3 us, 5.8 TB/s.
template <typename T, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_grad_kernel(NormGradArgs a)
{
    constexpr int E = Elem<T>::kCount;
    constexpr int WORKERS = THREADS < 256 ? 256 / THREADS : 1;
    constexpr bool kLean = THREADS == 1024;                 // 128 registers a thread: less is kept and fetched ahead
    __shared__ float lds[THREADS / kWave];
    const uint32_t worker = blockIdx.x * WORKERS + threadIdx.x / THREADS;
    if (worker >= a.workers) return;
    const uint32_t tid = threadIdx.x % THREADS;
    u32x4_t weight[VPT];                                    // kept as it lies in memory: half the registers
    float dw[VPT][E];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        if constexpr (!kLean)
            weight[k] = load_raw<T>(static_cast<const T*>(a.weight), k * THREADS + tid, a.hidden);
#pragma unroll
        for (int e = 0; e < E; ++e) dw[k][e] = 0.0f;
    }
    // a row's three inputs as they lie in memory, loaded while the row before is computed
    u32x4_t next[3][VPT];
    const auto fetch = [&](uint64_t row) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const uint32_t vec = k * THREADS + tid;
            next[0][k] = load_raw<T>(static_cast<const T*>(a.grad_out) + row * a.grad_out_stride, vec, a.hidden);
            next[1][k] = load_raw<T>(static_cast<const T*>(a.summed) + row * a.summed_stride, vec, a.hidden);
            if constexpr (!kLean)
                next[2][k] = a.grad_summed ? load_raw<T>(static_cast<const T*>(a.grad_summed) +
                                                         row * a.grad_summed_stride, vec, a.hidden)
                                       : u32x4_t{0, 0, 0, 0};
        }
    };
    fetch(worker);
    for (uint64_t row = worker; row < a.n; row += a.workers) {
        float u[VPT][E], g[VPT][E];
        u32x4_t through[VPT];
        const float r = a.rstd[row];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            Elem<T>::unpack(next[0][k], g[k]);
            Elem<T>::unpack(next[1][k], u[k]);
            through[k] = next[2][k];
            if constexpr (kLean) {
                through[k] = a.grad_summed ? load_raw<T>(static_cast<const T*>(a.grad_summed) +
                                                             row * a.grad_summed_stride, k * THREADS + tid, a.hidden)
                                           : u32x4_t{0, 0, 0, 0};
                weight[k] = load_raw<T>(static_cast<const T*>(a.weight), k * THREADS + tid, a.hidden);
            }
        }
        if (row + a.workers < a.n) fetch(row + a.workers);
        float inner = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float w[E];
            Elem<T>::unpack(weight[k], w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                u[k][e] *= r;
                dw[k][e] = __builtin_fmaf(g[k][e], u[k][e], dw[k][e]);
                g[k][e] *= w[e];
                inner = __builtin_fmaf(g[k][e], u[k][e], inner);
            }
        }
        inner = row_sum<THREADS>(inner, lds) / static_cast<float>(a.hidden);
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float past[E] = {};
            if (a.grad_summed) Elem<T>::unpack(through[k], past);
#pragma unroll
            for (int e = 0; e < E; ++e) g[k][e] = __builtin_fmaf(g[k][e] - u[k][e] * inner, r, past[e]);
            store_vec<T, E>(static_cast<T*>(a.grad_x) + row * a.grad_x_stride, k * THREADS + tid, a.hidden, g[k]);
        }
    }
    if (a.partial)
#pragma unroll
        for (int k = 0; k < VPT; ++k)
            store_vec<float, E>(a.partial + static_cast<uint64_t>(worker) * a.hidden, k * THREADS + tid, a.hidden,
                                dw[k]);
}

// Rows too long for registers: two passes over the row, dw in the workspace,
// where each column belongs to one thread.
template <typename T> __global__ __launch_bounds__(256) void long_norm_grad_kernel(NormGradArgs a)
{
    constexpr int E = Elem<T>::kCount;
    __shared__ float lds[4];
    const uint32_t vecs = ceil_div(a.hidden, static_cast<uint32_t>(E));
    float* mine = a.partial ? a.partial + static_cast<uint64_t>(blockIdx.x) * a.hidden : nullptr;
    for (uint64_t row = blockIdx.x; row < a.n; row += a.workers) {
        const float r = a.rstd[row];
        const T* grad_out = static_cast<const T*>(a.grad_out) + row * a.grad_out_stride;
        const T* summed = static_cast<const T*>(a.summed) + row * a.summed_stride;
        float inner = 0.0f;
        for (uint32_t vec = threadIdx.x; vec < vecs; vec += 256) {
            float g[E], u[E], w[E];
            load_vec<T>(grad_out, vec, a.hidden, g);
            load_vec<T>(summed, vec, a.hidden, u);
            load_vec<T>(static_cast<const T*>(a.weight), vec, a.hidden, w);
#pragma unroll
            for (int e = 0; e < E; ++e) inner = __builtin_fmaf(g[e] * w[e], u[e] * r, inner);
        }
        inner = row_sum<256>(inner, lds) / static_cast<float>(a.hidden);
        for (uint32_t vec = threadIdx.x; vec < vecs; vec += 256) {
            float g[E], u[E], w[E], past[E] = {}, dw[E] = {};
            load_vec<T>(grad_out, vec, a.hidden, g);
            load_vec<T>(summed, vec, a.hidden, u);
            load_vec<T>(static_cast<const T*>(a.weight), vec, a.hidden, w);
            if (a.grad_summed)
                load_vec<T>(static_cast<const T*>(a.grad_summed) + row * a.grad_summed_stride, vec, a.hidden, past);
            if (mine && row != blockIdx.x)
#pragma unroll
                for (int e = 0; e < E; ++e) dw[e] = vec * E + e < a.hidden ? mine[vec * E + e] : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                u[e] *= r;
                dw[e] = __builtin_fmaf(g[e], u[e], dw[e]);
                g[e] = __builtin_fmaf(g[e] * w[e] - u[e] * inner, r, past[e]);
            }
            store_vec<T, E>(static_cast<T*>(a.grad_x) + row * a.grad_x_stride, vec, a.hidden, g);
            if (mine) store_vec<float, E>(mine, vec, a.hidden, dw);
        }
    }
}

// dw: the workers' shares of a column, 16 interleaved sums added in order.  512
// shares of 4096 columns: 4.7 us.
template <typename W>
__global__ __launch_bounds__(1024) void join_weight_grad_kernel(const float* partial, uint32_t workers,
                                                                uint32_t hidden, W* grad_weight, int accumulate)
{
    __shared__ float lds[16][kWave];
    const uint32_t column = blockIdx.x * kWave + threadIdx.x % kWave;
    const uint32_t part = threadIdx.x / kWave;
    float sum = 0.0f;
    if (column < hidden)
#pragma unroll 8
        for (uint32_t k = part; k < workers; k += 16) sum += partial[static_cast<uint64_t>(k) * hidden + column];
    lds[part][threadIdx.x % kWave] = sum;
    __syncthreads();
    if (part == 0 && column < hidden) {
#pragma unroll
        for (int k = 1; k < 16; ++k) sum += lds[k][threadIdx.x];
        if (accumulate) sum += Elem<W>::to_f32(grad_weight[column]);
        grad_weight[column] = Elem<W>::from_f32(sum);
    }
}

// Workers that share the rows out, and the weight gradient's partials.
// A worker prefetches its next row, so few are enough to keep memory busy, and each
// costs a row of partials.  8192 rows: of 4096 (a workgroup each) 512 workers 53 us,
// 1024 62 us, without the prefetch 82 us; of 512 (a wave each) 1024 16 us, 512 20 us.
constexpr uint64_t kWaveWorkers = 1024;
constexpr uint64_t kGroupWorkers = 512;

uint64_t most_workers(uint64_t n) { return n < kWaveWorkers ? n : kWaveWorkers; }

template <typename T> int norm_grad_rows(NormGradArgs& a, hipStream_t st)
{
    const uint32_t vecs = ceil_div(a.hidden, static_cast<uint32_t>(Elem<T>::kCount));
    const uint64_t most = vecs <= 128 ? kWaveWorkers : kGroupWorkers;
    a.workers = static_cast<uint32_t>(a.n < most ? a.n : most);
    if (vecs <= 128 && vecs > 64)
        return launch(norm_grad_kernel<T, 64, 2>, dim3(ceil_div(a.workers, 4)), dim3(256), st, a);
    if (vecs <= 64) return launch(norm_grad_kernel<T, 64, 1>, dim3(ceil_div(a.workers, 4)), dim3(256), st, a);
    if (vecs <= 256) return launch(norm_grad_kernel<T, 256, 1>, dim3(a.workers), dim3(256), st, a);
    if (vecs <= 512) return launch(norm_grad_kernel<T, 256, 2>, dim3(a.workers), dim3(256), st, a);
    if (vecs <= 1024) return launch(norm_grad_kernel<T, 512, 2>, dim3(a.workers), dim3(512), st, a);
    if (vecs <= 2048) return launch(norm_grad_kernel<T, 1024, 2>, dim3(a.workers), dim3(1024), st, a);
    return launch(long_norm_grad_kernel<T>, dim3(a.workers), dim3(256), st, a);
}

template <typename W> int join_weight_grad(const NormGradArgs& a, void* grad_weight, int accumulate, hipStream_t st)
{
    return launch(join_weight_grad_kernel<W>, dim3(ceil_div(a.hidden, kWave)), dim3(1024), st, a.partial, a.workers,
                  a.hidden, static_cast<W*>(grad_weight), accumulate);
}

constexpr uint64_t kMaxHidden = 1ull << 24;
constexpr uint64_t kMaxRows = (1ull << 24) - 1;             // a launch has under 2^32 threads

bool reachable(const void* p) { return !p || la_ptr::device_accessible(p); }

}  // namespace

extern "C" {

int la_rms_norm(int dtype, const void* x, uint64_t x_stride, const void* residual, uint64_t residual_stride,
                const void* weight, uint64_t n, uint64_t hidden, float eps, void* summed, uint64_t summed_stride,
                int out_dtype, void* out, uint64_t out_stride, float* scales, float* rstd, la_stream_t stream)
{
    if (!is_float_dtype(dtype)) return LA_EDTYPE;
    const bool eight = out_dtype == LA_I8 || out_dtype == LA_F8E4M3;
    if (!eight && out_dtype != dtype) return LA_EDTYPE;
    if (n == 0 || hidden == 0) return LA_OK;
    if (n > kMaxRows || hidden > kMaxHidden) return LA_EINVAL;
    int rc = check_matrix(x, dtype, hidden, x_stride);
    if (rc == LA_OK && residual) rc = check_matrix(residual, dtype, hidden, residual_stride);
    if (rc == LA_OK) rc = check_matrix(weight, dtype, hidden, hidden);
    if (rc == LA_OK && summed) rc = check_matrix(summed, dtype, hidden, summed_stride);
    if (rc == LA_OK) rc = check_matrix(out, out_dtype, hidden, out_stride);
    if (rc == LA_OK && eight) rc = check_matrix(scales, LA_F32, 1, 1);
    if (rc == LA_OK && rstd) rc = check_matrix(rstd, LA_F32, 1, 1);
    if (rc != LA_OK) return rc;
    if (!reachable(x) || !reachable(residual) || !reachable(weight) || !reachable(summed) || !reachable(out) ||
        (eight && !reachable(scales)) || !reachable(rstd))
        return LA_EFAULT;
    const NormArgs a{x, residual, weight, summed, out, scales, rstd, n, x_stride, residual_stride, summed_stride,
                     out_stride, static_cast<uint32_t>(hidden), eps};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == LA_F32) return norm<float>(out_dtype, a, st);
    if (dtype == LA_BF16) return norm<__bf16>(out_dtype, a, st);
    return norm<_Float16>(out_dtype, a, st);
}

uint64_t la_rms_norm_grad_workspace(uint64_t n, uint64_t hidden)
{
    return n > kMaxRows || hidden > kMaxHidden ? 0 : most_workers(n) * hidden * sizeof(float);
}

int la_rms_norm_grad(int dtype, const void* grad_out, uint64_t grad_out_stride, const void* summed,
                     uint64_t summed_stride, const float* rstd, const void* weight, const void* grad_summed,
                     uint64_t grad_summed_stride, uint64_t n, uint64_t hidden, void* grad_x, uint64_t grad_x_stride,
                     int w_dtype, void* grad_weight, int accumulate, void* workspace, uint64_t workspace_bytes,
                     la_stream_t stream)
{
    if (!is_float_dtype(dtype) || (grad_weight && w_dtype != dtype && w_dtype != LA_F32)) return LA_EDTYPE;
    if (hidden == 0) return LA_OK;
    if (n > kMaxRows || hidden > kMaxHidden) return LA_EINVAL;
    int rc = LA_OK;
    if (n > 0) {
        rc = check_matrix(grad_out, dtype, hidden, grad_out_stride);
        if (rc == LA_OK) rc = check_matrix(summed, dtype, hidden, summed_stride);
        if (rc == LA_OK) rc = check_matrix(rstd, LA_F32, 1, 1);
        if (rc == LA_OK) rc = check_matrix(weight, dtype, hidden, hidden);
        if (rc == LA_OK && grad_summed) rc = check_matrix(grad_summed, dtype, hidden, grad_summed_stride);
        if (rc == LA_OK) rc = check_matrix(grad_x, dtype, hidden, grad_x_stride);
        if (rc == LA_OK && grad_weight)
            rc = check_workspace(workspace, workspace_bytes, most_workers(n) * hidden * sizeof(float), 16);
    }
    if (rc == LA_OK && grad_weight) rc = check_matrix(grad_weight, w_dtype, hidden, hidden);
    if (rc != LA_OK) return rc;
    if (!reachable(grad_weight) ||
        (n > 0 && (!reachable(grad_out) || !reachable(summed) || !reachable(rstd) || !reachable(weight) ||
                   !reachable(grad_summed) || !reachable(grad_x) || (grad_weight && !reachable(workspace)))))
        return LA_EFAULT;
    NormGradArgs a{grad_out, summed, rstd, weight, grad_summed, grad_x,
                         grad_weight ? static_cast<float*>(workspace) : nullptr, n, grad_out_stride, summed_stride,
                         grad_summed_stride, grad_x_stride, static_cast<uint32_t>(hidden),
                         0};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (n > 0) {
        rc = dtype == LA_F32    ? norm_grad_rows<float>(a, st)
             : dtype == LA_BF16 ? norm_grad_rows<__bf16>(a, st)
                                : norm_grad_rows<_Float16>(a, st);
        if (rc != LA_OK) return rc;
    }
    if (!grad_weight) return LA_OK;
    return w_dtype == LA_F32    ? join_weight_grad<float>(a, grad_weight, accumulate, st)
           : w_dtype == LA_BF16 ? join_weight_grad<__bf16>(a, grad_weight, accumulate, st)
                                : join_weight_grad<_Float16>(a, grad_weight, accumulate, st);
}

}  // extern "C"
