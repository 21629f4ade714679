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
#include "attention_tile.h"

#include <algorithm>

namespace {

using namespace att;

struct GradArgs {
    Heads q, k, v, out, grad_out;
    Heads grad_q, grad_k, grad_v;
    const float* lse;
    float *lse2, *delta;            // [heads][flat rows]: lse in base 2, and delta, by grad_q_kernel
    Sequences seq;
    uint32_t heads, kv_heads, dim, read_dim;
    uint32_t rows_all;              // flat rows
    float scale;
    int q_aligned, k_aligned, v_aligned;
    int keep_rest;
};

// dS in the operands' 16 bits.  bfloat16 has fp32's range.  fp16 has not: what a wave rounds is brought near the
// top of its range by a power of two for each column, which shrinks when a larger value comes, and its
// sums with it; P, at most 1, by a fixed one.
template <typename T> struct Range {
    static constexpr float kP = 0.0f;
    __device__ __forceinline__ float factor() const { return 1.0f; }
    template <int N> __device__ __forceinline__ void fit(f32x16&, f32x16 (&)[N]) {}
};
template <> struct Range<_Float16> {
    static constexpr float kP = 14.0f;                   // P is held times 2^14
    float up = 0x1p60f;
    __device__ __forceinline__ float factor() const { return up; }
    template <int N> __device__ __forceinline__ void fit(f32x16& x, f32x16 (&sums)[N])
    {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, __builtin_fabsf(x[i]));
        most = both_max(most);
        if (__any(most * up > 32768.0f)) {
            // to 2^10 .. 2^11: five doublings before it shrinks again
            int e;
            (void)frexpf(most, &e);
            e = 11 - e;
            e = e < -60 ? -60 : e > 60 ? 60 : e;
            const float now = most * up > 32768.0f && most < INFINITY ? __builtin_ldexpf(1.0f, e) : up;
            const float shrink = now / up;
            up = now;
#pragma unroll
            for (int n = 0; n < N; ++n) sums[n] *= shrink;
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

template <int D> __device__ __forceinline__ void load_row(s16x8 (&q)[D / 16], const char* row, bool there, uint32_t dim)
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

// 128 rows to a workgroup, 32 to a wave, tiles of 64 keys as in the forward pass.
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

    s16x8 q[D / 16], g[D / 16];
    load_row<D>(q, a.q.at(p.batch, p.first + token, head), there, a.read_dim);
    load_row<D>(g, a.grad_out.at(p.batch, p.first + token, head), there, a.read_dim);
    float delta, lse2;
    {
        s16x8 o[D / 16];
        load_row<D>(o, a.out.at(p.batch, p.first + token, head), there, a.read_dim);
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
        lse2 = there ? a.lse[flat * a.heads + head] * kLog2E : 0.0f;
        if (there && lane < 32) {
            const uint64_t at = static_cast<uint64_t>(head) * a.rows_all + flat;
            a.lse2[at] = lse2;
            a.delta[at] = delta;
        }
        asm volatile("" : "+v"(lse2));
    }

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

    f32x16 sums[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) sums[d] = zeros();
    Range<T> scaled;
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
                scaled.fit(d, sums);
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

// 128 keys to a workgroup, 32 to a wave; all waves go over the same tiles of 64 rows of one query
// head after the other.
template <typename T, int D> __global__ __launch_bounds__(256, 2) void grad_kv_kernel(GradArgs a)
{
    constexpr uint32_t kBytes = Tile<D>::kBytes;
    constexpr uint32_t kRowValues = kTileRows * 4;       // bytes of a tile's lse, and of its delta
    __shared__ __attribute__((aligned(1024))) char shared[4 * kBytes + 4 * 4 * kRowValues];
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    const Piece p = locate(a.seq, blockIdx.x / a.kv_heads, true, 1, 128);
    if (!p.valid) return;
    const uint32_t wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t group = a.seq.group;
    const uint32_t key = p.tile * 128 + wave * 32 + lane % 32;
    const bool there = key < p.keys;
    const int32_t shift = static_cast<int32_t>(p.keys) - static_cast<int32_t>(p.length);

    // the queries that see keys [from, to): those of row `from` .. where causal
    const auto rows_of = [&](uint32_t from, uint32_t to) {
        Seen r{0, static_cast<int32_t>(p.length)};
        if (!a.seq.causal) return r;
        r.lo = static_cast<int32_t>(from) - shift;
        r.lo = r.lo < 0 ? 0 : r.lo;
        const int32_t last = static_cast<int32_t>(to) - 1 - shift;       // sees key `to` - 1 as its last
        if (a.seq.window && last + static_cast<int64_t>(a.seq.window) < r.hi)
            r.hi = last + static_cast<int32_t>(a.seq.window);
        return r;
    };
    const Seen mine = rows_of(key, key + 1);
    const uint32_t first = p.tile * 128, wave_first = first + wave * 32;
    const uint32_t past = first + 128 < p.keys ? first + 128 : p.keys;
    const Seen all = p.rest ? Seen{0, 0} : rows_of(first, past);
    const Seen own = rows_of(wave_first, wave_first + 32);
    const Seen common{rows_of(wave_first + 31, wave_first + 32).lo, rows_of(wave_first, wave_first + 1).hi};
    const int32_t tile_from = all.lo / static_cast<int32_t>(kTileRows);
    const int32_t tile_to = all.hi > 0 ? (all.hi + static_cast<int32_t>(kTileRows) - 1) / static_cast<int32_t>(kTileRows) : 0;

    f32x16 sums_k[D / 32], sums_v[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) sums_k[d] = sums_v[d] = zeros();
    Range<T> scaled;
    if (tile_from < tile_to) {
        s16x8 k[D / 16], v[D / 16];
        load_row<D>(k, a.k.at(p.batch, p.key_first + key, kv_head), there, a.read_dim);
        load_row<D>(v, a.v.at(p.batch, p.key_first + key, kv_head), there, a.read_dim);
        Loader<D, kTileRows, 4> load_q, load_g;
        load_q.init(wave, static_cast<uint32_t>(a.q.row), a.read_dim);
        load_g.init(wave, static_cast<uint32_t>(a.grad_out.row), a.read_dim);
        Fragments<D> f;
        f.init();
        lds_char* lds = (lds_char*)shared;
        const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
        const uint32_t place = base + wave * 1024;
        const uint32_t values = 4 * kBytes + wave * 4 * kRowValues;      // this wave's own copy
        const float factor = a.scale * kLog2E;
        const auto load = [&](uint32_t head, int32_t tile, uint32_t buffer) {
            const Rows queries{reinterpret_cast<uint64_t>(a.q.at(p.batch, p.first, head)), static_cast<int32_t>(p.length)};
            const Rows grads{reinterpret_cast<uint64_t>(a.grad_out.at(p.batch, p.first, head)),
                             static_cast<int32_t>(p.length)};
            load_q.load(queries, tile * kTileRows, place + buffer * 2 * kBytes);
            load_g.load(grads, tile * kTileRows, place + buffer * 2 * kBytes + kBytes);
            const uint64_t at = static_cast<uint64_t>(head) * a.rows_all + static_cast<uint64_t>(p.batch) * a.seq.rows + p.first;
            const int32_t left = static_cast<int32_t>(p.length) - tile * static_cast<int32_t>(kTileRows);
            const uint32_t bytes = left <= 0 ? 0u : left < static_cast<int32_t>(kTileRows) ? left * 4u : kRowValues;
            load_values(reinterpret_cast<uint64_t>(a.lse2 + at + tile * kTileRows), bytes,
                        base + values + buffer * 2 * kRowValues);
            load_values(reinterpret_cast<uint64_t>(a.delta + at + tile * kTileRows), bytes,
                        base + values + buffer * 2 * kRowValues + kRowValues);
        };
        uint32_t head = kv_head * group, buffer = 0;
        const uint32_t head_end = head + group;
        load(head, tile_from, 0);
        for (int32_t tile = tile_from; head < head_end; buffer ^= 1) {
            arrive<0>();
            int32_t next = tile + 1;
            uint32_t next_head = head;
            if (next == tile_to) next = tile_from, ++next_head;
            if (next_head < head_end) load(next_head, next, buffer ^ 1);
            const lds_char *qs = lds + buffer * 2 * kBytes, *gs = qs + kBytes;
            const lds_char* rows = lds + values + buffer * 2 * kRowValues;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int32_t first_row = tile * static_cast<int32_t>(kTileRows) + b * 32;
                if (first_row >= own.hi || first_row + 32 <= own.lo) continue;
                f32x16 s = product<T, D>(qs, k, f, b);
                f32x16 d = product<T, D>(gs, v, f, b);
                const uint32_t half = lane / 32 * 16;
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const f32x4 lse2 = *reinterpret_cast<const lds_f32x4*>(rows + b * 128 + i * 8 + half);
                    const f32x4 delta = *reinterpret_cast<const lds_f32x4*>(rows + kRowValues + b * 128 + i * 8 + half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[i + e] = exp2_of(__builtin_fmaf(s[i + e], factor, Range<T>::kP - lse2[e]));
                        d[i + e] = s[i + e] * (d[i + e] - delta[e]);
                    }
                }
                if (first_row < common.lo || first_row + 32 > common.hi) {
                    hide(s, first_row, mine);
                    hide(d, first_row, mine);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const s16x8 p16 = rounded<T>(s, h);
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) sums_v[e] = mfma<T>(f.columns(gs, e, b * 2 + h), p16, sums_v[e]);
                }
                scaled.fit(d, sums_k);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const s16x8 ds = rounded<T>(d, h);
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) sums_k[e] = mfma<T>(f.columns(qs, e, b * 2 + h), ds, sums_k[e]);
                }
            }
            tile = next;
            head = next_head;
        }
    }
    constexpr float kShrinkP = Range<T>::kP == 0.0f ? 1.0f : 0x1p-14f;
    const bool stored = key < (a.keep_rest ? (p.rest ? 0u : p.keys) : p.key_stored);
    store_row<T, D>(const_cast<char*>(a.grad_v.at(p.batch, p.key_first + key, kv_head)), sums_v, kShrinkP, stored, a.dim,
                    a.v_aligned);
    store_row<T, D>(const_cast<char*>(a.grad_k.at(p.batch, p.key_first + key, kv_head)), sums_k,
                    a.scale * kShrinkP / scaled.factor(), stored, a.dim, a.k_aligned);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
uint64_t row_values_bytes(const la_attention_t& c) { return ceil_div(flat_rows(c) * c.heads * 4, 256ull) * 256; }

template <typename T, int D> int run(const la_attention_t& c, const GradArgs& a, hipStream_t stream)
{
    int rc = LA_OK;
    const uint64_t by_rows = pieces(a.seq, false, a.seq.group, 128) * c.kv_heads;
    const uint64_t by_keys = pieces(a.seq, true, 1, 128) * c.kv_heads;
    if (flat_rows(c) > 0) rc = launch(grad_q_kernel<T, D>, dim3(static_cast<uint32_t>(by_rows)), dim3(256), stream, a);
    if (rc == LA_OK && flat_keys(c) > 0)
        rc = launch(grad_kv_kernel<T, D>, dim3(static_cast<uint32_t>(by_keys)), dim3(256), stream, a);
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
    return 2 * row_values_bytes(c) + packed_bytes(c, c.q, true) + packed_bytes(c, c.k, false) +
           packed_bytes(c, c.v, false) + packed_bytes(c, c.out, true) + packed_bytes(c, c.grad_out, true);
}

int la_attention_grad(const la_attention_t* call, void* workspace, uint64_t workspace_bytes, la_stream_t stream)
{
    int rc = check_call(call);
    if (rc != LA_OK) return rc;
    const la_attention_t& c = *call;
    const bool rows = flat_rows(c) > 0, keys = flat_keys(c) > 0;
    if ((rows && (!there(c.q) || !there(c.out) || !there(c.grad_out) || !there(c.grad_q) || !c.lse ||
                  reinterpret_cast<uintptr_t>(c.lse) % 4)) ||
        (keys && (!there(c.k) || !there(c.v) || !there(c.grad_k) || !there(c.grad_v))))
        return LA_EINVAL;
    rc = check_workspace(workspace, workspace_bytes, la_attention_grad_workspace(call), 256);
    if (rc != LA_OK) return rc;
    const Sequences s = sequences_of(c);
    if (pieces(s, false, s.group, 128) * c.kv_heads >> 31 || pieces(s, true, 1, 128) * c.kv_heads >> 31) return LA_EINVAL;
    for (const void* p : {c.q.data, c.k.data, c.v.data, c.out.data, c.grad_out.data, c.grad_q.data, c.grad_k.data,
                          c.grad_v.data, static_cast<const void*>(c.lse)})
        if (!reachable(p)) return LA_EFAULT;
    if (!indices_reachable(c) || !reachable(workspace)) return LA_EFAULT;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    GradArgs a{};
    a.lse = c.lse;
    a.lse2 = reinterpret_cast<float*>(ws);
    a.delta = reinterpret_cast<float*>(ws + row_values_bytes(c));
    ws += 2 * row_values_bytes(c);
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
