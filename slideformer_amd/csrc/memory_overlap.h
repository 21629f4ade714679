// slideformer_amd: whether two sets of memory share a byte, where each lies in
// up to three strides, as the heads of a tensor do (host code, plain C++).
//
// Parts of one projection interleave row by row, so that their first and last bytes say little.
// Two runs of `width` bytes share one where the difference of their places is within their widths, and that
// difference is a sum of the strides, each times a number from a range: it is looked for stride by
// stride, the longest first, among the numbers after which the shorter ones can still make up the rest.  That
// is one or two for each stride where rows lie as in tensors, within one another.
#ifndef SLIDEFORMER_AMD_MEMORY_OVERLAP_H
#define SLIDEFORMER_AMD_MEMORY_OVERLAP_H

#include <cstdint>

namespace la_memory {

// The bytes [at + sum i[d] stride[d], + width) for all i[d] < count[d].
struct Place {
    uintptr_t at;
    uint64_t width;
    uint64_t count[3], stride[3];
};

inline Place flat(const void* at, uint64_t bytes) { return {reinterpret_cast<uintptr_t>(at), bytes, {1, 1, 1}, {0, 0, 0}}; }

inline bool nothing(const Place& p) { return !p.at || !p.width || !p.count[0] || !p.count[1] || !p.count[2]; }

// Whether both are the same bytes in the same order.
inline bool same(const Place& a, const Place& b)
{
    bool alike = a.at == b.at && a.width == b.width;
    for (int d = 0; d < 3; ++d)
        alike = alike && a.count[d] == b.count[d] && (a.count[d] < 2 || a.stride[d] == b.stride[d]);
    return alike;
}

constexpr uint64_t kEndless = 1ull << 62;                // lengths that no memory has

// Bytes from the first to past the last, kEndless at the most.
inline uint64_t length(const Place& p)
{
    uint64_t sum = p.width < kEndless ? p.width : kEndless;
    for (int d = 0; d < 3; ++d) {
        uint64_t more = 0;
        if (__builtin_mul_overflow(p.count[d] - 1, p.stride[d], &more) || more > kEndless) more = kEndless;
        sum = sum + more < kEndless ? sum + more : kEndless;
    }
    return sum;
}

struct Search {
    int64_t stride[6], lo[6], hi[6];                     // numbers of times, inclusive
    int64_t rest_lo[7], rest_hi[7];                      // what the strides from here on can add
    int64_t from, to;                                    // the differences that count
    int strides, steps;

    bool found(int k, int64_t sum)
    {
        if (k == strides) return sum >= from && sum <= to;
        const int64_t s = stride[k], least = from - sum - rest_hi[k + 1], most = to - sum - rest_lo[k + 1];
        const int64_t up = least >= 0 ? (least + s - 1) / s : -(-least / s), down = most >= 0 ? most / s : -((-most + s - 1) / s);
        for (int64_t x = up > lo[k] ? up : lo[k]; x <= hi[k] && x <= down; ++x) {
            if (--steps < 0) return true;                // not decided
            if (found(k + 1, sum + s * x)) return true;
        }
        return false;
    }
};

// Whether a and b share a byte; also where that is not found out in 2^14 steps.
inline bool shared(const Place& a, const Place& b)
{
    if (nothing(a) || nothing(b)) return false;
    const uint64_t of_a = length(a), of_b = length(b);
    if (a.at < b.at ? of_a <= b.at - a.at : of_b <= a.at - b.at) return false;
    if (of_a >= kEndless || of_b >= kEndless) return true;
    Search s{};
    s.steps = 1 << 14;
    s.from = -static_cast<int64_t>(a.width) + 1;
    s.to = static_cast<int64_t>(b.width) - 1;
    const auto add = [&s](uint64_t stride, int64_t lo, int64_t hi) {
        if (stride == 0 || lo == hi) return;
        int k = 0;
        while (k < s.strides && s.stride[k] > static_cast<int64_t>(stride)) ++k;
        if (k < s.strides && s.stride[k] == static_cast<int64_t>(stride)) {
            s.lo[k] += lo;
            s.hi[k] += hi;
            return;
        }
        for (int m = s.strides++; m > k; --m) {
            s.stride[m] = s.stride[m - 1];
            s.lo[m] = s.lo[m - 1];
            s.hi[m] = s.hi[m - 1];
        }
        s.stride[k] = static_cast<int64_t>(stride);
        s.lo[k] = lo;
        s.hi[k] = hi;
    };
    for (int d = 0; d < 3; ++d) {
        add(a.stride[d], 0, static_cast<int64_t>(a.count[d]) - 1);
        add(b.stride[d], 1 - static_cast<int64_t>(b.count[d]), 0);
    }
    for (int k = s.strides - 1; k >= 0; --k) {
        s.rest_lo[k] = s.rest_lo[k + 1] + s.stride[k] * s.lo[k];
        s.rest_hi[k] = s.rest_hi[k + 1] + s.stride[k] * s.hi[k];
    }
    return s.found(0, static_cast<int64_t>(a.at) - static_cast<int64_t>(b.at));
}

}  // namespace la_memory

#endif  // SLIDEFORMER_AMD_MEMORY_OVERLAP_H
