// la_memory::shared against counting every byte, and on layouts whose answer is known.
#include "memory_overlap.h"

#include <cstdio>
#include <random>
#include <set>

using la_memory::Place;

namespace {

int wrong = 0;

void show(const char* what, const Place& a, const Place& b, bool got)
{
    ++wrong;
    std::printf("%s: got %d\n", what, got);
    for (const Place* p : {&a, &b})
        std::printf("  at %zu width %llu counts %llu %llu %llu strides %llu %llu %llu\n", static_cast<size_t>(p->at),
                    static_cast<unsigned long long>(p->width), static_cast<unsigned long long>(p->count[0]),
                    static_cast<unsigned long long>(p->count[1]), static_cast<unsigned long long>(p->count[2]),
                    static_cast<unsigned long long>(p->stride[0]), static_cast<unsigned long long>(p->stride[1]),
                    static_cast<unsigned long long>(p->stride[2]));
}

void expect(const char* what, const Place& a, const Place& b, bool want)
{
    if (la_memory::shared(a, b) != want) show(what, a, b, !want);
    if (la_memory::shared(b, a) != want) show(what, b, a, !want);
}

std::set<uint64_t> bytes(const Place& p)
{
    std::set<uint64_t> s;
    for (uint64_t i = 0; i < p.count[0]; ++i)
        for (uint64_t j = 0; j < p.count[1]; ++j)
            for (uint64_t k = 0; k < p.count[2]; ++k)
                for (uint64_t w = 0; w < p.width; ++w) s.insert(p.at + i * p.stride[0] + j * p.stride[1] + k * p.stride[2] + w);
    return s;
}

// heads of rows of batches
Place heads(uint64_t at, uint64_t width, uint64_t batches, uint64_t rows, uint64_t heads, uint64_t batch, uint64_t row, uint64_t head)
{
    return {at, width, {batches, rows, heads}, {batch, row, head}};
}

}  // namespace

int main()
{
    std::mt19937 rng(1);
    const auto pick = [&](uint32_t n) { return rng() % n; };
    int cases = 0, sharing = 0;
    for (int n = 0; n < 200000; ++n) {
        Place p[2];
        const bool common = pick(2);                     // strides in common, as parts of one buffer have
        const uint64_t strides[3] = {pick(60), pick(25), pick(9)};
        for (Place& x : p) {
            x.at = 1000 + pick(120);
            x.width = pick(6);
            for (int d = 0; d < 3; ++d) {
                x.count[d] = pick(10) ? 1 + pick(4) : pick(2);
                x.stride[d] = common && pick(8) ? strides[d] : pick(40);
            }
        }
        const std::set<uint64_t> a = bytes(p[0]), b = bytes(p[1]);
        bool want = false;
        for (uint64_t x : a) want = want || b.count(x);
        const bool got = la_memory::shared(p[0], p[1]);
        if (got != want && wrong < 5) show("counted", p[0], p[1], got);
        ++cases;
        sharing += want;
    }
    // parts of one projection of 4096 rows, 32 and 8 and 8 heads of 256 bytes
    const uint64_t at = 1ull << 32, row = 48 * 256;
    const Place q = heads(at, 256, 1, 4096, 32, 0, row, 256), k = heads(at + 32 * 256, 256, 1, 4096, 8, 0, row, 256);
    const Place v = heads(at + 40 * 256, 256, 1, 4096, 8, 0, row, 256);
    expect("q, k", q, k, false);
    expect("k, v", k, v, false);
    expect("q, q a row on", q, heads(at + row, 256, 1, 4096, 32, 0, row, 256), true);
    expect("k, k a head on", k, heads(at + 33 * 256, 256, 1, 4096, 8, 0, row, 256), true);
    expect("k, v an element before", k, heads(at + 40 * 256 - 2, 256, 1, 4096, 8, 0, row, 256), true);
    // heads first beside rows first, in one buffer and one after the other
    expect("orders", heads(at, 128, 2, 512, 8, 512 * 8 * 128, 128, 512 * 128),
           heads(at, 128, 2, 512, 8, 512 * 8 * 128, 8 * 128, 128), true);
    expect("one after the other", heads(at, 128, 2, 512, 8, 512 * 8 * 128, 128, 512 * 128),
           heads(at + 2 * 512 * 8 * 128, 128, 2, 512, 8, 512 * 8 * 128, 8 * 128, 128), false);
    // a batch's keys and values in one cache, as neighbours in a row and as halves of a sequence
    expect("neighbours", heads(at, 128, 64, 8192, 8, 8192 * 16 * 128, 16 * 128, 256),
           heads(at + 128, 128, 64, 8192, 8, 8192 * 16 * 128, 16 * 128, 256), false);
    expect("halves", heads(at, 128, 64, 8192, 8, 2 * 8192 * 8 * 128, 8 * 128, 128),
           heads(at + 8192 * 8 * 128, 128, 64, 8192, 8, 2 * 8192 * 8 * 128, 8 * 128, 128), false);
    // one fp32 to a head beside the heads, and in them
    expect("values beside", q, heads(at + 47 * 256, 4, 1, 4096, 32, 0, row, 4), false);
    expect("values within", q, heads(at + 31 * 256, 4, 1, 4096, 32, 0, row, 4), true);
    // expanded inputs, nothing, and lengths that no memory has
    expect("one row", heads(at, 256, 16, 4096, 8, 0, 0, 256), heads(at + 8 * 256, 256, 1, 4096, 8, 0, row, 256), false);
    expect("empty", heads(at, 256, 1, 0, 8, 0, row, 256), q, false);
    expect("null", heads(0, 256, 1, 4096, 8, 0, row, 256), heads(0, 256, 1, 4096, 8, 0, row, 256), false);
    expect("endless", heads(at, 256, 2, 4096, 8, ~0ull, row, 256), k, true);
    expect("endless, behind", heads(at + (1ull << 40), 256, 1ull << 40, 4096, 8, ~0ull, row, 256), k, false);
    // Even and odd bytes in six strides, none within another: it is not found out that they never meet
    expect("not decided", {at, 1, {1000, 1001, 1002}, {9998, 10002, 10006}}, {at + 1, 1, {1003, 1004, 1005}, {9994, 10010, 10014}}, true);
    if (la_memory::same(q, k) || !la_memory::same(q, q) ||
        !la_memory::same(heads(at, 8, 1, 1, 4, 5, 6, 8), heads(at, 8, 1, 1, 4, 7, 9, 8)) ||
        la_memory::same(heads(at, 8, 1, 2, 4, 5, 6, 8), heads(at, 8, 1, 2, 4, 5, 9, 8))) {
        ++wrong;
        std::printf("same\n");
    }
    std::printf("%d cases, %d sharing, %d wrong\n", cases, sharing, wrong);
    return wrong != 0;
}
