// Walks every tile, step, wave and lane of the matrix products' operands over matrices of
// many sizes, with the arithmetic the kernels use (tile_range.h), and checks each
// 16-byte read against the matrix: one that the descriptor's range lets through lies inside
// it, and one whose element the tile has in the matrix is let through.
// Prints the cases walked; exits with 1 at the first read that is wrong.
#include <cinttypes>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "tile_range.h"

namespace {

using tile::kDepth;

struct Case {
    bool by_rows;
    int side;
    uint64_t count, width, stride, tile_at, k_at;
    uint32_t all, begin;
};

uint64_t cases = 0, excluded = 0;

[[noreturn]] void fail(const Case& c, const char* what, uint32_t step, uint64_t at, uint64_t extent)
{
    std::printf("%s: by_rows %d side %d count %" PRIu64 " width %" PRIu64 " stride %" PRIu64 " tile_at %" PRIu64
                " k_at %" PRIu64 " steps %u begin %u: step %u reads at %" PRIu64 " of %" PRIu64 " bytes\n",
                what, c.by_rows, c.side, c.count, c.width, c.stride, c.tile_at, c.k_at, c.all, c.begin, step, at, extent);
    std::exit(1);
}

void check(const Case& c)
{
    ++cases;
    const uint64_t extent = (c.count - 1) * c.stride + c.width * 2;
    tile::Walk walk;
    walk.init(c.by_rows, c.count, c.width, c.stride, c.tile_at, c.k_at, c.all, c.begin);
    // four steps more are turned to at the end, which read nothing
    for (uint32_t turned = 0; turned < c.all + 4; ++turned) {
        const uint64_t at = walk.at;
        const uint32_t range = walk.range(turned);
        walk.turn();
        if (range != 0 && at + range > extent) fail(c, "range past the end", turned, at + range, extent);
        if (turned >= c.all) {
            if (range != 0) fail(c, "a step too many", turned, at, extent);
            continue;
        }
        const uint64_t k_first = c.k_at + (c.begin + turned) % c.all * static_cast<uint64_t>(kDepth);
        for (uint32_t n = 0; n < static_cast<uint32_t>(c.side) / 64; ++n)
            for (uint32_t thread = 0; thread < 256; ++thread) {
                const uint32_t offset =
                    tile::load_offset(c.side, c.by_rows, n, thread / 64, thread % 64, static_cast<uint32_t>(c.stride));
                // which row and element the lane reads, from the tile's place alone
                const uint64_t row = (c.by_rows ? c.tile_at : k_first) + offset / c.stride;
                const uint64_t element = (c.by_rows ? k_first : c.tile_at) + offset % c.stride / 2;
                const bool inside = row < c.count && element + 8 <= c.width;
                const bool read = range >= 16 && offset <= range - 16;
                if (inside && at + offset != row * c.stride + element * 2) fail(c, "another place", turned, at + offset, extent);
                if (inside && !read) fail(c, "not read", turned, at + offset, extent);
                if (read && at + offset + 16 > extent) fail(c, "read past the end", turned, at + offset, extent);
                excluded += !read;
            }
    }
}

uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

}  // namespace

int main()
{
    for (int side : {128, 256}) {
        const uint64_t s = side;
        for (uint64_t gap : {0, 8, 776}) {
            // scores: a vocabulary matrix by rows, in whole pairs of steps, tiles over the columns padded to 256
            for (uint64_t base : {0, 256, 768})
                for (uint64_t rest : {0, 1, 2, 63, 127, 128, 129, 255}) {
                    const uint64_t vocab = base + rest, columns = up(vocab, 256);
                    if (vocab == 0) continue;
                    for (uint64_t width : {64, 192}) {
                        const uint32_t steps = static_cast<uint32_t>(width / kDepth);
                        for (uint64_t at = 0; at < columns; at += s)
                            for (uint32_t xcd = 0; xcd < 8; ++xcd)
                                check({true, side, vocab, width, (width + gap) * 2, at, 0, steps, xcd * steps / 8});
                    }
                    // the states' gradient: the same matrix by columns, k over the padded columns in runs
                    for (uint64_t hidden : {8, 72, 264, 320}) {
                        const uint32_t pairs = static_cast<uint32_t>(columns / 64);
                        for (uint32_t splits : {1u, 3u, 4u}) {
                            if (splits > pairs) continue;
                            for (uint32_t run = 0; run < splits; ++run) {
                                const uint32_t from = pairs * run / splits * 2, to = pairs * (run + 1) / splits * 2;
                                for (uint64_t at = 0; at < up(hidden, s); at += s)
                                    for (uint32_t xcd = 0; xcd < 8; xcd += 3)
                                        check({false, side, vocab, hidden, (hidden + gap) * 2, at,
                                               static_cast<uint64_t>(from) * kDepth, to - from,
                                               xcd * (to - from) / 8});
                            }
                        }
                    }
                }
            if (gap > 0) continue;
            // the softmax's gradient, whole tiles: by rows over runs of k, and by columns over the trained rows
            for (uint64_t piece : {256, 768})
                for (uint64_t columns : {256, 512}) {
                    for (uint64_t at = 0; at < piece; at += s)
                        for (uint32_t xcd = 0; xcd < 8; ++xcd)
                            for (uint64_t run = 0; run < 2; ++run) {
                                const uint32_t steps = static_cast<uint32_t>(columns / 2 / kDepth);
                                check({true, side, piece, columns, columns * 2, at, run * columns / 2, steps, xcd * steps / 8});
                            }
                    for (uint64_t rows : {1, 65, 250}) {
                        const uint32_t steps = static_cast<uint32_t>(up(rows, 64) / kDepth);
                        for (uint64_t at = 0; at < columns; at += s)
                            check({false, side, piece, columns, columns * 2, at, 0, steps, steps / 2});
                    }
                }
        }
    }
    std::printf("%" PRIu64 " walks, %" PRIu64 " reads excluded\n", cases, excluded);
    return 0;
}
