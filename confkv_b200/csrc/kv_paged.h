// Index arithmetic of the paged cache's operators, free of CUDA so that the CPU tests compile and replay it: what a
// request's change takes and gives back, and how attention cuts its work.
#pragma once

#include <cstdint>

#include "kv_layout.h"

namespace confkv {
namespace kv {

constexpr uint32_t kMaxRequests = 1u << 24;
constexpr uint32_t kMaxTokens = 0x7fffffffu;

// Most tokens that a row of `width` blocks names, as far as 31 bits count them.
KV_HD uint32_t row_limit(uint32_t width, uint32_t block_size)
{
    const uint64_t n = uint64_t{width} * block_size;
    return n < kMaxTokens ? static_cast<uint32_t>(n) : kMaxTokens;
}

KV_HD uint32_t blocks_of(const FastDiv& by_block, uint32_t tokens)
{
    const uint32_t q = quotient(by_block, tokens);
    return q + (tokens != q * by_block.d ? 1u : 0u);
}

// What a request does on its way from `held` to `length` tokens.
struct Change {
    uint32_t held, kept;        // tokens before, and after where it is not refused
    uint32_t before;            // its blocks before
    uint32_t take, give;        // blocks that it takes, or gives back
    uint32_t tokens;            // new tokens
};

KV_HD Change change_of(int32_t held, int32_t length, uint32_t limit, const FastDiv& by_block)
{
    Change c{};
    if (held < 0 || static_cast<uint32_t>(held) > limit) {
        return c;
    }
    c.held = c.kept = static_cast<uint32_t>(held);
    c.before = blocks_of(by_block, c.held);
    if (length < 0 || static_cast<uint32_t>(length) > limit) {
        return c;
    }
    c.kept = static_cast<uint32_t>(length);
    const uint32_t after = blocks_of(by_block, c.kept);
    c.take = after > c.before ? after - c.before : 0;
    c.give = after < c.before ? c.before - after : 0;
    c.tokens = c.kept > c.held ? c.kept - c.held : 0;
    return c;
}

// A cursor brought into the ring's range.
struct Cursor {
    uint32_t first, count;
};

KV_HD Cursor cursor_of(int32_t first, int32_t count, uint32_t ring)
{
    Cursor c{};
    if (ring != 0) {
        c.first = static_cast<uint32_t>(first);
        if (c.first >= ring) {
            const int64_t f = first % static_cast<int64_t>(ring);
            c.first = static_cast<uint32_t>(f < 0 ? f + ring : f);
        }
        c.count = count < 0 ? 0 : (static_cast<uint32_t>(count) < ring ? static_cast<uint32_t>(count) : ring);
    }
    return c;
}

// The tokens [first, end) that a request attends to.
struct Span {
    uint32_t first, end;
};

KV_HD Span span_of(int32_t length, uint32_t limit, uint32_t window)
{
    Span s{};
    s.end = length < 0 ? 0 : (static_cast<uint32_t>(length) < limit ? static_cast<uint32_t>(length) : limit);
    s.first = window != 0 && s.end > window ? s.end - window : 0;
    return s;
}

// Tiles of a row over a span; an empty row has one, so that its result is written like any other.
KV_HD uint32_t tiles_of(const Span& s, uint32_t tile)
{
    const uint32_t n = s.end - s.first;
    return n == 0 ? 1u : (n + tile - 1) / tile;
}

// Attention's work is counted in units: a row's tiles, and kRowUnits in front of them for its beginning and its end. The units of all rows, one row
// behind the other, are cut into equal parts for `workers` <= total workers: worker c has the units [part_start(c),
// part_start(c + 1)), one at least. total < 2^52, workers < 2^11. With one, two, three and five units in front of a row 64 ragged
// requests take 34.9, 31.4, 31.7 and 33.3 us, and 128 of one key head 22.6, 21.0, 19.2 and 18.8.
constexpr uint32_t kRowUnits = 3;

KV_HD uint64_t part_start(uint64_t total, uint32_t workers, uint32_t c)
{
    // 32 bits where they hold it: the division is a good part of a small call's beginning
    return total < (1u << 21) ? static_cast<uint32_t>(total) * c / workers : total * c / workers;
}

// The worker that has a unit: the largest c with total c / workers < unit + 1.
KV_HD uint32_t part_of(uint64_t total, uint32_t workers, uint64_t unit)
{
    return static_cast<uint32_t>(((unit + 1) * workers - 1) / total);
}

// How finely rows may be cut, a kernel's own: cutting costs more than some tiles do (the pieces have to be written and joined). A row of up to
// whole_tiles tiles stays whole, and few units are shared by fewer workers, 2^least_units each.
struct Cutting {
    uint32_t whole_tiles, least_units;
};

KV_HD uint32_t workers_for(const Cutting& k, uint64_t total, uint32_t most)
{
    const uint64_t n = total >> k.least_units;
    return n == 0 ? 1u : (n < most ? static_cast<uint32_t>(n) : most);
}

// Where a part's border at `x` units behind a row's first one (or before it) cuts the row: in front of which tile.
KV_HD uint32_t first_units(const Cutting& k, uint32_t tiles)      // up to there a border lies in front of the row
{
    return tiles <= k.whole_tiles ? (tiles + kRowUnits) / 2 : kRowUnits;
}

KV_HD uint32_t last_units(const Cutting& k, uint32_t tiles)       // beyond there it lies behind the row
{
    return tiles <= k.whole_tiles ? (tiles + kRowUnits) / 2 : kRowUnits + tiles - 1;
}

KV_HD uint32_t cut_at(const Cutting& k, int64_t x, uint32_t tiles)
{
    return x <= static_cast<int64_t>(first_units(k, tiles)) ? 0u
           : x > static_cast<int64_t>(last_units(k, tiles)) ? tiles
                                                            : static_cast<uint32_t>(x) - kRowUnits;
}

}  // namespace kv
}  // namespace confkv
