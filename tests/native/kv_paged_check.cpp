// Host build of the paged cache's index arithmetic (csrc/kv_paged.h) for the CPU tests: each function on arrays.
#include <cstdint>

#include "kv_paged.h"

using namespace confkv::kv;

extern "C" {

// held, length -> kept, before, take, give, tokens
void changes(const int32_t* held, const int32_t* length, int n, uint32_t width, uint32_t block_size, uint32_t* out)
{
    const FastDiv d = make_fast_div(block_size);
    const uint32_t limit = row_limit(width, block_size);
    for (int i = 0; i < n; ++i) {
        const Change c = change_of(held[i], length[i], limit, d);
        uint32_t* o = out + 5 * i;
        o[0] = c.kept;
        o[1] = c.before;
        o[2] = c.take;
        o[3] = c.give;
        o[4] = c.tokens;
    }
}

void cursors(const int32_t* first, const int32_t* count, int n, uint32_t ring, uint32_t* out)
{
    for (int i = 0; i < n; ++i) {
        const Cursor c = cursor_of(first[i], count[i], ring);
        out[2 * i] = c.first;
        out[2 * i + 1] = c.count;
    }
}

void spans(const int32_t* length, int n, uint32_t limit, uint32_t window, uint32_t tile, uint32_t* out)
{
    for (int i = 0; i < n; ++i) {
        const Span s = span_of(length[i], limit, window);
        out[3 * i] = s.first;
        out[3 * i + 1] = s.end;
        out[3 * i + 2] = tiles_of(s, tile);
    }
}

// 0 where the rows (of so many tiles each) are cut as joining takes it: every tile is one worker's; a row begins in the worker that
// part_of names for first_units, goes on in the next ones without a gap, and ends in the one named for last_units; rows of few
// tiles are whole.
int check_rows(const uint32_t* tiles, int rows, uint32_t most, uint32_t whole_tiles, uint32_t least_units)
{
    const Cutting k{whole_tiles, least_units};
    uint64_t total = 0;
    for (int r = 0; r < rows; ++r) {
        total += tiles[r] + kRowUnits;
    }
    const uint32_t workers = workers_for(k, total, most);
    if (workers > total || workers > most) {
        return 1;
    }
    uint64_t row_begin = 0;
    for (int r = 0; r < rows; ++r) {
        const uint32_t begins = part_of(total, workers, row_begin + first_units(k, tiles[r]));
        const uint32_t ends = part_of(total, workers, row_begin + last_units(k, tiles[r]));
        uint32_t next = 0;
        for (uint32_t c = 0; c < workers; ++c) {
            const int64_t a = static_cast<int64_t>(part_start(total, workers, c)) - static_cast<int64_t>(row_begin);
            const int64_t b = static_cast<int64_t>(part_start(total, workers, c + 1)) - static_cast<int64_t>(row_begin);
            if (b <= 0 || a >= static_cast<int64_t>(tiles[r] + kRowUnits)) {
                continue;
            }
            const uint32_t first = cut_at(k, a, tiles[r]), last = cut_at(k, b, tiles[r]);
            if ((last > first) != (c >= begins && c <= ends)) {
                return 2;
            }
            if (last <= first) {
                continue;
            }
            if (first != next) {
                return 3;
            }
            next = last;
        }
        if (next != tiles[r]) {
            return 5;
        }
        if (tiles[r] <= whole_tiles && begins != ends) {
            return 6;
        }
        row_begin += tiles[r] + kRowUnits;
    }
    return 0;
}

// 0 where all parts of `total` tiles are right: none empty, one behind the other, sizes at most one apart, every tile's worker
// the one whose part it lies in (at the parts' ends, and at every tile where there are few)
int check_parts(uint64_t total, uint32_t workers)
{
    if (part_start(total, workers, 0) != 0 || part_start(total, workers, workers) != total) {
        return 1;
    }
    const uint64_t least = total / workers;
    for (uint32_t c = 0; c < workers; ++c) {
        const uint64_t a = part_start(total, workers, c), b = part_start(total, workers, c + 1);
        if (b - a < least || b - a > least + 1 || a == b) {
            return 2;
        }
        if (part_of(total, workers, a) != c || part_of(total, workers, b - 1) != c) {
            return 3;
        }
        if (total < 5000) {
            for (uint64_t t = a; t < b; ++t) {
                if (part_of(total, workers, t) != c) {
                    return 4;
                }
            }
        }
    }
    return 0;
}
}
