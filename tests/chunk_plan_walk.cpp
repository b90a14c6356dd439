// Walks through the plan of the chunk attention: every unit of every item belongs to exactly one piece, and the pieces
// of an item that is cut are those of the workers from the one that begins it to the one worker_of() names.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "../qwencore_b200/csrc/kernels/chunk_plan.h"

using namespace qwc;

static int fail(const char* what) {
    std::printf("%s\n", what);
    return 1;
}

static int check(const std::vector<ChunkSequence>& sequences, int most_workers) {
    struct Item {
        int sequence, head, tile;
        long long at;
    };
    std::vector<Item> items;
    long long total = 0;
    for (int s = 0; s < static_cast<int>(sequences.size()); ++s) {
        for (int head = 0; head < kPlanHeads; ++head) {
            for (int tile = 0; tile < item_tiles(sequences[s]); ++tile) {
                items.push_back({s, head, tile, total});
                total += item_units(sequences[s], tile) + kItemLead;
            }
        }
    }
    const auto info = [&](int s) { return sequences[s]; };
    const int workers = plan_workers(total, most_workers);
    std::map<std::tuple<int, int, int>, std::vector<std::tuple<int, ChunkPiece>>> pieces;
    std::map<std::tuple<int, int, int>, int> last;
    long long most = 0, least = 1ll << 60;
    size_t start = 0;
    for (int w = 0; w < workers; ++w) {
        const long long begin = share_begin(total, w, workers), end = share_begin(total, w + 1, workers);
        most = end - begin > most ? end - begin : most;
        least = end - begin < least ? end - begin : least;
        if (begin == end) {
            continue;
        }
        while (start + 1 < items.size() && items[start + 1].at <= begin) {
            ++start;
        }
        ChunkWalk walk = {};
        walk.sequence = items[start].sequence;
        walk.head = items[start].head;
        walk.tile = items[start].tile;
        walk.skip = begin - items[start].at;
        walk.at = items[start].at;
        walk.left = end - begin;
        walk.info = sequences[walk.sequence];
        ChunkPiece piece;
        int cut_at_end = 0;
        for (bool first = true; next_piece(walk, first, static_cast<int>(sequences.size()), info, piece); first = false) {
            if (cut_at_end) return fail("a piece behind one that is cut at its end");
            if (piece.unit_begin < 0 || piece.unit_end > piece.units) return fail("units beyond the item");
            cut_at_end = piece.unit_end < piece.units;
            const auto key = std::make_tuple(walk.sequence, walk.head, walk.tile);
            if (piece.units != item_units(sequences[walk.sequence], walk.tile)) return fail("another item's units");
            pieces[key].push_back({w, piece});
            if (piece.unit_begin == 0) {
                last[key] = worker_of(total, walk.item_end - 1, workers);
            }
        }
    }
    if (most - least > 1) return fail("shares differ");
    for (const Item& item : items) {
        const auto key = std::make_tuple(item.sequence, item.head, item.tile);
        int unit = 0, worker = -1;
        for (const auto& [w, piece] : pieces[key]) {
            if (piece.unit_begin != unit || (worker >= 0 && w != worker + 1)) return fail("a gap, or a unit twice");
            unit = piece.unit_end;
            worker = w;
        }
        if (unit != item_units(sequences[item.sequence], item.tile)) return fail("units left over");
        if (last[key] != worker) return fail("another last worker");
    }
    return 0;
}

int main() {
    std::mt19937 rng(5);
    const auto log_uniform = [&](double high) {
        return static_cast<int>(std::exp(std::uniform_real_distribution<double>(0.0, std::log(high))(rng)));
    };
    for (int round = 0; round < 3000; ++round) {
        std::vector<ChunkSequence> sequences;
        const int count = log_uniform(129.0);
        int begin = 0;
        for (int s = 0; s < count; ++s) {
            const int length = rng() % 6 == 0 ? 0 : log_uniform(3000.0);
            const int past = rng() % 5 == 0 ? -static_cast<int>(rng() % (length + 1)) : log_uniform(40000.0);
            sequences.push_back({begin, length, length + past});
            begin += length;
        }
        if (check(sequences, 1 + static_cast<int>(rng() % 96)) != 0) {
            return 1;
        }
    }
    // contexts near the end of int
    if (check({{0, 50, 0x7fffffff}, {50, 1, 0x7fffff00}, {51, 1, 1}}, 74) != 0) {
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
