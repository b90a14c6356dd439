// How the attention of a batch of chunks is dealt out.  Plain arithmetic, the same on the device and on the host.
//
// An item is a tile of kItemTokens tokens of one chunk with one KV head; its units are the 128 positions of cache that go
// through the tensor cores at once, up to the last position that the tile's last token sees.  All items lie on a line,
// (sequence, head, tile) in order, each a lead of kItemLead and then its units: the lead is what an item costs besides, in
// units (2048 tokens: 80.5 us with a lead of 8, 81.9 with 6, 81.7 with 10; 13 chunks of a ragged batch: 86.4, 93.8, 91.7).
// Worker w of n has positions total * w / n .. total * (w + 1) / n: every worker the same work, whatever the lengths are
// (of a short line fewer workers have kSmallestShare each).  What of an item's units lies in a worker's share is a piece;
// pieces of an item that is cut are merged afterwards.  The lead stands in front, so the workers that have pieces of
// an item follow one another: from the one that has its first unit to the one that has the end of its line.

#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define QWC_CHUNK_PLAN_FUNCTION __host__ __device__ __forceinline__
#else
#define QWC_CHUNK_PLAN_FUNCTION inline
#endif

namespace qwc {

constexpr int kItemTokens = 42;
constexpr int kItemLead = 8;
constexpr int kSmallestShare = 4;
constexpr int kPlanUnitTokens = 128;
constexpr int kPlanHeads = 4;

struct ChunkSequence {
    int begin;    // first row
    int length;   // rows; none: no items
    int context;  // positions of the cache, the chunk's own among them
};

QWC_CHUNK_PLAN_FUNCTION int item_tiles(const ChunkSequence& s) { return (s.length + kItemTokens - 1) / kItemTokens; }

// Units of a tile; one at least, so that rows that see nothing are written too.
QWC_CHUNK_PLAN_FUNCTION int item_units(const ChunkSequence& s, int tile) {
    const int last = (tile + 1) * kItemTokens < s.length ? (tile + 1) * kItemTokens : s.length;
    const long long visible = static_cast<long long>(s.context) - s.length + last;
    return visible <= kPlanUnitTokens ? 1 : static_cast<int>((visible + kPlanUnitTokens - 1) / kPlanUnitTokens);
}

QWC_CHUNK_PLAN_FUNCTION int plan_workers(long long total, int workers) {
    const long long most = total / kSmallestShare;
    return most >= workers ? workers : most < 1 ? 1 : static_cast<int>(most);
}

// a / b; of 32 bits where they do (a division of 64 is a few hundred cycles).
QWC_CHUNK_PLAN_FUNCTION long long plan_divide(long long a, long long b) {
    if (a <= 0xffffffffll && b <= 0xffffffffll) {
        return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    }
    return a / b;
}

// (A line is below 2^37: 1689 tiles at most of 2^16 tokens, 4 heads, 2^24 units.)
QWC_CHUNK_PLAN_FUNCTION long long share_begin(long long total, int worker, int workers) {
    return plan_divide(total * worker, workers);
}

// The worker whose share holds `position` (below total): the last one with total * worker / workers < position + 1.
QWC_CHUNK_PLAN_FUNCTION int worker_of(long long total, long long position, int workers) {
    return static_cast<int>(plan_divide((position + 1) * workers - 1, total));
}

struct ChunkPiece {
    int unit_begin;
    int unit_end;
    int units;  // of the whole item
};

// Where a worker stands on the line.
struct ChunkWalk {
    int sequence, head, tile;
    long long skip;      // positions of the item at hand that lie before the worker's share
    long long left;      // positions of the share from there on
    long long item_end;  // line position behind the item of the piece handed out last
    long long at;        // line position of the item at hand
    ChunkSequence info;  // of `sequence`
};

// The next piece of the share that has units; false: there is none.  `sequence_info(s)` gives a ChunkSequence.
// The piece's item is w.sequence, w.head, w.tile until the next call, which goes on from there (`first`: the first call).
template <typename Info>
QWC_CHUNK_PLAN_FUNCTION bool next_piece(ChunkWalk& w, bool first, int sequences, const Info& sequence_info, ChunkPiece& piece) {
    for (bool moved = !first;; moved = true) {
        if (w.left <= 0) {
            return false;
        }
        if (moved) {
            if (++w.tile >= item_tiles(w.info)) {
                w.tile = 0;
                if (++w.head == kPlanHeads) {
                    w.head = 0;
                    do {
                        if (++w.sequence >= sequences) {
                            w.left = 0;
                            return false;
                        }
                        w.info = sequence_info(w.sequence);
                    } while (w.info.length == 0);
                }
            }
        }
        piece.units = item_units(w.info, w.tile);
        const long long length = piece.units + kItemLead;
        const long long take = w.left < length - w.skip ? w.left : length - w.skip;
        piece.unit_begin = w.skip > kItemLead ? static_cast<int>(w.skip - kItemLead) : 0;
        piece.unit_end = w.skip + take > kItemLead ? static_cast<int>(w.skip + take - kItemLead) : 0;
        w.left -= take;
        w.item_end = w.at + length;
        w.at = w.item_end;
        w.skip = 0;
        if (piece.unit_begin < piece.unit_end) {
            return true;
        }
    }
}

}  // namespace qwc
