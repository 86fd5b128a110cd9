// hyp_batch_attention's schedule (csrc/attention_batch_walk.h) run on the host: every worker's tiles as they would be
// walked and the pieces that the merge would join, checked against each other and against the keys that each row sees,
// for test_batch_walk_cpu.py.
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <map>
#include <memory>
#include <set>
#include <string>
#include <tuple>

#include "attention_batch_walk.h"

using namespace hyperion::hip;

namespace {

struct Fault : std::runtime_error {
    using std::runtime_error::runtime_error;
};

[[noreturn]] void fail(const char* format, ...) {
    char text[400];
    va_list args;
    va_start(args, format);
    vsnprintf(text, sizeof text, format, args);
    va_end(args);
    throw Fault(text);
}

struct Segment {
    uint32_t b0, b1, to, piece;
};

// A tile: wide or of few rows, its request (-1: the prefix), kv head, number.
using Tile = std::tuple<bool, int, uint32_t, uint32_t>;

template <bool kWide>
void check(BatchParams p, bool ordered) {
    const BatchView& b = p.b;
    std::vector<Record> request(b.requests + 1u, Record{});
    std::vector<RowRecord> row(b.max_rows + 1u, RowRecord{0xFFFFFFFFu, 0xFFFFFFFFu});
    const RowRecord guard = row.back();
    auto header = std::make_unique<Header>();
    std::memset(header.get(), 0xFF, sizeof(Header));
    p.request = request.data();
    p.row = row.data();
    p.header = header.get();

    std::map<Tile, std::vector<Segment>> tiles;
    std::map<Tile, Source> sources;
    std::set<uint32_t> few_pieces, wide_pieces;
    const auto piece_once = [&](bool wide, uint32_t piece) {
        const uint32_t end = 2u * p.groups * (wide ? 1u : kGroupWaves);
        if (piece >= end) fail("piece %u of %u (%s)", piece, end, wide ? "wide" : "few rows");
        if (!(wide ? wide_pieces : few_pieces).insert(piece).second) fail("piece %u twice", piece);
    };
    const auto rows_inside = [&](uint32_t row0, uint32_t rows, uint32_t hk, uint32_t tile, uint32_t tile_rows) {
        if (row0 > b.max_rows || rows > b.max_rows - row0) fail("rows %u + %u of %u", row0, rows, b.max_rows);
        if (hk >= p.KVH) fail("kv head %u of %u", hk, p.KVH);
        if (static_cast<uint64_t>(tile) * tile_rows >= static_cast<uint64_t>(rows) * p.G)
            fail("tile %u of %u rows", tile, rows * p.G);
    };
    const auto keys_inside = [&](int r, uint32_t keys) {   // own keys (r >= 0), or the prefix's
        const uint64_t held = r < 0 ? b.prefix : static_cast<uint64_t>(b.max_blocks) << b.shift;
        if (keys == 0u || keys > held) fail("%u keys of %llu", keys, static_cast<unsigned long long>(held));
    };
    // The request of a tile's rows, whose table it must be.
    const auto request_of = [&](uint32_t row0, uint32_t rows, const uint32_t* table) -> int {
        for (uint32_t r = 0; r < b.requests; ++r) {
            if (std::min(b.row_start[r], b.max_rows) != row0 || b.row_start[r + 1u] <= row0 ||
                std::min(b.row_start[r + 1u], b.max_rows) - row0 != rows) {
                continue;
            }
            if (table == b.tables + static_cast<size_t>(r) * b.max_blocks) return static_cast<int>(r);
        }
        fail("rows %u + %u with a table of no request's", row0, rows);
    };

    for (uint32_t chunk = 0; chunk <= b.requests; chunk += 64u)
        host_wave::run([&](uint32_t lane) { scribe<kWide>(p, chunk, lane); });
    if (row.back().request != guard.request) fail("a row record behind the last");
    for (uint32_t group = 0; group < p.groups; ++group) {
        for (uint32_t wave = 0; wave < kGroupWaves; ++wave) {
            bool wide_group = false;
            host_wave::run([&](uint32_t lane) {
                worker_units<kWide>(
                    p, group, wave, lane,
                    [&](const Sequence& s, uint32_t hk, uint32_t tile, uint32_t b0, uint32_t b1, uint32_t to, uint32_t piece) {
                        wide_group = true;
                        if (lane != 0u) return;
                        const int r = s.by_request ? -1 : request_of(s.row0, s.rows, s.own);
                        rows_inside(s.row0, s.rows, hk, tile, kChunkRows);
                        if (s.pre != 0u) keys_inside(-1, s.pre);
                        if (s.keys > s.pre) keys_inside(r, s.keys - s.pre);
                        if (s.keys == 0u || b0 >= b1 || b1 > (s.keys + kKeyBlock - 1u) / kKeyBlock) fail("blocks %u .. %u", b0, b1);
                        if (to == kToPiece) piece_once(true, piece);
                        tiles[{true, r, hk, tile}].push_back({b0, b1, to, piece});
                        Source at{s.row0, s.rows, 0u, s.keys, s.pos, 0u, 0u};
                        sources[{true, r, hk, tile}] = at;
                    },
                    [&](uint32_t piece) {
                        wide_group = true;
                        if (lane == 0u) piece_once(true, piece);
                    },
                    [&](const Source& s, const uint32_t* table, bool is_prefix, uint32_t hk, uint32_t tile, uint32_t b0,
                        uint32_t b1, uint32_t to, uint32_t piece) {
                        if (lane != 0u) return;
                        const int r = is_prefix ? -1 : request_of(s.row0, s.rows, table);
                        rows_inside(s.row0, s.rows, hk, tile, kTileRows);
                        keys_inside(r, s.hi);
                        if (s.lo >= s.hi || b0 >= b1 || s.lo + (b1 - 1u) * kKeyBlock >= s.hi) fail("blocks %u .. %u", b0, b1);
                        if (to == kToPiece) piece_once(false, piece);
                        tiles[{false, r, hk, tile}].push_back({b0, b1, to, piece});
                        sources[{false, r, hk, tile}] = s;
                    });
            });
            if (wide_group) break;   // (its waves go through the same tiles)
        }
    }
    if (!ordered) return;

    const uint32_t last_row = b.row_start[b.requests];
    std::vector<int> request_at(b.max_rows, -1);
    for (uint32_t r = 0; r < b.requests; ++r)
        for (uint32_t t = b.row_start[r]; t < b.row_start[r + 1u]; ++t) request_at[t] = static_cast<int>(r);
    std::set<Tile> merged;
    for (uint32_t t = 0; t < b.max_rows; ++t) {
        for (uint32_t h = 0; h < p.H; ++h) {
            const int r = request_at[t];
            Pieces found[2] = {};
            const bool todo = t < last_row && row_pieces(p, t, h, found[0], found[1]);
            if (r < 0) {
                if (todo) fail("row %u of no request is joined", t);
                continue;
            }
            const uint32_t hk = h / p.G, i = t - b.row_start[r];
            const uint64_t held = static_cast<uint64_t>(b.max_blocks) << b.shift;
            const int64_t own = static_cast<int64_t>(std::min<uint64_t>(b.lens[r], held));
            const int64_t pre = b.prefix;
            const int64_t n = b.row_start[r + 1u] - b.row_start[r];
            const int64_t pos = pre + own - n + i;
            const int64_t seen0 = p.window != 0u ? std::max<int64_t>(0, pos + 1 - p.window) : 0;
            const int64_t seen1 = std::min(pos + 1, pre + own);   // it sees [seen0, seen1)
            const bool apart = header->apart != 0u;
            const uint32_t at_all = t * p.G + h % p.G, at_own = i * p.G + h % p.G;
            // Its tiles: of the prefix, of its own tokens (with the prefix's before them where apart), in the kind that
            // was walked.
            for (int side = 0; side < 2; ++side) {
                const uint32_t at = side == 0 ? at_all : at_own;
                const std::vector<Segment>* segments = nullptr;
                Tile tile;
                Source src{};
                for (const bool wide : {false, true}) {
                    const Tile x{wide, side == 0 ? -1 : r, hk, at / (wide ? kChunkRows : kTileRows)};
                    const auto found_tile = tiles.find(x);
                    if (found_tile == tiles.end()) continue;
                    if (segments != nullptr) fail("row %u head %u in tiles of both kinds", t, h);
                    segments = &found_tile->second;
                    tile = x;
                    src = sources[x];
                }
                // The keys of this side that the row sees are in its segments, each once.
                const int64_t from = side == 0 ? 0 : (apart ? 0 : pre);
                const int64_t to = side == 0 ? (apart ? 0 : pre) : pre + own;
                const int64_t need0 = std::max(seen0, from), need1 = std::min(seen1, to);
                std::vector<std::pair<int64_t, int64_t>> ranges;
                if (segments != nullptr) {
                    for (const Segment& s : *segments)
                        ranges.emplace_back(from + src.lo + int64_t{kKeyBlock} * s.b0,
                                            std::min(from + src.lo + int64_t{kKeyBlock} * s.b1, from + src.hi));
                    std::sort(ranges.begin(), ranges.end());
                    for (size_t k = 1; k < ranges.size(); ++k)
                        if (ranges[k].first != ranges[k - 1u].second) fail("row %u head %u: key blocks twice or left out", t, h);
                    if (src.row0 + (side == 0 ? t : i) != t) fail("row %u head %u stands elsewhere", t, h);
                    const int64_t place = (side == 0 || apart ? pre : 0) + own - n;
                    if (side == 1 && src.pos != place) fail("row %u stands at %d, not %lld", t, src.pos, static_cast<long long>(place));
                }
                if (need0 < need1 && (ranges.empty() || ranges.front().first > need0 || ranges.back().second < need1))
                    fail("row %u head %u side %d: keys %lld .. %lld are not walked", t, h, side, static_cast<long long>(need0),
                         static_cast<long long>(need1));
                // What was written is what the merge reads.
                if (!todo) {
                    if (side == 0 ? segments != nullptr : segments == nullptr || segments->size() != 1u || (*segments)[0].to != kToOutput)
                        fail("row %u head %u is not joined and not whole", t, h);
                    continue;
                }
                const Pieces& f = found[side];
                if (f.count == 0u) {
                    if (segments != nullptr) fail("row %u head %u: the merge leaves out its pieces", t, h);
                    continue;
                }
                if (f.at != at % (f.wide ? kChunkRows : kTileRows)) fail("row %u head %u at %u of its tile", t, h, f.at);
                if (f.count == 1u) {
                    if (segments == nullptr || segments->size() != 1u || (*segments)[0].to != kToRows || std::get<0>(tile) != f.wide)
                        fail("row %u head %u: the merge reads rows that were not written", t, h);
                    continue;
                }
                if (f.count > kMaxParts) fail("%u pieces", f.count);
                std::set<uint32_t> read;
                for (uint32_t w = 0; w < f.count; ++w) read.insert(w == 0u ? f.place : f.next + 2u * (w - 1u));
                for (const uint32_t x : read)
                    if ((f.wide ? wide_pieces : few_pieces).count(x) == 0u) fail("row %u head %u: piece %u was not written", t, h, x);
                if (segments == nullptr) fail("row %u head %u: pieces of no tile", t, h);
                for (const Segment& s : *segments)
                    if (s.to != kToPiece || read.count(s.piece) == 0u) fail("row %u head %u: piece %u is not joined", t, h, s.piece);
            }
        }
    }
}

}  // namespace

// A batch's schedule for `groups` workgroups; 0, or 1 and what is wrong. ordered: the row starts do not decrease and end
// within max_rows (otherwise only the bounds are checked).
extern "C" int check_walk(const HypBatch* batch, uint32_t H, uint32_t KVH, uint32_t window, uint32_t groups, float wide_cost,
                          int wide, int ordered, char* message) {
    BatchParams p{};
    uint32_t shift = 0;
    while ((1u << shift) < batch->block_size) ++shift;
    p.b = {batch->requests, shift,         batch->num_blocks, batch->max_blocks, batch->max_rows, batch->prefix_len,
           batch->prefix_table, batch->tables, batch->lens,   batch->row_start,  batch->slots,    batch->positions};
    p.H = H;
    p.KVH = KVH;
    p.G = H / KVH;
    p.window = window;
    p.groups = groups;
    p.by_G = Divisor(p.G);
    p.wide_cost = wide_cost;
    try {
        if (wide) check<true>(p, ordered != 0); else check<false>(p, ordered != 0);
    } catch (const std::exception& e) {
        snprintf(message, 400, "%s", e.what());
        return 1;
    }
    return 0;
}
