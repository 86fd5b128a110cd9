// How hyp_batch_attention's work is cut (see attention_batch.hip).
//
// A unit is a block of 32 keys for a tile of query rows of one kv head. Tiles are of two kinds: of few rows
// (16, a wave each) and wide (128, a workgroup each; kTileCost units come before a wide tile's blocks, for what it
// costs to begin one). Units of a kind are numbered tile by tile: of few rows the prefix's tiles by kv head, then each
// request's by kv head; wide ones kv head by kv head, in each the prefix's, then request by request. Every
// workgroup finds its units itself from the lengths in device memory, 64 requests at a time across a wave's lanes; the
// launch has a fixed number of workgroups whatever the lengths, each with the same number of consecutive units of
// one kind.
#pragma once

#include "attention.h"
#include "batch.h"
#include "wave.h"

namespace hyperion::hip {

constexpr uint32_t kTileRows = 16;
constexpr uint32_t kComputeUnits = 256;
constexpr uint32_t kMaxParts = 256;     // of one tile: what the merge reads for a row
constexpr uint32_t kTileCost = 4;
constexpr uint32_t kXcds = 8;
constexpr uint32_t kGroupThreads = 256;
constexpr uint32_t kGroupWaves = kGroupThreads / 64u;

// n / d for a divisor that the host knows: n times 2^36 / d rounded up, exact while n d < 2^36 (rows times
// heads are below 2^25, heads at most 2^10). (A division is some 30 instructions, and a wave that takes a block
// or two forms several.)
struct Divisor {
    uint64_t inverse;   // 2^36 / d, rounded up
    uint32_t d;
    Divisor() = default;
    explicit Divisor(uint32_t d_) : inverse(((1ull << 36) + d_ - 1u) / d_), d(d_) {}
    __device__ uint32_t of(uint32_t n) const { return static_cast<uint32_t>((n * inverse) >> 36); }
};

// ceil(n / d): from fp32, then put right.
__device__ __forceinline__ uint32_t ceil_div(uint32_t n, uint32_t d) {
    uint32_t q = static_cast<uint32_t>(static_cast<float>(n) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
    while (static_cast<uint64_t>(q) * d > n) --q;   // q <= n / d
    while (static_cast<uint64_t>(q) * d < n) ++q;
    return q;
}
// floor(n / d), the same way.
__device__ __forceinline__ uint32_t floor_div(uint32_t n, uint32_t d) {
    const uint32_t q = ceil_div(n, d);
    return static_cast<uint64_t>(q) * d > n ? q - 1u : q;
}

// What the attention launch's scribes leave for the merge.
struct Header {
    uint32_t few_per, wide_per;            // units of a wave, of a workgroup; few_per 0: no batch
    uint32_t blocks, tiles;                // the prefix in tiles of few rows
    uint32_t wide_blocks, wide_tiles;      // the prefix in wide tiles
    uint32_t wide_head;                    // units of the wide tiles of one kv head
    uint32_t apart;                        // every request's tiles take the prefix's keys too
    uint32_t unused[8];
};
struct Record {
    uint32_t unit0, tiles, blocks;                 // few rows
    uint32_t wide_unit0, wide_units;               // wide tiles, within a kv head
    uint32_t unused[3];
};
struct RowRecord {
    uint32_t request, row;   // its request, its row there
};

struct BatchParams {
    BatchView b;
    const uint16_t* q;
    const uint16_t* ck;
    const uint16_t* cv;
    uint16_t* out;
    Header* header;
    Record* request;
    RowRecord* row;
    // Unnormalised rows with their (m, l). Tiles that one worker walked whole, by output row: [0] of
    // the prefix, [1] of the own tokens. Otherwise worker w's piece 2 w (its first) or 2 w + 1.
    float2* whole_ml[2];   // [max_rows][H]
    float* whole_o[2];     // [max_rows][H][D]
    float2* part_ml;       // [piece][kTileRows]
    float* part_o;         // [piece][kTileRows][D]
    float2* wide_ml;       // [piece][kChunkRows]
    float* wide_o;         // [piece][kChunkRows][D]
    uint32_t H, KVH, G, window, groups;   // groups: workgroups of the launch
    Divisor by_G;
    float scale;           // with log2(e)
    float wide_cost;       // a workgroup's time for a unit of a wide tile, by that of its waves for one of few rows
};

// A request's (or the prefix's) part of the work for few rows.
struct Source {
    uint32_t row0, rows;   // query rows (tokens)
    uint32_t lo, hi;       // keys [lo, hi) that some row sees
    int32_t pos;           // the first row's position, counted from the source's key 0
    uint32_t tiles, blocks;
    __device__ uint32_t units(uint32_t KVH) const { return KVH * tiles * blocks; }
};

__device__ __forceinline__ uint32_t tiles_of(uint32_t rows, uint32_t G) { return (rows * G + kTileRows - 1u) / kTileRows; }
__device__ __forceinline__ uint32_t wide_tiles_of(uint32_t rows, uint32_t G) { return (rows * G + kChunkRows - 1u) / kChunkRows; }

// sum over i < n of floor((a i + b) / m): the whole parts of a and b over m, then the same sum with m
// and a exchanged. (a n + b below 2^32, the sum too.)
__device__ __forceinline__ uint32_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    uint32_t sum = 0u;
    while (n != 0u) {
        const uint32_t qa = a / m, qb = b / m;
        sum += static_cast<uint32_t>(static_cast<uint64_t>(n) * (n - 1u) / 2u * qa) + n * qb;
        a -= qa * m;
        b -= qb * m;
        const uint32_t top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top - n * m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// The key blocks of a request's wide tiles. Tile k's rows end at position pos0 + (128 k + 127) / G, so its
// blocks end at floor((pos0 + (128 k + 127) / G + 32) / 32), which with pos0 + 32 = 32 q + r is
// end(k) = q + floor((128 k + G r + 127) / 32 G); at most all blocks, and with a window no more than `most`
// of them are seen.
struct WideSpan {
    uint32_t G, all, most, q, c;
    __device__ WideSpan(uint32_t G_, uint32_t keys, int32_t pos0, uint32_t window) : G(G_) {
        all = (keys + kKeyBlock - 1u) / kKeyBlock;
        most = all;
        if (window != 0u) {
            const uint64_t seen = (static_cast<uint64_t>(window) + 127u / G + 63u) / kKeyBlock;
            // (Rows before position 0 are counted from there: their tiles start as much earlier.)
            const uint64_t early = pos0 < 0 ? (31u - static_cast<int64_t>(pos0)) / kKeyBlock : 0u;
            if (seen + early < all) most = static_cast<uint32_t>(seen + early);
        }
        const uint32_t x = static_cast<uint32_t>(max(pos0, 0)) + kKeyBlock;
        q = x / kKeyBlock;
        c = G * (x % kKeyBlock) + 127u;
    }
    __device__ uint32_t end(uint32_t k) const { return min(q + (128u * k + c) / (32u * G), all); }
    __device__ uint32_t units(uint32_t k) const { return min(end(k), most); }
    __device__ uint32_t cost(uint32_t k) const { return units(k) + kTileCost; }
    // Units of the tiles before k, with what they cost: those whose end is below `most`, then `most` each.
    __device__ uint32_t before(uint32_t k) const {
        uint32_t rising = 0u;
        if (most > q) {
            const uint64_t full = 32ull * G * (most - q);
            if (full > c) rising = static_cast<uint32_t>(min(static_cast<uint64_t>(k), (full - c + 127u) >> 7));
        }
        return rising * q + floor_sum(rising, 32u * G, 128u, c) + (k - rising) * most + k * kTileCost;
    }
};

__device__ __forceinline__ Source request_source(const BatchParams& p, uint32_t r) {
    Source s{0u, 0u, 0u, 0u, 0, 0u, 0u};
    if (r >= p.b.requests) return s;
    s.row0 = min(p.b.row_start[r], p.b.max_rows);
    s.rows = max(min(p.b.row_start[r + 1u], p.b.max_rows), s.row0) - s.row0;
    const uint64_t held = min(static_cast<uint64_t>(p.b.max_blocks) << p.b.shift, static_cast<uint64_t>(1u << 30));
    s.hi = min(p.b.lens[r], static_cast<uint32_t>(held));
    s.pos = static_cast<int32_t>(s.hi) - static_cast<int32_t>(s.rows);
    if (p.window != 0u && static_cast<int64_t>(s.pos) + 1 > p.window) s.lo = s.pos + 1u - p.window;
    s.tiles = tiles_of(s.rows, p.G);
    s.blocks = s.rows != 0u && s.hi > s.lo ? (s.hi - s.lo + kKeyBlock - 1u) / kKeyBlock : 0u;
    return s;
}

// The same value in every lane, as a scalar.
__device__ __forceinline__ uint32_t scalar(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); }
__device__ __forceinline__ int32_t scalar(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// The batch as one wave sees it. Which rows go where: rows of one request that fill wide tiles by
// themselves read the prefix there, at one pass over all their keys, where that takes at most a quarter
// more tiles than the rows of all requests together would (apart). Otherwise the prefix is taken for all
// rows together, in wide tiles from 17 rows on, and a request's own tokens in wide tiles where its rows
// pass 16. Without kWide there are no wide tiles.
template <bool kWide>
struct Walk {
    uint32_t rows;              // of all requests
    int32_t first_pos;          // their least position
    bool apart;
    Source prefix;              // the prefix in tiles of few rows (its keys [lo, hi) in either kind)
    uint32_t wide_tiles, wide_lo, wide_blocks;   // and in wide ones
    uint32_t units, wide_units;                  // of all
    uint32_t wide_head_units;                    // of one kv head's wide tiles
    uint32_t wide_groups, wide_per, few_per;     // workgroups 0 .. wide_groups - 1 take wide tiles

    __device__ bool wide(const BatchParams& p, uint32_t n) const { return kWide && (apart || n * p.G > kTileRows); }
    __device__ uint32_t few_units(const BatchParams& p, const Source& s) const { return wide(p, s.rows) ? 0u : s.units(p.KVH); }
    // The keys that a request's wide tiles walk: the prefix's before its own where apart.
    __device__ WideSpan span(const BatchParams& p, const Source& s) const {
        const uint32_t pre = apart ? p.b.prefix : 0u;
        return WideSpan(p.G, pre + s.hi, static_cast<int32_t>(pre) + s.pos, p.window);
    }
    // Units of a request's wide tiles of one kv head. A tile has a block at least: a request without keys has no
    // tiles (the merge finds no pieces of its rows there).
    __device__ uint32_t wide_head(const BatchParams& p, const Source& s) const {
        if (!kWide || s.rows == 0u || !wide(p, s.rows)) return 0u;
        const WideSpan keys = span(p, s);
        return keys.all != 0u ? keys.before(wide_tiles_of(s.rows, p.G)) : 0u;
    }
    __device__ bool has_prefix() const { return prefix.blocks != 0u || wide_blocks != 0u; }
    // Units of the prefix's wide tiles of one kv head.
    __device__ uint32_t prefix_units() const { return wide_blocks != 0u ? wide_tiles * (wide_blocks + kTileCost) : 0u; }
    // The worker for workgroup i. Workgroups go to the XCDs in turn, and each of those has a cache of its own:
    // an XCD takes consecutive workers, whose tiles share keys (24 prompts of 9 to 250 rows behind 6000 tokens, window 1024
    // at head_dim 256: 159 us so, 171 with worker i; 478 and 490 at 128; 718 and 715 at 512).
    __device__ uint32_t worker(uint32_t i) const {
        const uint32_t n = wide_groups / kXcds, more = wide_groups % kXcds;
        const uint32_t x = i % kXcds;
        return x * n + min(x, more) + i / kXcds;
    }

    // False where the row starts are no rows of the batch (they would pass the workspace).
    __device__ bool open(const BatchParams& p, uint32_t lane) {
        const Source mine = request_source(p, lane);
        uint32_t sum = 0u, top = 0u, tiles = 0u;
        int32_t first = 0x7fffffff;
        for (uint32_t r = lane; r < p.b.requests; r += 64u) {
            const Source s = r == lane ? mine : request_source(p, r);
            sum = min(sum + s.rows, 1u << 25);
            top = max(top, s.row0 + s.rows);
            if (kWide) tiles += wide_tiles_of(s.rows, p.G);
            if (s.rows != 0u) first = min(first, s.pos);
        }
        if (wave_sum(sum) > p.b.max_rows) return false;
        rows = wave_max(top);
        first_pos = wave_min(first);
        apart = kWide && rows * p.G > kTileRows && 4u * wave_sum(tiles) <= 5u * wide_tiles_of(rows, p.G);
        uint32_t n = 0u, most = 0u, wide_n = 0u, wide_most = 0u;
        for (uint32_t r = lane; r < p.b.requests; r += 64u) {
            const Source s = r == lane ? mine : request_source(p, r);
            if (s.rows == 0u) continue;
            if (wide(p, s.rows)) {
                wide_n += wide_head(p, s);
                wide_most = max(wide_most, ((apart ? p.b.prefix : 0u) + s.hi) / kKeyBlock + 1u);
            } else {
                n += s.units(p.KVH);
                most = max(most, s.blocks);
            }
        }
        prefix = Source{0u, rows, 0u, p.b.prefix, 0, tiles_of(rows, p.G), 0u};
        wide_tiles = wide_lo = wide_blocks = 0u;
        if (rows != 0u && !apart) {
            first_pos += static_cast<int32_t>(p.b.prefix);
            prefix.pos = first_pos;
            if (p.window != 0u && static_cast<int64_t>(first_pos) + 1 > p.window) prefix.lo = first_pos + 1u - p.window;
            if (prefix.hi > prefix.lo) {
                if (wide(p, rows)) {
                    wide_tiles = wide_tiles_of(rows, p.G);
                    wide_lo = prefix.lo / kKeyBlock;
                    wide_blocks = (prefix.hi + kKeyBlock - 1u) / kKeyBlock - wide_lo;
                } else {
                    prefix.blocks = (prefix.hi - prefix.lo + kKeyBlock - 1u) / kKeyBlock;
                }
            }
        }
        most = max(wave_max(most), prefix.blocks);
        units = wave_sum(n) + prefix.units(p.KVH);
        wide_head_units = kWide ? prefix_units() : 0u;
        if (kWide && rows * p.G > kTileRows) {
            wide_head_units += wave_sum(wide_n);
            wide_most = max(wave_max(wide_most), wide_blocks);
        }
        wide_units = p.KVH * wide_head_units;
        wide_groups = 0u;
        wide_per = 1u;
        if (kWide && wide_units != 0u) {
            wide_groups = p.groups;
            if (units != 0u) {
                const float cost = static_cast<float>(wide_units) * p.wide_cost;
                const float share = cost * __builtin_amdgcn_rcpf(cost + static_cast<float>(units));
                wide_groups = min(max(static_cast<uint32_t>(static_cast<float>(p.groups) * share), 1u), p.groups - 1u);
            }
            wide_per = max(ceil_div(wide_units, wide_groups), (wide_most + kTileCost + kMaxParts - 2u) / (kMaxParts - 1u));
            wide_groups = ceil_div(wide_units, wide_per);
        }
        const uint32_t waves = max((p.groups - wide_groups) * kGroupWaves, 1u);
        few_per = max(max(ceil_div(units, waves), (most + kMaxParts - 2u) / (kMaxParts - 1u)), 1u);
        return true;
    }
};

// Requests 64 at a time, with running sums of their units of one kind.
template <typename W>
struct Chunk {
    Source mine;       // this lane's request
    uint32_t base;     // the first request
    uint32_t before;   // units before it
    uint32_t incl;     // with this lane's request
    uint32_t own;      // this lane's units (of wide tiles: in one kv head)
    bool wide;

    __device__ void load(const BatchParams& p, const W& w, uint32_t lane) {
        mine = request_source(p, base + lane);
        own = wide ? w.wide_head(p, mine) : w.few_units(p, mine);
        incl = wave_incl(own);
    }
    __device__ void open(const BatchParams& p, const W& w, uint32_t lane, bool wide_) {
        wide = wide_;
        base = 0u;
        before = wide ? w.prefix_units() : w.prefix.units(p.KVH);
        load(p, w, lane);
    }
    __device__ void next(const BatchParams& p, const W& w, uint32_t lane) {
        before += from_lane(incl, 63u);
        base += 64u;
        load(p, w, lane);
    }
    // The lane whose request holds unit u (u >= before); 64 where none does.
    __device__ uint32_t seek(const BatchParams& p, const W& w, uint32_t u, uint32_t lane) {
        while (base + 64u < p.b.requests && u >= before + from_lane(incl, 63u))
            next(p, w, lane);
        const uint64_t behind = __ballot(u < before + incl);
        return behind == 0u ? 64u : static_cast<uint32_t>(__builtin_ctzll(behind));
    }
};

__device__ __forceinline__ Source source_of_lane(const Source& s, uint32_t from) {
    return Source{from_lane(s.row0, from), from_lane(s.rows, from),  from_lane(s.lo, from),    from_lane(s.hi, from),
                  __builtin_amdgcn_readlane(s.pos, from), from_lane(s.tiles, from), from_lane(s.blocks, from)};
}

// Position of token row t, whatever its request (counted from the prefix's key 0).
__device__ __forceinline__ int32_t row_position(const BatchParams& p, uint32_t t) {
    uint32_t lo = 0u, hi = p.b.requests;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (p.b.row_start[mid] <= t) lo = mid; else hi = mid;
    }
    const Source s = request_source(p, lo);
    return static_cast<int32_t>(p.b.prefix) + s.pos + static_cast<int32_t>(t - s.row0);
}

// What the merge needs: a wave writes 64 requests and their rows.
template <bool kWide>
__device__ __forceinline__ void scribe(const BatchParams& p, uint32_t chunk, uint32_t lane) {
    Walk<kWide> w;
    if (!w.open(p, lane)) {
        if (chunk == 0u && lane == 0u) *p.header = Header{};
        return;
    }
    if (chunk == 0u && lane == 0u) {
        *p.header = Header{w.few_per, w.wide_per, w.prefix.blocks, w.prefix.tiles, w.wide_blocks, w.wide_tiles, w.wide_head_units, w.apart ? 1u : 0u, {}};
    }
    if (chunk >= p.b.requests) return;
    Chunk<Walk<kWide>> few, wide;
    few.open(p, w, lane, false);
    wide.open(p, w, lane, true);
    while (few.base < chunk) {
        few.next(p, w, lane);
        wide.next(p, w, lane);
    }
    const Source s = few.mine;
    const bool is_wide = w.wide(p, s.rows);
    if (chunk + lane < p.b.requests) {
        p.request[chunk + lane] = Record{few.before + few.incl - few.own, s.tiles, is_wide ? 0u : s.blocks,
                                         wide.before + wide.incl - wide.own, wide.own, {}};
    }
    for (uint32_t i = 0; i < 64u; ++i) {
        const uint32_t row0 = from_lane(s.row0, i);
        const uint32_t n = from_lane(s.rows, i);
        for (uint32_t t = lane; t < n; t += 64u) p.row[row0 + t] = RowRecord{chunk + i, t};
    }
}

// Where a segment's rows go: to the output (all their keys were in it), by output row, or to a piece.
enum : uint32_t { kToOutput = 0u, kToRows = 1u, kToPiece = 2u };

// The keys that a tile walks, positions 0 .. keys - 1: `pre` of the prefix's tokens, then own ones.
struct Sequence {
    const uint32_t* own;   // the request's row of tables
    uint32_t pre, keys;
    uint32_t row0, rows;   // query rows (tokens)
    int32_t pos;           // the first one's position among the keys
    bool by_request;       // rows of all requests: pos is their least position
};

// A workgroup's units of wide tiles: segment(sequence, kv head, tile, its blocks [b0, b1), where to, piece) of each
// tile in turn, and nothing(piece) for a piece without blocks.
template <typename Segment, typename Nothing>
__device__ __forceinline__ void wide_units(const BatchParams& p, uint32_t worker, uint32_t begin, uint32_t end, uint32_t lane,
                                           Segment&& segment, Nothing&& nothing) {
    uint32_t u = begin;
    while (u < end) {
        // (Formed again for each tile rather than kept in registers beside the tile's.)
        Walk<true> w;
        if (!w.open(p, lane)) return;
        Sequence s{nullptr, p.b.prefix, p.b.prefix, 0u, w.rows, w.first_pos, true};
        const uint32_t hk = floor_div(u, w.wide_head_units);
        const uint32_t in_head = u - hk * w.wide_head_units;
        uint32_t tile, off, blocks, block0;   // off: units before u, with kTileCost before the blocks
        if (in_head < w.prefix_units()) {
            blocks = w.wide_blocks;
            block0 = w.wide_lo;
            tile = floor_div(in_head, blocks + kTileCost);
            off = in_head - tile * (blocks + kTileCost);
        } else {
            Chunk<Walk<true>> c;
            c.open(p, w, lane, true);
            const uint32_t at = c.seek(p, w, in_head, lane);
            if (at == 64u) return;   // (not with u below the total)
            const Source src = source_of_lane(c.mine, at);
            const uint32_t x = in_head - (c.before + from_lane(c.incl, at) - from_lane(c.own, at));
            s.own = p.b.tables + static_cast<size_t>(c.base + at) * p.b.max_blocks;
            s.pre = w.apart ? p.b.prefix : 0u;
            s.keys = s.pre + src.hi;
            s.row0 = src.row0;
            s.rows = src.rows;
            s.pos = static_cast<int32_t>(s.pre) + src.pos;
            s.by_request = false;
            const WideSpan span = w.span(p, src);
            uint32_t t0 = 0u, t1 = wide_tiles_of(src.rows, p.G);   // the last tile with before() <= x
            while (t1 - t0 > 1u) {
                const uint32_t mid = (t0 + t1) / 2u;
                if (span.before(mid) <= x) t0 = mid; else t1 = mid;
            }
            tile = t0;
            off = x - span.before(tile);
            blocks = span.units(tile);
            block0 = span.end(tile) - blocks;
        }
        const uint32_t take = min(blocks + kTileCost - off, end - u);
        const bool complete = !s.by_request && !w.has_prefix();
        const uint32_t to = take < blocks + kTileCost ? kToPiece : (complete ? kToOutput : kToRows);
        const uint32_t piece = 2u * worker + (u == begin ? 0u : 1u);
        const uint32_t b0 = max(off, kTileCost) - kTileCost;
        const uint32_t b1 = max(off + take, kTileCost) - kTileCost;
        if (b0 < b1) {
            segment(s, scalar(hk), scalar(tile), scalar(block0 + b0), scalar(block0 + b1), to, piece);
        } else {
            nothing(piece);
        }
        u = scalar(u + take);
    }
}

// A wave's units of tiles of few rows: segment(source, its table, whether that is the prefix, kv head, tile, its blocks
// [b0, b1), where to, piece).
template <typename W, typename Segment>
__device__ __forceinline__ void few_units(const BatchParams& p, const W& w, uint32_t worker, uint32_t begin, uint32_t end,
                                          uint32_t lane, Segment&& segment) {
    Chunk<W> c;
    c.open(p, w, lane, false);
    uint32_t u = begin;
    while (u < end) {
        Source s = w.prefix;
        const uint32_t* table = p.b.prefix_table;
        uint32_t unit0 = 0u;
        const bool is_prefix = u < w.prefix.units(p.KVH);
        if (!is_prefix) {
            const uint32_t at = c.seek(p, w, u, lane);
            if (at == 64u) return;   // (not with u below the total)
            s = source_of_lane(c.mine, at);
            table = p.b.tables + static_cast<size_t>(c.base + at) * p.b.max_blocks;
            unit0 = c.before + from_lane(c.incl, at) - s.units(p.KVH);
        }
        const uint32_t g = floor_div(u - unit0, s.blocks);
        const uint32_t b0 = u - unit0 - g * s.blocks;
        const uint32_t b1 = min(s.blocks, b0 + (end - u));
        const uint32_t hk = floor_div(g, s.tiles);
        const uint32_t to = b1 - b0 < s.blocks ? kToPiece : (!is_prefix && !w.has_prefix() ? kToOutput : kToRows);
        segment(s, table, is_prefix, scalar(hk), scalar(g - hk * s.tiles), scalar(b0), scalar(b1), to,
                2u * worker + (u == begin ? 0u : 1u));
        u += b1 - b0;
    }
}

// The units of wave `wave` of workgroup `group`. Every wave of a workgroup that takes wide tiles goes through all of
// its units.
template <bool kWide, typename Wide, typename Nothing, typename Few>
__device__ __forceinline__ void worker_units(const BatchParams& p, uint32_t group, uint32_t wave, uint32_t lane, Wide&& wide,
                                             Nothing&& nothing, Few&& few) {
    Walk<kWide> w;
    if (!w.open(p, lane)) return;
    if (kWide && group < w.wide_groups) {
        const uint32_t worker = scalar(w.worker(group));
        const uint32_t begin = worker * w.wide_per;
        wide_units(p, worker, begin, min(begin + w.wide_per, w.wide_units), lane, wide, nothing);
    } else {
        const uint32_t worker = (group - w.wide_groups) * kGroupWaves + wave;
        const uint64_t begin = static_cast<uint64_t>(worker) * w.few_per;
        if (begin >= w.units) return;   // (no barrier follows)
        few_units(p, w, worker, static_cast<uint32_t>(begin), min(static_cast<uint32_t>(begin) + w.few_per, w.units), lane,
                  few);
    }
}

// Where a row's pieces lie, of the prefix or of its own tokens.
struct Pieces {
    uint32_t count;    // 0: no keys there
    uint32_t place;    // the first worker's piece, then 2 (first + 1), 2 (first + 2), ...
    uint32_t next;     // 2 (first + 1)
    uint32_t at;       // the row's place in its tile
    bool wide;

    __device__ void set(uint32_t unit0, uint32_t blocks, uint32_t per, uint32_t row, bool wide_) {
        const uint32_t tile_rows = wide_ ? kChunkRows : kTileRows;
        at = row % tile_rows;
        wide = wide_;
        count = 0u;
        if (blocks == 0u) return;
        const uint32_t first = floor_div(unit0, per);
        count = floor_div(unit0 + blocks - 1u, per) - first + 1u;
        place = 2u * first + (first * per < unit0 ? 1u : 0u);
        next = 2u * first + 2u;
    }
};

// The pieces of head h of row t, of the prefix (a) and of its own tokens (b); false where the output has that row already,
// or no request has it.
__device__ __forceinline__ bool row_pieces(const BatchParams& p, uint32_t t, uint32_t h, Pieces& a, Pieces& b) {
    const Header head = *p.header;
    const RowRecord row = p.row[t];
    // (Row starts that skip a row leave its record unwritten.)
    if (head.few_per == 0u || row.request >= p.b.requests || p.b.row_start[row.request] + row.row != t ||
        t >= p.b.row_start[row.request + 1u]) {
        return false;
    }
    const Record own = p.request[row.request];
    const uint32_t hk = p.by_G.of(h);
    const uint32_t pr = t * p.G + (h - hk * p.G);           // its row among all rows of the kv head
    const uint32_t orow = row.row * p.G + (h - hk * p.G);   // and among its request's
    if (head.wide_blocks != 0u) {
        const uint32_t cost = head.wide_blocks + kTileCost;
        a.set(hk * head.wide_head + pr / kChunkRows * cost, cost, head.wide_per, pr, true);
    } else {
        a.set((hk * head.tiles + pr / kTileRows) * head.blocks, head.blocks, head.few_per, pr, false);
    }
    if (own.wide_units != 0u) {
        const Source src = request_source(p, row.request);
        const uint32_t pre = head.apart != 0u ? p.b.prefix : 0u;
        const WideSpan span(p.G, pre + src.hi, static_cast<int32_t>(pre) + src.pos, p.window);
        const uint32_t tile = orow / kChunkRows;
        b.set(hk * head.wide_head + own.wide_unit0 + span.before(tile), span.cost(tile), head.wide_per, orow, true);
    } else {
        b.set(own.unit0 + (hk * own.tiles + orow / kTileRows) * own.blocks, own.blocks, head.few_per, orow, false);
    }
    return b.count != 1u || (head.apart == 0u && (head.blocks != 0u || head.wide_blocks != 0u));
}

}  // namespace hyperion::hip
