// Attention of a batch of requests over a paged cache, behind a prefix that all of them share
// (hyp_batch_attention): request r's row i stands at pos = prefix + len_r - n_r + i and sees the
// key positions p <= pos (with a window: p > pos - window) among the prefix's tokens and its own,
//   out = sum_p 2^(s_p - m) v_p / sum_p 2^(s_p - m),   s_p = scale log2(e) q.k_p,
// with no key visible: zeros. A sum over keys splits anywhere (each part keeps its own maximum m,
// sum l and unnormalised O, and parts join as sum_i 2^(m_i - m) O_i), so the prefix is taken for
// all rows of the batch at once, each request's own tokens for its rows, and the parts are joined.
//
// Work is cut evenly whatever the lengths: a unit is a block of 32 keys for a tile of query rows
// of one kv head (a group: the prefix's tiles, then request by request), and each of a fixed number of
// workers takes the same number of consecutive units. A worker that crosses from one group to the
// next leaves a part for each; part w + g (worker, group) is its place, different for every pair
// of the walk. Lengths live on the device, so every worker finds its units itself from the
// running sums over the requests, 64 requests at a time across its lanes.
//
// The kernel for few rows (attn_batch_rows_kernel): a worker is one wave, a tile 16 query rows of
// 16x16x32 products, transposed: S^T = K Q^T with the keys' rows straight from memory as the A
// operand, so a lane holds 8 of a block's keys for one query row and its probabilities are the B
// operand of O^T = V^T P^T as they stand. V rows go to the wave's own LDS (16-byte loads with the
// LDS as destination, chunks XOR-swizzled) and come back by transposing reads. The next block's K
// rows are requested before this one's softmax, its table entries a block earlier.
// Probabilities enter as two bf16 terms (p and what its rounding left): the products wait for
// memory here, and one term alone would add the error of a second rounding to the output's.
//
// What bounds it: HBM, each key row read once for up to 16 query rows.
#include <algorithm>

#include "attention.h"
#include "attention_tile.h"
#include "batch.h"
#include "common.h"
#include "q4_rmsnorm.h"

namespace hyperion::hip {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kTileRows = 16;
constexpr uint32_t kComputeUnits = 256;
constexpr uint32_t kMaxParts = 256;     // of one group: what a merge reads for a row
constexpr uint32_t kMergeThreads = 256;
constexpr uint32_t kScribeRequests = 64;

// What the first launch's scribes leave for the others.
struct Header {
    uint32_t per, blocks, tiles;         // few rows: units a worker; the prefix's blocks and tiles
    uint32_t wide_per, wide_units;       // wide tiles: units a worker, of all
    uint32_t wide_lo, wide_blocks, wide_tiles;   // the prefix's first block, blocks and tiles there
    uint32_t apart;                      // every request's tiles take the prefix's keys too
    uint32_t rows;                       // of all requests
    uint32_t unused[6];
};
struct Record {
    uint32_t unit0, tiles, blocks;                 // few rows
    uint32_t wide_unit0, wide_tiles, wide_head;    // wide tiles; units of one kv head
    uint32_t unused[2];
};
struct RowRecord {
    uint32_t request, row;   // its request, its row there
    int32_t pos;             // its position
    uint32_t unused;
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
    // the prefix, [1] of the own tokens. Otherwise the worker's piece 2 w (its first) or 2 w + 1.
    float2* whole_ml[2];   // [max_rows][H]
    float* whole_o[2];     // [max_rows][H][D]
    float2* part_ml;       // [piece][kTileRows]
    float* part_o;         // [piece][kTileRows][D]
    float2* wide_ml;       // [piece][kChunkRows]
    float* wide_o;         // [piece][kChunkRows][D]
    uint32_t H, KVH, G, window, workers, wide_workers;
    float scale;        // with log2(e)
};

// One wave in a workgroup: its LDS holds V rows of a block of 32 keys.
template <uint32_t D>
struct RowsLds {
    static constexpr uint32_t kRow = D * 2u;
    static constexpr uint32_t kChunks = D / 8u;
    static constexpr uint32_t kBytes = kKeyBlock * kRow;
    static constexpr uint32_t kWaves = D >= 512u ? 4u : (D == 256u ? 8u : (D == 128u ? 12u : 16u));   // of a compute unit
    // A transposing read takes 16 rows (4 kb + 0..3) at one pair of chunks: rows 8 apart share banks.
    static constexpr uint32_t swz(uint32_t row) { return D == 64u ? ((row >> 1) & 3u) << 1 : (row & 7u) << 1; }
};

template <uint32_t D>
constexpr uint32_t kWorkers = kComputeUnits * RowsLds<D>::kWaves;

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
// and a exchanged.
__device__ __forceinline__ uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
    uint64_t sum = 0u;
    while (n != 0u) {
        sum += n * (n - 1u) / 2u * (a / m) + n * (b / m);
        a %= m;
        b %= m;
        const uint64_t top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top % m;
        const uint64_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// The key blocks of a request's wide tiles. Tile k's rows end at position pos0 + (128 k + 127) / G, so
// its blocks end at end(k) = floor((128 k + 127 + G (pos0 + 32)) / 32 G), at most all of them, and with
// a window no more than `most` of them are seen.
struct WideSpan {
    uint32_t G, all, most;
    uint64_t c;
    __device__ WideSpan(uint32_t G_, uint32_t keys, int32_t pos0, uint32_t window) : G(G_) {
        all = (keys + kKeyBlock - 1u) / kKeyBlock;
        const uint64_t seen = (static_cast<uint64_t>(window) + 127u / G + 63u) / kKeyBlock;
        // (Rows before position 0 are counted from there: their tiles start as much earlier.)
        const uint64_t early = pos0 < 0 ? (31u - static_cast<int64_t>(pos0)) / kKeyBlock : 0u;
        most = window != 0u && seen + early < all ? static_cast<uint32_t>(seen + early) : all;
        c = 127u + static_cast<uint64_t>(G) * (static_cast<uint32_t>(max(pos0, 0)) + 32u);
    }
    __device__ uint32_t end(uint32_t k) const {
        const uint64_t e = (128ull * k + c) / (32ull * G);
        return e < all ? static_cast<uint32_t>(e) : all;
    }
    __device__ uint32_t units(uint32_t k) const { return min(end(k), most); }
    // Units of the tiles before k: those whose end is below `most`, then `most` each.
    __device__ uint32_t before(uint32_t k) const {
        const uint64_t full = 32ull * G * most;
        const uint64_t rising = full > c ? min(static_cast<uint64_t>(k), (full - c + 127u) / 128u) : 0u;
        return static_cast<uint32_t>(floor_sum(rising, 32ull * G, 128u, c) + (k - rising) * most);
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

__device__ __forceinline__ uint32_t wave_incl(uint32_t v, uint32_t lane) {
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t y = __shfl_up(v, d, 64);
        if (lane >= d) v += y;
    }
    return v;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(v, m, 64)));
    return v;
}

__device__ __forceinline__ int32_t wave_min(int32_t v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = min(v, static_cast<int32_t>(__shfl_xor(v, m, 64)));
    return v;
}

// Which rows go where. Rows of one request that fill wide tiles by themselves read the prefix there, at
// one pass over all their keys, where that takes at most a quarter more tiles than the rows of all
// requests together would (apart). Otherwise the prefix is taken for all rows together, in wide tiles
// from 17 rows on, and a request's own tokens in wide tiles where its rows pass 16.
struct Walk {
    Source mine;                // this lane's request of the chunk
    uint32_t chunk = 0;         // first request of the chunk
    uint32_t units0;            // before the chunk
    uint32_t units1;            // inclusive sums over the chunk's lanes
    Source prefix;              // of few rows
    uint32_t total;             // units of all
    uint32_t rows_all;
    int32_t first_pos;          // the least position of all rows
    bool apart;

    __device__ bool wide(const BatchParams& p, uint32_t rows) const { return apart || rows * p.G > kTileRows; }
    // A request as the workers for few rows see it.
    __device__ Source few(const BatchParams& p, uint32_t r) const {
        Source s = request_source(p, r);
        if (wide(p, s.rows)) s.blocks = 0u;
        return s;
    }
    __device__ void load(const BatchParams& p, uint32_t lane) {
        mine = few(p, chunk + lane);
        units1 = wave_incl(mine.units(p.KVH), lane);
    }
    // Totals of the batch and the prefix's part; then the first chunk. Returns units a worker; 0
    // where the row starts are no rows of the batch (they would pass the workspace).
    __device__ uint32_t open(const BatchParams& p, uint32_t lane) {
        uint32_t rows = 0u, sum = 0u, tiles = 0u;
        int32_t first = 0x7fffffff;
        for (uint32_t r = lane; r < p.b.requests; r += 64u) {
            const Source s = request_source(p, r);
            sum = min(sum + s.rows, 1u << 25);
            rows = max(rows, s.row0 + s.rows);
            tiles += wide_tiles_of(s.rows, p.G);
            if (s.rows != 0u) first = min(first, s.pos);
        }
        if (static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(wave_sum(sum))) > p.b.max_rows) return 0u;
        rows_all = __builtin_amdgcn_readfirstlane(wave_max(rows));
        tiles = __builtin_amdgcn_readfirstlane(wave_sum(tiles));
        first_pos = static_cast<int32_t>(p.b.prefix) + __builtin_amdgcn_readfirstlane(wave_min(first));
        apart = rows_all * p.G > kTileRows && 4u * tiles <= 5u * wide_tiles_of(rows_all, p.G);
        uint32_t units = 0u, most = 0u;
        for (uint32_t r = lane; r < p.b.requests; r += 64u) {
            const Source s = few(p, r);
            units += s.units(p.KVH);
            most = max(most, s.blocks);
        }
        units = __builtin_amdgcn_readfirstlane(wave_sum(units));
        most = __builtin_amdgcn_readfirstlane(wave_max(most));
        prefix = Source{0u, rows_all, 0u, p.b.prefix, 0, 0u, 0u};
        if (rows_all != 0u) {
            prefix.pos = first_pos;
            if (p.window != 0u && static_cast<int64_t>(first_pos) + 1 > p.window) prefix.lo = first_pos + 1u - p.window;
            prefix.tiles = tiles_of(rows_all, p.G);
            if (!wide(p, rows_all) && prefix.hi > prefix.lo)
                prefix.blocks = (prefix.hi - prefix.lo + kKeyBlock - 1u) / kKeyBlock;
        }
        most = max(most, prefix.blocks);
        total = units + prefix.units(p.KVH);
        units0 = prefix.units(p.KVH);
        load(p, lane);
        return max(max((total + p.workers - 1u) / p.workers, (most + kMaxParts - 2u) / (kMaxParts - 1u)), 1u);
    }
    // On to the chunk that holds unit u (u >= units0).
    __device__ void seek(const BatchParams& p, uint32_t u, uint32_t lane) {
        while (chunk + 64u < p.b.requests && u >= units0 + __builtin_amdgcn_readlane(units1, 63)) next(p, lane);
    }
    __device__ void next(const BatchParams& p, uint32_t lane) {
        units0 += __builtin_amdgcn_readlane(units1, 63);
        chunk += 64u;
        load(p, lane);
    }
    // Whether some rows see keys of the prefix outside their request's tiles.
    __device__ bool has_prefix(const BatchParams& p) const {
        return prefix.blocks != 0u || (!apart && wide(p, rows_all) && prefix.hi > prefix.lo);
    }
    // The keys that a request's wide tiles walk: the prefix's before its own where apart.
    __device__ WideSpan span(const BatchParams& p, const Source& s) const {
        const uint32_t pre = apart ? p.b.prefix : 0u;
        return WideSpan(p.G, s.rows != 0u ? pre + s.hi : 0u, static_cast<int32_t>(pre) + s.pos, p.window);
    }
    __device__ uint32_t wide_head(const BatchParams& p, const Source& s) const {
        return wide(p, s.rows) && s.rows != 0u ? span(p, s).before(wide_tiles_of(s.rows, p.G)) : 0u;
    }
};

__device__ __forceinline__ Source shfl_source(const Source& s, uint32_t from) {
    return Source{static_cast<uint32_t>(__builtin_amdgcn_readlane(s.row0, from)),
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(s.rows, from)),
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(s.lo, from)),
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(s.hi, from)),
                  __builtin_amdgcn_readlane(s.pos, from),
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(s.tiles, from)),
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(s.blocks, from))};
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

// One query row again over its visible keys [j0, j1) of a segment alone, against the same
// reference ref: the matrix products take masked keys with a probability of 0, which a value of V
// that is not finite turns into NaN (and the two terms of a probability make NaN of an infinity). Four keys at a time, 16 lanes each; the sums stay
// unnormalised, dims 64 c + 4 (lane % 16) + e of o[c][e], in every lane.
template <uint32_t D, typename SlotOf>
__device__ __forceinline__ void row_alone(const BatchParams& p, uint32_t hk, const uint16_t* q_row, uint32_t j0,
                                          uint32_t j1, float ref, uint32_t lane, SlotOf&& slot_of,
                                          float (&o)[D / 64u][4]) {
    constexpr uint32_t kC = D / 64u;
    const uint32_t at = (lane & 15u) * 4u;
    const auto value = [](const uint2& w, int e) {
        const uint32_t two = e < 2 ? w.x : w.y;
        return (e & 1) != 0 ? __uint_as_float(two & 0xFFFF0000u) : bf16_bits_to_f32(two & 0xFFFFu);
    };
#pragma unroll
    for (uint32_t c = 0; c < kC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][e] = 0.0f;
    for (uint32_t jb = j0; jb < j1; jb += 4u) {
        const uint32_t j = min(jb + (lane >> 4), j1 - 1u);
        const uint32_t slot = slot_of(j);
        const bool seen = jb + (lane >> 4) < j1 && slot != HYP_SLOT_NONE;
        const size_t row = (static_cast<size_t>(seen ? slot : 0u) * p.KVH + hk) * D;
        float s = 0.0f;
        uint2 v[kC];
#pragma unroll
        for (uint32_t c = 0; c < kC; ++c) {
            const uint2 k = *reinterpret_cast<const uint2*>(p.ck + row + 64u * c + at);
            const uint2 q = *reinterpret_cast<const uint2*>(q_row + 64u * c + at);
            v[c] = *reinterpret_cast<const uint2*>(p.cv + row + 64u * c + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf(value(q, e), value(k, e), s);
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) s += __shfl_xor(s, d);
        if (seen) {
            const float w = __builtin_amdgcn_exp2f(fmaf(s, p.scale, -ref));
#pragma unroll
            for (uint32_t c = 0; c < kC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][e] = fmaf(w, value(v[c], e), o[c][e]);
        }
    }
#pragma unroll
    for (uint32_t c = 0; c < kC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[c][e] += __shfl_xor(o[c][e], 16);
            o[c][e] += __shfl_xor(o[c][e], 32);
        }
}

// Where a segment's rows go: to the output (all their keys were in it), by output row, or to a piece.
enum : uint32_t { kToOutput = 0u, kToRows = 1u, kToPiece = 2u };

// Blocks [b0, b1) of tile `tile` of kv head hk of source s.
template <uint32_t D>
__device__ __forceinline__ void rows_segment(const BatchParams& p, const Source& s, const uint32_t* table, bool is_prefix,
                                             uint32_t hk, uint32_t tile, uint32_t b0, uint32_t b1, uint32_t to,
                                             uint32_t piece, uint32_t lds, uint32_t lane) {
    using Lds = RowsLds<D>;
    constexpr uint32_t kSteps = D / 32u;
    constexpr uint32_t kDTiles = D / 16u;
    constexpr uint32_t kUnitRows = 512u / D;                // V rows of one 1 KB load
    constexpr uint32_t kUnits = kKeyBlock / kUnitRows;
    const uint32_t j16 = lane & 15u;
    const uint32_t kb = lane >> 4;
    const uint32_t rows = s.rows * p.G;
    const uint32_t r = tile * kTileRows + j16;
    const bool live = r < rows;
    const uint32_t token = (live ? r : tile * kTileRows) / p.G;
    const uint32_t head = hk * p.G + (live ? r : tile * kTileRows) - token * p.G;
    const uint16_t* q_row = p.q + (static_cast<size_t>(s.row0 + token) * p.H + head) * D;

    // This lane's query row (column j16) and the keys [first, last] that it sees.
    bf16x8_t q[kSteps];
#pragma unroll
    for (uint32_t st = 0; st < kSteps; ++st) q[st] = *reinterpret_cast<const bf16x8_t*>(q_row + st * 32u + kb * 8u);
    int32_t last = static_cast<int32_t>(s.hi) - 1;
    int32_t first = 0;
    if (!is_prefix || p.window != 0u || s.pos < last) {
        const int32_t pos = is_prefix ? row_position(p, s.row0 + token) : s.pos + static_cast<int32_t>(token);
        last = min(last, pos);
        if (p.window != 0u) first = max(first, static_cast<int32_t>(max(static_cast<int64_t>(pos) + 1 - p.window, int64_t{0})));
    }

    const uint32_t last_key = s.hi - 1u;
    const uint32_t mask = (1u << p.b.shift) - 1u;
    const auto entry_of = [&](uint32_t j) { return table[min(j, last_key) >> p.b.shift]; };
    const auto slot_at = [&](uint32_t entry, uint32_t j) { return (entry << p.b.shift) + (min(j, last_key) & mask); };
    const auto slot_of = [&](uint32_t j) {
        const uint32_t e = entry_of(j);
        return e < p.b.num_blocks ? slot_at(e, j) : HYP_SLOT_NONE;
    };

    const size_t head_at = static_cast<size_t>(hk) * D;
    const size_t stride = static_cast<size_t>(p.KVH) * D;
    bf16x8_t kf[2][kSteps];
    const auto load_k = [&](const uint32_t (&slot)[2]) {
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
            const uint16_t* row = p.ck + static_cast<size_t>(slot[c]) * stride + head_at + kb * 8u;
#pragma unroll
            for (uint32_t st = 0; st < kSteps; ++st) kf[c][st] = *reinterpret_cast<const bf16x8_t*>(row + st * 32u);
        }
    };
    // Slots of keys jb + 16 c + j16 from their table entries; a block outside the pool gives slot 0
    // and its bit in the mask of keys that are there (bit 16 c + j16).
    uint32_t there = 0xFFFFFFFFu;
    const auto slots_from = [&](const uint32_t (&entry)[2], uint32_t jb, uint32_t (&slot)[2]) {
        bool ok[2];
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
            ok[c] = entry[c] < p.b.num_blocks;
            slot[c] = ok[c] ? slot_at(entry[c], jb + 16u * c + j16) : 0u;
        }
        there = (static_cast<uint32_t>(__ballot(ok[0])) & 0xFFFFu) | (static_cast<uint32_t>(__ballot(ok[1])) << 16);
    };

    f32x4_t o[kDTiles];
#pragma unroll
    for (uint32_t t = 0; t < kDTiles; ++t) o[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_huge_valf();
    float l = 0.0f;

    uint32_t entry[2], slot[2];
    const uint32_t j_first = s.lo + b0 * kKeyBlock;
#pragma unroll
    for (uint32_t c = 0; c < 2u; ++c) entry[c] = entry_of(j_first + 16u * c + j16);
    slots_from(entry, j_first, slot);
    load_k(slot);
#pragma unroll
    for (uint32_t c = 0; c < 2u; ++c) entry[c] = entry_of(j_first + kKeyBlock + 16u * c + j16);

    // V operand of dim tile t: group kb reads key rows 4 kb + 0..3 (then + 16), dims 16 t + 0..15.
    const uint32_t vrow = 4u * kb + (j16 >> 2);
    const uint32_t v_at = lds + vrow * Lds::kRow + ((((j16 >> 1) & 1u) ^ Lds::swz(vrow)) << 4) + (j16 & 1u) * 8u;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t jb = s.lo + b * kKeyBlock;
        const bool more = b + 1u < b1;
        const uint32_t now_there = there;
        // V of this block (the last block's reads of the LDS are done: their products are).
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // per-lane offsets formed here, not kept in registers over the walk
#pragma unroll
        for (uint32_t u = 0; u < kUnits; ++u) {
            const uint32_t vr = u * kUnitRows + ln / Lds::kChunks;
            const int own = static_cast<int>(slot[u * kUnitRows / 16u]);   // lane j16 holds row 16 c + j16's
            const uint32_t at = static_cast<uint32_t>(kUnitRows == 1u ? __builtin_amdgcn_readlane(own, u & 15u)
                                                                      : __shfl(own, static_cast<int>(vr & 15u), 64));
            const uint16_t* src = p.cv + static_cast<size_t>(at) * stride + head_at +
                                  (((ln % Lds::kChunks) ^ Lds::swz(vr)) * 8u);
            __builtin_amdgcn_global_load_lds((const HYP_GLOBAL void*)src,
                                             reinterpret_cast<HYP_LDS void*>(lds + u * 1024u), 16, 0, 0);
        }
        f32x4_t sc[2] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (uint32_t st = 0; st < kSteps; ++st)
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
                sc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[c][st], q[st], sc[c], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
            slots_from(entry, jb + kKeyBlock, slot);
            load_k(slot);
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) entry[c] = entry_of(jb + 2u * kKeyBlock + 16u * c + j16);
        }
        __builtin_amdgcn_sched_barrier(0);

        // sc[c][i] is key jb + 16 c + 4 kb + i of row j16.
        float pr[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) pr[i] = sc[i / 4u][i % 4u] * p.scale;
        if (now_there != 0xFFFFFFFFu || __any(static_cast<int32_t>(jb + kKeyBlock) - 1 > last || static_cast<int32_t>(jb) < first)) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                const uint32_t k = 16u * (i / 4u) + 4u * kb + i % 4u;
                const int32_t j = static_cast<int32_t>(jb + k);
                if (j > last || j < first || ((now_there >> k) & 1u) == 0u) pr[i] = -__builtin_huge_valf();
            }
        }
        float mx = pr[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, pr[i]);
        mx = max_lane_xor32(max_lane_xor16(mx));
        const float m_new = fmaxf(m, mx);
        const float ref = m_new > -__builtin_huge_valf() ? m_new : 0.0f;
        const float alpha = m_new > m ? __builtin_amdgcn_exp2f(m - ref) : 1.0f;
        m = m_new;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            pr[i] = __builtin_amdgcn_exp2f(pr[i] - ref);
            sum += pr[i];
        }
        l = l * alpha + sum;
        const bf16x8_t ph = round_p(pr);
#pragma unroll
        for (int i = 0; i < 8; ++i) pr[i] -= bf16_bits_to_f32(__builtin_bit_cast(u16x8_t, ph)[i]);
        const bf16x8_t pl = round_p(pr);
#pragma unroll
        for (uint32_t t = 0; t < kDTiles; ++t) o[t] *= alpha;
        // V has landed: of the loads behind it (the next block's 2 kSteps of K, its successor's
        // entries) no more than the K rows' number is outstanding.
        if (more) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2u * kSteps) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t t = 0; t < kDTiles; ++t) {
            const uint32_t c = 2u * t;
            const bf16x8_t v = lds_read_tr((v_at ^ ((c & 15u) << 4)) + (c & ~15u) * 16u, 16u * Lds::kRow);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph, o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl, o[t], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    l = add_lane_xor32(add_lane_xor16(l));

    // o[t][i] is dim 16 t + 4 kb + i of row j16.
    float odd = 0.0f;
#pragma unroll
    for (uint32_t t = 0; t < kDTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd = fmaf(o[t][i], 0.0f, odd);
    const size_t out_row = static_cast<size_t>(s.row0 + token) * p.H + head;
    const size_t prow = to == kToRows ? out_row : static_cast<size_t>(piece) * kTileRows + j16;
    float* const po = to == kToRows ? p.whole_o[is_prefix ? 0 : 1] : p.part_o;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    if (live && to == kToOutput) {
#pragma unroll
        for (uint32_t t = 0; t < kDTiles; ++t)
            *reinterpret_cast<uint2*>(p.out + out_row * D + 16u * t + 4u * kb) =
                make_uint2(cvt_pk_bf16(o[t][0] * inv, o[t][1] * inv), cvt_pk_bf16(o[t][2] * inv, o[t][3] * inv));
    } else if (live) {
#pragma unroll
        for (uint32_t t = 0; t < kDTiles; ++t)
            *reinterpret_cast<float4*>(po + prow * D + 16u * t + 4u * kb) =
                make_float4(o[t][0], o[t][1], o[t][2], o[t][3]);
        if (kb == 0u) (to == kToRows ? p.whole_ml[is_prefix ? 0 : 1] : p.part_ml)[prow] = make_float2(m, l);
    }
    // Rows with a value that is not finite are formed again, by themselves.
    const uint64_t odd_lanes = __ballot(odd != 0.0f && live);
    uint32_t odd_rows = static_cast<uint32_t>((odd_lanes | (odd_lanes >> 16) | (odd_lanes >> 32) | (odd_lanes >> 48)) & 0xFFFFu);
    if (odd_rows == 0u) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's own stores of these rows are done
    for (; odd_rows != 0u; odd_rows &= odd_rows - 1u) {
        const uint32_t i = __builtin_ctz(odd_rows);
        const uint32_t rr = tile * kTileRows + i;
        const uint32_t tok = rr / p.G;
        const uint16_t* src = p.q + (static_cast<size_t>(s.row0 + tok) * p.H + hk * p.G + (rr - tok * p.G)) * D;
        const int32_t j0 = max(__shfl(first, static_cast<int>(i)), static_cast<int32_t>(j_first));
        const int32_t j1 = min(__shfl(last, static_cast<int>(i)), static_cast<int32_t>(s.lo + b1 * kKeyBlock) - 1) + 1;
        const float ref = __shfl(m, static_cast<int>(i));
        float a[D / 64u][4];
        row_alone<D>(p, hk, src, static_cast<uint32_t>(j0), static_cast<uint32_t>(max(j1, j0)),
                     ref > -__builtin_huge_valf() ? ref : 0.0f, lane, slot_of, a);
        const size_t to_row = static_cast<size_t>(s.row0 + tok) * p.H + hk * p.G + (rr - tok * p.G);
        const float by = __shfl(inv, static_cast<int>(i));
        if (lane >= 16u) continue;
#pragma unroll
        for (uint32_t c = 0; c < D / 64u; ++c) {
            const uint32_t dim = 64u * c + 4u * lane;
            if (to == kToOutput) {
                *reinterpret_cast<uint2*>(p.out + to_row * D + dim) =
                    make_uint2(cvt_pk_bf16(a[c][0] * by, a[c][1] * by), cvt_pk_bf16(a[c][2] * by, a[c][3] * by));
            } else {
                *reinterpret_cast<float4*>(po + (to == kToRows ? to_row : static_cast<size_t>(piece) * kTileRows + i) * D + dim) =
                    make_float4(a[c][0], a[c][1], a[c][2], a[c][3]);
            }
        }
    }
}

// What the other launches need of the walk: the chunk's requests and their rows.
__device__ __forceinline__ void scribe(const BatchParams& p, Walk& w, uint32_t per, uint32_t chunk, uint32_t lane) {
    if (per == 0u) {
        if (chunk == 0u && lane == 0u) *p.header = Header{};
        return;
    }
    // The prefix's wide tiles (for all rows together) come first.
    uint32_t tiles = 0u, blocks = 0u, lo = 0u;
    if (!w.apart && w.wide(p, w.rows_all) && w.prefix.hi > w.prefix.lo) {
        tiles = wide_tiles_of(w.rows_all, p.G);
        lo = w.prefix.lo / kKeyBlock;
        blocks = (w.prefix.hi + kKeyBlock - 1u) / kKeyBlock - lo;
    }
    const uint32_t first_unit = p.KVH * tiles * blocks;
    uint32_t unit0 = first_unit;
    const auto head_of = [&](const Source& s) { return w.wide_head(p, s); };
    const auto tiles_here = [&](const Source& s) { return w.wide(p, s.rows) ? wide_tiles_of(s.rows, p.G) : 0u; };
    while (w.chunk < chunk) {
        unit0 += wave_sum(p.KVH * head_of(w.mine));
        w.next(p, lane);
    }
    const Source s = w.mine;
    const uint32_t r = chunk + lane;
    const uint32_t head = head_of(s);
    const uint32_t wt = tiles_here(s);
    const uint32_t units1 = wave_incl(p.KVH * head, lane);
    if (r < p.b.requests) {
        p.request[r] = Record{w.units0 + w.units1 - s.units(p.KVH), s.tiles, s.blocks, unit0 + units1 - p.KVH * head, wt, head,
                              {}};
    }
    for (uint32_t i = 0; i < 64u; ++i) {
        const uint32_t row0 = __builtin_amdgcn_readlane(s.row0, i);
        const uint32_t rows = __builtin_amdgcn_readlane(s.rows, i);
        const int32_t pos = static_cast<int32_t>(p.b.prefix) + __builtin_amdgcn_readlane(s.pos, i);
        for (uint32_t t = lane; t < rows; t += 64u)
            p.row[row0 + t] = RowRecord{chunk + i, t, pos + static_cast<int32_t>(t), 0u};
    }
    if (chunk + 64u < p.b.requests) return;
    // The last chunk knows all units.
    const uint32_t all = unit0 + __builtin_amdgcn_readlane(units1, 63);
    uint32_t most = max(blocks, wave_max(w.apart ? (p.b.prefix + s.hi) / kKeyBlock + 1u : s.hi / kKeyBlock + 1u));
    for (uint32_t c = lane; c < chunk; c += 64u) most = max(most, request_source(p, c).hi / kKeyBlock + 1u + (w.apart ? p.b.prefix / kKeyBlock + 1u : 0u));
    most = wave_max(most);
    if (lane == 0u) {
        const uint32_t wide_per = max(max((all + p.wide_workers - 1u) / p.wide_workers,
                                          (most + kMaxParts - 2u) / (kMaxParts - 1u)), 1u);
        *p.header = Header{per, w.prefix.blocks, w.prefix.tiles, wide_per, all, lo, blocks, tiles, w.apart ? 1u : 0u, w.rows_all, {}};
    }
}

template <uint32_t D>
__global__ __launch_bounds__(64, RowsLds<D>::kWaves / 4u) void attn_batch_rows_kernel(BatchParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[];
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((HYP_LDS uint8_t*)lds_mem));
    const uint32_t lane = threadIdx.x;
    Walk w;
    const uint32_t per = w.open(p, lane);
    if (blockIdx.x >= p.workers) {
        scribe(p, w, per, (blockIdx.x - p.workers) * kScribeRequests, lane);
        return;
    }
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * per;
    if (per == 0u || begin >= w.total) return;
    uint32_t u = static_cast<uint32_t>(begin);
    const uint32_t end = min(u + per, w.total);
    while (u < end) {
        Source s = w.prefix;
        const uint32_t* table = p.b.prefix_table;
        uint32_t unit0 = 0u;
        bool is_prefix = true;
        if (u >= w.prefix.units(p.KVH)) {
            w.seek(p, u, lane);
            const uint64_t behind = __ballot(u < w.units0 + w.units1);
            if (behind == 0u) return;   // (not with u below the total)
            const uint32_t at = __builtin_ctzll(behind);
            s = shfl_source(w.mine, at);
            table = p.b.tables + static_cast<size_t>(w.chunk + at) * p.b.max_blocks;
            unit0 = w.units0 + __builtin_amdgcn_readlane(w.units1, at) - s.units(p.KVH);
            is_prefix = false;
        }
        const uint32_t g = (u - unit0) / s.blocks;
        const uint32_t b0 = u - unit0 - g * s.blocks;
        const uint32_t b1 = min(s.blocks, b0 + (end - u));
        const uint32_t hk = g / s.tiles;
        const uint32_t to = b1 - b0 < s.blocks ? kToPiece : (!is_prefix && !w.has_prefix(p) ? kToOutput : kToRows);
        rows_segment<D>(p, s, table, is_prefix, __builtin_amdgcn_readfirstlane(hk),
                        __builtin_amdgcn_readfirstlane(g - hk * s.tiles), __builtin_amdgcn_readfirstlane(b0),
                        __builtin_amdgcn_readfirstlane(b1), to, 2u * blockIdx.x + (u == begin ? 0u : 1u), lds, lane);
        u += b1 - b0;
    }
}

// Wide tiles (attn_batch_tiles_kernel): the arithmetic of attention_chunk.hip's kernel - 128 query rows
// of one kv head, 32 a wave on 32x32x16 products, S^T = K Q^T and O^T = V^T P^T, K and V rows by loads
// straight to two LDS stages - over paged keys. A lane looks up the slot of key lane % 32 of the block
// after the next one, so its table entry has arrived a block before the rows are requested.
// Probabilities enter as one bf16 term here, where the matrix products are what is waited for, and the
// row's sum takes them as rounded: the output is then a weighted mean with slightly other weights, and a
// row that one key dominates is exact however old its maximum is. (Two terms cost half as many
// products again for an error of 1.7e-3 of the output's norm instead of 2.4e-3, most of both the
// output's own rounding.)
template <uint32_t D>
struct TilesLds {
    static constexpr uint32_t kRow = D * 2u;
    static constexpr uint32_t kChunks = D / 8u;
    static constexpr uint32_t kV = kKeyBlock * kRow;
    static constexpr uint32_t kStage = 2u * kKeyBlock * kRow;
    static constexpr uint32_t kOutRow = D * 2u + 16u;
    static constexpr uint32_t kOut = kChunkRows * kOutRow;
    static constexpr uint32_t kBytes = 2u * kStage > kOut ? 2u * kStage : kOut;
    static constexpr uint32_t k_swz(uint32_t row) { return (row & 15u) & (kChunks - 1u); }
    static constexpr uint32_t v_swz(uint32_t row) { return (((row & 3u) << 2) | ((row >> 1) & 2u)) & (kChunks - 1u); }
};

constexpr uint32_t kTileThreads = 256;
constexpr uint32_t kTileWaves = kTileThreads / 64u;
constexpr uint32_t kWaveRows = 32;
constexpr float kRescaleLog2 = 8.0f;

// Workers: as many workgroups as the device holds at once.
template <uint32_t D>
constexpr uint32_t kWideWorkers = kComputeUnits * (D >= 512u ? 1u : 2u);

// The keys that a tile walks, positions 0 .. keys - 1: `pre` of the prefix's tokens, then own ones.
struct Sequence {
    const uint32_t* own;   // the request's row of tables
    uint32_t pre, keys;
    uint32_t row0, rows;   // query rows (tokens)
    int32_t pos;           // the first one's position among the keys
    bool by_record;        // rows of many requests: their positions from the records
};

template <uint32_t D>
__device__ __forceinline__ void tile_segment(const BatchParams& p, const Sequence& s, uint32_t hk, uint32_t tile,
                                             uint32_t b0, uint32_t b1, uint32_t to, uint32_t piece, uint32_t lds,
                                             int32_t (*range)[2]) {
    using Lds = TilesLds<D>;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 31u;   // this lane's query row of the wave
    const uint32_t h = lane >> 5;
    const uint32_t rows = s.rows * p.G;
    const uint32_t wrow0 = tile * kChunkRows + wave * kWaveRows;
    const uint32_t qrow = min(wrow0 + n, rows - 1u);   // rows past the end repeat the last (not stored)
    const uint32_t qt = qrow / p.G;
    const size_t out_row = static_cast<size_t>(s.row0 + qt) * p.H + hk * p.G + (qrow - qt * p.G);

    constexpr uint32_t kSteps = D / 16u;
    constexpr uint32_t kDTiles = D / 32u;
    bf16x8_t q[kSteps];
    {
        const uint16_t* src = p.q + out_row * D + h * 8u;
#pragma unroll
        for (uint32_t st = 0; st < kSteps; ++st) q[st] = *reinterpret_cast<const bf16x8_t*>(src + st * 16u);
    }
    // The keys [first, last] that this lane's row sees, and the blocks that some row of the tile sees.
    const int32_t pos = s.by_record ? p.row[s.row0 + qt].pos : s.pos + static_cast<int32_t>(qt);
    const int32_t last = min(static_cast<int32_t>(s.keys) - 1, pos);
    const int32_t first = p.window != 0u ? max(0, static_cast<int32_t>(max(static_cast<int64_t>(pos) + 1 - p.window, int64_t{0}))) : 0;
    {
        const int32_t lo = wave_min(first), hi = -wave_min(-last);
        if (lane == 0u) {
            range[wave][0] = lo;
            range[wave][1] = hi;
        }
    }
    __syncthreads();
    int32_t lo = range[0][0], hi = range[0][1];
#pragma unroll
    for (uint32_t w = 1; w < kTileWaves; ++w) {
        lo = min(lo, range[w][0]);
        hi = max(hi, range[w][1]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    if (hi < lo) hi = lo - 1;
    b0 = max(b0, static_cast<uint32_t>(lo) / kKeyBlock);
    b1 = min(b1, static_cast<uint32_t>(hi + 1 + static_cast<int32_t>(kKeyBlock) - 1) / kKeyBlock);

    const uint32_t last_key = s.keys - 1u;
    const uint32_t mask = (1u << p.b.shift) - 1u;
    const auto entry_of = [&](uint32_t j) {
        j = min(j, last_key);
        return j < s.pre ? p.b.prefix_table[j >> p.b.shift] : s.own[(j - s.pre) >> p.b.shift];
    };
    const auto slot_at = [&](uint32_t entry, uint32_t j) {
        j = min(j, last_key);
        return (entry << p.b.shift) + ((j < s.pre ? j : j - s.pre) & mask);
    };
    const auto slot_of = [&](uint32_t j) {
        const uint32_t e = entry_of(j);
        return e < p.b.num_blocks ? slot_at(e, j) : HYP_SLOT_NONE;
    };
    // This lane's key (lane % 32) of a block from its entry; a block outside the pool gives slot 0 and
    // a 0 in the mask of keys that are there.
    uint32_t there = 0u;
    const auto slot_from = [&](uint32_t entry, uint32_t j) {
        const bool ok = entry < p.b.num_blocks;
        there = static_cast<uint32_t>(__ballot(ok));
        return ok ? slot_at(entry, j) : 0u;
    };

    constexpr uint32_t kUnitRows = 512u / D;
    constexpr uint32_t kUnits = kKeyBlock / kUnitRows / kTileWaves;   // of a wave
    const size_t stride = static_cast<size_t>(p.KVH) * D;
    const uint16_t* const ck = p.ck + static_cast<size_t>(hk) * D;
    const uint16_t* const cv = p.cv + static_cast<size_t>(hk) * D;
    // Unit i of the wave (1 KB of K rows and of V rows) of the block whose slots are given, into stage st.
    const auto load_unit = [&](uint32_t slots, uint32_t st, uint32_t i) {
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // per-lane addresses formed here, not kept in registers over the walk
        const uint32_t unit = wave + kTileWaves * i;
        const uint32_t r = unit * kUnitRows + ln / Lds::kChunks;
        const uint32_t phys = ln % Lds::kChunks;
        const uint32_t slot = static_cast<uint32_t>(kUnitRows == 1u ? __builtin_amdgcn_readlane(static_cast<int>(slots), unit)
                                                                    : __shfl(static_cast<int>(slots), static_cast<int>(r), 64));
        const size_t at = static_cast<size_t>(slot) * stride;
        HYP_LDS void* kd = reinterpret_cast<HYP_LDS void*>(lds + st * Lds::kStage + unit * 1024u);
        HYP_LDS void* vd = reinterpret_cast<HYP_LDS void*>(lds + st * Lds::kStage + Lds::kV + unit * 1024u);
        __builtin_amdgcn_global_load_lds((const HYP_GLOBAL void*)(ck + at + (phys ^ Lds::k_swz(r)) * 8u), kd, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const HYP_GLOBAL void*)(cv + at + (phys ^ Lds::v_swz(r)) * 8u), vd, 16, 0, 0);
    };

    f32x16_t o[kDTiles];
#pragma unroll
    for (uint32_t t = 0; t < kDTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -__builtin_huge_valf();   // the softmax reference (log2 domain) of row n
    float l = 0.0f;                     // the sum over this lane's keys

    const uint32_t k_at = lds + n * Lds::kRow + ((h ^ Lds::k_swz(n)) << 4);
    constexpr uint32_t kSpan = Lds::kChunks < 16u ? Lds::kChunks : 16u;   // chunks a swizzle permutes
    constexpr uint32_t kAhead = 4u;
    const uint32_t j16 = lane & 15u;
    const uint32_t vrow = 4u * h + (j16 >> 2);
    const uint32_t vchunk = 2u * ((lane >> 4) & 1u) + ((j16 >> 1) & 1u);
    const uint32_t v_at = lds + Lds::kV + vrow * Lds::kRow + ((vchunk ^ Lds::v_swz(vrow)) << 4) + (j16 & 1u) * 8u;

    uint32_t slots = 0u, entry = 0u;   // of the block whose rows are requested next
    if (b0 < b1) {
        slots = slot_from(entry_of(b0 * kKeyBlock + n), b0 * kKeyBlock + n);
        entry = entry_of((b0 + 1u) * kKeyBlock + n);
#pragma unroll
        for (uint32_t i = 0; i < kUnits; ++i) load_unit(slots, 0u, i);
    }
    const auto v_read = [&](uint32_t stage, uint32_t u) {
        const uint32_t c = 4u * (u / 2u);
        const uint32_t at = ((v_at + stage) ^ ((c % kSpan) << 4)) + (c / kSpan) * kSpan * 16u;
        return lds_read_tr(at + 16u * (u % 2u) * Lds::kRow, 8u * Lds::kRow);
    };
    constexpr uint32_t kProducts = 2u * kDTiles;
    constexpr bool kLazy = D >= 512u;
    float mx = 0.0f;
    // kLazy as in attention_chunk.hip: a block that outgrows the reference ends the inner loop before it
    // touches O, the outer loop rescales, and the inner loop takes the same block again.
    uint32_t b = b0;
    uint32_t now_there = there;
    bool again = false;
    do {
        for (; b < b1; ++b) {
            const uint32_t stage = ((b - b0) & 1u) * Lds::kStage;
            const uint32_t jb = b * kKeyBlock;
            if (!again) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();   // block b has landed, and every wave has left the other stage
                now_there = there;
                // (The last block loads what it loaded before once more: the same bytes.)
                if (b + 1u < b1) slots = slot_from(entry, jb + kKeyBlock + n);
                entry = entry_of(jb + 2u * kKeyBlock + n);
            }
            again = false;
            const uint32_t stage_n = (b + 1u - b0) & 1u;
            const auto k_read = [&](uint32_t st) {
                const uint32_t c = 2u * st;
                return lds_read16(((k_at + stage) ^ ((c % kSpan) << 4)) + (c / kSpan) * kSpan * 16u);
            };
            f32x16_t sc;
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
            bf16x8_t kf[kAhead];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t st = 0; st < kAhead; ++st) kf[st] = k_read(st);
#pragma unroll
            for (uint32_t st = 0; st < kSteps; ++st) {
                __builtin_amdgcn_sched_barrier(0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[st % kAhead], q[st], sc, 0, 0, 0);
                if (st + kAhead < kSteps) kf[st % kAhead] = k_read(st + kAhead);
                if (st % (kSteps / kUnits) == 0u) load_unit(slots, stage_n, st / (kSteps / kUnits));
            }
            __builtin_amdgcn_sched_barrier(0);
            bf16x8_t vf[kAhead];
            if constexpr (D != 256u) {   // (at 256 their registers are short)
#pragma unroll
                for (uint32_t u = 0; u < kAhead; ++u) vf[u] = v_read(stage, u);
                __builtin_amdgcn_sched_barrier(0);
            }

            // sc[i] is key jb + 8 (i / 4) + 4 h + i % 4 of row n.
            if (now_there != 0xFFFFFFFFu || __any(static_cast<int32_t>(jb + kKeyBlock) - 1 > last || static_cast<int32_t>(jb) < first)) {
#pragma unroll
                for (uint32_t i = 0; i < 16u; ++i) {
                    const uint32_t k = 8u * (i / 4u) + 4u * h + (i & 3u);
                    const int32_t j = static_cast<int32_t>(jb + k);
                    sc[i] = j <= last && j >= first && ((now_there >> k) & 1u) != 0u ? sc[i] * p.scale : -__builtin_huge_valf();
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] *= p.scale;
            }
            mx = sc[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
            mx = half_max(mx);
            if constexpr (kLazy) m = m == -__builtin_huge_valf() ? mx : m;   // O is still zero: nothing to rescale
            float alpha = 1.0f;
            if constexpr (kLazy) {
                if (__any(mx > m + kRescaleLog2)) {
                    again = true;
                    break;
                }
            } else {
                const float m_new = fmaxf(m, mx);
                alpha = m_new > m ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
                m = m_new;
                l *= alpha;
            }
            const float ref = m > -__builtin_huge_valf() ? m : 0.0f;
            float pr[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) pr[i] = __builtin_amdgcn_exp2f(sc[i] - ref);
            bf16x8_t pb[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) pb[t] = round_p(pr + 8 * t);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += bf16_bits_to_f32(__builtin_bit_cast(u16x8_t, pb[i / 8])[i % 8]);
            l += sum;
            if constexpr (!kLazy) {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[0][i] *= alpha;
            }
            if constexpr (D == 256u) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t u = 0; u < kAhead; ++u) vf[u] = v_read(stage, u);
            }
#pragma unroll
            for (uint32_t u = 0; u < kProducts; ++u) {
                __builtin_amdgcn_sched_barrier(0);
                o[u / 2u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[u % kAhead], pb[u % 2u], o[u / 2u], 0, 0, 0);
                if (u + kAhead < kProducts) vf[u % kAhead] = v_read(stage, u + kAhead);
                if (!kLazy && u / 2u + 1u < kDTiles) {   // the next tile, half of it in each product's shadow
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) o[u / 2u + 1u][8u * (u % 2u) + i] *= alpha;
                }
            }
        }
        if (again) {
            const float m_new = fmaxf(m, mx);
            const float alpha = m_new > m ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
            m = m_new;
            l *= alpha;
#pragma unroll
            for (uint32_t t = 0; t < kDTiles; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
        }
    } while (again);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last loads: none writes LDS past here
    l = half_sum(l);

    float zero = 0.0f;
#pragma unroll
    for (uint32_t dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = fmaf(o[dt][i], 0.0f, zero);
    const uint64_t odd_lanes = __ballot(zero != 0.0f && wrow0 + n < rows);
    const uint32_t odd_rows = static_cast<uint32_t>(odd_lanes) | static_cast<uint32_t>(odd_lanes >> 32);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const size_t prow = to == kToRows ? out_row : static_cast<size_t>(piece) * kChunkRows + wave * kWaveRows + n;
    float* const po = to == kToRows ? p.whole_o[s.by_record ? 0 : 1] : p.wide_o;

    // o[dt][i] is dim 32 dt + 8 (i / 4) + 4 h + i % 4 of row n.
    __syncthreads();   // every wave has left the stages
    if (to != kToOutput) {
        if (wrow0 + n < rows) {
#pragma unroll
            for (uint32_t dt = 0; dt < kDTiles; ++dt)
#pragma unroll
                for (uint32_t u = 0; u < 4u; ++u)
                    *reinterpret_cast<float4*>(po + prow * D + 32u * dt + 8u * u + 4u * h) =
                        make_float4(o[dt][4 * u], o[dt][4 * u + 1], o[dt][4 * u + 2], o[dt][4 * u + 3]);
            if (h == 0u) (to == kToRows ? p.whole_ml[s.by_record ? 0 : 1] : p.wide_ml)[prow] = make_float2(m, l);
        }
    } else {
        // The wave's rows through LDS (its own part of the stages), then out as 16-byte pieces of whole rows.
        const uint32_t out_lds = lds + wave * kWaveRows * Lds::kOutRow;
#pragma unroll
        for (uint32_t dt = 0; dt < kDTiles; ++dt)
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u) {
                u32x2_t w;
                w.x = cvt_pk_bf16(o[dt][4 * u] * inv, o[dt][4 * u + 1] * inv);
                w.y = cvt_pk_bf16(o[dt][4 * u + 2] * inv, o[dt][4 * u + 3] * inv);
                *reinterpret_cast<HYP_LDS u32x2_t*>(out_lds + n * Lds::kOutRow + (32u * dt + 8u * u + 4u * h) * 2u) = w;
            }
        __syncthreads();
        for (uint32_t c = lane; c < kWaveRows * Lds::kChunks; c += 64u) {
            const uint32_t r = c / Lds::kChunks;
            const uint32_t gr = wrow0 + r;
            if (gr >= rows) break;
            const uint32_t t = gr / p.G;
            const size_t dst = (static_cast<size_t>(s.row0 + t) * p.H + hk * p.G + (gr - t * p.G)) * D + (c % Lds::kChunks) * 8u;
            *reinterpret_cast<u32x4_t*>(p.out + dst) =
                *reinterpret_cast<const HYP_LDS u32x4_t*>(out_lds + r * Lds::kOutRow + (c % Lds::kChunks) * 16u);
        }
        __syncthreads();   // the next segment's loads go to the same place
    }
    if (odd_rows == 0u) return;
    // Rows with a value that is not finite are formed again, by themselves.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's own stores of these rows are done
    for (uint32_t todo = odd_rows; todo != 0u; todo &= todo - 1u) {
        const uint32_t i = __builtin_ctz(todo);
        const uint32_t tok = (wrow0 + i) / p.G;
        const size_t to_row = static_cast<size_t>(s.row0 + tok) * p.H + hk * p.G + (wrow0 + i - tok * p.G);
        const int32_t j0 = max(__shfl(first, static_cast<int>(i)), static_cast<int32_t>(b0 * kKeyBlock));
        const int32_t j1 = min(__shfl(last, static_cast<int>(i)), static_cast<int32_t>(b1 * kKeyBlock) - 1) + 1;
        const float ref = __shfl(m, static_cast<int>(i));
        const float by = __shfl(inv, static_cast<int>(i));
        float a[D / 64u][4];
        row_alone<D>(p, hk, p.q + to_row * D, static_cast<uint32_t>(j0), static_cast<uint32_t>(max(j1, j0)),
                     ref > -__builtin_huge_valf() ? ref : 0.0f, lane, slot_of, a);
        if (lane >= 16u) continue;
#pragma unroll
        for (uint32_t c = 0; c < D / 64u; ++c) {
            const uint32_t dim = 64u * c + 4u * lane;
            if (to == kToOutput) {
                *reinterpret_cast<uint2*>(p.out + to_row * D + dim) =
                    make_uint2(cvt_pk_bf16(a[c][0] * by, a[c][1] * by), cvt_pk_bf16(a[c][2] * by, a[c][3] * by));
            } else {
                const size_t at = to == kToRows ? to_row : static_cast<size_t>(piece) * kChunkRows + wave * kWaveRows + i;
                *reinterpret_cast<float4*>(po + at * D + dim) = make_float4(a[c][0], a[c][1], a[c][2], a[c][3]);
            }
        }
    }
}

template <uint32_t D>
__global__ __launch_bounds__(kTileThreads, D >= 512u ? 1 : 2) void attn_batch_tiles_kernel(BatchParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[];
    __shared__ int32_t range[kTileWaves][2];
    __shared__ uint32_t found;
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((HYP_LDS uint8_t*)lds_mem));
    const Header head = *p.header;
    const uint64_t from = static_cast<uint64_t>(blockIdx.x) * head.wide_per;
    if (head.wide_per == 0u || from >= head.wide_units) return;
    const uint32_t begin = static_cast<uint32_t>(from);
    const uint32_t end = min(begin + head.wide_per, head.wide_units);
    uint32_t u = begin;
    while (u < end) {
        Sequence s{nullptr, p.b.prefix, p.b.prefix, 0u, head.rows, 0, true};
        uint32_t hk, tile, off, blocks, block0;
        if (u < p.KVH * head.wide_tiles * head.wide_blocks) {
            const uint32_t g = u / head.wide_blocks;
            blocks = head.wide_blocks;
            block0 = head.wide_lo;
            off = u - g * blocks;
            hk = g / head.wide_tiles;
            tile = g - hk * head.wide_tiles;
        } else {
            __syncthreads();   // the last round's `found` has been read
            if (threadIdx.x == 0u) found = p.b.requests;
            __syncthreads();
            for (uint32_t r = threadIdx.x; r < p.b.requests; r += kTileThreads) {
                const Record rec = p.request[r];
                if (u >= rec.wide_unit0 && u - rec.wide_unit0 < p.KVH * rec.wide_head) found = r;
            }
            __syncthreads();
            const uint32_t r = __builtin_amdgcn_readfirstlane(found);
            if (r >= p.b.requests) return;   // (not with u below the total)
            const Record rec = p.request[r];
            const Source src = request_source(p, r);
            s.own = p.b.tables + static_cast<size_t>(r) * p.b.max_blocks;
            s.pre = head.apart != 0u ? p.b.prefix : 0u;
            s.keys = s.pre + src.hi;
            s.row0 = src.row0;
            s.rows = src.rows;
            s.pos = static_cast<int32_t>(s.pre) + src.pos;
            s.by_record = false;
            const WideSpan span(p.G, s.keys, s.pos, p.window);
            hk = (u - rec.wide_unit0) / rec.wide_head;
            const uint32_t x = u - rec.wide_unit0 - hk * rec.wide_head;
            uint32_t t0 = 0u, t1 = rec.wide_tiles;   // the last tile with before() <= x
            while (t1 - t0 > 1u) {
                const uint32_t mid = (t0 + t1) / 2u;
                if (span.before(mid) <= x) t0 = mid; else t1 = mid;
            }
            tile = t0;
            off = x - span.before(tile);
            blocks = span.units(tile);
            block0 = span.end(tile) - blocks;
        }
        const uint32_t take = min(blocks - off, end - u);
        const bool complete = !s.by_record && (head.apart != 0u || (head.blocks == 0u && head.wide_blocks == 0u));
        const uint32_t to = take < blocks ? kToPiece : (complete ? kToOutput : kToRows);
        tile_segment<D>(p, s, __builtin_amdgcn_readfirstlane(hk), __builtin_amdgcn_readfirstlane(tile),
                        __builtin_amdgcn_readfirstlane(block0 + off), __builtin_amdgcn_readfirstlane(block0 + off + take), to,
                        2u * blockIdx.x + (u == begin ? 0u : 1u), lds, range);
        u += take;
    }
}

// Joins a row's pieces of the prefix and of its own tokens: one workgroup per row and head, D/4
// lanes across the dims and as many pieces side by side as fit, then across those in LDS. Rows that
// one tile's walk finished are left alone.
template <uint32_t D>
__global__ __launch_bounds__(kMergeThreads) void attn_batch_merge_kernel(BatchParams p) {
    constexpr uint32_t kLanes = D / 4u;
    constexpr uint32_t kSide = kMergeThreads / kLanes;
    __shared__ float4 acc[kSide][kLanes];
    __shared__ float2 ml[kSide];
    const uint32_t t = blockIdx.x;
    if (t >= min(p.b.row_start[p.b.requests], p.b.max_rows)) return;
    const uint32_t h = blockIdx.y;
    const uint32_t side = threadIdx.x / kLanes;
    const uint32_t c = threadIdx.x % kLanes;
    const Header head = *p.header;
    const RowRecord row = p.row[t];
    // (Row starts that skip a row leave its record unwritten.)
    if (head.per == 0u || row.request >= p.b.requests || p.b.row_start[row.request] + row.row != t ||
        t >= p.b.row_start[row.request + 1u]) return;
    const Record own = p.request[row.request];
    const uint32_t hk = h / p.G;
    const size_t out_row = static_cast<size_t>(t) * p.H + h;
    // The pieces of the prefix [0] and of the own tokens [1]: none, the whole rows, or those of workers
    // first .. first + count - 1.
    struct Pieces {
        uint32_t count, first, at, tile_rows;
        bool whole, later;   // later: the first worker's piece is not its first
    };
    const auto pieces = [&](uint32_t unit0, uint32_t blocks, uint32_t per, uint32_t at, uint32_t tile_rows) {
        Pieces x{0u, 0u, at, tile_rows, false, false};
        if (blocks == 0u) return x;
        x.first = unit0 / per;
        x.count = (unit0 + blocks - 1u) / per - x.first + 1u;
        x.whole = x.count == 1u;
        x.later = x.first * per < unit0;
        return x;
    };
    const uint32_t pr = t * p.G + (h - hk * p.G);         // its row among all rows of the kv head
    const uint32_t orow = row.row * p.G + (h - hk * p.G);   // and among its request's
    Pieces part[2];
    part[0] = head.wide_blocks != 0u ? pieces((hk * head.wide_tiles + pr / kChunkRows) * head.wide_blocks, head.wide_blocks,
                                              head.wide_per, pr % kChunkRows, kChunkRows)
                                     : pieces((hk * head.tiles + pr / kTileRows) * head.blocks, head.blocks, head.per,
                                              pr % kTileRows, kTileRows);
    if (own.wide_head != 0u) {
        const Source src = request_source(p, row.request);
        const uint32_t pre = head.apart != 0u ? p.b.prefix : 0u;
        const WideSpan span(p.G, pre + src.hi, static_cast<int32_t>(pre) + src.pos, p.window);
        const uint32_t tile = orow / kChunkRows;
        part[1] = pieces(own.wide_unit0 + hk * own.wide_head + span.before(tile), span.units(tile), head.wide_per,
                         orow % kChunkRows, kChunkRows);
    } else {
        part[1] = pieces(own.unit0 + (hk * own.tiles + orow / kTileRows) * own.blocks, own.blocks, head.per, orow % kTileRows,
                         kTileRows);
    }
    if (part[1].whole && (head.apart != 0u || (head.blocks == 0u && head.wide_blocks == 0u))) return;
    float m = -__builtin_huge_valf();
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto join = [&](const float2& x, const float4& v) {
        if (x.y == 0.0f) return;   // nothing seen there
        const float m_new = fmaxf(m, x.x);
        const float ref = m_new > -__builtin_huge_valf() ? m_new : 0.0f;
        const float a = __builtin_amdgcn_exp2f(m - ref);
        const float b = __builtin_amdgcn_exp2f(x.x - ref);
        m = m_new;
        l = l * a + x.y * b;
        o = make_float4(o.x * a + v.x * b, o.y * a + v.y * b, o.z * a + v.z * b, o.w * a + v.w * b);
    };
    const uint32_t all = part[0].count + part[1].count;
    for (uint32_t i = side; i < all; i += kSide) {
        const uint32_t k = i < part[0].count ? 0u : 1u;
        const Pieces& x = part[k];
        const uint32_t w = k == 0u ? i : i - part[0].count;
        const uint32_t piece = 2u * (x.first + w) + (w == 0u && x.later ? 1u : 0u);
        const bool wide = x.tile_rows == kChunkRows;
        const size_t r = x.whole ? out_row : static_cast<size_t>(piece) * x.tile_rows + x.at;
        const float2* pml = x.whole ? p.whole_ml[k] : (wide ? p.wide_ml : p.part_ml);
        const float* po = x.whole ? p.whole_o[k] : (wide ? p.wide_o : p.part_o);
        join(pml[r], *reinterpret_cast<const float4*>(po + r * D + 4u * c));
    }
    acc[side][c] = o;
    if (c == 0u) ml[side] = make_float2(m, l);
    __syncthreads();
    if (side != 0u) return;
    for (uint32_t i = 1; i < kSide; ++i) join(ml[i], acc[i][c]);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    *reinterpret_cast<uint2*>(p.out + out_row * D + 4u * c) =
        make_uint2(cvt_pk_bf16(o.x * inv, o.y * inv), cvt_pk_bf16(o.z * inv, o.w * inv));
}

constexpr size_t align256(size_t n) { return (n + 255u) & ~size_t{255u}; }

// The workspace: the header, requests and rows, the rows of whole tiles, the workers' pieces.
struct Layout {
    size_t request, row, whole_ml[2], whole_o[2], ml, o, wide_ml, wide_o, bytes;
};

uint32_t workers_of(uint32_t D) {
    switch (D) {
        case 64: return kWorkers<64>;
        case 128: return kWorkers<128>;
        case 256: return kWorkers<256>;
        default: return kWorkers<512>;
    }
}
uint32_t wide_workers_of(uint32_t D) { return D >= 512u ? kWideWorkers<512> : kWideWorkers<256>; }

Layout layout_of(const BatchView& b, uint32_t H, uint32_t D) {
    const size_t rows = static_cast<size_t>(b.max_rows) * H;
    Layout l{};
    size_t at = 256u;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    l.request = take(b.requests * sizeof(Record));
    l.row = take(b.max_rows * sizeof(RowRecord));
    for (int k = b.prefix != 0u ? 0 : 1; k < 2; ++k) {
        l.whole_ml[k] = take(rows * sizeof(float2));
        l.whole_o[k] = take(rows * D * sizeof(float));
    }
    const size_t pieces = 2u * workers_of(D) * kTileRows, wide = 2u * wide_workers_of(D) * kChunkRows;
    l.ml = take(pieces * sizeof(float2));
    l.o = take(pieces * D * sizeof(float));
    l.wide_ml = take(wide * sizeof(float2));
    l.wide_o = take(wide * D * sizeof(float));
    l.bytes = at;
    return l;
}

template <uint32_t D>
void launch_d(BatchParams p, hipStream_t stream) {
    static_assert(RowsLds<D>::kBytes <= 65536u && sizeof(Header) <= 256u, "batch attention");
    constexpr size_t lds = TilesLds<D>::kBytes;
    if (lds > 65536u) {
        static thread_local int configured_device = -1;
        int dev = 0;
        HYP_HIP_CHECK(hipGetDevice(&dev));
        if (configured_device != dev) {
            HYP_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(attn_batch_tiles_kernel<D>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
            configured_device = dev;
        }
    }
    p.workers = kWorkers<D>;
    p.wide_workers = kWideWorkers<D>;
    const uint32_t scribes = (p.b.requests + kScribeRequests - 1u) / kScribeRequests;
    hipLaunchKernelGGL(attn_batch_rows_kernel<D>, dim3(p.workers + scribes), dim3(64), RowsLds<D>::kBytes, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    if (static_cast<uint64_t>(p.b.max_rows) * p.G > kTileRows) {   // (fewer rows make no wide tile)
        hipLaunchKernelGGL(attn_batch_tiles_kernel<D>, dim3(p.wide_workers), dim3(kTileThreads), lds, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(attn_batch_merge_kernel<D>, dim3(p.b.max_rows, p.H), dim3(kMergeThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace

size_t batch_attention_workspace_bytes(const BatchView& b, uint32_t n_heads, uint32_t head_dim) {
    return layout_of(b, n_heads, head_dim).bytes;
}

void launch_batch_attention(const BatchView& b, const BatchAttentionArgs& a, hipStream_t stream) {
    const Layout l = layout_of(b, a.n_heads, a.head_dim);
    HYP_REQUIRE(a.workspace_bytes >= l.bytes, HYP_STATUS_INVALID_ARGUMENT, "batch attention: workspace too small");
    // Units (tiles times key blocks) are counted in 32 bits.
    const uint64_t G = a.n_heads / a.n_kv_heads;
    const uint64_t tiles = (static_cast<uint64_t>(b.max_rows) * G / kTileRows + std::min(b.requests, b.max_rows) + 1u) * 2u;
    const uint64_t keys = b.prefix + std::min<uint64_t>(static_cast<uint64_t>(b.max_blocks) << b.shift, 1u << 30);
    HYP_REQUIRE(keys < (1ull << 30) && tiles * a.n_kv_heads * (keys / kKeyBlock + 1u) < (1ull << 31),
                HYP_STATUS_INVALID_ARGUMENT, "batch attention: too many rows for tables this long");
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    BatchParams p{};
    p.b = b;
    p.q = a.q;
    p.ck = a.cache_k;
    p.cv = a.cache_v;
    p.out = a.out;
    p.header = reinterpret_cast<Header*>(ws);
    p.request = reinterpret_cast<Record*>(ws + l.request);
    p.row = reinterpret_cast<RowRecord*>(ws + l.row);
    for (int k = 0; k < 2; ++k) {
        p.whole_ml[k] = reinterpret_cast<float2*>(ws + l.whole_ml[k]);
        p.whole_o[k] = reinterpret_cast<float*>(ws + l.whole_o[k]);
    }
    p.part_ml = reinterpret_cast<float2*>(ws + l.ml);
    p.part_o = reinterpret_cast<float*>(ws + l.o);
    p.wide_ml = reinterpret_cast<float2*>(ws + l.wide_ml);
    p.wide_o = reinterpret_cast<float*>(ws + l.wide_o);
    p.H = a.n_heads;
    p.KVH = a.n_kv_heads;
    p.G = static_cast<uint32_t>(G);
    p.window = a.window;
    p.scale = a.scale * kLog2e;
    switch (a.head_dim) {
        case 64: launch_d<64>(p, stream); break;
        case 128: launch_d<128>(p, stream); break;
        case 256: launch_d<256>(p, stream); break;
        case 512: launch_d<512>(p, stream); break;
        default: throw NativeError(HYP_STATUS_UNSUPPORTED, "batch attention: head_dim must be 64, 128, 256 or 512");
    }
}

}  // namespace hyperion::hip
