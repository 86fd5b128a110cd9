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

struct BatchParams {
    BatchView b;
    const uint16_t* q;
    const uint16_t* ck;
    const uint16_t* cv;
    uint16_t* out;
    uint4* header;      // {units a worker, prefix blocks, prefix tiles, 0}
    uint4* request;     // {first unit, first group, tiles, blocks}
    uint2* row;         // {request, row in the request}
    float2* part_ml;    // [part][kTileRows]
    float* part_o;      // [part][kTileRows][D]
    uint32_t H, KVH, G, window, workers;
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

// A request's (or the prefix's) part of the work.
struct Source {
    uint32_t row0, rows;   // query rows (tokens)
    uint32_t lo, hi;       // keys [lo, hi) that some row sees
    int32_t pos;           // the first row's position, counted from the source's key 0
    uint32_t tiles, blocks;
    __device__ uint32_t units(uint32_t KVH) const { return KVH * tiles * blocks; }
    __device__ uint32_t groups(uint32_t KVH) const { return blocks != 0u ? KVH * tiles : 0u; }
};

__device__ __forceinline__ uint32_t tiles_of(uint32_t rows, uint32_t G) { return (rows * G + kTileRows - 1u) / kTileRows; }

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

// The batch's walk as one wave sees it: 64 requests across its lanes at a time.
struct Walk {
    Source mine;                // this lane's request of the chunk
    uint32_t chunk = 0;         // first request of the chunk
    uint32_t units0, groups0;   // before the chunk
    uint32_t units1, groups1;   // inclusive sums over the chunk's lanes
    Source prefix;
    uint32_t total;             // units of all

    __device__ void load(const BatchParams& p, uint32_t lane) {
        mine = request_source(p, chunk + lane);
        units1 = wave_incl(mine.units(p.KVH), lane);
        groups1 = wave_incl(mine.groups(p.KVH), lane);
    }
    // Totals of the batch and the prefix's part; then the first chunk. Returns units a worker; 0
    // where the row starts are no rows of the batch (they would pass the workspace).
    __device__ uint32_t open(const BatchParams& p, uint32_t lane) {
        uint32_t units = 0u, most = 0u, rows = 0u, sum = 0u;
        int32_t first = 0x7fffffff;
        for (uint32_t r = lane; r < p.b.requests; r += 64u) {
            const Source s = request_source(p, r);
            sum = min(sum + s.rows, 1u << 25);
            units += s.units(p.KVH);
            most = max(most, s.blocks);
            rows = max(rows, s.row0 + s.rows);
            if (s.rows != 0u) first = min(first, s.pos);
        }
        if (static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(wave_sum(sum))) > p.b.max_rows) return 0u;
        units = __builtin_amdgcn_readfirstlane(wave_sum(units));
        most = __builtin_amdgcn_readfirstlane(wave_max(most));
        rows = __builtin_amdgcn_readfirstlane(wave_max(rows));
        first = __builtin_amdgcn_readfirstlane(wave_min(first));
        prefix = Source{0u, rows, 0u, p.b.prefix, 0, 0u, 0u};
        if (rows != 0u) {
            prefix.pos = static_cast<int32_t>(p.b.prefix) + first;   // the least of all rows
            if (p.window != 0u && static_cast<int64_t>(prefix.pos) + 1 > p.window) prefix.lo = prefix.pos + 1u - p.window;
            prefix.tiles = tiles_of(rows, p.G);
            if (prefix.hi > prefix.lo) prefix.blocks = (prefix.hi - prefix.lo + kKeyBlock - 1u) / kKeyBlock;
        }
        most = max(most, prefix.blocks);
        total = units + prefix.units(p.KVH);
        units0 = prefix.units(p.KVH);
        groups0 = prefix.groups(p.KVH);
        load(p, lane);
        return max(max((total + p.workers - 1u) / p.workers, (most + kMaxParts - 2u) / (kMaxParts - 1u)), 1u);
    }
    // On to the chunk that holds unit u (u >= units0).
    __device__ void seek(const BatchParams& p, uint32_t u, uint32_t lane) {
        while (chunk + 64u < p.b.requests && u >= units0 + __builtin_amdgcn_readlane(units1, 63)) next(p, lane);
    }
    __device__ void next(const BatchParams& p, uint32_t lane) {
        units0 += __builtin_amdgcn_readlane(units1, 63);
        groups0 += __builtin_amdgcn_readlane(groups1, 63);
        chunk += 64u;
        load(p, lane);
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

// Blocks [b0, b1) of tile `tile` of kv head hk of source s into part `part`.
template <uint32_t D>
__device__ __forceinline__ void rows_segment(const BatchParams& p, const Source& s, const uint32_t* table, bool is_prefix,
                                             uint32_t hk, uint32_t tile, uint32_t b0, uint32_t b1, uint32_t part,
                                             uint32_t lds, uint32_t lane) {
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
    const size_t prow = static_cast<size_t>(part) * kTileRows + j16;
    if (live) {
#pragma unroll
        for (uint32_t t = 0; t < kDTiles; ++t)
            *reinterpret_cast<float4*>(p.part_o + prow * D + 16u * t + 4u * kb) =
                make_float4(o[t][0], o[t][1], o[t][2], o[t][3]);
        if (kb == 0u) p.part_ml[prow] = make_float2(m, l);
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
        if (lane < 16u) {
#pragma unroll
            for (uint32_t c = 0; c < D / 64u; ++c)
                *reinterpret_cast<float4*>(p.part_o + (static_cast<size_t>(part) * kTileRows + i) * D + 64u * c + 4u * lane) =
                    make_float4(a[c][0], a[c][1], a[c][2], a[c][3]);
        }
    }
}

// What the merge needs of the walk: the chunk's requests and their rows.
__device__ __forceinline__ void scribe(const BatchParams& p, Walk& w, uint32_t per, uint32_t chunk, uint32_t lane) {
    if (chunk == 0u && lane == 0u) *p.header = make_uint4(per, w.prefix.blocks, w.prefix.tiles, 0u);
    if (per == 0u) return;
    while (w.chunk < chunk) w.next(p, lane);
    const Source& s = w.mine;
    const uint32_t r = chunk + lane;
    if (r < p.b.requests) {
        p.request[r] = make_uint4(w.units0 + w.units1 - s.units(p.KVH), w.groups0 + w.groups1 - s.groups(p.KVH), s.tiles,
                                  s.blocks);
    }
    for (uint32_t i = 0; i < 64u; ++i) {
        const uint32_t row0 = __builtin_amdgcn_readlane(s.row0, i);
        const uint32_t rows = __builtin_amdgcn_readlane(s.rows, i);
        for (uint32_t t = lane; t < rows; t += 64u) p.row[row0 + t] = make_uint2(chunk + i, t);
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
        uint32_t unit0 = 0u, group0 = 0u;
        bool is_prefix = true;
        if (u >= w.prefix.units(p.KVH)) {
            w.seek(p, u, lane);
            const uint64_t behind = __ballot(u < w.units0 + w.units1);
            if (behind == 0u) return;   // (not with u below the total)
            const uint32_t at = __builtin_ctzll(behind);
            s = shfl_source(w.mine, at);
            table = p.b.tables + static_cast<size_t>(w.chunk + at) * p.b.max_blocks;
            unit0 = w.units0 + __builtin_amdgcn_readlane(w.units1, at) - s.units(p.KVH);
            group0 = w.groups0 + __builtin_amdgcn_readlane(w.groups1, at) - s.groups(p.KVH);
            is_prefix = false;
        }
        const uint32_t g = (u - unit0) / s.blocks;
        const uint32_t b0 = u - unit0 - g * s.blocks;
        const uint32_t b1 = min(s.blocks, b0 + (end - u));
        const uint32_t hk = g / s.tiles;
        rows_segment<D>(p, s, table, is_prefix, __builtin_amdgcn_readfirstlane(hk),
                        __builtin_amdgcn_readfirstlane(g - hk * s.tiles), __builtin_amdgcn_readfirstlane(b0),
                        __builtin_amdgcn_readfirstlane(b1), blockIdx.x + group0 + g, lds, lane);
        u += b1 - b0;
    }
}

// Joins a row's parts of the prefix and of its own tokens: one workgroup per row and head, D/4
// lanes across the dims and as many parts side by side as fit, then across those in LDS.
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
    const uint4 head = *p.header;
    const uint2 row = p.row[t];
    // (Row starts that skip a row leave its record unwritten.)
    if (head.x == 0u || row.x >= p.b.requests || p.b.row_start[row.x] + row.y != t ||
        t >= p.b.row_start[row.x + 1u]) return;
    const uint4 own = p.request[row.x];
    const uint32_t hk = h / p.G;
    // Parts [first, first + count) at row `at` of their tile, of the prefix and of the own tokens.
    uint32_t first[2], count[2], at[2];
    const auto parts = [&](uint32_t k, uint32_t token, uint32_t unit0, uint32_t group0, uint32_t tiles, uint32_t blocks) {
        const uint32_t r = token * p.G + (h - hk * p.G);
        const uint32_t g = hk * tiles + r / kTileRows;
        at[k] = r % kTileRows;
        count[k] = 0u;
        if (blocks == 0u) return;
        const uint32_t u = unit0 + g * blocks;
        const uint32_t w0 = u / head.x;
        first[k] = w0 + group0 + g;
        count[k] = (u + blocks - 1u) / head.x - w0 + 1u;
    };
    parts(0u, t, 0u, 0u, head.z, head.y);
    parts(1u, row.y, own.x, own.y, own.z, own.w);
    const auto part_row = [&](uint32_t i) {
        return i < count[0] ? static_cast<size_t>(first[0] + i) * kTileRows + at[0]
                            : static_cast<size_t>(first[1] + (i - count[0])) * kTileRows + at[1];
    };
    const uint32_t all = count[0] + count[1];
    float m = -__builtin_huge_valf();
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto join = [&](float mi, float li, const float4& v) {
        const float m_new = fmaxf(m, mi);
        const float ref = m_new > -__builtin_huge_valf() ? m_new : 0.0f;
        const float a = __builtin_amdgcn_exp2f(m - ref);
        const float b = __builtin_amdgcn_exp2f(mi - ref);
        m = m_new;
        l = l * a + li * b;
        o = make_float4(o.x * a + v.x * b, o.y * a + v.y * b, o.z * a + v.z * b, o.w * a + v.w * b);
    };
    for (uint32_t i = side; i < all; i += kSide) {
        const size_t r = part_row(i);
        const float2 x = p.part_ml[r];
        join(x.x, x.y, *reinterpret_cast<const float4*>(p.part_o + r * D + 4u * c));
    }
    acc[side][c] = o;
    if (c == 0u) ml[side] = make_float2(m, l);
    __syncthreads();
    if (side != 0u) return;
    for (uint32_t i = 1; i < kSide; ++i) join(ml[i].x, ml[i].y, acc[i][c]);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(t) * p.H + h) * D + 4u * c) =
        make_uint2(cvt_pk_bf16(o.x * inv, o.y * inv), cvt_pk_bf16(o.z * inv, o.w * inv));
}

constexpr size_t align256(size_t n) { return (n + 255u) & ~size_t{255u}; }

// The workspace: the header, requests, rows, and the parts of every worker and group.
struct Layout {
    size_t request, row, ml, o, bytes;
    uint64_t groups, parts;
};

uint32_t workers_of(uint32_t D) {
    switch (D) {
        case 64: return kWorkers<64>;
        case 128: return kWorkers<128>;
        case 256: return kWorkers<256>;
        default: return kWorkers<512>;
    }
}

Layout layout_of(const BatchView& b, uint32_t H, uint32_t KVH, uint32_t D) {
    const uint64_t G = H / KVH;
    const uint64_t rows = b.max_rows;
    const uint64_t whole = (rows * G + kTileRows - 1u) / kTileRows;
    // A request's last tile may be short, so each adds at most one to the rows' own.
    const uint64_t own = rows * G / kTileRows + std::min<uint64_t>(b.requests, rows);
    Layout l{};
    l.groups = KVH * (own + (b.prefix != 0u ? whole : 0u));
    l.parts = workers_of(D) + l.groups;
    l.request = 256u;
    l.row = l.request + align256(b.requests * sizeof(uint4));
    l.ml = l.row + align256(rows * sizeof(uint2));
    l.o = l.ml + align256(l.parts * kTileRows * sizeof(float2));
    l.bytes = l.o + l.parts * kTileRows * D * sizeof(float);
    return l;
}

template <uint32_t D>
void launch_d(BatchParams p, hipStream_t stream) {
    static_assert(RowsLds<D>::kBytes <= 65536u, "batch attention LDS");
    p.workers = kWorkers<D>;
    const uint32_t scribes = (p.b.requests + kScribeRequests - 1u) / kScribeRequests;
    hipLaunchKernelGGL(attn_batch_rows_kernel<D>, dim3(p.workers + scribes), dim3(64), RowsLds<D>::kBytes, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(attn_batch_merge_kernel<D>, dim3(p.b.max_rows, p.H), dim3(kMergeThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace

size_t batch_attention_workspace_bytes(const BatchView& b, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
    return layout_of(b, n_heads, n_kv_heads, head_dim).bytes;
}

void launch_batch_attention(const BatchView& b, const BatchAttentionArgs& a, hipStream_t stream) {
    const Layout l = layout_of(b, a.n_heads, a.n_kv_heads, a.head_dim);
    HYP_REQUIRE(a.workspace_bytes >= l.bytes, HYP_STATUS_INVALID_ARGUMENT, "batch attention: workspace too small");
    // Units are counted in 32 bits.
    const uint64_t keys = std::max<uint64_t>(b.prefix, std::min<uint64_t>(static_cast<uint64_t>(b.max_blocks) << b.shift, 1u << 30));
    HYP_REQUIRE(l.groups * (keys / kKeyBlock + 1u) < (1ull << 31), HYP_STATUS_INVALID_ARGUMENT,
                "batch attention: too many rows for tables this long");
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    BatchParams p{};
    p.b = b;
    p.q = a.q;
    p.ck = a.cache_k;
    p.cv = a.cache_v;
    p.out = a.out;
    p.header = reinterpret_cast<uint4*>(ws);
    p.request = reinterpret_cast<uint4*>(ws + l.request);
    p.row = reinterpret_cast<uint2*>(ws + l.row);
    p.part_ml = reinterpret_cast<float2*>(ws + l.ml);
    p.part_o = reinterpret_cast<float*>(ws + l.o);
    p.H = a.n_heads;
    p.KVH = a.n_kv_heads;
    p.G = a.n_heads / a.n_kv_heads;
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
