// Attention of a batch of requests over a paged cache, behind a prefix that all of them share
// (hyp_batch_attention): request r's row i stands at pos = prefix + len_r - n_r + i and sees the
// key positions p <= pos (with a window: p > pos - window) among the prefix's tokens and its own,
//   out = sum_p 2^(s_p - m) v_p / sum_p 2^(s_p - m),   s_p = scale log2(e) q.k_p,
// with no key visible: zeros. A sum over keys splits anywhere (each part keeps its own maximum m,
// sum l and unnormalised O, and parts join as sum_i 2^(m_i - m) O_i), so the prefix is taken for
// all rows of the batch at once, each request's own tokens for its rows, and the parts are joined.
//
// Work is cut evenly whatever the lengths (attention_batch_walk.h): tiles of few rows (16, a wave each) and wide
// tiles (128, a workgroup each), the blocks of 32 keys of each kind dealt out in equal runs to a fixed number of workers.
// A worker that has all of a tile writes its rows; one that has a part leaves a piece, at most two: 2 w for the tile
// its run begins in, 2 w + 1 for the one it ends in. A second launch joins a row's pieces, prefix and own. The
// lengths live on the device, so every worker finds its run itself.
//
// Few rows: a worker is one wave on 16x16x32 products, transposed: S^T = K Q^T with the keys' rows straight from memory
// as the A operand, so a lane holds 8 of a block's keys for one query row and its probabilities are the B
// operand of O^T = V^T P^T as they stand. V rows go to the wave's own LDS (16-byte loads with the
// LDS as destination) and come back by transposing reads. The next block's K rows are requested
// before this one's softmax, its V rows behind its products, its table entries a block earlier; a compute
// unit's other waves keep the memory busy in between. Probabilities enter as two bf16 terms (p and what its
// rounding left): the products wait for memory here, and one term alone would add the error of a second
// rounding to the output's. What bounds it is HBM, each key row read once for up to 16 query rows: 64 decode rows of
// 1 to 1500 tokens without a prefix (8 kv heads of 256, window 1024) take 77 us, 4.7 TB/s; 96 rows of up to 3000 behind
// 777 tokens (8 of 128) 133 us, 4.5 TB/s; a copy reaches 5.0.
//
// Wide: four waves with 32 rows each on 32x32x16 products over K and V blocks that all of them read from LDS, with the
// same two terms of P: one alone halves the products with V but leaves the output 2.4e-3 from the
// 64-bit result in norm where its own rounding leaves 1.7e-3 (as two terms do), and a row would have fewer bits
// where more than 16 share its keys. 24 prompts of 9 to 250 rows behind 6000 tokens (16 heads on one of 512) take
// 718 us with their merge, 629 TFLOP/s of scores and values (943 with the second term) of 1270 that a large matrix
// product reaches, with one term 590; 50 decode rows behind 16001 95 us, with one term 84.
#include <algorithm>

#include "attention.h"
#include "attention_batch_walk.h"
#include "attention_tile.h"
#include "batch.h"
#include "common.h"
#include "q4_rmsnorm.h"

namespace hyperion::hip {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

#define HYP_INLINE __attribute__((always_inline))

constexpr uint32_t kMergeThreads = 256;
constexpr uint32_t kMergeRows = 64;        // (row, head) pairs of a workgroup, at most
constexpr uint32_t kMergeGroups = 2048;    // workgroups before one takes several

// A block of 32 keys in LDS: 1 KB units of 8 keys by 64 dims, the unit of keys 8 o and dims 64 g at
// o D/64 + g, in it each key's 128 bytes as eight 16-byte pieces. One load fills a unit from 8 whole cache
// lines: lane l brings piece l % 8 of key l / 8. (A load whose neighbouring lanes take 16 bytes of
// different rows each runs at half the rate.) Which piece of the row stands where is exchanged by key
// (swizzles below), so that the pieces one operand read takes lie on different banks.
template <uint32_t D>
struct BlockLds {
    static constexpr uint32_t kGroups = D / 64u;
    static constexpr uint32_t kOctet = kGroups * 1024u;       // 8 keys
    static constexpr uint32_t kBytes = 4u * kOctet;
};

// One query row again over its visible keys [j0, j1) of a segment alone, against the same
// reference ref: the matrix products take masked keys with a probability of 0, which a value of V
// that is not finite turns into NaN (and the two terms of a probability make NaN of an infinity). Four keys at a
// time, 16 lanes each; the sums stay unnormalised, dims 64 c + 4 (lane % 16) + e of o[c][e], in every lane.
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
        // (A score of -inf weighs nothing whatever the value is: 0 times one that is not finite would be NaN.)
        if (seen && s * p.scale != -__builtin_huge_valf()) {
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

// Blocks [b0, b1) of tile `tile` of kv head hk of source s.
template <uint32_t D>
__device__ __forceinline__ void rows_segment(const BatchParams& p, const Source& s, const uint32_t* table, bool is_prefix,
                                             uint32_t hk, uint32_t tile, uint32_t b0, uint32_t b1, uint32_t to,
                                             uint32_t piece, uint32_t lds, uint32_t lane) {
    constexpr uint32_t kSteps = D / 32u;
    constexpr uint32_t kDTiles = D / 16u;
    constexpr uint32_t kGroups = BlockLds<D>::kGroups;
    const uint32_t j16 = lane & 15u;
    const uint32_t kb = lane >> 4;
    const uint32_t rows = s.rows * p.G;
    const uint32_t r = tile * kTileRows + j16;
    const bool live = r < rows;
    const uint32_t token = p.by_G.of(live ? r : tile * kTileRows);
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
    const uint32_t stride = p.KVH * D;
    bf16x8_t kf[2][kSteps];
    // Rows of the block that is loaded next: K of keys 16 c + j16 (the operand's), V of keys 8 o + lane / 8.
    const uint16_t* const ck = p.ck + head_at + kb * 8u;
    const uint16_t* const cv = p.cv + head_at + (((lane & 7u) ^ (((lane >> 4) & 3u) << 1)) * 8u);
    uint32_t slot = 0u;   // of key lane % 32
    const auto row_of = [&](uint32_t key) {
        return static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(slot), static_cast<int>(key), 64))) * stride;
    };
    const auto load_k = [&] {
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
            const uint16_t* row = ck + row_of(16u * c + j16);
#pragma unroll
            for (uint32_t st = 0; st < kSteps; ++st) kf[c][st] = *reinterpret_cast<const bf16x8_t*>(row + st * 32u);
        }
    };
    const auto load_v = [&] {
#pragma unroll
        for (uint32_t oc = 0; oc < 4u; ++oc) {
            const uint16_t* row = cv + row_of(8u * oc + (lane >> 3));
#pragma unroll
            for (uint32_t g = 0; g < kGroups; ++g)
                __builtin_amdgcn_global_load_lds((const HYP_GLOBAL void*)(row + g * 64u),
                                                 reinterpret_cast<HYP_LDS void*>(lds + (oc * kGroups + g) * 1024u), 16, 0, 0);
        }
    };
    // From the keys' table entries; a block outside the pool gives slot 0 and a 0 in the mask of keys
    // that are there.
    uint32_t there = 0xFFFFFFFFu;
    const auto slot_from = [&](uint32_t entry, uint32_t j) {
        const bool ok = entry < p.b.num_blocks;
        there = static_cast<uint32_t>(__ballot(ok));
        return ok ? slot_at(entry, j) : 0u;
    };

    f32x4_t o[kDTiles];
#pragma unroll
    for (uint32_t t = 0; t < kDTiles; ++t) o[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_huge_valf();
    float l = 0.0f;

    const uint32_t n32 = lane & 31u;
    const uint32_t j_first = s.lo + b0 * kKeyBlock;
    slot = slot_from(entry_of(j_first + n32), j_first + n32);
    load_k();
    load_v();
    uint32_t entry = entry_of(j_first + kKeyBlock + n32);

    // V operand of dim tile t: group kb reads keys 4 kb + 0..3 (then + 16) at pieces 2 (t % 4) + 0..1 of unit
    // t / 4; pair t % 4 of key k stands at (t % 4) ^ (k / 2 % 4).
    const uint32_t vkey = 4u * kb + (j16 >> 2);
    const uint32_t v_at = lds + (vkey >> 3) * BlockLds<D>::kOctet + (vkey & 7u) * 128u + (((vkey >> 1) & 3u) << 5) +
                          ((j16 >> 1) & 1u) * 16u + (j16 & 1u) * 8u;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t jb = s.lo + b * kKeyBlock;
        const bool more = b + 1u < b1;
        const uint32_t now_there = there;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // K and V of this block have landed
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t sc[2] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (uint32_t st = 0; st < kSteps; ++st)
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
                sc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[c][st], q[st], sc[c], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
            slot = slot_from(entry, jb + kKeyBlock + n32);
            load_k();
            entry = entry_of(jb + 2u * kKeyBlock + n32);
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
#pragma unroll
        for (uint32_t t = 0; t < kDTiles; ++t) {
            const bf16x8_t v = lds_read_tr((v_at ^ ((t % 4u) << 5)) + (t / 4u) * 1024u, 2u * BlockLds<D>::kOctet);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph, o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl, o[t], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // (The products are issued, so their reads of the LDS are done.)
        if (more) load_v();
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
        const uint32_t tok = p.by_G.of(rr);
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

// Wide tiles (attn_batch_tiles_kernel): the arithmetic of attention_chunk.hip's kernel - 128 query rows
// of one kv head, 32 a wave on 32x32x16 products, S^T = K Q^T and O^T = V^T P^T, K and V rows by loads
// straight to two LDS stages - over paged keys. A lane looks up the slot of key lane % 32 of the block
// after the next one, so its table entry has arrived a block before the rows are requested.
// Probabilities enter as two bf16 terms (2^-16 of a weight), as attention_chunk.hip's do where O is rescaled
// lazily: a row's largest one need not be an exact 1.
template <uint32_t D>
struct TilesLds {
    static constexpr uint32_t kV = BlockLds<D>::kBytes;
    static constexpr uint32_t kStage = 2u * BlockLds<D>::kBytes;
    static constexpr uint32_t kOutRow = D * 2u + 16u;
    static constexpr uint32_t kOutChunks = D / 8u;
    static constexpr uint32_t kOut = kChunkRows * kOutRow;
    static constexpr uint32_t kBytes = 2u * kStage > kOut ? 2u * kStage : kOut;
};

constexpr uint32_t kWaveRows = 32;
constexpr float kRescaleLog2 = 8.0f;

struct TileShared {
    int32_t range[kGroupWaves][2];   // the waves' first and last keys
    int32_t pos[kChunkRows];         // positions of a prefix tile's tokens
};

template <uint32_t D>
__device__ __forceinline__ void tile_segment(const BatchParams& p, const Sequence& s, uint32_t hk, uint32_t tile,
                                             uint32_t b0, uint32_t b1, uint32_t to, uint32_t piece, uint32_t lds,
                                             TileShared& shared) {
    using Lds = TilesLds<D>;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 31u;   // this lane's query row of the wave
    const uint32_t h = lane >> 5;
    const uint32_t rows = s.rows * p.G;
    const uint32_t wrow0 = tile * kChunkRows + wave * kWaveRows;
    const uint32_t qrow = min(wrow0 + n, rows - 1u);   // rows past the end repeat the last (not stored)
    const uint32_t qt = p.by_G.of(qrow);
    constexpr uint32_t kSteps = D / 16u;
    constexpr uint32_t kDTiles = D / 32u;
    bf16x8_t q[kSteps];
    {
        const uint16_t* src = p.q + (static_cast<size_t>(s.row0 + qt) * p.H + hk * p.G + (qrow - qt * p.G)) * D + h * 8u;
#pragma unroll
        for (uint32_t st = 0; st < kSteps; ++st) q[st] = *reinterpret_cast<const bf16x8_t*>(src + st * 16u);
    }
    // The keys [first, last] that this lane's row sees, and the blocks that some row of the tile sees.
    int32_t pos = s.pos + static_cast<int32_t>(qt);
    if (s.by_request) {
        pos = 0x3fffffff;   // past the prefix
        if (p.window != 0u || s.pos < static_cast<int32_t>(s.keys) - 1) {
            const uint32_t t0 = p.by_G.of(tile * kChunkRows);
            const uint32_t t1 = p.by_G.of(min((tile + 1u) * kChunkRows, rows) - 1u);
            if (tid < kChunkRows) shared.pos[tid] = -1;   // (a row of no request)
            __syncthreads();
            for (uint32_t r = tid; r < p.b.requests; r += kGroupThreads) {
                const Source src = request_source(p, r);
                for (uint32_t t = max(t0, src.row0); t < src.row0 + src.rows && t <= t1; ++t)
                    shared.pos[t - t0] = static_cast<int32_t>(p.b.prefix) + src.pos + static_cast<int32_t>(t - src.row0);
            }
            __syncthreads();
            pos = shared.pos[qt - t0];
        }
    }
    const int32_t last = min(static_cast<int32_t>(s.keys) - 1, pos);
    const int32_t first = p.window != 0u ? max(0, static_cast<int32_t>(max(static_cast<int64_t>(pos) + 1 - p.window, int64_t{0}))) : 0;
    {
        const int32_t lo = wave_min(first), hi = -wave_min(-last);
        if (lane == 0u) {
            shared.range[wave][0] = lo;
            shared.range[wave][1] = hi;
        }
    }
    __syncthreads();
    int32_t lo = shared.range[0][0], hi = shared.range[0][1];
#pragma unroll
    for (uint32_t w = 1; w < kGroupWaves; ++w) {
        lo = min(lo, shared.range[w][0]);
        hi = max(hi, shared.range[w][1]);
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

    // Wave w loads keys 8 w .. 8 w + 7 of a block, K and V. Piece c of K of key k stands at c ^ k_swz(k), of V
    // at c ^ v_swz(k): an operand read takes one piece of 32 keys of K, four pieces of 8 keys of V.
    constexpr uint32_t kGroups = BlockLds<D>::kGroups;
    const uint32_t stride = p.KVH * D;
    const uint16_t* const ck = p.ck + hk * D;
    const uint16_t* const cv = p.cv + hk * D;
    // Registers are short at head_dim 256 and 512: what follows from the lane alone is formed where it is
    // used, from the lane's number counted anew.
    const auto lane_again = [] {
        uint32_t ln;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(ln));
        return ln;
    };
    size_t at = 0u;   // the row of this lane's key, of the block that is loaded next
    struct Pieces2 {
        const uint16_t *k, *v;
    };
    const auto pieces_at = [&] {
        const uint32_t ln = lane_again();
        const uint32_t k_piece = (ln & 7u) ^ (((ln >> 4) & 3u) | ((wave & 1u) << 2));
        const uint32_t v_piece = (ln & 7u) ^ (((ln >> 4) & 1u) << 2);
        return Pieces2{ck + at + k_piece * 8u, cv + at + v_piece * 8u};
    };
    const auto load_unit = [&](const Pieces2& from, uint32_t st, uint32_t g) {
        const uint32_t to_lds = lds + st * Lds::kStage + (wave * kGroups + g) * 1024u;
        __builtin_amdgcn_global_load_lds((const HYP_GLOBAL void*)(from.k + g * 64u), reinterpret_cast<HYP_LDS void*>(to_lds), 16,
                                         0, 0);
        __builtin_amdgcn_global_load_lds((const HYP_GLOBAL void*)(from.v + g * 64u),
                                         reinterpret_cast<HYP_LDS void*>(to_lds + Lds::kV), 16, 0, 0);
    };
    const auto row_of = [&](uint32_t slot) {
        const uint32_t key = 8u * wave + (lane_again() >> 3);
        return static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(slot), static_cast<int>(key), 64))) * stride;
    };

    f32x16_t o[kDTiles];
#pragma unroll
    for (uint32_t t = 0; t < kDTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -__builtin_huge_valf();   // the softmax reference (log2 domain) of row n
    float l = 0.0f;                     // the sum over this lane's keys

    // K operand of step st: key n, piece 2 (st % 4) + h of unit st / 4.
    constexpr uint32_t kAhead = D == 256u ? 3u : 4u;
    const auto k_address = [&] {
        const uint32_t ln = lane_again();
        const uint32_t key = ln & 31u;
        const uint32_t swz = ((key >> 1) & 3u) | (((key >> 3) & 1u) << 2);
        return lds + (key >> 3) * BlockLds<D>::kOctet + (key & 7u) * 128u + (((ln >> 5) ^ swz) << 4);
    };
    // V operand of dim tile dt, step t: 16-lane group g reads keys 16 t + 4 h + 0..3 (then + 8) at pieces
    // 4 (dt % 2) + 2 (g % 2) + 0..1 of unit dt / 2.
    const auto v_address = [&] {
        const uint32_t ln = lane_again();
        const uint32_t key = 4u * (ln >> 5) + ((ln >> 2) & 3u);
        return lds + Lds::kV + key * 128u + (((key >> 1) & 1u) << 6) + ((ln >> 4) & 1u) * 32u + ((ln >> 1) & 1u) * 16u +
               (ln & 1u) * 8u;
    };

    uint32_t entry = 0u;
    if (b0 < b1) {
        at = row_of(slot_from(entry_of(b0 * kKeyBlock + n), b0 * kKeyBlock + n));
        entry = entry_of((b0 + 1u) * kKeyBlock + n);
#pragma unroll
        for (uint32_t g = 0; g < kGroups; ++g) load_unit(pieces_at(), 0u, g);
    }
    const auto v_read = [&](uint32_t v_at, uint32_t v_odd, uint32_t u) {   // v_at, v_odd: of even and odd dim tiles
        const uint32_t dt = u / 2u;
        return lds_read_tr((dt % 2u == 0u ? v_at : v_odd) + (dt / 2u) * 1024u + (u % 2u) * 2u * BlockLds<D>::kOctet,
                           BlockLds<D>::kOctet);
    };
    constexpr uint32_t kProducts = 2u * kDTiles;
    float mx = 0.0f;
    // As attention_chunk.hip at head_dim 512: O is rescaled only when a row's maximum has grown by more than
    // 2^kRescaleLog2 since the last time. A block that outgrows the reference ends the inner loop before it
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
                if (b + 1u < b1) at = row_of(slot_from(entry, jb + kKeyBlock + (lane_again() & 31u)));
            }
            again = false;
            const uint32_t stage_n = (b + 1u - b0) & 1u;
            const uint32_t k_at = k_address() + stage;
            const auto k_read = [&](uint32_t st) { return lds_read16((k_at ^ ((st % 4u) << 5)) + (st / 4u) * 1024u); };
            f32x16_t sc;
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
            bf16x8_t kf[kAhead];
            const Pieces2 from = pieces_at();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t st = 0; st < kAhead; ++st) kf[st] = k_read(st);
#pragma unroll
            for (uint32_t st = 0; st < kSteps; ++st) {
                __builtin_amdgcn_sched_barrier(0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[st % kAhead], q[st], sc, 0, 0, 0);
                if (st + kAhead < kSteps) kf[st % kAhead] = k_read(st + kAhead);
                if (st % 4u == 1u) load_unit(from, stage_n, st / 4u);
            }
            __builtin_amdgcn_sched_barrier(0);
            const uint32_t entry_next = entry_of(jb + 2u * kKeyBlock + (lane_again() & 31u));
            bf16x8_t vf[kAhead];
            const uint32_t v_at = v_address() + stage;
            const uint32_t v_odd = v_at ^ 64u;
            if constexpr (D != 256u) {   // (at 256 their registers are short)
#pragma unroll
                for (uint32_t u = 0; u < kAhead; ++u) vf[u] = v_read(v_at, v_odd, u);
                __builtin_amdgcn_sched_barrier(0);
            }

            // sc[i] is key jb + 8 (i / 4) + 4 h + i % 4 of row n.
            if (now_there != 0xFFFFFFFFu || __any(static_cast<int32_t>(jb + kKeyBlock) - 1 > last || static_cast<int32_t>(jb) < first)) {
#pragma unroll
                for (uint32_t i = 0; i < 16u; ++i) {
                    const uint32_t k = 8u * (i / 4u) + 4u * h + (i & 3u);
                    const int32_t j = static_cast<int32_t>(jb + k);
                    sc[i] = j <= last && j >= first && ((now_there >> k) & 1u) != 0u ? sc[i] : -__builtin_huge_valf();
                }
            }
            mx = sc[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
            mx = half_max(mx) * p.scale;
            m = m == -__builtin_huge_valf() ? mx : m;   // O is still zero: nothing to rescale
            if (__any(mx > m + kRescaleLog2)) {
                again = true;
                break;
            }
            entry = entry_next;
            const float ref = m > -__builtin_huge_valf() ? m : 0.0f;
            float pr[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) pr[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], p.scale, -ref));
            // Two bf16 terms of each; the row's sum takes both, as the products do.
            bf16x8_t pb[2], pl[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t two[4], rest[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = pr[8 * t + 2 * i], b = pr[8 * t + 2 * i + 1];
                    two[i] = cvt_pk_bf16(a, b);
                    rest[i] = cvt_pk_bf16(a - bf16_bits_to_f32(two[i] & 0xFFFFu), b - __uint_as_float(two[i] & 0xFFFF0000u));
                    l += a + b;
                }
                pb[t] = __builtin_bit_cast(bf16x8_t, make_uint4(two[0], two[1], two[2], two[3]));
                pl[t] = __builtin_bit_cast(bf16x8_t, make_uint4(rest[0], rest[1], rest[2], rest[3]));
            }
            if constexpr (D == 256u) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t u = 0; u < kAhead; ++u) vf[u] = v_read(v_at, v_odd, u);
            }
#pragma unroll
            for (uint32_t u = 0; u < kProducts; ++u) {
                __builtin_amdgcn_sched_barrier(0);
                o[u / 2u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[u % kAhead], pb[u % 2u], o[u / 2u], 0, 0, 0);
                o[u / 2u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[u % kAhead], pl[u % 2u], o[u / 2u], 0, 0, 0);
                if (u + kAhead < kProducts) vf[u % kAhead] = v_read(v_at, v_odd, u + kAhead);
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

    const uint32_t ln = lane_again();
    const uint32_t on = ln & 31u, oh = ln >> 5;   // this lane's row and half again
    const bool live = wrow0 + on < rows;
    const uint32_t ot = p.by_G.of(wrow0 + on);
    const size_t out_row = static_cast<size_t>(s.row0 + ot) * p.H + hk * p.G + (wrow0 + on - ot * p.G);
    float zero = 0.0f;
#pragma unroll
    for (uint32_t dt = 0; dt < kDTiles; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = fmaf(o[dt][i], 0.0f, zero);
    const uint64_t odd_lanes = __ballot(zero != 0.0f && live);
    const uint32_t odd_rows = static_cast<uint32_t>(odd_lanes) | static_cast<uint32_t>(odd_lanes >> 32);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const size_t prow = to == kToRows ? out_row : static_cast<size_t>(piece) * kChunkRows + wave * kWaveRows + on;
    float* const po = to == kToRows ? p.whole_o[s.by_request ? 0 : 1] : p.wide_o;

    // o[dt][i] is dim 32 dt + 8 (i / 4) + 4 h + i % 4 of row n.
    __syncthreads();   // every wave has left the stages
    if (to != kToOutput) {
        if (live) {
#pragma unroll
            for (uint32_t dt = 0; dt < kDTiles; ++dt)
#pragma unroll
                for (uint32_t u = 0; u < 4u; ++u)
                    *reinterpret_cast<float4*>(po + prow * D + 32u * dt + 8u * u + 4u * oh) =
                        make_float4(o[dt][4 * u], o[dt][4 * u + 1], o[dt][4 * u + 2], o[dt][4 * u + 3]);
            if (oh == 0u) (to == kToRows ? p.whole_ml[s.by_request ? 0 : 1] : p.wide_ml)[prow] = make_float2(m, l);
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
                *reinterpret_cast<HYP_LDS u32x2_t*>(out_lds + on * Lds::kOutRow + (32u * dt + 8u * u + 4u * oh) * 2u) = w;
            }
        __syncthreads();
        for (uint32_t c = ln; c < kWaveRows * Lds::kOutChunks; c += 64u) {
            const uint32_t r = c / Lds::kOutChunks;
            const uint32_t gr = wrow0 + r;
            if (gr >= rows) break;
            const uint32_t t = p.by_G.of(gr);
            const size_t dst = (static_cast<size_t>(s.row0 + t) * p.H + hk * p.G + (gr - t * p.G)) * D + (c % Lds::kOutChunks) * 8u;
            *reinterpret_cast<u32x4_t*>(p.out + dst) =
                *reinterpret_cast<const HYP_LDS u32x4_t*>(out_lds + r * Lds::kOutRow + (c % Lds::kOutChunks) * 16u);
        }
        __syncthreads();   // the next segment's loads go to the same place
    }
    if (odd_rows == 0u) return;
    // Rows with a value that is not finite are formed again, by themselves.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's own stores of these rows are done
    for (uint32_t todo = odd_rows; todo != 0u; todo &= todo - 1u) {
        const uint32_t i = __builtin_ctz(todo);
        const uint32_t tok = p.by_G.of(wrow0 + i);
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

// Workgroups: as many as the device holds at once.
constexpr uint32_t groups_of(uint32_t D, bool wide) {
    return kComputeUnits * (D >= 512u ? 1u : (wide || D == 256u ? 2u : (D == 128u ? 3u : 4u)));
}

// Without kWide every tile is of few rows (Walk). Both kinds go in one launch: two launches, one after the
// other (wide tiles with one term of P), took 124 us for one's 107 (64 rows behind 2000 tokens at head_dim 256, window 1024), 173 for 133 (96
// rows behind 777 at 128) and 115 for 111 (50 rows behind 16001 at 512).
template <uint32_t D, bool kWide>
__global__ __launch_bounds__(kGroupThreads, groups_of(D, kWide) / kComputeUnits) void attn_batch_kernel(BatchParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds_mem[];
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((HYP_LDS uint8_t*)lds_mem));
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = scalar(threadIdx.x >> 6);
    constexpr uint32_t kGroups = groups_of(D, kWide);
    if (blockIdx.x >= kGroups) {
        scribe<kWide>(p, ((blockIdx.x - kGroups) * kGroupWaves + wave) * 64u, lane);
        return;
    }
    worker_units<kWide>(
        p, blockIdx.x, wave, lane,
        [&](const Sequence& s, uint32_t hk, uint32_t tile, uint32_t b0, uint32_t b1, uint32_t to, uint32_t piece) HYP_INLINE {
            if constexpr (kWide) {
                __shared__ TileShared shared;
                tile_segment<D>(p, s, hk, tile, b0, b1, to, piece, lds, shared);
            }
        },
        [&](uint32_t piece) HYP_INLINE {
            if (threadIdx.x < kChunkRows)
                p.wide_ml[static_cast<size_t>(piece) * kChunkRows + threadIdx.x] = make_float2(-__builtin_huge_valf(), 0.0f);
        },
        [&](const Source& s, const uint32_t* table, bool is_prefix, uint32_t hk, uint32_t tile, uint32_t b0, uint32_t b1,
            uint32_t to, uint32_t piece) HYP_INLINE {
            rows_segment<D>(p, s, table, is_prefix, hk, tile, b0, b1, to, piece, lds + wave * BlockLds<D>::kBytes, lane);
        });
}

// Joins the pieces of rows that one tile's walk did not finish. A workgroup takes `each` consecutive
// (row, head) pairs: its first threads find their pieces, one pair a thread, then all of it joins the
// pairs that have any left: D/4 lanes across the dims and as many pieces side by side as fit, then across
// those in LDS.
template <uint32_t D>
__global__ __launch_bounds__(kMergeThreads) void attn_batch_merge_kernel(BatchParams p, Divisor by_H, uint32_t each) {
    constexpr uint32_t kLanes = D / 4u;
    constexpr uint32_t kSide = kMergeThreads / kLanes;
    __shared__ float4 acc[kSide][kLanes];
    __shared__ float2 ml[kSide];
    __shared__ Pieces found[kMergeRows][2];
    __shared__ uint64_t todo_of;
    const uint32_t first_pair = blockIdx.x * each;
    if (threadIdx.x < 64u) {
        const uint32_t pair = first_pair + threadIdx.x;
        const uint32_t t = by_H.of(pair);
        const uint32_t h = pair - t * p.H;
        bool todo = threadIdx.x < each && t < min(p.b.row_start[p.b.requests], p.b.max_rows);
        if (todo) {
            Pieces a, b;
            todo = row_pieces(p, t, h, a, b);
            if (todo) {
                found[threadIdx.x][0] = a;
                found[threadIdx.x][1] = b;
            }
        }
        const uint64_t left = __ballot(todo);
        if (threadIdx.x == 0u) todo_of = left;
    }
    __syncthreads();
    const uint32_t side = threadIdx.x / kLanes;
    const uint32_t c = threadIdx.x % kLanes;
    for (uint64_t todo = todo_of; todo != 0u; todo &= todo - 1u) {
        const uint32_t i = static_cast<uint32_t>(__builtin_ctzll(todo));
        const size_t out_row = first_pair + i;
        const Pieces a = found[i][0], b = found[i][1];
        float m = -__builtin_huge_valf();
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const auto join = [&](const float2& x, const float4& v) {
            if (x.y == 0.0f) return;   // nothing seen there
            const float m_new = fmaxf(m, x.x);
            const float ref = m_new > -__builtin_huge_valf() ? m_new : 0.0f;
            const float f = __builtin_amdgcn_exp2f(m - ref);
            const float g = __builtin_amdgcn_exp2f(x.x - ref);
            m = m_new;
            l = l * f + x.y * g;
            o = make_float4(o.x * f + v.x * g, o.y * f + v.y * g, o.z * f + v.z * g, o.w * f + v.w * g);
        };
        const uint32_t all = a.count + b.count;
        const auto load = [&](uint32_t k, float2& x, float4& v) {
            const bool own = k >= a.count;
            const uint32_t w = own ? k - a.count : k;
            const bool whole = (own ? b.count : a.count) == 1u;
            const bool wide = own ? b.wide : a.wide;
            const uint32_t place = w == 0u ? (own ? b.place : a.place) : (own ? b.next : a.next) + 2u * (w - 1u);
            const size_t r = whole ? out_row : static_cast<size_t>(place) * (wide ? kChunkRows : kTileRows) + (own ? b.at : a.at);
            const float2* pml = whole ? p.whole_ml[own ? 1 : 0] : (wide ? p.wide_ml : p.part_ml);
            const float* po = whole ? p.whole_o[own ? 1 : 0] : (wide ? p.wide_o : p.part_o);
            x = pml[r];
            v = *reinterpret_cast<const float4*>(po + r * D + 4u * c);
        };
        // Four pieces in flight.
        for (uint32_t k = side; k < all; k += 4u * kSide) {
            float2 x[4];
            float4 v[4];
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u) {
                x[u] = make_float2(0.0f, 0.0f);
                if (k + u * kSide < all) load(k + u * kSide, x[u], v[u]);
            }
#pragma unroll
            for (uint32_t u = 0; u < 4u; ++u) join(x[u], v[u]);
        }
        acc[side][c] = o;
        if (c == 0u) ml[side] = make_float2(m, l);
        __syncthreads();
        if (side == 0u) {
            for (uint32_t k = 1; k < kSide; ++k) join(ml[k], acc[k][c]);
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            *reinterpret_cast<uint2*>(p.out + out_row * D + 4u * c) =
                make_uint2(cvt_pk_bf16(o.x * inv, o.y * inv), cvt_pk_bf16(o.z * inv, o.w * inv));
        }
        __syncthreads();
    }
}

constexpr size_t align256(size_t n) { return (n + 255u) & ~size_t{255u}; }

// The workspace: the header, requests and rows, the rows of whole tiles, the workers' pieces.
struct Layout {
    size_t request, row, whole_ml[2], whole_o[2], ml, o, wide_ml, wide_o, bytes;
};

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
    const size_t pieces = 2u * groups_of(D, false) * kGroupWaves * kTileRows, wide = 2u * groups_of(D, true) * kChunkRows;
    l.ml = take(pieces * sizeof(float2));
    l.o = take(pieces * D * sizeof(float));
    l.wide_ml = take(wide * sizeof(float2));
    l.wide_o = take(wide * D * sizeof(float));
    l.bytes = at;
    return l;
}

template <uint32_t D, bool kWide>
void launch_walk(BatchParams p, hipStream_t stream) {
    constexpr size_t few = kGroupWaves * BlockLds<D>::kBytes;
    constexpr size_t lds = kWide && TilesLds<D>::kBytes > few ? TilesLds<D>::kBytes : few;
    static_assert(lds + sizeof(TileShared) <= 160u * 1024u && sizeof(Header) <= 256u, "batch attention");
    if (lds + sizeof(TileShared) > 65536u) {
        static thread_local int configured_device = -1;
        int dev = 0;
        HYP_HIP_CHECK(hipGetDevice(&dev));
        if (configured_device != dev) {
            HYP_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(attn_batch_kernel<D, kWide>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
            configured_device = dev;
        }
    }
    p.groups = groups_of(D, kWide);
    // Of two kinds of tile each gets a share of the workgroups. Measured with half of these up to three times as much
    // (us, here first): head_dim 512, 50 rows behind 16001 tokens 92, 97 with 1, 100 with 3; 90 rows of up to 1500
    // behind 700 57, 71 with 1, 53 with 3. 256 (window 1024), 64 rows of up to 1500 behind 2000 97, 105 with 4, 98 with
    // 8. 128, 50 of up to 600 behind 16001 61, 56 with 3, 78 with 8; 96 of up to 3000 behind 777 132, 134, 134. 64, 48
    // of up to 600 behind 12000 34, 34 with 2, 41 with 4; 64 of up to 1500 behind 2000 37, 40, 38.
    p.wide_cost = D >= 512u ? 2.0f : (D == 256u ? 5.5f : (D == 128u ? 4.0f : 3.0f));
    const uint32_t scribes = (p.b.requests + 64u * kGroupWaves - 1u) / (64u * kGroupWaves);
    hipLaunchKernelGGL((attn_batch_kernel<D, kWide>), dim3(p.groups + scribes), dim3(kGroupThreads), lds, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

template <uint32_t D>
void launch_d(const BatchParams& p, hipStream_t stream) {
    // Tiles of few rows alone where no more than 16 rows of a kv head can be, and without a prefix where
    // there are no more rows than requests (a decode step; should one request hold many of them, its keys are
    // read for every 16). Without the wide tiles' registers 64 decode rows took 77 us, not 84 (head_dim 256,
    // no prefix), 4 rows behind 100 tokens 12.5, not 13.8.
    if (static_cast<uint64_t>(p.b.max_rows) * p.G <= kTileRows ||
        (p.b.prefix == 0u && p.b.max_rows <= p.b.requests && p.G <= kTileRows)) {
        launch_walk<D, false>(p, stream);
    } else {
        launch_walk<D, true>(p, stream);
    }
    const uint64_t pairs = static_cast<uint64_t>(p.b.max_rows) * p.H;
    const uint32_t each = static_cast<uint32_t>(std::min<uint64_t>((pairs + kMergeGroups - 1u) / kMergeGroups, kMergeRows));
    hipLaunchKernelGGL(attn_batch_merge_kernel<D>, dim3(static_cast<uint32_t>((pairs + each - 1u) / each)),
                       dim3(kMergeThreads), 0, stream, p, Divisor(p.H), each);
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
    HYP_REQUIRE(keys < (1ull << 30) && tiles * a.n_kv_heads * (keys / kKeyBlock + 1u + kTileCost) < (1ull << 31),
                HYP_STATUS_INVALID_ARGUMENT, "batch attention: too many rows for tables this long");
    const uint64_t q_bytes = static_cast<uint64_t>(b.max_rows) * a.n_heads * a.head_dim * 2u;
    HYP_REQUIRE(!overlap(a.out, q_bytes, a.q, q_bytes) && !overlap(a.workspace, l.bytes, a.q, q_bytes) &&
                    !overlap(a.workspace, l.bytes, a.out, q_bytes),
                HYP_STATUS_INVALID_ARGUMENT, "batch attention: q, out and workspace must not overlap");
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
    p.by_G = Divisor(p.G);
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
