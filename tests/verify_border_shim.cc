// hyp_verify_batch's search for the end of a row's filters (csrc/verify_border.h) run on the host, a wave of 64 lanes at a
// time: rows whose running sums and weights meet a filter's border to a few roundings, for test_verify_border_cpu.py.
#include <cmath>
#include <cstdio>
#include <random>

#include "verify_border.h"

using namespace hyperion::hip;

namespace {

constexpr uint32_t kLanes = 64, kSlots = 33;

struct Row {
    uint32_t n[kLanes][kSlots];
    double w[kLanes][kSlots];      // a value's own weight
    double rough[kLanes];          // a lane's mass by other roundings
    bool light[kLanes];
    double mass0;                  // of the waves before
    uint32_t count0;
    double enough, min_p;          // 0: off
};

double nudged(double v, int ulps) {
    for (; ulps > 0; --ulps) v = std::nextafter(v, 1e300);
    for (; ulps < 0; ++ulps) v = std::nextafter(v, 0.0);
    return v;
}

Row row_of(std::mt19937_64& rng) {
    const auto below = [&](uint32_t n) { return static_cast<uint32_t>(rng() % n); };
    const auto unit = [&] { return static_cast<double>(rng() >> 11) * 0x1p-53; };
    Row r{};
    double w = 1.0;
    const uint32_t fill = 1u + below(60u);
    const double fall = 0.01 + 0.5 * unit();
    for (uint32_t l = 0; l < kLanes; ++l)
        for (uint32_t s = 0; s < kSlots; ++s) {
            if (below(60u) >= fill / (1u + (l & 3u) * 8u) || w < 1e-6) continue;
            r.n[l][s] = 1u + below(100u);
            r.w[l][s] = w;
            w *= std::exp(-fall * unit() - 1e-3);
        }
    r.mass0 = below(2u) ? 0.0 : 50.0 * unit();
    r.count0 = r.mass0 != 0.0 ? 1u + below(1000u) : 0u;
    // A border on a token, to a few roundings, or anywhere.
    double sum = r.mass0;
    std::vector<double> sums, weights;
    for (uint32_t l = 0; l < kLanes; ++l)
        for (uint32_t s = 0; s < kSlots; ++s)
            if (r.n[l][s] != 0u) {
                sums.push_back(sum + (1u + below(r.n[l][s])) * r.w[l][s]);
                sum += r.n[l][s] * r.w[l][s];
                sums.push_back(sum);
                weights.push_back(r.w[l][s]);
            }
    if (sums.empty()) return r;
    const int ulps = static_cast<int>(below(9u)) - 4;
    switch (below(4u)) {
    case 0: r.enough = nudged(sums[below(static_cast<uint32_t>(sums.size()))], ulps); break;
    case 1: r.min_p = nudged(weights[below(static_cast<uint32_t>(weights.size()))], ulps); break;
    case 2:
        r.enough = nudged(sums[below(static_cast<uint32_t>(sums.size()))], ulps);
        r.min_p = nudged(weights[below(static_cast<uint32_t>(weights.size()))], -ulps);
        break;
    default:
        r.enough = sum * 1.2 * unit();
        r.min_p = unit() * unit();
    }
    for (uint32_t l = 0; l < kLanes; ++l)
        for (uint32_t s = 0; s < kSlots; ++s) {
            if (r.n[l][s] == 0u) continue;
            const double v = r.w[l][s] * (1.0 + 0x1p-46 * (2.0 * unit() - 1.0));
            r.rough[l] += r.n[l][s] * v;
            r.light[l] = r.light[l] || may_be_light(v, r.min_p);
        }
    return r;
}

uint32_t border_of(const Row& r) {
    uint32_t got[kLanes];
    host_wave::run([&](uint32_t lane) {
        uint32_t here = 0u;
        for (uint32_t s = 0; s < kSlots; ++s) here += r.n[lane][s];
        const double incl = r.mass0 + wave_incl64(r.rough[lane]);
        const uint32_t count = r.count0 + wave_incl(here);
        const bool by_mass = r.enough != 0.0;
        const uint64_t maybe = __ballot(here != 0u && (r.light[lane] || (by_mass && may_be_past(incl, r.enough))));
        got[lane] = wave_border(maybe, by_mass, r.enough, r.min_p, [&](uint32_t from) {
            OneValue o{0u, 0u, 0u, 0.0, 0.0};
            if (lane < kSlots) {
                o.n = r.n[from][lane];
                o.w = r.w[from][lane];
            }
            const double m = o.n * o.w;
            const double mass_before = incl - r.rough[lane];
            const uint64_t before = __builtin_bit_cast(uint64_t, mass_before);
            const uint64_t lo = from_lane(static_cast<uint32_t>(before), from);
            const uint64_t hi = from_lane(static_cast<uint32_t>(before >> 32), from);
            o.mass = __builtin_bit_cast(double, lo | hi << 32) + (wave_incl64(m) - m);
            o.before = from_lane(count - here, from) + (wave_incl(o.n) - o.n);
            return o;
        });
    });
    for (uint32_t l = 1; l < kLanes; ++l)
        if (got[l] != got[0]) throw std::runtime_error("the lanes have different borders");
    return got[0];
}

}  // namespace

// 0, or 1 with the first row that is wrong in `message`.
extern "C" int check_borders(uint64_t seed, uint32_t rows, char* message, size_t bytes) {
    std::mt19937_64 rng(seed);
    for (uint32_t i = 0; i < rows; ++i) {
        const Row r = row_of(rng);
        // The definition, the sum in more bits: what top-p keeps, what min-p does.
        long double mass = r.mass0;
        uint32_t count = r.count0, by_mass = 0xFFFFFFFFu, by_weight = 0xFFFFFFFFu;
        for (uint32_t l = 0; l < kLanes; ++l)
            for (uint32_t s = 0; s < kSlots; ++s) {
                if (r.n[l][s] != 0u && r.w[l][s] < r.min_p) by_weight = std::min(by_weight, count);
                for (uint32_t k = 0; k < r.n[l][s]; ++k, ++count, mass += r.w[l][s])
                    if (r.enough != 0.0 && !(mass < r.enough)) by_mass = std::min(by_mass, count);
            }
        const uint32_t want = std::min(std::min(by_mass, by_weight), count);
        uint32_t got;
        try {
            got = std::min(border_of(r), count);
        } catch (const std::exception& e) {
            snprintf(message, bytes, "row %u: %s", i, e.what());
            return 1;
        }
        // (A running sum is right to some roundings: a token either way. A weight is the value's own.)
        const bool ok = by_weight < by_mass ? got == want || (got < want && want - got <= 1u && by_mass <= by_weight + 1u)
                                            : got <= want + 1u && want <= got + 1u && got <= std::min(by_weight, count);
        if (!ok) {
            snprintf(message, bytes, "row %u: %u tokens kept, %u by mass, %u by weight, of %u (enough %a, min_p %a)", i, got, by_mass,
                     by_weight, count, r.enough, r.min_p);
            return 1;
        }
    }
    return 0;
}
