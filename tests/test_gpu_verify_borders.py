"""Rows whose running sum or weight meets a filter's border to a rounding: what hyp_verify_batch keeps of them against the
definition and against hyp_sample_batch. Every token is a draft once, at a uniform of 0: it is accepted iff it is kept.

Bars: a running sum is some hundred fp64 roundings, here within one of the border: the kept tokens end one token off at most.
A weight is one exponential of fp64, which of two that differ by its rounding is below min_p is open to it alone: so the
value at the border is in or out, as hyp_sample_batch, with the same exponential, has it."""
import numpy as np
import pytest

import hyperion_amd as hy
import pages_ref as R
from hyperion_amd import synthetic as syn
from test_gpu_batch import dev, say
from test_gpu_verify import Verify, config

pytestmark = pytest.mark.gpu

# Temperature, top-p, min-p, (logit, tokens) ...: found by a search over temperatures.
ROWS = [
    (1.22, 0.758066356, 0, ((8.1875, 17), (7.6875, 103), (6.15625, 144))),
    (1.19, 0.998272479, 0, ((13.6875, 14), (11.4375, 110), (5.1875, 67))),
    (0.664545655, 0.999897301, 0, ((-1.7890625, 21), (-3.3125, 108), (-8.375, 66), (-11.75, 1))),
    (0.967571974, 0.977481604, 0, ((-1.4765625, 20), (-3.171875, 99), (-5.03125, 28), (-7.53125, 76))),
    (0.907848001, 0.744553864, 0, ((-1.96875, 29), (-2.90625, 40), (-4.03125, 142), (-6.8125, 40))),
    (0.991171598, 0.867865086, 0, ((-0.435546875, 13), (-1.578125, 92), (-3.25, 92), (-4.59375, 68))),
    (1.04320014, 0.973505318, 0, ((8, 14), (6.03125, 85), (2.65625, 122), (-1.359375, 33))),
    (1.33588207, 0, 0.105235413, ((-1.4296875, 11), (-4.4375, 69), (-5.78125, 34), (-11.25, 13))),
    (0.540771604, 0, 0.00694487989, ((8.75, 18), (6.0625, 120), (5.03125, 65), (0.265625, 21))),
    (0.986763, 0, 0.0245929118, ((10.6875, 20), (7.03125, 4), (5.25, 91), (1.3515625, 28))),
    (0.54212153, 0, 0.00273590116, ((0.98046875, 25), (-2.21875, 114), (-3.765625, 34), (-8.625, 7))),
    (0.759048462, 0, 0.0245929118, ((1.1875, 26), (-1.625, 64), (-5.15625, 15), (-10.5625, 67))),
    (1.40882814, 0, 0.453745902, ((-0.26953125, 28), (-1.3828125, 99), (-4.15625, 92), (-7.59375, 7))),
    (0.60723877, 0, 0.0245929118, ((13.75, 30), (11.5, 19), (8.125, 135), (6.1875, 81))),
    (0.509264112, 0, 0.000874891935, ((2.546875, 6), (-1.0390625, 71), (-4.84375, 81), (-10.3125, 32))),
    (1.45191061, 0, 0.243868649, ((1.71875, 29), (-0.330078125, 108), (-3.125, 124), (-4.03125, 99))),
    (0.550310135, 0, 0.0245929118, ((3.921875, 7), (1.8828125, 25), (-0.59765625, 7), (-2.703125, 21))),
    (0.616726875, 0, 0.0245929118, ((1.3828125, 23), (-0.90234375, 9), (-1.5546875, 25), (-5, 88))),
    (1.81276476, 0, 0.632606149, ((1.1796875, 5), (0.349609375, 81), (-0.2353515625, 1), (-3.40625, 74))),
    (0.726060987, 0, 0.00485569937, ((-0.2255859375, 16), (-4.09375, 71), (-8.625, 109), (-13.625, 53))),
]


@pytest.mark.parametrize("temperature,top_p,min_p,values", ROWS)
def test_borders_met_to_a_rounding(stream, temperature, top_p, min_p, values):
    say(f"verify: a border at T={temperature}, top_p={top_p}, min_p={min_p}")
    setting = (temperature, 0, top_p, min_p)
    x = np.concatenate([np.full(n, v, np.float32) for v, n in values] + [np.full(6, -np.inf, np.float32)])
    x = x[np.random.default_rng(x.size).permutation(x.size)]
    bits = syn.bf16_bits(x).reshape(-1)
    assert np.array_equal(syn.bf16_to_f32(bits), x)
    vocab = x.size
    order = np.argsort(-x, kind="stable")

    ids = np.zeros((vocab, 2), np.uint32)
    ids[:, 1] = np.arange(vocab)
    v = Verify(stream, [2] * vocab, np.tile(bits, (2 * vocab, 1)), None, ids.reshape(-1), config([setting] * vocab), None,
               np.zeros(2 * vocab), logprobs=False)
    v.run()
    kept = v.results()["accepted"] == 1
    count = int(kept.sum())
    assert count >= 1 and kept[order[:count]].all(), "no prefix of the order"

    # hyp_sample_batch's last token: one of the border's values is more than 2^-20 of the kept sum.
    token = dev(np.zeros(1, np.uint32), stream)
    need = hy.sample_batch_workspace_bytes(1, vocab)
    work = dev(np.zeros(need, np.uint8), stream) if need else None
    hy.sample_batch(dev(bits, stream), 1, vocab, dev(config([setting]), stream), dev(np.array([0.99999994], np.float32), stream),
                    token, None, work, stream)
    drawn = int(np.flatnonzero(order == token.to_host(stream)[0])[0]) + 1

    if min_p:
        w = np.exp((x[order].astype(np.float64) - float(x.max())) / float(np.float32(temperature)))
        least, most = (int(np.count_nonzero(w >= float(np.float32(min_p)) * s)) for s in (1 + 1e-14, 1 - 1e-14))
        assert least < most, "the row meets no border"
        assert count in (least, most), (count, least, most)
        assert count == drawn, (count, drawn)
    else:
        want = int(np.count_nonzero(R.kept(x, *(float(np.float32(s)) for s in setting))[0]))
        assert abs(count - want) <= 1, (count, want)
        assert abs(count - drawn) <= 1, (count, drawn)
