"""Batched serving at the ends of what its calls define. Bars as test_gpu_batch.py's."""
import numpy as np
import pytest

from hyperion_amd import synthetic as syn
from test_gpu_batch import CONFIG, Scene, check_draw, f64, say

pytestmark = pytest.mark.gpu

NO_KEYS = [
    # lens, rows, H, KVH, D, prefix, window: requests of many rows without own tokens
    ([0] * 70 + [40], [70] * 70 + [40], 8, 8, 64, 0, 0),         # the output's rows: a worker has whole tiles of none
    ([0] * 70 + [40], [70] * 70 + [40], 8, 8, 64, 20, 0),        # beside a prefix that they do not see
    ([0, 30] * 40, [21, 9] * 40, 16, 8, 256, 33, 0),
    ([90, 0, 200] * 30, [1, 50, 33] * 30, 16, 8, 256, 64, 40),
    ([0] * 40, [130] * 40, 16, 1, 512, 0, 0),                    # nothing else in the batch
    ([0, 300, 0], [256, 290, 127], 2, 2, 128, 0, 0),             # rows that fill wide tiles by themselves
    ([0, 300, 0], [256, 290, 127], 2, 2, 128, 90, 0),
]


@pytest.mark.parametrize("lens,rows,H,KVH,D,prefix,window", NO_KEYS)
def test_many_rows_of_requests_without_tokens(stream, lens, rows, H, KVH, D, prefix, window):
    """Row i of n of a request without tokens stands n - i before the end of the prefix: it sees what the prefix
    has there, or nothing."""
    say(f"no own keys: {len(lens)} requests H={H} KVH={KVH} D={D} prefix={prefix} window={window}")
    s = Scene(D + prefix, stream, lens, rows, H, KVH, D, 16, prefix, window, extra_rows=2).place()
    for _ in range(2):
        s.run()
        s.check("without own keys")


def test_many_rows_behind_tables_without_entries(stream):
    """max_blocks 0: lengths end at the tables, so no request has tokens."""
    s = Scene(5, stream, [0] * 70, [70] * 70, 8, 8, 64, 16, 20, 0)
    s.tables = s.tables[:, :0]
    s.place()
    s.lens[:] = 50
    s.d_lens.upload(s.lens, stream)
    s.lens[:] = 0
    s.run()
    s.check("no entries")


@pytest.mark.parametrize("min_p", [1.0, 1.5, 2.0, 2.0**20, np.inf])
@pytest.mark.parametrize("vocab", [5, 999, 70000])
def test_sample_min_p_of_one_and_more(stream, vocab, min_p):
    """A weight is at most 1: min_p above 1 leaves one token, min_p 1 the largest logit's; +inf logits weigh 1."""
    rng = np.random.default_rng(vocab)
    rows = 12
    x = np.round(2.0 * rng.standard_normal((rows, vocab)))
    x[:, 1::2] = np.max(x, axis=1, keepdims=True)        # many of the largest
    x[::2, 3:] = np.where(rng.random((rows // 2, vocab - 3)) < 0.3, np.inf, x[::2, 3:])
    x[::2, 4] = np.inf
    x[::2, 3] = np.inf                                   # two at least
    configs = np.zeros(rows, CONFIG)
    configs["temperature"], configs["min_p"] = 0.8, min_p
    configs["top_k"][4:8], configs["top_p"][6:10] = 2, 0.9
    uniforms = np.resize(np.array([0.999, 0.5, 0.75], np.float32), rows)
    check_draw(stream, syn.bf16_bits(x.astype(np.float32)), configs, uniforms, f"min_p {min_p}")


UNWEIGHED = [
    # rows of each request, H, KVH, D, prefix
    (1, 2, 2, 64, 0),        # few rows, straight to the output
    (3, 8, 2, 256, 0),
    (1, 16, 1, 512, 20),     # and joined
    (40, 4, 2, 128, 0),      # wide tiles, straight to the output
    (40, 4, 2, 256, 0),
    (20, 16, 1, 512, 20),
]


@pytest.mark.parametrize("rows,H,KVH,D,prefix", UNWEIGHED)
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_keys_with_a_score_of_minus_infinity_weigh_nothing(stream, rows, H, KVH, D, prefix, bad):
    """Whatever their values are: a row whose every score is -inf gives zeros, one with others is their mean."""
    say(f"scores of -inf: rows={rows} H={H} KVH={KVH} D={D} prefix={prefix} V={bad}")
    s = Scene(D + rows, stream, [50, 90, 60], [rows] * 3, H, KVH, D, 16, prefix, 0)
    low, worst = (syn.bf16_bits(np.array([v], np.float32))[0] for v in (-np.inf, bad))
    one = syn.bf16_bits(np.ones(1, np.float32))[0]
    s.q[:, :, 0] = one
    at = np.arange(50)
    own = s.tables[0, at // 16].astype(np.int64) * 16 + at % 16
    s.ck[own, :, 0], s.cv[own] = low, worst                       # request 0: every own key
    at = np.arange(3, 40)
    own = s.tables[1, at // 16].astype(np.int64) * 16 + at % 16
    s.ck[own, :, 0], s.cv[own, :, ::3] = low, worst               # request 1: some
    if prefix:
        at = s.prefix_table[np.arange(prefix) // 16].astype(np.int64) * 16 + np.arange(prefix) % 16
        s.ck[at, :, 0], s.cv[at, :, 1] = low, worst               # the prefix
    s.place()
    s.run()
    out = s.check("scores of -inf")
    assert np.all(f64(out[:rows]) == 0.0)


@pytest.mark.parametrize("lens,rows,H,KVH,D,block,prefix,window,scale,spread", [
    ([300], [1], 64, 1, 64, 16, 0, 0, None, 2.0),                          # one row of 64 heads
    ([70, 300, 9], [60, 130, 9], 16, 8, 64, 16, 250, 0, None, 2.0),
    ([70, 300, 9], [60, 130, 9], 16, 4, 128, 16, 250, 0, None, 2.0),
    ([70, 300, 9], [60, 130, 9], 4, 2, 256, 16, 250, 100, 1.0, 2.0),
    ([64, 300, 9], [60, 130, 9], 4, 2, 256, 16, 250, 0, 1.0, 8.0),         # scores far apart: maxima grow late
    ([64, 300, 9], [60, 130, 9], 16, 1, 512, 16, 250, 0, 1.0, 8.0),
    ([20] * 40, [1] * 40, 16, 1, 512, 16, 1500, 0, 1.0, 2.0),
    ([20, 700], [20, 300], 16, 1, 512, 16, 70, 0, None, 0.5),              # many keys of like weight
])
def test_many_rows_weigh_in_two_terms(stream, lens, rows, H, KVH, D, block, prefix, window, scale, spread):
    """Wide tiles round a probability by no more than tiles of few rows do (2^-16 of itself): the bound of
    Scene.compare without its term for one rounding to bf16."""
    say(f"two terms: {len(lens)} requests H={H} KVH={KVH} D={D} prefix={prefix} spread={spread}")
    s = Scene(sum(lens) + D, stream, lens, rows, H, KVH, D, block, prefix, window, scale, spread=spread).place()
    s.one_term = lambda: False
    s.run()
    s.check("two terms")
