"""GPU parity of hyp_verify_batch against pages_ref.py's 64-bit reference.

Bars: accepted, rejected and tokens equal. A logprob is one rounding to fp32 of an fp64 value: 2^-24 of itself, plus
1e-12 for the fp64 sums (some hundred roundings each: weights are counted by value, and 2^23 tokens are 128 chunks).
"""
import numpy as np
import pytest

import batch_ref as B
import hyperion_amd as hy
import pages_ref as R
from hyperion_amd import synthetic as syn
from test_gpu_batch import CONFIG, dev, say

pytestmark = pytest.mark.gpu

GREEDY = (0.0, 0, 0.0, 0.0)
PLAIN = (1.0, 0, 0.0, 0.0)


def config(settings):
    c = np.zeros(len(settings), CONFIG)
    for i, s in enumerate(settings):
        c["temperature"][i], c["top_k"][i], c["top_p"][i], c["min_p"][i] = s
    return c


def setting(c):
    return float(c["temperature"]), int(c["top_k"]), float(c["top_p"]), float(c["min_p"])


class Verify:
    """The arrays of one call on the device."""

    def __init__(self, stream, counts, logits, draft, ids, configs, draft_configs, uniforms, extra=0, logprobs=True):
        rows, vocab = logits.shape
        n = len(counts)
        self.stream, self.counts, self.rows, self.vocab, self.n = stream, counts, rows, vocab, n
        self.start = np.concatenate(([0], np.cumsum(counts))).astype(np.uint32)
        assert self.start[-1] + extra == rows
        self.host = dict(logits=logits, draft=draft, ids=np.asarray(ids, np.uint32), configs=configs, draft_configs=draft_configs,
                         uniforms=np.asarray(uniforms, np.float32), start=self.start)
        empty = lambda a: a if a.size else np.zeros(1, a.dtype)  # noqa: E731
        self.d = {k: None if v is None else dev(empty(v), stream) for k, v in self.host.items()}
        self.out = {k: dev(np.full(n, 77, np.uint32), stream) for k in ("accepted", "rejected", "tokens")}
        self.logprobs = dev(np.full(max(rows, 1), 77.0, np.float32), stream) if logprobs else None
        need = hy.verify_batch_workspace_bytes(rows, vocab, n, draft is not None)
        self.work = dev(np.full(max(need, 16), 0xFF, np.uint8), stream)

    def run(self, stream=None):
        d, o = self.d, self.out
        hy.verify_batch(d["logits"], d["draft"], self.rows, self.vocab, d["start"], self.n, d["ids"], d["configs"],
                        d["draft_configs"], d["uniforms"], o["accepted"], o["rejected"], o["tokens"], self.logprobs, self.work,
                        stream or self.stream)

    def results(self):
        got = {k: v.to_host(self.stream) for k, v in self.out.items()}
        got["logprobs"] = None if self.logprobs is None else self.logprobs.to_host(self.stream)
        return got

    def check(self, what):
        h, got = self.host, self.results()
        values = syn.bf16_to_f32(h["logits"]).reshape(h["logits"].shape)
        guess = None if h["draft"] is None else syn.bf16_to_f32(h["draft"]).reshape(h["draft"].shape)
        seen = np.zeros(self.rows, bool)
        for r, n in enumerate(self.counts):
            if n == 0:
                assert (got["accepted"][r], got["rejected"][r], got["tokens"][r]) == (0, 0, 77), (what, r)
                continue
            at = slice(int(self.start[r]), int(self.start[r]) + n)
            mine = setting(h["configs"][r])
            theirs = mine if h["draft_configs"] is None else setting(h["draft_configs"][r])
            a, token, logs = R.verify(values[at], None if guess is None else guess[at], h["ids"][at], h["uniforms"][at], mine,
                                      theirs)
            assert got["accepted"][r] == a and got["rejected"][r] == n - 1 - a, (what, r, mine, theirs, got["accepted"][r], a, n)
            assert got["tokens"][r] == token, (what, r, mine, theirs, a, n, got["tokens"][r], token)
            if got["logprobs"] is not None:
                lp = got["logprobs"][at][:a + 1].astype(np.float64)
                ref = np.array(logs)
                sure = np.where(np.isfinite(ref), ref, 0.0)
                ok = (lp == ref) | (np.abs(np.where(np.isfinite(ref), lp, 1.0) - sure) <= 2.0**-24 * np.abs(sure) + 1e-12)
                assert np.all(ok), (what, r, lp, ref)
                seen[at.start:at.start + a + 1] = True
        if got["logprobs"] is not None:
            assert np.all(got["logprobs"][:self.rows][~seen] == 77.0), what
        return got


def rows_of(kind, rng, rows, vocab):
    """bf16 logits of a kind, and a drafting model's near them."""
    x = 2.5 * rng.standard_normal((rows, vocab))
    x[:, rng.integers(0, vocab, 12)] += 6.0
    y = x + 0.5 * rng.standard_normal((rows, vocab))
    at = rng.random((rows, vocab))
    if kind == "ties":
        x, y = np.round(x), np.round(y)
    elif kind == "same":
        y = x.copy()
    elif kind == "inf":
        x[at < 0.01], y[at < 0.03] = np.inf, np.inf
        x[:, 0] = y[:, 0] = np.inf
    elif kind == "nan":
        x[at < 0.1], y[at > 0.9] = np.nan, np.nan
    elif kind == "masked":
        x[at < 0.6], y[at < 0.5] = -np.inf, -np.inf
    elif kind == "lowest":
        x[at < 0.6], y[at < 0.5] = -3.3895314e38, -3.3895314e38
    elif kind == "deep":
        x[at < 0.7], y[at < 0.7] = -300.0 - 200.0 * at[at < 0.7], -290.0 - 210.0 * at[at < 0.7]
    elif kind == "large":
        x, y = 100.0 * x, 100.0 * y
    elif kind == "tiny":
        x, y = x * 2.0**-30, y * 2.0**-28
    elif kind == "none":
        x[::2] = -np.inf
        y[1::3] = -np.inf
    elif kind == "flat":
        x[:], y[:] = 1.0, 1.0
    with np.errstate(over="ignore"):
        return syn.bf16_bits(x.astype(np.float32)).reshape(rows, vocab), syn.bf16_bits(y.astype(np.float32)).reshape(rows, vocab)


def drafts(rng, guess, start):
    """Ids that the drafting model makes likely, some of anything."""
    rows, vocab = guess.shape
    y = syn.bf16_to_f32(guess).reshape(rows, vocab).astype(np.float64)
    y = np.where(np.isnan(y), -np.inf, y)
    gumbel = -np.log(-np.log(rng.random((rows, vocab)) * 0.999999 + 1e-7))
    ids = np.zeros(rows, np.uint32)
    with np.errstate(invalid="ignore"):
        ids[1:] = np.argmax(y / 0.7 + gumbel, -1)[:-1]
    any_at = rng.random(rows) < 0.1
    ids[any_at] = rng.integers(0, vocab, int(any_at.sum()))
    return ids


def settings(rng, n, vocab):
    return config([(rng.choice([0.0, 0.4, 0.8, 1.0, 1.5, -1.0, np.nan], p=[.12, .2, .3, .2, .1, .04, .04]),
                    rng.choice([0, 0, 1, 2, 5, 60, vocab, vocab + 9, max(1, 3 * vocab // 4)]),
                    rng.choice([0.0, 0.5, 0.9, 0.99, 1.0, 0.01]), rng.choice([0.0, 0.0, 0.05, 0.3, 1.0, 1.5, 1e-38]))
                   for _ in range(n)])


def scene(stream, seed, kind, counts, vocab, drafter, extra=0, own_configs=False, **kw):
    rng = np.random.default_rng(seed)
    rows = sum(counts) + extra
    x, y = rows_of(kind, rng, rows, vocab)
    ids = drafts(rng, y, None)
    u = rng.random(rows).astype(np.float32)
    return Verify(stream, counts, x, y if drafter else None, ids, settings(rng, len(counts), vocab),
                  settings(rng, len(counts), vocab) if own_configs else None, u, extra, **kw)


KINDS = ["usual", "ties", "same", "inf", "nan", "masked", "lowest", "deep", "large", "tiny", "none", "flat"]


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("kind", KINDS)
def test_kinds_of_rows(stream, kind, drafter):
    say(f"verify: rows of kind {kind}, drafter={drafter}")
    rng = np.random.default_rng(len(kind))
    counts = [1, 4, 0, 6, 2, 3, 5, 1, 4, 4, 3, 2, 6, 5] * 3
    for vocab in (1, 6, 999, 9001):
        v = scene(stream, rng.integers(1 << 30), kind, counts, vocab, drafter, extra=5, own_configs=vocab != 999)
        v.run()
        v.check((kind, vocab))


SHAPES = [
    # counts, vocab, extra rows
    ([1], 1, 0),
    ([5], 262144, 0),
    ([2], 2048, 0),          # a tile of the sums exactly
    ([3, 3], 2049, 0),
    ([3, 3], 2047, 1),
    ([0, 0, 4, 0], 50001, 3),
    ([100], 999, 0),
    ([600], 300, 2),         # more drafts than threads of a workgroup
    ([3] * 400, 640, 7),     # rows enough for one workgroup each
    ([2, 7] * 40, 40000, 0),
    ([4] * 130, 70001, 0),   # chunks of more than 32768 tokens
    ([1] * 4096, 64, 0),     # the most requests
    ([4, 0] * 2048, 33, 0),
]


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("counts,vocab,extra", SHAPES)
def test_shapes(stream, counts, vocab, extra, drafter):
    say(f"verify: {len(counts)} requests, {sum(counts)} rows of {vocab}, drafter={drafter}")
    v = scene(stream, vocab + len(counts), "usual", counts, vocab, drafter, extra)
    v.run()
    v.check("shape")


def test_every_draft_accepted_or_none(stream):
    say("verify: uniforms at their ends")
    for u in (0.0, 0.99999994, 1.0, 2.0, -1.0, np.nan, np.inf):
        v = scene(stream, 11, "usual", [4, 5, 1, 7] * 4, 3000, True)
        v.host["uniforms"][:] = u
        v.d["uniforms"].upload(v.host["uniforms"], stream)
        v.run()
        got = v.check(("uniform", u))
    v = scene(stream, 12, "same", [4, 5, 1, 7] * 4, 3000, True)
    v.host["uniforms"][:] = 0.9999
    v.d["uniforms"].upload(v.host["uniforms"], stream)
    for k in ("temperature", "top_k", "top_p", "min_p"):
        v.host["configs"][k] = 1.0 if k == "temperature" else 0
    v.d["configs"].upload(v.host["configs"], stream)
    v.run()
    got = v.check("the same model")
    assert not got["rejected"].any()


@pytest.mark.parametrize("drafter", [True, False])
def test_drafts_outside_the_vocabulary(stream, drafter):
    say(f"verify: ids of vocab and more, drafter={drafter}")
    v = scene(stream, 13, "usual", [6, 5, 4], 700, drafter)
    v.host["ids"][[0, 2, 6, 8]] = [0xFFFFFFFF, 700, 0x80000000, 0xFFFFFFFF]
    v.host["uniforms"][:] = 0.0
    for name in ("ids", "uniforms"):
        v.d[name].upload(v.host[name], stream)
    v.run()
    got = v.check("outside")
    assert got["accepted"][0] <= 1 and got["accepted"][1] <= 1


def test_equal_to_the_border(stream):
    """p(x) is 1/2 to the bit: a uniform of 1/2 rejects, the next one below accepts; a draw at the border takes the next."""
    say("verify: borders")
    x = syn.bf16_bits(np.tile(np.array([0.0, -np.inf, 0.0], np.float32), (6, 1))).reshape(6, 3)
    below = np.nextafter(np.float32(0.5), np.float32(0))
    v = Verify(stream, [2, 2, 1, 1], x, None, [9, 2, 9, 2, 9, 9], config([PLAIN] * 4), None,
               [0.5, 0.0, below, 0.5, below, 0.5])
    v.run()
    got = v.check("borders")
    assert got["accepted"].tolist() == [0, 1, 0, 0] and got["tokens"].tolist() == [0, 2, 0, 2]


@pytest.mark.parametrize("top_k", [3, 40, 600, 899, 900])
def test_cut_among_values_far_below(stream, top_k):
    """Tokens whose weights are far below the others' are still in or out by the filters: at a uniform of 0 a draft stands if p
    is above 0 at all."""
    say(f"verify: cut far below, top_k={top_k}")
    rng = np.random.default_rng(top_k)
    vocab = 900
    x = np.concatenate((rng.standard_normal(100), -300.0 - np.arange(800) // 7))
    order = rng.permutation(vocab)
    bits = syn.bf16_bits(np.tile(x[order].astype(np.float32), (40, 1))).reshape(40, vocab)
    v = Verify(stream, [2] * 20, bits, None, rng.integers(0, vocab, 40), config([(1.0, top_k, 0.0, 0.0)] * 20), None,
               np.zeros(40))
    v.run()
    v.check(("cut", top_k))


@pytest.mark.parametrize("vocab", [700, 20001])
def test_filters_end_anywhere_in_the_order(stream, vocab):
    """Logits on both sides of 2^7 and of 0, at temperatures under which all of them weigh something: the filters end among the
    large, the small, the negative or the far negative ones."""
    say(f"verify: a wide order of {vocab}")
    rng = np.random.default_rng(vocab)
    n = 96
    x = rng.uniform(-400.0, 300.0, (2 * n, vocab))
    x[:, ::9] = 1e-9 * x[:, ::9]
    x[::3] = np.where(x[::3] > 0.0, x[::3] * 1e-3, x[::3])     # (and some whose largest is small)
    bits = syn.bf16_bits(x.astype(np.float32)).reshape(x.shape)
    some = config([(rng.choice([20.0, 100.0, 400.0, 3000.0]), rng.choice([0, 0, vocab // 3, vocab - vocab // 9]),
                    rng.choice([0.0, 0.2, 0.6, 0.97, 0.99999]), rng.choice([0.0, 0.0, 0.9, 0.5, 0.02, 1e-5])) for _ in range(n)])
    v = Verify(stream, [2] * n, bits, None, rng.integers(0, vocab, 2 * n), some, None,
               np.where(rng.random(2 * n) < 0.3, 0.0, rng.random(2 * n)))
    v.run()
    v.check("wide")
    v = Verify(stream, [2] * n, bits, np.roll(bits, 1, 0), rng.integers(0, vocab, 2 * n), some, some[::-1].copy(), rng.random(2 * n))
    v.run()
    v.check("wide, drafted")


LOWEST = -3.3895314e38


@pytest.mark.parametrize("fill", [-127.5, -128.0, -129.0, -400.0, -2000.0, LOWEST, -np.inf, 0.0, 1e-9, np.inf, np.nan])
@pytest.mark.parametrize("allowed", [1, 5, 300])
def test_masked_tokens(stream, allowed, fill):
    """Masks of any value under any temperature, with fewer tokens left than top-k keeps; drafts that are masked among them."""
    say(f"verify: {allowed} tokens left of a mask of {fill}")
    rng = np.random.default_rng(allowed)
    vocab, n = 3000, 60
    x = 4.0 * rng.standard_normal((3 * n, vocab))
    at = np.argsort(rng.random((n, vocab)), -1)[:, allowed:].repeat(3, 0)
    y = x + rng.standard_normal(x.shape)
    np.put_along_axis(x, at, fill, -1)
    np.put_along_axis(y[::2], at[::2], fill, -1)   # (of some rows the target alone is masked)
    bits = [syn.bf16_bits(a.astype(np.float32)).reshape(a.shape) for a in (x, y)]
    some = config([(rng.choice([0.0, 0.3, 1.0, 1.9, 2.5, 60.0, 1e30]), rng.choice([0, 2, 64, 2000]), rng.choice([0.0, 0.95]),
                    rng.choice([0.0, 0.0, 0.02])) for _ in range(n)])
    u = np.where(rng.random(3 * n) < 0.2, 0.0, rng.random(3 * n))
    for draft in (bits[1], None):
        v = Verify(stream, [3] * n, bits[0], draft, drafts(rng, bits[1], None), some, None, u)
        v.run()
        v.check((allowed, fill, draft is None))


def test_largest_vocabulary(stream):
    say("verify: 2^23 tokens")
    vocab, keep = 1 << 23, 6000001
    flat = np.full((3, vocab), 0x3F80, np.uint16)
    v = Verify(stream, [3], flat, None, [0, keep - 1, keep], config([(1.0, keep, 0.0, 0.0)]), None, [0.0, 0.0, 0.7])
    v.run()
    got = v.check("flat")
    assert (got["accepted"][0], got["rejected"][0]) == (1, 1)
    v = scene(stream, 5, "usual", [2], vocab - 1, True)
    v.run()
    v.check("usual")


def test_rows_past_2_to_the_32_bytes(stream):
    """The last rows of 300 of 2^23 tokens, 5 GB: the same as those alone."""
    say("verify: rows far behind the first")
    vocab, rows, skip = 1 << 23, 300, 297
    rng = np.random.default_rng(8)
    x = syn.bf16_bits((2.5 * rng.standard_normal((3, vocab), np.float32))).reshape(3, vocab)
    ids = np.concatenate(([0], np.argmax(syn.bf16_to_f32(x[:2]).reshape(2, vocab), -1)))
    u, c = [0.0, 0.0, 0.6], config([(0.9, 0, 0.99, 0.0)])
    alone = Verify(stream, [3], x, None, ids, c, None, u)
    alone.run()
    want = alone.check("alone")
    logits = hy.DeviceArray((rows, vocab), np.uint16)
    hy.call("hyp_memcpy_htod", hy.ctypes.c_void_p(logits.ptr.value + skip * vocab * 2), x.ctypes.data_as(hy.ctypes.c_void_p),
            x.nbytes, stream.handle)
    pad = lambda a, t: dev(np.concatenate((np.zeros(skip, t), np.asarray(a, t))), stream)  # noqa: E731
    out = [dev(np.zeros(1, np.uint32), stream) for _ in range(3)]
    logprobs = dev(np.full(rows, 77.0, np.float32), stream)
    work = hy.DeviceArray((hy.verify_batch_workspace_bytes(rows, vocab, 1, False),), np.uint8)
    hy.verify_batch(logits, None, rows, vocab, dev(np.array([skip, rows], np.uint32), stream), 1, pad(ids, np.uint32), alone.d["configs"],
                    None, pad(u, np.float32), *out, logprobs, work, stream)
    got = [o.to_host(stream)[0] for o in out]
    assert got == [want[k][0] for k in ("accepted", "rejected", "tokens")]
    got = logprobs.to_host(stream)
    assert np.array_equal(got[skip:], want["logprobs"]) and np.all(got[:skip] == 77.0)


@pytest.mark.parametrize("vocab", [70, 5000, 262144])
def test_without_drafts_every_token_can_be_drawn(stream, vocab):
    """Requests of one row: the uniform's place in the running sum along the index."""
    say(f"verify: draws, vocab={vocab}")
    rng = np.random.default_rng(vocab)
    rows = 12
    x = syn.bf16_bits(rng.standard_normal((rows, vocab)).astype(np.float32)).reshape(rows, vocab)
    u = np.concatenate(([0.0, 0.99999994], rng.random(rows - 2)))
    v = Verify(stream, [1] * rows, x, None, np.zeros(rows), config([PLAIN] * rows), None, u)
    v.run()
    got = v.check("draws")
    assert got["tokens"][0] == 0 and got["tokens"][1] >= vocab - 2 - vocab // 1000
    v = Verify(stream, [1] * rows, x, None, np.zeros(rows), config([GREEDY] * rows), None, u, logprobs=False)
    v.run()
    got = v.check("greedy")
    values = syn.bf16_to_f32(x).reshape(x.shape)
    assert np.array_equal(got["tokens"], np.argmax(values, -1))
    assert [B.sample(r, *GREEDY, 0.5)[0] for r in values] == got["tokens"].tolist()


def test_unaligned_logits(stream):
    """Rows at odd addresses: logits are 2-byte aligned only."""
    say("verify: odd addresses")
    v = scene(stream, 31, "usual", [3, 4, 2], 4099, True)
    for name in ("logits", "draft"):
        flat = v.host[name].reshape(-1)
        held = dev(np.concatenate((np.zeros(1, np.uint16), flat)), stream)
        view = hy.DeviceArray.__new__(hy.DeviceArray)
        view.shape, view.dtype, view.nbytes = flat.shape, flat.dtype, flat.nbytes
        view._p = hy.ctypes.c_void_p(held.ptr.value + 2)
        view.close = lambda: None
        v.d[name], v.d[name + "_held"] = view, held
    v.run()
    v.check("odd addresses")


def test_row_starts_past_the_rows(stream):
    """Starts are cut off at the rows there are; what they then hold is the same as with true ones."""
    say("verify: row starts past the rows")
    v = scene(stream, 32, "usual", [3, 4, 2], 800, True)
    v.d["start"].upload(np.array([0, 3, 7, 5000], np.uint32), stream)
    v.run()
    v.check("past the rows")


def test_the_same_in_any_batch(stream):
    """A request's results do not depend on the batch that it is in, nor on the run."""
    say("verify: alone and in a batch")
    v = scene(stream, 41, "ties", [5, 3, 6, 1, 4, 4] * 12, 20011, True)
    v.run()
    first = v.check("batch")
    v.run()
    again = v.results()
    for k in first:
        assert np.array_equal(first[k], again[k])
    h = v.host
    for r in (0, 7, 38, 71):
        a, b = int(v.start[r]), int(v.start[r + 1])
        one = Verify(stream, [b - a], h["logits"][a:b], h["draft"][a:b], h["ids"][a:b], h["configs"][r:r + 1], None,
                     h["uniforms"][a:b])
        one.run()
        got = one.results()
        for k in ("accepted", "rejected", "tokens"):
            assert got[k][0] == first[k][r]
        n = int(got["accepted"][0]) + 1
        assert np.array_equal(got["logprobs"][:n], first["logprobs"][a:a + n])


@pytest.mark.parametrize("drafter", [True, False])
def test_replays_of_a_graph(stream, drafter):
    """Recorded once; each replay takes what is in the arrays then."""
    say(f"verify: graph, drafter={drafter}")
    counts = [4, 2, 0, 5, 1, 6]
    v = scene(stream, 51, "usual", counts, 30011, drafter, extra=3)
    with hy.Graph.capture(stream) as g:
        v.run()
    for seed in range(4):
        rng = np.random.default_rng(seed)
        counts = rng.permutation(counts).tolist()
        w = scene(stream, 60 + seed, "usual", counts, 30011, drafter, extra=3)
        for k in ("logits", "draft", "ids", "configs", "uniforms", "start"):
            if v.d[k] is not None:
                v.host[k] = w.host[k]
                v.d[k].upload(w.host[k], stream)
        v.counts, v.start = counts, w.start
        v.logprobs.upload(np.full(v.rows, 77.0, np.float32), stream)
        for o in v.out.values():
            o.upload(np.full(v.n, 77, np.uint32), stream)
        g.launch(stream)
        w.run()   # eager work of another call between the replays
        got = v.check(("replay", seed))
        eager = w.check(("eager", seed))
        assert all(np.array_equal(got[k], eager[k]) for k in got)
    g.close()


def test_two_streams(stream):
    """Calls that overlap, each with a workspace of its own."""
    say("verify: two streams")
    other = hy.Stream()
    a, b = (scene(stream, 70 + i, "usual", [5, 4, 6] * 8, 60001, True) for i in range(2))
    for _ in range(3):
        a.run()
        b.run(other)
    stream.synchronize()
    other.synchronize()
    a.check("first")
    b.check("second")
    other.close()
