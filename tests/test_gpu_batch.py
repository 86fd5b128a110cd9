"""GPU parity of batched serving (hyp_batch_*) against batch_ref.py's 64-bit references.

Bars: whole numbers (tables, slots, positions, tokens) equal. A bf16 output is one rounding of an
fp32 value, off by at most 2^-8 of itself, plus the fp32 arithmetic's own error, written per test.
"""
import ctypes
import sys

import numpy as np
import pytest

import batch_ref as R
import hyperion_amd as hy
from hyperion_amd import synthetic as syn

pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def dev(a, stream):
    return hy.DeviceArray.from_host(np.ascontiguousarray(a), stream)


def u32(*values):
    return np.array(values, np.uint32)


def fill_cache(cache, ck, cv, stream):
    for ptr, host in zip(cache.buffers(), (ck, cv)):
        hy.call("hyp_memcpy_htod", ptr, host.ctypes.data_as(ctypes.c_void_p), host.nbytes, stream.handle)
    stream.synchronize()


def read_cache(cache, shape, stream):
    out = []
    for ptr in cache.buffers():
        a = np.empty(shape, np.uint16)
        hy.call("hyp_memcpy_dtoh", a.ctypes.data_as(ctypes.c_void_p), ptr, a.nbytes, stream.handle)
        out.append(a)
    stream.synchronize()
    return out


# ---- plan ---------------------------------------------------------------------------------

class Plan:
    """The arrays of one plan on the device."""

    def __init__(self, lens, new, tables, free, taken, block, max_rows, prefix, stream, in_place=False):
        n = len(lens)
        self.stream, self.in_place = stream, in_place
        self.lens = dev(lens, stream) if n else hy.DeviceArray((0,), np.uint32)
        self.new = dev(new, stream) if n else hy.DeviceArray((0,), np.uint32)
        self.free, self.taken = dev(free, stream), dev(u32(taken), stream)
        self.tables = dev(tables, stream)
        self.lens_out = self.lens if in_place else dev(np.full(max(n, 0), 77, np.uint32), stream)
        self.taken_out = self.taken if in_place else dev(u32(77), stream)
        self.served = dev(u32(77), stream)
        self.row_start = dev(np.full(n + 1, 77, np.uint32), stream)
        self.slots, self.positions = (dev(np.full(max_rows, 77, np.uint32), stream) for _ in range(2))
        prefix_table = dev(np.zeros(R.blocks(prefix, block), np.uint32), stream) if prefix else None
        self.batch = hy.Batch(block, free.size, self.tables, self.lens_out, self.row_start, self.slots, self.positions,
                              prefix, prefix_table)

    def run(self):
        self.batch.plan(self.lens, self.new, self.free, self.taken, self.taken_out, self.served, self.stream)

    def results(self):
        s = self.stream
        return (self.tables.to_host(s), self.free.to_host(s), int(self.taken_out.to_host(s)[0]),
                int(self.served.to_host(s)[0]), self.lens_out.to_host(s), self.row_start.to_host(s),
                self.slots.to_host(s), self.positions.to_host(s))


def check_plan(got, ref):
    top = ref[2]
    assert got[2] == top and got[3] == ref[3], (got[2:4], ref[2:4])
    assert np.array_equal(got[1][top:], ref[1][top:])
    for i in (0, 4, 5, 6, 7):
        assert np.array_equal(got[i], ref[i]), i


def plan_case(seed, n, block, hi, new_hi, done, spare=5, extra=3, short_rows=0):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, hi + 1, n).astype(np.uint32)
    new = rng.integers(0 if new_hi > 1 else 1, new_hi + 1, n).astype(np.uint32)
    ended = rng.random(n) < done
    counts = [R.blocks(int(v), block) for v in lens]
    grown = [R.blocks(int(a) + int(b), block) for a, b in zip(lens, new)]
    num = max(1, sum(counts) + max(0, sum(g - c for g, c in zip(grown, counts)) + spare))
    order = rng.permutation(num).astype(np.uint32)
    tables = np.full((n, max(grown, default=0) + extra), R.NONE, np.uint32)
    at = 0
    for r, c in enumerate(counts):
        tables[r, :c] = order[at:at + c]
        at += c
    free = np.concatenate((np.full(at, 12345, np.uint32), order[at:]))
    rows = int(new.sum())
    new[ended] = R.DONE
    return lens, new, tables, free, at, block, max(1, rows - short_rows), 0


PLANS = [
    # n, block, hi, new_hi, done, spare, extra, short_rows, prefix
    (1, 16, 0, 1, 0.0, 5, 3, 0, 0),          # one new request
    (1, 1, 40, 3, 0.0, 5, 3, 0, 7),          # a block a token
    (64, 16, 4000, 1, 0.1, 5, 3, 0, 1000),   # a decode step
    (64, 8, 100, 1, 1.0, 5, 3, 0, 0),        # all done
    (65, 16, 300, 40, 0.3, -60, 3, 0, 5),    # too few blocks
    (65, 16, 300, 40, 0.0, 5, -2, 0, 0),     # a row of tables too short
    (65, 16, 300, 40, 0.2, 5, 3, 500, 0),    # too few rows
    (1025, 64, 900, 1, 0.05, 5, 3, 0, 0),    # two requests a thread
    (4096, 16, 60, 9, 0.1, 5, 3, 0, 0),      # the most requests, rows in a second launch
    (300, 128, 500, 700, 0.1, 5, 3, 0, 33),  # a large admission, rows in a second launch
    (7, 65536, 3000, 2000, 0.0, 5, 3, 0, 0),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,block,hi,new_hi,done,spare,extra,short_rows,prefix", PLANS)
def test_plan(stream, n, block, hi, new_hi, done, spare, extra, short_rows, prefix, in_place):
    say(f"plan n={n} block={block} hi={hi} new_hi={new_hi} done={done} in_place={in_place}")
    case = plan_case(n * 31 + block, n, block, hi, new_hi, done, spare, extra, short_rows)[:-1] + (prefix,)
    p = Plan(*case, stream, in_place=in_place)
    p.run()
    check_plan(p.results(), R.plan(*case))
    if not in_place:
        p.run()   # what was read has not changed
        check_plan(p.results(), R.plan(*case))


def test_plan_without_requests(stream):
    p = Plan(u32(), u32(), np.zeros((0, 4), np.uint32), u32(1, 0), 1, 16, 5, 0, stream)
    p.run()
    _, _, top, served, _, start, slots, pos = p.results()
    assert (top, served, start.tolist()) == (1, 0, [0])
    assert slots.tolist() == [R.NONE] * 5 and pos.tolist() == [0] * 5


def test_plan_at_the_last_position(stream):
    """Positions end below 2^24: the request that would pass it, and those behind it, wait."""
    block, prefix = 65536, 2**24 - 100
    for new, served in ((100, 3), (101, 1)):
        case = (u32(0, 0, 0), u32(1, new, 1), np.full((3, 1), R.NONE, np.uint32), u32(0, 1, 2), 0, block, 300, prefix)
        p = Plan(*case, stream)
        p.run()
        got = p.results()
        assert got[3] == served
        check_plan(got, R.plan(*case))


def test_plan_holds_its_bounds_on_damaged_state(stream):
    """A taken past the stack, lengths past their tables, ids outside the pool: nothing is written
    outside the arrays (guards around them), and such blocks have no slots."""
    n, block, max_blocks, num, rows = 3, 16, 2, 4, 40
    guard = 64

    def guarded(a):
        return dev(np.concatenate((np.full(guard, 0xABABABAB, np.uint32), np.asarray(a, np.uint32).ravel(),
                                   np.full(guard, 0xABABABAB, np.uint32))), stream)

    class At:
        def __init__(self, array, shape):
            self.array, self.shape = array, shape
            self.ptr = ctypes.c_void_p(array.ptr.value + 4 * guard)

    arrays = {k: (guarded(v), s) for k, (v, s) in dict(
        tables=([9, 9, 1, 9, 9, 9], (n, max_blocks)), lens=([0] * n, (n,)), row_start=([0] * (n + 1), (n + 1,)),
        slots=([0] * rows, (rows,)), positions=([0] * rows, (rows,)), free=([9, 0, 2, 3], (num,)), taken=([99], (1,)),
        out=([0], (1,)), served=([0], (1,)), have=([4000000000, 3, 17], (n,)),
        new=([R.DONE, 1, 4000000000], (n,))).items()}
    v = {k: At(a, s) for k, (a, s) in arrays.items()}
    b = hy.Batch(block, num, v["tables"], v["lens"], v["row_start"], v["slots"], v["positions"])
    b.plan(v["have"], v["new"], v["free"], v["taken"], v["out"], v["served"], stream)
    for k, (a, s) in arrays.items():
        host = a.to_host(stream)
        assert np.all(host[:guard] == 0xABABABAB) and np.all(host[-guard:] == 0xABABABAB), k
    got = {k: a.to_host(stream)[guard:-guard] for k, (a, s) in arrays.items()}
    assert got["served"][0] == 2                                # the last one asks for too much
    assert got["lens"].tolist() == [0, 4, 17] and got["row_start"].tolist() == [0, 0, 1, 1]
    assert got["out"][0] == 4 - 2                               # two entries came back
    assert got["slots"][0] == 1 * block + 3 and np.all(got["slots"][1:] == R.NONE)


def test_plan_steps_in_a_graph(stream):
    """A step recorded in place and replayed: each replay goes on from the last one's state."""
    lens, new, tables, free, taken, block, _, _ = plan_case(5, 40, 8, 50, 1, 0.0, spare=60, extra=12)
    case = [lens, new, tables, free, taken, block, 40, 0]
    p = Plan(*case, stream, in_place=True)
    other = hy.Stream()
    with hy.Graph.capture(other) as g:
        p.batch.plan(p.lens, p.new, p.free, p.taken, p.taken_out, p.served, other)
    for step in range(12):
        new = new.copy()
        if step in (4, 8):
            new[step::9] = R.DONE
        if step in (5, 9):
            new[:] = 1
        p.new.upload(new, stream)
        g.launch(other)
        other.synchronize()
        case[1] = new
        ref = R.plan(*case)
        check_plan(p.results(), ref)
        case[0], case[2], case[3], case[4] = ref[4], ref[0], p.free.to_host(stream), ref[2]
    g.close()
    other.close()


# ---- prepare --------------------------------------------------------------------------------

PREPARES = [
    # rows, H, KVH, D, rotated, base, own V, max_rows beyond the rows
    (1, 16, 8, 256, 256, 1e4, True, 0),
    (48, 16, 8, 256, 256, 1e4, True, 0),
    (33, 16, 1, 512, 128, 1e6, False, 5),
    (700, 16, 1, 512, 128, 1e6, True, 9),
    (5, 12, 12, 64, 64, 1e4, True, 1),
    (2100, 4, 2, 64, 16, 1e4, False, 0),
    (65, 32, 8, 128, 128, 5e5, True, 0),
    (3, 5, 1, 128, 0, 1e4, True, 0),         # nothing rotated; one pass is not filled
]


@pytest.mark.parametrize("rows,H,KVH,D,rotated,base,own_v,extra", PREPARES)
def test_prepare(stream, rows, H, KVH, D, rotated, base, own_v, extra):
    say(f"prepare rows={rows} H={H} KVH={KVH} D={D} rotated={rotated} own_v={own_v}")
    rng = np.random.default_rng(rows + D)
    bits = lambda *shape: syn.bf16_bits(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    block, max_rows = 16, rows + extra
    num = R.blocks(rows, block) + 2
    q, k, v = bits(max_rows, H, D), bits(max_rows, KVH, D), bits(max_rows, KVH, D)
    qn, kn = bits(D), bits(D)
    slots = rng.permutation(num * block)[:max_rows].astype(np.uint32)
    slots[1::7] = R.NONE
    if rows > 2:
        slots[2] = num * block + 5                           # outside the cache
    positions = rng.integers(0, 262144, max_rows).astype(np.uint32)
    positions[0] = 2**24 - 1
    cache = hy.KvCache(num * block, KVH, D)
    ck, cv = bits(num * block, KVH, D), bits(num * block, KVH, D)
    fill_cache(cache, ck, cv, stream)
    b = hy.Batch(block, num, dev(np.zeros((2, 1), np.uint32), stream), dev(u32(0, 0), stream),
                 dev(u32(0, 0, rows), stream), dev(slots, stream), dev(positions, stream))
    out = dev(np.full((max_rows, H, D), 0x7FC0, np.uint16), stream)
    qd = dev(q, stream)
    args = (dev(k, stream), dev(v, stream) if own_v else None, H, cache, dev(qn, stream), dev(kn, stream), 1e-6, rotated,
            base)
    b.prepare(qd, *args, out, stream)
    f = lambda a: syn.bf16_to_f32(a).astype(np.float64)  # noqa: E731

    def near(got, normed, what):
        """One rounding, 2^-8; below it the fp32 norm and rotation: some 30 roundings of either
        value of a pair (the row's sum of squares: 8 in a lane and 6 between lanes, halved by the root)."""
        ref = R.rope(normed, positions[:rows], rotated, base) if what != "v" else normed
        pair = np.abs(normed) + np.abs(np.roll(normed, D // 2, -1))
        err = np.abs(f(got) - ref)
        bound = 2.0**-8 * np.abs(ref) + 64 * 2.0**-24 * pair
        say(f"  {what}: worst {np.max(err / np.maximum(bound, 1e-30)):.3f} of the bound")
        assert np.all(err <= bound), what

    got = out.to_host(stream)
    near(got[:rows], R.rms(f(q[:rows]), f(qn)), "q")
    assert np.all(got[rows:] == 0x7FC0)                      # rows behind the last are left as they were
    gk, gv = read_cache(cache, ck.shape, stream)
    live = [t for t in range(rows) if slots[t] < num * block]
    at = slots[live].astype(np.int64)
    fk, fv = np.empty((rows, KVH, D), np.uint16), np.empty((rows, KVH, D), np.uint16)
    nk, nv = R.rms(f(k[:rows]), f(kn)), R.rms(f(v[:rows] if own_v else k[:rows]))
    fk[:], fv[:] = syn.bf16_bits(R.rope(nk, positions[:rows], rotated, base)), syn.bf16_bits(nv)
    fk[live], fv[live] = gk[at], gv[at]
    near(fk, nk, "k")
    near(fv, nv, "v")
    rest = np.setdiff1d(np.arange(num * block), at)
    assert np.array_equal(gk[rest], ck[rest]) and np.array_equal(gv[rest], cv[rest])
    b.prepare(qd, *args, qd, stream)                         # in place: the same bits
    assert np.array_equal(qd.to_host(stream)[:rows], got[:rows])


def test_prepare_turns_as_rope_does(stream):
    """A row whose norm is exact (values of one magnitude, weight 1, eps 0) has hyp_rope's bits."""
    D, H, rows = 256, 3, 40
    rng = np.random.default_rng(3)
    x = syn.bf16_bits(np.where(rng.random((rows, H, D)) < 0.5, -1.0, 1.0).astype(np.float32))
    one = dev(syn.bf16_bits(np.ones(D, np.float32)), stream)
    offset = 131072
    cache = hy.KvCache(64, H, D)
    b = hy.Batch(64, 1, dev(np.zeros((1, 1), np.uint32), stream), dev(u32(rows), stream), dev(u32(0, rows), stream),
                 dev(np.arange(rows, dtype=np.uint32), stream), dev(np.arange(offset, offset + rows, dtype=np.uint32), stream))
    xd, got, ref = dev(x, stream), hy.DeviceArray(x.shape, np.uint16), hy.DeviceArray(x.shape, np.uint16)
    b.prepare(xd, xd, None, H, cache, one, one, 0.0, D, 1e4, got, stream)
    hy.rope(xd, rows, H, D, D, 1e4, offset, ref, stream)
    assert np.array_equal(got.to_host(stream), ref.to_host(stream))
    assert np.array_equal(read_cache(cache, (64, H, D), stream)[0][:rows], ref.to_host(stream))


# ---- attention --------------------------------------------------------------------------------

def f64(bits):
    return syn.bf16_to_f32(bits).astype(np.float64)


class Scene:
    """A batch's cache, tables and rows for attention, on the host and the device."""

    def __init__(self, seed, stream, lens, rows, H, KVH, D, block=16, prefix=0, window=0, scale=None, extra_rows=0,
                 spread=2.0):
        rng = np.random.default_rng(seed)
        self.stream, self.H, self.KVH, self.D = stream, H, KVH, D
        self.block, self.prefix, self.window = block, prefix, window
        self.scale = D ** -0.5 if scale is None else scale
        counts = [R.blocks(prefix, block)] + [R.blocks(n, block) for n in lens]
        self.num = sum(counts) + 2
        order = rng.permutation(self.num).astype(np.uint32)
        self.prefix_table = order[:counts[0]]
        self.tables = np.full((len(lens), max(counts[1:]) + 1), R.NONE, np.uint32)
        at = counts[0]
        for r, c in enumerate(counts[1:]):
            self.tables[r, :c] = order[at:at + c]
            at += c
        self.lens = np.array(lens, np.uint32)
        self.row_start = np.concatenate(([0], np.cumsum(rows))).astype(np.uint32)
        self.rows = int(self.row_start[-1])
        bits = lambda size, *shape: syn.bf16_bits((size * rng.standard_normal(shape)).astype(np.float32))  # noqa: E731
        size = 1.0 if scale is None else D ** -0.25
        self.q = bits(spread * size, self.rows + extra_rows, H, D)
        self.ck, self.cv = bits(size, self.num * block, KVH, D), bits(1.0, self.num * block, KVH, D)

    def live_slots(self):
        """Slots that hold tokens."""
        at = [int(self.prefix_table[j // self.block]) * self.block + j % self.block for j in range(self.prefix)]
        for r, n in enumerate(self.lens):
            at += [int(self.tables[r, j // self.block]) * self.block + j % self.block for j in range(int(n))]
        at = np.array(at, np.int64)
        return at[at < self.num * self.block]

    def place(self):
        s = self.stream
        self.cache = hy.KvCache(self.num * self.block, self.KVH, self.D)
        fill_cache(self.cache, self.ck, self.cv, s)
        n = max(1, self.q.shape[0])
        self.d_lens, self.d_start = dev(self.lens, s), dev(self.row_start, s)
        self.d_tables = dev(self.tables, s)
        self.batch = hy.Batch(self.block, self.num, self.d_tables, self.d_lens, self.d_start,
                              dev(np.zeros(n, np.uint32), s), dev(np.zeros(n, np.uint32), s), self.prefix,
                              dev(self.prefix_table, s) if self.prefix else None)
        self.d_q, self.d_out = dev(self.q, s), dev(np.full(self.q.shape, 0x7FC0, np.uint16), s)
        need = self.batch.attention_workspace_bytes(self.H, self.cache)
        self.work = dev(np.full(need + 256, 0xFF, np.uint8), s)   # (parts are NaN until they are written)
        self.work.nbytes = need
        return self

    def run(self, stream=None):
        self.batch.attention(self.d_q, self.H, self.cache, self.window, self.scale, self.d_out, self.work,
                             stream or self.stream)

    def result(self):
        out = self.d_out.to_host(self.stream)
        self.work.nbytes += 256
        assert np.all(self.work.to_host(self.stream)[-256:] == 0xFF)   # nothing behind the workspace
        self.work.nbytes -= 256
        return out

    def check(self, what=""):
        out = self.result()
        assert np.all(out[self.rows:] == 0x7FC0)   # rows behind the last are left as they were
        self.compare(out, what)
        return out

    def one_term(self):
        """Whether some rows go through wide tiles, whose probabilities are one bf16 term."""
        G = self.H // self.KVH
        n = np.diff(self.row_start.astype(np.int64)) * G
        tiles = lambda r: -(-r // 128)  # noqa: E731
        return n.sum() > 16 and bool(self.prefix or np.any(n > 16) or 4 * tiles(n).sum() <= 5 * tiles(n.sum()))

    def compare(self, out, what=""):
        """One rounding, 2^-8. Below it: a score is off by the fp32 sums of its product (one rounding a step
        of 32 dims, and a few for its scaling), which moves every weight by as much, and a
        probability in two bf16 terms by 2^-16. One term moves a weight by up to 2^-8 of itself; the output
        is the mean by the moved weights, so off by at most 2^-8 / (1 - 2^-8) of its values' mean
        distance from it."""
        ck, cv = f64(self.ck), f64(self.cv)
        ref, size, apart = R.attention(f64(self.q[:self.rows]), ck, cv, self.tables, self.lens, self.row_start, self.block,
                                self.num, self.prefix, self.prefix_table, self.window, self.scale)
        got = f64(out[:self.rows])
        score = (self.D / 32 + 8) * 2.0**-24 * abs(self.scale) * size[..., None]
        vmax = np.max(np.abs(cv[self.live_slots()]), initial=0.0, where=np.isfinite(cv[self.live_slots()]))
        bound = 2.0**-8 * np.abs(ref) + vmax * (2.0**-15 + 2 * score)
        if self.one_term():
            bound += 2.0**-8 * (1 + 2.0**-7) * apart
        err = np.abs(got - ref)
        say(f"  attention {what}: worst {np.max(err / bound, initial=0.0):.3f} of the bound")
        assert np.all(err <= bound), what


SCENES = [
    # lens, rows, H, KVH, D, block, prefix, window, scale
    ([1], [1], 4, 2, 64, 16, 0, 0, None),                              # one token sees itself
    ([5, 1, 0, 33], [1, 1, 0, 1], 16, 8, 256, 16, 0, 0, 1.0),          # an idle request
    ([40, 7, 65, 64], [1, 1, 1, 1], 16, 8, 256, 16, 100, 0, 1.0),      # a prefix that ends inside a block
    ([40, 7, 165, 64], [1, 1, 1, 1], 16, 8, 256, 16, 90, 128, 1.0),    # a window across prefix and own tokens
    ([300, 20], [1, 1], 16, 8, 256, 32, 200, 64, 1.0),                 # a window past the prefix for one of them
    ([10, 3, 129], [1, 1, 1], 16, 1, 512, 16, 333, 0, 1.0),
    ([900, 2, 31], [1, 1, 1], 16, 1, 512, 64, 0, 0, 1.0),
    ([17, 50, 100], [1, 1, 1], 32, 8, 128, 8, 63, 0, None),
    ([17, 50, 100], [1, 1, 1], 12, 12, 64, 1, 5, 0, None),             # a block a token
    ([17, 50], [1, 1], 7, 1, 64, 16, 1000, 0, None),                   # odd heads
    ([30, 9, 64, 33], [5, 9, 1, 4], 16, 8, 256, 16, 50, 0, 1.0),       # drafts
    ([30, 90, 64, 33], [5, 70, 1, 33], 16, 8, 256, 16, 50, 40, 1.0),   # prompts' ends, window
    ([40, 33, 130], [40, 33, 64], 16, 1, 512, 16, 70, 0, 1.0),         # whole questions
    ([260, 1], [257, 1], 6, 2, 128, 128, 0, 0, None),
    ([30, 200, 1], [30, 99, 1], 8, 8, 64, 16, 45, 50, None),
    ([70] * 70, [1] * 70, 4, 2, 64, 16, 20, 0, None),                  # more requests than a wave has lanes
    ([3, 200] * 65, [1, 2] * 65, 4, 1, 128, 16, 64, 100, None),
    ([9000], [1], 8, 1, 128, 16, 0, 0, None),                          # one long request over many workers
    ([1], [1], 4, 1, 64, 32, 20000, 0, None),
]


@pytest.mark.parametrize("lens,rows,H,KVH,D,block,prefix,window,scale", SCENES)
def test_attention(stream, lens, rows, H, KVH, D, block, prefix, window, scale):
    say(f"attention {len(lens)} requests H={H} KVH={KVH} D={D} block={block} prefix={prefix} window={window}")
    s = Scene(sum(lens) + D, stream, lens, rows, H, KVH, D, block, prefix, window, scale, extra_rows=3).place()
    s.run()
    first = s.check()
    s.run()
    assert np.array_equal(first, s.result())   # the same bits again


@pytest.mark.parametrize("D,KVH", [(64, 4), (256, 2), (512, 1)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_attention_ignores_what_it_does_not_see(stream, D, KVH, bad):
    """Every slot without a token, the tokens that a draft row does not see yet, and those before a
    window hold what is not finite; so does a block outside the pool's place in the cache."""
    s = Scene(D, stream, [20, 37, 50], [3, 1, 18], 4 * KVH, KVH, D, 16, 45, 30)
    poison = syn.bf16_bits(np.array([bad], np.float32))[0]
    rest = np.setdiff1d(np.arange(s.num * s.block), s.live_slots())
    s.ck[rest], s.cv[rest] = poison, poison
    s.cv[int(s.tables[0, 1]) * 16 + 3] = poison         # request 0's token 19: seen by its last row alone
    s.ck[int(s.prefix_table[0]) * 16 + 2] = poison      # before every window
    s.cv[int(s.prefix_table[0]) * 16 + 2] = poison
    s.place()
    s.run()
    out = s.result()
    seen = out[2].copy()
    assert np.all(~np.isfinite(f64(seen)))              # that row takes it
    out[2] = 0
    s.cv[int(s.tables[0, 1]) * 16 + 3] = 0
    ck, cv = f64(s.ck), f64(s.cv)
    want, _, far = R.attention(f64(s.q), ck, cv, s.tables, s.lens, s.row_start, 16, s.num, s.prefix, s.prefix_table, s.window,
                          s.scale)
    got = f64(out)
    keep = np.arange(s.rows) != 2
    vmax = np.max(np.abs(cv), where=np.isfinite(cv), initial=0.0)
    assert np.all(np.abs(got - want)[keep] <= 2.0**-8 * np.abs(want[keep]) + vmax * 2.0**-12 + 2.0**-8 * 1.01 * far[keep])


def test_attention_scores_that_are_not_finite(stream):
    """Rows whose every score is -inf give zeros; a NaN score gives NaN; -inf scores beside finite ones
    weigh nothing; the lowest finite value is a value."""
    D = 64
    s = Scene(1, stream, [20, 20, 20, 20], [1, 1, 1, 1], 2, 2, D, 16, 0, 0, scale=1.0)
    at = [s.tables[r, :2].astype(np.int64) for r in range(4)]
    for r in range(4):
        s.q[r] = syn.bf16_bits(np.ones((2, D), np.float32))
    inf, nan, low = (syn.bf16_bits(np.array([v], np.float32))[0] for v in (-np.inf, np.nan, -3e38))
    for b in at[0]:
        s.ck[b * 16:(b + 1) * 16] = inf
    s.ck[at[1][0] * 16 + 5, :, 3] = nan
    s.ck[at[2][0] * 16 + 5, :, 3] = inf
    s.ck[at[3][0] * 16 + 7, :, 0] = low
    s.place()
    s.run()
    out = f64(s.result())
    assert np.all(out[0] == 0.0) and np.all(np.isnan(out[1]))
    ref, _, far = R.attention(f64(s.q[2:]), f64(s.ck), f64(s.cv), s.tables[2:], s.lens[2:], u32(0, 1, 2), 16, s.num, 0, u32(), 0,
                         1.0)
    assert np.all(np.abs(out[2:] - ref) <= 2.0**-8 * np.abs(ref) + 2.0**-12 + 2.0**-8 * 1.01 * far)


def test_attention_blocks_outside_the_pool_hold_no_tokens(stream):
    s = Scene(2, stream, [40, 40, 20], [1, 1, 2], 8, 2, 128, 8, 30, 0)
    s.tables[0, 1] = s.num                   # a block in the middle
    s.tables[1, :] = 0xFFFFFF00              # every own block
    s.prefix_table[2] = 4000000000
    s.place()
    s.run()
    s.check("with missing blocks")


def test_attention_lengths_at_odds_with_rows(stream):
    """More rows than tokens: the first rows stand before the own tokens, or before everything. Lengths
    past the tables end at the tables."""
    s = Scene(3, stream, [2, 0, 30, 1], [6, 4, 2, 9], 4, 2, 64, 16, 5, 0)
    s.lens[2] = 4000000000
    s.tables = s.tables[:, :2]
    s.place()
    s.run()
    out = f64(s.result())
    s.lens[2] = 32
    ref, _, far = R.attention(f64(s.q), f64(s.ck), f64(s.cv), s.tables, s.lens, s.row_start, 16, s.num, 5, s.prefix_table, 0,
                         s.scale)
    assert np.any(np.all(ref == 0, axis=(1, 2)))     # rows that see nothing are among them
    assert np.all(np.abs(out - ref) <= 2.0**-8 * np.abs(ref) + 2.0**-12 * 6 + 2.0**-8 * 1.01 * far)


@pytest.mark.parametrize("starts", [(0, 9, 3, 20, 5), (7, 3, 2, 1, 0), (0, 4000000000, 2, 9, 12), (0, 2, 4, 6, 99), (5, 6, 7, 8, 9),
                                    (0, 12, 0, 12, 12)])
def test_attention_holds_its_bounds_on_damaged_row_starts(stream, starts):
    s = Scene(4, stream, [30, 20, 9, 40], [3, 3, 3, 3], 4, 2, 64, 16, 20, 0)
    s.row_start = np.array(starts, np.uint32)
    s.rows = 0
    s.place()
    s.run()
    s.result()                               # (the workspace's end is untouched; the outputs are not defined)


def test_attention_recorded_and_replayed_with_new_lengths(stream):
    """A graph reads the lengths on the device; two recorded calls with a workspace each replay beside
    one another."""
    other = hy.Stream()
    scenes = [Scene(7 + i, stream, [30, 200, 64], [1, 1, 1], 16, 8, 256, 16, 70, 0, 1.0).place() for i in range(2)]
    graphs = []
    for s, st in zip(scenes, (stream, other)):
        with hy.Graph.capture(st) as g:
            s.run(st)
        graphs.append(g)
    for cut in (0, 29, 5, 17):
        for s in scenes:
            s.lens = np.array([30 - cut, 200 - 6 * cut, 64], np.uint32)
            s.d_lens.upload(s.lens, stream)
            s.d_out.upload(np.full(s.q.shape, 0x7FC0, np.uint16), stream)
        for g, st in zip(graphs, (stream, other)):
            g.launch(st)
        other.synchronize()
        for s in scenes:
            s.check(f"replayed, {cut} fewer")
    for g in graphs:
        g.close()
    other.close()


def test_attention_of_one_request_agrees_with_hyp_attention(stream):
    """Blocks in order and no prefix: the batch's attention is hyp_attention's over a linear cache, up
    to the latter's probabilities in one bf16 term."""
    H, KVH, D, n = 16, 8, 256, 700
    s = Scene(11, stream, [n], [1], H, KVH, D, 16, 0, 0, 1.0)
    s.tables[0, :R.blocks(n, 16)] = np.arange(R.blocks(n, 16))
    s.place()
    s.run()
    got = f64(s.check("in order"))
    out = hy.DeviceArray(s.q.shape, np.uint16)
    hy.call("hyp_attention", s.d_q.ptr, None, None, 1, H, s.cache.handle, n - 1, n - 1, 0, out.ptr, stream.handle)
    ref = f64(out.to_host(stream))
    assert np.all(np.abs(got - ref) <= 2.0**-7 * np.abs(ref) + 2.0**-9 * np.max(np.abs(f64(s.cv))))


# ---- sampling ---------------------------------------------------------------------------------

CONFIG = np.dtype([("temperature", "<f4"), ("top_k", "<i4"), ("top_p", "<f4"), ("min_p", "<f4"), ("seed", "<u8")])


def draw(stream, bits, configs, uniforms, logprobs=True, unaligned=False):
    """Tokens and logprobs of rows of logits; `unaligned` puts the rows 2 bytes past an aligned place."""
    rows, vocab = bits.shape
    flat = np.concatenate((np.zeros(1, np.uint16), bits.ravel())) if unaligned else bits
    d = dev(flat, stream)
    if unaligned:
        class Behind:
            ptr = ctypes.c_void_p(d.ptr.value + 2)
        at = Behind()
    else:
        at = d
    need = hy.sample_batch_workspace_bytes(rows, vocab)
    work = dev(np.full(need + 64, 0xA5, np.uint8), stream)
    work.nbytes = need
    tok = dev(np.full(rows + 1, 0xDEAD, np.uint32), stream)
    lp = dev(np.full(rows + 1, 7.0, np.float32), stream) if logprobs else None
    hy.sample_batch(at, rows, vocab, dev(configs, stream), dev(np.asarray(uniforms, np.float32), stream), tok, lp, work,
                    stream)
    tokens = tok.to_host(stream)
    assert tokens[rows] == 0xDEAD
    work.nbytes = need + 64
    assert np.all(work.to_host(stream)[need:] == 0xA5)
    if not logprobs:
        return tokens[:rows], None
    values = lp.to_host(stream)
    assert values[rows] == 7.0
    return tokens[:rows], values[:rows]


def check_draw(stream, bits, configs, uniforms, what, **kw):
    tokens, logprobs = draw(stream, bits, configs, uniforms, **kw)
    values = syn.bf16_to_f32(bits).reshape(bits.shape)
    for r in range(bits.shape[0]):
        c = configs[r]
        token, lp = R.sample(values[r], float(c["temperature"]), int(c["top_k"]), float(c["top_p"]), float(c["min_p"]),
                             float(np.float32(uniforms[r])))
        assert tokens[r] == token, (what, r, c, uniforms[r], int(tokens[r]), token)
        if logprobs is not None:
            # one rounding to fp32 of a value with an fp64 error far below it
            assert logprobs[r] == lp or abs(logprobs[r] - lp) <= 2.0**-24 * abs(lp) + 1e-12, (what, r, logprobs[r], lp)


def mixed(rng, rows, vocab):
    c = np.zeros(rows, CONFIG)
    c["temperature"] = np.where(rng.random(rows) < 0.15, 0.0, rng.uniform(0.2, 2.0, rows))
    c["top_k"] = np.where(rng.random(rows) < 0.4, 0, rng.integers(1, vocab + 3, rows))
    c["top_p"] = np.where(rng.random(rows) < 0.3, rng.integers(0, 2, rows), rng.uniform(0.05, 1.0, rows))
    c["min_p"] = np.where(rng.random(rows) < 0.5, 0.0, rng.uniform(0.0, 0.4, rows))
    c["seed"] = rng.integers(0, 2**63, rows)
    return c


@pytest.mark.parametrize("rows,vocab,spread", [(1, 1, 3.0), (1, 2, 3.0), (3, 7, 3.0), (5, 63, 8.0), (2, 513, 1.0),
                                               (40, 1000, 3.0), (300, 300, 2.0), (9, 8193, 0.05), (6, 50001, 3.0),
                                               (1, 262144, 3.0), (4, 262144, 9.0), (33, 20000, 3.0), (2, 1000003, 2.0)])
def test_sample(stream, rows, vocab, spread):
    say(f"sample rows={rows} vocab={vocab} spread={spread}")
    rng = np.random.default_rng(rows * 7 + vocab)
    bits = syn.bf16_bits(np.clip(spread * rng.standard_normal((rows, vocab)), -30, 30).astype(np.float32))
    configs, uniforms = mixed(rng, rows, vocab), rng.random(rows).astype(np.float32)
    check_draw(stream, bits, configs, uniforms, "mixed")
    check_draw(stream, bits, configs, uniforms, "unaligned rows", unaligned=True, logprobs=False)
    configs[:] = (1.0, 0, 0.0, 0.0, 0)
    check_draw(stream, bits, configs, np.linspace(0, 1, rows, dtype=np.float32), "temperature alone")


def shaped(kind, rng, vocab):
    x = 3.0 * rng.standard_normal(vocab)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "two values":
        x = np.where(rng.random(vocab) < 0.5, 2.0, 2.25)
    elif kind == "zeros":
        x = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    elif kind == "next to zero":
        x = 1e-9 * rng.standard_normal(vocab)
    elif kind == "some next to zero":
        x[::3] = 1e-9 * rng.standard_normal(x[::3].size)
    elif kind == "large":
        x = 90.0 * x
    elif kind == "largest":
        x = np.where(rng.random(vocab) < 0.01, 3.3e38, x)
    elif kind == "lowest masked":
        x = np.where(rng.random(vocab) < 0.9, -3.3895e38, x)   # bf16's lowest
    elif kind == "masked":
        x = np.where(rng.random(vocab) < 0.9, -np.inf, x)
    elif kind == "one left":
        x[:] = -np.inf
        x[vocab // 2] = -4.0
    elif kind == "nan":
        x = np.where(rng.random(vocab) < 0.1, np.nan, x)
    elif kind == "infinite":
        x = np.where(rng.random(vocab) < 0.02, np.inf, x)
    elif kind == "nothing":
        x = np.where(rng.random(vocab) < 0.5, np.nan, -np.inf)
    elif kind == "below":
        x = -200.0 - np.abs(40.0 * x)
    elif kind == "denormal":
        x = 1e-39 * rng.standard_normal(vocab)
    elif kind == "descending":
        x = np.linspace(20, -20, vocab)
    return syn.bf16_bits(x.astype(np.float32))


@pytest.mark.parametrize("vocab", [999, 70000])
@pytest.mark.parametrize("kind", ["equal", "two values", "zeros", "next to zero", "some next to zero", "large", "largest",
                                  "lowest masked", "masked", "one left", "nan", "infinite", "nothing", "below", "denormal",
                                  "descending"])
def test_sample_rows_of_every_kind(stream, kind, vocab):
    say(f"sample {kind} vocab={vocab}")
    rng = np.random.default_rng(vocab)
    rows = 8
    bits = np.stack([shaped(kind, rng, vocab) for _ in range(rows)])
    configs = mixed(rng, rows, vocab)
    configs["temperature"][:3] = (1.0, 0.0, 50.0)
    configs[4] = (1.0, 0, 0.5, 0.0, 0)
    configs[5] = (0.7, 0, 0.0, 0.0, 0)
    configs[6] = (30.0, 100, 0.0, 0.0, 0)
    check_draw(stream, bits, configs, rng.random(rows).astype(np.float32), kind)


def test_sample_configurations_at_their_ends(stream):
    """What a configuration may hold beyond its ranges: temperatures below 0, NaN, tiny, infinite;
    top_k below 0 and past the vocabulary; top_p of 0, 1, NaN; min_p of 1 and more; uniforms of
    0, next to 1, 1, NaN, negative."""
    rng = np.random.default_rng(8)
    vocab = 3000
    rows = [(t, k, p, m, 0) for t in (1.0, -1.0, np.nan, 1e-30, np.inf) for k in (0, -5, 1, vocab + 9)
            for p in (0.0, 1.0, np.nan, 1e-9, 0.3) for m in (0.0, 1.0, 2.0, np.nan, -1.0)]
    configs = np.array(rows, CONFIG)
    bits = syn.bf16_bits((2.0 * rng.standard_normal((len(rows), vocab))).astype(np.float32))
    uniforms = np.resize(np.array([0.0, 0.5, 1.0 - 2.0**-24, 1.0, np.nan, -3.0, 2.0**-40], np.float32), len(rows))
    check_draw(stream, bits, configs, uniforms, "ends")


def test_sample_rows_do_not_depend_on_their_batch(stream):
    """A row gives the same token and the same bits of its logprob alone and in batches of any size."""
    rng = np.random.default_rng(9)
    rows, vocab = 270, 40000
    bits = syn.bf16_bits((3.0 * rng.standard_normal((rows, vocab))).astype(np.float32))
    configs, uniforms = mixed(rng, rows, vocab), rng.random(rows).astype(np.float32)
    tokens, logprobs = draw(stream, bits, configs, uniforms)
    for n in (1, 2, 9, 64, 150):
        at = slice(7, 7 + n)
        some, values = draw(stream, bits[at], configs[at], uniforms[at])
        assert np.array_equal(some, tokens[at]) and np.array_equal(values.view(np.uint32), logprobs[at].view(np.uint32)), n


def test_sample_an_empty_vocabulary(stream):
    tokens, logprobs = draw(stream, np.zeros((2, 0), np.uint16), mixed(np.random.default_rng(0), 2, 1), [0.5, 0.5])
    assert tokens.tolist() == [0, 0] and np.all(logprobs == -np.inf)


def test_sample_in_a_graph(stream):
    """Recorded once, replayed with other logits, configurations and uniforms."""
    rng = np.random.default_rng(10)
    rows, vocab = 5, 30000
    d, c, u = hy.DeviceArray((rows, vocab), np.uint16), hy.DeviceArray((rows,), CONFIG), hy.DeviceArray((rows,), np.float32)
    tok, lp = hy.DeviceArray((rows,), np.uint32), hy.DeviceArray((rows,), np.float32)
    need = hy.sample_batch_workspace_bytes(rows, vocab)
    work = hy.DeviceArray((need,), np.uint8)
    with hy.Graph.capture(stream) as g:
        hy.sample_batch(d, rows, vocab, c, u, tok, lp, work, stream)
    for _ in range(4):
        bits = syn.bf16_bits((3.0 * rng.standard_normal((rows, vocab))).astype(np.float32))
        configs, uniforms = mixed(rng, rows, vocab), rng.random(rows).astype(np.float32)
        for a, host in ((d, bits), (c, configs), (u, uniforms)):
            a.upload(host, stream)
        g.launch(stream)
        tokens = tok.to_host(stream)
        same, _ = draw(stream, bits, configs, uniforms)
        assert np.array_equal(tokens, same)
        want = [R.sample(syn.bf16_to_f32(bits[r]), *(float(configs[r]["temperature"]), int(configs[r]["top_k"]),
                         float(configs[r]["top_p"]), float(configs[r]["min_p"]), float(uniforms[r])))[0] for r in range(rows)]
        assert tokens.tolist() == want
    g.close()
