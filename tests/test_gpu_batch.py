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
