"""GPU parity of the operations on a batch's blocks (hyp_batch_fork, rewind, compact, copy) against pages_ref.py.
Everything is whole numbers or moved bits, and equal."""
import numpy as np
import pytest

import hyperion_amd as hy
import pages_ref as R
from test_gpu_batch import dev, fill_cache, read_cache, say, u32

pytestmark = pytest.mark.gpu


def some(a, least=1):
    """A device array may not be empty; the call reads none of it then."""
    return a if a.size >= least else np.zeros(least, a.dtype)


class Pool:
    """Requests over one pool of blocks: host arrays, and a call's arrays on the device."""

    def __init__(self, seed, stream, n, block, hi, spare=9, extra=2, groups=0, prefix=0, shuffle=True):
        rng = np.random.default_rng(seed)
        self.stream, self.n, self.block, self.prefix, self.rng = stream, n, block, prefix, rng
        self.lens = rng.integers(0, hi + 1, n).astype(np.uint32)
        width = R.blocks(int(self.lens.max(initial=0)), block) + extra
        # requests of a group hold the first blocks in common
        group = rng.integers(0, groups, n) if groups else np.arange(n)
        common = {}
        need = [R.blocks(int(v), block) for v in self.lens]
        total = sum(need) + R.blocks(prefix, block)
        self.num = max(1, total + spare)
        order = (rng.permutation(self.num) if shuffle else np.arange(self.num)).astype(np.uint32)
        at = R.blocks(prefix, block)
        self.prefix_table = order[:at]
        self.tables = np.full((n, width), R.NONE, np.uint32)
        for r in range(n):
            c = need[r]
            shared = common.get(group[r], np.zeros(0, np.uint32))[:max(0, int(self.lens[r]) // block - 1)]
            fresh = order[at:at + c - shared.size]
            at += fresh.size
            self.tables[r, :c] = np.concatenate((shared, fresh))
            if group[r] not in common:
                common[group[r]] = self.tables[r, :int(self.lens[r]) // block]
        self.taken = at
        self.free = np.concatenate((np.full(at, 12345, np.uint32), order[at:]))

    def place(self, in_place=False):
        s = self.stream
        self.d_tables, self.d_lens = dev(some(self.tables), s), dev(some(self.lens), s)
        self.d_free, self.d_taken = dev(self.free, s), dev(u32(self.taken), s)
        self.lens_out = self.d_lens if in_place else dev(np.full(max(self.n, 1), 77, np.uint32), s)
        self.taken_out = self.d_taken if in_place else dev(u32(77), s)
        self.served, self.n_copies = dev(u32(77), s), dev(u32(77), s)
        self.copies = dev(np.full((max(self.n, self.num // 2, 1), 3), 77, np.uint32), s)
        self.d_prefix = dev(self.prefix_table, s) if self.prefix else None
        self.rows = [dev(np.full(some(np.zeros(k)).size, 77, np.uint32), s) for k in (self.n + 1, 1, 1)]
        self.batch = self.of(self.lens_out)
        self.work = dev(np.full(self.batch.pages_workspace_bytes(), 0xEE, np.uint8), s)
        return self

    def of(self, lens):
        """The batch with these lengths (hy.Batch takes its sizes from the arrays; here some are empty)."""
        f = hy.Batch.__new__(hy.Batch)
        f.arrays = (self.d_tables, lens, self.rows)
        f.fields = hy.BatchFields(self.n, self.block, self.num, self.tables.shape[1], 1, self.prefix,
                                  None if self.d_prefix is None else self.d_prefix.ptr, self.d_tables.ptr, lens.ptr,
                                  self.rows[0].ptr, self.rows[1].ptr, self.rows[2].ptr)
        f._ref = hy.ctypes.byref(f.fields)
        return f

    def host(self, a, shape=None):
        got = a.to_host(self.stream)
        return got if shape is None else got.reshape(-1)[:int(np.prod(shape))].reshape(shape)

    def check_copies(self, copies):
        assert int(self.host(self.n_copies)[0]) == len(copies), (int(self.host(self.n_copies)[0]), len(copies))
        got = self.host(self.copies)
        assert [tuple(map(int, c)) for c in got[:len(copies)]] == copies
        assert np.all(got[len(copies):] == 77)

    # ---- fork
    def fork(self, parents):
        self.d_parents = dev(some(parents), self.stream)
        self.batch.fork(self.d_lens, self.d_parents, self.d_free, self.d_taken, self.taken_out, self.served, self.copies,
                        self.n_copies, self.stream)

    def check_fork(self, parents):
        tables, lens, taken, served, copies = R.fork(self.lens, parents, self.tables, self.free, self.taken, self.block)
        assert np.array_equal(self.host(self.d_tables, tables.shape), tables)
        assert np.array_equal(self.host(self.lens_out)[:self.n], lens)
        assert int(self.host(self.taken_out)[0]) == taken and int(self.host(self.served)[0]) == served
        assert np.array_equal(self.host(self.d_free), self.free)
        self.check_copies(copies)
        return served

    # ---- rewind
    def rewind(self, drop):
        self.d_drop = dev(some(drop), self.stream)
        self.batch.rewind(self.d_lens, self.d_drop, self.d_free, self.d_taken, self.taken_out, self.copies, self.n_copies,
                          self.work, self.stream)

    def check_rewind(self, drop):
        tables, lens, free, top, copies = R.rewind(self.lens, drop, self.tables, self.free, self.taken, self.block)
        assert np.array_equal(self.host(self.lens_out)[:self.n], lens)
        assert int(self.host(self.taken_out)[0]) == top, (int(self.host(self.taken_out)[0]), top)
        assert np.array_equal(self.host(self.d_tables, tables.shape), tables)
        assert np.array_equal(self.host(self.d_free)[top:], free[top:])
        self.check_copies(copies)
        return lens, copies

    # ---- compact
    def compact(self, in_place):
        s = self.stream
        self.t_out = self.d_tables if in_place else dev(np.full(some(self.tables).shape, 77, np.uint32), s)
        self.p_out = self.d_prefix if in_place or not self.prefix else dev(np.full(self.prefix_table.size, 77, np.uint32), s)
        self.compact_batch = self.of(self.d_lens)
        self.compact_batch.compact(self.t_out, self.p_out, self.d_free, self.taken_out, self.copies, self.n_copies, self.work, s)

    def check_compact(self):
        tables, prefix, count, copies = R.compact(self.lens, self.tables, self.prefix_table, self.num, self.block)
        assert np.array_equal(self.host(self.t_out, tables.shape), tables)
        if self.prefix:
            assert np.array_equal(self.host(self.p_out), prefix)
        assert int(self.host(self.taken_out)[0]) == count
        free = self.host(self.d_free)
        assert np.array_equal(free[count:], np.arange(count, self.num))
        assert np.array_equal(free[:count], self.free[:count])
        self.check_copies(copies)
        return copies


POOLS = [
    # n, block, hi, spare, extra, groups
    (1, 16, 40, 9, 2, 0),
    (2, 1, 30, 40, 2, 0),        # a block a token
    (7, 16, 100, 9, 0, 3),
    (64, 16, 4000, 40, 8, 0),
    (65, 8, 700, 200, 3, 9),
    (300, 32, 2500, 100, 2, 40),
    (1025, 64, 900, 50, 1, 100),
    (4096, 16, 60, 700, 3, 500),  # the most requests
    (3, 65536, 200000, 4, 2, 0),
    (20, 16, 40000, 9, 2, 4),     # long tables
    (40, 16, 300, 33000, 2, 6),   # small tables, a pool beyond LDS
    (250, 16, 6000, 40, 3, 30),   # tables beyond one workgroup, marks that fit LDS or not
    (400, 8, 9000, 5000, 3, 20),
]


def parents_of(rng, p, share):
    """Some requests become copies of some that have tokens; odd values among the others."""
    n = p.n
    parents = np.full(n, R.NONE, np.uint32)
    child = rng.random(n) < share
    parents[child] = rng.integers(0, n, int(child.sum()))
    odd = rng.random(n) < 0.05
    parents[odd] = rng.choice(np.array([n, n + 5, 0xFFFFFFFE, 1 << 31], np.uint32), int(odd.sum()))
    return parents


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,block,hi,spare,extra,groups", POOLS)
def test_fork(stream, n, block, hi, spare, extra, groups, in_place):
    say(f"fork: n={n} block={block} hi={hi} in_place={in_place}")
    for share in (0.0, 0.3, 0.9):
        p = Pool(n + block, stream, n, block, hi, spare, extra, groups).place(in_place)
        parents = parents_of(p.rng, p, share)
        p.fork(parents)
        p.check_fork(parents)


def test_fork_without_free_blocks(stream):
    """Copies are served as far as free blocks go; those that need none behind the first that lacks one wait too."""
    say("fork: too few free blocks")
    for spare in (0, 1, 2, 7, 30):
        p = Pool(spare, stream, 60, 16, 300, spare)
        p.lens[::3] = p.lens[::3] // 16 * 16
        p.place()
        parents = np.full(60, R.NONE, np.uint32)
        parents[20:] = p.rng.integers(0, 20, 40)
        p.fork(parents)
        served = p.check_fork(parents)
        assert (served == 60) == (spare == 30)
    p.taken = p.num + 5   # more taken than there are
    p.place()
    p.fork(parents)
    p.taken = p.num
    p.check_fork(parents)


def test_fork_of_lengths_past_the_table(stream):
    say("fork: lengths past the table")
    p = Pool(3, stream, 8, 16, 100, 9, 0)
    p.lens[:4] = [0xFFFFFFFF, 100000, p.tables.shape[1] * 16 + 1, p.tables.shape[1] * 16]
    p.place()
    parents = np.array([R.NONE] * 4 + [0, 1, 2, 3], np.uint32)
    p.fork(parents)
    p.check_fork(parents)


def drops_of(rng, p, kind):
    n = p.n
    if kind == "none":
        return np.zeros(n, np.uint32)
    if kind == "all":
        return np.full(n, hy.REQUEST_DONE, np.uint32)
    drop = rng.integers(0, 8, n).astype(np.uint32)
    if kind == "far":
        drop = (p.lens * rng.random(n)).astype(np.uint32)
    drop[rng.random(n) < 0.15] = hy.REQUEST_DONE
    exact = rng.random(n) < 0.1
    drop[exact] = p.lens[exact]
    return drop


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,block,hi,spare,extra,groups", POOLS)
def test_rewind(stream, n, block, hi, spare, extra, groups, in_place):
    say(f"rewind: n={n} block={block} hi={hi} groups={groups} in_place={in_place}")
    copied = 0
    for kind in ("none", "few", "far", "all"):
        p = Pool(n + block, stream, n, block, hi, spare, extra, groups).place(in_place)
        drop = drops_of(p.rng, p, kind)
        p.rewind(drop)
        copied += len(p.check_rewind(drop)[1])
    assert copied or groups < 9


@pytest.mark.parametrize("spare", [0, 1, 5])
def test_rewind_into_shared_blocks_without_free_ones(stream, spare):
    """Requests that find no block of their own end where the shared one begins."""
    say(f"rewind: shared blocks, {spare} free")
    p = Pool(spare, stream, 40, 16, 400, spare, groups=5)
    p.place()
    drop = (p.lens * 0.6).astype(np.uint32)
    p.rewind(drop)
    lens, copies = p.check_rewind(drop)
    # none of the blocks that come back: only as many as are free
    p = Pool(spare, stream, 40, 64, 300, spare, groups=2)
    lens0 = p.lens.copy()
    p.tables[:], p.lens[:] = p.tables[int(np.argmax(lens0))], lens0.max()   # all hold the same
    p.place()
    drop = p.rng.integers(1, 60, 40).astype(np.uint32)
    drop[7] = 0
    p.rewind(drop)
    lens, copies = p.check_rewind(drop)
    assert len(copies) == min(p.num - p.taken, np.count_nonzero((p.lens - drop) % 64 * (drop > 0)))


def test_rewind_with_ids_outside_the_pool(stream):
    say("rewind: ids outside the pool")
    p = Pool(8, stream, 30, 16, 300, 9, groups=6)
    at = p.rng.random(p.tables.shape) < 0.1
    p.tables[at] = p.rng.choice(np.array([p.num, p.num + 7, R.NONE, 1 << 31], np.uint32), int(at.sum()))
    p.place()
    drop = drops_of(p.rng, p, "far")
    p.rewind(drop)
    p.check_rewind(drop)
    p = Pool(9, stream, 30, 16, 300, 9)
    p.lens[3], p.lens[4], p.taken = 0xFFFFFFFF, 10**6, 5   # lengths past the table; fewer taken than come back
    p.place()
    drop = np.full(30, hy.REQUEST_DONE, np.uint32)
    p.rewind(drop)
    p.check_rewind(drop)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("prefix", [0, 333])
@pytest.mark.parametrize("n,block,hi,spare,extra,groups", POOLS)
def test_compact(stream, n, block, hi, spare, extra, groups, prefix, in_place):
    say(f"compact: n={n} block={block} hi={hi} prefix={prefix} in_place={in_place}")
    for more in (0, 1, 3000):
        p = Pool(n + block, stream, n, block, hi, spare + more, extra, groups, prefix).place()
        if block * p.num >= 1 << 30:
            continue
        p.compact(in_place)
        p.check_compact()


def test_compact_of_ids_in_order_or_outside(stream):
    say("compact: nothing to move; ids outside the pool")
    p = Pool(1, stream, 20, 16, 300, 50, shuffle=False).place()
    p.compact(False)
    assert not p.check_compact()
    p = Pool(2, stream, 20, 16, 300, 50, prefix=40)
    p.tables[p.rng.random(p.tables.shape) < 0.2] = p.num + 3
    p.prefix_table[1] = R.NONE
    p.lens[5] = 0xFFFFFFFF
    p.place()
    p.compact(True)
    p.check_compact()
    p = Pool(3, stream, 1, 16, 0, 1).place()   # one block, none in use
    p.compact(False)
    p.check_compact()


def test_no_requests(stream):
    say("pages: no requests")
    p = Pool(4, stream, 0, 16, 0, 10, prefix=50).place()
    p.fork(np.zeros(0, np.uint32))
    p.check_fork(np.zeros(0, np.uint32))
    p.rewind(np.zeros(0, np.uint32))
    p.check_rewind(np.zeros(0, np.uint32))
    p.compact(False)
    p.check_compact()


# ---- copies ---------------------------------------------------------------------------------

COPIES = [
    # caches (KV heads, head dim), block, blocks, copies
    ([(2, 64)], 16, 10, 3),
    ([(1, 64)], 1, 40, 20),
    ([(8, 256), (1, 512), (3, 128)], 16, 30, 12),
    ([(4, 64)] * 130, 8, 12, 5),          # more caches than one launch takes
    ([(2, 128)], 4096, 6, 3),
    ([(1, 64), (2, 64)], 16, 3000, 1400),
]


@pytest.mark.parametrize("shapes,block,num,count", COPIES)
def test_copy(stream, shapes, block, num, count):
    say(f"copy: {len(shapes)} caches block={block} copies={count} of {num}")
    rng = np.random.default_rng(num)
    caches, host = [], []
    for kvh, d in shapes:
        caches.append(hy.KvCache(num * block + 5, kvh, d))
        kv = [rng.integers(0, 1 << 16, (num * block + 5, kvh, d), dtype=np.uint16) for _ in range(2)]
        fill_cache(caches[-1], *kv, stream)
        host.append(kv)
    ids = rng.permutation(num).astype(np.uint32)
    copies = np.stack((ids[:count], ids[count:2 * count], rng.integers(0, block + 1, count)), 1).astype(np.uint32)
    copies[0, 2] = block
    if count > 4:
        copies[1, 2] = 0xFFFFFFFF                                # as many as a block has
        copies[2, 0], copies[3, 1] = num, R.NONE                 # outside
        copies[4, 1] = copies[4, 0]                              # to itself
    one = dev(np.zeros(1, np.uint32), stream)
    batch = hy.Batch(block, num, dev(np.zeros((1, 1), np.uint32), stream), one, dev(u32(0, 0), stream), one, one)
    d_copies, n = dev(copies, stream), dev(u32(count - 1), stream)

    def expect(entries):
        for kv in host:
            for a in kv:
                old = a.copy()
                for f, t, tokens in entries.tolist():
                    if f < num and t < num:
                        m = min(tokens, block)
                        a[t * block:t * block + m] = old[f * block:f * block + m]

    def compare():
        for (kvh, d), c, kv in zip(shapes, caches, host):
            for a, b in zip(read_cache(c, (num * block + 5, kvh, d), stream), kv):
                assert np.array_equal(a, b)

    batch.copy(caches, d_copies, n, stream)      # all but the last
    expect(copies[:count - 1])
    compare()
    n.upload(u32(count + 1000), stream)          # no more than the list has
    batch.copy(caches, d_copies, n, stream)
    expect(copies)
    compare()
    n.upload(u32(0), stream)
    batch.copy(caches, d_copies, n, stream)
    compare()


@pytest.mark.parametrize("tokens", [65536, 40001, 16385, 1])
def test_copy_of_the_longest_blocks_in_many_caches(stream, tokens):
    """More pieces than a launch has workgroups: blocks of 65536 tokens, 128 caches (two, listed over and over)."""
    say(f"copy: {tokens} of 65536 tokens, 128 caches")
    rng = np.random.default_rng(tokens)
    block, num, kvh, d = 65536, 2, 1, 64
    caches, host = [hy.KvCache(num * block, kvh, d) for _ in range(2)], []
    for c in caches:
        host.append([rng.integers(0, 1 << 16, (num * block, kvh, d), dtype=np.uint16) for _ in range(2)])
        fill_cache(c, *host[-1], stream)
    one = dev(np.zeros(1, np.uint32), stream)
    batch = hy.Batch(block, num, dev(np.zeros((1, 1), np.uint32), stream), one, dev(u32(0, 0), stream), one, one)
    batch.copy(caches * 64, dev(np.array([[1, 0, tokens]], np.uint32), stream), dev(u32(1), stream), stream)
    for c, kv in zip(caches, host):
        for got, was in zip(read_cache(c, (num * block, kvh, d), stream), kv):
            was[:tokens] = was[block:block + tokens]
            assert np.array_equal(got, was)
        c.close()


def test_copy_past_2_to_the_32_bytes(stream):
    """A cache of more than 2^32 bytes: offsets need 64 bits."""
    say("copy: a large cache")
    block, num, kvh, d = 64, 36000, 8, 128               # 4.7 GB for K, as much for V
    cache = hy.KvCache(num * block, kvh, d)
    k, v = cache.buffers()
    rng = np.random.default_rng(1)
    nbytes = block * kvh * d * 2
    data = [rng.integers(0, 256, nbytes, dtype=np.uint8) for _ in range(4)]
    low, high = 3, num - 2
    at = lambda p, b: hy.ctypes.c_void_p(p.value + b * nbytes)  # noqa: E731
    host = lambda a: a.ctypes.data_as(hy.ctypes.c_void_p)  # noqa: E731
    for p, a, b in ((k, 0, 1), (v, 2, 3)):
        hy.call("hyp_memcpy_htod", at(p, low), host(data[a]), nbytes, stream.handle)
        hy.call("hyp_memcpy_htod", at(p, high), host(data[b]), nbytes, stream.handle)
    stream.synchronize()
    one = dev(np.zeros(1, np.uint32), stream)
    batch = hy.Batch(block, num, dev(np.zeros((1, 1), np.uint32), stream), one, dev(u32(0, 0), stream), one, one)
    batch.copy([cache], dev(np.array([[low, high - 1, block], [high, low + 1, block]], np.uint32), stream), dev(u32(2), stream),
               stream)
    for p, a, b in ((k, 0, 1), (v, 2, 3)):
        for where, want in ((low, a), (high, b), (high - 1, a), (low + 1, b)):
            got = np.empty(nbytes, np.uint8)
            hy.call("hyp_memcpy_dtoh", host(got), at(p, where), nbytes, stream.handle)
            stream.synchronize()
            assert np.array_equal(got, data[want]), where
    cache.close()


# ---- together ---------------------------------------------------------------------------------

def test_replays_of_a_graph(stream):
    """Fork, its copies, rewind and compaction recorded once, replayed over changed arrays with eager work between."""
    say("pages: graphs")
    n, block, hi = 40, 16, 300
    p = Pool(1, stream, n, block, hi, 200, 4, groups=6, prefix=60).place()
    cache = hy.KvCache(p.num * block, 2, 64)
    parents, drop = (dev(np.full(n, R.NONE, np.uint32), stream) for _ in range(2))
    t_out, p_out, free_c, taken_c = (dev(a, stream) for a in (p.tables, p.prefix_table, p.free, u32(0)))
    copies = [dev(np.full((p.num, 3), 77, np.uint32), stream) for _ in range(3)]
    counts = [dev(u32(77), stream) for _ in range(3)]
    lens2, taken2 = dev(p.lens, stream), dev(u32(0), stream)
    after = p.of(lens2)

    def calls():
        p.batch.fork(p.d_lens, parents, p.d_free, p.d_taken, p.taken_out, p.served, copies[0], counts[0], stream)
        p.batch.copy([cache], copies[0], counts[0], stream)
        after.rewind(p.lens_out, drop, p.d_free, p.taken_out, taken2, copies[1], counts[1], p.work, stream)
        p.batch.copy([cache], copies[1], counts[1], stream)
        after.compact(t_out, p_out, free_c, taken_c, copies[2], counts[2], p.work, stream)
        p.batch.copy([cache], copies[2], counts[2], stream)

    with hy.Graph.capture(stream) as g:
        calls()
    for seed in range(4):
        q = Pool(100 + seed, stream, n, block, hi, 0, 4, groups=6, prefix=60)
        if q.taken > p.num or q.tables.shape[1] > p.tables.shape[1]:
            q.tables = q.tables[:, :p.tables.shape[1]]
            q.lens = np.minimum(q.lens, np.uint32(p.tables.shape[1] * block))
        width = p.tables.shape[1]
        tables = np.full((n, width), R.NONE, np.uint32)
        tables[:, :min(width, q.tables.shape[1])] = q.tables[:, :width]
        # spread its ids over the larger pool
        ids = q.rng.permutation(p.num).astype(np.uint32)
        assert q.num <= p.num
        tables = np.where(tables < q.num, ids[np.minimum(tables, q.num - 1)], tables)
        prefix = ids[q.prefix_table]
        free = np.concatenate((np.full(q.num, 5, np.uint32), ids[q.num:]))
        lens = q.lens.copy()
        par = np.full(n, R.NONE, np.uint32)
        par[lens < 40] = int(np.argmax(lens))
        end = np.where(q.rng.random(n) < 0.3, R.NONE, (lens * 0.4)).astype(np.uint32)
        cells = q.rng.integers(0, 1 << 16, (p.num * block, 2, 64), dtype=np.uint16)
        results = []
        for replay in (True, False):
            for a, v in ((p.d_tables, tables), (p.d_lens, lens), (p.d_free, free), (p.d_taken, u32(q.num)), (parents, par),
                         (drop, end), (p.d_prefix, prefix)):
                a.upload(v, stream)
            for c in copies:
                c.upload(np.full((p.num, 3), 77, np.uint32), stream)
            fill_cache(cache, cells, cells, stream)
            if replay:
                g.launch(stream)
            else:
                calls()
            outs = (p.d_tables, lens2, p.d_free, p.taken_out, taken2, p.served, t_out, p_out, taken_c, *copies, *counts)
            results.append([a.to_host(stream) for a in outs] + read_cache(cache, cells.shape, stream))
        t1, l1, top, served, c1 = R.fork(lens, par, tables, free, q.num, block)
        t2, l2, f2, top2, c2 = R.rewind(l1, end, t1, free, top, block)
        t3, p3, count, c3 = R.compact(l2, t2, prefix, p.num, block)
        k = cells.copy()
        for c in (c1, c2, c3):
            old = k.copy()
            for a, b, m in c:
                k[b * block:b * block + m] = old[a * block:a * block + m]
        for got in results:
            assert np.array_equal(got[0], t2) and np.array_equal(got[1], l2) and np.array_equal(got[2][top2:], f2[top2:])
            assert [int(x[0]) for x in got[3:6]] == [top, top2, served]
            assert np.array_equal(got[6], t3) and np.array_equal(got[7], p3) and int(got[8][0]) == count
            for have, number, want in zip(got[9:12], got[12:15], (c1, c2, c3)):
                assert int(number[0]) == len(want) and [tuple(map(int, c)) for c in have[:len(want)]] == want
            assert np.array_equal(got[15], k) and np.array_equal(got[16], k)
    g.close()
    cache.close()
