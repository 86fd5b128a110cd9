"""Forked requests and verified drafts without a GPU: what the entry points refuse before they touch a device,
and the references of test_gpu_pages.py and test_gpu_verify.py against closed forms."""
import ctypes

import numpy as np
import pytest

import hyperion_amd as hy
import pages_ref as R
from test_batch_cpu import BAD_BATCHES, CACHE, STREAM, fields, handle, refused


def ptr(at):
    return ctypes.c_void_p(at)


A = [ptr(0x100000 * (i + 1)) for i in range(16)]   # addresses far apart, that no refused call reads
SMALL_MEM, SMALL = handle(0x48504B56, 64 * 16 - 1, 2, 128)   # a cache of one token less than the batch has


def batch(**over):
    f = fields(tables=A[10].value, lens=A[11].value, prefix_table=A[12].value)
    for k, v in over.items():
        setattr(f, k, v)
    return f


def fork_args(b, **over):
    a = dict(lens=A[0], parents=A[1], free=A[2], taken=A[3], taken_out=A[4], served=A[5], copies=A[6], n=A[7], stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), *a.values())


def rewind_args(b, **over):
    a = dict(lens=A[0], drop=A[1], free=A[2], taken=A[3], taken_out=A[4], copies=A[6], n=A[7], work=A[8], bytes=1 << 16,
             stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), *a.values())


def compact_args(b, **over):
    a = dict(tables=A[0], prefix=A[1], free=A[2], taken_out=A[4], copies=A[6], n=A[7], work=A[8], bytes=1 << 16, stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), *a.values())


def copy_args(b, of=(CACHE,), **over):
    handles = (ctypes.c_void_p * max(len(of), 1))(*[None if c is None else c.value for c in of])
    a = dict(caches=handles, n=len(of), copies=A[0], most=8, n_copies=A[1], stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), *a.values())


def verify_args(**over):
    a = dict(logits=A[0], draft=A[1], rows=6, vocab=1000, start=A[2], requests=2, ids=A[3], configs=A[4], draft_configs=A[5],
             uniforms=A[6], accepted=A[7], rejected=A[8], tokens=A[9], logprobs=A[10], work=A[11], bytes=1 << 24, stream=STREAM)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over,says", BAD_BATCHES)
def test_bad_batches_are_refused(over, says):
    b = batch(**over)
    refused("hyp_batch_fork", *fork_args(b), says=says)
    refused("hyp_batch_rewind", *rewind_args(b), says=says)
    refused("hyp_batch_compact", *compact_args(b), says=says)
    refused("hyp_batch_copy", *copy_args(b), says=says)
    refused("hyp_batch_pages_workspace", ctypes.byref(b), ctypes.byref(ctypes.c_size_t()), says=says)


def test_tables_of_too_many_entries_are_refused():
    for b in (batch(requests=4096, max_blocks=1 << 19), batch(requests=1, max_blocks=1 << 31)):
        refused("hyp_batch_fork", *fork_args(b), says="2^31")
        refused("hyp_batch_rewind", *rewind_args(b), says="2^31")
        refused("hyp_batch_compact", *compact_args(b), says="2^31")


ODD = ptr(0x100002)


@pytest.mark.parametrize("over,says", [
    (dict(lens=None), "null"), (dict(parents=None), "null"), (dict(free=None), "null"), (dict(taken=None), "null"),
    (dict(taken_out=None), "null"), (dict(served=None), "null"), (dict(copies=None), "null"), (dict(n=None), "null"),
    (dict(stream=None), "null"), (dict(stream=CACHE), "magic"), (dict(copies=ODD), "aligned"), (dict(lens=ODD), "aligned"),
    (dict(parents=A[11]), "overlap"), (dict(copies=A[10]), "overlap"), (dict(lens=ptr(A[11].value + 4)), "overlap"),
    (dict(n=A[5]), "overlap"), (dict(taken=ptr(A[4].value)), None), (dict(lens=A[11]), None), (dict(taken=A[5]), "overlap"),
    (dict(free=A[6]), "overlap")])
def test_fork_refusals(over, says):
    if says is None:   # the same array is allowed: the call goes on to the next refusal
        refused("hyp_batch_fork", *fork_args(batch(), **over, n=None), says="non-null")
    else:
        refused("hyp_batch_fork", *fork_args(batch(), **over), says=says)
    refused("hyp_batch_fork", None, *fork_args(batch())[1:], says="batch is null")


@pytest.mark.parametrize("over,says", [
    (dict(lens=None), "null"), (dict(drop=None), "null"), (dict(free=None), "null"), (dict(taken=None), "null"),
    (dict(taken_out=None), "null"), (dict(copies=None), "null"), (dict(n=None), "null"), (dict(stream=None), "null"),
    (dict(drop=ODD), "aligned"), (dict(work=None), "workspace too small"), (dict(bytes=5 * 64 - 1), "workspace too small"),
    (dict(work=ptr(0x900004)), "aligned"), (dict(work=ptr(A[2].value + 16)), "overlap"), (dict(drop=A[11]), "overlap"),
    (dict(drop=A[2]), "overlap"), (dict(copies=A[4]), "overlap"), (dict(taken=A[7]), "overlap")])
def test_rewind_refusals(over, says):
    refused("hyp_batch_rewind", *rewind_args(batch(), **over), says=says)


@pytest.mark.parametrize("over,says", [
    (dict(tables=None), "null"), (dict(prefix=None), "prefix"), (dict(free=None), "null"), (dict(taken_out=None), "null"),
    (dict(copies=None), "null"), (dict(n=None), "null"), (dict(work=None), "workspace too small"), (dict(bytes=100), "too small"),
    (dict(stream=None), "null"), (dict(tables=ODD), "aligned"), (dict(tables=ptr(A[10].value + 16)), "overlap"),
    (dict(prefix=ptr(A[12].value + 4)), "overlap"), (dict(prefix=A[10]), "overlap"), (dict(free=A[11]), "overlap"),
    (dict(copies=A[2]), "overlap")])
def test_compact_refusals(over, says):
    refused("hyp_batch_compact", *compact_args(batch(), **over), says=says)
    refused("hyp_batch_compact", *compact_args(batch(prefix_table=None)), says="prefix")


@pytest.mark.parametrize("over,says", [
    (dict(copies=None), "null"), (dict(n_copies=None), "null"), (dict(caches=None, n=1), "null"), (dict(stream=None), "null"),
    (dict(copies=ODD), "aligned")])
def test_copy_refusals(over, says):
    refused("hyp_batch_copy", *copy_args(batch(), **over), says=says)
    refused("hyp_batch_copy", *copy_args(batch(), (CACHE, None)), says="null")
    refused("hyp_batch_copy", *copy_args(batch(), (CACHE, STREAM)), says="magic")
    refused("hyp_batch_copy", *copy_args(batch(), (CACHE, SMALL)), says="must hold")


def test_copies_of_nothing():
    b = batch()
    for args in (copy_args(b, ()), copy_args(b, most=0)):
        assert hy.lib().hyp_batch_copy(*args) == 0, hy.last_error()


@pytest.mark.parametrize("over,says", [
    (dict(logits=None), "logits"), (dict(start=None), "row_start"), (dict(ids=None), "ids"), (dict(configs=None), "configs"),
    (dict(uniforms=None), "uniforms"), (dict(accepted=None), "accepted"), (dict(rejected=None), "rejected"),
    (dict(tokens=None), "tokens"), (dict(stream=None), "null"), (dict(vocab=(1 << 23) + 1), "2^23"),
    (dict(rows=(1 << 20) + 1), "2^20"), (dict(requests=4097), "4096"), (dict(work=None), "too small"), (dict(bytes=64), "too small"),
    (dict(work=ptr(0xC00008)), "aligned"), (dict(configs=ptr(0x500004)), "8-byte"), (dict(draft_configs=ptr(0x500004)), "8-byte"),
    (dict(logits=ptr(0x100001)), "2-byte"), (dict(draft=ptr(0x100001)), "2-byte"), (dict(ids=ODD), "4-byte"),
    (dict(logprobs=ODD), "4-byte"), (dict(tokens=A[3]), "overlap"), (dict(tokens=A[7]), "overlap"), (dict(logprobs=A[6]), "overlap"),
    (dict(accepted=A[2]), "overlap"), (dict(work=A[0]), "overlap"), (dict(work=A[1]), "overlap"), (dict(rejected=A[4]), "overlap")])
def test_verify_refusals(over, says):
    refused("hyp_verify_batch", *verify_args(**over), says=says)


def test_verify_of_no_requests():
    assert hy.lib().hyp_verify_batch(*verify_args(requests=0, rows=0, logits=None)) == 0, hy.last_error()


def test_workspaces():
    out = ctypes.c_size_t()
    assert hy.lib().hyp_batch_pages_workspace(ctypes.byref(batch()), ctypes.byref(out)) == 0
    assert out.value == 5 * 64
    refused("hyp_batch_pages_workspace", ctypes.byref(batch()), None, says="out_bytes")
    refused("hyp_verify_batch_workspace", 6, 1000, 2, 1, None, says="out_bytes")
    for args, says in (((6, (1 << 23) + 1, 2, 1), "2^23"), (((1 << 20) + 1, 5, 2, 1), "2^20"), ((6, 5, 4097, 1), "4096")):
        refused("hyp_verify_batch_workspace", *args, ctypes.byref(out), says=says)
    for rows, vocab, requests in ((6, 1000, 2), (5, 262144, 1), (300, 262144, 64), (2000, 70001, 400)):
        for drafted in (False, True):
            size = hy.verify_batch_workspace_bytes(rows, vocab, requests, drafted)
            refused("hyp_verify_batch", *verify_args(rows=rows, vocab=vocab, requests=requests, bytes=size - 1,
                                                     draft=ptr(1 << 44) if drafted else None, logits=ptr(1 << 45)),
                    says="too small")


# ---- the references -------------------------------------------------------------------------

def pool(rng, num, *, rows=6, width=9, block=4):
    """Requests of up to `width` blocks with ids of their own."""
    lens = rng.integers(0, width * block - 3, rows).astype(np.uint32)
    order = rng.permutation(num).astype(np.uint32)
    tables = np.full((rows, width), R.NONE, np.uint32)
    at = 0
    for r, n in enumerate(lens):
        c = R.blocks(int(n), block)
        tables[r, :c] = order[at:at + c]
        at += c
    return lens, tables, order, at


@pytest.mark.parametrize("seed", range(8))
def test_rewind_takes_back_what_fork_gave(seed):
    rng = np.random.default_rng(seed)
    lens, tables, free, taken = pool(rng, 80)
    lens[[1, 4]] = 0
    parents = np.full(6, R.NONE, np.uint32)
    parents[[1, 4]] = 0
    tables2, lens2, taken2, served, copies = R.fork(lens, parents, tables, free, taken, 4)
    assert served == 6 and len(copies) == (2 if lens[0] % 4 else 0) and taken2 == taken + len(copies)
    drop = np.where(parents == 0, R.NONE, 0).astype(np.uint32)
    tables3, lens3, free3, taken3, copies3 = R.rewind(lens2, drop, tables2, free, taken2, 4)
    assert taken3 == taken and np.array_equal(lens3, lens) and not copies3
    assert sorted(free3[taken3:]) == sorted(free[taken:])
    # all end: every block is free again
    end = np.full(6, R.NONE, np.uint32)
    _, lens4, free4, taken4, _ = R.rewind(lens2, end, tables2, free, taken2, 4)
    assert not lens4.any() and len(set(free4[taken4:])) == free4.size - taken4
    held = {b for r, n in enumerate(lens2) for b in R.held(tables2[r], n, 4)}
    assert set(free4[taken4:].tolist()) == held | set(free[taken2:].tolist())


def test_rewind_into_a_shared_block():
    tables = np.array([[5, 6, 7, 0], [5, 6, 1, 0], [5, 6, 2, 0]], np.uint32)
    lens = np.array([10, 11, 9], np.uint32)
    free = np.array([5, 6, 7, 1, 2, 3, 4, 0], np.uint32)
    # request 1 goes back into block 6, which 0 and 2 hold whole: it gets its own old third block
    t, n, f, top, copies = R.rewind(lens, np.array([0, 5, 0], np.uint32), tables, free, 5, 4)
    assert n.tolist() == [10, 6, 9] and copies == [(6, 1, 2)] and t[1].tolist() == [5, 1, 1, 0] and top == 5
    # all three: the last keeps it, and three blocks are free for two
    t, n, f, top, copies = R.rewind(lens, np.array([3, 5, 2], np.uint32), tables, free, 5, 4)
    assert n.tolist() == [7, 6, 7] and copies == [(6, 7, 3), (6, 1, 2)] and t[2, 1] == 6 and top == 4 and f[4] == 2
    # no block free: the rest of the block goes too
    tables[1, 2] = 9
    t, n, f, top, copies = R.rewind(lens, np.array([0, 5, 0], np.uint32), tables, free, 8, 4)
    assert n.tolist() == [10, 4, 9] and not copies and top == 8


@pytest.mark.parametrize("seed", range(8))
def test_compact_keeps_every_token(seed):
    rng = np.random.default_rng(seed)
    lens, tables, order, taken = pool(rng, 90)
    prefix = order[taken:taken + 3]
    t, p, count, copies = R.compact(lens, tables, prefix, 90, 4)
    cells = np.arange(90)
    moved = cells.copy()
    for a, b, _ in copies:
        moved[b] = cells[a]
    for r, n in enumerate(lens):
        assert [moved[b] for b in R.held(t[r], n, 4)] == R.held(tables[r], n, 4)
    assert np.array_equal(moved[p], prefix) and count == taken + 3
    assert max([b for r, n in enumerate(lens) for b in R.held(t[r], n, 4)] + p.tolist()) < count


@pytest.mark.parametrize("drafter", [True, False])
def test_verified_tokens_are_distributed_as_the_targets(drafter):
    """Summed over a grid of uniforms (and drafts as q draws them): the first token of the two has p's distribution, up to
    the grid's steps."""
    rng = np.random.default_rng(3)
    vocab, steps = 5, 200
    x, y = 2.0 * rng.standard_normal((2, vocab)), 2.0 * rng.standard_normal((2, vocab))
    setting, draft_setting = (0.8, 4, 1.0, 0.0), (1.1, 0, 0.9, 0.0)
    p = R.kept(x[0], *setting)[0]
    q = R.kept(y[0], *draft_setting)[0] if drafter else np.eye(vocab)[2]
    got = np.zeros(vocab)
    grid = (np.arange(steps) + 0.5) / steps
    for draft in np.flatnonzero(q):
        accept = R.kept(x[0], *setting)[0][draft]
        for u in grid:
            a, token, _ = R.verify(x, y if drafter else None, [0, draft], [u, 0.5], setting, draft_setting)
            assert (a == 1) == (u * q[draft] < accept)
            if a == 1:
                got[draft] += q[draft] / steps
            else:
                for v in grid[::10] - 0.5 / steps + 5 / steps:
                    got[R.verify(x, y if drafter else None, [0, draft], [u, v], setting, draft_setting)[1]] += q[draft] / steps / 20
    assert np.all(np.abs(got - p) <= 1 / steps + 1 / 20)   # a step of each grid
    assert np.all(got[p == 0] == 0)


def test_verify_closed_forms():
    x = np.log(np.array([[0.5, 0.25, 0.25, 1e-300]]))
    two = np.repeat(x, 2, 0)
    plain = (1.0, 0, 0.0, 0.0)
    # without a distribution: accepted below p, drawn from the others above
    assert R.verify(two, None, [9, 0], [0.4999, 0.0], plain, plain)[:2] == (1, 0)
    assert R.verify(two, None, [9, 0], [0.5001, 0.4], plain, plain)[:2] == (0, 1)
    assert R.verify(two, None, [9, 0], [0.5001, 0.6], plain, plain)[:2] == (0, 2)
    # the same distribution: always accepted, whatever the uniform
    assert R.verify(two, two, [9, 1], [0.99999, 0.8], plain, plain)[:2] == (1, 2)
    # a draft outside the vocabulary, one that the filters drop
    assert R.verify(two, two, [9, 77], [0.0, 0.1], plain, plain)[:2] == (0, 0)
    assert R.verify(two, two, [9, 2], [0.0, 0.9], (1.0, 2, 0.0, 0.0), plain)[:2] == (0, 1)
    # nothing to draw
    none = np.full((2, 4), -np.inf)
    assert R.verify(none, None, [9, 2], [0.0, 0.9], plain, plain) == (0, 0, [-np.inf])
