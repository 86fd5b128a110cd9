"""Batched serving without a GPU: what the entry points refuse before they touch a device, and
the references of test_gpu_batch.py against closed forms."""
import ctypes

import numpy as np
import pytest

import batch_ref as R
import hyperion_amd as hy

INVALID, UNSUPPORTED = 1, 5


def handle(magic, *words):
    """Host memory that opens like one of the library's handles: its magic, then `words`."""
    mem = (ctypes.c_uint32 * 64)(magic, *words)
    return mem, ctypes.c_void_p(ctypes.addressof(mem))


STREAM_MEM, STREAM = handle(0x48505354)
CACHE_MEM, CACHE = handle(0x48504B56, 64 * 16, 2, 128)   # capacity, KV heads, head_dim
P = ctypes.c_void_p(0x1000)                              # an aligned address that no refused call reads


def fields(**over):
    f = hy.BatchFields(requests=4, block_size=16, num_blocks=64, max_blocks=8, max_rows=32, prefix_len=20,
                       prefix_table=0x1000, tables=0x1000, lens=0x1000, row_start=0x1000, slots=0x1000,
                       positions=0x1000)
    for k, v in over.items():
        setattr(f, k, v)
    return f


def refused(name, *args, status=INVALID, says=""):
    got = getattr(hy.lib(), name)(*args)
    assert got == status, (got, hy.last_error())
    assert says in hy.last_error(), hy.last_error()


BAD_BATCHES = [
    (dict(requests=4097), "4096 requests"),
    (dict(block_size=0), "power of two"),
    (dict(block_size=24), "power of two"),
    (dict(block_size=131072), "power of two"),
    (dict(num_blocks=0), "positive"),
    (dict(num_blocks=1 << 26), "below 2^30"),
    (dict(max_rows=(1 << 20) + 1), "2^20 rows"),
    (dict(prefix_len=(1 << 24) + 1), "2^24"),
    (dict(tables=None), "tables"),
    (dict(lens=None), "lens"),
    (dict(row_start=None), "row_start"),
]


def plan_args(b, **over):
    a = dict(lens=P, new=P, free=P, taken=P, taken_out=P, served=P, stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), a["lens"], a["new"], a["free"], a["taken"], a["taken_out"], a["served"], a["stream"])


def prepare_args(b, **over):
    a = dict(q=P, k=P, v=P, heads=4, cache=CACHE, qn=P, kn=P, eps=1e-6, rotated=128, base=1e4, out=P, stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), a["q"], a["k"], a["v"], a["heads"], a["cache"], a["qn"], a["kn"], a["eps"], a["rotated"],
            a["base"], a["out"], a["stream"])


def attention_args(b, **over):
    a = dict(q=P, heads=4, cache=CACHE, window=0, scale=1.0, out=P, work=P, bytes=1 << 40, stream=STREAM)
    a.update(over)
    return (ctypes.byref(b), a["q"], a["heads"], a["cache"], a["window"], a["scale"], a["out"], a["work"], a["bytes"],
            a["stream"])


@pytest.mark.parametrize("over,says", BAD_BATCHES)
def test_bad_batches_are_refused_by_every_call(over, says):
    b = fields(**over)
    refused("hyp_batch_plan", *plan_args(b), says=says)
    refused("hyp_batch_prepare", *prepare_args(b), says=says)
    refused("hyp_batch_attention", *attention_args(b), says=says)
    refused("hyp_batch_attention_workspace", ctypes.byref(b), 4, CACHE, ctypes.byref(ctypes.c_size_t()), says=says)


@pytest.mark.parametrize("over", [dict(lens=None), dict(new=None), dict(free=None), dict(taken=None),
                                  dict(taken_out=None), dict(served=None), dict(stream=None)])
def test_plan_refusals(over):
    refused("hyp_batch_plan", *plan_args(fields(), **over), says="null")
    refused("hyp_batch_plan", None, *plan_args(fields())[1:], says="batch is null")
    refused("hyp_batch_plan", *plan_args(fields(slots=None)), says="slots")


@pytest.mark.parametrize("over,says", [
    (dict(q=None), "non-null"), (dict(k=None), "non-null"), (dict(qn=None), "non-null"), (dict(kn=None), "non-null"),
    (dict(out=None), "non-null"), (dict(q=ctypes.c_void_p(0x1002)), "aligned"), (dict(v=ctypes.c_void_p(0x1008)), "aligned"),
    (dict(out=ctypes.c_void_p(0x1004)), "aligned"), (dict(heads=0), "multiple"), (dict(heads=5), "multiple"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(rotated=130), "rotated"), (dict(rotated=7), "rotated"),
    (dict(base=0.0), "rope_base"), (dict(base=float("inf")), "rope_base"), (dict(cache=None), "null"),
    (dict(cache=STREAM), "magic"), (dict(stream=CACHE), "magic")])
def test_prepare_refusals(over, says):
    refused("hyp_batch_prepare", *prepare_args(fields(), **over), says=says)


@pytest.mark.parametrize("over,says", [
    (dict(q=None), "non-null"), (dict(out=None), "non-null"), (dict(work=None), "non-null"),
    (dict(q=ctypes.c_void_p(0x1002)), "aligned"), (dict(out=ctypes.c_void_p(0x1008)), "aligned"),
    (dict(work=ctypes.c_void_p(0x1004)), "aligned"), (dict(heads=0), "multiple"), (dict(heads=3), "multiple"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(heads=1026), "1024"), (dict(bytes=1000), "workspace too small"),
    (dict(cache=None), "null"), (dict(stream=None), "null")])
def test_attention_refusals(over, says):
    refused("hyp_batch_attention", *attention_args(fields(), **over), says=says)


def workspace(b, heads=4):
    out = ctypes.c_size_t()
    assert hy.lib().hyp_batch_attention_workspace(ctypes.byref(b), heads, CACHE, ctypes.byref(out)) == 0, hy.last_error()
    return out.value


def test_attention_workspace_is_what_the_call_asks_for():
    b = fields()
    need = workspace(b)
    refused("hyp_batch_attention", *attention_args(b, bytes=need - 1), says="too small")
    assert workspace(fields(max_rows=64)) > need > workspace(fields(prefix_len=0))
    refused("hyp_batch_attention_workspace", ctypes.byref(b), 4, CACHE, None, says="out_bytes")


def test_attention_refuses_what_its_counters_do_not_hold():
    b = fields(num_blocks=16, block_size=64, max_blocks=1 << 24, max_rows=1 << 20)
    refused("hyp_batch_attention", *attention_args(b, bytes=1 << 60), says="too many rows")


def test_a_pool_beyond_the_cache_is_refused():
    refused("hyp_batch_prepare", *prepare_args(fields(num_blocks=65)), says="must hold")
    refused("hyp_batch_attention", *attention_args(fields(num_blocks=65)), says="must hold")
    refused("hyp_batch_attention", *attention_args(fields(prefix_table=None)), says="prefix_table")
    refused("hyp_batch_prepare", *prepare_args(fields(max_rows=1 << 20), heads=32), says="too large")


def test_binding_checks_the_arrays():
    class Fake:
        def __init__(self, *shape):
            self.shape, self.ptr = shape, P

    good = [Fake(3, 4), Fake(3), Fake(4), Fake(7), Fake(7)]
    hy.Batch(16, 8, *good)
    for i, bad in ((1, Fake(4)), (2, Fake(3)), (4, Fake(8))):
        with pytest.raises(ValueError):
            hy.Batch(16, 8, *(bad if k == i else a for k, a in enumerate(good)))
    with pytest.raises(ValueError):
        hy.Batch(16, 8, *good, prefix_len=33, prefix_table=Fake(2))


def test_plan_reference_walks_blocks_as_defined():
    tables = np.array([[7, 9, R.NONE], [5, R.NONE, R.NONE], [3, 4, R.NONE]], np.uint32)
    free = np.array([100, 100, 100, 100, 100, 2, 1, 0, 6, 8], np.uint32)
    t, f, top, served, lens, start, slots, pos = R.plan(
        np.array([5, 4, 8], np.uint32), np.array([4, R.DONE, 1], np.uint32), tables, free, 5, 4, 8, 100)
    # request 1's block 5 returns as entry 4 and is dealt first, to request 0
    assert top == 6 and served == 3 and t[0].tolist() == [7, 9, 5] and t[2].tolist() == [3, 4, 2]
    assert lens.tolist() == [9, 0, 9] and start.tolist() == [0, 4, 4, 5]
    assert slots.tolist() == [37, 38, 39, 20, 8, R.NONE, R.NONE, R.NONE]
    assert pos.tolist() == [105, 106, 107, 108, 108, 0, 0, 0]


def test_rope_reference_turns_pairs():
    x = np.zeros((1, 1, 8))
    x[0, 0, 1] = 1.0
    y = R.rope(x, np.array([3]), 8, 100.0)
    theta = float(np.float32(3) * np.float32(100.0 ** -0.25))
    assert np.allclose(y[0, 0, [1, 5]], [np.cos(theta), np.sin(theta)], atol=1e-15)
    assert np.array_equal(R.rope(x, np.array([3]), 2, 100.0), x)   # pair 1 lies past the rotated dims


def sample_args(**over):
    a = dict(logits=P, rows=3, vocab=1000, configs=P, uniforms=P, tokens=P, logprobs=P, work=P, bytes=1 << 40, stream=STREAM)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over,says", [
    (dict(logits=None), "logits"), (dict(configs=None), "configs"), (dict(uniforms=None), "uniforms"),
    (dict(tokens=None), "tokens"), (dict(vocab=(1 << 23) + 1), "2^23"), (dict(rows=(1 << 20) + 1), "2^20"),
    (dict(configs=ctypes.c_void_p(0x1004)), "aligned"), (dict(work=ctypes.c_void_p(0x1008)), "aligned"),
    (dict(stream=None), "null"), (dict(stream=CACHE), "magic")])
def test_sample_refusals(over, says):
    refused("hyp_sample_batch", *sample_args(**over), says=says)


def test_sample_workspace_is_what_the_call_asks_for():
    for rows, vocab in ((1, 262144), (64, 262144), (300, 262144), (2, 100)):
        need = hy.sample_batch_workspace_bytes(rows, vocab)
        if need:
            refused("hyp_sample_batch", *sample_args(rows=rows, vocab=vocab, bytes=need - 1), says="too small")
            refused("hyp_sample_batch", *sample_args(rows=rows, vocab=vocab, work=None), says="too small")
    refused("hyp_sample_batch_workspace", 1, 10, None, says="out_bytes")
    refused("hyp_sample_batch_workspace", 1, (1 << 23) + 1, ctypes.byref(ctypes.c_size_t()), says="2^23")
    assert hy.lib().hyp_sample_batch(None, 0, 0, None, None, None, None, None, 0, STREAM) == 0   # no rows: nothing to do


def test_sample_reference_closed_forms():
    x = np.log(np.array([0.1, 0.4, 0.1, 0.4]))
    for u, token in ((0.0, 1), (0.39, 1), (0.41, 3), (0.79, 3), (0.81, 0), (0.91, 2), (0.999, 2), (1.0, 2)):
        assert R.sample(x, 1.0, 0, 0.0, 0.0, u)[0] == token       # value descending, then index ascending
    assert R.sample(x, 0.0, 0, 0.0, 0.0, 0.9) == (1, pytest.approx(np.log(0.4)))
    assert R.sample(x, 1.0, 3, 0.0, 0.0, 0.95)[0] == 0            # 0.4, 0.4, 0.1 kept
    assert R.sample(x, 1.0, 0, 0.79, 0.0, 0.99)[0] == 3           # the nucleus ends with the token that reaches it
    assert R.sample(x, 1.0, 0, 0.0, 0.3, 0.99)[0] == 3
    assert R.sample(np.array([-np.inf, np.nan]), 1.0, 0, 0.0, 0.0, 0.5) == (0, -np.inf)
    assert R.sample(np.array([3.0, np.inf, np.inf]), 1.0, 0, 0.0, 0.0, 0.7) == (2, pytest.approx(np.log(0.5)))


AT = 0x10000000   # an address of its own
Q_BYTES, KV_BYTES = 32 * 4 * 128 * 2, 32 * 2 * 128 * 2   # fields()' arrays


@pytest.mark.parametrize("over,says", [
    (dict(q=P, k=AT, v=2 * AT, out=AT), "k_raw or v_raw"),
    (dict(q=P, k=AT, v=2 * AT, out=AT + KV_BYTES - 16), "k_raw or v_raw"),
    (dict(q=P, k=AT, v=2 * AT, out=2 * AT - Q_BYTES + 16), "k_raw or v_raw"),
    (dict(q=AT, k=2 * AT, v=None, out=AT + 16), "must be q or not overlap"),
])
def test_prepare_refuses_outputs_over_its_inputs(over, says):
    refused("hyp_batch_prepare", *prepare_args(fields(), **over), says=says)


@pytest.mark.parametrize("over", [
    dict(q=AT, out=AT, work=2 * AT),
    dict(q=AT, out=AT + Q_BYTES - 16, work=2 * AT),
    dict(q=AT, out=2 * AT, work=AT + Q_BYTES - 16),
    dict(q=AT, out=2 * AT, work=2 * AT - 16),
])
def test_attention_refuses_arrays_over_each_other(over):
    refused("hyp_batch_attention", *attention_args(fields(), **over), says="must not overlap")


@pytest.mark.parametrize("over,says", [
    (dict(logits=AT + 1), "2-byte"), (dict(uniforms=AT + 2), "4-byte"), (dict(tokens=AT + 1), "4-byte"),
    (dict(logprobs=AT + 2), "4-byte"),
])
def test_sample_refuses_odd_addresses(over, says):
    refused("hyp_sample_batch", *sample_args(**over), says=says)
