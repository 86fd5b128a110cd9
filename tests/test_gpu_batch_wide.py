"""hyp_batch_attention where many rows share keys, at the borders of its tiles, from several streams and far into a large
cache; hyp_batch_plan's large steps; hyp_sample_batch over long rows and many. Bars as test_gpu_batch.py's."""
import ctypes

import numpy as np
import pytest

import batch_ref as R
import hyperion_amd as hy
from hyperion_amd import synthetic as syn
from test_gpu_batch import Plan, Scene, check_draw, check_plan, dev, draw, f64, mixed, plan_case, say, u32

pytestmark = pytest.mark.gpu

SCENES = [
    # lens, rows, H, KVH, D, block, prefix, window, scale, spread
    ([64, 300, 9], [60, 130, 9], 16, 1, 512, 16, 250, 0, 1.0, 8.0),        # scores far apart: maxima grow late
    ([64, 300, 9], [60, 130, 9], 4, 2, 256, 16, 250, 0, 1.0, 8.0),
    ([64, 300, 9], [60, 130, 9], 4, 2, 64, 16, 250, 0, 1.0, 30.0),
    ([700, 40], [300, 40], 4, 2, 256, 16, 0, 200, 1.0, 2.0),               # a window over several wide tiles
    ([700, 40], [300, 40], 4, 2, 256, 16, 500, 300, 1.0, 2.0),             # and back into the prefix
    ([300, 300], [290, 290], 2, 2, 128, 16, 40, 1, None, 2.0),             # a row sees itself alone
    ([45, 3, 160], [45, 1, 77], 12, 4, 64, 16, 33, 0, None, 2.0),          # three heads a kv head
    ([45, 3, 160], [45, 1, 77], 10, 2, 128, 32, 100, 50, None, 2.0),       # five
    ([200, 1], [128, 1], 1, 1, 256, 16, 0, 0, None, 2.0),                  # a wide tile filled to its last row
    ([200, 1], [129, 1], 1, 1, 256, 16, 0, 0, None, 2.0),                  # and one row more
    ([31, 32, 33, 64], [16, 17, 1, 16], 2, 2, 128, 16, 32, 0, None, 2.0),  # the borders of the two kinds
    ([50] * 70, [20] * 70, 2, 2, 64, 16, 30, 0, None, 2.0),                # more requests with wide tiles than lanes
    ([30, 41] * 65, [9, 1] * 65, 8, 2, 64, 16, 0, 20, None, 2.0),
    ([60] + [1] * 24, [21] + [0] * 24, 4, 2, 64, 16, 0, 0, None, 2.0),     # one request has all rows of a decode step
    ([2000, 90], [3, 90], 8, 1, 128, 128, 3100, 0, None, 2.0),             # tiles split over many workers
    ([5] * 40, [1] * 40, 16, 1, 512, 16, 2500, 0, 1.0, 2.0),
    ([20, 20], [20, 20], 64, 1, 64, 16, 10, 0, None, 2.0),                 # 64 heads on one kv head
]


@pytest.mark.parametrize("lens,rows,H,KVH,D,block,prefix,window,scale,spread", SCENES)
def test_many_rows(stream, lens, rows, H, KVH, D, block, prefix, window, scale, spread):
    say(f"attention {len(lens)} requests H={H} KVH={KVH} D={D} prefix={prefix} window={window} spread={spread}")
    s = Scene(sum(lens) + D, stream, lens, rows, H, KVH, D, block, prefix, window, scale, extra_rows=2,
              spread=spread).place()
    s.run()
    first = s.check()
    s.run()
    assert np.array_equal(first, s.result())


def test_two_streams_at_once(stream):
    """Calls on two streams, each with its workspace, beside one another."""
    other = hy.Stream()
    scenes = [Scene(3, stream, [70, 200, 33], [70, 1, 33], 8, 2, 128, 16, 90, 0, None).place(),
              Scene(4, stream, [250] * 30, [1] * 30, 16, 8, 256, 16, 300, 100, 1.0).place()]
    stream.synchronize()
    for _ in range(5):
        for s, st in zip(scenes, (stream, other)):
            s.run(st)
    other.synchronize()
    for s in scenes:
        s.check("two streams")
    other.close()


def test_slots_behind_the_32nd_bit(stream):
    """A cache of more than 2^32 elements: appended to and read at its end."""
    H, KVH, D, block, n = 4, 1, 512, 1024, 300
    num = 2**23 // block + 3
    rng = np.random.default_rng(12)
    cache = hy.KvCache(num * block, KVH, D)
    slots = ((num - 1) * block + np.arange(n)).astype(np.uint32)
    assert int(slots[0]) * KVH * D >= 2**32
    bits = lambda *shape: syn.bf16_bits(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    q, k, v, one = bits(n, H, D), bits(n, KVH, D), bits(n, KVH, D), syn.bf16_bits(np.ones(D, np.float32))
    b = hy.Batch(block, num, dev(np.array([[num - 1]], np.uint32), stream), dev(u32(n), stream), dev(u32(0, n), stream),
                 dev(slots, stream), dev(np.arange(n, dtype=np.uint32), stream))
    d_q, d_out, d_one = dev(q, stream), dev(np.zeros_like(q), stream), dev(one, stream)
    b.prepare(d_q, dev(k, stream), dev(v, stream), H, cache, d_one, d_one, 1e-6, D, 1e4, d_q, stream)
    kv = []
    for ptr in cache.buffers():
        a = np.empty((n, KVH, D), np.uint16)
        hy.call("hyp_memcpy_dtoh", a.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(ptr.value + int(slots[0]) * KVH * D * 2),
                a.nbytes, stream.handle)
        stream.synchronize()
        kv.append(f64(a))
    ref = R.rope(R.rms(f64(k)), np.arange(n, dtype=np.uint32), D, 1e4)
    pair = np.abs(R.rms(f64(k))) + np.abs(np.roll(R.rms(f64(k)), D // 2, -1))
    assert np.all(np.abs(kv[0] - ref) <= 2.0**-8 * np.abs(ref) + 64 * 2.0**-24 * pair)
    work = dev(np.full(b.attention_workspace_bytes(H, cache), 0xFF, np.uint8), stream)
    b.attention(d_q, H, cache, 0, 1.0 / 16, d_out, work, stream)
    turned = f64(d_q.to_host(stream))
    want, size, apart = R.attention(turned, *kv, np.zeros((1, 1), np.uint32), u32(n), u32(0, n), block, 1, 0, u32(), 0, 1.0 / 16)
    score = (D / 32 + 8) * 2.0**-24 / 16 * size[..., None]
    bound = 2.0**-8 * np.abs(want) + np.max(np.abs(kv[1])) * (2.0**-15 + 2 * score) + 2.0**-8 * (1 + 2.0**-7) * apart
    assert np.all(np.abs(f64(d_out.to_host(stream)) - want) <= bound)
    cache.close()


@pytest.mark.parametrize("n,block,hi,new_hi,done,spare,short_rows", [
    (64, 16, 4000, 200, 0.1, 5, 0),       # one launch with thousands of rows
    (200, 16, 300, 400, 0.3, -900, 0),    # too few blocks, two launches
    (200, 1, 30, 300, 0.1, 5, 0),         # a block a token
    (200, 32, 300, 400, 0.2, 5, 9000),    # too few rows
    (4096, 8, 30, 40, 0.1, 5, 0),         # the most requests
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_of_many_rows(stream, n, block, hi, new_hi, done, spare, short_rows, in_place):
    say(f"plan n={n} block={block} hi={hi} new_hi={new_hi} in_place={in_place}")
    case = plan_case(n + block, n, block, hi, new_hi, done, spare, 3, short_rows)[:-1] + (41,)
    p = Plan(*case, stream, in_place=in_place)
    p.run()
    check_plan(p.results(), R.plan(*case))
    if not in_place:
        p.run()
        check_plan(p.results(), R.plan(*case))


@pytest.mark.parametrize("vocab", [2**22 + 5, 2**23])
def test_sample_rows_of_many_chunks(stream, vocab):
    """More chunks than a wave has lanes; the drawn value stands in many of them."""
    rng = np.random.default_rng(vocab)
    bits = syn.bf16_bits((0.5 * np.round(2.0 * rng.standard_normal((2, vocab)))).astype(np.float32))
    bits[1, ::5] = 0xFF80
    configs = mixed(rng, 2, vocab)
    configs["temperature"], configs["top_k"] = (1.0, 3.0), (0, 5000)
    for uniforms in ([0.37, 0.9], [0.99999, 1e-6]):
        check_draw(stream, bits, configs, np.array(uniforms, np.float32), f"vocab {vocab}")


def test_sample_rows_alone_and_among_more_than_the_device_holds(stream):
    """From 512 rows on a row is one workgroup's: the same tokens and bits of logprobs as a row alone."""
    rng = np.random.default_rng(3)
    rows, vocab = 530, 20001
    bits = syn.bf16_bits((3.0 * rng.standard_normal((rows, vocab))).astype(np.float32))
    bits[7, 100:400] = syn.bf16_bits(np.full(300, 200.0, np.float32))     # above the fine values
    bits[8, ::2] = syn.bf16_bits(np.full(10001, -300.0, np.float32))      # and below
    bits[9] = syn.bf16_bits((1e-9 * rng.standard_normal(vocab)).astype(np.float32))
    configs, uniforms = mixed(rng, rows, vocab), rng.random(rows).astype(np.float32)
    tokens, logprobs = draw(stream, bits, configs, uniforms)
    for r in (0, 7, 8, 9, 300, 529):
        one, value = draw(stream, bits[r:r + 1], configs[r:r + 1], uniforms[r:r + 1])
        assert one[0] == tokens[r] and value.view(np.uint32)[0] == logprobs.view(np.uint32)[r], r
