"""Batched serving at the ends of what its calls define. Bars as test_gpu_batch.py's."""
import pytest

from test_gpu_batch import Scene, say

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
