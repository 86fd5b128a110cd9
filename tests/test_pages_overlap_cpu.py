"""hyp_batch_copy refuses a list that lies in the memory of a cache it writes, before it touches a device."""
import ctypes

import pytest

from test_batch_cpu import handle, refused
from test_pages_cpu import A, batch, copy_args

CELLS = 64 * 16                     # tokens of the batch's pool and of the caches
BYTES = CELLS * 2 * 128 * 2


def cache(k, v):
    """A cache's handle: magic, capacity, KV heads, head dim, then K and V as address and bytes."""
    words = [w for at in (k, v) for w in (at & 0xFFFFFFFF, at >> 32, BYTES, 0)]
    return handle(0x48504B56, CELLS, 2, 128, *words)


FIRST_MEM, FIRST = cache(0x10000000, 0x20000000)
SECOND_MEM, SECOND = cache(0x30000000, 0x40000000)


@pytest.mark.parametrize("start", [0x10000000, 0x20000000, 0x30000000, 0x40000000])
@pytest.mark.parametrize("at", [0, BYTES // 2, BYTES - 4, -4])
def test_lists_within_a_cache_are_refused(start, at):
    inside = ctypes.c_void_p(start + at)
    refused("hyp_batch_copy", *copy_args(batch(), (FIRST, SECOND), copies=inside), says="overlap")
    if at >= 0:
        refused("hyp_batch_copy", *copy_args(batch(), (FIRST, SECOND), n_copies=inside), says="overlap")


def test_lists_beside_a_cache_go_on():
    """Up to the first byte and from behind the last: the call goes on to the next cache, which is none."""
    for copies, n in ((0x10000000 - 12 * 8, 0x10000000 + BYTES), (0x20000000 + BYTES, 0x20000000 - 4)):
        refused("hyp_batch_copy", *copy_args(batch(), (FIRST, SECOND, None), copies=ctypes.c_void_p(copies),
                                             n_copies=ctypes.c_void_p(n)), says="null")
    refused("hyp_batch_copy", *copy_args(batch(), (FIRST, FIRST, None), copies=A[0]), says="null")
