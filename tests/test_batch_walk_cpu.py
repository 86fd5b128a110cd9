"""The schedule of hyp_batch_attention (csrc/attention_batch_walk.h, compiled here with the host compiler and run a wave's
64 lanes at a time): over batches of every shape each worker's tiles stay inside the batch, a row's tiles hold every key
that it sees once, and the merge joins what the workers wrote of a row, all of it and nothing else."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

import hyperion_amd as hy

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# Query heads, kv heads and the kernel's workgroups' shares (wide_cost) of some forms.
FORMS = [(16, 8, 5.5), (16, 1, 2.0), (32, 8, 4.0), (12, 12, 3.0), (7, 1, 3.0), (6, 2, 4.0), (40, 2, 3.0)]


@pytest.fixture(scope="session")
def walk(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("walk") / "walk.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-U_FORTIFY_SOURCE", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "tests", "host_device"), "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "hyperion_amd", "csrc"), os.path.join(ROOT, "tests", "batch_walk_shim.cc"),
                    "-o", so], check=True)
    return ctypes.CDLL(so)


def check(walk, lens, row_start, H, KVH, cost, groups, block=16, prefix=0, window=0, max_blocks=None, spare_rows=0,
          max_rows=None, kinds=(True, False), ordered=True):
    n = len(lens)
    row_start = np.ascontiguousarray(row_start, np.uint32)
    lens = np.array(lens, np.uint32)
    if max_blocks is None:
        max_blocks = -(-int(lens.max(initial=0)) // block) + 1
    if max_rows is None:
        max_rows = int(row_start[-1]) + spare_rows
    tables = np.zeros(max(1, n * max_blocks), np.uint32)   # (only their addresses matter here)
    p = lambda a: a.ctypes.data  # noqa: E731
    fields = hy.BatchFields(n, block, 1 << 14, max_blocks, max_rows, prefix, p(tables), p(tables), p(lens), p(row_start),
                            None, None)
    for wide in kinds:
        message = ctypes.create_string_buffer(400)
        bad = walk.check_walk(ctypes.byref(fields), H, KVH, window, groups, ctypes.c_float(cost), int(wide), int(ordered),
                              message)
        assert not bad, (message.value.decode(), wide, lens.tolist(), row_start.tolist(), H, KVH, groups, block, prefix, window)


def starts(rows, first=0):
    return np.concatenate(([first], first + np.cumsum(rows)))


@pytest.mark.parametrize("lens,rows,form,groups,prefix,window", [
    ([0] * 70 + [40], [70] * 70 + [40], (8, 8, 3.0), 512, 0, 0),      # many rows of requests without keys
    ([0] * 70 + [40], [70] * 70 + [40], (8, 8, 3.0), 512, 20, 0),
    ([0, 300, 0], [256, 290, 127], (2, 2, 4.0), 16, 0, 0),            # and where rows fill tiles by themselves
    ([0, 300, 0], [256, 290, 127], (2, 2, 4.0), 16, 90, 50),
    ([3000] * 7 + [0] * 3, [100] * 7 + [40] * 3, (16, 8, 5.5), 512, 64, 0),
    ([9000], [1], (8, 1, 4.0), 768, 0, 0),                            # one request over all workers
    ([1], [1], (4, 1, 3.0), 512, 20000, 0),
    ([64, 300, 9], [60, 130, 9], (16, 1, 2.0), 256, 250, 0),
    ([700, 40], [300, 40], (4, 2, 5.5), 512, 500, 300),
    ([300, 300], [290, 290], (2, 2, 4.0), 64, 40, 1),
    ([50] * 70, [20] * 70, (2, 2, 4.0), 512, 30, 0),
    ([20], [1], (1, 1, 3.0), 4, 0, 0),
    ([], [], (4, 2, 3.0), 4, 50, 0),                                  # no requests
    ([5, 9], [0, 0], (4, 2, 3.0), 4, 50, 0),                          # none with rows
])
def test_schedules(walk, lens, rows, form, groups, prefix, window):
    check(walk, lens, starts(rows), *form, groups, prefix=prefix, window=window, spare_rows=3)


@pytest.mark.parametrize("seed", range(24))
def test_schedules_of_drawn_batches(walk, seed):
    rng = random.Random(seed)
    for _ in range(6):
        form = rng.choice(FORMS)
        n = rng.choice((1, 2, 3, 5, 9, 17, 64, 65, 130))
        top = rng.choice((3, 40, 400, 2500))
        most = rng.choice((1, 1, 3, 20, 90))
        lens = [rng.choice((0, 1, top, rng.randint(0, top), rng.randint(0, top))) for _ in range(n)]
        covered = rng.random() < 0.6        # lengths that hold their rows
        rows = [min(rng.randint(0, most), v) if covered else rng.randint(0, most) for v in lens]
        if sum(rows) == 0:
            rows[0], lens[0] = 1, max(lens[0], 1)
        block = rng.choice((1, 16, 64))
        check(walk, lens, starts(rows, rng.choice((0, 0, 0, 5))), *form, rng.choice((2, 7, 16, 40, 64)), block=block,
              prefix=rng.choice((0, 0, 1, rng.randint(1, 200), rng.randint(1, 3000))),
              window=rng.choice((0, 0, 1, rng.randint(1, 100), rng.randint(1, 2000))),
              max_blocks=rng.choice((None, None, None, 0, 2)), spare_rows=rng.choice((0, 7)))


@pytest.mark.parametrize("seed", range(6))
def test_schedules_of_large_batches(walk, seed):
    """The kernel's own numbers of workgroups."""
    rng = random.Random(100 + seed)
    form, groups = rng.choice((((16, 8, 5.5), 512), ((16, 1, 2.0), 256), ((32, 8, 4.0), 512), ((12, 12, 3.0), 512)))
    n, hi, most = rng.choice(((64, 1500, 1), (24, 330, 60), (96, 3000, 1), (40, 700, 9)))
    lens = [rng.randint(1, hi) for _ in range(n)]
    rows = [min(v, rng.randint(1, most)) for v in lens]
    check(walk, lens, starts(rows), *form, groups, prefix=rng.choice((0, 777, 6000)), window=rng.choice((0, 1024)),
          kinds=(True,) if rng.random() < 0.7 else (False,))


@pytest.mark.parametrize("row_start", [(0, 9, 3, 20, 5), (7, 3, 2, 1, 0), (0, 4000000000, 2, 9, 12), (0, 2, 4, 6, 99),
                                       (5, 6, 7, 8, 9), (0, 12, 0, 12, 12), (0, 300, 300, 300, 300), (299, 0, 299, 0, 300)])
def test_damaged_row_starts_stay_in_bounds(walk, row_start):
    for form in FORMS[:4]:
        for max_rows in (12, 300):
            check(walk, [30, 20, 9, 4000], np.array(row_start, np.uint32), *form, 16, prefix=20, max_blocks=4,
                  max_rows=max_rows, ordered=False)
