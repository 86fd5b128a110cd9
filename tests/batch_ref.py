"""Batched serving in numpy, in 64 bits: the references of test_batch_cpu.py and
test_gpu_batch.py, written from the entry points' definitions."""
import numpy as np

NONE = 0xFFFFFFFF
DONE = 0xFFFFFFFF


def blocks(tokens, size):
    return -(-tokens // size)


def plan(lens, new, tables, free, taken, block, max_rows, prefix):
    """hyp_batch_plan one request and one block at a time, as a list is walked. Returns tables,
    free, taken, served, lens, row_start, slots, positions; entries of free below the returned
    taken are not defined."""
    tables, free = tables.copy(), free.copy()
    num, max_blocks = free.size, tables.shape[1]
    back = [int(b) for r, (n, m) in enumerate(zip(lens, new)) if m == DONE
            for b in tables[r, :min(blocks(int(n), block), max_blocks)]][:int(taken)]
    top = int(taken) - len(back)
    free[top:int(taken)] = back
    out, start, slots, positions, served = [], [0], [], [], None
    for r, (n, m) in enumerate(zip(lens.tolist(), new.tolist())):
        if m == DONE:
            out.append(0)
            start.append(len(slots))
            continue
        have, need = blocks(n, block), blocks(n + m, block)
        if served is None and (len(slots) + m > max_rows or top + need - have > num or need > max_blocks or
                               prefix + n + m > 2**24):
            served = r
        if served is not None:
            out.append(n)
            start.append(len(slots))
            continue
        tables[r, have:need] = free[top:top + need - have]
        top += need - have
        for j in range(n, n + m):
            b = int(tables[r, j // block])
            slots.append(b * block + j % block if b < num else NONE)
            positions.append(prefix + j)
        out.append(n + m)
        start.append(len(slots))
    rest = max_rows - len(slots)
    return (tables, free, top, len(lens) if served is None else served, np.array(out, np.uint32),
            np.array(start, np.uint32), np.array(slots + [NONE] * rest, np.uint32),
            np.array(positions + [0] * rest, np.uint32))


def rms(x, weight=None, eps=1e-6):
    x = x.astype(np.float64)
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    return y if weight is None else y * weight.astype(np.float64)


def rope(x, positions, rotated, base):
    """x [rows, heads, d] float64; angles are float32 products, as hyp_rope defines them."""
    d = x.shape[-1]
    i = np.arange(rotated // 2)
    inv = (float(np.float32(base)) ** (-2.0 * i / d)).astype(np.float32)
    theta = (positions.astype(np.float32)[:, None] * inv).astype(np.float64)[:, None]
    y = x.copy()
    a, b = x[..., :rotated // 2], x[..., d // 2:d // 2 + rotated // 2]
    y[..., :rotated // 2] = a * np.cos(theta) - b * np.sin(theta)
    y[..., d // 2:d // 2 + rotated // 2] = a * np.sin(theta) + b * np.cos(theta)
    return y


def attention(q, ck, cv, tables, lens, row_start, block, num_blocks, prefix, prefix_table, window, scale):
    """hyp_batch_attention in float64, a row at a time: q [rows, H, D], ck / cv [slots, KVH, D] float64.
    Returns the output, for each row the largest sum |q||k| over its keys (for the error of its scores),
    and the weighted mean distance of its values from the output (for the error of its weights). NaN of
    keys that a row does not see is never touched."""
    rows, H, D = q.shape
    KVH = ck.shape[1]
    G = H // KVH
    out, size, apart = np.zeros(q.shape), np.zeros((rows, H)), np.zeros(q.shape)
    shared = [(j, int(prefix_table[j // block]) * block + j % block) for j in range(prefix)
              if prefix_table[j // block] < num_blocks]
    for r, n in enumerate(lens):
        t0, t1 = int(row_start[r]), int(row_start[r + 1])
        if t0 == t1:
            continue
        n = min(int(n), tables.shape[1] * block)
        own = [(prefix + j, int(tables[r, j // block]) * block + j % block) for j in range(n)
               if tables[r, j // block] < num_blocks]
        keys = np.array(shared + own, np.int64).reshape(-1, 2)
        for t in range(t0, t1):
            pos = prefix + n - (t1 - t0) + (t - t0)
            seen = keys[:, 0] <= pos
            if window:
                seen &= keys[:, 0] > pos - window
            at = keys[seen, 1]
            if at.size == 0:
                continue
            k, v = ck[at], cv[at]
            for h in range(H):
                s = scale * (k[:, h // G] @ q[t, h])
                size[t, h] = np.max(np.abs(k[:, h // G]) @ np.abs(q[t, h]), initial=0.0)
                m = np.max(s)
                if m == -np.inf:
                    continue
                w = np.exp(s - m)
                live = w != 0
                out[t, h] = (w[live] @ v[live, h // G]) / w.sum()
                apart[t, h] = (w[live] @ np.abs(v[live, h // G] - out[t, h])) / w.sum()
    return out, size, apart


def sample(logits, temperature, top_k, top_p, min_p, u):
    """hyp_sample_batch of one row of float values, in float64: (token, logprob)."""
    x = logits.astype(np.float64) + 0.0
    live = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
    if live.size == 0:
        return 0, -np.inf
    order = live[np.argsort(-x[live], kind="stable")]
    v = x[order]
    greedy = not temperature > 0
    t = 1.0 if greedy else float(temperature)
    w = (v == np.inf).astype(np.float64) if v[0] == np.inf else np.exp((v - v[0]) / t)
    mass = np.cumsum(w)
    keep = v.size if top_k <= 0 else min(v.size, top_k)
    if 0 < top_p < 1:
        keep = min(keep, int(np.count_nonzero(mass - w < float(top_p) * mass[-1])))
    if min_p > 0:
        keep = min(keep, int(np.count_nonzero(w >= float(min_p))))
    keep = 1 if greedy else max(1, keep)
    goal = (min(float(u), 1.0 - 2.0**-24) if u > 0 else 0.0) * mass[keep - 1]
    j = min(int(np.count_nonzero(mass[:keep] <= goal)), keep - 1)
    return int(order[j]), float(np.log(w[j] / mass[-1])) if w[j] > 0 else -np.inf
