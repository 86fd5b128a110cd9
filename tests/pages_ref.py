"""Forked requests and verified drafts in numpy, in 64 bits: the references of test_pages_cpu.py,
test_gpu_pages.py and test_gpu_verify.py, written from the entry points' definitions."""
import numpy as np

from batch_ref import NONE, blocks  # noqa: F401


def held(table, tokens, block):
    """The entries of a row of tables that so many tokens take."""
    return [int(b) for b in table[:min(blocks(int(tokens), block), table.size)]]


def fork(lens, parents, tables, free, taken, block):
    """hyp_batch_fork, one copy after the other: tables, lens, taken, served, copies."""
    n, out, tables, copies, top = len(lens), lens.copy(), tables.copy(), [], int(taken)
    for r in range(n):
        p = int(parents[r])
        if p >= n or parents[p] != NONE:
            continue
        length = int(lens[p])
        whole = min(length // block, tables.shape[1])
        part = length % block if length // block < tables.shape[1] else 0
        if part and top == free.size:
            return tables, out, top, r, copies
        tables[r, :whole] = tables[p, :whole]
        if part:
            copies.append((int(tables[p, whole]), int(free[top]), part))
            tables[r, whole] = free[top]
            top += 1
        out[r] = length
    return tables, out, top, n, copies


def rewind(lens, drop, tables, free, taken, block):
    """hyp_batch_rewind: tables, lens, free, taken, copies; entries of free below the returned taken
    are not defined."""
    num, tables, free = free.size, tables.copy(), free.copy()
    keep = [int(n) - min(int(n), int(d)) for n, d in zip(lens, drop)]
    holders = {}
    for r, k in enumerate(keep):
        for b in held(tables[r], k, block):
            holders.setdefault(b, []).append(r)
    back = []
    for r, (n, k) in enumerate(zip(lens, keep)):
        for b in held(tables[r], n, block)[blocks(k, block):]:
            if b < num and b not in holders and b not in back:
                back.append(b)
    back = back[max(0, len(back) - int(taken)):]   # (a stack holds no more than was taken from it)
    top = int(taken) - len(back)
    free[top:int(taken)] = back
    cut = {}   # block -> the requests that were shortened into it
    for r, (n, k) in enumerate(zip(lens, keep)):
        if k < n and k % block and k // block < tables.shape[1]:
            cut.setdefault(int(tables[r, k // block]), []).append(r)
    copies = []
    for r, k in enumerate(keep):
        if not (k < lens[r] and k % block and k // block < tables.shape[1]):
            continue
        b = int(tables[r, k // block])
        if b >= num or (set(holders[b]) == set(cut[b]) and r == max(cut[b])):
            continue
        if top == num:
            keep[r] = k // block * block
            continue
        copies.append((b, int(free[top]), k % block))
        tables[r, k // block] = free[top]
        top += 1
    return tables, np.array(keep, np.uint32).reshape(len(lens)), free, top, copies


def compact(lens, tables, prefix_table, num, block):
    """hyp_batch_compact: tables, prefix table, the number of blocks in use, copies."""
    live = {b for r, n in enumerate(lens) for b in held(tables[r], n, block) if b < num}
    live |= {int(b) for b in prefix_table if b < num}
    movers = sorted(b for b in live if b >= len(live))
    holes = [b for b in range(len(live)) if b not in live]
    to = dict(zip(movers, holes))
    tables = tables.copy()
    for r, n in enumerate(lens):
        ids = held(tables[r], n, block)
        tables[r, :len(ids)] = [to.get(b, b) for b in ids]
    prefix = np.array([to.get(int(b), int(b)) for b in prefix_table], np.uint32)
    return tables, prefix, len(live), [(b, to[b], block) for b in movers]


def kept(logits, temperature, top_k, top_p, min_p):
    """One row of float values: the tokens' probabilities after the filters, ln of their shares before."""
    x = logits.astype(np.float64) + 0.0
    p, share = np.zeros(x.size), np.full(x.size, -np.inf)
    live = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
    if live.size == 0:
        return p, share
    order = live[np.argsort(-x[live], kind="stable")]
    v = x[order]
    greedy = not temperature > 0
    t = 1.0 if greedy else float(temperature)
    gap = np.where(v == np.inf, 0.0, -np.inf) if v[0] == np.inf else (v - v[0]) / t
    w = np.exp(gap)
    mass = np.cumsum(w)
    keep = v.size if top_k <= 0 else min(v.size, top_k)
    if 0 < top_p < 1:
        keep = min(keep, int(np.count_nonzero(mass - w < float(top_p) * mass[-1])))
    if min_p > 0:
        keep = min(keep, int(np.count_nonzero(w >= float(min_p))))
    keep = 1 if greedy else max(1, keep)
    p[order[:keep]] = w[:keep] / mass[keep - 1]
    share[order] = gap - np.log(mass[-1])
    return p, share


def uniform(u):
    return min(float(u), 1.0 - 2.0**-24) if u > 0 else 0.0


def verify(logits, draft_logits, ids, uniforms, setting, draft_setting):
    """hyp_verify_batch for one request's rows (float values): how many drafts are accepted, the next token,
    ln shares of the tokens that follow the rows up to it."""
    n, logs = len(ids), []
    for t in range(n):
        p, share = kept(logits[t], *setting)
        rest = p
        if t + 1 < n:
            x = int(ids[t + 1])
            if draft_logits is not None:
                q = kept(draft_logits[t], *draft_setting)[0]
            else:
                q = np.zeros(p.size)
                if x < p.size:
                    q[x] = 1.0
            if x < p.size and uniform(uniforms[t]) * q[x] < p[x]:
                logs.append(share[x])
                continue
            rest = np.maximum(0.0, p - q)
            if not rest.sum() > 0:
                rest = p
        if not rest.sum() > 0:
            return t, 0, logs + [-np.inf]
        running = np.cumsum(rest)
        token = int(np.count_nonzero(running <= uniform(uniforms[n - 1]) * running[-1]))
        token = min(token, int(np.flatnonzero(rest)[-1]))
        return t, token, logs + [share[token]]
