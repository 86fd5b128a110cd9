"""Speculative decoding and forked requests as a program runs them: drafts drawn from a small model, verified beside each other
over the paged caches, the ones that fall rewound; requests forked into several answers, ended, the pool compacted.
The host keeps its own account of tables, lengths and of every token's K and V."""
import numpy as np
import pytest

import hyperion_amd as hy
import pages_ref as R
from hyperion_amd import synthetic as syn
from test_gpu_batch import CONFIG, dev, read_cache, say, u32
from test_gpu_batch_serving import HIDDEN, VOCAB, Server

pytestmark = pytest.mark.gpu

DRAFTS = 3


class Speculator:
    """What the program keeps beside the server's arrays: the drafting model (a head on the embedding), the arrays of a
    verification and of the calls on blocks."""

    def __init__(self, sv, step):
        s, n, rows = sv.stream, sv.host["lens"].size, step.rows
        self.sv, self.rows, self.n = sv, rows, n
        self.head = hy.QWeight.from_host(*syn.q4_weights(VOCAB, HIDDEN, seed=77))
        self.x, self.last = dev(np.zeros((n, HIDDEN), np.uint16), s), dev(np.zeros(n, np.uint32), s)
        self.guess = [dev(np.zeros((n, VOCAB), np.uint16), s) for _ in range(DRAFTS)]
        self.drawn = [dev(np.zeros(n, np.uint32), s) for _ in range(DRAFTS)]
        self.configs, self.uniforms = dev(np.zeros(n, CONFIG), s), dev(np.zeros(n, np.float32), s)
        self.sample_work = dev(np.zeros(max(16, hy.sample_batch_workspace_bytes(n, VOCAB)), np.uint8), s)
        self.draft_logits = dev(np.zeros((rows, VOCAB), np.uint16), s)
        self.ids, self.row_uniforms = dev(np.zeros(rows, np.uint32), s), dev(np.zeros(rows, np.float32), s)
        self.accepted, self.rejected, self.tokens = (dev(np.zeros(n, np.uint32), s) for _ in range(3))
        self.logprobs = dev(np.zeros(rows, np.float32), s)
        self.verify_work = dev(np.full(hy.verify_batch_workspace_bytes(rows, VOCAB, n, True), 0xFF, np.uint8), s)
        self.parents, self.served = dev(np.full(n, R.NONE, np.uint32), s), dev(u32(0), s)
        self.copies, self.n_copies = dev(np.zeros((max(n, sv.num // 2), 3), np.uint32), s), dev(u32(0), s)
        self.work = dev(np.full(step.batch.pages_workspace_bytes(), 0xEE, np.uint8), s)
        self.graph = None

    def draft(self, last, settings, rng):
        """DRAFTS tokens behind `last` for every slot, one after the other, and the logits that each was drawn from."""
        s = self.sv.stream
        self.configs.upload(settings, s)
        self.last.upload(last, s)
        at = self.last
        for j in range(DRAFTS):
            self.uniforms.upload(rng.random(self.n).astype(np.float32), s)
            hy.embed(self.sv.table, at, self.n, self.x, s)
            hy.qmatmul(self.head, self.x, self.n, self.guess[j], s, softcap=30.0)
            hy.sample_batch(self.guess[j], self.n, VOCAB, self.configs, self.uniforms, self.drawn[j], None, self.sample_work, s)
            at = self.drawn[j]
        s.synchronize()
        return [d.to_host(s) for d in self.drawn], [g.to_host(s) for g in self.guess]

    def judge(self, step):
        """Verify the step's rows, drop what fell, copy what that leaves shared: calls that a graph records."""
        sv, s = self.sv, self.sv.stream
        hy.verify_batch(step.logits, self.draft_logits, self.rows, VOCAB, sv.row_start, self.n, self.ids, self.configs, None,
                        self.row_uniforms, self.accepted, self.rejected, self.tokens, self.logprobs, self.verify_work, s)
        step.batch.rewind(sv.lens, self.rejected, sv.free, sv.taken, sv.taken, self.copies, self.n_copies, self.work, s)
        step.batch.copy([la.cache for la in sv.layers], self.copies, self.n_copies, s)


class Account:
    """Every token's K and V of each request, as they were stored."""

    def __init__(self, sv):
        self.sv = sv
        self.kv = [[] for _ in range(sv.host["lens"].size)]   # per request, per token: (K, V) of every layer

    def cells(self):
        sv = self.sv
        return [read_cache(la.cache, (sv.num * sv.block, la.KVH, la.D), sv.stream) for la in sv.layers]

    def slots(self, r):
        h, j = self.sv.host, np.arange(int(self.sv.host["lens"][r]))
        return h["tables"][r, j // self.sv.block].astype(np.int64) * self.sv.block + j % self.sv.block

    def append(self):
        cells = self.cells()
        for r in range(len(self.kv)):
            at = self.slots(r)
            for j in range(len(self.kv[r]), at.size):
                self.kv[r].append([(k[at[j]].copy(), v[at[j]].copy()) for k, v in cells])

    def check(self, what):
        cells = self.cells()
        for r, tokens in enumerate(self.kv):
            at = self.slots(r)
            assert at.size == len(tokens), (what, r)
            for j, mine in zip(at, tokens):
                for (k, v), (mk, mv) in zip(cells, mine):
                    assert np.array_equal(k[j], mk) and np.array_equal(v[j], mv), (what, r, j)


def serve(stream, from_graph):
    rng = np.random.default_rng(123)
    n = 8
    sv = Server(stream, n, 16, 90, 8, 37)
    h = sv.host
    prompts, step = sv.step_of(120), sv.step_of(n * (1 + DRAFTS))
    sp, account = Speculator(sv, step), Account(sv)
    lens_of = lambda: sv.lens.to_host(stream)  # noqa: E731

    def same(what):
        assert np.array_equal(lens_of(), h["lens"]) and int(sv.taken.to_host(stream)[0]) == h["taken"], what
        assert np.array_equal(sv.tables.to_host(stream), h["tables"]), what
        assert np.array_equal(sv.free.to_host(stream)[h["taken"]:], h["free"][h["taken"]:]), what
        account.check(what)

    def prompt(lengths):
        new = np.array(lengths, np.uint32)
        tokens, start = prompts.run(new, rng.integers(0, VOCAB, new.sum()), rng)
        account.append()
        for r in np.flatnonzero(new):
            last[r] = tokens[start[r + 1] - 1]
        same("prompt")

    def rewound(drop, what):
        h["tables"], h["lens"], free, h["taken"], copies = R.rewind(h["lens"], drop, h["tables"], h["free"], h["taken"], 16)
        h["free"][h["taken"]:] = free[h["taken"]:]
        for r in range(n):
            del account.kv[r][int(h["lens"][r]):]
        same(what)
        return copies

    def end(which):
        drop = np.zeros(n, np.uint32)
        drop[which] = hy.REQUEST_DONE
        sv.new.upload(drop, stream)
        step.batch.rewind(sv.lens, sv.new, sv.free, sv.taken, sv.taken, sp.copies, sp.n_copies, sp.work, stream)
        assert not rewound(drop, "end")

    def fork(parents):
        p = np.full(n, R.NONE, np.uint32)
        for r, of in parents.items():
            p[r] = of
            last[r] = last[of]
            account.kv[r] = list(account.kv[of])
        sp.parents.upload(p, stream)
        step.batch.fork(sv.lens, sp.parents, sv.free, sv.taken, sv.taken, sp.served, sp.copies, sp.n_copies, stream)
        step.batch.copy([la.cache for la in sv.layers], sp.copies, sp.n_copies, stream)
        h["tables"], h["lens"], h["taken"], served, copies = R.fork(h["lens"], p, h["tables"], h["free"], h["taken"], 16)
        assert served == n and int(sp.served.to_host(stream)[0]) == n
        same("fork")

    def rewind_into(drop):
        sv.new.upload(drop, stream)
        step.batch.rewind(sv.lens, sv.new, sv.free, sv.taken, sv.taken, sp.copies, sp.n_copies, sp.work, stream)
        step.batch.copy([la.cache for la in sv.layers], sp.copies, sp.n_copies, stream)
        return rewound(drop, "rewind")

    def compact():
        step.batch.compact(sv.tables, sv.d_prefix, sv.free, sv.taken, sp.copies, sp.n_copies, sp.work, stream)
        step.batch.copy([la.cache for la in sv.layers], sp.copies, sp.n_copies, stream)
        h["tables"], sv.prefix_table, h["taken"], copies = R.compact(h["lens"], h["tables"], sv.prefix_table, sv.num, 16)
        h["free"][h["taken"]:] = np.arange(h["taken"], sv.num)
        assert np.array_equal(sv.d_prefix.to_host(stream), sv.prefix_table)
        same("compact")
        return copies

    last = np.zeros(n, np.uint32)
    log = []
    prompt([1, 40, 17, 0, 33, 0, 0, 16])
    for at in range(9):
        if at == 2:
            fork({3: 1, 5: 1, 6: 2})
        if at == 4:
            end([1, 4])
        if at == 5:
            prompt([0, 7, 0, 0, 21, 0, 0, 0])
            drop = np.zeros(n, np.uint32)
            drop[5] = h["lens"][5] - 20   # back into what it has in common with request 3
            assert rewind_into(drop)
        if at == 6:
            assert compact()
        live = h["lens"] > 0
        settings = np.zeros(n, CONFIG)
        settings["temperature"] = rng.choice([0.0, 0.6, 1.0], n)
        settings["top_k"], settings["top_p"] = rng.choice([0, 5, 50], n), rng.choice([0.0, 0.8], n)
        drawn, guess = sp.draft(last, settings, rng)
        new = np.where(live, 1 + rng.integers(0, DRAFTS + 1, n), 0).astype(np.uint32)
        ids, rows_guess = [], np.zeros((step.rows, VOCAB), np.uint16)
        for r in range(n):
            for j in range(int(new[r])):
                if j + 1 < new[r]:
                    rows_guess[len(ids)] = guess[j][r]   # what the next row's token was drawn from
                ids.append(last[r] if j == 0 else drawn[j - 1][r])
        step.run(new, ids, rng)   # plan, layers, LM head, all checked
        account.append()
        all_ids = np.zeros(step.rows, np.uint32)
        all_ids[:len(ids)] = ids
        u = rng.random(step.rows).astype(np.float32)
        for a, v in ((sp.draft_logits, rows_guess), (sp.ids, all_ids), (sp.row_uniforms, u)):
            a.upload(v, stream)
        if from_graph and at == 0:
            with hy.Graph.capture(stream) as sp.graph:
                sp.judge(step)
        if sp.graph is not None:
            sp.graph.launch(stream)
        else:
            sp.judge(step)
        stream.synchronize()
        start = np.concatenate(([0], np.cumsum(new)))
        logits = syn.bf16_to_f32(step.logits.to_host(stream)).reshape(step.rows, VOCAB)
        drafted = syn.bf16_to_f32(rows_guess).reshape(step.rows, VOCAB)
        accepted, rejected, tokens = (a.to_host(stream) for a in (sp.accepted, sp.rejected, sp.tokens))
        for r in np.flatnonzero(new):
            rows = slice(int(start[r]), int(start[r + 1]))
            c = settings[r]
            setting = (float(c["temperature"]), int(c["top_k"]), float(c["top_p"]), float(c["min_p"]))
            a, token, _ = R.verify(logits[rows], drafted[rows], all_ids[rows], u[rows], setting, setting)
            assert (accepted[r], rejected[r], tokens[r]) == (a, new[r] - 1 - a, token), (at, r)
            last[r] = token
        assert not rewound(np.where(new > 0, rejected, 0).astype(np.uint32), ("step", at))
        log.append((accepted.copy(), last.copy(), h["lens"].copy()))
    if sp.graph is not None:
        sp.graph.close()
    assert sum(int(a.sum()) for a, _, _ in log) > 0   # some drafts stood
    return log


def test_drafts_forks_and_rewinds(stream):
    say("speculative decoding, eager and from a graph")
    for a, b in zip(serve(stream, False), serve(stream, True)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))


def test_ends_without_rows_give_zeroes(stream):
    """A step in which nobody has rows: no draft, nothing dropped."""
    say("speculative decoding: no rows")
    n, vocab = 5, 700
    ids = dev(np.zeros(4, np.uint32), stream)
    logits = dev(np.zeros((4, vocab), np.uint16), stream)
    out = [dev(np.full(n, 7, np.uint32), stream) for _ in range(3)]
    work = dev(np.zeros(hy.verify_batch_workspace_bytes(4, vocab, n, False), np.uint8), stream)
    hy.verify_batch(logits, None, 4, vocab, dev(np.zeros(n + 1, np.uint32), stream), n, ids, dev(np.zeros(n, CONFIG), stream), None,
                    dev(np.zeros(4, np.float32), stream), *out, None, work, stream)
    accepted, rejected, tokens = (o.to_host(stream) for o in out)
    assert not accepted.any() and not rejected.any() and np.all(tokens == 7)
    hy.verify_batch(logits, None, 0, vocab, dev(np.zeros(n + 1, np.uint32), stream), n, ids, dev(np.zeros(n, CONFIG), stream), None,
                    dev(np.zeros(4, np.float32), stream), *out, None, work, stream)
    assert not out[0].to_host(stream).any()
