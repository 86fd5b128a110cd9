"""Batched serving as a program runs it: plan, embed, project, prepare, attend, LM head, sample, step after step,
with requests that come, end and wait, eager and from graphs. Each step is checked against batch_ref.py with
the host's own account of tables and lengths."""
import numpy as np
import pytest

import batch_ref as R
import hyperion_amd as hy
from hyperion_amd import synthetic as syn
from test_gpu_batch import CONFIG, dev, f64, read_cache, say, u32

pytestmark = pytest.mark.gpu

HIDDEN, VOCAB = 256, 1000
LAYERS = [   # n_heads, kv heads, head dim, window, rotated dims, base, V of its own, scale
    (4, 2, 64, 24, 64, 1e4, True, 1.0),
    (8, 1, 128, 0, 32, 1e6, False, 128**-0.5),
]


class Layer:
    def __init__(self, i, shape, slots):
        self.H, self.KVH, self.D, self.window, self.rotated, self.base, self.own_v, self.scale = shape
        w = lambda n, s, k=HIDDEN: hy.QWeight.from_host(*syn.q4_weights(n, k, seed=100 * i + s))  # noqa: E731
        self.q, self.k, self.v = w(self.H * self.D, 1), w(self.KVH * self.D, 2), w(self.KVH * self.D, 3)
        self.o = w(HIDDEN, 4, self.H * self.D)
        self.cache = hy.KvCache(slots, self.KVH, self.D)
        rng = np.random.default_rng(i)
        norm = lambda: syn.bf16_bits((0.5 + rng.random(self.D)).astype(np.float32))  # noqa: E731
        self.q_norm, self.k_norm = norm(), norm()


class Server:
    """The device's state of a few requests, and the host's account of it."""

    def __init__(self, stream, requests, block, num_blocks, max_blocks, prefix):
        self.stream, self.block, self.num, self.prefix = stream, block, num_blocks, prefix
        rng = np.random.default_rng(5)
        order = rng.permutation(num_blocks).astype(np.uint32)
        n_prefix = R.blocks(prefix, block)
        self.prefix_table = order[:n_prefix]
        self.host = dict(lens=np.zeros(requests, np.uint32), tables=np.full((requests, max_blocks), R.NONE, np.uint32),
                         free=order.copy(), taken=n_prefix)   # (the prefix's blocks are the stack's first)
        h = self.host
        self.lens, self.tables, self.free = dev(h["lens"], stream), dev(h["tables"], stream), dev(h["free"], stream)
        self.taken, self.served = dev(u32(h["taken"]), stream), dev(u32(0), stream)
        self.new, self.row_start = dev(h["lens"], stream), dev(np.zeros(requests + 1, np.uint32), stream)
        self.d_prefix = dev(self.prefix_table, stream)
        self.layers = [Layer(i, s, num_blocks * block) for i, s in enumerate(LAYERS)]
        self.table = hy.QWeight.from_host(*syn.q4_weights(VOCAB, HIDDEN, seed=9))
        for la in self.layers:
            la.d_qn, la.d_kn = dev(la.q_norm, stream), dev(la.k_norm, stream)
        self.fill_prefix(rng)

    def fill_prefix(self, rng):
        """The prefix's K and V, stored as a request's would be."""
        n, s = self.prefix, self.stream
        at = np.arange(n)
        slots = (self.prefix_table[at // self.block] * self.block + at % self.block).astype(np.uint32)
        b = hy.Batch(self.block, self.num, dev(np.zeros((1, 1), np.uint32), s), dev(u32(n), s), dev(u32(0, n), s),
                     dev(slots, s), dev(at.astype(np.uint32), s))
        for la in self.layers:
            k, v, q = (dev(syn.bf16_bits(rng.standard_normal((n, h, la.D)).astype(np.float32)), s)
                       for h in (la.KVH, la.KVH, la.H))
            b.prepare(q, k, v if la.own_v else None, la.H, la.cache, la.d_qn, la.d_kn, 1e-6, la.rotated, la.base, q, s)
            s.synchronize()

    def step_of(self, max_rows):
        return Step(self, max_rows)


class Step:
    """The arrays of a step of up to max_rows rows, and its calls."""

    def __init__(self, server, rows):
        self.sv, self.rows, self.graphs = server, rows, []
        s = server.stream
        z = lambda *shape: dev(np.zeros(shape, np.uint16), s)  # noqa: E731
        self.slots, self.positions = dev(np.zeros(rows, np.uint32), s), dev(np.zeros(rows, np.uint32), s)
        self.batch = hy.Batch(server.block, server.num, server.tables, server.lens, server.row_start, self.slots,
                              self.positions, server.prefix, server.d_prefix)
        self.ids, self.tokens = dev(np.zeros(rows, np.uint32), s), dev(np.zeros(rows, np.uint32), s)
        self.configs, self.uniforms = dev(np.zeros(rows, CONFIG), s), dev(np.zeros(rows, np.float32), s)
        self.logprobs = dev(np.zeros(rows, np.float32), s)
        self.x, self.logits = z(rows, HIDDEN), z(rows, VOCAB)
        self.bufs = [dict(q=z(rows, la.H, la.D), k=z(rows, la.KVH, la.D), v=z(rows, la.KVH, la.D), turned=z(rows, la.H, la.D),
                          out=z(rows, la.H, la.D), y=z(rows, HIDDEN)) for la in server.layers]
        need = max(self.batch.attention_workspace_bytes(la.H, la.cache) for la in server.layers)
        self.work = dev(np.full(need, 0xFF, np.uint8), s)
        self.sample_work = dev(np.full(hy.sample_batch_workspace_bytes(rows, VOCAB), 0xFF, np.uint8), s)

    def plan(self):
        sv = self.sv
        self.batch.plan(sv.lens, sv.new, sv.free, sv.taken, sv.taken, sv.served, sv.stream)

    def attend(self, la, b):
        s = self.sv.stream
        self.batch.prepare(b["q"], b["k"], b["v"] if la.own_v else None, la.H, la.cache, la.d_qn, la.d_kn, 1e-6, la.rotated,
                           la.base, b["turned"], s)
        self.batch.attention(b["turned"], la.H, la.cache, la.window, la.scale, b["out"], self.work, s)

    def sample(self):
        hy.sample_batch(self.logits, self.rows, VOCAB, self.configs, self.uniforms, self.tokens, self.logprobs,
                        self.sample_work, self.sv.stream)

    def capture(self):
        """The batch's calls as graphs (hyp_qmatmul of more than 4 rows, between them, is not recorded)."""
        sv = self.sv
        self.graphs = []
        for f in [self.plan] + [lambda la=la, b=b: self.attend(la, b) for la, b in zip(sv.layers, self.bufs)] + [self.sample]:
            with hy.Graph.capture(sv.stream) as g:
                f()
            self.graphs.append(g)

    def calls(self, graphs):
        sv, s, n = self.sv, self.sv.stream, self.rows
        plan, *attend, sample = [lambda g=g: g.launch(s) for g in graphs] if graphs else (
            [self.plan] + [lambda la=la, b=b: self.attend(la, b) for la, b in zip(sv.layers, self.bufs)] + [self.sample])
        plan()
        hy.embed(sv.table, self.ids, n, self.x, s)
        x = self.x
        for la, b, f in zip(sv.layers, self.bufs, attend):
            for w, y in ((la.q, b["q"]), (la.k, b["k"]), (la.v, b["v"])):
                hy.qmatmul(w, x, n, y, s)
            f()
            hy.qmatmul(la.o, b["out"], n, b["y"], s)
            x = b["y"]
        hy.qmatmul(sv.table, x, n, self.logits, s, softcap=30.0)
        sample()

    def run(self, new, ids, rng):
        """One step with these new tokens: its sampled tokens, checked throughout."""
        sv, s, h = self.sv, self.sv.stream, self.sv.host
        configs = np.zeros(self.rows, CONFIG)
        configs["temperature"] = rng.choice([0.0, 0.5, 1.0], self.rows)
        configs["top_k"] = rng.choice([0, 3, 50], self.rows)
        configs["top_p"] = rng.choice([0.0, 0.5, 0.9], self.rows)
        uniforms = rng.random(self.rows).astype(np.float32)
        all_ids = np.zeros(self.rows, np.uint32)
        all_ids[:len(ids)] = ids
        for a, v in ((sv.new, new), (self.ids, all_ids), (self.configs, configs), (self.uniforms, uniforms)):
            a.upload(v, s)
        self.calls(self.graphs)
        s.synchronize()
        h["tables"], free, h["taken"], served, h["lens"], start, slots, positions = R.plan(
            h["lens"], new, h["tables"], h["free"], h["taken"], self.sv.block, self.rows, sv.prefix)
        h["free"][h["taken"]:] = free[h["taken"]:]
        got = sv.lens.to_host(s), sv.row_start.to_host(s), self.slots.to_host(s), self.positions.to_host(s)
        for a, b in zip(got, (h["lens"], start, slots, positions)):
            assert np.array_equal(a, b)
        assert int(sv.taken.to_host(s)[0]) == h["taken"] and int(sv.served.to_host(s)[0]) == served
        assert np.array_equal(sv.tables.to_host(s), h["tables"])
        rows = int(start[-1])
        at = slots[:rows].astype(np.int64)
        for la, b in zip(sv.layers, self.bufs):
            ck, cv = (f64(c) for c in read_cache(la.cache, (sv.num * sv.block, la.KVH, la.D), s))
            q, k, v = (f64(b[n].to_host(s))[:rows] for n in "qkv")

            def near(got, normed, turned, what):   # as test_prepare's
                ref = R.rope(normed, positions[:rows], la.rotated, la.base) if turned else normed
                pair = np.abs(normed) + np.abs(np.roll(normed, la.D // 2, -1))
                assert np.all(np.abs(got - ref) <= 2.0**-8 * np.abs(ref) + 64 * 2.0**-24 * pair), what

            turned = b["turned"].to_host(s)
            near(f64(turned)[:rows], R.rms(q, f64(la.q_norm)), True, "q")
            near(ck[at], R.rms(k, f64(la.k_norm)), True, "k")
            near(cv[at], R.rms(v if la.own_v else k), False, "v")
            ref, size, apart = R.attention(f64(turned)[:rows], ck, cv, h["tables"], h["lens"], start, sv.block, sv.num,
                                           sv.prefix, sv.prefix_table, la.window, la.scale)
            score = (la.D / 32 + 8) * 2.0**-24 * la.scale * size[..., None]   # as Scene.compare's, one term
            bound = (2.0**-8 * np.abs(ref) + np.max(np.abs(cv[np.isfinite(cv)])) * (2.0**-15 + 2 * score) +
                     2.0**-8 * (1 + 2.0**-7) * apart)
            assert np.all(np.abs(f64(b["out"].to_host(s))[:rows] - ref) <= bound)
        logits = syn.bf16_to_f32(self.logits.to_host(s))
        tokens = self.tokens.to_host(s)
        for t in range(rows):
            c = configs[t]
            assert tokens[t] == R.sample(logits[t], float(c["temperature"]), int(c["top_k"]), float(c["top_p"]),
                                         float(c["min_p"]), float(uniforms[t]))[0]
        return tokens, start


def serve(stream, from_graph):
    """Ten requests' slots: prompts of 1 .. 60 tokens, then decode steps while some end and others come."""
    rng = np.random.default_rng(77)
    requests = 10
    sv = Server(stream, requests, 16, 80, 8, 37)
    prompts, decode = sv.step_of(300), sv.step_of(requests)
    last = np.zeros(requests, np.uint32)
    log = []

    def prompt(lengths):
        new = np.array(lengths, np.uint32)
        tokens, start = prompts.run(new, rng.integers(0, VOCAB, new.sum()), rng)
        for r in range(requests):
            if new[r]:
                last[r] = tokens[start[r + 1] - 1]
        log.append(last.copy())

    prompt([1, 60, 17, 0, 33, 16, 0, 5, 48, 29])
    for step in range(8):
        new = (sv.host["lens"] > 0).astype(np.uint32)
        if step == 3:
            new[[1, 7]] = hy.REQUEST_DONE
        if step == 5:
            new[4] = 0   # waits
        if from_graph and step == 1:   # (the first step was eager)
            decode.capture()
        rows = np.flatnonzero(new == 1)
        tokens, start = decode.run(new, last[rows], rng)
        last[rows] = tokens[:len(rows)]
        log.append(last.copy())
        if step == 4:
            prompt([0, 7, 0, 44, 0, 0, 1, 0, 0, 0])
        if step == 6:
            new = (sv.host["lens"] > 0).astype(np.uint32)   # drafts of some requests verified beside a prompt
            new[[0, 2]] = 4
            new[7] = 31
            prompt(new)
    stream.synchronize()
    for g in decode.graphs:
        g.close()
    return np.array(log)


def test_requests_come_and_go(stream):
    say("serving, eager and from graphs")
    eager = serve(stream, False)
    assert np.array_equal(eager, serve(stream, True))
