"""Performance cases of batched serving: many requests decoded together over one paged cache
per layer, with a prefix that all of them share.

Kinds:
  plan       block tables, slot map and positions of one step, from the requests' lengths
  prepare    q/k norms, RoPE at each row's own position and the cache append by slot
  attention  every request's rows over the shared prefix and its own paged tokens
  sample     one token a row from given uniforms: temperature, top-k, top-p, min-p

Layer forms: the 12B decoder's sliding layers (16 query heads, 8 KV heads x 256, 1024-token
window) and global layers (1 KV head x 512, K = V, 128 rotated dims), and two generic ones,
grouped heads of 128 and ungrouped heads of 64. Index tensors are int32 with the entry
points' 32-bit patterns: -1 is HYP_SLOT_NONE, and in `new` a request that is done.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
GOLDEN = 0.6180339887498949
MAX_POSITION = 1 << 24
# name -> query heads, KV heads, head dim, window, rotated dims, base, V of its own, q.k scale
LAYERS = {
    "sliding": (16, 8, 256, 1024, 256, 1e4, True, 1.0),
    "global": (16, 1, 512, 0, 128, 1e6, False, 1.0),
    "grouped": (32, 8, 128, 0, 128, 1e4, True, 128 ** -0.5),
    "ungrouped": (12, 12, 64, 0, 64, 1e4, True, 64 ** -0.5),
}


def listed():
    return [
        # One decode step of 64 conversations of mixed lengths, some of which have just ended.
        {"name": "plan-decode", "kind": "plan", "requests": 64, "block": 16, "prefix": 1000, "lo": 1, "hi": 4000,
         "new_hi": 1, "done_every": 9},
        # Admission of many prompts of very different lengths in one step.
        {"name": "plan-prompts", "kind": "plan", "requests": 509, "block": 32, "prefix": 0, "lo": 0, "hi": 300,
         "new_hi": 1500, "done_every": 13},
        # The append of one decode step of 48 requests, sliding layer.
        {"name": "prepare-decode", "kind": "prepare", "layer": "sliding", "rows": 48, "block": 16, "far": 9000},
        # A whole chunk of prompt rows behind a long context, global layer.
        {"name": "prepare-chunk", "kind": "prepare", "layer": "global", "rows": 2047, "block": 64, "far": 120000},
        # Four conversations that have just begun behind a short instruction: the smallest call.
        {"name": "attn-few", "kind": "attention", "layer": "sliding", "requests": 4, "block": 16, "prefix": 100,
         "lo": 1, "hi": 60, "rows_hi": 1},
        # A decode step of 64 conversations; the window reaches back into the shared prefix for some of them.
        {"name": "attn-sliding", "kind": "attention", "layer": "sliding", "requests": 64, "block": 16, "prefix": 2000,
         "lo": 20, "hi": 1500, "rows_hi": 1},
        # A decode step behind a long shared document, global layer: the prefix is most of the keys.
        {"name": "attn-global", "kind": "attention", "layer": "global", "requests": 50, "block": 32, "prefix": 16001,
         "lo": 1, "hi": 1800, "rows_hi": 1},
        # A decode step whose own tokens are most of the keys, grouped heads.
        {"name": "attn-own", "kind": "attention", "layer": "grouped", "requests": 96, "block": 64, "prefix": 777,
         "lo": 33, "hi": 3000, "rows_hi": 1},
        # Questions of different lengths prefilled together behind one document.
        {"name": "attn-questions", "kind": "attention", "layer": "global", "requests": 24, "block": 16, "prefix": 6000,
         "lo": 9, "hi": 330, "rows_hi": 250},
        # One conversation alone.
        {"name": "sample-one", "kind": "sample", "rows": 1, "vocab": 262144, "filters": "usual"},
        # A batch whose requests ask for different filters.
        {"name": "sample-mixed", "kind": "sample", "rows": 64, "vocab": 262144, "filters": "mixed"},
        # A large batch at temperature alone: every token can be drawn. An odd vocabulary.
        {"name": "sample-free", "kind": "sample", "rows": 200, "vocab": 50001, "filters": "free"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "prepare", "attention", "attention", "attention", "sample"))
    if kind == "plan":
        decode = rng.random() < 0.5
        return {"kind": kind, "requests": _log(rng, 1, 500), "block": rng.choice((8, 16, 32, 64, 128)),
                "prefix": rng.choice((0, _log(rng, 1, 30000))), "lo": rng.randint(0, 40), "hi": _log(rng, 50, 4000),
                "new_hi": 1 if decode else _log(rng, 2, 1500), "done_every": rng.randint(3, 40)}
    if kind == "prepare":
        return {"kind": kind, "layer": rng.choice(tuple(LAYERS)), "rows": _log(rng, 1, 2040),
                "block": rng.choice((8, 16, 32, 64, 128)), "far": _log(rng, 100, 250000)}
    if kind == "sample":
        rows = _log(rng, 1, 200)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 1000, min(262143, 64 * 262144 // rows)),
                "filters": rng.choice(("usual", "mixed", "free"))}
    layer = rng.choice(tuple(LAYERS))
    case = {"kind": kind, "layer": layer, "block": rng.choice((8, 16, 32, 64, 128)), "lo": rng.randint(1, 50)}
    if rng.random() < 0.7:   # a decode step
        n = _log(rng, 1, 96)
        hi = _log(rng, 60, 3000 if layer == "grouped" else 1500)
        return dict(case, requests=n, prefix=rng.choice((0, _log(rng, 1, 16000))), hi=hi, rows_hi=1)
    n = _log(rng, 1, 24)   # drafts verified, or questions prefilled
    return dict(case, requests=n, prefix=rng.choice((0, _log(rng, 1, 6000))), hi=_log(rng, 60, 330),
                rows_hi=_log(rng, 2, 250))


# ---- inputs -----------------------------------------------------------------------------

def _spread(n, lo, hi, turn=0.0):
    """n whole numbers over [lo, hi], evenly and in no order."""
    return [lo + int((hi - lo + 1) * ((GOLDEN * (i + 1) + turn) % 1.0)) for i in range(n)]


def _blocks(tokens, block):
    return (tokens + block - 1) // block


def _plan_lens(case):
    """Tokens held, tokens new (None: done) of each request."""
    n = case["requests"]
    new = [None if i % case["done_every"] == case["done_every"] - 1 else v
           for i, v in enumerate(_spread(n, 1, case["new_hi"], 0.3))]
    return _spread(n, case["lo"], case["hi"]), new


def _attn_lens(case):
    """Own tokens (this step's among them) and rows of each request."""
    lens = _spread(case["requests"], case["lo"], case["hi"])
    rows = [min(r, n) for r, n in zip(_spread(case["requests"], 1, case["rows_hi"], 0.3), lens)]
    return lens, rows


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _norm(g, n, around=1.0):
    return (around * (1.0 + 0.1 * _randn(g, n))).to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _full(value, *shape):
    return torch.full(shape, value, dtype=torch.int32, device="cuda")


def _tables(g, held, block, max_blocks, spare):
    """Random blocks for `held` tokens of each request, the unused entries -1; then the blocks that
    are left, in random order, and how many the pool has."""
    counts = [_blocks(n, block) for n in held]
    num = sum(counts) + spare
    order = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    tables = _full(-1, len(held), max_blocks)
    at = 0
    for i, c in enumerate(counts):
        tables[i, :c] = order[at:at + c]
        at += c
    return tables, order[at:], num


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = _gen(seed)
    kind = case["kind"]
    t = {}
    if kind == "plan":
        lens, new = _plan_lens(case)
        block = case["block"]
        rows = sum(n for n in new if n is not None)
        grown = [_blocks(n + (m or 0), block) for n, m in zip(lens, new)]
        t["tables"], left, num = _tables(g, lens, block, max(grown) + 8, sum(grown) + 5)
        taken = num - left.numel()
        t["free"] = torch.cat((_full(-1, taken), left))
        t["lens"], t["new"] = _ints(lens), _ints([-1 if n is None else n for n in new])
        t["taken"], t["taken_out"], t["served"] = _ints([taken]), _full(0, 1), _full(0, 1)
        t["lens_out"], t["row_start"] = _full(0, len(lens)), _full(0, len(lens) + 1)
        t["slots"], t["positions"] = _full(0, rows + 7), _full(0, rows + 7)
        t["num"] = num
    elif kind == "prepare":
        h, kvh, d, _, _, _, own_v, _ = LAYERS[case["layer"]]
        rows, block = case["rows"], case["block"]
        num = _blocks(rows, block) + 3
        t["num"] = num
        t["slots"] = torch.randperm(num * block, generator=g, device="cuda")[:rows].to(torch.int32)
        t["positions"] = torch.randint(0, case["far"], (rows,), generator=g, device="cuda").to(torch.int32)
        t["row_start"] = _ints([0, rows])
        t["tables"], t["lens"] = _full(-1, 1, num), _ints([rows])
        t["q"] = _randn(g, rows, h, d).to(torch.bfloat16)
        t["k"] = _randn(g, rows, kvh, d).to(torch.bfloat16)
        if own_v:
            t["v"] = _randn(g, rows, kvh, d).to(torch.bfloat16)
        t["q_norm"], t["k_norm"] = _norm(g, d, d ** -0.25), _norm(g, d, d ** -0.25)
        t["pool_k"], t["pool_v"] = (_randn(g, num * block, kvh, d).to(torch.bfloat16) for _ in range(2))
        t["q_out"] = torch.zeros_like(t["q"])
    elif kind == "attention":
        h, kvh, d, _, _, _, _, scale = LAYERS[case["layer"]]
        lens, rows = _attn_lens(case)
        block, prefix = case["block"], case["prefix"]
        held = [prefix] + lens
        tables, _, num = _tables(g, held, block, max(_blocks(n, block) for n in held), 3)
        t["num"] = num
        t["prefix_table"] = tables[0, :_blocks(prefix, block)].contiguous()
        t["tables"] = tables[1:, :max(_blocks(n, block) for n in lens) + 2].contiguous()
        t["lens"] = _ints(lens)
        t["row_start"] = _ints(np.concatenate(([0], np.cumsum(rows))).tolist())
        total = sum(rows)
        t["slots"], t["positions"] = _full(-1, total), _full(0, total)
        size = d ** -0.25 if scale == 1.0 else 1.0   # (scores of a standard deviation of 2)
        t["q"] = (2.0 * size * _randn(g, total, h, d)).to(torch.bfloat16)
        t["pool_k"] = (size * _randn(g, num * block, kvh, d)).to(torch.bfloat16)
        t["pool_v"] = _randn(g, num * block, kvh, d).to(torch.bfloat16)
        t["out"] = torch.zeros_like(t["q"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        t["logits"] = (30.0 * torch.tanh(3.0 * _randn(g, rows, vocab) / 30.0)).to(torch.bfloat16)
        t["uniforms"] = torch.rand((rows,), generator=g, device="cuda", dtype=torch.float32)
        cfg = torch.zeros((rows, 6), dtype=torch.int32, device="cuda")   # HypSamplingConfig, 24 bytes a row
        pick = torch.randint(0, 1000, (4, rows), generator=g, device="cuda")
        if case["filters"] == "usual":
            temperature, top_k, top_p, min_p = (torch.full((rows,), v, device="cuda") for v in (0.8, 64, 0.95, 0.05))
        elif case["filters"] == "free":
            temperature = 0.5 + pick[0] / 1000.0
            top_k, top_p, min_p = pick[1] * 0, 1.0 + pick[2] * 0.0, pick[3] * 0.0
        else:
            temperature = torch.where(pick[0] < 120, pick[0] * 0.0, 0.3 + pick[0] / 800.0)
            top_k = torch.where(pick[1] < 400, 0, pick[1] - 399)
            top_p = torch.where(pick[2] < 300, 1.0, 0.7 + pick[2] * 3e-4)
            min_p = torch.where(pick[3] < 600, 0.0, pick[3] * 1e-4)
        for i, v in enumerate((temperature, None, top_p, min_p)):
            if v is not None:
                cfg[:, i] = v.to(torch.float32).view(torch.int32)
        cfg[:, 1] = top_k.to(torch.int32)
        t["configs"], t["tokens"] = cfg, _full(0, rows)
        t["logprobs"] = torch.zeros((rows,), dtype=torch.float32, device="cuda")
    return t


# ---- the framework's side -----------------------------------------------------------------

_stream = None


def _the_stream():
    """The one stream of this program."""
    global _stream
    if _stream is None:
        import hyperion_amd as hy
        _stream = hy.Stream()
    return _stream


class _Raw:
    """A cache's memory for torch.as_tensor; the tensor keeps this object, and with it the cache, alive."""

    def __init__(self, owner, address, shape):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (address, False), "shape": tuple(shape), "typestr": "<i2",
                                         "version": 2}


def _handles(case, st):
    """What a program using the entry points keeps: the cache, the step's batch, workspaces."""
    import hyperion_amd as hy
    kind = case["kind"]
    st["stream"] = _the_stream()
    st["dev"] = dev = {k: hy.DeviceView(v) for k, v in st.items() if isinstance(v, torch.Tensor)}
    if kind in ("prepare", "attention"):
        _, kvh, d = LAYERS[case["layer"]][:3]
        slots = st["num"] * case["block"]
        st["cache"] = cache = hy.KvCache(slots, kvh, d)
        for name, p in zip(("pool_k", "pool_v"), cache.buffers()):
            view = torch.as_tensor(_Raw(cache, p.value, (slots, kvh, d)), device="cuda").view(torch.bfloat16)
            view.copy_(st[name])
            st[name] = view
    if kind != "sample":
        st["batch"] = hy.Batch(case["block"], st["num"], dev["tables"], dev["lens_out" if kind == "plan" else "lens"],
                               dev["row_start"], dev["slots"], dev["positions"], case.get("prefix", 0),
                               dev.get("prefix_table"))
    need = 0
    if kind == "attention":
        need = st["batch"].attention_workspace_bytes(LAYERS[case["layer"]][0], st["cache"])
    elif kind == "sample":
        need = hy.sample_batch_workspace_bytes(case["rows"], case["vocab"])
    st["workspace"] = hy.DeviceArray((need,), np.uint8) if need else None


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        _handles(case, st)
    torch.cuda.synchronize()
    return st


def _run_own(st):
    case, dev, s = st["case"], st["dev"], st["stream"]
    kind = case["kind"]
    if kind == "plan":
        st["batch"].plan(dev["lens"], dev["new"], dev["free"], dev["taken"], dev["taken_out"], dev["served"], s)
    elif kind == "prepare":
        h, _, _, _, rotated, base, _, _ = LAYERS[case["layer"]]
        st["batch"].prepare(dev["q"], dev["k"], dev.get("v"), h, st["cache"], dev["q_norm"], dev["k_norm"], EPS, rotated,
                            base, dev["q_out"], s)
    elif kind == "attention":
        h, _, _, window, _, _, _, scale = LAYERS[case["layer"]]
        st["batch"].attention(dev["q"], h, st["cache"], window, scale, dev["out"], st["workspace"], s)
    else:
        from hyperion_amd import sample_batch
        sample_batch(dev["logits"], case["rows"], case["vocab"], dev["configs"], dev["uniforms"], dev["tokens"],
                     dev["logprobs"], st["workspace"], s)


# ---- the plain forms ------------------------------------------------------------------------

def _plan_plain(st):
    case = st["case"]
    block, prefix, num = case["block"], case["prefix"], st["num"]
    lens, new = st["lens"].long(), st["new"].long()
    max_blocks, max_rows = st["tables"].shape[1], st["slots"].shape[0]
    done = new < 0
    have = _blocks(lens, block)
    new = torch.where(done, 0, new)
    need = torch.where(done, 0, _blocks(lens + new, block))
    grow = torch.where(done, 0, need - have)
    entry = torch.arange(max_blocks, device="cuda")
    back = done[:, None] & (entry < have[:, None])               # the blocks that return, in order
    returned = back.sum()
    first = st["taken"].long() - returned
    ok = (new.cumsum(0) <= max_rows) & (grow.cumsum(0) <= num - first) & (need <= max_blocks)
    ok &= prefix + lens + new <= MAX_POSITION
    served = ok.long().cumprod(0).sum()
    serve = torch.arange(lens.shape[0], device="cuda") < served
    new, need = torch.where(serve, new, 0), torch.where(serve & ~done, need, 0)
    at = torch.where(back.flatten(), first + back.flatten().cumsum(0) - 1, num)
    free = torch.cat((st["free"], st["free"][:1]))
    free[at] = st["tables"].flatten()
    st["free"].copy_(free[:num])
    fresh = (entry >= have[:, None]) & (entry < need[:, None])
    at = (first + fresh.flatten().cumsum(0) - 1).clamp(0, num - 1)
    st["tables"].copy_(torch.where(fresh, st["free"][at].view(fresh.shape), st["tables"]))
    st["taken_out"].copy_(first + fresh.sum())
    st["served"].copy_(served)
    st["lens_out"].copy_(torch.where(done, 0, lens + new))
    st["row_start"][1:] = new.cumsum(0)
    row = torch.arange(max_rows, device="cuda")
    request = torch.searchsorted(st["row_start"][1:].long(), row, right=True)
    live = request < lens.shape[0]
    request = request.clamp(max=lens.shape[0] - 1)
    own_at = lens[request] + row - st["row_start"].long()[request]
    entry = st["tables"][request, (own_at // block).clamp(max=max_blocks - 1)].long()
    st["slots"].copy_(torch.where(live, entry * block + own_at % block, -1))
    st["positions"].copy_(torch.where(live, prefix + own_at, 0))


def _rotate(x, positions, rotated, base):
    """x [rows, heads, d] float32; the angles are float32 products, as every RoPE here defines them."""
    d = x.shape[-1]
    half = d // 2
    inv = (base ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / d)).float()
    theta = (positions.float()[:, None] * inv).double()
    theta[:, rotated // 2:] = 0.0
    c, s = torch.cos(theta).float()[:, None], torch.sin(theta).float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def _rms(x, weight=None):
    x = x.float()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if weight is None else y * weight.float()


def _prepare_plain(st):
    _, _, _, _, rotated, base, own_v, _ = LAYERS[st["case"]["layer"]]
    at = st["slots"].long()
    st["q_out"].copy_(_rotate(_rms(st["q"], st["q_norm"]), st["positions"], rotated, base))
    st["pool_k"][at] = _rotate(_rms(st["k"], st["k_norm"]), st["positions"], rotated, base).to(torch.bfloat16)
    st["pool_v"][at] = _rms(st["v"] if own_v else st["k"]).to(torch.bfloat16)


def _weigh(scores, seen, values):
    """Maximum, sum and weighted values of score rows [..., rows, keys] over the keys seen."""
    scores = scores.masked_fill(~seen, -math.inf)
    m = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - m.clamp(min=-1e30))
    return m, w.sum(-1, keepdim=True), w @ values


def _token_slots(table, tokens, block):
    """Slots of the first `tokens` tokens of tables [..., blocks]."""
    j = torch.arange(tokens, device="cuda")
    return table.long()[..., j // block].clamp(min=0) * block + j % block


def _attention_plain(st):
    case = st["case"]
    h, kvh, d, window, _, _, _, scale = LAYERS[case["layer"]]
    n, prefix, block, g = case["requests"], case["prefix"], case["block"], h // kvh
    longest, most, total = case["hi"], case["rows_hi"], st["q"].shape[0]
    q = st["q"].float() * scale
    row = torch.arange(total, device="cuda")
    start = st["row_start"].long()
    request = torch.searchsorted(start[1:], row, right=True)
    i = row - start[request]
    lens = st["lens"].long()
    pos = prefix + lens[request] - (start[1:] - start[:-1])[request] + i

    def back(x):   # [n, kvh, most * g, e] -> [total, h, e]
        return x.view(n, kvh, most, g, -1)[request, :, i].reshape(total, h, -1)

    # Each request's own tokens, rows and keys padded to the longest.
    padded = torch.zeros((n, most, kvh, g, d), device="cuda")
    padded[request, i] = q.view(total, kvh, g, d)
    padded = padded.permute(0, 2, 1, 3, 4).reshape(n, kvh, most * g, d)
    at = _token_slots(st["tables"], min(longest, st["tables"].shape[1] * block), block)
    k, v = (st[p][at].float().permute(0, 2, 1, 3) for p in ("pool_k", "pool_v"))
    key = torch.arange(at.shape[1], device="cuda")
    where = torch.full((n, most), -1, device="cuda")
    where[request, i] = pos - prefix
    where = where[:, None, :, None].expand(n, 1, most, g).reshape(n, 1, most * g, 1)
    seen = (key <= where) & (key < lens[:, None, None, None])
    if window:
        seen &= key > where - window
    m, l, o = (back(x) for x in _weigh(padded @ k.transpose(-1, -2), seen, v))
    if prefix:
        # The prefix once: every row of a KV head against the same keys.
        at = _token_slots(st["prefix_table"], prefix, block)
        k, v = (st[p][at].float().permute(1, 0, 2) for p in ("pool_k", "pool_v"))
        rows = q.view(total, kvh, g, d).permute(1, 0, 2, 3).reshape(kvh, total * g, d)
        key = torch.arange(prefix, device="cuda")
        where = pos[:, None].expand(total, g).reshape(1, total * g, 1)
        seen = key <= where
        if window:
            seen = seen & (key > where - window)
        mp, lp, op = (x.view(kvh, total, g, -1).permute(1, 0, 2, 3).reshape(total, h, -1)
                      for x in _weigh(rows @ k.transpose(-1, -2), seen, v))
        top = torch.maximum(m, mp)
        a, b = torch.exp(m - top), torch.exp(mp - top)
        l, o = l * a + lp * b, o * a + op * b
    st["out"].copy_(o / l)


def _sample_plain(st):
    cfg = st["configs"]
    temperature, top_p, min_p = (cfg[:, c:c + 1].view(torch.float32).double() for c in (0, 2, 3))
    top_k = cfg[:, 1:2]
    x, index = torch.sort(st["logits"].float() + 0.0, dim=-1, descending=True, stable=True)
    vocab = x.shape[1]
    t = torch.where(temperature > 0, temperature, 1.0)
    w = torch.exp((x - x[:, :1]).double() / t)
    running = w.cumsum(-1)
    total = running[:, -1:]
    rank = torch.arange(vocab, device="cuda")
    kept = torch.where(top_p < 1, running - w < top_p * total, True) & (w >= min_p)
    kept &= torch.where(top_k > 0, rank < top_k, True) & torch.where(temperature > 0, True, rank < 1)
    count = kept.long().cumprod(-1).sum(-1, keepdim=True)
    goal = st["uniforms"].double()[:, None] * running.gather(-1, count - 1)
    at = torch.minimum((running <= goal).sum(-1, keepdim=True), count - 1)
    st["tokens"].copy_(index.gather(-1, at)[:, 0])
    st["logprobs"].copy_(((x.gather(-1, at) - x[:, :1]).double() / t - torch.log(total))[:, 0])


def run(st):
    kind = st["case"]["kind"]
    if own:
        _run_own(st)
    elif kind == "plan":
        _plan_plain(st)
    elif kind == "prepare":
        _prepare_plain(st)
    elif kind == "attention":
        _attention_plain(st)
    else:
        _sample_plain(st)
    names = {"plan": ("tables", "free", "taken_out", "served", "lens_out", "row_start", "slots", "positions"),
             "prepare": ("q_out", "pool_k", "pool_v"), "attention": ("out",), "sample": ("tokens", "logprobs")}[kind]
    return {name: st[name] for name in names}


# ---- what a pass has to do -------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        lens, new = _plan_lens(case)
        block = case["block"]
        rows = sum(n for n in new if n is not None)
        fresh = sum(_blocks(a + (b or 0), block) - _blocks(a, block) for a, b in zip(lens, new))
        back = sum(_blocks(a, block) for a, b in zip(lens, new) if b is None)
        # lengths in and out, row starts, a partly filled block's entry; blocks moved; rows written
        return {"bytes": 20 * len(lens) + 8 * (fresh + back) + 8 * (rows + 7), "flops": 0}
    if kind == "prepare":
        h, kvh, d, _, _, _, own_v, _ = LAYERS[case["layer"]]
        rows = case["rows"]
        values = rows * d
        read, written = h + kvh + (kvh if own_v else 0), h + 2 * kvh
        return {"bytes": 2 * values * (read + written) + 8 * rows + 4 * d, "flops": values * (4 * read + 6 * (h + kvh))}
    if kind == "sample":
        return {"bytes": case["rows"] * (2 * case["vocab"] + 36), "flops": 0}
    h, kvh, d, window, _, _, _, _ = LAYERS[case["layer"]]
    prefix = case["prefix"]
    lens, rows = _attn_lens(case)
    keys, pairs, oldest = 0, 0, prefix
    for n, r in zip(lens, rows):
        first = prefix + n - r                               # the first row's position
        low = max(0, first + 1 - window) if window else 0    # its first key
        oldest = min(oldest, low)
        keys += prefix + n - max(low, prefix)
        for pos in range(first, prefix + n):
            pairs += min(pos + 1, window) if window else pos + 1
    total = sum(rows)
    size = 2 * 2 * kvh * d * (keys + prefix - oldest) + 2 * 2 * h * d * total
    return {"bytes": size + 4 * (len(lens) * 2 + keys // case["block"]), "flops": 4 * h * d * pairs}


# ---- the same in 64 bits ---------------------------------------------------------------------

def _exact_prepare(case, t):
    _, _, d, _, rotated, base, own_v, _ = LAYERS[case["layer"]]
    pair = torch.arange(rotated // 2, dtype=torch.float64, device="cuda")
    angle = t["positions"].to(torch.float32)[:, None] * torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"),
                                                                   -2.0 * pair / d).to(torch.float32)[None, :]
    turn = torch.polar(torch.ones_like(angle, dtype=torch.float64), angle.double())[:, None, :]

    def normed(x, weight):
        x = x.double()
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        return x if weight is None else x * weight.double()

    def turned(x):
        z = torch.complex(x[..., :rotated // 2].contiguous(), x[..., d // 2:d // 2 + rotated // 2].contiguous()) * turn
        y = x.clone()
        y[..., :rotated // 2], y[..., d // 2:d // 2 + rotated // 2] = z.real, z.imag
        return y

    pool_k, pool_v = t["pool_k"].double(), t["pool_v"].double()
    at = t["slots"].long()
    pool_k[at] = turned(normed(t["k"], t["k_norm"]))
    pool_v[at] = normed(t["v"] if own_v else t["k"], None)
    return {"q_out": turned(normed(t["q"], t["q_norm"])), "pool_k": pool_k, "pool_v": pool_v}


def _exact_attention(case, t):
    h, kvh, d, window, _, _, _, scale = LAYERS[case["layer"]]
    block, prefix = case["block"], case["prefix"]
    lens, rows = _attn_lens(case)

    def tokens(pool, table, count):   # [kvh, count, d]
        slots = torch.cat([torch.arange(b * block, b * block + block) for b in table.tolist()] or
                          [torch.zeros(0, dtype=torch.long)])[:count]
        return pool[slots.cuda()].double().transpose(0, 1)

    shared = [tokens(t[p], t["prefix_table"], prefix) for p in ("pool_k", "pool_v")]
    out = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        table = t["tables"][b, :_blocks(n, block)]
        k, v = (torch.cat((s, tokens(t[p], table, n)), 1) for s, p in zip(shared, ("pool_k", "pool_v")))
        q = t["q"][row:row + r].double().reshape(r, kvh, h // kvh, d).permute(1, 2, 0, 3)
        s = scale * torch.matmul(q, k.transpose(1, 2)[:, None].contiguous())       # [kvh, g, r, keys]
        ago = (prefix + n - r + torch.arange(r, device="cuda"))[:, None] - torch.arange(prefix + n, device="cuda")
        hidden = (ago < 0) | (ago >= window) if window else ago < 0
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        out[row:row + r] = torch.matmul(p, v[:, None].contiguous()).permute(2, 0, 1, 3).reshape(r, h, d)
        row += r
    return {"out": out}


def _exact_sample(t):
    logits = t["logits"].float().cpu().numpy().astype(np.float64)
    raw = np.ascontiguousarray(t["configs"].cpu().numpy())
    values, counts = raw.view(np.float32).astype(np.float64), raw[:, 1]
    uniforms = t["uniforms"].cpu().numpy().astype(np.float64)
    tokens, logprobs = [], []
    for x, f, top_k, u in zip(logits, values, counts, uniforms):
        temperature, top_p, min_p = f[0], f[2], f[3]
        greedy = temperature <= 0
        order = np.argsort(-x, kind="stable")
        w = np.exp((x[order] - x[order[0]]) / (1.0 if greedy else temperature))
        mass = np.cumsum(w)
        keep = x.size if top_k <= 0 else min(x.size, int(top_k))
        if top_p < 1:
            keep = min(keep, int(np.searchsorted(mass, top_p * mass[-1], side="left")) + 1)
        keep = min(keep, int(np.count_nonzero(w >= min_p)))
        keep = 1 if greedy else max(1, keep)
        j = min(int(np.searchsorted(mass[:keep], u * mass[keep - 1], side="right")), keep - 1)
        tokens.append(int(order[j]))
        logprobs.append(math.log(w[j] / mass[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None   # whole numbers
    t = _inputs(case, seed)
    if kind == "prepare":
        return _exact_prepare(case, t)
    return _exact_attention(case, t) if kind == "attention" else _exact_sample(t)
