"""Performance cases of speculative decoding and of forked requests, next to batched serving: drafts
verified against the target's logits, and the operations on a paged cache's blocks that go with it.

Kinds:
  verify   drafted tokens against the target's filtered probabilities, from given uniforms
  fork     requests that become copies of others: shared blocks, one block of their own each
  rewind   requests that lose their last tokens or end: blocks that nobody holds are free again
  compact  the blocks in use moved to the pool's lowest ids: tables, free blocks, list of copies
  copy     such a list carried out in the caches of all layers

Index tensors are int32 with the entry points' 32-bit patterns: -1 is HYP_PARENT_NONE, HYP_REQUEST_DONE,
or a table's unused entry.
"""
import math

import numpy as np
import torch

own = False

GOLDEN = 0.6180339887498949
# name -> (layers, KV heads, head dim) of the layers that share one batch's blocks
MODELS = {
    "decoder12b": ((25, 8, 256), (5, 1, 512)),   # 30 of its 48 layers, sliding and global
    "grouped": ((16, 8, 128),),
    "ungrouped": ((12, 12, 64),),
}


def listed():
    return [
        # One conversation with four drafts of a small model: the smallest call.
        {"name": "verify-one", "kind": "verify", "requests": 1, "rows_lo": 5, "rows_hi": 5, "vocab": 262144,
         "filters": "usual", "drafter": True},
        # A batch with a drafting model; every request has filters and a number of drafts of its own.
        {"name": "verify-mixed", "kind": "verify", "requests": 64, "rows_lo": 1, "rows_hi": 8, "vocab": 262144,
         "filters": "mixed", "drafter": True},
        # Drafts found by lookup in the text: no distribution of their own.
        {"name": "verify-lookup", "kind": "verify", "requests": 48, "rows_lo": 4, "rows_hi": 6, "vocab": 262144,
         "filters": "usual", "drafter": False},
        # Temperature alone: every token can be drawn. An odd vocabulary.
        {"name": "verify-free", "kind": "verify", "requests": 100, "rows_lo": 1, "rows_hi": 6, "vocab": 50001,
         "filters": "free", "drafter": True},
        # Two more answers for each of a few conversations.
        {"name": "fork-few", "kind": "fork", "groups": 4, "fan": 2, "block": 16, "lo": 100, "hi": 3000},
        # Prompts that were just read, seven more answers each.
        {"name": "fork-answers", "kind": "fork", "groups": 60, "fan": 7, "block": 16, "lo": 500, "hi": 8000},
        # After verification: every request gives up the drafts that were not taken.
        {"name": "rewind-drafts", "kind": "rewind", "requests": 64, "fan": 0, "block": 16, "lo": 20, "hi": 4000,
         "own_hi": 60, "drop_hi": 7, "done_every": 65},
        # Many answers to common prompts, a part of which have ended.
        {"name": "rewind-answers", "kind": "rewind", "requests": 500, "fan": 4, "block": 32, "lo": 100, "hi": 9000,
         "own_hi": 700, "drop_hi": 20, "done_every": 7},
        # A small pool behind a short prefix.
        {"name": "compact-few", "kind": "compact", "requests": 16, "fan": 0, "block": 16, "lo": 50, "hi": 2000,
         "own_hi": 60, "prefix": 300, "loose": 2.0},
        # A large pool with forked requests, most of it free.
        {"name": "compact-large", "kind": "compact", "requests": 400, "fan": 3, "block": 16, "lo": 100, "hi": 6000,
         "own_hi": 900, "prefix": 5000, "loose": 2.5},
        # The partly filled blocks of a few forked conversations, layers of the 12B decoder.
        {"name": "copy-fork", "kind": "copy", "model": "decoder12b", "copies": 8, "block": 16, "whole": False},
        # A compaction's moves, grouped heads of 128.
        {"name": "copy-compact", "kind": "copy", "model": "grouped", "copies": 500, "block": 16, "whole": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("verify", "verify", "verify", "fork", "rewind", "compact", "copy"))
    block = rng.choice((8, 16, 32, 64, 128))
    if kind == "verify":
        requests = _log(rng, 1, 100)
        hi = rng.randint(1, 8)
        return {"kind": kind, "requests": requests, "rows_lo": rng.randint(1, hi), "rows_hi": hi,
                "vocab": _log(rng, 1000, min(262144, 100000000 // (requests * hi))),
                "filters": rng.choice(("usual", "mixed", "free")), "drafter": rng.random() < 0.6}
    if kind == "fork":
        fan = rng.randint(1, 9)
        return {"kind": kind, "groups": _log(rng, 1, 500 // (fan + 1)), "fan": fan, "block": block,
                "lo": rng.randint(1, 200), "hi": _log(rng, 200, 8000)}
    if kind == "rewind":
        return {"kind": kind, "requests": _log(rng, 1, 500), "fan": rng.choice((0, 0, rng.randint(1, 8))), "block": block,
                "lo": rng.randint(1, 200), "hi": _log(rng, 200, 9000), "own_hi": _log(rng, 20, 700),
                "drop_hi": _log(rng, 1, 40), "done_every": rng.randint(2, 70)}
    if kind == "compact":
        return {"kind": kind, "requests": _log(rng, 1, 400), "fan": rng.choice((0, 0, rng.randint(1, 8))), "block": block,
                "lo": rng.randint(1, 200), "hi": _log(rng, 200, 6000), "own_hi": _log(rng, 20, 900),
                "prefix": rng.choice((0, _log(rng, 1, 5000))), "loose": rng.uniform(1.0, 2.5)}
    model = rng.choice(tuple(MODELS))
    return {"kind": kind, "model": model, "copies": _log(rng, 1, (1024 if model == "decoder12b" else 8000) // block),
            "block": block, "whole": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------

def _spread(n, lo, hi, turn=0.0):
    """n whole numbers over [lo, hi], evenly and in no order."""
    return [lo + int((hi - lo + 1) * ((GOLDEN * (i + 1) + turn) % 1.0)) for i in range(n)]


def _blocks(tokens, block):
    return (tokens + block - 1) // block


def _verify_rows(case):
    return _spread(case["requests"], case["rows_lo"], case["rows_hi"])


def _fork_lens(case):
    """(parents' lengths, slots a parent and its children take)."""
    return _spread(case["groups"], case["lo"], case["hi"]), case["fan"] + 1


def _held(case):
    """For each request: its group, the blocks that the group shares, its length. Requests of a group have a
    prompt's whole blocks in common."""
    n = case["requests"]
    groups = (n + case["fan"]) // (case["fan"] + 1)
    prompts = _spread(groups, case["lo"], case["hi"])
    extra = _spread(n, 0, case["own_hi"], 0.3)
    return [(r % groups, prompts[r % groups] // case["block"], prompts[r % groups] + extra[r]) for r in range(n)]


def _drops(case):
    """Tokens that each request gives up (None: all). What a group shares stays whole."""
    every, block = case["done_every"], case["block"]
    return [None if r % every == every - 1 else min(d, n - shared * block)
            for r, (d, (_, shared, n)) in enumerate(zip(_spread(case["requests"], 0, case["drop_hi"], 0.7), _held(case)))]


def _live_blocks(case):
    """Blocks in use, and how many of those only one request holds."""
    held = _held(case)
    shared = sum({g: s for g, s, _ in held}.values())
    single = sum(_blocks(n, case["block"]) - s for _, s, n in held)
    return shared + single, single


def _copy_tokens(case):
    return [case["block"]] * case["copies"] if case["whole"] else _spread(case["copies"], 1, case["block"] - 1)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(values):
    return torch.tensor(np.asarray(values, np.int32), dtype=torch.int32, device="cuda")


def _full(value, *shape):
    return torch.full(shape, value, dtype=torch.int32, device="cuda")


def _tables(case, order, width):
    """Tables of _held()'s requests over the ids `order`, the unused entries -1, and how many ids they took."""
    held = _held(case)
    tables = np.full((len(held), width), -1, np.int32)
    at, common = 0, {}
    for r, (g, shared, n) in enumerate(held):
        if g not in common:
            common[g] = order[at:at + shared]
            at += shared
        rest = _blocks(n, case["block"]) - shared
        tables[r, :shared] = common[g]
        tables[r, shared:shared + rest] = order[at:at + rest]
        at += rest
    return tables, at


def _verify_inputs(case, seed):
    g = _gen(seed)
    t = {}
    rows, vocab, n = _verify_rows(case), case["vocab"], case["requests"]
    total = sum(rows)
    # A model's logits: most tokens far below, a few likely ones; the drafting model has nearly the same.
    x = 2.0 * _randn(g, total, vocab)
    likely = torch.randint(0, vocab, (total, 24), generator=g, device="cuda")
    x.scatter_add_(1, likely, 10.0 + 3.0 * _randn(g, total, 24))
    t["logits"] = (30.0 * torch.tanh(x / 30.0)).to(torch.bfloat16)
    guess = x + 0.5 * _randn(g, total, vocab)
    guess.scatter_add_(1, likely, 0.7 * _randn(g, total, 24))
    if case["drafter"]:
        t["draft_logits"] = (30.0 * torch.tanh(guess / 30.0)).to(torch.bfloat16)
    u = torch.rand((total, vocab), generator=g, device="cuda", dtype=torch.float32).clamp_(1e-20, 0.9999999)
    drafts = (guess / 0.8 - torch.log(-torch.log(u))).argmax(-1)
    t["ids"] = _full(0, total)
    t["ids"][1:] = drafts[:-1]          # row t + 1 holds what was drafted to follow row t
    t["row_start"] = _ints(np.concatenate(([0], np.cumsum(rows))))
    t["uniforms"] = torch.rand((total,), generator=g, device="cuda", dtype=torch.float32)
    cfg = torch.zeros((n, 6), dtype=torch.int32, device="cuda")   # HypSamplingConfig, 24 bytes a request
    pick = torch.randint(0, 1000, (4, n), generator=g, device="cuda")
    if case["filters"] == "usual":
        temperature, top_k, top_p, min_p = (torch.full((n,), v, device="cuda") for v in (0.8, 64, 0.95, 0.05))
    elif case["filters"] == "free":
        temperature = 0.5 + pick[0] / 1000.0
        top_k, top_p, min_p = pick[1] * 0, 1.0 + pick[2] * 0.0, pick[3] * 0.0
    else:
        temperature = torch.where(pick[0] < 120, pick[0] * 0.0, 0.3 + pick[0] / 800.0)
        top_k = torch.where(pick[1] < 400, 0, pick[1] - 399)
        top_p = torch.where(pick[2] < 300, 1.0, 0.7 + pick[2] * 3e-4)
        min_p = torch.where(pick[3] < 600, 0.0, pick[3] * 1e-4)
    for i, v in ((0, temperature), (2, top_p), (3, min_p)):
        cfg[:, i] = v.to(torch.float32).view(torch.int32)
    cfg[:, 1] = top_k.to(torch.int32)
    t["configs"] = cfg
    t["accepted"], t["rejected"], t["tokens"] = _full(0, n), _full(0, n), _full(0, n)
    t["logprobs"] = torch.zeros((total,), dtype=torch.float32, device="cuda")
    return t


def _copy_inputs(case, seed):
    g = _gen(seed)
    n, block = case["copies"], case["block"]
    num = 2 * n + 3
    ids = torch.randperm(num, generator=g, device="cuda").to(torch.int32)
    t = {"num": num, "copies": torch.stack((ids[:n], ids[n:2 * n], _ints(_copy_tokens(case))), 1).contiguous(),
         "n_copies": _ints([n]), "pools": []}
    for layers, heads, dim in MODELS[case["model"]]:
        for _ in range(2 * layers):
            t["pools"].append(_randn(g, num * block, heads, dim).to(torch.bfloat16))
    return t


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    kind = case["kind"]
    if kind == "verify":
        return _verify_inputs(case, seed)
    if kind == "copy":
        return _copy_inputs(case, seed)
    rng = np.random.default_rng(seed)
    block = case["block"]
    t = {}
    if kind == "fork":
        lens, size = _fork_lens(case)
        n = len(lens) * size
        slot = rng.permutation(n)                        # which slot a parent or child has
        mine = [_blocks(v, block) for v in lens]
        num = sum(mine) + n + 5
        order = rng.permutation(num).astype(np.int32)
        tables = np.full((n, max(mine) + 8), -1, np.int32)
        all_lens, parents = np.zeros(n, np.int32), np.full(n, -1, np.int32)
        at = 0
        for i, (v, c) in enumerate(zip(lens, mine)):
            p = slot[i * size]
            tables[p, :c] = order[at:at + c]
            at += c
            all_lens[p] = v
            parents[slot[i * size + 1:(i + 1) * size]] = p
        t["tables"], t["lens"], t["parents"] = _ints(tables), _ints(all_lens), _ints(parents)
        t["free"] = _ints(np.concatenate((np.full(at, -1, np.int32), order[at:])))
        t["taken"], t["served"] = _ints([at]), _full(0, 1)
        t["copies"] = _full(0, n, 3)
    else:
        live, _ = _live_blocks(case)
        held = _held(case)
        prefix = _blocks(case.get("prefix", 0), block)
        num = int((live + prefix) * case.get("loose", 1.0)) + 5
        order = rng.permutation(num).astype(np.int32)
        tables, at = _tables(case, order[prefix:], max(_blocks(m, block) for _, _, m in held) + 8)
        n = len(held)
        t["tables"], t["lens"] = _ints(tables), _ints([m for _, _, m in held])
        if kind == "rewind":
            t["drop"] = _ints([-1 if d is None else d for d in _drops(case)])
            t["free"] = _ints(np.concatenate((np.full(at, -1, np.int32), order[at:])))
            t["taken"], t["copies"] = _ints([at]), _full(0, n, 3)
        else:
            t["prefix_table"], t["tables_out"] = _ints(order[:prefix]), _full(0, *tables.shape)
            t["prefix_out"], t["free"], t["copies"] = _full(0, prefix), _full(0, num), _full(0, num // 2, 3)
    t["num"] = num
    t["n_copies"], t["taken_out"] = _full(0, 1), _full(0, 1)
    t["lens_out"], t["row_start"] = _full(0, n), _full(0, n + 1)
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
    """What a program using the entry points keeps: the caches, the batch, workspaces."""
    import hyperion_amd as hy
    kind = case["kind"]
    st["stream"] = _the_stream()
    st["dev"] = dev = {k: hy.DeviceView(v) for k, v in st.items() if isinstance(v, torch.Tensor)}
    need = 0
    if kind == "verify":
        need = hy.verify_batch_workspace_bytes(st["logits"].shape[0], case["vocab"], case["requests"], case["drafter"])
    elif kind == "copy":
        slots = st["num"] * case["block"]
        st["caches"] = []
        for layers, heads, dim in MODELS[case["model"]]:
            for _ in range(layers):
                cache = hy.KvCache(slots, heads, dim)
                for side, p in enumerate(cache.buffers()):
                    at = 2 * len(st["caches"]) + side
                    view = torch.as_tensor(_Raw(cache, p.value, (slots, heads, dim)), device="cuda").view(torch.bfloat16)
                    view.copy_(st["pools"][at])
                    st["pools"][at] = view
                st["caches"].append(cache)
        empty = hy.DeviceView(_full(0, 1))
        st["batch"] = hy.Batch(case["block"], st["num"], hy.DeviceView(_full(-1, 1, 1)), empty, hy.DeviceView(_full(0, 2)),
                               empty, empty)
    else:
        lens = dev["lens"] if kind == "compact" else dev["lens_out"]
        rows = hy.DeviceView(_full(0, 1))
        st["batch"] = hy.Batch(case["block"], st["num"], dev["tables"], lens, dev["row_start"], rows, rows,
                               case.get("prefix", 0), dev.get("prefix_table"))
        need = 0 if kind == "fork" else st["batch"].pages_workspace_bytes()
    st["workspace"] = hy.DeviceArray((need,), np.uint8) if need else None


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        _handles(case, st)
    torch.cuda.synchronize()
    return st


def _run_own(st):
    case, dev, s = st["case"], st.get("dev"), st["stream"]
    kind = case["kind"]
    if kind == "verify":
        from hyperion_amd import verify_batch
        verify_batch(dev["logits"], dev.get("draft_logits"), st["logits"].shape[0], case["vocab"], dev["row_start"],
                     case["requests"], dev["ids"], dev["configs"], None, dev["uniforms"], dev["accepted"], dev["rejected"],
                     dev["tokens"], dev["logprobs"], st["workspace"], s)
    elif kind == "fork":
        st["batch"].fork(dev["lens"], dev["parents"], dev["free"], dev["taken"], dev["taken_out"], dev["served"],
                         dev["copies"], dev["n_copies"], s)
    elif kind == "rewind":
        st["batch"].rewind(dev["lens"], dev["drop"], dev["free"], dev["taken"], dev["taken_out"], dev["copies"],
                           dev["n_copies"], st["workspace"], s)
    elif kind == "compact":
        st["batch"].compact(dev["tables_out"], dev["prefix_out"], dev["free"], dev["taken_out"], dev["copies"],
                            dev["n_copies"], st["workspace"], s)
    else:
        st["batch"].copy(st["caches"], dev["copies"], dev["n_copies"], s)


# ---- the plain forms ------------------------------------------------------------------------

def _filtered(logits, cfg):
    """Rows of probabilities after the filters, in the tokens' order, and ln of every token's share before them."""
    temperature, top_p, min_p = (cfg[:, c:c + 1].view(torch.float32).double() for c in (0, 2, 3))
    top_k = cfg[:, 1:2]
    x, index = torch.sort(logits.float() + 0.0, dim=-1, descending=True, stable=True)
    t = torch.where(temperature > 0, temperature, 1.0)
    w = torch.exp((x - x[:, :1]).double() / t)
    running = w.cumsum(-1)
    total = running[:, -1:]
    rank = torch.arange(x.shape[1], device="cuda")
    kept = torch.where(top_p < 1, running - w < top_p * total, True) & (w >= min_p)
    kept &= torch.where(top_k > 0, rank < top_k, True) & torch.where(temperature > 0, True, rank < 1)
    count = kept.long().cumprod(-1).sum(-1, keepdim=True)
    p = torch.where(rank < count, w, 0.0) / running.gather(-1, count - 1)
    share = (logits.double() - x[:, :1].double()) / t - torch.log(total)
    return torch.zeros_like(w).scatter_(-1, index, p), share


def _verify_plain(st):
    start = st["row_start"].long()
    n, total = start.shape[0] - 1, st["logits"].shape[0]
    row = torch.arange(total, device="cuda")
    request = torch.searchsorted(start[1:], row, right=True)
    rows = start[1:] - start[:-1]
    cfg = st["configs"][request]
    p, share = _filtered(st["logits"], cfg)
    last = row == start[1:][request] - 1
    draft = st["ids"].long().roll(-1)
    px = p.gather(-1, draft[:, None])[:, 0]
    if "draft_logits" in st:
        q, _ = _filtered(st["draft_logits"], cfg)
    else:
        q = torch.zeros_like(p).scatter_(-1, draft[:, None], 1.0)
    qx = q.gather(-1, draft[:, None])[:, 0]
    fails = last | (st["uniforms"].double() * qx >= px)
    first = torch.full((n,), total, device="cuda").scatter_reduce(0, request, torch.where(fails, row, total), "amin")
    accepted = first - start[:-1]
    st["accepted"].copy_(accepted)
    st["rejected"].copy_(rows - 1 - accepted)
    q = torch.where(last[first][:, None], 0.0, q[first])
    p = p[first]
    r = (p - q).clamp(min=0.0)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p)
    running = r.cumsum(-1)
    goal = st["uniforms"].double()[start[1:] - 1][:, None] * running[:, -1:]
    vocab = p.shape[1]
    most = torch.where(r > 0, torch.arange(vocab, device="cuda"), 0).amax(-1)
    token = torch.minimum((running <= goal).sum(-1), most)
    st["tokens"].copy_(token)
    follows = torch.where(row < first[request], draft, token[request])
    logprob = share.gather(-1, follows[:, None])[:, 0].float()
    st["logprobs"].copy_(torch.where(row <= first[request], logprob, st["logprobs"]))


def _fork_plain(st):
    block, num = st["case"]["block"], st["num"]
    lens, parents = st["lens"].long(), st["parents"].long()
    n = lens.shape[0]
    slot = torch.arange(n, device="cuda")
    p = parents.clamp(min=0)
    child = (parents >= 0) & (parents[p] < 0)
    have = torch.where(child, lens[p], 0)
    need = child & (have % block != 0)
    rank = need.long().cumsum(0)
    taken = st["taken"].long()
    ok = ~need | (rank <= num - taken)
    served = ok.long().cumprod(0).sum()
    child &= slot < served
    need &= slot < served
    entry = torch.arange(st["tables"].shape[1], device="cuda")
    held = child[:, None] & (entry < _blocks(have, block)[:, None])
    tables = torch.where(held, st["tables"][p], st["tables"])
    fresh = st["free"][(taken + rank - 1).clamp(max=num - 1)]
    tables = torch.where(need[:, None] & (entry == (have // block)[:, None]), fresh[:, None], tables)
    at = torch.where(need, rank - 1, n)
    copies = torch.cat((st["copies"], st["copies"][:1]))
    source = st["tables"][p].gather(1, (have // block)[:, None])[:, 0]
    copies[at] = torch.stack((source, fresh, (have % block).int()), 1)
    st["copies"].copy_(copies[:n])
    st["tables"].copy_(tables)
    st["lens_out"].copy_(torch.where(child, have, lens))
    st["n_copies"].copy_(need.sum())
    st["taken_out"].copy_(taken + need.sum())
    st["served"].copy_(served)


def _rewind_plain(st):
    """(No case here leaves a shared block partly filled, so there is nothing to copy.)"""
    block, num = st["case"]["block"], st["num"]
    lens, drop = st["lens"].long(), st["drop"].long()
    keep = torch.where((drop < 0) | (drop > lens), 0, lens - drop)
    entry = torch.arange(st["tables"].shape[1], device="cuda")
    held = entry < _blocks(keep, block)[:, None]
    gone = ~held & (entry < _blocks(lens, block)[:, None])
    table = st["tables"].long()
    kept = torch.zeros(num + 1, dtype=torch.bool, device="cuda")
    kept[torch.where(held, table, num).flatten()] = True
    kept[num] = True
    at = torch.arange(table.numel(), device="cuda")
    flat = torch.where(gone, table, num).flatten()
    place = torch.where(gone.flatten(), flat, num + 1 + at)   # (what is not given up in places of its own)
    first = torch.full((num + 1 + table.numel(),), table.numel(), device="cuda").scatter_reduce(0, place, at, "amin")
    back = ~kept[flat] & (first[place] == at)
    top = st["taken"].long() - back.sum()
    free = torch.cat((st["free"], st["free"][:1]))
    free[torch.where(back, top + back.cumsum(0) - 1, num)] = flat.int()
    st["free"].copy_(free[:num])
    st["taken_out"].copy_(top)
    st["lens_out"].copy_(keep)
    st["n_copies"].zero_()


def _compact_plain(st):
    block, num = st["case"]["block"], st["num"]
    table = st["tables"].long()
    entry = torch.arange(table.shape[1], device="cuda")
    held = entry < _blocks(st["lens"].long(), block)[:, None]
    live = torch.zeros(num + 1, dtype=torch.bool, device="cuda")
    live[torch.where(held, table, num).flatten()] = True
    live[st["prefix_table"].long()] = True
    live = live[:num]
    count = live.sum()
    ids = torch.arange(num, device="cuda")
    mover, hole = live & (ids >= count), ~live & (ids < count)
    cap = st["copies"].shape[0]
    copies = torch.cat((st["copies"], st["copies"][:1]))
    copies[torch.where(mover, mover.cumsum(0) - 1, cap), 0] = ids.int()
    copies[torch.where(hole, hole.cumsum(0) - 1, cap), 1] = ids.int()
    moves = mover.sum()
    copies[:, 2] = torch.where(torch.arange(cap + 1, device="cuda") < moves, block, copies[:, 2]).int()
    st["copies"].copy_(copies[:cap])
    to = torch.where(mover, copies[(mover.cumsum(0) - 1).clamp(min=0), 1].long(), ids).int()
    st["tables_out"].copy_(torch.where(held, to[table.clamp(min=0)], st["tables"]))
    st["prefix_out"].copy_(to[st["prefix_table"].long()])
    st["free"].copy_(torch.where(ids >= count, ids, st["free"]))
    st["taken_out"].copy_(count)
    st["n_copies"].copy_(moves)


def _copy_plain(st):
    block = st["case"]["block"]
    copies = st["copies"].long()
    j = torch.arange(block, device="cuda")
    there = (j < copies[:, 2:]).flatten()
    source, to = ((copies[:, c:c + 1] * block + j).flatten()[there] for c in (0, 1))
    for pool in st["pools"]:
        pool[to] = pool[source]


def run(st):
    kind = st["case"]["kind"]
    if own:
        _run_own(st)
    else:
        {"verify": _verify_plain, "fork": _fork_plain, "rewind": _rewind_plain, "compact": _compact_plain,
         "copy": _copy_plain}[kind](st)
    names = {"verify": ("accepted", "rejected", "tokens", "logprobs"),
             "fork": ("tables", "lens_out", "taken_out", "served", "copies", "n_copies"),
             "rewind": ("tables", "lens_out", "free", "taken_out", "n_copies"),
             "compact": ("tables_out", "prefix_out", "free", "taken_out", "copies", "n_copies"), "copy": ("pools",)}[kind]
    return {name: st[name] for name in names}


# ---- what a pass has to do -------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "verify":
        rows, n = _verify_rows(case), case["requests"]
        read = sum(rows) + (sum(rows) - n if case["drafter"] else 0)   # (nothing follows a request's last row)
        return {"bytes": 2 * case["vocab"] * read + 12 * sum(rows) + 40 * n, "flops": 0}
    if kind == "copy":
        token = sum(2 * 2 * layers * heads * dim for layers, heads, dim in MODELS[case["model"]])
        return {"bytes": 2 * token * sum(_copy_tokens(case)) + 12 * case["copies"], "flops": 0}
    block = case["block"]
    if kind == "fork":
        lens, size = _fork_lens(case)
        entries = sum(_blocks(n, block) for n in lens)
        part = sum(n % block != 0 for n in lens) * (size - 1)
        return {"bytes": 12 * size * len(lens) + 4 * entries * size + 20 * part, "flops": 0}
    held = _held(case)
    entries = sum(_blocks(n, block) for _, _, n in held)
    if kind == "rewind":
        back = sum(_blocks(n, block) - _blocks(n - (n if d is None else d), block) for d, (_, _, n) in zip(_drops(case), held))
        return {"bytes": 12 * len(held) + 4 * entries + 4 * back, "flops": 0}
    live = _live_blocks(case)[0] + _blocks(case["prefix"], block)
    num = int(live * case["loose"]) + 5
    moves = live * (num - live) // num   # of ids in random order
    return {"bytes": 4 * len(held) + 8 * entries + 8 * _blocks(case["prefix"], block) + 4 * (num - live) + 12 * moves,
            "flops": 0}


# ---- the same in 64 bits ---------------------------------------------------------------------

def _kept_weights(x, temperature, top_k, top_p, min_p):
    """One row's probabilities after the filters and ln of its tokens' shares before them, float64 on the device."""
    x = x.double()
    order = torch.sort(x, descending=True, stable=True).indices
    greedy = temperature <= 0
    w = torch.exp((x[order] - x[order[0]]) / (1.0 if greedy else temperature))
    mass = torch.cumsum(w, 0)
    keep = x.numel() if top_k <= 0 else min(x.numel(), top_k)
    if top_p < 1:
        keep = min(keep, int(torch.searchsorted(mass, top_p * mass[-1:]).item()) + 1)
    keep = min(keep, int((w >= min_p).sum().item()))
    keep = 1 if greedy else max(1, keep)
    p = torch.zeros_like(x)
    p[order[:keep]] = w[:keep] / mass[keep - 1]
    logs = torch.empty_like(x)
    logs[order] = torch.log(w / mass[-1])
    return p, logs


def _exact_verify(case, t):
    raw = np.ascontiguousarray(t["configs"].cpu().numpy())
    values = raw.view(np.float32).astype(np.float64)
    ids, u = t["ids"].tolist(), t["uniforms"].double().tolist()
    out = {"accepted": [], "rejected": [], "tokens": []}
    logprobs = [0.0] * len(ids)
    first = 0
    for n, f, top_k in zip(_verify_rows(case), values, raw[:, 1].tolist()):
        setting = (f[0], top_k, f[2], f[3])
        taken = 0
        while True:
            row = first + taken
            p, logs = _kept_weights(t["logits"][row], *setting)
            rest = p
            if taken == n - 1:
                break
            x = ids[row + 1]
            if case["drafter"]:
                q, _ = _kept_weights(t["draft_logits"][row], *setting)
            else:
                q = torch.zeros_like(p)
                q[x] = 1.0
            if not u[row] * q[x].item() < p[x].item():
                rest = torch.relu(p - q)
                if not rest.sum().item() > 0.0:
                    rest = p
                break
            logprobs[row] = logs[x].item()
            taken += 1
        running = torch.cumsum(rest, 0)
        token = int(torch.searchsorted(running, u[first + n - 1] * running[-1:], right=True).item())
        token = min(token, int(torch.nonzero(rest).max().item()))
        logprobs[first + taken] = logs[token].item()
        out["accepted"].append(taken)
        out["rejected"].append(n - 1 - taken)
        out["tokens"].append(token)
        first += n
    out = {k: torch.tensor(v, dtype=torch.int32) for k, v in out.items()}
    out["logprobs"] = torch.tensor(logprobs, dtype=torch.float64)
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return _exact_verify(case, _verify_inputs(case, seed))
    if kind != "copy":
        return None   # whole numbers
    t = _copy_inputs(case, seed)
    block = case["block"]
    source, to = [], []
    for a, b, tokens in t["copies"].tolist():
        source += range(a * block, a * block + tokens)
        to += range(b * block, b * block + tokens)
    pools = []
    for pool in t["pools"]:
        moved = pool.double()
        moved[to] = pool[source].double()
        pools.append(moved)
    return {"pools": pools}
