"""The serving-side operators of the framework: what is measured of each, on which cases, and their plain forms.

Five operators work on one another's data: rotary positions for queries and keys, a paged key/value cache with its
append, attention for a tree of drafted tokens over that cache, the attention weight that each cached key gathers, and
the eviction that goes by it.

A cache is ``k_pages``/``v_pages`` [pages, kv heads, page size, head dimension] with a ``block_table`` [batch, pages of a
sequence] and ``lengths`` [batch], both int32: slot ``s`` of sequence ``b`` is row ``s % page_size`` of page
``block_table[b, s // page_size]``. ``weights`` (fp32) and ``positions`` (int32) of the slots are [batch, kv heads, slots].
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step of 32 sequences: queries and keys of one token each; a call of a few microseconds
        {"name": "rotary decode", "op": "rotary", "batch": 32, "heads": 32, "kv_heads": 8, "tokens": 1, "dim": 64,
         "rotary_dim": 64, "layout": "half", "scaling": "linear", "far": 16384, "dtype": "fp16", "rows_first": False,
         "backward": False},
        # one layer's queries and keys of a training step, as a projection lays them out ([B, N, H, D]), one token short
        # of 8192, forward and backward
        {"name": "rotary training", "op": "rotary", "batch": 4, "heads": 32, "kv_heads": 32, "tokens": 8191, "dim": 64,
         "rotary_dim": 64, "layout": "interleaved", "scaling": "yarn", "far": 0, "dtype": "fp16", "rows_first": True,
         "backward": True},
        # the rows of a prompt's chunk go into the cache
        {"name": "append chunk", "op": "append", "batch": 4, "kv_heads": 8, "tokens": 2048, "dim": 64, "page": 64,
         "length": 6000, "spread": 0.5, "dtype": "fp16", "path": False},
        # the accepted nodes of each sequence's drafted tree go into the cache
        {"name": "append accepted", "op": "append", "batch": 32, "kv_heads": 8, "tokens": 16, "dim": 128, "page": 16,
         "length": 4000, "spread": 0.5, "dtype": "bf16", "path": True},
        # one token of one sequence of 1024, as many key heads as query heads: latency
        {"name": "decode one sequence", "op": "tree", "batch": 1, "heads": 8, "kv_heads": 8, "tokens": 1, "dim": 64,
         "page": 64, "length": 1024, "spread": 0.0, "dtype": "fp16"},
        # one token each of 32 sequences of unequal length, grouped heads: bandwidth
        {"name": "decode batch", "op": "tree", "batch": 32, "heads": 32, "kv_heads": 8, "tokens": 1, "dim": 64,
         "page": 16, "length": 16384, "spread": 0.5, "dtype": "fp16"},
        # drafted trees of 29 nodes for 8 sequences
        {"name": "tree batch", "op": "tree", "batch": 8, "heads": 32, "kv_heads": 8, "tokens": 29, "dim": 128,
         "page": 64, "length": 8192, "spread": 0.3, "dtype": "bf16"},
        # a wide tree over one long cache
        {"name": "tree long", "op": "tree", "batch": 1, "heads": 32, "kv_heads": 4, "tokens": 64, "dim": 64,
         "page": 128, "length": 65500, "spread": 0.0, "dtype": "fp16"},
        # the weight that the keys of 32 caches gather in a decoding step
        {"name": "weight decode", "op": "weight", "batch": 32, "heads": 32, "kv_heads": 8, "tokens": 1, "dim": 64,
         "page": 16, "length": 4096, "spread": 0.5, "dtype": "fp16"},
        # the weight that a long prompt's keys gather from its last 32 queries
        {"name": "weight window", "op": "weight", "batch": 1, "heads": 32, "kv_heads": 8, "tokens": 32, "dim": 128,
         "page": 64, "length": 65536, "spread": 0.0, "dtype": "bf16"},
        # 32 caches that grew by a sixteenth go back to their budget
        {"name": "evict batch", "op": "evict", "batch": 32, "kv_heads": 8, "dim": 64, "page": 16, "length": 4352,
         "spread": 0.1, "budget": 4096, "recent": 256, "sinks": 4, "dtype": "fp16"},
        # one long prompt's cache is cut to a quarter
        {"name": "evict prompt", "op": "evict", "batch": 1, "kv_heads": 8, "dim": 128, "page": 64, "length": 65536,
         "spread": 0.0, "budget": 16384, "recent": 1024, "sinks": 16, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["rotary", "append", "tree", "tree", "weight", "evict"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    c = {"op": op, "dim": dim, "kv_heads": kv_heads, "dtype": rng.choice(["fp16", "bf16"])}
    if op == "rotary":
        tokens = _log(rng, 1, 8192)
        batch = max(1, min(_log(rng, 1, 64), 16384 // tokens))
        return c | {"batch": batch, "heads": kv_heads * rng.choice([1, 2, 4]), "tokens": tokens,
                    "rotary_dim": rng.choice([dim, dim // 2, 48]), "layout": rng.choice(["half", "interleaved"]),
                    "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "far": rng.choice([0, 5000, 1000000]),
                    "dtype": rng.choice(["fp16", "bf16", "fp32"]), "rows_first": rng.random() < 0.5,
                    "backward": rng.random() < 0.5}
    page = rng.choice([16, 32, 64, 128])
    c |= {"page": page, "spread": rng.choice([0.0, 0.3, 0.9])}
    if op == "append":
        tokens = _log(rng, 1, 2048)
        batch = max(1, min(_log(rng, 1, 64), 8192 // tokens))
        return c | {"batch": batch, "tokens": tokens, "length": _log(rng, 1, 8000), "path": rng.random() < 0.5}
    length = _log(rng, 1, 65536)
    batch = max(1, min(_log(rng, 1, 64), 200000 // length))
    if op == "evict":
        budget = max(1, int(length * rng.uniform(0.2, 1.0)))
        recent = int(budget * rng.uniform(0.0, 0.5))
        return c | {"batch": batch, "length": length, "budget": budget, "recent": recent,
                    "sinks": min(4, budget - recent)}
    group = rng.choice([1, 2, 4, 7, 8])
    tokens = max(1, min(_log(rng, 1, 64), 60000000 // (batch * kv_heads * group * length)))
    return c | {"batch": batch, "heads": kv_heads * group, "tokens": tokens, "length": length}


def _lengths(case):
    """Lengths of the sequences: from (1 - spread) * length up to length, in a scattered order."""
    b, top = case["batch"], case["length"]
    return [max(1, top - int(case["spread"] * top * ((i * 37 + 11) % b) / b)) for i in range(b)]


def _counts(case):
    """How many of a sequence's new rows are appended."""
    t = case["tokens"]
    return [1 + (i * 5 + 3) % t if case["path"] else t for i in range(case["batch"])]


# --------------------------------------------------------------------------------------------------------- inputs

def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _pages(case, g, slots):
    """A cache whose pages lie scattered among a few more than it uses; every slot holds something."""
    per = -(-slots // case["page"])
    n = case["batch"] * per
    total = n + 3
    dtype, shape = DTYPES[case["dtype"]], (total, case["kv_heads"], case["page"], case["dim"])
    table = torch.randperm(total, generator=g, device="cuda")[:n].reshape(case["batch"], per).int()
    return {"k_pages": torch.randn(shape, generator=g, device="cuda", dtype=dtype),
            "v_pages": torch.randn(shape, generator=g, device="cuda", dtype=dtype), "block_table": table,
            "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")}


def _tree(case, g):
    """Parents drawn at random: node i hangs below one of the nodes before it, node 0 is the root; a node sees its
    ancestors and itself (the places where a high power of "itself or its parent" is not zero)."""
    b, t = case["batch"], case["tokens"]
    parent = (torch.rand((b, t), generator=g, device="cuda") * torch.arange(t, device="cuda")).long()
    step = torch.nn.functional.one_hot(parent, t).double()
    step[:, 0] = 0
    return torch.linalg.matrix_power(step + torch.eye(t, dtype=torch.float64, device="cuda"), 64) > 0


def _log_sum_exp(s, case):
    """The row statistics that an attention over the cache alone has handed out."""
    length = int(s["lengths"].max())
    k = _rows(s["k_pages"], s["block_table"])[:, :, :length].float()
    b, h, t, d = s["query"].shape
    q = s["query"].float().reshape(b, case["kv_heads"], -1, d)
    score = q @ k.transpose(-1, -2) * s["scale"]
    score = score.masked_fill(_behind(s["lengths"], length)[:, None, None], -math.inf)
    return torch.logsumexp(score, -1).reshape(b, h, t)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dtype, d = case["op"], DTYPES[case["dtype"]], case["dim"]
    b, t = case["batch"], case.get("tokens")
    s = {"op": op, "case": case}
    if op == "rotary":
        s |= {"layout": case["layout"], "backward": case["backward"]}
        for name, heads in (("query", case["heads"]), ("key", case["kv_heads"])):
            shape = (b, t, heads, d) if case["rows_first"] else (b, heads, t, d)
            for kind in (name, "grad_" + name) if case["backward"] else (name,):
                x = _randn(g, *(shape if kind == name else (b, heads, t, d)), dtype=dtype)
                s[kind] = x.transpose(1, 2) if case["rows_first"] and kind == name else x
        first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")
        s["frequencies"], s["factor"] = _frequencies(case)
        return s
    if op == "append":
        top = case["length"] + t
        s |= _pages(case, g, top)
        s["key"], s["value"] = (_randn(g, b, case["kv_heads"], t, d, dtype=dtype) for _ in range(2))
        slots = s["block_table"].shape[1] * case["page"]
        s["weights"] = torch.rand((b, case["kv_heads"], slots), generator=g, device="cuda")
        s["positions"] = torch.arange(slots, device="cuda", dtype=torch.int32).repeat(b, case["kv_heads"], 1)
        s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
        s["path"], s["new_positions"] = None, (s["lengths"][:, None] + torch.arange(t, device="cuda")).int()
        if case["path"]:  # accepted nodes: the first `count` of an increasing choice
            some = torch.rand((b, t), generator=g, device="cuda").argsort(-1)
            at = torch.arange(t, device="cuda")
            s["path"] = torch.where(at < s["counts"][:, None], some, t).sort(-1).values.clamp(max=t - 1).int()
        return s
    s |= _pages(case, g, case["length"])
    if op in ("tree", "weight"):
        s["scale"] = d ** -0.5
        # a spread of scores as attention has it: a few keys stand out for each query
        s["query"] = _randn(g, b, case["heads"], t, d, dtype=dtype, scale=1.5)
    if op == "tree":
        s["k_tree"], s["v_tree"] = (_randn(g, b, case["kv_heads"], t, d, dtype=dtype) for _ in range(2))
        s["tree_mask"] = _tree(case, g)
    elif op == "weight":
        slots = s["block_table"].shape[1] * case["page"]
        s["lse"] = _log_sum_exp(s, case)
        s["weights"] = torch.rand((b, case["kv_heads"], slots), generator=g, device="cuda")
    else:
        slots = s["block_table"].shape[1] * case["page"]
        # weights of a cache in use: over several orders of magnitude, a good part of them zero (equal)
        w = torch.exp(3 * _randn(g, b, case["kv_heads"], slots) - 4)
        s["weights"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.2, 0.0, w)
        # an earlier eviction has left the slots in no order
        order = torch.rand(w.shape, generator=g, device="cuda").masked_fill(_behind(s["lengths"], slots)[:, None], 2.0)
        s["positions"] = order.argsort(-1).argsort(-1).int()
    return s


# ------------------------------------------------------------------------------------------------------ plain forms

def _frequencies(case):
    """Angles a position apart (radians, fp64) and the factor on the rotated elements, for contexts longer than trained."""
    r, base, longer, trained = case["rotary_dim"], 10000.0, 4.0, 4096
    if case["scaling"] == "ntk":
        base *= longer ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if case["scaling"] == "linear":
        f = f / longer
    if case["scaling"] == "yarn":
        def pair(turns):
            return r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / longer * ramp + f * (1 - ramp)
        return f.cuda(), 0.1 * math.log(longer) + 1
    return f.cuda(), 1.0


def _rows(pages, table):
    """The slots of each sequence in order: [B, Hk, slots, D]."""
    x = pages[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _behind(lengths, slots):
    return torch.arange(slots, device=lengths.device) >= lengths[:, None]


def _rotate(x, positions, frequencies, factor, layout, wide):
    """The rotation in the type `wide`, unrounded; the angles always in fp64."""
    angle = (positions.double()[:, None, :, None] * frequencies)
    c, s = (angle.cos() * factor).to(wide), (angle.sin() * factor).to(wide)
    r = 2 * frequencies.numel()
    x = x.to(wide)
    y = x.clone()
    one, two = ((slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r)))
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    return y


def _run_rotary(s):
    args = (s["positions"], s["frequencies"], s["factor"], s["layout"], torch.float32)
    q, k = s["query"], s["key"]
    out = [_rotate(x, *args).to(x.dtype).contiguous() for x in (q, k)]
    if s["backward"]:  # a rotation's transpose turns the other way
        back = (s["positions"], -s["frequencies"], s["factor"], s["layout"], torch.float32)
        out += [_rotate(x, *back).to(x.dtype) for x in (s["grad_query"], s["grad_key"])]
    return out


def _run_append(s):
    b, hk, n, d = s["key"].shape
    at = s["lengths"].long()[:, None] + torch.arange(n, device="cuda")
    new = torch.arange(n, device="cuda") < s["counts"][:, None]
    pages, size = s["block_table"].long(), s["k_pages"].shape[2]
    page, row = pages.gather(1, at // size), at % size
    rows = torch.arange(n, device="cuda").expand(b, n) if s["path"] is None else s["path"].long()
    pick = rows[:, None, :, None].expand(b, hk, n, d)
    put = new[:, :, None, None]  # behind a sequence's count its slots keep what they hold
    s["k_pages"][page, :, row] = torch.where(put, s["key"].gather(2, pick).transpose(1, 2), s["k_pages"][page, :, row])
    s["v_pages"][page, :, row] = torch.where(put, s["value"].gather(2, pick).transpose(1, 2), s["v_pages"][page, :, row])
    at = at[:, None].expand(b, hk, n)
    new = new[:, None]
    s["weights"].scatter_(2, at, torch.where(new, 0.0, s["weights"].gather(2, at)))
    given = s["new_positions"].gather(1, rows)[:, None]
    s["positions"].scatter_(2, at, torch.where(new, given, s["positions"].gather(2, at)))
    return s["k_pages"], s["v_pages"], s["weights"], s["positions"], s["lengths"] + s["counts"]


def _run_tree(s):
    b, h, t, d = s["query"].shape
    hk = s["k_tree"].shape[1]
    q = s["query"].float().reshape(b, hk, h // hk * t, d)
    k = torch.cat([_rows(s["k_pages"], s["block_table"]).float(), s["k_tree"].float()], 2)
    v = torch.cat([_rows(s["v_pages"], s["block_table"]).float(), s["v_tree"].float()], 2)
    slots = k.shape[2] - t
    hidden = torch.cat([_behind(s["lengths"], slots)[:, None].expand(b, t, slots), ~s["tree_mask"]], -1)
    hidden = hidden[:, None, None].expand(b, 1, h // hk, t, slots + t).reshape(b, 1, h // hk * t, -1)
    score = (q @ k.transpose(-1, -2)).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)  # nothing to see: every weight is zero
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, h, t, d).to(s["query"].dtype), (top + total.log()).reshape(b, h, t)


def _run_weight(s):
    b, h, t, d = s["query"].shape
    hk = s["k_pages"].shape[1]
    q = s["query"].float().reshape(b, hk, -1, d)
    k = _rows(s["k_pages"], s["block_table"]).float()
    p = (q @ k.transpose(-1, -2)).mul_(s["scale"]).sub_(s["lse"].reshape(b, hk, -1, 1)).exp_()
    p.masked_fill_(_behind(s["lengths"], k.shape[2])[:, None, None], 0.0)
    s["weights"] += p.sum(2)
    return s["weights"]


def _run_evict(s):
    c = s["case"]
    budget = c["budget"]
    b, hk, slots = s["weights"].shape
    at = torch.arange(slots, device="cuda")
    behind = _behind(s["lengths"], slots)[:, None].expand(b, hk, slots)
    last = s["positions"].masked_fill(behind, -1).amax(-1, keepdim=True)
    safe = (s["positions"] > last - c["recent"]) | (s["positions"] < c["sinks"])
    value = torch.where(safe, math.inf, s["weights"]).masked_fill(behind, -math.inf)
    order = value.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(behind).scatter_(-1, order[..., :budget], True) & ~behind
    # the i-th dropped slot before the budget takes the i-th kept slot behind it
    hole, mover = ~kept & (at < budget) & ~behind, kept & (at >= budget)
    to = (~hole).to(torch.int8).sort(dim=-1, stable=True).indices
    come = (~mover).to(torch.int8).sort(dim=-1, stable=True).indices
    n = min(budget, max(slots - budget, 0))  # no more of them than that
    to, come = to[..., :n], come[..., :n]
    come = torch.where(at[:n] < mover.sum(-1, keepdim=True), come, to)
    bi, hi = torch.arange(b, device="cuda")[:, None, None], torch.arange(hk, device="cuda")[:, None]
    page, table = s["k_pages"].shape[2], s["block_table"].long()
    page_to, page_come = table[bi, to // page], table[bi, come // page]
    s["k_pages"][page_to, hi, to % page] = s["k_pages"][page_come, hi, come % page]
    s["v_pages"][page_to, hi, to % page] = s["v_pages"][page_come, hi, come % page]
    lengths = s["lengths"].clamp(max=budget)
    gone = _behind(lengths, slots)[:, None]
    weights = s["weights"].scatter(2, to, s["weights"].gather(2, come)).masked_fill_(gone, 0.0)
    positions = s["positions"].scatter(2, to, s["positions"].gather(2, come)).masked_fill_(gone, -1)
    return s["k_pages"], s["v_pages"], weights, positions, lengths


# -------------------------------------------------------------------------------------------------- the calls users make

def _own(s):
    import flash_attention_2_lab_b200 as fa

    op = s["op"]
    if op == "rotary":
        q, k = s["query"], s["key"]
        if s["backward"]:
            q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = fa.apply_rotary(q, k, s["positions"], s["frequencies"], layout=s["layout"], attention_factor=s["factor"])
        if not s["backward"]:
            return out
        return [*out, *torch.autograd.grad(out, (q, k), (s["grad_query"], s["grad_key"]))]
    if op == "append":
        lengths = fa.append_to_cache(s["key"], s["value"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"],
                                     path=s["path"], counts=s["counts"], weights=s["weights"],
                                     positions=s["positions"], new_positions=s["new_positions"])
        return s["k_pages"], s["v_pages"], s["weights"], s["positions"], lengths
    if op == "tree":
        return fa.tree_attention(s["query"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"], s["k_tree"],
                                 s["v_tree"], tree_mask=s["tree_mask"], scale=s["scale"])
    if op == "weight":
        return fa.accumulate_attention_weight(s["weights"], s["query"], s["k_pages"], s["block_table"], s["lengths"],
                                              s["lse"], scale=s["scale"])
    c = s["case"]
    weights, positions, lengths = fa.evict_from_cache(s["k_pages"], s["v_pages"], s["block_table"], s["lengths"],
                                                      s["weights"], s["positions"], c["budget"], recent=c["recent"],
                                                      sinks=c["sinks"])
    return s["k_pages"], s["v_pages"], weights, positions, lengths


PLAIN = {"rotary": _run_rotary, "append": _run_append, "tree": _run_tree, "weight": _run_weight, "evict": _run_evict}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------- work

def work(case):
    op, d, hk, b = case["op"], case["dim"], case["kv_heads"], case["batch"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "rotary":
        rows = b * case["tokens"] * (case["heads"] + hk)
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * (2 * rows * d * size + 8 * b * case["tokens"] + 4 * case["rotary_dim"]),
                "flops": passes * 3 * rows * case["rotary_dim"]}
    if op == "append":  # rows of K and V, their weights and positions
        n = sum(_counts(case)) * hk
        return {"bytes": n * (2 * 2 * d * size + 8), "flops": 0}
    n = sum(_lengths(case))
    if op == "evict":
        # every slot's weight and position are looked at and written anew; of the rows only those move whose place is
        # behind the budget: about as many as a random choice leaves there
        top = case["budget"]
        moved = sum(max(0, x - top) * top / x for x in _lengths(case)) * hk
        slots = -(-case["length"] // case["page"]) * case["page"] * b * hk
        return {"bytes": 8 * n * hk + 8 * slots + moved * 2 * 2 * d * size, "flops": 0}
    rows, t = b * case["heads"] * case["tokens"], case["tokens"]
    pairs = case["heads"] * t * n
    if op == "weight":
        return {"bytes": n * hk * (d * size + 8) + rows * (d * size + 4), "flops": 2 * d * pairs}
    own_keys = b * case["heads"] * t * t
    return {"bytes": 2 * (n + b * t) * hk * d * size + rows * (2 * d * size + 4) + b * t * t,
            "flops": 4 * d * (pairs + own_keys)}


# ------------------------------------------------------------------------------------------------------------ exact

def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rotary":  # as products of complex numbers
        def turned(x, sign):
            x, r = x.double(), case["rotary_dim"]
            head = x[..., :r]
            z = (torch.view_as_complex(head.reshape(*head.shape[:-1], r // 2, 2).contiguous())
                 if case["layout"] == "interleaved" else torch.complex(*(h.contiguous() for h in head.chunk(2, -1))))
            angle = sign * s["positions"].double()[:, None, :, None] * s["frequencies"]
            z = z * torch.polar(torch.full_like(angle, s["factor"]), angle)
            y = (torch.view_as_real(z).flatten(-2) if case["layout"] == "interleaved" else torch.cat([z.real, z.imag], -1))
            return torch.cat([y, x[..., r:]], -1)
        out = [turned(s["query"], 1), turned(s["key"], 1)]
        return out + [turned(s["grad_query"], -1), turned(s["grad_key"], -1)] if case["backward"] else out
    if op in ("append", "evict"):
        return None  # rows are copied and whole numbers are compared: nothing is computed
    # attention one sequence at a time, over just the slots that it has
    hk, group, t = case["kv_heads"], case["heads"] // case["kv_heads"], case["tokens"]
    outs, stats, weights = [], [], []
    for b, n in enumerate(_lengths(case)):
        at = s["block_table"][b].long()
        k = s["k_pages"][at].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()
        q = s["query"][b].double().unflatten(0, (hk, group))
        score = torch.einsum("hgtd,hnd->hgtn", q, k) * s["scale"]
        if op == "weight":
            got = s["weights"][b].double()
            got[:, :n] += torch.exp(score - s["lse"][b].double().unflatten(0, (hk, group))[..., None]).sum((1, 2))
            weights.append(got)
            continue
        v = s["v_pages"][at].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()
        drafted = torch.einsum("hgtd,hnd->hgtn", q, s["k_tree"][b].double()) * s["scale"]
        drafted = torch.where(s["tree_mask"][b], drafted, -math.inf)
        lse = torch.logaddexp(torch.logsumexp(score, -1), torch.logsumexp(drafted, -1))
        o = (torch.einsum("hgtn,hnd->hgtd", torch.exp(score - lse[..., None]), v)
             + torch.einsum("hgtn,hnd->hgtd", torch.exp(drafted - lse[..., None]), s["v_tree"][b].double()))
        outs.append(o.flatten(0, 1))
        stats.append(lse.flatten(0, 1))
    return torch.stack(weights) if op == "weight" else (torch.stack(outs), torch.stack(stats))
