"""Operators of drafted decoding over a paged K/V cache, and the cases they are measured on.

Five operators: the plan of a step (block tables, slot map, positions, tree masks, work units), the write of K/V rows
into pages, attention of a tree of drafted tokens over the pages, acceptance of the tree against the logits, and the
compaction of the accepted rows.  `run` computes them in plain torch, or, where `own` is true, calls
``manual_whisper_amd.paged``.

Request b has kept[b] tokens in its pages and appends fresh[b] rows in this step: the nodes of its tree, parents
before children, node 0 the root (or a plain chain of tokens where there are no parents).
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64          # keys: the granule of the work units


def listed():
    return [
        # a step of 16 recordings with a tree of 8 drafted tokens each: pages of 64, at most 448 + 64 positions
        {"name": "plan, a step of trees", "op": "plan", "batch": 16, "page": 64, "max_pages": 8, "kept_min": 20, "kept": 430,
         "fresh_min": 8, "fresh": 8, "tree": True, "tight": 0.0},
        # admission of a queue of prompts of very different lengths into small pages; the pool holds most of them
        {"name": "plan, prompts", "op": "plan", "batch": 256, "page": 16, "max_pages": 2304, "kept_min": 0, "kept": 30000,
         "fresh_min": 1, "fresh": 5000, "tree": False, "tight": 0.1},
        # the K/V rows of that step's trees, one layer of large-v3's decoder (20 heads of 64), from the fused q|k|v rows
        {"name": "write, a step, f16", "op": "write", "batch": 16, "heads": 20, "kv_heads": 20, "dim": 64, "page": 64,
         "kept_min": 20, "kept": 430, "fresh_min": 8, "fresh": 8, "type": "f16", "cache": "f16"},
        # the rows of long prompts into an e4m3 cache (grouped heads of 128)
        {"name": "write, prompts, e4m3", "op": "write", "batch": 12, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "kept_min": 0, "kept": 900, "fresh_min": 300, "fresh": 4000, "type": "bf16", "cache": "e4m3"},
        # the attention of that step: 16 recordings, 20 heads of 64, trees of 8
        {"name": "attend, a step, f16", "op": "attend", "batch": 16, "heads": 20, "kv_heads": 20, "dim": 64, "page": 64,
         "kept_min": 20, "kept": 430, "fresh_min": 8, "fresh": 8, "tree": True, "type": "f16", "cache": "f16"},
        # one token per request over long, ragged caches (no draft at hand)
        {"name": "attend, one row, bf16", "op": "attend", "batch": 8, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "kept_min": 4000, "kept": 65000, "fresh_min": 1, "fresh": 1, "tree": False, "type": "bf16", "cache": "bf16"},
        # wide trees over caches of some thousand tokens: the products count here
        {"name": "attend, wide trees, bf16", "op": "attend", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "kept_min": 300, "kept": 8000, "fresh_min": 20, "fresh": 61, "tree": True, "type": "bf16", "cache": "bf16"},
        # chains of drafted tokens, eight query heads to one K/V head, the cache in e4m3
        {"name": "attend, chains, e4m3", "op": "attend", "batch": 24, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "kept_min": 1000, "kept": 16000, "fresh_min": 3, "fresh": 16, "tree": False, "type": "f16", "cache": "e4m3"},
        # 16 trees of 8 against the vocabulary of large-v3, with the suppressed ids
        {"name": "accept, a step, f32", "op": "accept", "batch": 16, "nodes_min": 8, "nodes": 8, "vocab": 51866, "type": "f32",
         "suppress": True},
        # larger trees of many requests against a large vocabulary
        {"name": "accept, many rows, bf16", "op": "accept", "batch": 48, "nodes_min": 9, "nodes": 45, "vocab": 128000,
         "type": "bf16", "suppress": False},
        # the accepted rows of that step in all 32 layers
        {"name": "compact, a step, f16", "op": "compact", "batch": 16, "layers": 32, "kv_heads": 20, "dim": 64, "page": 64,
         "kept_min": 20, "kept": 430, "nodes_min": 8, "nodes": 8, "cache": "f16"},
        # deep accepted paths of many requests in a deep model, e4m3
        {"name": "compact, long paths, e4m3", "op": "compact", "batch": 64, "layers": 48, "kv_heads": 8, "dim": 128, "page": 16,
         "kept_min": 0, "kept": 160, "nodes_min": 16, "nodes": 60, "cache": "e4m3"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "accept", "compact"])
    page = rng.choice([16, 32, 64, 128])
    heads, kv_heads, dim = rng.choice([(20, 20, 64), (6, 6, 64), (16, 1, 64), (12, 4, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128)])
    if op == "plan":
        tree = rng.random() < 0.5
        fresh = _log(rng, 1, 128) if tree else _log(rng, 1, 5000)
        kept = _log(rng, 1, 30000)
        return {"op": op, "batch": _log(rng, 1, 256), "page": page, "max_pages": (kept + fresh) // page + rng.randint(1, 9),
                "kept_min": kept // 4, "kept": kept, "fresh_min": max(1, fresh // 3), "fresh": fresh, "tree": tree,
                "tight": rng.choice([0.0, 0.0, 0.2])}
    if op == "write":
        cache = rng.choice(["f16", "bf16", "e4m3"])
        fresh = _log(rng, 1, 2000)
        return {"op": op, "batch": _log(rng, 1, 24), "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "kept_min": 0,
                "kept": _log(rng, 1, 900), "fresh_min": max(1, fresh // 3), "fresh": fresh,
                "type": cache if cache != "e4m3" else rng.choice(["f16", "bf16"]), "cache": cache}
    if op == "attend":
        cache = rng.choice(["f16", "bf16", "e4m3"])
        fresh = _log(rng, 1, 64)
        kept = _log(rng, 1, 16000)
        batch = max(1, min(_log(rng, 1, 64), 250000 // (kept + 64), 60000000 // (heads * fresh * (kept + fresh))))
        return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "kept_min": kept // 5,
                "kept": kept, "fresh_min": max(1, fresh // 2), "fresh": fresh, "tree": rng.random() < 0.6,
                "type": cache if cache != "e4m3" else rng.choice(["f16", "bf16"]), "cache": cache}
    if op == "accept":
        nodes = _log(rng, 1, 60)
        vocab = _log(rng, 1000, 128000)
        return {"op": op, "batch": max(1, min(_log(rng, 1, 64), 100000000 // (nodes * vocab))), "nodes_min": max(1, nodes // 2),
                "nodes": nodes, "vocab": vocab, "type": rng.choice(["f32", "f16", "bf16"]), "suppress": rng.random() < 0.5}
    nodes = _log(rng, 2, 64)
    return {"op": op, "batch": _log(rng, 1, 48), "layers": _log(rng, 1, 40), "kv_heads": min(kv_heads, 8), "dim": dim,
            "page": min(page, 64), "kept_min": 0, "kept": _log(rng, 1, 160), "nodes_min": max(1, nodes // 2), "nodes": nodes,
            "cache": rng.choice(["f16", "bf16", "e4m3"])}


# ------------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(g, n, *ranges):
    """For each (low, high) n lengths spread evenly over their logarithm, high among them, paired anyhow but always the same
    way; the seed says which request has which."""
    order = torch.randperm(n, generator=g, device="cuda")
    fixed = torch.Generator()
    fixed.manual_seed(n)
    got = []
    for low, high in ranges:
        u = 1 - torch.randperm(n, generator=fixed) / n
        x = torch.exp(math.log(low + 1) + u * (math.log(high + 1) - math.log(low + 1))) - 1
        got.append(x.round().clamp(low, high).to(torch.int32).cuda()[order])
    return got


def _parents(g, rows, row_start, seq, own_index):
    """Drafts as they come: mostly one long branch with others beside it; node 0 is the root."""
    u = torch.rand(rows, generator=g, device="cuda")
    back = torch.where(u < 0.55, torch.ones_like(u), 1 + torch.floor(torch.rand(rows, generator=g, device="cuda") * 6)).to(torch.int32)
    return torch.where(own_index == 0, torch.full_like(own_index, -1), (own_index - back).clamp(min=0)).to(torch.int32)


def _rows_of(fresh):
    """row_start [B + 1], and for each row its request and its index there."""
    start = torch.zeros(fresh.numel() + 1, dtype=torch.int32, device=fresh.device)
    start[1:] = torch.cumsum(fresh, 0)
    rows = int(start[-1])
    seq = torch.repeat_interleave(torch.arange(fresh.numel(), device=fresh.device), fresh.long(), output_size=rows)
    return start, rows, seq, (torch.arange(rows, device=fresh.device) - start[seq]).to(torch.int32)


def _table(g, lengths, page, spare):
    """Pages of a pool in no order, given to requests of these lengths; -1 behind a request's last page."""
    need = (lengths + page - 1) // page
    most, total = max(1, int(need.max())), int(need.sum())
    n_pages = total + spare
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(most, device="cuda")
    at = (torch.cumsum(need, 0) - need)[:, None] + col[None]
    return torch.where(col[None] < need[:, None], order[at.clamp(max=n_pages - 1)], torch.full_like(at, -1, dtype=torch.int32)), n_pages


def _fill(g, shape, cache):
    """A cache's values as a model leaves them: heads of different size."""
    x = torch.empty(shape, dtype=torch.bfloat16 if cache == "bf16" else torch.float16, device="cuda").normal_(generator=g)
    x *= (0.5 + torch.rand(shape[-3], generator=g, device="cuda"))[:, None, None].to(x.dtype)
    return x


def _caches(g, shape, cache):
    """k, v (and row scales of an e4m3 cache): [..., pages, heads, page, dim]."""
    if cache != "e4m3":
        return {"k": _fill(g, shape, cache), "v": _fill(g, shape, cache)}
    s = {}
    for name in ("k", "v"):
        code = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
        code[(code & 0x7F) == 0x7F] = 0x3C                     # no NaN codes: 1.5 in their place
        s[name] = code
        s[name + "_scale"] = (0.5 + torch.rand(shape[:-1], generator=g, device="cuda")) / 448
    return s


def prepare(case, seed):
    g = _generator(seed)
    op, batch = case["op"], case["batch"]
    s = {"op": op}
    if op in ("plan", "write", "attend"):
        s["kept"], s["fresh"] = _lengths(g, batch, (case["kept_min"], case["kept"]), (case["fresh_min"], case["fresh"]))
        start, rows, seq, index = _rows_of(s["fresh"])
        s["rows"] = rows
    if op == "plan":
        page = case["page"]
        held = (s["kept"] + page - 1) // page                  # what the kept tokens occupy; every sixth holds pages too many
        extra = torch.where(torch.rand(batch, generator=g, device="cuda") < 1 / 6, 1 + (s["fresh"] + page - 1) // page + 1, torch.zeros_like(held))
        s["pages"] = torch.minimum(held + extra, torch.full_like(held, case["max_pages"])).to(torch.int32)
        grow = ((s["kept"] + s["fresh"] + page - 1) // page - s["pages"]).clamp(min=0)
        n_free = max(0, int(int(grow.sum()) * (1 - case["tight"])) + (8 if case["tight"] == 0 else 0))
        total = int(s["pages"].sum())
        order = torch.randperm(total + n_free, generator=g, device="cuda").to(torch.int32)
        col = torch.arange(case["max_pages"], device="cuda")
        at = (torch.cumsum(s["pages"], 0) - s["pages"])[:, None] + col[None]
        s["table"] = torch.where(col[None] < s["pages"][:, None], order[at.clamp(max=max(0, total + n_free - 1))], torch.full_like(at, -1, dtype=torch.int32))
        s["free"] = torch.cat([order[total:], torch.full((total,), -1, dtype=torch.int32, device="cuda")])
        s["n_free"] = torch.tensor([n_free], dtype=torch.int32, device="cuda")
        s["page"], s["units"], s["chunk"] = page, _cut(8, case["max_pages"] * page), 512
        s["parents"] = _parents(g, rows, start, seq, index) if case["tree"] else None
        s["words"] = (case["fresh"] + 31) // 32
    elif op == "write":
        table, n_pages = _table(g, s["kept"] + s["fresh"], case["page"], 3)
        at = s["kept"][seq] + index
        s["slots"] = table[seq, at // case["page"]].long() * case["page"] + at % case["page"]
        s["slots"][torch.rand(rows, generator=g, device="cuda") < 0.01] = -1            # rows of requests that were refused
        s.update(_caches(g, (n_pages, case["kv_heads"], case["page"], case["dim"]), case["cache"]))
        qkv = torch.empty((rows, case["heads"] + 2 * case["kv_heads"], case["dim"]), dtype=TYPES[case["type"]], device="cuda").normal_(generator=g)
        s["k_rows"], s["v_rows"] = qkv[:, case["heads"]:case["heads"] + case["kv_heads"]], qkv[:, case["heads"] + case["kv_heads"]:]
    elif op == "attend":
        s["table"], n_pages = _table(g, s["kept"] + s["fresh"], case["page"], 3)
        s["row_start"], s["nodes"] = start, case["fresh"]
        s["mask"] = None
        if case["tree"]:
            parents = _parents(g, rows, start, seq, index)
            s["mask"] = _words(_ancestors(parents, start, seq, index, batch, case["fresh"])[seq, index.long()], (case["fresh"] + 31) // 32)
        columns = case["fresh"] * (case["heads"] // case["kv_heads"])        # query columns that share a K/V head
        s["units"], s["unit_start"] = _units(s["kept"], s["fresh"], torch.ones_like(s["kept"]),
                                             _cut(case["kv_heads"], s["table"].shape[1] * case["page"]), max(512, 4 * columns))
        s.update(_caches(g, (n_pages, case["kv_heads"], case["page"], case["dim"]), case["cache"]))
        qkv = torch.empty((rows, case["heads"] + 2 * case["kv_heads"], case["dim"]), dtype=TYPES[case["type"]], device="cuda").normal_(generator=g)
        s["q"] = qkv[:, :case["heads"]] * 1
        if case["kv_heads"] == case["heads"]:
            s["q"] = qkv[:, :case["heads"]]                    # a view into the fused rows
    elif op == "accept":
        fresh, = _lengths(g, batch, (case["nodes_min"], case["nodes"]))
        start, rows, seq, index = _rows_of(fresh)
        s["row_start"], s["depth"] = start, case["nodes"]
        s["parents"] = _parents(g, rows, start, seq, index)
        s["logits"] = torch.empty((rows, case["vocab"]), dtype=TYPES[case["type"]], device="cuda").normal_(generator=g)
        s["suppress"] = (torch.rand(case["vocab"], generator=g, device="cuda") < 0.01).to(torch.uint8) if case["suppress"] else None
        s["tokens"] = torch.randint(0, case["vocab"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        # a draft that is right four times out of five: the parent's choice, as the model would make it
        choice = torch.where(s["suppress"][None].bool(), torch.full_like(s["logits"], -math.inf), s["logits"]).argmax(1) if case["suppress"] else s["logits"].argmax(1)
        right = torch.rand(rows, generator=g, device="cuda") < 0.8
        up = (start[seq] + s["parents"].clamp(min=0)).long()
        s["tokens"] = torch.where(right, choice[up].to(torch.int32), s["tokens"])
    else:
        kept, fresh = _lengths(g, batch, (case["kept_min"], case["kept"]), (case["nodes_min"], case["nodes"]))
        s["kept"] = kept
        s["table"], n_pages = _table(g, kept + fresh, case["page"], 3)
        # accepted paths: an ascending choice of about half the nodes of each tree, from node 0 on
        nodes = torch.arange(case["nodes"], device="cuda")
        taken = (torch.rand((batch, case["nodes"]), generator=g, device="cuda") < 0.5) & (nodes[None] < fresh[:, None])
        taken[:, 0] = True
        s["count"] = taken.sum(1).to(torch.int32)
        s["path"] = torch.where(nodes[None] < s["count"][:, None], torch.argsort((~taken).to(torch.uint8), dim=1, stable=True), torch.full_like(taken, -1, dtype=torch.int64)).to(torch.int32)
        s.update(_caches(g, (case["layers"], n_pages, case["kv_heads"], case["page"], case["dim"]), case["cache"]))
    return s


def _mean(low, high):
    """Mean of _lengths (about)."""
    return (high - low) / math.log((high + 1) / (low + 1)) - 1 if high > low else float(high)


def work(case):
    op, b = case["op"], case["batch"]
    if op == "plan":
        rows = b * _mean(case["fresh_min"], case["fresh"])
        return {"bytes": b * 24 + rows * (12 + ((4 + 4 * ((case["fresh"] + 31) // 32)) if case["tree"] else 0)) + 8 * rows / case["page"], "flops": 0}
    if op == "accept":
        rows = b * _mean(case["nodes_min"], case["nodes"])
        return {"bytes": rows * (case["vocab"] * (4 if case["type"] == "f32" else 2) + 12), "flops": rows * case["vocab"]}
    row = case["kv_heads"] * (2 * case["dim"] + 8 if case["cache"] == "e4m3" else 4 * case["dim"])      # bytes of K and V of one token
    if op == "compact":
        return {"bytes": b * _mean(case["nodes_min"], case["nodes"]) * 0.45 * case["layers"] * row * 2, "flops": 0}
    rows = b * _mean(case["fresh_min"], case["fresh"])
    if op == "write":
        return {"bytes": rows * (4 * case["kv_heads"] * case["dim"] + row + 8), "flops": 0}
    keys = _mean(case["kept_min"], case["kept"]) + rows / b
    return {"bytes": b * keys * row + 4 * rows * case["heads"] * case["dim"], "flops": 4.0 * case["dim"] * case["heads"] * rows * keys}


# ------------------------------------------------------------------------------------------------ plain forms

def _ancestors(parents, start, seq, index, batch, nodes):
    """[B, N, N]: whether node j is node i or one of its ancestors: the inverse of (1 - parent matrix), exact in 32 bits."""
    step = torch.zeros((batch, nodes, nodes), device=parents.device)
    fine = (parents >= 0) & (parents < index)
    step[seq, index.long(), parents.clamp(min=0).long()] = fine.float()
    step[seq, index.long(), index.long()] = 0
    eye = torch.eye(nodes, device=parents.device).expand(batch, nodes, nodes).contiguous()
    return torch.linalg.solve_triangular(eye - step, eye, upper=False, unitriangular=True) > 0.5


def _words(bits, words):
    """[R, N] truth values -> [R, words] int32, bit j of word w for node 32 w + j."""
    wide = torch.zeros((bits.shape[0], words * 32), dtype=torch.int64, device=bits.device)
    wide[:, :bits.shape[1]] = bits
    value = (wide.view(-1, words, 32) << torch.arange(32, device=bits.device)).sum(2)
    return torch.where(value >= 2**31, value - 2**32, value).to(torch.int32)


def _cut(kv_heads, longest):
    """How many work units a program asks for: enough for all compute units, or no cuts where no request is long."""
    return 0 if longest <= 512 else max(16, 2048 // kv_heads)


def _units(kept, fresh, admitted, target, least):
    """The work units of attention: {request, first key, key behind the last, units of the request}, -1 behind the last unit;
    every request with rows is cut into equal pieces of whole granules, about `target` of them in all (0: none is cut)."""
    batch = kept.numel()
    length = torch.where(admitted.bool(), kept.long() + fresh, torch.zeros_like(kept, dtype=torch.int64))
    length = torch.where(fresh > 0, length, torch.zeros_like(length))
    most = (length.sum() + target - 1) // target if target else length.sum()
    most = torch.maximum((most + CHUNK - 1) // CHUNK * CHUNK, torch.full_like(most, (least + CHUNK - 1) // CHUNK * CHUNK))
    count = torch.where(fresh > 0, ((length + most - 1) // most).clamp(min=1), torch.zeros_like(length))
    each = (length + count.clamp(min=1) - 1) // count.clamp(min=1)
    each = (each + CHUNK - 1) // CHUNK * CHUNK
    start = torch.zeros(batch + 1, dtype=torch.int32, device=kept.device)
    start[1:] = torch.cumsum(count, 0)
    u = torch.arange(batch + target, device=kept.device)
    b = torch.searchsorted(start[1:].contiguous(), u.to(torch.int32), right=True)
    real = b < batch
    b = b.clamp(max=batch - 1)
    first = (u - start[b]) * each[b]
    units = torch.stack([b, torch.minimum(first, length[b]), torch.minimum(first + each[b], length[b]), count[b]], 1)
    return torch.where(real[:, None], units, torch.full_like(units, -1)).to(torch.int32), start


def _plain_plan(s):
    kept, fresh, held, table, free, page = s["kept"].long(), s["fresh"].long(), s["pages"].long(), s["table"], s["free"], s["page"]
    batch, columns, rows = kept.numel(), table.shape[1], s["rows"]
    start = torch.zeros(batch + 1, dtype=torch.int64, device=kept.device)
    start[1:] = torch.cumsum(fresh, 0)
    need = (kept + fresh + page - 1) // page
    valid = (need <= columns) & (start[1:] <= rows)
    back = torch.where(valid, (held - need).clamp(min=0), torch.zeros_like(need))
    grow = torch.where(valid, (need - held).clamp(min=0), torch.zeros_like(need))
    # pages that come back lie on the stack in request order
    col = torch.arange(columns, device=kept.device)
    gone = (col[None] >= (held - back)[:, None]) & (col[None] < held[:, None])
    n_free = s["n_free"].long()
    at = n_free + torch.cumsum(back, 0)[:, None] - held[:, None] + col[None]
    free[at[gone]] = table[gone]
    stack = n_free + back.sum()
    upto = torch.cumsum(grow, 0)
    admitted = valid & ((grow == 0) | (upto <= stack))
    grow = torch.where(admitted, grow, torch.zeros_like(grow))
    new = (col[None] >= held[:, None]) & (col[None] < (held + grow)[:, None])
    from_top = stack - 1 - (upto - grow)[:, None] - (col[None] - held[:, None])
    table[new] = free[from_top[new]]
    pages = torch.where(admitted, need, held)
    seq = torch.repeat_interleave(torch.arange(batch, device=kept.device), fresh, output_size=rows)
    index = torch.arange(rows, device=kept.device) - start[seq]
    place = kept[seq] + index
    slots = torch.where(admitted[seq], table[seq, (place // page).clamp(max=columns - 1)].long() * page + place % page, torch.full_like(place, -1))
    out = {"row_start": start.to(torch.int32), "admitted": admitted.to(torch.int32), "pages": pages.to(torch.int32),
           "n_free": (stack - grow.sum()).to(torch.int32), "slots": slots, "table": table}
    if s["parents"] is None:
        out["positions"] = place.to(torch.int32)
    else:
        up = _ancestors(s["parents"], start, seq, index.to(torch.int32), batch, s["words"] * 32)[seq, index]
        out["positions"] = (kept[seq] + up.sum(1) - 1).to(torch.int32)
        out["mask"] = _words(up, s["words"])
    out["units"], out["unit_start"] = _units(s["kept"], s["fresh"], admitted, s["units"], s["chunk"])
    return out


def _e4m3(x):
    """Codes and scales of rows: scale = max |x| / 448."""
    scale = x.abs().amax(-1) / 448
    return (x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _plain_write(s):
    page = s["k"].shape[2]
    keep = s["slots"] >= 0
    p, o = s["slots"][keep] // page, s["slots"][keep] % page
    if "k_scale" in s:
        s["k"][p, :, o], s["k_scale"][p, :, o] = _e4m3(s["k_rows"][keep].float())
        s["v"][p, :, o], s["v_scale"][p, :, o] = _e4m3(s["v_rows"][keep].float())
    else:
        s["k"][p, :, o], s["v"][p, :, o] = s["k_rows"][keep], s["v_rows"][keep]
    return _cache_values(s)


def _cache_values(s):
    """A cache's contents: 16-bit values as they are, codes as the numbers they stand for beside their scales."""
    if "k_scale" in s:
        return {"k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"k": s["k"], "v": s["v"]}


def _gathered(s, name, page, offset):
    """[B, L, heads, dim] in 32 bits."""
    x = s[name][page, :, offset]
    if name + "_scale" in s:
        return x.view(torch.float8_e4m3fn).float() * s[name + "_scale"][page, :, offset][..., None]
    return x.float()


def _plain_attend(s):
    q, start = s["q"], s["row_start"].long()
    rows, heads, dim = q.shape
    batch, kv_heads, page = s["kept"].numel(), s["k"].shape[1], s["k"].shape[2]
    kept, fresh = s["kept"].long(), s["fresh"].long()
    nodes, most = s["nodes"], s["table"].shape[1] * page
    key = torch.arange(most, device=q.device)
    inside = key[None] < (kept + fresh)[:, None]
    where = s["table"].long().repeat_interleave(page, 1).clamp(min=0)
    k = _gathered(s, "k", where, key[None] % page).permute(0, 2, 3, 1).contiguous()                 # [B, Hkv, D, L]
    v = torch.where(inside[:, :, None, None], _gathered(s, "v", where, key[None] % page), 0.0).permute(0, 2, 1, 3).contiguous()
    node = torch.arange(nodes, device=q.device)
    row = (start[:-1, None] + node[None]).clamp(max=rows - 1)                                       # [B, N]
    wide = q.float()[row].view(batch, nodes, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, -1, dim)
    score = torch.matmul(wide, k).view(batch, kv_heads, nodes, heads // kv_heads, most) * (1.0 / math.sqrt(dim))
    j = key[None] - kept[:, None]                                                                   # [B, L]: node of a key, < 0 in the context
    if s["mask"] is None:
        sees = j[:, None, :] <= node[None, :, None]
    else:
        bits = s["mask"][row].long() & 0xFFFFFFFF                                                   # [B, N, W]
        word = (j.clamp(min=0) // 32).clamp(max=bits.shape[2] - 1)
        sees = (j[:, None, :] < 0) | ((bits.gather(2, word[:, None, :].expand(batch, nodes, most)) >> (j.clamp(min=0) % 32)[:, None, :]) & 1).bool()
    sees = (sees & inside[:, None, :])[:, None, :, None, :]
    score = torch.where(sees, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p.view(batch, kv_heads, -1, most), v).view(batch, kv_heads, nodes, -1, dim).permute(0, 2, 1, 3, 4).reshape(batch, nodes, heads, dim)
    return o[node[None] < fresh[:, None]].to(q.dtype)


def _plain_accept(s):
    logits, start = s["logits"].float(), s["row_start"].long()
    rows, batch, nodes = logits.shape[0], start.numel() - 1, s["depth"]
    logits = torch.where(torch.isnan(logits), torch.full_like(logits, -math.inf), logits)
    if s["suppress"] is not None:
        logits = torch.where(s["suppress"].bool()[None], torch.full_like(logits, -math.inf), logits)
    best = logits.argmax(1)
    seq = torch.repeat_interleave(torch.arange(batch, device=logits.device), start[1:] - start[:-1], output_size=rows)
    index = torch.arange(rows, device=logits.device) - start[seq]
    up = s["parents"].long()
    hangs = (up >= 0) & (up < index)
    agrees = hangs & (s["tokens"].long() == best[(start[seq] + up.clamp(min=0))])
    # of siblings with the same token the first one counts
    padded = torch.full((batch, nodes), -1, dtype=torch.int64, device=logits.device)
    padded[seq, index] = torch.where(hangs, s["tokens"].long() * nodes + up, torch.full_like(up, -1))
    earlier = torch.ones((nodes, nodes), dtype=torch.bool, device=logits.device).tril(-1)
    repeated = ((padded[:, :, None] == padded[:, None, :]) & earlier[None]).any(2)[seq, index] & hangs
    good = torch.zeros((batch, nodes), dtype=torch.bool, device=logits.device)
    good[seq, index] = (agrees & ~repeated) | (index == 0)
    line = _ancestors(s["parents"], start, seq, index.to(torch.int32), batch, nodes)
    real = torch.zeros((batch, nodes), dtype=torch.bool, device=logits.device)
    real[seq, index] = True
    taken = ~(line & ~good[:, None, :]).any(2) & real & line[:, :, 0]
    path = torch.full((batch, nodes), -1, dtype=torch.int64, device=logits.device)
    b, i = taken.nonzero(as_tuple=True)
    path[b, line[b, i].sum(1) - 1] = i
    ids = torch.where(path >= 0, best[(start[:-1, None] + path.clamp(min=0)).clamp(max=rows - 1)], torch.full_like(path, -1))
    return {"best": best.to(torch.int32), "path": path.to(torch.int32), "count": taken.sum(1).to(torch.int32), "tokens": ids.to(torch.int32)}


def _plain_compact(s):
    page = s["k"].shape[3]
    col = torch.arange(s["path"].shape[1], device=s["path"].device)
    b, i = ((col[None] < s["count"][:, None]) & (s["path"] != col[None])).nonzero(as_tuple=True)
    old, new = s["kept"][b] + s["path"][b, i], s["kept"][b] + i
    p0, o0, p1, o1 = s["table"][b, old // page].long(), old % page, s["table"][b, new // page].long(), new % page
    s["k"][:, p1, :, o1], s["v"][:, p1, :, o1] = s["k"][:, p0, :, o0], s["v"][:, p0, :, o0]
    if "k_scale" in s:
        s["k_scale"][:, p1, :, o1], s["v_scale"][:, p1, :, o1] = s["k_scale"][:, p0, :, o0], s["v_scale"][:, p0, :, o0]
    return _cache_values(s)


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    s, op = state, state["op"]
    if not own:
        return {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend, "accept": _plain_accept, "compact": _plain_compact}[op](s)
    from manual_whisper_amd import paged
    if op == "plan":
        pool = paged.PagePool(s["table"], s["pages"], s["free"], s["n_free"], s["page"])
        p = pool.plan(s["kept"], s["fresh"], s["rows"], parents=s["parents"], mask_words=s["words"], units=s["units"], chunk=s["chunk"])
        out = {"row_start": p.row_start, "admitted": p.admitted, "pages": p.pages, "n_free": p.n_free, "slots": p.slots, "table": s["table"],
               "positions": p.positions, "units": p.units, "unit_start": p.unit_start}
        if s["parents"] is not None:
            out["mask"] = p.mask
        return out
    if op == "accept":
        best, path, count, tokens = paged.accept(s["logits"], s["tokens"], s["parents"], s["row_start"], s["depth"], suppress=s["suppress"])
        return {"best": best, "path": path, "count": count, "tokens": tokens}
    cache = paged.PagedCache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    if op == "write":
        paged.write(cache, s["k_rows"], s["v_rows"], s["slots"])
        return _cache_values(s)
    if op == "attend":
        return paged.tree_attention(s["q"], cache, s["table"], s["kept"], s["row_start"], s["units"], s["unit_start"], s["nodes"], mask=s["mask"])
    paged.compact(cache, s["table"], s["kept"], s["path"], s["count"])
    return _cache_values(s)


# ------------------------------------------------------------------------------------------------ 64 bits

def _numbers(s, name):
    """What a cache holds, as 64-bit numbers: values and (e4m3) scales apart."""
    x = s[name]
    return x.view(torch.float8_e4m3fn).to(torch.float32).double() if x.dtype == torch.uint8 else x.double()


def exact(case, seed):
    if case["op"] in ("plan", "accept"):
        return None                                            # whole numbers only
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "attend":
        rows, heads, dim = s["q"].shape
        group = heads // case["kv_heads"]
        out = torch.zeros((rows, heads, dim), dtype=torch.float64, device="cuda")
        kept, start = s["kept"].tolist(), s["row_start"].tolist()
        scales = "k_scale" in s
        for b in range(case["batch"]):
            n = start[b + 1] - start[b]
            length = kept[b] + n
            pages = s["table"][b, :(length + page - 1) // page].long()
            seen = torch.ones((n, length), dtype=torch.bool, device="cuda")
            if s["mask"] is None:
                seen[:, kept[b]:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
            else:
                for j in range(n):
                    seen[:, kept[b] + j] = ((s["mask"][start[b]:start[b + 1], j // 32] >> (j % 32)) & 1).bool()
            for h in range(case["kv_heads"]):
                part = {}
                for name in ("k", "v"):
                    x = s[name][pages, h].reshape(-1, dim)[:length]
                    x = x.view(torch.float8_e4m3fn).to(torch.float32).double() if scales else x.double()
                    part[name] = x * s[name + "_scale"][pages, h].reshape(-1)[:length].double()[:, None] if scales else x
                for c in range(h * group, (h + 1) * group):
                    z = (s["q"][start[b]:start[b + 1], c].double() @ part["k"].T) / math.sqrt(dim)
                    z = z.masked_fill(~seen, -math.inf)
                    out[start[b]:start[b + 1], c] = torch.softmax(z, 1) @ part["v"]
        return out
    got = {name: _numbers(s, name) for name in ("k", "v")}
    if "k_scale" in s:
        got.update({name: s[name].double() for name in ("k_scale", "v_scale")})
    if case["op"] == "write":
        slots = s["slots"].tolist()
        live = [r for r, t in enumerate(slots) if t >= 0]
        at = torch.tensor([slots[r] for r in live], device="cuda")
        for name in ("k", "v"):
            x = s[name + "_rows"][torch.tensor(live, device="cuda")].double()
            if "k_scale" in s:
                scale = x.abs().max(2).values / 448
                got[name + "_scale"][at // page, :, at % page] = scale
                x = x / scale.clamp(min=1e-300)[:, :, None]
            got[name][at // page, :, at % page] = x
        return got
    path, count, kept, table = s["path"].tolist(), s["count"].tolist(), s["kept"].tolist(), s["table"].tolist()
    old, new = [], []
    for b in range(case["batch"]):
        for i in range(count[b]):
            a, z = kept[b] + path[b][i], kept[b] + i
            old.append(table[b][a // page] * page + a % page)
            new.append(table[b][z // page] * page + z % page)
    old, new = torch.tensor(old, device="cuda"), torch.tensor(new, device="cuda")
    for name, x in got.items():
        x[:, new // page, :, new % page] = x[:, old // page, :, old % page]
    return got
