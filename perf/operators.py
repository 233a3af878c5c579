"""The operators that move a model's rows around the table, as measured cases.

Two families, each in a plain form (elementary torch operations) and as the
calls of the framework (`hkv_b200`):

* tokens sorted by group (an expert, a table, an owner) and back with weights,
  and the gradients of both ways: `group_tokens`, `dispatch_rows`,
  `combine_rows`, `combine_rows_backward`;
* the pages of a cache whose index is a table: `PagePool.copy`, `fork`,
  `resize`, `free` and `compact`.

A case names its operator in "op". Every pass can be repeated on its state:
a branch pass gives its branches away and takes them again, and a compaction
writes the new page table beside the old one.
"""
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u64": torch.int64}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "u64": 8}
IDS = {"i32": torch.int32, "i64": torch.int64}


def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "hierarchicalkv-ascend_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import hkv_b200

    return hkv_b200


# ---- cases -----------------------------------------------------------------


def listed():
    return [
        # one decode step: few tokens, each to several experts; latency counts
        {"name": "dispatch decode", "op": "dispatch", "tokens": 32, "slots": 4, "groups": 64,
         "dim": 1024, "type": "bf16", "ids": "i64", "dropped": 0, "train": False},
        # one batch of keys for a model with a table per feature (eight tables)
        {"name": "dispatch keys to tables", "op": "dispatch", "tokens": 1000003, "slots": 1,
         "groups": 8, "dim": 1, "type": "u64", "ids": "i32", "dropped": 4099, "train": False},
        # one layer of a training step, there and the gradient back, some tokens over capacity
        {"name": "dispatch training", "op": "dispatch", "tokens": 16384, "slots": 8,
         "groups": 128, "dim": 2048, "type": "bf16", "ids": "i64", "dropped": 2621,
         "train": True},
        # the way back of the decode step
        {"name": "combine decode", "op": "combine", "tokens": 32, "slots": 4, "dim": 1024,
         "type": "bf16", "weights": "f32", "sorted": True, "dropped": 0, "train": False},
        # weighted sum of looked-up rows: bags of up to 19 keys, two fifths of the places empty
        {"name": "combine looked-up bags", "op": "combine", "tokens": 50021, "slots": 19,
         "dim": 64, "type": "f32", "weights": "f32", "sorted": False, "dropped": 380159,
         "train": False},
        # the way back of one layer of a training step with both gradients
        {"name": "combine training", "op": "combine", "tokens": 8192, "slots": 8, "dim": 4096,
         "type": "bf16", "weights": "f32", "sorted": True, "dropped": 655, "train": True},
        # a dozen pages moved between requests
        {"name": "copy a few pages", "op": "copy", "pages": 512, "pairs": 12, "planes": 4,
         "page_bytes": 16384},
        # a large part of a cache copied
        {"name": "copy many pages", "op": "copy", "pages": 4096, "pairs": 1800, "planes": 8,
         "page_bytes": 16384},
        # beams of two requests take one more token; half of the beams end
        {"name": "branch beams", "op": "branch", "prompts": 2, "branches": 4, "pages": 512,
         "max_pages": 64, "page_tokens": 16, "shortest": 203, "longest": 331, "grow": 1,
         "freed": 4, "planes": 4, "page_bytes": 8192},
        # many samples of long prompts: 64 prompts, 15 branches each
        {"name": "branch samples", "op": "branch", "prompts": 64, "branches": 15,
         "pages": 32768, "max_pages": 512, "page_tokens": 16, "shortest": 1021,
         "longest": 7919, "grow": 33, "freed": 480, "planes": 4, "page_bytes": 4096},
        # a small cache after some requests ended
        {"name": "compact a small cache", "op": "compact", "pages": 500, "live": 301,
         "moved": 37, "rows": 7, "max_pages": 50, "page_tokens": 16, "shared": 3, "planes": 2,
         "page_bytes": 8192},
        # a large cache, two fifths of it free in scattered places
        {"name": "compact a large cache", "op": "compact", "pages": 16384, "live": 9830,
         "moved": 3600, "rows": 256, "max_pages": 64, "page_tokens": 16, "shared": 8,
         "planes": 4, "page_bytes": 16384},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return max(low, min(high, round(2.0 ** rng.uniform(np.log2(low), np.log2(high + 0.49)))))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "copy", "branch", "compact"])
    if op in ("dispatch", "combine"):
        train = rng.random() < 0.5
        kind = rng.choice(["f32", "f16", "bf16"])
        dim = _spread(rng, 8, 4096)
        if rng.random() < 0.6:
            dim = max(8, dim // 8 * 8)
        if op == "dispatch" and not train and rng.random() < 0.3:
            kind, dim = "u64", rng.choice([1, 1, 2, 5])
        slots = rng.randint(1, 8 if op == "dispatch" else 20)
        most = min(1 << 20, (1 << 29) // (slots * dim * BYTES[kind]), (1 << 20) // slots)
        tokens = _spread(rng, 1, max(1, most))
        dropped = rng.choice([0, tokens * slots // 50, tokens * slots * 2 // 5])
        if op == "dispatch":
            groups = max(slots, _spread(rng, 2, 256))
            return {"op": op, "tokens": tokens, "slots": slots, "groups": groups, "dim": dim,
                    "type": kind, "ids": rng.choice(["i32", "i64"]), "dropped": dropped,
                    "train": train}
        return {"op": op, "tokens": tokens, "slots": slots, "dim": dim, "type": kind,
                "weights": rng.choice(["f32", "f32", kind, "none"]),
                "sorted": rng.random() < 0.6, "dropped": dropped, "train": train}
    planes = _spread(rng, 1, 16)
    page_bytes = rng.choice([16, 1]) * 16 * _spread(rng, 4, 128)
    if op == "copy":
        pages = _spread(rng, 16, min(8192, (1 << 29) // (planes * page_bytes)))
        return {"op": op, "pages": pages, "pairs": _spread(rng, 1, pages // 2),
                "planes": planes, "page_bytes": page_bytes}
    if op == "branch":
        prompts, branches = _spread(rng, 1, 48), rng.randint(1, 12)
        page_tokens = rng.choice([8, 16, 32, 64])
        shortest = _spread(rng, 1, 2048)
        longest = shortest + rng.randint(0, 2048)
        grow = rng.choice([1, 1, 5, 70])
        max_pages = (longest + grow) // page_tokens + rng.randint(1, 9)
        each = (longest + page_tokens - 1) // page_tokens
        pages = prompts * each + prompts * branches * (grow // page_tokens + 2) + rng.randint(0, 99)
        page_bytes = max(16, min(page_bytes, (1 << 29) // (planes * pages) // 16 * 16))
        return {"op": op, "prompts": prompts, "branches": branches, "pages": pages,
                "max_pages": max_pages, "page_tokens": page_tokens, "shortest": shortest,
                "longest": longest, "grow": grow, "freed": rng.randint(0, prompts * branches),
                "planes": planes, "page_bytes": page_bytes}
    pages = _spread(rng, 32, min(16384, (1 << 29) // (planes * page_bytes)))
    live = rng.randint(1, pages)
    rows = _spread(rng, 1, 128)
    per_row = max(1, live // rows)
    return {"op": op, "pages": pages, "live": live, "moved": rng.randint(0, min(live, pages - live)),
            "rows": rows, "max_pages": per_row + rng.randint(0, 7),
            "page_tokens": rng.choice([8, 16, 32, 64]), "shared": rng.randint(0, per_row // 2),
            "planes": planes, "page_bytes": page_bytes}


# ---- inputs ----------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def _perm(g, n):
    return torch.randperm(n, generator=g, device=DEVICE)


def _routes(g, tokens, slots, groups, dropped):
    """Group numbers as a router gives them: distinct in a token, some groups
    asked for more than others, -1 for a token that is not sent."""
    favour = torch.randn(groups, generator=g, device=DEVICE)
    score = torch.rand((tokens, groups), generator=g, device=DEVICE).mul_(3).add_(favour)
    ids = score.topk(slots, dim=1).indices if slots > 1 else score.argmax(1, keepdim=True)
    ids.view(-1)[_perm(g, tokens * slots)[:dropped]] = -1
    return ids


def _pages_of(lengths, page_tokens):
    return (lengths + page_tokens - 1) // page_tokens


def _row_tokens(case):
    """The prompts' lengths, from the shortest to the longest."""
    n = case["prompts"]
    return [case["shortest"] + (case["longest"] - case["shortest"]) * i // max(1, n - 1)
            for i in range(n)]


def _planes(g, case):
    shape = (case["planes"], case["pages"], case["page_bytes"] // 2)
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.bfloat16)


def _page_state(case, planes, refs, table, lengths):
    state = {"op": case["op"], "case": case, "planes": planes, "refs": refs, "table": table,
             "lengths": lengths}
    if own:  # the handle that a serving program keeps
        state["pool"] = _package().PagePool(list(planes), case.get("page_tokens", 16),
                                            refs=refs, table=table, lengths=lengths)
    return state


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op in ("dispatch", "combine"):
        tokens, slots, dim = case["tokens"], case["slots"], case["dim"]
        n, kind = tokens * slots, TYPES[case["type"]]
        state = {"op": op, "case": case}
    if op == "dispatch":
        state["ids"] = _routes(g, tokens, slots, case["groups"], case["dropped"]).to(IDS[case["ids"]])
        if kind == torch.int64:
            state["x"] = torch.randint(1, 1 << 62, (tokens, dim), generator=g, device=DEVICE)
        else:
            state["x"] = _randn(g, (tokens, dim), kind)
        state["offsets"] = torch.zeros(case["groups"] + 1, dtype=torch.int32, device=DEVICE)
        state["positions"] = torch.zeros((tokens, slots), dtype=torch.int32, device=DEVICE)
        state["order"] = torch.zeros(n, dtype=torch.int32, device=DEVICE)
        state["rows"] = torch.zeros((n, dim), dtype=kind, device=DEVICE)
        if case["train"]:
            state["grad_rows"] = _randn(g, (n, dim), kind)
            state["grad_x"] = torch.zeros((tokens, dim), dtype=kind, device=DEVICE)
        if own:
            size = _package().group_workspace(n, case["groups"])
            state["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEVICE)
        return state
    if op == "combine":
        state["rows"] = _randn(g, (n, dim), kind)
        if case["sorted"]:
            positions = _perm(g, n)
        else:
            positions = torch.arange(n, device=DEVICE)
        positions[_perm(g, n)[:case["dropped"]]] = -1
        state["positions"] = positions.to(torch.int32).view(tokens, slots)
        state["weights"] = None
        if case["weights"] != "none":
            score = torch.randn((tokens, slots), generator=g, device=DEVICE)
            state["weights"] = torch.softmax(score, 1).to(TYPES[case["weights"]])
        state["out"] = torch.zeros((tokens, dim), dtype=kind, device=DEVICE)
        if case["train"]:
            state["grad_out"] = _randn(g, (tokens, dim), kind)
            state["grad_rows"] = torch.zeros((n, dim), dtype=kind, device=DEVICE)
            state["grad_weights"] = None
            if state["weights"] is not None:
                state["grad_weights"] = torch.zeros_like(state["weights"])
        return state
    planes, pages = _planes(g, case), case["pages"]
    refs = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    if op == "copy":
        some = _perm(g, pages).to(torch.int32)
        refs += 1
        table = torch.zeros((1, 1), dtype=torch.int32, device=DEVICE)
        state = _page_state(case, planes, refs, table, torch.zeros(1, dtype=torch.int32, device=DEVICE))
        state["src"] = some[:case["pairs"]].contiguous()
        state["dst"] = some[pages - case["pairs"]:].contiguous()
        return state
    width, size = case["max_pages"], case["page_tokens"]
    if op == "branch":
        prompts, branches = case["prompts"], case["branches"]
        count = prompts * branches
        rows = _perm(g, prompts + count)
        parents, children = rows[:prompts], rows[prompts:]
        tokens = torch.tensor(_row_tokens(case), device=DEVICE)[_perm(g, prompts)]
        table = torch.full((prompts + count, width), -1, dtype=torch.int32, device=DEVICE)
        lengths = torch.zeros(prompts + count, dtype=torch.int32, device=DEVICE)
        lengths[parents] = tokens.to(torch.int32)
        used = _pages_of(tokens, size)
        on = torch.arange(width, device=DEVICE) < used[:, None]
        taken = _perm(g, pages)[:int(used.sum())]
        table[parents] = torch.full_like(table[parents], -1).masked_scatter_(on, taken.to(torch.int32))
        refs[taken] = 1
        state = _page_state(case, planes, refs, table, lengths)
        which = _perm(g, count) % prompts
        state["parents"] = parents[which].to(torch.int32)
        state["children"] = children.to(torch.int32)
        state["longer"] = (tokens[which] + case["grow"]).to(torch.int32)
        state["ended"] = children[_perm(g, count)[:case["freed"]]].to(torch.int32)
        state["served"] = torch.zeros(count, dtype=torch.bool, device=DEVICE)
        return state
    # compact: `live` pages in use, `moved` of them behind the first `live`
    live, moved, rows = case["live"], case["moved"], case["rows"]
    low = _perm(g, live)[:live - moved]
    high = live + _perm(g, pages - live)[:moved]
    used = torch.cat([low, high])[_perm(g, live)].to(torch.int32)
    each = max(1, live // rows)
    at = (torch.arange(rows, device=DEVICE)[:, None] * each + torch.arange(each, device=DEVICE)) % live
    table = torch.full((rows, width), -1, dtype=torch.int32, device=DEVICE)
    table[:, :each] = used[at]
    table[:, :case["shared"]] = table[:1, :case["shared"]].clone()
    refs[used.long()] = 1  # what no row holds any more is held by the index of prefixes
    refs += torch.bincount(table[:, :each].reshape(-1).long(), minlength=pages).to(torch.int32)
    lengths = torch.full((rows,), each * size - size // 2, dtype=torch.int32, device=DEVICE)
    state = _page_state(case, planes, refs, table, lengths)
    state["page_map"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    state["new_table"] = torch.full_like(table, -1)
    state["new_refs"] = torch.zeros_like(refs)
    return state


# ---- plain forms -----------------------------------------------------------


def _plain_dispatch(s):
    case = s["case"]
    slots, groups = case["slots"], case["groups"]
    ids = s["ids"].reshape(-1).long()
    n = ids.numel()
    kept = ids >= 0
    key = torch.where(kept, ids, groups)
    ordered, order = key.sort(stable=True)
    places = torch.arange(n, device=ids.device)
    offsets = torch.searchsorted(ordered, torch.arange(groups + 1, device=ids.device))
    positions = torch.empty_like(order)
    positions[order] = places
    positions = torch.where(kept, positions, -1)
    sent = places < offsets[groups]
    rows = torch.where(sent[:, None], s["x"][order // slots], 0)
    out = {"offsets": offsets.to(torch.int32), "order": torch.where(sent, order, -1).to(torch.int32),
           "positions": positions.view(-1, slots).to(torch.int32), "rows": rows}
    if case["train"]:
        picked = s["grad_rows"].float()[positions.clamp(min=0)]
        picked = torch.where(kept[:, None], picked, 0.0).view(-1, slots, picked.shape[1])
        out["grad_x"] = picked.sum(1).to(s["x"].dtype)
    return out


def _plain_combine(s):
    kind, positions = s["rows"].dtype, s["positions"].long()
    kept = positions >= 0
    at = positions.clamp(min=0)
    weights = torch.ones_like(kept, dtype=torch.float32)
    if s["weights"] is not None:
        weights = s["weights"].float()
    weights = torch.where(kept, weights, 0.0)
    picked = torch.where(kept[:, :, None], s["rows"][at].float(), 0.0)
    out = {"out": (picked * weights[:, :, None]).sum(1).to(kind)}
    if s["case"]["train"]:
        grad = s["grad_out"].float()
        spread = (weights[:, :, None] * grad[:, None, :]).to(kind)
        buffer = torch.zeros((at.numel() + 1, grad.shape[1]), dtype=kind, device=grad.device)
        buffer[torch.where(kept, at, at.numel()).reshape(-1)] = spread.reshape(-1, grad.shape[1])
        out["grad_rows"] = buffer[:-1]
        if s["weights"] is not None:
            out["grad_weights"] = (picked * grad[:, None, :]).sum(2).to(s["weights"].dtype)
    return out


def _plain_fork(s, src, dst):
    table, lengths, refs, size = s["table"], s["lengths"], s["refs"], s["case"]["page_tokens"]
    src, dst = src.long(), dst.long()
    j = torch.arange(table.shape[1], device=table.device)
    new, old = table[src], table[dst]
    new_on = j < _pages_of(lengths[src], size)[:, None]
    old_on = j < _pages_of(lengths[dst], size)[:, None]
    refs.index_add_(0, new.clamp(min=0).reshape(-1).long(), new_on.reshape(-1).to(torch.int32))
    refs.index_add_(0, old.clamp(min=0).reshape(-1).long(), -old_on.reshape(-1).to(torch.int32))
    table[dst] = torch.where(new_on, new, old)
    lengths[dst] = lengths[src]


def _plain_resize(s, rows, longer):
    table, lengths, refs, planes = s["table"], s["lengths"], s["refs"], s["planes"]
    size, rows, longer = s["case"]["page_tokens"], rows.long(), longer.long()
    j = torch.arange(table.shape[1], device=table.device)
    entries, old = table[rows], lengths[rows].long()
    before, after = _pages_of(old, size), _pages_of(longer, size)
    last = entries.gather(1, (before - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0).long()
    copied = (longer > old) & (old % size != 0) & (refs[last] > 1)
    need = (after - before).clamp(min=0) + copied
    fits = (longer >= 0) & (after <= table.shape[1])
    need = torch.where(fits, need, 0)
    upto = need.cumsum(0)
    free = (refs == 0).nonzero()[:, 0]
    served = fits & ((need == 0) | (upto <= free.numel()))
    copied = copied & served
    first = upto - need
    grown = served[:, None] & (j >= before[:, None]) & (j < after[:, None])
    gone = served[:, None] & (j >= after[:, None]) & (j < before[:, None])
    given = (first + copied)[:, None] + j - before[:, None]
    entries = entries.clone()
    freed, took = entries[gone].long(), free[given[grown]]
    entries[grown] = took.to(torch.int32)
    fresh, shared = free[first[copied]], last[copied]
    entries[copied, before[copied] - 1] = fresh.to(torch.int32)
    refs.index_add_(0, freed, torch.full_like(freed, -1, dtype=torch.int32))
    refs.index_add_(0, shared, torch.full_like(shared, -1, dtype=torch.int32))
    refs[took] = 1
    refs[fresh] = 1
    planes[:, fresh] = planes[:, shared]
    table[rows] = entries
    lengths[rows] = torch.where(served, longer, old).to(torch.int32)
    return served


def _plain_free(s, rows):
    table, lengths, refs = s["table"], s["lengths"], s["refs"]
    rows = rows.long()
    j = torch.arange(table.shape[1], device=table.device)
    on = j < _pages_of(lengths[rows], s["case"]["page_tokens"])[:, None]
    refs.index_add_(0, table[rows].clamp(min=0).reshape(-1).long(), -on.reshape(-1).to(torch.int32))
    lengths[rows] = 0


def _plain_compact(s):
    refs, table, planes = s["refs"], s["table"], s["planes"]
    live = refs > 0
    number = torch.arange(refs.numel(), device=refs.device)
    count = live.sum()
    holes = (~live & (number < count)).nonzero()[:, 0]
    movers = (live & (number >= count)).nonzero()[:, 0]
    page_map = torch.where(live, number, -1)
    page_map[movers] = holes
    planes[:, holes] = planes[:, movers]
    new_refs = refs.clone()
    new_refs[holes] = refs[movers]
    new_refs[movers] = 0
    on = torch.arange(table.shape[1], device=table.device) < _pages_of(
        s["lengths"], s["case"]["page_tokens"])[:, None]
    new_table = torch.where(on, page_map[table.clamp(min=0).long()], -1).to(torch.int32)
    return {"page_map": page_map.to(torch.int32), "table": new_table, "refs": new_refs,
            "planes": planes}


# ---- one pass --------------------------------------------------------------


def run(state):
    s, case, op = state, state["case"], state["op"]
    if op == "dispatch":
        if not own:
            return _plain_dispatch(s)
        hkv = _package()
        hkv.group_tokens(s["order"].numel(), s["ids"], case["groups"], s["offsets"],
                         s["positions"], s["order"], s["workspace"])
        hkv.dispatch_rows(case["tokens"], s["x"], s["positions"], s["rows"])
        out = {"offsets": s["offsets"], "order": s["order"], "positions": s["positions"],
               "rows": s["rows"]}
        if case["train"]:
            hkv.combine_rows(case["tokens"], s["grad_rows"], s["positions"], None, s["grad_x"])
            out["grad_x"] = s["grad_x"]
        return out
    if op == "combine":
        if not own:
            return _plain_combine(s)
        hkv = _package()
        hkv.combine_rows(case["tokens"], s["rows"], s["positions"], s["weights"], s["out"])
        out = {"out": s["out"]}
        if case["train"]:
            hkv.combine_rows_backward(case["tokens"], s["rows"], s["positions"], s["weights"],
                                      s["grad_out"], s["grad_rows"], s["grad_weights"])
            out["grad_rows"] = s["grad_rows"]
            if s["weights"] is not None:
                out["grad_weights"] = s["grad_weights"]
        return out
    if op == "copy":
        if own:
            s["pool"].copy(case["pairs"], s["src"], s["dst"])
        else:
            s["planes"][:, s["dst"].long()] = s["planes"][:, s["src"].long()]
        return {"planes": s["planes"]}
    if op == "branch":
        count = case["prompts"] * case["branches"]
        if own:
            served = s["served"]
            s["pool"].fork(count, s["parents"], s["children"])
            s["pool"].resize(count, s["children"], s["longer"], served)
            s["pool"].free(case["freed"], s["ended"])
        else:
            _plain_fork(s, s["parents"], s["children"])
            served = _plain_resize(s, s["children"], s["longer"])
            _plain_free(s, s["ended"])
        return {"served": served, "table": s["table"], "lengths": s["lengths"],
                "refs": s["refs"], "planes": s["planes"]}
    if not own:
        return _plain_compact(s)
    s["pool"].compact(s["page_map"], s["new_table"], s["new_refs"])
    return {"page_map": s["page_map"], "table": s["new_table"], "refs": s["new_refs"],
            "planes": s["planes"]}


# ---- what a pass cannot do without -----------------------------------------


def work(case):
    op = case["op"]
    if op in ("dispatch", "combine"):
        tokens, slots, dim = case["tokens"], case["slots"], case["dim"]
        n, width = tokens * slots, dim * BYTES[case["type"]]
        kept = n - case["dropped"]
    if op == "dispatch":
        size = n * (4 if case["ids"] == "i32" else 8) + 4 * (case["groups"] + 1) + 8 * n
        size += tokens * width + kept * width
        if case["train"]:
            size += kept * width + tokens * width
        return {"bytes": size, "flops": kept * dim if case["train"] else 0}
    if op == "combine":
        weights = 0 if case["weights"] == "none" else BYTES[case["weights"]]
        size = 4 * n + weights * n + kept * width + tokens * width
        flops = 2 * kept * dim
        if case["train"]:
            size += tokens * width + kept * width + weights * n
            flops += 3 * kept * dim
        return {"bytes": size, "flops": flops}
    page = case["planes"] * case["page_bytes"]
    if op == "copy":
        return {"bytes": case["pairs"] * (2 * page + 8), "flops": 0}
    if op == "branch":
        size, grow, branches = case["page_tokens"], case["grow"], case["branches"]
        bytes_ = 4 * case["pages"] + 12 * case["prompts"] * branches + 4 * case["freed"]
        for tokens in _row_tokens(case):
            old, new = -(-tokens // size), -(-(tokens + grow) // size)
            # the prompt's entries, the branches' entries, the counts that change
            bytes_ += 4 * old + 4 * branches * new + 8 * old + 8 * branches * (new - old)
            if tokens % size:  # the last page of the prompt, one copy for each branch
                bytes_ += page * (1 + branches)
        return {"bytes": bytes_, "flops": 0}
    each = max(1, case["live"] // case["rows"])
    return {"bytes": 2 * page * case["moved"] + 12 * case["pages"] + 8 * case["rows"] * each,
            "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------


def _exact_dispatch(s):
    case = s["case"]
    slots, groups = case["slots"], case["groups"]
    ids = s["ids"].reshape(-1).cpu().numpy().astype(np.int64)
    order = np.full(ids.size, -1, np.int64)
    positions = np.full(ids.size, -1, np.int64)
    offsets = np.zeros(groups + 1, np.int64)
    for group in range(groups):
        members = np.flatnonzero(ids == group)
        start = offsets[group]
        offsets[group + 1] = start + members.size
        order[start:start + members.size] = members
        positions[members] = start + np.arange(members.size)
    sent = int(offsets[-1])
    source = torch.from_numpy(order[:sent] // slots).to(DEVICE)
    x = s["x"] if s["x"].dtype == torch.int64 else s["x"].double()
    rows = torch.zeros((ids.size, x.shape[1]), dtype=x.dtype, device=DEVICE)
    rows[:sent] = x[source]
    out = {"offsets": torch.from_numpy(offsets), "order": torch.from_numpy(order),
           "positions": torch.from_numpy(positions.reshape(-1, slots)), "rows": rows}
    if case["train"]:
        grad = torch.zeros(x.shape, dtype=torch.float64, device=DEVICE)
        out["grad_x"] = grad.index_add_(0, source, s["grad_rows"][:sent].double())
    return out


def _exact_combine(s):
    tokens, slots = s["positions"].shape
    dim, n = s["rows"].shape[1], tokens * slots
    out = torch.zeros((tokens, dim), dtype=torch.float64, device=DEVICE)
    grad_rows = torch.zeros((n, dim), dtype=torch.float64, device=DEVICE)
    grad_weights = torch.zeros((tokens, slots), dtype=torch.float64, device=DEVICE)
    for slot in range(slots):
        who = (s["positions"][:, slot] >= 0).nonzero()[:, 0]
        at = s["positions"][who, slot].long()
        weight = torch.ones(who.numel(), dtype=torch.float64, device=DEVICE)
        if s["weights"] is not None:
            weight = s["weights"][who, slot].double()
        rows = s["rows"][at].double()
        out.index_add_(0, who, rows * weight[:, None])
        if s["case"]["train"]:
            grad = s["grad_out"][who].double()
            grad_rows[at] = grad * weight[:, None]
            grad_weights[who, slot] = (rows * grad).sum(1)
    result = {"out": out}
    if s["case"]["train"]:
        result["grad_rows"] = grad_rows
        if s["weights"] is not None:
            result["grad_weights"] = grad_weights
    return result


def _exact_branch(s):
    size, width = s["case"]["page_tokens"], s["case"]["max_pages"]
    table, lengths = s["table"].cpu().numpy(), s["lengths"].tolist()
    refs, moves = s["refs"].cpu().numpy(), []
    whole = [table[r].copy() for r in range(len(lengths))]
    used = [-(-n // size) for n in lengths]
    for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
        refs[whole[parent][:used[parent]]] += 1
        table[child][:used[parent]] = whole[parent][:used[parent]]
        lengths[child] = lengths[parent]
    free, served = np.flatnonzero(refs == 0).tolist(), []
    counts = refs.copy()
    place = wanted = 0
    for row, length in zip(s["children"].tolist(), s["longer"].tolist()):
        old = lengths[row]
        have, want = -(-old // size), -(-length // size)
        shared = length > old and old % size and counts[table[row][have - 1]] > 1
        need = max(0, want - have) + bool(shared) if want <= width else 0
        wanted += need
        served.append(want <= width and (need == 0 or wanted <= len(free)))
        place = wanted - need
        if not served[-1]:
            continue
        if shared:
            moves.append((int(table[row][have - 1]), free[place]))
            refs[table[row][have - 1]] -= 1
            refs[free[place]] = 1
            table[row][have - 1] = free[place]
            place += 1
        for k in range(have, want):
            table[row][k] = free[place]
            refs[free[place]] = 1
            place += 1
        for k in range(want, have):
            refs[table[row][k]] -= 1
        lengths[row] = length
    for row in s["ended"].tolist():
        refs[table[row][:-(-lengths[row] // size)]] -= 1
        lengths[row] = 0
    planes = s["planes"].clone()
    if moves:
        pairs = torch.tensor(moves, device=DEVICE)
        planes[:, pairs[:, 1]] = s["planes"][:, pairs[:, 0]]
    return {"served": torch.tensor(served), "table": torch.from_numpy(table),
            "lengths": torch.tensor(lengths), "refs": torch.from_numpy(refs), "planes": planes}


def _exact_compact(s):
    size = s["case"]["page_tokens"]
    refs = s["refs"].cpu().numpy()
    live = int((refs > 0).sum())
    holes = [p for p in range(live) if refs[p] == 0]
    movers = [p for p in range(live, refs.size) if refs[p] > 0]
    page_map = np.where(refs > 0, np.arange(refs.size), -1)
    new_refs = np.where(np.arange(refs.size) < live, refs, 0)
    planes = s["planes"].clone()
    if movers:
        page_map[movers] = holes
        new_refs[holes] = refs[movers]
        planes[:, torch.tensor(holes, device=DEVICE)] = s["planes"][:, torch.tensor(movers, device=DEVICE)]
    table = s["table"].cpu().numpy()
    new_table = np.full_like(table, -1)
    for row, length in enumerate(s["lengths"].tolist()):
        n = -(-length // size)
        new_table[row, :n] = page_map[table[row, :n]]
    return {"page_map": torch.from_numpy(page_map), "table": torch.from_numpy(new_table),
            "refs": torch.from_numpy(new_refs), "planes": planes}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "dispatch":
        return _exact_dispatch(s)
    if op == "combine":
        return _exact_combine(s)
    if op == "copy":
        planes = s["planes"].clone()
        planes[:, s["dst"].long()] = s["planes"][:, s["src"].long()]
        return {"planes": planes}
    return _exact_branch(s) if op == "branch" else _exact_compact(s)
