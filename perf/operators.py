"""What is timed and compared of the serving operators on the paged K/V cache: attention of ragged
new tokens over the cache (with a window and first tokens that stay visible), forks of sequences,
compaction of kept tokens, and the turnover of pages.

A case is a dict of plain values. "op" says which operator:

  "extend"    attention of a batch in which every sequence brings its own number of new tokens over
              its cached keys and the new ones. `cache`: "ring" (a sliding layer's ring) or "full".
              `window` keys are visible to a row (0: all), and the first `sinks` ones always.
              `singles` of the sequences bring one token, the others min_rows..max_rows.
  "fork"      sequences become branches of others: whole pages are shared, what may still be
              written to is copied, in every layer. The branches of the step before are dropped.
  "compact"   sequences keep some of their tokens, which close up, in every layer.
  "turnover"  pages of ranges of positions go back to the pool and others are taken from it.

Geometries: 8 KV heads x 256 and 1 KV head x 512, 16 query heads, bf16. Lengths come from the case's
"lengths", data and the order of the pages from the seed.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
QUERY_HEADS = 16
WINDOW = 1024
EVERYTHING = 2**31 - 1


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # One conversation's next token on a sliding layer, ring long wrapped: the smallest call.
        {"name": "extend_token_sliding_b1", "op": "extend", "heads": 8, "dim": 256, "cache": "ring",
         "page": 1, "window": WINDOW, "sinks": 0, "batch": 1, "singles": 1, "min_rows": 1,
         "max_rows": 1, "min_prior": 8192, "max_prior": 8192, "lengths": 0},
        # The next tokens of 24 conversations of all lengths on a global layer.
        {"name": "extend_tokens_global512_b24", "op": "extend", "heads": 1, "dim": 512,
         "cache": "full", "page": 64, "window": 0, "sinks": 0, "batch": 24, "singles": 24,
         "min_rows": 1, "max_rows": 1, "min_prior": 200, "max_prior": 12000, "lengths": 1},
        # One step of a server on a global layer: next tokens, drafts to verify, short messages.
        {"name": "extend_mixed_global512_b10", "op": "extend", "heads": 1, "dim": 512,
         "cache": "full", "page": 64, "window": 0, "sinks": 0, "batch": 10, "singles": 5,
         "min_rows": 2, "max_rows": 300, "min_prior": 0, "max_prior": 8000, "lengths": 2},
        # The same on a sliding layer, with longer messages in the batch.
        {"name": "extend_mixed_sliding_b12", "op": "extend", "heads": 8, "dim": 256,
         "cache": "ring", "page": 16, "window": WINDOW, "sinks": 0, "batch": 12, "singles": 6,
         "min_rows": 2, "max_rows": 777, "min_prior": 0, "max_prior": 5000, "lengths": 3},
        # Endless streams: a window over a full-length cache, its first tokens kept, the pages
        # between them given back.
        {"name": "extend_sinks_global256_b16", "op": "extend", "heads": 8, "dim": 256,
         "cache": "full", "page": 16, "window": 2000, "sinks": 4, "batch": 16, "singles": 8,
         "min_rows": 2, "max_rows": 33, "min_prior": 100, "max_prior": 16000, "lengths": 4},
        # A long prompt's chunk on a global layer: the largest call.
        {"name": "extend_prompt_global512_2048", "op": "extend", "heads": 1, "dim": 512,
         "cache": "full", "page": 64, "window": 0, "sinks": 0, "batch": 1, "singles": 0,
         "min_rows": 2048, "max_rows": 2048, "min_prior": 6144, "max_prior": 6144, "lengths": 5},
        # A second answer to one prompt: all sliding layers' rings are copied.
        {"name": "fork_ring_1", "op": "fork", "heads": 8, "dim": 256, "cache": "ring", "page": 64,
         "layers": 40, "window": WINDOW, "parents": 1, "children": 1, "min_len": 5000,
         "max_len": 5000, "lengths": 6},
        # A beam step on the global layers: whole pages shared, the begun ones copied.
        {"name": "fork_global512_18", "op": "fork", "heads": 1, "dim": 512, "cache": "full",
         "page": 64, "layers": 8, "window": 0, "parents": 6, "children": 18, "min_len": 700,
         "max_len": 8191, "lengths": 7},
        # A verified draft tree: a few of each sequence's newest tokens stay.
        {"name": "compact_drafts_sliding_b8", "op": "compact", "heads": 8, "dim": 256,
         "cache": "ring", "page": 64, "layers": 10, "window": WINDOW, "batch": 8, "min_len": 1500,
         "max_len": 6000, "tail": 32, "kept": 7, "lengths": 8},
        # Long prompts thinned out to the tokens worth keeping.
        {"name": "compact_thinned_global512_b4", "op": "compact", "heads": 1, "dim": 512,
         "cache": "full", "page": 64, "layers": 8, "window": 0, "batch": 4, "min_len": 4000,
         "max_len": 8000, "tail": 0, "kept": 3001, "lengths": 9},
        # A server's step: a few sequences end, others begin or reach a new page.
        {"name": "turnover_b64", "op": "turnover", "page": 64, "batch": 64, "max_pages": 512,
         "pool": 16384, "ending": 4, "beginning": 6, "max_len": 20000, "lengths": 10},
        # A small one.
        {"name": "turnover_b5", "op": "turnover", "page": 16, "batch": 5, "max_pages": 64,
         "pool": 200, "ending": 1, "beginning": 1, "max_len": 700, "lengths": 11},
    ]


def _log_int(rng, low, high):
    high = max(low, high)
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _draw_extend(rng):
    heads, dim = rng.choice([(8, 256), (1, 512)])
    ring = heads == 8 and rng.random() < 0.5
    window = WINDOW if ring else rng.choice([0, 0, _log_int(rng, 16, 4096)])
    batch = _log_int(rng, 1, 32)
    # At most 150 000 cached tokens (80 000 of 8 x 256), and as many row x key pairs, padded to the
    # longest of the batch, as half of the largest listed case.
    prior = _log_int(rng, 1, min(14000, (150_000 if heads == 1 else 80_000) // batch))
    rows = _log_int(rng, 1, 2000)
    span = min(window, prior) if window else prior
    while rows > 1 and batch * rows * (span + rows) > 8_000_000:
        rows = rows * 3 // 4
    return {"op": "extend", "heads": heads, "dim": dim, "cache": "ring" if ring else "full",
            "page": rng.choice([1, 16, 64]) if ring else rng.choice([16, 64]), "window": window,
            "sinks": rng.choice([0, 1, 4, 67]) if window and not ring else 0, "batch": batch,
            "singles": rng.randint(0, batch) if rows > 1 else batch,
            "min_rows": _log_int(rng, 1, rows), "max_rows": rows,
            "min_prior": rng.choice([0, _log_int(rng, 1, prior)]), "max_prior": prior,
            "lengths": rng.randrange(1 << 20)}


def _draw_fork(rng):
    heads, dim, cache = rng.choice([(8, 256, "ring"), (8, 256, "full"), (1, 512, "full")])
    children = _log_int(rng, 1, 4 if cache == "ring" else 24)
    length = _log_int(rng, 20, 6000)
    return {"op": "fork", "heads": heads, "dim": dim, "cache": cache, "page": rng.choice([16, 64]),
            "layers": rng.randint(1, 20 // children if cache == "ring" else 8),
            "window": WINDOW if cache == "ring" else 0, "parents": rng.randint(1, min(3, children)),
            "children": children, "min_len": _log_int(rng, 1, length), "max_len": length,
            "lengths": rng.randrange(1 << 20)}


def _draw_compact(rng):
    heads, dim, cache = rng.choice([(8, 256, "ring"), (8, 256, "full"), (1, 512, "full")])
    batch = _log_int(rng, 1, 12)
    length = _log_int(rng, 80, 4000)
    tail = rng.randint(2, 64) if cache == "ring" or rng.random() < 0.5 else 0
    return {"op": "compact", "heads": heads, "dim": dim, "cache": cache,
            "page": rng.choice([16, 64]), "layers": rng.randint(1, 6),
            "window": WINDOW if cache == "ring" else 0, "batch": batch, "min_len": 70,
            "max_len": length, "tail": tail, "kept": rng.randint(1, tail or length // 2),
            "lengths": rng.randrange(1 << 20)}


def _draw_turnover(rng):
    batch, page = _log_int(rng, 1, 128), rng.choice([16, 64])
    max_pages = _log_int(rng, 4, 512)
    changing = rng.randint(1, batch)
    ending = rng.randint(0, changing)
    return {"op": "turnover", "page": page, "batch": batch, "max_pages": max_pages,
            "pool": batch * max_pages, "ending": ending, "beginning": changing - ending,
            "max_len": _log_int(rng, page, max_pages * page - 1), "lengths": rng.randrange(1 << 20)}


def draw(rng):
    return rng.choice([_draw_extend] * 6 + [_draw_fork, _draw_compact, _draw_turnover])(rng)


# ---- what a user's program holds ---------------------------------------------------------------

def _lengths(case):
    """(rows, prior lengths) of an extending batch, as the scheduler knows them."""
    rng = random.Random(case["lengths"])
    batch = case["batch"]
    rows = [1] * case["singles"]
    rows += [_log_int(rng, case["min_rows"], case["max_rows"]) for _ in range(batch - len(rows))]
    if case["singles"] < batch:
        rows[-1] = case["max_rows"]
    prior = [rng.randint(case["min_prior"], case["max_prior"]) for _ in range(batch)]
    prior[rng.randrange(batch)] = case["max_prior"]
    rng.shuffle(rows)
    return rows, prior


def _sequence_lengths(case, count):
    rng = random.Random(case["lengths"])
    lens = [rng.randint(min(case["min_len"], case["max_len"]), case["max_len"]) for _ in range(count)]
    lens[rng.randrange(count)] = case["max_len"]
    return lens


def _ring_pages(window, page):
    return (window + 2 * page - 2) // page


def _max_pages(case, longest):
    return _ring_pages(case["window"], case["page"]) if case["cache"] == "ring" else -(-longest // case["page"])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


class _Inputs:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed * 1_000_003 + 29)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device=DEVICE, dtype=torch.bfloat16)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=DEVICE).to(torch.int32)


def _table(mapped, max_pages, order):
    """Page table of sequences whose logical slots `mapped[b]` (a list) hold pages, in the order of
    a pool that has been in use for a while."""
    flat, used = [], 0
    for slots in mapped:
        row = [-1] * max_pages
        for s in slots:
            row[s] = used
            used += 1
        flat.append(row)
    at = torch.tensor(flat, device=DEVICE, dtype=torch.int64)
    return torch.where(at >= 0, order[at.clamp(min=0)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()


def _make_extend(case, seed):
    i = _Inputs(seed)
    rows, prior = _lengths(case)
    heads, dim, page, batch = case["heads"], case["dim"], case["page"], case["batch"]
    max_pages = _max_pages(case, max(n + p for n, p in zip(rows, prior)))
    window, sinks = case["window"], case["sinks"]
    mapped = []
    for n, p in zip(rows, prior):
        if case["cache"] == "ring":
            mapped.append(range(min(max_pages, -(-(n + p) // page))))
        else:  # pages that no row sees any more were given back
            first = max(0, p - window + 1) // page if window else 0
            mapped.append([s for s in range(-(-(n + p) // page)) if s >= first or s * page < sinks])
    pages = sum(len(m) for m in mapped)
    total = sum(rows)
    off = [sum(rows[:b]) for b in range(batch + 1)]
    s = {"rows": rows, "prior": prior, "pages": pages, "max_pages": max_pages, "total": total,
         "page_table": _table(mapped, max_pages, i.order(pages)), "row_offsets": _int32(off),
         "prior_lengths": _int32(prior), "scale": 1.0 / math.sqrt(dim)}
    s["cache_k"], s["cache_v"] = (i.normal(pages * page, heads, dim) for _ in range(2))
    s["q"] = i.normal(total, QUERY_HEADS, dim)
    s["k"], s["v"] = (i.normal(total, heads, dim) for _ in range(2))
    s["out"] = torch.empty_like(s["q"])
    return s


def _make_fork(case, seed):
    i = _Inputs(seed)
    rng = random.Random(case["lengths"] + 1)
    parents, children, page = case["parents"], case["children"], case["page"]
    lens = _sequence_lengths(case, parents)
    parent_of = [rng.randrange(parents) for _ in range(children)]
    old = [max(1, lens[p] - rng.randint(0, page)) for p in parent_of]  # the branches of before
    max_pages = _max_pages(case, max(lens) + page)
    held = [range(min(max_pages, -(-n // page))) for n in lens + old]
    batch = parents + children
    pool = batch * max_pages
    order = i.order(pool)
    # (child, slot, rows) of the pages to copy, as the scheduler knows them: a ring's, or begun ones.
    if case["cache"] == "ring":
        copied = [(c, j, page) for c, p in enumerate(parent_of) for j in held[p]]
    else:
        copied = [(c, lens[p] // page, lens[p] % page) for c, p in enumerate(parent_of) if lens[p] % page]
    s = {"copied": [torch.tensor(x, device=DEVICE) for x in zip(*copied)] if copied else None,
         "max_pages": max_pages, "batch": batch, "pages": pool,
         "page_table": _table(held, max_pages, order), "seq_lengths": _int32(lens + old),
         "parents": _int32(parent_of), "children": _int32(list(range(parents, batch))),
         "first": _int32([EVERYTHING] * parents + [0] * children), "end": _int32([EVERYTHING] * batch),
         "status": _int32([0])}
    refs = torch.zeros(pool, dtype=torch.int32, device=DEVICE)
    refs[order[:sum(len(h) for h in held)].long()] = 1
    s["page_refs"] = refs
    s["cache_k"], s["cache_v"] = (i.normal(case["layers"], pool * page, case["heads"], case["dim"]) for _ in range(2))
    return s


def _make_compact(case, seed):
    i = _Inputs(seed)
    rng = random.Random(case["lengths"] + 1)
    page, batch = case["page"], case["batch"]
    lens = _sequence_lengths(case, batch)
    max_pages = _max_pages(case, max(lens))
    first, kept = [], []
    for n in lens:  # what stays of the last `tail` tokens, or of all
        begin = n - min(case["tail"], n) if case["tail"] else 0
        keep = min(case["kept"], n - begin)
        first.append(begin)
        kept.append(sorted(rng.sample(range(begin, n), keep)))
    pool = batch * max_pages
    order = i.order(pool)
    held = [range(min(max_pages, -(-n // page))) for n in lens]
    s = {"max_pages": max_pages, "batch": batch, "pages": pool,
         "page_table": _table(held, max_pages, order), "sequences": _int32(list(range(batch))),
         "first": _int32(first), "kept_offsets": _int32([sum(map(len, kept[:b])) for b in range(batch + 1)]),
         "kept_positions": _int32([p for k in kept for p in k]), "total": sum(map(len, kept)),
         "status": torch.zeros(batch, dtype=torch.int32, device=DEVICE)}
    refs = torch.zeros(pool, dtype=torch.int32, device=DEVICE)
    refs[order[:sum(len(h) for h in held)].long()] = 1
    s["page_refs"] = refs
    s["cache_k"], s["cache_v"] = (i.normal(case["layers"], pool * page, case["heads"], case["dim"]) for _ in range(2))
    return s


def _make_turnover(case, seed):
    i = _Inputs(seed)
    rng = random.Random(case["lengths"])
    page, batch, max_pages = case["page"], case["batch"], case["max_pages"]
    room = case["pool"] // batch * page
    longest = min(case["max_len"], max_pages * page - 1, max(1, room - 1))
    lens = [rng.randint(1, longest) for _ in range(batch)]
    ending, beginning = case["ending"], case["beginning"]
    for b in range(ending, ending + beginning):
        lens[b] = 0
    held = [range(-(-n // page)) for n in lens]
    order = i.order(case["pool"])
    refs = torch.zeros(case["pool"], dtype=torch.int32, device=DEVICE)
    refs[order[:sum(len(h) for h in held)].long()] = 1
    release = [0] * ending + [EVERYTHING] * (batch - ending)
    # New sequences take their prompt's pages, the others the page of their next token.
    end = [0] * ending + [rng.randint(1, longest) for _ in range(beginning)] + [n + 1 for n in lens[ending + beginning:]]
    begin = [0 if n == 0 else n for n in lens]
    return {"batch": batch, "max_pages": max_pages, "pages": case["pool"], "page_table": _table(held, max_pages, order),
            "page_refs": refs, "release_first": _int32(release), "release_end": _int32([EVERYTHING] * batch),
            "reserve_first": _int32(begin), "reserve_end": _int32(end), "status": _int32([0])}


_MAKE = {"extend": _make_extend, "fork": _make_fork, "compact": _make_compact, "turnover": _make_turnover}


def _library():
    path = str(Path.cwd() / "gemma.c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gemma_kv
    return gemma_kv


def prepare(case, seed):
    s = _MAKE[case["op"]](case, seed)
    s["case"] = case
    if own:
        gk = _library()
        s["gk"] = gk
        s["config"] = gk.make_config(
            case.get("layers", 1), s["pages"], case["page"], s["max_pages"], s.get("batch", case.get("batch")),
            case.get("heads", 8), case.get("dim", 256), case["window"] if case.get("cache") == "ring" else 0)
        if case["op"] == "extend":  # a step's plan serves all of its layers
            shape = (s["config"], case["batch"], s["total"])
            s["plan_bytes"] = gk.flash_attention_extend_plan_bytes(*shape)
            s["workspace_bytes"] = gk.flash_attention_extend_workspace_bytes(*shape)
            s["plan"] = torch.empty(s["plan_bytes"], dtype=torch.uint8, device=DEVICE)
            s["workspace"] = torch.empty(s["workspace_bytes"], dtype=torch.uint8, device=DEVICE)
            gk.check(gk.flash_attention_extend_plan(
                s["plan"], s["plan_bytes"], s["row_offsets"], s["prior_lengths"], *shape, case["window"], case["sinks"]))
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _bits(t):
    return t.view(torch.int16)


def run(s):
    op = s["case"]["op"]
    if own:
        return {"extend": _own_extend, "fork": _own_fork, "compact": _own_compact, "turnover": _own_turnover}[op](s)
    return {"extend": _plain_extend, "fork": _plain_fork, "compact": _plain_compact, "turnover": _plain_turnover}[op](s)


def _own_extend(s):
    gk, case = s["gk"], s["case"]
    gk.check(gk.flash_attention_extend_paged_bf16(
        s["out"], s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["page_table"], s["plan"], s["plan_bytes"],
        s["config"], 0, case["batch"], s["total"], s["scale"], s["workspace"], s["workspace_bytes"]))
    return s["out"]


def _own_fork(s):
    gk = s["gk"]
    gk.check(gk.kv_cache_release_pages(s["page_table"], s["page_refs"], s["config"], s["first"], s["end"]))
    gk.check(gk.kv_cache_fork_bf16(
        s["cache_k"], s["cache_v"], s["config"], s["page_table"], s["page_refs"], s["seq_lengths"], s["parents"],
        s["children"], s["case"]["children"], s["status"]))
    return {"k": _bits(s["cache_k"]), "v": _bits(s["cache_v"]), "table": s["page_table"], "refs": s["page_refs"],
            "lengths": s["seq_lengths"]}


def _own_compact(s):
    gk = s["gk"]
    gk.check(gk.kv_cache_compact_bf16(
        s["cache_k"], s["cache_v"], s["config"], s["page_table"], s["page_refs"], s["sequences"], s["first"],
        s["kept_offsets"], s["kept_positions"], s["batch"], s["total"], s["status"]))
    return {"k": _bits(s["cache_k"]), "v": _bits(s["cache_v"])}


def _own_turnover(s):
    gk = s["gk"]
    gk.check(gk.kv_cache_release_pages(s["page_table"], s["page_refs"], s["config"], s["release_first"], s["release_end"]))
    gk.check(gk.kv_cache_reserve_pages(s["page_table"], s["page_refs"], s["config"], s["reserve_first"],
                                       s["reserve_end"], s["status"]))
    return {"table": s["page_table"], "refs": s["page_refs"]}


def _plain_extend(s):
    """softmax(scale q K^T + mask) V over the batch, padded to its longest sequence."""
    case, rows, prior = s["case"], s["rows"], s["prior"]
    batch, page, window, sinks = case["batch"], case["page"], case["window"], case["sinks"]
    heads, dim, total = case["heads"], case["dim"], s["total"]
    group, most = QUERY_HEADS // heads, max(rows)
    span = max(p + n - (max(0, p - window + 1) if window else 0) for n, p in zip(rows, prior))
    sinks = sinks if window else 0
    P, O = s["prior_lengths"].long()[:, None], s["row_offsets"].long()
    first = (P - window + 1).clamp(min=0) if window else torch.zeros_like(P)
    # Key positions: the sinks, then from the first key on that row 0's window holds.
    pos = torch.cat([torch.arange(sinks, device=DEVICE).expand(batch, sinks), first + torch.arange(span, device=DEVICE)], 1)
    once = torch.arange(sinks + span, device=DEVICE) < sinks
    once = once | (pos >= sinks)
    n_rows = (O[1:] - O[:-1])[:, None]
    there = once & (pos < P + n_rows)
    slot = (pos // page) % s["max_pages"]
    at = torch.gather(s["page_table"].long(), 1, slot) * page + pos % page
    new = pos >= P
    there = there & (new | (at >= 0))
    chunk = (O[:-1, None] + pos - P).clamp(0, total - 1)
    at = at.clamp(min=0)
    pick = lambda c, x: torch.where(new[..., None, None], x[chunk], c[at]).float().permute(0, 2, 1, 3).contiguous()  # noqa: E731
    line = torch.arange(most, device=DEVICE)
    q = s["q"][(O[:-1, None] + line).clamp(max=total - 1)].float()
    q = q.view(batch, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, dim)
    score = torch.matmul(q, pick(s["cache_k"], s["k"]).transpose(2, 3)) * s["scale"]
    at_row = (P + line)[:, :, None]
    seen = there[:, None] & (pos[:, None] <= at_row)
    if window:
        seen = seen & ((pos[:, None] > at_row - window) | (pos[:, None] < sinks))
    score = score.view(batch, heads, group, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(weight.view(batch, heads, group * most, -1), pick(s["cache_v"], s["v"]))
    out = out.view(batch, heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, QUERY_HEADS, dim)
    of = torch.repeat_interleave(torch.arange(batch, device=DEVICE), n_rows[:, 0], output_size=total)
    return out[of, torch.arange(total, device=DEVICE) - O[:-1][of]].bfloat16()


def _plain_release(s, first, end):
    """Whole pages in [first, end) leave the table; each costs its page one reference."""
    page = s["case"]["page"]
    at = torch.arange(s["max_pages"], device=DEVICE) * page
    table, refs = s["page_table"], s["page_refs"]
    out = (at >= first[:, None]) & (at + page <= end[:, None].long()) & (table >= 0)
    refs.scatter_add_(0, table.clamp(min=0).long().view(-1), -out.int().view(-1))
    table.masked_fill_(out, -1)


def _plain_take(s, wanted):
    """The lowest free pages, in order, for the true places of `wanted`, and -1 elsewhere."""
    refs = s["page_refs"]
    free = torch.argsort((refs > 0).int(), stable=True).int()
    rank = (torch.cumsum(wanted.view(-1).int(), 0) - 1).clamp(0, refs.numel() - 1)
    taken = torch.where(wanted.view(-1), free[rank.long()], torch.full_like(rank, -1, dtype=torch.int32))
    refs.scatter_add_(0, taken.clamp(min=0).long(), (taken >= 0).int())
    return taken.view(wanted.shape)


def _plain_turnover(s):
    _plain_release(s, s["release_first"], s["release_end"])
    page, table = s["case"]["page"], s["page_table"]
    at = torch.arange(s["max_pages"], device=DEVICE) * page
    first, end = s["reserve_first"][:, None], s["reserve_end"][:, None]
    wanted = (at + page > first) & (at < end) & (first < end) & (table < 0)
    table.copy_(torch.where(wanted, _plain_take(s, wanted), table))
    return {"table": table, "refs": s["page_refs"]}


def _plain_fork(s):
    case = s["case"]
    table, refs, lens, page, mp = s["page_table"], s["page_refs"], s["seq_lengths"], case["page"], s["max_pages"]
    _plain_release(s, s["first"], s["end"])
    parents, children = s["parents"].long(), s["children"].long()
    of = table[parents]
    slot = torch.arange(mp, device=DEVICE)
    n = lens[parents][:, None]
    if case["cache"] == "ring":
        shared, copied = torch.zeros_like(of, dtype=torch.bool), of >= 0
    else:
        shared, copied = (of >= 0) & ((slot + 1) * page <= n), (of >= 0) & (slot * page < n) & ((slot + 1) * page > n)
    taken = _plain_take(s, copied)
    refs.scatter_add_(0, of.clamp(min=0).long().view(-1), shared.int().view(-1))
    table[children] = torch.where(shared, of, taken)
    lens[children] = lens[parents]
    if s["copied"] is not None:
        c, j, rows = s["copied"]
        line = torch.arange(page, device=DEVICE)
        line = line[None] * (line[None] < rows[:, None])  # past the last row: row 0 again
        src, dst = ((x[c, j].long()[:, None] * page + line).view(-1) for x in (of, taken))
        for cache in (s["cache_k"], s["cache_v"]):
            cache[:, dst] = cache[:, src]
    return {"k": _bits(s["cache_k"]), "v": _bits(s["cache_v"]), "table": table, "refs": refs, "lengths": lens}


def _plain_compact(s):
    page, mp = s["case"]["page"], s["max_pages"]
    off, src = s["kept_offsets"].long(), s["kept_positions"].long()
    of = torch.repeat_interleave(torch.arange(s["batch"], device=DEVICE), off[1:] - off[:-1], output_size=s["total"])
    dst = s["first"].long()[of] + torch.arange(s["total"], device=DEVICE) - off[of]
    table = s["page_table"].long()[s["sequences"].long()[of]]
    row = lambda p: torch.gather(table, 1, ((p // page) % mp)[:, None])[:, 0] * page + p % page  # noqa: E731
    src, dst = row(src), row(dst)
    for cache in (s["cache_k"], s["cache_v"]):
        cache[:, dst] = cache[:, src]
    return {"k": _bits(s["cache_k"]), "v": _bits(s["cache_v"])}


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    op = case["op"]
    row_bytes = case.get("heads", 0) * case.get("dim", 0) * 2
    if op == "extend":
        rows, prior = _lengths(case)
        window, sinks = case["window"], case["sinks"] if case["window"] else 0
        keys = pairs = 0
        for n, p in zip(rows, prior):
            lo = max(0, p - window + 1) if window else 0
            keys += p - min(lo, p) + min(sinks, lo, p)
            for r in range(n):
                at = p + r
                low = max(0, at - window + 1) if window else 0
                pairs += at + 1 - low + min(sinks, low)
        total = sum(rows)
        return {"bytes": 2 * keys * row_bytes + 2 * total * row_bytes + 2 * total * QUERY_HEADS * case["dim"] * 2,
                "flops": 4 * QUERY_HEADS * case["dim"] * pairs}
    if op == "fork":
        rng = random.Random(case["lengths"] + 1)
        lens, page = _sequence_lengths(case, case["parents"]), case["page"]
        rows, entries = 0, 0
        for _ in range(case["children"]):
            n = lens[rng.randrange(case["parents"])]
            mp = _ring_pages(case["window"], page) if case["cache"] == "ring" else 0
            rows += min(mp, -(-n // page)) * page if mp else n % page
            entries += min(mp, -(-n // page)) if mp else -(-n // page)
        return {"bytes": 2 * 2 * case["layers"] * rows * row_bytes + 5 * 4 * entries, "flops": 0}
    if op == "compact":
        rng = random.Random(case["lengths"] + 1)
        rows = 0
        for n in _sequence_lengths(case, case["batch"]):
            begin = n - min(case["tail"], n) if case["tail"] else 0
            kept = sorted(rng.sample(range(begin, n), min(case["kept"], n - begin)))
            rows += sum(p != begin + j for j, p in enumerate(kept))
        return {"bytes": 2 * 2 * case["layers"] * rows * row_bytes + 4 * rows, "flops": 0}
    # The changing sequences' entries and their pages' counts, and four bounds for each sequence.
    entries = (case["ending"] + case["beginning"]) * -(-case["max_len"] // 2 // case["page"]) + case["batch"]
    return {"bytes": 16 * entries + 16 * case["batch"], "flops": 0}


# ---- the definition in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    """softmax(q.k scale) v over each row's visible keys, sequence by sequence; the other operators move
    values and count pages: nothing is computed."""
    if case["op"] != "extend":
        return None
    s = _make_extend(case, seed)
    page, window, sinks, heads = case["page"], case["window"], case["sinks"], case["heads"]
    out = torch.zeros(s["total"], QUERY_HEADS, case["dim"], dtype=torch.float64, device=DEVICE)
    start = 0
    for b, (n, p) in enumerate(zip(s["rows"], s["prior"])):
        keys = torch.arange(p, device=DEVICE)
        if window:
            keys = keys[(keys > p - window) | (keys < sinks)]
        held = s["page_table"][b].long()[(keys // page) % s["max_pages"]]
        keys, held = keys[held >= 0], held[held >= 0]
        row = held * page + keys % page
        positions = torch.cat([keys, p + torch.arange(n, device=DEVICE)])
        k = torch.cat([s["cache_k"][row], s["k"][start:start + n]]).double()
        v = torch.cat([s["cache_v"][row], s["v"][start:start + n]]).double()
        for r0 in range(0, n, 256):
            at = p + torch.arange(r0, min(n, r0 + 256), device=DEVICE)[:, None]
            seen = positions <= at
            if window:
                seen &= (positions > at - window) | (positions < sinks)
            for h in range(QUERY_HEADS):
                kv = h * heads // QUERY_HEADS
                x = s["q"][start + r0:start + r0 + len(at), h].double() @ k[:, kv].t() / math.sqrt(case["dim"])
                x = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[start + r0:start + r0 + len(at), h] = x @ v[:, kv]
        start += n
    return out
