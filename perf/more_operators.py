"""What is timed and compared of the operators that prepare rows for the paged K/V cache, hold it in
8 bits, and share a prefix's keys among sequences.

A case is a dict of plain values. "op" says which operator:

  "rope"    RMSNorm and rotary positions of a batch's ragged rows, taken out of a projection's wider
            rows. `rotary` leading dims are rotated, in pairs (i, i + rotary / 2) or, `interleaved`,
            (2 i, 2 i + 1); `scaling` of the frequencies for long contexts; `norm`: with RMSNorm of
            q, k and v (of v from the raw k at 1 x 512), else rotation only.
  "write"   rows quantised to e4m3 and written to the paged cache
  "read"    rows of a quantised cache back as bf16
  "decode"  one token per sequence over a quantised cache: its K/V rows appended, then attention
  "shared"  attention of ragged new tokens in groups of sequences whose page tables begin with the
            same pages: `groups` prompts, each with up to `members` sequences behind it

Geometries: 8 KV heads x 256 and 1 KV head x 512, 16 query heads. Lengths come from the case's
"lengths", data and the order of the pages from the seed. A quantised value is code * scale, the
scale fixed for a layer's KV head.
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
EPS = 1e-6
TOP = 448.0  # the largest e4m3 value


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # A server's step on a sliding layer: next tokens, drafts and messages, with q/k norms.
        {"name": "rope_mixed_sliding_b12", "op": "rope", "heads": 8, "dim": 256, "rotary": 256,
         "interleaved": False, "norm": True, "scaling": "none", "batch": 12, "singles": 6,
         "min_rows": 2, "max_rows": 777, "max_prior": 5000, "lengths": 0},
        # A prompt's chunk deep in a context stretched to a million tokens, a quarter of the head.
        {"name": "rope_prompt_global512_2048", "op": "rope", "heads": 1, "dim": 512, "rotary": 128,
         "interleaved": False, "norm": True, "scaling": "parts", "batch": 1, "singles": 0,
         "min_rows": 2048, "max_rows": 2048, "max_prior": 1_000_000, "lengths": 1},
        # The next tokens' K/V of 24 conversations: the smallest call.
        {"name": "write_tokens_global512_b24", "op": "write", "heads": 1, "dim": 512,
         "cache": "full", "page": 64, "window": 0, "batch": 24, "singles": 24, "min_rows": 1,
         "max_rows": 1, "max_prior": 12000, "strided": False, "lengths": 2},
        # Long prompts' rows of a layer, out of the projection's rows.
        {"name": "write_prompts_global256_b4", "op": "write", "heads": 8, "dim": 256,
         "cache": "full", "page": 16, "window": 0, "batch": 4, "singles": 0, "min_rows": 1500,
         "max_rows": 4096, "max_prior": 300, "strided": True, "lengths": 3},
        # A conversation's keys before its next prompt chunk.
        {"name": "read_global512_8000", "op": "read", "heads": 1, "dim": 512, "cache": "full",
         "page": 64, "window": 0, "batch": 1, "min_len": 8000, "max_len": 8000, "lengths": 4},
        # The rings of a batch, all live keys.
        {"name": "read_sliding_b24", "op": "read", "heads": 8, "dim": 256, "cache": "ring",
         "page": 16, "window": WINDOW, "batch": 24, "min_len": 100, "max_len": 6000, "lengths": 5},
        # One conversation's next token on a sliding layer, ring long wrapped.
        {"name": "decode_sliding_b1", "op": "decode", "heads": 8, "dim": 256, "cache": "ring",
         "page": 1, "window": WINDOW, "batch": 1, "min_len": 8193, "max_len": 8193, "lengths": 6},
        # A global layer of the model, 24 conversations of all lengths.
        {"name": "decode_global512_b24", "op": "decode", "heads": 1, "dim": 512, "cache": "full",
         "page": 64, "window": 0, "batch": 24, "min_len": 200, "max_len": 12001, "lengths": 7},
        # A full-length cache of 8 KV heads under a serving batch: the largest read.
        {"name": "decode_global256_b48", "op": "decode", "heads": 8, "dim": 256, "cache": "full",
         "page": 64, "window": 0, "batch": 48, "min_len": 512, "max_len": 16384, "lengths": 8},
        # Samples of one long prompt, a little behind it.
        {"name": "shared_samples_global512_b32", "op": "shared", "heads": 1, "dim": 512, "page": 64,
         "groups": 1, "members": 32, "min_members": 32, "min_prefix": 8000, "max_prefix": 8000,
         "min_own": 10, "max_own": 400, "singles": 32, "min_rows": 1, "max_rows": 1, "lengths": 9},
        # Three system prompts under conversations of all lengths, some with drafts to verify.
        {"name": "shared_mixed_global256_b40", "op": "shared", "heads": 8, "dim": 256, "page": 16,
         "groups": 3, "members": 24, "min_members": 6, "min_prefix": 1500, "max_prefix": 6000,
         "min_own": 0, "max_own": 1500, "singles": 24, "min_rows": 2, "max_rows": 9, "lengths": 10},
        # A beam of 4.
        {"name": "shared_beam_global512_b4", "op": "shared", "heads": 1, "dim": 512, "page": 64,
         "groups": 1, "members": 4, "min_members": 4, "min_prefix": 2000, "max_prefix": 2000,
         "min_own": 30, "max_own": 30, "singles": 4, "min_rows": 1, "max_rows": 1, "lengths": 11},
    ]


def _log_int(rng, low, high):
    high = max(low, high)
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _geometry(rng):
    return rng.choice([(8, 256), (1, 512)])


def _draw_rope(rng):
    heads, dim = _geometry(rng)
    batch = _log_int(rng, 1, 24)
    rows = _log_int(rng, 1, 4000 // batch)
    return {"op": "rope", "heads": heads, "dim": dim,
            "rotary": rng.choice([dim, dim // 2, dim // 4, 16 * rng.randint(1, dim // 16)]),
            "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.7,
            "scaling": rng.choice(["none", "linear", "base", "parts"]), "batch": batch,
            "singles": rng.randint(0, batch) if rows > 1 else batch, "min_rows": _log_int(rng, 1, rows),
            "max_rows": rows, "max_prior": _log_int(rng, 1, 2_000_000), "lengths": rng.randrange(1 << 20)}


def _draw_write(rng):
    heads, dim = _geometry(rng)
    ring = heads == 8 and rng.random() < 0.5
    batch = _log_int(rng, 1, 48)
    rows = _log_int(rng, 1, min(WINDOW if ring else 4096, 9000 // batch))
    return {"op": "write", "heads": heads, "dim": dim, "cache": "ring" if ring else "full",
            "page": rng.choice([1, 16, 64]) if ring else rng.choice([16, 64]), "window": WINDOW if ring else 0,
            "batch": batch, "singles": rng.randint(0, batch) if rows > 1 else batch,
            "min_rows": _log_int(rng, 1, rows), "max_rows": rows,
            "max_prior": _log_int(rng, 1, 20000 if ring else 150_000 // batch // heads),
            "strided": rng.random() < 0.5, "lengths": rng.randrange(1 << 20)}


def _draw_read(rng):
    heads, dim = _geometry(rng)
    ring = heads == 8 and rng.random() < 0.5
    batch = _log_int(rng, 1, 24)
    length = _log_int(rng, 1, 6000 if ring else 24_000 // batch)
    return {"op": "read", "heads": heads, "dim": dim, "cache": "ring" if ring else "full",
            "page": rng.choice([1, 16, 64]) if ring else rng.choice([16, 64]), "window": WINDOW if ring else 0,
            "batch": batch, "min_len": _log_int(rng, 1, length), "max_len": length,
            "lengths": rng.randrange(1 << 20)}


def _draw_decode(rng):
    heads, dim = _geometry(rng)
    ring = heads == 8 and rng.random() < 0.4
    batch = _log_int(rng, 1, 64)
    length = _log_int(rng, 1, 20000 if ring else min(40_000, (700_000 if heads == 1 else 400_000) // batch))
    return {"op": "decode", "heads": heads, "dim": dim, "cache": "ring" if ring else "full",
            "page": rng.choice([1, 16, 64]) if ring else rng.choice([16, 64]), "window": WINDOW if ring else 0,
            "batch": batch, "min_len": _log_int(rng, 1, length), "max_len": length,
            "lengths": rng.randrange(1 << 20)}


def _draw_shared(rng):
    heads, dim = _geometry(rng)
    groups = _log_int(rng, 1, 4)
    members = _log_int(rng, 2, 64 // groups)
    prefix = _log_int(rng, 16, 16000 // groups)
    behind = _log_int(rng, 1, 40_000 // (groups * members))
    rows = _log_int(rng, 1, 12)
    return {"op": "shared", "heads": heads, "dim": dim, "page": rng.choice([16, 64]), "groups": groups,
            "members": members, "min_members": rng.randint(1, members),
            "min_prefix": _log_int(rng, 1, prefix), "max_prefix": prefix,
            "min_own": rng.choice([0, _log_int(rng, 1, behind)]), "max_own": behind,
            "singles": rng.choice([groups * members, rng.randint(0, groups * members)]), "min_rows": 1,
            "max_rows": rows, "lengths": rng.randrange(1 << 20)}


def draw(rng):
    return rng.choice([_draw_decode] * 3 + [_draw_shared] * 3 + [_draw_rope, _draw_write, _draw_read])(rng)


# ---- what a user's program holds ---------------------------------------------------------------

def _spread(rng, low, high, count):
    """`count` lengths of low..high, one of them high."""
    out = [rng.randint(min(low, high), high) for _ in range(count)]
    out[rng.randrange(count)] = high
    return out


def _rows(rng, case, batch):
    """New rows of each sequence."""
    singles = min(case["singles"], batch)
    rows = [1] * singles + [_log_int(rng, case["min_rows"], case["max_rows"]) for _ in range(batch - singles)]
    if singles < batch:
        rows[-1] = case["max_rows"]
    rng.shuffle(rows)
    return rows


def _lengths(case):
    """What the scheduler knows of the batch, by operator: lists of numbers."""
    rng = random.Random(case["lengths"])
    op = case["op"]
    if op in ("rope", "write"):
        rows = _rows(rng, case, case["batch"])
        return rows, _spread(rng, 0, case["max_prior"], case["batch"])
    if op in ("read", "decode"):
        return _spread(rng, case["min_len"], case["max_len"], case["batch"])
    page = case["page"]
    sizes = _spread(rng, case["min_members"], case["members"], case["groups"])
    prefix = [p // page * page for p in _spread(rng, case["min_prefix"], case["max_prefix"], case["groups"])]
    behind = _spread(rng, case["min_own"], case["max_own"], sum(sizes))
    return sizes, prefix, behind, _rows(rng, case, sum(sizes))


def _ring_pages(window, page):
    return (window + 2 * page - 2) // page


def _max_pages(case, longest):
    return _ring_pages(case["window"], case["page"]) if case["cache"] == "ring" else -(-longest // case["page"])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


class _Inputs:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed * 1_000_003 + 31)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device=DEVICE, dtype=torch.bfloat16)

    def weight(self, n):
        return (1 + 0.3 * torch.randn(n, generator=self.gen, device=DEVICE)).bfloat16()

    def scales(self, heads):
        """What a calibration found for each KV head."""
        return 0.01 + 0.04 * torch.rand(1, heads, generator=self.gen, device=DEVICE)

    def codes(self, rows, heads, dim):
        """e4m3 bytes of a cache in use."""
        out = torch.empty(rows, heads, dim, dtype=torch.uint8, device=DEVICE)
        for at in range(0, rows, 1 << 16):
            part = out[at:at + (1 << 16)]
            x = torch.randn(part.shape, generator=self.gen, device=DEVICE, dtype=torch.bfloat16) * 40
            part.copy_(x.clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(torch.uint8))
        return out

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=DEVICE).to(torch.int32)


def _table(mapped, max_pages, order):
    """Page table of sequences whose logical pages `mapped[b]` (a list) are the pool's pages of these
    numbers, in the order of a pool that has been in use for a while."""
    at = torch.tensor([list(m) + [-1] * (max_pages - len(m)) for m in mapped], device=DEVICE, dtype=torch.int64)
    return torch.where(at >= 0, order[at.clamp(min=0)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()


def _counted(counts):
    """Pages of sequences that share none."""
    used = [sum(counts[:b]) for b in range(len(counts) + 1)]
    return [range(used[b], used[b + 1]) for b in range(len(counts))], used[-1]


def _offsets(counts):
    return [sum(counts[:b]) for b in range(len(counts) + 1)]


def _tokens(rows, first):
    """(sequence, position) of the packed rows."""
    return (_int32([b for b, n in enumerate(rows) for _ in range(n)]),
            _int32([p + r for n, p in zip(rows, first) for r in range(n)]))


def _turns(case):
    """Rotations per position of each pair, and the amplitude: theta^(-2 i / rotary) / 2 pi, scaled."""
    factor, context, rotary = 8.0, 32768.0, case["rotary"]
    theta = 1e4 if case["heads"] == 8 else 1e6
    i = torch.arange(rotary // 2, dtype=torch.float64)
    if case["scaling"] == "base":
        theta *= factor ** (rotary / (rotary - 2))
    turns = theta ** (-2 * i / rotary) / (2 * math.pi)
    if case["scaling"] == "linear":
        turns = turns / factor
    if case["scaling"] == "parts":
        kept = ((turns * context - 1) / (32 - 1)).clamp(0, 1)
        turns = turns * (kept + (1 - kept) / factor)
    return turns.to(DEVICE), 0.1 * math.log(factor) + 1 if case["scaling"] == "parts" else 1.0


def _make_rope(case, seed):
    i = _Inputs(seed)
    rows, prior = _lengths(case)
    heads, dim, total = case["heads"], case["dim"], sum(rows)
    own_v = heads > 1  # at 1 x 512 the value is the raw key's
    width = QUERY_HEADS * dim, heads * dim
    projected = i.normal(total, width[0] + (2 if own_v else 1) * width[1])
    q, k, *v = projected.split([width[0], width[1]] + [width[1]] * own_v, 1)
    s = {"q": q, "k": k, "v": v[0] if own_v else None, "stride": projected.shape[1], "total": total,
         "q_weight": i.weight(dim), "k_weight": i.weight(dim), "position": _tokens(rows, prior)[1],
         "q_out": i.normal(total, QUERY_HEADS, dim), "k_out": i.normal(total, heads, dim)}
    s["turns"], s["amplitude"] = _turns(case)
    s["v_out"] = torch.empty_like(s["k_out"]) if case["norm"] else None
    return s


def _make_write(case, seed):
    i = _Inputs(seed)
    rows, prior = _lengths(case)
    heads, dim, page, total = case["heads"], case["dim"], case["page"], sum(rows)
    max_pages = _max_pages(case, max(n + p for n, p in zip(rows, prior)))
    mapped, pages = _counted([min(max_pages, -(-(n + p) // page)) for n, p in zip(rows, prior)])
    s = {"pages": pages, "max_pages": max_pages, "total": total,
         "page_table": _table(mapped, max_pages, i.order(pages))}
    s["batch_of"], s["position"] = _tokens(rows, prior)
    projected = i.normal(total, heads * dim * (4 if case["strided"] else 2))
    if case["strided"]:
        s["k"], s["v"] = projected[:, heads * dim:2 * heads * dim], projected[:, 2 * heads * dim:3 * heads * dim]
    else:
        s["k"], s["v"] = (projected.view(2, total, heads * dim)[j] for j in range(2))
    s["cache_k"], s["cache_v"] = (i.codes(pages * page, heads, dim) for _ in range(2))
    s["k_scales"], s["v_scales"] = i.scales(heads), i.scales(heads)
    return s


def _make_cache(case, i, lens):
    page = case["page"]
    max_pages = _max_pages(case, max(lens))
    mapped, pages = _counted([min(max_pages, -(-n // page)) for n in lens])
    s = {"pages": pages, "max_pages": max_pages, "page_table": _table(mapped, max_pages, i.order(pages))}
    s["cache_k"], s["cache_v"] = (i.codes(pages * page, case["heads"], case["dim"]) for _ in range(2))
    s["k_scales"], s["v_scales"] = i.scales(case["heads"]), i.scales(case["heads"])
    return s


def _make_read(case, seed):
    i = _Inputs(seed)
    lens = _lengths(case)
    s = _make_cache(case, i, lens)
    live = [min(n, case["window"]) if case["window"] else n for n in lens]
    s["batch_of"], s["position"] = _tokens(live, [n - m for n, m in zip(lens, live)])
    s["total"] = sum(live)
    s["k_out"], s["v_out"] = (torch.empty(s["total"], case["heads"], case["dim"], dtype=torch.bfloat16, device=DEVICE)
                              for _ in range(2))
    return s


def _make_decode(case, seed):
    i = _Inputs(seed)
    lens, batch = _lengths(case), case["batch"]
    s = _make_cache(case, i, lens)
    s |= {"lens": lens, "seq_lengths": _int32(lens), "position": _int32([n - 1 for n in lens]),
          "q": i.normal(batch, QUERY_HEADS, case["dim"]), "scale": 1.0 / math.sqrt(case["dim"])}
    s["k"], s["v"] = (i.normal(batch, case["heads"], case["dim"]) for _ in range(2))
    s["out"] = torch.empty_like(s["q"])
    return s


def _make_shared(case, seed):
    i = _Inputs(seed)
    sizes, prefix, behind, rows = _lengths(case)
    heads, dim, page = case["heads"], case["dim"], case["page"]
    group_of = [g for g, n in enumerate(sizes) for _ in range(n)]
    prior = [prefix[g] + b for g, b in zip(group_of, behind)]
    shared, used = _counted([p // page for p in prefix])
    rest, more = _counted([-(-(b + n) // page) for b, n in zip(behind, rows)])
    mapped = [list(shared[g]) + [used + p for p in r] for g, r in zip(group_of, rest)]
    pages, max_pages, total = used + more, max(map(len, mapped)), sum(rows)
    s = {"rows": rows, "prior": prior, "prefix": prefix, "sizes": sizes, "behind": behind, "pages": pages,
         "max_pages": max_pages, "total": total, "page_table": _table(mapped, max_pages, i.order(pages)),
         "row_offsets": _int32(_offsets(rows)), "prior_lengths": _int32(prior),
         "group_offsets": _int32(_offsets(sizes)), "group_of": torch.tensor(group_of, device=DEVICE),
         "prefix_lengths": torch.tensor(prefix, device=DEVICE), "scale": 1.0 / math.sqrt(dim)}
    s["cache_k"], s["cache_v"] = (i.normal(pages * page, heads, dim) for _ in range(2))
    s["q"] = i.normal(total, QUERY_HEADS, dim)
    s["k"], s["v"] = (i.normal(total, heads, dim) for _ in range(2))
    s["out"] = torch.empty_like(s["q"])
    return s


_MAKE = {"rope": _make_rope, "write": _make_write, "read": _make_read, "decode": _make_decode, "shared": _make_shared}


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
        op = case["op"]
        if op != "rope":
            batch = sum(s["sizes"]) if op == "shared" else case["batch"]
            s["batch"] = batch
            s["config"] = gk.make_config(1, s["pages"], case["page"], s["max_pages"], batch, case["heads"],
                                         case["dim"], case.get("window", 0) if case.get("cache") == "ring" else 0)
        if op == "decode":  # the splits of the batch's longest sequence, and their partial sums
            live = max(min(n, case["window"]) if case["window"] else n for n in s["lens"])
            s["split_size"], s["num_splits"] = gk.decode_split_plan_fp8(s["config"], case["batch"], live)
            slots = case["batch"] * QUERY_HEADS * s["num_splits"]
            s["m"], s["l"], s["acc"] = (torch.empty(slots * n, dtype=torch.float32, device=DEVICE)
                                        for n in (1, 1, case["dim"]))
        if op == "shared":  # a step's plan serves all of its layers
            shape = (s["config"], batch, s["total"])
            s["plan_bytes"] = gk.flash_attention_extend_shared_plan_bytes(*shape)
            s["workspace_bytes"] = gk.flash_attention_extend_shared_workspace_bytes(*shape)
            s["plan"] = torch.empty(s["plan_bytes"], dtype=torch.uint8, device=DEVICE)
            s["workspace"] = torch.empty(s["workspace_bytes"], dtype=torch.uint8, device=DEVICE)
            gk.check(gk.flash_attention_extend_shared_plan(
                s["plan"], s["plan_bytes"], s["row_offsets"], s["prior_lengths"], s["page_table"],
                s["group_offsets"], case["groups"], *shape))
    return s


# ---- one pass ----------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"rope": _own_rope, "write": _own_write, "read": _own_read, "decode": _own_decode,
                "shared": _own_shared}[op](s)
    return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "decode": _plain_decode,
            "shared": _plain_shared}[op](s)


def _values(codes):
    return codes.view(torch.float8_e4m3fn)


def _own_rope(s):
    gk, case = s["gk"], s["case"]
    norm = case["norm"]
    gk.check(gk.rope_rows_bf16(
        s["q_out"], s["k_out"], s["v_out"], s["q"], s["k"], s["v"] if norm else None,
        s["q_weight"] if norm else None, s["k_weight"] if norm else None, s["position"], s["turns"],
        s["amplitude"], case["rotary"], case["interleaved"], case["heads"], case["dim"], s["total"],
        q_stride=s["stride"], kv_stride=s["stride"]))
    return [s["q_out"], s["k_out"]] + ([s["v_out"]] if norm else [])


def _own_write(s):
    gk = s["gk"]
    gk.check(gk.kv_cache_write_fp8(
        s["cache_k"], s["cache_v"], s["config"], s["page_table"], s["batch_of"], s["position"], s["total"], 0,
        s["k"], s["v"], s["k_scales"], s["v_scales"], kv_stride=s["k"].stride(0)))
    return _values(s["cache_k"]), _values(s["cache_v"])


def _own_read(s):
    gk = s["gk"]
    gk.check(gk.kv_cache_read_fp8(
        s["k_out"], s["v_out"], s["cache_k"], s["cache_v"], s["config"], s["page_table"], s["batch_of"],
        s["position"], s["total"], 0, s["k_scales"], s["v_scales"]))
    return s["k_out"], s["v_out"]


def _own_decode(s):
    gk = s["gk"]
    gk.check(gk.flash_attention_append_decode_paged_fp8(
        s["out"], s["m"], s["l"], s["acc"], s["q"], s["cache_k"], s["cache_v"], s["k_scales"], s["v_scales"],
        s["page_table"], s["seq_lengths"], s["position"], s["k"], s["v"], s["config"], 0, s["scale"],
        s["split_size"], s["num_splits"], s["batch"]))
    return s["out"], _values(s["cache_k"]), _values(s["cache_v"])


def _own_shared(s):
    gk = s["gk"]
    gk.check(gk.flash_attention_extend_shared_paged_bf16(
        s["out"], s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["page_table"], s["plan"], s["plan_bytes"],
        s["config"], 0, s["batch"], s["total"], s["scale"], s["workspace"], s["workspace_bytes"]))
    return s["out"]


def _plain_rope(s):
    case = s["case"]
    rotary, heads, dim = case["rotary"], case["heads"], case["dim"]
    # The angle's whole turns go in 64 bits: a far position has thousands of them.
    part = s["position"].double()[:, None] * s["turns"]
    angle = ((part - part.floor()) * (2 * math.pi))
    cos, sin = (f(angle).float()[:, None] * s["amplitude"] for f in (torch.cos, torch.sin))

    def normed(x, n):
        x = x.unflatten(1, (n, dim)).float()
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) if case["norm"] else x

    def rotated(x, n, weight):
        x = normed(x, n)
        if case["norm"]:
            x = x * weight.float()
        turned, rest = x[..., :rotary], x[..., rotary:]
        if case["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([turned, rest], -1).bfloat16()

    out = [rotated(s["q"], QUERY_HEADS, s["q_weight"]), rotated(s["k"], heads, s["k_weight"])]
    return out + ([normed(s["k"] if s["v"] is None else s["v"], heads).bfloat16()] if case["norm"] else [])


def _row_of(s, batch_of, position):
    """Cache row of (sequence, position)."""
    page = s["case"]["page"]
    slot = (position // page) % s["max_pages"]
    return s["page_table"].long()[batch_of, slot] * page + position % page


def _quantised(x, scales):
    """e4m3 bytes of [rows][heads][dim]."""
    return (x.float() / scales[0, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_write(s):
    shape = (s["case"]["heads"], s["case"]["dim"])
    row = _row_of(s, s["batch_of"].long(), s["position"].long())
    s["cache_k"][row] = _quantised(s["k"].unflatten(1, shape), s["k_scales"])
    s["cache_v"][row] = _quantised(s["v"].unflatten(1, shape), s["v_scales"])
    return _values(s["cache_k"]), _values(s["cache_v"])


def _read(s, cache, scales, row):
    return _values(cache[row]).float() * scales[0, :, None]


def _plain_read(s):
    row = _row_of(s, s["batch_of"].long(), s["position"].long())
    return (_read(s, s["cache_k"], s["k_scales"], row).bfloat16(),
            _read(s, s["cache_v"], s["v_scales"], row).bfloat16())


def _plain_decode(s):
    """The append, then softmax(scale q K^T) V over the live keys, padded to the longest."""
    case, lens = s["case"], s["lens"]
    batch, heads, dim, window = case["batch"], case["heads"], case["dim"], case["window"]
    line = torch.arange(batch, device=DEVICE)
    at = _row_of(s, line, s["position"].long())
    s["cache_k"][at] = _quantised(s["k"], s["k_scales"])
    s["cache_v"][at] = _quantised(s["v"], s["v_scales"])
    span = min(max(lens), window) if window else max(lens)
    length = s["seq_lengths"].long()[:, None]
    first = (length - window).clamp(min=0) if window else torch.zeros_like(length)
    position = first + torch.arange(span, device=DEVICE)
    there = position < length
    row = _row_of(s, line[:, None], torch.where(there, position, first))
    pick = lambda cache, scales: (_values(cache[row]).float() * scales[0, :, None]).permute(0, 2, 1, 3).contiguous()  # noqa: E731
    q = s["q"].float().view(batch, heads, QUERY_HEADS // heads, dim)
    score = torch.matmul(q, pick(s["cache_k"], s["k_scales"]).transpose(2, 3)) * s["scale"]
    score = score.masked_fill(~there[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, pick(s["cache_v"], s["v_scales"])).view(batch, QUERY_HEADS, dim).bfloat16()
    return out, _values(s["cache_k"]), _values(s["cache_v"])


def _plain_shared(s):
    """softmax(scale q K^T + mask) V: each group's rows over its prefix in one product, and over the keys
    behind it in another, padded to the longest; one softmax over both."""
    case, sizes, rows = s["case"], s["sizes"], s["rows"]
    heads, dim, page, total = case["heads"], case["dim"], case["page"], s["total"]
    group, batch, groups, most = QUERY_HEADS // heads, len(rows), case["groups"], max(rows)
    span, reach = max(s["prefix"]), max(b + n for b, n in zip(s["behind"], rows))
    O, P = s["row_offsets"].long(), s["prior_lengths"].long()[:, None]
    L = s["prefix_lengths"][s["group_of"]][:, None]
    table = s["page_table"].long()
    line = torch.arange(most, device=DEVICE)
    q = s["q"][(O[:-1, None] + line).clamp(max=total - 1)].float()
    q = q.view(batch, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, dim)
    # Behind the prefix: cached keys, then the rows'.
    position = L + torch.arange(reach, device=DEVICE)
    n_rows = (O[1:] - O[:-1])[:, None]
    slot = (position // page).clamp(max=s["max_pages"] - 1)
    at = torch.where(position < P, torch.gather(table, 1, slot) * page + position % page, 0)
    fresh = (O[:-1, None] + position - P).clamp(0, total - 1)
    pick = lambda c, x: torch.where((position >= P)[..., None, None], x[fresh], c[at]).float().permute(0, 2, 1, 3).contiguous()  # noqa: E731
    score = torch.matmul(q, pick(s["cache_k"], s["k"]).transpose(2, 3)).view(batch, heads, group, most, reach)
    seen = (position < P + n_rows)[:, None] & (position[:, None] <= (P + line)[:, :, None])
    score = (score * s["scale"]).masked_fill(~seen[:, None, None], -math.inf)
    if not span:
        parts = [score]
    else:  # the prefix, by groups padded to the largest
        leader = s["group_offsets"].long()[:-1, None]
        widest = max(sizes)
        member = (leader + torch.arange(widest, device=DEVICE)).clamp(max=batch - 1)
        key = torch.arange(span, device=DEVICE)[None]
        held = key < s["prefix_lengths"][:, None]
        at_prefix = torch.where(held, table[leader, (key // page).clamp(max=s["max_pages"] - 1)] * page + key % page, 0)
        take = lambda c: c[at_prefix].float().permute(0, 2, 1, 3).contiguous()  # noqa: E731
        flat = q[member].permute(0, 2, 1, 3, 4).reshape(groups, heads, widest * group * most, dim)
        first = torch.matmul(flat, take(s["cache_k"]).transpose(2, 3)) * s["scale"]
        first = first.masked_fill(~held[:, None, None], -math.inf).view(groups, heads, widest, group, most, span)
        of = torch.arange(batch, device=DEVICE) - leader[s["group_of"], 0]
        parts = [first[s["group_of"], :, of], score]
    score = torch.cat(parts, -1)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(weight[..., -reach:].reshape(batch, heads, group * most, reach), pick(s["cache_v"], s["v"]))
    if span:
        flat = weight[..., :span][member].permute(0, 2, 1, 3, 4, 5).reshape(groups, heads, widest * group * most, span)
        first = torch.matmul(flat, take(s["cache_v"])).view(groups, heads, widest, group * most, dim)
        out = out + first[s["group_of"], :, of]
    out = out.view(batch, heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, QUERY_HEADS, dim)
    of = torch.repeat_interleave(torch.arange(batch, device=DEVICE), n_rows[:, 0], output_size=total)
    return out[of, torch.arange(total, device=DEVICE) - O[:-1][of]].bfloat16()


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    op, heads, dim = case["op"], case["heads"], case["dim"]
    kv, q = heads * dim, QUERY_HEADS * dim  # elements of a token's K (or V) row, and of its query
    if op == "rope":
        total = sum(_lengths(case)[0])
        norm = case["norm"]
        read = q + kv + (kv if norm and heads > 1 else 0)
        return {"bytes": 2 * total * (read + q + kv + (kv if norm else 0)) + 4 * total,
                "flops": total * 4 * (q + kv)}
    if op == "write":
        total = sum(_lengths(case)[0])
        return {"bytes": total * (2 * kv * 3 + 8), "flops": 0}
    if op == "read":
        total = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
        return {"bytes": total * (2 * kv * 3 + 8), "flops": 0}
    if op == "decode":
        keys = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
        return {"bytes": 2 * keys * kv + case["batch"] * (4 * q + 4 * kv), "flops": 4 * q * keys}
    sizes, prefix, behind, rows = _lengths(case)
    group_of = [g for g, n in enumerate(sizes) for _ in range(n)]
    keys = sum(prefix) + sum(behind)
    pairs = sum(n * (prefix[g] + b) + n * (n + 1) // 2 for g, b, n in zip(group_of, behind, rows))
    total = sum(rows)
    return {"bytes": 4 * keys * kv + 4 * total * kv + 4 * total * q, "flops": 4 * q * pairs}


# ---- the definition in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = _MAKE[case["op"]](case, seed)
    s["case"] = case
    return {"rope": _exact_rope, "write": _exact_write, "read": _exact_read, "decode": _exact_decode,
            "shared": _exact_shared}[case["op"]](s)


def _exact_rope(s):
    """Pairs as complex numbers, turned by amplitude * exp(2 pi i position turns)."""
    case = s["case"]
    dim, half = case["dim"], case["rotary"] // 2
    angle = torch.remainder(s["position"].double()[:, None] * s["turns"], 1.0) * 2 * math.pi
    by = torch.polar(torch.full_like(angle, s["amplitude"]), angle)
    first = torch.arange(half, device=DEVICE) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    got = []
    for name, weight in (("q", "q_weight"), ("k", "k_weight")):
        x = s[name].double().reshape(s["total"], -1, dim)
        if case["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * s[weight].double()
        y = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * by[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        got.append(y)
    if case["norm"]:
        x = s["k" if s["v"] is None else "v"].double().reshape(s["total"], -1, dim)
        got.append(x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt())
    return got


def _exact_codes(x, scale):
    """The nearest e4m3 value to x / scale, ties to even: 3 bits behind the leading one, exponents from -6."""
    x = x.double() / scale.double()[:, None]
    size = x.abs().clamp(max=TOP)
    step = torch.exp2((torch.frexp(size)[1].double() - 1).clamp(min=-6) - 3)
    return torch.copysign(torch.round(size / step) * step, x)


def _exact_rows(s, b, positions):
    page = s["case"]["page"]
    return s["page_table"][b].long()[(positions // page) % s["max_pages"]] * page + positions % page


def _exact_write(s):
    got, case = [], s["case"]
    row = torch.empty(s["total"], dtype=torch.int64, device=DEVICE)
    for b in range(case["batch"]):
        mine = s["batch_of"] == b
        row[mine] = _exact_rows(s, b, s["position"][mine].long())
    for name in ("k", "v"):
        out = _values(s["cache_" + name]).double()
        out[row] = _exact_codes(s[name].reshape(s["total"], case["heads"], case["dim"]), s[name + "_scales"][0])
        got.append(out)
    return tuple(got)


def _exact_read(s):
    got = []
    for name in ("k", "v"):
        parts = []
        for b in range(s["case"]["batch"]):
            row = _exact_rows(s, b, s["position"][s["batch_of"] == b].long())
            parts.append(_values(s["cache_" + name][row]).double() * s[name + "_scales"][0].double()[:, None])
        got.append(torch.cat(parts))
    return tuple(got)


def _exact_decode(s):
    case = s["case"]
    heads, dim, window = case["heads"], case["dim"], case["window"]
    out = torch.zeros(case["batch"], QUERY_HEADS, dim, dtype=torch.float64, device=DEVICE)
    new_k, new_v = (_exact_codes(s[n], s[n + "_scales"][0]) for n in ("k", "v"))
    for name, new in (("cache_k", new_k), ("cache_v", new_v)):
        for b, n in enumerate(s["lens"]):
            row = _exact_rows(s, b, torch.tensor([n - 1], device=DEVICE))
            s[name][row] = new[b].float().to(torch.float8_e4m3fn).view(torch.uint8)
    for b, n in enumerate(s["lens"]):
        row = _exact_rows(s, b, torch.arange(max(0, n - window) if window else 0, n, device=DEVICE))
        k, v = (_values(s["cache_" + c][row]).double() * s[c + "_scales"][0].double()[:, None] for c in ("k", "v"))
        for h in range(QUERY_HEADS):
            kv = h * heads // QUERY_HEADS
            out[b, h] = torch.softmax(k[:, kv] @ s["q"][b, h].double() / math.sqrt(dim), 0) @ v[:, kv]
    whole = [_values(s[c]).double() if s[c].numel() < 1 << 28 else None for c in ("cache_k", "cache_v")]
    return (out, *whole)


def _exact_shared(s):
    case, page = s["case"], s["case"]["page"]
    out = torch.zeros(s["total"], QUERY_HEADS, case["dim"], dtype=torch.float64, device=DEVICE)
    start = 0
    for b, (n, p) in enumerate(zip(s["rows"], s["prior"])):
        keys = torch.arange(p, device=DEVICE)
        row = s["page_table"][b].long()[keys // page] * page + keys % page
        k = torch.cat([s["cache_k"][row], s["k"][start:start + n]]).double()
        v = torch.cat([s["cache_v"][row], s["v"][start:start + n]]).double()
        hidden = torch.arange(p + n, device=DEVICE) > p + torch.arange(n, device=DEVICE)[:, None]
        for h in range(QUERY_HEADS):
            kv = h * case["heads"] // QUERY_HEADS
            x = s["q"][start:start + n, h].double() @ k[:, kv].t() / math.sqrt(case["dim"])
            out[start:start + n, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[:, kv]
        start += n
    return out
