"""Cases for the attention operators over the paged KV pool.

Three operators read (and one rearranges) the pool that ``tcx_kv_gather`` gathers from:

* ``attention``: the newest tokens of every sequence attend over the sequence's pages, with an
  optional sliding window and a few first tokens that stay visible (sinks); one query token per
  sequence (decode) or many (a prompt, or the last chunk of one);
* ``shared``: the same for a batch whose sequences share one long prefix, held in pages of its own;
* ``weights``: attention that also adds every visible token's softmax weight to the accumulators
  that ``evict`` ranks by, and ``evict``: each sequence's first tokens, newest tokens and highest
  accumulated weights are kept, copied in order into new pages.

``run`` computes them with elementary torch operations, or through the package where ``own`` is set.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one chat session generating a token: latency counts
        {"name": "decode_one", "op": "attention", "seqs": 1, "lo": 777, "hi": 777, "queries": 1, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 0, "sinks": 0},
        # a serving batch of the paged-KV benchmark's lengths (64-4096 tokens), one token each
        {"name": "decode_batch", "op": "attention", "seqs": 96, "lo": 64, "hi": 4096, "queries": 1, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 0, "sinks": 0},
        # streaming sessions with long caches: a window and four first tokens
        {"name": "decode_window", "op": "attention", "seqs": 16, "lo": 9000, "hi": 40000, "queries": 1,
         "q_heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "type": "fp16", "window": 4096, "sinks": 4},
        # several prompts at once, whole, behind a window with sinks
        {"name": "prompt_window", "op": "attention", "seqs": 6, "lo": 100, "hi": 4000, "queries": 0, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 1024, "sinks": 4},
        # the last chunk of a long prompt
        {"name": "prompt_chunk", "op": "attention", "seqs": 1, "lo": 40011, "hi": 40011, "queries": 2048,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 0, "sinks": 0},
        # a handful of requests behind one system prompt, a small model's heads
        {"name": "shared_few", "op": "shared", "seqs": 5, "lo": 1, "hi": 60, "queries": 1, "q_heads": 8,
         "kv_heads": 2, "dim": 64, "page": 16, "type": "bf16", "window": 0, "sinks": 0, "prefix": 1003},
        # many samples of one long document
        {"name": "shared_batch", "op": "shared", "seqs": 64, "lo": 1, "hi": 700, "queries": 1, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 0, "sinks": 0, "prefix": 8200},
        # a large batch behind a long prefix
        {"name": "shared_large", "op": "shared", "seqs": 128, "lo": 90, "hi": 1000, "queries": 1, "q_heads": 64,
         "kv_heads": 8, "dim": 128, "page": 32, "type": "fp16", "window": 0, "sinks": 0, "prefix": 20000},
        # decode that keeps the accumulators up to date
        {"name": "weights_decode", "op": "weights", "seqs": 40, "lo": 500, "hi": 4096, "queries": 1, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 0, "sinks": 0},
        # the last tokens of two prompts rank the prompts' tokens before the first eviction
        {"name": "weights_prompt", "op": "weights", "seqs": 2, "lo": 5001, "hi": 6100, "queries": 256, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "window": 0, "sinks": 0},
        # one layer of one session goes back to its budget
        {"name": "evict_one", "op": "evict", "seqs": 1, "lo": 700, "hi": 700, "layers": 1, "kv_heads": 8, "dim": 128,
         "page": 16, "type": "bf16", "budget": 512, "sinks": 4, "recent": 128},
        # a batch's caches cut to a budget, several layers at once; the shorter sequences keep all
        {"name": "evict_batch", "op": "evict", "seqs": 24, "lo": 500, "hi": 8192, "layers": 4, "kv_heads": 8,
         "dim": 128, "page": 16, "type": "bf16", "budget": 2048, "sinks": 4, "recent": 256},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "shared", "weights", "evict"])
    kv_heads, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128])
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([8, 16, 24, 32, 64, 128]),
            "type": rng.choice(["bf16", "fp16"])}
    if op == "evict":
        case |= {"seqs": _log(rng, 1, 24), "layers": rng.randint(1, 4), "lo": _log(rng, 1, 500),
                 "hi": _log(rng, 500, 8192), "sinks": rng.randint(0, 8), "recent": _log(rng, 1, 60),
                 "budget": _log(rng, 70, 2048)}
        return case
    case |= {"q_heads": kv_heads * rng.choice([1, 2, 4, 5, 8]), "window": 0, "sinks": 0}
    if rng.random() < 0.4:
        case |= {"window": _log(rng, 1, 4096), "sinks": rng.randint(0, 5)}
    if op == "attention" and rng.random() < 0.5:  # prompts, whole or their last chunk
        case |= {"seqs": rng.randint(1, 4), "lo": _log(rng, 1, 300), "hi": _log(rng, 300, 4000),
                 "queries": rng.choice([0, _log(rng, 2, 1000)])}
    elif op == "weights" and rng.random() < 0.4:
        case |= {"seqs": rng.randint(1, 3), "lo": _log(rng, 1, 300), "hi": _log(rng, 300, 4000),
                 "queries": _log(rng, 2, 128)}
    elif op == "shared":
        case |= {"seqs": _log(rng, 2, 100), "lo": _log(rng, 1, 20), "hi": _log(rng, 20, 800), "queries": 1,
                 "prefix": _log(rng, 30, 9000)}
    else:
        case |= {"seqs": _log(rng, 1, 64), "lo": _log(rng, 1, 400), "hi": _log(rng, 400, 6000),
                 "queries": rng.choice([1, 1, 1, 2, 4])}
    return case


def _lengths(case):
    """Tokens and query tokens of each sequence: a case has the same ones for every seed."""
    rng = random.Random("%(seqs)d %(lo)d %(hi)d %(page)d" % case)
    tokens = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    queries = case.get("queries", 0)
    return tokens, [min(n, queries) if queries else n for n in tokens]


def _visible(case, tokens, queries):
    """(tokens that any of the sequence's queries sees, pairs of a query and a token that it sees), with
    positions counted from the start of the prefix."""
    prefix, window, sinks = case.get("prefix", 0), case["window"], case["sinks"]
    pos = np.arange(prefix + tokens - queries, prefix + tokens, dtype=np.int64)
    if not window:
        return prefix + tokens, int((pos + 1).sum())
    low = np.maximum(pos - window + 1, 0)
    pairs = pos + 1 - np.maximum(low - sinks, 0) if sinks else pos + 1 - low
    first = int(low[0])
    return prefix + tokens - max(first - sinks, 0), int(pairs.sum())


def work(case):
    tokens, queries = _lengths(case)
    size, kv_heads, dim = 2, case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in tokens)
        heads = case["layers"] * kv_heads
        # weights read; indices, weights and both planes' rows written; the rows read
        return {"bytes": heads * (4 * sum(tokens) + kept * (8 + 4 * dim * size)), "flops": 2 * heads * sum(tokens)}
    seen = [_visible(case, n, m) for n, m in zip(tokens, queries)]
    prefix = case.get("prefix", 0)
    if prefix:  # the prefix is read once: what the sequence that sees most of it sees
        own_part = [min(n, s[0]) for n, s in zip(tokens, seen)]
        rows = sum(own_part) + max(s[0] - o for s, o in zip(seen, own_part))
    else:
        rows = sum(s[0] for s in seen)
    pairs, total = sum(s[1] for s in seen), sum(queries)
    moved = rows * kv_heads * dim * 2 * size + total * case["q_heads"] * (2 * dim * size + 4)
    flops = pairs * case["q_heads"] * 4 * dim
    if case["op"] == "weights":
        moved += 8 * rows * kv_heads
        flops += pairs * case["q_heads"] * 2
    return {"bytes": moved, "flops": flops}


class _Pages:
    """Page tables of `tokens`, their slots taken from `slots` in turn."""

    def __init__(self, tokens, page, slots):
        pages = [-(-n // page) for n in tokens]
        self.tokens = np.array(tokens, np.uint32)
        self.offsets = np.concatenate([[0], np.cumsum(pages)]).astype(np.uint64)
        self.table = slots[: int(self.offsets[-1])].astype(np.uint32)
        self.capacity = int(self.offsets[-1]) * page


def _token_rows(pages, page, tokens, device):
    """[sequence, token] -> row of the pool (slot * page + place), with 0 for tokens behind the last."""
    longest = max(max(tokens), 1)
    rows = np.zeros((len(tokens), longest), np.int64)
    for s, n in enumerate(tokens):
        at = np.arange(n)
        rows[s, :n] = pages.table[int(pages.offsets[s]) + at // page].astype(np.int64) * page + at % page
    return torch.from_numpy(rows).to(device)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 7919 + 17)
    kind = TYPES[case["type"]]
    tokens, queries = _lengths(case)
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    layers = case.get("layers", 1)
    kept = [min(n, case["budget"]) for n in tokens] if case["op"] == "evict" else []
    prefix = case.get("prefix", 0)
    need = sum(-(-n // page) for n in tokens + kept + [prefix])
    pool_pages = need + 5
    slots = np.random.default_rng(int(seed)).permutation(pool_pages)
    pages = _Pages(tokens, page, slots)
    slots = slots[len(pages.table):]
    pool = torch.randn((2 * layers, pool_pages * page, kv_heads, dim), generator=g, device=device).to(kind)
    st = {"case": case, "pool": pool, "tokens": tokens, "queries": queries, "pages": pages, "pool_pages": pool_pages,
          "rows": _token_rows(pages, page, tokens, device), "length": torch.tensor(tokens, device=device),
          "scale": dim ** -0.5}
    if case["op"] in ("weights", "evict"):
        # accumulated softmax weights: a few tokens hold most of the mass
        st["weights"] = torch.exp(2.5 * torch.randn((layers, kv_heads, pages.capacity), generator=g, device=device))
        col = [int(pages.offsets[s]) * page + np.arange(n) for s, n in enumerate(tokens)]
        at = [s * st["rows"].shape[1] + np.arange(n) for s, n in enumerate(tokens)]
        st["columns"] = torch.from_numpy(np.concatenate(col)).to(device)
        st["places"] = torch.from_numpy(np.concatenate(at)).to(device)
    if case["op"] == "evict":
        dst = _Pages(kept, page, slots)
        st |= {"dst": dst, "budget": case["budget"], "kept": torch.tensor(kept, device=device)}
        at = [s * max(kept) + np.arange(n) for s, n in enumerate(kept)]
        col = [int(dst.offsets[s]) * page + np.arange(n) for s, n in enumerate(kept)]
        st["kept_places"] = torch.from_numpy(np.concatenate(at)).to(device)
        st["kept_columns"] = torch.from_numpy(np.concatenate(col)).to(device)
        st["kept_rows"] = _token_rows(dst, page, kept, device).reshape(-1)[st["kept_places"]]
    else:
        total, heads = sum(queries), case["q_heads"]
        # the queries are a part of the fused projection's output, as the model has them
        fused = torch.randn((total, (heads + 2 * kv_heads) * dim), generator=g, device=device) * 1.5
        st["q"] = fused.to(kind)[:, : heads * dim].unflatten(1, (heads, dim))
        most = max(queries)
        first = np.cumsum([0] + queries)
        where = np.stack([first[s] + np.minimum(np.arange(most), m - 1) for s, m in enumerate(queries)])
        st["q_rows"] = torch.from_numpy(where).to(device)
        st["q_places"] = torch.from_numpy(np.concatenate(
            [s * most + np.arange(m) for s, m in enumerate(queries)])).to(device)
        st["first"] = torch.tensor([n - m for n, m in zip(tokens, queries)], device=device)
        st["q_count"] = torch.tensor(queries, device=device)
        if prefix:
            st["prefix"] = _Pages([prefix], page, slots)
            st["prefix_rows"] = _token_rows(st["prefix"], page, [prefix], device)[0]
    if own:
        _handles(st)
    return st


def _handles(st):
    """What a serving program builds once for a batch: its tables on the device."""
    from tensorcast_b200.kvattention import KvAttention, KvEvict
    from tensorcast_b200.kvcache import KvWorkload
    case, pages = st["case"], st["pages"]
    kind, page = TYPES[case["type"]], case["page"]
    token_bytes = case["kv_heads"] * case["dim"] * 2
    tables = lambda p: KvWorkload(st["pool"].shape[0], st["pool_pages"], page, token_bytes,  # noqa: E731
                                  p.tokens, p.offsets, p.table)
    if case["op"] == "evict":
        st["handle"] = KvEvict(tables(pages), tables(st["dst"]), case["kv_heads"], sinks=case["sinks"],
                               recent=case["recent"])
        return
    more = {"prefix_pages": st["prefix"].table, "prefix_tokens": case["prefix"]} if "prefix" in st else {}
    st["handle"] = KvAttention(tables(pages), case["q_heads"], case["kv_heads"], kind, query_tokens=st["queries"],
                               window=case["window"], sinks=case["sinks"], **more)


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "evict":
            keep, weights, tokens = state["handle"].run(state["pool"], state["weights"])
            return {"keep": keep, "weights": weights, "tokens": tokens, "pool": state["pool"]}
        if op == "weights":
            out, lse = state["handle"].run(state["pool"], 0, state["q"], weights=state["weights"][0])
            return {"out": out, "lse": lse, "weights": state["weights"]}
        out, lse = state["handle"].run(state["pool"], 0, state["q"])
        return {"out": out, "lse": lse}
    return _evict(state) if op == "evict" else _attention(state)


def _attention(st):
    """softmax(scale q k^T) v over the visible tokens, all sequences padded to the longest."""
    case, pool = st["case"], st["pool"]
    heads, kv_heads, dim = case["q_heads"], case["kv_heads"], case["dim"]
    group, prefix = heads // kv_heads, case.get("prefix", 0)
    rows = st["rows"]
    batch, longest = rows.shape
    if prefix:
        rows = torch.cat([st["prefix_rows"].expand(batch, prefix), rows], 1)
    spots = torch.arange(longest + prefix, device=rows.device)
    valid = spots < st["length"][:, None] + prefix
    k = pool[0][rows].float().permute(0, 2, 3, 1)                                   # [batch, kv head, dim, token]
    v = torch.where(valid[:, :, None, None], pool[1][rows].float(), 0.0).permute(0, 2, 1, 3)
    most = st["q_rows"].shape[1]
    q = st["q"][st["q_rows"]].float().view(batch, most, kv_heads, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, most * group, dim)
    s = torch.matmul(q * st["scale"], k)
    pos = prefix + st["first"][:, None] + torch.arange(most, device=rows.device)      # [batch, query]
    see = (spots <= pos[:, :, None]) & valid[:, None]
    if case["window"]:
        see &= (spots > pos[:, :, None] - case["window"]) | (spots < case["sinks"])
    see &= (torch.arange(most, device=rows.device) < st["q_count"][:, None])[:, :, None]
    see = see[:, None, :, None].expand(batch, 1, most, group, -1).reshape(batch, 1, most * group, -1)
    s = torch.where(see, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).view(batch, kv_heads, most, group).permute(0, 2, 1, 3)
    p = p / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, v).view(batch, kv_heads, most, group, dim).permute(0, 2, 1, 3, 4)
    out = out.reshape(batch * most, heads, dim)[st["q_places"]].to(st["q"].dtype)
    got = {"out": out, "lse": lse.reshape(batch * most, heads)[st["q_places"]]}
    if case["op"] == "weights":
        added = p.sum(2).permute(1, 0, 2).reshape(kv_heads, -1)[:, st["places"]]
        st["weights"][0].index_add_(1, st["columns"], added)
        got["weights"] = st["weights"]
    return got


def _evict(st):
    """Stable descending sort of the weights, the protected tokens first; kept rows copied in their old order."""
    case, pool = st["case"], st["pool"]
    layers, kv_heads, page = case["layers"], case["kv_heads"], case["page"]
    batch, longest = st["rows"].shape
    weights = torch.full((layers, kv_heads, batch * longest), float("-inf"), device=pool.device)
    weights[:, :, st["places"]] = st["weights"][:, :, st["columns"]]
    weights = weights.view(layers, kv_heads, batch, longest)
    spots = torch.arange(longest, device=pool.device)
    safe = (spots < case["sinks"]) | (spots >= st["length"][:, None] - case["recent"])
    safe &= spots < st["length"][:, None]
    order = torch.sort(torch.where(safe, float("inf"), weights), dim=-1, descending=True, stable=True).indices
    order = torch.where(spots < st["kept"][:, None], order, longest)
    most = int(min(case["budget"], longest))
    index = torch.sort(order, dim=-1).values[..., :most].reshape(layers, kv_heads, batch * most)[:, :, st["kept_places"]]
    flat = index + (st["kept_places"] // most) * longest
    keep = torch.full((layers, kv_heads, st["dst"].capacity), -1, dtype=torch.int32, device=pool.device)
    keep[:, :, st["kept_columns"]] = index.int()
    left = torch.zeros((layers, kv_heads, st["dst"].capacity), device=pool.device)
    left[:, :, st["kept_columns"]] = weights.view(layers, kv_heads, -1).gather(2, flat)
    source = st["rows"].reshape(-1)[flat].transpose(1, 2).repeat_interleave(2, 0)     # [plane, kept, kv head]
    rows = pool.gather(1, source[..., None].expand(-1, -1, -1, case["dim"]))
    pool[:, st["kept_rows"]] = rows
    return {"keep": keep, "weights": left, "tokens": st["kept"].int(), "pool": pool}


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_evict(st) if case["op"] == "evict" else _exact_attention(st)


def _exact_attention(st):
    """One sequence and one kv head after the other, in 64 bits."""
    case, pool = st["case"], st["pool"]
    prefix, group, page = case.get("prefix", 0), case["q_heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=pool.device)
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device=pool.device)
    weights = st["weights"].double() if "weights" in st else None
    first = 0
    for s, (n, m) in enumerate(zip(st["tokens"], st["queries"])):
        rows = st["rows"][s, :n]
        if prefix:
            rows = torch.cat([st["prefix_rows"], rows])
        at = torch.arange(prefix + n, device=pool.device)
        pos = at[prefix + n - m:]
        ahead = pos[:, None] - at
        see = ahead >= 0
        if case["window"]:
            see &= (ahead < case["window"]) | (at < case["sinks"])
        for h in range(case["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            q = st["q"][first:first + m, mine].double()
            k, v = pool[0][rows, h].double(), pool[1][rows, h].double()
            for j in range(group):
                z = (q[:, j] @ k.t()).div_(math.sqrt(case["dim"])).masked_fill_(~see, -math.inf)
                norm = torch.logsumexp(z, 1)
                z.sub_(norm[:, None]).exp_()
                lse[first:first + m, h * group + j] = norm
                out[first:first + m, h * group + j] = z @ v
                if weights is not None:
                    c = int(st["pages"].offsets[s]) * page
                    weights[0, h, c:c + n] += z.sum(0)[prefix:]
        first += m
    got = {"out": out, "lse": lse}
    if weights is not None:
        got["weights"] = weights
    return got


def _exact_evict(st):
    """Each sequence's and head's tokens ranked on the host."""
    case, page = st["case"], st["case"]["page"]
    pool, weights = st["pool"].double(), st["weights"].cpu().numpy()
    layers, kv_heads = weights.shape[:2]
    keep = np.full((layers, kv_heads, st["dst"].capacity), -1, np.int32)
    left = np.zeros(keep.shape, np.float64)
    for s, n in enumerate(st["tokens"]):
        m = min(n, case["budget"])
        old, new = int(st["pages"].offsets[s]) * page, int(st["dst"].offsets[s]) * page
        r = np.arange(m)
        to = st["dst"].table[int(st["dst"].offsets[s]) + r // page].astype(np.int64) * page + r % page
        for a in range(layers):
            for h in range(kv_heads):
                w = weights[a, h, old:old + n].astype(np.float64)
                key = w.copy()
                key[: case["sinks"]] = np.inf
                key[max(n - case["recent"], 0):] = np.inf
                best = np.sort(np.lexsort((np.arange(n), -key))[:m])
                keep[a, h, new:new + m], left[a, h, new:new + m] = best, w[best]
                table = st["pages"].table[int(st["pages"].offsets[s]) + best // page].astype(np.int64)
                src = torch.from_numpy(table * page + best % page).to(pool.device)
                dst = torch.from_numpy(to).to(pool.device)
                pool[2 * a:2 * a + 2, dst, h] = pool[2 * a:2 * a + 2, src, h]
    return {"keep": torch.from_numpy(keep), "weights": torch.from_numpy(left), "tokens": st["kept"].int(), "pool": pool}
