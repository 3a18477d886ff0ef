"""Performance cases of the operators around the sampler in a round of speculative decoding on a paged cache.

A round puts the drafted rows' keys and values into the lanes' pages, lets the
rows attend to them, constrains the logits before the tokens are decided, and
cuts the cache back to what was accepted.  A case is a dict of plain values:

=========  ====================================================================
kind       entry point of ``voidinfer_amd``
=========  ====================================================================
logits     ``process_logits``: penalties over token histories (and each row's
           drafted prefix), biases, grammar masks
append     ``norm_rotate_append``: per-head norms and the rotation of queries
           and keys, keys and values written to the lanes' pages
attention  ``prefix_attention``: rows over the paged cache, the prefix that the
           lanes of a group share read once for all of them
fork       ``pages_fork``, ``pages_extend``: lanes forked for parallel samples,
           their shared last page copied as they grow
round      ``pages_extend``, ``keep_rows``, ``pages_truncate``: the page work of
           one speculative round
compact    ``pages_truncate``, ``pages_compact``, ``pages_extend``: half of the
           lanes retire, the pool is compacted, new lanes are admitted
=========  ====================================================================

A cache is one tensor [layers, 2 (keys, values), pages, kv_heads, page_size,
head_dim]; ``tables`` int32 [lanes, pages per lane] (-1: no page), ``lengths``
int32 [lanes] and ``refs`` int32 [pages] (how many lanes hold a page) describe
who holds what.  Page ids are a random order, as after hours of serving.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_DEV = "cuda:0"
_PARAMS = np.dtype([   # the sampler's row parameters
    ("temperature", "<f4"), ("top_p", "<f4"), ("min_p", "<f4"), ("repetition_penalty", "<f4"),
    ("presence_penalty", "<f4"), ("frequency_penalty", "<f4"), ("top_k", "<i4"), ("lane", "<u4"), ("seed", "<u8"),
    ("position", "<i4"), ("reserved", "<u4")])
_PENALTIES = ("repetition_penalty", "presence_penalty", "frequency_penalty")


def listed():
    return [
        # One interactive lane under a JSON grammar, with the most biases that a request may bring.
        dict(name="logits-1-f32", kind="logits", lanes=1, drafts=0, vocab=151936, dtype="f32", history=256, biases=300,
             masked=1.0),
        # A ragged vocabulary, no grammar: penalties and a few biases, every second row off a 16-byte boundary.
        dict(name="logits-64-f16-odd", kind="logits", lanes=64, drafts=0, vocab=65537, dtype="f16", history=1000,
             biases=20, masked=0.0),
        # A verified block: 8 lanes x (16 drafted rows and the bonus row), each row with the drafted tokens before
        # it in its history, half of the rows under a grammar.
        dict(name="logits-8x17-bf16", kind="logits", lanes=8, drafts=16, vocab=248320, dtype="bf16", history=4096,
             biases=50, masked=0.5),
        # One decode step of a small batch: 8 rows.
        dict(name="append-8-bf16", kind="append", lanes=8, rows=1, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, page=16, dtype="bf16", context=4096),
        # A verified block with wide heads, a quarter of each rotated.
        dict(name="append-8x17-f16", kind="append", lanes=8, rows=17, heads=24, kv_heads=4, dim=256, rotary=64,
             interleaved=True, page=32, dtype="f16", context=1000),
        # A prompt of 16,384 tokens (4 lanes of 4,096).
        dict(name="append-4x4096-bf16", kind="append", lanes=4, rows=4096, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, page=16, dtype="bf16", context=0),
        # Four samples of one short prompt, one token each: the smallest attention, latency only.
        dict(name="attention-4x1-f16", kind="attention", groups=1, lanes=4, rows=1, heads=16, kv_heads=4, dim=64,
             page=16, dtype="f16", prefix=512, own=100, tree=False),
        # A verified block: 8 lanes x up to 17 rows of a verification tree over a shared system prompt.
        dict(name="attention-8x17-bf16", kind="attention", groups=1, lanes=8, rows=17, heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16", prefix=4096, own=1500, tree=True),
        # A large decode batch over one long document: 64 lanes, 32,768 shared tokens.
        dict(name="attention-64x1-bf16", kind="attention", groups=1, lanes=64, rows=1, heads=64, kv_heads=8, dim=128,
             page=16, dtype="bf16", prefix=32768, own=2048, tree=False),
        # Parallel samples: 4 prompts forked into 4 lanes each, the shared last pages copied.
        dict(name="fork-4x4", kind="fork", parents=4, children=4, layers=16, kv_heads=8, dim=128, page=16,
             dtype="bf16", pages=1024, length=1000),
        # The pages of a round: 64 lanes grow by 17 rows, keep an accepted path, give the rest back.
        dict(name="round-64x17", kind="round", lanes=64, rows=17, layers=16, kv_heads=8, dim=128, page=16,
             dtype="bf16", pages=2048, length=300),
        # Half of 16 lanes retire, the pool's live pages move together, eight lanes are admitted.
        dict(name="compact-16", kind="compact", lanes=16, layers=16, kv_heads=8, dim=128, page=16, dtype="bf16",
             pages=2048, length=1700),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["logits", "logits", "append", "append", "attention", "attention", "attention", "fork", "round",
                       "compact"])
    if kind == "logits":
        vocab = _spread(rng, 32000, 248320)
        vocab = vocab | 1 if rng.random() < 0.3 else vocab // 64 * 64
        drafts = rng.choice([0, 0, 3, 7, 16])
        return dict(kind=kind, lanes=_spread(rng, 1, 128 // (drafts + 1)), drafts=drafts, vocab=vocab,
                    dtype=rng.choice(["bf16", "f16", "f32"]) if vocab < 130000 else rng.choice(["bf16", "f16"]),
                    history=_spread(rng, 16, 8192), biases=rng.choice([0, _spread(rng, 1, 300)]),
                    masked=rng.choice([0.0, 0.5, 1.0]))
    dim, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "f16"])
    layout = dict(kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if kind == "append":
        rows = rng.choice([1, 1, _spread(rng, 2, 17), _spread(rng, 100, 4096)])
        return dict(kind=kind, lanes=_spread(rng, 1, 4 if rows > 17 else 128), rows=rows,
                    heads=kv_heads * rng.choice([1, 2, 3, 4]), rotary=rng.choice([dim, dim // 4]),
                    interleaved=rng.random() < 0.3, context=_spread(rng, 1, 8192),
                    **{**layout, "dim": min(dim, 128) if rows > 17 else dim})
    if kind == "attention":
        groups = rng.choice([1, 1, 2, 4])
        rows = rng.choice([1, 1, rng.randrange(2, 18)])
        most, longest = (64, 32768) if rows == 1 else (8, 8192)
        return dict(kind=kind, groups=groups, lanes=groups * _spread(rng, 1, most // groups), rows=rows,
                    heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8] if kv_heads < 8 else [1, 2, 4]),
                    prefix=_spread(rng, 64, longest // groups) // page * page, own=_spread(rng, 1, 2048),
                    tree=rows > 1 and rng.random() < 0.5, **layout)
    layout["layers"] = rng.choice([1, 4, 16]) if page * kv_heads * dim <= 16384 else 1
    if kind == "fork":
        parents, children = _spread(rng, 1, 8), _spread(rng, 1, 8)
        length = _spread(rng, 1, 1000)
        return dict(kind=kind, parents=parents, children=children, length=length,
                    pages=parents * (-(-length // page) + 1) + parents * children * 2 + _spread(rng, 1, 500), **layout)
    if kind == "round":
        lanes, rows, length = _spread(rng, 1, 64), rng.choice([2, 5, 9, 17]), _spread(rng, 1, 400)
        return dict(kind=kind, lanes=lanes, rows=rows, length=length,
                    pages=lanes * (-(-(length + rows) // page) + 1) + _spread(rng, 1, 500), **layout)
    lanes, length = 2 * _spread(rng, 1, 8), _spread(rng, 16, 1700)
    return dict(kind=kind, lanes=lanes, length=length, pages=lanes * -(-length // page) + _spread(rng, 1, 300),
                **layout)


# ---- sizes that follow from a case ------------------------------------------------------------------------------------
def _row_counts(c):
    """Rows of each lane: ragged where a lane verifies a tree."""
    return [c["rows"] - (3 * i) % (1 + c["rows"] // 2) if c.get("tree") else c["rows"] for i in range(c["lanes"])]


def _own_lengths(c):
    """Tokens of each lane beyond the shared prefix, before its rows."""
    return [c["own"] - (37 * i) % (1 + c["own"] // 2) for i in range(c["lanes"])]


def _lengths(c, lanes):
    return [max(1, c["length"] - (53 * i) % (1 + c["length"] // 4)) for i in range(lanes)]


def _kept(c):
    """Rows that each lane of a round keeps: the anchor, some of the chain, sometimes a sibling row behind it."""
    return [1 + (5 * i + 3) % c["rows"] for i in range(c["lanes"])]


def _pages(c, tokens):
    return -(-tokens // c["page"])


def _page_bytes(c):
    return 2 * c["layers"] * c["kv_heads"] * c["page"] * c["dim"] * _SIZE[c["dtype"]]


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    host = np.random.default_rng(seed)
    kind = "pages" if case["kind"] in ("fork", "round", "compact") else case["kind"]
    state = {"logits": _prepare_logits, "append": _prepare_append, "attention": _prepare_attention,
             "pages": _prepare_pages}[kind](case, g, host)
    state["case"] = case
    return state


def _i32(values):
    return torch.tensor(np.asarray(values, dtype=np.int32), device=_DEV)


def _i64(values):
    return torch.tensor(np.asarray(values, dtype=np.int64), device=_DEV)


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=_DEV) * std).to(dtype)


def _prepare_logits(c, g, host):
    lanes, per, vocab, dt = c["lanes"], c["drafts"] + 1, c["vocab"], _DT[c["dtype"]]
    rows = lanes * per
    logits = _normal(g, rows, vocab, std=2.0)
    logits += 8.0 / (1.0 + torch.rand(rows, vocab, generator=g, device=_DEV) * vocab) ** 0.5   # a few likely tokens
    p = np.zeros(lanes, dtype=_PARAMS)
    p["temperature"], p["top_p"], p["lane"] = 0.7, 0.95, np.arange(lanes)
    p["repetition_penalty"] = host.choice([1.0, 1.05, 1.1, 1.3], lanes)
    p["presence_penalty"] = host.choice([0.0, 0.2, 0.5], lanes)
    p["frequency_penalty"] = host.choice([0.1, 0.3], lanes)
    lens = np.maximum(1, c["history"] - (29 * np.arange(lanes)) % (1 + c["history"] // 2))
    hist = np.minimum(host.zipf(1.3, int(lens.sum())) * 7 % vocab, vocab - 1)   # text repeats few tokens often
    s = dict(logits=logits.to(dt), params=torch.from_numpy(p.view(np.uint8).reshape(-1).copy()).to(_DEV),
             penalties=torch.tensor(np.stack([p[n] for n in _PENALTIES]), device=_DEV),
             histories=_i32(hist), offsets=_i64(np.concatenate([[0], np.cumsum(lens)])), max_history=int(lens.max()),
             lanes=_i32(np.repeat(np.arange(lanes), per)), out=torch.empty(rows, vocab, dtype=dt, device=_DEV),
             extra=None, extra_offsets=None, bias_ids=None, bias_values=None, bias_offsets=None, masks=None,
             mask_index=None)
    if c["drafts"]:
        drafted = host.integers(0, vocab, (lanes, c["drafts"]))
        s["extra"] = _i32(np.concatenate([drafted[l, :j] for l in range(lanes) for j in range(per)]))
        s["extra_offsets"] = _i64(np.concatenate([[0], np.cumsum(np.tile(np.arange(per), lanes))]))
    if c["biases"]:
        n = c["biases"] - np.arange(lanes) % (1 + c["biases"] // 2)
        s["bias_ids"] = _i32(np.concatenate([host.choice(vocab, k, replace=False) for k in n]))
        s["bias_values"] = torch.tensor(host.uniform(-5, 5, int(n.sum())).astype(np.float32), device=_DEV)
        s["bias_offsets"] = _i64(np.concatenate([[0], np.cumsum(n)]))
    if c["masked"]:
        # each masked row stands at a place of its grammar: free text, where most tokens may follow, or syntax
        count = max(1, int(rows * c["masked"]))
        words = -(-vocab // 32)
        share = torch.tensor(host.choice([0.97, 0.3, 0.003], count).astype(np.float32), device=_DEV)
        bits = torch.rand(count, words, 32, generator=g, device=_DEV) < share[:, None, None]
        word = (bits.to(torch.int64) << torch.arange(32, device=_DEV)).sum(2)
        s["masks"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)
        index = np.full(rows, -1)
        index[host.choice(rows, count, replace=False)] = host.permutation(count)
        s["mask_index"] = _i32(index)
    return s


def _tables(host, pages, counts, width):
    """Tables of lanes that hold counts[l] pages each, ids in a random order."""
    order, tables, at = host.permutation(pages), np.full((len(counts), width), -1), 0
    for i, n in enumerate(counts):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables


def _prepare_append(c, g, host):
    lanes, n, dt, d = c["lanes"], c["rows"], _DT[c["dtype"]], c["dim"]
    rows, hk = lanes * n, c["kv_heads"]
    ctx = np.array([max(0, c["context"] - (37 * i) % (1 + c["context"] // 2)) for i in range(lanes)])
    held = [_pages(c, int(x) + n) for x in ctx]
    pages = sum(held) + 5
    width = max(held)
    qkv = _normal(g, rows, (c["heads"] + 2 * hk) * d, std=1.5, dtype=dt)   # one projection's output
    q, k, v = qkv.split([c["heads"] * d, hk * d, hk * d], dim=1)
    limit = int(ctx.max()) + n
    angle = torch.arange(limit, device=_DEV, dtype=torch.float64)[:, None] \
        * 10000.0 ** (-torch.arange(0, c["rotary"], 2, device=_DEV, dtype=torch.float64) / c["rotary"])
    return dict(q=q.view(rows, c["heads"], d), k=k.view(rows, hk, d), v=v.view(rows, hk, d),
                pool=_normal(g, 2, pages, hk, c["page"], d, dtype=dt), tables=_i32(_tables(host, pages, held, width)),
                offsets=_i32(np.arange(lanes + 1) * n), context=_i32(ctx), cos=angle.cos().float(),
                sin=angle.sin().float(), q_weight=1 + _normal(g, d, std=0.2, dtype=dt),
                k_weight=1 + _normal(g, d, std=0.2, dtype=dt), eps=1e-6,
                out=torch.empty(rows, c["heads"], d, dtype=dt, device=_DEV))


def _prepare_attention(c, g, host):
    lanes, dt, ps = c["lanes"], _DT[c["dtype"]], c["page"]
    counts, more = _row_counts(c), _own_lengths(c)
    shared, each = c["prefix"] // ps, lanes // c["groups"]
    held = [_pages(c, m + n) for m, n in zip(more, counts)]
    pages = c["groups"] * shared + sum(held) + 3
    order, at = host.permutation(pages), c["groups"] * shared
    tables = np.full((lanes, shared + max(held)), -1)
    for i in range(lanes):
        p = i // each * shared
        tables[i, :shared] = order[p:p + shared]
        tables[i, shared:shared + held[i]] = order[at:at + held[i]]
        at += held[i]
    rows = sum(counts)
    s = dict(q=_normal(g, rows, c["heads"], c["dim"], std=1.5, dtype=dt),
             pool=_normal(g, 2, pages, c["kv_heads"], ps, c["dim"], dtype=dt), tables=_i32(tables),
             offsets=_i32(np.concatenate([[0], np.cumsum(counts)])), context=_i32(c["prefix"] + np.array(more)),
             group_offsets=_i32(np.arange(c["groups"] + 1) * each), prefix_lens=_i32([c["prefix"]] * c["groups"]),
             most=dict(max_rows=max(counts), max_own=max(more) + max(counts), max_prefix=c["prefix"],
                       max_group_rows=max(sum(counts[i:i + each]) for i in range(0, lanes, each))),
             tree=None, out=torch.empty(rows, c["heads"], c["dim"], dtype=dt, device=_DEV),
             lse=torch.empty(rows, c["heads"], device=_DEV))
    if c["tree"]:
        # the anchor and a chain, then siblings of chain tokens: a row sees its ancestors and itself
        seen = []
        for n in counts:
            chain = max(1, n - n // 3)
            seen += [(1 << (i + 1)) - 1 if i < chain else (1 << int(host.integers(1, chain + 1))) - 1 | 1 << i
                     for i in range(n)]
        s["tree"] = _i64(seen)
    return s


def _prepare_pages(c, g, host):
    kind, dt, ps = c["kind"], _DT[c["dtype"]], c["page"]
    s = dict(pool=torch.randn(c["layers"], 2, c["pages"], c["kv_heads"], ps, c["dim"], generator=g, device=_DEV,
                              dtype=dt), status=torch.zeros(3, dtype=torch.int32, device=_DEV))
    lanes = c["parents"] if kind == "fork" else c["lanes"]
    lens = _lengths(c, lanes)
    grown = lens if kind != "round" else [n + c["rows"] for n in lens]
    total = lanes * (1 + c["children"]) if kind == "fork" else lanes
    tables = np.full((total, max(_pages(c, n) for n in grown) + 1), -1)
    tables[:lanes] = _tables(host, c["pages"], [_pages(c, n) for n in lens], tables.shape[1])
    refs = np.zeros(c["pages"], dtype=np.int32)
    refs[tables[tables >= 0]] = 1
    s |= dict(tables=_i32(tables), refs=_i32(refs), lengths=_i32(lens + [0] * (total - lanes)))
    if kind == "fork":
        s |= dict(parents=_i32(np.repeat(np.arange(lanes), c["children"])), children=_i32(np.arange(lanes, total)),
                  grown=_i32(np.repeat(np.array(lens) + 1, c["children"])))
    elif kind == "round":
        kept = _kept(c)
        paths = np.zeros((lanes, c["rows"]))
        for i, n in enumerate(kept):   # a chain, its last row a sibling further behind where there is one
            paths[i, :n] = np.arange(n)
            paths[i, n - 1] = host.integers(n - 1, c["rows"])
        s |= dict(lanes=_i32(np.arange(lanes)), context=_i32(lens), grown=_i32(grown), paths=_i32(paths),
                  kept=_i32(kept), cut=_i32(np.array(lens) + kept))
    else:
        halves = [np.arange(lanes)[k::2] for k in (0, 1)]
        s |= dict(halves=[_i32(h) for h in halves], again=[_i32(np.array(lens)[h]) for h in halves], turn=0,
                  none=[_i32(np.zeros(len(h))) for h in halves])
    return s


# ---- the calls --------------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        import voidinfer_amd as vi
        return _OWN[kind](vi, state)
    return _PLAIN[kind](state)


def _own_logits(vi, s):
    return vi.process_logits(s["logits"], s["params"], lanes=s["lanes"], histories=s["histories"],
                             offsets=s["offsets"], max_history=s["max_history"], extra=s["extra"],
                             extra_offsets=s["extra_offsets"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                             bias_offsets=s["bias_offsets"], masks=s["masks"], mask_index=s["mask_index"],
                             out=s["out"])


def _own_append(vi, s):
    vi.norm_rotate_append(s["q"], s["k"], s["v"], s["pool"][0], s["pool"][1], s["tables"], s["offsets"], s["context"],
                          s["cos"], s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"],
                          interleaved=s["case"]["interleaved"], out=s["out"])
    return s["out"], s["pool"]


def _own_attention(vi, s):
    vi.prefix_attention(s["q"], s["pool"][0], s["pool"][1], s["tables"], s["offsets"], s["context"],
                        group_offsets=s["group_offsets"], prefix_lens=s["prefix_lens"], tree=s["tree"], out=s["out"],
                        lse=s["lse"], **s["most"])
    return s["out"], s["lse"]


def _own_fork(vi, s):
    vi.pages_fork(s["refs"], s["tables"], s["lengths"], s["parents"], s["children"], s["case"]["page"], s["status"])
    vi.pages_extend(s["refs"], s["tables"], s["lengths"], s["children"], s["grown"], s["pool"], s["status"])
    return s["refs"], s["tables"], s["lengths"], s["status"], s["pool"]


def _own_round(vi, s):
    vi.pages_extend(s["refs"], s["tables"], s["lengths"], s["lanes"], s["grown"], s["pool"], s["status"])
    vi.keep_rows(s["pool"], s["tables"], s["lanes"], s["context"], s["paths"], s["kept"])
    vi.pages_truncate(s["refs"], s["tables"], s["lengths"], s["lanes"], s["cut"], s["case"]["page"])
    return s["refs"], s["tables"], s["lengths"], s["status"], s["pool"]


def _own_compact(vi, s):
    k = s["turn"]
    s["turn"] ^= 1   # the other half retires in the next pass
    vi.pages_truncate(s["refs"], s["tables"], s["lengths"], s["halves"][k], s["none"][k], s["case"]["page"])
    vi.pages_compact(s["refs"], s["tables"], s["pool"], s["status"])
    vi.pages_extend(s["refs"], s["tables"], s["lengths"], s["halves"][k], s["again"][k], s["pool"], s["status"])
    return s["refs"], s["tables"], s["lengths"], s["status"], s["pool"]


_OWN = {"logits": _own_logits, "append": _own_append, "attention": _own_attention, "fork": _own_fork,
        "round": _own_round, "compact": _own_compact}


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _expand(offsets, values):
    """(segment of each entry, entries) of lists laid end to end."""
    n = offsets[1:] - offsets[:-1]
    return torch.repeat_interleave(torch.arange(n.numel(), device=_DEV), n, output_size=values.numel())


def _plain_logits(s):
    x, lane = s["logits"].float(), s["lanes"].long()
    rows, vocab = x.shape
    lanes = s["offsets"].numel() - 1
    count = torch.zeros(lanes, vocab, device=_DEV)
    ones = torch.ones(1, device=_DEV)
    hist = s["histories"].long()
    count.index_put_((_expand(s["offsets"], hist), hist), ones, accumulate=True)
    count = count[lane]
    if s["extra"] is not None:
        extra = s["extra"].long()
        count.index_put_((_expand(s["extra_offsets"], extra), extra), ones, accumulate=True)
    rep, presence, frequency = s["penalties"][:, lane, None]
    x = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep) - frequency * count - presence, x)
    if s["bias_ids"] is not None:
        bias, ids = torch.zeros(lanes, vocab, device=_DEV), s["bias_ids"].long()
        bias[_expand(s["bias_offsets"], ids), ids] = s["bias_values"]
        x = x + bias[lane]
    if s["masks"] is not None:
        bits = (s["masks"][s["mask_index"].clamp_min(0).long(), :, None] >> torch.arange(32, device=_DEV)) & 1
        allowed = bits.reshape(rows, -1)[:, :vocab].bool() | (s["mask_index"] < 0)[:, None]
        x = torch.where(allowed, x, -math.inf)
    return x.to(s["logits"].dtype)


def _places(s):
    """(lane, page, place in the page) of every row's own token, and its position."""
    n = (s["offsets"][1:] - s["offsets"][:-1]).long()
    lane = torch.repeat_interleave(torch.arange(n.numel(), device=_DEV), n, output_size=s["q"].shape[0])
    at = s["context"][lane].long() + torch.arange(lane.numel(), device=_DEV) - s["offsets"][lane].long()
    ps = s["case"]["page"]
    return s["tables"][lane, at // ps].long(), at % ps, at


def _rotated(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_append(s):
    page, place, at = _places(s)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = s["q"].float(), s["k"].float()
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + s["eps"]) * s["q_weight"].float()
    k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + s["eps"]) * s["k_weight"].float()
    turned = s["case"]["interleaved"]
    out = _rotated(q, cos, sin, turned).to(s["q"].dtype)
    s["pool"][0][page, :, place] = _rotated(k, cos, sin, turned).to(s["k"].dtype)
    s["pool"][1][page, :, place] = s["v"]
    return out, s["pool"]


def _plain_attention(s):
    c, q = s["case"], s["q"].float()
    rows, heads, d = q.shape
    groups, lanes, hk, ps, most = c["groups"], c["lanes"], c["kv_heads"], c["page"], s["most"]["max_rows"]
    g, each, scale = heads // hk, lanes // groups, 1.0 / math.sqrt(d)
    off = s["offsets"].long()
    n = off[1:] - off[:-1]
    lane = torch.repeat_interleave(torch.arange(lanes, device=_DEV), n, output_size=rows)
    slot = torch.arange(rows, device=_DEV) - off[lane]
    padded = torch.zeros(lanes, most, heads, d, device=_DEV)
    padded[lane, slot] = q
    padded = padded.view(lanes, most, hk, g, d).permute(0, 2, 1, 3, 4)                       # lanes, hk, most, g, d
    # the prefix, once for a group's rows
    shared = c["prefix"] // ps
    ids = s["tables"].view(groups, each, -1)[:, 0, :shared].long()
    kp, vp = (s["pool"][i][ids].permute(0, 2, 1, 3, 4).reshape(groups, hk, shared * ps, d).float() for i in (0, 1))
    qp = padded.reshape(groups, each, hk, most * g, d).transpose(1, 2).reshape(groups, hk, each * most * g, d)
    sp = qp @ kp.transpose(2, 3) * scale
    # each lane's own tokens
    wide = s["most"]["max_own"]
    at = c["prefix"] + torch.arange(wide, device=_DEV)
    place = (at % ps).expand(lanes, -1)
    ids = s["tables"][:, (at // ps).clamp_max(s["tables"].shape[1] - 1)].clamp_min(0).long()
    ko, vo = (s["pool"][i][ids, :, place].permute(0, 2, 1, 3).float() for i in (0, 1))       # lanes, hk, wide, d
    so = (padded.reshape(lanes, hk, most * g, d) @ ko.transpose(2, 3) * scale).view(lanes, hk, most, g, wide)
    later = at[None] - s["context"][:, None].long()                                          # index among the rows
    if s["tree"] is None:
        seen = later[:, None] <= torch.arange(most, device=_DEV)[None, :, None]
    else:
        bits = torch.zeros(lanes, most, dtype=torch.int64, device=_DEV)
        bits[lane, slot] = s["tree"]
        seen = (later < 0)[:, None] | ((bits[:, :, None] >> later.clamp(0, 63)[:, None]) & 1).bool() \
            & (later < n[:, None])[:, None]
    so = torch.where(seen[:, None, :, None], so, -math.inf)
    sp = sp.view(groups, hk, each, most * g, -1).transpose(1, 2).reshape(lanes, hk, most, g, -1)
    m = torch.maximum(sp.amax(-1), so.amax(-1))[..., None]
    sp, so = torch.exp(sp - m), torch.exp(so - m)
    total = sp.sum(-1) + so.sum(-1)
    back = sp.view(groups, each, hk, most * g, -1).transpose(1, 2).reshape(groups, hk, each * most * g, -1) @ vp
    back = back.view(groups, hk, each, most * g, d).transpose(1, 2).reshape(lanes, hk, most, g, d)
    out = (back + (so.view(lanes, hk, most * g, wide) @ vo).view(lanes, hk, most, g, d)) / total[..., None]
    lse = m[..., 0] + torch.log(total)
    out, lse = out.permute(0, 2, 1, 3, 4)[lane, slot], lse.permute(0, 2, 1, 3)[lane, slot]
    return out.reshape(rows, heads, d).to(s["q"].dtype), lse.reshape(rows, heads)


def _add_refs(refs, pages, value):
    pages = pages[pages >= 0].long()
    refs.index_add_(0, pages, torch.full((pages.numel(),), value, dtype=torch.int32, device=_DEV))


def _plain_truncate(s, lanes, lengths):
    lanes = lanes.long()
    t = s["tables"][lanes]
    beyond = torch.arange(t.shape[1], device=_DEV)[None] >= (lengths[:, None] + s["case"]["page"] - 1) // s["case"]["page"]
    _add_refs(s["refs"], torch.where(beyond, t, -1), -1)
    s["tables"][lanes] = torch.where(beyond, -1, t)
    s["lengths"][lanes] = lengths


def _plain_extend(s, lanes, lengths):
    refs, tables, ps, lanes = s["refs"], s["tables"], s["case"]["page"], lanes.long()
    now = s["lengths"][lanes]
    held, wanted = (now + ps - 1) // ps, (lengths + ps - 1) // ps
    last = torch.where((now % ps > 0) & (lengths > now), tables[lanes, (held - 1).clamp_min(0).long()], -1)
    earlier = ((last[:, None] == last[None]) & (last >= 0)).int().tril(-1).sum(1)   # lanes before, on the same page
    copied = (last >= 0) & (refs[last.clamp_min(0).long()] - earlier > 1)
    need = (wanted - held).clamp_min(0) + copied
    base, total = torch.cumsum(need, 0) - need, int(need.sum())
    free = torch.nonzero(refs == 0)[:total, 0].int()
    if free.numel() < total:
        raise RuntimeError("the pool has too few free pages")
    who = torch.repeat_interleave(torch.arange(lanes.numel(), device=_DEV), need, output_size=total)
    slot = held[who] - copied[who].int() + torch.arange(total, device=_DEV) - base[who]
    tables[lanes[who], slot] = free
    refs[free.long()] = 1
    source, target = last[copied], free[base[copied].long()]
    _add_refs(refs, source, -1)
    s["pool"][:, :, target.long()] = s["pool"][:, :, source.long()]
    s["lengths"][lanes] = lengths
    s["status"][:] = torch.tensor([0, total, source.numel()], dtype=torch.int32, device=_DEV)


def _plain_fork(s):
    parents, children, t = s["parents"].long(), s["children"].long(), s["tables"]
    _add_refs(s["refs"], t[children], -1)
    t[children] = t[parents]
    _add_refs(s["refs"], t[children], 1)
    s["lengths"][children] = s["lengths"][parents]
    _plain_extend(s, s["children"], s["grown"])
    return s["refs"], t, s["lengths"], s["status"], s["pool"]


def _plain_round(s):
    ps = s["case"]["page"]
    _plain_extend(s, s["lanes"], s["grown"])
    width = s["paths"].shape[1]
    lane, i = torch.nonzero(torch.arange(width, device=_DEV)[None] < s["kept"][:, None], as_tuple=True)
    source, target = (s["context"][lane].long() + x for x in (s["paths"][lane, i].long(), i))
    moved = s["pool"][:, :, s["tables"][lane, source // ps].long(), :, source % ps]
    s["pool"][:, :, s["tables"][lane, target // ps].long(), :, target % ps] = moved
    _plain_truncate(s, s["lanes"], s["cut"])
    return s["refs"], s["tables"], s["lengths"], s["status"], s["pool"]


def _plain_compact(s):
    k, refs, tables = s["turn"], s["refs"], s["tables"]
    s["turn"] ^= 1
    _plain_truncate(s, s["halves"][k], s["none"][k])
    live = refs > 0
    count = int(live.sum())
    holes, movers = torch.nonzero(~live[:count])[:, 0], torch.nonzero(live[count:])[:, 0] + count
    to = torch.arange(refs.numel(), dtype=torch.int32, device=_DEV)
    to[movers] = holes.int()
    s["tables"][:] = torch.where(tables >= 0, to[tables.clamp_min(0).long()], -1)
    refs[holes] = refs[movers]
    refs[movers] = 0
    s["pool"][:, :, holes] = s["pool"][:, :, movers]
    _plain_extend(s, s["halves"][k], s["again"][k])
    return refs, tables, s["lengths"], s["status"], s["pool"]


_PLAIN = {"logits": _plain_logits, "append": _plain_append, "attention": _plain_attention, "fork": _plain_fork,
          "round": _plain_round, "compact": _plain_compact}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(c):
    kind = c["kind"]
    if kind == "logits":
        rows = c["lanes"] * (c["drafts"] + 1)
        masked = max(1, int(rows * c["masked"])) if c["masked"] else 0
        size = 2 * rows * c["vocab"] * _SIZE[c["dtype"]] + masked * c["vocab"] // 8
        return {"bytes": size + 4 * c["lanes"] * c["history"], "flops": 3 * rows * c["vocab"]}
    if kind == "append":
        rows, heads, hk, d = c["lanes"] * c["rows"], c["heads"], c["kv_heads"], c["dim"]
        return {"bytes": 2 * rows * (heads + 2 * hk) * d * _SIZE[c["dtype"]] + 4 * rows * c["rotary"],
                "flops": 8 * rows * (heads + hk) * d}
    if kind == "attention":
        counts, more = _row_counts(c), _own_lengths(c)
        tokens = c["groups"] * c["prefix"] + sum(more) + sum(counts)
        pairs = sum(n * (c["prefix"] + m + n) for n, m in zip(counts, more))
        line = c["dim"] * _SIZE[c["dtype"]]
        return {"bytes": 2 * tokens * c["kv_heads"] * line + sum(counts) * c["heads"] * (2 * line + 4),
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    if kind == "fork":
        lens = _lengths(c, c["parents"])
        copied = sum(c["children"] for n in lens if n % c["page"])
        held = sum(_pages(c, n) for n in lens)
        return {"bytes": 2 * copied * _page_bytes(c) + 4 * c["pages"] + 12 * c["children"] * held, "flops": 0}
    if kind == "round":
        moved = sum(1 for n in _kept(c) if n < c["rows"])   # the sibling rows that stand behind their place
        tables = 8 * sum(_pages(c, n + c["rows"]) - _pages(c, n) for n in _lengths(c, c["lanes"]))
        return {"bytes": 2 * moved * _page_bytes(c) // c["page"] + 4 * c["pages"] + tables, "flops": 0}
    held = [_pages(c, n) for n in _lengths(c, c["lanes"])]
    moved = sum(held) // 2   # the half that was admitted last lies behind the half that retires
    return {"bytes": 2 * moved * _page_bytes(c) + 8 * sum(held) + 8 * c["pages"], "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "round", "compact"):
        return None   # whole numbers and copies
    s = prepare(case, seed)
    return {"logits": _exact_logits, "append": _exact_append, "attention": _exact_attention}[kind](case, s)


def _exact_logits(c, s):
    rep, presence, frequency = s["penalties"].double().tolist()
    out = s["logits"].double()
    offs, hist = s["offsets"].tolist(), s["histories"].long()
    for r, l in enumerate(s["lanes"].tolist()):
        tokens = hist[offs[l]:offs[l + 1]]
        if s["extra"] is not None:
            a, b = s["extra_offsets"][r:r + 2].tolist()
            tokens = torch.cat([tokens, s["extra"][a:b].long()])
        ids, n = torch.unique(tokens, return_counts=True)
        x = out[r, ids]
        out[r, ids] = torch.where(x > 0, x / rep[l], x * rep[l]) - frequency[l] * n - presence[l]
        if s["bias_ids"] is not None:
            a, b = s["bias_offsets"][l:l + 2].tolist()
            out[r, s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        if s["masks"] is not None and (i := int(s["mask_index"][r])) >= 0:
            word = s["masks"][i].long()
            bits = torch.stack([word >> b & 1 for b in range(32)], 1).flatten()[:c["vocab"]]
            out[r, bits == 0] = -math.inf
    return out


def _exact_append(c, s):
    rows, half, ps = c["lanes"] * c["rows"], c["rotary"] // 2, c["page"]
    lane = torch.arange(rows, device=_DEV) // c["rows"]
    at = s["context"].long()[lane] + torch.arange(rows, device=_DEV) % c["rows"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]

    def turned(x, weight):
        x = x.double()
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["dim"] + s["eps"]) * weight.double()
        first = slice(0, 2 * half, 2) if c["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if c["interleaved"] else slice(half, 2 * half)
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out, pool = turned(s["q"], s["q_weight"]), s["pool"].double()
    page = s["tables"].long()[lane, at // ps]
    pool[0].transpose(1, 2)[page, at % ps] = turned(s["k"], s["k_weight"])
    pool[1].transpose(1, 2)[page, at % ps] = s["v"].double()
    return out, pool


def _exact_attention(c, s):
    off, ctx, ps = s["offsets"].tolist(), s["context"].tolist(), c["page"]
    g, out, lse = c["heads"] // c["kv_heads"], [], []
    for l in range(c["lanes"]):
        n, length = off[l + 1] - off[l], ctx[l] + off[l + 1] - off[l]
        ids = s["tables"][l, :-(-length // ps)].long()
        k, v = (x[ids].transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :length].double() for x in s["pool"])
        q = s["q"][off[l]:off[l + 1]].double().view(n, c["kv_heads"], g, -1).permute(1, 2, 0, 3).reshape(
            c["kv_heads"], g * n, -1)
        score = torch.bmm(q, k.transpose(1, 2).contiguous()).div_(math.sqrt(c["dim"])).view(-1, g, n, length)
        for i in range(n):
            if s["tree"] is None:
                score[:, :, i, ctx[l] + i + 1:] = -math.inf
            else:
                seen = int(s["tree"][off[l] + i])
                hidden = [ctx[l] + j for j in range(n) if not seen >> j & 1]
                score[:, :, i, hidden] = -math.inf
        total = torch.logsumexp(score, -1)
        p = torch.exp(score - total[..., None]).view(c["kv_heads"], g * n, length)
        out.append(torch.bmm(p, v).view(-1, g, n, c["dim"]).permute(2, 0, 1, 3).reshape(n, c["heads"], -1))
        lse.append(total.permute(2, 0, 1).reshape(n, c["heads"]))
    return torch.cat(out), torch.cat(lse)
