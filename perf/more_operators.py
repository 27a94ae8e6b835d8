"""More of what a server over a paged cache has its layers and its pages do: the rotary forms of other models, attention whose scores are capped, biased or
masked otherwise, and the bookkeeping of the pages.

The pool, its pages and ragged batches are those of the paged cache: position j of a sequence lies in slot j % page of page table[sequence][j // page], a call takes the
rows starts[s] .. starts[s + 1] of the activations, which are a sequence's newest tokens, and lengths[s] counts those among the cached positions.

  rotate   a layer's queries and keys rotated from a table of angles -- halves (i, i + dims/2) or neighbours (2i, 2i + 1), the first `dims` of a head, frequencies
           scaled for long contexts -- beside their norms, the gate split off the queries, keys and values quantised and written into their pages; read back as fp16
  attend   attention over the pages with scores cap * tanh(x / cap), less slope * |i - j|, and what a token sees given by a range of its own (documents that do not see one
           another, a prefix that sees itself in both directions) beside the window and the first `sinks`
  copy     pages from one pool to another, in all layers
  fork     sequences that go on from others': whole pages shared and counted, the last one copied; then room for a token of each
  compact  sequences end, the pages of the others are moved together, new ones get theirs

Two shapes: `dense` (32 query / 8 kv heads of 128) and `hybrid` (24 / 4 heads of 256, norms, gated output).  A cache is `q8_0` (an fp16 scale for 32 int8), `row` (int8, one
scale a row), `f16`, or `mixed` (q8_0 keys, fp16 values).
"""
import math
import random

import numpy as np
import torch

own = False

SHAPES = {"dense": dict(hq=32, hkv=8, d=128), "hybrid": dict(hq=24, hkv=4, d=256)}
THETA, EPSILON = 1.0e6, 1.0e-6


def listed():
    return [
        # the first tokens of a chat with a model that caps its scores: one sequence, one token, where latency is the time
        {"name": "attend-token-60", "kind": "attend", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 16, "sequences": 1, "shortest": 59, "longest": 59, "chunks": 0,
         "tokens": 1, "mix": 1, "window": 0, "sinks": 0, "lse": False, "cap": 30.0, "slopes": False, "sight": "causal"},
        # a decode step of a server whose model weighs positions by their distance, pages of 32
        {"name": "attend-tokens-48", "kind": "attend", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 32, "sequences": 48, "shortest": 300, "longest": 14000, "chunks": 0,
         "tokens": 1, "mix": 2, "window": 0, "sinks": 0, "lse": True, "cap": 50.0, "slopes": True, "sight": "causal"},
        # a piece of a long prompt, capped scores, a layer that sees everything
        {"name": "attend-chunk-cap", "kind": "attend", "shape": "dense", "cache": "f16", "act": "f16", "page": 64, "sequences": 1, "shortest": 6500, "longest": 6500, "chunks": 1,
         "tokens": 1333, "mix": 3, "window": 0, "sinks": 0, "lse": True, "cap": 50.0, "slopes": False, "sight": "causal"},
        # two prompts of many documents that see themselves and a common head of 40 positions
        {"name": "attend-documents", "kind": "attend", "shape": "hybrid", "cache": "q8_0", "act": "f16", "page": 64, "sequences": 2, "shortest": 0, "longest": 900, "chunks": 2,
         "tokens": 4100, "mix": 4, "window": 0, "sinks": 40, "lse": False, "cap": 0.0, "slopes": False, "sight": "documents"},
        # a decode step: neighbours, half of the head, frequencies scaled by their wavelength
        {"name": "rotate-tokens-40", "kind": "rotate", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 16, "sequences": 40, "shortest": 50, "longest": 120000, "chunks": 0,
         "tokens": 1, "mix": 5, "dims": 64, "layout": "neighbours", "scaling": "bands", "norms": False},
        # three prompts of the gated model, halves of the whole head, a ramp over the frequencies
        {"name": "rotate-prompts-3", "kind": "rotate", "shape": "hybrid", "cache": "row", "act": "f16", "page": 64, "sequences": 3, "shortest": 0, "longest": 700, "chunks": 3,
         "tokens": 2700, "mix": 6, "dims": 256, "layout": "halves", "scaling": "ramp", "norms": True},
        # a short prompt's pages into another pool
        {"name": "copy-pages-24", "kind": "copy", "shape": "dense", "cache": "q8_0", "page": 16, "layers": 4, "pages": 200, "count": 24, "mix": 7},
        # the pages of many sequences on their way out of a pool that has become too small
        {"name": "copy-pages-700", "kind": "copy", "shape": "hybrid", "cache": "f16", "page": 64, "layers": 6, "pages": 900, "count": 700, "mix": 8},
        # eight answers to one prompt
        {"name": "fork-answers-8", "kind": "fork", "shape": "dense", "cache": "q8_0", "page": 64, "layers": 12, "parents": 1, "children": 8, "shortest": 1000, "longest": 1000,
         "mix": 9},
        # a step of a search over 24 prompts
        {"name": "fork-search-144", "kind": "fork", "shape": "hybrid", "cache": "row", "page": 128, "layers": 8, "parents": 24, "children": 6, "shortest": 300, "longest": 3500,
         "mix": 10},
        # three of twelve sequences end
        {"name": "compact-12", "kind": "compact", "shape": "dense", "cache": "q8_0", "page": 16, "layers": 4, "stay": 6, "turn": 3, "shortest": 60, "longest": 700, "mix": 11},
        # a third of a full server turns over
        {"name": "compact-96", "kind": "compact", "shape": "dense", "cache": "mixed", "page": 32, "layers": 6, "stay": 48, "turn": 24, "shortest": 100, "longest": 3000, "mix": 12},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "rotate", "copy", "fork", "compact"])
    case = {"kind": kind, "shape": rng.choice(["dense", "hybrid"]), "cache": rng.choice(["q8_0", "q8_0", "row", "f16", "mixed"]), "page": rng.choice([16, 32, 64, 128]),
            "mix": rng.randrange(1 << 20)}
    s = SHAPES[case["shape"]]
    page_bytes = s["hkv"] * case["page"] * (_row_bytes(case, 0) + _row_bytes(case, 1))
    if kind == "copy":
        case["layers"] = rng.randint(1, 12)
        case["pages"] = max(8, min(_spread(rng, 16, 4000), int(1.2e9 / (page_bytes * case["layers"]))))
        case["count"] = _spread(rng, 1, case["pages"] * 3 // 4)
        return case
    if kind in ("fork", "compact"):
        case["layers"] = rng.randint(1, 12)
        case["longest"] = _spread(rng, 32, 4000)
        case["shortest"] = rng.randint(1, case["longest"])
        most = int(1.2e9 / (page_bytes * case["layers"]))      # pages of a pool
        each = -(-case["longest"] // case["page"]) + 1
        if kind == "fork":
            case["parents"] = max(1, min(_spread(rng, 1, 32), most // (4 * each)))
            case["children"] = max(1, min(_spread(rng, 1, 16), most // (4 * case["parents"])))
        else:
            case["turn"] = max(1, min(_spread(rng, 1, 32), most // (4 * each)))
            case["stay"] = max(1, min(_spread(rng, 1, 64), most // (4 * each)))
        return case
    case["act"] = rng.choice(["f16", "f16", "f32"])
    sequences = _spread(rng, 1, 64)
    decode = rng.random() < 0.5
    tokens = 1 if decode else _spread(rng, 2, 2048)
    longest = _spread(rng, 64, 14000 if kind == "attend" else 120000)
    chunks = 0 if decode else min(sequences, rng.choice([1, 1, 2, 4]))
    if kind == "attend":
        # the plain form's padded rows and scores stay within those of the largest listed cases
        while sequences > 1 and (sequences * (longest + tokens) * s["hkv"] * s["d"] > 5.0e8 or sequences * s["hq"] * tokens * (longest + tokens) > 5.0e8):
            sequences -= 1
        while s["hq"] * tokens * (longest + tokens) * s["d"] * 4 * sequences > 9.0e10 and longest > 64:
            longest = longest * 3 // 4
    else:
        while sequences > 1 and sequences * (longest + tokens) > 3000000:
            sequences -= 1
    case.update(sequences=sequences, shortest=rng.randint(0, longest), longest=longest, chunks=min(chunks, sequences), tokens=tokens)
    if kind == "rotate":
        case.update(dims=rng.choice([s["d"], s["d"], 64, 32, 96, 16]), layout=rng.choice(["halves", "neighbours"]), scaling=rng.choice(["none", "linear", "base", "bands", "ramp"]),
                    norms=rng.random() < 0.5)
        return case
    window = rng.choice([0, 0, _spread(rng, 16, 4096)])
    sight = rng.choice(["causal", "documents", "prefix"])
    cap = rng.choice([0.0, 15.0, 30.0, 50.0])
    slopes = rng.random() < 0.5 or (cap == 0.0 and sight == "causal")
    case.update(window=window, sinks=rng.choice([0, 4, 40]) if window or sight != "causal" else 0, cap=cap, slopes=slopes, sight=sight,
                lse=case["act"] == "f16" and (decode or case["cache"] == "f16"))
    return case


def _batch(case):
    """(new tokens, cached positions) of each sequence: the first `chunks` bring a piece of a prompt, the others a token."""
    rng = random.Random(case["mix"])
    got = []
    for i in range(case["sequences"]):
        n = 1
        if i < case["chunks"]:
            n = case["tokens"] if i == 0 else rng.randint((case["tokens"] + 1) // 2, case["tokens"])
        got.append((n, n + rng.randint(case["shortest"], case["longest"])))
    return got


def _row_bytes(case, side):
    """Bytes of one row of K (0) or V (1)."""
    d = SHAPES[case["shape"]]["d"]
    return {"q8_0": d + 2 * (d // 32), "row": d + 2, "f16": 2 * d, "mixed": 2 * d if side else d + 2 * (d // 32)}[case["cache"]]


def _sight(case):
    """Per sequence an array [new tokens][2]: the first position that a token sees and the one behind the last, its window aside."""
    rng, got = random.Random(case["mix"] + 1), []
    for n, length in _batch(case):
        i = np.arange(length - n, length)
        low, upto = np.zeros(n, np.int64), i + 1
        if case["sight"] == "documents":     # of very different lengths, the last one open
            starts = [0]
            while starts[-1] < length:
                starts.append(starts[-1] + _spread(rng, 16, max(64, length // 4)))
            low = np.array(starts)[np.searchsorted(starts, i, side="right") - 1]
        elif case["sight"] == "prefix":      # a part that is read in both directions, behind the cached positions or among them
            prefix = rng.randint(length // 4, length)
            upto = np.where(i < prefix, prefix, i + 1)
        got.append(np.stack([low, upto], 1))
    return got


def _seen(case):
    """Per sequence: pairs of a new token and a position it sees, and positions that any of them sees."""
    got = []
    for (n, length), sight in zip(_batch(case), _sight(case)):
        low, upto = sight[:, 0], sight[:, 1]
        if case["window"]:
            low = np.maximum(low, np.arange(length - n, length) + 1 - case["window"])
        first = np.minimum(case["sinks"], np.minimum(low, upto))
        edges = np.zeros(length + 2, np.int64)
        for a, b in ((low, np.maximum(upto, low)), (np.zeros(n, np.int64), first)):
            np.add.at(edges, a, 1)
            np.add.at(edges, b, -1)
        got.append((int((np.maximum(upto - low, 0) + first).sum()), int((np.cumsum(edges) > 0).sum())))
    return got


def _lengths(case, count, salt=0):
    rng = random.Random(case["mix"] + salt)
    return [rng.randint(case["shortest"], case["longest"]) for _ in range(count)]


def work(case):
    s = SHAPES[case["shape"]]
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    row = _row_bytes(case, 0) + _row_bytes(case, 1)
    if case["kind"] in ("copy", "fork", "compact"):
        page = hkv * case["page"] * row * case["layers"]
        if case["kind"] == "copy":
            return {"bytes": case["count"] * (2 * page + 8), "flops": 0}
        if case["kind"] == "fork":
            shared = [n // case["page"] for n in _lengths(case, case["parents"])]
            tails = sum(n % case["page"] > 0 for n in _lengths(case, case["parents"]))
            return {"bytes": tails * page + case["children"] * (tails * page + sum(8 * n + 24 for n in shared)), "flops": 0}
        moved = sum(-(-n // case["page"]) for n in _lengths(case, case["turn"]))
        held = sum(-(-n // case["page"]) for n in _lengths(case, case["stay"], 1))
        return {"bytes": moved * (2 * page + 24) + held * 8, "flops": 0}
    batch = _batch(case)
    act, total = (2 if case["act"] == "f16" else 4), sum(n for n, _ in batch)
    gate = 4 if case["shape"] == "hybrid" else 0
    if case["kind"] == "rotate":    # in, out, to the pages, and read back
        return {"bytes": total * (hq * d * (2 * act + gate + (act if gate else 0)) + hkv * (2 * d * act + row + 4 * d)), "flops": 0}
    seen = _seen(case)
    pairs, positions = sum(p for p, _ in seen), sum(u for _, u in seen)
    return {"bytes": positions * hkv * row + total * hq * (d * (act + gate + 2) + (4 if case["lse"] else 0)) + (8 * total if case["sight"] != "causal" else 0),
            "flops": 4.0 * d * hq * pairs}


def _quantise(x, block):
    """int8 and fp16 scales of rows of fp32: amax / 127 of each block, nearest even."""
    b = x.unflatten(-1, (-1, block))
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    return (b * (1 / scale)).round().clamp(-128, 127).to(torch.int8).flatten(-2), scale.squeeze(-1).half()


def _quant(case):
    d = SHAPES[case["shape"]]["d"]
    return {"q8_0": (32, 32), "row": (d, d), "f16": (0, 0), "mixed": (32, 0)}[case["cache"]]


def _mode(case):
    return (1 if _quant(case)[0] else 0) + (2 if _quant(case)[1] else 0)


def _tables(lists, width):
    t = np.full((len(lists), max(1, width)), -1, np.int32)
    for i, pages in enumerate(lists):
        t[i, :len(pages)] = pages
    return torch.from_numpy(t).cuda()


def prepare(case, seed):
    return _prepare_pages(case, seed) if case["kind"] in ("copy", "fork", "compact") else _prepare_batch(case, seed)


def _pools(case, seed, pages, pools=1):
    """Planes [pool][layer][k, k scales, v, v scales] of any bytes that are numbers."""
    s = SHAPES[case["shape"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    shape, got = (pages, s["hkv"], case["page"]), []
    for _ in range(pools):
        got.append([])
        for _ in range(case["layers"]):
            planes = []
            for block in _quant(case):
                if block:
                    planes += [torch.randint(-127, 128, (*shape, s["d"]), generator=g, dtype=torch.int8, device="cuda"),
                               torch.rand(*shape, s["d"] // block, generator=g, dtype=torch.float16, device="cuda")]
                else:
                    planes += [torch.randn(*shape, s["d"], generator=g, dtype=torch.float16, device="cuda"), None]
            got[-1].append(planes)
    return got


def _views(case, pool):
    from miinfer_b200 import paged

    return [paged.PagedView.of(*planes, _mode(case)) for planes in pool]


def _prepare_pages(case, seed):
    rng, page = np.random.default_rng(seed), case["page"]
    ints = lambda v: torch.tensor(list(v), dtype=torch.int32, device="cuda")
    held = lambda lengths: [-(-n // page) for n in lengths]
    if case["kind"] == "copy":
        pools = _pools(case, seed, case["pages"], 2)
        st = dict(case=case, pools=pools, source=ints(rng.permutation(case["pages"])[:case["count"]]), target=ints(rng.permutation(case["pages"])[:case["count"]]))
        if own:
            st["views"] = [_views(case, pool) for pool in pools]
        return st
    if case["kind"] == "fork":
        # the parents' pages scattered over the lower three quarters, where the others belong to sequences that only wait
        parents, children = case["parents"], case["parents"] * case["children"]
        lengths = _lengths(case, parents)
        need, more = held(lengths), 3 * children + 8
        pages = 2 * sum(need) + more
        order = rng.permutation(pages)
        at, lists = 0, []
        for n in need:
            lists.append(order[at:at + n])
            at += n
        refs = np.zeros(pages, np.int32)
        refs[order[:2 * sum(need)]] = 1
        lengths += [0] * children
        st = dict(parents=ints(np.repeat(np.arange(parents), case["children"])), children=ints(range(parents, parents + children)), add=ints([1] * children))
        width = max(need) + 2
    else:
        # what stays and what ends next scattered over the lower pages, the newest sequences behind them: as every turn leaves it
        turn, stay = _lengths(case, case["turn"]), _lengths(case, case["stay"], 1)
        low = sum(held(turn)) + sum(held(stay))
        pages = low + sum(held(turn)) + 5
        order, top = rng.permutation(low), low + rng.permutation(sum(held(turn)))
        lists, at, up = [], 0, 0
        for n in held(stay) + held(turn):
            lists.append(order[at:at + n])
            at += n
        for n in held(turn):
            lists.append(top[up:up + n])
            up += n
        refs = np.zeros(pages, np.int32)
        refs[:low + sum(held(turn))] = 1
        lengths = stay + turn + turn
        first = len(stay)
        st = dict(ending=[ints(range(first, first + len(turn))), ints(range(first + len(turn), first + 2 * len(turn)))], add=ints(turn), turn=0,
                  moved=torch.zeros(pages, dtype=torch.int32, device="cuda"))
        width = max(held(lengths)) + 1
    lists += [[]] * (len(lengths) - len(lists))
    st.update(case=case, page=page, refs=ints(refs), tables=_tables(lists, width), lengths=ints(lengths), planes=_pools(case, seed, pages)[0])
    if own:     # what a program keeps: the views of its layers, the book, its workspace
        from miinfer_b200 import paged

        st["views"] = _views(case, st["planes"])
        st["book"] = paged.PageBook(st["refs"], st["tables"], st["lengths"], page_size=page)
        st["workspace"] = paged.pages_workspace(st["book"])
    return st


def _prepare_batch(case, seed):
    s, batch = SHAPES[case["shape"]], _batch(case)
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], case["page"]
    hybrid = case["shape"] == "hybrid"
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    act = torch.float16 if case["act"] == "f16" else torch.float32
    count = len(batch)
    tokens, lengths = [n for n, _ in batch], [length for _, length in batch]
    total, most = sum(tokens), max(lengths)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    st = dict(case=case, hq=hq, hkv=hkv, d=d, page=page, scale=d ** -0.5, total=total, most=most, max_tokens=max(tokens), sum_lengths=sum(lengths),
              starts=ints([sum(tokens[:i]) for i in range(count + 1)]), lengths=ints(lengths), blocks=_quant(case))

    # the pool: every sequence's pages scattered over it, three pages nobody has.  What a rotation writes is its tokens' pages; the rest of a long sequence is not looked at and lies,
    # as a prefix that all have in common, in the same pages.
    first = [(length - n) // page if case["kind"] == "rotate" else 0 for n, length in batch]
    need = [-(-length // page) - f for f, length in zip(first, lengths)]
    pages = sum(need) + 3
    order, at, lists = np.random.default_rng(seed).permutation(pages), 0, []
    for f, n in zip(first, need):
        lists.append(np.concatenate([np.full(f, order[-1]), order[at:at + n]]))
        at += n
    st["table"] = _tables(lists, max(len(x) for x in lists))
    planes = []
    for block in st["blocks"]:
        x = normal(pages, hkv, page, d)
        planes += list(_quantise(x, block)) if block else [x.half(), None]
        del x
    st["k"], st["ks"], st["v"], st["vs"] = planes

    if case["kind"] == "rotate":
        # queries, keys and values are columns of one matrix, as the product that makes them leaves it; the gated shape's heads are a query and its gate
        wide = hq * d * (2 if hybrid else 1)
        rows = normal(total, wide + 2 * hkv * d).to(act)
        st.update(q=rows[:, :wide], key=rows[:, wide:wide + hkv * d], value=rows[:, wide + hkv * d:], q_out=torch.zeros(total, hq, d, dtype=act, device="cuda"),
                  gate=torch.zeros(total, hq, d, device="cuda") if hybrid else None, q_norm=1 + 0.1 * normal(d) if case["norms"] else None,
                  k_norm=1 + 0.1 * normal(d) if case["norms"] else None, **{side: torch.zeros(total, hkv, d, dtype=torch.float16, device="cuda") for side in ("key_out", "value_out")})
        st["frequencies"], st["magnitude"] = _frequencies(case)
    else:
        st.update(q=((3.0 if case["cap"] else 1.5) * normal(total, hq, d)).to(act), gate=normal(total, hq, d) if hybrid else None,
                  out=torch.zeros(total, hq, d, dtype=torch.float16, device="cuda"), lse=torch.zeros(total, hq, device="cuda") if case["lse"] else None,
                  slopes=torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda") / hq) if case["slopes"] else None,
                  ranges=torch.from_numpy(np.concatenate(_sight(case)).astype(np.int32)).cuda() if case["sight"] != "causal" else None)
    if own:     # what a program keeps from call to call: the view, the batch's description, the table of angles or the workspace
        from miinfer_b200 import paged

        st["view"] = paged.PagedView.of(st["k"], st["ks"], st["v"], st["vs"], _mode(case))
        st["batch"] = paged.PagedBatch(st["table"], st["starts"], st["lengths"], total_tokens=total, max_tokens=st["max_tokens"], max_length=most,
                                       total_length=st["sum_lengths"])
        if case["kind"] == "rotate":
            scaling = dict(none=paged.RotaryScaling.NONE, linear=paged.RotaryScaling.LINEAR, base=paged.RotaryScaling.BASE, bands=paged.RotaryScaling.BANDS,
                           ramp=paged.RotaryScaling.RAMP)[case["scaling"]]
            st["rotary"] = paged.RotaryTable(case["dims"], theta=THETA, layout=paged.RotaryLayout.HALVES if case["layout"] == "halves" else paged.RotaryLayout.NEIGHBOURS,
                                             scaling=scaling, **({} if case["scaling"] == "none" else SCALINGS[case["scaling"]]))
        else:
            st["scoring"] = paged.PagedScoring(cap=case["cap"], slopes=st["slopes"], ranges=st["ranges"])
            st["workspace"] = paged.paged_workspace(st["view"], st["batch"], hq, window=case["window"], sinks=case["sinks"], scoring=st["scoring"])
    return st


SCALINGS = {"linear": dict(factor=4.0), "base": dict(factor=4.0), "bands": dict(factor=8.0, original_length=8192, low=1.0, high=4.0),
            "ramp": dict(factor=4.0, original_length=32768, low=1.0, high=32.0)}


def _frequencies(case):
    """Radians a position of every pair, in 64 bits, and what sine and cosine are multiplied by.

    linear: all divided by the factor.  base: theta * factor^(dims / (dims - 2)).  bands: those that turn less than `low` times in the original length are divided by the
    factor, those that turn more than `high` times are not, those between in part.  ramp: in part from the pair that turns `high` times to the one that turns `low` times,
    straight over the pairs' numbers, and 0.1 log(factor) + 1 as the magnitude."""
    n, half = case["dims"], case["dims"] // 2
    scaling = SCALINGS.get(case["scaling"], {})
    base = THETA * (scaling["factor"] ** (n / (n - 2)) if case["scaling"] == "base" else 1.0)
    f = base ** (-np.arange(half) * 2.0 / n)
    if case["scaling"] == "linear":
        return f / scaling["factor"], 1.0
    if case["scaling"] == "bands":
        part = np.clip((scaling["original_length"] * f / (2 * np.pi) - scaling["low"]) / (scaling["high"] - scaling["low"]), 0, 1)
        return part * f + (1 - part) * f / scaling["factor"], 1.0
    if case["scaling"] == "ramp":
        pair = lambda turns: n * math.log(scaling["original_length"] / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        a, b = max(math.floor(pair(scaling["high"])), 0), min(math.ceil(pair(scaling["low"])), n - 1)
        part = np.clip((np.arange(half) - a) / (b - a if b > a else 0.001), 0, 1)
        return part * f / scaling["factor"] + (1 - part) * f, 0.1 * math.log(scaling["factor"]) + 1.0
    return f, 1.0


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------------


def _rows(st, plane, scales, block):
    """A side of every sequence's pages as fp32 [sequence][kv_head][position][d]; positions past a sequence's pages show some other page's."""
    j = torch.arange(st["most"], device="cuda")
    at = st["table"].long()[:, j // st["page"]].clamp(min=0)
    x = plane[at, :, j % st["page"]].float()
    if block:
        x = (x.unflatten(-1, (-1, block)) * scales[at, :, j % st["page"]].float().unsqueeze(-1)).flatten(-2)
    return x.transpose(1, 2)


def _padded(st, x):
    """Rows of the activations padded to [sequence][token][...], and which of them exist."""
    n = st["starts"][1:] - st["starts"][:-1]
    t = torch.arange(st["max_tokens"], device="cuda")
    return x[(st["starts"][:-1, None] + t).clamp(max=st["total"] - 1).long()], st["lengths"][:, None] - n[:, None] + t, t < n[:, None]


def _flat(st, x):
    """[sequence][kv_head][head of it][token][...] back to [row][query head][...]."""
    row = torch.arange(st["total"], device="cuda")
    s = torch.searchsorted(st["starts"][1:].contiguous(), row, right=True)
    return x[s, :, :, row - st["starts"][s]].flatten(1, 2)


def _plain_attend(st):
    case = st["case"]
    q, at, live = _padded(st, st["q"])
    q = q.float().unflatten(2, (st["hkv"], -1)).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.flatten(2, 3), _rows(st, st["k"], st["ks"], st["blocks"][0]).transpose(2, 3)).unflatten(2, q.shape[2:4]).mul_(st["scale"])
    if case["cap"]:
        e = x.mul_(2.0 / case["cap"]).exp_()          # tanh, its argument bounded by the scores'
        x = e.add_(1.0).reciprocal_().mul_(-2.0).add_(1.0).mul_(case["cap"])
    j = torch.arange(st["most"], device="cuda")
    if st["slopes"] is not None:
        away = (at[..., None] - j).abs().float()
        for h in range(st["hq"]):
            x[:, h // (st["hq"] // st["hkv"]), h % (st["hq"] // st["hkv"])] -= st["slopes"][h] * away
    low, upto = (torch.zeros_like(at), at + 1) if st["ranges"] is None else _padded(st, st["ranges"])[0].unbind(-1)
    if case["window"]:
        low = torch.maximum(low, at + 1 - case["window"])
    seen = (j < upto[..., None]) & ((j >= low[..., None]) | (j < case["sinks"])) & live[..., None]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _rows(st, st["v"], st["vs"], st["blocks"][1])).unflatten(2, p.shape[2:4])
    o = _flat(st, torch.where(total > 0, o / total, torch.zeros_like(o)))
    if st["gate"] is not None:
        o = o / (1 + torch.exp(-st["gate"]))
    out = {"out": o.half()}
    if st["lse"] is not None:
        out["lse"] = _flat(st, (m + torch.log(total)).squeeze(-1))
    return out


def _plain_rotate(st):
    case, d, n = st["case"], st["d"], st["case"]["dims"]
    row = torch.arange(st["total"], device="cuda")
    s = torch.searchsorted(st["starts"][1:].contiguous(), row, right=True)
    at = st["lengths"][s] - st["starts"][s + 1] + row
    page, slot = st["table"][s, (at // st["page"]).long()].long(), (at % st["page"]).long()
    angle = at.double()[:, None] * torch.from_numpy(st["frequencies"]).cuda()
    c, sn = ((f(angle) * st["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x, weight):
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * weight
        if case["layout"] == "halves":
            a, b = x[..., :n // 2], x[..., n // 2:n]
            return torch.cat((a * c - b * sn, a * sn + b * c, x[..., n:]), -1)
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        return torch.cat((torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2), x[..., n:]), -1)

    q = st["q"].float().unflatten(1, (st["hq"], -1))
    out = {"q": turned(q[..., :d], st["q_norm"]).to(st["q"].dtype)}
    if st["gate"] is not None:
        out["gate"] = q[..., d:].clone()
    for new, plane, scales, block, name in ((turned(st["key"].float().unflatten(1, (st["hkv"], d)), st["k_norm"]), "k", "ks", st["blocks"][0], "key"),
                                            (st["value"].float().unflatten(1, (st["hkv"], d)), "v", "vs", st["blocks"][1], "value")):
        if block:
            st[plane][page, :, slot], st[scales][page, :, slot] = _quantise(new, block)
            r = st[plane][page, :, slot].float().unflatten(-1, (-1, block)) * st[scales][page, :, slot].float().unsqueeze(-1)
            out[name] = r.flatten(-2).half()
        else:
            st[plane][page, :, slot] = new.half()
            out[name] = st[plane][page, :, slot]
    return out


def _plain_copy(st):
    for here, there in zip(*st["pools"]):
        for a, b in zip(here, there):
            if a is not None:
                b[st["target"].long()] = a[st["source"].long()]
    return _pool_outputs(st["pools"][1])


def _pool_outputs(pool):
    return {f"{name}{i}": plane for i, planes in enumerate(pool) for name, plane in zip(("k", "ks", "v", "vs"), planes) if plane is not None}


def _free(st, slots):
    slots = slots.long()
    held = (st["lengths"][slots] + st["page"] - 1) // st["page"]
    mine = torch.arange(st["tables"].shape[1], device="cuda") < held[:, None]
    st["refs"].scatter_add_(0, st["tables"][slots].long().clamp(min=0).flatten(), -mine.int().flatten())
    st["tables"][slots] = -1
    st["lengths"][slots] = 0


def _free_pages(st):
    return torch.argsort((st["refs"] > 0).int(), stable=True).int()      # the free ones first, the lowest ahead


def _grow(st, slots, add):
    slots = slots.long()
    held, want = ((n + st["page"] - 1) // st["page"] for n in (st["lengths"][slots], st["lengths"][slots] + add))
    column = torch.arange(st["tables"].shape[1], device="cuda")
    new = (column >= held[:, None]) & (column < want[:, None])
    rank = torch.cumsum(want - held, 0)[:, None] - want[:, None] + column
    pages = torch.where(new, _free_pages(st)[rank.clamp(0, st["refs"].numel() - 1).long()], 0)
    st["tables"][slots] = torch.where(new, pages, st["tables"][slots])
    st["refs"].scatter_add_(0, pages.long().flatten(), new.int().flatten())
    st["lengths"][slots] += add


def _plain_fork(st):
    _free(st, st["children"])
    parents, children = st["parents"].long(), st["children"].long()
    lengths = st["lengths"][parents]
    whole, tail = (lengths // st["page"])[:, None], (lengths % st["page"] > 0).int()
    fresh = _free_pages(st)[(torch.cumsum(tail, 0) - tail).long()]
    column = torch.arange(st["tables"].shape[1], device="cuda")
    rows = st["tables"][parents]
    old = rows.gather(1, whole.clamp(max=rows.shape[1] - 1).long())[:, 0]
    st["tables"][children] = torch.where(column < whole, rows, torch.where((column == whole) & (tail > 0)[:, None], fresh[:, None], -1)).int()
    st["refs"].scatter_add_(0, rows.long().clamp(min=0).flatten(), (column < whole).int().flatten())
    st["refs"].scatter_add_(0, fresh.long(), tail)
    source, target = torch.where(tail > 0, old, rows[:, 0]).long(), torch.where(tail > 0, fresh, rows[:, 0]).long()     # without a last page the first one, over itself
    for planes in st["planes"]:
        for plane in planes:
            if plane is not None:
                plane[target] = plane[source]
    st["lengths"][children] = lengths
    _grow(st, st["children"], st["add"])
    return {"refs": st["refs"], "tables": st["tables"], "lengths": st["lengths"]} | _pool_outputs(st["planes"])


def _plain_compact(st):
    ending = st["ending"][st["turn"] % 2]
    st["turn"] += 1
    _free(st, ending)
    live = st["refs"] > 0
    page = torch.arange(live.numel(), device="cuda")
    count = live.sum()
    moves = live & (page >= count)
    holes, movers = _free_pages(st).long(), torch.argsort((~moves).int(), stable=True)      # the k-th hole gets the k-th page behind the others
    valid = page < moves.sum()
    stays = torch.where(live, page, -1)
    moved = stays.scatter(0, movers, torch.where(valid, holes, stays[movers]))
    source = torch.cat((page, page[:1])).scatter(0, torch.where(valid, holes, live.numel()), movers)[:-1]
    st["refs"].copy_(torch.where(page < count, st["refs"][source], 0))
    st["tables"].copy_(torch.where(st["tables"] >= 0, moved[st["tables"].long().clamp(min=0)], -1))
    for planes in st["planes"]:
        for plane in planes:
            if plane is not None:
                plane.copy_(plane[source])
    st["moved"].copy_(moved)
    _grow(st, ending, st["add"])
    return {"refs": st["refs"], "tables": st["tables"], "lengths": st["lengths"], "moved": st["moved"]} | _pool_outputs(st["planes"])


# ---- the framework's calls ----------------------------------------------------------------------------------------------------------------


def _own(st):
    from miinfer_b200 import paged

    case = st["case"]
    if case["kind"] == "attend":
        paged.launch_paged_attention(st["view"], st["batch"], st["q"], st["out"], query_heads=st["hq"], scale=st["scale"], window=case["window"], sinks=case["sinks"],
                                     gate=st["gate"], lse=st["lse"], workspace=st["workspace"], scoring=st["scoring"])
        return {"out": st["out"]} | ({} if st["lse"] is None else {"lse": st["lse"]})
    if case["kind"] == "rotate":
        paged.launch_paged_rotary(st["view"], st["batch"], st["rotary"], st["key"], st["value"], st["q"], st["q_out"], query_heads=st["hq"], gate=st["gate"],
                                  q_norm_weight=st["q_norm"], k_norm_weight=st["k_norm"], epsilon=EPSILON)
        paged.launch_paged_load(st["view"], st["batch"], st["key_out"], st["value_out"])
        return {"q": st["q_out"], "key": st["key_out"], "value": st["value_out"]} | ({} if st["gate"] is None else {"gate": st["gate"]})
    if case["kind"] == "copy":
        paged.launch_pages_copy(st["views"][0], st["views"][1], st["source"], st["target"])
        return _pool_outputs(st["pools"][1])
    if case["kind"] == "fork":
        paged.launch_pages_free(st["book"], st["children"])
        paged.launch_pages_fork(st["book"], st["views"], st["parents"], st["children"], workspace=st["workspace"])
        paged.launch_pages_grow(st["book"], st["children"], st["add"], workspace=st["workspace"])
        return {"refs": st["refs"], "tables": st["tables"], "lengths": st["lengths"]} | _pool_outputs(st["planes"])
    ending = st["ending"][st["turn"] % 2]
    st["turn"] += 1
    paged.launch_pages_free(st["book"], ending)
    paged.launch_pages_compact(st["book"], st["views"], st["moved"], workspace=st["workspace"])
    paged.launch_pages_grow(st["book"], ending, st["add"], workspace=st["workspace"])
    return {"refs": st["refs"], "tables": st["tables"], "lengths": st["lengths"], "moved": st["moved"]} | _pool_outputs(st["planes"])


def run(st):
    if own:
        return _own(st)
    return {"attend": _plain_attend, "rotate": _plain_rotate, "copy": _plain_copy, "fork": _plain_fork, "compact": _plain_compact}[st["case"]["kind"]](st)


# ---- from the definitions, in 64 bits, one sequence and kv head after the other -----------------------------------------------------------------


def _cached(st, s, h, plane, scales, block):
    """Rows of one sequence's kv head."""
    length = int(st["lengths"][s])
    pages = st["table"][s, :-(-length // st["page"])].long()
    x = st[plane][pages, h].double().flatten(0, 1)[:length]
    return x if not block else (x.unflatten(1, (-1, block)) * st[scales][pages, h].double().flatten(0, 1)[:length, :, None]).flatten(1)


def _exact_attend(case, st):
    group = st["hq"] // st["hkv"]
    out = torch.zeros(st["total"], st["hq"], st["d"], dtype=torch.float64, device="cuda")
    lse = torch.full((st["total"], st["hq"]), -math.inf, dtype=torch.float64, device="cuda")
    sight = _sight(case)
    for s in range(case["sequences"]):
        begin, end, length = int(st["starts"][s]), int(st["starts"][s + 1]), int(st["lengths"][s])
        at = torch.arange(length - (end - begin), length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        first, behind = (torch.from_numpy(sight[s][:, i]).cuda()[:, None] for i in (0, 1))
        hidden = j < first
        if case["window"]:
            hidden = hidden | (at - j >= case["window"])
        hidden = (hidden & (j >= case["sinks"])) | (j >= behind)
        for h in range(st["hkv"]):
            heads = slice(h * group, (h + 1) * group)
            k, v = _cached(st, s, h, "k", "ks", st["blocks"][0]), _cached(st, s, h, "v", "vs", st["blocks"][1])
            x = st["q"][begin:end, heads].double().transpose(0, 1) @ k.T * st["scale"]
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - st["slopes"][heads].double()[:, None, None] * (at - j).abs().double()
            x = x.masked_fill(hidden, -math.inf)
            lse[begin:end, heads] = torch.logsumexp(x, -1).T
            out[begin:end, heads] = torch.nan_to_num(torch.softmax(x, -1)).matmul(v).transpose(0, 1)
    if st["gate"] is not None:
        out *= torch.sigmoid(st["gate"].double())
    return {"out": out} | ({"lse": lse} if case["lse"] else {})


def _exact_rotate(case, st):
    d, n = st["d"], case["dims"]
    frequencies, magnitude = _frequencies(case)
    positions = np.concatenate([np.arange(length - k, length) for k, length in _batch(case)])
    turn = torch.polar(torch.tensor(float(magnitude), dtype=torch.float64, device="cuda"), torch.from_numpy(positions[:, None] * frequencies).cuda())[:, None]

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPSILON).sqrt() * weight.double()
        pairs = x[..., :n].reshape(*x.shape[:2], 2, n // 2).transpose(2, 3) if case["layout"] == "halves" else x[..., :n].reshape(*x.shape[:2], n // 2, 2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(2, 3) if case["layout"] == "halves" else z
        return torch.cat((z.reshape(*x.shape[:2], n), x[..., n:]), -1)

    q = st["q"].reshape(st["total"], st["hq"], -1)
    got = {"q": turned(q[..., :d], st["q_norm"])}
    if st["gate"] is not None:
        got["gate"] = q[..., d:].double()
    for name, block in (("key", st["blocks"][0]), ("value", st["blocks"][1])):
        x = st[name].reshape(st["total"], st["hkv"], d)
        x = turned(x, st["k_norm"]) if name == "key" else x.double()
        if block:
            b = x.reshape(st["total"], st["hkv"], d // block, block)
            step = b.abs().amax(-1, keepdim=True) / 127
            step = torch.where(step > 0, step, 1.0)
            x = (torch.round(b / step).clamp(-128, 127) * step.half().double()).reshape(st["total"], st["hkv"], d)
        got[name] = x
    return got


def _move(planes, source, target, into=None):
    for here, there in zip(planes, planes if into is None else into):
        for a, b in zip(here, there):
            if a is not None:
                b[int(target)].copy_(a[int(source)])


def _exact_pages(case, st):
    """The book, entry by entry, and copies of the pages one by one."""
    refs, tables, lengths = (st[name].cpu().numpy().copy() for name in ("refs", "tables", "lengths"))
    page = case["page"]
    held = lambda slot: -(-int(lengths[slot]) // page)
    lowest = lambda: int(np.flatnonzero(refs == 0)[0])

    def grow(slots, add):
        for slot, n in zip(slots, add):
            first = held(slot)
            lengths[slot] += n
            for c in range(first, held(slot)):
                tables[slot, c] = lowest()
                refs[tables[slot, c]] = 1

    got = {}
    if case["kind"] == "fork":
        children = st["children"].tolist()
        for parent, child in zip(st["parents"].tolist(), children):
            n, lengths[child] = int(lengths[parent]), lengths[parent]
            tables[child, :n // page] = tables[parent, :n // page]
            refs[tables[parent, :n // page]] += 1
            if n % page:
                tables[child, n // page] = lowest()
                refs[tables[child, n // page]] = 1
                _move(st["planes"], tables[parent, n // page], tables[child, n // page])
        grow(children, st["add"].tolist())
    else:
        ending = st["ending"][0].tolist()
        for slot in ending:
            refs[tables[slot, :held(slot)]] -= 1
            tables[slot], lengths[slot] = -1, 0
        live = np.flatnonzero(refs > 0)
        moved = np.where(refs > 0, np.arange(len(refs)), -1)
        movers = live[live >= len(live)]
        moved[movers] = np.flatnonzero(refs == 0)[:len(movers)]
        for source in movers:
            _move(st["planes"], source, moved[source])
        after = np.zeros_like(refs)
        after[moved[live]] = refs[live]
        refs[:] = after
        tables[tables >= 0] = moved[tables[tables >= 0]]
        got["moved"] = moved
        grow(ending, st["add"].tolist())
    got.update(refs=refs, tables=tables, lengths=lengths)
    return {name: torch.from_numpy(x.astype(np.int32)) for name, x in got.items()} | _pool_outputs(st["planes"])


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "copy":
        for source, target in zip(st["source"].tolist(), st["target"].tolist()):
            _move(st["pools"][0], source, target, st["pools"][1])
        return _pool_outputs(st["pools"][1])
    return (_exact_attend if case["kind"] == "attend" else _exact_rotate if case["kind"] == "rotate" else _exact_pages)(case, st)
