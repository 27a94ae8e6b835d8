"""The operators over a paged cache: what a server that keeps many sequences in one pool of pages has them do, layer by layer.

A pool's planes are [page][kv_head][slot][...]; position j of a sequence lies in slot j % page of page table[sequence][j // page].  A call
takes a ragged batch: sequence s has the rows starts[s] .. starts[s + 1] of the activations, its newest tokens, and lengths[s] cached
positions, those tokens among them.

  store   K norm, RoPE, quantisation and the write of the new tokens' rows into their pages; read back as fp16
  attend  attention of every new token over its sequence's pages: causal, with a sliding window of `window` positions beside the first
          `sinks`, if one is set; times sigmoid(gate) for the hybrid shape; with `lse`, each row's log of the sum of exponentials as well
  weigh   the weight that each cached position gets from the (last `observe`) new tokens, summed over tokens and heads of the kv head,
          added to what it had
  evict   of each sequence and kv head keep `keep` positions -- the first `sinks`, the last `recent`, and those with the largest weights of
          the others -- in order, in the pages of another table

Two shapes: `dense` (32 query / 8 kv heads of 128, NeoX RoPE) and `hybrid` (24 / 4 heads of 256, sectioned RoPE, K norm, gated output).  A cache is
`q8_0` (an fp16 scale for 32 int8), `row` (int8, one scale a row), `f16`, or `mixed` (q8_0 keys, fp16 values).
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
        # the first tokens of a chat: one sequence, one token, where latency is the time
        {"name": "attend-token-100", "kind": "attend", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 16, "sequences": 1, "shortest": 99,
         "longest": 99, "chunks": 0, "tokens": 1, "mix": 1, "window": 0, "sinks": 0, "lse": False},
        # a decode step of a busy server
        {"name": "attend-tokens-64", "kind": "attend", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 64, "sequences": 64, "shortest": 512,
         "longest": 16383, "chunks": 0, "tokens": 1, "mix": 42, "window": 0, "sinks": 0, "lse": True},
        # decode steps of long sequences under a sliding window with sinks
        {"name": "attend-tokens-window", "kind": "attend", "shape": "hybrid", "cache": "row", "act": "f16", "page": 32, "sequences": 24,
         "shortest": 2000, "longest": 30000, "chunks": 0, "tokens": 1, "mix": 7, "window": 4096, "sinks": 4, "lse": False},
        # a piece of a long prompt
        {"name": "attend-chunk-512-8192", "kind": "attend", "shape": "hybrid", "cache": "q8_0", "act": "f16", "page": 64, "sequences": 1,
         "shortest": 8192, "longest": 8192, "chunks": 1, "tokens": 512, "mix": 3, "window": 0, "sinks": 0, "lse": False},
        # pieces of two prompts beside decoding sequences, small pages, odd lengths
        {"name": "attend-mixed-16", "kind": "attend", "shape": "dense", "cache": "q8_0", "act": "f32", "page": 16, "sequences": 16, "shortest": 100,
         "longest": 5000, "chunks": 2, "tokens": 333, "mix": 11, "window": 0, "sinks": 0, "lse": False},
        # the same in a model whose layers see a window, cache left in fp16
        {"name": "attend-chunk-window", "kind": "attend", "shape": "dense", "cache": "f16", "act": "f16", "page": 64, "sequences": 1, "shortest": 6001,
         "longest": 6001, "chunks": 1, "tokens": 2048, "mix": 5, "window": 1024, "sinks": 4, "lse": True},
        # one token of each of 48 sequences
        {"name": "store-tokens-48", "kind": "store", "shape": "hybrid", "cache": "row", "act": "f32", "page": 16, "sequences": 48, "shortest": 50,
         "longest": 4000, "chunks": 0, "tokens": 1, "mix": 13, "shift": 500},
        # four fresh prompts
        {"name": "store-prompts-4", "kind": "store", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 64, "sequences": 4, "shortest": 0,
         "longest": 0, "chunks": 4, "tokens": 2500, "mix": 17, "shift": 0},
        # keeping account of the weights in a decode step
        {"name": "weigh-tokens-32", "kind": "weigh", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 64, "sequences": 32, "shortest": 512,
         "longest": 12000, "chunks": 0, "tokens": 1, "mix": 19, "window": 0, "sinks": 0, "observe": 0},
        # what the last 64 tokens of a prompt looked at
        {"name": "weigh-chunk-12000", "kind": "weigh", "shape": "hybrid", "cache": "q8_0", "act": "f16", "page": 32, "sequences": 2, "shortest": 7000,
         "longest": 12000, "chunks": 2, "tokens": 300, "mix": 23, "window": 0, "sinks": 0, "observe": 64},
        # eight sequences back to 2048 positions
        {"name": "evict-8", "kind": "evict", "shape": "dense", "cache": "q8_0", "act": "f16", "page": 64, "sequences": 8, "shortest": 3000,
         "longest": 9000, "chunks": 0, "tokens": 1, "mix": 29, "keep": 2048, "sinks": 4, "recent": 256},
        # one very long document
        {"name": "evict-70000", "kind": "evict", "shape": "hybrid", "cache": "f16", "act": "f16", "page": 16, "sequences": 1, "shortest": 70000,
         "longest": 70000, "chunks": 0, "tokens": 1, "mix": 31, "keep": 4000, "sinks": 4, "recent": 512},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "store", "weigh", "evict"])
    case = {"kind": kind, "shape": rng.choice(["dense", "hybrid"]), "cache": rng.choice(["q8_0", "q8_0", "row", "f16", "mixed"]),
            "act": rng.choice(["f16", "f16", "f32"]) if kind in ("attend", "store") else "f16", "page": rng.choice([16, 32, 64, 128]), "mix": rng.randrange(1 << 20)}
    s = SHAPES[case["shape"]]
    sequences = _spread(rng, 1, 64)
    decode = kind == "evict" or rng.random() < 0.5
    tokens = 1 if decode else _spread(rng, 2, 2048)
    longest = _spread(rng, 64, 16000 if kind != "evict" else 60000)
    chunks = 0 if decode else min(sequences, rng.choice([1, 1, 2, 4]))
    # the plain form's padded rows, scores and rounded planes stay within those of the largest listed cases
    while sequences > 1 and (sequences * (longest + tokens) * s["hkv"] * s["d"] > 5.0e8 or sequences * s["hq"] * tokens * (longest + tokens) > 5.0e8):
        sequences -= 1
    while s["hq"] * tokens * (longest + tokens) * s["d"] * 4 * sequences > 9.0e10 and longest > 64:
        longest = longest * 3 // 4
    case.update(sequences=sequences, shortest=rng.randint(0 if kind != "evict" else 16, longest), longest=longest, chunks=min(chunks, sequences), tokens=tokens)
    if kind == "store":
        case.update(shift=rng.choice([0, rng.randint(1, 30000)]))
    elif kind == "evict":
        keep = _spread(rng, 16, 8192)
        case.update(keep=keep, sinks=rng.randint(0, keep // 8), recent=rng.randint(0, keep // 2))
    else:
        window = rng.choice([0, 0, _spread(rng, 16, 4096)])
        case.update(window=window, sinks=rng.choice([0, 4, 17]) if window else 0)
        if kind == "attend":
            case.update(lse=decode or case["cache"] == "f16")
        else:
            case.update(observe=rng.choice([0, 16, 64]))
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


def _seen(case, n, length, observe=0):
    """Pairs of a new token and a position it sees, and positions that any of them sees."""
    first = n - min(n, observe) if observe else 0
    window, sinks = case["window"], case["sinks"]
    pairs = 0
    for t in range(first, n):
        upto = length - n + t + 1
        pairs += upto if window == 0 or upto <= window else min(upto, window + min(sinks, upto - window))
    lowest = length - n + first + 1 - window if window else 0
    return pairs, length if lowest <= 0 else min(length, length - lowest + min(sinks, lowest))


def work(case):
    s, batch = SHAPES[case["shape"]], _batch(case)
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    act, total = (2 if case["act"] == "f16" else 4), sum(n for n, _ in batch)
    row = _row_bytes(case, 0) + _row_bytes(case, 1)
    if case["kind"] == "store":     # in, to the pages, and read back
        return {"bytes": total * hkv * (2 * d * act + row + 4 * d), "flops": 0}
    if case["kind"] == "evict":
        kept = [min(length, case["keep"]) for _, length in batch]
        return {"bytes": sum(hkv * (4 * length + k * (2 * row + 8)) for k, (_, length) in zip(kept, batch)), "flops": 0}
    seen = [_seen(case, n, length, case.get("observe", 0)) for n, length in batch]
    pairs, positions = sum(p for p, _ in seen), sum(u for _, u in seen)
    if case["kind"] == "attend":
        gate = 4 if case["shape"] == "hybrid" else 0
        return {"bytes": positions * hkv * row + total * hq * (d * (act + gate + 2) + (4 if case["lse"] else 0)), "flops": 4.0 * d * hq * pairs}
    observed = sum(min(n, case["observe"]) if case["observe"] else n for n, _ in batch)
    return {"bytes": positions * hkv * (_row_bytes(case, 0) + 8) + observed * hq * (d * 2 + 4), "flops": 2.0 * d * hq * pairs}


def _quantise(x, block):
    """int8 and fp16 scales of rows of fp32: amax / 127 of each block, nearest even."""
    b = x.unflatten(-1, (-1, block))
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    return (b * (1 / scale)).round().clamp(-128, 127).to(torch.int8).flatten(-2), scale.squeeze(-1).half()


def prepare(case, seed):
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
    starts = [sum(tokens[:i]) for i in range(count + 1)]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    st = dict(case=case, hq=hq, hkv=hkv, d=d, page=page, scale=d ** -0.5, total=total, most=most, max_tokens=max(tokens), sum_lengths=sum(lengths),
              starts=ints(starts), lengths=ints(lengths))

    # the pool: every sequence's pages scattered over it, three pages nobody has; for evict the kept rows' pages behind them
    need = [-(-length // page) for length in lengths]
    kept = [-(-min(length, case["keep"]) // page) for length in lengths] if case["kind"] == "evict" else []
    pages = sum(need) + sum(kept) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    def table(sizes, first):
        columns = torch.arange(max(1, max(sizes)), device="cuda")
        begin = torch.tensor([first + sum(sizes[:i]) for i in range(count)], device="cuda")
        inside = columns < torch.tensor(sizes, device="cuda")[:, None]
        return torch.where(inside, order[(begin[:, None] + columns).clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    st["table"] = table(need, 0)
    quant = {"q8_0": (32, 32), "row": (d, d), "f16": (0, 0), "mixed": (32, 0)}[case["cache"]]
    st["blocks"], st["pages"] = quant, pages
    planes = []
    for block in quant:
        x = normal(pages, hkv, page, d)
        planes += list(_quantise(x, block)) if block else [x.half(), None]
        del x
    st["k"], st["ks"], st["v"], st["vs"] = planes

    if case["kind"] == "store":
        st.update(key=normal(total, hkv * d).to(act), value=normal(total, hkv * d).to(act), weight=1.0 + 0.1 * normal(d) if hybrid else None,
                  positions=None, key_out=torch.zeros(total, hkv, d, dtype=torch.float16, device="cuda"), value_out=torch.zeros(total, hkv, d, dtype=torch.float16, device="cuda"))
        if case["shift"]:   # an earlier eviction left the slots behind the positions
            st["positions"] = ints([length - n + t + case["shift"] + i for i, (n, length) in enumerate(batch) for t in range(n)])
    elif case["kind"] == "evict":
        st["target"] = table(kept, sum(need))
        w = torch.exp(1.5 * normal(count, hkv, most))
        st.update(weights=torch.where(w < 0.25, (w * 64).round() / 64, w), kept=torch.full((count, hkv, case["keep"]), -1, dtype=torch.int32, device="cuda"),
                  new_weights=torch.zeros(count, hkv, case["keep"], device="cuda"), new_lengths=torch.zeros(count, dtype=torch.int32, device="cuda"))
    else:
        st["q"] = (1.5 * normal(total, hq, d)).to(act)
        if case["kind"] == "attend":
            st.update(gate=normal(total, hq, d) if hybrid else None, out=torch.zeros(total, hq, d, dtype=torch.float16, device="cuda"),
                      lse=torch.zeros(total, hq, device="cuda") if case["lse"] else None)
        else:
            looks = hq // hkv * min(max(tokens), case["observe"] or max(tokens))     # of the order that one call adds
            st["weights"] = 2.0 * looks / most * torch.rand(count, hkv, most, generator=g, device="cuda")
            st["lse"] = _statistics(st).float()     # the attention call before has left them
    if own:     # what a program keeps from call to call: the view, the batch's description, the workspace
        from miinfer_b200 import paged

        mode = (1 if quant[0] else 0) + (2 if quant[1] else 0)
        st["view"] = paged.PagedView.of(st["k"], st["ks"], st["v"], st["vs"], mode)
        st["batch"] = paged.PagedBatch(st["table"], st["starts"], st["lengths"], total_tokens=total, max_tokens=st["max_tokens"], max_length=most,
                                       total_length=st["sum_lengths"])
        st["workspace"] = paged.paged_workspace(st["view"], st["batch"], hq, window=case.get("window", 0), sinks=case.get("sinks", 0)) if case["kind"] == "attend" else None
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------------


def _rows(st, plane, scales, block):
    """A side of every sequence's pages as fp32 [sequence][kv_head][position][d]; positions past a sequence's pages show some other page's."""
    j = torch.arange(st["most"], device="cuda")
    at = st["table"].long()[:, j // st["page"]].clamp(min=0)
    x = plane[at, :, j % st["page"]].float()
    if block:
        x = (x.unflatten(-1, (-1, block)) * scales[at, :, j % st["page"]].float().unsqueeze(-1)).flatten(-2)
    return x.transpose(1, 2)


def _queries(st):
    """The query rows padded to [sequence][kv_head][head of it][token][d], the tokens' positions, and which of them exist."""
    n = st["starts"][1:] - st["starts"][:-1]
    t = torch.arange(st["max_tokens"], device="cuda")
    at = (st["starts"][:-1, None] + t).clamp(max=st["total"] - 1).long()
    q = st["q"][at].float().unflatten(2, (st["hkv"], -1)).permute(0, 2, 3, 1, 4)
    return q, st["lengths"][:, None] - n[:, None] + t, t < n[:, None]


def _flat(st, x):
    """[sequence][kv_head][head of it][token][...] back to [row][query head][...]."""
    row = torch.arange(st["total"], device="cuda")
    s = torch.searchsorted(st["starts"][1:].contiguous(), row, right=True)
    return x[s, :, :, row - st["starts"][s]].flatten(1, 2)


def _scores(st):
    """Scores [sequence][kv_head][head of it][token][position], minus infinity where a token does not see the position."""
    case = st["case"]
    q, at, live = _queries(st)
    k = _rows(st, st["k"], st["ks"], st["blocks"][0])
    x = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).unflatten(2, q.shape[2:4]).mul_(st["scale"])
    j = torch.arange(st["most"], device="cuda")
    seen = (j <= at[..., None]) & live[..., None]
    if case["window"]:
        seen &= (j > at[..., None] - case["window"]) | (j < case["sinks"])
    if case.get("observe"):
        seen &= (at >= st["lengths"][:, None] - case["observe"])[..., None]
    return x.masked_fill_(~seen[:, None, None], -math.inf)


def _plain_attend(st):
    x = _scores(st)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = _rows(st, st["v"], st["vs"], st["blocks"][1])
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, p.shape[2:4])
    o = _flat(st, torch.where(total > 0, o / total, torch.zeros_like(o)))
    if st["gate"] is not None:
        o = o / (1 + torch.exp(-st["gate"]))
    out = {"out": o.half()}
    if st["lse"] is not None:
        out["lse"] = _flat(st, (m + torch.log(total)).squeeze(-1))
    return out


def _plain_weigh(st):
    x = _scores(st)
    q_rows = _queries(dict(st, q=st["lse"].unsqueeze(-1)))[0]      # the statistics, laid out as the queries are
    st["weights"] += x.sub_(q_rows).exp_().sum((2, 3))
    return st["weights"]


def _slots(st):
    """Page and slot of every new token, and its position for the RoPE."""
    row = torch.arange(st["total"], device="cuda")
    s = torch.searchsorted(st["starts"][1:].contiguous(), row, right=True)
    at = st["lengths"][s] - st["starts"][s + 1] + row
    return st["table"][s, (at // st["page"]).long()].long(), (at % st["page"]).long(), at if st["positions"] is None else st["positions"]


def _plain_store(st):
    d, page, slot, at = st["d"], *_slots(st)
    x = st["key"].float().unflatten(1, (st["hkv"], d))
    if st["weight"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * st["weight"]
    half = d // 2 if st["case"]["shape"] == "dense" else 32        # NeoX: pairs (i, i + d/2); sectioned: (i, i + 32) of the first 64
    angle = at.double()[:, None] * THETA ** (-torch.arange(half, device="cuda").double() / half)
    c, s = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))
    a, b = x[..., :half], x[..., half:2 * half]
    x = torch.cat((a * c - b * s, a * s + b * c, x[..., 2 * half:]), -1)
    got = []
    for new, plane, scales, block in ((x, "k", "ks", st["blocks"][0]), (st["value"].float().unflatten(1, (st["hkv"], d)), "v", "vs", st["blocks"][1])):
        if block:
            st[plane][page, :, slot], st[scales][page, :, slot] = _quantise(new, block)
            r = st[plane][page, :, slot].float().unflatten(-1, (-1, block)) * st[scales][page, :, slot].float().unsqueeze(-1)
            got.append(r.flatten(-2).half())
        else:
            st[plane][page, :, slot] = new.half()
            got.append(st[plane][page, :, slot])
    return {"key": got[0], "value": got[1]}


def _plain_evict(st):
    case, keep, page = st["case"], st["case"]["keep"], st["page"]
    j = torch.arange(st["most"], device="cuda")
    length = st["lengths"][:, None, None]
    pinned = (j < case["sinks"]) | (j >= length - case["recent"])
    w = torch.where(pinned, math.inf, st["weights"]).masked_fill(j >= length, -math.inf)
    first = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]       # ties: the lowest position
    missing = keep - first.shape[-1]
    if missing > 0:
        first = torch.nn.functional.pad(first, (0, missing), value=st["most"])
    kept = first.masked_fill(first >= length, st["most"]).sort(-1).values
    there = kept < length
    at = kept.clamp(max=st["most"] - 1)
    s, h, r = (x.flatten() for x in torch.broadcast_tensors(torch.arange(at.shape[0], device="cuda")[:, None, None], torch.arange(st["hkv"], device="cuda")[:, None], torch.arange(keep, device="cuda")))
    ok = there.flatten()
    s, h, r, at_ok = s[ok], h[ok], r[ok], at.flatten()[ok]
    old, new = st["table"][s, at_ok // page].long(), st["target"][s, r // page].long()
    for plane in ("k", "ks", "v", "vs"):
        if st[plane] is not None:
            st[plane][new, h, r % page] = st[plane][old, h, at_ok % page]
    got = {"kept": torch.where(there, kept, -1).int(), "lengths": st["lengths"].clamp(max=keep),
           "weights": torch.where(there, st["weights"].gather(2, at), torch.zeros_like(st["new_weights"]))}
    return got | {plane: st[plane] for plane in ("k", "ks", "v", "vs") if st[plane] is not None}


# ---- the framework's calls ----------------------------------------------------------------------------------------------------------------


def _own(st):
    from miinfer_b200 import kv, paged

    case = st["case"]
    if case["kind"] == "attend":
        paged.launch_paged_attention(st["view"], st["batch"], st["q"], st["out"], query_heads=st["hq"], scale=st["scale"], window=case["window"],
                                     sinks=case["sinks"], gate=st["gate"], lse=st["lse"], workspace=st["workspace"])
        return {"out": st["out"]} | ({} if st["lse"] is None else {"lse": st["lse"]})
    if case["kind"] == "weigh":
        paged.launch_paged_weights(st["view"], st["batch"], st["q"], st["lse"], st["weights"], query_heads=st["hq"], scale=st["scale"],
                                   window=case["window"], sinks=case["sinks"], observe=case["observe"])
        return st["weights"]
    if case["kind"] == "store":
        paged.launch_paged_store(st["view"], st["batch"], st["key"], st["value"], st["weight"], theta=THETA, epsilon=EPSILON, positions=st["positions"],
                                 rope_mode=kv.RopeMode.NEOX_FULL if case["shape"] == "dense" else kv.RopeMode.SECTIONED64)
        paged.launch_paged_load(st["view"], st["batch"], st["key_out"], st["value_out"])
        return {"key": st["key_out"], "value": st["value_out"]}
    paged.launch_paged_evict(st["view"], st["batch"], st["target"], st["weights"], keep=case["keep"], sinks=case["sinks"], recent=case["recent"],
                             new_weights=st["new_weights"], kept=st["kept"], new_lengths=st["new_lengths"])
    return {"kept": st["kept"], "lengths": st["new_lengths"], "weights": st["new_weights"]} | {p: st[p] for p in ("k", "ks", "v", "vs") if st[p] is not None}


def run(st):
    if own:
        return _own(st)
    return {"attend": _plain_attend, "weigh": _plain_weigh, "store": _plain_store, "evict": _plain_evict}[st["case"]["kind"]](st)


# ---- from the definitions, in 64 bits, one sequence and kv head after the other -----------------------------------------------------------------


def _cached(st, s, h, plane, scales, block):
    """Rows of one sequence's kv head."""
    length = int(st["lengths"][s])
    pages = st["table"][s, :-(-length // st["page"])].long()
    x = st[plane][pages, h].double().flatten(0, 1)[:length]
    return x if not block else (x.unflatten(1, (-1, block)) * st[scales][pages, h].double().flatten(0, 1)[:length, :, None]).flatten(1)


def _each(st):
    """Per sequence and kv head: the rows of its tokens, its query heads, and the scores with what is not seen at minus infinity."""
    case, group = st["case"], st["hq"] // st["hkv"]
    for s in range(case["sequences"]):
        begin, end, length = int(st["starts"][s]), int(st["starts"][s + 1]), int(st["lengths"][s])
        if begin == end:
            continue
        at = torch.arange(length - (end - begin), length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        hidden = j > at
        if case["window"]:
            hidden = hidden | ((at - j >= case["window"]) & (j >= case["sinks"]))
        if case.get("observe"):
            hidden = hidden | (length - at > case["observe"])
        for h in range(st["hkv"]):
            k = _cached(st, s, h, "k", "ks", st["blocks"][0])
            q = st["q"][begin:end, h * group:(h + 1) * group].double().transpose(0, 1)
            yield s, h, slice(begin, end), slice(h * group, (h + 1) * group), (q @ k.T * st["scale"]).masked_fill(hidden, -math.inf)


def _statistics(st):
    lse = torch.full((st["total"], st["hq"]), -math.inf, dtype=torch.float64, device="cuda")
    for _, _, rows, heads, x in _each(dict(st, case=dict(st["case"], observe=0))):
        lse[rows, heads] = torch.logsumexp(x, -1).T
    return lse


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "attend":
        out = torch.zeros(st["total"], st["hq"], st["d"], dtype=torch.float64, device="cuda")
        for s, h, rows, heads, x in _each(st):
            out[rows, heads] = (torch.softmax(x, -1) @ _cached(st, s, h, "v", "vs", st["blocks"][1])).transpose(0, 1)
        if st["gate"] is not None:
            out *= torch.sigmoid(st["gate"].double())
        return {"out": out} | ({"lse": _statistics(st)} if case["lse"] else {})
    if case["kind"] == "weigh":
        weights = st["weights"].double()
        for s, h, rows, heads, x in _each(st):
            weights[s, h, :x.shape[2]] += torch.exp(x - st["lse"][rows, heads].double().T[..., None]).sum((0, 1))
        return weights
    if case["kind"] == "evict":
        weights = torch.zeros(case["sequences"], st["hkv"], case["keep"], dtype=torch.float64)     # the rest is a choice and copies: nothing is computed
        for s in range(case["sequences"]):
            length = int(st["lengths"][s])
            for h in range(st["hkv"]):
                w = st["weights"][s, h, :length].double().cpu().numpy()
                rank = w.copy()
                rank[:case["sinks"]] = rank[max(0, length - case["recent"]):] = np.inf
                chosen = np.sort(np.lexsort((np.arange(length), -rank))[:case["keep"]])
                weights[s, h, :len(chosen)] = torch.from_numpy(w[chosen])
        return {"weights": weights}
    d, hkv = st["d"], st["hkv"]
    got = {}
    for name, block in (("key", st["blocks"][0]), ("value", st["blocks"][1])):
        x = st[name].double().view(st["total"], hkv, d)
        if name == "key":
            if st["weight"] is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPSILON).sqrt() * st["weight"].double()
            width = d if case["shape"] == "dense" else 64
            positions = [length - n + t + (case["shift"] + i if case["shift"] else 0) for i, (n, length) in enumerate(_batch(case)) for t in range(n)]
            power = torch.arange(0, width, 2, dtype=torch.float64, device="cuda") / width
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.tensor(positions, dtype=torch.float64, device="cuda")[:, None] / THETA ** power)
            z = torch.complex(x[..., :width // 2].contiguous(), x[..., width // 2:width].contiguous()) * turn[:, None]
            x = torch.cat((z.real, z.imag, x[..., width:]), -1)
        if block:
            b = x.reshape(st["total"], hkv, d // block, block)
            step = b.abs().amax(-1, keepdim=True) / 127
            step = torch.where(step > 0, step, 1.0)
            x = (torch.round(b / step).clamp(-128, 127) * step.half().double()).reshape(st["total"], hkv, d)
        got[name] = x
    return got
