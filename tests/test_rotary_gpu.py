"""The rotary store against plain arithmetic in 64 bits: queries, gates and the cache's rows, at the layouts, scalings, strides and positions where it can go wrong."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from miinfer_b200 import kv, paged

pytestmark = pytest.mark.gpu

MODES = [(0, 32), (3, 32), (3, None), (1, 32), (2, None)]      # (quant mode, qblock; None = head_dim)
HALVES, NEIGHBOURS = paged.RotaryLayout.HALVES, paged.RotaryLayout.NEIGHBOURS


@pytest.fixture
def status():
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv.set_status_word(word)
    yield word
    kv.set_status_word(None)


def rotated(x, positions, frequencies, magnitude, layout, weight=None, epsilon=1e-6):
    """(x', its bound before any rounding to fewer bits) of rows [token][head][d], float64."""
    d, n = x.shape[2], 2 * len(frequencies)
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + epsilon) * weight.astype(np.float64)
    angle = np.asarray(positions, np.float64)[:, None] * frequencies
    c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if layout == HALVES else (x[..., 0:n:2], x[..., 1:n:2])
    y, size = x.copy(), np.abs(x)
    u, v, w = a * c - b * s, a * s + b * c, (np.abs(a) + np.abs(b)) * magnitude
    if layout == HALVES:
        y[..., :n // 2], y[..., n // 2:n], size[..., :n // 2], size[..., n // 2:n] = u, v, w, w
    else:
        y[..., 0:n:2], y[..., 1:n:2], size[..., 0:n:2], size[..., 1:n:2] = u, v, w, w
    # sine and cosine are off by 2^-22 (a polynomial good to 3e-8 and its roundings), the angle by 2^-32 of a turn, products and sums by 2^-24 each; a norm's sum of 256 squares, in runs of
    # eight and a tree of five, by 2^-21, its root by half of that, and three more roundings.  Float64 angles of positions below 2^31 are good to 2^-53 of 2^31: 2^-22.
    far = np.abs(angle).max(initial=0) * 2.0 ** -52
    return y, size * (2.0 ** -20.5 + far + (2.0 ** -20 if weight is not None else 0.0)) if n or weight is not None else np.zeros_like(y)


def frequencies(dims, theta=1e6):
    return theta ** (-np.arange(dims // 2) * 2.0 / dims) if dims else np.zeros(0)


def cache_bound(y, e, q8, qblock):
    """How far a cache row may be from y: fp16's rounding, or half a step of its block and the rounding of its scale."""
    if not q8:
        return e + (np.abs(y) + e) * po.HALF_STEP + 2.0 ** -25
    most = np.repeat(np.abs(y).reshape(*y.shape[:2], -1, qblock).max(-1), qblock, axis=-1)
    spread = np.repeat(e.reshape(*y.shape[:2], -1, qblock).max(-1), qblock, axis=-1)
    return e + (most + spread) / 254 * (1 + 2.0 ** -20) + (np.abs(y) + most / 254 + e) * po.HALF_STEP + 2.0 ** -24


class Setup:
    def __init__(self, seed, tokens, lengths, *, d, hq, heads, page, mode, qblock, act, gated=False, pad_rows=2, packed=True, scale=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.pool = po.Pool(rng, lengths, d=d, heads=heads, page=page, mode=mode, qblock=qblock or d)
        self.view = self.pool.upload()
        self.batch, self.starts = po.batch_of(self.pool, tokens, pad_rows=pad_rows)
        total, wide = self.batch.total_tokens, hq * d * (2 if gated else 1)
        self.tokens, self.lengths, self.hq, self.d, self.heads, self.gated, self.total = tokens, lengths, hq, d, heads, gated, total
        rows = (rng.standard_normal((total, wide + 2 * heads * d)) * scale).astype(act)
        self.rows = rows
        dev = torch.from_numpy(rows).cuda()
        self.q, self.key, self.value = dev[:, :wide], dev[:, wide:wide + heads * d], dev[:, wide + heads * d:]
        if not packed:
            self.q, self.key, self.value = (t.contiguous() for t in (self.q, self.key, self.value))
        self.hk, self.hv = (rows[:, wide + i * heads * d:wide + (i + 1) * heads * d].reshape(total, heads, d) for i in (0, 1))
        hqs = rows[:, :wide].reshape(total, hq, -1)
        self.hq_rows, self.hgate = hqs[..., :d], hqs[..., d:]
        self.live = np.concatenate([np.arange(self.starts[s], self.starts[s] + n) for s, n in enumerate(tokens)]).astype(int)
        self.places = np.concatenate([np.arange(length - n, length) for n, length in zip(tokens, lengths)])

    def check_cache(self, positions, f, magnitude, layout, weight, epsilon=1e-6):
        p = self.pool
        p.k, p.ks, p.v, p.vs = (None if t is None else t.cpu().numpy() for t in p.dev)
        y, e = rotated(self.hk[self.live], positions, f, magnitude, layout, weight, epsilon)
        bounds = (cache_bound(y, e, p.mode in (1, 3), p.qblock), cache_bound(self.hv[self.live].astype(np.float64), np.zeros_like(y), p.mode in (2, 3), p.qblock))
        for s, n in enumerate(self.tokens):
            rows = slice(sum(self.tokens[:s]), sum(self.tokens[:s + 1]))
            for h in range(self.heads):
                for side, want, bound in ((0, y, bounds[0]), (1, self.hv[self.live].astype(np.float64), bounds[1])):
                    off = np.abs(p.rows(s, h, side)[self.lengths[s] - n:] - want[rows, h])
                    assert (off <= bound[rows, h]).all(), (s, h, side, off.max())


@pytest.mark.parametrize("mode,qblock", MODES)
@pytest.mark.parametrize("d,hq,heads,page,act,dims,layout,gated,norm", [
    (128, 8, 2, 16, np.float16, 128, HALVES, False, False), (128, 7, 7, 32, np.float32, 64, NEIGHBOURS, False, True), (256, 6, 1, 64, np.float16, 256, HALVES, True, True),
    (256, 5, 5, 16, np.float32, 96, HALVES, True, False), (128, 3, 1, 128, np.float16, 16, NEIGHBOURS, True, True), (256, 2, 2, 256, np.float16, 240, NEIGHBOURS, False, False),
    (128, 1, 1, 16, np.float32, 112, HALVES, False, True), (256, 4, 4, 32, np.float16, 48, HALVES, False, True)])
def test_rows_against_the_formula(cuda, status, mode, qblock, d, hq, heads, page, act, dims, layout, gated, norm):
    s = Setup(100 * mode + d + dims, [3, 0, 1, 40, 17], [19, 5, 1, 40, 300], d=d, hq=hq, heads=heads, page=page, mode=mode, qblock=qblock, act=act, gated=gated)
    weights = [(1 + 0.2 * s.rng.standard_normal(d)).astype(np.float32) if norm else None for _ in range(2)]
    qw, kw = (None if w is None else torch.from_numpy(w).cuda() for w in weights)
    table = paged.RotaryTable(dims, layout=layout, magnitude=1.25)
    before = [None if p is None else p.clone() for p in s.pool.dev]
    for out_type in (torch.float16, torch.float32):
        out = torch.full((s.total, hq, d), 7.0, dtype=out_type, device="cuda")
        gate = torch.full((s.total, hq, d), 7.0, device="cuda") if gated else None
        paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value, s.q, out, query_heads=hq, gate=gate, q_norm_weight=qw, k_norm_weight=kw, epsilon=1e-5)
        y, e = rotated(s.hq_rows[s.live], s.places, frequencies(dims), 1.25, layout, weights[0], 1e-5)
        if out_type == torch.float16:
            e = e + (np.abs(y) + e) * po.HALF_STEP + 2.0 ** -25
        assert (np.abs(out.cpu().numpy()[s.live].astype(np.float64) - y) <= e + np.abs(y) * 2.0 ** -23).all()
        assert bool((out[-2:] == 7).all())
        if gated:
            assert np.array_equal(gate.cpu().numpy()[s.live], s.hgate[s.live].astype(np.float32)) and bool((gate[-2:] == 7).all())
    s.check_cache(s.places, frequencies(dims), 1.25, layout, weights[1], 1e-5)
    written = np.zeros((s.pool.pages, page), bool)
    for q, (n, length) in enumerate(zip(s.tokens, s.lengths)):
        for j in range(length - n, length):
            written[s.pool.place(q, j)] = True
    for now, old in zip(s.pool.dev, before):      # no other row of the pool
        if now is not None:
            assert not ((now != old).any(-1).any(1).cpu().numpy() & ~written).any()
    assert int(status) == 0


@pytest.mark.parametrize("mode,qblock", MODES + [(2, 32), (1, None)])
@pytest.mark.parametrize("d,heads,act", [(128, 8, np.float16), (128, 3, np.float32), (256, 4, np.float32), (256, 1, np.float16)])
def test_without_a_rotation_the_bits_are_the_store_s(cuda, mode, qblock, d, heads, act):
    s = Setup(mode + d, [5, 33, 1], [20, 33, 129], d=d, hq=4, heads=heads, page=32, mode=mode, qblock=qblock, act=act)
    s.key[0].zero_()                                 # a block of zeros, infinities and NaN among the numbers
    s.value[1, :40] = float("inf")
    s.key[2, 3], s.value[3, 7], s.value[4, 100] = float("nan"), float("nan"), -float("inf")
    key, value = s.key.contiguous(), s.value.contiguous()
    paged.launch_paged_store(s.view, s.batch, key, value, None, rope_mode=kv.RopeMode.NONE)
    want = [None if p is None else p.clone() for p in s.pool.dev]
    for p in s.pool.dev:
        if p is not None:
            p.zero_()
    first = [None if p is None else p.clone() for p in s.pool.dev]
    table = paged.RotaryTable(16, frequencies=[0.0] * 8)
    table.dims = 0
    paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value)
    for q, (n, length) in enumerate(zip(s.tokens, s.lengths)):
        for j in range(length - n, length):
            page, slot = s.pool.place(q, j)
            for got, w in zip(s.pool.dev, want):
                if got is not None:
                    assert torch.equal(got[page, :, slot].contiguous().view(torch.uint8), w[page, :, slot].contiguous().view(torch.uint8)), (q, j)
    assert all(f is None or not torch.equal(f.view(torch.uint8), g.view(torch.uint8)) for f, g in zip(first, s.pool.dev))


@pytest.mark.parametrize("layout", [HALVES, NEIGHBOURS])
def test_far_positions(cuda, status, layout):
    """Angles of positions up to 2^31 - 1, against rational turns of the table; negative ones count as 0."""
    s = Setup(3, [9], [30], d=128, hq=2, heads=1, page=16, mode=0, qblock=32, act=np.float32, pad_rows=0)
    positions = [0, 1, -5, 131071, 1 << 20, 16777217, 1 << 30, (1 << 31) - 1, 2000000011]
    table = paged.RotaryTable(128, layout=layout)
    out = torch.zeros(9, 2, 128, device="cuda")
    paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value, s.q, out, query_heads=2, positions=po.ints(positions))
    turns = [int(t) % 2 ** 64 for t in table.table.cpu().tolist()]
    angle = np.array([[(max(p, 0) * t % 2 ** 64) / 2.0 ** 64 for t in turns] for p in positions])[:, None] * 2 * np.pi
    x = s.hq_rows.astype(np.float64)
    a, b = (x[..., :64], x[..., 64:]) if layout == HALVES else (x[..., 0::2], x[..., 1::2])
    u, v, size = a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle), (np.abs(a) + np.abs(b)) * 2.0 ** -20.5
    got = out.cpu().numpy().astype(np.float64)
    g, h = (got[..., :64], got[..., 64:]) if layout == HALVES else (got[..., 0::2], got[..., 1::2])
    assert (np.abs(g - u) <= size).all() and (np.abs(h - v) <= size).all()
    assert int(status) == 0
    s.pool.k = s.pool.dev[0].cpu().numpy()
    k = s.hk.astype(np.float64)[:, 0]
    a, b = (k[:, :64], k[:, 64:]) if layout == HALVES else (k[:, 0::2], k[:, 1::2])
    rows = s.pool.rows(0, 0, 0)[21:]
    g = rows[:, :64] if layout == HALVES else rows[:, 0::2]
    want = a * np.cos(angle[:, 0]) - b * np.sin(angle[:, 0])
    assert (np.abs(g - want) <= np.abs(want) * po.HALF_STEP + (np.abs(a) + np.abs(b)) * 2.0 ** -20 + 2.0 ** -24).all()


def test_in_place_queries_only_keys_only_and_a_single_row(cuda, status):
    s = Setup(8, [4, 1], [10, 70], d=128, hq=6, heads=2, page=16, mode=3, qblock=32, act=np.float16, packed=False, pad_rows=1)
    table = paged.RotaryTable(64)
    out = torch.zeros(6, 6, 128, dtype=torch.float16, device="cuda")
    clean = [p.clone() for p in s.pool.dev]
    paged.launch_paged_rotary(s.view, s.batch, table, None, None, s.q, out, query_heads=6)
    assert all(torch.equal(a, b) for a, b in zip(s.pool.dev, clean))                  # queries only
    last = s.q[-1].clone()
    paged.launch_paged_rotary(s.view, s.batch, table, None, None, s.q, s.q, query_heads=6)
    assert torch.equal(s.q[:5].view(5, 6, 128), out[:5]) and torch.equal(s.q[-1], last)   # where they lie
    paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value)                 # keys only
    s.check_cache(s.places, frequencies(64), 1.0, HALVES, None)
    one = Setup(9, [1], [1], d=256, hq=1, heads=1, page=16, mode=0, qblock=32, act=np.float32, pad_rows=0)
    table = paged.RotaryTable(256, layout=NEIGHBOURS)
    out = torch.zeros(1, 1, 256, device="cuda")
    paged.launch_paged_rotary(one.view, one.batch, table, one.key, one.value, one.q, out, query_heads=1)
    assert np.array_equal(out.cpu().numpy()[0], one.hq_rows[0])                       # position 0
    one.check_cache(one.places, frequencies(256), 1.0, NEIGHBOURS, None)
    assert int(status) == 0


def test_many_tokens_and_rows_behind_the_last_sequence(cuda, status):
    """More tokens than warps at a time (one warp a token), arrays that end before the activations do."""
    s = Setup(10, [3000, 2500, 0, 700], [3000, 2501, 4, 900], d=128, hq=3, heads=1, page=64, mode=3, qblock=32, act=np.float16, pad_rows=50)
    table = paged.RotaryTable(128, layout=NEIGHBOURS, scaling=paged.RotaryScaling.LINEAR, factor=4.0)
    out = torch.full((s.total, 3, 128), -3.0, dtype=torch.float16, device="cuda")
    paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value, s.q, out, query_heads=3)
    y, e = rotated(s.hq_rows[s.live], s.places, frequencies(128) / 4, 1.0, NEIGHBOURS)
    assert (np.abs(out.cpu().numpy()[s.live].astype(np.float64) - y) <= e + (np.abs(y) + e) * po.HALF_STEP + 2.0 ** -25).all()
    assert bool((out[-50:] == -3).all()) and int(status) == 0
    s.check_cache(s.places, frequencies(128) / 4, 1.0, NEIGHBOURS, None)


def test_pages_outside_the_pool_and_lengths_below_the_tokens(cuda, status):
    s = Setup(11, [12, 3], [40, 33], d=128, hq=2, heads=2, page=16, mode=3, qblock=32, act=np.float16, pad_rows=0)
    good = s.pool.table.copy()
    s.pool.table_dev[0, 2] = s.pool.pages
    before = [p.clone() for p in s.pool.dev]
    out = torch.zeros(15, 2, 128, dtype=torch.float16, device="cuda")
    table = paged.RotaryTable(128)
    paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value, s.q, out, query_heads=2)
    assert int(status) == paged.STATUS_BAD_PAGE
    changed = (s.pool.dev[0] != before[0]).any(-1).any(1).cpu().numpy()
    allowed = np.zeros_like(changed)
    for j in range(28, 32):
        allowed[good[0, j // 16], j % 16] = True
    for j in range(30, 33):
        allowed[good[1, j // 16], j % 16] = True
    assert not (changed & ~allowed).any()
    y, e = rotated(s.hq_rows, s.places, frequencies(128), 1.0, HALVES)                # the queries are there all the same
    assert (np.abs(out.cpu().numpy().astype(np.float64) - y) <= e + (np.abs(y) + e) * po.HALF_STEP + 2.0 ** -25).all()
    status.zero_()
    for p, b in zip(s.pool.dev, before):
        p.copy_(b)
    batch, _ = po.batch_of(s.pool, [12, 3])
    batch.tensors[2].copy_(po.ints([5, 33]))                                          # seven of the tokens have no place
    paged.launch_paged_rotary(s.view, batch, table, s.key, s.value, s.q, out, query_heads=2)
    changed = (s.pool.dev[0] != before[0]).any(-1).any(1).cpu().numpy()
    allowed[:] = False
    allowed[good[0, 0], :5] = True
    for j in range(30, 33):
        allowed[good[1, j // 16], j % 16] = True
    assert not (changed & ~allowed).any() and changed[good[0, 0], :5].all()


def test_captured_and_on_a_stream_of_its_own(cuda, status):
    s = Setup(12, [2, 1], [20, 70], d=128, hq=4, heads=2, page=16, mode=3, qblock=32, act=np.float16, pad_rows=0)
    table = paged.RotaryTable(128, scaling=paged.RotaryScaling.BANDS, factor=8.0, original_length=64, low=1.0, high=4.0)
    eager, got = (torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    positions = po.ints([3, 4, 9])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value, s.q, got, query_heads=4, positions=positions)
    for p in ([3, 4, 9], [100000, 7, 70]):
        positions.copy_(po.ints(p))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        paged.launch_paged_rotary(s.view, s.batch, table, s.key, s.value, s.q, eager, query_heads=4, positions=positions, stream=stream)
        stream.synchronize()
        want = [t.clone() for t in s.pool.dev]
        got.zero_()
        graph.replay()
        assert torch.equal(eager, got) and all(torch.equal(a, b) for a, b in zip(want, s.pool.dev))
    assert int(status) == 0


def test_tensors_that_are_refused(cuda):
    s = Setup(13, [2, 1], [20, 70], d=128, hq=4, heads=2, page=16, mode=3, qblock=32, act=np.float16, pad_rows=0)
    table, out = paged.RotaryTable(128), torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    go = lambda key=s.key, value=s.value, q=s.q, o=out, table=table, heads=4, **k: paged.launch_paged_rotary(s.view, s.batch, table, key, value, q, o, query_heads=heads, **k)
    go()
    for bad in (dict(key=s.key.float()), dict(q=s.q.float()), dict(key=s.key[:2]), dict(key=s.key[:, :128]), dict(value=s.value.view(3, 2, 128)), dict(q=s.q.t()), dict(q=s.q.cpu()),
                dict(o=out[:2]), dict(o=out.long()), dict(heads=0), dict(heads=8), dict(gate=torch.zeros(3, 4, 128, device="cuda")), dict(positions=po.ints([1, 2])),
                dict(k_norm_weight=torch.ones(64, device="cuda")), dict(q_norm_weight=torch.ones(128, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            go(**bad)
    with pytest.raises(TypeError):
        go(table=s.view)
    for bad in (dict(key=None), dict(o=None), dict(epsilon=float("nan")), dict(q=torch.zeros(3, 516, dtype=torch.float16, device="cuda")[:, :512])):
        with pytest.raises(paged._lib.B200KvError):
            go(**bad)
    for bad in (dict(dims=0), dict(dims=24), dict(dims=272), dict(dims=64, frequencies=[1.0] * 31), dict(dims=64, frequencies=[1.0] * 32, scaling=1)):
        with pytest.raises(ValueError):
            paged.RotaryTable(**bad)
    with pytest.raises(paged._lib.B200KvError):
        paged.RotaryTable(64, scaling=paged.RotaryScaling.BANDS, factor=2.0)
