"""The paged cache's operators at the edges of their types and arguments:
probabilities far below the largest, scores that leave one slot, evictions of
sequences that miss pages, and sizes at the limits of a launch. Bounds as in
paged_util, or derived beside the test."""
import ctypes as C

import numpy as np
import pytest

import lfm3amd as L
import paged_util as P

pytestmark = pytest.mark.gpu
F16, BF16, F32 = L.TYPE_F16, L.TYPE_BF16, L.TYPE_F32
PAIRS = [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)]
TILINGS = [(16, 4096), (16, 64), (128, 4096), (128, 192), (256, 4096), (256, 320)]


def seeded(seed, kv, page, dim, kind, rows, lengths):
    counts = [-(-n // page) for n in lengths]
    pool = P.Pool(seed, sum(counts) + 1, kv, page, dim, kind)
    return pool, P.Batch(rows, lengths, P.tables(seed + 1, counts, pool.pages))


@pytest.mark.parametrize("kind,row_kind", PAIRS)
@pytest.mark.parametrize("columns,span", TILINGS)
@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 128), (8, 4, 64)])
@pytest.mark.parametrize("gap", [11.0, 17.0])
def test_attention_sink_and_long_tail(gap, heads, kv, dim, columns, span, kind, row_kind):
    """A first slot without a value takes nearly all of the weight, and what the
    output holds is the sum of probabilities e^-gap below it: each of them has
    to keep its own accuracy. (Their products with values of one sign add up, so
    that roundings of one direction would show.)"""
    pool, b = seeded(201, kv, 32, dim, kind, [40, 1], [2000, 1500])
    rng = np.random.default_rng(202)
    k = rng.standard_normal(pool.shape, np.float32) * np.float32(0.2)
    v = 1 + 0.25 * rng.standard_normal(pool.shape, np.float32)
    k[..., 0] = 0
    for s in range(b.seqs):
        p = int(b.table[s, 0])
        k[p, :, 0] = 0
        k[p, :, 0, 0] = gap * np.sqrt(dim) / 8
        v[p, :, 0] = 0
    pool.k, pool.v = P.to_bits(k, kind), P.to_bits(v, kind)
    q = rng.standard_normal((b.rows, heads, dim), np.float32)
    q[..., 0] = 8
    pool.upload(), b.upload()
    call = P.AttentionCall(pool, b, q, heads, 0, None, row_kind,
                           items=P.tiled(b, heads, kv, 0, columns, span))
    call.launch()
    L.synchronize()
    got, _ = call.results()
    got = got.reshape(q.shape)
    want, tol, _, _, _ = P.attention(pool, b, call.q.values, heads, 0, None, row_kind)
    if kind == F16:  # parts of a probability end at 2^-40 of the largest; the sum is at least 1
        slots = np.repeat(np.asarray(b.lengths), b.counts)
        tol = tol + 2.0 ** -40 * (slots * np.abs(v).max())[:, None, None]
        tol += 2.0 ** -25 * (row_kind == F16)   # half of F16's lowest step, below 2^-14
    assert want[5].max() > 2.0 ** -14       # a normal value in either type
    far = np.abs(got - want) - tol
    worst = np.unravel_index(np.argmax(far), far.shape)
    assert not (far > 0).any(), (worst, got[worst], want[worst], tol[worst])


@pytest.mark.parametrize("kind,row_kind,key,query", [
    (*pair, *size) for pair in PAIRS
    for size in ((4.0, 20.0), (300.0, 500.0), (3000.0, 30000.0), (3000.0, 3e9))
    if size[1] < 65504 or pair[1] != F16])
@pytest.mark.parametrize("columns,span", TILINGS)
@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 128), (8, 4, 64)])
def test_attention_of_one_winner(key, query, heads, kv, dim, columns, span, kind, row_kind):
    """Keys of random signs and a query along one of them: its score is hundreds
    to 10^14 above every other, the output is its value and lse its score."""
    pool, b = seeded(211, kv, 32, dim, kind, [40, 1], [700, 500])
    rng = np.random.default_rng(212)
    sign = rng.choice(np.array([-1, 1], np.float32), pool.shape)
    pool.k = P.to_bits(key * sign, kind)
    q = np.zeros((b.rows, heads, dim), np.float32)
    want, value = np.zeros(q.shape), P.from_bits(pool.v, kind)
    for s in range(b.seqs):
        before = int(b.lengths[s]) - b.counts[s]
        for j in range(b.counts[s]):
            r = int(b.starts[s]) + j
            for h in range(heads):
                t = int(rng.integers(0, before + j + 1))
                at = (int(b.table[s, t // 32]), h // (heads // kv), t % 32)
                q[r, h], want[r, h] = query * sign[at], value[at]
    pool.upload(), b.upload()
    gate = rng.standard_normal((b.rows, heads), np.float32)
    call = P.AttentionCall(pool, b, q, heads, 0, gate, row_kind,
                           items=P.tiled(b, heads, kv, 0, columns, span))
    call.launch()
    L.synchronize()
    raw, lse = call.results()
    k0, q0 = np.abs(P.from_bits(pool.k, kind)).max(), np.abs(call.q.values).max()
    score = k0 * q0 * np.sqrt(dim)
    # The next largest score: each row's other keys, in units of the winner's.
    for s in range(b.seqs):
        page, off, _ = P.slots_of(pool, b.table[s], int(b.lengths[s]))
        rows = slice(int(b.starts[s]), int(b.starts[s + 1]))
        for g in range(kv):
            unit = np.sign(q[rows, g * (heads // kv):(g + 1) * (heads // kv)])
            second = np.sort((unit @ sign[page, g, off].T / dim), -1)[..., -2].max()
            assert score * (1 - second) > 40
    want = want / (1 + np.exp(-gate.astype(np.float64)))[:, :, None]
    # The probability's rounding (FP32 rows: its parts, 2^-21) and the output's.
    step = P.HALF_STEP[row_kind]
    # F16 values below 2^-14 lie 2^-24 apart: half of that.
    tol = np.abs(want) * (2 * step + 2.0 ** -20) + 2.0 ** -25 * (row_kind == F16)
    got = raw.reshape(q.shape)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()
    # FP32 sums of dim terms of one sign, and the scale's rounding.
    assert np.abs(lse - score).max() <= score * (dim + 8) * 2.0 ** -24


# Sequences: (length, the table entries that name no page). Sinks and recent
# slots lie on pages, as the call asks.
MISSING = [
    # fewer present than the budget; none missing; all but the first and last page
    (16, 96, 4, 10, [(200, range(1, 9)), (100, []), (160, range(1, 9)), (7, [])]),
    # a length within the budget, with and without holes; one slot past it
    (16, 128, 4, 16, [(128, [2, 5]), (90, [1]), (60, []), (129, [3]), (0, [])]),
    # nothing between the sinks and the recent slots
    (32, 64, 32, 32, [(640, [3, 9]), (64, []), (40, [])]),
    # no sinks: the first pages are gone, as a sliding window leaves them
    (64, 1000, 0, 100, [(3000, range(0, 40)), (900, [0, 1]), (1500, range(0, 20))]),
    # in slices: too few present, enough, and lengths within the budget
    (64, 5000, 4, 64, [(20000, range(1, 300)), (20000, range(1, 100)), (4000, [3, 20]),
                       (300, [])]),
    # longer than a block's ranks and all within the budget; nothing left of the last
    (128, 20000, 0, 0, [(18000, [0, 7, 100]), (17000, []), (100, [0])]),
]


@pytest.mark.parametrize("kind,dim", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("shape", range(len(MISSING)))
def test_evict_drops_slots_on_no_page(shape, kind, dim):
    """A sequence keeps what lies on a page, up to the budget; what the new pages
    held before is seen by no row and ranks nowhere afterwards."""
    page, budget, sinks, recent, sequences = MISSING[shape]
    kv, heads, n = 2, 4, len(sequences)
    lengths = [length for length, _ in sequences]
    counts = [max(-(-length // page), 1) for length in lengths]
    new_counts = [max(-(-(min(length, budget) + 1) // page), 1) for length in lengths]
    pool = P.Pool(221, sum(counts) + sum(new_counts) + 1, kv, page, dim, kind)
    both = P.tables(222, counts + new_counts, pool.pages)
    table, new = both[:n, :max(counts)].copy(), both[n:, :max(new_counts)].copy()
    for s, (_, missing) in enumerate(sequences):
        table[s, list(missing)] = [0xFFFFFFFF, pool.pages, 0x80000000][s % 3]
    nan = P.to_bits(np.float32(np.nan), kind)
    fresh = new[new < pool.pages]
    pool.k[fresh], pool.v[fresh], pool.w[fresh] = nan, nan, np.nan
    pool.upload()
    # The call, restated: what is on a page, less the lightest between the ends.
    old_k, old_v, old_w = pool.k.copy(), pool.v.copy(), pool.w.copy()
    room = min(budget, max(lengths))
    kept = np.full((n, kv, budget), 0xABABABAB, np.uint32)
    left = []
    for s, length in enumerate(lengths):
        at, off, present = (x[:length] for x in P.slots_of(pool, table[s], max(length, 1)))
        t = np.arange(length)
        always = (t < sinks) | (t + recent >= length)
        left.append(min(int(present.sum()), budget))
        for g in range(kv):
            ranked = t[present & ~always]
            ranked = ranked[np.argsort(-old_w[at[ranked], g, off[ranked]], kind="stable")]
            mine = np.sort(np.concatenate([t[always], ranked[:left[s] - always.sum()]]))
            assert len(mine) == left[s]
            kept[s, g, :len(mine)] = mine
            to, to_off, _ = P.slots_of(pool, new[s], max(len(mine), 1))
            to, to_off = to[:len(mine)], to_off[:len(mine)]
            for x, old in ((pool.k, old_k), (pool.v, old_v), (pool.w, old_w)):
                x[to, g, to_off] = old[at[mine], g, off[mine]]
    assert room <= new.shape[1] * page
    dt, dn, dl = (L.DeviceBuffer.of(np.ascontiguousarray(x, np.uint32))
                  for x in (table, new, lengths))
    out = L.DeviceBuffer.of(np.full(kept.size, 0xABABABAB, np.uint32))
    need = L.lib().lfm3_paged_evict_workspace_bytes(n, kv, budget, max(lengths))
    ws = L.DeviceBuffer.of(np.full(max(need, 16), 0x5A, np.uint8))
    L.check(L.lib().lfm3_paged_evict(
        C.byref(pool.cache), dt.addr, table.shape[1], dl.addr, n, max(lengths), dn.addr,
        new.shape[1], budget, sinks, recent, out.addr, ws.addr, need, None))
    L.synchronize()
    assert np.array_equal(out.download(np.uint32, kept.size).reshape(kept.shape), kept)
    gk, gv, gw = pool.download()
    assert np.array_equal(gk, pool.k) and np.array_equal(gv, pool.v)
    assert np.array_equal(gw.view(np.uint32), pool.w.view(np.uint32))
    # One more token a sequence: heads, attention and weights on the new table.
    b = P.Batch([1] * n, np.array(left) + 1, new).upload()
    rng = np.random.default_rng(223)
    call = P.AttentionCall(pool, b, rng.standard_normal((n, heads, dim), np.float32), heads, 0)
    x = L.DeviceBuffer.of(rng.standard_normal((n, heads * dim), np.float32))
    ones = L.DeviceBuffer.of(np.ones(dim, np.float32))
    L.check(L.lib().lfm3_paged_heads(
        C.byref(pool.cache), C.byref(b.batch), call.q.addr, x.addr, x.addr, heads * dim,
        ones.addr, ones.addr, ones.addr, None, call.q.addr, call.q.ld, F32, heads, 1e-5, None))
    call.launch()
    L.check(L.lib().lfm3_paged_weights(
        C.byref(pool.cache), C.byref(b.batch), call.q.addr, call.q.ld, F32, call.lse.addr, heads,
        0, max(left) + 1, None))
    L.synchronize()
    pool.k, pool.v, gw = pool.download()
    call.q.values = call.q.download().reshape(n, heads, dim)
    P.check_attention(call, shape)
    for s in range(n):
        at, off, _ = P.slots_of(pool, new[s], left[s] + 1)
        assert np.isfinite(gw[at, :, off]).all()


def test_heads_of_more_rows_than_a_launch():
    """Rows up to 2^25: those of 2^24 and more, all but a few of no sequence."""
    kv, heads, dim, far = 1, 1, 64, (1 << 24) + 3
    pool, b = seeded(231, kv, 16, dim, F16, [2, 1], [20, 1])
    b.starts = b.starts + np.uint32(far)
    b.rows = far + 4
    pool.upload(), b.upload()
    rng = np.random.default_rng(232)
    x = rng.standard_normal((3, dim), np.float32)
    rows = L.DeviceBuffer(b.rows * dim * 4)
    out = L.DeviceBuffer(b.rows * dim * 4)
    rows.upload(x, far * dim * 4)
    out.upload(np.full((5, dim), 7.0, np.float32), (far - 1) * dim * 4)
    out.upload(np.full((1, dim), 7.0, np.float32))
    ones = L.DeviceBuffer.of(np.ones(dim, np.float32))
    freq = L.DeviceBuffer.of((1e4 ** (-2.0 * np.arange(dim // 2) / dim)).astype(np.float32))
    L.check(L.lib().lfm3_paged_heads(
        C.byref(pool.cache), C.byref(b.batch), rows.addr, rows.addr, rows.addr, dim, ones.addr,
        ones.addr, freq.addr, None, out.addr, dim, F32, heads, 1e-5, None))
    L.synchronize()
    near = P.Batch([2, 1], b.lengths, b.table)
    wq, eq, _, _ = P.heads_rows(near, x[:, None], x[:, None], x[:, None], np.ones(dim),
                                np.ones(dim), (1e4 ** (-2.0 * np.arange(dim // 2) / dim)
                                               ).astype(np.float32), None, 1e-5)
    got = out.download(np.float32, 5 * dim, (far - 1) * dim * 4).reshape(5, 1, dim)
    assert (got[0] == 7).all() and (got[4] == 7).all()
    assert (out.download(np.float32, dim) == 7).all()
    assert (np.abs(got[1:4] - wq) <= eq + np.abs(wq) * 2.0 ** -23).all()
    _, gv, gw = pool.download()
    for r, (s, t) in enumerate(((0, 18), (0, 19), (1, 0))):
        at = (int(b.table[s, t // 16]), 0, t % 16)
        assert np.array_equal(gv[at], P.to_bits(x[r], F16)) and gw[at] == 0


def test_attention_of_more_items_than_a_launch():
    """A work list past 2^23 items, whose last ones alone hold work; one tile's
    spans lie on both sides of 2^23."""
    kv, heads, dim, room = 2, 8, 64, (1 << 23) + 3
    pool, b = seeded(241, kv, 16, dim, F16, [1, 20], [900, 20])
    pool.upload(), b.upload()
    rng = np.random.default_rng(242)
    call = P.AttentionCall(pool, b, rng.standard_normal((21, heads, dim), np.float32), heads, 0,
                           items=P.tiled(b, heads, kv, 0, 16, 128))
    assert sum(it.parts > 1 for it in call.items) > 8
    size = C.sizeof(L.PagedItem)
    items = L.DeviceBuffer(room * size)     # those left zero have no rows
    items.upload(np.frombuffer(bytes(call.items), np.uint8), (room - len(call.items)) * size)
    L.check(L.lib().lfm3_paged_attention(
        C.byref(pool.cache), C.byref(b.batch), items.addr, room, call.q.addr, call.q.ld, None,
        heads, call.out.addr, call.out.ld, F32, call.lse.addr, heads, 0, call.ws.addr, call.need,
        None))
    L.synchronize()
    P.check_attention(call, "items")


@pytest.mark.parametrize("budget", [1000, (1 << 28) + 5])
def test_evict_within_bounds_of_many_slots(budget):
    """Bounds (max_length, the budget) far above the lengths: more blocks to move
    slots than a launch has."""
    kv, dim, page, longest = 1, 128, 256, (1 << 28) + 300
    lengths = [1500, 40]
    pool = P.Pool(251, 14, kv, page, dim, F16)
    width = -(-longest // page)
    table, new = (np.full((2, width), 0xFFFFFFFF, np.uint32) for _ in range(2))
    order = np.random.default_rng(252).permutation(14).astype(np.uint32)
    table[0, :6], table[1, 0], new[0, :6], new[1, 0] = order[:6], order[6], order[7:13], order[13]
    pool.upload()
    kept, k, v, w = P.evict(pool, table, lengths, new, min(budget, 1500), 3, 20)
    dt, dn, dl = (L.DeviceBuffer.of(np.asarray(x, np.uint32)) for x in (table, new, lengths))
    out = L.DeviceBuffer(2 * budget * 4)
    need = L.lib().lfm3_paged_evict_workspace_bytes(2, kv, budget, longest)
    ws = L.DeviceBuffer(max(need, 16))
    L.check(L.lib().lfm3_paged_evict(
        C.byref(pool.cache), dt.addr, width, dl.addr, 2, longest, dn.addr, width, budget, 3, 20,
        out.addr, ws.addr, need, None))
    L.synchronize()
    for s in range(2):
        n = len(kept[s][0])
        got = out.download(np.uint32, n + 1, s * budget * 4)
        assert np.array_equal(got[:n], kept[s][0]) and got[n] == 0
    gk, gv, gw = pool.download()
    assert np.array_equal(gk, k) and np.array_equal(gv, v) and np.array_equal(gw, w)
