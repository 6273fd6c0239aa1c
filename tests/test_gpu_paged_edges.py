"""The paged cache's operators at the edges of their types and arguments:
probabilities far below the largest. Bounds as in paged_util, or derived beside
the test."""
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
