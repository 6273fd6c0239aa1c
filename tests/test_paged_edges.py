"""CPU checks of the paged cache's entry points at the limits of their sizes. No
kernel runs here."""
import ctypes as C

import pytest

import lfm3amd as L


@pytest.mark.parametrize("seqs,kv,length", [(64, 16, 1 << 30), (65535, 16, 1 << 30),
                                            (2, 1023, 1 << 30), (64, 1023, 1 << 25)])
def test_weights_refuse_more_slots_than_their_units_count(seqs, kv, length):
    """Sequences of mostly absent pages may be long; 64 of them times the KV heads
    have to stay within 2^31 units of 512 slots."""
    assert min(seqs, 64) * kv * length // 512 > 0x7FFFFFFF
    a = 0x10000
    cache = L.PagedCache(a, a, a, L.TYPE_F16, 4, 256, kv, 64)
    batch = L.PagedBatch(a, 1 << 22, a, a, a, seqs, 1)
    assert L.lib().lfm3_paged_weights(C.byref(cache), C.byref(batch), a, kv * 64, L.TYPE_F32, a,
                                      kv, 0, length, None) == L.E_INVALID
    assert b"too many slots" in L.lib().lfm3_last_error()
