"""Batches over an 8-bit paged cache whose sequences hold the same first pages."""

from __future__ import annotations

from test_gpu_serving import Batch, _filled, _g


def shared_batch(lengths, shared_rows, *, kv, d, page, seed, **places):
    """A ``Batch`` whose parts of the table begin with sequence 0's first
    ``shared_rows // page`` pages; the rows that a sequence sees are numbers."""

    b = Batch(lengths, kv=kv, d=d, page=page, seed=seed, **places)
    whole = shared_rows // page
    pages = b.k_bytes.shape[0]
    front = [at if 0 <= at < pages else 0 for at in b.table[0][:whole]]
    for line in b.table:
        line[:whole] = front
    for at in front:
        for stored in (b.k_bytes[at], b.v_bytes[at]):
            stored[(stored & 0x7f) == 0x7f] = 0x31
    _filled(b, seed + 1)
    b.scales *= 2.0**-3
    return b


def generator(seed):
    return _g(seed)
