"""Attention behind shared rows where the table has room for long histories: one long
conversation among short ones is split, as tests/test_shared_plan.py says. Bounds as in
tests/test_gpu_shared_attention.py."""

from __future__ import annotations

import pytest
import torch
from long_batches import generator, shared_batch
from test_gpu_serving import _say
from test_gpu_shared_attention import run_and_check
from test_shared_plan import splits

from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


@pytest.mark.parametrize("batch,kv,d,page,out_dtype", [(40, 8, 64, 64, torch.float32), (70, 8, 64, 16, torch.bfloat16),
                                                       (34, 8, 128, 32, torch.bfloat16), (40, 8, 256, 128, torch.float32)])
def test_one_long_conversation_among_short_ones(batch, kv, d, page, out_dtype):
    _say("shared skew", batch, kv, d, page)
    shared = 130
    lengths = [(shared + 5 * (i % 40), 1) for i in range(batch)]
    lengths[7] = (shared + 12800, 1)
    lengths[9] = (shared + 700, 2)   # a few splits
    lengths[11] = (20, 1)            # some of the shared rows alone
    lengths[12] = (shared, 0)
    b = shared_batch(lengths, shared, kv=kv, d=d, page=page, seed=951, ahead=1, behind=1)
    assert splits(b.tokens, batch, kv, kv, d, page, len(b.table[0]), shared)[0] == 2
    q = torch.randn(b.tokens, kv, d, generator=generator(952)).to(torch.bfloat16)
    run_and_check(b, shared, q, kv, page=page, d=d, out_dtype=out_dtype)
