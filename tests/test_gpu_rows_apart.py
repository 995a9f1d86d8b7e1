"""Query rows that share a wave change no bit of each other's results: what one row's
values make the kernels do (scores beyond what fp32 resolves) is its own."""

from __future__ import annotations

import pytest
import torch
from long_batches import generator, shared_batch
from test_gpu_serving import DEV, _say

from conftest import gpu_available
from nanoquant_amd.runtime import shell_ops as ops

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

LOUD = (1, 2)  # token and q head whose query grows


def others(b, q_heads):
    """The query rows of the batch but the loud one."""
    mine = torch.ones(b.tokens, q_heads, dtype=torch.bool)
    mine[LOUD] = False
    return mine


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,shared,d", [
    ([(300, 3)], 0, 64),                # slots of one sequence's rows
    ([(300, 40), (150, 2)], 0, 128),
    ([(200, 3)], 0, 256),
    ([(400, 1), (390, 1), (450, 2)], 320, 128),  # slots of rows of all sequences
])
def test_attention_beside_a_row_of_huge_scores(lengths, shared, d, q_dtype):
    _say("rows apart", lengths, shared, d, q_dtype)
    b = shared_batch(lengths, shared, kv=1, d=d, page=64, seed=701)
    cache, batch = b.device()
    quiet = torch.randn(b.tokens, 4, d, generator=generator(702))
    loud = quiet.clone()
    loud[LOUD] *= 1e12
    mine = others(b, 4)
    args = {"scaling": d**-0.5, "out_dtype": torch.float32, **batch}

    def run(q):
        lse = torch.empty(b.tokens, 4, device=DEV)
        paged = ops.launch_paged_attention(q.to(q_dtype).to(DEV), cache, **args)
        out = ops.launch_shared_attention(q.to(q_dtype).to(DEV), cache, shared_rows=shared, lse=lse, **args)
        return [x.cpu().view(b.tokens, 4, -1)[mine] for x in (paged, out, lse)]

    for beside, alone in zip(run(loud), run(quiet)):
        assert not torch.isnan(alone).any()
        assert torch.equal(beside, alone)
