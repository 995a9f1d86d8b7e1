"""Query rows that share a wave change no bit of each other's results: what one row's
values make the kernels do (scores or log-sum-exps beyond what fp32 resolves) is its own."""

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


@pytest.mark.parametrize("q_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,d", [([(300, 2)], 128), ([(300, 12)], 64), ([(100, 80)], 128), ([(100, 80)], 256)])
def test_attention_weights_beside_a_row_of_a_huge_lse(lengths, d, q_dtype):
    """The held-back weights of a row beyond fp32's reach are its own: the others', which a log-sum-exp
    below theirs brings above 1, stay what they are. All that the loud row itself adds is 0."""

    _say("weights apart", lengths, d, q_dtype)
    b = shared_batch(lengths, 0, kv=1, d=d, page=64, seed=711)
    cache, batch = b.device()
    q = torch.randn(b.tokens, 4, d, generator=generator(712)).to(q_dtype).to(DEV)
    lse = torch.empty(b.tokens, 4, device=DEV)
    ops.launch_shared_attention(q, cache, shared_rows=0, scaling=d**-0.5, lse=lse, **batch)
    lse -= 20.0  # every row's weights sum to e^20
    none = torch.zeros(b.k_bytes.shape[0], 1, 64, device=DEV)

    def run(of):
        quiet = lse.clone()
        quiet[LOUD] = of
        return ops.launch_attention_weights(q, cache, quiet, none, scaling=d**-0.5, out=torch.zeros_like(none), **batch)

    alone, beside = run(500.0), run(1e6)  # e^(s - 500) and e^(s - 10^6) are 0
    assert float(alone.max()) > 4.0 * b.tokens
    assert torch.equal(beside, alone)
