"""The decoder with a 4-bit output projection: logits are the final norm's rows times
the matrix that the 4 bits stand for, greedy tokens their largest, with and without graphs."""

from __future__ import annotations

import pytest
import torch
from test_gpu_int4 import check
from test_gpu_serving import DEV, SMALL, _check_logprobs, _g

from conftest import gpu_available
from nanoquant_amd import synthetic as syn
from nanoquant_amd.runtime import shell_ops as ops
from nanoquant_amd.runtime.decoder_shell import DecoderShellError, PackedDecoder, dense_tensors

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]


def decoder_with(group, act=torch.float32, cache=torch.bfloat16):
    weights = syn.synthetic_decoder(SMALL, seed=syn.BASE_SEED + 91, random_norms=True)
    weights.lm_head = ops.int4_matrix(weights.lm_head.to(DEV), group)
    return weights, PackedDecoder(SMALL, weights, device=DEV, max_positions=300, activation_dtype=act, cache_dtype=cache)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn])
def test_logits_tokens_and_graphs(group, cache):
    weights, decoder = decoder_with(group, cache=cache)
    prompt = torch.randint(0, SMALL.vocab, (60,), generator=_g(601)).to(DEV)
    logits = decoder.prefill(prompt).clone()
    _, buffers = decoder._prefill(prompt, 0)
    head = ops.Int4Matrix(*(None if t is None else t.cpu() for t in weights.lm_head))
    check(logits[None], buffers.final[59:60].cpu(), head, group)
    eager = decoder.generate_greedy(prompt, 21, use_graph=False).tolist()
    assert eager[0] == int(logits.argmax())
    assert decoder.generate_greedy(prompt, 21).tolist() == eager
    tokens, scores = decoder.generate_greedy_scored(prompt, 21, top=3)
    assert tokens.tolist() == eager
    assert torch.equal(scores.top_ids[:, 0], tokens)


def test_a_text_is_scored_by_its_rows_logits():
    _, decoder = decoder_with(64)
    ids = torch.randint(0, SMALL.vocab, (290,), generator=_g(602))
    got = decoder.score(ids, top=5)
    assert torch.equal(decoder.logits, decoder.prefill(ids))
    _, buffers = decoder._prefill(ids, 0)
    logits = torch.cat([ops.launch_int4_projection(buffers.final[:256], decoder.lm_head),
                        ops.launch_int4_projection(buffers.final[256:289], decoder.lm_head)])
    _check_logprobs(got, logits, ids[1:], 5)
    for row in (0, 100, 288):  # rows alone: the same but for the order of a few fp32 sums
        one = ops.launch_int4_projection(buffers.final[row:row + 1], decoder.lm_head)
        assert torch.allclose(one[0], logits[row], rtol=1e-5, atol=1e-5 * float(logits[row].abs().max()))


def test_a_matrix_of_another_shape_is_refused():
    weights, _ = decoder_with(64)
    with pytest.raises(DecoderShellError, match="dense"):
        dense_tensors(weights)
    weights.lm_head = ops.int4_matrix(torch.randn(SMALL.vocab - 1, SMALL.hidden, device=DEV))
    with pytest.raises(DecoderShellError, match="lm_head"):
        PackedDecoder(SMALL, weights, device=DEV)
