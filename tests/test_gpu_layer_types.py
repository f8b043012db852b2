"""DynamicLinearAttention in 16 bits: whole sequences, pieces and single tokens of one another, and of float64.

A layer's value passes through about eight roundings to the type (projections, convolutions, scores, states, o, norm, gate),
each of at most u of a value and independent of the others, and sums of many terms between them, so that the outputs' error
has a standard deviation of about 2 u of their own (u = 2^-8, 2^-11).  The largest of a few thousand is within 5 of them,
and the largest output is over 3 deviations of the outputs: 16 u of it leaves room for four times that."""

import pytest
import torch

from helpers import gen, max_rel, randn
from test_gpu_layer import _layer, _ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
TOL = {BF: 16 * 2.0**-8, HF: 16 * 2.0**-11}


@pytest.mark.parametrize("W", [4, 1])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_prompt_pieces_and_tokens(dtype, W):
    m = _layer(W=W, dtype=dtype)
    B, T = 3, 140
    x = randn(gen(2), B, T, 128).to(dtype)
    ref, S = _ref(m, x.double())
    x = x.to(DEV)
    with torch.no_grad():
        whole, last = m(x, return_state=True)
        a, state = m(x[:, :2], return_state=True)
        b, state = m(x[:, 2:100], state=state, return_state=True)
        parts = [a, b] + [m.step(x[:, t], state)[:, None] for t in range(100, T)]
    assert whole.dtype == dtype and state.conv.dtype == dtype and state.attn.dtype == torch.float32
    assert max_rel(whole, ref) < TOL[dtype] and max_rel(torch.cat(parts, 1), ref) < TOL[dtype]
    assert max_rel(last.attn, S) < TOL[dtype] and max_rel(state.attn, S) < TOL[dtype]
    assert torch.equal(last.conv, state.conv)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_tokens_from_a_cache(dtype):
    """Single tokens of some of a cache's sequences, from nothing, and rows of others left alone."""
    m = _layer(dtype=dtype)
    x = randn(gen(5), 2, 20, 128).to(dtype)
    ref, S = _ref(m, x.double())
    cache = m.new_state(5)
    cache.attn[[0, 2, 3]] = 7.0
    slots = torch.tensor([4, -1, 1], dtype=torch.int32, device=DEV)
    rows = []
    for t in range(20):
        token = torch.stack([x[0, t], torch.full((128,), float("nan"), dtype=dtype), x[1, t]]).to(DEV)
        rows.append(m.step(token, cache, slots=slots)[[0, 2]])
    assert max_rel(torch.stack(rows, 1), ref) < TOL[dtype] and max_rel(cache.attn[[4, 1]], S) < TOL[dtype]
    assert (cache.attn[[0, 2, 3]] == 7).all() and (cache.conv[[0, 2, 3]] == 0).all()
