"""The calls of a decoding step in CUDA graphs, replayed on inputs that were copied in after the capture."""

from __future__ import annotations

from functools import cache

import pytest
import torch

from spalmer_b200 import (
    add_rms_norm,
    add_rms_norm_mxfp8,
    linear_attention_step,
    rotary_embed,
    rotary_frequencies,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _bf16(*shape):
    return torch.randn(shape, device=DEV).to(torch.bfloat16)


@cache
def _frequencies():
    return rotary_frequencies(64, device=DEV)[0]


CALLS = {
    # name: (the call, fresh inputs for it)
    "norm": (lambda x, r, w: add_rms_norm(x, r, w), lambda: (_bf16(5, 768), _bf16(5, 768), _bf16(768))),
    "norm_mxfp8": (lambda x, r, w: add_rms_norm_mxfp8(x, r, w, rows=True),
                   lambda: (_bf16(5, 768), torch.randn(5, 768, device=DEV), _bf16(768))),
    "rotary": (lambda q, k, p: rotary_embed(q, k, p, _frequencies()),
               lambda: (_bf16(48, 12, 64), _bf16(48, 12, 64), torch.randint(0, 8192, (48,), device=DEV))),
    "step": (lambda q, k, v, a, s, at: (linear_attention_step(q, k, v, a, s, slots=at), s),
             lambda: (_bf16(3, 12, 64), _bf16(3, 4, 64), _bf16(3, 4, 64), -torch.rand(3, 12, device=DEV),
                      torch.randn(6, 12, 64, 64, device=DEV), torch.randperm(6, device=DEV)[:3])),
}


@pytest.mark.parametrize("name", CALLS)
def test_graph(name):
    fn, fresh = CALLS[name]
    with torch.no_grad():
        static = fresh()
        fn(*static)  # the library is loaded before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = fn(*static)
        for _ in range(2):
            new = fresh()
            for x, y in zip(static, new):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(got, fn(*new)):
                assert torch.equal(x, y)
