"""examples/paged_generate.py: the paged ops together, as a server uses them."""

import os
import sys

import pytest
import torch

import ssa_b200 as ssa

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _model():
    import paged_generate as pg

    torch.manual_seed(0)
    return pg, pg.Decoder(layers=2).cuda()


def test_chunked_serving_equals_the_dense_model():
    pg, model = _model()
    prompts = [torch.randint(0, 512, (n,)) for n in (130, 1, 33)]
    seqs, last, cache = pg.serve(model, prompts, new_tokens=9, chunk=32)
    ssa.check_errors()
    for i, (p, s) in enumerate(zip(prompts, seqs)):
        assert len(s) == len(p) + 9 and s[:len(p)] == p.tolist() and cache.length(i) == len(s) - 1
        with torch.no_grad():
            ref = model.dense(torch.tensor(s[:-1], device="cuda"))
        # fp32 all through: logits of order 10, sums of a few hundred terms
        assert (last[i] - ref[-1]).abs().max() < 1e-3
        assert s[len(p):] == ref[len(p) - 1:].argmax(-1).tolist()


def test_serving_within_a_budget():
    pg, model = _model()
    prompts = [torch.randint(0, 512, (n,)) for n in (200, 20)]
    seqs, last, cache = pg.serve(model, prompts, new_tokens=12, chunk=64, budget=48, recent=8)
    ssa.check_errors()
    assert [len(s) for s in seqs] == [212, 32]
    assert cache.length(0) == 48 and cache.length(1) == 31
    assert all(bool(torch.isfinite(x).all()) for x in last)
