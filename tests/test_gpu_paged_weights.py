"""Slot weights of chunks where their work is cut: many CTAs on the slots of one
item, items of one row tile, sequences without work between others.

Tolerance: a slot's weight is a sum of positive fp32 terms, each off by 1e-6 of
itself, added in up to a few hundred steps of 2^-24: 3e-5 of the sum, and one
rounding where it is added to the weight that was there.
"""

import pytest
import torch

import ssa_b200 as ssa
from test_gpu_paged import make, oracle

pytestmark = pytest.mark.gpu


def _add(c, causal):
    ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], is_causal=causal,
                        weights=c["w"])


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,q_lens,h_q,h_kv", [
    ([200], [3000], 4, 1),                          # one item, a row tile or two for every CTA; rows that see nothing
    ([3000], [3000], 8, 1),                         # the whole triangle of one head
    ([5000], [40], 8, 2),                           # items of one or two row tiles
    ([0, 700, 0, 31, 2049, 0], [9, 257, 40, 31, 130, 0], 14, 2),
    ([300 + 13 * s for s in range(40)], [17 + 5 * s for s in range(40)], 7, 1),
    ([5], [600], 3, 3),
    ([600, 600], [600, 1], 16, 1),
])
def test_weights_of_cut_items(lens, q_lens, h_q, h_kv, causal, dtype, d):
    c = make(lens, q_lens, h_q, h_kv, d, 32, dtype, seed=len(lens), weights=True)
    start = c["w"].clone()
    _add(c, causal)
    once = c["w"].clone()
    _, _, _, add = oracle(c, causal=causal)
    err = (once.double() - start.double() - add).abs()
    assert (err <= 3e-5 * add + 2.0 ** -23 * (start.double() + add)).all(), float((err / (add + 1e-9)).max())
    for _ in range(3):                              # the same bits again, after other lengths in between
        other = make([900], [70], h_q, h_kv, d, 32, dtype, seed=2, weights=True)
        _add(other, causal)
        c["w"].copy_(start)
        _add(c, causal)
        assert torch.equal(c["w"], once)
    ssa.check_errors()
