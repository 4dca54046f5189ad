"""Slot weights of single tokens where the table is much wider than what is filled: the
same weights, and a bounded workspace.  Tolerances as in test_gpu_paged_weights.py."""

import pytest
import torch

import ssa_b200 as ssa
from test_gpu_paged import check_attention, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 96)])
@pytest.mark.parametrize("h_q,h_kv", [(32, 8), (28, 4)])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_with_a_wide_table(dtype, d, h_q, h_kv, causal):
    lens = [300, 70, 1, 0, 2049, 64, 65, 5000]
    c = make(lens, [1, 1, 1, 1, 1, 1, 0, 2], h_q, h_kv, d, 64, dtype, seed=d, weights=True)
    wide = torch.zeros((8, 131072), dtype=torch.int32, device="cuda")         # 8 M slots a row
    wide[:, :c["page_table"].shape[1]] = c["page_table"]
    w0 = c["w"].double()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ssa.paged_attention(c["q"], c["k"], c["v"], wide, c["q_starts"], c["kv_lens"], is_causal=causal,
                              weights=c["w"], return_lse=True)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1.25 * 2 ** 30
    check_attention(c, causal=causal, got=got)
    _, _, _, add = oracle(c, causal=causal)
    assert ((c["w"].double() - w0 - add).abs() <= 3e-5 * add + 2.0 ** -23 * (w0 + add)).all()
    ssa.check_errors()
