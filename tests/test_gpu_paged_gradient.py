"""The paged ops serve: a backward pass through paged_attention raises, and no gradient is
dropped in silence."""

import pytest
import torch

import ssa_b200 as ssa
from test_gpu_paged import make

pytestmark = pytest.mark.gpu


def _case(dtype=torch.bfloat16):
    c = make([300, 40], [60, 1], 8, 2, 64, 16, dtype, seed=1)
    return c["q"], (c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])


@pytest.mark.parametrize("copied", [False, True])           # both argument paths
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_backward_raises(which, copied):
    q, args = _case()
    want, want_lse = ssa.paged_attention(q, *args, return_lse=True)
    if copied:
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    leaf = {"q": q, "k": args[0], "v": args[1]}[which].requires_grad_()
    for result, ref in zip(ssa.paged_attention(q, *args, return_lse=True), (want, want_lse)):
        assert result.requires_grad and torch.equal(result, ref)
        with pytest.raises(RuntimeError, match="no gradient"):
            result.float().nan_to_num().sum().backward()
    out = ssa.paged_attention(q, *args)
    out.mul_(2)                                             # a result like any other
    assert torch.equal(out, 2 * want)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(out.sum(), leaf)
    assert leaf.grad is None


def test_results_without_a_history():
    q, args = _case()
    assert not ssa.paged_attention(q, *args).requires_grad
    q.requires_grad_()
    with torch.no_grad():
        assert not ssa.paged_attention(q, *args).requires_grad
        assert not any(x.requires_grad for x in ssa.paged_attention(q, *args, return_lse=True))
    with torch.inference_mode():
        ssa.paged_attention(q, *args)
    ssa.check_errors()


def test_a_layer_in_front_of_it_learns_of_it():
    """A projection whose output is attended, with gradients on: the loss has a history, and
    asking for the projection's gradient raises."""
    q, args = _case(torch.float32)
    proj = torch.nn.Linear(64, 64, device="cuda")
    loss = ssa.paged_attention(proj(q), *args).square().sum()
    with pytest.raises(RuntimeError, match="no gradient"):
        loss.backward()
    assert proj.weight.grad is None
