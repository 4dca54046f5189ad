"""The paged ops' error words: what the host reads, and when (words in plain memory here;
on the GPU a replayed graph's errors)."""

import types

import pytest
import torch

import ssa_b200 as ssa
from ssa_b200 import _lib as L
from ssa_b200 import _status as S


@pytest.fixture
def words(monkeypatch):
    """Words of device 0 that no GPU writes; notes the waits."""
    waits = []
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    monkeypatch.setattr(torch.cuda, "synchronize", waits.append)
    monkeypatch.setattr(S, "_words", {})
    monkeypatch.setattr(S, "_rings", {})
    monkeypatch.setattr(S, "_ring", lambda dev: types.SimpleNamespace(pending=[]))
    monkeypatch.setattr(S, "workspaces", {})
    monkeypatch.delenv("SSA_CHECKED", raising=False)
    return waits


def test_check_errors_looks_at_words_that_no_call_named_since_the_last_check(words):
    """A replayed graph writes the word that its capture was given."""
    S.host_word(0, 1)
    ssa.check_errors()
    assert words == [0]
    S._words[0].host[1] = L.SSA_DEVICE_BAD_LENGTH           # as a replay would
    with pytest.raises(ValueError, match="paged_attention"):
        ssa.check_errors()
    assert words == [0, 0]
    ssa.check_errors()
    S._words[0].host[0] = L.SSA_DEVICE_BAD_PAGE
    ssa.check_errors(torch.device("cuda", 1))               # another device's
    with pytest.raises(IndexError, match="paged_append"):
        ssa.check_errors(torch.device("cuda", 0))


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 40])
def test_errors_of_a_replayed_graph(q_len):
    from test_gpu_paged import make

    c = make([500, 90], [q_len, q_len], 8, 2, 128, 32, torch.bfloat16, seed=2)
    args = (c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ssa.paged_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ssa.paged_attention(*args)
    graph.replay()
    ssa.check_errors()
    good = out.clone()
    for _ in range(2):
        c["kv_lens"][0] = 10 ** 6                           # past the table: refused on the device
        graph.replay()
        with pytest.raises(ValueError):
            ssa.check_errors()
        c["kv_lens"][0] = 500
        graph.replay()
        ssa.check_errors()
        assert torch.equal(out, good)
