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


BITS = [L.SSA_DEVICE_BAD_PAGE, L.SSA_DEVICE_BAD_LENGTH, L.SSA_DEVICE_TIMEOUT]


def test_kinds_of_errors_have_a_byte_each():
    """The kernels store a kind's byte alone, so that none hides another."""
    at = [(b.bit_length() - 1) // 8 for b in BITS]
    assert len(set(at)) == len(BITS) and all(b & (b - 1) == 0 for b in BITS)


def _store(word, bits):
    """What a kernel does: one byte of the word."""
    at = (bits.bit_length() - 1) // 8
    word.view(torch.uint8)[at] = bits >> 8 * at


@pytest.mark.parametrize("first", BITS)
@pytest.mark.parametrize("second", BITS)
def test_a_timeout_drops_the_workspaces_whatever_else_is_found(words, first, second):
    S.host_word(0, 1)
    S.workspaces[0, 7] = S.Workspace(torch.zeros(1))
    word = S._words[0].host[1:2]
    _store(word, first)
    _store(word, second)
    with pytest.raises((IndexError, ValueError, RuntimeError)) as e:
        S.host_word(0, 0)
    timed_out = L.SSA_DEVICE_TIMEOUT in (first, second)
    assert (not S.workspaces) == timed_out and ("timed out" in str(e.value)) == timed_out
    seen = 1
    while True:                                    # each kind is raised once
        try:
            S.host_word(0, 0)
            break
        except (IndexError, ValueError, RuntimeError):
            seen += 1
    assert seen == len({first, second}) and not word.any()


def test_timeouts_count_without_checks_too(words, monkeypatch):
    monkeypatch.setenv("SSA_CHECKED", "0")
    address, sync = S.host_word(0, 1)
    assert address and not sync                    # a word all the same
    S.workspaces[0, 7] = S.Workspace(torch.zeros(1))
    base = S._words[0].host.data_ptr()
    word = S._words[0].host[(address - base) // 4:][:1]
    _store(word, L.SSA_DEVICE_BAD_PAGE)
    S.host_word(0, 1)
    assert S.workspaces                            # no error is raised, and nothing else happens
    _store(word, L.SSA_DEVICE_TIMEOUT)
    S.host_word(0, 1)
    assert not S.workspaces and not word.any()
    monkeypatch.delenv("SSA_CHECKED")
    _store(word, L.SSA_DEVICE_BAD_LENGTH)          # a call made without checks is not reported later
    S.host_word(0, 0)
    ssa.check_errors()


@pytest.mark.gpu
def test_a_bad_page_and_a_bad_length_of_one_call_are_both_reported():
    from test_gpu_paged import make

    c = make([100, 64], [2, 1], 4, 2, 64, 16, torch.bfloat16, seed=1)
    c["page_table"][1, 0] = -1
    c["kv_lens"][0] = 10 ** 6
    ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    found = set()
    for _ in range(2):
        with pytest.raises((IndexError, ValueError)) as e:
            ssa.check_errors()
        found.add(e.type)
    assert found == {IndexError, ValueError}
    ssa.check_errors()
