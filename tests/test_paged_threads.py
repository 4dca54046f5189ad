"""Threads that share a stream: a call of paged_attention is several launches that hand
partial results through one kept workspace, so no other call may put its launches
between them.  On the CPU with stand-ins for the launches; on the GPU against the
results of one thread."""

import contextlib
import threading
import time
import types

import pytest
import torch

import ssa_b200 as ssa
from ssa_b200 import _lib as L
from ssa_b200 import _status as S
from ssa_b200 import paged as P


class _Launches:
    """Stands in for both argument paths; notes calls that overlap on a workspace."""

    def __init__(self):
        self.busy, self.overlaps, self.calls, self.lock = {}, 0, [], threading.Lock()

    @contextlib.contextmanager
    def on(self, at, kind):
        with self.lock:
            self.calls.append(kind)
            self.overlaps += self.busy.get(at, 0)
            self.busy[at] = self.busy.get(at, 0) + 1
        yield time.sleep(0.05)                       # the interpreter is free, as in a ctypes call
        with self.lock:
            self.busy[at] -= 1

    def attend(self, q, *args):                      # the extension module: takes contiguous queries
        if not q.is_contiguous():
            return None
        with self.on(args[-1].data_ptr(), "module"):
            return 0, q, None

    def ssa_paged_attn_workspace_size(self, c, a):
        return 32768

    def ssa_paged_attn(self, c, a, ws, nbytes, stream):
        with self.on(ws, "ctypes"):
            return 0
    ssa_paged_attn.__name__ = "ssa_paged_attn"


@pytest.fixture
def launches(monkeypatch):
    fake = _Launches()
    fake.append = fake.evict = None
    monkeypatch.setattr(L, "_lib", fake)
    monkeypatch.setattr(L, "_call", fake)
    monkeypatch.setattr(S, "workspaces", {})
    monkeypatch.setattr(S, "host_word", lambda key, op: (None, False))
    monkeypatch.setattr(P, "_raw_stream", lambda key: 7)
    monkeypatch.setattr(P, "_cache_args", lambda *a: (0, types.SimpleNamespace(batch=1, h_kv=2, d=64), False, ()))
    for name in ("_check_rows", "_index"):
        monkeypatch.setattr(P, name, lambda t, *a: t)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda key: contextlib.nullcontext())
    return fake


def _attend(q):
    pages = types.SimpleNamespace(is_cuda=True, get_device=lambda: 0, dtype=q.dtype, requires_grad=False)
    starts = torch.zeros(2, dtype=torch.int32)
    return ssa.paged_attention(q, pages, pages, starts, starts, starts)


def test_calls_of_two_threads_do_not_overlap_on_a_workspace(launches):
    plain = torch.zeros((5, 4, 64))
    copied = torch.zeros((4, 5, 64)).transpose(0, 1)
    _attend(plain)                                   # the stream's workspace
    launches.calls.clear()
    threads = [threading.Thread(target=lambda q=q: [_attend(q) for _ in range(4)]) for q in (plain, copied, copied)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert launches.calls.count("module") == 4 and launches.calls.count("ctypes") == 8
    assert launches.overlaps == 0


def test_a_workspace_is_handed_out_zeroed(launches, monkeypatch):
    """Another thread may take it as soon as it is kept."""
    seen = []

    class _Kept(dict):
        def __setitem__(self, at, kept):
            seen.append(bool(getattr(kept, "buffer", kept)[:L.SSA_PAGED_ZEROED].any()))
            super().__setitem__(at, kept)

    monkeypatch.setattr(S, "workspaces", _Kept())
    like = types.SimpleNamespace(new_empty=lambda shape, dtype: torch.full(shape, 7, dtype=dtype))
    P._workspace(0, 32768, like)
    P._workspace(0, 65536, like)
    assert seen == [False, False]


def test_a_workspace_dropped_by_an_errors_look_up_is_not_used(launches, monkeypatch):
    """A timeout leaves the head of a workspace undefined: the call that learns of it takes
    another one."""
    plain = torch.zeros((5, 4, 64))
    _attend(plain)
    old = S.workspaces[0, 7].buffer
    launches.calls.clear()
    monkeypatch.setattr(S, "host_word", lambda key, op: (S.workspaces.clear(), (None, False))[1])
    used = []
    monkeypatch.setattr(launches, "attend", lambda *args: used.append(args[-1]) and None)
    _attend(plain)
    assert not any(u is old for u in used) and S.workspaces[0, 7].buffer is not old


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [70, 300, 5]])
@pytest.mark.parametrize("weighted", [False, True])
def test_two_threads_on_one_stream(dtype, d, q_lens, weighted):
    from test_gpu_paged import make

    lens = [900, 700, 2000]
    sets = [make(lens, q_lens, 8, 2, d, 32, dtype, seed=s, weights=True) for s in (1, 2)]
    q = [sets[0]["q"], sets[1]["q"].transpose(1, 2).contiguous().transpose(1, 2)]     # the second needs a copy
    assert q[1].stride(2) != 1

    def attend(i):
        c = sets[i]
        w = c["w"].clone() if weighted else None
        out, lse = ssa.paged_attention(q[i], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], weights=w,
                                       return_lse=True)
        return (out, lse) + ((w,) if weighted else ())

    want = [attend(0), attend(1)]
    wrong, raised = [0, 0], []

    def work(i):
        try:
            for _ in range(40):
                wrong[i] += not all(torch.equal(a, b) for a, b in zip(attend(i), want[i]))
        except Exception as e:                       # noqa: BLE001 - reported below
            raised.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not raised and wrong == [0, 0]
    ssa.check_errors()
