"""The argument path of the paged ops: the extension module takes the plain calls
and leaves every other to the Python code, and both make the same call."""

import pytest
import torch

import ssa_b200 as ssa
from ssa_b200 import _lib as L
from ssa_b200 import paged as P
from ssa_b200.build import build


class _Nothing:
    """Stands in for the extension module: takes no call."""

    def __init__(self):
        self.asked = 0

    def _none(self, *args):
        self.asked += 1

    append = attend = evict = _none


def _tensors(device, dtype=torch.bfloat16, d=64):
    g = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=g).to(dtype).to(device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return dict(q=rand(5, 4, d), k_new=rand(5, 2, d), v_new=rand(5, 2, d), k=rand(8, 16, 2, d), v=rand(8, 16, 2, d),
                w=torch.rand((8, 16, 2), generator=g).to(device), table=i32([[3, 1, 7], [0, 5, 2]]), starts=i32([0, 2, 5]),
                lens=i32([33, 20]), new=i32([[4], [6]]))


def test_the_module_leaves_cpu_tensors_and_wrong_counts_to_python():
    build()
    call, t = L.paged_call(), _tensors("cpu")
    assert call.append(t["k_new"], t["v_new"], t["k"], t["v"], t["table"], t["starts"], t["lens"], None, None) is None
    assert call.attend(t["q"], t["k"], t["v"], t["table"], t["starts"], t["lens"], None, True, None, False, None,
                       t["w"]) is None
    assert call.evict(t["k"], t["v"], t["w"], t["table"], t["lens"], t["new"], 16, 0, None) is None
    assert call.append() is None and call.attend(1, 2) is None and call.evict(None) is None
    assert call.append(*[None] * 9) is None and call.attend(*["x"] * 12) is None
    with pytest.raises(TypeError):
        call.bind(1)


def _run(t):
    args = t["k"], t["v"], t["table"]
    assert ssa.paged_append(t["k_new"], t["v_new"], *args, t["starts"], t["lens"], t["w"]) is None
    out = [ssa.paged_attention(t["q"], *args, t["starts"], t["lens"]),
           *ssa.paged_attention(t["q"], *args, t["starts"], t["lens"], 3, False, t["w"], True)]
    return out + list(ssa.paged_evict(t["k"], t["v"], t["w"], t["table"], t["lens"], t["new"], 16, 4)) + [
        t["k"].clone(), t["v"].clone(), t["w"].clone()]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_both_paths_make_the_same_call(monkeypatch, dtype):
    _run(_tensors("cuda", dtype))                   # the stream's workspace
    with monkeypatch.context() as m:                # the Python path alone
        none = _Nothing()
        m.setattr(L, "_call", none)
        want = _run(_tensors("cuda", dtype))
        assert none.asked == 4
    with monkeypatch.context() as m:                # the module alone
        def refuse(*a):
            raise AssertionError("a plain call reached the Python path")
        m.setattr(P, "_cache_args", refuse)
        got = _run(_tensors("cuda", dtype))
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)
    ssa.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("name,change", [
    ("starts", lambda x: x.repeat_interleave(2)[::2]),
    ("lens", lambda x: x.repeat_interleave(2)[::2]),
    ("table", lambda x: x.t().contiguous().t()),
    ("q", lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)),
    ("k_new", lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)),
    ("new", lambda x: x.repeat(1, 2).t().contiguous().t()),
])
def test_tensors_that_need_a_copy_still_work(name, change):
    want = _run(_tensors("cuda"))
    t = _tensors("cuda")
    t[name] = change(t[name])
    for a, b in zip(_run(t), want):
        assert torch.equal(a, b)
    ssa.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("name,change", [
    ("starts", lambda x: x.long()), ("lens", lambda x: x.float()), ("table", lambda x: x[:1]), ("table", lambda x: x.cpu()),
    ("k", lambda x: x.half()), ("k", lambda x: x[0]), ("v", lambda x: x[:, :8]), ("q", lambda x: x.cpu()),
    ("q", lambda x: x[:, :3]), ("q", lambda x: x[..., :32]), ("k_new", lambda x: x.float()), ("v_new", lambda x: x[:4]),
    ("w", lambda x: x.double()), ("w", lambda x: x[:, :8]), ("new", lambda x: x.long()), ("new", lambda x: x[:1]),
    ("starts", lambda x: x[:2]),
])
def test_what_the_module_refuses_is_named_by_python(name, change):
    t = _tensors("cuda")
    _run(_tensors("cuda"))
    before = {k: v.clone() for k, v in t.items()}
    t[name] = change(t[name])
    args = t["k"], t["v"], t["table"]
    calls = [lambda: ssa.paged_append(t["k_new"], t["v_new"], *args, t["starts"], t["lens"], t["w"]),
             lambda: ssa.paged_attention(t["q"], *args, t["starts"], t["lens"], weights=t["w"]),
             lambda: ssa.paged_evict(t["k"], t["v"], t["w"], t["table"], t["lens"], t["new"], 16, 4)]
    uses = {"q": [1], "k_new": [0], "v_new": [0], "starts": [0, 1], "new": [2]}.get(name, [0, 1, 2])
    for i in uses:
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            calls[i]()
    for k in ("k", "v", "w"):
        if k != name:
            assert torch.equal(t[k], before[k])


@pytest.mark.gpu
def test_a_cache_without_heads_is_refused():
    t = _tensors("cuda")
    with pytest.raises(ValueError):
        ssa.paged_attention(t["q"], t["k"][:, :, :0], t["v"][:, :, :0], t["table"], t["starts"], t["lens"])
