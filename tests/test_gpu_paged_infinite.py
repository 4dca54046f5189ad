"""Infinite and NaN values that rows see: the paged attention gives what the formula
gives -- the same infinities, NaN where it has NaN, and its tolerance elsewhere."""

import math

import pytest
import torch

import ssa_b200 as ssa
from test_gpu_paged import U, make, oracle, slots

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64), (torch.float32, 64),
         (torch.bfloat16, 96)]


def _check(c, causal=True):
    out = ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], is_causal=causal)
    ref, amp, _, _ = oracle(c, causal=causal)
    for same in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(same(out), same(ref)), same.__name__
    fine = torch.isfinite(ref)
    u = U[out.dtype]
    assert ((out.double() - ref).abs() <= u * ref.abs() + (u + 2e-5) * amp + 1e-7)[fine].all()
    return out


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("q_len", [1, 3, 200])
@pytest.mark.parametrize("sharp", [1.0, 5.0])
def test_infinite_values(dtype, d, q_len, sharp):
    """Weights down to some 2^-60 of a row's largest: of every infinite value a part, and no
    NaN but where infinities of both signs or a NaN are seen."""
    c = make([700, 320], [q_len, 1], 8, 2, d, 32, dtype, seed=d, weights=True)
    c["q"].mul_(sharp)
    pg, sl = slots(c, 0, 700)
    v = c["v"]
    v[pg[5], sl[5], 0, 3] = math.inf               # a tile that every row sees
    v[pg[70], sl[70], 0, 4] = -math.inf
    v[pg[200], sl[200], 0, 5] = math.nan
    v[pg[6], sl[6], 0, 6] = math.inf
    v[pg[300], sl[300], 0, 6] = -math.inf
    v[pg[699], sl[699], 1, 7] = math.inf           # the last row alone sees it
    v[pg[3], sl[3], 1, 7] = math.inf
    pg, sl = slots(c, 1, 320)
    v[pg[:], sl[:], 1, 0] = -math.inf
    out = _check(c)
    assert torch.isposinf(out[:q_len, :4, 3]).all() and torch.isneginf(out[:q_len, :4, 4]).all()
    assert torch.isnan(out[:q_len, :4, 5:7]).all() and torch.isneginf(out[-1, 4:, 0]).all()
    _check(c, causal=False)
    ssa.check_errors()


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("h_q,h_kv", [(28, 4), (3, 1), (13, 1), (8, 2)])
@pytest.mark.parametrize("q_lens", [[200, 1], [1, 1], [300, 129]])
def test_slot_weights_beside_an_infinite_key(dtype, d, h_q, h_kv, q_lens):
    """A key with an infinite entry that every query meets with the other sign: its weight is
    0 in every row, and all else stays finite."""
    c = make([700, 320], q_lens, h_q, h_kv, d, 32, dtype, seed=d + h_q, weights=True)
    c["q"][..., 3] = -c["q"][..., 3].abs() - 0.25
    pg, sl = slots(c, 0, 700)
    for at in (5, 130, 380):                       # tiles that every row sees
        c["k"][pg[at], sl[at], 0, 3] = math.inf
    w0 = c["w"].double()
    ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], weights=c["w"])
    _, _, _, add = oracle(c)
    assert bool(torch.isfinite(add).all()) and not add[pg[5], sl[5], 0].any()
    err = (c["w"].double() - w0 - add).abs()
    assert (err <= 3e-5 * add + 2.0 ** -23 * (w0 + add)).all()
    _check(c)
    ssa.check_errors()


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("fill", [math.nan, math.inf])
def test_many_items_with_infinite_values_past_their_lengths(dtype, d, fill):
    """Several items on every CTA: tiles that hold such values, hidden, and tiles without them
    take turns."""
    lens = [130 + 37 * s % 500 for s in range(48)]
    c = make(lens, [1 + 11 * s % 40 for s in range(48)], 8, 8, d, 64, dtype, seed=d, fill=fill)
    _check(c)
    _check(c, causal=False)
    ssa.check_errors()
