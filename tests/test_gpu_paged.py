"""The paged key/value cache (ssa_b200.paged) on the GPU against its formulas in
64 bits.

Attention tolerance, elementwise, with u the largest relative error of one
rounding to the tensors' type (bf16 2^-8, fp16 2^-11, fp32 2^-24): the output is
rounded once (u |ref|), and the weights of the product with the values may be
held in that type too, each off by at most u, which moves the output by at most
u A with A = sum_j softmax_ij |v_j|.  What is left is fp32 arithmetic: a logit
is a sum of d products, off by a few 2^-24 sum_x |q_x k_x| / scale (about 7 for
normal vectors of d = 128), so a softmax weight is off by some 1e-6 of itself;
2e-5 A is allowed.  Slot weights are fp32 sums of such weights: 3e-5 relative.
"""

import math

import pytest
import torch

import ssa_b200 as ssa
from ssa_b200 import _lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make(lens, q_lens, h_q, h_kv, d, page, dtype, layout="hnd", seed=0, spare=3, weights=False, fill=None):
    """A cache holding ``lens`` slots per sequence in randomly placed pages."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.zeros((len(lens), max(max(need), 1)), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n

    def paged(*tail, dt):
        if layout == "hnd":
            return torch.empty((pages, h_kv, page) + tail, dtype=dt, device=DEV).transpose(1, 2)
        return torch.empty((pages, page, h_kv) + tail, dtype=dt, device=DEV)

    c = dict(page=page, lens=list(lens), q_lens=list(q_lens), table=table, h_kv=h_kv, h_q=h_q, d=d)
    for name in ("k", "v"):
        t = paged(d, dt=dtype)
        t.copy_(torch.randn((pages, page, h_kv, d), generator=g))
        if fill is not None:                       # what the slots past a length hold
            used = torch.zeros((pages, page), dtype=torch.bool)
            for s, n in enumerate(lens):
                j = torch.arange(n)
                used[table[s][j // page].long(), j % page] = True
            t[~used.to(DEV)] = fill
        c[name] = t
    c["w"] = None
    if weights:
        c["w"] = paged(dt=torch.float32)
        c["w"].copy_(torch.rand((pages, page, h_kv), generator=g))
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    c["starts"] = starts
    c["q"] = torch.randn((starts[-1], h_q, d), generator=g).to(DEV, dtype)
    c["page_table"] = table.to(DEV)
    c["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    c["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return c


def slots(c, s, n, table=None):
    j = torch.arange(n)
    t = c["table"] if table is None else table
    return t[s][j // c["page"]].long().to(DEV), (j % c["page"]).to(DEV)


def oracle(c, scale=None, causal=True):
    """(out, A, lse, added slot weights) in 64 bits; A is the tolerance's factor."""
    scale = scale or math.sqrt(c["d"])
    g = c["h_q"] // c["h_kv"]
    T = c["starts"][-1]
    out = torch.zeros((T, c["h_q"], c["d"]), dtype=torch.float64, device=DEV)
    amp = torch.zeros_like(out)
    lse = torch.full((T, c["h_q"]), -math.inf, dtype=torch.float64, device=DEV)
    add = torch.zeros(c["k"].shape[:3], dtype=torch.float64, device=DEV)
    for s, (n, L_) in enumerate(zip(c["q_lens"], c["lens"])):
        if n == 0 or L_ == 0:
            continue
        pg, sl = slots(c, s, L_)
        r = slice(c["starts"][s], c["starts"][s + 1])
        lim = torch.arange(L_ - n, L_, device=DEV)[:, None] if causal else torch.full((n, 1), L_, device=DEV)
        hide = torch.arange(L_, device=DEV)[None] > lim
        for e in range(c["h_q"]):
            k, v = c["k"][pg, sl, e // g].double(), c["v"][pg, sl, e // g].double()
            x = (c["q"][r, e].double() @ k.T / scale).masked_fill(hide, -math.inf)
            z = torch.logsumexp(x, 1)
            p = torch.where(hide, 0.0, torch.exp(x - z[:, None]))
            # a hidden slot's value takes no part, whatever it holds
            for i in range(n) if not torch.isfinite(v).all() else ():
                see = ~hide[i]
                out[r.start + i, e] = p[i, see] @ v[see]
                amp[r.start + i, e] = p[i, see] @ v[see].abs()
            if torch.isfinite(v).all():
                out[r, e], amp[r, e] = p @ v, p @ v.abs()
            lse[r, e] = z
            add[pg, sl, e // g] += p.sum(0)
    return out, amp, lse, add


def check_attention(c, scale=None, causal=True, got=None):
    out, lse = got or ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"],
                                          scale=scale, is_causal=causal, return_lse=True)
    ref, amp, ref_lse, _ = oracle(c, scale, causal)
    assert out.dtype == c["q"].dtype and out.shape == c["q"].shape and lse.dtype == torch.float32
    u = U[out.dtype]
    err = (out.double() - ref).abs()
    tol = u * ref.abs() + (u + 2e-5) * amp + 1e-7
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} elements off, worst {float((err / tol)[bad].max()):.3g} x the tolerance"
    seen = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse), seen) and bool((lse[~seen] == -math.inf).all())
    assert ((lse.double() - ref_lse)[seen].abs() <= 1e-5 + 1e-6 * ref_lse[seen].abs()).all()
    assert not out[~seen].any()
    return out, lse


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,q_lens,h_q,h_kv,d,page,layout", [
    ([1], [1], 8, 2, 64, 16, "hnd"),                                   # one token, nothing before it
    ([1000], [1], 32, 8, 128, 64, "hnd"),                              # one token
    ([5, 700, 64, 63, 65, 128, 1], [1] * 7, 28, 4, 128, 64, "hnd"),    # tokens of seven sequences, g = 7
    ([2049, 17], [1, 1], 8, 8, 64, 32, "nhd"),                         # no head sharing
    ([300], [300], 8, 2, 64, 16, "nhd"),                               # a whole prompt
    ([777], [130], 16, 1, 128, 16, "hnd"),                             # a group of 16
    ([513, 200, 1, 0, 90], [513, 3, 1, 0, 0], 4, 2, 64, 128, "hnd"),   # empty chunk, empty sequence
    ([40, 7], [50, 9], 4, 2, 64, 16, "nhd"),                           # rows before slot 0 see nothing
    ([260, 129], [33, 70], 6, 2, 96, 24, "hnd"),                       # odd head size and page
    ([50, 3], [20, 2], 3, 3, 8, 1, "nhd"),                             # smallest head, pages of one slot
    ([400], [65], 8, 1, 256, 100, "nhd"),                              # largest head
    ([1100, 1023, 1025], [255, 256, 257], 8, 2, 128, 256, "hnd"),      # tile edges
    ([4000], [9], 14, 2, 128, 1024, "nhd"),                            # few rows, long context, large pages
])
def test_attention_matches_formula(lens, q_lens, h_q, h_kv, d, page, layout, dtype):
    check_attention(make(lens, q_lens, h_q, h_kv, d, page, dtype, layout, seed=len(lens) + d))


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 200, 5]])
def test_attention_without_causal_mask_and_with_a_scale(dtype, d, q_lens):
    c = make([90, 333, 5], q_lens, 8, 2, d, 32, dtype, seed=4)
    check_attention(c, scale=3.0, causal=False)
    check_attention(c, scale=0.5, causal=True)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64),
                                     (torch.bfloat16, 96)])
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [60, 200, 5]])
def test_what_lies_past_a_length_takes_no_part(dtype, d, fill, q_lens):
    check_attention(make([70, 391, 5], q_lens, 8, 2, d, 64, dtype, seed=2, fill=fill))


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_later_rows_infinite_value_does_not_reach_earlier_rows(dtype, d, bad):
    c = make([300], [200], 8, 2, d, 32, dtype, seed=3)
    pg, sl = slots(c, 0, 300)
    at = 250                                       # seen by rows 150 .. 199
    c["v"][pg[at], sl[at], 1, 5] = bad
    c["k"][pg[at + 20], sl[at + 20], 0, 3] = math.nan
    out = ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    ref, amp, _, _ = oracle(c)
    fine = torch.isfinite(ref)
    # hidden: every row before, and every other column of the rows that see it
    assert fine[:150].all() and not fine[150:, 4:, 5].any() and not fine[170:, :4].any()
    assert torch.equal(torch.isfinite(out), fine)
    u = U[dtype]
    assert ((out.double() - ref).abs() <= u * ref.abs() + (u + 2e-5) * amp + 1e-7)[fine].all()


def test_large_logits_stay_finite():
    for dtype, d in ((torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 64)):
        for q_lens in ([1, 1], [100, 300]):
            c = make([200, 301], q_lens, 8, 2, d, 16, dtype, seed=6)
            c["q"].mul_(30.0)
            out, lse = ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"],
                                           return_lse=True)
            ref, amp, ref_lse, _ = oracle(c)
            assert torch.isfinite(out).all()
            # logits of some hundreds: their fp32 error (4e-7 of 30 * 7) reaches 1e-4
            assert ((lse.double() - ref_lse).abs() <= 2e-4 + 1e-6 * ref_lse.abs()).all()
            u = U[dtype]
            assert ((out.double() - ref).abs() <= u * ref.abs() + (u + 1e-3) * amp + 1e-7).all()


def test_strided_queries_and_pages():
    c = make([400, 33], [50, 1], 8, 2, 128, 16, torch.bfloat16, seed=9)
    wide = torch.randn((51, 12, 136), device=DEV).to(torch.bfloat16)
    wide[:, 2:10, :128] = c["q"]
    c["q"] = wide[:, 2:10, :128]
    both = torch.empty((c["k"].shape[0], 2, 16, 2, 128), dtype=torch.bfloat16, device=DEV)   # K and V interleaved
    both[:, 0], both[:, 1] = c["k"], c["v"]
    c["k"], c["v"] = both[:, 0], both[:, 1]
    check_attention(c)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, its used pages at the end."""
    page, h_kv, d = 64, 2, 128
    pages = (2 ** 31) // (page * h_kv * d) + 40
    for q_lens in ([1], [150]):
        c = make([900], q_lens, 8, h_kv, d, page, torch.bfloat16, seed=1, spare=0, weights=True)
        big = {}
        for name in ("k", "v"):
            big[name] = torch.zeros((pages, page, h_kv, d), dtype=torch.bfloat16, device=DEV)
            big[name][pages - 15:] = c[name]
        wbig = torch.zeros((pages, page, h_kv), device=DEV)
        wbig[pages - 15:] = c["w"]
        c.update(big)
        c["table"] = c["table"] + pages - 15
        c["page_table"] = c["table"].to(DEV)
        check_attention(c)
        _, _, _, add = oracle({**c, "k": c["k"], "v": c["v"]})
        before = wbig.clone()
        ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], weights=wbig)
        assert ((wbig - before).double() - add).abs().max() <= 3e-5 * add.max() + 1e-6
        del big, add
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 64)])
def test_results_do_not_depend_on_the_rest_of_the_batch_or_the_run(dtype, d):
    c = make([1500, 40, 700], [1, 1, 1], 8, 2, d, 32, dtype, seed=5, weights=True)
    w0 = c["w"].clone()
    args = (c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    a, la = ssa.paged_attention(c["q"], *args, weights=c["w"], return_lse=True)
    w1 = c["w"].clone()
    c["w"].copy_(w0)
    b, lb = ssa.paged_attention(c["q"], *args, weights=c["w"], return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(w1, c["w"])
    check_attention(c, got=(a, la))


# ---------------------------------------------------------------------------
# slot weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,q_lens,h_q,h_kv,d,page,layout,causal", [
    ([900, 1, 64, 0], [1, 1, 1, 0], 32, 8, 128, 64, "hnd", True),
    ([2000, 333], [1, 1], 14, 2, 64, 16, "nhd", True),
    ([300, 130], [300, 70], 8, 2, 128, 32, "hnd", True),
    ([700, 40, 129], [129, 50, 1], 28, 4, 128, 128, "nhd", True),
    ([257, 100], [40, 100], 4, 4, 64, 16, "hnd", False),
    ([120], [30], 6, 2, 40, 12, "nhd", True),
])
def test_slot_weights_match_formula(lens, q_lens, h_q, h_kv, d, page, layout, causal, dtype):
    c = make(lens, q_lens, h_q, h_kv, d, page, dtype, layout, seed=d, weights=True)
    w0 = c["w"].double()
    got = ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"],
                              is_causal=causal, weights=c["w"], return_lse=True)
    check_attention(c, causal=causal, got=got)
    _, _, _, add = oracle(c, causal=causal)
    err = (c["w"].double() - w0 - add).abs()
    assert (err <= 3e-5 * add + 2.0 ** -23 * (w0 + add)).all(), float((err / (add + 1e-9)).max())
    assert torch.equal(c["w"][add == 0].double(), w0[add == 0])


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("q_len", [1, 200])
def test_nan_in_a_key_reaches_every_weight_of_the_rows_that_see_it(dtype, d, q_len):
    c = make([300], [q_len], 8, 2, d, 32, dtype, seed=13, weights=True)
    pg, sl = slots(c, 0, 300)
    c["k"][pg[250], sl[250], 0, 7] = math.nan          # the last row sees it, and all 300 slots
    w0 = c["w"].clone()
    ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], weights=c["w"])
    assert torch.isnan(c["w"][pg, sl, 0]).all()
    assert torch.isfinite(c["w"][pg, sl, 1]).all() and (c["w"][pg, sl, 1] >= w0[pg, sl, 1]).all()


def test_a_page_shared_by_two_sequences_collects_both():
    c = make([64, 64], [1, 1], 8, 2, 64, 32, torch.bfloat16, seed=8, weights=True)
    c["table"][1] = c["table"][0]
    c["page_table"] = c["table"].to(DEV)
    w0 = c["w"].double()
    ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], weights=c["w"])
    _, _, _, add = oracle(c)
    assert ((c["w"].double() - w0 - add).abs() <= 3e-5 * add + 1e-6).all()
    assert abs(float(add.sum()) - 2 * 8) < 1e-6        # every row and head gives 1


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,d", [(torch.float32, 8), (torch.bfloat16, 128), (torch.float16, 72)])
@pytest.mark.parametrize("page,layout", [(16, "hnd"), (7, "nhd")])
@pytest.mark.parametrize("lens,q_lens", [([1], [1]), ([9, 40, 3, 0, 100], [2, 40, 0, 0, 61]), ([300], [300])])
def test_append_writes_its_slots_and_nothing_else(dtype, d, page, layout, lens, q_lens):
    c = make(lens, q_lens, 4, 2, d, page, dtype, layout, seed=7, weights=True)
    T = c["starts"][-1]
    wide = torch.randn((2, T, 3, d + 8), device=DEV).to(dtype)
    k_new, v_new = wide[0, :, 1:, :d], wide[1, :, 1:, :d]
    ref = {n: c[n].clone() for n in ("k", "v", "w")}
    for s, (n, L_) in enumerate(zip(q_lens, lens)):
        pg, sl = slots(c, s, L_)
        pg, sl = pg[L_ - n:], sl[L_ - n:]
        r = slice(c["starts"][s], c["starts"][s + 1])
        ref["k"][pg, sl], ref["v"][pg, sl], ref["w"][pg, sl] = k_new[r], v_new[r], 0.0
    ssa.paged_append(k_new, v_new, c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], c["w"])
    for n in ("k", "v", "w"):
        assert torch.equal(c[n], ref[n]), n


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def evict_oracle(c, budget, recent):
    """Kept slots by a plain sort: recent first, then by (weight, -slot)."""
    kept = torch.full((len(c["lens"]), c["h_kv"], budget), -1, dtype=torch.int32)
    for s, n in enumerate(c["lens"]):
        pg, sl = slots(c, s, n)
        size = min(n, budget)
        for h in range(c["h_kv"]):
            w = c["w"][pg, sl, h].double().cpu().tolist()
            w = [-math.inf if x != x else x for x in w]
            rank = sorted(range(n), key=lambda j: (j < n - recent, -w[j], j))
            kept[s, h, :size] = torch.tensor(sorted(rank[:size]), dtype=torch.int32)
    return kept


def run_evict(c, budget, recent):
    page = c["page"]
    need = [-(-min(n, budget) // page) for n in c["lens"]]
    used = set(int(x) for s, n in enumerate(c["lens"]) for x in c["table"][s][:-(-n // page)])
    free = [p for p in range(c["k"].shape[0]) if p not in used]
    new = torch.zeros((len(need), max(max(need), 1)), dtype=torch.int32)
    for s, n in enumerate(need):
        for i in range(n):
            new[s, i] = free.pop()
    before = {n: c[n].clone() for n in ("k", "v", "w")}
    kept, lens = ssa.paged_evict(c["k"], c["v"], c["w"], c["page_table"], c["kv_lens"], new.to(DEV), budget, recent)
    ref = evict_oracle({**c, **before}, budget, recent)
    assert torch.equal(kept.cpu(), ref)
    assert lens.tolist() == [min(n, budget) for n in c["lens"]]
    for s, n in enumerate(c["lens"]):
        size = min(n, budget)
        pg, sl = slots(c, s, n)
        to_pg, to_sl = slots(c, s, size, new)
        for h in range(c["h_kv"]):
            j = ref[s, h, :size].long().to(DEV)
            for name in ("k", "v", "w"):
                before[name][to_pg, to_sl, h] = before[name][pg[j], sl[j], h]
    for name in ("k", "v", "w"):
        a, b = c[name], before[name]
        assert torch.equal(torch.nan_to_num(a, nan=-7.0), torch.nan_to_num(b, nan=-7.0)), name


@pytest.mark.parametrize("dtype,d,layout", [(torch.bfloat16, 128, "hnd"), (torch.float32, 16, "nhd"),
                                            (torch.float16, 64, "nhd")])
@pytest.mark.parametrize("lens,budget,recent,page", [
    ([1], 1, 0, 16), ([1], 1, 1, 16), ([100], 1, 0, 16), ([100], 1, 1, 16),
    ([500, 64, 0, 65, 1000], 64, 10, 16),
    ([3000, 1025], 1024, 0, 64), ([777], 300, 300, 7), ([130, 90], 129, 64, 32),
    ([5000], 4999, 5, 128),
])
def test_evict_keeps_the_heaviest_and_the_recent(dtype, d, layout, lens, budget, recent, page):
    spare = sum(-(-min(n, budget) // page) for n in lens) + 1
    c = make(lens, [0] * len(lens), 4, 2, d, page, dtype, layout, seed=budget, spare=spare, weights=True)
    run_evict(c, budget, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "zero", "nan", "inf", "negative"])
def test_evict_ties_and_special_weights(kind):
    c = make([700, 301], [0, 0], 4, 2, 64, 32, torch.bfloat16, seed=3, spare=24, weights=True)
    w = c["w"]
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few":
        w.copy_((w * 3).floor())
    elif kind == "zero":
        w.copy_(torch.where(w < 0.5, 0.0, -0.0))           # -0 and 0 are equal
    elif kind == "nan":
        w[w < 0.6] = math.nan
        w[w > 0.9] = -math.inf                             # a tie with NaN: the lower slot first
    elif kind == "inf":
        w[w < 0.6] = math.inf
    else:
        w.neg_()
    run_evict(c, 300, 20)


# ---------------------------------------------------------------------------
# errors, streams, graphs
# ---------------------------------------------------------------------------
def test_bad_page_and_bad_lengths_are_reported():
    def fresh():
        return make([100, 64], [2, 1], 4, 2, 64, 16, torch.bfloat16, seed=1, weights=True)

    def attend(c):
        return ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])

    def append(c):
        ssa.paged_append(c["q"][:, :2], c["q"][:, :2], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])

    ref = attend(fresh())
    for page in (-1, 10 ** 6):
        c = fresh()
        c["page_table"][0, 6] = page                      # holds slots 96 .. 99
        out = attend(c)
        with pytest.raises(IndexError):
            ssa.check_errors()
        assert torch.equal(out[2], ref[2])                # the other sequence is right
        k = c["k"].clone()
        append(c)
        with pytest.raises(IndexError):
            ssa.check_errors()
        pg, sl = int(c["table"][1][3]), 15                # slot 63 of the other sequence
        k[pg, sl] = c["q"][2, :2]
        assert torch.equal(c["k"], k)
    for name, at, v in (("kv_lens", 0, 7 * 16 + 1), ("kv_lens", 0, -1), ("q_starts", 1, -1), ("q_starts", 1, 4)):
        c = fresh()
        c[name][at] = v
        if name == "q_starts":
            c["q_starts"][2] = max(3, v)
        attend(c)
        with pytest.raises(ValueError):
            ssa.check_errors()
    c = fresh()
    c["kv_lens"][0] = 1                                   # two rows appended to one slot
    append(c)
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        attend(fresh())                                   # raised by the next call
    ssa.check_errors()
    c = fresh()
    new = torch.zeros((2, 2), dtype=torch.int32, device=DEV) + c["k"].shape[0]
    ssa.paged_evict(c["k"], c["v"], c["w"], c["page_table"], c["kv_lens"], new, 32)
    with pytest.raises(IndexError):
        ssa.check_errors()
    ssa.paged_evict(c["k"], c["v"], c["w"], c["page_table"], c["kv_lens"], new[:, :1] * 0, 32)
    with pytest.raises(ValueError):
        ssa.check_errors()
    ssa.check_errors()


def test_sync_mode_raises_in_the_failing_call(monkeypatch):
    c = make([20], [1], 4, 2, 64, 16, torch.bfloat16)
    c["page_table"][0, 1] = 99
    monkeypatch.setenv("SSA_CHECKED", "sync")
    with pytest.raises(IndexError):
        ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    monkeypatch.setenv("SSA_CHECKED", "0")
    ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    monkeypatch.delenv("SSA_CHECKED")
    ssa.check_errors()


def test_refusals():
    c = make([20, 30], [1, 4], 4, 2, 64, 16, torch.bfloat16, weights=True)
    k, v, t, qs, kl, q, w = (c[n] for n in ("k", "v", "page_table", "q_starts", "kv_lens", "q", "w"))

    def attend(q=q, k=k, v=v, t=t, qs=qs, kl=kl, **kw):
        return ssa.paged_attention(q, k, v, t, qs, kl, **kw)

    bad = [
        (RuntimeError, dict(q=q.cpu())), (RuntimeError, dict(t=t.cpu())), (TypeError, dict(q=q.float())),
        (TypeError, dict(v=v.half())), (TypeError, dict(t=t.long())), (TypeError, dict(qs=qs.float())),
        (ValueError, dict(q=q[:, :3])), (ValueError, dict(q=q[..., :32])), (ValueError, dict(q=q[0])),
        (ValueError, dict(v=v[:2])), (ValueError, dict(t=t[:1])), (ValueError, dict(qs=qs[:2])),
        (ValueError, dict(kl=kl[:1])), (ValueError, dict(k=k.transpose(2, 3), v=v.transpose(2, 3))),
        (TypeError, dict(weights=w.double())), (ValueError, dict(weights=w[:1])),
        (RuntimeError, dict(weights=w.cpu())), (L.SSAError, dict(scale=0.0)), (L.SSAError, dict(scale=math.nan)),
        (TypeError, dict(k=k.double(), v=v.double(), q=q.double())),
        (L.SSAError, dict(q=torch.empty((5, 4, 72), device=DEV, dtype=q.dtype)[..., 4:68])),      # 8-byte start
        (L.SSAError, dict(q=torch.empty((5, 34, 64), device=DEV, dtype=q.dtype))),                # g = 17
        (L.SSAError, dict(q=torch.empty((5, 4, 4), device=DEV, dtype=q.dtype),                    # d = 4
                          k=torch.empty((9, 16, 2, 4), device=DEV, dtype=q.dtype),
                          v=torch.empty((9, 16, 2, 4), device=DEV, dtype=q.dtype))),
        (L.SSAError, dict(k=torch.empty((2, 1025, 2, 64), device=DEV, dtype=q.dtype),
                          v=torch.empty((2, 1025, 2, 64), device=DEV, dtype=q.dtype))),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            attend(**kw)
    new = torch.zeros((2, 2), dtype=torch.int32, device=DEV)
    for budget, recent in ((0, 0), (8, 9), (8, -1)):
        with pytest.raises(ValueError):
            ssa.paged_evict(k, v, w, t, kl, new, budget, recent)
    with pytest.raises(ValueError):
        ssa.paged_evict(k, v, None, t, kl, new, 8)
    with pytest.raises(ValueError):
        ssa.paged_evict(k, v, w, t, kl, new[:1], 8)
    for kn in (q[:, :1], q[:, :2, :32], q[:4, :2]):
        with pytest.raises(ValueError):
            ssa.paged_append(kn, q[:, :2], k, v, t, qs, kl)
    with pytest.raises(TypeError):
        ssa.paged_append(q[:, :2].float(), q[:, :2].float(), k, v, t, qs, kl)
    ssa.check_errors()


def test_empty_calls():
    c = make([20, 30], [0, 0], 4, 2, 64, 16, torch.bfloat16, weights=True)
    out = ssa.paged_attention(c["q"], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], weights=c["w"])
    assert out.shape == (0, 4, 64)
    e = torch.empty((0, 2), dtype=torch.int32, device=DEV)
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ssa.paged_attention(c["q"], c["k"], c["v"], e, z, e[:, 0]).shape == (0, 4, 64)
    ssa.paged_append(c["q"][:, :2], c["q"][:, :2], c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    kept, lens = ssa.paged_evict(c["k"], c["v"], c["w"], e, e[:, 0], e, 4)
    assert kept.shape == (0, 2, 4) and lens.shape == (0,)
    ssa.check_errors()


@pytest.mark.parametrize("q_len", [1, 40])
def test_another_stream_and_a_graph_with_new_lengths(q_len):
    c = make([500, 90], [q_len, q_len], 8, 2, 128, 32, torch.bfloat16, seed=2, weights=True)
    args = (c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"])
    ref = ssa.paged_attention(c["q"], *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ssa.paged_attention(c["q"], *args)
        ssa.paged_attention(c["q"], *args, weights=c["w"])        # warm-up of every kernel of the graph
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    c["w"].zero_()
    with torch.cuda.graph(graph):
        out, lse = ssa.paged_attention(c["q"], *args, weights=c["w"], return_lse=True)
    for lens in ([500, 90], [350, 41], [41, 90]):
        c["lens"] = lens
        c["kv_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["w"].zero_()
        graph.replay()
        check_attention(c, got=(out, lse))
        _, _, _, add = oracle(c)
        assert ((c["w"].double() - add).abs() <= 3e-5 * add + 1e-7).all()
    ssa.check_errors()


# ---------------------------------------------------------------------------
# the cache object
# ---------------------------------------------------------------------------
def test_cache_steps_equal_dense_attention_and_eviction_frees_pages():
    torch.manual_seed(0)
    h_q, h_kv, d = 8, 2, 64
    cache = ssa.PagedCache(num_pages=40, page_size=16, num_kv_heads=h_kv, head_dim=d, num_layers=2,
                           dtype=torch.float32, device=DEV, track_weights=True)
    ids = [cache.add(), cache.add()]
    kept = {s: [torch.empty((0, n, d), device=DEV) for n in (h_kv, h_kv)] for s in ids}
    for new in ([37, 5], [1, 1], [20, 1], [1, 60]):
        batch = cache.extend(ids, new)
        T = sum(new)
        q, k, v = (torch.randn((T, h, d), device=DEV) for h in (h_q, h_kv, h_kv))
        for layer in (0, 1):
            cache.append(batch, k, v * (layer + 1), layer)
        outs = [cache.attend(batch, q, layer) for layer in (0, 1)]
        assert torch.allclose(outs[1], 2 * outs[0], rtol=1e-5, atol=1e-5)
        at = 0
        for s, n in zip(ids, new):
            kept[s] = [torch.cat((old, x[at:at + n])) for old, x in zip(kept[s], (k, v))]
            full = kept[s][0].shape[0]
            mask = ssa.build_causal_mask(full, device=DEV)[full - n:]
            ref = ssa.dense_attention(q[at:at + n].double(), *(x.double() for x in kept[s]), causal_mask=mask)
            assert (outs[0][at:at + n].double() - ref).abs().max() < 1e-5
            at += n
    assert [cache.length(s) for s in ids] == [59, 67]
    free = cache.free_pages
    assert cache.evict(ids, budget=64, recent=8) == [ids[1]]
    assert [cache.length(s) for s in ids] == [59, 64] and cache.free_pages == free + 1
    assert cache.evict(ids, budget=20, recent=8) == ids
    assert cache.free_pages == 40 - 4
    batch = cache.extend(ids, [1, 1])
    q = torch.randn((2, h_q, d), device=DEV)
    cache.append(batch, q[:, :2], q[:, :2])
    assert torch.isfinite(cache.attend(batch, q)).all()
    with pytest.raises(RuntimeError, match="full"):
        cache.extend([ids[0]], [40 * 16])
    assert cache.length(ids[0]) == 21
    cache.remove(ids[0])
    cache.remove(ids[1])
    assert cache.free_pages == 40
    ssa.check_errors()


def test_cache_refusals():
    cache = ssa.PagedCache(4, 16, 1, 64, device=DEV)
    s = cache.add()
    with pytest.raises(ValueError):
        cache.extend([s, s], [1, 1])
    with pytest.raises(ValueError):
        cache.extend([s], [-1])
    with pytest.raises(ValueError, match="track_weights"):
        cache.evict([s], 4)
    tracked = ssa.PagedCache(4, 16, 1, 64, device=DEV, track_weights=True)
    t = tracked.add()
    tracked.extend([t], [60])
    with pytest.raises(RuntimeError, match="free pages"):
        tracked.evict([t], 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_sequences(dtype):
    """A padded q and an empty batch: nothing to do, and nothing is done."""
    c = make([20], [5], 4, 2, 64, 16, dtype, weights=True)
    none, start = torch.empty((0, 2), dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    before = c["w"].clone()
    out, lse = ssa.paged_attention(c["q"], c["k"], c["v"], none, start, none[:, 0], weights=c["w"], return_lse=True)
    assert out.shape == (5, 4, 64) and lse.shape == (5, 4) and torch.equal(c["w"], before)
    ssa.check_errors()


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("lens,q_lens,bad", [([9, 40, 30], [2, 41, 5], 1), ([1, 20], [300, 20], 0), ([0, 7], [3, 1], 0)])
def test_append_of_more_rows_than_a_sequence_holds_writes_none_of_them(lens, q_lens, bad, layout):
    c = make(lens, q_lens, 4, 2, 64, 16, torch.bfloat16, layout, seed=5, weights=True)
    k_new, v_new = torch.randn((2, c["starts"][-1], 2, 64), device=DEV).to(torch.bfloat16).unbind()
    ref = {n: c[n].clone() for n in ("k", "v", "w")}
    for s, (n, L_) in enumerate(zip(q_lens, lens)):
        if s != bad:
            pg, sl = slots(c, s, L_)
            pg, sl, r = pg[L_ - n:], sl[L_ - n:], slice(c["starts"][s], c["starts"][s + 1])
            ref["k"][pg, sl], ref["v"][pg, sl], ref["w"][pg, sl] = k_new[r], v_new[r], 0.0
    ssa.paged_append(k_new, v_new, c["k"], c["v"], c["page_table"], c["q_starts"], c["kv_lens"], c["w"])
    with pytest.raises(ValueError, match="paged_append"):
        ssa.check_errors()
    for n in ("k", "v", "w"):
        assert torch.equal(c[n], ref[n]), n
