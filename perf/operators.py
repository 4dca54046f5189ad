"""Timed cases of the paged key/value cache operators, with their plain forms.

Four operators work on one cache of fixed-size pages (``k_pages``, ``v_pages``
``[pages, page, h_kv, d]``; sequence ``s`` keeps its slot ``j`` in page
``page_table[s, j // page]`` at row ``j % page``):

* ``append``  -- the chunk's new keys and values are written to their slots;
* ``attend``  -- causal softmax attention of a chunk of new tokens (one token
  per sequence while decoding) over everything the sequence has cached;
* ``weigh``   -- the same attention, which also adds to every cached slot the
  attention weight it received, summed over the chunk's rows and the heads of
  its group;
* ``evict``   -- every sequence keeps, per KV head, its ``recent`` last slots and
  the heaviest of the others, ``budget`` in all, copied in order to new pages.

A batch is ragged: sequence ``s`` owns rows ``q_starts[s] .. q_starts[s + 1]`` of
the chunk, which are its last cached positions (``kv_lens`` counts them).
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _case(name, op, dtype, heads, page, batch, q, kv, ragged, layout="hnd", budget=0, recent=0):
    """``ragged``: 0 every sequence has ``q`` new rows and ``kv`` keys; 1 lengths
    spread below those; 2 as 1, and every other sequence has one new row."""
    h_q, h_kv, d = heads
    c = dict(op=op, dtype=dtype, h_q=h_q, h_kv=h_kv, d=d, page=page, batch=batch, q=q, kv=kv, ragged=ragged,
             layout=layout, budget=budget, recent=recent)
    if name:
        c["name"] = name
    return c


# the head layouts of this repository's op-level sweep, its dense check and its decoder stack
_SWEEP, _DENSE, _STACK = (32, 8, 128), (8, 2, 64), (28, 4, 128)


def listed():
    return [
        # one sequence's next token enters the cache: latency only
        _case("append_one_token", "append", "bf16", _SWEEP, 64, 1, 1, 1024, 0),
        # the prompts of a batch enter the cache, token-major pages of 16
        _case("append_prompts", "append", "bf16", _STACK, 16, 16, 2048, 2048, 1, "nhd"),
        # one sequence decodes at a short context: the smallest call of a serving loop
        _case("attend_one_token", "attend", "bf16", _SWEEP, 64, 1, 1, 1024, 0),
        # a decoding batch of unequal contexts (group of 7 heads)
        _case("attend_token_batch", "attend", "bf16", _STACK, 64, 64, 1, 16384, 1),
        # prompts' chunks and single tokens in one batch, as a scheduler mixes them
        _case("attend_mixed_batch", "attend", "bf16", _SWEEP, 32, 24, 512, 6000, 2),
        # odd ragged chunks, small heads, small token-major pages
        _case("attend_odd_chunks", "attend", "f16", _DENSE, 16, 7, 301, 2477, 1, "nhd"),
        # a long prompt's chunk against its long cached prefix
        _case("attend_long_chunk", "attend", "bf16", _SWEEP, 128, 1, 2048, 32768, 0),
        # full precision, as a check of a model runs it
        _case("attend_f32", "attend", "f32", _DENSE, 32, 3, 129, 1500, 1),
        # a decoding batch that keeps count of the attention its cache receives
        _case("weigh_token_batch", "weigh", "bf16", _SWEEP, 64, 16, 1, 8192, 1),
        # two prompts' chunks, weights kept
        _case("weigh_chunks", "weigh", "bf16", _SWEEP, 64, 2, 1024, 8192, 0),
        # caches a few pages over their budget are cut back
        _case("evict_pages", "evict", "bf16", _SWEEP, 64, 8, 0, 4352, 0, budget=4096, recent=64),
        # long prompts' caches are cut to an eighth of the longest
        _case("evict_prompts", "evict", "f16", _SWEEP, 64, 16, 0, 32768, 1, budget=4096, recent=512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "attend", "attend", "attend", "weigh", "weigh", "evict"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        heads = rng.choice([_SWEEP, _DENSE, _STACK])
        page = rng.choice([16, 32, 64, 128])
        layout = rng.choice(["hnd", "nhd"])
        ragged = rng.choice([0, 1, 2])
        batch = _log(rng, 1, 64)
        kv = _log(rng, 1, 32768)
        if op == "evict":
            c = _case("", op, dtype, heads, page, batch, 0, kv, min(ragged, 1), layout,
                      budget=max(1, int(kv * rng.uniform(0.05, 0.95))))
            c["recent"] = rng.randrange(0, c["budget"] + 1)
        else:
            q = 1 if rng.random() < 0.4 else _log(rng, 1, min(kv, 2048))
            c = _case("", op, dtype, heads, page, batch, q, kv, ragged, layout)
        # no dearer than the largest listed case of the kind: the scores of the plain form, the
        # keys it gathers in 32 bits, the cache itself, and what the CUDA cores do in full precision
        scores = batch * max(1, c["q"]) * kv * c["h_q"]
        keys = batch * kv * c["h_kv"] * c["d"]
        if c["op"] in ("attend", "weigh") and (scores > 2 ** 31 or dtype == "f32" and scores > 2 ** 28):
            continue
        if keys > (2 ** 29 if dtype != "f32" else 2 ** 28) or c["op"] == "append" and batch * c["q"] > 32768:
            continue
        return c


def _lens(case):
    """New rows and cached keys of every sequence, by the case alone."""
    rng = random.Random(case["batch"] * 1000003 + case["kv"] * 31 + case["q"])
    q, kv = [], []
    for s in range(case["batch"]):
        n, m = case["kv"], case["q"]
        if case["ragged"] and s:
            n = max(1, int(n * rng.uniform(0.02, 1.0)))
            m = max(1, int(m * rng.uniform(0.05, 1.0))) if m else 0
        if case["ragged"] == 2 and s % 2:
            m = min(m, 1)
        if case["op"] == "append" and case["q"] == case["kv"]:
            m = n                                             # whole prompts
        kv.append(n)
        q.append(min(m, n))
    return q, kv


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _paged(pages, page, h_kv, tail, layout, dtype):
    """``[pages, page, h_kv, *tail]``, a head's rows side by side ("hnd") or a token's heads ("nhd")."""
    if layout == "hnd":
        return torch.empty((pages, h_kv, page, *tail), dtype=dtype, device="cuda").transpose(1, 2)
    return torch.empty((pages, page, h_kv, *tail), dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, page, h_q, h_kv, d = _DTYPES[case["dtype"]], case["page"], case["h_q"], case["h_kv"], case["d"]
    q_lens, kv_lens = _lens(case)
    need = [-(-n // page) for n in kv_lens]
    keep = [-(-min(n, case["budget"]) // page) for n in kv_lens] if case["op"] == "evict" else [0] * len(need)
    pages = sum(need) + sum(keep)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    # the pages of a sequence lie anywhere in the cache
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros((len(need), max(need)), dtype=torch.int32)
    new_table = torch.zeros((len(need), max(max(keep), 1)), dtype=torch.int32)
    at = 0
    for s, (a, b) in enumerate(zip(need, keep)):
        table[s, :a] = order[at:at + a]
        new_table[s, :b] = order[at + a:at + a + b]
        at += a + b
    starts = torch.zeros(len(q_lens) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(q_lens, dtype=torch.int32).cumsum(0)
    st = dict(op=case["op"], page=page, budget=case["budget"], recent=case["recent"], rows=sum(q_lens),
              q_max=max(q_lens), kv_max=max(kv_lens), group=h_q // h_kv, page_table=table.cuda(),
              new_table=new_table.cuda(), q_starts=starts.cuda(),
              kv_lens=torch.tensor(kv_lens, dtype=torch.int32).cuda())

    # keys lie around 64 centroids at the rate of one in twenty, the rest are spread (the planted
    # clusters of this repository's sweep); half of the queries look for a centroid, so rows of
    # sharp and of flat attention meet
    cent = randn(64, d)

    def near(rows, heads, share):
        x = randn(rows, heads, d)
        at = torch.rand(rows, heads, 1, generator=g, device="cuda") < share
        which = torch.randint(0, 64, (rows, heads), generator=g, device="cuda")
        return torch.where(at, cent[which] + 0.1 * x, x)

    st["k_pages"] = _paged(pages, page, h_kv, (d,), case["layout"], dt)
    st["v_pages"] = _paged(pages, page, h_kv, (d,), case["layout"], dt)
    st["k_pages"].copy_(near(pages * page, h_kv, 0.05).view(pages, page, h_kv, d))
    st["v_pages"].copy_(randn(pages, page, h_kv, d))
    st["weights"] = None
    if case["op"] == "append":
        st["k_new"], st["v_new"] = near(sum(q_lens), h_kv, 0.05).to(dt), randn(sum(q_lens), h_kv, d).to(dt)
    else:
        st["q"] = near(sum(q_lens), h_q, 0.5).to(dt) if sum(q_lens) else None
    if case["op"] in ("weigh", "evict"):
        # weight collected by earlier steps: a few slots hold most of it
        st["weights"] = _paged(pages, page, h_kv, (), case["layout"], torch.float32)
        st["weights"].copy_(torch.exp(2.0 * randn(pages, page, h_kv)))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


def _run_own(st):
    import ssa_b200 as ssa

    cache = st["k_pages"], st["v_pages"]
    if st["op"] == "append":
        ssa.paged_append(st["k_new"], st["v_new"], *cache, st["page_table"], st["q_starts"], st["kv_lens"])
        return cache
    if st["op"] == "evict":
        kept, lens = ssa.paged_evict(*cache, st["weights"], st["page_table"], st["kv_lens"], st["new_table"],
                                     st["budget"], st["recent"])
        return kept, lens, *cache, st["weights"]
    out, lse = ssa.paged_attention(st["q"], *cache, st["page_table"], st["q_starts"], st["kv_lens"],
                                   weights=st["weights"], return_lse=True)
    return (out, lse) if st["weights"] is None else (out, lse, st["weights"])


def _row_places(st):
    """Sequence of every chunk row and its number there."""
    t = torch.arange(st["rows"], device="cuda", dtype=torch.int32)
    s = torch.searchsorted(st["q_starts"], t, right=True) - 1
    return s, t - st["q_starts"][s]


def _slots(st, n, table):
    """Page and row of slots 0 .. n-1 of every sequence, ``[B, n]``."""
    j = torch.arange(n, device="cuda")
    return table[:, j // st["page"]].long(), (j % st["page"]).expand(table.shape[0], n)


def _plain_append(st):
    s, i = _row_places(st)
    n_new = st["q_starts"][1:] - st["q_starts"][:-1]
    j = st["kv_lens"][s] - n_new[s] + i
    where = st["page_table"][s, j // st["page"]].long(), (j % st["page"]).long()
    st["k_pages"][where] = st["k_new"]
    st["v_pages"][where] = st["v_new"]
    return st["k_pages"], st["v_pages"]


def _plain_attend(st):
    dt, n_max, kv_max, g = st["q"].dtype, st["q_max"], st["kv_max"], st["group"]
    B, (T, h_q, d) = st["kv_lens"].shape[0], st["q"].shape
    h = h_q // g
    where = _slots(st, kv_max, st["page_table"])
    k, v = st["k_pages"][where].float(), st["v_pages"][where].float()           # [B, kv, h, d]
    # the chunk's rows, padded to the longest chunk
    starts, lens = st["q_starts"].long(), st["kv_lens"].long()
    i = torch.arange(n_max, device="cuda")
    n_new = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + i).clamp_(max=max(T - 1, 0))
    q = st["q"][rows].float().view(B, n_max, h, g, d) / math.sqrt(d)
    s = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, h, g * n_max, d), k.permute(0, 2, 3, 1))
    s = s.view(B, h, g, n_max, kv_max)
    j = torch.arange(kv_max, device="cuda")
    seen = (j <= (lens - n_new)[:, None, None] + i[:, None]) & (i < n_new[:, None])[..., None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(-1)                                         # [B, h, g, n]
    p /= total.clamp(min=1e-30)
    o = torch.matmul(p.view(B, h, g * n_max, kv_max), v.transpose(1, 2)).view(B, h, g, n_max, d)
    at = _row_places(st)
    out = o.permute(0, 3, 1, 2, 4)[at].reshape(T, h_q, d).to(dt)
    lse = lse.permute(0, 3, 1, 2)[at].reshape(T, h_q)
    if st["weights"] is None:
        return out, lse
    st["weights"].index_put_(where, p.sum((2, 3)).transpose(1, 2), accumulate=True)
    return out, lse, st["weights"]


def _plain_evict(st):
    lens, budget, recent, kv_max = st["kv_lens"].long(), st["budget"], st["recent"], st["kv_max"]
    where = _slots(st, kv_max, st["page_table"])
    w = st["weights"][where].transpose(1, 2)                                    # [B, h, kv]
    j = torch.arange(kv_max, device="cuda")
    w = w.masked_fill((j >= (lens - recent)[:, None])[:, None], math.inf)
    w = w.masked_fill((j >= lens[:, None])[:, None], -math.inf)
    best = w.argsort(dim=-1, descending=True, stable=True)[..., :budget]
    best = torch.where(best < lens[:, None, None], best, kv_max).sort(-1).values
    best = torch.nn.functional.pad(best, (0, max(0, budget - best.shape[-1])), value=kv_max)
    fine = best < kv_max
    kept = torch.where(fine, best, -1).to(torch.int32)
    # survivors, in order, to the first slots of the new pages (a lane without one rewrites its slot 0)
    b = torch.arange(lens.shape[0], device="cuda")[:, None, None]
    h = torch.arange(best.shape[1], device="cuda")[:, None]
    src = torch.where(fine, best, 0)
    src = st["page_table"][b, src // st["page"]].long(), src % st["page"], h
    to = torch.arange(budget, device="cuda").expand_as(best)
    width = st["new_table"].shape[1] * st["page"]
    to_page = st["new_table"][b, to.clamp(max=width - 1) // st["page"]].long()
    dst = torch.where(fine, to_page, src[0]), torch.where(fine, to % st["page"], src[1]), h
    for t in (st["k_pages"], st["v_pages"], st["weights"]):
        t[dst] = t[src]
    return kept, lens.clamp(max=budget).to(torch.int32), st["k_pages"], st["v_pages"], st["weights"]


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_attend, "evict": _plain_evict}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    q_lens, kv_lens = _lens(case)
    size = 4 if case["dtype"] == "f32" else 2
    h_q, h, d = case["h_q"], case["h_kv"], case["d"]
    row = 2 * h * d * size                                    # one position's key and value
    if case["op"] == "append":
        return {"bytes": 2.0 * sum(q_lens) * row, "flops": 0.0}
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in kv_lens)
        return {"bytes": float(sum(kv_lens) * h * 4 + kept * (2 * row + 2 * h * 4)), "flops": 0.0}
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(q_lens, kv_lens))   # (row, key) pairs in sight
    total = float(sum(kv_lens) * row + sum(q_lens) * h_q * (2 * d * size + 4))
    if case["op"] == "weigh":
        total += 2.0 * sum(kv_lens) * h * 4
    return {"bytes": total, "flops": 4.0 * pairs * h_q * d}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    page, h_kv, g = case["page"], case["h_kv"], case["h_q"] // case["h_kv"]
    q_lens, kv_lens = _lens(case)
    table = st["page_table"].cpu()
    ends = st["q_starts"].cpu().tolist()

    def places(s, first, last, which=table):
        j = torch.arange(first, last)
        return which[s][j // page].long().cuda(), (j % page).cuda()

    if case["op"] == "append":
        for s, (m, n) in enumerate(zip(q_lens, kv_lens)):
            pg, sl = places(s, n - m, n)
            for t, new in ((st["k_pages"], st["k_new"]), (st["v_pages"], st["v_new"])):
                t.index_put_((pg, sl), new[ends[s]:ends[s + 1]])
        return st["k_pages"].double(), st["v_pages"].double()
    weights = st["weights"].double() if st["weights"] is not None else None
    if case["op"] == "evict":
        k, v = st["k_pages"].double(), st["v_pages"].double()
        kept = torch.full((case["batch"], h_kv, case["budget"]), -1, dtype=torch.int32)
        for s, n in enumerate(kv_lens):
            size = min(n, case["budget"])
            pg, sl = places(s, 0, n)
            to_pg, to_sl = places(s, 0, size, st["new_table"].cpu())
            for h in range(h_kv):
                w = weights[pg, sl, h].clone()
                w[max(0, n - case["recent"]):] = math.inf
                # ascending by (-weight, position): a stable sort keeps the lower position first
                top = torch.sort(-w, stable=True).indices[:size].sort().values
                kept[s, h, :size] = top.to(torch.int32).cpu()
                for t in (k, v, weights):
                    t[to_pg, to_sl, h] = t[pg[top], sl[top], h]
        lens = torch.tensor([min(n, case["budget"]) for n in kv_lens], dtype=torch.int32)
        return kept, lens, k, v, weights
    out = torch.zeros((sum(q_lens), case["h_q"], case["d"]), dtype=torch.float64, device="cuda")
    lse = torch.zeros((sum(q_lens), case["h_q"]), dtype=torch.float64, device="cuda")
    for s, (m, n) in enumerate(zip(q_lens, kv_lens)):
        pg, sl = places(s, 0, n)
        last = torch.arange(n - m, n, device="cuda")           # a row's own position: the last key it sees
        hidden = torch.arange(n, device="cuda")[None, :] > last[:, None]
        for h in range(h_kv):
            k, v = st["k_pages"][pg, sl, h].double(), st["v_pages"][pg, sl, h].double()
            for e in range(h * g, (h + 1) * g):
                x = st["q"][ends[s]:ends[s + 1], e].double() @ k.T / math.sqrt(case["d"])
                x[hidden] = -math.inf
                norm = torch.logsumexp(x, 1)
                x = torch.exp(x - norm[:, None])
                out[ends[s]:ends[s + 1], e] = x @ v
                lse[ends[s]:ends[s + 1], e] = norm
                if weights is not None:
                    weights[pg, sl, h] += x.sum(0)
    return (out, lse) if weights is None else (out, lse, weights)
