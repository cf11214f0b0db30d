"""The paged-cache serving operators: plain forms, the framework's calls, and the cases both are measured on.

Four operators that act on one paged KV cache (pages ``[num_pages, kv_heads, page_size, head_dim]`` for K and for V, a
table of page ids per sequence):

* ``append``: rotary embedding of new tokens' q and k, their K and V rows into the pages;
* ``attention``: one new token per sequence over its pages, optionally adding every key's attention weight to a running sum;
* ``evict``: keeps, per sequence and head, the newest tokens, the first ones and the heaviest of the rest;
* ``beam``: log-softmax and the best continuations over beams and vocabulary, then the page tables and partly filled
  pages of the new beams (every layer).

With ``own`` false, ``run`` computes them in elementary torch operations; with ``own`` true it calls the framework.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_ITEM = {"float32": 4, "bfloat16": 2}


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one sequence of a 7B-shaped model takes one token: the smallest call of a decode step
        dict(name="append_one_token", op="append", batch=1, new_max=1, past_max=130, q_heads=32, kv_heads=32,
             head_dim=128, page_size=16, dtype="bfloat16", track=False),
        # eight ragged prompts of up to 2048 tokens enter the cache, with the per-slot state that eviction needs
        dict(name="append_prompts", op="append", batch=8, new_max=2048, past_max=0, q_heads=32, kv_heads=32,
             head_dim=128, page_size=16, dtype="bfloat16", track=True),
        # single-stream decoding early in a conversation: latency
        dict(name="attention_one_row", op="attention", batch=1, len_min=130, len_max=130, q_heads=32, kv_heads=32,
             head_dim=128, page_size=16, dtype="bfloat16", track=False),
        # batched decoding of 64 sequences near context 4096, a head of keys per query head: bandwidth
        dict(name="attention_batched", op="attention", batch=64, len_min=4030, len_max=4110, q_heads=32, kv_heads=32,
             head_dim=128, page_size=16, dtype="bfloat16", track=False),
        # continuous batching with shared key heads: lengths from empty to 8192
        dict(name="attention_ragged_shared_heads", op="attention", batch=40, len_min=0, len_max=8192, q_heads=64,
             kv_heads=8, head_dim=128, page_size=32, dtype="bfloat16", track=False),
        # two long documents, the attention weights summed for eviction
        dict(name="attention_long_tracked", op="attention", batch=2, len_min=30001, len_max=65536, q_heads=32,
             kv_heads=8, head_dim=128, page_size=64, dtype="bfloat16", track=True),
        # fp32 with small heads (the tiny configuration's type), weights summed
        dict(name="attention_fp32_tracked", op="attention", batch=16, len_min=1, len_max=1023, q_heads=8, kv_heads=4,
             head_dim=64, page_size=8, dtype="float32", track=True),
        # steady state of a bounded cache: every sequence is one token over its budget
        dict(name="evict_one_over", op="evict", batch=16, len_min=1025, len_max=1025, kv_heads=8, head_dim=128,
             page_size=16, dtype="bfloat16", budget=1024, recent=128, sink=4),
        # long prompts cut down to a quarter at once
        dict(name="evict_prompts", op="evict", batch=8, len_min=1500, len_max=8190, kv_heads=32, head_dim=128,
             page_size=16, dtype="bfloat16", budget=2048, recent=256, sink=4),
        # beam search of one prompt on the 7B shape: latency
        dict(name="beam_one_prompt", op="beam", batch=1, beams=4, vocab=32000, length=201, layers=32, kv_heads=32,
             head_dim=128, page_size=16, dtype="bfloat16", finished=False),
        # many prompts, some beams finished
        dict(name="beam_batched", op="beam", batch=32, beams=8, vocab=32000, length=77, layers=8, kv_heads=32,
             head_dim=128, page_size=16, dtype="bfloat16", finished=True),
        # wide beams over a large vocabulary in fp32
        dict(name="beam_wide_fp32", op="beam", batch=8, beams=16, vocab=131072, length=1000, layers=4, kv_heads=8,
             head_dim=128, page_size=64, dtype="float32", finished=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "evict", "beam"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    hd = rng.choice([32, 64, 128, 128])
    ps = rng.choice([8, 16, 32, 64, 128, 256])
    hkv = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
    hq = hkv * rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 12, 16] if hkv <= 8 else [1, 2])
    base = dict(op=op, kv_heads=hkv, head_dim=hd, page_size=ps, dtype=dtype)
    if op == "append":
        batch = _log(rng, 1, 128)
        most = max(1, min(4096, 16384 * 4096 // (batch * (hq + 2 * hkv) * hd)))
        return dict(base, batch=batch, q_heads=hq, new_max=_log(rng, 1, most), past_max=_log(rng, 1, 2048),
                    track=rng.random() < 0.5)
    if op == "attention":
        batch = _log(rng, 1, 128)
        most = min(131072, (1 << 31) // (batch * hkv * hd * 2 * _ITEM[dtype]))
        most = max(2, min(most, (1 << 32) // (batch * hq * hd)))
        hi = _log(rng, 1, most)
        return dict(base, batch=batch, q_heads=hq, len_max=hi, len_min=rng.randint(0, hi), track=rng.random() < 0.4)
    if op == "evict":
        batch = _log(rng, 1, 32)
        most = max(16, min(32768, (1 << 30) // (batch * hkv * hd * 2 * _ITEM[dtype])))
        hi = _log(rng, 8, most)
        budget = _log(rng, 2, hi)
        recent = rng.randint(0, budget // 2)
        return dict(base, batch=batch, len_max=hi, len_min=rng.randint(0, hi), budget=budget, recent=recent,
                    sink=rng.randint(0, min(4, budget - recent)))
    beams = rng.choice([2, 3, 4, 5, 6, 8, 12, 16])
    batch = _log(rng, 1, 32)
    most = min(200000, (1 << 25) // (batch * beams))
    layers = rng.choice([1, 2, 4, 8])
    return dict(base, batch=batch, beams=beams, vocab=_log(rng, 1000, max(1500, most)), length=_log(rng, 1, 600),
                layers=layers, finished=rng.random() < 0.5)


def _lengths(n, lo, hi):
    """Lengths of n sequences between lo and hi, spread evenly in an order that is not sorted: both ends are met."""
    if n == 1:
        return [hi]
    got = [lo + int((hi - lo) * ((b * 0.6180339887498949) % 1.0)) for b in range(n)]
    got[n // 2] = hi
    return got


def _pages_of(lengths, ps):
    return [-(-n // ps) for n in lengths]


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(g, lengths, ps):
    """A page table over randomly ordered pages (a few of the pool stay unused) and the pool's size."""
    need = _pages_of(lengths, ps)
    width, total = max(max(need), 1), sum(need)
    pool = total + 5
    order = torch.randperm(pool, generator=g, device="cuda")
    table = torch.zeros(len(lengths), width, dtype=torch.int32, device="cuda")
    mask = torch.arange(width, device="cuda")[None, :] < _ints(need)[:, None]
    table[mask] = order[:total].to(torch.int32)
    return table, pool


def _package():
    pkg = str(Path(__file__).resolve().parent.parent / "flagos-pim-compiler_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from backend import cuda_paged

    return cuda_paged


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = globals()["_prepare_" + case["op"]](case, g)
    s["case"] = case
    if own:  # the handle that a program makes once for its buffers and calls at every step
        s["call"] = globals()["_bind_" + case["op"]](case, s)
    return s


def _prepare_append(c, g):
    dt, b = _DTYPES[c["dtype"]], c["batch"]
    hq, hkv, hd, ps = c["q_heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    new = _lengths(b, 1, c["new_max"])
    past = _lengths(b, 0, c["past_max"])
    table, pool = _tables(g, [m + n for m, n in zip(past, new)], ps)
    tokens = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    # the projection's output rows [q | k | v]: strided views of one buffer, as a decoder layer has them
    qkv = _randn(g, tokens, (hq + 2 * hkv) * hd, dtype=dt)
    top = max(m + n for m, n in zip(past, new)) + 100
    inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    ang = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    width = table.shape[1] * ps
    s = dict(q=qkv[:, :hq * hd].view(tokens, hq, hd), k=qkv[:, hq * hd:(hq + hkv) * hd].view(tokens, hkv, hd),
             v=qkv[:, (hq + hkv) * hd:].view(tokens, hkv, hd), cu=_ints(cu), lengths=_ints(past),
             positions=_ints([m + 100 * (i % 2) for i, m in enumerate(past)]),  # some sequences were cut before
             cos=ang.cos().float(), sin=ang.sin().float(), table=table,
             k_pages=_randn(g, pool, hkv, ps, hd, dtype=dt), v_pages=_randn(g, pool, hkv, ps, hd, dtype=dt),
             q_out=torch.zeros(tokens, hq, hd, dtype=dt, device="cuda"),
             lengths_out=torch.zeros(b, dtype=torch.int32, device="cuda"),
             positions_out=torch.zeros(b, dtype=torch.int32, device="cuda"))
    if c["track"]:
        s["slot_positions"] = torch.zeros(b, hkv, width, dtype=torch.int32, device="cuda")
        s["weights"] = _randn(g, b, hkv, width).abs()
    return s


def _prepare_attention(c, g):
    dt, b = _DTYPES[c["dtype"]], c["batch"]
    hq, hkv, hd, ps = c["q_heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    lens = _lengths(b, c["len_min"], c["len_max"])
    table, pool = _tables(g, lens, ps)
    s = dict(q=_randn(g, b, hq, hd, dtype=dt), table=table, lengths=_ints(lens),
             k_pages=_randn(g, pool, hkv, ps, hd, dtype=dt), v_pages=_randn(g, pool, hkv, ps, hd, dtype=dt),
             out=torch.zeros(b, hq, hd, dtype=dt, device="cuda"))
    if c["track"]:
        s["weights"] = _randn(g, b, hkv, table.shape[1] * ps).abs() * 0.01
    return s


def _prepare_evict(c, g):
    dt, b = _DTYPES[c["dtype"]], c["batch"]
    hkv, hd, ps = c["kv_heads"], c["head_dim"], c["page_size"]
    lens = _lengths(b, c["len_min"], c["len_max"])
    table, pool = _tables(g, lens, ps)
    width = table.shape[1] * ps
    # sums of attention weights: a heavy tail, and tokens that nothing has looked at yet
    w = torch.exp(1.5 * _randn(g, b, hkv, width))
    w[torch.rand(b, hkv, width, generator=g, device="cuda") < 0.05] = 0
    # slots hold tokens in no order: earlier evictions moved them
    pos = torch.argsort(torch.rand(b, hkv, width, generator=g, device="cuda"), dim=-1)
    near = torch.arange(width, device="cuda").expand(b, hkv, width)
    lens_t = _ints(lens)
    pos = torch.argsort(torch.where(near < lens_t[:, None, None], pos, pos + width), dim=-1).argsort(dim=-1)
    return dict(table=table, lengths=lens_t, positions=lens_t.clone(), weights=w, slot_positions=pos.to(torch.int32),
                k_pages=_randn(g, pool, hkv, ps, hd, dtype=dt), v_pages=_randn(g, pool, hkv, ps, hd, dtype=dt),
                weights_out=torch.zeros_like(w), slot_positions_out=torch.zeros_like(pos, dtype=torch.int32),
                lengths_out=torch.zeros_like(lens_t))


def _prepare_beam(c, g):
    dt, b, w, ps, n = _DTYPES[c["dtype"]], c["batch"], c["beams"], c["page_size"], c["length"]
    full = n // ps
    width = full + 2  # the partly filled page and one more that is reserved
    pool = b * full + 2 * b * w + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    shared = order[:b * full].view(b, 1, full).expand(b, w, full)
    mine = order[b * full:b * full + 2 * b * w].view(b, w, 2)
    table = torch.cat([shared, mine], dim=2).reshape(b * w, width).contiguous()
    done = torch.zeros(b, w, dtype=torch.int32, device="cuda")
    if c["finished"]:
        done = (torch.rand(b, w, generator=g, device="cuda") < 0.2).to(torch.int32)
    return dict(logits=(3.0 * _randn(g, b, w, c["vocab"])).to(dt), scores=-20.0 + 2.0 * _randn(g, b, w), done=done,
                pages=_randn(g, c["layers"], 2, pool, c["kv_heads"], ps, c["head_dim"], dtype=dt), table=table,
                lengths=_ints([n] * b), eos=2, pad=0,
                scores_out=torch.zeros(b, w, device="cuda"), parents=torch.zeros(b, w, dtype=torch.int32, device="cuda"),
                tokens=torch.zeros(b, w, dtype=torch.int32, device="cuda"),
                done_out=torch.zeros(b, w, dtype=torch.int32, device="cuda"), table_out=torch.zeros_like(table))


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _bind_append(c, s):
    return _package().PagedAppend(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["lengths_out"],
                                  q=s["q"], q_out=s["q_out"], cos=s["cos"], sin=s["sin"], positions=s["positions"],
                                  positions_out=s["positions_out"], starts=s["cu"],
                                  slot_positions=s.get("slot_positions"), weights=s.get("weights"))


def _bind_attention(c, s):
    return _package().PagedAttention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["out"],
                                     weights=s.get("weights"))


def _bind_evict(c, s):
    return _package().PagedEvict(s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["weights"],
                                 s["slot_positions"], s["positions"], s["weights_out"], s["slot_positions_out"],
                                 s["lengths_out"], budget=c["budget"], recent=c["recent"], sink=c["sink"])


def _bind_beam(c, s):
    p = _package()
    select = p.BeamSelect(s["logits"], s["scores"], s["scores_out"], s["parents"], s["tokens"], done=s["done"],
                          done_out=s["done_out"], eos=s["eos"], pad=s["pad"])
    reorder = p.BeamReorder(s["pages"], s["table"], s["lengths"], s["parents"], s["table_out"])

    def call():
        select()
        reorder()

    return call


def _outputs(s):
    op = s["case"]["op"]
    names = {"append": ["k_pages", "v_pages", "q_out", "lengths_out", "positions_out", "slot_positions", "weights"],
             "attention": ["out", "weights"],
             "evict": ["k_pages", "v_pages", "weights_out", "slot_positions_out", "lengths_out"],
             "beam": ["pages", "table_out", "scores_out", "parents", "tokens", "done_out"]}[op]
    return {n: s[n] for n in names if n in s}


def run(state):
    if own:
        state["call"]()
    else:
        globals()["_plain_" + state["case"]["op"]](state)
    return _outputs(state)


# ---- plain forms --------------------------------------------------------------------------------------------------------

def _rotate(x, cos, sin):
    """x [tokens, heads, head_dim], halves rotated against one another, in 32 bits, rounded once."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def _plain_append(s):
    cu, ps = s["cu"].long(), s["k_pages"].shape[2]
    tokens = s["k"].shape[0]
    t = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(cu, t, right=True) - 1
    off = t - cu[row]
    slot = s["lengths"].long()[row] + off
    pos = s["positions"].long()[row] + off
    page = s["table"][row, slot // ps].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    s["q_out"].copy_(_rotate(s["q"], cos, sin))
    s["k_pages"][page, :, slot % ps] = _rotate(s["k"], cos, sin)
    s["v_pages"][page, :, slot % ps] = s["v"]
    new = (cu[1:] - cu[:-1]).to(torch.int32)
    torch.add(s["lengths"], new, out=s["lengths_out"])
    torch.add(s["positions"], new, out=s["positions_out"])
    if "weights" in s:
        s["slot_positions"][row, :, slot] = pos.to(torch.int32)[:, None].expand(-1, s["k"].shape[1])
        s["weights"][row, :, slot] = 0.0


def _rows_of(pages, table, count):
    """The first `count` slots of every sequence, in 32 bits: [rows, kv_heads, count, head_dim]."""
    ps = pages.shape[2]
    j = torch.arange(count, device=pages.device)
    page = table[:, j // ps].long()
    return pages[page, :, (j % ps)[None, :]].transpose(1, 2).float()


def _plain_attention(s):
    q, hkv = s["q"].float(), s["k_pages"].shape[1]
    b, hq, hd = q.shape
    n = max(1, min(s["case"]["len_max"], s["table"].shape[1] * s["k_pages"].shape[2]))
    valid = torch.arange(n, device="cuda")[None, :] < s["lengths"][:, None]
    k = _rows_of(s["k_pages"], s["table"], n)
    sc = torch.matmul(q.view(b, hkv, hq // hkv, hd) * (1.0 / math.sqrt(hd)), k.transpose(2, 3))
    del k
    sc = sc.masked_fill(~valid[:, None, None, :], -math.inf)
    top = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p, _rows_of(s["v_pages"], s["table"], n))
    s["out"].copy_(o.view(b, hq, hd).to(s["out"].dtype))
    if "weights" in s:
        s["weights"][:, :, :n] += p.sum(dim=2)


def _plain_evict(s):
    c, table, ps = s["case"], s["table"], s["k_pages"].shape[2]
    b, h, width = s["weights"].shape
    budget = c["budget"]
    n = s["lengths"].long()
    j = torch.arange(width, device="cuda").expand(b, h, width)
    valid = j < n[:, None, None]
    p = s["slot_positions"].long()
    safe = valid & ((p >= (s["positions"].long() - c["recent"])[:, None, None]) | (p < c["sink"]))
    rank_by = torch.where(safe, math.inf, torch.where(valid, s["weights"].double(), -math.inf))
    order = torch.sort(rank_by, dim=-1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(2, order, j)  # each slot's rank, the heaviest first
    left = n.clamp_max(budget)
    keep = valid & (place < left[:, None, None])
    inside = j < left[:, None, None]
    hole, source = inside & ~keep, keep & ~inside
    # the i-th hole takes the i-th source
    nth_source = torch.where(source, source.cumsum(-1) - 1, width)
    where_source = torch.zeros(b, h, width + 1, dtype=torch.long, device="cuda").scatter_(2, nth_source, j)
    from_slot = torch.where(hole, torch.gather(where_source, 2, (hole.cumsum(-1) - 1).clamp_min(0)), j)
    for name in ("weights", "slot_positions"):
        torch.where(inside, torch.gather(s[name], 2, from_slot), s[name + "_out"], out=s[name + "_out"])
    s["lengths_out"].copy_(left)
    bi, hi, ji = hole.nonzero(as_tuple=True)
    si = from_slot[bi, hi, ji]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[table[bi, ji // ps].long(), hi, ji % ps] = pages[table[bi, si // ps].long(), hi, si % ps]


def _plain_beam(s):
    b, w, vocab = s["logits"].shape
    ps = s["pages"].shape[4]
    # 64 bits: candidates next to one another decide which tokens come out
    x = s["logits"].double()
    top = x.amax(dim=-1, keepdim=True)
    logp = x - top - torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))
    cand = s["scores"].double()[:, :, None] + logp
    done = s["done"].bool()
    only = torch.full_like(cand, -math.inf)
    only[:, :, s["pad"]] = s["scores"].double()
    cand = torch.where(done[:, :, None], only, cand).view(b, w * vocab)
    best = torch.sort(cand, dim=-1, descending=True, stable=True)
    val, idx = best.values[:, :w], best.indices[:, :w]
    parent, token = idx // vocab, idx % vocab
    none = torch.isinf(val)
    s["scores_out"].copy_(val)
    s["parents"].copy_(torch.where(none, 0, parent))
    s["tokens"].copy_(torch.where(none, s["pad"], token))
    s["done_out"].copy_(none | (token == s["eos"]) | torch.gather(done, 1, parent))
    # the new beams' states: a parent's first child takes its partly filled page, further children copy it into the
    # pages of beams without a child
    parent = s["parents"].long()
    beam = torch.arange(w, device="cuda")
    before = (parent[:, :, None] == parent[:, None, :]) & (beam[None, :] < beam[:, None])
    first = ~before.any(dim=2)
    childless = ~(parent[:, :, None] == beam).any(dim=1)
    nth = torch.cumsum(~first, dim=1) - 1
    free = torch.argsort((~childless).to(torch.int32), dim=1, stable=True)
    takes = torch.where(first, parent, torch.gather(free, 1, nth.clamp_min(0)))
    rows = s["table"].view(b, w, -1).long()
    n = s["lengths"].long()[:, None, None]
    at = torch.arange(rows.shape[2], device="cuda")[None, None, :]
    take = lambda which: torch.gather(rows, 1, which[:, :, None].expand(-1, -1, rows.shape[2]))  # noqa: E731
    tail = (at == n // ps) & (n % ps != 0)
    new = torch.where(at < n // ps, take(parent), torch.where(tail, take(takes), rows))
    s["table_out"].copy_(new.view(b * w, -1))
    bi, wi = ((~first) & (n[:, :, 0] % ps != 0)).nonzero(as_tuple=True)
    at = s["lengths"].long()[bi] // ps
    src, dst = rows[bi, parent[bi, wi], at], new[bi, wi, at]
    fill = s["case"]["length"] % ps
    s["pages"][:, :, dst, :, :fill] = s["pages"][:, :, src, :, :fill]


# ---- what one pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    c, e = case, _ITEM[case["dtype"]]
    hd, ps, hkv, b = c["head_dim"], c["page_size"], c["kv_heads"], c["batch"]
    if c["op"] == "append":
        tokens = sum(_lengths(b, 1, c["new_max"]))
        rows = tokens * (c["q_heads"] + 2 * hkv)
        return {"bytes": 2 * rows * hd * e + tokens * (hd * 4 + 4) + (8 * tokens * hkv if c["track"] else 0),
                "flops": 3 * tokens * (c["q_heads"] + hkv) * hd}
    if c["op"] == "attention":
        lens = _lengths(b, c["len_min"], c["len_max"])
        keys = sum(lens)
        return {"bytes": 2 * keys * hkv * hd * e + 2 * b * c["q_heads"] * hd * e + 4 * sum(_pages_of(lens, ps)) +
                (8 * keys * hkv if c["track"] else 0),
                "flops": 4 * keys * c["q_heads"] * hd}
    if c["op"] == "evict":
        lens = _lengths(b, c["len_min"], c["len_max"])
        # kept tokens are spread evenly over the slots: the share beyond the budget moves
        moved = sum(c["budget"] * (n - c["budget"]) / n for n in lens if n > c["budget"])
        kept = sum(min(n, c["budget"]) for n in lens)
        return {"bytes": hkv * (8 * sum(lens) + 8 * kept + 4 * moved * hd * e), "flops": 4 * hkv * sum(lens)}
    w = c["beams"]
    copies = b * w * (1 - 1 / w) ** w if c["length"] % ps else 0
    return {"bytes": b * w * c["vocab"] * e + 4 * copies * c["layers"] * hkv * (c["length"] % ps) * hd * e,
            "flops": 4 * b * w * c["vocab"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](case, s)


def _exact_append(c, s):
    ps, hd = c["page_size"], c["head_dim"]
    out = {"k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double(),
           "q_out": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    if c["track"]:
        out["slot_positions"], out["weights"] = s["slot_positions"].clone(), s["weights"].double()
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    cu, past, first = s["cu"].tolist(), s["lengths"].tolist(), s["positions"].tolist()

    def turned(x, pos):
        z = torch.complex(x[..., :hd // 2].double(), x[..., hd // 2:].double()) * turn[pos][:, None]
        return torch.cat([z.real, z.imag], dim=-1)

    for b in range(c["batch"]):
        part = slice(cu[b], cu[b + 1])
        m = cu[b + 1] - cu[b]
        pos = torch.arange(first[b], first[b] + m, device="cuda")
        out["q_out"][part] = turned(s["q"][part], pos)
        at = torch.arange(past[b], past[b] + m, device="cuda")
        flat = s["table"][b].long()[at.div(ps, rounding_mode="floor")], at.remainder(ps)
        out["k_pages"].transpose(1, 2)[flat] = turned(s["k"][part], pos)
        out["v_pages"].transpose(1, 2)[flat] = s["v"][part].double()
        if c["track"]:
            out["slot_positions"][b, :, past[b]:past[b] + m] = pos.to(torch.int32)
            out["weights"][b, :, past[b]:past[b] + m] = 0
    count = torch.tensor([cu[b + 1] - cu[b] for b in range(c["batch"])], dtype=torch.int32, device="cuda")
    out["lengths_out"], out["positions_out"] = s["lengths"] + count, s["positions"] + count
    return out


def _exact_attention(c, s):
    hkv, hd, ps = c["kv_heads"], c["head_dim"], c["page_size"]
    group = c["q_heads"] // hkv
    out = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    if c["track"]:
        out["weights"] = s["weights"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // ps)].long()
        k, v = (s[name][pages].double().permute(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :n] for name in ("k_pages", "v_pages"))
        q = s["q"][b].double().view(hkv, group, hd)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(hd), dim=-1)
        out["out"][b] = torch.einsum("hgn,hnd->hgd", p, v).reshape(-1, hd)
        if c["track"]:
            out["weights"][b, :, :n] += p.sum(dim=1)
    return out


def _exact_evict(c, s):
    ps, budget = c["page_size"], c["budget"]
    kept_lengths = [min(n, budget) for n in s["lengths"].tolist()]
    out = {"k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double(), "weights_out": s["weights_out"].double(),
           "slot_positions_out": s["slot_positions_out"].clone(),
           "lengths_out": torch.tensor(kept_lengths, dtype=torch.int32, device="cuda")}
    weights, where, table = s["weights"].cpu().numpy(), s["slot_positions"].cpu().numpy(), s["table"].cpu().numpy()
    rows, to, taken = [], [], []
    for b, (n, nxt) in enumerate(zip(s["lengths"].tolist(), s["positions"].tolist())):
        m = kept_lengths[b]
        for h in range(c["kv_heads"]):
            w, p = weights[b, h, :n].astype("f8"), where[b, h, :n]
            must = (p >= nxt - c["recent"]) | (p < c["sink"])
            w[must] = math.inf
            keep = set((-w).argsort(kind="stable")[:m].tolist())
            src = list(range(m))
            spare = iter(sorted(i for i in keep if i >= m))
            for i in range(m):
                if i not in keep:
                    src[i] = next(spare)
                    rows.append((b, h))
                    to.append(i)
                    taken.append(src[i])
            out["weights_out"][b, h, :m] = torch.from_numpy(weights[b, h, src].astype("f8")).cuda()
            out["slot_positions_out"][b, h, :m] = torch.from_numpy(where[b, h, src]).cuda()
    if rows:
        bh = torch.tensor(rows, device="cuda")
        to, taken = torch.tensor(to, device="cuda"), torch.tensor(taken, device="cuda")
        page = torch.from_numpy(table).cuda().long()
        for name in ("k_pages", "v_pages"):
            old = out[name].clone()
            out[name][page[bh[:, 0], to // ps], bh[:, 1], to % ps] = old[page[bh[:, 0], taken // ps], bh[:, 1], taken % ps]
    return out


def _exact_beam(c, s):
    b, w, vocab, ps, n = c["batch"], c["beams"], c["vocab"], c["page_size"], c["length"]
    pages, table_out = s["pages"].double(), s["table"].clone()
    table = s["table"].tolist()
    scores, parents, tokens, flags = [], [], [], []
    done = s["done"].tolist()
    for i in range(b):
        got = []
        for j in range(w):
            base = float(s["scores"][i, j])
            if done[i][j]:
                got.append((-base, j * vocab + s["pad"]))
                continue
            lp = torch.log_softmax(s["logits"][i, j].double(), dim=-1)
            least = torch.topk(lp, min(w, vocab)).values[-1]
            at = torch.nonzero(lp >= least).view(-1)
            got += [(-(base + x), j * vocab + t) for x, t in zip(lp[at].tolist(), at.tolist())]
        got = sorted(got)[:w]
        scores.append([-x for x, _ in got])
        parents.append([k // vocab for _, k in got])
        tokens.append([k % vocab for _, k in got])
        flags.append([int(t == s["eos"] or done[i][p] == 1) for p, t in zip(parents[-1], tokens[-1])])
        unused = [j for j in range(w) if j not in parents[-1]]
        full, seen = n // ps, set()
        for j, p in enumerate(parents[-1]):
            mine = i * w + j
            table_out[mine, :full] = s["table"][i * w + p, :full]
            if n % ps == 0:
                continue
            if p not in seen:
                seen.add(p)
                table_out[mine, full] = table[i * w + p][full]
            else:
                to = table[i * w + unused.pop(0)][full]
                table_out[mine, full] = to
                pages[:, :, to, :, :n % ps] = pages[:, :, table[i * w + p][full], :, :n % ps]
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"pages": pages, "table_out": table_out, "scores_out": torch.tensor(scores, dtype=torch.float64, device="cuda"),
            "parents": whole(parents), "tokens": whole(tokens), "done_out": whole(flags)}
