"""Host-side checks of the paged-cache operators, and their fp64 statements (no GPU needed).

The C entry points check their arguments before any CUDA call, so dummy non-null pointers are never dereferenced; the
Python classes check shapes, types and overlaps before they ask for a CUDA device.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as ref

P = 1 << 20  # a non-null, 16-byte aligned dummy address


def _kv(**kw):
    from backend import _native as nat

    base = dict(k_pages=P, v_pages=P, page_stride=2 * 16 * 64, table=P, table_stride=4, rows=3, max_pages=4, num_pages=12,
                page_size=16, kv_heads=2, head_dim=64)
    return nat.PagedKV(**{**base, **kw})


def _status(name, args, dtype=1, ws=True):
    from backend import _native as nat

    fn = getattr(nat.lib, name)
    extra = ()
    if name + "_workspace_bytes" in nat.EXPORTS:
        extra = (P if ws else None, 1 << 40 if ws else 0)
    rc = fn(ctypes.byref(args), dtype, *extra, None)
    return rc, nat.lib.pim_last_error().decode()


BAD_KV = [(dict(k_pages=None), "null pages"), (dict(table=None), "null pages"), (dict(page_size=24), "page_size"),
          (dict(page_size=512), "page_size"), (dict(head_dim=96), "head_dim"), (dict(kv_heads=0), "kv_heads"),
          (dict(rows=0), "bad rows"), (dict(num_pages=0), "bad rows"), (dict(max_pages=0), "bad rows"),
          (dict(table_stride=3), "table_stride"), (dict(page_stride=2047), "page_stride"),
          (dict(page_stride=2049), "aligned"), (dict(k_pages=P + 8), "aligned"),
          (dict(max_pages=1 << 27, table_stride=1 << 27), "2^30")]


def _attention(kv=None, **kw):
    from backend import _native as nat

    base = dict(kv=kv or _kv(), q=P, out=P, q_stride=256, out_stride=256, lengths=P, q_heads=4)
    return nat.PagedAttentionArgs(**{**base, **kw})


def _append(kv=None, **kw):
    from backend import _native as nat

    base = dict(kv=kv or _kv(), k=P, v=P, k_stride=128, v_stride=128, k_head_stride=64, v_head_stride=64, tokens=3,
                lengths=P)
    return nat.PagedAppendArgs(**{**base, **kw})


def _evict(kv=None, **kw):
    from backend import _native as nat

    base = dict(kv=kv or _kv(), lengths=P, positions=P, weights=P, slot_positions=P, weights_out=P, slot_positions_out=P,
                lengths_out=P + 64, state_row_stride=128, state_head_stride=64, budget=16)
    return nat.PagedEvictArgs(**{**base, **kw})


@pytest.mark.parametrize("kw,message", BAD_KV)
@pytest.mark.parametrize("name,make", [("pim_paged_attention", _attention), ("pim_paged_append", _append),
                                       ("pim_paged_evict", _evict)])
def test_bad_pages_are_refused_before_any_cuda_call(name, make, kw, message):
    rc, said = _status(name, make(_kv(**kw)))
    assert rc == 1 and message in said and said.startswith(name), said


@pytest.mark.parametrize("kw,message", [
    (dict(q=None), "null q"), (dict(lengths=None), "null q"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(q_stride=255), "stride"), (dict(out_stride=260), "aligned"), (dict(out=P + 2), "aligned"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(weights=P, weights_head_stride=63, weights_row_stride=128), "weights strides"),
    (dict(weights=P, weights_head_stride=64, weights_row_stride=127), "weights strides")])
def test_attention_refusals(kw, message):
    from backend import _native as nat

    a = _attention(**kw)
    rc, said = _status("pim_paged_attention", a)
    assert rc == 1 and message in said, said
    assert nat.lib.pim_paged_attention_workspace_bytes(ctypes.byref(a), 1) == -1
    assert _status("pim_paged_attention", _attention(), dtype=2)[0] == 1


def test_attention_refuses_grids_beyond_its_index_range():
    rc, said = _status("pim_paged_attention", _attention(_kv(rows=65535, kv_heads=4, page_stride=4 * 16 * 64), q_heads=4096,
                                                         q_stride=4096 * 64, out_stride=4096 * 64))
    assert rc == 1 and "2^27" in said
    rc, said = _status("pim_paged_attention", _attention(_kv(rows=65536)))
    assert rc == 1 and "65535 rows" in said


def test_workspace_follows_the_form():
    """Short rows run in one launch without a workspace; long ones need the partials, and with weights the scores too."""
    from backend import _native as nat

    def need(**kw):
        return nat.lib.pim_paged_attention_workspace_bytes(ctypes.byref(_attention(**kw)), 1)

    assert need() == 0
    long = _kv(max_pages=1000, table_stride=1000)
    plain = need(kv=long)
    assert plain > 0
    tracked = need(kv=long, weights=P, weights_head_stride=16000, weights_row_stride=32000)
    assert tracked >= plain + 3 * 4 * 16000 * 4  # rows x heads x slots, fp32
    rc, said = _status("pim_paged_attention", _attention(kv=long), ws=False)
    assert rc == 1 and "workspace" in said


@pytest.mark.parametrize("kw,message", [
    (dict(tokens=-1), "number of tokens"), (dict(k=None), "null k"), (dict(lengths=None), "null k"),
    (dict(tokens=4), "one token per row"), (dict(q=P), "go together"), (dict(q=P, q_out=P, q_heads=0), "q_heads"),
    (dict(rope_cos=P), "go together"), (dict(rope_cos=P, rope_sin=P), "max_pos"), (dict(weights=P), "go together"),
    (dict(weights=P, slot_positions=P, state_head_stride=64, state_row_stride=64), "state strides"),
    (dict(lengths_out=P), "of their own"), (dict(positions=P + 64, positions_out=P + 64), "of their own"),
    (dict(positions_out=P), "of their own"), (dict(lengths_out=P + 64, positions_out=P + 64), "of their own"),
    (dict(q=P, q_out=P + 4096, q_heads=2, q_stride=64, q_out_stride=128), "q strides"),
    (dict(q=P, q_out=P, q_heads=2, q_stride=128, q_out_stride=128, pair_order=1), "in place"),
    (dict(q=P, q_out=P, q_heads=2, q_stride=128, q_out_stride=256), "in place"),
    (dict(k_stride=129), "aligned"), (dict(v_head_stride=65), "aligned"), (dict(v=P + 4), "aligned")])
def test_append_refusals(kw, message):
    rc, said = _status("pim_paged_append", _append(**kw))
    assert rc == 1 and message in said, said


@pytest.mark.parametrize("kw,message", [
    (dict(weights=None), "null state"), (dict(slot_positions_out=None), "null state"), (dict(lengths_out=P), "of its own"),
    (dict(budget=0), "budget"), (dict(recent=-1), "budget"), (dict(recent=10, sink=7), "budget"),
    (dict(recent=2**31 - 1, sink=2**31 - 1), "budget"), (dict(state_head_stride=63), "state strides"),
    (dict(state_row_stride=127), "state strides")])
def test_evict_refusals(kw, message):
    rc, said = _status("pim_paged_evict", _evict(**kw))
    assert rc == 1 and message in said, said
    rc, said = _status("pim_paged_evict", _evict(), ws=False)
    assert rc == 1 and "workspace" in said


def _beam(**kw):
    from backend import _native as nat

    base = dict(logits=P, logits_stride=1000, scores=P, scores_out=P + 64, parents=P, tokens=P, batch=2, beams=4,
                beams_out=4, vocab=1000, eos=2, pad=0)
    return nat.BeamSelectArgs(**{**base, **kw})


@pytest.mark.parametrize("kw,message", [
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(beams=65), "beams"), (dict(beams_out=0), "beams"),
    (dict(beams_out=65), "beams"), (dict(batch=0), "batch"), (dict(batch=20000), "batch"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 19) + 1, logits_stride=1 << 20), "vocab"), (dict(logits_stride=999), "logits_stride"),
    (dict(logits=P + 1), "aligned"), (dict(eos=1000), "eos"), (dict(pad=-1), "pad"), (dict(pad=1000), "pad"),
    (dict(scores_out=P), "of their own"), (dict(done=P, done_out=P), "of their own")])
def test_beam_select_refusals(kw, message):
    rc, said = _status("pim_beam_select", _beam(**kw))
    assert rc == 1 and message in said, said
    assert _status("pim_beam_select", _beam(), ws=False)[0] == 1


def _reorder(**kw):
    from backend import _native as nat

    base = dict(pages=P, block_stride=12 * 2048, page_stride=2048, table=P, table_out=P + 4096, table_stride=4, lengths=P,
                parents=P, batch=2, beams=4, num_blocks=4, max_pages=4, num_pages=12, page_size=16, kv_heads=2,
                head_dim=64)
    return nat.BeamReorderArgs(**{**base, **kw})


@pytest.mark.parametrize("kw,message", [
    (dict(pages=None), "null"), (dict(parents=None), "null"), (dict(table_out=P), "of its own"), (dict(page_size=10), "page_size"),
    (dict(beams=65), "beams"), (dict(batch=0), "batch"), (dict(num_blocks=0), "counts"), (dict(table_stride=3), "counts"),
    (dict(page_stride=2040), "strides"), (dict(block_stride=8), "strides"), (dict(block_stride=12 * 2048 + 1), "aligned"),
    (dict(pages=P + 8), "aligned")])
def test_beam_reorder_refusals(kw, message):
    rc, said = _status("pim_beam_reorder", _reorder(**kw))
    assert rc == 1 and message in said, said


# ---- the Python classes ---------------------------------------------------------------------------------------------------

def _tensors(rows=3, heads=2, ps=16, hd=64, pages=12, width=4, dt=torch.bfloat16):
    return dict(k_pages=torch.zeros(pages, heads, ps, hd, dtype=dt), v_pages=torch.zeros(pages, heads, ps, hd, dtype=dt),
                table=torch.zeros(rows, width, dtype=torch.int32), lengths=torch.zeros(rows, dtype=torch.int32))


def test_attention_class_checks_shapes_types_and_overlap():
    from backend.cuda_paged import PagedAttention

    t = _tensors()
    q, out = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 4, 64, dtype=torch.bfloat16)

    def make(**kw):
        a = {**t, "q": q, "out": out, **kw}
        return PagedAttention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("table"), a.pop("lengths"),
                              a.pop("out"), **a)

    for kw, message in [(dict(q=q[:2]), "expected shape"), (dict(q=q.float()), "expected bfloat16"),
                        (dict(out=q), "shares memory"), (dict(v_pages=t["k_pages"]), "shares memory"),
                        (dict(v_pages=t["v_pages"][:5]), "k_pages and v_pages"),
                        (dict(k_pages=t["k_pages"].half(), v_pages=t["v_pages"].half()), "expected float16|has no kernel"),
                        (dict(table=t["table"].long()), "expected int32"), (dict(lengths=t["lengths"][:2]), "expected shape"),
                        (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
                        (dict(weights=torch.zeros(3, 2, 63)), "slots a row"), (dict(scale=0.0), "scale"),
                        (dict(k_pages=t["k_pages"].transpose(1, 2)), "k_pages and v_pages|must be contiguous"),
                        (dict(), "needs CUDA tensors")]:
        with pytest.raises(ValueError, match=message):
            make(**kw)


def test_append_class_tells_parts_of_one_row_from_overlap():
    from backend.cuda_paged import PagedAppend

    t = _tensors()
    pages = (t["k_pages"], t["v_pages"], t["table"], t["lengths"])
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    q, k, v = (x.view(3, -1, 64) for x in qkv.split([256, 128, 128], dim=1))
    with pytest.raises(ValueError, match="needs CUDA"):  # in place, beside k and v: everything else is in order
        PagedAppend(k, v, *pages, q=q, q_out=q)
    with pytest.raises(ValueError, match="q_out shares memory with q"):
        PagedAppend(k, v, *pages, q=q, q_out=qkv[:, 64:320].view(3, 4, 64))
    with pytest.raises(ValueError, match="q_out shares memory with k"):
        PagedAppend(k, v, *pages, q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), q_out=qkv[:, 192:448].view(3, 4, 64))
    with pytest.raises(ValueError, match="lengths_out shares memory"):
        PagedAppend(k, v, *pages, t["lengths"])
    with pytest.raises(ValueError, match="go together"):
        PagedAppend(k, v, *pages, q=q)
    with pytest.raises(ValueError, match="3 tokens, k has 2"):
        PagedAppend(k[:2], v, *pages, starts=torch.zeros(3, dtype=torch.int32))


def test_evict_class_takes_its_state_in_place_or_apart():
    from backend.cuda_paged import PagedEvict

    t = _tensors()
    w, p = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, dtype=torch.int32)
    n, out = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    pages = (t["k_pages"], t["v_pages"], t["table"], t["lengths"])
    with pytest.raises(ValueError, match="needs CUDA"):
        PagedEvict(*pages, w, p, n, w, p, out, budget=8)
    big = torch.zeros(3 * 2 * 64 + 8)
    with pytest.raises(ValueError, match="its input or apart"):
        PagedEvict(*pages, big[:384].view(3, 2, 64), p, n, big[8:].view(3, 2, 64), p, out, budget=8)
    with pytest.raises(ValueError, match="strides must be those"):
        PagedEvict(*pages, w, p, n, torch.zeros(3, 2, 70), p, out, budget=8)
    with pytest.raises(ValueError, match="lengths_out shares memory"):
        PagedEvict(*pages, w, p, n, w, p, t["lengths"], budget=8)


def test_beam_classes_check_their_shapes():
    from backend.cuda_paged import BeamReorder, BeamSelect

    lg, sc = torch.zeros(2, 4, 100), torch.zeros(2, 4)
    outs = (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="needs CUDA"):
        BeamSelect(lg, sc, *outs)
    with pytest.raises(ValueError, match="shares memory"):
        BeamSelect(lg, sc, sc, *outs[1:])
    with pytest.raises(ValueError, match="evenly spaced"):
        BeamSelect(torch.zeros(2, 5, 100)[:, :4], sc, *outs)
    with pytest.raises(ValueError, match="expected shape"):
        BeamSelect(lg, sc, outs[0], outs[1][:, :3], outs[2])
    table = torch.zeros(8, 3, dtype=torch.int32)
    pages = torch.zeros(2, 2, 6, 1, 8, 32)
    with pytest.raises(ValueError, match="needs CUDA"):
        BeamReorder(pages, table, torch.zeros(2, dtype=torch.int32), outs[1], table.clone())
    with pytest.raises(ValueError, match="shares memory"):
        BeamReorder(pages, table, torch.zeros(2, dtype=torch.int32), outs[1], table)
    with pytest.raises(ValueError, match="expected shape"):
        BeamReorder(pages, table[:6], torch.zeros(2, dtype=torch.int32), outs[1], table)


# ---- the fp64 statements ----------------------------------------------------------------------------------------------------

def test_oracle_attention_is_softmax_attention():
    rng = np.random.default_rng(0)
    table = np.array([[3, 1], [0, 2]])
    k, v = rng.standard_normal((2, 4, 2, 8, 16))
    q = rng.standard_normal((2, 4, 16))
    for b, (out, p, _, _) in enumerate(ref.attention(q, k, v, table, [11, 16])):
        n = [11, 16][b]
        ks, vs = (torch.tensor(np.repeat(ref.slots(x, table[b], n), 2, 0)) for x in (k, v))
        want = torch.nn.functional.scaled_dot_product_attention(torch.tensor(q[b])[:, None], ks, vs)[:, 0]
        assert np.abs(out - want.numpy()).max() < 1e-12 and np.abs(p.sum(1) - 1).max() < 1e-12


def test_oracle_evict_keeps_what_a_full_sort_keeps():
    rng = np.random.default_rng(1)
    for n, budget, recent, sink in ((30, 12, 3, 2), (30, 12, 12, 0), (12, 12, 0, 0), (13, 12, 0, 0)):
        w, pos = rng.integers(0, 4, n).astype(np.float32), rng.permutation(n)
        src = ref.evict(n, n, w, pos, budget, recent, sink)
        must = {int(i) for i in range(n) if pos[i] >= n - recent or pos[i] < sink}
        rest = sorted((i for i in range(n) if i not in must), key=lambda i: (-w[i], i))
        assert set(src.tolist()) == must | set(rest[:budget - len(must)])
        stay = [i for i in range(budget) if i in set(src.tolist())]
        assert all(src[i] == i for i in stay)


def test_oracle_beam_select_is_the_top_of_all_continuations():
    rng = np.random.default_rng(2)
    lg, sc = rng.standard_normal((3, 20)), rng.standard_normal(3)
    s, p, t, d = ref.beam_select(lg, sc, 6, eos=4)
    full = (torch.log_softmax(torch.tensor(lg), -1) + torch.tensor(sc)[:, None]).flatten()
    best = torch.sort(full, descending=True, stable=True)
    assert np.abs(s - best.values[:6].numpy()).max() < 1e-12
    assert (p * 20 + t).tolist() == best.indices[:6].tolist() and d.tolist() == [int(x == 4) for x in t]


def test_oracle_beam_reorder_gives_every_beam_its_parents_slots():
    rng = np.random.default_rng(3)
    for length, parents in ((13, [2, 2, 0, 2]), (16, [1, 1, 1, 1]), (5, [3, 2, 1, 0])):
        full = length // 8
        table = np.concatenate([np.repeat(np.arange(full)[None], 4, 0), (full + np.arange(8)).reshape(4, 2)], 1)
        pages = rng.standard_normal((2, full + 8, 1, 8, 4))
        after, out = ref.beam_reorder(pages, table, length, np.array(parents))
        for j, p in enumerate(parents):
            for blk in range(2):
                assert np.array_equal(ref.slots(after[blk], out[j], length), ref.slots(pages[blk], table[p], length))
        tails = out[:, full:].flatten().tolist()
        assert sorted(tails) == sorted(table[:, full:].flatten().tolist())  # no page is lost or held twice


def test_pools_that_overlap_are_refused_and_interleaved_ones_are_not():
    """K and V as halves of each page of one buffer share nothing; V half a page behind K does, as do single pages."""
    from backend.cuda_paged import PagedAttention

    heads, ps, hd, num = 2, 16, 64, 6
    page = heads * ps * hd
    t = _tensors(heads=heads, ps=ps, hd=hd)
    q, out = torch.zeros(3, 4, hd, dtype=torch.bfloat16), torch.zeros(3, 4, hd, dtype=torch.bfloat16)
    buf = torch.zeros(3 * num * page, dtype=torch.bfloat16)

    def pool(at, pitch, n=num):
        return buf.as_strided((n, heads, ps, hd), (pitch, ps * hd, hd, 1), at)

    for k, v, ok in ((pool(0, 2 * page), pool(page, 2 * page), True), (pool(page, 2 * page), pool(0, 2 * page), True),
                     (pool(0, 2 * page), pool(page // 2, 2 * page), False), (pool(0, 2 * page), pool(page + 8, 2 * page), False),
                     (pool(0, 3 * page), pool(page + page // 2, 3 * page), True),
                     (pool(0, 2 * page), pool(2 * page, 2 * page), False), (pool(0, page), pool(num * page, page), True),
                     (pool(0, page, 1), pool(page - 8, page, 1), False), (pool(0, page, 1), pool(page, page, 1), True)):
        with pytest.raises(ValueError, match="needs CUDA" if ok else "k_pages shares memory with v_pages"):
            PagedAttention(q, k, v, t["table"], t["lengths"], out)


def test_append_class_keeps_all_that_it_writes_apart():
    from backend.cuda_paged import PagedAppend

    t = _tensors()
    k, v = (torch.zeros(3, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    w, p = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, dtype=torch.int32)
    f = torch.float32
    both = torch.zeros(3, 2, 2, 64)  # [rows, heads, positions | weights, slots]: interleaved, nothing shared
    floats = torch.zeros(12 * 2 * 16 * 64 // 2)
    paged = floats.view(torch.bfloat16).view(12, 2, 16, 64)

    def make(pages=None, **kw):
        a = {**t, **(pages or {})}
        PagedAppend(k, v, a["k_pages"], a["v_pages"], a["table"], a["lengths"], **kw)

    for said, pages, kw in [
            ("needs CUDA", None, dict(slot_positions=p, weights=w)),
            ("needs CUDA", None, dict(slot_positions=both[:, :, 0].view(torch.int32), weights=both[:, :, 1])),
            ("slot_positions shares memory with weights", None, dict(slot_positions=w.view(torch.int32), weights=w)),
            ("slot_positions shares memory with weights", None,
             dict(slot_positions=both.view(3, 2, 128)[:, :, 8:72].view(torch.int32), weights=both[:, :, 0])),
            ("weights shares memory with k_pages", dict(k_pages=paged), dict(slot_positions=p, weights=floats[:384].view(3, 2, 64))),
            ("slot_positions shares memory with v_pages", dict(v_pages=paged),
             dict(slot_positions=floats[:384].view(3, 2, 64).view(torch.int32), weights=w)),
            ("slot_positions shares memory with lengths", dict(lengths=p.view(-1)[:3]), dict(slot_positions=p, weights=w)),
            ("slot_positions shares memory with table", dict(table=p.view(-1)[:12].view(3, 4)), dict(slot_positions=p, weights=w)),
            ("lengths_out shares memory with k_pages", dict(k_pages=paged), dict(lengths_out=floats[:3].view(torch.int32))),
            ("k_pages shares memory with table", dict(k_pages=paged, table=floats.view(torch.int32)[:12].view(3, 4)), {}),
            ("k_pages shares memory with cos", dict(k_pages=paged), dict(cos=floats[:320].view(10, 32), sin=torch.zeros(10, 32, dtype=f))),
            ("q_out shares memory with lengths", dict(lengths=floats[:3].view(torch.int32)),
             dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), q_out=floats.view(torch.bfloat16)[:768].view(3, 4, 64)))]:
        with pytest.raises(ValueError, match=said):
            make(pages, **kw)


def test_evict_and_reorder_classes_keep_the_pages_apart_from_what_they_read():
    from backend.cuda_paged import BeamReorder, PagedEvict

    t = _tensors()
    w, p = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, dtype=torch.int32)
    n, out = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    floats = torch.zeros(12 * 2 * 16 * 64 // 2)
    paged = floats.view(torch.bfloat16).view(12, 2, 16, 64)
    with pytest.raises(ValueError, match="v_pages shares memory with positions"):
        PagedEvict(t["k_pages"], paged, t["table"], t["lengths"], w, p, floats.view(torch.int32)[:3], w.clone(), p.clone(), out, budget=8)
    with pytest.raises(ValueError, match="k_pages shares memory with weights"):
        PagedEvict(paged, t["v_pages"], t["table"], t["lengths"], floats[:384].view(3, 2, 64), p, n, w, p.clone(), out, budget=8)
    pool = torch.zeros(2, 2, 6, 1, 8, 32)
    ints = pool.view(-1).view(torch.int32)
    table, lengths, parents = (torch.zeros(s, dtype=torch.int32) for s in ((8, 3), (2,), (2, 4)))
    for kw, said in ((dict(table=ints[:24].view(8, 3)), "table"), (dict(lengths=ints[:2]), "lengths"),
                     (dict(parents=ints[:8].view(2, 4)), "parents")):
        a = {**dict(table=table, lengths=lengths, parents=parents), **kw}
        with pytest.raises(ValueError, match=f"pages shares memory with {said}"):
            BeamReorder(pool, a["table"], a["lengths"], a["parents"], torch.zeros(8, 3, dtype=torch.int32))


def test_numbers_that_the_argument_structs_cannot_hold_are_refused():
    """A budget of 2^32 + 1 is not one of 1, and a scale that fp32 rounds to 0 is not the default scale."""
    from backend.cuda_paged import BeamSelect, PagedAttention, PagedEvict

    t = _tensors()
    w, p = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, dtype=torch.int32)
    n, out = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    pages = (t["k_pages"], t["v_pages"], t["table"], t["lengths"])
    for kw, said in ((dict(budget=2**32 + 1), "budget"), (dict(budget=9, recent=2**32), "recent"),
                     (dict(budget=9, sink=-2**31 - 1), "sink")):
        with pytest.raises(ValueError, match=f"{said}=.* 32 bits"):
            PagedEvict(*pages, w, p, n, w, p, out, **kw)
    q, o = (torch.zeros(3, 4, 64, dtype=torch.bfloat16) for _ in range(2))
    for scale in (1e-50, 1e39, float("inf"), float("nan"), -1.0):
        with pytest.raises(ValueError, match="scale must be"):
            PagedAttention(q, *pages, o, scale=scale)
    lg, sc = torch.zeros(2, 4, 100), torch.zeros(2, 4)
    outs = (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32))
    for kw, said in ((dict(eos=2**32 + 5), "eos"), (dict(pad=2**32), "pad")):
        with pytest.raises(ValueError, match=f"{said}=.* 32 bits"):
            BeamSelect(lg, sc, *outs, **kw)
