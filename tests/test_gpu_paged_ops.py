"""The paged-cache operators against fp64 statements of the same formulas (GPU).

Tolerances are derived, not tuned: the last rounding costs half a step of the type (``eps / 2`` of the value), and what
comes before it is bounded by the arithmetic stated in ``oracle.paged.attention`` or beside the check.  Pages, tables and
state outside what an operator may touch are compared bit for bit, and slots beyond a row's length hold NaN, so that a
kernel which reads them shows.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0**-24, "bfloat16": 2.0**-8}
EXP = {"float32": 2.0**-21, "bfloat16": 2.0**-17}


def _torch():
    import torch

    return torch


def _tdt(dt):
    torch = _torch()
    return {"float32": torch.float32, "bfloat16": torch.bfloat16}[dt]


def _host(t):
    """fp64 copy of a device tensor (exact for every type used here)."""
    torch = _torch()
    torch.cuda.synchronize()
    return t.detach().to(torch.float64).cpu().numpy()


def _ints(a):
    return _torch().tensor(np.asarray(a), dtype=_torch().int32, device="cuda")


class Pool:
    """Pages of rows with the given numbers of slots in use, in shuffled order; unused slots and pages hold NaN."""

    def __init__(self, lengths, *, heads, ps, hd, dt, seed=0, room=0, spare=3, k_scale=1.0):
        torch = _torch()
        rng = np.random.default_rng(seed)
        need = [-(-(n + room) // ps) for n in lengths]
        self.width = max(max(need), 1)
        total = sum(need) + spare
        order = rng.permutation(total).astype(np.int32)
        table = np.full((len(lengths), self.width), order[-1] if spare else 0, np.int32)
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = order[at:at + m]
            at += m
        self.table_np, self.lengths_np = table, np.asarray(lengths, np.int32)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def pages(scale):
            p = torch.full((total, heads, ps, hd), float("nan"), device="cuda", dtype=_tdt(dt))
            for b, n in enumerate(lengths):
                for i in range(need[b]):
                    m = min(ps, n - i * ps)
                    if m > 0:
                        p[table[b, i], :, :m] = (scale * torch.randn(heads, m, hd, device="cuda", generator=g)).to(p.dtype)
            return p

        self.k, self.v = pages(k_scale), pages(1.0)
        self.table, self.lengths = _ints(table), _ints(lengths)
        self.ps = ps
        self.slots = self.width * ps


# ---- attention ------------------------------------------------------------------------------------------------------------

def _attention_case(lengths, group, heads, ps, hd, dt, seed=0, track=False, scale=None, k_scale=1.0):
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    pool = Pool(lengths, heads=heads, ps=ps, hd=hd, dt=dt, seed=seed, k_scale=k_scale)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(len(lengths), heads * group, hd, device="cuda", generator=g).to(_tdt(dt))
    out = torch.full_like(q, float("nan"))
    w0 = None
    if track:
        w0 = torch.rand(len(lengths), heads, pool.slots + 3, device="cuda", generator=g)[..., :pool.slots]
    weights = None if w0 is None else w0.clone(memory_format=torch.preserve_format)
    op = PagedAttention(q, pool.k, pool.v, pool.table, pool.lengths, out, weights=weights, scale=scale)
    return pool, q, out, w0, weights, op


def _check_attention(pool, q, out, w0, weights, dt, scale=None, lengths=None):
    lengths = pool.lengths_np if lengths is None else lengths
    want = ref.attention(_host(q), _host(pool.k), _host(pool.v), pool.table_np, lengths, scale, EXP[dt])
    got = _host(out)
    heads = pool.k.shape[1]
    for b, (o, p, bound, rel) in enumerate(want):
        tol = HALF[dt] * np.abs(o) + bound + 1e-30
        off = np.abs(got[b] - o)
        assert (off <= tol).all(), (b, lengths[b], float((off / tol).max()), float(off.max()))
        if weights is None:
            continue
        n = lengths[b]
        got_w, old = _host(weights[b]), _host(w0[b])
        add = p.reshape(heads, p.shape[0] // heads, n).sum(1)
        # one rounding of the sum and one per head added to it
        tol = (1 + p.shape[0] // heads) * 2.0**-24 * (old[:, :n] + add) + rel * add
        assert (np.abs(got_w[:, :n] - (old[:, :n] + add)) <= tol).all(), b
        assert np.array_equal(got_w[:, n:], old[:, n:])


# One CTA per unit, a cluster per unit, and the split: by the slots that the table holds.
LENGTHS = {"one": [1, 0, 7, 8, 9, 63, 64, 65, 130, 200, 0, 256], "cluster": [1, 0, 7, 8, 9, 63, 64, 65, 130, 257, 0, 513],
           "split": [1, 0, 7, 8, 9, 63, 64, 65, 130, 257, 0, 4200]}


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group,heads,ps", [(1, 3, 16), (2, 2, 8), (4, 1, 32), (7, 2, 64), (8, 1, 16), (12, 1, 128),
                                            (16, 2, 16), (33, 1, 8)])
@pytest.mark.parametrize("form", list(LENGTHS))
def test_attention_groups_and_dims(form, group, heads, ps, hd, dt, track):
    lengths = LENGTHS[form]
    pool, q, out, w0, weights, op = _attention_case(lengths, group, heads, ps, hd, dt, track=track)
    assert op() is out
    _check_attention(pool, q, out, w0, weights, dt)
    op.check()


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths", [[1], [130], [0], [0, 0, 5, 0], [4090], [4097], [1025], [2, 9001, 1, 3000], [300] * 70,
                                     [1] * 3 + [2000] + [5] * 12])
def test_attention_lengths(lengths, dt, track):
    pool, q, out, w0, weights, op = _attention_case(lengths, 4, 2, 16, 128, dt, seed=3, track=track)
    op()
    _check_attention(pool, q, out, w0, weights, dt)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_attention_many_rows_and_heads(dt):
    rng = np.random.default_rng(5)
    pool, q, out, w0, weights, op = _attention_case(list(rng.integers(0, 200, 150)), 1, 32, 16, 128, dt, seed=5, track=True)
    op()
    _check_attention(pool, q, out, w0, weights, dt)


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,heads,group,most,hd", [(80, 32, 1, 17, 64), (90, 8, 4, 129, 32), (40, 16, 12, 60, 128),
                                                      (90, 27, 2, 65, 128)])
def test_attention_of_many_short_rows(rows, heads, group, most, hd, dt, track):
    """Units by the thousand, of a warp or two each; 12 heads a group make a second, partly filled tile in fp32."""
    lengths = list(np.random.default_rng(rows).integers(0, most, rows))
    pool, q, out, w0, weights, op = _attention_case(lengths, group, heads, 8, hd, dt, seed=6, track=track)
    op()
    _check_attention(pool, q, out, w0, weights, dt)
    op.check()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_attention_of_one_long_row_lies_in_every_cta(dt):
    """A unit in some hundred parts, with and without weights, and keys of -inf that leave whole parts empty."""
    for track in (False, True):
        pool, q, out, w0, weights, op = _attention_case([30011], 3, 1, 16, 64, dt, seed=14, track=track)
        op()
        _check_attention(pool, q, out, w0, weights, dt)
    for page in pool.table_np[0, :1200]:
        pool.k[page, 0, :, 0] = -float("inf")
    q[:] = 0
    q[:, :, 0] = 1
    weights.zero_()
    op()
    v = ref.slots(_host(pool.v), pool.table_np[0], 30011)[0][19200:].astype(np.float64)
    s = ref.slots(_host(pool.k), pool.table_np[0], 30011)[0][19200:, 0].astype(np.float64) / 8
    p = np.exp(s - s.max())
    p /= p.sum()
    want = p @ v
    # as in ref.attention: the scores' roundings, the exponentials', and those of two sums of as many terms
    rel = 2 * (64 + 2) * 2.0**-23 * np.abs(s).max() + EXP[dt] + 2 * len(p) * 2.0**-23
    assert (np.abs(_host(out)[0] - want) <= HALF[dt] * np.abs(want) + rel * (p @ np.abs(v)) + 1e-30).all()
    assert (_host(weights)[0, 0, :19200] == 0).all()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_attention_scale_and_sharp_scores(dt):
    """Scores of tens: all the weight on few keys, and a running maximum that grows along the row."""
    pool, q, out, w0, weights, op = _attention_case([700, 33], 2, 2, 32, 64, dt, seed=8, track=True, scale=0.5,
                                                    k_scale=4.0)
    op()
    _check_attention(pool, q, out, w0, weights, dt, scale=0.5)


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("form,slot", [("one", 70), ("one", 199), ("cluster", 0), ("cluster", 300), ("split", 64),
                                       ("split", 4000)])
def test_attention_nan_in_a_key_comes_out_and_stays_in_its_head(form, slot, dt, track):
    """A NaN key makes its row's outputs of the heads that read it NaN, and their probabilities; nothing else."""
    lengths = {"one": [256, 5], "cluster": [513, 5], "split": [4200, 300, 5] + [1000] * 40}[form]
    pool, q, out, w0, weights, op = _attention_case(lengths, 4, 2, 16, 64, dt, seed=4, track=track)
    pool.k[pool.table_np[0, slot // 16], 1, slot % 16, 3] = float("nan")
    op()
    op.check()
    got = _host(out)
    assert np.isnan(got[0, 4:]).all()
    got[0, 4:] = 0
    assert np.isfinite(got).all()
    if track:
        w = _host(weights)
        assert np.isnan(w[0, 1, :lengths[0]]).all()
        w[0, 1, :lengths[0]] = 0
        assert np.isfinite(w).all()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("group", [1, 5, 12])
@pytest.mark.parametrize("form", ["one", "cluster", "split"])
def test_attention_probabilities_keep_32_bits_where_their_products_cancel(form, group, dt):
    """Three keys of probabilities 1 : p : 2^-10 whose values are such that the sum of p v all but vanishes, so that what is
    left of a probability's rounding shows.  Scores are exact: q is one-hot, keys are short binary fractions and the scale
    is log 2, so a score is a power of two's exponent.  Off by at most, before the last rounding: 2^-22 of p v = 1 (the
    exponential; 2^-24 for the scale's rounding) and six steps of 2^-23 of sums whose terms are 1."""
    torch = _torch()
    heads, hd, rows = 2, 128, 9
    scale = float(np.float32(np.log(2)))
    lengths = [3] * rows + {"one": [200], "cluster": [513], "split": [4200]}[form]
    pool, q, out, w0, weights, op = _attention_case(lengths, group, heads, 16, hd, dt, seed=21, scale=scale)
    rng = np.random.default_rng(group)
    q.zero_()
    q[:, :, 0] = 1
    bf16 = lambda x: torch.tensor(x).to(torch.bfloat16).double().numpy()  # noqa: E731
    for b in range(rows):
        page = int(pool.table_np[b, 0])
        a = rng.integers(1, 256, heads) / 256.0
        p2, p3 = np.exp(-scale * a)[:, None], np.exp(-scale * 10)
        v2 = bf16(bf16(1 / p2) + (np.arange(hd) % 4 - 2) * 2.0**-7)
        v3 = bf16((1 - p2 * v2) / p3)
        for j, (key, value) in enumerate(((0 * a, -np.ones((heads, hd))), (-a, v2), (-10 + 0 * a, v3))):
            pool.k[page, :, j] = 0
            pool.k[page, :, j, 0] = torch.tensor(key, device="cuda").to(pool.k.dtype)
            pool.v[page, :, j] = torch.tensor(value, device="cuda").to(pool.v.dtype)
    op()
    want = ref.attention(_host(q), _host(pool.k), _host(pool.v), pool.table_np, lengths, scale)
    for b in range(rows):
        o, p = want[b][:2]
        one = p.max(1, keepdims=True)  # what a probability of 1 became by the division
        off = np.abs(_host(out)[b] - o) / one
        assert (off <= HALF[dt] * np.abs(o) / one + 2.0**-22 + 2.0**-24 + 6 * 2.0**-23).all(), (b, float(off.max() * 2.0**20))


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("group", [1, 12])
def test_attention_sums_over_long_rows_round_to_nearest(group, dt):
    """Keys of the second half repeat the first half's with V negated: the sum is 0, and what comes out is what its additions
    lost.  A warp adds its keys in up to S = 260 steps (448 units of 256 tiles on 444 CTAs or fewer, twice that where a group
    makes two tiles); rounded to nearest, each is off by at most 2^-24 of a partial sum that grows to half of its share W of
    the row's weight, as if at random: a deviation of 2^-24 / sqrt(3) sqrt(S / 3) W / 2 = 2.7 x 2^-24 W, halved again by the
    four warps (and over more and shorter ones in fp32).  Eight deviations, doubled for units that two CTAs share: 22 x 2^-24.
    Additions that round towards zero lose some 140 x 2^-24 here."""
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    n, ps, hd, rows = 16384, 256, 32, 448
    rng = np.random.default_rng(group)
    key = -rng.integers(0, 257, n // 2) / 256.0
    value = np.where(rng.random((1, hd)) < 0.5, -1.0, 1.0) * np.ones((n // 2, hd))
    key[::8], value[::8] = 0, 0  # every step begins with the largest score: the running maximum never moves
    k = torch.zeros(n, hd, device="cuda")
    k[:, 0] = torch.tensor(np.tile(key, 2), device="cuda")
    v = torch.tensor(np.concatenate([value, -value]), device="cuda")
    k, v = (x.to(_tdt(dt)).view(n // ps, 1, ps, hd) for x in (k, v))
    table = _ints(np.tile(np.arange(n // ps), (rows, 1)))  # all rows read the same pages
    q = torch.zeros(rows, group, hd, device="cuda", dtype=_tdt(dt))
    q[:, :, 0] = 1
    out = torch.full_like(q, float("nan"))
    PagedAttention(q, k, v, table, _ints([n] * rows), out, scale=1.0)()
    assert np.abs(_host(out)).max() <= 2.0**-19, np.abs(_host(out)).max() * 2.0**24


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("group", [1, 6, 12])
@pytest.mark.parametrize("form", ["one", "cluster", "split"])
def test_attention_infinite_values_come_out_as_the_sum_has_them(form, group, dt):
    """An infinite V element that is attended to makes its dim infinite, of both signs NaN; whatever the probability is (here
    also 1 before the division, and powers of two, which short formats hold exactly).  The other dims stay as they are."""
    torch = _torch()
    inf = float("inf")
    lengths = [40, {"one": 200, "cluster": 513, "split": 4200}[form], 9]
    pool, q, out, w0, weights, op = _attention_case(lengths, group, 2, 16, 64, dt, seed=23, scale=float(np.float32(np.log(2))))
    q.zero_()
    q[:, :, 0] = 1
    pool.k[..., 0] = torch.round(pool.k[..., 0] * 2)  # scores are whole powers of two
    n = lengths[1]
    for row, slot, dim, x in ((0, 3, 5, inf), (0, 39, 6, -inf), (1, n - 1, 7, inf), (1, 0, 7, -inf), (1, n // 2, 8, -inf),
                              (2, 0, 9, inf), (2, 8, 9, inf), (2, 4, 10, float("nan"))):
        pool.v[pool.table_np[row, slot // 16], :, slot % 16, dim] = x
    op()
    op.check()
    got = _host(out)
    with np.errstate(invalid="ignore"):
        want = ref.attention(_host(q), _host(pool.k), _host(pool.v), pool.table_np, lengths, np.float32(np.log(2)), EXP[dt])
    for b, (o, _, bound, _) in enumerate(want):
        fine = np.isfinite(o)
        assert (~fine).any() and np.array_equal(got[b][~fine], o[~fine], equal_nan=True), b
        assert (np.abs(got[b][fine] - o[fine]) <= HALF[dt] * np.abs(o[fine]) + bound[fine]).all(), b


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_attention_keys_of_minus_infinity_get_no_weight(dt):
    """A key whose score is -inf (here alone in its first tiles) has probability 0; the row's sum stays finite."""
    torch = _torch()
    pool, q, out, w0, weights, op = _attention_case([200], 1, 1, 16, 64, dt, seed=9, track=True)
    q[:] = 0
    q[:, :, 0] = 1
    for slot in list(range(0, 70)) + [120]:
        pool.k[pool.table_np[0, slot // 16], 0, slot % 16, 0] = -float("inf")
    op()
    got = _host(out)
    k = ref.slots(_host(pool.k), pool.table_np[0], 200)[0]
    v = ref.slots(_host(pool.v), pool.table_np[0], 200)[0]
    s = k[:, 0] / 8.0
    p = np.exp(s - s.max())
    p /= p.sum()
    assert (p[:70] == 0).all()
    want = p @ v
    rel = 2 * 66 * 2.0**-23 * np.abs(s[np.isfinite(s)]).max() + EXP[dt] + 400 * 2.0**-23
    assert (np.abs(got[0, 0] - want) <= HALF[dt] * np.abs(want) + rel * (p @ np.abs(v))).all()
    assert np.array_equal(_host(weights)[0, 0, :70], _host(w0)[0, 0, :70])


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_attention_strided_rows_shared_pages_and_repeats(dt):
    """q and out as parts of wider rows; two rows read the same pages; a second call gives the same bits."""
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    pool = Pool([90, 70], heads=2, ps=16, hd=64, dt=dt, seed=11)
    table = pool.table_np.copy()
    table[1, :4] = table[0, :4]
    pool.table_np, pool.table = table, _ints(table)
    wide = torch.randn(2, 4 + 2, 6, 64, device="cuda").to(_tdt(dt))
    q = wide[:, 1, :4]
    hold = torch.full((2, 8, 64), float("nan"), device="cuda", dtype=_tdt(dt))
    out = hold[:, 2:6]
    op = PagedAttention(q, pool.k, pool.v, pool.table, pool.lengths, out)
    op()
    _check_attention(pool, q, out, None, None, dt)
    assert bool(torch.isnan(hold[:, :2]).all()) and bool(torch.isnan(hold[:, 6:]).all())
    first = out.clone()
    op()
    assert torch.equal(first, out)


def test_attention_bad_pages_and_lengths_raise_the_flag_and_hide_the_slots():
    """A page id outside the pool hides its slots, a length outside the table is clamped; both are reported."""
    torch = _torch()
    pool, q, out, _, _, op = _attention_case([40, 40, 40], 2, 2, 16, 64, "bfloat16", seed=12)
    table = pool.table_np.copy()
    table[0, 1], table[1, 0] = pool.k.shape[0], -1
    pool.table.copy_(_ints(table))
    pool.lengths.copy_(_ints([40, 16, -5]))
    op()
    with pytest.raises(ValueError, match="out of range"):
        op.check()
    op.check()  # cleared
    keep = np.r_[0:16, 32:40]
    k, v = (np.repeat(ref.slots(_host(p), pool.table_np[0], 40)[:, keep], 2, 0) for p in (pool.k, pool.v))
    s = np.einsum("hd,hnd->hn", _host(q)[0], k) / 8.0
    p = np.exp(s - s.max(1, keepdims=True))
    want = np.einsum("hn,hnd->hd", p / p.sum(1, keepdims=True), v)
    # (a coarse bound: the values are what is asked, the arithmetic is held to its bound above)
    assert np.abs(_host(out)[0] - want).max() <= 2 * HALF["bfloat16"] * np.abs(want).max()
    assert not _host(out)[1].any() and not _host(out)[2].any()
    pool.lengths.copy_(_ints([0, 0, 10**6]))
    pool.k.nan_to_num_(), pool.v.nan_to_num_()
    op()
    with pytest.raises(ValueError):
        op.check()
    assert np.isfinite(_host(out)).all()


def test_attention_offsets_beyond_32_bits():
    """Pages behind the 2^31-th element of the pool."""
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    heads, ps, hd = 4, 32, 128
    num = (1 << 31) // (heads * ps * hd) + 40
    k, v = (torch.empty(num, heads, ps, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = np.array([[num - 1 - 2 * i for i in range(6)]], np.int32)
    n = 6 * ps - 5
    for p in (k, v):
        for i in table[0]:
            p[int(i)] = torch.randn(heads, ps, hd, device="cuda").to(torch.bfloat16)
    q = torch.randn(1, heads * 2, hd, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    PagedAttention(q, k, v, _ints(table), _ints([n]), out)()
    small = [_host(p[table[0].tolist()]) for p in (k, v)]
    (o, _, bound, _), = ref.attention(_host(q), *small, np.arange(6)[None], [n])
    assert (np.abs(_host(out)[0] - o) <= HALF["bfloat16"] * np.abs(o) + bound).all()


# ---- append -----------------------------------------------------------------------------------------------------------------

def _rope(hd, top):
    torch = _torch()
    inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    ang = torch.arange(top, dtype=torch.float64)[:, None] * inv[None]
    return ang.cos().float().cuda(), ang.sin().float().cuda()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("pair_order", [False, True])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("hq,heads,hd,ps,new,past", [
    (4, 4, 128, 16, [1], [0]), (4, 2, 64, 8, [5, 0, 17, 1], [3, 9, 0, 40]), (3, 1, 32, 32, [0, 0, 70], [1, 2, 31]),
    (32, 32, 128, 16, [1] * 9, list(range(9))), (8, 1, 128, 256, [300, 1], [0, 255])])
def test_append(hq, heads, hd, ps, new, past, rotate, pair_order, dt):
    from backend.cuda_paged import PagedAppend

    torch = _torch()
    rows = len(new)
    pool = Pool([0] * rows, heads=heads, ps=ps, hd=hd, dt=dt, seed=1, room=max(m + n for m, n in zip(past, new)) + 1)
    before = [p.clone() for p in (pool.k, pool.v)]
    tokens = sum(new)
    pad = 3  # tokens behind the last row: left out
    torch.manual_seed(hq + hd + tokens)
    qkv = torch.randn(tokens + pad, (hq + 2 * heads) * hd, device="cuda").to(_tdt(dt))
    q, k, v = (x.view(tokens + pad, -1, hd) for x in qkv.split([hq * hd, heads * hd, heads * hd], dim=1))
    starts = np.r_[0, np.cumsum(new)].astype(np.int32)
    positions = np.asarray(past) + 7 * (np.arange(rows) % 2)
    cos, sin = _rope(hd, int(max(positions + new)) + 1) if rotate else (None, None)
    q_out = torch.full((tokens + pad, hq, hd), 5.0, device="cuda", dtype=_tdt(dt))
    lengths_out, positions_out = _ints([-1] * rows), _ints([-1] * rows)
    slot_positions = torch.full((rows, heads, pool.slots), -9, dtype=torch.int32, device="cuda")
    weights = torch.full((rows, heads, pool.slots), 3.0, device="cuda")
    op = PagedAppend(k, v, pool.k, pool.v, pool.table, _ints(past), lengths_out, q=q, q_out=q_out, cos=cos, sin=sin,
                     positions=_ints(positions), positions_out=positions_out, starts=_ints(starts),
                     slot_positions=slot_positions, weights=weights, pair_order=pair_order)
    op()
    op.check()
    c, s = (None, None) if cos is None else (_host(cos), _host(sin))
    args = (pool.table_np, past, starts, positions, _host(q), _host(k), _host(v))
    wk, wv, wq = ref.append(_host(before[0]), _host(before[1]), *args, c, s, pair_order)
    # |x1 c - x2 s| in fp32: two rounded products and their sum, each off by 2^-24 of at most |x1 c| + |x2 s|
    # (and c, s are of one angle: |x1 c| + |x2 s| <= sqrt 2 max |x|)
    mk, mv, mq = (4.0 * 2.0**-24 * 2.0**0.5 * float(qkv.float().abs().max()) if rotate else 0.0,) * 3
    for got, want, m in ((pool.k, wk, mk), (pool.v, wv, mv)):
        got = _host(got)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        ok = ~np.isnan(want)
        assert (np.abs(got - want)[ok] <= HALF[dt] * np.abs(want)[ok] + m).all()
    assert np.array_equal(_host(pool.v)[~np.isnan(wv)], wv[~np.isnan(wv)])  # v is copied
    got = _host(q_out)
    assert (np.abs(got - wq)[:tokens] <= HALF[dt] * np.abs(wq)[:tokens] + mq).all() and (got[tokens:] == 5.0).all()
    assert _host(lengths_out).tolist() == [m + n for m, n in zip(past, new)]
    assert _host(positions_out).tolist() == (positions + new).tolist()
    for b in range(rows):
        at = np.full(pool.slots, -9.0)
        at[past[b]:past[b] + new[b]] = positions[b] + np.arange(new[b])
        assert (_host(slot_positions)[b] == at).all()
        assert (_host(weights)[b] == np.where(at == -9, 3.0, 0.0)).all()


def test_append_one_token_a_row_in_place_and_from_a_contiguous_block():
    """Without starts: a token per row, q rotated in place; then K / V taken from [heads][k|v][seq][dim] blocks."""
    from backend.cuda_paged import PagedAppend

    torch = _torch()
    hd, heads, rows = 64, 2, 5
    past = [0, 7, 8, 15, 16]
    pool = Pool([0] * rows, heads=heads, ps=8, hd=hd, dt="float32", room=40)
    q, k, v = (torch.randn(rows, n, hd, device="cuda") for n in (6, heads, heads))
    cos, sin = _rope(hd, 40)
    want = ref.append(_host(pool.k), _host(pool.v), pool.table_np, past, np.arange(rows + 1), past, _host(q), _host(k),
                      _host(v), _host(cos), _host(sin))
    op = PagedAppend(k, v, pool.k, pool.v, pool.table, _ints(past), q=q, q_out=q, cos=cos, sin=sin)
    op()
    op.check()
    for got, w in zip((pool.k, pool.v, q), want):
        got, ok = _host(got), ~np.isnan(w)
        assert np.array_equal(np.isnan(got), np.isnan(w))
        assert (np.abs(got - w)[ok] <= HALF["float32"] * np.abs(w)[ok] + 4 * 2.0**-24 * 8.0).all()
    block = torch.randn(heads, 2, 30, hd, device="cuda")
    pool = Pool([0], heads=heads, ps=8, hd=hd, dt="float32", room=40)
    PagedAppend(block[:, 0, :21].transpose(0, 1), block[:, 1, :21].transpose(0, 1), pool.k, pool.v, pool.table,
                _ints([3]), starts=_ints([0, 21]))()
    for pages, i in ((pool.k, 0), (pool.v, 1)):
        assert np.array_equal(ref.slots(_host(pages), pool.table_np[0], 24)[:, 3:], _host(block[:, i, :21]))


def test_append_leaves_out_what_does_not_fit():
    """A slot beyond the table, a page id outside the pool and a position outside the rotary table: reported, and
    neither written nor rotated; the other rows' tokens are."""
    from backend.cuda_paged import PagedAppend

    torch = _torch()
    pool = Pool([0] * 4, heads=1, ps=8, hd=32, dt="float32", room=16)
    table = pool.table_np.copy()
    table[1, 0] = pool.k.shape[0]
    pool.table.copy_(_ints(table))
    k = torch.randn(4, 1, 32, device="cuda")
    q = torch.randn(4, 1, 32, device="cuda")
    q_out = torch.zeros_like(q)
    cos, sin = _rope(32, 10)
    op = PagedAppend(k, k.clone(), pool.k, pool.v, pool.table, _ints([16, 3, 2, 4]), q=q, q_out=q_out, cos=cos, sin=sin,
                     positions=_ints([1, 1, 10, 9]))
    op()
    with pytest.raises(ValueError, match="out of range"):
        op.check()
    written = ~torch.isnan(pool.v).all(dim=-1)
    assert int(written.sum()) == 1 and bool(written[int(table[3, 0]), 0, 4])
    assert not _host(q_out)[:3].any() and _host(q_out)[3].any()


@pytest.mark.parametrize("outs", [True, False])
def test_append_reports_starts_that_decrease(outs):
    """Rows never lose slots by them, and what is written stays within the rows' new slots."""
    from backend.cuda_paged import PagedAppend

    torch = _torch()
    past, rows = [4, 5, 6], 3
    for starts in ([0, 5, 3, 8], [0, -1, 2, 8], [8, 8, 8, 0], [2, 1, 1, 8], [0, 9, 8, 8]):
        pool = Pool([0] * rows, heads=1, ps=8, hd=32, dt="float32", room=24)
        k = torch.randn(8, 1, 32, device="cuda")
        lengths_out, positions_out = (_ints([-1] * rows) for _ in range(2)) if outs else (None, None)
        op = PagedAppend(k, k.clone(), pool.k, pool.v, pool.table, _ints(past), lengths_out, positions=_ints([9, 9, 9]),
                         positions_out=positions_out, starts=_ints(starts))
        op()
        with pytest.raises(ValueError, match="out of range"):
            op.check()
        new = np.maximum(np.diff(starts), 0)
        if outs:
            assert lengths_out.tolist() == (past + new).tolist() and positions_out.tolist() == (9 + new).tolist()
        for b in range(rows):
            written = ~np.isnan(ref.slots(_host(pool.v), pool.table_np[b], 24)[0]).all(-1)
            assert not written[:past[b]].any() and not written[past[b] + new[b]:].any()


# ---- eviction -----------------------------------------------------------------------------------------------------------------

def _evict_case(lengths, heads, ps, hd, dt, budget, recent, sink, seed=0, ties=False, in_place=False, weights=None,
                seen=None):
    from backend.cuda_paged import PagedEvict

    torch = _torch()
    rng = np.random.default_rng(seed)
    pool = Pool(lengths, heads=heads, ps=ps, hd=hd, dt=dt, seed=seed)
    rows, slots = len(lengths), pool.slots
    if weights is None:
        weights = rng.exponential(size=(rows, heads, slots)).astype(np.float32)
        if ties:
            weights = np.round(weights).astype(np.float32)
    seen = [n + 5 for n in lengths] if seen is None else seen
    pos = np.full((rows, heads, slots), -77, np.int32)
    for b, n in enumerate(lengths):
        for h in range(heads):
            pos[b, h, :n] = np.sort(rng.permutation(seen[b])[:n])[rng.permutation(n)] if n else []
    w_in, p_in = torch.tensor(weights, device="cuda"), _ints(pos)
    w_out, p_out = (w_in, p_in) if in_place else (torch.full_like(w_in, -3.0), torch.full_like(p_in, -3))
    lengths_out = _ints([-1] * rows)
    before = [p.clone() for p in (pool.k, pool.v)]
    op = PagedEvict(pool.k, pool.v, pool.table, pool.lengths, w_in, p_in, _ints(seen), w_out, p_out, lengths_out,
                    budget=budget, recent=recent, sink=sink)
    op()
    op.check()
    got_w, got_p = _host(w_out), _host(p_out)
    want = [_host(p) for p in before]
    for b, n in enumerate(lengths):
        left = min(n, budget)
        for h in range(heads):
            src = ref.evict(n, seen[b], weights[b, h], pos[b, h], budget, recent, sink)
            assert np.array_equal(got_w[b, h, :left], weights[b, h][src], equal_nan=True), (b, h)
            assert np.array_equal(got_p[b, h, :left], pos[b, h][src])
            if in_place:
                assert np.array_equal(got_w[b, h, left:], weights[b, h, left:], equal_nan=True)
                assert np.array_equal(got_p[b, h, left:], pos[b, h, left:])
            else:
                assert (got_w[b, h, left:] == -3).all() and (got_p[b, h, left:] == -3).all()
            for w, old in zip(want, before):
                rows_of = ref.slots(_host(old), pool.table_np[b], n)[h][src] if n else []
                for j in range(left):
                    w[pool.table_np[b, j // ps], h, j % ps] = rows_of[j]
    assert _host(lengths_out).tolist() == [min(n, budget) for n in lengths]
    for pages, w in zip((pool.k, pool.v), want):
        assert np.array_equal(_host(pages), w, equal_nan=True)
    return pool, op


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dt,hd", [("float32", 32), ("bfloat16", 64), ("bfloat16", 128), ("float32", 128)])
@pytest.mark.parametrize("lengths,heads,ps,budget,recent,sink", [
    ([33], 2, 16, 32, 8, 2), ([0, 1, 2, 5, 17, 64, 65, 200], 2, 8, 17, 5, 1), ([100, 3], 1, 32, 1, 0, 0),
    ([90, 40], 3, 16, 64, 64, 0), ([90, 40], 1, 16, 20, 0, 20), ([50, 60], 2, 64, 128, 10, 4), ([1500], 1, 16, 700, 100, 4)])
def test_evict(lengths, heads, ps, budget, recent, sink, dt, hd, in_place):
    _evict_case(lengths, heads, ps, hd, dt, budget, recent, sink, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("over", [1, 2, 3, 8, 9, 30])
def test_evict_a_few_tokens_over_the_budget(over, in_place):
    """The steps of a bounded cache: rows one or a few tokens over, with ties and protected tokens among the lightest."""
    for budget in (1, 16, 40, 200):
        lengths = [budget + over, budget, budget + 1, max(budget - 3, 0)]
        _evict_case(lengths, 2, 8, 64, "bfloat16", budget, min(3, budget - 1), min(1, budget - 1), seed=over, ties=True,
                    in_place=in_place)
        _evict_case(lengths, 1, 8, 32, "float32", budget, 0, 0, seed=over + 1)


@pytest.mark.parametrize("budget", [1, 13, 64, 255])
def test_evict_ties_go_to_the_lower_slot(budget):
    _evict_case([256, 199], 2, 16, 32, "bfloat16", budget, 0, 0, seed=4, ties=True)
    _evict_case([256], 1, 16, 32, "bfloat16", budget, 0, 0, weights=np.zeros((1, 1, 256), np.float32))


def test_evict_ranks_infinities_zeros_of_both_signs_and_nan():
    rng = np.random.default_rng(6)
    w = rng.choice(np.array([0.0, -0.0, 1.0, -1.0, np.inf, -np.inf, np.nan, 1e-42, 3e38], np.float32), size=(1, 2, 304))
    for budget in (5, 100, 250, 303):
        _evict_case([301], 2, 16, 32, "float32", budget, 2, 1, seed=budget, weights=w.copy())


def test_evict_rows_longer_than_shared_memory():
    _evict_case([70001], 1, 256, 32, "bfloat16", 20000, 300, 4, seed=7)
    _evict_case([52000, 48000], 1, 64, 32, "bfloat16", 40001, 0, 0, seed=8, ties=True, in_place=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lengths,heads,ps,budget,recent,sink", [
    ([4096], 3, 64, 1000, 100, 4), ([9000, 5, 0, 6000], 1, 8, 2000, 0, 0), ([16500, 20, 9001], 2, 256, 90, 10, 2),
    ([8193], 8, 32, 8000, 50, 0), ([8200, 8100] * 6, 1, 16, 2500, 40, 4), ([33000], 1, 128, 16384, 1, 1)])
def test_evict_long_rows_of_few_units(lengths, heads, ps, budget, recent, sink, in_place):
    """Several CTAs share a row's slots: short rows leave some of them none, and lists start where others end."""
    for ties in (False, True):
        _evict_case(lengths, heads, ps, 32, "bfloat16", budget, recent, sink, seed=11, ties=ties, in_place=in_place)
    weights = np.zeros((len(lengths), heads, -(-max(lengths) // ps) * ps), np.float32)
    _evict_case(lengths, heads, ps, 32, "bfloat16", budget, 0, 0, weights=weights, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("over", [1, 2, 5, 8, 9, 40])
def test_evict_a_few_tokens_of_long_rows(over, in_place):
    budget = 8190
    _evict_case([budget + over, budget, budget + 1, 17], 2, 64, 64, "bfloat16", budget, 20, 3, seed=over, in_place=in_place)
    _evict_case([budget + over], 1, 64, 32, "float32", budget, 0, 0, seed=over, ties=True, in_place=in_place)


def test_evict_long_rows_that_one_cta_takes():
    """Too many units for clusters, and rows too long for the shared memory of one."""
    _evict_case([50000] + [30] * 74, 1, 256, 32, "bfloat16", 300, 20, 4, seed=12)
    _evict_case([400001], 1, 256, 32, "bfloat16", 250, 20, 4, seed=13, ties=True)


def test_evict_reports_bad_lengths_and_pages():
    from backend.cuda_paged import PagedEvict

    torch = _torch()
    pool, op = _evict_case([40, 40], 1, 8, 32, "float32", 16, 4, 0)
    op.check()
    w, p = torch.rand(2, 1, 40, device="cuda"), torch.arange(40, device="cuda", dtype=torch.int32).repeat(2, 1, 1)
    table = pool.table.clone()
    table[1, 1:] = 10**6
    k = pool.k.clone()
    op = PagedEvict(pool.k, pool.v, table, _ints([99, 40]), w, p, _ints([40, 40]), torch.zeros_like(w),
                    torch.zeros_like(p), _ints([0, 0]), budget=16, recent=4)
    op()
    with pytest.raises(ValueError, match="out of range"):
        op.check()
    assert _host(op.lengths_out).tolist() == [16, 16]
    same = (k == pool.k) | (torch.isnan(k) & torch.isnan(pool.k))
    for page in pool.table_np[1]:
        assert bool(same[int(page)].all())


# ---- beam search ----------------------------------------------------------------------------------------------------------------

def _select(logits, scores, k, done=None, eos=-1, pad=0):
    from backend.cuda_paged import BeamSelect

    torch = _torch()
    b = logits.shape[0]
    outs = (torch.full((b, k), 9.0, device="cuda"), *(torch.full((b, k), -5, dtype=torch.int32, device="cuda") for _ in range(3)))
    op = BeamSelect(logits, scores, *outs[:3], done=done, done_out=outs[3], eos=eos, pad=pad)
    op()
    return [_host(t) for t in outs]


def _check_select(logits, scores, k, done=None, eos=-1, pad=0):
    got = _select(logits, scores, k, done, eos, pad)
    lg, sc = _host(logits), _host(scores)
    for b in range(lg.shape[0]):
        want = ref.beam_select(lg[b], sc[b], k, None if done is None else _host(done)[b], eos, pad)
        for name, g, w in zip(("parents", "tokens", "done"), (x[b] for x in got[1:]), want[1:]):
            assert g.tolist() == w.tolist(), (name, b, g, w, want[0])
        fine = np.isfinite(want[0])
        # fp32 exponentials (2 units in the last place) under an fp64 sum: 2^-22 in the sum, so in its logarithm, and
        # the last rounding
        assert (np.abs(got[0][b][fine] - want[0][fine]) <= 2.0**-24 * np.abs(want[0])[fine] + 2.0**-22).all()
        assert (got[0][b][~fine] == -np.inf).all()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("b,w,vocab,k", [(1, 4, 32000, 4), (1, 1, 1024, 5), (3, 5, 1003, 5), (2, 8, 4096, 16), (2, 3, 7, 4),
                                         (1, 2, 1, 2), (2, 16, 50001, 16), (1, 64, 5000, 64), (4, 1, 9000, 64),
                                         (1, 33, 4097, 33)])
def test_beam_select(b, w, vocab, k, dt):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(b * 1000 + w)
    logits = (3 * torch.randn(b, w, vocab, device="cuda", generator=g)).to(_tdt(dt))
    scores = -10 + torch.randn(b, w, device="cuda", generator=g)
    _check_select(logits, scores, k)
    done = (torch.rand(b, w, device="cuda", generator=g) < 0.4).to(torch.int32)
    _check_select(logits, scores, k, done, eos=min(2, vocab - 1), pad=vocab - 1)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_beam_select_ties(dt):
    """Equal logits, equal beams and constant rows: the lowest beam, then the lowest token."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(2)
    few = torch.randint(0, 3, (2, 4, 9001), device="cuda", generator=g).to(_tdt(dt))
    few[:, 2] = few[:, 0]
    scores = torch.zeros(2, 4, device="cuda")
    _check_select(few, scores, 8)
    _check_select(torch.zeros(1, 3, 20000, device="cuda", dtype=_tdt(dt)), torch.zeros(1, 3, device="cuda"), 64)
    zeros = torch.zeros(1, 2, 64, device="cuda", dtype=_tdt(dt))
    zeros[0, 0, ::2] = -0.0
    _check_select(zeros, torch.zeros(1, 2, device="cuda"), 5)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_beam_select_infinities_and_ended_beams(dt):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(3, 3, 5003, device="cuda", generator=g).to(_tdt(dt))
    inf = float("inf")
    logits[0, 0] = -inf                      # a beam with nothing left
    logits[0, 1, 5:] = -inf                  # five tokens left
    logits[0, 2, :] = -inf
    logits[0, 2, 7] = 1.0
    logits[1, :, 100:4000] = torch.finfo(logits.dtype).min  # masked with the type's lowest value: a logit like any other
    logits[1, 0, 17], logits[1, 1, 18], logits[1, 2, 19] = inf, float("nan"), -inf
    scores = torch.randn(3, 3, device="cuda", generator=g)
    scores[2, 0], scores[2, 2] = -inf, float("nan")
    _check_select(logits, scores, 8)  # entry 0: six candidates for eight places
    done = torch.tensor([[1, 0, 0], [0, 1, 1], [1, 1, 1]], dtype=torch.int32, device="cuda")
    _check_select(logits, scores, 8, done, eos=3, pad=4)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [40, 9001, 70000])
def test_beam_select_logits_near_the_types_limits(vocab, dt):
    """Rows masked whole or in part with the type's lowest value, and logits of its largest: the formula still."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    lim = torch.finfo(_tdt(dt))
    logits = torch.randn(1, 6, vocab, device="cuda", generator=g).to(_tdt(dt))
    logits[0, 0] = lim.min                   # a constant row: every token at -log(vocab)
    logits[0, 1, : vocab - 3] = lim.min      # whole chunks of nothing else
    logits[0, 2, 7] = lim.max                # one token has it all
    logits[0, 3, 3:9] = lim.max              # six have
    logits[0, 4, ::2], logits[0, 4, 1::2] = lim.max, lim.min
    _check_select(logits, torch.tensor([[0.0, 0.3, -4.0, -2.0, 3.0, 0.1]], device="cuda"), 20)
    _check_select(logits[:, :1], torch.tensor([[-1.5]], device="cuda"), 5)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [30, 5003, 70000])
def test_beam_select_reports_nan_and_infinity(vocab, dt):
    """-inf is a mask and no error, and nothing of an ended beam's logits is looked at; the results are as without it."""
    from backend.cuda_paged import BeamSelect

    torch = _torch()
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device="cuda").manual_seed(vocab)
    clean = torch.randn(2, 3, vocab, device="cuda", generator=g).to(_tdt(dt))
    clean[1, 0, ::2] = -inf
    clean[0, 2] = -inf
    logits, scores, done = clean.clone(), torch.zeros(2, 3, device="cuda"), _ints([[0, 0, 0], [0, 1, 0]])
    scores[1, 2] = -inf
    outs = (torch.zeros(2, 4, device="cuda"), *(torch.zeros(2, 4, dtype=torch.int32, device="cuda") for _ in range(2)))
    op = BeamSelect(logits, scores, *outs, done=done)
    logits[1, 1] = nan  # (ended)
    op()
    op.check()
    for bad in (nan, inf):
        for b, w, t in ((0, 0, 0), (0, 1, vocab - 1), (1, 0, vocab // 2)):
            logits[b, w, t] = bad
            op()
            with pytest.raises(ValueError, match="a logit or score was NaN"):
                op.check()
            logits[b, w, t] = clean[b, w, t]
            op()
            op.check()
    scores[0, 1] = nan
    op()
    with pytest.raises(ValueError, match="a logit or score was NaN"):
        op.check()


def _crowded_rows(vocab, dt):
    """Rows whose sums of exponentials have as many equal terms as can be: a rounding of one is a rounding of the sum."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = torch.empty(6, vocab, device="cuda")
    for i, rest in enumerate((-0.1, -0.7, -3.3, -9.0, -17.0)):
        rows[i] = rest
        rows[i, vocab // 3] = 0.0
    rows[5] = torch.linspace(-12, 4, vocab, device="cuda")[torch.randperm(vocab, device="cuda", generator=g)]
    return rows.to(_tdt(dt))


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [7, 1003, 8192, 50001, 131072])
def test_beam_select_sums_in_64_bits(vocab, dt):
    """A beam's score is chosen so that it all but cancels the logarithm of its sum: what is left comes out rounded once.
    The sum's own error: 2^-50 a term (an exponential in 64 bits) and 2^-53 an addition, of which a term passes fewer than
    200 (32 in a thread, 13 across a CTA, 128 chunks); its logarithm and the subtractions, at numbers below 32, 2^-48."""
    torch = _torch()
    logits = _crowded_rows(vocab, dt)[:, None]
    x = _host(logits)[:, 0]
    lse = np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) + x.max(1)
    scores = torch.tensor(lse - x.max(1), dtype=torch.float32, device="cuda")[:, None]
    got = _select(logits, scores, 1)
    want = _host(scores)[:, 0] + (x.max(1) - lse)
    assert (got[2][:, 0] == x.argmax(1)).all()
    assert (np.abs(got[0][:, 0] - want) <= 2.0**-24 * np.abs(want) + 2.0**-50 + 200 * 2.0**-53 + 2.0**-48).all()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [1003, 8192, 131072])
def test_beam_select_orders_beams_that_lie_close_together(vocab, dt):
    """A beam against an ended one whose score is 2e-9 above or below its best candidate's: the better one comes first."""
    torch = _torch()
    rows = _crowded_rows(vocab, dt)
    x = _host(rows)
    below = x.max(1) - (np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) + x.max(1))  # the best token's log-probability
    score = (-below - 1e-3).astype(np.float32)
    best = score.astype(np.float64) + below  # about -1e-3, where fp32 has steps of 1e-10
    logits = torch.stack([rows, rows], dim=1)
    done = _ints([[0, 1]] * 6)
    for off in (-2e-9, 2e-9):
        scores = torch.tensor(np.stack([score, best + off], 1), dtype=torch.float32, device="cuda")
        got = _select(logits, scores, 2, done, pad=5)
        assert got[1][:, 0].tolist() == [1 if off > 0 else 0] * 6, off


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [8200, 26080, 4100])
def test_beam_select_of_rows_that_crowd_in_a_few_warps(vocab, dt):
    """Ranges masked to nothing or to one value, sorted rows and vocabularies a little longer than a chunk."""
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(1, 7, vocab, device="cuda", generator=g).to(_tdt(dt))
    logits[0, 0, 1500:] = -float("inf")
    logits[0, 1, :-700] = -float("inf")
    logits[0, 2, 900:] = torch.finfo(_tdt(dt)).min
    logits[0, 3] = torch.arange(vocab, device="cuda") / 1000
    logits[0, 4] = -torch.arange(vocab, device="cuda") / 1000
    logits[0, 5] = torch.randint(0, 5, (vocab,), device="cuda", generator=g).to(logits.dtype)
    scores = torch.tensor([[0.0, -0.5, 0.25, 1.0, 1.5, 3.0, 0.1]], device="cuda")
    _check_select(logits, scores, 64)
    for w in range(7):
        _check_select(logits[:, w:w + 1], scores[:, w:w + 1].contiguous(), 13)


def test_beam_select_strided_logits():
    torch = _torch()
    for dt in ("float32", "bfloat16"):
        wide = torch.randn(6, 1050, device="cuda").to(_tdt(dt))
        logits = wide.view(2, 3, 1050)[:, :, 1:1042]
        _check_select(logits, torch.zeros(2, 3, device="cuda"), 3)
    stack = torch.randn(2, 3, 1040, device="cuda")
    _check_select(stack[:, :, :1024], torch.zeros(2, 3, device="cuda"), 3)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("layers,heads,ps,hd,length", [(2, 3, 16, 64, 37), (1, 1, 8, 32, 8), (3, 2, 32, 128, 0),
                                                       (1, 2, 16, 128, 5), (2, 1, 64, 32, 191), (2, 2, 8, 64, 48)])
def test_beam_reorder(layers, heads, ps, hd, length, dt):
    from backend.cuda_paged import BeamReorder

    torch = _torch()
    rng = np.random.default_rng(length)
    cases = [[0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [2, 2, 2, 2, 2], [1, 1, 0, 0, 4], [0, 0, 0, 4, 4], [3, 1, 3, 1, 3]]
    b, w, full = len(cases), 5, length // ps
    width = full + 2
    pool = b * full + 2 * b * w + 2
    order = rng.permutation(pool)
    table = np.zeros((b, w, width), np.int32)
    table[:, :, :full] = order[:b * full].reshape(b, 1, full)
    table[:, :, full:] = order[b * full:b * full + 2 * b * w].reshape(b, w, 2)
    pages = torch.randn(layers, 2, pool, heads, ps, hd, device="cuda").to(_tdt(dt))
    before = _host(pages).reshape(layers * 2, pool, heads, ps, hd)
    parents = _ints(cases)
    table_out = torch.full((b * w, width), -1, dtype=torch.int32, device="cuda")
    op = BeamReorder(pages, _ints(table.reshape(b * w, width)), _ints([length] * b), parents, table_out)
    op()
    op.check()
    want = before
    rows = []
    for i in range(b):
        want, t = ref.beam_reorder(want, table[i], length, np.asarray(cases[i]))
        rows.append(t)
    assert np.array_equal(_host(table_out), np.concatenate(rows))
    assert np.array_equal(_host(pages).reshape(want.shape), want)
    first = pages.clone()
    op()  # the tables have not changed: a repeat writes the same copies
    assert torch.equal(first, pages)


def test_beam_reorder_reports_bad_parents_and_keeps_the_tables():
    from backend.cuda_paged import BeamReorder

    torch = _torch()
    pages = torch.randn(1, 2, 12, 1, 8, 32, device="cuda")
    table = _ints([[0, 1], [0, 2], [3, 4], [3, 5]])
    for parents, lengths, bad in (([[0, 2], [1, 1]], [12, 12], 0), ([[0, 0], [-1, 0]], [12, 12], 1),
                                  ([[1, 0], [1, 1]], [12, 17], 1), ([[1, 0], [0, 0]], [-1, 12], 0)):
        out = torch.zeros_like(table)
        op = BeamReorder(pages, table, _ints(lengths), _ints(parents), out)
        op()
        with pytest.raises(ValueError, match="out of range"):
            op.check()
        assert torch.equal(out[2 * bad:2 * bad + 2], table[2 * bad:2 * bad + 2])


# ---- streams and graphs -------------------------------------------------------------------------------------------------------------

def test_calls_on_another_stream_and_captured_replays_follow_the_device_values():
    """One captured graph of append + attention + eviction is replayed with new lengths, positions and values."""
    from backend.cuda_paged import PagedAppend, PagedAttention, PagedEvict

    torch = _torch()
    heads, hd, ps, rows, budget = 2, 64, 8, 3, 24
    dt = "float32"

    def build(seed):
        pool = Pool([20, 5, 24], heads=heads, ps=ps, hd=hd, dt=dt, seed=seed, room=10)
        g = torch.Generator(device="cuda").manual_seed(seed)
        s = dict(pool=pool, q=torch.randn(rows, 4, hd, device="cuda", generator=g),
                 k=torch.randn(rows, heads, hd, device="cuda", generator=g),
                 v=torch.randn(rows, heads, hd, device="cuda", generator=g))
        s["n1"], s["n2"], s["pos2"] = _ints([0] * rows), _ints([0] * rows), _ints([0] * rows)
        s["pos"] = _ints([20, 5, 24])
        s["q_out"], s["out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["q"])
        s["w"] = torch.rand(rows, heads, pool.slots, device="cuda", generator=g)
        s["sp"] = torch.arange(pool.slots, device="cuda", dtype=torch.int32).expand(rows, heads, -1).contiguous()
        cos, sin = _rope(hd, 100)
        ops = [PagedAppend(s["k"], s["v"], pool.k, pool.v, pool.table, pool.lengths, s["n1"], q=s["q"], q_out=s["q_out"],
                           cos=cos, sin=sin, positions=s["pos"], positions_out=s["pos2"], slot_positions=s["sp"],
                           weights=s["w"]),
               PagedAttention(s["q_out"], pool.k, pool.v, pool.table, s["n1"], s["out"], weights=s["w"]),
               PagedEvict(pool.k, pool.v, pool.table, s["n1"], s["w"], s["sp"], s["pos2"], s["w"], s["sp"], s["n2"],
                          budget=budget, recent=4)]

        def step():
            for op in ops:
                op()
            pool.lengths.copy_(s["n2"])
            s["pos"].copy_(s["pos2"])

        return s, ops, step

    one, ops1, step1 = build(3)
    two, ops2, step2 = build(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step2()  # a warm-up on another stream, then the capture
    torch.cuda.current_stream().wait_stream(side)
    step1()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step2()
    torch.cuda.synchronize()
    for i in range(8):
        for s in (one, two):
            g = torch.Generator(device="cuda").manual_seed(50 + i)
            for name in ("q", "k", "v"):
                s[name].copy_(torch.randn(s[name].shape, device="cuda", generator=g))
        step1()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("out", "w", "sp", "n2", "pos"):
            assert torch.equal(one[name], two[name]), (i, name)
        for a, b in ((one["pool"].k, two["pool"].k), (one["pool"].v, two["pool"].v)):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        assert bool(torch.isfinite(one["out"]).all())
    assert one["n2"].tolist() == [24, 14, 24]
    for op in ops1 + ops2:
        op.check()


def test_first_call_inside_a_capture():
    """A capture of calls that have not run before (kernels are loaded and sized during it) replays to the right result."""
    from backend.cuda_paged import BeamSelect, PagedEvict

    torch = _torch()
    pool, q, out, _, _, op = _attention_case([5000, 77], 8, 1, 64, 32, "bfloat16", seed=31)
    logits = torch.randn(1, 3, 777, device="cuda")
    outs = (torch.zeros(1, 9, device="cuda"), *(torch.zeros(1, 9, dtype=torch.int32, device="cuda") for _ in range(2)))
    select = BeamSelect(logits, torch.zeros(1, 3, device="cuda"), *outs)
    w = torch.rand(2, 1, pool.slots, device="cuda")
    p = torch.arange(pool.slots, device="cuda", dtype=torch.int32).repeat(2, 1, 1)
    n = _ints([0, 0])
    evict = PagedEvict(pool.k.clone(), pool.v.clone(), pool.table, pool.lengths, w, p, pool.lengths, torch.zeros_like(w),
                       torch.zeros_like(p), n, budget=1500, recent=10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op()
        select()
        evict()
    graph.replay()
    _check_attention(pool, q, out, None, None, "bfloat16")
    want = ref.beam_select(_host(logits)[0], np.zeros(3), 9)
    assert _host(outs[1])[0].tolist() == want[1].tolist() and _host(outs[2])[0].tolist() == want[2].tolist()
    assert n.tolist() == [1500, 77]


def test_two_operators_at_once_on_two_streams():
    """Each with its own workspace and outputs, over the same pages; as if one ran after the other."""
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    pool, q, out, _, _, op = _attention_case([9000, 4500, 3, 0], 4, 2, 16, 128, "bfloat16", seed=32)
    q2 = torch.randn_like(q)
    out2 = torch.empty_like(q2)
    op2 = PagedAttention(q2, pool.k, pool.v, pool.table, pool.lengths, out2)
    op(), op2()
    want, want2 = out.clone(), out2.clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        out.zero_(), out2.zero_()
        torch.cuda.synchronize()
        for st, o in zip(streams, (op, op2)):
            with torch.cuda.stream(st):
                o()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want2)


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_attention_of_many_rows(dt):
    """More rows than a scan's threads take one each, most of them empty or short, one long; more CTAs than tiles and fewer."""
    rng = np.random.default_rng(33)
    lengths = list(rng.integers(0, 3, 700)) + [5000] + list(rng.integers(0, 90, 300))
    pool, q, out, w0, weights, op = _attention_case(lengths, 2, 1, 8, 32, dt, seed=33, track=True)
    op()
    _check_attention(pool, q, out, w0, weights, dt)


def test_an_operator_dropped_while_its_work_is_pending_keeps_its_memory():
    """The workspace of an operator used on another stream is not handed out again before that stream's work is done."""
    torch = _torch()
    want = None
    for i in range(6):
        pool, q, out, _, _, op = _attention_case([30000, 20000], 8, 2, 64, 128, "bfloat16", seed=34)
        if want is None:
            op()
            want = out.clone()
            out.zero_()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(20):
                op()
        op = None
        junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(32)]  # would land in a freed workspace
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        del junk


def _wait_a_moment():
    _torch().cuda._sleep(100_000_000)  # about 50 ms of the current stream


def test_check_sees_errors_of_calls_on_other_streams():
    """A call that is still waiting on another stream when ``check`` is asked on this one."""
    torch = _torch()
    pool, q, out, _, _, op = _attention_case([40, 30], 2, 2, 16, 64, "bfloat16", seed=41)
    pool.lengths.copy_(_ints([40, -1]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            _wait_a_moment()
            op()
        with pytest.raises(ValueError, match="out of range"):
            op.check()
    op.check()  # cleared


def test_an_operator_made_behind_pending_work_keeps_what_another_stream_reports():
    """The flag's zero waits on the stream that the operator was made on: a call on another one comes behind it."""
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    pool, q, out, _, _, first = _attention_case([9000, 30], 2, 2, 16, 64, "bfloat16", seed=42)
    first()
    want = out.clone()
    bad = _ints([9000, 10**6])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for lengths in (bad, pool.lengths):
        out.zero_()
        torch.cuda.synchronize()
        _wait_a_moment()
        op = PagedAttention(q, pool.k, pool.v, pool.table, lengths, out)
        with torch.cuda.stream(side):
            op()
        torch.cuda.synchronize()
        if lengths is bad:
            with pytest.raises(ValueError, match="out of range"):
                op.check()
        else:
            op.check()
            assert torch.equal(out, want)


def test_an_operator_made_and_called_inside_a_capture():
    """Its flag and workspace belong to the graph; replays report what they meet."""
    from backend.cuda_paged import PagedAttention

    torch = _torch()
    pool, q, out, _, _, first = _attention_case([9000, 30], 2, 2, 16, 64, "bfloat16", seed=43)
    first()
    want = out.clone()
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op = PagedAttention(q, pool.k, pool.v, pool.table, pool.lengths, out)
        op()
    graph.replay()
    op.check()
    assert torch.equal(out, want)
    pool.lengths.copy_(_ints([9000, -3]))
    graph.replay()
    with pytest.raises(ValueError, match="out of range"):
        op.check()
