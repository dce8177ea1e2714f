"""Attention over the 8-bit cache (mossgpu_attention_kv8) at the ends of its range -- queries, scales, scores
and V scales of any size, NaN in some rows only -- in each of its forms, against the 64-bit form."""
from __future__ import annotations

import functools

import pytest
import torch

import kv8_ref as R
from test_op_kv8 import L, M, attend, batch, ok, status, stream  # noqa: F401 (L and M are fixtures)

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# New rows of a sequence, query heads of a kv head, pages of a slot: a table of up to 192 pages takes the one-launch
# form of few or of some rows, a wider one the forms that cut the positions into runs, for 4, some and many rows.
FORMS = {"few_one": (2, 2, 130), "few": (2, 2, 300), "some_one": (3, 4, 130), "some": (3, 4, 300), "many": (9, 8, 300)}
SLOTS = [2, 0, 1]
CTX = [1990, 31, 0]  # several tiles for every warp of the one-launch forms; runs of several tiles with 12 kv heads


@functools.lru_cache(maxsize=None)
def filled(fmt, dim, kvh, new):
    cache = R.Cache(fmt, kvh, dim, len(CTX), 130, spare=1, seed=3)
    for s, slot in enumerate(SLOTS):
        cache.fill(slot, CTX[s] + new, 20 + s)
    return cache


def setup(form, fmt, dim, t, kvh=12):
    new, group, pps = FORMS[form]
    cache = R.Cache.__new__(R.Cache)
    cache.__dict__.update(filled(fmt, dim, kvh, new).__dict__)
    cache.codes, cache.scales = cache.codes.clone(), cache.scales.clone()
    cache.table = torch.nn.functional.pad(cache.table, (0, pps - cache.pps), value=-1)  # a wider table, which ends as the slots do
    cache.pps = pps
    starts = [i * new for i in range(len(CTX) + 1)]
    q = torch.randn(starts[-1], kvh * group, dim, generator=torch.Generator().manual_seed(3)).to(t)
    return cache, q, starts, SLOTS, new, group


def exact(cache, q, starts, slots, scale, mask=None):
    """As kv8_ref.attend64, the rows of a sequence at once."""
    rows, qh, dim = q.shape
    group = qh // cache.kvh
    out, mass, top = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(rows, qh, dtype=torch.float64)
    for s, slot in enumerate(slots):
        n = starts[s + 1] - starts[s]
        at = slice(starts[s], starts[s + 1])
        # NaN counts as 0: what rows that do not see it have, and the others are not compared
        k, v = (torch.nan_to_num(cache.heads(slot, CTX[s] + n, half)) for half in (0, 1))
        see = torch.ones(n, CTX[s] + n, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                see[i, CTX[s] + j] = j <= i if mask is None else bool(int(mask[starts[s] + i, 0]) >> j & 1)
        qs, see = q[at].view(n, cache.kvh, group, dim), see[:, None, None]
        a = (torch.einsum("ikgd,jkd->ikgj", qs, k) * scale).masked_fill(~see, float("-inf"))
        p = torch.nan_to_num(torch.softmax(a, -1))  # nothing seen: zeros
        out[at] = torch.einsum("ikgj,jkd->ikgd", p, v).reshape(n, qh, dim)
        mass[at] = torch.einsum("ikgj,jkd->ikgd", p, v.abs()).reshape(n, qh, dim)
        size = torch.einsum("ikgd,jkd->ikgj", qs.abs(), k.abs()) * abs(scale)
        top[at] = size.masked_fill(~see, 0.0).amax(-1).view(n, qh)
    return out, mass, top


def each_place(cache, slot, pos):
    return int(cache.table[slot, pos // 16]), pos % 16


def run(M, L, cache, q, starts, slots, scale, mask=None):
    out = torch.full_like(q, 7.25, device="cuda")
    keep, seqs = batch(M, starts, slots, CTX, starts[-1])
    ws = attend(M, L, cache.cuda(), seqs, q.cuda(), out, scale, mask.cuda() if mask is not None else None)
    assert status(L) == 0
    del ws, keep
    return out.cpu().double()


def seen_scale(cache, starts, slots, mask=None):
    """Of each row and kv head: the largest V scale it sees, and how many positions that may be."""
    top = torch.zeros(starts[-1], cache.kvh, dtype=torch.float64)
    count = torch.zeros(starts[-1], 1, dtype=torch.float64)
    for s, slot in enumerate(slots):
        n = starts[s + 1] - starts[s]
        pos = torch.arange(CTX[s] + n)
        sv = cache.scales[cache.table[slot].long()[pos // 16], 1, :, pos % 16].double()
        for i in range(n):
            r = starts[s] + i
            see = torch.ones(len(pos), dtype=torch.bool)
            for j in range(n):
                see[CTX[s] + j] = j <= i if mask is None else bool(int(mask[r, 0]) >> j & 1)
            if see.any():
                top[r] = torch.nan_to_num(sv[see]).amax(0)
            count[r] = see.sum()
    return top, count


def tolerance(form, cache, q, want, mass, top, starts, slots, t, group, mask=None):
    """attend_tolerance, and what a weight's fp16 parts lose below 2^-14 of their range: half a step of 2^-24 where the
    largest weight times the largest V scale lies in [2^13, 2^14), so 2^-38 of that scale, for every position and its
    largest code, relative to a sum of weights of at least 1 (the largest).  The form for many rows leaves bf16 outputs
    2^6 of room above, so 2^-32."""
    low = 2.0**-32 if form == "many" and t == BF16 else 2.0**-38
    sv, count = seen_scale(cache, starts, slots, mask)
    sv = sv.repeat_interleave(group, 1)
    return R.attend_tolerance(mass, top, want, t) + (low * R.CODE_MAX[cache.fmt] * count * sv)[..., None]


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt,dim", [(R.INT8, 64), (R.E4M3, 128)])
@pytest.mark.parametrize("size", [1e-37, 1e-30, 1e25, 2e37])
def test_queries_and_v_scales_of_any_size(M, L, form, t, fmt, dim, size):
    # queries up to 2^126, which the scale takes back; V scales that grow along the sequence by 2^40
    cache, q, starts, slots, new, group = setup(form, fmt, dim, t)
    for s, slot in enumerate(slots):
        for p in range(CTX[s] + new):
            page, off = each_place(cache, slot, p)
            cache.scales[page, 1, :, off] *= 2.0 ** (p * 40.0 / 2000 - 20)
    q = (q.float().clamp(-4, 4) * size).to(t)
    scale = float(torch.tensor(0.125 / size, dtype=torch.float32))
    want, mass, top = exact(cache, q.double(), starts, slots, scale)
    got = run(M, L, cache, q, starts, slots, scale)
    assert ((got - want).abs() <= tolerance(form, cache, q, want, mass, top, starts, slots, t, group)).all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("scale", [1e-6, 1e-12, 1e-30, 1e-45])
def test_zero_queries_at_any_scale(M, L, form, t, scale):
    # every position that is seen weighs the same, and none that is not, however small the scale
    cache, q, starts, slots, new, group = setup(form, R.INT8, 64, t)
    q.zero_()
    want, mass, top = exact(cache, q.double(), starts, slots, scale)
    got = run(M, L, cache, q, starts, slots, scale)
    assert ((got - want).abs() <= R.attend_tolerance(mass, top, want, t)).all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt,dim", [(R.INT8, 64), (R.E4M3, 128)])
@pytest.mark.parametrize("scale", [2.0**8, -(2.0**12), 2.0**16, 1.7 * 2.0**20, 2.0**40, -(2.0**100)])
def test_scores_of_any_size(M, L, form, t, fmt, dim, scale):
    # Whole numbers throughout, so that scores are exact: a few positions share the largest and lie at least
    # |scale| above all others, which leaves the mean of their V
    cache, q, starts, slots, new, group = setup(form, fmt, dim, t)
    cache.scales[:, 0] = 1.0
    g = torch.Generator().manual_seed(8)
    base = torch.randint(0, 2, (dim,), generator=g) * 2 - 1
    small = torch.randint(-12, 13, (cache.pages, cache.kvh, R.PAGE, dim), generator=g)
    peak = (base * 64).float()
    code = (lambda x: x.to(torch.int8).view(torch.uint8)) if fmt == R.INT8 else (lambda x: x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    cache.codes[:, 0] = code(small)
    for p in (5, 6, 700, 1989):  # of the long context; the short ones keep what they have
        page, off = each_place(cache, slots[0], p)
        cache.codes[page, 0, :, off] = code(peak)
    times = torch.randint(1, 5, (q.shape[0], q.shape[1], 1), generator=g)
    q = (base * times).to(t) * (1 if scale > 0 else -1)
    long_rows = slice(0, new)
    want, mass, _ = exact(cache, q.double(), starts, slots, scale)
    v = cache.heads(slots[0], CTX[0], 1)[[5, 6, 700, 1989]].mean(0).repeat_interleave(group, 0)
    assert ((want[long_rows] - v).abs() <= 1e-12 * mass[long_rows]).all()
    got = run(M, L, cache, q, starts, slots, scale)
    tol = tolerance(form, cache, q, want, mass, torch.zeros(q.shape[:2], dtype=torch.float64), starts, slots, t, group)
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("fmt,dim", [(R.INT8, 64), (R.E4M3, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_hidden_v_scales_do_not_count(M, L, form, t, fmt, dim, causal):
    # A drafted token with a V scale 2^45 above the others', which some rows see and others do not: the rows that do not
    # are as exact as without it.  Outputs that hold such values pass the range of fp16: those rows go unread there.
    cache, q, starts, slots, new, group = setup(form, fmt, dim, t)
    hidden = new - 1 if causal else 0
    for s, slot in enumerate(slots):
        page, off = each_place(cache, slot, CTX[s] + hidden)
        cache.scales[page, 1, :, off] *= 2.0**45
    mask = None
    if not causal:  # every row sees itself and, from the second on, the one before it unless that is the first
        mask = torch.tensor([[1 << i | (1 << (i - 1) if i > 1 else 0)] for _ in CTX for i in range(new)], dtype=torch.int32)
    want, mass, top = exact(cache, q.double(), starts, slots, 0.125, mask)
    got = run(M, L, cache, q, starts, slots, 0.125, mask)
    tol = tolerance(form, cache, q, want, mass, top, starts, slots, t, group, mask)
    rows = torch.tensor([t != F16 or r % new != hidden for r in range(starts[-1])])
    assert ((got - want).abs() <= tol)[rows].all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("fmt,dim", [(R.INT8, 64), (R.E4M3, 128)])
@pytest.mark.parametrize("half", [0, 1])
def test_nan_only_where_it_is_seen(M, L, form, t, fmt, dim, half):
    # NaN scales at a context position of the second sequence, and at the first draft of the first, which the odd rows see
    kvh = 12
    cache, q, starts, slots, new, group = setup(form, fmt, dim, t)
    for slot, pos, head in ((slots[1], 17, 3), (slots[0], CTX[0], 5)):
        page, off = each_place(cache, slot, pos)
        cache.scales[page, half, head, off] = float("nan")
        cache.codes[page, half, head, off] = 0
    mask = torch.tensor([[(1 << i) & ~1 | (i & 1)] for _ in CTX for i in range(new)], dtype=torch.int32)
    got = run(M, L, cache, q, starts, slots, 0.125, mask)
    want = torch.zeros(starts[-1], kvh, dtype=torch.bool)
    want[starts[1] : starts[2], 3] = True
    want[[i for i in range(new) if i & 1], 5] = True
    want = want.repeat_interleave(group, 1)
    assert torch.equal(torch.isnan(got).all(-1), want) and torch.equal(torch.isnan(got).any(-1), want)
    clean, mass, top = exact(cache, q.double(), starts, slots, 0.125, mask)
    fine = ~want
    assert ((got - clean).abs() <= R.attend_tolerance(mass, top, clean, t))[fine].all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt,dim", [(R.INT8, 64), (R.E4M3, 128)])
def test_sums_of_the_largest_values(M, L, form, t, fmt, dim):
    # 2000 equal weights of values of about 2^120, whose sum is past the range of fp32
    cache, q, starts, slots, new, group = setup(form, fmt, dim, t)
    q.zero_()
    cache.codes[:, 1] = 100 if fmt == R.INT8 else 0x6c  # 96 in e4m3
    cache.scales[:, 1] = 2.0**114
    value = 2.0**114 * (100 if fmt == R.INT8 else 96)
    got = run(M, L, cache, q, starts, slots, 0.125)
    assert ((got - value).abs() <= value * (2.0**-19 + (2.0**-11 + 2.0**-8 if t == BF16 else 0.0))).all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt,dim", [(R.INT8, 64), (R.E4M3, 128)])
@pytest.mark.parametrize("k,v", [(2.0**100, 2.0**-87), (2.0**-100, 2.0**100)])
def test_scales_at_the_ends_of_their_range(M, L, form, t, fmt, dim, k, v):
    cache, q, starts, slots, new, group = setup(form, fmt, dim, t)
    for s, slot in enumerate(slots):
        n = CTX[s] + new
        for half, size in ((0, k), (1, v)):
            pos = torch.arange(n)
            page = cache.table[slot].long()[pos // 16]
            cache.scales[page, half, :, pos % 16] = torch.ldexp(0.5 + torch.rand(n, cache.kvh, generator=torch.Generator().manual_seed(half)) / 2,
                                                                torch.tensor(float(torch.tensor(size).log2())))
    q = (q.double() / k / 50).to(t)
    want, mass, top = exact(cache, q.double(), starts, slots, 0.125)
    got = run(M, L, cache, q, starts, slots, 0.125)
    assert ((got - want).abs() <= tolerance(form, cache, q, want, mass, top, starts, slots, t, group)).all()
