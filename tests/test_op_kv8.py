"""Rotary positions and the 8-bit paged cache (append, read-back, attention over it) through the C
ABI, against plain 64-bit forms (kv8_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SENTINEL = 7.25  # exact in every type


@pytest.fixture(scope="module")
def M():
    import moss_b200
    moss_b200.build()
    return moss_b200


@pytest.fixture(scope="module")
def L(M):
    return M.lib()


def ok(L, rc):
    assert rc == 0, L.mossgpu_op_last_error().decode()


def status(L):
    import ctypes as C
    torch.cuda.synchronize()
    code = C.c_int(-1)
    ok(L, L.mossgpu_op_device_status(C.byref(code)))
    return code.value


def stream():
    return torch.cuda.current_stream().cuda_stream


def strided(rows, heads, dim, t, pad=0, lead=0, fill=SENTINEL):
    """(buffer, view [rows][heads][dim]) with `pad` elements between heads and rows and `lead` in front."""
    hs = dim + pad
    rs = heads * hs + 3 * pad
    buf = torch.full((lead + rows * rs + 16,), fill, dtype=t, device="cuda")
    return buf, buf[lead : lead + rows * rs].as_strided((rows, heads, dim), (rs, hs, 1), lead)


# ---- rotary positions ------------------------------------------------------------------------


def run_rope(M, L, x, out, pos, steps, rot, inter, mag=1.0, inverse=False, rc=0):
    rope = M.Rope(steps.data_ptr(), rot, int(inter), mag)
    a = M.RopeArgs(x=x.data_ptr(), out=out.data_ptr(), pos=pos.data_ptr(), x_row_stride=x.stride(0), x_head_stride=x.stride(1),
                   out_row_stride=out.stride(0), out_head_stride=out.stride(1), rows=x.shape[0], heads=x.shape[1],
                   head_dim=x.shape[2], type=R.type_id(x.dtype), inverse=int(inverse))
    ok(L, L.mossgpu_rope_rotate(rope, a, stream()))


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("rows,heads,dim,rot,pad", [(1, 1, 64, 64, 0), (3, 5, 64, 20, 0), (7, 2, 80, 80, 8), (2, 33, 96, 62, 0),
                                                    (5, 3, 256, 256, 0), (4, 3, 128, 96, 5), (2, 2, 8, 2, 1), (130, 12, 64, 48, 0)])
def test_rope(M, L, t, inter, rows, heads, dim, rot, pad):
    g = torch.Generator().manual_seed(rows * dim + rot)
    x64 = torch.randn(rows, heads, dim, generator=g).to(t).double()
    pos = torch.randint(-(2**31), 2**31 - 1, (rows,), generator=g, dtype=torch.int64).int()
    pos[: min(rows, 3)] = torch.tensor([0, 1, 2**31 - 1][: min(rows, 3)], dtype=torch.int32)
    freq = R.freqs(rot)
    steps = torch.from_numpy(R.steps_of(freq).view(np.int64)).cuda()
    _, x = strided(rows, heads, dim, t, pad)
    buf, out = strided(rows, heads, dim, t, pad, lead=pad)
    x.copy_(x64)
    mag = 1.25
    run_rope(M, L, x, out, pos.cuda(), steps, rot, inter, mag)
    # the angle the steps stand for, reduced exactly in whole 2^-64 turns
    turns = np.array([[int(p) * int(s) % 2**64 for s in R.steps_of(freq).tolist()] for p in pos.tolist()], dtype=object)
    ang = np.array([[float(v) / 2**64 for v in row] for row in turns], np.float64).reshape(rows, rot // 2) * 2 * np.pi
    c, s = np.cos(ang)[:, None] * mag, np.sin(ang)[:, None] * mag
    xn = x64.numpy()
    ia = np.arange(0, rot, 2) if inter else np.arange(rot // 2)
    ib = ia + 1 if inter else ia + rot // 2
    want = xn.copy()
    want[..., ia] = xn[..., ia] * c - xn[..., ib] * s
    want[..., ib] = xn[..., ib] * c + xn[..., ia] * s
    # cos, sin: the angle to 2^-24 of half a turn (2^-22), sincospif to 2 ulp (2^-23), times mag (2^-24); two products and a sum
    tol = np.abs(want) * R.half_step(t) + 1e-38
    size = (np.abs(xn[..., ia]) + np.abs(xn[..., ib])) * mag * (2.0**-22 + 2.0**-23 + 4 * 2.0**-24)
    tol[..., ia] += size
    tol[..., ib] += size
    got = out.cpu().double().numpy()
    assert (np.abs(got - want) <= tol).all()
    assert np.array_equal(got[..., rot:], xn[..., rot:])  # copied
    gaps = torch.ones_like(buf, dtype=torch.bool)
    gaps.as_strided(out.shape, out.stride(), out.storage_offset()).fill_(False)
    assert (buf[gaps] == SENTINEL).all()  # nothing outside the heads
    # in place: the same bits
    run_rope(M, L, x, x, pos.cuda(), steps, rot, inter, mag)
    assert torch.equal(x, out)


@pytest.mark.parametrize("inter", [True, False])
def test_rope_inverse_is_the_gradient(M, L, inter):
    # <R x, g> = <x, R' g>, and differences of the forward in single elements
    rows, heads, dim, rot, mag = 3, 2, 64, 40, 1.1
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, heads, dim, generator=g).cuda()
    w = torch.randn(rows, heads, dim, generator=g).cuda()
    pos = torch.tensor([0, 77, 4000], dtype=torch.int32).cuda()
    steps = torch.from_numpy(R.steps_of(R.freqs(rot)).view(np.int64)).cuda()
    y, grad = torch.empty_like(x), torch.empty_like(x)
    run_rope(M, L, x, y, pos, steps, rot, inter, mag)
    run_rope(M, L, w, grad, pos, steps, rot, inter, mag, inverse=True)
    a, b = (y.double() * w.double()).sum(), (x.double() * grad.double()).sum()
    size = (y.double().abs() * w.double().abs()).sum() + (x.double().abs() * grad.double().abs()).sum()
    assert abs(a - b) <= size * 2.0**-20
    for e in (0, 1, 19, 20, 39, 40, 63):
        up = x.clone()
        up[1, 1, e] += 1.0
        y2 = torch.empty_like(x)
        run_rope(M, L, up, y2, pos, steps, rot, inter, mag)
        d = ((y2.double() - y.double()) * w.double()).sum().item()
        assert abs(d - grad[1, 1, e].item()) <= 64 * 2.0**-20  # rounding of two passes over values of up to about 4


# ---- append and read back --------------------------------------------------------------------


def batch(M, starts, slots, ctx, rows):
    keep = [torch.tensor(v, dtype=torch.int32).cuda() for v in (starts, slots, ctx)]
    return keep, M.SeqBatch(keep[0].data_ptr(), keep[1].data_ptr(), keep[2].data_ptr(), len(slots), rows)


def append_args(M, k, v, q=None, q_out=None, pos=None):
    a = M.KV8AppendArgs(k=k.data_ptr(), v=v.data_ptr(), k_row_stride=k.stride(0), k_head_stride=k.stride(1),
                        v_row_stride=v.stride(0), v_head_stride=v.stride(1), type=R.type_id(k.dtype),
                        pos=pos.data_ptr() if pos is not None else None)
    if q is not None:
        a.q, a.q_out, a.q_heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
        a.q_row_stride, a.q_head_stride, a.q_out_row_stride, a.q_out_head_stride = *q.stride()[:2], *q_out.stride()[:2]
    return a


LENGTHS = {  # (new rows, context) of each sequence
    "one": [(1, 0)],
    "ragged": [(3, 13), (0, 9), (1, 31), (17, 15), (5, 0)],
    "many": [((7 * i) % 4, (5 * i) % 40) for i in range(70)],
}


def layout(lengths, lead=0):
    starts, n = [lead], lead
    for new, _ in lengths:
        n += new
        starts.append(n)
    order = np.random.RandomState(len(lengths)).permutation(len(lengths)).tolist()
    return starts, order, [c for _, c in lengths]


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("fmt", [R.INT8, R.E4M3])
@pytest.mark.parametrize("dim,kvh,pad", [(64, 12, 0), (128, 3, 8), (64, 1, 3)])
def test_append_codes_and_read_back(M, L, lengths, t, fmt, dim, kvh, pad):
    starts, slots, ctx = layout(LENGTHS[lengths], lead=2)  # rows before the first sequence and after the last
    rows = starts[-1] + 3
    cache = R.Cache(fmt, kvh, dim, len(slots) + 1, 6, seed=5)
    before_codes, before_scales = cache.codes.clone(), cache.scales.clone()
    g = torch.Generator().manual_seed(9)
    kv = []
    for _ in range(2):
        x = (torch.randn(rows, kvh, dim, generator=g) * torch.exp(2 * torch.randn(rows, kvh, 1, generator=g))).to(t)
        x[starts[0], 0] = 0                                     # a head of zeros
        if rows > 8:
            x[5, kvh - 1] = 1e-39                               # a scale that would be subnormal (0 in fp16)
            x[6, 0, 3] = float("nan")
            x[7, 0, dim - 1] = float("-inf")
        _, view = strided(rows, kvh, dim, t, pad, lead=pad)
        view.copy_(x)
        kv.append((x, view))
    dev = cache.cuda()
    keep, seqs = batch(M, starts, slots, ctx, rows)
    ok(L, L.mossgpu_kv8_append(dev.struct(M), seqs, None, append_args(M, kv[0][1], kv[1][1]), stream()))
    assert status(L) == 0
    for half in (0, 1):
        codes, scales = R.quantise32(kv[half][0], fmt)
        for s, slot in enumerate(slots):
            for i in range(starts[s + 1] - starts[s]):
                cache.put(slot, ctx[s] + i, half, codes[starts[s] + i], scales[starts[s] + i])
    assert torch.equal(dev.codes.cpu(), cache.codes)  # every cell: written ones exactly, all others untouched
    assert torch.equal(dev.scales.cpu().view(torch.int32).isfinite(), cache.scales.view(torch.int32).isfinite())
    a, b = dev.scales.cpu(), cache.scales
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))
    assert (before_codes != cache.codes).any() or starts[-1] == starts[0]
    # back, in every type, and each half alone
    for out_t in R.TYPES:
        views = [strided(rows, kvh, dim, out_t, pad, lead=2 * pad) for _ in range(2)]
        ra = M.KV8ReadArgs(k=views[0][1].data_ptr(), v=views[1][1].data_ptr(), k_row_stride=views[0][1].stride(0),
                           k_head_stride=views[0][1].stride(1), v_row_stride=views[1][1].stride(0),
                           v_head_stride=views[1][1].stride(1), type=R.type_id(out_t))
        ok(L, L.mossgpu_kv8_read(dev.struct(M), seqs, ra, stream()))
        alone = torch.full_like(views[1][0], SENTINEL)
        ra.k, ra.v = None, alone.data_ptr() + views[1][1].storage_offset() * alone.element_size()
        ok(L, L.mossgpu_kv8_read(dev.struct(M), seqs, ra, stream()))
        assert status(L) == 0
        assert torch.equal(torch.nan_to_num(alone.float()), torch.nan_to_num(views[1][0].float()))
        for half in (0, 1):
            buf, view = views[half]
            want = torch.full(view.shape, SENTINEL, dtype=out_t)
            for s, slot in enumerate(slots):
                n = starts[s + 1] - starts[s]
                if n:
                    # one fp32 product of a code of 8 bits and the scale, then the type's rounding
                    want[starts[s] : starts[s + 1]] = cache.heads(slot, ctx[s] + n, half)[ctx[s] :].float().to(out_t)
            got = view.cpu()
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))
            gaps = torch.ones_like(buf, dtype=torch.bool)
            gaps.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(False)
            assert (buf[gaps] == SENTINEL).all()


@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("given_pos", [True, False])
def test_append_turns_keys_and_queries(M, L, t, inter, given_pos):
    dim, kvh, group, rot, mag, fmt = 128, 4, 3, 96, 1.1, R.INT8
    starts, slots, ctx = layout(LENGTHS["ragged"], lead=1)
    rows = starts[-1] + 2
    cache = R.Cache(fmt, kvh, dim, len(slots), 4, seed=1)
    g = torch.Generator().manual_seed(2)
    k, v, q = (torch.randn(rows, h, dim, generator=g).to(t) for h in (kvh, kvh, kvh * group))
    freq = R.freqs(rot)
    steps = torch.from_numpy(R.steps_of(freq).view(np.int64)).cuda()
    pos = torch.randint(0, 100000, (rows,), generator=g, dtype=torch.int32)
    at = np.zeros(rows, np.int64)
    for s in range(len(slots)):
        for i in range(starts[s + 1] - starts[s]):
            at[starts[s] + i] = int(pos[starts[s] + i]) if given_pos else ctx[s] + i
    dev = cache.cuda()
    keep, seqs = batch(M, starts, slots, ctx, rows)
    qd, kd, vd, pd = q.cuda(), k.cuda(), v.cuda(), pos.cuda()
    q_out = torch.full_like(qd, SENTINEL)
    rope = M.Rope(steps.data_ptr(), rot, int(inter), mag)
    ok(L, L.mossgpu_kv8_append(dev.struct(M), seqs, rope, append_args(M, kd, vd, qd, q_out, pd if given_pos else None), stream()))
    assert status(L) == 0
    live = slice(starts[0], starts[-1])
    q64 = torch.from_numpy(R.rope64(q.double().numpy(), at, freq, inter, mag))[live]
    size = torch.nn.functional.pad(torch.full((rot,), 1.0, dtype=torch.float64), (0, dim - rot)) * 4.5 * 2 * mag * 2.0**-20
    got = q_out.cpu().double()
    # inputs stay below 4.5 (normal, a few thousand of them); angle and products as in test_rope
    assert (q.abs() < 4.5).all() and ((got[live] - q64).abs() <= q64.abs() * R.half_step(t) + size).all()
    assert (q_out[: starts[0]] == SENTINEL).all() and (q_out[starts[-1] :] == SENTINEL).all()
    k64 = torch.from_numpy(R.rope64(k.double().numpy(), at, freq, inter, mag))
    out = cache.cuda()
    out.codes, out.scales = dev.codes.cpu(), dev.scales.cpu()
    out.table = cache.table
    for s, slot in enumerate(slots):
        n = starts[s + 1] - starts[s]
        rows_s = slice(starts[s], starts[s + 1])
        for half, want in ((0, k64[rows_s]), (1, v.double()[rows_s])):
            got = out.heads(slot, ctx[s] + n, half)[ctx[s] :]
            scale = want.abs().amax(-1, keepdim=True) / 127
            # half a code, and the rotation's own error
            assert ((got - want).abs() <= scale * (0.5 + 127 * 2.0**-22) + (2.0**-18 if half == 0 else 0)).all()
    # in place: q_out is q
    again = cache.cuda()
    ok(L, L.mossgpu_kv8_append(again.struct(M), seqs, rope, append_args(M, kd, vd, qd, qd, pd if given_pos else None), stream()))
    torch.cuda.synchronize()
    assert torch.equal(qd[live], q_out[live]) and torch.equal(qd[: starts[0]].cpu(), q[: starts[0]])
    assert torch.equal(again.codes, dev.codes)


# ---- attention -------------------------------------------------------------------------------


def attend(M, L, dev, seqs, q, out, scale, mask=None, ws=None):
    need = L.mossgpu_attention_kv8_workspace_bytes(dev.struct(M), q.shape[1], q.shape[0])
    if ws is None:
        ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")  # any contents
    a = M.AttentionKV8Args(q=q.data_ptr(), out=out.data_ptr(), mask=mask.data_ptr() if mask is not None else None,
                           workspace=ws.data_ptr(), workspace_bytes=ws.numel(), q_row_stride=q.stride(0),
                           q_head_stride=q.stride(1), out_row_stride=out.stride(0), out_head_stride=out.stride(1),
                           q_heads=q.shape[1], type=R.type_id(q.dtype), mask_words=mask.shape[1] if mask is not None else 0,
                           scale=scale)
    ok(L, L.mossgpu_attention_kv8(dev.struct(M), seqs, a, stream()))
    return ws


def tree(starts, words, seed):
    """Random trees: a row sees itself and the ancestors of a parent before it; the second row of the first sequence
    that has two sees none of the new rows."""
    rng = np.random.RandomState(seed)
    mask = np.zeros((starts[-1], words), np.uint32)
    for s in range(len(starts) - 1):
        for i in range(starts[s + 1] - starts[s]):
            up = rng.randint(-1, i) if i else -1
            r = starts[s] + i
            if up >= 0:
                mask[r] = mask[starts[s] + up]
            if i // 32 < words:
                mask[r, i // 32] |= np.uint32(1 << (i % 32))
    blank = next((starts[s] + 1 for s in range(len(starts) - 1) if starts[s + 1] - starts[s] > 1), None)
    if blank is not None:
        mask[blank] = 0
    return torch.from_numpy(mask.view(np.int32))


ATTEND = {  # (new rows, context)
    "single": [(1, 0)],
    "edges": [(1, c) for c in (0, 1, 14, 15, 16, 30, 31, 32, 33, 47, 63, 64, 100)],
    "new": [(2, 0), (9, 7), (0, 5), (16, 31), (33, 40), (17, 0)],
    "long": [(1, 1500), (3, 2000), (2, 3)],
    "empty": [(0, 10), (1, 5), (0, 0)],
}


@pytest.mark.parametrize("lengths", list(ATTEND))
@pytest.mark.parametrize("use_mask", [False, True])
@pytest.mark.parametrize("t", R.TYPES)
@pytest.mark.parametrize("fmt,dim,kvh,group", [(R.INT8, 64, 12, 1), (R.E4M3, 64, 2, 4), (R.INT8, 128, 2, 3), (R.E4M3, 128, 1, 16)])
def test_attention(M, L, lengths, use_mask, t, fmt, dim, kvh, group):
    starts, slots, ctx = layout(ATTEND[lengths])
    rows = starts[-1] + 2
    need = max(c + n for n, c in ATTEND[lengths])
    cache = R.Cache(fmt, kvh, dim, len(slots), need // 16 + 2, seed=3)
    for s, slot in enumerate(slots):
        cache.fill(slot, ctx[s] + starts[s + 1] - starts[s], 100 + s)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(rows, kvh * group, dim, generator=g).to(t)
    mask = tree(starts, 1, 5) if use_mask else None  # one word: new rows from 32 on are not seen
    scale = dim**-0.5 * 1.3
    want, mass, top = R.attend64(cache, q[: starts[-1]].double(), starts, slots, ctx, scale, mask)
    pad = 0 if dim == 64 else 8
    _, qv = strided(rows, kvh * group, dim, t, pad)
    qv.copy_(q)
    buf, out = strided(rows, kvh * group, dim, t, pad)
    dev = cache.cuda()
    keep, seqs = batch(M, starts, slots, ctx, rows)
    dm = mask.cuda() if use_mask else None
    if use_mask:
        dm = torch.cat([dm, torch.full((2, 1), -1, dtype=torch.int32, device="cuda")])
    ws = attend(M, L, dev, seqs, qv, out, scale, dm)
    assert status(L) == 0
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    assert ((got[: starts[-1]] - want).abs() <= R.attend_tolerance(mass, top, want, t)).all()
    live = torch.zeros_like(buf, dtype=torch.bool)
    live.as_strided(out[: starts[-1]].shape, out.stride(), out.storage_offset()).fill_(True)
    assert (buf[~live] == SENTINEL).all()  # rows behind the last sequence, and the gaps
    # the same workspace again: the same bits
    again = torch.zeros_like(buf).as_strided(out.shape, out.stride(), out.storage_offset())
    attend(M, L, dev, seqs, qv, again, scale, dm, ws)
    torch.cuda.synchronize()
    assert torch.equal(again[: starts[-1]], out[: starts[-1]])


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("new,group", [(1, 1), (3, 4), (20, 4), (60, 4)])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_attention_any_sign_of_the_scale(M, L, t, new, group, scale):
    # the forms for few, some and many rows, each with and without a split over positions
    for seqs_n in (2, 300):
        lengths = [(new, 37 * (i % 3)) for i in range(seqs_n)]
        starts, slots, ctx = layout(lengths)
        cache = R.Cache(R.E4M3, 2, 64, seqs_n, 9, seed=3)
        for s in range(min(seqs_n, 6)):
            cache.fill(slots[s], ctx[s] + new, s)
        for s in range(6, seqs_n):  # the others share the first ones' pages: they are read only
            cache.table[slots[s]] = cache.table[slots[s % 6]]
        q = torch.randn(starts[-1], 2 * group, 64, generator=torch.Generator().manual_seed(1)).to(t)
        out = torch.empty_like(q, device="cuda")
        keep, seqs = batch(M, starts, slots, ctx, starts[-1])
        attend(M, L, cache.cuda(), seqs, q.cuda(), out, scale)
        assert status(L) == 0
        n = 6 if seqs_n > 6 else seqs_n
        want, mass, top = R.attend64(cache, q[: starts[n]].double(), starts[: n + 1], slots[:n], ctx[:n], scale)
        assert ((out[: starts[n]].cpu().double() - want).abs() <= R.attend_tolerance(mass, top, want, t)).all()
        if seqs_n > 6:  # later sequences have the cache of one of the first six, but its own queries
            for s in (6, 47, 299):
                own = R.attend64(cache, q[starts[s] : starts[s + 1]].double(), [0, new], [slots[s]], [ctx[s]], scale)
                assert ((out[starts[s] : starts[s + 1]].cpu().double() - own[0]).abs() <= R.attend_tolerance(own[1], own[2], own[0], t)).all()


@pytest.mark.parametrize("dim,new,group,t", [(64, 1, 1, F32), (128, 1, 2, BF16), (64, 2, 3, F32), (128, 2, 8, BF16), (64, 3, 8, F16)])
def test_attention_the_most_sequences(M, L, dim, new, group, t):
    # 4096 sequences, some without rows, that all read a few slots' pages
    n = 4096
    lengths = [(0 if i % 7 == 3 else new, i % 50) for i in range(n)]
    starts, slots, ctx = layout(lengths)
    cache = R.Cache(R.INT8, 1, dim, n, 4, seed=3)
    for s in range(50):
        cache.fill(slots[s], 49 + new, s)
    for s in range(50, n):
        cache.table[slots[s]] = cache.table[slots[s % 50]]
    q = torch.randn(starts[-1], group, dim, generator=torch.Generator().manual_seed(1)).to(t)
    buf = torch.full((starts[-1] + 1, group, dim), SENTINEL, dtype=t, device="cuda")
    keep, seqs = batch(M, starts, slots, ctx, starts[-1])
    attend(M, L, cache.cuda(), seqs, q.cuda(), buf[: starts[-1]], dim**-0.5)
    assert status(L) == 0 and (buf[-1] == SENTINEL).all()
    got = buf[: starts[-1]].cpu().double()
    assert torch.isfinite(got).all()
    for s in list(range(0, n, 97)) + [n - 1]:
        if starts[s + 1] > starts[s]:
            rows = slice(starts[s], starts[s + 1])
            want, mass, top = R.attend64(cache, q[rows].double(), [0, new], [slots[s]], [ctx[s]], float(np.float32(dim**-0.5)))
            assert ((got[rows] - want).abs() <= R.attend_tolerance(mass, top, want, t)).all()


def test_attention_misaligned_rows(M, L):
    # odd strides and a base off 16 bytes: element-wise loads and stores
    for t in R.TYPES:
        starts, slots, ctx = layout(ATTEND["new"])
        cache = R.Cache(R.INT8, 3, 64, len(slots), 6, seed=3)
        for s, slot in enumerate(slots):
            cache.fill(slot, ctx[s] + starts[s + 1] - starts[s], s)
        q = torch.randn(starts[-1], 6, 64, generator=torch.Generator().manual_seed(1)).to(t)
        want, mass, top = R.attend64(cache, q.double(), starts, slots, ctx, 0.125)
        _, qv = strided(starts[-1], 6, 64, t, pad=1, lead=3)
        qv.copy_(q)
        buf, out = strided(starts[-1], 6, 64, t, pad=5, lead=1)
        keep, seqs = batch(M, starts, slots, ctx, starts[-1])
        attend(M, L, cache.cuda(), seqs, qv, out, 0.125)
        assert ((out.cpu().double() - want).abs() <= R.attend_tolerance(mass, top, want, t)).all()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("scale_of", [1e-30, 1e-5, 1e4, 1e25])
def test_attention_far_ranges(M, L, t, scale_of):
    # tiny and huge queries, and V scales that grow along the sequence by 2^40
    dim, kvh = 64, 2
    cache = R.Cache(R.INT8, kvh, dim, 1, 10, seed=3)
    cache.fill(0, 150, 1)
    grow = torch.exp2(torch.arange(150) * 40.0 / 150 - 20)
    for p in range(150):
        page = int(cache.table[0, p // 16])
        cache.scales[page, 1, :, p % 16] *= grow[p]
    q = (torch.randn(1, kvh, dim, generator=torch.Generator().manual_seed(2)) * scale_of).to(t)
    scale = 0.125 / scale_of
    want, mass, top = R.attend64(cache, q.double(), [0, 1], [0], [149], float(np.float32(scale)))
    out = torch.empty_like(q, device="cuda")
    keep, seqs = batch(M, [0, 1], [0], [149], 1)
    attend(M, L, cache.cuda(), seqs, q.cuda(), out, scale)
    # a weight whose V scale is far below the largest keeps an absolute error of 2^-25 * 2^-13 of that one: below the rest
    assert ((out.cpu().double() - want).abs() <= 1.5 * R.attend_tolerance(mass, top, want, t)).all()


def test_attention_nan_only_where_it_is_seen(M, L):
    # NaN scales at a context position (seen by all), and at a drafted one (seen by its descendants only)
    dim, kvh = 64, 2
    for fmt in (R.INT8, R.E4M3):
        for half in (0, 1):
            cache = R.Cache(fmt, kvh, dim, 2, 4, seed=1)
            cache.fill(0, 40, 1)
            cache.fill(1, 40, 2)
            for slot, pos in ((0, 36), (1, 5)):
                page = int(cache.table[slot, pos // 16])
                cache.scales[page, half, 1, pos % 16] = float("nan")
                cache.codes[page, half, 1, pos % 16] = 0
            mask = torch.tensor([[1], [3], [5], [13], [1], [2]], dtype=torch.int32)  # of rows 0..3 rows 1 alone sees new row 1
            q = torch.randn(6, kvh, dim, generator=torch.Generator().manual_seed(2))
            out = torch.zeros_like(q, device="cuda")
            keep, seqs = batch(M, [0, 4, 6], [0, 1], [35, 38], 6)
            attend(M, L, cache.cuda(), seqs, q.cuda(), out, 0.125, mask.cuda())
            got = out.cpu()
            bad = torch.isnan(got).all(-1)
            want = torch.zeros(6, kvh, dtype=torch.bool)
            want[1, 1] = True   # the drafted token
            want[4:, 1] = True  # the context
            assert torch.equal(bad, want) and torch.equal(torch.isnan(got).any(-1), want)


def test_bad_device_values_are_skipped_and_reported(M, L):
    dim, kvh = 64, 2
    cache = R.Cache(R.INT8, kvh, dim, 2, 2, seed=1)
    cache.fill(0, 32, 1)
    cache.fill(1, 32, 1)
    k = torch.randn(4, kvh, dim).cuda()
    out = torch.full((4, kvh, dim), SENTINEL, device="cuda")

    def ops(starts, slots, ctx, table=None):
        dev = cache.cuda()
        if table is not None:
            dev.table = table.cuda()
        keep, seqs = batch(M, starts, slots, ctx, 4)
        codes = []
        assert status(L) == 0
        ok(L, L.mossgpu_kv8_append(dev.struct(M), seqs, None, append_args(M, k, k), stream()))
        codes.append(status(L))
        assert status(L) == 0  # reading clears it
        ra = M.KV8ReadArgs(k=out.data_ptr(), v=None, k_row_stride=kvh * dim, k_head_stride=dim, type=0)
        ok(L, L.mossgpu_kv8_read(dev.struct(M), seqs, ra, stream()))
        codes.append(status(L))
        o = torch.zeros_like(out)
        attend(M, L, dev, seqs, k, o, 0.125)
        codes.append(status(L))
        return codes, dev, o

    codes, dev, _ = ops([0, 4], [0], [30])          # the slot ends two rows early
    assert codes == [9, 9, 9]
    assert (out[2:] == SENTINEL).all() and (out[:2] != SENTINEL).any()
    for slots, ctx in (([2], [0]), ([-1], [0]), ([0], [-1]), ([0], [2**31 - 1]), ([0], [33])):
        codes, dev, _ = ops([0, 4], slots, ctx)
        assert codes == [9, 9, 9]
        assert torch.equal(dev.codes.cpu(), cache.codes)
    table = cache.table.clone()
    table[0, 0], table[0, 1] = cache.pages, -5
    codes, dev, o = ops([0, 4], [0], [14], table)   # pages outside the pool
    assert codes == [10, 10, 10]
    assert torch.equal(dev.codes.cpu(), cache.codes) and (o == 0).all()  # no position there: nothing seen
    codes, dev, _ = ops([0, 2**30], [0], [0])       # row bounds past the rows are cut
    assert codes == [0, 0, 0]
    codes, dev, _ = ops([3, -7], [0], [0])
    assert codes == [0, 0, 0]
    assert torch.equal(dev.codes.cpu(), cache.codes)


def test_streams_and_graphs(M, L):
    # a step of append and attention captured twice, with a workspace each, replayed on two streams at once
    dim, kvh, fmt, t = 64, 4, R.E4M3, F32
    starts, slots, ctx = layout(ATTEND["long"])
    rows = starts[-1]
    freq = R.freqs(64)
    steps = torch.from_numpy(R.steps_of(freq).view(np.int64)).cuda()
    rope = M.Rope(steps.data_ptr(), 64, 1, 1.0)
    base = R.Cache(fmt, kvh, dim, len(slots), 130, seed=3)
    for s, slot in enumerate(slots):
        base.fill(slot, ctx[s] + starts[s + 1] - starts[s], s)
    runs = []
    for i in range(2):
        g = torch.Generator().manual_seed(i)
        k, v, q = (torch.randn(rows, kvh, dim, generator=g).cuda() for _ in range(3))
        dev = base.cuda()
        keep, seqs = batch(M, starts, slots, ctx, rows)
        q_out, out = torch.empty_like(q), torch.empty_like(q)
        ws = torch.empty(L.mossgpu_attention_kv8_workspace_bytes(dev.struct(M), kvh, rows), dtype=torch.uint8, device="cuda")

        def step(dev=dev, seqs=seqs, k=k, v=v, q=q, q_out=q_out, out=out, ws=ws):
            ok(L, L.mossgpu_kv8_append(dev.struct(M), seqs, rope, append_args(M, k, v, q, q_out), stream()))
            attend(M, L, dev, seqs, q_out, out, 0.125, None, ws)

        step()
        torch.cuda.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((graph, out, want, torch.cuda.Stream(), (k, v, q, q_out, ws, keep, dev)))
    for _ in range(20):
        for graph, out, want, st, _keep in runs:
            with torch.cuda.stream(st):
                out.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for graph, out, want, st, _keep in runs:
        assert torch.equal(out, want)
    assert status(L) == 0


def test_long_pool_offsets(M, L):
    # pages whose byte offsets pass 2^32: 3 million pages of 2 heads
    dim, kvh = 128, 1
    pages = (2**32) // (2 * kvh * 16 * dim) + 1000
    codes = torch.zeros(pages * 2 * kvh * 16 * dim, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(pages * 2 * kvh * 16, device="cuda")
    table = torch.tensor([[pages - 1, pages - 3, 0, pages - 2]], dtype=torch.int32, device="cuda")
    c = M.KV8Cache(codes.data_ptr(), scales.data_ptr(), table.data_ptr(), pages, 1, 4, kvh, dim, R.INT8)
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(64, kvh, dim, generator=g).cuda(), torch.randn(64, kvh, dim, generator=g).cuda()
    keep, seqs = batch(M, [0, 64], [0], [0], 64)
    ok(L, L.mossgpu_kv8_append(c, seqs, None, append_args(M, k, v), stream()))
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    ra = M.KV8ReadArgs(k=kb.data_ptr(), v=vb.data_ptr(), k_row_stride=dim, k_head_stride=dim, v_row_stride=dim,
                       v_head_stride=dim, type=0)
    ok(L, L.mossgpu_kv8_read(c, seqs, ra, stream()))
    assert status(L) == 0
    for x, b in ((k, kb), (v, vb)):
        assert ((x - b).abs() <= x.abs().amax(-1, keepdim=True) / 127 * 0.5001).all()
    q = torch.randn(64, 2, dim, generator=g).cuda()
    out = torch.empty_like(q)
    ws = torch.empty(L.mossgpu_attention_kv8_workspace_bytes(c, 2, 64), dtype=torch.uint8, device="cuda")
    a = M.AttentionKV8Args(q=q.data_ptr(), out=out.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                           q_row_stride=2 * dim, q_head_stride=dim, out_row_stride=2 * dim, out_head_stride=dim, q_heads=2,
                           type=0, scale=0.1)
    ok(L, L.mossgpu_attention_kv8(c, seqs, a, stream()))
    s = torch.einsum("ihd,jd->hij", q.double(), kb[:, 0].double()) * 0.1
    s.masked_fill_(~torch.ones(64, 64, dtype=torch.bool, device="cuda").tril(), float("-inf"))
    want = torch.einsum("hij,jd->ihd", torch.softmax(s, -1), vb[:, 0].double())
    # the scores stay below 2^6 with |q||k| sums of that order: attend_tolerance gives under 1e-3 of max |v| (about 4)
    assert ((out.double() - want).abs() <= 2.5e-4).all()


@pytest.mark.parametrize("fmt", [R.INT8, R.E4M3])
@pytest.mark.parametrize("t", [F32, BF16])
def test_prompt_draft_score_and_next_token(M, L, fmt, t):
    # the operators as a server runs them, one layer: a prompt, a tree of drafted tokens that share rotary positions by
    # depth, the drafts' log-probabilities, the accepted branch moved (read, appended again), one more token
    import test_op_logprobs as P
    kvh, group, dim, vocab, rot = 2, 3, 64, 777, 48
    qh = kvh * group
    g = torch.Generator().manual_seed(7)
    cache = R.Cache(fmt, kvh, dim, 2, 6, seed=2)
    dev = cache.cuda()
    steps, mag = M.rope_steps(rot)
    steps = torch.from_numpy(steps.view(np.int64)).cuda()
    rope = M.Rope(steps.data_ptr(), rot, 0, mag)
    head = torch.randn(qh * dim, vocab, generator=g).cuda()

    def step(starts, ctx, mask=None, pos=None):
        rows = starts[-1]
        k, v, q = (torch.randn(rows, h, dim, generator=g).to(t).cuda() for h in (kvh, kvh, qh))
        keep, seqs = batch(M, starts, [1, 0], ctx, rows)
        pd = torch.tensor(pos, dtype=torch.int32).cuda() if pos is not None else None
        md = mask.cuda() if mask is not None else None
        out = torch.empty_like(q)
        ok(L, L.mossgpu_kv8_append(dev.struct(M), seqs, rope, append_args(M, k, v, q, q, pd), stream()))
        attend(M, L, dev, seqs, q, out, 0.125, md)
        assert status(L) == 0
        host = R.Cache.__new__(R.Cache)
        host.__dict__.update(cache.__dict__)
        host.codes, host.scales = dev.codes.cpu(), dev.scales.cpu()
        want, mass, top = R.attend64(host, q.cpu().double(), starts, [1, 0], ctx, 0.125, mask)
        assert ((out.cpu().double() - want).abs() <= R.attend_tolerance(mass, top, want, t)).all()
        return out

    step([0, 37, 60], [0, 0])                                   # prompts of 37 and 23
    # drafts: 0 -> 1 -> 3, 0 -> 2 for the first, a chain of two for the second
    mask = torch.tensor([[0b1], [0b11], [0b101], [0b1011], [0b1], [0b11]], dtype=torch.int32)
    out = step([0, 4, 6], [37, 23], mask, [37, 38, 38, 39, 23, 24])
    logits = (out.float().view(6, -1) @ head).contiguous()
    drafted = torch.randint(0, vocab, (6,), generator=g, dtype=torch.int32)
    P.check(logits.cpu(), drafted, 5, 1.0, P.run(M, logits, drafted.cuda(), 5))
    # the first sequence accepts 0, 2: position 39 (draft 2) moves to 38, without another rounding of the codes' values
    k1 = torch.empty(1, kvh, dim, device="cuda")
    v1 = torch.empty_like(k1)
    keep, seqs = batch(M, [0, 1], [1], [39], 1)
    ok(L, L.mossgpu_kv8_read(dev.struct(M), seqs, M.KV8ReadArgs(k=k1.data_ptr(), v=v1.data_ptr(), k_row_stride=kvh * dim,
                             k_head_stride=dim, v_row_stride=kvh * dim, v_head_stride=dim, type=0), stream()))
    keep2, seqs = batch(M, [0, 1], [1], [38], 1)
    ok(L, L.mossgpu_kv8_append(dev.struct(M), seqs, None, append_args(M, k1, v1), stream()))
    assert status(L) == 0
    page, was, now = int(cache.table[1, 2]), 39 - 32, 38 - 32
    assert torch.equal(dev.codes[page, :, :, now], dev.codes[page, :, :, was])
    step([0, 1, 2], [39, 25])                                   # the next token of both
