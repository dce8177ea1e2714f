"""The standalone 8-bit-cache, rotary, drafted-token attention and log-probability operators:
their cases, their plain forms, their calls and their values in 64 bits.

`run` computes a case's operator in elementary torch operations (`own` false) or through the
library's C ABI (`own` true).  Sequences are ragged: lengths are spread evenly between a case's
bounds and dealt to the sequences by the seed, so that the work of a case does not depend on it.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CTYPE = {"f32": 0, "f16": 1, "bf16": 2}
FORMAT = {"int8": 0, "e4m3": 1}
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -----------------------------------------------------------------------------------


def listed():
    return [
        # the queries of one decode step of 8 streams of the framework's own model (12 heads of 64)
        dict(name="rope_step", op="rope", rows=8, heads=12, dim=64, rot=64, inter=True, scaled=False, inverse=False,
             top=4608, type="f32"),
        # the q and k heads of a long prompt, part of a 128-wide head, positions far past the trained length
        dict(name="rope_prompt", op="rope", rows=8191, heads=40, dim=128, rot=96, inter=False, scaled=True,
             inverse=False, top=1 << 20, type="bf16"),
        # one new token of each of 64 streams goes into an e4m3 cache, its query rotated in the same call
        dict(name="append_step", op="append", seqs=64, new_min=1, new_max=1, ctx_min=64, ctx_max=1024, qh=12, kvh=12,
             dim=64, rot=64, inter=True, scaled=False, type="f32", format="e4m3"),
        # 16 prompts of up to 512 tokens, grouped heads, half layout
        dict(name="append_prompts", op="append", seqs=16, new_min=17, new_max=512, ctx_min=0, ctx_max=900, qh=32,
             kvh=8, dim=128, rot=128, inter=False, scaled=True, type="bf16", format="e4m3"),
        # new tokens are written and the same positions read back, as a draft is when it is accepted elsewhere
        dict(name="append_read", op="round", seqs=24, new_min=1, new_max=63, ctx_min=0, ctx_max=700, qh=0, kvh=12,
             dim=64, rot=64, inter=True, scaled=False, type="f16", format="int8"),
        # whole contexts leave the 8-bit cache in 16 bits, for a prefix that is handed on
        dict(name="read_contexts", op="read", seqs=48, new_min=300, new_max=4096, ctx_min=0, ctx_max=0, kvh=8, dim=128,
             type="bf16", format="e4m3"),
        # one stream's next token: latency
        dict(name="attend_one", op="attend", seqs=1, new_min=1, new_max=1, ctx_min=300, ctx_max=300, qh=12, kvh=12,
             dim=64, tree=False, type="f32", format="int8"),
        # 512 streams of the framework's model, 256 to 4096 cached positions, one token each
        dict(name="attend_512", op="attend", seqs=512, new_min=1, new_max=1, ctx_min=256, ctx_max=4096, qh=12, kvh=12,
             dim=64, tree=False, type="f32", format="int8"),
        # trees of 5 to 24 drafted tokens over long contexts, grouped heads
        dict(name="attend_trees", op="attend", seqs=48, new_min=5, new_max=24, ctx_min=700, ctx_max=8000, qh=32, kvh=8,
             dim=128, tree=True, type="bf16", format="e4m3"),
        # the 16 audio heads of one stream's frame: latency
        dict(name="score_frame", op="score", rows=16, vocab=1024, top=5, hot=1.0, type="f32"),
        # the 16 audio heads of 512 streams
        dict(name="score_512", op="score", rows=8192, vocab=1024, top=8, hot=0.8, type="f32"),
        # drafted text tokens over a large vocabulary
        dict(name="score_vocab", op="score", rows=160, vocab=128001, top=20, hot=1.3, type="bf16"),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["rope", "append", "round", "read", "attend", "attend", "score", "score"])
    kind = rng.choice(["f32", "f16", "bf16"])
    form = rng.choice(["int8", "e4m3"])
    dim = rng.choice([64, 128])
    kvh = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        return dict(op=op, rows=log(1, 4000), heads=rng.choice([1, 5, 12, 24, 32]), dim=dim,
                    rot=2 * rng.randint(1, dim // 2), inter=rng.random() < 0.5, scaled=rng.random() < 0.5,
                    inverse=rng.random() < 0.3, top=log(100, 1 << 20), type=kind)
    if op in ("append", "round"):
        new_max = log(1, 400)
        # the rounded bits of int8 codes come back through the read, in 16 bits
        return dict(op=op, seqs=log(1, 60), new_min=rng.randint(0, 1) if new_max > 1 else 1, new_max=new_max, ctx_min=0,
                    ctx_max=log(1, 1500), qh=kvh * group if op == "append" else 0, kvh=kvh, dim=dim,
                    rot=2 * rng.randint(1, dim // 2), inter=rng.random() < 0.5, scaled=rng.random() < 0.5,
                    type=kind if op == "append" else rng.choice(["f16", "bf16"]),
                    format="e4m3" if op == "append" else form)
    if op == "read":
        return dict(op=op, seqs=log(1, 40), new_min=1, new_max=log(2, 3000), ctx_min=0, ctx_max=log(1, 500), kvh=kvh,
                    dim=dim, type=kind, format=form)
    if op == "attend":
        tree = rng.random() < 0.5
        new_max = log(2, 64) if tree else rng.choice([1, 1, 1, log(2, 90)])
        seqs = log(1, 300)
        new_max = max(1, min(new_max, 3000 // seqs))
        # positions a sequence that keep the case below the largest
        room = min(400_000_000 // (seqs * kvh * dim), 30_000_000_000 // (seqs * new_max * kvh * group * dim))
        return dict(op=op, seqs=seqs, new_min=1, new_max=new_max, ctx_min=0, ctx_max=log(16, max(17, min(16000, room))),
                    qh=kvh * group, kvh=kvh, dim=dim, tree=tree, type=kind, format=form)
    vocab = log(40, 200_000)
    return dict(op="score", rows=log(1, max(2, min(8000, 20_000_000 // vocab))), vocab=vocab, top=rng.randint(0, 32),
                hot=rng.choice([0.7, 1.0, 1.6]), type=kind)


def spread(lo, hi, n):
    """n whole lengths, evenly between lo and hi."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def work(case):
    c, op = case, case["op"]
    if op == "rope":
        n = c["rows"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * SIZE[c["type"]] + 4 * c["rows"], "flops": 3 * n * c["rot"]}
    if op == "score":
        return {"bytes": c["rows"] * (c["vocab"] * SIZE[c["type"]] + 12 + 8 * c["top"]), "flops": 4 * c["rows"] * c["vocab"]}
    new, ctx = spread(c["new_min"], c["new_max"], c["seqs"]), spread(c["ctx_min"], c["ctx_max"], c["seqs"])
    rows, size, cell = sum(new), SIZE[c["type"]], c["kvh"] * (c["dim"] + 4)
    if op == "read":
        return {"bytes": 2 * rows * (cell + c["kvh"] * c["dim"] * size), "flops": 2 * rows * c["kvh"] * c["dim"]}
    if op in ("append", "round"):
        moved = 2 * rows * (c["kvh"] * c["dim"] * size + cell) + 2 * rows * c["qh"] * c["dim"] * size
        if op == "round":  # read back
            moved += 2 * rows * (cell + c["kvh"] * c["dim"] * size)
        return {"bytes": moved, "flops": rows * (3 * (c["qh"] + c["kvh"]) * c["rot"] + 6 * c["kvh"] * c["dim"])}
    # the lengths are dealt so that the i-th context belongs to the i-th number of new tokens
    seen = sum(x + n for x, n in zip(ctx, new))
    pairs = sum(n * x + n * (n + 1) // 2 for x, n in zip(ctx, new))
    return {"bytes": 2 * seen * cell + 2 * rows * c["qh"] * c["dim"] * size, "flops": 4 * pairs * c["qh"] * c["dim"]}


# ---- inputs ----------------------------------------------------------------------------------


def frequencies(rot, scaled):
    """Angle a position, by pair: 10000^(-2i / rot); scaled ones are stretched 8-fold below one turn
    in 4096 positions, left as they are above 32 turns, and between the two in proportion."""
    f = 10000.0 ** (-2.0 * np.arange(rot // 2, dtype=np.float64) / rot)
    if scaled:
        turns = 4096.0 * f / (2.0 * np.pi)
        keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
        f = f * keep + f / 8.0 * (1.0 - keep)
    return f


def rotary(case, dev):
    """The angles and the same as whole 2^-64 turns a position, which is the form the library takes."""
    f = frequencies(case["rot"], case["scaled"])
    steps = [int(round(math.ldexp(x / (2.0 * math.pi), 64))) % (1 << 64) for x in f.tolist()]
    steps = torch.tensor([s - (1 << 64) if s >= 1 << 63 else s for s in steps], dtype=torch.int64, device=dev)
    return torch.tensor(f, dtype=torch.float64, device=dev), steps, 0.1 * math.log(8.0) + 1.0 if case["scaled"] else 1.0


def pool(case, g, dev, total, filled):
    """A paged pool in which every sequence's positions lie on pages of their own in mixed order.  What no
    position fills holds whatever was there before: random codes, scales that are no numbers."""
    n, kvh, dim = case["seqs"], case["kvh"], case["dim"]
    need = [-(-t // PAGE) for t in total]
    width, pages = max(1, max(need)), max(1, sum(need))
    order = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    col = torch.arange(width, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table[col] = order[: sum(need)]
    x = torch.randn(pages, 2, kvh, PAGE, dim, generator=g, device=dev)
    if case["format"] == "int8":
        codes = (x * 36.0).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        codes = (x * 130.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    del x
    scales = torch.exp(0.3 * torch.randn(pages, 2, kvh, PAGE, generator=g, device=dev)) * (3.4 / CODE_MAX[case["format"]])
    place = torch.full((pages * PAGE,), False, device=dev)
    at = torch.arange(width * PAGE, device=dev)
    live = at[None, :] < torch.tensor(filled, device=dev)[:, None]
    cell = (table.long().clamp(min=0) * PAGE).repeat_interleave(PAGE, 1) + at % PAGE
    place[cell[live]] = True
    scales.masked_fill_(~place.view(pages, 1, 1, PAGE), float("nan"))
    return codes, scales, table


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    c, op = case, case["op"]
    kind = TYPES[c["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(kind)

    s = {"case": dict(c)}
    if op == "rope":
        s["x"] = normal(c["rows"], c["heads"], c["dim"])
        s["pos"] = torch.randint(0, c["top"], (c["rows"],), generator=g, device=dev, dtype=torch.int32)
        s["freq"], s["steps"], s["mag"] = rotary(c, dev)
        s["out"] = torch.empty_like(s["x"])
        return s
    if op == "score":
        s["x"] = (torch.randn(c["rows"], c["vocab"], generator=g, device=dev) * 2.5).to(kind)
        banned = torch.rand(c["rows"], c["vocab"], generator=g, device=dev) < 0.02
        s["x"].masked_fill_(banned, float("-inf"))
        del banned
        s["tok"] = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=dev, dtype=torch.int32)
        s["tok"][torch.rand(c["rows"], generator=g, device=dev) < 0.05] = -1
        s["lp"] = torch.empty(c["rows"], device=dev)
        s["ent"] = torch.empty(c["rows"], device=dev)
        s["ids"] = torch.empty(c["rows"], c["top"], dtype=torch.int32, device=dev)
        s["top"] = torch.empty(c["rows"], c["top"], device=dev)
        return s
    n = c["seqs"]
    deal = torch.randperm(n, generator=g, device=dev).tolist()
    new, ctx = spread(c["new_min"], c["new_max"], n), spread(c["ctx_min"], c["ctx_max"], n)
    new, ctx = [new[i] for i in deal], [ctx[i] for i in deal]
    total = [a + b for a, b in zip(new, ctx)]
    s["codes"], s["scales"], s["table"] = pool(c, g, dev, total, total if op in ("attend", "read") else ctx)
    start = np.concatenate([[0], np.cumsum(new)])
    rows = s["rows"] = int(start[-1])
    s["start"] = torch.tensor(start, dtype=torch.int32, device=dev)
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=dev)
    s["slot"] = torch.arange(n, dtype=torch.int32, device=dev)
    s["width"], s["longest"] = max(total), max(new)
    if op != "attend":
        s["k_out"] = torch.empty(rows, c["kvh"], c["dim"], dtype=kind, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
    if op in ("append", "round"):
        s["k"], s["v"] = normal(rows, c["kvh"], c["dim"]), normal(rows, c["kvh"], c["dim"])
        s["freq"], s["steps"], s["mag"] = rotary(c, dev)
        if c["qh"]:
            s["q"] = normal(rows, c["qh"], c["dim"])
            s["q_out"] = torch.empty_like(s["q"])
    if op == "attend":
        s["q"] = normal(rows, c["qh"], c["dim"])
        s["out"] = torch.empty_like(s["q"])
        s["mask"] = None
        if c["tree"]:
            # each drafted token's parent is an earlier one or the context; it sees its ancestors and itself
            words = -(-s["longest"] // 32)
            rng = np.random.RandomState(seed % (1 << 31))
            mask = np.zeros((rows, words), np.uint32)
            for b in range(n):
                for i in range(new[b]):
                    up = rng.randint(-1, i) if i else -1
                    r = start[b] + i
                    if up >= 0:
                        mask[r] = mask[start[b] + up]
                    mask[r, i // 32] |= np.uint32(1 << (i % 32))
            s["mask"] = torch.from_numpy(mask.view(np.int32)).to(dev)
    return s


# ---- plain forms -----------------------------------------------------------------------------


def p_rope(x, pos, freq, mag, inter, inverse=False):
    rot = 2 * freq.numel()
    t = pos.double()[:, None] * freq[None, :]
    if inverse:
        t = -t
    cos, sin = (torch.cos(t) * mag).float()[:, None, :], (torch.sin(t) * mag).float()[:, None, :]
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if inter else (y[..., : rot // 2], y[..., rot // 2 : rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if inter else torch.cat([u, w], -1)
    return torch.cat([turned, y[..., rot:]], -1)


def p_quantise(x, form):
    """Codes and scales of heads x[..., dim] in fp32."""
    top = x.abs().amax(-1)
    scale = top / CODE_MAX[form]
    sound = torch.isfinite(top)
    zero = (scale < 2.0**-126) | ~sound
    y = torch.where(zero[..., None], torch.zeros_like(x), x) / torch.where(zero, torch.ones_like(scale), scale)[..., None]
    if form == "int8":
        codes = y.round().clamp(-127, 127).to(torch.int8)
    else:
        codes = y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), torch.where(sound, torch.where(zero, torch.zeros_like(scale), scale), torch.full_like(scale, float("nan")))


def p_places(s):
    """Of each new row: its sequence, its position, and the page and offset of that."""
    start = s["start"].long()
    r = torch.arange(s["rows"], device=start.device)
    b = torch.searchsorted(start, r, right=True) - 1
    pos = s["ctx"].long()[b] + r - start[b]
    return b, pos, s["table"].long()[s["slot"].long()[b], pos // PAGE], pos % PAGE


def p_values(codes, form):
    return codes.view(torch.int8).float() if form == "int8" else codes.view(torch.float8_e4m3fn).float()


def p_append(s):
    c = s["case"]
    _, pos, page, off = p_places(s)
    k = p_rope(s["k"], pos, s["freq"], s["mag"], c["inter"])
    for half, x in enumerate((k, s["v"].float())):
        codes, scale = p_quantise(x, c["format"])
        s["codes"][page, half, :, off] = codes
        s["scales"][page, half, :, off] = scale
    return p_rope(s["q"], pos, s["freq"], s["mag"], c["inter"]).to(s["q"].dtype) if c["qh"] else None


def p_read(s):
    c = s["case"]
    _, _, page, off = p_places(s)
    return [(p_values(s["codes"][page, half, :, off], c["format"]) * s["scales"][page, half, :, off][..., None])
            .to(TYPES[c["type"]]) for half in (0, 1)]


def p_attend(s):
    c = s["case"]
    n, kvh, dim, group = c["seqs"], c["kvh"], c["dim"], c["qh"] // c["kvh"]
    b, pos, _, _ = p_places(s)
    i = pos - s["ctx"].long()[b]
    q = torch.zeros(n, s["longest"], kvh, group, dim, device=b.device)
    q[b, i] = s["q"].float().view(-1, kvh, group, dim)
    wide = -(-s["width"] // PAGE)
    page = s["table"].long()[s["slot"].long(), :wide].clamp(min=0)
    at = torch.arange(wide * PAGE, device=b.device)
    total = s["ctx"].long() + (s["start"][1:] - s["start"][:-1]).long()
    kv = []
    for half in (0, 1):
        x = p_values(s["codes"][page, half], c["format"]) * s["scales"][page, half][..., None]  # [n][pages][kvh][16][dim]
        x = torch.where((at[None, :] < total[:, None]).view(n, wide, 1, PAGE, 1), x, torch.zeros_like(x))
        kv.append(x.transpose(2, 3).reshape(n, wide * PAGE, kvh, dim))
    score = torch.einsum("bikgd,bjkd->bkgij", q, kv[0]) * dim**-0.5
    seen = torch.zeros(n, s["longest"], wide * PAGE, dtype=torch.bool, device=b.device)
    ctx = s["ctx"].long()[b][:, None]
    j = at[None, :] - ctx  # which new token, for each row
    if s["mask"] is None:
        allowed = j <= i[:, None]
    else:
        word = s["mask"].long().gather(1, (j.clamp(0, s["longest"] - 1) // 32))
        allowed = (j < 0) | (((word >> (j.clamp(min=0) % 32)) & 1) != 0)
    seen[b, i] = allowed & (at[None, :] < total[b][:, None])
    seen = seen[:, None, None]
    score = torch.where(seen, score, torch.full_like(score, float("-inf")))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    mass = p.sum(-1, keepdim=True)
    p = p / torch.where(mass > 0, mass, torch.ones_like(mass))
    out = torch.einsum("bkgij,bjkd->bikgd", p, kv[1])
    return out[b, i].reshape(s["q"].shape).to(s["q"].dtype)


def p_score(s):
    c = s["case"]
    x = s["x"].float()
    y = x / c["hot"]
    top = y.amax(-1, keepdim=True)
    e = torch.exp(y - top)
    z = e.sum(-1, keepdim=True)
    norm = top + torch.log(z)
    tok = s["tok"].long()
    lp = torch.where(tok < 0, torch.zeros_like(norm[:, 0]), (y.gather(1, tok.clamp(min=0)[:, None]) - norm)[:, 0])
    ent = (torch.log(z) - (torch.where(e > 0, (y - top) * e, torch.zeros_like(e))).sum(-1, keepdim=True) / z)[:, 0]
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, : c["top"]]
    return {"logprob": lp, "entropy": ent, "top_ids": ids.int(), "top_logprobs": y.gather(1, ids) - norm}


# ---- the library's calls ---------------------------------------------------------------------


def package():
    import importlib.util
    import sys
    from pathlib import Path
    if "moss_b200" not in sys.modules:
        home = Path(__file__).resolve().parents[1] / "dsh-moss-tts_b200"
        spec = importlib.util.spec_from_file_location("moss_b200", home / "__init__.py", submodule_search_locations=[str(home)])
        sys.modules["moss_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["moss_b200"])
    return sys.modules["moss_b200"]


def descriptors(s):
    """The argument structs over this state's buffers; a program keeps them as it keeps the buffers."""
    M, c, op = package(), s["case"], s["case"]["op"]
    d = {"lib": M.lib()}
    kind = CTYPE[c["type"]]
    if "steps" in s:
        d["rope"] = M.Rope(s["steps"].data_ptr(), c["rot"], int(c["inter"]), s["mag"])
    if op == "rope":
        wide = c["heads"] * c["dim"]
        d["args"] = M.RopeArgs(x=s["x"].data_ptr(), out=s["out"].data_ptr(), pos=s["pos"].data_ptr(), x_row_stride=wide,
                               x_head_stride=c["dim"], out_row_stride=wide, out_head_stride=c["dim"], rows=c["rows"],
                               heads=c["heads"], head_dim=c["dim"], type=kind, inverse=int(c["inverse"]))
        return d
    if op == "score":
        d["args"] = M.LogprobArgs(logits=s["x"].data_ptr(), tokens=s["tok"].data_ptr(), logprob=s["lp"].data_ptr(),
                                  entropy=s["ent"].data_ptr(), top_ids=s["ids"].data_ptr(),
                                  top_logprobs=s["top"].data_ptr(), row_stride=c["vocab"], rows=c["rows"],
                                  vocab=c["vocab"], type=kind, top_k=c["top"], temperature=c["hot"])
        return d
    d["cache"] = M.KV8Cache(s["codes"].data_ptr(), s["scales"].data_ptr(), s["table"].data_ptr(), s["codes"].shape[0],
                            c["seqs"], s["table"].shape[1], c["kvh"], c["dim"], FORMAT[c["format"]])
    d["seqs"] = M.SeqBatch(s["start"].data_ptr(), s["slot"].data_ptr(), s["ctx"].data_ptr(), c["seqs"], s["rows"])
    wide = c["kvh"] * c["dim"]
    if op in ("append", "round"):
        q = dict(q=s["q"].data_ptr(), q_out=s["q_out"].data_ptr(), q_row_stride=c["qh"] * c["dim"],
                 q_head_stride=c["dim"], q_out_row_stride=c["qh"] * c["dim"], q_out_head_stride=c["dim"]) if c["qh"] else {}
        d["append"] = M.KV8AppendArgs(k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_row_stride=wide, k_head_stride=c["dim"],
                                      v_row_stride=wide, v_head_stride=c["dim"], q_heads=c["qh"], type=kind, **q)
    if op in ("read", "round"):
        d["read"] = M.KV8ReadArgs(k=s["k_out"].data_ptr(), v=s["v_out"].data_ptr(), k_row_stride=wide,
                                  k_head_stride=c["dim"], v_row_stride=wide, v_head_stride=c["dim"], type=kind)
    if op == "attend":
        wide = c["qh"] * c["dim"]
        need = d["lib"].mossgpu_attention_kv8_workspace_bytes(d["cache"], c["qh"], s["rows"])
        d["space"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        d["args"] = M.AttentionKV8Args(q=s["q"].data_ptr(), out=s["out"].data_ptr(),
                                       mask=s["mask"].data_ptr() if s["mask"] is not None else None,
                                       workspace=d["space"].data_ptr(), workspace_bytes=need, q_row_stride=wide,
                                       q_head_stride=c["dim"], out_row_stride=wide, out_head_stride=c["dim"],
                                       q_heads=c["qh"], type=kind,
                                       mask_words=s["mask"].shape[1] if s["mask"] is not None else 0,
                                       scale=c["dim"]**-0.5)
    return d


def called(d, status):
    if status != 0:
        raise RuntimeError(d["lib"].mossgpu_op_last_error().decode())


def run(s):
    c, op = s["case"], s["case"]["op"]
    if own:
        d = s.get("own") or s.setdefault("own", descriptors(s))
        stream = torch.cuda.current_stream().cuda_stream  # of this pass: a later one may run on another
        if op == "rope":
            called(d, d["lib"].mossgpu_rope_rotate(d["rope"], d["args"], stream))
            return s["out"]
        if op == "score":
            called(d, d["lib"].mossgpu_token_logprobs(d["args"], stream))
            return {"logprob": s["lp"], "entropy": s["ent"], "top_ids": s["ids"], "top_logprobs": s["top"]}
        if op == "attend":
            called(d, d["lib"].mossgpu_attention_kv8(d["cache"], d["seqs"], d["args"], stream))
            return s["out"]
        if op != "read":
            called(d, d["lib"].mossgpu_kv8_append(d["cache"], d["seqs"], d["rope"], d["append"], stream))
        if op != "append":
            called(d, d["lib"].mossgpu_kv8_read(d["cache"], d["seqs"], d["read"], stream))
            return {"k": s["k_out"], "v": s["v_out"]}
        return {"codes": s["codes"].view(torch.float8_e4m3fn), "scales": s["scales"], "q": s["q_out"]}
    if op == "rope":
        return p_rope(s["x"], s["pos"], s["freq"], s["mag"], c["inter"], c["inverse"]).to(s["x"].dtype)
    if op == "score":
        return p_score(s)
    if op == "attend":
        return p_attend(s)
    if op != "read":
        q = p_append(s)
    if op != "append":
        k, v = p_read(s)
        return {"k": k, "v": v}
    return {"codes": s["codes"].view(torch.float8_e4m3fn), "scales": s["scales"], "q": q}


# ---- the definitions in 64 bits --------------------------------------------------------------


def turn(x, pos, case, sign=1.0):
    """x [rows][heads][dim] in 64 bits, each pair as a complex number times m e^(i pos f)."""
    rot = case["rot"]
    f = torch.tensor(frequencies(rot, case["scaled"]), device=x.device)
    mag = 0.1 * math.log(8.0) + 1.0 if case["scaled"] else 1.0
    w = torch.polar(torch.full_like(pos.double()[:, None] * f, mag), sign * pos.double()[:, None] * f)[:, None]
    y = x.clone()
    first = slice(0, rot, 2) if case["inter"] else slice(0, rot // 2)
    second = slice(1, rot, 2) if case["inter"] else slice(rot // 2, rot)
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * w
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    c, op = case, case["op"]
    if op == "rope":
        return turn(s["x"].double(), s["pos"], c, -1.0 if c["inverse"] else 1.0)
    if op == "score":
        lp, ent, top = [], [], []
        for r0 in range(0, c["rows"], 256):
            y = s["x"][r0 : r0 + 256].double() / c["hot"]
            logp = y - torch.logsumexp(y, -1, keepdim=True)
            tok = s["tok"][r0 : r0 + 256].long()
            lp.append(torch.where(tok < 0, 0.0, logp[torch.arange(len(y), device=y.device), tok.clamp(min=0)]))
            p = torch.exp(logp)
            ent.append(-torch.where(p > 0, p * logp, 0.0).sum(-1))
            top.append(torch.sort(logp, dim=-1, descending=True)[0][:, : c["top"]])
        return {"logprob": torch.cat(lp), "entropy": torch.cat(ent), "top_ids": None, "top_logprobs": torch.cat(top)}
    form, start, ctx, table = c["format"], s["start"].tolist(), s["ctx"].tolist(), s["table"].long()
    codes, scales = s["codes"], s["scales"].double()

    def held(b, half, lo, hi):
        """Positions lo..hi-1 of a sequence, [positions][kvh][dim]."""
        page = table[b, lo // PAGE : -(-hi // PAGE)]
        x = codes[page, half].view(torch.int8 if form == "int8" else torch.float8_e4m3fn).float().double()
        x = (x * scales[page, half][..., None]).permute(0, 2, 1, 3).reshape(-1, c["kvh"], c["dim"])
        return x[lo % PAGE : lo % PAGE + hi - lo]

    if op == "attend":
        group, out = c["qh"] // c["kvh"], []
        for b in range(c["seqs"]):
            n = start[b + 1] - start[b]
            q = s["q"][start[b] : start[b + 1]].double().view(n, c["kvh"], group, c["dim"])
            k, v = held(b, 0, 0, ctx[b] + n), held(b, 1, 0, ctx[b] + n)
            a = torch.einsum("ikgd,jkd->ikgj", q, k) / math.sqrt(c["dim"])
            ok = torch.ones(n, ctx[b] + n, dtype=torch.bool, device=a.device)
            if s["mask"] is None:
                ok[:, ctx[b] :] = torch.ones(n, n, dtype=torch.bool, device=a.device).tril()
            else:
                word = s["mask"][start[b] : start[b + 1]].long()
                bit = torch.arange(n, device=a.device)
                ok[:, ctx[b] :] = (word[:, bit // 32] >> (bit % 32)) & 1 > 0
            a = a.masked_fill(~ok[:, None, None, :], float("-inf"))
            out.append(torch.einsum("ikgj,jkd->ikgd", torch.softmax(a, -1), v).reshape(n, c["qh"], c["dim"]))
        return torch.cat(out)
    where = torch.cat([torch.arange(ctx[b], ctx[b] + start[b + 1] - start[b]) for b in range(c["seqs"])]).to(codes.device)
    if op == "read":
        return {name: torch.cat([held(b, half, ctx[b], ctx[b] + start[b + 1] - start[b]) for b in range(c["seqs"])])
                for half, name in ((0, "k"), (1, "v"))}
    turned = turn(s["k"].double(), where, c), s["v"].double()
    scale = [x.abs().amax(-1) / CODE_MAX[form] for x in turned]
    if op == "round":
        rounded = [torch.round(x / t[..., None]) if form == "int8" else
                   (x / t[..., None]).float().clamp(-448, 448).to(torch.float8_e4m3fn).double() for x, t in zip(turned, scale)]
        return {name: x * t[..., None] for name, x, t in zip("kv", rounded, scale)}
    # the codes before their one rounding, as for every other output
    values = codes.view(torch.float8_e4m3fn).float().double()
    seq = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(start[1:]) - torch.tensor(start[:-1])).to(codes.device)
    page = table[seq, where // PAGE]
    for half in (0, 1):
        values[page, half, :, where % PAGE] = turned[half] / scale[half][..., None]
        scales[page, half, :, where % PAGE] = scale[half]
    return {"codes": values, "scales": scales, "q": turn(s["q"].double(), where, c)}
