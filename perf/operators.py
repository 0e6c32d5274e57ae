"""What is measured of the attention operators for voxel tokens, and their plain forms.

Four operators of the transformer between the sparse stages of the SLat generator, on rows of voxel
tokens (several objects of a batch follow one another as ragged sequences):

  rope    rotation of every head by the voxel position, several axes (s3dsp_rope)
  qk      RMS norm of q and k for each head and the rotation in the same pass (s3dsp_qk_norm_rope)
  select  the key blocks (64 rows) with the largest mean-by-mean score, for each block of 128 query
          rows and each head (s3dsp_block_select)
  attend  softmax attention over the listed key blocks, or over all (s3dsp_block_attention)

A case is a dict of numbers and texts; `lens` / `klens` are the sequences' rows of queries / keys
(klens "" = the same rows). Plain forms are elementary torch operations in 32 bits (angles, block means
and block scores in 64).
"""
import os
import sys

import numpy as np
import torch

own = False

Q_ROWS, K_ROWS = 128, 64
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one small object's tokens after its projection: the time is the call's
        dict(name="rope 37 rows", op="rope", dtype="bf16", out="bf16", n=37, heads=12, d=64, pad=0, far=0, half=0,
             inverse=0),
        # the row limit of one object, f32 path, pairs apart by half a head, positions over the whole domain
        dict(name="rope 42000 rows f32", op="rope", dtype="f32", out="f32", n=42000, heads=16, d=64, pad=0, far=1,
             half=1, inverse=1),
        # a small object out of a fused 768-channel projection (row stride 2304)
        dict(name="qk 300 rows of 2304", op="qk", dtype="bf16", out="bf16", n=300, heads=12, kv_heads=12, d=64,
             pad=1536, far=0, half=0, gamma="heads"),
        # an f32 projection made ready for the tensor cores
        dict(name="qk 7583 rows f32 to bf16", op="qk", dtype="f32", out="bf16", n=7583, heads=12, kv_heads=12, d=64,
             pad=0, far=0, half=0, gamma="heads"),
        # the row limit, wide heads, one weight for all heads
        dict(name="qk 42000 rows d128", op="qk", dtype="bf16", out="bf16", n=42000, heads=16, kv_heads=16, d=128,
             pad=0, far=0, half=1, gamma="shared"),
        # one object of coarse voxels
        dict(name="select 1900 rows", op="select", dtype="bf16", lens="1900", klens="", heads=16, kv_heads=16, d=64,
             top=8, local=1),
        # a ragged batch, one of its objects empty, one of a single row
        dict(name="select ragged batch", op="select", dtype="bf16", lens="15159,0,4211,1,8190,2777", klens="",
             heads=16, kv_heads=16, d=64, top=16, local=1),
        # one large volume
        dict(name="select 65500 rows", op="select", dtype="bf16", lens="65500", klens="", heads=16, kv_heads=16, d=64,
             top=32, local=0),
        # single queries over long key rows, heads in groups, wide heads: the serving form
        dict(name="attend 8 single rows", op="attend", dtype="bf16", lens="1,1,1,1,1,1,1,1",
             klens="6007,42000,1,128,15159,20000,333,9000", heads=16, kv_heads=4, d=128, top=0, pad=0),
        # dense attention of the coarse rows of one object, f16, out of rows of a fused projection
        dict(name="attend dense 7583 f16", op="attend", dtype="f16", lens="7583", klens="", heads=12, kv_heads=12,
             d=64, top=0, pad=1536),
        # sparse attention of a ragged batch
        dict(name="attend sparse ragged batch", op="attend", dtype="bf16", lens="15159,0,4211,1,8190,2777", klens="",
             heads=16, kv_heads=16, d=64, top=16, pad=0),
        # the row limit, sparse
        dict(name="attend sparse 42000", op="attend", dtype="bf16", lens="42000", klens="", heads=16, kv_heads=16,
             d=64, top=32, pad=0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rope", "qk", "select", "attend", "attend"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    d = c["d"] = rng.choice([64, 64, 128])
    heads = c["heads"] = rng.choice([4, 6, 8, 12, 16])
    if op in ("rope", "qk"):
        c.update(n=_spread(rng, 1, 42000), pad=8 * rng.choice([0, 0, 1, 5, 32]), far=rng.randint(0, 1),
                 half=rng.randint(0, 1))
        c["out"] = c["dtype"] if op == "rope" else rng.choice([c["dtype"], "bf16"])
        if op == "rope":
            c["inverse"] = rng.randint(0, 1)
        else:
            c.update(kv_heads=heads if rng.random() < 0.6 else heads // 2, gamma=rng.choice(["heads", "shared", "none"]))
        return c
    c["kv_heads"] = heads if rng.random() < 0.6 else heads // 2
    if c["dtype"] == "f32" and op == "attend":
        c["dtype"] = "bf16"
    if op == "select":
        total, parts = _spread(rng, 1000, 32000), rng.choice([1, 1, 2, 5])
    else:
        c.update(top=rng.choice([0, 0, 4, rng.randint(1, 24)]), pad=8 * rng.choice([0, 0, 3, 16]))
        total, parts = _spread(rng, 100, 6000 if c["top"] == 0 else 20000), rng.choice([1, 1, 3, 6])
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    c["lens"], c["klens"] = ",".join(map(str, lens)), ""
    if rng.random() < 0.4:  # keys of their own: an image's tokens, a longer cache
        c["klens"] = ",".join(str(_spread(rng, 300 if op == "select" else 1, 6000)) for _ in lens)
    if op == "select":  # fewer than the blocks there are, so that there is something to select
        most = max(-(-m // K_ROWS) for n, m in zip(lens, _lens(c["klens"] or c["lens"])) if n)
        c["local"] = rng.randint(0, 1) if most >= 8 and not c["klens"] else 0
        c["top"] = rng.randint(4 if c["local"] else 1, max(1, min(32, most // 2)))
    return c


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, n, width, pad, dtype, scale=1.0):
    """[n, width] rows inside rows that are `pad` wider."""
    x = torch.randn((n, width + pad), generator=g, device="cuda") * scale
    return x.to(dtype)[:, :width]


def _tokens(g, lens, width, pad, dtype):
    """Rows of voxel tokens: a part shared by near rows (what block means see) beside each row's own."""
    n = sum(lens)
    x = torch.randn((n, width + pad), generator=g, device="cuda")
    near = torch.randn(((n + 95) // 96 + 1, width + pad), generator=g, device="cuda")
    x += 0.7 * near[torch.arange(n, device="cuda") // 96]
    return x.to(dtype)[:, :width]


def _lens(text):
    return [int(t) for t in text.split(",")]


def _pairs(d):
    """Pairs of each of the three axes: a third of the head's pairs, rounded down; the rest stay."""
    return [d // 6] * 3


def _blocks(lens, rows):
    """Block tables of ragged sequences: rows of each block [nb, rows] (clamped), their mask, each
    block's sequence, the sequences' first block, and each row's place in the padded blocks."""
    first, start, seq, first_block, slot = [], 0, [], [0], []
    for s, m in enumerate(lens):
        nb = -(-m // rows)
        first += [(start + b * rows, min(rows, m - b * rows)) for b in range(nb)]
        seq += [s] * nb
        slot += [(first_block[-1] + np.arange(m) // rows) * rows + np.arange(m) % rows]
        first_block.append(first_block[-1] + nb)
        start += m
    at = np.array(first, np.int64).reshape(-1, 2)
    idx = at[:, :1] + np.arange(rows)[None]
    mask = np.arange(rows)[None] < at[:, 1:]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return dict(idx=dev(np.where(mask, idx, 0)), mask=dev(mask), count=dev(at[:, 1]), seq=dev(np.array(seq, np.int64)),
                first=dev(np.array(first_block, np.int64)), slot=dev(np.concatenate(slot).astype(np.int64)),
                row_seq=dev(np.repeat(np.arange(len(lens)), lens)))


def _lists(g, bq, bk, heads, top):
    """Ascending lists of up to `top` different blocks for each query block and head, -1 behind: the
    blocks around the query's own place and random others, as a selection gives them."""
    nkb = (bk["first"][1:] - bk["first"][:-1])[bq["seq"]]
    most = int(nkb.max()) if len(nkb) else 0
    at = (torch.arange(len(nkb), device="cuda") - bq["first"][bq["seq"]]) * (Q_ROWS // K_ROWS)
    block = torch.arange(max(most, top), device="cuda")
    key = torch.rand((len(nkb), heads, len(block)), generator=g, device="cuda")
    key = torch.where((block[None] - at[:, None]).abs().lt(3)[:, None], 2.0, key)
    key = torch.where((block[None] < nkb[:, None])[:, None], key, -1.0)
    best, pick = torch.topk(key, top, dim=-1)
    pick = torch.where(best >= 0, pick, 1 << 30).sort(dim=-1).values
    return torch.where(pick < (1 << 30), pick, -1).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case)
    d, heads, op = case["d"], case["heads"], case["op"]
    dt = DT[case["dtype"]]
    if op in ("rope", "qk"):
        n = case["n"]
        span = 30000 if case["far"] else 64
        pos = torch.randint(-span if case["far"] else 0, span, (n, 4), generator=g, device="cuda", dtype=torch.int32)
        s["pos"] = pos[:, 1:]  # rows (batch, x, y, z)
        pairs = s["pairs"] = _pairs(d)
        rest = d // 2 - sum(pairs)
        s["axis"] = torch.tensor([a for a, p in enumerate(pairs) for _ in range(p)] + [0] * rest, device="cuda")
        s["freq"] = torch.tensor([10000.0 ** (-i / p) for p in pairs for i in range(p)] + [0.0] * rest,
                                 dtype=torch.float64, device="cuda")
        s["q"] = _rows(g, n, heads * d, case["pad"], dt, 1.7)
        if op == "qk":
            kv = case["kv_heads"]
            s["k"] = _rows(g, n, kv * d, case["pad"], dt, 0.6)
            gamma = lambda h: torch.randn((h, d), generator=g, device="cuda") * 0.2 + 1.0  # noqa: E731
            if case["gamma"] == "heads":
                s["gq"], s["gk"] = gamma(heads), gamma(kv)
            elif case["gamma"] == "shared":
                s["gq"], s["gk"] = gamma(1)[0], gamma(1)[0]
            else:
                s["gq"] = s["gk"] = None
    else:
        lens, klens = _lens(case["lens"]), _lens(case["klens"] or case["lens"])
        kv, pad = case["kv_heads"], case.get("pad", 0)
        s["bq"], s["bk"] = _blocks(lens, Q_ROWS), _blocks(klens, K_ROWS)
        s["q"] = _tokens(g, lens, heads * d, pad, dt)
        s["k"] = _tokens(g, klens, kv * d, pad, dt)
        s["kv_of"] = torch.arange(heads, device="cuda") // (heads // kv)
        if op == "attend":
            s["v"] = _rows(g, sum(klens), kv * d, pad, dt)
            s["sel"] = _lists(g, s["bq"], s["bk"], heads, case["top"]) if case["top"] else None
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a user's program of the framework keeps between calls: its context, the plan of the batch
    and the output buffers."""
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sam3d.cpp_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import s3dsp
    c = s["case"]
    ctx = s["ctx"] = s3dsp.Context(0)
    new = lambda x, dt: torch.empty((x.shape[0], x.shape[1]), dtype=dt, device="cuda")  # noqa: E731
    if c["op"] in ("rope", "qk"):
        s["q_out"] = new(s["q"], DT[c["out"]])
        if c["op"] == "qk":
            s["k_out"] = new(s["k"], DT[c["out"]])
        return
    s["plan"] = ctx.attn_plan(_offsets(c["lens"]), _offsets(c["klens"]) if c["klens"] else None)
    if c["op"] == "select":
        s["out"] = torch.empty((s["bq"]["idx"].shape[0], c["heads"], c["top"]), dtype=torch.int32, device="cuda")
    else:
        s["out"] = new(s["q"], DT[c["dtype"]])


def _offsets(text):
    return np.concatenate([[0], np.cumsum(_lens(text))])


# --------------------------------------------------------------------------------------------------
# the operators: plain forms, or the framework's calls
# --------------------------------------------------------------------------------------------------
def run(s):
    return {"rope": _rope, "qk": _qk, "select": _select, "attend": _attend}[s["case"]["op"]](s)


def _turn(x, s):
    """x [n, h, d] f32, every pair turned by its angle."""
    c = s["case"]
    angle = s["pos"][:, s["axis"]].double() * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if c.get("inverse"):
        sin = -sin
    if c["half"]:
        a, b = x[..., : c["d"] // 2], x[..., c["d"] // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)


def _rope(s):
    c = s["case"]
    if own:
        s["ctx"].rope(s["q"], s["pos"], c["heads"], s["q_out"], s["pairs"], half=bool(c["half"]),
                      inverse=bool(c["inverse"]))
        return s["q_out"]
    x = s["q"].float().unflatten(1, (c["heads"], c["d"]))
    return _turn(x, s).flatten(1).to(DT[c["out"]])


def _qk(s):
    c = s["case"]
    if own:
        s["ctx"].qk_norm_rope(s["q"], c["heads"], s["gq"], s["q_out"], s["k"], c["kv_heads"], s["gk"], s["k_out"],
                              eps=1e-6, positions=s["pos"], axis_pairs=s["pairs"], half=bool(c["half"]))
        return [s["q_out"], s["k_out"]]
    return [_normed(s["q"], s["gq"], c["heads"], s), _normed(s["k"], s["gk"], c["kv_heads"], s)]


def _normed(x, gamma, heads, s):
    c = s["case"]
    x = x.float().unflatten(1, (heads, c["d"]))
    x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6)
    if gamma is not None:
        x = x * gamma
    return _turn(x, s).flatten(1).to(DT[c["out"]])


def _means(x, b, heads, d):
    """Block means [nb, heads, d] in 64 bits."""
    rows = x.unflatten(1, (heads, d))[b["idx"]].double() * b["mask"][..., None, None]
    return rows.sum(dim=1) / b["count"][:, None, None]


def _select(s):
    c = s["case"]
    if own:
        s["ctx"].block_select(s["plan"], s["q"], s["k"], c["heads"], c["kv_heads"], s["out"],
                              keep_local=bool(c["local"]))
        return s["out"]
    bq, bk, top = s["bq"], s["bk"], c["top"]
    qm = _means(s["q"], bq, c["heads"], c["d"])
    km = _means(s["k"], bk, c["kv_heads"], c["d"])[:, s["kv_of"]]
    score = torch.einsum("bhd,chd->bhc", qm, km)
    block = torch.arange(score.shape[2], device="cuda")
    first = bk["first"][bq["seq"]]
    mine = (block >= first[:, None]) & (block < bk["first"][1:][bq["seq"]][:, None])
    if c["local"]:
        at = first + (torch.arange(len(first), device="cuda") - bq["first"][bq["seq"]]) * (Q_ROWS // K_ROWS)
        near = (block >= at[:, None]) & (block < at[:, None] + Q_ROWS // K_ROWS)
        score = torch.where((near & mine)[:, None], torch.inf, score)
    score = torch.where(mine[:, None], score, -torch.inf)
    score = torch.nn.functional.pad(score, (0, max(0, top - score.shape[2])), value=-torch.inf)
    best, pick = torch.sort(score, dim=-1, descending=True, stable=True)
    pick = torch.where(best[..., :top] > -torch.inf, pick[..., :top] - first[:, None, None], 1 << 30).sort(dim=-1).values
    return torch.where(pick < (1 << 30), pick, -1).to(torch.int32)


def _attend(s):
    c = s["case"]
    if own:
        s["ctx"].block_attention(s["plan"], s["q"], s["k"], s["v"], c["heads"], c["kv_heads"], s["out"], sel=s["sel"])
        return s["out"]
    h, kv, d = c["heads"], c["kv_heads"], c["d"]
    bq, bk = s["bq"], s["bk"]
    q = s["q"].float().unflatten(1, (h, d)) * d ** -0.5
    k, v = (s[x].float().unflatten(1, (kv, d))[:, s["kv_of"]] for x in ("k", "v"))
    if s["sel"] is None:
        score = torch.einsum("qhd,khd->hqk", q, k)
        score = score.masked_fill(bq["row_seq"][:, None] != bk["row_seq"], -torch.inf)
        p, total = _weights(score)
        out = torch.einsum("hqk,khd->qhd", p, v) / total.permute(1, 0, 2)
        return torch.where(total.permute(1, 0, 2) > 0, out, 0).flatten(1).to(DT[c["dtype"]])
    sel, head = s["sel"].long(), torch.arange(h, device="cuda")[:, None]
    block = (sel + bk["first"][bq["seq"]][:, None, None]).clamp(min=0, max=max(0, bk["idx"].shape[0] - 1))
    rows = bk["idx"][block]
    seen = (bk["mask"][block] & (sel >= 0)[..., None]).flatten(2)
    kg, vg = (x[rows.flatten(2), head[None]] for x in (k, v))
    score = torch.einsum("bqhd,bhkd->bhqk", q[bq["idx"]], kg)
    score = score.masked_fill(~seen[:, :, None], -torch.inf)
    p, total = _weights(score)
    out = torch.einsum("bhqk,bhkd->bhqd", p, vg) / total
    out = torch.where(total > 0, out, 0).permute(0, 2, 1, 3).flatten(0, 1).flatten(1)
    return out[bq["slot"]].to(DT[c["dtype"]])


def _weights(score):
    """exp(score - row maximum) and its sum; a row with nothing: zeros."""
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -torch.inf, top, 0))
    return p, p.sum(dim=-1, keepdim=True)


# --------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] in ("rope", "qk"):
        w = c["n"] * c["d"] * (c["heads"] + c.get("kv_heads", 0))
        return {"bytes": w * (SIZE[c["dtype"]] + SIZE[c["out"]]) + 12 * c["n"],
                "flops": w * (3 if c["op"] == "rope" else 7)}
    lens, klens = _lens(c["lens"]), _lens(c["klens"] or c["lens"])
    nqb, nkb = [-(-m // Q_ROWS) for m in lens], [-(-m // K_ROWS) for m in klens]
    h, kv, d, e = c["heads"], c["kv_heads"], c["d"], SIZE[c["dtype"]]
    if c["op"] == "select":
        return {"bytes": d * e * (sum(lens) * h + sum(klens) * kv) + 4 * sum(nqb) * h * c["top"],
                "flops": d * (sum(lens) * h + sum(klens) * kv) + 2 * d * h * sum(a * b for a, b in zip(nqb, nkb))}
    listed_rows = [min(m, K_ROWS * c["top"]) if c["top"] else m for m in klens]
    return {"bytes": d * e * (2 * sum(lens) * h + 2 * sum(klens) * kv) + 4 * sum(nqb) * h * c["top"],
            "flops": 4 * d * h * sum(a * b for a, b in zip(lens, listed_rows))}


# --------------------------------------------------------------------------------------------------
# the definitions in 64 bits, row by row and head by head
# --------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    c = case
    d, heads = c["d"], c["heads"]
    if c["op"] in ("rope", "qk"):
        rates = [10000.0 ** (-i / p) for p in s["pairs"] for i in range(p)]
        axes = [a for a, p in enumerate(s["pairs"]) for _ in range(p)]
        outs = []
        for name, gamma, hs in [("q", "gq", heads)] + ([("k", "gk", c["kv_heads"])] if c["op"] == "qk" else []):
            x = s[name].double().reshape(c["n"], hs, d)
            if c["op"] == "qk":
                x = x / ((x ** 2).sum(dim=2, keepdim=True) / d + 1e-6) ** 0.5
                x = x if s[gamma] is None else x * s[gamma].double()
            y = x.clone()
            for j, (rate, a) in enumerate(zip(rates, axes)):
                turn = torch.polar(torch.ones(c["n"], dtype=torch.float64, device="cuda"), s["pos"][:, a].double() * rate)
                turn = turn.conj() if c.get("inverse") else turn
                i0, i1 = (j, j + d // 2) if c["half"] else (2 * j, 2 * j + 1)
                z = torch.complex(x[:, :, i0], x[:, :, i1]) * turn[:, None]
                y[:, :, i0], y[:, :, i1] = z.real, z.imag
            outs.append(y.reshape(c["n"], hs * d))
        return outs if c["op"] == "qk" else outs[0]
    if c["op"] == "select":
        return None  # whole numbers: they have to be the plain form's
    lens, klens = _lens(c["lens"]), _lens(c["klens"] or c["lens"])
    group = heads // c["kv_heads"]
    out = torch.zeros((sum(lens), heads * d), dtype=torch.float64, device="cuda")
    q0 = k0 = b0 = 0
    for m, mk in zip(lens, klens):
        nb, nk = -(-m // Q_ROWS), -(-mk // K_ROWS)
        for h in range(heads if m and mk else 0):
            cols, kcols = slice(h * d, h * d + d), slice(h // group * d, h // group * d + d)
            k, v = s["k"][k0:k0 + mk, kcols].double(), s["v"][k0:k0 + mk, kcols].double()
            for r0 in range(0, m, 4096):
                r1 = min(m, r0 + 4096)
                score = s["q"][q0 + r0:q0 + r1, cols].double() @ k.T / d ** 0.5
                if s["sel"] is not None:
                    sel = s["sel"][b0:b0 + nb, h].long()
                    table = torch.zeros((nb, nk + 1), dtype=torch.bool, device="cuda")
                    table.scatter_(1, torch.where(sel < 0, nk, sel), True)
                    rows = torch.arange(r0, r1, device="cuda") // Q_ROWS
                    seen = table[rows][:, torch.arange(mk, device="cuda") // K_ROWS]
                    score[~seen] = -torch.inf
                out[q0 + r0:q0 + r1, cols] = torch.softmax(score, dim=1).nan_to_num(0.0) @ v
        q0, k0, b0 = q0 + m, k0 + mk, b0 + nb
    return out
