"""The attention operators over voxel tokens against their definitions in 64
bits: s3dsp_rope, s3dsp_qk_norm_rope, s3dsp_block_select, s3dsp_block_attention
alone, at the sizes and masks where they can go wrong, and run together.

Tolerances count roundings (u = eps / 2 of the output type, 2^-24 an f32 one):

rope      an angle's remainder is rounded once (at most half a turn: pi 2^-25), sincospif is within 2 ulp
          (2^-23), two products and a sum follow: below (|a| + |b|) 6 * 2^-24 before the output's rounding.
          The f64 angle itself: frequency / 2 pi carries a pow (1 ulp: 2^-52), the constant 2 pi and a division
          (2^-53 each), the product with the position 2^-53; the definition here a pow and a product (2^-53 each):
          together at most |pos| 7 * 2^-53 of the pair's size (1.7e-6 at 2^31, nothing at voxel positions).
qk        the mean square adds at most 8 + 5 additions, a division, a sum, a square root, a division and
          two products: below 20 roundings more on each value.
attention P is rounded to the type (u of sum p |v| / sum p); a score errs by the f32 accumulation of d products,
          which may truncate (d 2^-23 sum |q k| scale), its exponential by that and a few 2^-22, in the
          numerator and in the sum; then the output's rounding.
"""
import numpy as np
import pytest
import torch

import s3dsp
import slat
import workloads
from gates import gate

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return s3dsp.Context(0)


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def strided(shape, seed, dtype, pad=0, offset=0, scale=1.0):
    """Rows inside a wider buffer, `offset` elements in."""
    n, w = shape
    return randn((n, w + pad + offset), seed, dtype, scale)[:, offset:offset + w]


def within(got, want, tol, u):
    """|got - want| <= tol + u |want|, elementwise (f16 adds its smallest step)."""
    got = got.double()
    tiny = 2.0 ** -24 if u == 2.0 ** -11 else 2.0 ** -133
    off = (got - want).abs() - (tol + u * (want.abs() + tol) + tiny)
    assert torch.isfinite(got).all()
    worst = int(off.argmax())
    assert off.max() <= 0, f"off by {float((got - want).abs().flatten()[worst]):.3e} at {worst}, want {float(want.flatten()[worst]):.6e}"


def unit(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------------------------------
# rope, qk_norm_rope
# ---------------------------------------------------------------------------------------------------
def turned(x, pos, heads, pairs, theta, half, inverse):
    """x [n, heads * d] f64 turned, and |a| + |b| of each value's pair."""
    n, d = x.shape[0], x.shape[1] // heads
    x = x.reshape(n, heads, d)
    y, size = x.clone(), x.abs()
    j = 0
    for a, p in enumerate(pairs):
        for i in range(p):
            ang = pos[:, a].double() * theta ** (-i / p)
            c, s = ang.cos()[:, None], ang.sin()[:, None] * (-1 if inverse else 1)
            i0, i1 = (j, j + d // 2) if half else (2 * j, 2 * j + 1)
            y[:, :, i0], y[:, :, i1] = x[:, :, i0] * c - x[:, :, i1] * s, x[:, :, i0] * s + x[:, :, i1] * c
            size[:, :, i0] = size[:, :, i1] = x[:, :, i0].abs() + x[:, :, i1].abs()
            j += 1
    return y.reshape(n, heads * d), size.reshape(n, heads * d)


ROPE = [
    # n, heads, d, pairs, in, out, pad, offset, span
    (1, 1, 8, [1, 1, 1], "f32", "f32", 0, 0, 64),
    (5, 3, 64, [10, 10, 10], "bf16", "bf16", 0, 0, 64),
    (1000, 12, 64, [10, 10, 10], "bf16", "bf16", 0, 0, 32768),
    (777, 16, 128, [21, 21, 21], "f16", "f16", 8, 0, 64),
    (300, 4, 96, [48], "f32", "bf16", 0, 0, 2 ** 31 - 1),
    (300, 4, 80, [0, 40], "bf16", "f32", 3, 1, 2 ** 31 - 1),
    (131, 2, 256, [32, 32, 32, 32], "f32", "f32", 1, 3, 1000),
    (64, 5, 24, [2, 3, 4], "f16", "bf16", 5, 0, 100),
    (9, 70, 64, [16, 16], "bf16", "f16", 0, 8, 100),
    (40, 2, 64, [], "bf16", "bf16", 0, 0, 100),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n,heads,d,pairs,di,do,pad,offset,span", ROPE)
def test_rope(ctx, n, heads, d, pairs, di, do, pad, offset, span, half, inverse):
    x = strided((n, heads * d), 1, DT[di], pad, offset, 1.7)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    pos = torch.randint(-span, span, (n, 5), generator=g, device="cuda", dtype=torch.int32)[:, 1:]
    keep = torch.full((n, heads * d + pad), 7.0, dtype=DT[do], device="cuda")
    out = keep[:, :heads * d]
    ctx.rope(x, pos, heads, out, pairs, theta=100.0, half=half, inverse=inverse)
    want, size = turned(x.double(), pos, heads, pairs, 100.0, half, inverse)
    within(out, want, size * (6 * F32 + span * 7 * 2.0 ** -53), unit(DT[do]))
    assert (keep[:, heads * d:] == 7.0).all()


def test_rope_in_place_and_back(ctx):
    """In place, then by the inverse: the rows come back; and the inverse is the transpose (what a gradient takes)."""
    n, heads, d, pairs = 500, 4, 64, [10, 10, 10]
    x = randn((n, heads * d), 3)
    pos = torch.randint(0, 64, (n, 3), device="cuda", dtype=torch.int32)
    y = x.clone()
    ctx.rope(y, pos, heads, y, pairs)
    back = torch.empty_like(y)
    ctx.rope(y, pos, heads, back, pairs, inverse=True)
    size = turned(x.double(), pos, heads, pairs, 1e4, False, False)[1]
    assert ((back - x).double().abs() <= 4 * 6 * F32 * size).all()
    w = randn((n, heads * d), 4)
    wt = torch.empty_like(w)
    ctx.rope(w, pos, heads, wt, pairs, inverse=True)
    a, b = (w.double() * y.double()).sum(), (wt.double() * x.double()).sum()  # <w, R x> = <R^T w, x>
    assert abs(a - b) <= 2 * 6 * F32 * float((w.abs() * 2 * size).sum())
    # and against differences along a direction: R is linear
    e = randn((n, heads * d), 5)
    y2 = torch.empty_like(y)
    ctx.rope(x + e, pos, heads, y2, pairs)
    diff = (w.double() * (y2.double() - y.double())).sum()
    assert abs(diff - (wt.double() * ((x + e).double() - x.double())).sum()) <= 6 * 6 * F32 * float((w.abs() * 3 * size).sum()) + \
        6 * 6 * F32 * float((w.abs() * e.abs()).sum() * 3)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("gamma", ["heads", "shared", "none"])
@pytest.mark.parametrize("n,heads,kv,d,pairs,di,do,pad,offset", [
    (1, 2, 1, 64, [10, 10, 10], "bf16", "bf16", 0, 0),
    (2500, 12, 12, 64, [10, 10, 10], "bf16", "bf16", 1536, 0),
    (311, 16, 4, 128, [21, 21, 21], "f32", "bf16", 0, 0),
    (100, 3, 0, 40, [20], "f16", "f32", 1, 1),
    (77, 6, 2, 256, [], "bf16", "f16", 0, 0),
])
def test_qk_norm_rope(ctx, n, heads, kv, d, pairs, di, do, pad, offset, gamma, half):
    q = strided((n, heads * d), 1, DT[di], pad, offset, 2.0)
    k = strided((n, kv * d), 2, DT[di], pad, offset, 0.01) if kv else None
    pos = torch.randint(0, 64, (n, 4), device="cuda", dtype=torch.int32)
    shape = {"heads": lambda h: (h, d), "shared": lambda h: (d,)}.get(gamma)
    gq = randn(shape(heads), 5, scale=0.3) + 1.0 if shape else None
    gk = randn(shape(kv), 6, scale=0.3) + 1.0 if shape and kv else None
    qo = torch.empty((n, heads * d), dtype=DT[do], device="cuda")
    ko = torch.empty((n, kv * d), dtype=DT[do], device="cuda") if kv else None
    ctx.qk_norm_rope(q, heads, gq, qo, k, kv, gk, ko, eps=1e-6, positions=pos[:, 1:], axis_pairs=pairs, half=half)
    for x, g, h, out in [(q, gq, heads, qo)] + ([(k, gk, kv, ko)] if kv else []):
        x = x.double().reshape(n, h, d)
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        x = (x if g is None else x * g.double()).reshape(n, h * d)
        want, size = turned(x, pos[:, 1:], h, pairs, 1e4, half, False)
        within(out, want, size * (6 + 20) * F32, unit(DT[do]))


def test_qk_norm_of_zero_rows_and_in_place(ctx):
    x = torch.zeros((3, 128), dtype=torch.bfloat16, device="cuda")
    ctx.qk_norm_rope(x, 2, None, x)
    assert (x == 0).all()  # 0 / sqrt(eps)
    ctx.qk_norm_rope(x[:0], 2, None, x[:0])


def test_rows_beyond_32_bits(ctx):
    """Rows whose element offsets pass 2^32: each is where its stride says."""
    n, stride = 40000, 120000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    big = torch.empty((n, stride), dtype=torch.bfloat16, device="cuda")
    x = big[:, 64:192]
    x.copy_(randn((n, 128), 1, torch.bfloat16))
    src = x.clone()
    pos = torch.randint(0, 64, (n, 3), device="cuda", dtype=torch.int32)
    out, ref = torch.empty_like(src), torch.empty_like(src)
    ctx.rope(x, pos, 2, out, [10, 10, 10])
    ctx.rope(src, pos, 2, ref, [10, 10, 10])
    assert torch.equal(out, ref)
    plan = ctx.attn_plan([0, 30000, n])
    sel, sref = (torch.empty((plan.q_blocks, 2, 4), dtype=torch.int32, device="cuda") for _ in range(2))
    ctx.block_select(plan, x, x, 2, 2, sel)
    ctx.block_select(plan, src, src, 2, 2, sref)
    assert torch.equal(sel, sref)
    ctx.block_attention(plan, x, x, x, 2, 2, out, sel=sel)
    ctx.block_attention(plan, src, src, src, 2, 2, ref, sel=sel)
    assert torch.equal(out, ref)
    wide = big[:, 256:384]
    ctx.block_attention(plan, src, src, src, 2, 2, wide, sel=sel)
    assert torch.equal(wide, ref)
    ctx.check()


# ---------------------------------------------------------------------------------------------------
# block_select
# ---------------------------------------------------------------------------------------------------
def offsets(lens, start=0):
    return np.concatenate([[0], np.cumsum(lens)]) + start


def chosen(q, k, lens, klens, heads, kv, top, local):
    """The selection by its definition: f64 means and scores, numpy's stable sort."""
    q, k = q.double(), k.double()
    d = q.shape[1] // heads
    rows, q0, k0 = [], 0, 0
    for m, mk in zip(lens, klens):
        nb, nk = -(-m // 128), -(-mk // 64)
        qm = torch.stack([q[q0 + 128 * b:q0 + min(m, 128 * b + 128)].mean(0) for b in range(nb)]) if nb else q[:0]
        km = torch.stack([k[k0 + 64 * c:k0 + min(mk, 64 * c + 64)].mean(0) for c in range(nk)]) if nk else k[:0]
        qm = qm.reshape(nb, heads, d).permute(1, 0, 2)
        km = km.reshape(nk, kv, d).permute(1, 0, 2).repeat_interleave(heads // kv, 0)
        score = torch.where((s := qm @ km.transpose(1, 2)).isnan(), -torch.inf, s).cpu().numpy()
        for b in range(nb):
            if local:
                score[:, b, 2 * b:2 * b + 2] = np.inf
            order = np.argsort(-score[:, b], axis=1, kind="stable")[:, :top]
            pad = np.full((heads, top - order.shape[1]), -1)
            rows.append(np.concatenate([np.sort(order, axis=1), pad], axis=1))
        q0, k0 = q0 + m, k0 + mk
    return torch.from_numpy(np.array(rows, np.int32).reshape(-1, heads, top))


SELECT = [
    # lens, klens, heads, kv, d, dtype, top, local, pad, offset
    ([1], None, 1, 1, 64, "bf16", 1, False, 0, 0),
    ([1000], None, 4, 4, 64, "bf16", 5, True, 0, 0),
    ([1000], None, 4, 2, 128, "f32", 5, False, 3, 1),
    ([0, 700, 1, 0, 129, 64, 5000], None, 6, 3, 64, "f16", 9, True, 8, 0),
    ([300, 20], [5000, 64], 2, 1, 64, "bf16", 16, False, 0, 0),
    ([300, 20, 5], [0, 640, 65], 2, 2, 40, "bf16", 3, False, 1, 0),
    ([2600], None, 3, 3, 256, "bf16", 1024, False, 0, 0),
    ([9000], None, 2, 2, 64, "bf16", 64, True, 0, 0),
]


@pytest.mark.parametrize("lens,klens,heads,kv,d,dt,top,local,pad,offset", SELECT)
def test_block_select(ctx, lens, klens, heads, kv, d, dt, top, local, pad, offset):
    q = strided((sum(lens), heads * d), 1, DT[dt], pad, offset)
    k = strided((sum(klens or lens), kv * d), 2, DT[dt], pad, offset)
    plan = ctx.attn_plan(offsets(lens), offsets(klens) if klens else None)
    sel = torch.full((plan.q_blocks, heads, top), -7, dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, k, heads, kv, sel, keep_local=local)
    assert torch.equal(sel.cpu(), chosen(q, k, lens, klens or lens, heads, kv, top, local))


def test_block_select_ties_and_nan(ctx):
    """Equal scores (whole numbers, exact in any order, and signed zeros): the lowest index; NaN scores last."""
    n, top = 64 * 40, 7
    q = torch.ones((n, 64), device="cuda")
    k = torch.zeros((n, 64), device="cuda")
    level = torch.tensor([3, 1, 2, 2, 0, 3, 2, 2, 2, 1] * 4, dtype=torch.float32)
    k[:, 0] = level.repeat_interleave(64).cuda()
    plan = ctx.attn_plan([0, n])
    sel = torch.empty((plan.q_blocks, 1, top), dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, k, 1, 1, sel)
    want = np.sort(np.argsort(-level.numpy(), kind="stable")[:top])
    assert (sel.cpu().numpy() == want).all(), sel[0]
    k.zero_()
    k[64 * 3:64 * 5] = -0.0
    ctx.block_select(plan, q, k, 1, 1, sel)
    assert (sel.cpu().numpy() == np.arange(top)).all()
    k[:64 * 38] = float("nan")
    ctx.block_select(plan, q, k, 1, 1, sel)
    assert (sel.cpu().numpy() == np.array([0, 1, 2, 3, 4, 38, 39])).all()
    k.fill_(-float("inf"))
    ctx.block_select(plan, q, k, 1, 1, sel)
    assert (sel.cpu().numpy() == np.arange(top)).all()


@pytest.mark.parametrize("copies", [3, 40])
@pytest.mark.parametrize("n", [64 * 50, 64 * 900, 64 * 1500])
def test_block_select_equal_blocks(ctx, n, copies):
    """Copies of one key block anywhere have one score, bit by bit: the first of them are taken."""
    q, k = randn((600, 128), 1, torch.bfloat16), randn((n, 128), 2, torch.bfloat16)
    g = np.random.default_rng(n + copies)
    at = np.sort(g.permutation(n // 64)[:copies])
    for c in at[1:]:
        k[64 * c:64 * c + 64] = k[64 * at[0]:64 * at[0] + 64]
    plan = ctx.attn_plan([0, 600], [0, n])
    for top in (1, 9, copies, 45):
        sel = torch.empty((plan.q_blocks, 2, top), dtype=torch.int32, device="cuda")
        ctx.block_select(plan, q, k, 2, 2, sel)
        for row in sel.reshape(-1, top).cpu().numpy():
            taken = np.isin(at, row)
            assert taken[:taken.sum()].all(), (at, row)
        assert (sel[..., 1:] > sel[..., :-1]).all()


@pytest.mark.parametrize("n", [64 * 20, 64 * 50, 64 * 700, 64 * 1500])
@pytest.mark.parametrize("q0,k0,q1,k1", [
    (1.0, 2.0**20, 1.0, 2.0**-10),      # apart by less than f32 keeps
    (1.0, -2.0**20, 2.0**-20, 2.0**10),
    (2.0**100, 2.0**100, 2.0**100, 2.0**80),     # beyond f32's range
    (2.0**100, -2.0**100, 2.0**100, 2.0**100),   # beyond it in the middle of a sum
    (2.0**-140, 2.0**100, 2.0**-149, 2.0**60),   # subnormal means
    (2.0**-70, 2.0**-70, 2.0**-70, 2.0**-79),    # subnormal products
])
def test_block_select_close_and_extreme_scores(ctx, n, q0, k0, q1, k1):
    """Scores q0 k0 + q1 k1 r for a permutation r of the blocks: exact in f64, equal, infinite or 0 in f32."""
    blocks = n // 64
    q, k = torch.zeros((200, 64), device="cuda"), torch.zeros((n, 64), device="cuda")
    r = torch.from_numpy(np.random.default_rng(n).permutation(blocks).astype(np.float32))
    q[:, 3], q[:, 40], k[:, 3] = q0, q1, k0
    k[:, 40] = (r * k1).repeat_interleave(64).cuda()
    plan = ctx.attn_plan([0, 200], [0, n])
    for top in (1, 9, 33):
        sel = torch.empty((plan.q_blocks, 1, top), dtype=torch.int32, device="cuda")
        ctx.block_select(plan, q, k, 1, 1, sel)
        assert torch.equal(sel.cpu(), chosen(q, k, [200], [n], 1, 1, top, False))


@pytest.mark.parametrize("n,inf", [(64 * 30, False), (64 * 30, True), (64 * 1100, True)])
@pytest.mark.parametrize("top", [1, 2, 3, 20])
def test_block_select_keep_local_short_lists(ctx, n, inf, top):
    """The own blocks come first, the lower one in a list of one; with infinite means beside them too."""
    q, k = randn((n, 64), 5, torch.bfloat16), randn((n, 64), 6, torch.bfloat16)
    if inf:
        k[64 * 7:64 * 7 + 10, 5] = float("inf")
        k[64 * 9:64 * 9 + 10, 5] = -float("inf")
        k[64 * 11:64 * 11 + 10, 5] = float("nan")
    plan = ctx.attn_plan([0, n])
    sel = torch.empty((plan.q_blocks, 1, top), dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, k, 1, 1, sel, keep_local=True)
    score = q.double().reshape(-1, 128, 64).mean(1) @ k.double().reshape(-1, 64, 64).mean(1).T
    score = torch.where(score.isnan(), -torch.inf, score).cpu().numpy()
    for b in range(n // 128):
        c = np.arange(n // 64)
        own = c // 2 == b
        order = np.lexsort((c, np.where(own, 0, -score[b]), ~own))  # own first, then by score, then by index
        assert (np.sort(order[:top]) == sel[b, 0].cpu().numpy()).all()


@pytest.mark.parametrize("top", [1, 31, 33, 64, 129, 500])
@pytest.mark.parametrize("n", [64 * 640, 64 * 1100])
def test_block_select_list_lengths(ctx, n, top):
    q, k = randn((300, 128), 3, torch.bfloat16), randn((n, 128), 4, torch.bfloat16)
    plan = ctx.attn_plan([0, 300], [0, n])
    sel = torch.empty((plan.q_blocks, 2, top), dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, k, 2, 2, sel)
    assert torch.equal(sel.cpu(), chosen(q, k, [300], [n], 2, 2, top, False))


@pytest.mark.parametrize("n", [120000, 300000])
def test_block_select_long_sequence(ctx, n):
    """More key blocks than sixteen score rows leave room for (groups of fewer query blocks)."""
    q, k = randn((200, 64), 1, torch.bfloat16), randn((n, 64), 2, torch.bfloat16)
    plan = ctx.attn_plan([0, 200], [0, n])
    sel = torch.empty((plan.q_blocks, 1, 50), dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, k, 1, 1, sel)
    assert torch.equal(sel.cpu(), chosen(q, k, [200], [n], 1, 1, 50, False))


def test_block_select_refuses_too_long_a_sequence(ctx):
    q = torch.zeros((1, 64), device="cuda")
    k = torch.zeros((1, 64), device="cuda").expand(1 << 21, 64)  # never read
    plan = ctx.attn_plan([0, 1], [0, 1 << 21])
    with pytest.raises(s3dsp.S3dError, match="key blocks"):
        s3dsp._call(s3dsp.load().s3dsp_block_select, ctx.handle, plan.handle, q.data_ptr(), 64, 1, k.data_ptr(), 64, 1,
                    s3dsp.F32, 64, 4, 0, q.data_ptr())


# ---------------------------------------------------------------------------------------------------
# block_attention
# ---------------------------------------------------------------------------------------------------
def attention(q, k, v, lens, klens, heads, kv, scale, sel=None):
    """The definition in f64, block by block, and the tolerance's two sums: out, sum p |v| / sum p, max sum |q k| scale."""
    d = q.shape[1] // heads
    out = torch.zeros((sum(lens), heads, d), dtype=torch.float64, device="cuda")
    mass, size = torch.zeros_like(out), torch.zeros((sum(lens), heads, 1), dtype=torch.float64, device="cuda")
    q0 = k0 = b0 = 0
    for m, mk in zip(lens, klens):
        nb, nk = -(-m // 128), -(-mk // 64)
        kh = k[k0:k0 + mk].double().reshape(mk, kv, d).repeat_interleave(heads // kv, 1)
        vh = v[k0:k0 + mk].double().reshape(mk, kv, d).repeat_interleave(heads // kv, 1)
        for b in range(nb if mk else 0):
            r = slice(q0 + 128 * b, q0 + min(m, 128 * b + 128))
            qh = q[r].double().reshape(-1, heads, d)
            for h in range(heads):
                if sel is None:
                    rows = torch.arange(mk, device="cuda")
                else:
                    rows = [torch.arange(64 * c, min(mk, 64 * c + 64), device="cuda") for c in sel[b0 + b, h].tolist() if 0 <= c < nk]
                    if not rows:
                        continue
                    rows = torch.cat(rows)
                s = qh[:, h] @ kh[rows, h].T * scale
                p = torch.softmax(s, dim=1)
                out[r, h], mass[r, h] = p @ vh[rows, h], p @ vh[rows, h].abs()
                size[r, h, 0] = (qh[:, h].abs() @ kh[rows, h].abs().T).amax(1) * scale
        q0, k0, b0 = q0 + m, k0 + mk, b0 + nb
    return out.flatten(1), (mass, size)


def check(got, q, k, v, lens, klens, heads, kv, scale, sel=None):
    want, (mass, size) = attention(q, k, v, lens, klens, heads, kv, scale, sel)
    d, u = q.shape[1] // heads, unit(q.dtype)
    tol = (mass * (u + 2 * (size * d * 2.0 ** -23 + 4 * 2.0 ** -22) + 16 * F32)).flatten(1)
    # f16: weights below the smallest step of f16 (2^-24) are lost or rounded to it
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * v.abs().max().double() * max(klens)
    within(got, want, tol, u)


def lists(plan, heads, top, lens, klens, seed, holes=True):
    """Random lists without order, with -1 anywhere."""
    g = np.random.default_rng(seed)
    sel = np.full((plan.q_blocks, heads, top), -1, np.int32)
    b = 0
    for m, mk in zip(lens, klens):
        nk = -(-mk // 64)
        for _ in range(-(-m // 128)):
            for h in range(heads):
                pick = g.permutation(nk)[:top]
                at = np.sort(g.permutation(top)[:len(pick)])
                sel[b, h, at] = pick
                if holes and top > 1:
                    sel[b, h, g.random(top) < 0.2] = -1
            b += 1
    return torch.from_numpy(sel).cuda()


ATTEND = [
    # lens, klens, heads, kv, d, top, pad
    ([1], None, 1, 1, 64, 0, 0),
    ([1], [64], 1, 1, 64, 0, 0),
    ([5], [63], 2, 1, 64, 0, 8),
    ([64], [65], 1, 1, 128, 0, 0),
    ([128], None, 1, 1, 64, 0, 0),
    ([129], [128], 3, 3, 128, 0, 24),
    ([1000], None, 12, 12, 64, 0, 1536),
    ([2000], None, 4, 2, 128, 0, 0),
    ([0, 300, 1, 0, 77, 640], None, 4, 4, 64, 0, 0),
    ([0, 300, 1, 0, 77, 640], None, 4, 2, 128, 4, 8),
    ([1, 1, 1, 1], [700, 1, 64, 5000], 8, 2, 64, 0, 0),
    ([1, 1, 1], [700, 1, 3000], 8, 2, 128, 8, 0),
    ([3, 200, 40], [0, 1000, 130], 2, 2, 64, 0, 0),
    ([3, 200, 40], [0, 1000, 130], 2, 2, 64, 3, 0),
    ([1500], None, 6, 6, 64, 1, 0),
    ([1500], None, 6, 3, 64, 40, 0),
    ([1500], None, 2, 2, 128, 1024, 0),
    ([4000], None, 2, 2, 64, 16, 0),
    ([260], [9000], 2, 1, 64, 0, 0),
    ([50], [20000], 2, 1, 128, 0, 0),
    ([2600, 129], [600, 3000], 16, 8, 64, 0, 0),     # tiles for more than a wave
    ([2600, 129], [600, 3000], 16, 16, 128, 7, 0),
    ([128 * 19, 50], [64 * 30, 64 * 60], 16, 16, 64, 0, 0),  # a wave of whole tiles, then shared ones
    ([128 * 19, 50], [64 * 30, 64 * 60], 16, 4, 128, 40, 0),
    ([7, 1, 30], [3000, 200, 5000], 12, 2, 64, 0, 0),  # groups of 6: tiles of 2 heads
    ([7, 1, 3], [3000, 0, 5000], 32, 1, 128, 0, 0),    # 16 heads a tile
]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("lens,klens,heads,kv,d,top,pad", ATTEND)
def test_block_attention(ctx, lens, klens, heads, kv, d, top, pad, dt):
    kl = klens or lens
    q = strided((sum(lens), heads * d), 1, DT[dt], pad)
    k = strided((sum(kl), kv * d), 2, DT[dt], pad)
    v = strided((sum(kl), kv * d), 3, DT[dt], pad)
    plan = ctx.attn_plan(offsets(lens), offsets(klens) if klens else None)
    sel = lists(plan, heads, top, lens, kl, 4) if top else None
    out = torch.full((sum(lens), heads * d + pad), 7.0, dtype=DT[dt], device="cuda")
    ctx.block_attention(plan, q, k, v, heads, kv, out[:, :heads * d], sel=sel)
    ctx.check()
    check(out[:, :heads * d], q, k, v, lens, kl, heads, kv, d ** -0.5, sel)
    assert (out[:, heads * d:] == 7.0).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("lens,klens,heads,kv,d,top", [
    ([700, 0, 600, 3], [5000, 70, 40, 0], 4, 2, 64, 0),
    ([700, 0, 600, 3], [5000, 70, 40, 0], 4, 2, 64, 60),
    ([1280], [6000], 4, 4, 128, 0),
    ([101] * 13, [2000 + 64 * i for i in range(13)], 3, 1, 128, 0),  # rows to join that are no multiple of eight
])
def test_attention_split_lists_of_many_rows(ctx, lens, klens, heads, kv, d, top, dt):
    """Few tiles of many rows and long lists: several CTAs a list, the rows joined by a warp each."""
    q = randn((sum(lens), heads * d), 1, DT[dt])
    k, v = randn((sum(klens), kv * d), 2, DT[dt]), randn((sum(klens), kv * d), 3, DT[dt])
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    sel = lists(plan, heads, top, lens, klens, 4) if top else None
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, heads, kv, out, sel=sel)
    ctx.check()
    check(out, q, k, v, lens, klens, heads, kv, d ** -0.5, sel)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("lens,klens,heads,kv,d", [
    ([500] * 8, [100] * 3 + [9000] + [0, 64, 65, 1], 8, 8, 64),             # one long sequence among many tiles
    ([1] * 90 + [100, 3, 0], [64] * 90 + [20000, 9000, 8000], 16, 4, 128),  # and tiles of few rows
    ([700, 130, 400, 128, 900], [3000, 40, 12000, 9000, 500], 12, 6, 64),   # several, in no order
    ([128, 0, 1000, 64, 300, 1, 500], [100, 0, 1000, 64, 0, 1, 400], 12, 4, 128),  # none split, the longest first
])
def test_attention_long_lists_among_many(ctx, lens, klens, heads, kv, d, dt):
    """More tiles than CTA slots, a few of them far longer: those are split, the others are not."""
    q = randn((sum(lens), heads * d), 1, DT[dt])
    k, v = randn((sum(klens), kv * d), 2, DT[dt]), randn((sum(klens), kv * d), 3, DT[dt])
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, heads, kv, out)
    ctx.check()
    check(out, q, k, v, lens, klens, heads, kv, d ** -0.5)


@pytest.mark.parametrize("top", [0, 12])
@pytest.mark.parametrize("scale,size", [(1.0, 3.0), (0.001, 1.0), (4.0, 3.0), (1e-4, 0.1)])
def test_attention_peaked_and_flat(ctx, scale, size, top):
    """Scores hundreds apart (the maximum keeps growing, weights underflow) and almost equal ones."""
    n, heads, d = 1200, 2, 64
    q, k, v = (randn((n, heads * d), s, torch.bfloat16, size) for s in (1, 2, 3))
    k *= torch.linspace(0.1, 2.0, n, device="cuda")[:, None].to(torch.bfloat16)  # later keys reach higher
    plan = ctx.attn_plan([0, n])
    sel = lists(plan, heads, top, [n], [n], 4) if top else None
    out = torch.empty_like(q)
    ctx.block_attention(plan, q, k, v, heads, heads, out, scale=scale, sel=sel)
    check(out, q, k, v, [n], [n], heads, heads, scale, sel)


def test_attention_leaves_other_rows(ctx):
    """Sequences that begin after row 0 and end before the last: the other rows stay, whatever the inputs hold there."""
    heads, d, lens = 2, 64, [100, 0, 90, 200]
    q, k, v = (randn((500, heads * d), s, torch.bfloat16) for s in (1, 2, 3))
    for x in (q, k, v):
        x[:30] = float("nan")
        x[30 + sum(lens):] = float("inf")
    plan = ctx.attn_plan(offsets(lens, 30))
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, heads, heads, out)
    inner = slice(30, 30 + sum(lens))
    check(out[inner], q[inner], k[inner], v[inner], lens, lens, heads, heads, d ** -0.5)
    assert (out[:30] == 7.0).all() and (out[inner.stop:] == 7.0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.0e38])
def test_attention_ignores_what_it_does_not_attend_to(ctx, bad, d):
    """NaN, infinities and the type's largest values in the neighbouring sequences and in blocks not listed."""
    heads, lens = 2, [70, 200, 130]
    q, k, v = (randn((400, heads * d), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan(offsets(lens))
    sel = torch.full((plan.q_blocks, heads, 2), -1, dtype=torch.int32, device="cuda")
    sel[1:3, :, 1] = 3  # the middle sequence's short last block (8 rows), listed alone
    mid = slice(70, 270)
    clean = [x.clone() for x in (q, k, v)]
    k[:70], k[270:], v[:70], v[270:] = bad, bad, bad, bad
    k[70:70 + 192], v[70:70 + 192] = bad, bad
    out = torch.empty_like(q)
    ctx.block_attention(plan, q, k, v, heads, heads, out, sel=sel)
    full = torch.full((2, heads, 1), 3)
    check(out[mid], clean[0][mid], clean[1][mid], clean[2][mid], [200], [200], heads, heads, d ** -0.5, full)
    assert (out[:70] == 0).all() and (out[270:] == 0).all()  # nothing listed


def test_attention_passes_nan_and_infinity_on(ctx):
    """A NaN score makes its row NaN and no other; a value row's infinity shows where its weight is not 0."""
    n, d = 300, 64
    q, k, v = (randn((n, d), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan([0, n])
    out, ref = torch.empty_like(q), torch.empty_like(q)
    ctx.block_attention(plan, q, k, v, 1, 1, ref)
    for row in (0, 127, 200):
        q2 = q.clone()
        q2[row, 5] = float("nan")
        ctx.block_attention(plan, q2, k, v, 1, 1, out)
        assert out[row].isnan().all()
        out[row] = ref[row]
        assert torch.equal(out, ref)
    for col in range(0, n, 7):
        k2 = k.clone()
        k2[col, 3] = float("nan")
        ctx.block_attention(plan, q, k2, v, 1, 1, out)
        assert out.isnan().all(), col
    v2 = v.clone()
    v2[299, 9] = float("inf")
    ctx.block_attention(plan, q, k, v2, 1, 1, out)
    assert (out[:, 9] == float("inf")).all()
    out[:, 9] = ref[:, 9]
    assert torch.equal(out, ref)


def test_attention_of_minus_infinity_scores_is_zero(ctx):
    n, d = 130, 64
    q = torch.ones((n, d), dtype=torch.bfloat16, device="cuda")
    k, v = torch.full_like(q, -float("inf")), randn((n, d), 3, torch.bfloat16)
    plan = ctx.attn_plan([0, n])
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, 1, 1, out)
    assert (out == 0).all()
    k[77] = 0.25  # one key left
    ctx.block_attention(plan, q, k, v, 1, 1, out)
    assert torch.equal(out, v[77].expand_as(out))


def test_attention_counts_a_block_as_often_as_it_is_listed(ctx):
    n, d = 256, 64
    q, k, v = (randn((n, d), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan([0, n])
    sel = torch.tensor([2, 2, -1, 0, 2], dtype=torch.int32, device="cuda").expand(2, 1, 5).contiguous()
    out = torch.empty_like(q)
    ctx.block_attention(plan, q, k, v, 1, 1, out, sel=sel)
    check(out, q, k, v, [n], [n], 1, 1, d ** -0.5, sel)


def test_attention_reports_a_block_that_is_not_there(ctx):
    n, d = 256, 64
    q, k, v = (randn((n, d), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan([0, n])
    good = torch.tensor([1, 3, -1], dtype=torch.int32, device="cuda").expand(2, 1, 3).contiguous()
    out, ref = torch.empty_like(q), torch.empty_like(q)
    ctx.block_attention(plan, q, k, v, 1, 1, ref, sel=good)
    ctx.check()
    for wrong in (4, 1 << 30, 2 ** 31 - 1):
        sel = good.clone()
        sel[1, 0, 2] = wrong
        ctx.block_attention(plan, q, k, v, 1, 1, out, sel=sel)
        with pytest.raises(s3dsp.S3dError):
            ctx.check()
        assert torch.equal(out, ref)  # skipped
        ctx.check()


def test_attention_refuses_to_write_over_its_inputs(ctx):
    q, k, v = (randn((128, 64), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan([0, 128])
    for bad in (q, k, v):
        with pytest.raises(s3dsp.S3dError, match="overlap"):
            ctx.block_attention(plan, q, k, v, 1, 1, bad)


def test_attention_is_deterministic_and_plans_are_reusable(ctx):
    lens = [1111, 30, 2049]
    n = sum(lens)
    q, k, v = (randn((n, 256), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan(offsets(lens))
    sel = lists(plan, 4, 6, lens, lens, 1)
    a, b = torch.empty_like(q), torch.empty_like(q)
    for s in (sel, None):
        ctx.block_attention(plan, q, k, v, 4, 4, a, sel=s)
        for _ in range(3):
            ctx.block_attention(plan, q, k, v, 4, 4, b, sel=s)
            assert torch.equal(a, b)


def test_empty_calls(ctx):
    plan = ctx.attn_plan([0, 0, 0])
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert plan.q_blocks == 0 and plan.k_blocks == 0
    ctx.block_attention(plan, x, x, x, 1, 1, x)
    ctx.block_select(plan, x, x, 1, 1, torch.empty((0, 1, 4), dtype=torch.int32, device="cuda"))
    ctx.attn_plan([0])
    # queries without a single key row anywhere: zeros
    plan = ctx.attn_plan([0, 70, 300], [0, 0, 0])
    q = randn((300, 64), 1, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, x, x, 1, 1, out)
    assert (out == 0).all()
    sel = torch.full((plan.q_blocks, 1, 3), 9, dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, x, 1, 1, sel)
    assert (sel == -1).all()
    out.fill_(7.0)
    ctx.block_attention(plan, q, x, x, 1, 1, out, sel=sel)
    assert (out == 0).all()


# ---------------------------------------------------------------------------------------------------
# streams, graphs, contexts
# ---------------------------------------------------------------------------------------------------
def _chain(c, plan, qkv, pos, gq, gk, buf, heads, d):
    """Norms and rotation out of one projection's rows, selection, attention."""
    w = heads * d
    c.qk_norm_rope(qkv[:, :w], heads, gq, buf["q"], qkv[:, w:2 * w], heads, gk, buf["k"], positions=pos,
                   axis_pairs=[d // 6] * 3)
    c.block_select(plan, buf["q"], buf["k"], heads, heads, buf["sel"], keep_local=True)
    c.block_attention(plan, buf["q"], buf["k"], qkv[:, 2 * w:], heads, heads, buf["out"], sel=buf["sel"])
    c.block_attention(plan, buf["q"][:], buf["k"], qkv[:, 2 * w:], heads, heads, buf["dense"])


def _chain_data(lens, heads, d, top, seed, plan):
    n, w = sum(lens), heads * d
    new = lambda: torch.full((n, w), 7.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    return (randn((n, 3 * w), seed, torch.bfloat16), torch.randint(0, 64, (n, 4), device="cuda", dtype=torch.int32)[:, 1:],
            randn((heads, d), seed + 1) * 0.1 + 1, randn((heads, d), seed + 2) * 0.1 + 1,
            dict(q=new(), k=new(), out=new(), dense=new(),
                 sel=torch.empty((plan.q_blocks, heads, top), dtype=torch.int32, device="cuda")))


def test_two_captured_graphs_and_an_eager_call(ctx):
    """Two graphs captured on one context and replayed on two streams at once, an eager call beside them."""
    heads, d, top, lens = 4, 64, 4, [900, 33, 1500]
    stream = torch.cuda.Stream()
    side = torch.cuda.Stream()
    c = s3dsp.Context(0, stream=stream.cuda_stream, flags=s3dsp.CONTEXT_DEFERRED_CHECKS)
    plan = c.attn_plan(offsets(lens))
    data = [_chain_data(lens, heads, d, top, s, plan) for s in (10, 20, 30)]
    torch.cuda.synchronize()
    want = []
    for x in data:
        _chain(c, plan, *x, heads, d)
        stream.synchronize()
        want.append({k: t.clone() for k, t in x[4].items()})
        for t in x[4].values():
            t.fill_(5)
    torch.cuda.synchronize()
    graphs = []
    for x in data[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            _chain(c, plan, *x, heads, d)
        graphs.append(g)
    for x in data:
        for t in x[4].values():
            t.fill_(5)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(stream):
            graphs[1].replay()
            _chain(c, plan, *data[2], heads, d)
    torch.cuda.synchronize()
    for x, w in zip(data, want):
        for name, t in w.items():
            assert torch.equal(x[4][name], t), name
    c.check()


def test_a_plan_is_not_made_inside_a_capture():
    stream = torch.cuda.Stream()
    c = s3dsp.Context(0, stream=stream.cuda_stream)
    x = torch.zeros(16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        x += 1
        with pytest.raises(s3dsp.S3dError, match="capture"):
            c.attn_plan([0, 100])
    g.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()


def test_contexts_on_their_own_streams(ctx):
    """Several contexts at once, each on its own stream, on inputs of their own."""
    heads, d, top = 2, 64, 3
    runs = []
    torch.cuda.synchronize()
    for s, lens in enumerate(([700], [5, 2000], [1, 1, 1, 400], [1300])):
        c = s3dsp.Context(0, stream=0, flags=s3dsp.CONTEXT_OWN_STREAM)
        plan = c.attn_plan(offsets(lens))
        runs.append((c, plan, _chain_data(lens, heads, d, top, 50 + s, plan), lens))
    torch.cuda.synchronize()
    for _ in range(5):
        for c, plan, x, _ in runs:
            _chain(c, plan, *x, heads, d)
    for c, *_ in runs:
        c.check()
    for c, plan, x, lens in runs:
        ref = _chain_data(lens, heads, d, top, 0, plan)[4]
        plan2 = ctx.attn_plan(offsets(lens))
        _chain(ctx, plan2, *x[:4], ref, heads, d)
        torch.cuda.synchronize()
        for name, t in ref.items():
            assert torch.equal(x[4][name], t), name


def test_sm_limit_changes_nothing(ctx):
    c = s3dsp.Context(0)
    c.set_sm_limit(4)
    lens, heads, d = [300, 1], 2, 64
    plan = c.attn_plan(offsets(lens), [0, 4000, 9000])
    q = randn((301, 128), 1, torch.bfloat16)
    k, v = (randn((9000, 128), s, torch.bfloat16) for s in (2, 3))
    out = torch.empty_like(q)
    c.block_attention(plan, q, k, v, heads, heads, out)
    check(out, q, k, v, lens, [4000, 5000], heads, heads, d ** -0.5)


# ---------------------------------------------------------------------------------------------------
# together: a self-attention layer on the coarse rows of the SLat generator
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("top", [0, 3])
def test_together_in_the_middle_of_the_sparse_stages(ctx, top):
    """slat.CoarseAttention as SlatSparse.forward's mid at the generator's width, two objects: every step against its
    definition on the step's own inputs, and the layer as a whole within the BF16 gate."""
    coords = np.concatenate([workloads.ellipsoid_shell(32, 0), workloads.ellipsoid_shell(24, 1, batch=1)])
    device = torch.device("cuda", 0)
    heads, c = 16, slat.MODEL_CH
    d = c // heads
    params = slat.attention_params(c, heads)
    layer = slat.CoarseAttention(s3dsp, ctx, params, heads, device, top=top)
    net = slat.SlatSparse(s3dsp, ctx, slat.slat_params(), s3dsp.PREC_BF16, device)
    tb = slat.SlatTablesDev(s3dsp, ctx, torch.from_numpy(np.ascontiguousarray(coords)).cuda(), torch)
    tables = layer.tables(tb)
    pos, plan = tables[0][:, 1:], tables[1]
    lens = torch.bincount(tables[0][:, 0].long()).tolist()
    assert sum(lens) == tb.nc == plan.n_q and min(lens) > 300
    t, seen = {}, {}

    def mid(h):
        seen["h"] = h.clone()
        seen["y"] = layer.forward(tables, h, taps=t)
        return seen["y"]

    out = net.forward(tb, randn((tb.nf, slat.IN_CH), 1), net.mods_to_device(slat.slat_mods()), mid=mid)
    ctx.check()
    assert out.shape == (tb.nf, slat.OUT_CH) and torch.isfinite(out).all()

    w = {k: (torch.from_numpy(params[k]["w"]).cuda().to(torch.bfloat16).double(), torch.from_numpy(params[k]["b"]).cuda().double())
         for k in ("q", "kv", "out")}
    x = torch.nn.functional.layer_norm(seen["h"].double(), (c,), eps=1e-6)
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    gate(rel(t["x"], x), 1e-2, "layer norm")
    lin = {k: t["x"].double() @ w[k][0].T + w[k][1] for k in ("q", "kv")}
    gate(rel(t["v"], lin["kv"][:, c:]), 1e-2, "v")
    heads_of = {"q": lin["q"], "k": lin["kv"][:, :c]}
    for name in ("q", "k"):
        g = torch.from_numpy(params[name + "_gamma"]).cuda().double()
        a = heads_of[name].reshape(-1, heads, d)
        a = (a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * g).reshape(-1, c)
        gate(rel(t[name], turned(a, pos, heads, [d // 6] * 3, 1e4, False, False)[0]), 1e-2, name)
    if top:
        assert torch.equal(t["sel"].cpu(), chosen(t["q"], t["k"], lens, lens, heads, heads, top, True))
    check(t["a"], t["q"], t["k"], t["v"], lens, lens, heads, heads, d ** -0.5, t["sel"])
    gate(rel(seen["y"], t["a"].double() @ w["out"][0].T + w["out"][1] + seen["h"].double()), 1e-2, "layer")


# ---------------------------------------------------------------------------------------------------
# batches whose longest key sequence has no query rows
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("lens,klens,heads,kv,d", [
    ([0, 1], [42000, 100], 16, 4, 128),                       # few tiles
    ([0, 300], [6000, 200], 12, 12, 64),
    ([0, 4000, 100], [6000, 300, 100], 16, 16, 64),           # more tiles than CTA slots
    ([2, 0, 1], [9000, 90000, 64], 16, 4, 128),               # another list is split
    ([500] * 7 + [0], [100] * 3 + [9000] + [0, 64, 65, 60000], 8, 8, 64),
])
def test_attention_longest_keys_without_queries(ctx, lens, klens, heads, kv, d, dt):
    q = randn((sum(lens), heads * d), 1, DT[dt])
    k, v = randn((sum(klens), kv * d), 2, DT[dt]), randn((sum(klens), kv * d), 3, DT[dt])
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    assert plan.max_k_blocks == max(-(-m // 64) for m in klens)
    for top in (0, 5):
        sel = lists(plan, heads, top, lens, klens, 4) if top else None
        out = torch.full_like(q, 7.0)
        ctx.block_attention(plan, q, k, v, heads, kv, out, sel=sel)
        ctx.check()
        check(out, q, k, v, lens, klens, heads, kv, d ** -0.5, sel)


@pytest.mark.parametrize("lens,klens,top", [
    ([0, 300], [64 * 1100, 3000], 5), ([200, 0, 5], [700, 64 * 28001, 64 * 20], 3), ([0, 300], [9000, 200], 5),
])
def test_block_select_longest_keys_without_queries(ctx, lens, klens, top):
    """Key blocks that no query row sees count neither for the limit nor for the lists."""
    q, k = randn((sum(lens), 128), 1, torch.bfloat16), randn((sum(klens), 128), 2, torch.bfloat16)
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    sel = torch.full((plan.q_blocks, 2, top), -7, dtype=torch.int32, device="cuda")
    ctx.block_select(plan, q, k, 2, 2, sel)
    assert torch.equal(sel.cpu(), chosen(q, k, lens, klens, 2, 2, top, False))


@pytest.mark.parametrize("own", [False, True])
def test_coarse_attention_on_a_stream_that_is_not_current(ctx, own):
    """tables() and forward() on a context whose stream is busy and not torch's current one (its own, or another torch
    stream): the row counts are read after the coordinates are written, and buffers that torch hands out again
    meanwhile are not the layer's."""
    device = torch.device("cuda", 0)
    coords = np.concatenate([workloads.ellipsoid_shell(24, b, batch=b) for b in range(3)])
    d_coords = torch.from_numpy(np.ascontiguousarray(coords)).cuda()
    heads, c = 4, 256
    params = slat.attention_params(c, heads)
    layer = slat.CoarseAttention(s3dsp, ctx, params, heads, device, top=3)
    tb = slat.SlatTablesDev(s3dsp, ctx, d_coords, torch)
    want_tables = layer.tables(tb)
    h = randn((tb.nc, c), 1)
    want = layer.forward(want_tables, h)
    torch.cuda.synchronize()

    stream = torch.cuda.Stream()
    other = s3dsp.Context(0, stream=0 if own else stream.cuda_stream, flags=s3dsp.CONTEXT_OWN_STREAM if own else 0)
    layer = slat.CoarseAttention(s3dsp, other, params, heads, device, top=3)
    tb2 = slat.SlatTablesDev(s3dsp, other, d_coords, torch)
    other.check()
    junk = [torch.full((tb.nc, w), -1, dtype=torch.int32, device="cuda") for w in (4, c, c // 2)]
    torch.cuda.synchronize()
    del junk  # torch's stream gets these rows of -1 next
    with torch.cuda.stream(layer.stream):
        torch.cuda._sleep(20_000_000)
    tables = layer.tables(tb2)
    assert torch.equal(tables[0], want_tables[0])
    assert (tables[1].n_q, tables[1].q_blocks) == (want_tables[1].n_q, want_tables[1].q_blocks)
    for _ in range(3):
        with torch.cuda.stream(layer.stream):
            torch.cuda._sleep(20_000_000)
        got = layer.forward(tables, h)
        for w in (4, c // 2, c, 2 * c):  # torch's stream writes wherever it may
            torch.full((tb.nc, w), 7, dtype=torch.int32, device="cuda")
        other.check()
        assert torch.equal(got, want)


# ---------------------------------------------------------------------------------------------------
# the range of values and weights
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("grow", [7.5, 8.5, 16.0, 20.0, 23.9, 40.0])
@pytest.mark.parametrize("lens,klens,heads,kv,d", [
    ([130], [300], 2, 2, 64), ([130], [300], 2, 1, 128), ([1, 3], [6000, 200], 2, 2, 64),  # the last: a split list
])
def test_attention_of_large_values(ctx, lens, klens, heads, kv, d, grow):
    """bf16 values whose plain sum with weights of at most 1 fits f32 (|v| times the keys up to 2^127), and a maximum
    that grows by so many powers of two after the first block of keys."""
    big = 2.0 ** 124 / max(klens)  # a normal value of more than 8 sigma does not come up
    q = torch.zeros((sum(lens), heads * d), dtype=torch.bfloat16, device="cuda")
    q[:, ::d] = 1.0
    k = randn((sum(klens), kv * d), 2, torch.bfloat16, 0.25)
    v = randn((sum(klens), kv * d), 3, torch.bfloat16, big)
    at = 0
    for m in klens:
        k[at + 64:at + m, ::d] += grow * np.log(2.0)
        at += m
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, heads, kv, out, scale=1.0)
    ctx.check()
    check(out, q, k, v, lens, klens, heads, kv, 1.0)


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("gap", [12.3, 17.7, 20.4, 23.6, 25.2, 29.5])
@pytest.mark.parametrize("lens,klens,heads,kv,d", [
    ([130], [4000], 2, 2, 64), ([130], [4000], 2, 1, 128), ([1, 3], [20000, 4000], 2, 2, 64),  # split lists
    ([2000], [4000], 16, 4, 64), ([2000], [4000], 16, 4, 128),                                 # whole ones
])
def test_attention_f16_of_small_weights(ctx, lens, klens, heads, kv, d, gap, last):
    """f16: one key (the first or the last) with a score far above the others', which are equal, and with value 0: the
    others' weights, 2^-gap of its, all round the same way. A weight is off by u of it or 2^-25 2^-7 of the largest."""
    q = torch.zeros((sum(lens), heads * d), dtype=torch.float16, device="cuda")
    q[:, ::d] = 1.0
    k = torch.zeros((sum(klens), kv * d), dtype=torch.float16, device="cuda")
    v = randn((sum(klens), kv * d), 3, torch.float16, 0.25) + 1.0
    at = 0
    for m in klens:
        one = at + (m - 1 if last else 0)
        k[one, ::d], v[one] = gap * np.log(2.0), 0.0
        at += m
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, heads, kv, out, scale=1.0)
    ctx.check()
    want, (mass, size) = attention(q, k, v, lens, klens, heads, kv, 1.0)
    u = unit(torch.float16)
    tol = (mass * (u + 2 * (size * d * 2.0 ** -23 + 4 * 2.0 ** -22) + 16 * F32)).flatten(1)
    within(out, want, tol + 2.0 ** -32 * float(v.abs().max()) * max(klens), u)


# ---------------------------------------------------------------------------------------------------
# the scratch of a selection
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,klens,heads,top", [
    ([330000], [64 * 28000], 2, 9),                             # cut inside a sequence, one head at a time
    ([1] * 2500 + [300] + [1] * 2500, [64] * 2500 + [64 * 28000] + [200] * 2500, 1, 5),
])
def test_block_select_holds_at_most_512_mb_of_scores(ctx, lens, klens, heads, top):
    """A head's scores (a row as long as the longest sequence for each query block) beyond that take several passes."""
    d = 64
    q, k = randn((sum(lens), heads * d), 1, torch.bfloat16), randn((sum(klens), heads * d), 2, torch.bfloat16)
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    assert plan.q_blocks * plan.max_k_blocks * 8 > 1 << 29
    sel = torch.full((plan.q_blocks, heads, top), -7, dtype=torch.int32, device="cuda")
    ctx.check()
    used = s3dsp.memory_stats(0, reset_high=True)["used"]
    ctx.block_select(plan, q, k, heads, heads, sel)
    ctx.check()
    means = (plan.q_blocks + plan.k_blocks) * heads * d * 8
    assert s3dsp.memory_stats(0)["used_high"] - used <= (1 << 29) + means + (1 << 16)
    q0 = k0 = b0 = 0
    for m, mk in zip(lens, klens):
        nb, nk = -(-m // 128), -(-mk // 64)
        if nk <= top:
            want = torch.arange(top, device="cuda").where(torch.arange(top, device="cuda") < nk, -1).expand(nb, heads, top)
        else:
            mean = lambda x, rows: torch.stack([c.double().mean(0) for c in x.split(rows)]).reshape(-1, heads, d)  # noqa: E731
            score = torch.einsum("bhd,chd->bhc", mean(q[q0:q0 + m], 128), mean(k[k0:k0 + mk], 64))
            want = score.topk(top, dim=-1).indices.sort(dim=-1).values
        assert torch.equal(sel[b0:b0 + nb].long(), want)
        q0, k0, b0 = q0 + m, k0 + mk, b0 + nb


@pytest.mark.parametrize("n,long,short,d", [(84, 6213, 50, 128), (149, 6000, 50, 128), (90, 5000, 40, 64)])
def test_attention_partial_sums_are_bounded(ctx, n, long, short, d):
    """One long list among many that are a little longer than a chunk: at most 256 MB of partial sums."""
    lens, klens = [128] * n, [64 * short] * 20 + [64 * long] + [64 * short] * (n - 21)
    q = randn((sum(lens), d), 1, torch.bfloat16)
    k, v = randn((sum(klens), d), 2, torch.bfloat16), randn((sum(klens), d), 3, torch.bfloat16)
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    out = torch.full_like(q, 7.0)
    ctx.check()
    used = s3dsp.memory_stats(0, reset_high=True)["used"]
    ctx.block_attention(plan, q, k, v, 1, 1, out)
    ctx.check()
    assert s3dsp.memory_stats(0)["used_high"] - used <= 1 << 28
    check(out, q, k, v, lens, klens, 1, 1, d ** -0.5)


def test_a_plan_outlives_its_context():
    """Freed after its context: the block tables go back to the pool."""
    c = s3dsp.Context(0)
    c.check()
    torch.cuda.synchronize()
    used = s3dsp.memory_stats(0)["used"]
    plan = c.attn_plan(offsets([5000] * 2000))
    assert s3dsp.memory_stats(0)["used"] >= used + plan.q_blocks * 32 + plan.k_blocks * 8
    c.close()
    plan.free()
    torch.cuda.synchronize()
    assert s3dsp.memory_stats(0)["used"] <= used


@pytest.mark.parametrize("pairs", [(), (5, 0, 20), None])
def test_coarse_attention_axis_pairs(ctx, pairs):
    """The layer without a rotation (rows that carry their position already), with pairs dealt otherwise, and as it is
    by default: q and k against the norm's definition and the rotation's."""
    device = torch.device("cuda", 0)
    coords = torch.from_numpy(np.ascontiguousarray(workloads.ellipsoid_shell(24, 1))).cuda()
    heads, c = 4, 256
    d = c // heads
    params = slat.attention_params(c, heads)
    layer = slat.CoarseAttention(s3dsp, ctx, params, heads, device, axis_pairs=pairs)
    tb = slat.SlatTablesDev(s3dsp, ctx, coords, torch)
    tables, t = layer.tables(tb), {}
    layer.forward(tables, randn((tb.nc, c), 1), taps=t)
    ctx.check()
    for name, wk, rows in (("q", "q", slice(0, c)), ("k", "kv", slice(0, c))):
        w = torch.from_numpy(params[wk]["w"][rows]).cuda().to(torch.bfloat16).double()
        a = (t["x"].double() @ w.T + torch.from_numpy(params[wk]["b"][rows]).cuda().double()).reshape(-1, heads, d)
        a = a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * torch.from_numpy(params[name + "_gamma"]).cuda().double()
        used = [d // 6] * 3 if pairs is None else list(pairs)
        want = turned(a.reshape(-1, c), tables[0][:, 1:], heads, used, 1e4, False, False)[0]
        gate(float((t[name].double() - want).norm() / want.norm()), 1e-2, name)
    check(t["a"], t["q"], t["k"], t["v"], [tb.nc], [tb.nc], heads, heads, d ** -0.5)


# ---------------------------------------------------------------------------------------------------
# scores far from 0: a softmax sees their differences
# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("offset", ["all", "later", "below", "below at first", "rows"])
@pytest.mark.parametrize("power", [10, 13, 16, 20, 30])
@pytest.mark.parametrize("lens,klens,heads,kv,d", [
    ([130], [1500], 2, 1, 64), ([130], [1500], 2, 1, 128),                # split lists
    ([700], [1500], 32, 8, 64), ([700], [1500], 32, 8, 128), ([5, 100], [40, 200], 2, 2, 64),
])
def test_attention_of_far_scores(ctx, lens, klens, heads, kv, d, power, offset, dt):
    """Scores (offset + x) / 2, exact in f32: an offset of 2^power to all keys, to those after the first 100, below 0,
    below 0 for the first 100 only, or of another size for each row; x whole numbers that grow along the keys. Each
    score's exponential is then off by less than 2^-18 (the rounding of an exponent up to 60, and ex2's 2^-22)."""
    if power == 30 and (offset != "below at first" or min(klens) <= 100):
        return  # a row whose scores are all 2^30 + x, which is no f32 (31 bits)
    nq, nk = sum(lens), sum(klens)
    q = torch.zeros((nq, heads, d), dtype=DT[dt], device="cuda")
    k = torch.zeros((nk, kv, d), dtype=DT[dt], device="cuda")
    v = randn((nk, kv * d), 3, DT[dt])
    place = torch.cat([torch.arange(m, device="cuda") for m in klens])
    x = (place * 60.0 / max(klens) + 12.0 * torch.rand(nk, generator=torch.Generator("cuda").manual_seed(1), device="cuda")).round()
    q[:, :, 1], k[:, :, 1] = 1.0, x[:, None]
    a, b = 2.0 ** (power // 2), 2.0 ** (power - power // 2)
    q[:, :, 5] = a
    if offset == "rows":
        q[:, :, 5] *= 2.0 ** -(torch.arange(nq, device="cuda") % 8)[:, None]
    sign = {"all": (1, 1), "later": (0, 1), "below": (-1, -1), "below at first": (-1, 0), "rows": (1, 1)}[offset]
    k[:, :, 5] = torch.where(place < 100, sign[0] * b, sign[1] * b)[:, None]
    q, k = q.flatten(1), k.flatten(1)
    plan = ctx.attn_plan(offsets(lens), offsets(klens))
    out = torch.full_like(q, 7.0)
    ctx.block_attention(plan, q, k, v, heads, kv, out, scale=0.5)
    ctx.check()
    want, (mass, _) = attention(q, k, v, lens, klens, heads, kv, 0.5)
    u = unit(DT[dt])
    tol = mass.flatten(1) * (u + 2.0 ** -17 + 16 * F32)
    if dt == "f16":
        tol = tol + 2.0 ** -32 * float(v.abs().max()) * max(klens)
    within(out, want, tol, u)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [1.0, 0.3, 1e-3])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_far_apart_scores(ctx, d, scale, dt):
    """Exact scores up to 2^36 apart by 2^28 and more: each row is the value of its largest key, whatever its place."""
    n = 300
    q = torch.full((n, d), 2.0 ** 15, dtype=DT[dt], device="cuda")
    q[::3] *= -1.0
    order = torch.from_numpy(np.random.default_rng(d).permutation(n).astype(np.float32)).cuda() - 100.0
    order = torch.where(order.abs() > 120, order.sign() * 119, order)  # whole numbers that both types keep, with ties
    order[17], order[211] = 127.0, -126.0
    k = (order * 128.0).to(DT[dt])[:, None].expand(n, d).contiguous()
    v = randn((n, d), 3, DT[dt])
    plan = ctx.attn_plan([0, n])
    out = torch.empty_like(q)
    ctx.block_attention(plan, q, k, v, 1, 1, out, scale=scale)
    ctx.check()
    best = torch.full((n,), 17, device="cuda")
    best[::3] = 211
    assert torch.equal(out, v[best])


def test_coarse_attention_in_a_graph():
    """The layer captured on its context's stream and replayed, on new rows, beside an eager call."""
    device = torch.device("cuda", 0)
    stream = torch.cuda.Stream()
    c = s3dsp.Context(0, stream=stream.cuda_stream, flags=s3dsp.CONTEXT_DEFERRED_CHECKS)
    width = 256
    layer = slat.CoarseAttention(s3dsp, c, slat.attention_params(width, 4), 4, device, top=3)
    coords = np.concatenate([workloads.ellipsoid_shell(24, b, batch=b) for b in range(2)])
    with torch.cuda.stream(stream):
        tb = slat.SlatTablesDev(s3dsp, c, torch.from_numpy(np.ascontiguousarray(coords)).cuda(), torch)
        tables = layer.tables(tb)
        h = [randn((tb.nc, width), seed) for seed in (1, 2, 3)]
        want = [layer.forward(tables, x).clone() for x in h]
        held = h[0].clone()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = layer.forward(tables, held)
    for x, w in zip(h, want):
        with torch.cuda.stream(stream):
            held.copy_(x)
            graph.replay()
            eager = layer.forward(tables, h[0])
        stream.synchronize()
        assert torch.equal(y, w) and torch.equal(eager, want[0])
    c.check()


def test_the_report_of_an_absent_block_names_it(ctx):
    q, k, v = (randn((128, 64), s, torch.bfloat16) for s in (1, 2, 3))
    plan = ctx.attn_plan([0, 128])
    ctx.block_attention(plan, q, k, v, 1, 1, torch.empty_like(q),
                        sel=torch.tensor([[[0, 2]]], dtype=torch.int32, device="cuda"))
    with pytest.raises(s3dsp.S3dError, match="listed key block"):
        ctx.check()
