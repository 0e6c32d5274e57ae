"""The arguments that the attention operators refuse, on the host: every check
comes before the first CUDA call, so zeroed memory stands in for a context
and a plan (device 0, no blocks) and no GPU is needed."""
import ctypes

import pytest
import torch

import s3dsp

BLANK = ctypes.create_string_buffer(4096)  # a context / plan with every field zero
FAKE = ctypes.addressof(BLANK)
X = torch.zeros(64, 512, dtype=torch.bfloat16)
POS = torch.zeros(64, 4, dtype=torch.int32)
PAIRS = (ctypes.c_int32 * 4)(10, 10, 10, 0)


def status(fn, args):
    buf = ctypes.create_string_buffer(256)
    st = fn(*args, buf, 256)
    return st, buf.value.decode()


def rope_args(**kw):
    a = dict(ctx=FAKE, x=X.data_ptr(), xd=s3dsp.BF16, n=64, xs=512, heads=8, d=64, pos=POS.data_ptr(), ps=4, axes=3,
             pairs=PAIRS, theta=10000.0, flags=0, y=X.data_ptr() + 16, yd=s3dsp.BF16, ys=512)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(ctx=None), "ctx"), (dict(xd=7), "dtype"), (dict(yd=3), "dtype"), (dict(flags=8), "flags"),
    (dict(n=-1), "row count"), (dict(n=1 << 31), "row count"), (dict(d=0), "head dimension"),
    (dict(d=60), "head dimension"), (dict(d=264), "head dimension"), (dict(axes=5), "axes"), (dict(axes=-1), "axes"),
    (dict(pairs=None), "axes"), (dict(pos=None), "positions"), (dict(ps=2), "positions"), (dict(theta=0.0), "theta"),
    (dict(theta=float("inf")), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(pairs=(ctypes.c_int32 * 3)(16, 16, 1)), "axis_pairs"), (dict(pairs=(ctypes.c_int32 * 3)(-1, 1, 1)), "axis_pairs"),
    (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(heads=0), "head count"), (dict(heads=-3), "head count"),
    (dict(xs=511), "row stride"), (dict(ys=511), "row stride"), (dict(x=X.data_ptr() + 1), "aligned"),
    (dict(y=X.data_ptr() + 1), "aligned"), (dict(y=X.data_ptr(), ys=520), "in place"),
    (dict(y=X.data_ptr(), yd=s3dsp.F32), "in place"),
])
def test_rope_refuses(kw, word):
    st, msg = status(s3dsp.load().s3dsp_rope, rope_args(**kw))
    assert st == s3dsp.S3D_INVALID_ARGUMENT and word in msg, msg


def test_rope_of_no_rows_is_done():
    assert status(s3dsp.load().s3dsp_rope, rope_args(n=0))[0] == s3dsp.S3D_OK


def qk_args(**kw):
    a = dict(ctx=FAKE, q=X.data_ptr(), qs=512, heads=8, gq=None, k=X.data_ptr(), ks=512, kv=4, gk=None, xd=s3dsp.BF16,
             n=64, d=64, eps=1e-6, pos=POS.data_ptr(), ps=4, axes=3, pairs=PAIRS, theta=10000.0, flags=0,
             qo=X.data_ptr(), qos=512, ko=X.data_ptr(), kos=512, yd=s3dsp.BF16)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(ctx=None), "ctx"), (dict(xd=9), "dtype"), (dict(flags=s3dsp.ROPE_INVERSE), "flags"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(k=None), "no k"),
    (dict(k=None, kv=0), "no k"), (dict(kv=0), "k: bad head"), (dict(q=None), "q: NULL"), (dict(qo=None), "q: NULL"),
    (dict(ko=None), "k: NULL"), (dict(qs=500), "q: row stride"), (dict(kos=200), "k: row stride"),
    (dict(d=4), "head dimension"), (dict(qos=1024), "in place"),
])
def test_qk_norm_rope_refuses(kw, word):
    st, msg = status(s3dsp.load().s3dsp_qk_norm_rope, qk_args(**kw))
    assert st == s3dsp.S3D_INVALID_ARGUMENT and word in msg, msg


def plan_args(q, k=None, ctx=FAKE, n=None, out=True):
    qo = (ctypes.c_int64 * len(q))(*q)
    ko = (ctypes.c_int64 * len(k))(*k) if k is not None else None
    h = ctypes.c_void_p()
    return [ctx, qo, ko, len(q) - 1 if n is None else n, ctypes.byref(h) if out else None]


@pytest.mark.parametrize("args,word", [
    (plan_args([0, 5], ctx=None), "NULL"), (plan_args([0, 5], out=False), "NULL"), (plan_args([0, 5], n=-1), "sequence"),
    (plan_args([0, 5, 4]), "offsets"), (plan_args([-1, 5]), "offsets"), (plan_args([0, 1 << 31]), "offsets"),
    (plan_args([0, 5], [3, 2]), "offsets"), (plan_args([0, 5], [0, (1 << 31) - 255]), "offsets"),
])
def test_plan_refuses(args, word):
    st, msg = status(s3dsp.load().s3dsp_attn_plan_create, args)
    assert st == s3dsp.S3D_INVALID_ARGUMENT and word in msg, msg


def select_args(**kw):
    a = dict(ctx=FAKE, plan=FAKE, q=X.data_ptr(), qs=512, heads=8, k=X.data_ptr(), ks=512, kv=4, dt=s3dsp.BF16, d=64,
             top=4, local=0, sel=POS.data_ptr())
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(ctx=None), "NULL"), (dict(plan=None), "NULL"), (dict(dt=5), "dtype"), (dict(d=12), "head dimension"),
    (dict(d=512), "head dimension"), (dict(kv=3), "heads over"), (dict(heads=0), "heads over"),
    (dict(kv=0), "heads over"), (dict(heads=8192, kv=1, qs=1 << 20), "heads over"), (dict(qs=511), "row stride"),
    (dict(ks=255), "row stride"), (dict(top=0), "top"), (dict(top=1025), "top"), (dict(local=1), "keep_local"),
])
def test_select_refuses(kw, word):
    st, msg = status(s3dsp.load().s3dsp_block_select, select_args(**kw))
    assert st == s3dsp.S3D_INVALID_ARGUMENT and word in msg, msg


def attend_args(**kw):
    a = dict(ctx=FAKE, plan=FAKE, q=X.data_ptr(), qs=512, heads=8, k=X.data_ptr(), ks=512, v=X.data_ptr(), vs=512, kv=4,
             dt=s3dsp.BF16, d=64, scale=0.125, sel=POS.data_ptr(), top=4, out=X.data_ptr(), os=512)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(ctx=None), "NULL"), (dict(plan=None), "NULL"), (dict(dt=s3dsp.F32), "dtype"), (dict(d=32), "head dimension"),
    (dict(d=96), "head dimension"), (dict(kv=5), "heads over"), (dict(heads=-8), "heads over"),
    (dict(qs=504), "row stride"), (dict(vs=248), "row stride"), (dict(os=8), "row stride"),
    (dict(qs=516), "multiples of 8"), (dict(ks=513), "multiples of 8"), (dict(os=1 << 40 | 4), "multiples of 8"),
    (dict(ks=1 << 39), "multiples of 8"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(top=0), "top"),
    (dict(top=2000), "top"), (dict(sel=None), "top"),
])
def test_attention_refuses(kw, word):
    st, msg = status(s3dsp.load().s3dsp_block_attention, attend_args(**kw))
    assert st == s3dsp.S3D_INVALID_ARGUMENT and word in msg, msg


def test_calls_on_an_empty_plan_are_done():
    assert status(s3dsp.load().s3dsp_block_select, select_args())[0] == s3dsp.S3D_OK
    assert status(s3dsp.load().s3dsp_block_attention, attend_args())[0] == s3dsp.S3D_OK


class Ctx(s3dsp.Context):
    """The binding's own checks, without a device behind them."""

    def __init__(self):
        self.handle = None


class Plan:
    handle, n_q, n_k, q_blocks, k_blocks = FAKE, 64, 64, 1, 1


def test_binding_refuses():
    c, x = Ctx(), torch.zeros(64, 512, dtype=torch.bfloat16)
    sel = torch.zeros(1, 8, 4, dtype=torch.int32)
    bad = [
        lambda: c.rope(x, POS, 7, x, [10, 10, 10]),                                # columns are no 7 heads
        lambda: c.rope(x, POS, 8, x[:, :256], [10, 10, 10]),                       # shapes differ
        lambda: c.rope(x.t(), POS, 8, x.t(), [1]),                                 # columns not contiguous
        lambda: c.rope(x, POS.long(), 8, x, [10, 10, 10]),                         # positions not int32
        lambda: c.rope(x, POS[:5], 8, x, [10, 10, 10]),                            # too few positions
        lambda: c.rope(x, POS[:, :2], 8, x, [10, 10, 10]),                         # too few axes
        lambda: c.qk_norm_rope(x, 8, torch.zeros(4, 64), x),                       # gamma shape
        lambda: c.qk_norm_rope(x, 8, torch.zeros(8, 64).double(), x),              # gamma type
        lambda: c.qk_norm_rope(x, 8, torch.zeros(64), x, x, 8, torch.zeros(8, 64), x),  # shared and not
        lambda: c.qk_norm_rope(x, 8, None, x, x, 4, None, x),                      # head dimensions differ
        lambda: c.qk_norm_rope(x, 8, None, x, x.float(), 8, None, x),              # types differ
        lambda: c.attn_plan([]),
        lambda: c.attn_plan([0, 4], [0, 4, 5]),
        lambda: c.block_select(Plan, x[:9], x, 8, 8, sel),                         # rows missing
        lambda: c.block_select(Plan, x, x, 8, 8, sel.long()),
        lambda: c.block_select(Plan, x, x, 8, 8, sel[:, :4]),
        lambda: c.block_attention(Plan, x, x, x[:9], 8, 8, x),                     # v unlike k
        lambda: c.block_attention(Plan, x, x, x, 8, 8, x.half()),
        lambda: c.block_attention(Plan, x, x, x, 8, 8, x, sel=sel[:, :, ::2]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(s3dsp.S3dError):
            f()
            pytest.fail(f"call {i} was accepted")



def test_binding_refuses_tensors_elsewhere():
    c, x = Ctx(), torch.zeros(64, 512, dtype=torch.bfloat16)
    c.device = 0
    sel = torch.zeros(1, 8, 4, dtype=torch.int32)
    for f in (
        lambda: c.rope(x, POS, 8, x, [10, 10, 10]),
        lambda: c.qk_norm_rope(x, 8, torch.ones(64), x),
        lambda: c.block_select(Plan, x, x, 8, 8, sel),
        lambda: c.block_attention(Plan, x, x, x, 8, 8, x.clone(), sel=sel),
    ):
        with pytest.raises(s3dsp.S3dError, match="a tensor on cpu"):
            f()


def test_binding_refuses_k_without_its_output():
    c, x = Ctx(), torch.zeros(64, 512, dtype=torch.bfloat16)
    with pytest.raises(s3dsp.S3dError, match="k_out"):
        c.qk_norm_rope(x, 8, None, x, x, 8)
