"""CPU checks of the attention, LayerNorm and preference entry points: what the C ABI refuses (before any
HIP call, with addresses that are never read), what the Python functions refuse, and their fakes."""
import ctypes

import pytest
import torch

import sparton_amd
from sparton_amd import _lib
from sparton_amd.attention import attention
from sparton_amd.loss import preference_loss, preference_margin
from sparton_amd.norm import SpartonLayerNorm, layer_norm

P = 0x10000  # 16- and 256-byte aligned address that is never read


def desc(**kw):
    a = dict(B=2, Hq=4, Hk=2, Sq=8, Sk=16, D=64, mask_batch=16, scale=0.125, causal=0, dtype=1, mask_dtype=0)
    s = dict(q=(2048, 64, 256), k=(2048, 64, 128), v=(2048, 64, 128), o=(2048, 64, 256), d_o=(2048, 64, 256),
             d_q=(2048, 64, 256), d_k=(2048, 64, 128), d_v=(2048, 64, 128))
    for n in list(kw):
        if n in s:
            s[n] = kw.pop(n)
    a.update(kw)
    d = _lib.AttentionDesc(**a)
    for n, v in s.items():
        getattr(d, n)[:] = v
    return ctypes.byref(d)


def fwd(d=None, **kw):
    a = dict(q=P, k=P, v=P, mask=P, out=P, lse=P, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.load().sparton_attention_fwd(desc(**(d or {})), *a.values())


def bwd(d=None, **kw):
    a = dict(q=P, k=P, v=P, mask=P, out=P, lse=P, do=P, dq=P, dk=P, dv=P, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.load().sparton_attention_bwd(desc(**(d or {})), *a.values())


BAD_DESC = [
    (dict(B=-1), -1), (dict(Hq=-4), -1), (dict(Sq=-1), -1), (dict(Sk=-1), -1), (dict(D=0), -1), (dict(D=60), -1),
    (dict(D=62, dtype=0), -1), (dict(dtype=3), -1), (dict(dtype=0x100), -1), (dict(mask_dtype=3), -1),
    (dict(mask_dtype=-1), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("inf")), -1),
    (dict(scale=float("nan")), -1), (dict(Hq=3), -1), (dict(Hk=0), -1), (dict(D=136), -3),
    (dict(Sk=1 << 31), -3), (dict(Sq=1 << 31), -3), (dict(B=1 << 30, Hq=4), -3), (dict(Sq=1 << 29, Hq=8, Hk=1), -3),
    (dict(B=1 << 20, Sk=1 << 20), -3),
    (dict(q=(2048, 60, 256)), -2), (dict(k=(2048, 64, 124)), -2), (dict(v=(2044, 64, 128)), -2),
]


@pytest.mark.parametrize("d,code", BAD_DESC)
def test_attention_description_is_checked(d, code):
    assert fwd(d) == code and bwd(d) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(q=P + 8), -2),
    (dict(out=P + 2), -2), (dict(v=P + 4), -2),
])
def test_attention_fwd_pointers_are_checked(kw, code):
    assert fwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(lse=None), -1), (dict(do=None), -1), (dict(dq=None), -1), (dict(dk=None), -1),
    (dict(dv=None), -1), (dict(dk=P + 8), -2), (dict(do=P + 8), -2), (dict(ws=None), -4), (dict(ws_bytes=16), -4),
    (dict(ws=P + 16), -2),
])
def test_attention_bwd_pointers_are_checked(kw, code):
    assert bwd(**kw) == code


def test_attention_sizes_with_nothing_to_do():
    assert fwd(dict(B=0)) == 0 and bwd(dict(B=0)) == 0 and fwd(dict(Hq=0, Hk=0)) == 0 and fwd(dict(Sq=0)) == 0
    assert _lib.load().sparton_attention_fwd(None, P, P, P, P, P, P, P, 0, None) == -1
    # a dimension of one may have any stride
    L = _lib.load()
    assert L.sparton_attention_workspace_bytes(desc(B=1, q=(7, 64, 256))) >= 0


THREADS = 1 << 32  # a launch of as many threads leaves workgroups out, and reports nothing
MOST = THREADS // 256 - 1


@pytest.mark.parametrize("sizes", [
    dict(B=1 << 24, Hq=1, Hk=1, Sq=1, Sk=1),             # a workgroup a (batch row, key head)
    dict(B=1 << 12, Hq=1 << 12, Hk=1 << 12, Sq=1, Sk=1),
    dict(B=1 << 23, Hq=2, Hk=1, Sq=100, Sk=1),           # two workgroups of 128 rows each
    dict(B=1 << 22, Hq=1, Hk=1, Sq=385, Sk=1),
], ids=str)
def test_attention_launches_hold_fewer_than_32_bits_of_threads(sizes):
    assert fwd(sizes) == -3 and bwd(sizes) == -3
    assert _lib.load().sparton_attention_workspace_bytes(desc(**sizes)) == 0
    assert _lib.load().sparton_attention_bwd_workspace_bytes(desc(**sizes)) == 0


def test_attention_backward_launches_over_keys():
    """dk and dv take a workgroup for 128 keys, where the forward walks any number of keys in one."""
    d = dict(B=1 << 22, Hq=1, Hk=1, Sq=1, Sk=385)
    assert bwd(d) == -3 and _lib.load().sparton_attention_bwd_workspace_bytes(desc(**d)) == 0
    assert fwd(d, ws=None, q=P + 8) == -2                # accepted so far: the next check is what answers
    assert bwd(dict(d, Sk=384, B=(1 << 22) + ((1 << 22) - 1) // 3), q=P + 8) == -2


@pytest.mark.parametrize("sizes", [
    dict(B=MOST, Hq=1, Hk=1, Sq=1, Sk=1), dict(B=MOST, Hq=1, Hk=1, Sq=32, Sk=128),
    dict(B=1, Hq=1, Hk=1, Sq=1 << 29, Sk=1), dict(B=1, Hq=1, Hk=1, Sq=1, Sk=(1 << 30) - 1),
], ids=str)
def test_attention_sizes_below_that_are_taken(sizes):
    assert fwd(sizes, q=P + 8) == -2 and bwd(sizes, q=P + 8) == -2


def test_attention_workspace():
    L = _lib.load()
    need = lambda **kw: L.sparton_attention_workspace_bytes(desc(**kw))
    assert need(B=32, Hq=12, Hk=12, Sq=256, Sk=256) == 0              # enough workgroups: no split
    # four rows to a key head against 20001 keys: splits of (D + 1) floats a row
    few = need(B=4, Hq=32, Hk=8, Sq=1, Sk=20001, D=128)
    assert few > 0 and few % (4 * 32 * 129 * 4) == 0 and few <= 64 * 4 * 32 * 129 * 4
    back = L.sparton_attention_bwd_workspace_bytes(desc(B=3, Hq=6, Hk=2, Sq=50))
    assert back == 3 * 6 * 50 * 4
    assert need(D=136) == 0 and need(B=0) == 0
    d = dict(B=4, Hq=32, Hk=8, Sq=1, Sk=20001, D=128)
    assert fwd(d, ws=None) == -4 and fwd(d, ws_bytes=few - 1) == -4 and fwd(d, ws=P + 16) == -2


def attention_kernels(B, Hq, Hk, Sq, Sk, D, dt, *_):
    """The kernels that a training step of these sizes launches: (kernel, type, head block, rows or keys of a
    workgroup, split). The rules of sparton_attention.hip once more."""
    cdiv, es, pairs, R = lambda a, b: -(-a // b), 4 if dt == "fp32" else 2, B * Hk, Hq // Hk * Sq
    block = 32 if D <= 32 else 64 if D <= 64 else 128
    small = lambda n: pairs * cdiv(n, 128) < (512 if es == 4 else 200)
    rows = 32 if R <= 32 else 64 if small(R) and (es == 4 or Sk <= 2048) else 128
    groups, tiles = pairs * cdiv(R, rows), cdiv(Sk, 128 if rows == 32 else 64 if rows == 64 or block <= 64 else 32)
    n = 1 if groups >= 192 else min(cdiv(512, groups), max(tiles // 4, 1), 64)
    return {("fwd", dt, block, rows, cdiv(tiles, cdiv(tiles, n)) > 1), ("dq", dt, block, 64 if small(R) else 128),
            ("dkv", dt, block, 64 if small(Sk) else 128)}


def test_the_attention_cases_reach_every_kernel():
    from test_gpu_attention import EVERY
    every = {(k, dt, block, n) for k in ("dq", "dkv") for dt in ("bf16", "fp16", "fp32") for block in (32, 64, 128)
             for n in (64, 128)}
    every |= {("fwd", dt, block, rows, split) for dt in ("bf16", "fp16", "fp32") for block in (32, 64, 128)
              for rows in (32, 64, 128) for split in (False, True)}
    # fp32 has 128 rows a workgroup only where workgroups are too many to be split
    every -= {("fwd", "fp32", block, 128, True) for block in (32, 64, 128)}
    assert set().union(*(attention_kernels(*c) for c in EVERY)) == every


def test_the_rules_above_are_the_librarys():
    """The workspace tells which forward calls are split, and over how many workgroups."""
    from test_gpu_attention import CASES, EVERY, FEW
    for B, Hq, Hk, Sq, Sk, D, dt, *_ in [*CASES, *EVERY, *FEW]:
        D += -D % (4 if dt == "fp32" else 8)
        need = _lib.load().sparton_attention_workspace_bytes(
            desc(B=B, Hq=Hq, Hk=Hk, Sq=Sq, Sk=Sk, D=D, dtype=("fp32", "bf16", "fp16").index(dt)))
        (split,) = (k[4] for k in attention_kernels(B, Hq, Hk, Sq, Sk, D, dt) if k[0] == "fwd")
        assert (need > 0) == split, (B, Hq, Hk, Sq, Sk, D, dt)


def q4(B=2, H=4, S=8, D=64, **kw):
    return torch.zeros(B, H, S, D, **kw)


@pytest.mark.parametrize("args,kw,error", [
    ((q4()[0], q4(), q4()), {}, ValueError),                                    # rank
    ((q4(), q4(H=2), q4(H=4)), {}, ValueError),                                 # k and v differ
    ((q4(), q4(H=3), q4(H=3)), {}, ValueError),                                 # heads not shared evenly
    ((q4(), q4(B=3), q4(B=3)), {}, ValueError),
    ((q4(), q4(D=32), q4(D=32)), {}, ValueError),
    ((q4(D=136), q4(D=136), q4(D=136)), {}, ValueError),                        # head too wide
    ((q4(), q4(), q4().half()), {}, TypeError),
    ((q4().double(), q4().double(), q4().double()), {}, TypeError),
    ((q4(), q4(), q4(), torch.ones(2, 9)), {}, ValueError),                     # mask shape
    ((q4(), q4(), q4(), torch.ones(2, 8)), {}, TypeError),                      # a float mask says two things
    ((q4(), q4(), q4(), torch.ones(2, 8, dtype=torch.int16)), {}, TypeError),
    ((q4(), q4(), q4()), dict(scale=0.0), ValueError),
    ((q4(), q4(), q4()), dict(scale=-0.1), ValueError),
    ((q4(), q4(), q4()), dict(scale=float("nan")), ValueError),
    ((q4(), q4(), q4()), {}, RuntimeError),                                     # CPU tensors
    ((q4(), q4(), q4(), torch.ones(2, 8, dtype=torch.int64)), dict(causal=True), RuntimeError),
])
def test_attention_refusals(args, kw, error):
    with pytest.raises(error):
        attention(*args, **kw)


@pytest.mark.parametrize("q", [q4(D=0), torch.zeros(()), torch.zeros(3, 0)], ids=["empty heads", "0-d", "2-d"])
def test_attention_default_scale_of_other_shapes(q):
    with pytest.raises(ValueError, match="attention"):
        attention(q, q, q)


def nfwd(**kw):
    a = dict(x=P, r=P, w=P, b=P, vec=0, eps=1e-5, y=P, mean=P, rstd=P, M=4, D=64, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_layer_norm_fwd(*a.values())


def nbwd(**kw):
    a = dict(dy=P, x=P, r=P, w=P, vec=0, mean=P, rstd=P, dx=P, dw=P, db=P, ws=P, ws_bytes=1 << 30, M=4, D=64, dtype=1,
             stream=None)
    a.update(kw)
    return _lib.load().sparton_layer_norm_bwd(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(D=0), -1), (dict(dtype=3), -1), (dict(vec=2), -1), (dict(x=None), -1), (dict(w=None), -1),
    (dict(y=None), -1), (dict(mean=None), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
    (dict(eps=float("inf")), -1), (dict(D=16385), -3), (dict(M=1 << 60), -3), (dict(x=P + 1), -2), (dict(w=P + 2), -2),
    (dict(M=0), 0), (dict(vec=1, w=P + 1), -2),
])
def test_layer_norm_fwd_checks(kw, code):
    assert nfwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -1), (dict(dtype=-1), -1), (dict(vec=2), -1), (dict(dy=None), -1), (dict(dx=None), -1),
    (dict(mean=None), -1), (dict(D=20000), -3), (dict(ws=None), -4), (dict(ws_bytes=8), -4), (dict(ws=P + 16), -2),
    (dict(dy=P + 1), -2), (dict(dw=P + 2), -2), (dict(M=0, dw=None, db=None), 0),
])
def test_layer_norm_bwd_checks(kw, code):
    assert nbwd(**kw) == code


def test_layer_norm_workspace():
    size = _lib.load().sparton_layer_norm_workspace_bytes
    assert size(0, 64) == 0 and size(5, 0) == 0 and size(5, 20000) == 0
    assert size(1, 768) == 2 * 768 * 4                    # one workgroup's column sums
    assert size(10 ** 9, 4096) <= 512 * 2 * 4096 * 4      # bounded however many rows


@pytest.mark.parametrize("args,kw,error", [
    ((torch.zeros(3, 8).double(), torch.ones(8).double()), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(9)), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8).half()), {}, ValueError),
    ((torch.zeros(3, 8).half(), torch.ones(8), torch.ones(8).half()), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8), torch.ones(7)), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8)), dict(residual=torch.zeros(8)), ValueError),   # no broadcast
    ((torch.zeros(3, 8), torch.ones(8)), dict(residual=torch.zeros(3, 8).half()), ValueError),
    ((torch.zeros(3, 8), torch.ones(8)), dict(eps=-1e-5), ValueError),
    ((torch.zeros(3, 0), torch.ones(0)), {}, ValueError),
    ((torch.zeros(3, 16385), torch.ones(16385)), {}, ValueError),
    ((torch.zeros(3, 8), torch.ones(8)), {}, RuntimeError),
])
def test_layer_norm_refusals(args, kw, error):
    with pytest.raises(error):
        layer_norm(*args, **kw)


def test_layer_norm_module_surface():
    ln = torch.nn.LayerNorm(32, eps=1e-7)
    m = SpartonLayerNorm.of(ln)
    assert m.weight is ln.weight and m.bias is ln.bias and m.eps == ln.eps and isinstance(m, torch.nn.LayerNorm)
    assert list(m.state_dict()) == list(ln.state_dict())
    for bad in (torch.nn.LayerNorm((4, 8)), torch.nn.LayerNorm(32, elementwise_affine=False), torch.nn.LayerNorm(16400)):
        with pytest.raises(ValueError):
            SpartonLayerNorm.of(bad)
    with pytest.raises(RuntimeError, match="ROCm/HIP device"):
        m(torch.zeros(2, 32))
    assert SpartonLayerNorm(16).weight.shape == (16,)
    assert sparton_amd.SpartonLayerNorm is SpartonLayerNorm


def test_layer_norm_module_needs_its_weight():
    for bad in (dict(elementwise_affine=False), dict(normalized_shape=(4, 8)), dict(normalized_shape=16400)):
        with pytest.raises(ValueError, match="SpartonLayerNorm"):
            SpartonLayerNorm(**{"normalized_shape": 16, **bad})
    assert SpartonLayerNorm(16, bias=False).bias is None


def pfwd(**kw):
    a = dict(q=P, p=P, n=P, ref=P, B=4, V=100, T=1.0, beta=1.0, eps=0.0, loss=P, margin=P, coef=P, ws=P,
             ws_bytes=1 << 30, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_preference_fwd(*a.values())


def pbwd(**kw):
    a = dict(q=P, p=P, n=P, coef=P, g=P, B=4, V=100, dq=P, dp=P, dn=P, dtype=1, stream=None)
    a.update(kw)
    return _lib.load().sparton_preference_bwd(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), -1), (dict(V=0), -1), (dict(dtype=3), -1), (dict(T=0.0), -1), (dict(T=float("nan")), -1),
    (dict(T=float("inf")), -1), (dict(beta=0.0), -1), (dict(beta=float("inf")), -1), (dict(eps=-0.1), -1),
    (dict(eps=0.6), -1), (dict(eps=float("nan")), -1), (dict(q=None), -1), (dict(margin=None), -1),
    (dict(loss=None), -1), (dict(coef=None), -1), (dict(B=1 << 30), -3), (dict(V=1 << 31), -3), (dict(q=P + 1), -2),
    (dict(ref=P + 2), -2), (dict(ws=None), -4), (dict(ws_bytes=4), -4), (dict(ws=P + 4), -2),
])
def test_preference_fwd_checks(kw, code):
    assert pfwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), -1), (dict(dtype=-1), -1), (dict(coef=None), -1), (dict(g=None), -1), (dict(dn=None), -1),
    (dict(V=1 << 31), -3), (dict(dq=P + 1), -2), (dict(g=P + 2), -2),
])
def test_preference_bwd_checks(kw, code):
    assert pbwd(**kw) == code


def test_preference_launches_hold_fewer_than_32_bits_of_threads():
    size = _lib.load().sparton_preference_workspace_bytes
    for B in (MOST + 1, (1 << 25) - 1):
        assert pfwd(B=B) == -3 and pbwd(B=B) == -3 and size(B, 100, 1) == 0
    assert pfwd(B=MOST, q=P + 1) == -2 and pbwd(B=MOST, q=P + 1) == -2
    assert size(MOST, 100, 1) == MOST * 4


def test_preference_workspace():
    size = _lib.load().sparton_preference_workspace_bytes
    assert size(0, 10, 1) == 0 and size(4, 0, 1) == 0 and size(4, 10, 9) == 0
    assert size(5000, 30522, 1) == 5000 * 4       # a row a workgroup
    assert size(1, 250002, 1) <= 64 * 4


R = torch.zeros(4, 10)


@pytest.mark.parametrize("args,kw,error", [
    ((R[0], R[0], R[0]), {}, ValueError),
    ((R, R[:3], R), {}, ValueError),
    ((R, R, R.half()), {}, ValueError),
    ((R.long(), R.long(), R.long()), {}, ValueError),
    ((R[:0], R[:0], R[:0]), {}, ValueError),
    ((R, R, R, torch.zeros(3)), {}, ValueError),
    ((R, R, R, torch.zeros(4).half()), {}, ValueError),
    ((R, R, R, torch.zeros(4, requires_grad=True)), {}, ValueError),   # the reference model is frozen
    ((R, R, R), dict(temperature=0.0), ValueError),
    ((R, R, R), dict(beta=-1.0), ValueError),
    ((R, R, R), dict(label_smoothing=0.7), ValueError),
    ((R, R, R), dict(label_smoothing=float("nan")), ValueError),
    ((R, R, R), {}, RuntimeError),
])
def test_preference_refusals(args, kw, error):
    with pytest.raises(error):
        preference_loss(*args, **kw)


def test_preference_margin_refuses_cpu():
    with pytest.raises(RuntimeError, match="ROCm/HIP device"):
        preference_margin(R, R, R)


def test_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty(2, 4, 8, 64, dtype=torch.bfloat16)
        k = torch.empty(2, 2, 16, 64, dtype=torch.bfloat16)
        out, lse = torch.ops.sparton.attention_fwd(q, k, k, None, False, 0.125)
        assert out.shape == q.shape and out.transpose(1, 2).is_contiguous() and lse.shape == (2, 4, 8)
        dq, dk, dv = torch.ops.sparton.attention_bwd(out, q, k, k, None, out, lse, False, 0.125)
        assert dq.shape == q.shape and dk.shape == k.shape == dv.shape and dk.dtype == torch.bfloat16
        x, w = torch.empty(3, 5, 32, dtype=torch.float16), torch.empty(32)
        y, mean, rstd = torch.ops.sparton.layer_norm_fwd(x, x, w, w, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == (15,) == rstd.shape
        dx, dw, db = torch.ops.sparton.layer_norm_bwd(y, x, x, w, True, mean, rstd)
        assert dx.dtype == x.dtype and dw.shape == (32,) == db.shape and dw.dtype == torch.float32
        r = torch.empty(4, 10, dtype=torch.bfloat16)
        loss, margin, coef = torch.ops.sparton.preference_fwd(r, r, r, None, 1.0, 1.0, 0.0)
        assert loss.shape == () and margin.shape == (4,) == coef.shape and loss.dtype == torch.float32
        assert all(g.shape == r.shape and g.dtype == r.dtype
                   for g in torch.ops.sparton.preference_bwd(loss, r, r, r, coef))
