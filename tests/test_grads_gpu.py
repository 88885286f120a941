"""The gradient operators (tikun_b200.grads) against plain 64-bit forms.

Tolerances, from the roundings that each operator makes (u = 2^-24, half a step
of f32):

* norm: f32 elements are squared exactly and summed in f64, so that only the
  last rounding to f32 is left: u.  bf16 and f16 elements are first added by
  eights in f32 as two chains of four and their sum, at most four roundings on
  the way of each value, which is 4 u of an L1 norm and half of that of an L2
  norm: 5 u with the last one.  The largest magnitude is exact.
* clipping: given the norm, scale and products are separately rounded f32
  operations: equal bits.
* the sum over micro-batches: one f32 rounding of alpha * g + acc: u, and half
  of the smallest subnormal.  (The 64-bit form rounds once before, which the
  factor 1.001 covers.)
"""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import tikun_b200
from tikun_b200 import GradTable, _native, accumulate_grads_, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
NORMS = [2.0, 1.0, math.inf]


def tensors(sizes, dtype, seed=0, offsets=(0,), std=None):
    """Tensors of one buffer each, the first element `offset` elements into it."""
    gen = torch.Generator().manual_seed(seed)
    std = std if std is not None else (0.5 if dtype == torch.float16 else 1e-3)
    out = []
    for i, n in enumerate(sizes):
        off = offsets[i % len(offsets)]
        buf = torch.zeros(off + n + 9, dtype=dtype, device="cuda")
        buf[off:off + n] = (torch.randn(n, generator=gen) * std).to(dtype)
        out.append(buf[off:off + n])
    return out


def norm64(ts, p):
    vals = [t.detach().double().abs().cpu().reshape(-1) for t in ts if t.numel()]
    if not vals:
        return 0.0
    v = torch.cat(vals)
    if torch.isnan(v).any():
        return math.nan
    if p == math.inf:
        return v.max().item()
    return math.sqrt((v * v).sum().item()) if p == 2.0 else v.sum().item()


def assert_norm(got, want, dtype, p):
    got = got.item() if isinstance(got, torch.Tensor) else got
    if math.isnan(want) or math.isinf(want) or p == math.inf:
        assert got == want or (math.isnan(got) and math.isnan(want)), (got, want)
        return
    tol = (1 if dtype == torch.float32 else 5) * U * 1.001
    assert abs(got - want) <= tol * want + 2.0 ** -150, (got, want, abs(got - want) / max(want, 1e-300))


def clip_bits(g, norm, max_norm, dtype):
    """The clipped gradient from the norm that the call returned, in f32 steps."""
    norm = np.float32(norm.item())
    scale = np.float32(1)
    if norm > np.float32(max_norm):
        with np.errstate(all="ignore"):
            scale = np.float32(max_norm) / (norm + np.float32(1e-6))
    return (g.detach().cpu().float() * torch.tensor(scale)).to(dtype)


def same_bits(a, b):
    a, b = a.detach().cpu(), b.detach().cpu()
    assert a.dtype == b.dtype and a.shape == b.shape
    i = torch.int32 if a.dtype == torch.float32 else torch.int16
    nan = torch.isnan(a) & torch.isnan(b)
    return bool(((a.view(i) == b.view(i)) | nan).all())


SIZES = {
    "none": [],
    "empty": [0, 0],
    "one": [1],
    "tiny": [1, 0, 7, 8, 9, 0],
    "unit-edges": list(range(1, 26)),
    "block-edges": [2047, 2048, 2049, 4097, 256, 65536],
    "uneven": [1_000_003, 3, 17, 250_000, 1],
    "many-small": [(i * 37) % 97 for i in range(700)],
    "three-launches": [(i * 53) % 211 for i in range(2100)],
    "big-and-small": [5_000_011] + [768] * 40 + [2_000_000],
}


@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_norm(sizes, dtype, p):
    ts = tensors(sizes, dtype, offsets=(0, 1, 5, 0, 3))
    got, each = grad_norm(ts, norm_type=p, per_tensor=True)
    assert got.shape == () and got.dtype == torch.float32 and each.shape == (len(ts),)
    assert_norm(got, norm64(ts, p), dtype, p)
    assert_norm(grad_norm(ts, norm_type=p), norm64(ts, p), dtype, p)
    for t, e in zip(ts, each.tolist()):
        assert_norm(e, norm64([t], p), dtype, p)


@pytest.mark.parametrize("target", ["in-place", "f32", "bf16", "f16"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_clip(sizes, dtype, target):
    ts = tensors(sizes, dtype, offsets=(0, 1, 5, 0, 3))
    before = [t.clone() for t in ts]
    want = norm64(ts, 2.0)
    odt = dtype if target == "in-place" else dict(zip(IDS, DTYPES))[target]
    for max_norm in (want * 0.3 + 1e-9, want * 3 + 1e-9):
        for t, b in zip(ts, before):
            t.copy_(b)
        # out in phase with its gradient, and not
        outs = None if target == "in-place" else tensors(sizes, odt, seed=1, offsets=(0, 1, 4, 2, 3))
        norm = clip_grad_norm_(ts, max_norm, out=outs)
        assert_norm(norm, want, dtype, 2.0)
        for b, t, o in zip(before, ts, outs or ts):
            assert same_bits(o, clip_bits(b, norm, max_norm, odt))
            if outs is not None:
                assert same_bits(t, b)


@pytest.mark.parametrize("p", NORMS)
def test_clip_by_other_norms(p):
    ts = tensors([70_001, 33, 8], torch.bfloat16)
    before = [t.clone() for t in ts]
    max_norm = 0.5 * norm64(ts, p)
    norm = clip_grad_norm_(ts, max_norm, norm_type=p)
    assert_norm(norm, norm64(before, p), torch.bfloat16, p)
    for b, t in zip(before, ts):
        assert same_bits(t, clip_bits(b, norm, max_norm, torch.bfloat16))


def test_what_lies_around_the_tensors_stays():
    """Nothing outside the elements is written, at any start and length of a unit."""
    for dtype in DTYPES:
        for off in range(9):
            for n in (1, 6, 8, 9, 17, 4099):
                buf = torch.full((off + n + 16,), 2.0, dtype=dtype, device="cuda")
                acc = torch.full((off + n + 16,), 3.0, device="cuda")
                g = buf[off:off + n]
                accumulate_grads_([g], [acc[off:off + n]], alpha=0.5)
                clip_grad_norm_([g], 1e-3)
                for t, v in ((buf, 2.0), (acc, 3.0)):
                    assert (t[:off] == v).all() and (t[off + n:] == v).all()
                assert (acc[off:off + n] == 4.0).all() and (g < 1.0).all()


@pytest.mark.parametrize("p", [None] + NORMS)
@pytest.mark.parametrize("overwrite", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_accumulate(sizes, dtype, overwrite, p):
    ts = tensors(sizes, dtype, offsets=(0, 1, 5, 0, 3))
    acc = tensors(sizes, torch.float32, seed=2, offsets=(0, 1, 4, 2, 3))
    alpha = 0.3
    want = [np.float32(alpha).item() * t.double() + (0 if overwrite else a.double())
            for t, a in zip(ts, acc)]
    norm = accumulate_grads_(ts, acc, alpha=alpha, overwrite=overwrite, norm_type=p)
    for a, w in zip(acc, want):
        err = (a.double() - w).abs()
        assert (err <= U * 1.001 * w.abs() + 2.0 ** -150).all()
    if p is None:
        assert norm is None
    else:
        assert_norm(norm, norm64(acc, p), torch.float32, p)


def test_types_mixed_in_one_call():
    ts = [t for d in DTYPES for t in tensors([1000, 3, 70_000], d, std=0.25)]
    outs = [torch.empty_like(t, dtype=d) for t, d in zip(ts, DTYPES * 3)]
    got, each = grad_norm(ts, per_tensor=True)
    assert_norm(got, norm64(ts, 2.0), torch.bfloat16, 2.0)
    for t, e in zip(ts, each.tolist()):
        assert_norm(e, norm64([t], 2.0), t.dtype, 2.0)
    norm = clip_grad_norm_(ts, 1.0, out=outs)
    assert same_bits(norm, got)
    for t, o in zip(ts, outs):
        assert same_bits(o, clip_bits(t, norm, 1.0, o.dtype))
    before = [t.clone() for t in ts]
    assert same_bits(clip_grad_norm_(ts, 1.0), norm)
    for t, b in zip(ts, before):
        assert same_bits(t, clip_bits(b, norm, 1.0, t.dtype))


@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("value", ["large", "small", "subnormal", "mixed", "zeros", "inf", "-inf", "nan"])
def test_values_at_the_ends_of_the_range(value, dtype, p):
    info = torch.finfo(dtype)
    n = 5003
    x = torch.zeros(n, dtype=torch.float64)
    if value == "large":  # squares, and sums of f32, overflow f32
        x[:] = info.max
    elif value == "small":  # squares underflow f32
        x[:] = info.tiny * 3
    elif value == "subnormal":
        x[:] = info.smallest_normal * info.eps * 5
    elif value == "mixed":  # eights of both kinds, and some whose squares underflow beside ones
        x[:] = 1e-30
        x[5::64] = -info.max / 4
        x[2::40] = 1.0
    elif value != "zeros":
        x[:] = 0.5
        x[n // 2] = float(value)
    t = x.to(dtype).cuda()
    ts = [t[:2000], t[2000:2001], t[2001:]]
    got, each = grad_norm(ts, norm_type=p, per_tensor=True)
    assert_norm(got, f32_range(norm64(ts, p)), dtype, p)
    for s, e in zip(ts, each.tolist()):
        assert_norm(e, f32_range(norm64([s], p)), dtype, p)


def f32_range(v):
    """A norm above f32's range is infinity."""
    return math.inf if v >= 2.0 ** 128 else v


@pytest.mark.parametrize("value", ["inf", "nan"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_clip_of_non_finite_gradients(dtype, value):
    """A NaN norm leaves the gradients, an infinite one scales them by 0."""
    ts = tensors([1000, 50], dtype)
    ts[1][7] = float(value)
    before = [t.clone() for t in ts]
    with pytest.raises(RuntimeError, match="norm of order 2.0 is " + value):
        clip_grad_norm_(ts, 1.0, error_if_nonfinite=True)
    assert all(same_bits(t, b) for t, b in zip(ts, before))
    with pytest.raises(RuntimeError, match="is " + value):
        grad_norm(ts, error_if_nonfinite=True)
    norm = clip_grad_norm_(ts, 1.0)
    for b, t in zip(before, ts):
        assert same_bits(t, clip_bits(b, norm, 1.0, dtype))
    if value == "inf":
        assert (ts[0] == 0).all() and math.isnan(ts[1][7].item())


def test_equal_inputs_give_equal_bits():
    for dtype in DTYPES:
        ts = tensors([3_000_001, 77, 1_000_000], dtype)
        a = [grad_norm(ts, norm_type=p, per_tensor=True) for p in NORMS]
        b = [grad_norm(ts, norm_type=p, per_tensor=True) for p in NORMS]
        for (x, xe), (y, ye) in zip(a, b):
            assert same_bits(x, y) and same_bits(xe, ye)


def test_dense_views_in_other_orders():
    w = torch.randn(40, 70, device="cuda")
    g = w.t()  # a transposed weight's gradient
    assert not g.is_contiguous()
    assert_norm(grad_norm([g]), norm64([w], 2.0), torch.float32, 2.0)
    out = torch.empty_like(g, dtype=torch.bfloat16)  # keeps the strides
    assert out.stride() == g.stride()
    norm = clip_grad_norm_([g], 1.0, out=[out])
    assert same_bits(out, clip_bits(g, norm, 1.0, torch.bfloat16))
    with pytest.raises(ValueError, match="strides"):
        clip_grad_norm_([g], 1.0, out=[torch.empty(70, 40, device="cuda")])
    with pytest.raises(ValueError, match="lazily negated"):
        grad_norm([torch._neg_view(w)])
    for sparse in (w.to_sparse(), w.to_sparse_csr()):
        with pytest.raises(ValueError, match="dense CUDA tensor"):
            grad_norm([w, sparse])
    with pytest.raises(ValueError, match="dense CUDA tensor"):
        grad_norm([w, torch.empty(3, device="meta")])
    for bad in (w[:, ::2], w[:, 1:], torch.zeros(3, 1, device="cuda").expand(3, 4)):
        with pytest.raises(ValueError, match="one stretch of memory"):
            grad_norm([bad])


def test_refusals_with_device_tensors():
    a = torch.zeros(64, device="cuda")
    with pytest.raises(TypeError, match="float64"):
        grad_norm([a.double()])
    with pytest.raises(ValueError, match="1 out tensors for 2 gradients"):
        clip_grad_norm_([a, a.clone()], 1.0, out=[a.clone()])
    with pytest.raises(ValueError, match="out 0 has shape"):
        clip_grad_norm_([a], 1.0, out=[torch.zeros(63, device="cuda")])
    # twice the same tensor: counted twice by the norm, refused by the clip
    a += 1.0
    assert grad_norm([a, a]).item() == np.float32(math.sqrt(128.0))
    with pytest.raises(ValueError, match="shares memory"):
        clip_grad_norm_([a, a], 1.0)
    with pytest.raises(ValueError, match="shares memory"):
        clip_grad_norm_([a, a[8:9]], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        clip_grad_norm_([a[:32]], 1.0, out=[a[16:48]])
    assert (a == 1.0).all()
    # sums go into f32 buffers of their own
    for acc in (a, torch.zeros(64, device="cuda", dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="f32 out buffers of their own"):
            accumulate_grads_([a], [acc])
    with pytest.raises(ValueError, match="f32 out buffers of their own"):
        accumulate_grads_(GradTable([a]))
    with pytest.raises(ValueError, match="has its out tensors"):
        clip_grad_norm_(GradTable([a]), 1.0, out=[a])
    pinned = torch.zeros(8).pin_memory()
    arr = (_native.TkGrad * 1)(_native.TkGrad(pinned.data_ptr(), 0, 8, 0, 0))
    h = ctypes.c_void_p()
    with pytest.raises(ValueError, match="not device memory"):
        _native.check(_native.lib().tk_grad_table_create(arr, 1, ctypes.byref(h)))


@pytest.mark.parametrize("sizes", [[4097], [1_000_003, 5, 300_000]], ids=["small", "large"])
def test_workspace_of_the_caller_or_the_pool(sizes):
    """The C calls give the same bits with either, write nothing behind the
    bytes they ask for, and refuse what is not device memory."""
    L = _native.lib()
    ts = tensors(sizes, torch.bfloat16)
    acc = [torch.zeros(n, device="cuda") for n in sizes]
    t = GradTable(ts, out=acc)
    b, be = ctypes.c_uint64(), ctypes.c_uint64()
    _native.check(L.tk_grad_workspace(t._handle, ctypes.byref(b), ctypes.byref(be)))
    assert (b.value == 0) == (len(sizes) == 1) and be.value > 0 and be.value % 8 == 0
    s = torch.cuda.current_stream().cuda_stream
    got = []
    for with_ws in (False, True):
        res = torch.zeros(4 + len(sizes), device="cuda")
        at = [res[i:].data_ptr() for i in range(5)]
        ws = torch.full((be.value // 8 + 8,), 7.0, dtype=torch.float64, device="cuda")
        w = ws.data_ptr() if with_ws else None
        _native.check(L.tk_grad_norm(t._handle, 0, 0.5, at[0], at[4], at[1], w, s))
        _native.check(L.tk_clip_grad_norm(t._handle, 1, 0.5, at[2], None, w, s))
        clipped = [a.clone() for a in acc]
        _native.check(L.tk_accumulate_grads(t._handle, 0.5, 1, 2, at[3], w, s))
        assert (ws[be.value // 8:] == 7.0).all()
        got.append([res] + clipped + [a.clone() for a in acc])
    for x, y in zip(*got):
        assert same_bits(x, y)
    host = torch.zeros(8, dtype=torch.float64)
    pinned = torch.zeros(8, dtype=torch.float64).pin_memory()
    dev = torch.zeros(8, dtype=torch.float64, device="cuda")
    for bad in (host.data_ptr(), pinned.data_ptr(), dev.data_ptr() + 4):
        with pytest.raises(ValueError, match="for a workspace"):
            _native.check(L.tk_grad_norm(t._handle, 0, 0.0, dev.data_ptr(), None, None, bad, s))
    for bad in (host.data_ptr(), pinned.data_ptr(), dev.data_ptr() + 2):
        for args in ((bad, None, None), (None, bad, None), (None, None, bad)):
            with pytest.raises(ValueError, match="for a result"):
                _native.check(L.tk_grad_norm(t._handle, 0, 0.0, *args, None, s))
        with pytest.raises(ValueError, match="for a result"):
            _native.check(L.tk_clip_grad_norm(t._handle, 0, 1.0, bad, None, None, s))
        with pytest.raises(ValueError, match="for a result"):
            _native.check(L.tk_accumulate_grads(t._handle, 1.0, 1, 0, bad, None, s))
    with pytest.raises(ValueError, match="norm_dev is NULL"):
        _native.check(L.tk_accumulate_grads(t._handle, 1.0, 1, 0, None, None, s))
    for call in (lambda: L.tk_grad_norm(t._handle, 3, 0.0, None, None, None, None, s),
                 lambda: L.tk_grad_norm(t._handle, -1, 0.0, None, None, None, None, s),
                 lambda: L.tk_clip_grad_norm(t._handle, 7, 1.0, None, None, None, s),
                 lambda: L.tk_accumulate_grads(t._handle, 1.0, 1, 5, None, None, s)):
        with pytest.raises(ValueError, match="unknown norm"):
            _native.check(call())
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="is not positive"):
            _native.check(L.tk_clip_grad_norm(t._handle, 0, bad, None, None, None, s))


def test_parameters_stand_for_their_gradients():
    lin = torch.nn.Linear(33, 17, device="cuda")
    frozen = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    lin(torch.randn(8, 33, device="cuda")).square().sum().backward()
    want = norm64([p.grad for p in lin.parameters()], 2.0)
    table = GradTable({"a": list(lin.parameters()), "b": frozen, "c": None})
    assert len(table) == 2
    assert_norm(grad_norm(table), want, torch.float32, 2.0)
    assert_norm(grad_norm(lin.parameters()), want, torch.float32, 2.0)
    ref = [p.grad.clone() for p in lin.parameters()]
    norm = clip_grad_norm_(lin.parameters(), want / 2)
    for p, b in zip(lin.parameters(), ref):
        assert same_bits(p.grad, clip_bits(b, norm, want / 2, torch.float32))
    lin.zero_grad(set_to_none=True)
    with pytest.raises(RuntimeError, match="build the table anew"):
        grad_norm(table)
    assert grad_norm(lin.parameters()).item() == 0.0


def test_a_table_keeps_its_memory_and_is_not_copied():
    import copy
    import pickle

    g = torch.full((1 << 20,), 2.0, device="cuda")
    table = GradTable([g])
    g.data = torch.zeros(4, device="cuda")
    junk = [torch.full((1 << 20,), 9.0, device="cuda") for _ in range(4)]
    assert grad_norm(table, norm_type=1.0).item() == 2.0 * (1 << 20) and len(junk) == 4
    for dup in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="build another"):
            dup(table)
    p = torch.nn.Parameter(torch.zeros(1 << 20, device="cuda"))
    with pytest.raises(TypeError, match="not parameters"):
        GradTable(table.grads, out=[p])


def test_micro_batches_norm_clip_and_step_together():
    """Sum, norm, clip and an AdamW step that does not clip give the bits of the
    fused clipped step on the same sums; the clipped bf16 gradients, too, of
    the torch form of the whole path."""
    sizes = [4099, 768, 1, 250_000]
    parts = [tensors(sizes, torch.bfloat16, seed=s) for s in range(3)]
    acc = [torch.empty(n, device="cuda") for n in sizes]
    for k, gs in enumerate(parts):
        norm = accumulate_grads_(gs, acc, alpha=1 / 3, overwrite=k == 0,
                                 norm_type=2.0 if k == 2 else None)
    max_norm = 0.25 * norm.item()
    params = [torch.randn(n, device="cuda") * 0.02 for n in sizes]
    a = [torch.nn.Parameter(p.clone()) for p in params]
    b = [torch.nn.Parameter(p.clone()) for p in params]
    opt_a = tikun_b200.AdamW(a, max_norm=max_norm)
    opt_a.step([t.clone() for t in acc])
    low = [torch.empty_like(t, dtype=torch.bfloat16) for t in acc]
    clip_grad_norm_(acc, max_norm, out=low)
    again = clip_grad_norm_(acc, max_norm)
    assert same_bits(again, norm)
    opt_b = tikun_b200.AdamW(b)
    opt_b.step(acc)
    for x, y, t, l in zip(a, b, acc, low):
        assert same_bits(x, y)
        assert same_bits(l, t.to(torch.bfloat16))
    plain = [sum(np.float32(1 / 3).item() * gs[i].double() for gs in parts) for i in range(len(sizes))]
    n64 = math.sqrt(sum((x * x).sum().item() for x in plain))
    for x, t in zip(plain, acc):
        want = x * (max_norm / (n64 + 1e-6))
        # three sums, norm, scale (two roundings) and product
        assert ((t.double() - want).abs() <= 8 * U * x.abs().max() + 2.0 ** -149).all()


def muon_params(seed=3):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(256, 384), (384, 256), (96, 40), (3, 64, 32), (768,), (5,)]
    return [torch.randn(s, generator=gen).cuda() * 0.02 for s in shapes]


@pytest.mark.parametrize("over", [True, False], ids=["over", "under"])
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
def test_muon_nd_clips_by_the_common_norm(dtype, over):
    """Three clipped steps give the bits of steps on gradients multiplied by
    the scale in f32, which is what the norm of all leaves calls for."""
    a = [torch.nn.Parameter(t) for t in muon_params()]
    b = [torch.nn.Parameter(t.clone()) for t in muon_params()]
    opt_a = tikun_b200.MuonND(a, max_norm=0.01 if over else 100.0)
    opt_b = tikun_b200.MuonND(b)
    for step in range(3):
        gs = [t.to(dtype) * 0.1 for t in muon_params(seed=10 + step)]
        for p, g in zip(a, gs):
            p.grad_dtype = None  # it may have another type than its parameter
            p.grad = g
        opt_a.step()
        want = norm64(gs, 2.0)
        assert_norm(opt_a.grad_norm, want, dtype, 2.0)
        scale = opt_a.clip_scale.cpu()
        assert (scale.item() < 1.0) == over
        for p, g in zip(b, gs):
            p.grad = (g.cpu().float() * scale).cuda()
        opt_b.step()
        for x, y, g in zip(a, b, gs):
            assert same_bits(x, y)
            assert same_bits(x.grad, g)  # the gradients stay as they are


def test_muon_clips_its_two_groups_together():
    def build(**kw):
        ps = [torch.nn.Parameter(t) for t in muon_params()]
        return ps, tikun_b200.Muon(ps[:3], ps[4:], **kw)

    a, opt_a = build(max_norm=0.05)
    b, opt_b = build()
    c, opt_c = build()
    used = [0, 1, 2, 4, 5]
    for step in range(2):
        gs = [t * 0.1 for t in muon_params(seed=20 + step)]
        for i in used:
            a[i].grad, c[i].grad = gs[i].clone(), gs[i].clone()
        opt_a.step()
        assert_norm(opt_a.grad_norm, norm64([gs[i] for i in used], 2.0), torch.float32, 2.0)
        norm, scale = tikun_b200.clip_scale([gs[i] for i in used], 0.05)
        assert same_bits(norm, opt_a.grad_norm) and same_bits(scale, opt_a.clip_scale)
        assert scale.item() == (np.float32(0.05) / (np.float32(norm.item()) + np.float32(1e-6)))
        opt_c.step(clip_scale=scale)
        for i in used:
            b[i].grad = gs[i] * scale
        opt_b.step()
        for i in used:
            assert same_bits(a[i], b[i]) and same_bits(c[i], b[i])


@pytest.mark.parametrize("form", ["adamw", "lion", "sgd", "arena", "torch-adamw"])
def test_optimizers_take_a_common_scale(form):
    from tikun_b200.optimizer import AdamW as TorchAdamW

    def build(ts):
        ps = [torch.nn.Parameter(t.clone()) for t in ts]
        if form == "torch-adamw":
            return ps, TorchAdamW(ps)
        if form == "arena":
            return ps, tikun_b200.AdamW(ps, arena=True)
        return ps, tikun_b200.Optimizer(ps, algorithm=form)

    ts = muon_params()
    (a, opt_a), (b, opt_b) = build(ts), build(ts)
    other = torch.randn(1000, device="cuda")
    for step in range(2):
        gs = [t * 0.1 for t in muon_params(seed=30 + step)]
        norm, scale = tikun_b200.clip_scale([gs, other], 0.5)
        assert_norm(norm, norm64(gs + [other], 2.0), torch.float32, 2.0)
        assert scale.item() < 1.0
        for p, q, g in zip(a, b, gs):
            if form == "arena":
                p.grad.copy_(g)
                q.grad.copy_(g * scale)
            else:
                p.grad, q.grad = g, g * scale
        opt_a.step(clip_scale=scale)
        opt_b.step()
        for x, y in zip(a, b):
            assert same_bits(x, y)
    with pytest.raises(ValueError, match="one float32 value"):
        opt_a.step(clip_scale=scale.double())


def test_clip_scale_refusals():
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    p.grad = torch.ones(8, device="cuda")
    norm, scale = tikun_b200.clip_scale([p], 1.0)
    for opt in (tikun_b200.AdamW([p], max_norm=1.0), tikun_b200.MuonND([p], max_norm=1.0)):
        with pytest.raises(ValueError, match="forms its own clip scale"):
            opt.step(clip_scale=scale)
    with pytest.raises(ValueError, match="before a common norm is known"):
        tikun_b200.AdamW([p], in_backward=True).step(clip_scale=scale)
    w = np.zeros((4, 4), np.float32)
    leaf = (_native.TkMuonLeaf * 1)(_native.TkMuonLeaf(w.ctypes.data, w.ctypes.data + 16,
                                                      w.ctypes.data + 32, 1, 2, 2, 0, 0))
    hp = _native.TkMuonHParams(0.02, 0.95, 1, 5, _native.TK_NS_F16)
    L = _native.lib()
    for ptr, text in ((None, "scale_dev is NULL"), (scale.data_ptr(), "takes device buffers")):
        with pytest.raises(ValueError, match=text):
            _native.check(L.tk_muon_step_clipped(leaf, 1, ctypes.byref(hp), ptr, None))


def test_captured_calls_and_graphs_side_by_side():
    """Two captured graphs on two streams, replayed at once on new contents,
    beside eager calls on a third."""
    sizes = [100_003, 768, 5]
    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, state = [], []
    for k in range(2):
        ts = tensors(sizes, torch.bfloat16, seed=k)
        outs = [torch.empty_like(t, dtype=torch.float32) for t in ts]
        table = GradTable(ts, out=outs)
        clip_grad_norm_(table, 0.01)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[k]):
            norm = clip_grad_norm_(table, 0.01)
            total, each = grad_norm(ts, per_tensor=True)
        graphs.append(g)
        state.append((ts, outs, norm, total, each))
    eager = tensors(sizes, torch.float32, seed=9)
    for round_ in range(3):
        for k in range(2):
            for t, n in zip(state[k][0], tensors(sizes, torch.bfloat16, seed=10 * round_ + k)):
                t.copy_(n)
        torch.cuda.synchronize()
        for _ in range(4):
            for k in range(2):
                with torch.cuda.stream(side[k]):
                    graphs[k].replay()
            e = grad_norm(eager)
        torch.cuda.synchronize()
        assert_norm(e, norm64(eager, 2.0), torch.float32, 2.0)
        for ts, outs, norm, total, each in state:
            want = norm64(ts, 2.0)
            assert_norm(norm, want, torch.bfloat16, 2.0)
            assert same_bits(norm, total)
            for t, o, x in zip(ts, outs, each.tolist()):
                assert same_bits(o, clip_bits(t, norm, 0.01, torch.float32))
                assert_norm(x, norm64([t], 2.0), torch.bfloat16, 2.0)


@pytest.mark.parametrize("limit", [0.5, 2.0], ids=["over", "under"])
def test_captured_clip_in_place_replays(limit):
    """Every replay of a clip in place scales each element once."""
    sizes = [700_001, 768, 0, 1_300_000]
    ts = [t for d in DTYPES for t in tensors(sizes, d, offsets=(0, 3))]
    table = GradTable(ts)
    clip_grad_norm_(table, 1.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = clip_grad_norm_(table, limit)
    for round_ in range(3):
        fresh = [t for d in DTYPES for t in tensors(sizes, d, seed=round_, std=1.0 / 2400)]
        for t, f in zip(ts, fresh):
            t.copy_(f)
        g.replay()
        torch.cuda.synchronize()
        assert_norm(norm, norm64(fresh, 2.0), torch.bfloat16, 2.0)
        assert (norm.item() > limit) == (limit == 0.5)
        for t, f in zip(ts, fresh):
            assert same_bits(t, clip_bits(f, norm, limit, t.dtype))


def test_streams_and_threads():
    """Calls on a side stream order after that stream's work; threads share a table."""
    n = 3_000_000
    s = torch.cuda.Stream()
    g = torch.zeros(n, device="cuda")
    table = GradTable([g])
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            g.add_(1.0)
        norm = grad_norm(table, norm_type=1.0)
        g.zero_()
    s.synchronize()
    assert norm.item() == 20.0 * n
    g.fill_(2.0)
    torch.cuda.synchronize()
    got = [[] for _ in range(4)]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got[k].append(grad_norm(table, norm_type=[2.0, 1.0, math.inf, 2.0][k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    want = [np.float32(2.0 * math.sqrt(n)), 2.0 * n, 2.0, np.float32(2.0 * math.sqrt(n))]
    for k in range(4):
        assert len(got[k]) == 50 and all(x.item() == want[k] for x in got[k])


def test_more_than_two_to_the_32_elements():
    """Element offsets and byte offsets past 32 bits."""
    n = 2 ** 32 + 4099
    g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g[-1] = 3.0
    total, each = grad_norm([g[:5], g[5:]], norm_type=1.0, per_tensor=True)
    assert total.item() == np.float32(n + 2) and each[0].item() == 5.0
    assert grad_norm([g], norm_type=math.inf).item() == 3.0
    norm = clip_grad_norm_([g], 0.5 * n, norm_type=1.0)
    assert norm.item() == np.float32(n + 2)
    assert same_bits(g[-5000:], clip_bits(torch.cat([torch.ones(4999), torch.tensor([3.0])]).bfloat16(),
                                          norm, 0.5 * n, torch.bfloat16))
    assert same_bits(g[2 ** 31 - 8:2 ** 31 + 8], g[:16]) and same_bits(g[2 ** 32 - 8:2 ** 32 + 8], g[:16])
