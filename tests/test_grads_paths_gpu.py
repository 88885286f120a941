"""The gradient operators at the sizes where their launches change: one cluster,
two launches, a fold between, a cluster's fold, more than a wave of tickets.

Norms are held to the tolerances that test_grads_gpu derives; a clip has the
bits of the f32 product with the scale that the call reports, in every element.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_grads_gpu import DTYPES, IDS, NORMS, assert_norm
from tikun_b200 import (GradTable, _native, accumulate_grads_, clip_grad_norm_, clip_scale,
                        grad_norm)

pytestmark = pytest.mark.gpu

F32 = torch.float32


def tile_elements(dtype):
    return 8192 if dtype == F32 else 16384


def table_of(dtype, tiles, seed):
    """One buffer of `tiles` tiles as three tensors, the last two off a unit's start."""
    per = tile_elements(dtype)
    a = max(1, tiles // 3)
    sizes = [a * per, 5, (tiles - a - 1) * per - 13]
    flat = torch.empty(sum(sizes), dtype=dtype, device="cuda")
    fill(flat, seed)
    return flat, list(flat.split(sizes))


def fill(flat, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    flat.normal_(0.0, 0.5 if flat.dtype == torch.float16 else 1e-3, generator=gen)


def norm64(flat, p):
    parts = [x.double().abs() for x in flat.split(1 << 25)]
    if p == math.inf:
        return max(x.max().item() for x in parts)
    total = math.fsum((x * x if p == 2.0 else x).sum().item() for x in parts)
    return math.sqrt(total) if p == 2.0 else total


def same(a, b):
    i = torch.int32 if a.dtype == F32 else torch.int16
    return a.dtype == b.dtype and torch.equal(a.view(i), b.view(i))


def scaled(flat, scale):
    return (flat.float() * scale).to(flat.dtype)


def clip_scale_of(norm, max_norm):
    norm, max_norm = np.float32(norm), np.float32(max_norm)
    return float(max_norm / (norm + np.float32(1e-6))) if norm > max_norm else 1.0


def call(fn, table, p, max_norm, res, ws):
    code = {2.0: 0, 1.0: 1, math.inf: 2}[p]
    _native.check(getattr(_native.lib(), fn)(
        table._handle, code, max_norm, res[0:].data_ptr(), res[1:].data_ptr(),
        ws.data_ptr() if ws is not None else None, torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("mixed", [False, True], ids=["one-type", "two-types"])
@pytest.mark.parametrize("start", [0, 1, 6, 15])
def test_the_scale_shares_no_line_with_the_partials(start, mixed):
    """A clip's scale is written while other CTAs read partials, so neither it
    nor the tickets may lie on a 128-byte line with one."""
    ts = table_of(F32, 1203 if not mixed else 5, 0)[1]
    if mixed:
        ts += table_of(torch.bfloat16, 4, 1)[1]
    table = GradTable(ts)
    words = table._scratch_each // 8
    buf = torch.full((start + words + 32,), 7.0, dtype=torch.float64, device="cuda")
    assert buf.data_ptr() % 128 == 0
    res = torch.zeros(2, device="cuda")
    call("tk_clip_grad_norm", table, 2.0, 1e-3, res, buf[start:])
    changed = (buf.view(torch.int64) != torch.tensor(7.0, dtype=torch.float64).view(torch.int64).item())
    at = changed.nonzero().flatten().tolist()
    assert at[0] == start and at[-1] < start + words
    end = next(i for i, x in enumerate(at) if x != start + i)  # behind the partials
    assert end == (1203 if not mixed else 9)
    assert all(x // 16 != at[end - 1] // 16 for x in at[end:])
    assert buf[at[end]:].view(F32)[0].item() == res[1].item() < 1.0


def test_each_call_scales_by_its_own_scale():
    """Clips of more than 8192 slots (a cluster's fold) and then less work with
    one workspace and another scale each time."""
    for tiles in (8197, 1201):
        flat, ts = table_of(F32, tiles, 2)
        out = torch.empty_like(flat)
        table = GradTable(ts, out=list(out.split([t.numel() for t in ts])))
        ws = torch.empty(table._scratch // 8, dtype=torch.float64, device="cuda")
        res = torch.zeros(2, device="cuda")
        norm = norm64(flat, 2.0)
        for k in range(12):
            call("tk_clip_grad_norm", table, 2.0, norm * (0.9 - 0.07 * k), res, ws)
            assert res[1].item() < 1.0 - 0.05 * k
            assert same(out, scaled(flat, res[1]))


@pytest.mark.parametrize("n", [1, 64, 320, 321, 400, 961, 2000])
def test_tables_of_empty_tensors_only(n):
    """As a rank may have whose shards are all empty: a norm of 0, nothing to scale."""
    ts = [torch.empty(0, dtype=DTYPES[i % 3] if n == 64 else F32, device="cuda") for i in range(n)]
    table = GradTable(ts, out=[torch.empty(0, device="cuda") for _ in ts])
    for p in NORMS:
        norm, each = grad_norm(ts, norm_type=p, per_tensor=True)
        assert norm.item() == 0.0 and each.shape == (n,) and (each == 0.0).all()
        for got in (grad_norm(ts, norm_type=p), clip_grad_norm_(ts, 1.0, norm_type=p),
                    clip_grad_norm_(table, 1.0, norm_type=p),
                    accumulate_grads_(table, norm_type=p)):
            assert got.item() == 0.0
        norm, scale = clip_scale(ts, 1.0, norm_type=p)
        assert norm.item() == 0.0 and scale.item() == 1.0
    accumulate_grads_(table)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = clip_grad_norm_(ts, 1.0)
        norm, each = grad_norm(ts, per_tensor=True)
    for x in (norm, each):
        x.fill_(7.0)
    g.replay()
    assert norm.item() == 0.0 and (each == 0.0).all()
