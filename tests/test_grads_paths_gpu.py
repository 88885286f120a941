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


def tile_counts(dtype):
    """The one-cluster limit of units and one more, the limit of a fold in the scaling and
    one more, above 52 MB of tiles that stay in L2, and a fold by a cluster."""
    units = 32 if dtype == F32 else 16
    return [units, units + 1, 1200, 1201, 1700, 8300]


PATHS = [(d, t) for d in DTYPES for t in tile_counts(d)]
PATH_IDS = [f"{dict(zip(DTYPES, IDS))[d]}-{t}" for d, t in PATHS]


@pytest.mark.parametrize("limit", ["over", "under"])
@pytest.mark.parametrize("target", ["in-place", "out"])
@pytest.mark.parametrize("dtype,tiles", PATHS, ids=PATH_IDS)
def test_clip_on_each_path(dtype, tiles, target, limit):
    """Three calls on one table, each with fresh values, and every element compared."""
    p = NORMS[tiles % 3]
    flat, ts = table_of(dtype, tiles, 3)
    out = flat if target == "in-place" else torch.empty_like(flat)
    table = GradTable(ts, out=None if target == "in-place"
                      else list(out.split([t.numel() for t in ts])))
    for seed in range(3):
        fill(flat, seed)
        want = norm64(flat, p)
        before = flat.clone()
        max_norm = want * (0.3 if limit == "over" else 3.0)
        norm = clip_grad_norm_(table, max_norm, norm_type=p)
        assert_norm(norm, want, dtype, p)
        scale = clip_scale_of(norm.item(), max_norm)
        assert (scale < 1.0) == (limit == "over")
        assert same(out, scaled(before, torch.tensor(scale, device="cuda")))


@pytest.mark.parametrize("dtype,tiles", PATHS, ids=PATH_IDS)
def test_norm_and_sum_on_each_path(dtype, tiles):
    flat, ts = table_of(dtype, tiles, 4)
    sizes = [t.numel() for t in ts]
    acc = torch.randn(flat.numel(), device="cuda",
                      generator=torch.Generator(device="cuda").manual_seed(5))
    table = GradTable(ts, out=list(acc.split(sizes)))
    for p in NORMS:
        want = norm64(flat, p)
        norm, each = grad_norm(table, norm_type=p, per_tensor=True)
        assert_norm(norm, want, dtype, p)
        assert_norm(grad_norm(table, norm_type=p), want, dtype, p)
        for t, e in zip(ts, each.tolist()):
            assert_norm(e, norm64(t, p), dtype, p)
    for overwrite in (True, False):
        # a product with a power of two is exact: one rounding of the sum on either side
        plain = flat.float() * 0.5 + (0.0 if overwrite else acc)
        norm = accumulate_grads_(table, alpha=0.5, overwrite=overwrite, norm_type=2.0)
        assert torch.equal(acc, plain)
        assert_norm(norm, norm64(acc, 2.0), F32, 2.0)


@pytest.mark.parametrize("n", [96, 97])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_clip_of_many_small_tensors(dtype, n):
    """The one-cluster limit of tiles and one more."""
    flat = torch.empty(n * 777, dtype=dtype, device="cuda")
    fill(flat, 6)
    before, want = flat.clone(), norm64(flat, 2.0)
    norm = clip_grad_norm_(list(flat.split(777)), want / 3)
    assert_norm(norm, want, dtype, 2.0)
    assert same(flat, scaled(before, torch.tensor(clip_scale_of(norm.item(), want / 3), device="cuda")))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_captured_clips_over_a_wave_of_tickets(dtype):
    """Two graphs, in place and out of it, with scratch of their own, replayed
    at once on two streams with fresh values: every element scaled once."""
    parts = []
    for k in range(2):
        flat, ts = table_of(dtype, 1700, 7 + k)
        out = flat if k == 0 else torch.empty_like(flat)
        table = GradTable(ts, out=None if k == 0 else list(out.split([t.numel() for t in ts])))
        limit = 0.4 * norm64(flat, 2.0)
        stream = torch.cuda.Stream()
        clip_grad_norm_(table, 1e9)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            norm = clip_grad_norm_(table, limit)
        parts.append((flat, out, limit, stream, graph, norm))
    for seed in range(3):
        before = []
        for k, (flat, *_) in enumerate(parts):
            fill(flat, 20 * seed + k)
            before.append(flat.clone())
        torch.cuda.synchronize()
        for _, _, _, stream, graph, _ in parts:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for b, (_, out, limit, _, _, norm) in zip(before, parts):
            assert_norm(norm, norm64(b, 2.0), dtype, 2.0)
            scale = clip_scale_of(norm.item(), limit)
            assert scale < 1.0
            assert same(out, scaled(b, torch.tensor(scale, device="cuda")))
