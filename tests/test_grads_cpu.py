"""The gradient operators' refusals, which come before any launch: no GPU."""
import ctypes

import pytest
import torch

import tikun_b200
from tikun_b200 import _native, grads


def create(entries):
    """tk_grad_table_create over (g, out, n, g dtype, out dtype) tuples: status and message."""
    arr = (_native.TkGrad * max(len(entries), 1))()
    for i, e in enumerate(entries):
        arr[i] = _native.TkGrad(*e)
    h = ctypes.c_void_p()
    st = _native.lib().tk_grad_table_create(arr, len(entries), ctypes.byref(h))
    assert st != 0 and not h.value
    return st, _native.lib().tk_last_error().decode()


F32, BF16, F16 = _native.TK_F32, _native.TK_BF16, _native.TK_F16


@pytest.mark.parametrize("entries,text", [
    ([(0, 0, 4, F32, 0)], "gradient 0: g is NULL"),
    ([(64, 0, 4, F32, 0), (4096, 0, 4, 3, 0)], "gradient 1: g dtype 3 is not f32, bf16 or f16"),
    ([(64, 4096, 4, F32, -1)], "gradient 0: out dtype -1"),
    ([(66, 0, 4, F32, 0)], "not aligned to its element size"),
    ([(65, 0, 4, BF16, 0)], "not aligned to its element size"),
    ([(64, 4098, 4, F16, F32)], "out at 0x1002 is not aligned"),
    ([(64, 0, 1 << 41, F32, 0)], "too many"),
    ([(64, 0, 1 << 40, F32, 0)] * 3, "too many elements for one table"),
    # an out buffer over its own gradient in another type, another's, another out
    ([(64, 64, 4, F32, BF16)], "overlap"),
    ([(64, 72, 4, F32, F32)], "overlap"),
    ([(64, 4096, 4, F32, F32), (4104, 0, 1, F32, 0)], "overlap"),
    ([(64, 4096, 4, F32, F32), (128, 4108, 1, F32, F32)], "overlap"),
])
def test_table_refuses(entries, text):
    st, msg = create(entries)
    assert st == _native.TK_ERR_INVALID and text in msg, msg


def test_null_arguments():
    L = _native.lib()
    h = ctypes.c_void_p()
    assert L.tk_grad_table_create(None, 0, None) == _native.TK_ERR_INVALID
    assert L.tk_grad_table_create(None, 3, ctypes.byref(h)) == _native.TK_ERR_INVALID
    assert L.tk_grad_table_destroy(None) == 0
    assert L.tk_grad_workspace(None, None, None) == _native.TK_ERR_INVALID
    for st in (L.tk_grad_norm(None, 0, 0.0, None, None, None, None, None),
               L.tk_clip_grad_norm(None, 0, 1.0, None, None, None, None),
               L.tk_accumulate_grads(None, 1.0, 0, -1, None, None, None)):
        assert st == _native.TK_ERR_INVALID and b"null gradient table" in L.tk_last_error()


@pytest.mark.parametrize("bad,error,text", [
    ([1.0], TypeError, "expected a torch tensor, got float"),
    ([torch.zeros(3)], ValueError, "expected a dense CUDA tensor"),
    ([(4096, 7)], TypeError, "expected a torch tensor, got tuple"),
    ({"w": torch.zeros(3), "b": None}, ValueError, "gradient 0"),
])
def test_front_end_refuses_what_is_not_a_cuda_tensor(bad, error, text):
    with pytest.raises(error, match=text):
        tikun_b200.grad_norm(bad)


def test_front_end_refuses_arguments():
    with pytest.raises(ValueError, match="norm_type is 2, 1 or inf"):
        tikun_b200.grad_norm([], norm_type=3)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm is positive"):
            tikun_b200.clip_grad_norm_([], bad)
    with pytest.raises(ValueError, match="needs acc"):
        tikun_b200.accumulate_grads_([])


def test_dense_views():
    t = torch.zeros(4, 6, 5)
    for v in (t, t.transpose(0, 2), t.permute(1, 2, 0), t[1], t[:, :1, :][:1], t.reshape(-1)[3:9],
              torch.zeros(2, 1, 3).transpose(0, 1), torch.zeros(())):
        assert grads._dense(v)
    for v in (t[:, ::2], t[:, 1:], t[..., 0], torch.zeros(3, 1).expand(3, 4)):
        assert not grads._dense(v)


def test_clip_scale_is_refused_before_a_step():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    for opt in (tikun_b200.AdamW([p]), tikun_b200.MuonND([p]), tikun_b200.Muon([p])):
        for bad in (0.5, torch.tensor(0.5)):
            with pytest.raises(ValueError, match="one float32 value on a CUDA device"):
                opt.step(clip_scale=bad)
        assert opt.step_count == 0
    with pytest.raises(ValueError, match="max_norm is positive"):
        tikun_b200.clip_scale([p], 0.0)
    with pytest.raises(ValueError, match="expected a dense CUDA tensor"):
        tikun_b200.MuonND([p], max_norm=1.0).step()
