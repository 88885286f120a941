"""Steps with a clip scale of the caller's between steps without one, on the GPU."""
import pytest
import torch

import tikun_b200
from tikun_b200.optimizer import AdamW as TorchAdamW

pytestmark = pytest.mark.gpu

SHAPES = [(64, 96), (96, 40), (3, 32, 16), (768,), (5,)]


def values(seed, std):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * std).cuda() for s in SHAPES]


BUILD = {
    "adamw": lambda ps: tikun_b200.AdamW(ps),
    "lion": lambda ps: tikun_b200.Lion(ps),
    "sgd": lambda ps: tikun_b200.SGD(ps),
    "arena": lambda ps: tikun_b200.AdamW(ps, arena=True),
    "torch": lambda ps: TorchAdamW(ps),
    "muon": lambda ps: tikun_b200.Muon(ps[:2], ps[3:]),
    "muon_nd": lambda ps: tikun_b200.MuonND(ps),
}


@pytest.mark.parametrize("form", BUILD)
def test_a_scale_of_the_callers_stays_as_it_is(form):
    """step(clip_scale=s), step() and step with a limit of its own: s keeps its value, and the
    parameters have the bits of an optimizer that never saw s."""
    def build():
        ps = [torch.nn.Parameter(t) for t in values(1, 0.02)]
        return ps, BUILD[form](ps)

    def give(ps, gs):
        for p, g in zip(ps, gs):
            if form == "arena":
                p.grad.copy_(g)
            else:
                p.grad = g

    def limit(opt, value):
        if form == "torch":
            opt.param_groups[0]["max_norm"] = value
        else:
            opt.max_norm = value

    (a, opt_a), (b, opt_b) = build(), build()
    history = torch.tensor([0.25, 0.5, 0.75], device="cuda")
    scale = history[1]
    for step, max_norm in enumerate((0.0, 0.0, 0.01, 0.0)):
        gs = values(10 + step, 0.1)
        limit(opt_a, 0.0 if step in (0, 3) else max_norm)
        limit(opt_b, max_norm)
        give(a, gs)
        if step in (0, 3):
            opt_a.step(clip_scale=scale)
            give(b, [g * 0.5 for g in gs])  # exact: the bits of the folded scale
        else:
            opt_a.step()
            give(b, gs)
        opt_b.step()
        assert history.tolist() == [0.25, 0.5, 0.75]
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("ns_steps", [0, 5])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_clipped_muon_step_at_odd_row_lengths(dtype, nesterov, ns_steps):
    """Rows that are no multiple of four, wide, tall and by heads, with and
    without Newton-Schulz: the bits of a step on gradients that were multiplied
    by the scale in f32."""
    shapes = [(33, 57), (57, 33), (1, 7), (9, 1), (3, 17, 29), (2, 70, 35), (64, 128)]
    gen = torch.Generator().manual_seed(4)
    ps = [torch.randn(s, generator=gen).cuda() * 0.02 for s in shapes]
    a, b = ([torch.nn.Parameter(t.clone()) for t in ps] for _ in range(2))
    opt_a, opt_b = (tikun_b200.MuonND(x, nesterov=nesterov, ns_steps=ns_steps) for x in (a, b))
    for scale in (0.37, 1.0, 2.0 ** -13):
        s = torch.tensor(scale, device="cuda")
        for x, y in zip(a, b):
            g = torch.randn(x.shape, generator=gen).cuda().to(dtype) * 0.1
            x.grad_dtype = y.grad_dtype = None  # it may have another type than its parameter
            x.grad, y.grad = g, g.float() * s
        opt_a.step(clip_scale=s)
        opt_b.step()
        for x, y in zip(a, b):
            assert torch.equal(x, y) and torch.isfinite(x).all()
