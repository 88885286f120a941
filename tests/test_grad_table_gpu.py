"""GradTable and its parameters, on the GPU."""
import pytest
import torch

from tikun_b200 import GradTable, accumulate_grads_, clip_grad_norm_, clip_scale, grad_norm

pytestmark = pytest.mark.gpu


def test_a_first_gradient_after_the_build_is_refused():
    """A table that was built before a parameter had a gradient does not leave
    that gradient out of the norm."""
    w, late = (torch.nn.Parameter(torch.zeros(8, device="cuda")) for _ in range(2))
    empty = GradTable([w, late])
    assert grad_norm(empty).item() == 0.0
    w.grad = torch.full((8,), 2.0, device="cuda")
    table = GradTable([w, late], out=[torch.zeros(8, device="cuda")])
    assert grad_norm(table, norm_type=1.0).item() == 16.0
    late.grad = torch.full((8,), 3.0, device="cuda")
    for t in (empty, table):
        for call in (lambda: grad_norm(t), lambda: clip_grad_norm_(t, 1.0),
                     lambda: clip_scale(t, 1.0), lambda: accumulate_grads_(t)):
            with pytest.raises(RuntimeError, match="build the table anew"):
                call()
    assert (w.grad == 2.0).all() and (late.grad == 3.0).all()
    assert grad_norm([w, late], norm_type=1.0).item() == 40.0
