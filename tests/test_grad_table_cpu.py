"""What a GradTable remembers of its parameters, with the native table stubbed out."""
import pytest
import torch

from tikun_b200 import GradTable, _native, grads


@pytest.fixture
def table(monkeypatch):
    """A table of parameters that have no gradient."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(grads, "_on_device", lambda t, call: None)
    monkeypatch.setattr(_native, "check", lambda status: None)

    def build(tree):
        t = GradTable.__new__(GradTable)
        t._build(tree, None)
        return t

    return build


def test_a_first_gradient_after_the_build_is_noticed(table):
    a, b = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    t = table({"a": a, "b": [b, None]})
    assert len(t) == 0 and t._standing() is t
    b.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="build the table anew"):
        t._standing()
    b.grad = None
    assert t._standing() is t
