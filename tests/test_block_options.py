"""What the block operators' options and modes mean beyond plain calls, with the kernels replaced by recorders (no GPU
needed)."""
import sys

import pytest
import torch

F = torch.float32


@pytest.fixture
def recorded(pkg, monkeypatch):
    """The three operators on CPU tensors that pass for device tensors; a kernel call leaves its keyword arguments in
    the list and gives tensors like its first ones."""
    calls = []
    for name in ("attention", "joint", "rotary"):
        module = sys.modules[f"{pkg.__name__}.{name}"]
        monkeypatch.setattr(module, "_meta", lambda t: None if t is None else (t.shape, t.dtype, torch.device("cuda", 0)))

    def kernel(n):
        def run(*args, **kw):
            calls.append(kw)
            first = args[0] if isinstance(args[0], (list, tuple)) else args
            return [t.detach().clone() for t in first[:n]]
        return run

    monkeypatch.setattr(pkg.kernels, "cross_attention", kernel(2))
    monkeypatch.setattr(pkg.kernels, "joint", kernel(2))
    monkeypatch.setattr(pkg.kernels, "rotary_axes", kernel(1))
    return calls


def heads():
    return torch.randn(1, 3, 2, 16)


def options(pkg):
    """(the option's name under the kernel, a call that takes it as a value) of every number that an operator takes."""
    pos = torch.zeros(3, 1, dtype=torch.int32)
    rows = torch.randn(1, 3, 16)
    return [("scale", lambda v: pkg.cross_attention(heads(), heads(), heads(), scale=v)),
            ("alpha", lambda v: pkg.gated_residual_norm(rows, rows, residual_scale=v)),
            ("eps", lambda v: pkg.gated_residual_norm(rows, rows, eps=v)),
            ("theta", lambda v: pkg.rotary_axes(heads(), pos, (16,), theta=v)),
            ("eps", lambda v: pkg.rotary_axes(heads(), pos, (16,), eps=v))]


@pytest.mark.parametrize("which", range(5))
def test_numbers_given_as_tensors_are_read_at_every_call(pkg, recorded, which):
    name, call = options(pkg)[which]
    value = torch.tensor(0.5)
    for now in (0.5, 0.25, 0.125):
        value.fill_(now)
        call(value)
        call(now)
        assert recorded[-2][name] == recorded[-1][name] == now


@pytest.mark.parametrize("which", range(5))
def test_numbers_have_no_gradient(pkg, recorded, which):
    """A value that wants one is refused and not used as a constant; without autograd it is a number like others."""
    name, call = options(pkg)[which]
    value = torch.nn.Parameter(torch.tensor(0.5))
    with pytest.raises(RuntimeError, match="no gradient"):
        call(value)
    assert not recorded
    with torch.no_grad():
        call(value)
    assert recorded[-1][name] == 0.5
    with pytest.raises(RuntimeError, match="number"):
        call("wide")


def test_unit_offset_is_read_at_every_call(pkg, recorded):
    x, w, flag = torch.randn(1, 3, 16), torch.ones(16), torch.tensor(True)
    for now in (True, False):
        flag.fill_(now)
        pkg.gated_residual_norm(x, x, scale=w, unit_offset=flag)
        assert recorded[-1]["unit_offset"] is now
