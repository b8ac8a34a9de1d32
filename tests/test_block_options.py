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


def calls(pkg):
    """(tensors, the operator on them) for every tensor operand that can carry a tangent."""
    pos, rows, w = torch.zeros(3, 1), torch.randn(1, 3, 16), torch.ones(16)
    q, k, v = heads(), heads(), heads()
    one = torch.ones(32)
    out = [([q, k, v], lambda *t: pkg.cross_attention(*t)),
           ([rows, rows + 1, w, w + 1, w + 2, w + 3], lambda *t: pkg.gated_residual_norm(*t[:5], post_norm="rms", post_weight=t[5])),
           ([q, k, one, one + 1, pos], lambda *t: pkg.rotary_axes_qk(t[0], t[1], t[4], (16,), q_weight=t[2], k_weight=t[3]))]
    return [(tensors, i, f) for tensors, f in out for i in range(len(tensors))]


@pytest.mark.parametrize("which", range(14))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(pkg, recorded, which, grad):
    """No operator has a forward-mode derivative: a tangent is never dropped without a word, with or without
    torch.no_grad (which does not switch forward mode off)."""
    from torch.autograd import forward_ad

    tensors, at, f = calls(pkg)[which]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        f(*tensors)  # a level without tangents changes nothing
        recorded.clear()
        tensors = [forward_ad.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate(tensors)]
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(*tensors)


def test_forward_mode_over_a_backward_is_refused(pkg, recorded):
    from torch.autograd import forward_ad

    q = heads().requires_grad_()
    out = pkg.cross_attention(q, heads(), heads())
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, [q], [g])


def test_forward_mode_numbers_are_refused(pkg, recorded):
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        value = forward_ad.make_dual(torch.tensor(0.5), torch.tensor(1.0))
        with pytest.raises(RuntimeError, match="forward-mode"):
            pkg.cross_attention(heads(), heads(), heads(), scale=value)


def test_grids_take_whole_numbers(pkg):
    """A start between two positions (a clip at another rate) was cut to a whole one: positions are int32 here, and a
    fractional start is refused; so is one whose grid leaves int32."""
    assert pkg.grid_positions([[1, 2.0]], 2, start=(torch.tensor(3), 4.0))[0].tolist() == [[3, 4], [3, 5]]
    for kw in (dict(start=0.5), dict(start=(0, 1.25)), dict(start=torch.tensor(0.5)), dict(start=float("nan")),
               dict(start=2 ** 31 - 2), dict(start=(0, -2 ** 31 - 1)), dict(start="x")):
        with pytest.raises(RuntimeError, match="start"):
            pkg.grid_positions([[1, 4]], 5, **kw)
    with pytest.raises(RuntimeError, match="grid_sizes"):
        pkg.grid_positions([[1, 2.5]], 5)
    assert pkg.grid_positions([[1, 2]], 2, start=2 ** 31 - 2)[0].tolist() == [[2 ** 31 - 2, 2 ** 31 - 2], [2 ** 31 - 2, 2 ** 31 - 1]]


def test_axis_dims_are_whole_numbers(pkg, recorded):
    pos = torch.zeros(3, 2, dtype=torch.int32)
    pkg.rotary_axes(heads(), pos, (8.0, torch.tensor(8)))
    assert recorded[-1]["axis_dims"] == (8, 8)
    with pytest.raises(RuntimeError, match="axis_dims"):
        pkg.rotary_axes(heads(), pos, (8.9, 8.9))
