"""What the training operators hand to their kernels, without a GPU: CPU tensors go through the CUDA path with the launches recorded."""
import contextlib

import pytest
import torch

from oxibonsai_b200 import training as TR
from oxibonsai_b200.ops import train_ops


class _Gpu:
    """Stands for the device of CPU tensors that are taken for CUDA ones."""
    type, index = "cuda", -1          # what get_device() says of a CPU tensor
    __hash__ = object.__hash__

    def __eq__(self, other):
        return True

    def __ne__(self, other):
        return False


@pytest.fixture
def launches(monkeypatch):
    """The Adam launches: (addresses of the parameters, sizes)."""
    seen = []

    class Lib:
        def bonsai_mt_partials(self, n):
            return n

        def bonsai_mt_adam(self, n, p, g, m, v, numel, *rest):
            seen.append((list(p)[:n], list(numel)[:n]))
            return 0

    monkeypatch.setattr(train_ops, "_lib", Lib)
    monkeypatch.setattr(train_ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(train_ops, "_stream", lambda device: 0)
    return seen


def _optimizer(params):
    opt = TR.FusedAdam(params)
    opt.device = _Gpu()
    opt._place()
    return opt


def _parameter(*shape, dtype=torch.float32):
    p = torch.ones(*shape, dtype=dtype, requires_grad=True)
    p.grad = torch.ones_like(p)
    return p


def _set(p, data):
    p.grad = None
    p.data = data
    p.grad = torch.ones_like(p)


@pytest.mark.parametrize("cpu", [False, True])
@pytest.mark.parametrize("change", [lambda x: x[:500], lambda x: x.view(500, 2), lambda x: x.view(2, 500), lambda x: x[::2], lambda x: x[:0]])
def test_adam_refuses_a_parameter_that_changed_in_place(change, cpu, launches):
    a, b = _parameter(1000), _parameter(7)
    opt = TR.FusedAdam([a, b]) if cpu else _optimizer([a, b])
    opt.step(max_norm=1.0)
    m, steps = opt.m[0].clone(), opt.t
    at = a.data_ptr()
    _set(a, change(a.data))
    assert a.data_ptr() in (at, 0)
    with pytest.raises(ValueError, match="shape"):
        opt.step(max_norm=1.0)
    assert len(launches) == (0 if cpu else 1) and torch.equal(opt.m[0], m) and opt.t == steps


def test_adam_refuses_a_parameter_that_is_shorter_than_its_gradient(launches):
    a = _parameter(1000)
    opt = _optimizer([a])
    a.data = a.data[:500]                         # the gradient still has its thousand values
    with pytest.raises(ValueError):
        opt.step()
    assert not launches


def test_adam_steps_a_type_that_changed_in_place(launches):
    a = _parameter(64, dtype=torch.float16)
    opt = _optimizer([a])
    opt.step()
    _set(a, a.data.view(torch.bfloat16))
    opt.step()
    assert launches[0] == launches[1] and opt._fixed[0].types[0] == train_ops.TYPE_CODES[torch.bfloat16]


def test_adam_takes_the_same_parameter_at_a_new_place(launches):
    a = _parameter(1000)
    opt = _optimizer([a])
    _set(a, torch.zeros(1000))
    opt.step()
    assert launches == [([a.data_ptr()], [1000])]


def test_tables_of_other_sizes_are_refused(launches):
    table = train_ops.TensorTable([torch.ones(10), torch.ones(3)])
    train_ops.TensorTable([torch.zeros(10), torch.zeros(3)], like=table)
    for bad in ([torch.zeros(5), torch.zeros(3)], [torch.zeros(10), torch.zeros(4)]):
        with pytest.raises(ValueError):
            train_ops.TensorTable(bad, like=table)


def test_adam_refuses_gradients_that_no_kernel_walks(launches):
    a = _parameter(8, 4)
    opt = _optimizer([a])
    a.grad = torch.eye(8)[:, :4].to_sparse()
    with pytest.raises(TypeError):
        opt.step()
    assert not launches


@pytest.mark.parametrize("cpu", [False, True])
def test_adam_counts_versions_of_the_parameters_that_it_steps(cpu, launches):
    a, b = _parameter(5), _parameter(7)
    opt = TR.FusedAdam([a, b]) if cpu else _optimizer([a, b])
    loss = (b * b).sum()                                # keeps b for its backward pass
    b.grad = None
    was = a._version
    opt.step(max_norm=1.0)
    assert a._version > was
    loss.backward()                                     # b has not been written
    opt.step()
    loss = (b * b).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
