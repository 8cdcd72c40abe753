"""What the row operators hand to the library, without a GPU: host tensors that say they are on one, and a library that notes its calls."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import bournemouth_forced_aligner_amd as bfa
from bournemouth_forced_aligner_amd import _lib, rows


class _Device(torch.Tensor):
    """a host tensor that says it is on the GPU and whose numbers cannot be read by the host"""
    is_cuda = property(lambda self: True)

    def _read(self, *args):
        raise AssertionError("read by the host")

    __bool__ = __float__ = __int__ = __index__ = item = tolist = cpu = _read


def _device(t):
    return t.as_subclass(_Device)


@pytest.fixture
def calls(monkeypatch):
    """the C entries as {name: arguments of its last call}"""
    seen = {}

    class Library:
        def __getattr__(self, name):
            def entry(*args):
                seen[name] = args
                return 0
            return entry

    monkeypatch.setattr(rows, "_call", lambda dev: (Library(), None, 0))
    return seen


def _sample_params(calls):
    return calls["bfa_sample_labels"][7]._obj


@pytest.mark.parametrize("name,value", [("temperature", 0.5), ("top_p", 0.25), ("min_p", 0.125), ("top_k", 3)])
def test_one_number_on_the_device_is_not_read_by_the_host(calls, name, value):
    x = _device(torch.zeros(4, 3, 8))
    bfa.sample_labels(x, torch.zeros(4, 3), **{name: _device(torch.tensor(value))})
    p = _sample_params(calls)
    assert getattr(p, name + "_B")  # an array of B numbers, not a number
    bfa.sample_labels(x, torch.zeros(4, 3), **{name: torch.tensor(value)})  # (one on the host is a number like any other)
    p = _sample_params(calls)
    assert not getattr(p, name + "_B") and getattr(p, name) == value


@pytest.mark.parametrize("k,want", [(2 ** 32 + 5, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (-2 ** 33 - 1, 0), (7, 7), (-1, 0)])
def test_a_wide_top_k_is_as_much_as_fits(calls, monkeypatch, k, want):
    given = []
    kept = rows._per_row
    monkeypatch.setattr(rows, "_per_row", lambda *args: given.append(kept(*args)) or given[-1])
    bfa.sample_labels(_device(torch.zeros(2, 3, 8)), torch.zeros(2, 3), top_k=torch.tensor([k, 4]))
    assert given[-1].dtype == torch.int32 and given[-1].tolist() == [want, 4]
    bfa.sample_labels(_device(torch.zeros(2, 3, 8)), torch.zeros(2, 3), top_k=k)
    assert _sample_params(calls).top_k == want


def test_weights_that_require_a_gradient_are_refused(calls):
    x, labels = _device(torch.zeros(2, 3, 8)), torch.zeros(2, 3, dtype=torch.int32)
    w = torch.ones(2, 3, requires_grad=True)
    for rows_in in (x, _device(torch.zeros(2, 3, 8)).requires_grad_()):
        with pytest.raises(ValueError, match="no gradient goes to the weights"):
            bfa.label_loss(rows_in, labels, weights=w)
    bfa.label_loss(x, labels, weights=w.detach())
    with torch.no_grad():
        bfa.label_loss(x, labels, weights=w)
    bfa.label_loss_and_grad(x, labels, weights=w)  # (builds no graph: the gradient it returns is the logits')


def test_tangents_are_refused_not_dropped(calls):
    x, w, labels = torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(2, 3, dtype=torch.int32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(_device(x), _device(torch.ones_like(x)))
        dual_w = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: bfa.layer_norm(dual), lambda: bfa.layer_norm(_device(x), dual_w), lambda: bfa.label_loss(dual, labels)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        with pytest.raises(ValueError, match="no gradient goes to the weights"):
            bfa.label_loss(_device(x), labels, weights=forward_ad.make_dual(torch.ones(2, 3), torch.ones(2, 3)))
        bfa.layer_norm(_device(x), w)  # (without a tangent: as ever)
        bfa.label_loss(_device(x), labels)
    assert {"bfa_layer_norm", "bfa_label_loss"} <= set(calls)
