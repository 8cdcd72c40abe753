"""The row operators (layer_norm, label_loss, sample_labels) without a GPU: the C entries and what is refused before any launch."""
import ctypes

import pytest
import torch

import bournemouth_forced_aligner_amd as bfa
from bournemouth_forced_aligner_amd import _lib, rows


def test_public_names():
    for name in ("layer_norm", "layer_norm_forward", "layer_norm_backward", "label_loss", "label_loss_and_grad", "sample_labels"):
        assert callable(getattr(bfa, name)) and name in bfa.__all__


def test_host_tensors_are_refused():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        bfa.layer_norm(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        bfa.label_loss(x, torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        bfa.sample_labels(x, torch.zeros(2, 3))


def test_workspace_sizes():
    L = _lib.lib()
    assert L.bfa_layer_norm_workspace_bytes(0, 5, 8) == 0
    assert L.bfa_layer_norm_workspace_bytes(1 << 16, 1 << 15, 8) == 0  # more rows than a call takes
    assert L.bfa_layer_norm_workspace_bytes(1, 1, 8) == 8 * 2 * 4       # one workgroup, dweight and dbias, float32
    assert L.bfa_layer_norm_workspace_bytes(64, 1000, 4096) >= 2 * 4096 * 4
    assert L.bfa_label_loss_workspace_bytes(4, 4, 67) > 0
    assert L.bfa_label_loss_workspace_bytes(-1, 4, 67) == 0


def test_null_handle_is_an_error_not_a_crash():
    L = _lib.lib()
    r = _lib.BfaRows(None, 0, 0, 0)
    assert L.bfa_layer_norm(None, ctypes.byref(r), 1, 1, 1, None, None, None, 0, 1e-5, ctypes.byref(r), None, None, None) == _lib.BFA_ERR_INVALID_ARGUMENT
    assert L.bfa_layer_norm_backward(None, ctypes.byref(r), ctypes.byref(r), 1, 1, 1, None, None, 0, None, None, None, None, None, None, 0,
                                     None) == _lib.BFA_ERR_INVALID_ARGUMENT
    assert L.bfa_label_loss(None, ctypes.byref(r), 1, 1, 1, None, None, None, 0, 1.0, None, None, None, None, 0, None) == _lib.BFA_ERR_INVALID_ARGUMENT
    p = _lib.BfaSampleParams(1.0, 1.0, 0.0, 0, None, None, None, None)
    assert L.bfa_sample_labels(None, ctypes.byref(r), 1, 1, 1, None, None, ctypes.byref(p), None, None, None) == _lib.BFA_ERR_INVALID_ARGUMENT


class _Meta(torch.Tensor):
    """a host tensor that says it is on the GPU: the argument checks in front of any launch look at nothing else"""
    is_cuda = property(lambda self: True)


def _meta(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Meta)


def test_shapes_and_types_are_checked():
    x = _meta(2, 3, 8)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        bfa.layer_norm(_meta(2, 3, 8, dtype=torch.float64))
    with pytest.raises(TypeError, match="weight must be"):
        bfa.layer_norm(x, torch.zeros(8, dtype=torch.float64))
    with pytest.raises(ValueError, match="weight must have shape"):
        bfa.layer_norm(x, torch.zeros(7))
    with pytest.raises(TypeError, match="one type"):
        bfa.layer_norm(x, torch.zeros(8), torch.zeros(8, dtype=torch.float16))
    with pytest.raises(ValueError, match="eps"):
        bfa.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        bfa.layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError, match="lengths must have one entry"):
        bfa.layer_norm(x, lengths=[3])
    with pytest.raises(ValueError, match="lengths go with rows"):
        bfa.layer_norm(_meta(2, 2, 3, 8), lengths=[3, 3])
    with pytest.raises(ValueError, match="reduction"):
        bfa.label_loss(x, torch.zeros(2, 3, dtype=torch.int32), reduction="average")
    with pytest.raises(ValueError, match="labels must have the shape"):
        bfa.label_loss(x, torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(TypeError, match="whole numbers"):
        bfa.label_loss(x, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="weights must have the shape"):
        bfa.label_loss(x, torch.zeros(2, 3, dtype=torch.int32), weights=torch.ones(3, 2))
    with pytest.raises(ValueError, match="uniform must have the shape"):
        bfa.sample_labels(x, torch.zeros(6))
    u = torch.zeros(2, 3)
    for bad in (dict(temperature=-1.0), dict(top_p=0.0), dict(min_p=1.5), dict(min_p=-0.1), dict(temperature=float("nan")),
                dict(top_p=float("nan")), dict(min_p=float("nan"))):
        with pytest.raises(ValueError, match=next(iter(bad))):
            bfa.sample_labels(x, u, **bad)
    with pytest.raises(ValueError, match="top_k must have the shape"):
        bfa.sample_labels(x, u, top_k=torch.tensor([1, 2, 3]))
    with pytest.raises(ValueError, match="grad must match"):
        bfa.layer_norm_backward(torch.zeros(2, 3, 7), x, torch.zeros(2, 3), torch.zeros(2, 3))
    with pytest.raises(ValueError, match="mean must be float32"):
        bfa.layer_norm_backward(torch.zeros(2, 3, 8), x, torch.zeros(3), torch.zeros(2, 3))


def test_views_are_described_not_copied():
    """padded rows, swapped leading dimensions and broadcast rows go to the kernels as they are"""
    store = torch.arange(2 * 3 * 10, dtype=torch.float32).reshape(2, 3, 10)
    t, r = rows._rows(store[..., :8], 2, 3)
    assert t.data_ptr() == store.data_ptr() and (r.strideB, r.strideT) == (30, 10)
    t, r = rows._rows(store.transpose(0, 1), 3, 2)
    assert t.data_ptr() == store.data_ptr() and (r.strideB, r.strideT) == (10, 30)
    t, r = rows._rows(torch.zeros(8).expand(2, 3, 8), 2, 3)
    assert (r.strideB, r.strideT) == (0, 0)
    t, r = rows._rows(store.transpose(1, 2), 2, 10)  # the last stride is not 1: copied
    assert t.is_contiguous() and (r.strideB, r.strideT) == (30, 3)
    t, r = rows._rows(torch.zeros(5), 1, 1)
    assert t.shape == (1, 1, 5)
