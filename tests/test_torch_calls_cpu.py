"""CPU: the module between torch tensors and the library answers None to what it cannot take, before anything of the
library is called, and ops says what it was."""
import ctypes as C

import pytest
import torch

from gcn_amd import lib as L
from gcn_amd import ops


@pytest.fixture(scope="module")
def calls():
    return L.calls()


def test_tensors_in_host_memory_are_not_taken(calls):
    x, y, d = torch.zeros(4, 13), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    table = (L.AdamwTensor * 1)((d.data_ptr(), 4, 0, 0, 0.0, L.TYPE_F32))
    for device in (0, -1, 7):
        assert calls.log_probs(0, device, x, y, 0, True) is None
        assert calls.log_probs_grad(0, device, x, y, torch.zeros(4, 4), d, d, None, None) is None
        assert calls.grad_norm(0, device, [d], 1.0) is None
        assert calls.adamw_step(0, device, [d], [d], C.addressof(table), 32, d, d, None, None, None, d, 1e-3, 0.9, 0.999,
                                1e-8, None) is None


def test_what_is_not_a_tensor_is_not_taken(calls):
    for odd in (None, 3, "x", [1.0], object()):
        assert calls.log_probs(0, 0, odd, odd, 0, True) is None
        assert calls.log_probs_grad(0, 0, odd, odd, odd, odd, odd, odd, odd) is None
        assert calls.grad_norm(0, 0, odd, 1.0) is None
        assert calls.grad_norm(0, 0, [odd], 1.0) is None
        assert calls.adamw_step(0, 0, odd, odd, 0, 32, odd, odd, odd, odd, odd, odd, 1e-3, 0.9, 0.999, 1e-8, odd) is None
        assert calls.adamw_step(0, 0, [odd], [odd], 0, 32, odd, odd, odd, odd, odd, odd, 1e-3, 0.9, 0.999, 1e-8, odd) is None
    assert calls.grad_norm(0, 0, [], 1.0) is None


def test_arguments_are_counted_and_numbers_are_numbers(calls):
    x, y = torch.zeros(4, 13), torch.zeros(4, dtype=torch.int32)
    for name in ("bind", "log_probs", "log_probs_grad", "grad_norm", "adamw_step"):
        with pytest.raises(TypeError):
            getattr(calls, name)(1)
    with pytest.raises(TypeError):
        calls.log_probs(0, 0, x, y, "many", True)
    with pytest.raises(TypeError):
        calls.grad_norm(0, 0, [x], "much")


def test_ops_says_what_is_wrong():
    x, y = torch.zeros(4, 13), torch.zeros(4, dtype=torch.int32)
    scored = ops.LogProbs(x[:, 0], x[:, 0], None, None, torch.zeros(4, 4))
    for call in (lambda: ops.log_probs(x, y), lambda: ops.log_probs(None, y), lambda: ops.log_probs_grad(x, y, scored, x[:, 0]),
                 lambda: ops.grad_norm([x]), lambda: ops.grad_norm([3]), lambda: ops.AdamW([x])):
        with pytest.raises(TypeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="at least one"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="max_norm"):
        ops.grad_norm([x], -1.0)


def test_the_table_of_a_step_is_an_array_with_a_length(calls):
    """Its entries are looked at up to its own length, which has to be that of the lists."""
    d = torch.zeros(4)
    table = (L.AdamwTensor * 1)((d.data_ptr(), 4, 0, 0, 0.0, L.TYPE_F32))
    for count in (1, 2, 500):
        for odd in (table, bytes(table), memoryview(b"")[::1], b"", "x", None, 3.5, 1 << 70, [table]):
            assert calls.adamw_step(0, 0, [d] * count, [d] * count, odd, 32, d, d, None, None, None, d, 1e-3, 0.9, 0.999,
                                    1e-8, None) is None


def test_a_read_out_takes_an_array_and_tensors_of_its_sizes(calls):
    d = torch.zeros(4)
    table = (L.AdamwTensor * 2)((d.data_ptr(), 4, 0, 0, 0.0, L.TYPE_F32), (d.data_ptr(), 4, 4, 1, 0.0, L.TYPE_F32))
    codes, scales = torch.zeros(512, dtype=torch.uint8), torch.zeros(2)
    for odd in (table, bytes(table)[:-1], b"", None, 3, "x"):
        for device in (0, -1):
            assert calls.adamw_moments(0, device, odd, codes, codes, scales, scales, None) is None
            assert calls.adamw_moments(0, device, odd, None, None, None, None, None) is None
    with pytest.raises(TypeError):
        calls.adamw_moments(0, 0, table)
