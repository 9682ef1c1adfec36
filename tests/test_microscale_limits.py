"""CPU: refusals of the microscaled operators at the limits of their arguments.  No kernel is launched."""
import pytest
import torch

from mapping_challenge_amd import microscale as mx


def test_packed_tensor_of_an_unknown_type_is_refused():
    codes, scales = torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    assert mx.MxTensor(codes, scales, 40).dtype is None
    assert mx.MxTensor(codes, scales, 40, dtype=torch.bfloat16).dtype == torch.bfloat16
    with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
        mx.MxTensor(codes, scales, 40, dtype=torch.float64)
