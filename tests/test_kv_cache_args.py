"""Arguments of KvCache that are refused before a tensor is made or looked at."""
import pytest
import torch

from frisk_amd import runtime as rt


@pytest.mark.parametrize("dtype,block", [
    (torch.int8, 0), (torch.float8_e4m3fn, 0), (torch.int8, -32), (torch.bfloat16, 0), (torch.bfloat16, 16),
    (torch.float16, -1)])
def test_blocks_of_no_slots(dtype, block):
    with pytest.raises(ValueError, match=f"scale_block must be 1 or more, and is for 8-bit caches .got {block}."):
        rt.KvCache.empty(4, 2, 16, 64, dtype, scale_block=block, device="cpu")
