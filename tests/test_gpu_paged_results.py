"""What the results of the paged calls hold on to."""
import pytest
import torch

import butterfly_b200 as bb

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [16, 4])
def test_outputs_and_sums_have_storages_of_their_own(bits):
    """A caller that keeps the sums of many steps does not keep their outputs, 2 dh / 4 times the size."""
    c = bb.PagedKVCache(num_layers=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=128, max_requests=2, max_tokens_per_request=32,
                        cache_bits=bits)
    rows = torch.randn(7, 2, 128, device=DEV).bfloat16()
    c.append(0, rows, rows, c.reserve([3, 4]).slot_map)
    q = torch.randn(2, 4, 1, 128, device=DEV).bfloat16()
    out, lse = c.attend(0, q, return_lse=True)
    assert out.untyped_storage().nbytes() == out.numel() * 2 and lse.untyped_storage().nbytes() == lse.numel() * 4
    assert out.untyped_storage().data_ptr() != lse.untyped_storage().data_ptr() and lse.storage_offset() == 0
    assert torch.equal(out, c.attend(0, q))
