"""Views that the paged-cache functions take: strides of dimensions of one element say nothing."""
import pytest
import torch

from mojo_llm_lab_b200 import ops

F16, I32 = torch.float16, torch.int32
# One KV head, and one page: caches [pages, heads, page, dim] whose strides differ there only.
CACHES = [(torch.zeros(6, 16, 1, 128, dtype=F16).transpose(1, 2), torch.zeros(6, 1, 16, 128, dtype=F16)),
          (torch.zeros(1, 2, 16, 128, dtype=F16), torch.zeros(2, 2, 16, 128, dtype=F16).as_strided((1, 2, 16, 128), (8, 2048, 128, 1)))]


@pytest.mark.parametrize("k,v", CACHES)
def test_caches_whose_strides_differ_in_dimensions_of_one(k, v):
    """Past the checks of the views: what is missing then is a GPU."""
    assert k.stride() != v.stride()
    heads, table, ints = k.shape[1], torch.zeros(3, 2, dtype=I32), torch.zeros(3, dtype=I32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_qkv_append(torch.zeros(3, (4 + 2 * heads) * 128), ints, ints, table, k, v, 4, torch.zeros(64, dtype=torch.float64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(torch.zeros(3, 4, 128, dtype=F16), k, v, table, ints)
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_reorder(torch.zeros(1, 3, dtype=I32), table, ints, ints, k, v)
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_reorder(torch.zeros(1, 3, dtype=I32), table, ints, ints, k[None], v[None])
