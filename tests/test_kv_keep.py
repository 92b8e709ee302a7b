"""KVCache.keep and QuantKVCache.keep: shapes that do not fit are refused on the host (a
row past the cache's sequences would be an index that the device stops at)."""
import pytest
import torch

from torchplusplus_amd.llmops.kvcache import KVCache, QuantKVCache


@pytest.mark.parametrize("kind", [KVCache, QuantKVCache])
def test_shapes_that_do_not_fit(kind):
    cache = kind(16, 2, 64, torch.float16, "cpu", 2)
    path, start = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cache.keep(start, path)
    cache.keep(start[:1], path[:1])
    for s, p in ((torch.zeros(3, dtype=torch.int32), torch.zeros(3, 3, dtype=torch.int32)), (start[:1], path),
                 (start, path[:1]), (start, path[0]), (start.view(2, 1), path)):
        with pytest.raises(ValueError, match="start"):
            cache.keep(s, p)
