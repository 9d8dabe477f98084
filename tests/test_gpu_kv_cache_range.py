"""The int8 cache of keys and values at the ends of its ranges."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from megcc_b200 import ops  # noqa: E402
from test_gpu_kv_cache import IDS, TYPES, angles, cache_of, gen, ints, table_of  # noqa: E402


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("before", [2 ** 31 - 1, 2 ** 31 - 10, 2 ** 31 - 16, 2 ** 31 - 17, 2 ** 31 - 40])
def test_positions_next_to_two_to_the_31(before, dtype):
    """They are positions beyond the table, and beyond the rotation's: reported, keys and queries returned all the same."""
    table, pages = table_of([16], 16, 3)
    cache = cache_of(pages, 2, 16, 32, 4)
    kept = [t.clone() for t in cache]
    x = torch.randn((30, 2, 32), generator=gen(1), device="cuda").to(dtype)
    junk = torch.full((64, 2, 32), 7.0, device="cuda").to(dtype)  # (what the results' memory may hold)
    del junk
    _, k = ops.kv_append_s8(cache, table, ints([before]), x, x, cu_tokens=ints([0, 30]), turned_keys=True)
    torch.cuda.synchronize()
    assert ops.device_status() == 0x201
    assert torch.equal(k, x)
    cos, sin = angles(40, 16)
    q, k = ops.kv_append_s8(cache, table, ints([before]), x, x, x, cos, sin, cu_tokens=ints([0, 30]), turned_keys=True)
    torch.cuda.synchronize()
    assert ops.device_status() in (0x201, 0x202)
    for got in (q, k):
        assert bool(torch.isnan(got[..., :16]).all()) and torch.equal(got[..., 16:], x[..., 16:])
    assert all(torch.equal(a, b) for a, b in zip(cache, kept))
