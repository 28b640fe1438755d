"""The 8-bit KV cache on the GPU where its calls end: rows that overlap."""
import numpy as np
import pytest

from hllm_b200._lib import StageError
from tests.gpu_util import torch_cuda
from tests.test_kv8_gpu import ints, random_cache, tables_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return torch_cuda()


@pytest.fixture(scope="module")
def kv8(torch):
    from hllm_b200 import kv8
    return kv8


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("turns", [2, 5, 40])
def test_decreasing_offsets_stay_inside_the_workspace(torch, kv8, d, turns):
    """cu_seqlens that run back make rows overlap: more tiles of queries than a
    batch of these tokens can have.  It is reported, nothing behind the workspace
    is written, and the calls after it are as before."""
    hq, hkv, T, n = 64, 8, 64, 1024
    rng = np.random.default_rng(d)
    cache = random_cache(torch, kv8, rng, 70, hkv, d)
    table = tables_for(torch, rng, [64], 70)
    rows = 2 * turns - 1
    cu = ints(torch, [0, T] * turns)
    lengths = ints(torch, np.linspace(T, n, rows).astype(np.int32))  # the last rows' tiles are taken first
    tables = ints(torch, np.repeat(table, rows, 0))
    q = torch.randn((T, hq * d), device="cuda").half()
    need = kv8.attention_workspace(rows, T, T, hq, hkv, d).numel()
    buffer = torch.full((need + (64 << 20),), 0xa5, dtype=torch.uint8, device="cuda")
    out = torch.full((T + 1, hq * d), 9.0, dtype=torch.float16, device="cuda")
    good = (ints(torch, [0, T]), ints(torch, [n]), ints(torch, table))
    clean = kv8.attention(cache, q, *good, max_tokens=T)
    for _ in range(2):
        kv8.attention(cache, q, cu, lengths, tables, max_tokens=T, out=out[:T], workspace=buffer[:need])
        with pytest.raises(StageError, match="out of range"):
            cache.check()
        assert bool((buffer[need:] == 0xa5).all())
        assert bool((out[T:] == 9).all()) and bool(out.isfinite().all())
        again = kv8.attention(cache, q, *good, max_tokens=T, workspace=buffer[:need])
        cache.check()
        assert torch.equal(again, clean)
