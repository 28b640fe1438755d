"""The 8-bit KV cache on the GPU where its calls end: rows that overlap,
keys that a token may not see, sizes far apart, tails of small weights."""
import math

import numpy as np
import pytest

from hllm_b200._lib import StageError
from tests import kv8_util
from tests.gpu_util import torch_cuda
from tests.test_kv8_gpu import bytes_of, ints, random_cache, tables_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return torch_cuda()


@pytest.fixture(scope="module")
def kv8(torch):
    from hllm_b200 import kv8
    return kv8


def normal(torch, shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g)


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
    q = normal(torch, (T, hq * d), turns).half()
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


def check_nan(torch, kv8, heads, n, count, keys, most=None):
    """NaN codes in K and in V rows reach the tokens at their position and later
    ones, of their kv head, in V their dimension alone; everything else keeps its bits."""
    hq, hkv, d = heads
    rng = np.random.default_rng(n + count + d)
    pages = (n + 15) // 16
    cache = random_cache(torch, kv8, rng, pages + 3, hkv, d)
    table = tables_for(torch, rng, [pages], pages + 3)
    q = normal(torch, (count, hq * d), n).half()
    args = (ints(torch, [0, count]), ints(torch, [n]), ints(torch, table))
    clean = kv8.attention(cache, q, *args, max_tokens=most or count).view(count, hq, d)
    assert not bool(clean.isnan().any())
    position = torch.arange(n - count, n, device="cuda")
    for which in (0, 2):
        codes = bytes_of(torch, cache)[which]
        keep = codes.clone()
        want = torch.zeros_like(clean, dtype=torch.bool)
        for i, key in enumerate(keys):
            head, dim = (key + i) % hkv, key * 7 % d
            codes[table[0, key // 16], head, key % 16, dim] = 0x7f if i % 2 else 0xff
            mine = slice(head * (hq // hkv), (head + 1) * (hq // hkv))
            want[position >= key, mine, dim if which else slice(None)] = True
        got = kv8.attention(cache, q, *args, max_tokens=most or count).view(count, hq, d)
        assert torch.equal(got.isnan(), want)
        assert torch.equal(got[~want], clean[~want])
        codes.copy_(keep)
    cache.check()


@pytest.mark.parametrize("heads", [(8, 2, 128), (32, 8, 128), (8, 8, 64), (4, 2, 64), (6, 2, 256), (3, 1, 32),
                                   (12, 4, 96), (4, 4, 160), (7, 1, 192), (2, 1, 224), (16, 1, 128), (20, 1, 64)])
@pytest.mark.parametrize("past,count", [(0, 3), (29, 2), (100, 3), (14, 15)])
def test_nan_in_keys_that_some_tokens_do_not_see(torch, kv8, heads, past, count):
    count = min(count, 63 * heads[1] // heads[0])  # few enough columns for the stream pass
    n = past + count
    check_nan(torch, kv8, heads, n, count, sorted({0, past // 2, past, past + 1, n - 2, n - 1} & set(range(n))))


@pytest.mark.parametrize("heads", [(6, 2, 256), (4, 4, 96), (3, 1, 32)])
def test_nan_in_the_middle_of_chunks_at_other_head_sizes(torch, kv8, heads):
    check_nan(torch, kv8, heads, 150, 90, (35, 60, 97, 113, 149))
    check_nan(torch, kv8, heads, 3000, 40, (7, 2959, 2960, 2975, 2976, 2998))


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 2, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128)])
@pytest.mark.parametrize("past,count", [(0, 140), (80, 70), (1000, 130), (2900, 100), (5, 400)])
def test_nan_in_the_middle_of_prompt_chunks(torch, kv8, heads, past, count):
    n = past + count
    keys = {0, 35, past, past + 1, past + count // 2, past + 63, past + 127, n - 2, n - 1}
    check_nan(torch, kv8, heads, n, count, sorted(k for k in keys if k < n))


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("n,count", [(3, 6), (20, 90), (40, 300)])
def test_nan_where_early_tokens_have_no_key(torch, kv8, heads, n, count):
    """More new tokens than keys: the first see none, and give zeros."""
    check_nan(torch, kv8, heads, n, count, (0, 1, n - 1))


@pytest.mark.parametrize("d", [64, 128])
def test_nan_in_the_middle_of_a_long_chunk(torch, kv8, d):
    """CTAs of two query tiles."""
    check_nan(torch, kv8, (16, 8, d), 2600, 2500, (35, 100, 127, 128, 1000, 1383, 2047, 2500, 2599))


def attend(torch, k, v, q, position, scale, spread=0):
    """One head of one row in 64 bits, with the error that its arithmetic may
    have: k, v [n, d], q [count, d], position [count].  A score's error counts by
    its own terms, so a key's size loosens nothing for the others:
      * score j, in F32: r_j = 2 (d + 8) 2^-23 sum_i |q_i k_ji| scale + 2^-20 (exp2 and
        scales), absolutely, which moves weight j by r_j of itself;
      * weight j to F16: 2^-11 of it, or half of F16's least step, 2^-25, where the
        largest weight times value scale is 2^7 at least: 2^-32 of that.  Where the
        reference counts a tile's largest value scale (exponents within 2^spread of
        it, 2^8 at most), the largest may be 2^spread less: 2^(spread - 32);
      * the sums of n terms: 2 n 2^-23 each, over all keys that there are;
      * the normaliser: sum_j p_j r_j and the sum's, of the output;
      * the output to F16: 2^-11 of it, or 2^-25."""
    n, d = k.shape
    hidden = torch.arange(n, device=q.device)[None, :] > position[:, None]
    p = torch.softmax((q @ k.T * scale).masked_fill(hidden, -math.inf), -1)
    o = p @ v
    r = 2 * (d + 8) * 2.0 ** -23 * (q.abs() @ k.abs().T * scale) + 2.0 ** -20
    pr = torch.where(p > 0, p * r, 0.0)
    sums = 2 * n * 2.0 ** -23
    share = p @ v.abs()
    amax = (p * 2 * v.abs().amax(-1)).amax(-1, keepdim=True)  # a value is at most 2 amax of its row
    tol = (pr @ v.abs() + (2.0 ** -11 + sums) * share + n * 2.0 ** (min(spread, 8) - 32) * amax +
           (pr.sum(-1, keepdim=True) + sums) * share + 2.0 ** -11 * o.abs() + 2.0 ** -25)
    return o, tol


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 2, 64), (16, 8, 128), (8, 8, 64), (6, 2, 256)])
@pytest.mark.parametrize("past,count", [(60, 100), (300, 5), (700, 600), (2, 3000)])
@pytest.mark.parametrize("octaves", [14, 18, 34, 44])
def test_large_keys_coarsen_no_others(torch, kv8, heads, past, count, octaves):
    """Keys 2^octaves times the others, along a direction of their own in which
    all queries point away from them: their weight is 0 where they are seen, and
    they are hidden from early tokens.  Others' scores keep their precision."""
    hq, hkv, d = heads
    n = past + count
    rng = np.random.default_rng(octaves)
    pages = (n + 15) // 16
    cache = random_cache(torch, kv8, rng, pages + 3, hkv, d)
    table = tables_for(torch, rng, [pages], pages + 3)
    kc, ks, vc, vs = bytes_of(torch, cache)
    kc[..., 0] = 0
    for key in sorted({0, past // 2, past, past + count // 3, n - 2}):
        at = int(table[0, key // 16]), slice(None), key % 16
        kc[at] = 0
        kc[at[0], :, at[2], 0] = 0xc0  # -2
        ks[at] = min(122 + octaves, 127 + 39)
    q = (1.5 * normal(torch, (count, hq, d), octaves)).half()
    q[..., 0] = 16.0
    got = kv8.attention(cache, q.view(count, hq * d), ints(torch, [0, count]), ints(torch, [n]),
                        ints(torch, table)).view(count, hq, d).double()
    cache.check()
    at = torch.as_tensor(table[0], device="cuda").long()
    k, v = (kv8_util.values(torch, c[at], e[at]).transpose(1, 2).reshape(-1, hkv, d)[:n]
            for c, e in ((kc, ks), (vc, vs)))
    position = torch.arange(past, n, device="cuda")
    spread = int(vs.max()) - int(vs.min())
    for h in range(hq):
        want, tol = attend(torch, k[:, h // (hq // hkv)], v[:, h // (hq // hkv)], q[:, h].double(), position,
                           1 / math.sqrt(d), spread)
        err = (got[:, h] - want).abs() / tol
        assert bool((err <= 1).all()), (h, float(err.max()), err.amax(-1).nonzero()[:5])


@pytest.mark.parametrize("heads", [(2, 1, 128), (4, 2, 64), (1, 1, 256), (16, 1, 128), (8, 2, 128)])
@pytest.mark.parametrize("n,count,rows", [(131072, 1, 1), (100001, 2, 1), (4000, 1, 1), (70003, 64, 1), (3001, 600, 1),
                                          (4000, 1, 1500), (3000, 2, 700)])
@pytest.mark.parametrize("octaves", [12, 20, 25])
def test_a_long_tail_of_small_weights_counts(torch, kv8, heads, n, count, rows, octaves):
    """One key 2^octaves times as heavy as each of all the others, whose values
    are 1 in every dimension and its own 0 in all but one: what the output holds is
    the others' share, 2^-8 for 2^17 of them at 25 octaves.  (Of one row the keys are
    split, and most splits do not have the key; of many rows they are not.)"""
    hq, hkv, d = heads
    rng = np.random.default_rng(octaves)
    pages = (n + 15) // 16
    cache = kv8.Cache(pages + 2, hkv, d)
    table = tables_for(torch, rng, [pages], pages + 2)
    kc, ks, vc, vs = bytes_of(torch, cache)
    vc[...] = 0x38  # 1
    heavy = n // 3
    at = int(table[0, heavy // 16]), heavy % 16
    kc[at[0], :, at[1], 0] = 0x38
    vc[at[0], :, at[1]] = 0
    vc[at[0], :, at[1], 1] = 0x38
    q = torch.zeros((count * rows, hq, d), device="cuda", dtype=torch.float16)
    q[..., 0] = octaves
    scale = math.log(2.0)
    got = kv8.attention(cache, q.view(-1, hq * d), ints(torch, np.arange(rows + 1) * count), ints(torch, [n] * rows),
                        ints(torch, np.repeat(table, rows, 0)), max_tokens=count, scale=scale)
    got = got.view(rows, count, hq, d).double()
    cache.check()
    pages_at = torch.as_tensor(table[0], device="cuda").long()
    k, v = (kv8_util.values(torch, c[pages_at, 0], e[pages_at, 0]).reshape(-1, d)[:n]
            for c, e in ((kc, ks), (vc, vs)))
    want, tol = attend(torch, k, v, q[:count, 0].double(), torch.arange(n - count, n, device="cuda"), scale)
    err = (got - want[:, None]).abs() / tol[:, None]
    assert bool((err <= 1).all()), float(err.max())


def test_a_single_row_may_have_any_step(torch, kv8):
    """torch leaves the stride of a dimension of one row open: a column's transpose,
    a row of a matrix of odd width, a row said to be repeated."""
    hq, hkv, d = 4, 2, 64
    rng = np.random.default_rng(1)
    cache = random_cache(torch, kv8, rng, 6, hkv, d)
    args = (ints(torch, [0, 1]), ints(torch, [40]), ints(torch, tables_for(torch, rng, [3], 6)))
    q = normal(torch, (1, hq * d), 1).half()
    want = kv8.attention(cache, q, *args)
    column = q.t().contiguous()
    odd = torch.empty((2, hq * d + 5), dtype=torch.float16, device="cuda")
    odd[0, :hq * d] = q[0]
    for given in (column.t(), odd[:1, :hq * d], q[0].expand(1, hq * d)):
        assert torch.equal(kv8.attention(cache, given, *args), want)
    for out in (torch.empty_like(column).t(), odd[:1, :hq * d]):
        assert torch.equal(kv8.attention(cache, q, *args, out=out), want)
        assert torch.equal(out, want)
    cache.check()


def test_read_reports_offsets_out_of_range(torch, kv8):
    """Rows that the output has no room for, or that end before they begin."""
    rng = np.random.default_rng(2)
    rows, n = 300, 20
    cache = random_cache(torch, kv8, rng, 2 * rows, 2, 64)
    table = ints(torch, tables_for(torch, rng, [2] * rows, 2 * rows))
    lengths = ints(torch, [n] * rows)
    good = np.arange(rows + 1) * n
    T = rows * n
    k, v = kv8.read(cache, table, lengths, ints(torch, good), T)
    cache.check()
    for change, kept in ((lambda c: c[-1:].__iadd__(1), T), (lambda c: c[280:].__iadd__(7), 280 * n),
                         (lambda c: c[5:6].__isub__(200), 0), (lambda c: c[:1].__isub__(n), 0)):
        cu = good.copy()
        change(cu)
        out = tuple(torch.full_like(k, 7.0) for _ in range(2))
        kv8.read(cache, table, lengths, ints(torch, cu), T, out=out)
        with pytest.raises(StageError, match="out of range"):
            cache.check()
        assert torch.equal(out[0][:kept], k[:kept]) and torch.equal(out[1][:kept], v[:kept])
    # A shorter output: the rows that fit are whole.
    out = tuple(torch.full_like(k, 7.0) for _ in range(2))
    kv8.read(cache, table, lengths, ints(torch, good), T - 2 * n, out=(out[0][:T - 2 * n], out[1][:T - 2 * n]))
    with pytest.raises(StageError, match="out of range"):
        cache.check()
    assert torch.equal(out[0][:T - 2 * n], k[:T - 2 * n]) and bool((out[0][T - 2 * n:] == 7).all())
    assert torch.equal(out[1][:T - 2 * n], v[:T - 2 * n]) and bool((out[1][T - 2 * n:] == 7).all())
