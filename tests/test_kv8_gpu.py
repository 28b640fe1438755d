"""The 8-bit KV cache on the GPU against its definition in 64 bits
(tests/kv8_util.py): the write with every rotary form, the read-back, the
attention over it, and a decoder layer's run of all three."""
import math

import numpy as np
import pytest

from hllm_b200 import _lib
from hllm_b200._lib import StageError
from tests import kv8_util
from tests.gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

SCALINGS = {"none": None, "linear": {"type": "linear", "factor": 4.0},
            "llama3": {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                       "high_freq_factor": 4.0, "original_max_position": 8192},
            "yarn": {"type": "yarn", "factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0,
                     "original_max_position": 32768}}


@pytest.fixture(scope="module")
def torch():
    return torch_cuda()


@pytest.fixture(scope="module")
def kv8(torch):
    from hllm_b200 import kv8
    return kv8


def ints(torch, values):
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def bytes_of(torch, cache):
    return [t.view(torch.uint8) for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]


def random_cache(torch, kv8, rng, blocks, hkv, d, spread=0.4):
    """A cache whose every row holds codes of a random row."""
    cache = kv8.Cache(blocks, hkv, d)
    kc, ks, vc, vs = bytes_of(torch, cache)
    g = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    for codes, scales in ((kc, ks), (vc, vs)):
        x = torch.randn(codes.shape, device="cuda", generator=g)
        x = x * torch.exp(spread * torch.randn(scales.shape, device="cuda", generator=g))[..., None]
        e = torch.ceil(torch.log2(x.abs().amax(-1) / 448)).clamp(-24, 39)
        codes.copy_((x / torch.exp2(e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8))
        scales.copy_((e + 127).to(torch.uint8))
    return cache


def tables_for(torch, rng, needs, blocks):
    perm = rng.permutation(blocks)[:sum(needs)]
    table = np.full((len(needs), max(1, max(needs))), -1, np.int32)
    at = 0
    for r, n in enumerate(needs):
        table[r, :n] = perm[at:at + n]
        at += n
    return table


# ----------------------------------------------------------------------------- write
def check_write(torch, kv8, hq, hkv, d, rot, inter, scaling, dtype, norm, positions, slots, blocks,
                seed=0, theta=1e6, qkv=None):
    rng = np.random.default_rng(seed)
    T = len(positions)
    x = rng.standard_normal((T, (hq + 2 * hkv) * d)) if qkv is None else qkv
    xd = torch.tensor(x, device="cuda").to(dtype)
    x = xd.double().cpu().numpy().reshape(T, -1, d)
    qn, kn = ((1 + 0.1 * rng.standard_normal((2, d))).astype(np.float32) if norm else (None, None))
    cache = random_cache(torch, kv8, rng, blocks, hkv, d)
    before = [t.cpu().numpy() for t in bytes_of(torch, cache)]
    rope = kv8.Rope(d, theta, rotary_dim=rot, interleaved=inter, scaling=scaling)
    dev = lambda w: None if w is None else torch.tensor(w, device="cuda")  # noqa: E731
    q = kv8.write(cache, xd, ints(torch, positions), ints(torch, slots), rope, q_norm=dev(qn),
                  k_norm=dev(kn), eps=1e-6)
    cache.check()
    f, factor = kv8_util.frequencies(rot, theta, scaling)
    pos = np.asarray(positions)
    yq = kv8_util.normed_rotated(x[:, :hq], pos, qn, 1e-6, rot, f, factor, inter)
    yk = kv8_util.normed_rotated(x[:, hq:hq + hkv], pos, kn, 1e-6, rot, f, factor, inter)
    yv = x[:, hq + hkv:]
    # The F32 chain (norm: a sum of d squares over lanes, a root, a quotient, two products; the
    # angle's sine and cosine to 2 ulp, the factor; two products and a sum) is under 32 roundings
    # of 2^-24, on values of at most 2 max |row|.  F16 rounds by 2^-11, or half of 2^-24.
    top = np.abs(yq).max(-1, keepdims=True)
    got = q.double().cpu().numpy().reshape(T, hq, d)
    tol = 2.0 ** -11 * np.abs(yq) + 2.0 ** -25 + 32 * 2.0 ** -24 * 2 * top
    assert np.all(np.abs(got - yq) <= tol), np.max(np.abs(got - yq) / tol)
    after = [t.cpu().numpy() for t in bytes_of(torch, cache)]
    table = kv8_util.e4m3_values()
    touched = np.zeros((blocks, 16), bool)
    for t, slot in enumerate(slots):
        if slot < 0:
            continue
        b, o = divmod(int(slot), 16)
        touched[b, o] = True
        for h in range(hkv):
            for y, codes, scales in ((yk[t, h], after[0], after[1]), (yv[t, h], after[2], after[3])):
                e = int(scales[b, h, o]) - 127
                top = np.abs(y).max()
                slack = 64 * 2.0 ** -24 * top
                assert -24 <= e <= 39
                assert top - slack <= 448 * 2.0 ** e
                assert e == -24 or top + slack > 224 * 2.0 ** e
                z = np.abs(y) * 2.0 ** -e
                # Half a step of e4m3: 2^-4 of the value, or 2^-10 below its least normal.
                tol = np.maximum(2.0 ** -4 * z, 2.0 ** -10) * 2.0 ** e + slack
                assert np.all(np.abs(table[codes[b, h, o]] * 2.0 ** e - y) <= tol)
    for a, b in zip(after, before):
        keep = ~touched
        moved = np.swapaxes(a, 1, 2)[keep] != np.swapaxes(b, 1, 2)[keep]
        assert not moved.any()
    # Values go in as they are: the codes are the one right rounding of each.
    for t, slot in enumerate(slots):
        if slot >= 0:
            b, o = divmod(int(slot), 16)
            for h in range(hkv):
                e = kv8_util.exponent(np.abs(yv[t, h]).max())
                assert int(after[3][b, h, o]) == e + 127
                np.testing.assert_array_equal(table[after[2][b, h, o]],
                                              kv8_util.e4m3_round(yv[t, h] * 2.0 ** -e))


@pytest.mark.parametrize("heads", [(32, 8, 128), (4, 2, 64), (6, 2, 256), (3, 1, 32), (5, 5, 96),
                                   (4, 1, 192), (2, 2, 224), (2, 1, 160)])
@pytest.mark.parametrize("inter", [False, True])
def test_write_head_sizes(torch, kv8, heads, inter):
    hq, hkv, d = heads
    rng = np.random.default_rng(d + inter)
    for T, rot, dtype, norm in ((1, d, torch.float32, True), (37, d // 2, torch.float16, False),
                                (18, d - 2, torch.bfloat16, True), (5, 2, torch.float32, False),
                                (2, d // 4, torch.float16, True)):
        slots = rng.choice(8 * 16, T, replace=False)
        check_write(torch, kv8, hq, hkv, d, rot, inter, None, dtype, norm,
                    rng.integers(0, 4000, T), slots, 8, seed=T)


@pytest.mark.parametrize("name", SCALINGS)
@pytest.mark.parametrize("inter", [False, True])
def test_write_scaled_positions_near_and_far(torch, kv8, name, inter):
    positions = [0, 1, 15, 16, 4095, 8191, 8192, 32767, 131071, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1]
    slots = np.random.default_rng(3).choice(64, len(positions), replace=False)
    check_write(torch, kv8, 4, 2, 128, 128, inter, SCALINGS[name], torch.float32, True, positions,
                slots, 4, theta=500000.0)


def test_write_many_tokens_and_padding(torch, kv8):
    """More tokens than one CTA a head takes, tokens without a slot among them."""
    rng = np.random.default_rng(5)
    T = 700
    slots = rng.choice(64 * 16, T, replace=False)
    slots[rng.random(T) < 0.1] = -1
    for hq, hkv, d in ((4, 2, 64), (3, 1, 128)):
        check_write(torch, kv8, hq, hkv, d, d, False, None, torch.float16, True,
                    rng.integers(0, 9000, T), slots, 64, seed=6)


def test_write_special_values(torch, kv8):
    """Zeros, borders of the scale, subnormals, and values that no code stands for."""
    d = 64
    rows = [np.zeros(d)]
    for k in (-24, -23, -3, 0, 7, 39):
        top = np.float32(448.0 * 2.0 ** k)
        rows += [np.full(d, x) for x in (top, np.nextafter(top, np.float32(0)), -top)]
        if k < 39:
            rows.append(np.full(d, np.nextafter(top, np.float32(np.inf))))
    rows.append(np.full(d, 1e-38))
    rows.append(np.float32(2.0) ** -np.arange(d))
    rows.append(np.float32(2.0) ** np.arange(d) * np.float32(2.0 ** -20))
    qkv = np.stack([np.concatenate([np.zeros(2 * d), r]) for r in rows]).astype(np.float32)
    T = len(rows)
    check_write(torch, kv8, 1, 1, d, d, False, None, torch.float32, False, [0] * T, list(range(T)),
                (T + 15) // 16, qkv=qkv)
    # Not finite, or past 448 * 2^39: NaN, and the others of the row as if it were not there.
    bad = [np.nan, np.inf, -np.inf, np.nextafter(np.float32(448.0 * 2.0 ** 39), np.float32(np.inf)), 3e38]
    x = np.zeros((len(bad), 3 * d), np.float32)
    rest = np.linspace(-3, 5, d).astype(np.float32)
    x[:, 2 * d:] = rest
    for i, b in enumerate(bad):
        x[i, 2 * d + 7] = b
    cache = kv8.Cache(1, 1, d)
    kv8.write(cache, torch.tensor(x, device="cuda"), ints(torch, [0] * 5), ints(torch, range(5)),
              kv8.Rope(d, 1e4))
    cache.check()
    e = kv8_util.exponent(5.0)
    for i in range(len(bad)):
        row = kv8_util.e4m3_values()[cache.v.view(torch.uint8)[0, 0, i].cpu().numpy()]
        assert int(cache.v_scale.view(torch.uint8)[0, 0, i]) == e + 127
        assert np.isnan(row[7])
        want = kv8_util.e4m3_round(rest.astype(np.float64) * 2.0 ** -e)
        np.testing.assert_array_equal(np.delete(row, 7), np.delete(want, 7))


def test_write_reports_and_skips_slots_out_of_range(torch, kv8):
    cache = kv8.Cache(2, 1, 64)
    x = torch.randn((4, 3 * 64), device="cuda")
    kv8.write(cache, x, ints(torch, [1, 2, 3, 4]), ints(torch, [5, 32, 2 ** 31 - 1, -7]),
              kv8.Rope(64, 1e4))
    used = cache.v.view(torch.uint8).reshape(32, 64).any(-1).nonzero().flatten().tolist()
    assert used == [5]
    with pytest.raises(StageError) as e:
        cache.check()
    assert e.value.code == _lib.INTERNAL and "out of range" in e.value.message
    cache.check()


# ----------------------------------------------------------------------------- read
@pytest.mark.parametrize("heads", [(2, 64), (8, 128), (1, 32), (3, 96), (2, 256)])
@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_read_is_exact(torch, kv8, heads, kind):
    hkv, d = heads
    rng = np.random.default_rng(d)
    dtype = getattr(torch, kind)
    lengths = [1, 16, 0, 17, 100, 33, 15] + [int(x) for x in rng.integers(0, 40, 40)]
    first = [0, 3, 0, 17, 50, 32, 14] + [int(rng.integers(0, n + 1)) for n in lengths[7:]]
    needs = [(n + 15) // 16 for n in lengths]
    blocks = sum(needs) + 3
    cache = random_cache(torch, kv8, rng, blocks, hkv, d, spread=1.5)
    table = tables_for(torch, rng, needs, blocks)
    for use_first in (True, False):
        begin = first if use_first else [0] * len(lengths)
        n = [e - f for e, f in zip(lengths, begin)]
        cu = np.concatenate([[0], np.cumsum(n)])
        total = int(cu[-1])
        out = tuple(torch.full((total + 5, hkv, d), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        kv8.read(cache, ints(torch, table), ints(torch, lengths), ints(torch, cu), total + 5,
                 first=ints(torch, first) if use_first else None, dtype=dtype, out=out)
        cache.check()
        kc, ks, vc, vs = bytes_of(torch, cache)
        for got, codes, scales in ((out[0], kc, ks), (out[1], vc, vs)):
            value = kv8_util.values(torch, codes, scales).float()  # exact: 4 bits and a power of two
            for r, e in enumerate(lengths):
                for p in range(begin[r], e):
                    want = value[table[r, p // 16], :, p % 16].to(dtype)
                    assert torch.equal(got[cu[r] + p - begin[r]], want)
            assert bool((got[total:] == 7).all())


def test_read_reports_missing_pages(torch, kv8):
    rng = np.random.default_rng(0)
    cache = random_cache(torch, kv8, rng, 4, 2, 64)
    table = ints(torch, [[1, -1, 4]])
    k, v = kv8.read(cache, table, ints(torch, [48]), ints(torch, [0, 48]), 48)
    for x in (k, v):
        assert bool(x[:16].any(-1).all()) and not x[16:].any()
    with pytest.raises(StageError):
        cache.check()


# ----------------------------------------------------------------------------- attention
def reference(torch, cache, table, rows, q, hq, scale=None):
    """(o, tolerance) of a packed batch; rows: (keys, new tokens)."""
    hkv, d = cache.kv_heads, cache.head_dim
    kc, ks, vc, vs = bytes_of(torch, cache)
    out, tol, t = [], [], 0
    for r, (n, count) in enumerate(rows):
        pages = torch.as_tensor(table[r, :(n + 15) // 16], device="cuda").long()
        k, v = (kv8_util.values(torch, c[pages], s[pages]).transpose(1, 2).reshape(-1, hkv, d)[:n]
                for c, s in ((kc, ks), (vc, vs)))
        o, e = kv8_util.attend(torch, k, v, q[t:t + count].double().view(count, hq, d),
                               np.arange(n - count, n), 1 / math.sqrt(d) if scale is None else scale)
        out.append(o.view(count, hq * d))
        tol.append(e.view(count, hq * d))
        t += count
    return torch.cat(out), torch.cat(tol)


def check_attention(torch, kv8, hq, hkv, d, rows, seed=0, spread=0.4, cache=None, table=None,
                    sharp=1.5, scale=None, max_tokens=None):
    rng = np.random.default_rng(seed)
    needs = [(n + 15) // 16 for n, _ in rows]
    if cache is None:
        blocks = sum(needs) + 3
        cache = random_cache(torch, kv8, rng, blocks, hkv, d, spread)
        table = tables_for(torch, rng, needs, blocks)
    counts = [c for _, c in rows]
    T = sum(counts)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (sharp * torch.randn((T, hq * d), device="cuda", generator=g)).half()
    cu = np.concatenate([[0], np.cumsum(counts)])
    most = max(counts) if max_tokens is None else max_tokens
    got = kv8.attention(cache, q, ints(torch, cu), ints(torch, [n for n, _ in rows]),
                        ints(torch, table), max_tokens=most, scale=scale)
    cache.check()
    want, tol = reference(torch, cache, table, rows, q, hq, scale)
    err = (got.double() - want).abs() / tol
    # F16 ends at 65504: 65520, half a step of 32 above it, and more round to infinity.
    err[(want.abs() + tol >= 65520) & (got.double() == want.sign() * math.inf)] = 0
    assert bool((err <= 1).all()), (float(err.max()), int((err > 1).sum()), got.numel())
    return got


HEADS = [(32, 8, 128), (8, 8, 64), (4, 2, 64), (6, 2, 256), (3, 1, 32), (12, 4, 96), (4, 4, 160),
         (7, 1, 192), (2, 1, 224), (16, 1, 128), (20, 1, 64), (9, 1, 256)]


@pytest.mark.parametrize("heads", HEADS)
def test_decode_short_rows(torch, kv8, heads):
    """Lengths from none to a few pages, ends inside, at and after a page."""
    rows = [(n, 1) for n in (1, 2, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 100)]
    check_attention(torch, kv8, *heads, rows, seed=heads[2])


@pytest.mark.parametrize("heads", HEADS)
def test_decode_one_row_each_length(torch, kv8, heads):
    for n in (0, 1, 16, 130, 1000):
        check_attention(torch, kv8, *heads, [(n, 1)], seed=n)


@pytest.mark.parametrize("heads", [(32, 8, 128), (4, 2, 64), (6, 2, 256), (16, 1, 128)])
def test_decode_ragged_batches(torch, kv8, heads):
    rng = np.random.default_rng(1)
    check_attention(torch, kv8, *heads, [(int(n), 1) for n in np.exp(rng.uniform(0, 8, 50))], seed=2)
    # More rows than one scan of 128, some of them without tokens.
    rows = [(int(n), int(rng.random() < 0.8)) for n in rng.integers(0, 300, 300)]
    check_attention(torch, kv8, *heads, rows, seed=3)


@pytest.mark.parametrize("heads,n", [((2, 1, 128), 70001), ((4, 2, 64), 131072), ((1, 1, 256), 33333)])
def test_decode_long_rows(torch, kv8, heads, n):
    check_attention(torch, kv8, *heads, [(n, 1), (5, 1)], seed=4)


@pytest.mark.parametrize("heads", HEADS)
def test_chunks_and_mixes(torch, kv8, heads):
    """Chunks at the start, behind earlier keys, of one token and of many, and
    rows that leave early tokens no key (more new tokens than keys)."""
    rows = [(5, 5), (40, 1), (17, 16), (130, 70), (0, 1), (64, 33), (3, 7), (200, 2), (0, 4), (257, 129)]
    check_attention(torch, kv8, *heads, rows, seed=5)


@pytest.mark.parametrize("heads", [(32, 8, 128), (8, 2, 64), (16, 8, 128), (8, 8, 64), (8, 1, 128),
                                   (4, 4, 128), (6, 2, 128)])
@pytest.mark.parametrize("rows", [[(512, 512)], [(1536, 512)], [(300, 300), (1, 1), (700, 128), (900, 129)],
                                  [(2049, 65), (128, 128), (127, 127), (129, 129)],
                                  [(4000, 40), (4000, 33), (100, 32)]], ids=str)
def test_prompt_chunks(torch, kv8, heads, rows):
    check_attention(torch, kv8, *heads, rows, seed=6)


@pytest.mark.parametrize("heads", [(8, 2, 128), (2, 1, 64), (3, 1, 256)])
def test_one_key_decides(torch, kv8, heads):
    """A query along one key's direction: the output is that key's value, so a
    key that is dropped, doubled or misplaced shows whole."""
    hq, hkv, d = heads
    rng = np.random.default_rng(8)
    for n in (1, 16, 17, 97, 1000):
        needs = [(n + 15) // 16]
        cache = random_cache(torch, kv8, rng, needs[0] + 2, hkv, d)
        table = tables_for(torch, rng, needs, needs[0] + 2)
        kc, ks, vc, vs = bytes_of(torch, cache)
        pages = torch.as_tensor(table[0], device="cuda").long()
        k = kv8_util.values(torch, kc[pages], ks[pages]).transpose(1, 2).reshape(-1, hkv, d)
        v = kv8_util.values(torch, vc[pages], vs[pages]).transpose(1, 2).reshape(-1, hkv, d)
        keys = sorted({0, n // 2, n - 1, min(15, n - 1), min(16, n - 1)})
        for j in keys:
            unit = k[j] / k[j].pow(2).sum(-1, keepdim=True)
            q = (unit * 900).repeat_interleave(hq // hkv, 0).reshape(1, hq * d).half()
            got = kv8.attention(cache, q, ints(torch, [0, 1]), ints(torch, [n]), ints(torch, table),
                                max_tokens=1, scale=1.0)
            want, tol = reference(torch, cache, table, [(n, 1)], q, hq, 1.0)
            assert bool(((got.double() - want).abs() <= tol).all())
            alone = v[j].repeat_interleave(hq // hkv, 0).reshape(1, -1)
            if float((want - alone).abs().max()) < 1e-3:
                assert float((got.double() - alone).abs().max()) <= 1e-3 + 2.0 ** -10 * float(alone.abs().max())
    cache.check()


@pytest.mark.parametrize("count", [1, 3, 80])
def test_rows_of_very_different_size(torch, kv8, count):
    """K and V rows from 2^-20 to 2^12 times their neighbours, sizes of V that
    oppose the weights, and a large scale."""
    check_attention(torch, kv8, 8, 2, 128, [(500, count), (90, min(count, 90))], seed=9, spread=3.0)
    check_attention(torch, kv8, 4, 2, 64, [(700, count)], seed=10, spread=4.0, sharp=0.2)


@pytest.mark.parametrize("count", [1, 2, 100])
def test_what_lies_past_the_last_key_is_not_read(torch, kv8, count):
    """NaN codes and scales in the last page's free rows, in pages that no
    table names, and table entries past the last page."""
    rng = np.random.default_rng(11)
    for hq, hkv, d in ((8, 2, 128), (4, 2, 64), (3, 1, 256)):
        for n in (count + 1, 130, 200):
            needs = [(n + 15) // 16]
            blocks = needs[0] + 4
            cache = random_cache(torch, kv8, rng, blocks, hkv, d)
            table = tables_for(torch, rng, needs, blocks)
            wide = np.full((1, needs[0] + 20), 10 ** 9, np.int32)
            wide[:, :needs[0]] = table
            rows = [(n, min(count, n))]
            clean = check_attention(torch, kv8, hq, hkv, d, rows, seed=12, cache=cache, table=table)
            free = np.ones((blocks, 16), bool)
            for p in range(n):
                free[table[0, p // 16], p % 16] = False
            mask = torch.as_tensor(free, device="cuda")[:, None].expand(blocks, hkv, 16)
            for t in bytes_of(torch, cache):
                t[mask] = 255
            g = torch.Generator(device="cuda").manual_seed(12)
            q = (1.5 * torch.randn((rows[0][1], hq * d), device="cuda", generator=g)).half()
            got = kv8.attention(cache, q, ints(torch, [0, rows[0][1]]), ints(torch, [n]),
                                ints(torch, wide), max_tokens=rows[0][1])
            cache.check()
            assert torch.equal(got, clean)


@pytest.mark.parametrize("count", [1, 70])
def test_nan_in_a_seen_key_reaches_its_heads_alone(torch, kv8, count):
    rng = np.random.default_rng(13)
    hq, hkv, d, n = 8, 2, 128, 150
    for which in (0, 2):
        cache = random_cache(torch, kv8, rng, 12, hkv, d)
        table = tables_for(torch, rng, [10], 12)
        q = torch.randn((count, hq * d), device="cuda").half()
        args = (ints(torch, [0, count]), ints(torch, [n]), ints(torch, table))
        clean = kv8.attention(cache, q, *args, max_tokens=count)
        bytes_of(torch, cache)[which][table[0, 2], 1, 3, 5] = 0x7f  # key 35 of kv head 1
        got = kv8.attention(cache, q, *args, max_tokens=count).view(count, hq, d)
        assert torch.equal(got[:, :4], clean.view(count, hq, d)[:, :4])
        seen = torch.arange(n - count, n, device="cuda") >= 35
        if which == 0:
            assert bool(got[seen, 4:].isnan().all())
        else:
            assert bool(got[seen][:, 4:, 5].isnan().all())


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 64)])
def test_many_chunks(torch, kv8, heads):
    """More chunk rows than are looked at together, of any order of lengths,
    among single tokens and rows without any."""
    rng = np.random.default_rng(34)
    counts = rng.choice([0, 1, 3, 16, 17, 40, 64, 129], 75)
    rows = [(int(c + rng.integers(0, 300)), int(c)) for c in counts]
    check_attention(torch, kv8, *heads, rows, seed=35)
    check_attention(torch, kv8, *heads, [(n, c) for n, c in rows if c >= 16][:40], seed=36)


@pytest.mark.parametrize("d", [64, 128])
def test_two_query_tiles_a_cta(torch, kv8, d):
    """Enough columns for CTAs of two query tiles: sharp and flat scores, weights
    far below the largest, rows that begin before the first key, a NaN key."""
    hq, hkv = 16, 8
    for sharp, rows in ((0.01, [(1500, 1300), (700, 700)]), (1.5, [(2300, 2000), (90, 130), (40, 1)]),
                        (40.0, [(1900, 1900), (1, 1)])):
        check_attention(torch, kv8, hq, hkv, d, rows, seed=21, sharp=sharp, spread=3.0)
    rng = np.random.default_rng(22)
    n, count = 2600, 2500
    cache = random_cache(torch, kv8, rng, 170, hkv, d)
    table = tables_for(torch, rng, [163], 170)
    q = torch.randn((count, hq * d), device="cuda").half()
    args = (ints(torch, [0, count]), ints(torch, [n]), ints(torch, table))
    clean = kv8.attention(cache, q, *args)
    bytes_of(torch, cache)[0][table[0, 2], 1, 3, 5] = 0x7f  # key 35 of kv head 1: all tokens see it
    got = kv8.attention(cache, q, *args).view(count, hq, d)
    keep = [h for h in range(hq) if h // 2 != 1]
    assert torch.equal(got[:, keep], clean.view(count, hq, d)[:, keep])
    assert bool(got[:, 2:4].isnan().all())


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 2, 64), (3, 1, 96)])
def test_strided_rows_and_rows_of_no_sequence(torch, kv8, heads):
    hq, hkv, d = heads
    rng = np.random.default_rng(14)
    rows = [(40, 1), (90, 70), (33, 1)]
    blocks = 16
    cache = random_cache(torch, kv8, rng, blocks, hkv, d)
    table = tables_for(torch, rng, [3, 6, 3], blocks)
    T = 72
    wide = torch.randn((T + 9, hq * d + 24), device="cuda").half()
    q = wide[:, 8:8 + hq * d]
    store = torch.full((T + 9, hq * d + 40), 5.0, dtype=torch.float16, device="cuda")
    out = store[:, 16:16 + hq * d]
    args = (ints(torch, [2, 3, 73, 74]), ints(torch, [40, 90, 33]), ints(torch, table))
    kv8.attention(cache, q, *args, max_tokens=70, out=out)
    cache.check()
    want, tol = reference(torch, cache, table, rows, q[2:74], hq)
    assert bool(((out[2:74].double() - want).abs() <= tol).all())
    assert bool((out[:2] == 5).all() and (out[74:] == 5).all())
    assert bool((store[:, :16] == 5).all() and (store[:, 16 + hq * d:] == 5).all())
    plain = kv8.attention(cache, q.contiguous(), *args, max_tokens=70)
    assert torch.equal(plain[2:74], out[2:74])


def test_rows_out_of_bounds_are_reported_and_skipped(torch, kv8):
    rng = np.random.default_rng(15)
    hq, hkv, d = 4, 2, 64
    cache = random_cache(torch, kv8, rng, 16, hkv, d)
    table = tables_for(torch, rng, [4, 4, 4], 16)
    q = torch.randn((12, hq * d), device="cuda").half()
    good = ([0, 4, 8, 12], [64, 64, 64])
    clean = kv8.attention(cache, q, ints(torch, good[0]), ints(torch, good[1]), ints(torch, table),
                          max_tokens=4)
    cache.check()
    for cu, lengths, most, left in (([0, 4, 8, 13], good[1], 5, [8, 9, 10, 11]),
                                    (good[0], [64, 65, 64], 4, [4, 5, 6, 7]),
                                    (good[0], [64, 64, -3], 4, [8, 9, 10, 11]),
                                    ([0, 4, 9, 12], good[1], 4, [4, 5, 6, 7, 8])):
        out = torch.full_like(clean, 9.0)
        kv8.attention(cache, q, ints(torch, cu), ints(torch, lengths), ints(torch, table),
                      max_tokens=most, out=out)
        with pytest.raises(StageError):
            cache.check()
        assert bool((out[left] == 9).all())
        if cu == good[0]:
            rest = [i for i in range(12) if i not in left]
            assert torch.equal(out[rest], clean[rest])
    # A missing page: its keys are left out.
    hole = table.copy()
    hole[1, 3] = -1
    out = kv8.attention(cache, q, ints(torch, good[0]), ints(torch, good[1]), ints(torch, hole),
                        max_tokens=4)
    with pytest.raises(StageError):
        cache.check()
    assert torch.equal(out[:4], clean[:4]) and torch.equal(out[8:], clean[8:])
    assert bool(out.isfinite().all())


def test_pools_past_32_bit_offsets(torch, kv8):
    """Pages whose codes lie past 2^32 bytes of the pool, written, read and attended."""
    hq, hkv, d = 8, 8, 128
    blocks = (5 << 30) // (hkv * 16 * d)
    pool = [torch.empty((blocks, hkv, 16, d), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scale = [torch.empty((blocks, hkv, 16), dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache = kv8.Cache.wrap(pool[0], scale[0], pool[1], scale[1])
    table = np.int32([[blocks - 1, 0, blocks - 2, blocks // 2]])
    n = 60
    slots = [int(table[0, p // 16]) * 16 + p % 16 for p in range(n)]
    x = torch.randn((n, (hq + 2 * hkv) * d), device="cuda")
    q = kv8.write(cache, x, ints(torch, range(n)), ints(torch, slots), kv8.Rope(d, 1e4))
    k, v = kv8.read(cache, ints(torch, table), ints(torch, [n]), ints(torch, [0, n]), n,
                    dtype=torch.float32)
    raw = x.view(n, -1, d)[:, hq + hkv:]
    assert bool(((v - raw).abs() <= 2.0 ** -4 * raw.abs() + 2.0 ** -10 * raw.abs().amax(-1, keepdim=True) / 224).all())
    for count in (1, n):
        got = kv8.attention(cache, q[n - count:], ints(torch, [0, count]), ints(torch, [n]),
                            ints(torch, table), max_tokens=count)
        want, tol = kv8_util.attend(torch, k.double(), v.double(), q[n - count:].double().view(count, hq, d),
                                    np.arange(n - count, n), 1 / math.sqrt(d))
        assert bool(((got.double().view(count, hq, d) - want).abs() <= tol).all())
    cache.check()


# ----------------------------------------------------------------------------- how calls are made
def layer_case(torch, kv8, seed, hq=8, hkv=2, d=128, rows=3, keys=40):
    rng = np.random.default_rng(seed)
    cache = kv8.Cache(rows * 8, hkv, d)
    table = rng.permutation(rows * 8).reshape(rows, 8).astype(np.int32)
    return rng, cache, table


def test_captured_calls_serve_new_lengths(torch, kv8):
    """A captured write + attention replayed for growing rows equals eager calls."""
    hq, hkv, d, rows = 8, 2, 128, 3
    rng, cache, table = layer_case(torch, kv8, 16)
    twin = kv8.Cache(rows * 8, hkv, d)
    rope = kv8.Rope(d, 1e4)
    tab = ints(torch, table)
    x = torch.zeros((rows, (hq + 2 * hkv) * d), device="cuda")
    positions, slots, lengths = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(3))
    cu = ints(torch, range(rows + 1))
    work = [kv8.attention_workspace(rows, rows, 1, hq, hkv, d) for _ in range(2)]
    out = torch.zeros((rows, hq * d), dtype=torch.float16, device="cuda")

    def step(c, w, o):
        q = kv8.write(c, x, positions, slots, rope)
        return kv8.attention(c, q, cu, lengths, tab, max_tokens=1, out=o, workspace=w)
    slots.fill_(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, work[0], out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, work[0], out)
    for p in range(100):
        at = np.array([p, p // 2, min(p, 20)])
        x.copy_(torch.tensor(rng.standard_normal(tuple(x.shape)), device="cuda"))
        positions.copy_(ints(torch, at))
        slots.copy_(ints(torch, [table[r, a // 16] * 16 + a % 16 for r, a in enumerate(at)]))
        lengths.copy_(ints(torch, at + 1))
        graph.replay()
        want = step(twin, work[1], None)
        assert torch.equal(out, want), p
    for a, b in zip(bytes_of(torch, cache), bytes_of(torch, twin)):
        assert torch.equal(a, b)
    cache.check()


def test_a_layers_run_prompt_chunks_then_decode(torch, kv8):
    """Two prompt chunks and then single tokens through write + attention, the
    rows packed together, against 64-bit attention over what the cache holds;
    and the cache read back into F16 pages serves the F16 attention alike."""
    hq, hkv, d, rows = 8, 2, 128, 3
    rng, cache, table = layer_case(torch, kv8, 17)
    rope = kv8.Rope(d, 5e5, scaling=SCALINGS["llama3"])
    norms = [1 + 0.1 * torch.randn(d, device="cuda") for _ in range(2)]
    tab = ints(torch, table)
    held = np.zeros(rows, int)
    for counts in ([37, 1, 16], [20, 44, 1], [1, 1, 1], [1, 1, 1], [1, 0, 30]):
        cu = np.concatenate([[0], np.cumsum(counts)])
        pos = np.concatenate([np.arange(h, h + c) for h, c in zip(held, counts)])
        row = np.repeat(np.arange(rows), counts)
        slots = table[row, pos // 16] * 16 + pos % 16
        x = torch.tensor(rng.standard_normal((len(pos), (hq + 2 * hkv) * d)), device="cuda").half()
        q = kv8.write(cache, x, ints(torch, pos), ints(torch, slots), rope, *norms)
        held = held + counts
        got = kv8.attention(cache, q, ints(torch, cu), ints(torch, held), tab, max_tokens=max(counts))
        cache.check()
        want, tol = reference(torch, cache, table, list(zip(held, counts)), q, hq)
        assert bool(((got.double() - want).abs() <= tol).all())
    # The same keys as F16 pages: values of 4 bits and a power of two are exact there.
    cu = np.concatenate([[0], np.cumsum(held)])
    k, v = kv8.read(cache, tab, ints(torch, held), ints(torch, cu), int(cu[-1]))
    pages = [torch.zeros((rows * 8, hkv, 16, d), dtype=torch.float16, device="cuda") for _ in range(2)]
    for r in range(rows):
        for p in range(held[r]):
            for dst, src in zip(pages, (k, v)):
                dst[table[r, p // 16], :, p % 16] = src[cu[r] + p]
    q = torch.randn((rows, hq * d), device="cuda").half()
    one = ints(torch, [1] * rows)
    splits = ints(torch, np.concatenate([[0], np.cumsum((held + 63) // 64)]))
    none = ints(torch, [0] * (rows + 1))
    out = torch.zeros_like(q)
    status = ints(torch, [0])
    lens, starts, firsts = ints(torch, held), ints(torch, range(rows + 1)), ints(torch, held - 1)
    _lib.check(_lib.lib().hllm_b200_attention(
        q.data_ptr(), pages[0].data_ptr(), pages[1].data_ptr(), firsts.data_ptr(), one.data_ptr(),
        starts.data_ptr(), lens.data_ptr(), tab.data_ptr(), splits.data_ptr(), none.data_ptr(), rows,
        int(splits[-1]), 0, hq, hkv, d, 8, 64, out.data_ptr(), hq * d, rows, rows * 8,
        status.data_ptr(), torch.cuda.current_stream().cuda_stream))
    got = kv8.attention(cache, q, starts, lens, tab, max_tokens=1)
    want, tol = reference(torch, cache, table, [(n, 1) for n in held], q, hq)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert bool(((out.double() - want).abs() <= 2 * tol).all())
    assert int(status) == 0


def test_streams_repeats_and_workspaces(torch, kv8):
    """The same call on other streams at once, each with its workspace, gives
    the same bits; so does a workspace full of NaN."""
    rng = np.random.default_rng(18)
    hq, hkv, d = 16, 4, 128
    rows = [(700, 1), (2000, 90), (1, 1), (300, 5)]
    cache = random_cache(torch, kv8, rng, 220, hkv, d)
    table = tables_for(torch, rng, [(n + 15) // 16 for n, _ in rows], 220)
    T = sum(c for _, c in rows)
    q = torch.randn((T, hq * d), device="cuda").half()
    args = (ints(torch, np.concatenate([[0], np.cumsum([c for _, c in rows])])),
            ints(torch, [n for n, _ in rows]), ints(torch, table))
    first = kv8.attention(cache, q, *args, max_tokens=90)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    spaces = [kv8.attention_workspace(len(rows), T, 90, hq, hkv, d).fill_(255) for _ in streams]
    outs = [torch.empty_like(first) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, w, o in zip(streams, spaces, outs):
            with torch.cuda.stream(s):
                kv8.attention(cache, q, *args, max_tokens=90, out=o, workspace=w)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)
    cache.check()


def test_write_in_one_call_or_many(torch, kv8):
    """How a call's tokens and heads are spread over warps leaves no trace."""
    rng = np.random.default_rng(30)
    T, hq, hkv, d = 11000, 3, 1, 64
    x = torch.randn((T, (hq + 2 * hkv) * d), device="cuda").bfloat16()
    positions = ints(torch, rng.integers(0, 1 << 20, T))
    slots = ints(torch, rng.permutation(700 * 16)[:T])
    norm = torch.rand(d, device="cuda") + 0.5
    for rope, norms in ((kv8.Rope(d, 1e4), dict(q_norm=norm)),
                        (kv8.Rope(d, 1e4, rotary_dim=40, interleaved=True), dict(k_norm=norm)),
                        (kv8.Rope(d, 1e4, rotary_dim=24), {})):
        one, many = kv8.Cache(700, hkv, d), kv8.Cache(700, hkv, d)
        q = kv8.write(one, x, positions, slots, rope, **norms)
        got = torch.empty_like(q)
        at = 0
        for n in (1, 2, 5, 60, 400, 1500, T - 1968):
            part = slice(at, at + n)
            kv8.write(many, x[part], positions[part], slots[part], rope, out=got[part], **norms)
            at += n
        assert at == T and torch.equal(got, q)
        for a, b in zip(bytes_of(torch, one), bytes_of(torch, many)):
            assert torch.equal(a, b)


def test_read_of_many_rows(torch, kv8):
    """Rows without tokens, and several rows to a CTA's tokens, past 256 rows."""
    rng = np.random.default_rng(31)
    hkv, d = 2, 64
    lengths = np.where(rng.random(700) < 0.5, 0, rng.integers(0, 40, 700))
    first = np.minimum(rng.integers(0, 3, 700), lengths)
    needs = [(int(n) + 15) // 16 for n in lengths]
    cache = random_cache(torch, kv8, rng, sum(needs), hkv, d)
    table = tables_for(torch, rng, needs, sum(needs))
    offsets = 5 + np.concatenate([[0], np.cumsum(lengths - first)])
    T = int(offsets[-1]) + 9
    out = tuple(torch.full((T, hkv, d), 7.0, device="cuda") for _ in range(2))
    kv8.read(cache, ints(torch, table), ints(torch, lengths), ints(torch, offsets), T,
             first=ints(torch, first), dtype=torch.float32, out=out)
    cache.check()
    kc, ks, vc, vs = bytes_of(torch, cache)
    row = np.repeat(np.arange(700), lengths - first)
    at = np.arange(len(row)) - (offsets[:-1] - 5)[row] + first[row]
    page, line = torch.as_tensor(table[row, at // 16]).long().cuda(), torch.as_tensor(at % 16).cuda()
    for c, s, o in ((kc, ks, out[0]), (vc, vs, out[1])):
        values = kv8_util.values(torch, c, s).transpose(1, 2)  # [page][16][head][d]
        want = torch.full((T, hkv, d), 7.0, device="cuda", dtype=torch.float64)
        want[5:5 + len(row)] = values[page, line]
        assert torch.equal(o.double(), want)


def test_tokens_without_a_page(torch, kv8):
    """Rows all of whose keys lie on missing pages give zeros, others what they see."""
    rng = np.random.default_rng(32)
    for hq, hkv, d, count in ((8, 2, 128, 1), (8, 2, 128, 90), (4, 2, 64, 40), (4, 4, 96, 3)):
        rows = [(200, count), (150, count), (0, 0), (180, count)]
        cache = random_cache(torch, kv8, rng, 40, hkv, d)
        table = tables_for(torch, rng, [13, 10, 0, 12], 40)
        holes = table.copy()
        holes[1] = -1
        holes[3, :] = 40
        T = 3 * count
        q = torch.randn((T, hq * d), device="cuda").half()
        args = (ints(torch, [0, count, 2 * count, 2 * count, T]), ints(torch, [n for n, _ in rows]))
        got = kv8.attention(cache, q, *args, ints(torch, holes), max_tokens=count)
        with pytest.raises(StageError, match="out of range"):
            cache.check()
        want, tol = reference(torch, cache, table, rows, q, hq)
        assert bool(((got.double() - want).abs() <= tol)[:count].all())
        assert bool((got[count:] == 0).all())


def test_a_workspace_serves_smaller_calls(torch, kv8):
    """A workspace for large counts is enough for any smaller ones, whose split
    over CTAs may be finer; and graphs may share one, replayed in turn."""
    rng = np.random.default_rng(33)
    hq, hkv, d = 16, 4, 128
    work = kv8.attention_workspace(64, 1024, 1024, hq, hkv, d)
    cache = random_cache(torch, kv8, rng, 300, hkv, d)
    calls = []
    for rows in ([(4000, 20)], [(700, 1)], [(64, 64)], [(1500, 100), (900, 1)], [(1024, 1024)]):
        table = tables_for(torch, rng, [(n + 15) // 16 for n, _ in rows], 300)
        T = sum(c for _, c in rows)
        q = torch.randn((T, hq * d), device="cuda").half()
        args = (q, ints(torch, np.concatenate([[0], np.cumsum([c for _, c in rows])])),
                ints(torch, [n for n, _ in rows]), ints(torch, table))
        want = kv8.attention(cache, *args)
        out = torch.empty_like(want)
        kv8.attention(cache, *args, out=out, workspace=work)
        assert torch.equal(out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kv8.attention(cache, *args, out=out, workspace=work)
        calls.append((graph, out, want, args))
    for _ in range(3):
        for graph, out, _, _ in calls:
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in calls:
            assert torch.equal(out, want)
    cache.check()


@pytest.mark.parametrize("heads", [(32, 8, 128), (16, 4, 64), (6, 2, 256)])
def test_cold_memory(torch, kv8, heads):
    """Caches, tables and queries that are in no cache of the GPU arrive late:
    many streams a warp, new queries each time, and everything else written
    over in between."""
    hq, hkv, d = heads
    rng = np.random.default_rng(20)
    rows = [(int(n), 1) for n in rng.integers(20, 1500, 64)]
    needs = [(n + 15) // 16 for n, _ in rows]
    cache = random_cache(torch, kv8, rng, sum(needs), hkv, d)
    table = tables_for(torch, rng, needs, sum(needs))
    args = (ints(torch, np.arange(len(rows) + 1)), ints(torch, [n for n, _ in rows]), ints(torch, table))
    sweep = torch.empty(320 << 20, dtype=torch.uint8, device="cuda")
    work = kv8.attention_workspace(len(rows), len(rows), 1, hq, hkv, d)
    for i in range(6):
        q = (1.5 * torch.randn((len(rows), hq * d), device="cuda")).half()
        sweep.fill_(i)
        got = kv8.attention(cache, q, *args, max_tokens=1, workspace=work)
        want, tol = reference(torch, cache, table, rows, q, hq)
        assert bool(((got.double() - want).abs() <= tol).all()), i
    cache.check()


def test_gpu_side_refusals(torch, kv8):
    cache = kv8.Cache(4, 2, 64)
    rope = kv8.Rope(64, 1e4)
    x = torch.zeros((3, 8 * 64), device="cuda")
    p = ints(torch, [0, 1, 2])
    q = torch.zeros((3, 4 * 64), dtype=torch.float16, device="cuda")
    tab, cu, n = ints(torch, [[0, 1]]), ints(torch, [0, 3]), ints(torch, [3])
    small = torch.empty(64, dtype=torch.uint8, device="cuda")
    for call, why in (
            (lambda: kv8.write(cache, x.double(), p, p, rope), "float32"),
            (lambda: kv8.write(cache, x[:, :500], p, p, rope), "rows of 500"),
            (lambda: kv8.write(cache, x[:, :256], p, p, rope), "rows of 256"),
            (lambda: kv8.write(cache, x, p[:2], p, rope), "positions"),
            (lambda: kv8.write(cache, x, p, p.long(), rope), "slots"),
            (lambda: kv8.write(cache, x.cpu(), p, p, rope), "cpu"),
            (lambda: kv8.write(cache, x, p, p, rope, q_norm=torch.ones(63, device="cuda")), "q_norm"),
            (lambda: kv8.write(cache, x, p, p, kv8.Rope(128, 1e4)), "head of 64"),
            (lambda: kv8.write(cache, x, p, p, rope, q_norm=torch.ones(65, device="cuda")[1:]), "aligned"),
            (lambda: kv8.read(cache, tab, n, p, 3), "offsets"),
            (lambda: kv8.read(cache, tab, n, cu, 3, dtype=torch.int8), "dtype"),
            (lambda: kv8.attention(cache, q.float(), cu, n, tab), "float16"),
            (lambda: kv8.attention(cache, q[:, :192], cu, n, tab), "192"),
            (lambda: kv8.attention(cache, q, n, n, tab), "cu_seqlens"),
            (lambda: kv8.attention(cache, q, cu, n, tab, out=q[:2]), "out"),
            (lambda: kv8.attention(cache, q.t().contiguous().t(), cu, n, tab), "contiguous rows"),
            (lambda: kv8.attention(cache, q, cu, n, tab, scale=float("inf")), "scale"),
            (lambda: kv8.attention(cache, q, cu, n, tab, workspace=small), "too small")):
        with pytest.raises(StageError) as e:
            call()
        assert why in e.value.message, e.value.message
        assert e.value.code in (_lib.INVALID_REQUEST, _lib.RESOURCE_EXHAUSTED)
    empty = kv8.attention(cache, q[:0], ints(torch, [0, 0]), n, tab)
    assert tuple(empty.shape) == (0, 256)
    cache.check()
