"""The 8-bit KV cache without a GPU: its number format, the rotary tables, and
what its entry points refuse (before any device call)."""
import ctypes as C

import numpy as np
import pytest

from hllm_b200 import _lib
from hllm_b200._lib import StageError
from tests import kv8_util

SCALINGS = [None, {"type": "linear", "factor": 4.0},
            {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position": 8192.0},
            {"type": "yarn", "factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0,
             "original_max_position": 32768.0},
            {"type": "yarn", "factor": 1.0, "beta_fast": 2.0, "beta_slow": 1.0,
             "original_max_position": 10.0}]
KINDS = {"none": 0, "linear": 1, "llama3": 2, "yarn": 3}


def rope(rot=128, theta=1e6, inter=0, scaling=None, attention=0.0, **more):
    s = {"factor": 1.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "beta_fast": 32.0,
         "beta_slow": 1.0, "original_max_position": 0.0, **(scaling or {"type": "none"}), **more}
    kind = s["type"]
    return _lib.Rope(rot, inter, theta, KINDS.get(kind, kind), s["factor"], s["low_freq_factor"],
                     s["high_freq_factor"], s["beta_fast"], s["beta_slow"],
                     s["original_max_position"], attention)


def turns_of(desc):
    out = (C.c_double * 128)()
    factor = C.c_float()
    st = _lib.lib().hllm_b200_rope_turns(C.byref(desc), out, C.byref(factor))
    return st, np.array(out[:max(0, desc.rotary_dim // 2)]), factor.value


@pytest.mark.parametrize("rot,theta", [(2, 10000.0), (64, 500000.0), (128, 1e6), (20, 1e4)])
@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["type"] if s else "none")
def test_rope_turns_match_the_formulas(rot, theta, scaling):
    st, turns, factor = turns_of(rope(rot, theta, 0, scaling))
    assert st == _lib.OK
    f, m = kv8_util.frequencies(rot, theta, scaling)
    # Both sides are a few roundings of 64-bit values.
    np.testing.assert_allclose(turns * 2 * np.pi, f, rtol=64 * 2.0 ** -53)
    assert factor == np.float32(m)


def test_rope_attention_factor_overrides_the_scalings_own():
    assert turns_of(rope(64, 1e4, 0, SCALINGS[3], attention=1.25))[2] == 1.25
    assert turns_of(rope(64, 1e4, 0, None, attention=0.5))[2] == 0.5


@pytest.mark.parametrize("desc,why", [
    (rope(0), "rotary_dim"), (rope(7), "rotary_dim"), (rope(258), "rotary_dim"),
    (rope(theta=1.0), "theta"), (rope(theta=float("nan")), "theta"),
    (rope(attention=-1.0), "attention_factor"), (rope(scaling={"type": 9}), "unknown"),
    (rope(scaling={"type": "linear"}, factor=0.5), "factor"),
    (rope(scaling={"type": "llama3"}, factor=8.0), "original_max_position"),
    (rope(scaling=SCALINGS[2], low_freq_factor=4.0), "low_freq_factor"),
    (rope(scaling=SCALINGS[3], beta_slow=32.0), "beta_fast"),
    (rope(scaling=SCALINGS[3], beta_fast=float("inf")), "beta_fast")])
def test_rope_refusals(desc, why):
    st, _, _ = turns_of(desc)
    assert st == _lib.INVALID_REQUEST
    assert why in _lib.last_error()


def test_exponent_and_rounding_of_the_restated_format():
    for k in range(-10, 20):
        top = 448.0 * 2.0 ** k
        assert kv8_util.exponent(top) == k
        assert kv8_util.exponent(np.nextafter(top, np.inf)) == k + 1
        assert kv8_util.exponent(np.nextafter(top, 0)) == k
    assert kv8_util.exponent(0.0) == -24 and kv8_util.exponent(1e-30) == -24
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).standard_normal(20000) * 10.0 ** np.random.default_rng(1).uniform(-5, 2, 20000)
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn)
    np.testing.assert_array_equal(kv8_util.e4m3_round(x.astype(np.float64)), want.double().numpy())
    codes = torch.arange(256, dtype=torch.uint8)
    np.testing.assert_array_equal(kv8_util.e4m3_values(),
                                  codes.view(torch.float8_e4m3fn).double().numpy())


# Addresses that no call may touch: every refusal comes before the device is asked.
A = 1 << 20


def cache(**more):
    d = {"k_codes": A, "k_scales": A, "v_codes": A, "v_scales": A, "blocks": 8, "kv_heads": 2,
         "head_dim": 64, **more}
    return _lib.KV8(*d.values())


BAD_CACHES = [({"k_codes": None}, "null"), ({"v_scales": None}, "null"), ({"v_codes": A + 8}, "aligned"),
              ({"k_scales": A + 1}, "aligned"), ({"head_dim": 0}, "head_dim"),
              ({"head_dim": 48}, "head_dim"), ({"head_dim": 288}, "head_dim"),
              ({"kv_heads": 0}, "kv_heads"), ({"blocks": 0}, "blocks"),
              ({"blocks": 1 << 27}, "blocks")]


def write_args(**more):
    d = dict(qkv=A, dtype=_lib.F32, tokens=3, hq=4, positions=A, slots=A, q_norm=None, k_norm=None,
             eps=1e-6, turns=A, rotary=64, inter=0, factor=1.0, q_out=A, status=A, stream=None)
    d.update(more)
    return list(d.values())


def read_args(**more):
    d = dict(tables=A, rows=2, max_blocks=4, first=None, lengths=A, offsets=A, tokens=5,
             dtype=_lib.F16, k=A, v=A, status=A, stream=None)
    d.update(more)
    return list(d.values())


def attention_args(**more):
    d = dict(q=A, ld_q=256, cu=A, lengths=A, tables=A, rows=2, tokens=5, most=4, hq=4, max_blocks=4,
             scale=0.125, out=A, ld_out=256, workspace=A, bytes=1 << 40, status=A, stream=None)
    d.update(more)
    return list(d.values())


CALLS = {"hllm_b200_kv8_write": write_args, "hllm_b200_kv8_read": read_args,
         "hllm_b200_kv8_attention": attention_args}


@pytest.mark.parametrize("name", CALLS)
def test_bad_caches_are_refused(name):
    f = getattr(_lib.lib(), name)
    assert f(None, *CALLS[name]()) == _lib.INVALID_REQUEST
    for more, why in BAD_CACHES:
        assert f(C.byref(cache(**more)), *CALLS[name]()) == _lib.INVALID_REQUEST, more
        assert why in _lib.last_error()


@pytest.mark.parametrize("name,more,why", [
    ("hllm_b200_kv8_write", {"hq": 0}, "query heads"), ("hllm_b200_kv8_write", {"hq": 3}, "query heads"),
    ("hllm_b200_kv8_write", {"dtype": 7}, "F32"), ("hllm_b200_kv8_write", {"tokens": 1 << 31}, "tokens"),
    ("hllm_b200_kv8_write", {"rotary": 66}, "rotary"), ("hllm_b200_kv8_write", {"rotary": 7}, "rotary"),
    ("hllm_b200_kv8_write", {"eps": -1.0}, "eps"), ("hllm_b200_kv8_write", {"eps": float("nan")}, "eps"),
    ("hllm_b200_kv8_write", {"factor": float("inf")}, "factor"),
    ("hllm_b200_kv8_write", {"status": None}, "status"), ("hllm_b200_kv8_write", {"qkv": None}, "null"),
    ("hllm_b200_kv8_write", {"turns": None}, "null"), ("hllm_b200_kv8_write", {"slots": None}, "null"),
    ("hllm_b200_kv8_write", {"qkv": A + 4}, "aligned"), ("hllm_b200_kv8_write", {"q_out": A + 2}, "aligned"),
    ("hllm_b200_kv8_read", {"dtype": 3}, "output"), ("hllm_b200_kv8_read", {"tokens": 1 << 31}, "tokens"),
    ("hllm_b200_kv8_read", {"rows": 1 << 31}, "rows"), ("hllm_b200_kv8_read", {"max_blocks": 0}, "null"),
    ("hllm_b200_kv8_read", {"offsets": None}, "null"), ("hllm_b200_kv8_read", {"v": A + 8}, "aligned"),
    ("hllm_b200_kv8_read", {"status": None}, "status"),
    ("hllm_b200_kv8_attention", {"hq": 5}, "query heads"),
    ("hllm_b200_kv8_attention", {"ld_q": 248}, "strides"),
    ("hllm_b200_kv8_attention", {"ld_out": 260}, "strides"),
    ("hllm_b200_kv8_attention", {"scale": float("nan")}, "scale"),
    ("hllm_b200_kv8_attention", {"max_blocks": 1 << 30}, "max_blocks"),
    ("hllm_b200_kv8_attention", {"max_blocks": 0}, "null"), ("hllm_b200_kv8_attention", {"most": 0}, "null"),
    ("hllm_b200_kv8_attention", {"workspace": None}, "null"),
    ("hllm_b200_kv8_attention", {"workspace": A + 4}, "aligned"),
    ("hllm_b200_kv8_attention", {"q": A + 8}, "aligned"),
    ("hllm_b200_kv8_attention", {"status": None}, "status")])
def test_bad_arguments_are_refused(name, more, why):
    assert getattr(_lib.lib(), name)(C.byref(cache()), *CALLS[name](**more)) == _lib.INVALID_REQUEST
    assert why in _lib.last_error()


@pytest.mark.parametrize("name,more", [
    ("hllm_b200_kv8_write", {"tokens": 0}), ("hllm_b200_kv8_read", {"tokens": 0}),
    ("hllm_b200_kv8_read", {"rows": 0}), ("hllm_b200_kv8_attention", {"tokens": 0}),
    ("hllm_b200_kv8_attention", {"rows": 0})])
def test_empty_calls_do_nothing(name, more):
    assert getattr(_lib.lib(), name)(C.byref(cache()), *CALLS[name](**more)) == _lib.OK


def test_structs_match_the_header(tmp_path):
    import subprocess
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{_lib.HEADER}"', 'int main(void) {']
    for name, cls in (("hllm_b200_kv8", _lib.KV8), ("hllm_b200_rope", _lib.Rope)):
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in (_lib.KV8, _lib.Rope):
        want.append(C.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def test_python_refusals_need_no_gpu():
    torch = pytest.importorskip("torch")
    from hllm_b200 import kv8
    codes, scales = torch.zeros((2, 2, 16, 64), dtype=torch.uint8), torch.zeros((2, 2, 16), dtype=torch.uint8)
    for args, why in (((codes, scales, codes, scales), "CUDA"), ((codes[0], scales, codes, scales), "codes"),
                      ((codes, scales, None, scales), "four")):
        with pytest.raises(StageError) as e:
            kv8.Cache.wrap(*args)
        assert e.value.code == _lib.INVALID_REQUEST and why in e.value.message
    for more, why in (({"rotary_dim": 66}, "rotary_dim"), ({"scaling": {"type": "magic"}}, "unknown"),
                      ({"scaling": {"type": "linear", "factor": 2.0, "fctor": 1}}, "unknown"),
                      ({"theta": 0.5}, "theta")):
        with pytest.raises(StageError) as e:
            kv8.Rope(64, **{"theta": 1e4, "device": "cpu", **more})
        assert why in e.value.message
    r = kv8.Rope(64, 1e4, rotary_dim=32, scaling={"type": "linear", "factor": 2.0}, device="cpu")
    np.testing.assert_allclose(r.turns.numpy() * 2 * np.pi, 1e4 ** (-np.arange(16) / 16.0) / 2, rtol=1e-14)
