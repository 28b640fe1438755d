"""The 8-bit KV cache's operators restated in 64 bits, for its tests: the
number format from its definition, rotary positions, and attention over the
cache's values, with the error that the kernels' arithmetic may have."""
import math

import numpy as np

E_MIN, E_MAX, LIMIT = -24, 39, 448.0 * 2.0 ** 39


def e4m3_values():
    """The value of each of the 256 codes."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


def e4m3_round(x):
    """float64 values of at most 448 in size, to the nearest e4m3 value, ties to even."""
    size = np.maximum(np.abs(x), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(size)) - 3)
    return np.round(x / step) * step


def exponent(top):
    """The scale exponent of a row with largest finite size `top`."""
    if top == 0:
        return E_MIN
    e = math.frexp(top / 448.0)
    return min(max(e[1] if e[0] > 0.5 else e[1] - 1, E_MIN), E_MAX)


def frequencies(rot, theta, scaling):
    """Radians per position of the pairs, and the factor on cos and sin."""
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if not scaling:
        return np.array(f), 1.0
    kind, factor = scaling["type"], scaling["factor"]
    if kind == "linear":
        return np.array(f) / factor, 1.0
    old = scaling["original_max_position"]
    out = []
    if kind == "llama3":
        lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
        for x in f:
            turns = old * x / (2 * math.pi)  # within the original length
            if turns > hi:
                out.append(x)
            elif turns < lo:
                out.append(x / factor)
            else:
                mix = (turns - lo) / (hi - lo)
                out.append((1 - mix) * x / factor + mix * x)
        return np.array(out), 1.0
    pair = [rot * math.log(old / (2 * math.pi * b)) / (2 * math.log(theta))
            for b in (scaling["beta_fast"], scaling["beta_slow"])]
    low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
    for i, x in enumerate(f):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(x / factor * ramp + x * (1 - ramp))
    return np.array(out), 0.1 * math.log(factor) + 1


def normed_rotated(x, positions, w, eps, rot, freq, factor, interleaved):
    """x float64 [T, heads, d]: RMSNorm (w None: none), then rotation."""
    y = x.copy()
    if w is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * w
    a = positions[:, None].astype(np.float64) * freq
    c, s = (factor * np.cos(a))[:, None], (factor * np.sin(a))[:, None]
    i0 = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    i1 = i0 + (1 if interleaved else rot // 2)
    z = y.copy()
    z[..., i0] = y[..., i0] * c - y[..., i1] * s
    z[..., i1] = y[..., i1] * c + y[..., i0] * s
    return z


def values(torch, codes, scales):
    """float64 values of uint8 codes [..., d] and scale bytes [...]."""
    table = torch.from_numpy(e4m3_values()).to(codes.device)
    return table[codes.long()] * torch.exp2(scales.double() - 127)[..., None]


def attend(torch, k, v, q, positions, scale):
    """Attention of one row: k, v float64 [L, Hkv, d], q float64 [count, Hq, d],
    positions [count] (keys up to it; negative: none).  Returns (o, tolerance).

    The tolerance, by where the kernels round (u = 2^-24 for F32; a product's
    sum on the tensor cores may truncate, so 2u a step):
      * the output to F16: 2^-11 |o|, or half a subnormal step, 2^-25;
      * a weight to F16: 2^-11 of it, or 2^-25 of a reference that the largest
        weight reaches, so n 2^-25 max_j (p_j 2 amax_j) in all, since a value is
        at most its row's 448 * 2^e < 2 amax;
      * a score: (d + 8) 2u sum_i |q_i k_i| scale, which moves a weight and the
        normaliser by that much each, relatively; 2^-20 covers exp2 and scales;
      * sums of n weighted values and of n weights: n 2u each.
    All but the first two multiply sum_j p_j |v_j|."""
    count, hq, d = q.shape
    n, hkv = k.shape[0], k.shape[1]
    g = hq // hkv
    o = torch.zeros((count, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.full_like(o, 2.0 ** -25)
    key = torch.arange(n, device=q.device)
    pos = torch.as_tensor(positions, device=q.device)
    some = pos >= 0
    if n == 0 or not bool(some.any()):
        return o, tol
    hidden = key[None, :] > pos[some, None]
    u2 = 2.0 ** -23
    for h in range(hq):
        kh, vh = k[:, h // g], v[:, h // g]
        s = (q[some, h] @ kh.T * scale).masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1)
        o[some, h] = p @ vh
        size = (q[some, h].abs() @ kh.abs().T * abs(scale)).masked_fill(hidden, 0.0).amax(-1)
        share = p @ vh.abs()
        part = (p * 2 * vh.abs().amax(-1)[None]).amax(-1)
        rel = 2.0 ** -11 + 2.0 ** -20 + 2 * (d + 8) * u2 * size + 2 * n * u2
        tol[some, h] += (2.0 ** -11 * o[some, h].abs() + rel[:, None] * share +
                         (n * 2.0 ** -25 * part)[:, None])
    return o, tol
