"""Cases of the 8-bit paged KV cache: its write (q/k norm, rotary positions,
quantisation), its read-back, and the attention that reads it.

The cache holds, per (token, kv head) of K and of V, ``d`` e4m3 codes and one
power-of-two scale 2^e: e is the least integer in [-24, 39] with
max |x| <= 448 * 2^e.  Pages are 16 tokens: codes [blocks][Hkv][16][d], scales
[blocks][Hkv][16].  ``run`` computes in plain torch operations in 32 bits, or,
where ``own`` is set, calls ``hllm_b200.kv8``.
"""
import math

import torch

own = False

PAGE = 16
E_MIN, E_MAX = -24, 39
LIMIT = 448.0 * 2.0 ** E_MAX
IN_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
#: (query heads, kv heads, head size) of the configurations and their tests.
HEADS = ((32, 8, 128), (16, 8, 128), (32, 8, 64), (8, 8, 64), (6, 2, 256), (4, 2, 64))
SCALINGS = ("none", "linear", "llama3", "yarn")


# ---------------------------------------------------------------- the cases
def _write(name, tokens, heads, dtype, norm, rot, inter, scaling, decode, top, pad=0):
    hq, hkv, d = heads
    return {"name": name, "op": "write", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d,
            "dtype": dtype, "norm": norm, "rot": rot, "inter": inter, "scaling": scaling,
            "decode": decode, "top": top, "pad": pad}


def _read(name, rows, lo, hi, heads, dtype, tail):
    hq, hkv, d = heads
    return {"name": name, "op": "read", "rows": rows, "lo": lo, "hi": hi, "hkv": hkv, "d": d,
            "dtype": dtype, "tail": tail}


def _attention(name, heads, rows=0, lo=1, hi=1, chunks=0, count_lo=2, count_hi=2, past_lo=0,
               past_hi=0):
    hq, hkv, d = heads
    return {"name": name, "op": "attention", "hq": hq, "hkv": hkv, "d": d, "rows": rows, "lo": lo,
            "hi": hi, "chunks": chunks, "count_lo": count_lo, "count_hi": count_hi,
            "past_lo": past_lo, "past_hi": past_hi}


def listed():
    return [
        # One request decoding: the write of its single token, where only latency counts.
        _write("write_1", 1, (32, 8, 128), "f32", True, 128, False, "none", True, 4096),
        # A prompt chunk of a long-context model: scaled half-layout positions past 100,000.
        _write("write_chunk_575", 575, (32, 8, 64), "f32", False, 64, False, "llama3", False, 120000),
        # A large prefill pass; interleaved pairs over half of the head, half-precision input,
        # and rows that a captured batch pads.
        _write("write_prefill_8192", 8192, (32, 8, 128), "f16", True, 64, True, "yarn", False, 32768, 23),
        # One sequence handed to another worker or to the F16 path.
        _read("read_1x4096", 1, 4096, 4096, (32, 8, 128), "f16", False),
        # The newer part of many sequences, in 32 bits.
        _read("read_37_ragged", 37, 33, 6000, (6, 2, 256), "f32", True),
        # One request decoding at a short context.
        _attention("decode_1x1000", (32, 8, 128), 1, 1000, 1000),
        # The steady state of a serving batch: 64 rows of about a thousand keys.
        _attention("decode_64_steady", (32, 8, 128), 64, 132, 4416),
        # A batch of long contexts, the most KV bytes of the cases.
        _attention("decode_64_long", (32, 8, 128), 64, 1024, 16384),
        # One request at a very long context: the split over the length is all there is.
        _attention("decode_1x131071", (16, 8, 128), 1, 131071, 131071),
        # A prompt chunk behind earlier ones.
        _attention("prefill_512_at_1024", (32, 8, 128), chunks=1, count_lo=512, count_hi=512,
                   past_lo=1024, past_hi=1024),
        # A mixed pass: decode rows beside ragged chunks.
        _attention("mixed_24_and_5", (32, 8, 64), 24, 100, 3001, 5, 3, 401, 0, 1500),
        # A long prompt's last large chunk.
        _attention("prefill_2048_at_8192", (32, 8, 128), chunks=1, count_lo=2048, count_hi=2048,
                   past_lo=8192, past_hi=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = rng.choice(HEADS)
    op = rng.choice(("write", "write", "read", "decode", "decode", "prefill", "prefill", "mixed"))
    hq, hkv, d = heads
    if op == "write":
        decode = rng.random() < 0.5
        tokens = _log(rng, 1, 256) if decode else _log(rng, 2, 8192 * 6144 // ((hq + 2 * hkv) * d * 2))
        rot = rng.choice((d, d, d // 2, d // 4))
        c = _write("", tokens, heads, rng.choice(tuple(IN_TYPES)), rng.random() < 0.5, rot,
                   rng.random() < 0.5, rng.choice(SCALINGS), decode, _log(rng, 16, 1 << 20),
                   rng.choice((0, 0, rng.randint(0, min(40, tokens)))))
    elif op == "read":
        rows = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, min(8192, 48000 * 512 // (rows * hkv * d))))
        c = _read("", rows, rng.randint(1, hi), hi, heads, rng.choice(tuple(IN_TYPES)),
                  rng.random() < 0.5)
    elif op == "decode":
        rows = _log(rng, 1, 64)
        hi = _log(rng, 1, min(131072, 64 * 16384 * 1024 // (2 * rows * hkv * d)))
        c = _attention("", heads, rows, rng.randint(1, hi), hi)
    elif op == "prefill":
        chunks = _log(rng, 1, 4)
        hi = _log(rng, 2, 2048 // chunks)
        past = _log(rng, 1, 8192) if rng.random() < 0.7 else 0
        c = _attention("", heads, 0, 1, 1, chunks, rng.randint(2, hi), hi, past // 2, past)
    else:
        chunks = rng.randint(1, 6)
        hi = _log(rng, 2, 600)
        past = _log(rng, 1, 3000) if rng.random() < 0.7 else 0
        rows = _log(rng, 1, 48)
        ctx = _log(rng, 1, 6000)
        c = _attention("", heads, rows, rng.randint(1, ctx), ctx, chunks, rng.randint(2, hi), hi,
                       past // 2, past)
    del c["name"]
    return c


def _spread(n, lo, hi):
    """n whole numbers between lo and hi, spread over their logarithm; the last is hi."""
    if n == 0:
        return []
    base = max(lo, 1)
    got = [int(round(base * (max(hi, 1) / base) ** (((i + 1) * 0.6180339887498949) % 1.0)))
           for i in range(n - 1)] + [hi]
    return [min(max(x, lo), hi) for x in got]


def _rows(case):
    """(earlier keys, new tokens) of each row of an attention case, decode rows first."""
    return ([(x - 1, 1) for x in _spread(case["rows"], case["lo"], case["hi"])] +
            list(zip(_spread(case["chunks"], case["past_lo"], case["past_hi"]),
                     _spread(case["chunks"], case["count_lo"], case["count_hi"]))))


def _spans(case):
    """(first, end) positions of each row of a read case."""
    ends = _spread(case["rows"], case["lo"], case["hi"])
    return [(e // 3 if case["tail"] else 0, e) for e in ends]


def work(case):
    hkv, d = case["hkv"], case["d"]
    if case["op"] == "write":
        t, hq, size = case["tokens"], case["hq"], SIZES[case["dtype"]]
        kept = t - case["pad"]
        return {"bytes": t * hq * d * (size + 2) + kept * 2 * hkv * (d * size + d + 1) + 8 * t,
                "flops": t * (hq + 2 * hkv) * d * 6}
    if case["op"] == "read":
        n = sum(e - f for f, e in _spans(case))
        return {"bytes": n * 2 * hkv * (d + 1 + d * SIZES[case["dtype"]]), "flops": n * 2 * hkv * d}
    rows, hq = _rows(case), case["hq"]
    keys = sum(p + c for p, c in rows)
    pairs = sum(c * p + c * (c + 1) // 2 for p, c in rows)
    return {"bytes": keys * hkv * 2 * (d + 1) + sum(c for _, c in rows) * hq * d * 4 +
            sum(-(-(p + c) // PAGE) for p, c in rows) * 4,
            "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------- the inputs
def _rope_options(case):
    """theta and scaling of a write case, as a model's configuration gives them."""
    kind = case["scaling"]
    if kind == "linear":
        return 10000.0, {"type": "linear", "factor": 4.0}
    if kind == "llama3":
        return 500000.0, {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                          "high_freq_factor": 4.0, "original_max_position": 8192}
    if kind == "yarn":
        return 1000000.0, {"type": "yarn", "factor": 4.0, "original_max_position": 32768,
                           "beta_fast": 32.0, "beta_slow": 1.0}
    return 1000000.0, None


def _fill(generator, blocks, hkv, d, spread):
    """A pool's codes and scale bytes for values whose size differs from token to token."""
    codes = torch.empty((blocks, hkv, PAGE, d), dtype=torch.uint8, device="cuda")
    scales = torch.empty((blocks, hkv, PAGE), dtype=torch.uint8, device="cuda")
    for b in range(0, blocks, 4096):
        n = min(4096, blocks - b)
        x = torch.randn((n, hkv, PAGE, d), device="cuda", generator=generator)
        x *= torch.exp(spread * torch.randn((n, hkv, PAGE, 1), device="cuda", generator=generator))
        codes[b:b + n], scales[b:b + n] = _quantise(x)
    return codes, scales


def _tables(generator, needs, spare=8):
    """Pages of each row [rows][most pages] (-1 past a row's last), and the pool's size."""
    blocks = int(sum(needs) * 1.05) + spare
    perm = torch.randperm(blocks, device="cuda", generator=generator)[:sum(needs)].to(torch.int32)
    width = max(needs)
    starts = torch.tensor([sum(needs[:i]) for i in range(len(needs))], device="cuda")
    counts = torch.tensor(needs, device="cuda")
    at = torch.arange(width, device="cuda")
    index = (starts[:, None] + at).clamp(max=sum(needs) - 1)
    return torch.where(at < counts[:, None], perm[index], -1).to(torch.int32).contiguous(), blocks


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hkv, d = case["hkv"], case["d"]
    s = {"case": case}
    if case["op"] == "write":
        t, hq = case["tokens"], case["hq"]
        x = torch.randn((t, (hq + 2 * hkv) * d), device="cuda", generator=g)
        s["qkv"] = x.to(IN_TYPES[case["dtype"]])
        blocks = t // PAGE + 8
        kept = t - case["pad"]
        if case["decode"]:  # tokens of many sequences, each somewhere in its last page
            slots = torch.randperm(blocks * PAGE, device="cuda", generator=g)[:t]
            s["positions"] = torch.randint(0, case["top"], (t,), device="cuda", generator=g).int()
        else:
            at = torch.arange(t, device="cuda")
            slots = torch.randperm(blocks, device="cuda", generator=g)[at // PAGE] * PAGE + at % PAGE
            first = int(torch.randint(0, case["top"], (1,), device="cuda", generator=g))
            s["positions"] = (first + at).int()
        s["slots"] = torch.where(torch.arange(t, device="cuda") < kept, slots, -1).int()
        s["k"], s["ks"] = _fill(g, blocks, hkv, d, 0.3)
        s["v"], s["vs"] = _fill(g, blocks, hkv, d, 0.3)
        s["q_norm"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if case["norm"] else None
        s["k_norm"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if case["norm"] else None
        s["out"] = torch.empty((t, hq * d), dtype=torch.float16, device="cuda")
    elif case["op"] == "read":
        spans = _spans(case)
        s["tables"], blocks = _tables(g, [-(-e // PAGE) for _, e in spans])
        s["k"], s["ks"] = _fill(g, blocks, hkv, d, 0.5)
        s["v"], s["vs"] = _fill(g, blocks, hkv, d, 0.5)
        s["first"], s["end"] = _ints([f for f, _ in spans]), _ints([e for _, e in spans])
        s["total"] = sum(e - f for f, e in spans)
        s["cu"] = _ints([sum(e - f for f, e in spans[:i]) for i in range(len(spans) + 1)])
    else:
        rows, hq = _rows(case), case["hq"]
        s["tables"], blocks = _tables(g, [-(-(p + c) // PAGE) for p, c in rows])
        s["k"], s["ks"] = _fill(g, blocks, hkv, d, 0.2)
        s["v"], s["vs"] = _fill(g, blocks, hkv, d, 0.5)
        t = sum(c for _, c in rows)
        s["q"] = (1.5 * torch.randn((t, hq * d), device="cuda", generator=g)).half()
        s["cu"] = _ints([sum(c for _, c in rows[:i]) for i in range(len(rows) + 1)])
        s["lengths"] = _ints([p + c for p, c in rows])
        s["out"] = torch.empty((t, hq * d), dtype=torch.float16, device="cuda")
    if own:
        from hllm_b200 import kv8
        s["cache"] = kv8.Cache.wrap(s["k"], s["ks"], s["v"], s["vs"])
        if case["op"] == "write":
            theta, scaling = _rope_options(case)
            s["rope"] = kv8.Rope(d, theta, rotary_dim=case["rot"], interleaved=case["inter"],
                                 scaling=scaling)
        if case["op"] == "attention":
            s["most"] = max(c for _, c in rows)
            s["workspace"] = kv8.attention_workspace(len(rows), t, s["most"], hq, hkv, d)
    return s


# ---------------------------------------------------------------- the plain forms
def _quantise(x):
    """Codes and scale bytes of rows of float32 values."""
    fit = x.abs() <= LIMIT
    top = torch.where(fit, x.abs(), 0.0).amax(-1)
    m, k = torch.frexp(top)
    e = torch.where(top > 0, torch.where(m <= 0.875, k - 9, k - 8), E_MIN).clamp(E_MIN, E_MAX)
    y = torch.where(fit, torch.ldexp(x, -e[..., None]), math.nan)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The float32 values of codes [..., d] and scale bytes [...]."""
    return codes.view(torch.float8_e4m3fn).float() * torch.exp2(scales.float() - 127.0)[..., None]


def _frequencies(rot, theta, scaling):
    """Radians per position of each pair (float64), and the factor on cos and sin."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = theta ** (-2.0 * i / rot)
    if scaling is None:
        return f, 1.0
    factor = scaling["factor"]
    if scaling["type"] == "linear":
        return f / factor, 1.0
    old = scaling["original_max_position"]
    if scaling["type"] == "llama3":
        lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
        wave = 2 * math.pi / f
        mix = (old / wave - lo) / (hi - lo)
        mixed = (1 - mix) * f / factor + mix * f
        return torch.where(wave < old / hi, f, torch.where(wave > old / lo, f / factor, mixed)), 1.0

    def dim(turns):  # the pair that turns so often within the original length
        return rot * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))
    low = max(math.floor(dim(scaling["beta_fast"])), 0)
    high = min(math.ceil(dim(scaling["beta_slow"])), rot - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _normed(x, w, eps):
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)) * w


def _rotated(x, c, s, rot, inter):
    """x [T, heads, d] with its first `rot` values rotated by cos / sin [T, 1, rot / 2]."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    y0, y1 = a * c - b * s, b * c + a * s
    y = torch.stack((y0, y1), -1).flatten(-2) if inter else torch.cat((y0, y1), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_write(s):
    case = s["case"]
    t, hq, hkv, d, rot = (case[n] for n in ("tokens", "hq", "hkv", "d", "rot"))
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if case["norm"]:
        q, k = _normed(q, s["q_norm"], 1e-6), _normed(k, s["k_norm"], 1e-6)
    f, factor = _frequencies(rot, *_rope_options(case))
    angle = s["positions"].double()[:, None] * f
    c, sn = (factor * angle.cos()).float()[:, None], (factor * angle.sin()).float()[:, None]
    q, k = _rotated(q, c, sn, rot, case["inter"]), _rotated(k, c, sn, rot, case["inter"])
    # A token without a slot (-1) is rotated and not stored.
    slot = s["slots"].long()
    kept = slot >= 0
    page, at = (slot.clamp(min=0) // PAGE)[kept], (slot.clamp(min=0) % PAGE)[kept]
    kc, ke = _quantise(k[kept])
    vc, ve = _quantise(v[kept])
    s["k"][page, :, at], s["ks"][page, :, at] = kc, ke
    s["v"][page, :, at], s["vs"][page, :, at] = vc, ve
    return q.half().view(t, hq * d)


def _plain_read(s):
    case = s["case"]
    cu, total = s["cu"].long(), s["total"]
    n = cu[1:] - cu[:-1]
    row = torch.repeat_interleave(torch.arange(case["rows"], device="cuda"), n, output_size=total)
    pos = torch.arange(total, device="cuda") - cu[row] + s["first"].long()[row]
    page = s["tables"].long()[row, pos // PAGE]
    kind = IN_TYPES[case["dtype"]]
    return [_values(c[page, :, pos % PAGE], e[page, :, pos % PAGE]).to(kind)
            for c, e in ((s["k"], s["ks"]), (s["v"], s["vs"]))]


def _attend(s, r0, r1, tokens):
    """Rows [r0, r1) with at most `tokens` new tokens each, padded to the longest."""
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    rows, g = r1 - r0, hq // hkv
    table = s["tables"][r0:r1].long().clamp(min=0)
    lengths, cu = s["lengths"][r0:r1].long(), s["cu"].long()
    count = (cu[1:] - cu[:-1])[r0:r1]
    at = torch.arange(tokens, device="cuda")
    valid = at < count[:, None]
    index = torch.where(valid, cu[:-1][r0:r1, None] + at, 0)
    q = s["q"][index].float().view(rows, tokens, hkv, g, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(rows, hkv, g * tokens, d)

    def of(codes, scales):
        x = _values(codes[table], scales[table])  # [rows, pages, hkv, 16, d]
        return x.permute(0, 2, 1, 3, 4).reshape(rows, hkv, -1, d)
    k = of(s["k"], s["ks"])
    scores = (q @ k.transpose(-1, -2)).view(rows, hkv, g, tokens, -1) / math.sqrt(d)
    position = (lengths - count)[:, None] + at
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= position[..., None]) & (key < lengths[:, None, None])
    del k
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = (p.view(rows, hkv, g * tokens, -1) @ of(s["v"], s["vs"])).view(rows, hkv, g, tokens, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(rows, tokens, hq * d)[valid].half()


def _plain_attention(s):
    case = s["case"]
    rows = case["rows"]
    got = [_attend(s, 0, rows, 1)] if rows else []
    if case["chunks"]:
        got.append(_attend(s, rows, rows + case["chunks"], case["count_hi"]))
    return torch.cat(got)


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from hllm_b200 import kv8
        if op == "write":
            q = kv8.write(s["cache"], s["qkv"], s["positions"], s["slots"], s["rope"],
                          q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, out=s["out"])
        elif op == "read":
            k, v = kv8.read(s["cache"], s["tables"], s["end"], s["cu"], s["total"],
                            first=s["first"], dtype=IN_TYPES[s["case"]["dtype"]])
        else:
            return kv8.attention(s["cache"], s["q"], s["cu"], s["lengths"], s["tables"],
                                 max_tokens=s["most"], out=s["out"], workspace=s["workspace"])
    elif op == "write":
        q = _plain_write(s)
    elif op == "read":
        k, v = _plain_read(s)
    else:
        return _plain_attention(s)
    if op == "read":
        return {"k": k, "v": v}
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return {"q": q, "k": s["k"].view(e4m3), "k_scale": s["ks"].view(e8m0),
            "v": s["v"].view(e4m3), "v_scale": s["vs"].view(e8m0)}


# ---------------------------------------------------------------- in 64 bits
def _code_values(codes, scales):
    """float64 values of e4m3 codes by their sign, exponent and mantissa fields, times 2^e."""
    c = codes.long()
    exponent, mantissa = (c >> 3) & 15, (c & 7).double()
    size = torch.where(exponent == 0, mantissa * 2.0 ** -9,
                       (8 + mantissa) * torch.pow(2.0, (exponent - 10).double()))
    size = torch.where((c & 127) == 127, math.nan, size)
    return torch.where(c >= 128, -size, size) * torch.pow(2.0, scales.double() - 127)[..., None]


def _e4m3_of(x):
    """float64 x, at most 448 in size, rounded to the nearest e4m3 value (ties to even)."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.pow(2.0, torch.floor(torch.log2(size)) - 3)
    return torch.round(x / step) * step


def _exact_write(case, s):
    t, hq, hkv, d, rot = (case[n] for n in ("tokens", "hq", "hkv", "d", "rot"))
    x = s["qkv"].double().view(t, -1, d)
    if case["norm"]:
        x = x.clone()
        for lo, hi, w in ((0, hq, s["q_norm"]), (hq, hq + hkv, s["k_norm"])):
            h = x[:, lo:hi]
            x[:, lo:hi] = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / d + 1e-6) * w.double()
    theta, scaling = _rope_options(case)
    f, factor = _frequencies(rot, theta, scaling)
    turn = torch.polar(torch.full((t, rot // 2), factor, dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * f)
    head = x[:, :hq + hkv, :rot]
    if case["inter"]:
        z = torch.view_as_complex(head.reshape(t, hq + hkv, rot // 2, 2).contiguous()) * turn[:, None]
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
        z = z * turn[:, None]
        head = torch.cat((z.real, z.imag), -1)
    x = torch.cat((torch.cat((head, x[:, :hq + hkv, rot:]), -1), x[:, hq + hkv:]), 1)
    got = {"q": x[:, :hq].reshape(t, hq * d)}
    slots = s["slots"].long()
    rows = torch.nonzero(slots >= 0)[:, 0]
    page, at = slots[rows] // PAGE, slots[rows] % PAGE
    ones = torch.full_like(s["ks"], 127)
    for n, lo, codes, scales in (("k", hq, s["k"], s["ks"]), ("v", hq + hkv, s["v"], s["vs"])):
        y = x[rows, lo:lo + hkv]
        e = torch.ceil(torch.log2(y.abs().amax(-1) / 448)).clamp(E_MIN, E_MAX)
        pool, scale = _code_values(codes, ones), torch.pow(2.0, scales.double() - 127)
        pool[page, :, at] = _e4m3_of(y / torch.pow(2.0, e)[..., None])
        scale[page, :, at] = torch.pow(2.0, e)
        got[n], got[n + "_scale"] = pool, scale
    return got


def _exact_read(case, s):
    got = {"k": [], "v": []}
    for r, (first, end) in enumerate(_spans(case)):
        pages = s["tables"][r, :-(-end // PAGE)].long()
        for n, codes, scales in (("k", s["k"], s["ks"]), ("v", s["v"], s["vs"])):
            x = _code_values(codes[pages], scales[pages]).transpose(1, 2)
            got[n].append(x.reshape(-1, case["hkv"], case["d"])[first:end])
    return {n: torch.cat(x) for n, x in got.items()}


def _exact_attention(case, s):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out, t = [], 0
    for r, (past, count) in enumerate(_rows(case)):
        end = past + count
        pages = s["tables"][r, :-(-end // PAGE)].long()
        o = torch.empty((count, hq, d), dtype=torch.float64, device="cuda")
        hidden = torch.arange(end, device="cuda") > past + torch.arange(count, device="cuda")[:, None]
        for h in range(hkv):
            k = _code_values(s["k"][pages, h], s["ks"][pages, h]).reshape(-1, d)[:end]
            v = _code_values(s["v"][pages, h], s["vs"][pages, h]).reshape(-1, d)[:end]
            for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                q = s["q"][t:t + count, j * d:(j + 1) * d].double()
                a = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                o[:, j] = a @ v
        out.append(o.view(count, hq * d))
        t += count
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(case, s)
    if case["op"] == "read":
        return _exact_read(case, s)
    return _exact_attention(case, s)
