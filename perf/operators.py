"""The 8-bit paged K/V cache and the attention that reads it, as cases that can be timed.

Each case is a dict of plain values; `kind` names the operator:

  append   rotate Q and K, put K and V into the cache in 8 bits, and read the rows back
  decode   single-token GQA attention over a batch of sequences' 8-bit caches
  prefill  causal attention of query rows after earlier tokens, over the 8-bit cache

Where `own` is false, run() computes them in elementary torch operations in 32
bits; where it is true, with the library's entry points.

Inputs are what those paths meet: queries, keys and values ~ N(0, 1) in BF16,
every sixteenth key channel eight times as large (the outlier channels of
trained models), pages in random order in a shared pool, and caches filled by
the format's own rule.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 16  # tokens that share a scale
THETA = 500000.0
# Largest value of a format: E4M3 (sign, four exponent and three mantissa bits) and symmetric INT8.
LARGEST = {"e4m3": 448.0, "int8": 127.0}
# Query heads, kv heads, head dimension: the benchmark's two, a group of seven, a head of 64.
HEADS = ((32, 8, 128), (64, 8, 128), (28, 4, 128), (32, 8, 64))


def _case(name, kind, batch, rows, low, high, heads, fmt, page):
    """rows: new tokens (append) or query rows (prefill, decode) of each sequence; low, high: tokens
    before them (append, prefill) or in all (decode)."""
    return {"name": name, "kind": kind, "batch": batch, "rows": rows, "low": low, "high": high, "q_heads": heads[0],
            "kv_heads": heads[1], "head_dim": heads[2], "format": fmt, "page": page}


def listed():
    return [
        # One chat session's decode step: the smallest append, launch and latency.
        _case("append_step", "append", 1, 1, 1000, 1000, HEADS[0], "e4m3", 16),
        # A server's decode step: 64 sessions of mixed age.
        _case("append_step64", "append", 64, 1, 0, 4000, HEADS[0], "int8", 16),
        # A prompt chunk of the runner that starts inside a block.
        _case("append_chunk", "append", 1, 512, 1000, 1000, HEADS[0], "e4m3", 16),
        # A whole long prompt at once.
        _case("append_prompt", "append", 1, 8192, 0, 0, HEADS[1], "e4m3", 16),
        # One chat session early in its context.
        _case("decode_single", "decode", 1, 1, 1000, 1000, HEADS[0], "e4m3", 16),
        # A server's decode step over 32 sessions of mixed age.
        _case("decode_ragged", "decode", 32, 1, 512, 8192, HEADS[0], "e4m3", 16),
        # Four sessions with long documents: the benchmark's decode shape.
        _case("decode_long", "decode", 4, 1, 32768, 32768, HEADS[1], "e4m3", 16),
        # An odd batch of a model with seven query heads per kv head, larger pages.
        _case("decode_group7", "decode", 9, 1, 1, 4000, HEADS[2], "int8", 64),
        # Checking four drafted tokens and one more of each of 16 sessions.
        _case("prefill_verify", "prefill", 16, 5, 300, 4000, HEADS[0], "e4m3", 16),
        # The last 512-token chunk of a 4,096-token prompt.
        _case("prefill_chunk", "prefill", 1, 512, 3584, 3584, HEADS[0], "e4m3", 16),
        # An odd-length turn after an odd-length history, seven query heads per kv head.
        _case("prefill_odd", "prefill", 1, 333, 777, 777, HEADS[2], "int8", 64),
        # The second half of an 8,192-token prompt: the largest call.
        _case("prefill_long", "prefill", 1, 4096, 4096, 4096, HEADS[1], "e4m3", 16),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "prefill", "prefill"))
    heads, fmt, page = rng.choice(HEADS), rng.choice(sorted(LARGEST)), rng.choice((16, 64, 256))
    if kind == "append":
        if rng.random() < 0.5:
            batch, rows = _log_uniform(rng, 1, 64), 1
        else:
            batch, rows = rng.choice((1, 1, 3)), _log_uniform(rng, 2, 2700)
        high = _log_uniform(rng, 16, 4096)
    elif kind == "decode":
        batch, rows = _log_uniform(rng, 1, 64), 1
        high = _log_uniform(rng, 16, min(32768, 131072 // batch))
    elif rng.random() < 0.5:
        batch, rows = _log_uniform(rng, 1, 32), rng.randint(2, 8)
        high = _log_uniform(rng, 16, min(16384, 65536 // batch))
    else:
        batch, rows, high = 1, _log_uniform(rng, 9, 2048), _log_uniform(rng, 16, 4096)
    low = high if rng.random() < 0.25 else max(1, int(high * rng.uniform(0.05, 0.9)))
    case = _case("", kind, batch, rows, low, high, heads, fmt, page)
    del case["name"]
    return case


# ---- inputs -------------------------------------------------------------------


def _lengths(case, seed):
    """Tokens of each sequence before the call's own rows; a decode's one row is in the cache already."""
    rng = random.Random(seed * 7919 + 17)
    return [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]


def _normal(gen, shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _keys(gen, shape):
    x = _normal(gen, shape)
    x[..., ::16] *= 8.0
    return x


def _scale_of(largest, amax):
    """The smallest power of two with amax <= largest * scale, 2^-126 at least."""
    top, exponent = math.frexp(largest)
    f, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - exponent + (f > top), torch.full_like(e, -126)).clamp_min(-126)
    # its bits: a power function need not be exact
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _encode(x, fmt):
    """The bytes of values already divided by their scale."""
    if fmt == "e4m3":
        return x.to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.round(x).to(torch.int8).view(torch.uint8)


def _decode_bytes(x, fmt):
    return x.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float()


def _fill(x, fmt, pages, kvh, page, d):
    """Bytes [pages][kvh][page][d] and scales [pages][kvh][page/16] of a pool of values."""
    x = x.view(pages, kvh, page // BLOCK, BLOCK, d)
    s = _scale_of(LARGEST[fmt], x.abs().amax((-1, -2)))
    return _encode(x / s[..., None, None], fmt).view(pages, kvh, page, d), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    b, n, kvh, d, page = c["batch"], c["rows"], c["kv_heads"], c["head_dim"], c["page"]
    before = _lengths(c, seed)
    total = [t if c["kind"] == "decode" else t + n for t in before]
    pages = [-(-t // page) for t in total]
    order = torch.randperm(sum(pages), generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((b, max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for i, count in enumerate(pages):
        table[i, :count] = order[at:at + count]
        at += count
    k8, ks = _fill(_keys(gen, (sum(pages), kvh, page, d)), c["format"], sum(pages), kvh, page, d)
    v8, vs = _fill(_normal(gen, (sum(pages), kvh, page, d)), c["format"], sum(pages), kvh, page, d)
    s = {"case": c, "before": before, "table": table, "pages": sum(pages), "pps": max(pages), "k_pool": k8,
         # four tokens of one dimension side by side: [block][4][d][4]
         "v_pool": v8.view(sum(pages), kvh, page // BLOCK, 4, 4, d).transpose(-1, -2).contiguous(),
         "scales": torch.stack((ks, vs), -1).contiguous()}
    s["q"] = _normal(gen, (b, n, c["q_heads"], d)).bfloat16()
    s["out"] = torch.empty_like(s["q"])
    if c["kind"] == "append":
        s["k"], s["v"] = _keys(gen, (b, n, kvh, d)).bfloat16(), _normal(gen, (b, n, kvh, d)).bfloat16()
        s["positions"] = torch.tensor(before, dtype=torch.int32, device="cuda")
        s["first"] = s["positions"] - (BLOCK - 1)
        s["k_rows"] = torch.empty((b, n + BLOCK - 1, kvh, d), dtype=torch.bfloat16, device="cuda")
        s["v_rows"] = torch.empty_like(s["k_rows"])
    return s


# ---- plain forms --------------------------------------------------------------


def _rows_of(s, rows):
    """Where logical rows [batch][n] (clamped into the table) are in a pool seen as [rows][kv heads]."""
    page = s["case"]["page"]
    at = rows.clamp(0, s["pps"] * page - 1)
    return torch.gather(s["table"].long(), 1, at // page), at % page


def _cached(s, rows):
    """Byte values and scales of K and V at rows [batch][n]: [batch][n][kv heads][head dim], [batch][n][kv heads]."""
    c = s["case"]
    p, r = _rows_of(s, rows)
    k = _decode_bytes(s["k_pool"][p, :, r], c["format"])
    v = _decode_bytes(s["v_pool"][p, :, r // BLOCK, r % BLOCK // 4, :, r % 4], c["format"])
    scales = s["scales"][p, :, r // BLOCK]
    return k, scales[..., 0], v, scales[..., 1]


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    c = s["case"]
    n, d = c["rows"], c["head_dim"]
    pos = s["positions"].long()[:, None]
    inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    angle = (pos + torch.arange(n, device="cuda"))[..., None, None] * inv
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _rotate(s["q"].float(), cos, sin).bfloat16()
    # whole blocks from the one that holds row pos - 15
    count = (n + 2 * BLOCK - 3) // BLOCK + 1
    start = torch.div(pos - (BLOCK - 1), BLOCK, rounding_mode="floor") * BLOCK
    rows = start + torch.arange(count * BLOCK, device="cuda")
    new = ((rows >= pos) & (rows < pos + n))[..., None, None]
    old = ((rows >= 0) & (rows < pos))[..., None, None]
    take = (rows - pos).clamp(0, n - 1)[..., None, None].expand(-1, -1, c["kv_heads"], d)
    k8, ks, v8, vs = _cached(s, rows)
    read = (pos - (BLOCK - 1) - start + torch.arange(n + BLOCK - 1, device="cuda"))
    outs = []
    for x, x8, xs in ((_rotate(s["k"].float(), cos, sin), k8, ks), (s["v"].float(), v8, vs)):
        x = torch.gather(x, 1, take) * new
        split = (x.shape[0], count, BLOCK) + x.shape[2:]
        amax = x.view(split).abs().amax((2, 4))
        fresh = new.view(split[:3]).any(2)[..., None]
        had = old.view(split[:3]).any(2)[..., None]
        before = xs.view(split[:4])[:, :, 0]
        scale = torch.where(fresh, _scale_of(LARGEST[c["format"]], amax), torch.zeros_like(amax))
        scale = torch.where(had, torch.maximum(scale, before), scale)[:, :, None, :, None]
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        kept = x8.view(split) * (before[:, :, None, :, None] / scale)
        value = torch.where(new.view(split[:3] + (1, 1)), x.view(split) / scale, kept)
        value = _decode_bytes(_encode(value, c["format"]), c["format"]) * scale
        value = torch.where(old | new, value.view(x.shape), torch.zeros_like(x))
        outs.append(torch.gather(value, 1, read[..., None, None].expand((-1, -1) + x.shape[2:])).bfloat16())
    return [q] + outs


def _plain_attention(s, lens, mask_rows):
    """q [batch][n][q heads][d] over tokens < lens - mask_rows + i + 1 for row i."""
    c = s["case"]
    b, n, qh, kvh, d = c["batch"], c["rows"], c["q_heads"], c["kv_heads"], c["head_dim"]
    tokens = torch.arange(max(lens), device="cuda")
    k8, ks, v8, vs = _cached(s, tokens.expand(b, -1))
    k = (k8 * ks[..., None]).permute(0, 2, 3, 1).contiguous()
    v = (v8 * vs[..., None]).permute(0, 2, 1, 3).contiguous()
    del k8, v8
    q = s["q"].float().view(b, n, kvh, qh // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, d)
    scores = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    last = torch.tensor(lens, device="cuda")[:, None] - mask_rows + torch.arange(n, device="cuda") + 1
    seen = tokens < last.repeat_interleave(qh // kvh, 1)[:, None, :, None]
    scores = scores.masked_fill_(~seen, float("-inf"))
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(b, kvh, n, qh // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, n, qh, d).bfloat16()


# ---- the library's calls ------------------------------------------------------

_library = None


def _calls():
    """The binding, and one library context on torch's current stream, as a program keeps them."""
    global _library
    if _library is None:
        package = os.path.join(os.getcwd(), "vk-shei_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import mslim_attn

        context = mslim_attn.Context()
        context.use_torch_stream()
        _library = mslim_attn, context
    return _library


def _cache(s):
    """The cache's description, made once per state like the page table that it names."""
    if "cache" not in s:
        c, (lib, _) = s["case"], _calls()
        s["cache"] = lib.Kv8Cache(s["k_pool"], s["v_pool"], s["scales"], s["table"], s["pages"], s["pps"], c["page"],
                                  c["kv_heads"], c["head_dim"], lib.FORMAT_E4M3 if c["format"] == "e4m3" else lib.FORMAT_INT8)
    return s["cache"]


def _own_append(s):
    c, ctx = s["case"], _calls()[1]
    ctx.rope_append_kv8(_cache(s), s["q"], s["k"], s["v"], s["out"], c["batch"], c["rows"], s["positions"],
                        c["q_heads"], THETA)
    ctx.pages_gather_kv8(s["cache"], c["batch"], c["rows"] + BLOCK - 1, s["first"], s["k_rows"], s["v_rows"])
    return [s["out"], s["k_rows"], s["v_rows"]]


def _own_attention(s):
    c, ctx = s["case"], _calls()[1]
    if c["kind"] == "decode":
        ctx.decode_kv8(_cache(s), s["q"], s["out"], s["before"], c["q_heads"])
    else:
        ctx.prefill_kv8(_cache(s), s["q"], s["out"], c["rows"], s["before"], c["q_heads"])
    return s["out"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own_append(state) if kind == "append" else _own_attention(state)
    if kind == "append":
        return _plain_append(state)
    n = state["case"]["rows"]
    return _plain_attention(state, [t + (n if kind == "prefill" else 0) for t in state["before"]], n)


# ---- what a pass cannot do without --------------------------------------------


def work(case):
    b, n, qh, kvh, d = case["batch"], case["rows"], case["q_heads"], case["kv_heads"], case["head_dim"]
    before = b * (case["low"] + case["high"]) / 2
    q = 2 * b * n * qh * d * 2  # read and written
    row = 2 * kvh * (d + 4 / BLOCK)  # K and V of one token in the cache, with its share of the scales
    if case["kind"] == "append":
        # the new rows in BF16, their bytes written; the rows read back, in bytes and in BF16
        kept = min(before, b * (BLOCK - 1))
        return {"bytes": q + b * n * 2 * kvh * d * 2 + b * n * row + (kept + b * n) * (row + 2 * kvh * d * 2),
                "flops": 6 * b * n * (qh + kvh) * d}
    seen = before if case["kind"] == "decode" else n * before + b * n * (n + 1) / 2
    cached = before + (0 if case["kind"] == "decode" else b * n)
    return {"bytes": q + cached * row, "flops": 4 * qh * d * seen}


# ---- the definition in 64 bits ------------------------------------------------


def _power(e):
    """2 ** e for whole numbers e, from its bits: a power function need not be exact."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _value(byte, fmt):
    """What a byte stands for, from the format's definition."""
    byte = byte.long()
    if fmt == "int8":
        return torch.where(byte > 127, byte - 256, byte).double()
    exponent, mantissa = byte // 8 % 16, (byte % 8).double()
    size = torch.where(exponent > 0, (8 + mantissa) * _power(exponent - 10), mantissa * 2.0 ** -9)
    return torch.where(byte > 127, -size, size)


def _nearest(x, fmt):
    """x rounded to a value of the format, halves to even."""
    if fmt == "int8":
        return torch.round(x)
    _, e = torch.frexp(x)
    step = _power(e.clamp_min(-5) - 4)
    return torch.round(x / step) * step


def _exact_rows(s, i, tokens):
    """K and V values of the first `tokens` rows of sequence i, and the scale of each row."""
    c = s["case"]
    page, fmt = c["page"], c["format"]
    pages = s["table"][i, :-(-tokens // page)].long()
    kvh, d = c["kv_heads"], c["head_dim"]
    room = pages.numel() * page
    k = _value(s["k_pool"][pages], fmt).permute(0, 2, 1, 3).reshape(room, kvh, d)[:tokens]
    v = _value(s["v_pool"][pages], fmt).permute(0, 2, 3, 5, 1, 4).reshape(room, kvh, d)[:tokens]
    scale = s["scales"][pages].double().permute(0, 2, 1, 3).reshape(room // BLOCK, kvh, 2)
    scale = scale.repeat_interleave(BLOCK, 0)[:tokens]
    return k, v, scale


def _exact_append(s):
    c = s["case"]
    n, d, fmt = c["rows"], c["head_dim"], c["format"]
    q_out, rows_out = [], ([], [])
    for i, pos in enumerate(s["before"]):
        where = torch.arange(pos, pos + n, dtype=torch.float64, device="cuda")
        pair = torch.arange(d // 2, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((n, 1, d // 2), dtype=torch.float64, device="cuda"),
                           (where[:, None] * torch.exp(-2 * pair / d * math.log(THETA)))[:, None])

        def rotated(x):
            y = torch.complex(x[..., :d // 2].double(), x[..., d // 2:].double()) * turn
            return torch.cat((y.real, y.imag), -1)

        q_out.append(rotated(s["q"][i]))
        fresh = (rotated(s["k"][i]), s["v"][i].double())
        low = max(0, pos // BLOCK * BLOCK)
        k, v, scale = _exact_rows(s, i, pos)
        for which, (x, cached) in enumerate(zip(fresh, (k, v))):
            out = [cached[:low] * scale[:low, :, which, None]]
            for at in range(low, pos + n, BLOCK):
                here = x[max(0, at - pos):at + BLOCK - pos]
                amax = here.abs().amax((0, 2)).clamp_min(1e-300)
                # a logarithm is rounded: an exact power must not come out above itself
                step = _power(torch.ceil(torch.log2(amax / LARGEST[fmt]) - 1e-12).clamp_min(-126))
                if at < pos:
                    before = scale[at, :, which]
                    step = torch.maximum(step, before)
                    out.append(_nearest(cached[at:] * (before / step)[:, None], fmt) * step[:, None])
                out.append(_nearest(here / step[:, None], fmt) * step[:, None])
            rows = torch.cat(out)[max(0, pos - BLOCK + 1):]
            missing = n + BLOCK - 1 - rows.shape[0]
            rows_out[which].append(torch.cat((rows.new_zeros((missing,) + rows.shape[1:]), rows)))
    return [torch.stack(q_out), torch.stack(rows_out[0]), torch.stack(rows_out[1])]


def _exact_attention(s):
    c = s["case"]
    n, kvh, d = c["rows"], c["kv_heads"], c["head_dim"]
    group = c["q_heads"] // kvh
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, before in enumerate(s["before"]):
        tokens = before if c["kind"] == "decode" else before + n
        k, v, scale = _exact_rows(s, i, tokens)
        hidden = torch.ones((n, tokens), dtype=torch.bool, device="cuda").triu(tokens - n + 1)
        for h in range(kvh):
            keys, values = k[:, h] * scale[:, h, :1], v[:, h] * scale[:, h, 1:]
            for g in range(group):
                x = s["q"][i, :, h * group + g].double() @ keys.T / math.sqrt(d)
                out[i, :, h * group + g] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ values
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attention(s)
