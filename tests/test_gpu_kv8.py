"""The 8-bit paged K/V cache on the GPU against the rule in numpy and 64 bits.

What is stored without a rotation, and every byte that a call has no business
with, is compared bit for bit.  Rotated keys are f32 (angle in 64 bits, cos and
sin within 2 units, two products and a sum: below 2^-21 of the pair's size):
a byte may differ from the 64-bit rule's only where the value lies that near
to the middle between two bytes, a scale only where the largest value lies
that near to a scale's edge.
"""
import numpy as np
import pytest
import torch

import mslim_attn
import oracle
from _data import from_torch, normal_bf16, to_torch
from _kv8 import E4M3, INT8, LARGEST, Pool, attend, bound, half_step, nearest, rotate, scale_of, values

pytestmark = pytest.mark.gpu

THETA = 500000.0


class Cache:
    """A pool on the host and the device, pages in random order, sequences of up to `tokens` tokens."""

    def __init__(self, rng, tokens, kvh, d, fmt, page, spare=3):
        self.kvh, self.d, self.fmt, self.page = kvh, d, fmt, page
        self.pps = max(1, max(-(-t // page) for t in tokens))
        pages = len(tokens) * self.pps + spare
        self.pool = Pool(pages, kvh, page, d, fmt)
        self.table = rng.permutation(pages)[:len(tokens) * self.pps].reshape(len(tokens), -1).astype(np.int32)
        # what an earlier user of the pages left there, NaN bytes and scales among it
        self.pool.k8[:] = rng.integers(0, 256, self.pool.k8.shape)
        self.pool.v8[:] = rng.integers(0, 256, self.pool.v8.shape)
        self.pool.scales[:] = rng.choice([np.nan, np.inf, 0.0, 1e30, 0.5], self.pool.scales.shape)
        self.upload()

    def upload(self):
        p = self.pool
        self.k, self.v = torch.from_numpy(p.k8).cuda(), torch.from_numpy(p.v_bytes()).cuda()
        self.s, self.t = torch.from_numpy(p.scales).cuda(), torch.from_numpy(self.table).cuda()
        self.desc = mslim_attn.Kv8Cache(self.k, self.v, self.s, self.t, p.pages, self.pps, self.page, self.kvh, self.d,
                                        self.fmt)

    def download(self):
        p = Pool(self.pool.pages, self.kvh, self.page, self.d, self.fmt)
        p.k8, p.scales = self.k.cpu().numpy(), self.s.cpu().numpy()
        p.set_v_bytes(self.v.cpu().numpy())
        return p

    def fill(self, rng, lens):
        """Random tokens by the format's rule: lens[b] of sequence b, stale bytes behind them."""
        p = self.pool
        for b, n in enumerate(lens):
            for t in range(0, n, 16):
                m = min(16, n - t)
                page, blk = self.table[b, t // self.page], t % self.page // 16
                if not 0 <= page < p.pages:
                    continue
                for which, bytes_ in enumerate((p.k8, p.v8)):
                    x = rng.standard_normal((self.kvh, m, self.d)) * 2.0 ** rng.integers(-3, 3)
                    if which == 0:
                        x[..., ::16] *= 8
                    s = scale_of(np.abs(x).max((1, 2)), self.fmt)
                    bytes_[page, :, blk * 16:blk * 16 + m] = encode(x / s[:, None, None], self.fmt)
                    p.scales[page, :, blk, which] = s
        self.upload()


def encode(x, fmt):
    """Bytes of the format's values nearest to x."""
    if fmt == INT8:
        return np.rint(x).astype(np.int8).view(np.uint8)
    table = values(fmt)
    keep = np.flatnonzero(np.isfinite(table) & (np.arange(256) != 128))
    order = keep[np.argsort(table[keep])]
    at = np.searchsorted(table[order], nearest(x, fmt))
    return (order[at] | np.where((table[order[at]] == 0) & np.signbit(x), 128, 0)).astype(np.uint8)


def check_append(cache, k, v, q, q_out, positions, theta, scaling=None, label=""):
    """Compare cache.download() with cache.pool after appending k, v [b][n][kvh][d] (f64), and q_out with q."""
    before, after, fmt = cache.pool, cache.download(), cache.fmt
    expected_k8, expected_v8, expected_s = before.k8.copy(), before.v8.copy(), before.scales.copy()
    slack = 2.0 ** -20 if theta else 0.0
    n = k.shape[1]
    loose = 0
    for b, pos in enumerate(positions):
        at = pos + np.arange(n)
        if theta:
            want = rotate(q[b], at, theta, scaling)
            got = oracle.read_bf16(from_torch(q_out[b]).reshape(-1)).astype(np.float64).reshape(want.shape)
            pair = np.abs(q[b]) + np.abs(np.roll(q[b], cache.d // 2, -1))
            assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -8 + pair * slack).all(), label
        keys = rotate(k[b], at, theta, scaling) if theta else k[b]
        stored = (at >= 0) & (at < cache.pps * cache.page)
        for first in sorted({t // 16 * 16 for t in at[stored]}):
            page, blk = cache.table[b, first // cache.page], first % cache.page // 16
            if not 0 <= page < before.pages:
                continue
            new = stored & (at >= first) & (at < first + 16)
            lo, rows = int(at[new][0] - first), int(new.sum())
            for h in range(cache.kvh):
                for which, x in enumerate((keys[new, h], v[b][new, h])):
                    bytes_, out = (before.k8, before.v8)[which], (expected_k8, expected_v8)[which]
                    got8 = (after.k8, after.v8)[which][page, h, blk * 16:blk * 16 + 16]
                    old = before.scales[page, h, blk, which].astype(np.float64)
                    amax = np.abs(x).max() if np.isfinite(x).all() else np.nan
                    scales = {float(scale_of(np.float64(amax * f), fmt)) for f in (1 - slack, 1, 1 + slack)}
                    if lo:
                        scales = {old if not (f > old or f != f) else f for f in scales}
                    got_s = float(after.scales[page, h, blk, which])
                    assert got_s in scales or (got_s != got_s and any(s != s for s in scales)), (label, got_s, scales)
                    expected_s[page, h, blk, which] = got_s
                    sl = slice(blk * 16, blk * 16 + 16)
                    kept = bytes_[page, h, sl].copy()
                    if lo and got_s > old:
                        with np.errstate(invalid="ignore"):
                            kept[:lo] = encode(np.nan_to_num(values(fmt)[kept[:lo]]) * (old / got_s), fmt)
                    if got_s == got_s:
                        exact = x / got_s
                        want8 = encode(np.clip(exact, -LARGEST[fmt], LARGEST[fmt]), fmt)
                    else:
                        want8 = np.zeros(x.shape, np.uint8)
                    differ = want8 != got8[lo:lo + rows]
                    if differ.any():
                        assert slack, (label, which)
                        off = np.abs(values(fmt)[got8[lo:lo + rows]] - exact)[differ]
                        pair = np.abs(x) + np.abs(np.roll(x, cache.d // 2, -1))
                        room = half_step(exact, fmt)[differ] + pair[differ] / got_s * slack
                        assert (off <= room).all(), (label, which)
                        loose += int(differ.sum())
                    kept[lo:lo + rows] = got8[lo:lo + rows]
                    out[page, h, sl] = kept
    # nothing else has changed, and older rows are what the rule makes of them
    assert np.array_equal(after.k8, expected_k8) and np.array_equal(after.v8, expected_v8), label
    assert np.array_equal(after.scales, expected_s, equal_nan=True), label
    assert loose <= 1e-3 * k.size, (label, loose)
    cache.pool = after


def f64(bits):
    return oracle.read_bf16(bits.reshape(-1)).astype(np.float64).reshape(bits.shape)


def append(ctx, cache, rng, positions, n, qh, theta, scaling=None, spread=1.0):
    b = len(positions)
    qb = normal_bf16(rng, (b, n, qh, cache.d))
    kb, vb = (normal_bf16(rng, (b, n, cache.kvh, cache.d), s) for s in (2.0 * spread, 0.5 * spread))
    q, k, v = to_torch(qb), to_torch(kb), to_torch(vb)
    q_out = torch.full_like(q, -1)
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    more = {} if scaling is None else dict(zip(("factor", "low_freq_factor", "high_freq_factor",
                                                "original_max_position"), scaling), llama3_scaling=True)
    ctx.rope_append_kv8(cache.desc, q if theta else None, k, v, q_out if theta else None, b, n, pos, qh, theta, **more)
    torch.cuda.synchronize()
    check_append(cache, f64(kb), f64(vb), f64(qb), q_out, positions, theta, scaling, f"{positions} x {n}")
    return q_out, f64(vb)


# (q heads, kv heads, head_dim, page): the benchmark's, a group of seven, odd
# pieces of 16, the smallest and the largest head, one kv head.
GEOMETRY = [(32, 8, 128, 16), (14, 2, 128, 64), (6, 3, 96, 32), (5, 5, 16, 16), (10, 1, 256, 128), (8, 2, 64, 4096),
            (40, 1, 208, 16)]


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("qh,kvh,d,page", GEOMETRY)
def test_append_then_gather(ctx, qh, kvh, d, page, fmt):
    rng = np.random.default_rng(d * 10 + qh)
    cache = Cache(rng, [200] * 4, kvh, d, fmt, page)
    # a chunk that starts blocks, then single tokens at every place of a
    # block, larger and larger ones, then a chunk from inside a block on
    append(ctx, cache, rng, [0, 16, 48, 32], 33, qh, THETA)
    for step in range(17):
        append(ctx, cache, rng, [33 + step, 49 + step, 81 + step, 65 + step], 1, qh, THETA, spread=1.3 ** step)
    append(ctx, cache, rng, [50, 66, 98, 82], 29, qh, 0.0, spread=4.0)
    append(ctx, cache, rng, [79, 95, 127, 111], 2, qh, 10000.0, spread=30.0)
    # some rows back again, from before the first to behind the last of the table
    first = [-3, 5, cache.pps * page - 4, 77]
    rows = 9
    k_rows = torch.empty((4, rows, kvh, d), dtype=torch.bfloat16, device="cuda")
    v_rows = torch.empty_like(k_rows)
    ctx.pages_gather_kv8(cache.desc, 4, rows, torch.tensor(first, dtype=torch.int32, device="cuda"), k_rows, v_rows)
    torch.cuda.synchronize()
    for b in range(4):
        for which, got in enumerate((k_rows, v_rows)):
            with np.errstate(invalid="ignore", over="ignore"):
                every, _ = cache.pool.rows(cache.table[b], cache.pps * page, which)
            for i in range(rows):
                t = first[b] + i
                want = every[t] if 0 <= t < len(every) else np.zeros((kvh, d))
                with np.errstate(over="ignore", invalid="ignore"):
                    bits = oracle.write_bf16(want.astype(np.float32).reshape(-1))
                x, y = oracle.read_bf16(from_torch(got[b, i]).reshape(-1)), oracle.read_bf16(bits)
                assert np.array_equal(x, y, equal_nan=True), (b, which, i)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_append_far_positions_and_scaled_rope(ctx, fmt):
    rng = np.random.default_rng(3)
    cache = Cache(rng, [200000], 1, 128, fmt, 4096, spare=0)
    for pos in (131072, 199984, 8192):
        append(ctx, cache, rng, [pos], 5, 4, THETA, scaling=(8.0, 1.0, 4.0, 8192.0))
        append(ctx, cache, rng, [pos + 5], 1, 4, THETA)


def test_append_at_the_table_s_edges(ctx):
    rng = np.random.default_rng(4)
    cache = Cache(rng, [64] * 6, 2, 64, E4M3, 16)
    cache.fill(rng, [64] * 6)
    cache.table[3] = -1                       # a padded slot
    cache.table[4, 1] = cache.pool.pages      # a page that is none
    cache.table[5, 2] = 2 ** 31 - 1
    cache.upload()
    append(ctx, cache, rng, [-1, 60, 64, 0, 10, 30], 20, 4, THETA)
    append(ctx, cache, rng, [-2147483648, 2147483647, 63, 5, 17, 33], 1, 4, THETA)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_append_values_at_their_limits(ctx, fmt):
    cache = Cache(np.random.default_rng(5), [64] * 8, 1, 32, fmt, 16)
    top = LARGEST[fmt]
    cases = [0.0, 1e-40, 3.3e38, top, top * 2.0 ** -7, np.inf, np.nan, -top * 2]
    x = np.zeros((8, 16, 1, 32), np.float32)
    x[:, 3, 0, 5] = cases
    bits = oracle.write_bf16(x.reshape(-1)).reshape(x.shape)
    rows = to_torch(bits)
    pos = torch.zeros(8, dtype=torch.int32, device="cuda")
    ctx.rope_append_kv8(cache.desc, None, rows, rows, None, 8, 16, pos, 1, 0.0)
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        check_append(cache, f64(bits), f64(bits), None, None, [0] * 8, 0.0)
    # a block with a NaN scale keeps it as long as rows are added, and loses it when begun anew
    one = to_torch(oracle.write_bf16(np.ones(8 * 32, np.float32)).reshape(8, 1, 1, 32))
    for at, poisoned in ((7, True), (0, False)):
        ctx.rope_append_kv8(cache.desc, None, one, one, None, 8, 1, pos + at, 1, 0.0)
        torch.cuda.synchronize()
        s = cache.download().scales[cache.table[:, 0], 0, 0]
        assert np.isnan(s[5:7]).all() == poisoned and not np.isnan(s[[0, 1, 2, 3, 4, 7]]).any()


def attention_inputs(rng, cache, rows, qh):
    qb = normal_bf16(rng, (len(cache.table), rows, qh, cache.d))
    return qb, to_torch(qb)


def check_attention(cache, qb, out, lens, queries, label, scale=None):
    scale = scale or float(mslim_attn.default_scale(cache.d))
    got = f64(from_torch(out)).reshape(qb.shape)
    for b, n in enumerate(lens):
        with np.errstate(invalid="ignore", over="ignore"):
            k, known = cache.pool.rows(cache.table[b], max(n, 1), 0)
            v, _ = cache.pool.rows(cache.table[b], max(n, 1), 1)
        limit = [max(0, n - queries + i + 1) for i in range(queries)]
        ref, size = attend(f64(qb[b]), np.nan_to_num(k), np.nan_to_num(v), limit, known & (np.arange(max(n, 1)) < n),
                           scale)
        over = np.abs(got[b] - ref) > bound(ref, size)
        assert not over.any(), (label, b, n, int(over.sum()), float((np.abs(got[b] - ref) / (bound(ref, size) + 1e-30)).max()))


LENS = [1, 0, 15, 16, 17, 33, 127, 128, 129, 300, 1025]


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("qh,kvh,d,page", GEOMETRY)
def test_decode(ctx, qh, kvh, d, page, fmt):
    rng = np.random.default_rng(d + qh)
    cache = Cache(rng, LENS, kvh, d, fmt, page)
    cache.fill(rng, LENS)
    qb, q = attention_inputs(rng, cache, 1, qh)
    out = torch.full_like(q, -1)
    ctx.decode_kv8(cache.desc, q, out, LENS, qh)
    torch.cuda.synchronize()
    check_attention(cache, qb, out, LENS, 1, "decode")
    again = torch.empty_like(out)
    ctx.decode_kv8(cache.desc, q, again, LENS, qh)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("qh,kvh,d,page", GEOMETRY)
@pytest.mark.parametrize("queries", [1, 3, 16, 65])
def test_prefill(ctx, qh, kvh, d, page, queries, fmt):
    rng = np.random.default_rng(d + qh + queries)
    priors = [0, 1, 15, 111, 128, 1000]
    lens = [p + queries for p in priors]
    cache = Cache(rng, lens, kvh, d, fmt, page)
    cache.fill(rng, lens)
    qb, q = attention_inputs(rng, cache, queries, qh)
    out = torch.full_like(q, -1)
    ctx.prefill_kv8(cache.desc, q, out, queries, priors, qh)
    torch.cuda.synchronize()
    check_attention(cache, qb, out, lens, queries, "prefill")


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("queries,prior", [(257, 0), (300, 777), (513, 100)])
@pytest.mark.parametrize("qh,kvh,d,page", [(8, 2, 128, 16), (7, 1, 128, 64), (4, 2, 64, 16), (3, 3, 96, 16),
                                           (2, 1, 256, 16)])
def test_long_prefill(ctx, qh, kvh, d, page, queries, prior, fmt):
    rng = np.random.default_rng(d + qh + queries)
    lens = [prior + queries] * 2
    cache = Cache(rng, lens, kvh, d, fmt, page)
    cache.fill(rng, lens)
    qb, q = attention_inputs(rng, cache, queries, qh)
    out = torch.full_like(q, -1)
    ctx.prefill_kv8(cache.desc, q, out, queries, [prior] * 2, qh)
    torch.cuda.synchronize()
    check_attention(cache, qb, out, lens, queries, "prefill")


def test_pages_that_are_none_weigh_nothing(ctx):
    rng = np.random.default_rng(11)
    lens = [100, 64, 40]
    cache = Cache(rng, lens, 2, 128, E4M3, 16)
    cache.fill(rng, lens)
    cache.table[0, 2] = -1
    cache.table[0, 6] = cache.pool.pages
    cache.table[1] = -7
    cache.upload()
    qb, q = attention_inputs(rng, cache, 1, 8)
    out = torch.full_like(q, -1)
    ctx.decode_kv8(cache.desc, q, out, lens, 8)
    torch.cuda.synchronize()
    check_attention(cache, qb, out, lens, 1, "pages")
    assert not out[1].any()


def test_what_a_row_does_not_see_stays_out(ctx):
    # a NaN block after the row, infinite and NaN scales and bytes behind the end
    rng = np.random.default_rng(12)
    queries, prior = 40, 30
    cache = Cache(rng, [prior + queries], 1, 64, E4M3, 16)
    cache.fill(rng, [prior + queries])
    page = cache.table[0, 3]  # tokens 48 .. 63
    clean = cache.pool.scales[page].copy()
    cache.pool.scales[page] = np.nan
    cache.upload()
    qb, q = attention_inputs(rng, cache, queries, 2)
    out = torch.empty_like(q)
    ctx.prefill_kv8(cache.desc, q, out, queries, [prior], 2)
    torch.cuda.synchronize()
    got = f64(from_torch(out)).reshape(qb.shape)
    assert np.isfinite(got[0, :18]).all() and np.isnan(got[0, 18:]).all()
    cache.pool.scales[page] = clean
    k, known = cache.pool.rows(cache.table[0], prior + queries, 0)
    v, _ = cache.pool.rows(cache.table[0], prior + queries, 1)
    ref, size = attend(f64(qb[0]), k, v, [prior + i + 1 for i in range(queries)], known,
                       float(mslim_attn.default_scale(64)))
    assert (np.abs(got[0, :18] - ref[:18]) <= bound(ref, size)[:18]).all()


def test_many_sequences(ctx):
    rng = np.random.default_rng(13)
    lens = [int(x) for x in rng.integers(0, 90, 200)]
    cache = Cache(rng, lens, 2, 64, INT8, 16)
    cache.fill(rng, lens)
    qb, q = attention_inputs(rng, cache, 1, 4)
    out = torch.full_like(q, -1)
    ctx.decode_kv8(cache.desc, q, out, lens, 4, scale=0.2)
    torch.cuda.synchronize()
    check_attention(cache, qb, out, lens, 1, "many", scale=float(np.float32(0.2)))


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_prompt_then_steps(ctx, fmt):
    """The calls together: two chunks of a prompt, then decode steps, every
    output against 64-bit attention over what the cache then holds."""
    rng = np.random.default_rng(14)
    qh, kvh, d, b = 8, 2, 128, 3
    cache = Cache(rng, [120] * b, kvh, d, fmt, 16)
    position = 0
    for n in (50, 37, 1, 1, 1, 1):
        qb = normal_bf16(rng, (b, n, qh, d))
        k, v = to_torch(normal_bf16(rng, (b, n, kvh, d))), to_torch(normal_bf16(rng, (b, n, kvh, d)))
        q, turned = to_torch(qb), torch.empty((b, n, qh, d), dtype=torch.int16, device="cuda")
        out = torch.full_like(q, -1)
        pos = torch.full((b,), position, dtype=torch.int32, device="cuda")
        ctx.rope_append_kv8(cache.desc, q, k, v, turned, b, n, pos, qh, THETA)
        if n == 1:
            ctx.decode_kv8(cache.desc, turned, out, [position + 1] * b, qh)
        else:
            ctx.prefill_kv8(cache.desc, turned, out, n, [position] * b, qh)
        torch.cuda.synchronize()
        cache.pool = cache.download()
        position += n
        check_attention(cache, from_torch(turned).reshape(qb.shape), out, [position] * b, n, f"at {position}")
