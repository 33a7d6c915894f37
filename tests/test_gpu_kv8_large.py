"""Attention over the 8-bit K/V cache at sizes that take the kernels of large
calls: prompt chunks on the MFMA-bound kernel, caches that the Infinity Cache
does not hold.  The 64-bit reference runs on the GPU; sequences share the pages
of a small pool, which reading allows."""
import numpy as np
import pytest
import torch

import mslim_attn
from _kv8 import E4M3, INT8, values

pytestmark = pytest.mark.gpu

PAGES = 600


class Pool:
    """Random bytes (no E4M3 NaN) and scales: scores of a standard deviation up to about 8."""

    def __init__(self, seed, kvh, d, page, fmt, lens, holes=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.kvh, self.d, self.page, self.fmt = kvh, d, page, fmt
        self.pages = max(2, PAGES * 16 // page)

        def byte(*shape):
            x = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.int32)
            if fmt == E4M3:
                x = torch.where((x & 127) == 127, x & 128, x)
            return x.to(torch.uint8)

        self.k = byte(self.pages, kvh, page, d)
        self.v = byte(self.pages, kvh, page // 16, 4, d, 4)
        grow = torch.randint(0, 4, (self.pages, kvh, page // 16, 2), generator=g, device="cuda")
        # E4M3 bytes spread over its range have a standard deviation of about 130, INT8's of 74
        self.s = ((2.0 ** -9 if fmt == E4M3 else 2.0 ** -8) * (1 << grow)).float().contiguous()
        self.pps = -(-max(lens) // page)
        self.table = torch.randint(0, self.pages, (len(lens), self.pps), generator=g, device="cuda", dtype=torch.int32)
        if holes:
            self.table[0, 1::7] = -1
            self.table[-1, ::5] = self.pages
        self.desc = mslim_attn.Kv8Cache(self.k, self.v, self.s, self.table, self.pages, self.pps, page, kvh, d, fmt)
        self.value = torch.from_numpy(np.nan_to_num(values(fmt))).cuda()

    def rows(self, b, head, tokens):
        """f64 K and V [tokens][d] of a kv head of sequence b, and which tokens have a page."""
        at = torch.arange(tokens, device="cuda")
        page = self.table[b, at // self.page].long()
        known = (page >= 0) & (page < self.pages)
        page = torch.where(known, page, 0)
        off = at % self.page
        s = self.s[page, head, off // 16].double()
        k = self.value[self.k[page, head, off].long()] * s[:, :1]
        v = self.value[self.v[page, head, off // 16, off % 16 // 4, :, off % 4].long()] * s[:, 1:]
        return k, v, known


def check(pool, q, out, lens, queries, qh, rows=None, label=""):
    """`rows` (a slice of the queries): the others are not compared."""
    group, scale = qh // pool.kvh, float(mslim_attn.default_scale(pool.d))
    rows = rows or slice(0, queries)
    worst = 0.0
    for b, n in enumerate(lens):
        for h in range(pool.kvh):
            k, v, known = pool.rows(b, h, n)
            limit = torch.arange(n - queries + 1, n + 1, device="cuda")[rows].repeat_interleave(group)
            qq = q[b, rows, h * group:(h + 1) * group].reshape(-1, pool.d).double()
            x = qq @ k.t().contiguous() * scale
            seen = known[None] & (torch.arange(n, device="cuda")[None] < limit[:, None])
            x = torch.where(seen, x, float("-inf"))
            p = torch.exp(x - x.max(1, keepdim=True).values.clamp(min=-1e300))
            p /= p.sum(1, keepdim=True).clamp(min=1e-300)
            want, size = p @ v, p @ v.abs()
            got = out[b, rows, h * group:(h + 1) * group].reshape(-1, pool.d).double()
            # the bound of _kv8.bound: the value's own rounding, the probabilities' and their
            # sum's, and scores of 32 bits (sum |q k| * scale < 128 here too)
            room = want.abs() * 2.0 ** -8 + size * (2.0 ** -7 + 2.0 ** -10)
            over = (got - want).abs() > room
            worst = max(worst, float(((got - want).abs() / (room + 1e-30)).max()))
            assert not over.any() and not got.isnan().any(), (label, b, h, n, int(over.sum()), worst)


def inputs(seed, batch, queries, qh, d):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn((batch, queries, qh, d), generator=g, device="cuda").bfloat16()
    return q, torch.full_like(q, -1)


# q heads, kv heads, head_dim, page, priors, queries
CHUNKS = [
    (32, 8, 128, 16, [3584], 512), (28, 4, 128, 64, [777, 2000, 0], 700), (6, 6, 96, 16, [1500, 0, 64, 2999], 1001),
    (16, 2, 64, 32, [100] * 20, 300), (64, 8, 128, 16, [2000, 1], 1025), (60, 3, 48, 4096, [999] * 3, 600),
    (256, 1, 16, 16, [700], 200), (200, 1, 112, 128, [500, 3], 150), (16, 2, 64, 16, [90, 300] * 35, 100),
    # two tiles of 16 rows at once: segments alike, ragged ones, head_dim over 128
    (32, 8, 128, 16, [300], 512), (12, 6, 96, 16, [5, 500, 40] * 16, 50), (16, 8, 256, 16, [77] * 6, 90)]


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("qh,kvh,d,page,priors,queries", CHUNKS)
def test_chunks(ctx, qh, kvh, d, page, priors, queries, fmt):
    lens = [n + queries for n in priors]
    pool = Pool(qh + d, kvh, d, page, fmt, lens, holes=page <= 32 and len(lens) < 5)
    q, out = inputs(qh + d, len(lens), queries, qh, d)
    ctx.prefill_kv8(pool.desc, q, out, queries, priors, qh)
    torch.cuda.synchronize()
    check(pool, q, out, lens, queries, qh)
    again = torch.empty_like(out)
    ctx.prefill_kv8(pool.desc, q, again, queries, priors, qh)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


# q heads, kv heads, head_dim, page, lengths, queries; over 200 MiB of K and V each
LONG = [
    (32, 8, 128, 16, [25600] * 5, 1), (32, 8, 128, 64, list(range(300, 7100, 200)), 1), (28, 4, 112, 16, [31000] * 8, 1),
    (28, 4, 112, 16, list(range(1000, 15000, 500)) + [40000], 1), (32, 8, 128, 16, [25600] * 5, 5),
    (32, 8, 128, 16, [25601, 30000, 17, 70000], 12), (32, 8, 128, 32, [3000] * 40, 5), (8, 2, 256, 16, [53000] * 4, 6),
    (5, 1, 208, 16, [131000] * 4, 9), (20, 5, 80, 16, [70000, 69999, 71003, 70000], 7), (16, 8, 64, 16, [60000] * 4, 9),
    (32, 8, 128, 16, list(range(500, 8000, 230)), 5), (24, 8, 112, 64, list(range(500, 8000, 230)), 6)]


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_large_caches(ctx, case, fmt):
    qh, kvh, d, page, lens, queries = LONG[case]
    assert sum(lens) * kvh * d * 2 >= 200 << 20
    pool = Pool(case, kvh, d, page, fmt, lens, holes=case % 2 == 0)
    q, out = inputs(case, len(lens), queries, qh, d)
    if queries == 1:
        ctx.decode_kv8(pool.desc, q, out, lens, qh)
    else:
        ctx.prefill_kv8(pool.desc, q, out, queries, [n - queries for n in lens], qh)
    torch.cuda.synchronize()
    check(pool, q, out, lens, queries, qh)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
@pytest.mark.parametrize("which", [0, 1])
def test_nan_scale_inside_a_chunk(ctx, which, fmt):
    # K's or V's scale of one block: rows before it are what they were, rows that see it are NaN
    qh, kvh, d, queries, prior = 16, 4, 128, 700, 1300
    lens = [prior + queries]
    pool = Pool(7, kvh, d, 16, fmt, lens)
    # every page once, so that the block is one of the sequence
    pool.table[0] = torch.randperm(pool.pages, device="cuda")[:pool.pps].int()
    q, out = inputs(7, 1, queries, qh, d)
    block = 100  # tokens 1600 .. 1615: rows 300 on see it
    page = int(pool.table[0, block])
    kept = pool.s[page].clone()
    pool.s[page, :, :, which] = float("nan")
    ctx.prefill_kv8(pool.desc, q, out, queries, [prior], qh)
    torch.cuda.synchronize()
    first = block * 16 - prior
    assert out[0, first:].isnan().all()
    pool.s[page] = kept
    check(pool, q, out, lens, queries, qh, rows=slice(0, first))


@pytest.mark.parametrize("case", [(16, 4, 128, 16, [1500], 700), (16, 2, 64, 32, [100] * 20, 300)])
def test_chunk_first_recorded(case):
    # nothing is allocated yet, so the recorded chunk runs unsplit; later eager calls are split
    qh, kvh, d, page, priors, queries = case
    c = mslim_attn.Context()
    lens = [n + queries for n in priors]
    pool = Pool(9, kvh, d, page, E4M3, lens)
    q, out = inputs(9, len(lens), queries, qh, d)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    c.set_stream(stream.cuda_stream)
    with torch.cuda.graph(graph, stream=stream):
        c.prefill_kv8(pool.desc, q, out, queries, priors, qh)
    c.use_torch_stream()
    eager = torch.empty_like(out)
    for _ in range(3):
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        check(pool, q, out, lens, queries, qh, label="recorded")
        c.prefill_kv8(pool.desc, q, eager, queries, priors, qh)
        torch.cuda.synchronize()
        check(pool, q, eager, lens, queries, qh, label="eager")
    del graph
    c.close()


def test_chunk_graph_after_eager(ctx):
    # recorded with its buffers there: split, and the same bits as the eager call
    qh, kvh, d, page, priors, queries = CHUNKS[0]
    lens = [n + queries for n in priors]
    pool = Pool(10, kvh, d, page, INT8, lens)
    q, out = inputs(10, 1, queries, qh, d)
    eager = torch.empty_like(out)
    ctx.prefill_kv8(pool.desc, q, eager, queries, priors, qh)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(stream.cuda_stream)
    with torch.cuda.graph(graph, stream=stream):
        ctx.prefill_kv8(pool.desc, q, out, queries, priors, qh)
    ctx.use_torch_stream()
    for _ in range(3):
        out.fill_(-1)
        other = torch.empty_like(eager)
        ctx.prefill_kv8(pool.desc, q, other, queries, priors, qh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(other, eager)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_pool_past_32_bits(ctx, fmt):
    """Pages beyond 4 GiB of a pool: the bits that the same calls give over a small pool."""
    qh, kvh, d, page, n = 16, 4, 128, 1024, 1500
    results = []
    for pages in (4, 8704 + 4):  # 512 KiB a page: the last four lie past 4.25 GiB
        k, v = (torch.empty((pages, kvh, page, d), dtype=torch.uint8, device="cuda") for _ in range(2))
        s = torch.empty((pages, kvh, page // 16, 2), device="cuda")
        table = torch.tensor([[1, 3]], dtype=torch.int32, device="cuda") + (pages - 4)
        cache = mslim_attn.Kv8Cache(k, v, s, table, pages, 2, page, kvh, d, fmt)
        q, out = inputs(20, 1, n, qh, d)
        rows = torch.randn((2, 1, n, kvh, d), generator=torch.Generator(device="cuda").manual_seed(3),
                           device="cuda").bfloat16()
        turned = torch.empty_like(q)
        ctx.rope_append_kv8(cache, q, rows[0].contiguous(), rows[1].contiguous(), turned, 1, n,
                            torch.zeros(1, dtype=torch.int32, device="cuda"), qh, 1e4)
        ctx.prefill_kv8(cache, turned, out, n, [0], qh)
        few, one, back = torch.empty_like(q[:, :9]), torch.empty_like(q[:, :1]), torch.zeros_like(rows)
        ctx.prefill_kv8(cache, turned[:, -9:].contiguous(), few, 9, [n - 9], qh)
        ctx.decode_kv8(cache, turned[:, -1:].contiguous(), one, [n], qh)
        ctx.pages_gather_kv8(cache, 1, n, None, back[0], back[1])
        torch.cuda.synchronize()
        results.append((turned, out, few, one, back))
        del k, v, s, cache
    assert not any(x.isnan().any() for x in results[0])
    # a value is within half a step of its byte, and 2^-4 of itself or 2^-6 of the block's largest covers both formats
    v = results[0][4][1]
    assert ((v - rows[1]).abs() <= rows[1].abs() * 2.0 ** -4 + rows[1].abs().max() * 2.0 ** -6).all()
    for small, large in zip(*results):
        assert torch.equal(small, large)
