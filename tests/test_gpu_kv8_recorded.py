"""Calls of the 8-bit K/V cache recorded into graphs, on other streams, and by
two contexts at once.  Every replay is compared with the eager result, with
eager work and synchronisations between them."""
import numpy as np
import pytest
import torch

import mslim_attn
from _data import normal_bf16, to_torch
from _kv8 import E4M3, INT8
from test_gpu_kv8 import THETA, Cache, check_attention

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh():
    c = mslim_attn.Context()
    c.use_torch_stream()
    yield c
    torch.cuda.synchronize()
    c.close()


def record(c, call):
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    c.set_stream(stream.cuda_stream)
    with torch.cuda.graph(graph, stream=stream):
        call()
    c.use_torch_stream()
    return graph


def filled(seed, lens, kvh, d, fmt):
    rng = np.random.default_rng(seed)
    cache = Cache(rng, lens, kvh, d, fmt, 16)
    cache.fill(rng, lens)
    return rng, cache


def attention(c, cache, q, lens, rows, qh):
    if rows == 1:
        return lambda out: c.decode_kv8(cache.desc, q, out, lens, qh)
    return lambda out: c.prefill_kv8(cache.desc, q, out, rows, [n - rows for n in lens], qh)


# lengths, query rows, q heads, kv heads, head_dim; and a call of the same
# context that needs larger buffers.
CALLS = {
    "decode": (([700, 3, 0], 1, 8, 2, 128), ([3000] * 40, 1, 64, 8, 128)),
    "decode, one long": (([4000], 1, 4, 1, 64), ([9000] * 4, 1, 32, 8, 128)),
    "few rows": (([900, 20], 5, 8, 2, 128), ([3000] * 8, 8, 64, 8, 128)),
    "many rows": (([700], 200, 8, 2, 128), ([2500], 1200, 32, 8, 128)),
    "wide heads": (([500], 60, 4, 2, 256), ([2000] * 2, 60, 16, 4, 256)),
}


@pytest.mark.parametrize("name", CALLS)
def test_first_call_under_capture(fresh, name):
    # nothing is allocated yet: the recorded call runs unsplit
    lens, rows, qh, kvh, d = CALLS[name][0]
    rng, cache = filled(31, lens, kvh, d, E4M3)
    qb = normal_bf16(rng, (len(lens), rows, qh, d))
    call = attention(fresh, cache, to_torch(qb), lens, rows, qh)
    got, want = (torch.full((len(lens), rows, qh, d), -1, dtype=torch.int16, device="cuda") for _ in range(2))
    graph = record(fresh, lambda: call(got))
    for _ in range(3):
        got.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(cache, qb, got, lens, rows, "recorded")
        call(want)
        torch.cuda.synchronize()
        check_attention(cache, qb, want, lens, rows, "eager")


@pytest.mark.parametrize("name", CALLS)
def test_replay_after_a_larger_call(fresh, name):
    made = []
    for k, (lens, rows, qh, kvh, d) in enumerate(CALLS[name]):
        rng, cache = filled(40 + k, [min(n, 200) for n in lens], kvh, d, INT8)
        # the table's rows repeat their pages, so long sequences need no long pool
        need = -(-max(lens) // 16)
        cache.table = np.tile(cache.table, (1, -(-need // cache.table.shape[1])))[:, :need].copy()
        cache.pool.scales[np.isnan(cache.pool.scales) | np.isinf(cache.pool.scales)] = 0.5
        cache.pps = need
        cache.upload()
        q = to_torch(normal_bf16(rng, (len(lens), rows, qh, d)))
        made.append((attention(fresh, cache, q, lens, rows, qh), torch.zeros_like(q), cache, q))
    (call, want, *_), (big_call, big, *_) = made
    call(want)
    torch.cuda.synchronize()
    got = torch.zeros_like(want)
    graph = record(fresh, lambda: call(got))
    for _ in range(3):
        big_call(big)
        again = torch.zeros_like(want)
        call(again)
        got.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, want)
    big_again = torch.zeros_like(big)
    big_call(big_again)
    torch.cuda.synchronize()
    assert torch.equal(big, big_again)


@pytest.mark.parametrize("fmt", [E4M3, INT8])
def test_recorded_step_follows_its_positions(fresh, fmt):
    # a step's append and attention recorded once: the positions are device
    # memory, so replays append wherever they say; every replay against the
    # same calls made eagerly on a copy of the cache
    qh, kvh, d, lens = 8, 2, 128, [60, 17, 33]
    rng, cache = filled(50, [n + 8 for n in lens], kvh, d, fmt)
    _, other = filled(50, [n + 8 for n in lens], kvh, d, fmt)
    b = len(lens)
    q, k, v, turned, out = (torch.zeros((b, h, d), dtype=torch.int16, device="cuda") for h in (qh, kvh, kvh, qh, qh))
    turned2, out2 = torch.zeros_like(turned), torch.zeros_like(out)
    pos = torch.zeros(b, dtype=torch.int32, device="cuda")
    full = [n + 8 for n in lens]

    def step(c, at, rot, to):
        fresh.rope_append_kv8(c.desc, q, k, v, rot, b, 1, at, qh, THETA)
        fresh.decode_kv8(c.desc, rot, to, full, qh)

    step(cache, pos - 1, turned, out)  # rows before the table: nothing is stored, buffers are made
    graph = record(fresh, lambda: step(cache, pos, turned, out))
    for i in range(8):
        for t, h in ((q, qh), (k, kvh), (v, kvh)):
            t.copy_(to_torch(normal_bf16(rng, (b, h, d), 1.5 ** i)))
        pos.copy_(torch.tensor([n + i for n in lens], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        step(other, pos, turned2, out2)
        torch.cuda.synchronize()
        assert torch.equal(turned, turned2) and torch.equal(out, out2), i
        for x, y in ((cache.k, other.k), (cache.v, other.v), (cache.s.view(torch.int32), other.s.view(torch.int32))):
            assert torch.equal(x, y), i


def test_two_contexts_on_two_streams():
    # each with its own buffers, at once, many times
    made = []
    for seed, (lens, rows, qh, kvh, d) in ((60, ([3000, 500], 1, 32, 8, 128)), (61, ([800], 300, 8, 2, 128))):
        c, stream = mslim_attn.Context(), torch.cuda.Stream()
        c.set_stream(stream.cuda_stream)
        rng, cache = filled(seed, lens, kvh, d, E4M3)
        q = to_torch(normal_bf16(rng, (len(lens), rows, qh, d)))
        call = attention(c, cache, q, lens, rows, qh)
        want = torch.zeros_like(q)
        torch.cuda.synchronize()
        call(want)
        c.synchronize()
        made.append((c, call, want, [torch.zeros_like(q) for _ in range(20)], cache, q))
    torch.cuda.synchronize()
    for i in range(20):
        for _, call, _, outs, *_ in made:
            call(outs[i])
    torch.cuda.synchronize()
    for c, _, want, outs, *_ in made:
        assert all(torch.equal(o, want) for o in outs)
        c.close()


def test_both_decodes_share_a_context(ctx):
    # the BF16 decode and this one use the same partials and counters in turn
    lens, qh, kvh, d = [2000, 300], 32, 8, 128
    rng, cache = filled(70, lens, kvh, d, E4M3)
    q = to_torch(normal_bf16(rng, (2, qh, d)))
    k, v = (to_torch(normal_bf16(rng, (2, 2000, kvh, d))) for _ in range(2))
    outs = [[torch.zeros_like(q) for _ in range(2)] for _ in range(5)]
    for a, b in outs:
        ctx.decode_dense(q, k, v, a, lens, qh, kvh, d, seq_stride_tokens=2000)
        ctx.decode_kv8(cache.desc, q, b, lens, qh)
    torch.cuda.synchronize()
    for a, b in outs[1:]:
        assert torch.equal(a, outs[0][0]) and torch.equal(b, outs[0][1])
