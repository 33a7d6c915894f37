"""The decoder runner on 8-bit K/V pages: bit for bit the library's calls made
one by one, near the runner on BF16 pages, and its refusals."""
import numpy as np
import pytest
import torch

import mslim_attn
from mslim_attn import MslimAttnError
from mslim_attn.model import Model, ModelSpec
from oracle.decoder import Spec, random_weights
from _data import logit_error, to_torch

pytestmark = pytest.mark.gpu

SPEC = Spec(layers=2, hidden=256, q_heads=8, kv_heads=2, head_dim=64, intermediate=512, vocab=1000)
FORMATS = {"paged_e4m3": mslim_attn.FORMAT_E4M3, "paged_int8": mslim_attn.FORMAT_INT8}
CONTEXT, SLOTS, CHUNK = 80, 3, 16


@pytest.fixture(scope="module")
def weights():
    return {k: to_torch(v) for k, v in random_weights(SPEC, np.random.default_rng(20261206)).items()}


def _model(ctx, weights, layout):
    spec = ModelSpec(SPEC.layers, SPEC.hidden, SPEC.q_heads, SPEC.kv_heads, SPEC.head_dim, SPEC.intermediate,
                     SPEC.vocab, SPEC.rms_eps, SPEC.rope_theta)
    return Model(ctx, spec, weights, max_batch=SLOTS, chunk_tokens=CHUNK, max_context=CONTEXT, kv_layout=layout)


class Calls:
    """The runner's layer loop as calls through the binding."""

    def __init__(self, ctx, w, fmt):
        self.ctx, self.w, s = ctx, w, SPEC
        self.pps = CONTEXT // 16
        pages = SLOTS * self.pps
        order = np.random.default_rng(1).permutation(pages).reshape(SLOTS, self.pps).astype(np.int32)
        self.table = torch.from_numpy(order).cuda()
        self.caches = []
        for _ in range(s.layers):
            k = torch.full((pages, s.kv_heads, 16, s.head_dim), 255, dtype=torch.uint8, device="cuda")
            scales = torch.full((pages, s.kv_heads, 1, 2), float("nan"), device="cuda")
            self.caches.append([mslim_attn.Kv8Cache(k, v, scales, table, pages, self.pps, 16, s.kv_heads, s.head_dim, fmt)
                                for v in (torch.full_like(k, 255),)
                                for table in [self.table] + [self.table[i] for i in range(SLOTS)]])

    def forward(self, ids, positions, slot=None):
        """Logits of the last row (a chunk of one slot) or of every row (a step of slots 0 ..)."""
        s, c, n = SPEC, self.ctx, len(ids)
        new = lambda *shape: torch.empty(shape, dtype=torch.int16, device="cuda")  # noqa: E731
        qd, kvd = s.q_heads * s.head_dim, s.kv_heads * s.head_dim
        x, q, qr, attn, k, v, act = (new(n, z) for z in (s.hidden, qd, qd, qd, kvd, kvd, s.intermediate))
        c.embed(self.w["embed"], s.vocab, s.hidden, torch.tensor(ids, dtype=torch.int32, device="cuda"), n, x)
        pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
        for layer in range(s.layers):
            w = {t: self.w[f"layers.{layer}.{t}"] for t in ("input_norm", "q", "k", "v", "o", "post_norm", "gate",
                                                            "up", "down")}
            cache = self.caches[layer][0 if slot is None else slot + 1]
            c.rmsnorm_gemm_qkv(w["input_norm"], s.rms_eps, w["q"], w["k"], w["v"], x, q, k, v, s.hidden, qd, kvd, n)
            batch, tokens = (n, 1) if slot is None else (1, n)
            c.rope_append_kv8(cache, q, k, v, qr, batch, tokens, pos, s.q_heads, s.rope_theta)
            if slot is None:
                c.decode_kv8(cache, qr, attn, [p + 1 for p in positions], s.q_heads)
            else:
                c.prefill_kv8(cache, qr, attn, n, positions[:1], s.q_heads)
            c.gemm_bf16_add(w["o"], attn, x, x, qd, s.hidden, n)
            c.rmsnorm_gemm_swiglu(w["post_norm"], s.rms_eps, w["gate"], w["up"], x, act, s.hidden, s.intermediate, n)
            c.gemm_bf16_add(w["down"], act, x, x, s.intermediate, s.hidden, n)
        rows = x if slot is None else x[-1:].contiguous()
        logits = new(len(rows), s.vocab)
        c.rmsnorm_gemm_bf16(self.w["final_norm"], s.rms_eps, self.w["lm_head"], rows, logits, s.hidden, s.vocab,
                            len(rows))
        torch.cuda.synchronize()
        return logits.cpu().numpy().view(np.uint16)


PROMPTS = [41, 3, 17]


@pytest.mark.parametrize("layout", sorted(FORMATS))
def test_runner_is_the_calls_one_by_one(ctx, weights, layout):
    rng = np.random.default_rng(9)
    calls, model = Calls(ctx, weights, FORMATS[layout]), _model(ctx, weights, layout)
    exact = _model(ctx, weights, "paged")
    try:
        for turn in range(2):  # the second after a reset, into pages that hold the first
            toks, at = [], []
            for slot, n in enumerate(PROMPTS):
                prompt = [int(t) for t in rng.integers(0, SPEC.vocab, n)]
                model.reset(slot)
                exact.reset(slot)
                toks.append(model.prefill_only(slot, prompt))
                exact.prefill_only(slot, prompt)
                for a in range(0, n, CHUNK):
                    want = calls.forward(prompt[a:a + CHUNK], [a], slot)
                assert np.array_equal(model.logits().reshape(-1), want.reshape(-1)), (turn, slot)
                at.append(n)
            for step in range(6):
                nxt = model.forward_batch(toks)
                want = calls.forward(toks, at)
                assert np.array_equal(model.logits().reshape(-1), want.reshape(-1)), (turn, step)
                exact.forward_batch(toks)
                # Each cached value is off by at most half a step of 2^-4 of
                # its size (E4M3; INT8 by 2^-7 of the block's largest): the
                # logits of two layers of it stay well within a quarter.
                assert logit_error(model.logits(), exact.logits())[1] < 0.25, (turn, step)
                toks, at = nxt, [p + 1 for p in at]
    finally:
        model.close()
        exact.close()


def test_runner_refuses_what_needs_exact_pages(ctx, weights, tmp_path):
    model = _model(ctx, weights, "paged_int8")
    try:
        model.prefill_only(0, [1, 2, 3])
        with pytest.raises(MslimAttnError, match="digest"):
            model.logical_kv_sha256(0)
        with pytest.raises(MslimAttnError, match="ColdStore"):
            model.attach_cold_store(1, str(tmp_path))
        model.forward_batch([5])  # and goes on
    finally:
        model.close()
