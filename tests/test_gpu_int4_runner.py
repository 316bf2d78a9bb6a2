"""GPU: the runner's Step over a 4-bit pool, the model's rows normed and rotated by qk_norm_rope, for
several consecutive steps with drafts, rejections and truncated tables. Each step's layer-0 attention
equals float64 attention over what the pool holds, its rows' keys are within half a step of the
normed and rotated ones in float64, and the decision equals the oracle's."""
import math

import numpy as np
import pytest
import torch

import int4_ref as ref
from gollmgo_amd._lib import DType
from gollmgo_amd.blocks import BlockPool, BlockTable
from gollmgo_amd.runner import ACCEPT_GREEDY, RunnerConfig, SamplingParams, VerifyRunner
from helpers import say
from oracle import oracle as ora
from test_gpu_rope import tolerance, want
from test_gpu_runner_step import Seq, SynthModel, engine_batch, prefill

pytestmark = pytest.mark.gpu


class RopeModel(SynthModel):
    """SynthModel with one fused projection per layer whose rows qk_norm_rope norms and rotates."""

    def __init__(self, **kw):
        super().__init__(**kw)
        import gollmgo_amd.verify as gv
        self.gv = gv
        g = torch.Generator().manual_seed(99)
        self.Wqkv = [torch.cat([q, k, v], 1).contiguous() for q, k, v in zip(self.Wq, self.Wk, self.Wv)]
        D = self.head_dim
        self.wq, self.wk = ((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().cuda() for _ in range(2))
        self.freq = torch.from_numpy((10000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)).cuda()

    def qkv(self, layer, positions):
        hq, hk, d = self.num_q_heads, self.num_kv_heads, self.head_dim
        n = self.B * self.R
        if positions is None:  # the prefill's rows: 0, 1, ... of each sequence
            positions = torch.arange(self.R, dtype=torch.int32, device="cuda").repeat(self.B, 1)
        x = (self.x.to(torch.bfloat16) @ self.Wqkv[layer]).view(n, hq + 2 * hk, d)
        pos = positions.reshape(n).contiguous()
        q, k = self.gv.qk_norm_rope(x[:, :hq], x[:, hq:hq + hk], pos, self.freq, self.wq, self.wk)
        if layer == 0:
            self.q0, self.k_raw, self.pos = q.view(self.B, self.R, hq, d), x[:, hq:hq + hk].clone(), pos
        return q.view(self.B, self.R, hq, d), k, x[:, hq + hk:].contiguous()


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 4, 64)])
def test_runner_steps_on_a_4_bit_pool(Hq, Hkv, D):
    B, K, P, steps, bs = 12, 4, 20, 8, 16
    model = RopeModel(seed=4, Hq=Hq, Hkv=Hkv, D=D)
    cfg = RunnerConfig(num_blocks=300, block_size=bs, kv_dtype=DType.INT4, max_drafts=K,
                       sampling=SamplingParams(temperature=0.0, seed=1), acceptance=ACCEPT_GREEDY)
    runner = VerifyRunner(model, cfg)
    runner.warmup(B, P + steps * (K + 1) + 8)
    pool = BlockPool(cfg.num_blocks, bs, order=np.random.default_rng(5).permutation(cfg.num_blocks).tolist())
    rng = np.random.default_rng(8)
    succ = model.succ.cpu().numpy()
    seqs = []
    for i in range(B):
        t = [int(rng.integers(0, model.vocab))]
        while len(t) < P:
            t.append(int(succ[t[-1]]) if rng.random() < 0.95 else int(rng.integers(0, model.vocab)))
        seqs.append(Seq(i, t, BlockTable(pool)))
    say(f"4-bit runner prefill D={D}")
    last = prefill(runner, model, seqs, P)
    for i, s in enumerate(seqs):
        s.tokens.append(int(ora.argmax(last[i])))
    scale = 1 / math.sqrt(D)
    accepted = rejected = 0
    for step in range(steps):
        say(f"4-bit runner step {step}")
        batch = engine_batch(seqs, K, 3)
        runner.step(batch)
        torch.cuda.synchronize()
        inp = runner.last_inputs
        acc, tok = runner.last_decision
        L = runner.last_logits.float().cpu().numpy()
        ea, et = ora.accept_greedy(L, inp.drafts, inp.n_drafts)
        assert np.array_equal(acc, ea) and np.array_equal(tok, et)
        Kv, Vv, k_span, v_span = ref.pool_values(runner.kv, 0, spans=True)
        q = model.q0.double().cpu().numpy()
        out, mag, reach, least = ref.attention(q, Kv, Vv, inp.ctx_lens, inp.row_counts, inp.block_tables, scale,
                                               np.zeros(q.shape), v_span)
        tol = ref.attention_tolerance(q, Kv, k_span, scale, out, mag, reach, least, "bf16", "bf16")
        got = model.out0.double().cpu().numpy()
        for b in range(B):
            n = int(inp.row_counts[b])
            assert (np.abs(got[b, :n] - out[b, :n]) <= tol[b, :n]).all()
        # The step's keys in the pool: normed, rotated, rounded to bf16, then to the row's codes.
        pos = model.pos.cpu().numpy()
        kw, km = want(model.k_raw.float().cpu().numpy(), model.wk.float().cpu().numpy(), 1e-6, pos[None], np.zeros(D // 2, int),
                      model.freq.cpu().numpy(), "halves")
        near = tolerance(kw, km, D, float(pos.max()), "bf16")
        for b in range(B):
            n = int(inp.row_counts[b])
            p = inp.ctx_lens[b] - n + np.arange(n)
            rows = slice(b * inp.rows_per_seq, b * inp.rows_per_seq + n)
            held = Kv[inp.block_tables[b, p // bs], :, p % bs]
            reach_k = np.maximum(kw[rows].max(-1), 0) - np.minimum(kw[rows].min(-1), 0) + 2 * near[rows].max(-1)
            assert (np.abs(held - kw[rows]) <= near[rows] + (reach_k / 15 * (17 / 32) * (1 + 2.0 ** -20))[..., None]).all()
        for b, s in enumerate(seqs):
            n, a = int(inp.n_drafts[b]), int(acc[b])
            s.table.truncate(n - a)
            s.tokens += [int(x) for x in inp.drafts[b, :a]] + [int(tok[b])]
            accepted += a
            rejected += n - a
    assert accepted > 0 and rejected > 0
    runner.close()
