"""The dense operators as a verify step uses them, with the cache, the attention and the MoE block between them: hidden states
-> q, k, v projection -> norms, rotary positions, store -> paged attention -> output projection + residual -> MoE block ->
language-model head -> which drafts stay.  Each operator's inputs are what the one before it has left on the device, so each is
held to its own 64-bit definition on exactly those values; the first call's results are also what a captured graph replays."""
import numpy as np
import pytest
import torch

import on_device_sd_amd as odsd
from on_device_sd_amd import ops
from on_device_sd_amd.workloads import MoEWorkload, LayerInputs
from oracle import dense_oracle as orc
from tests import helpers

pytestmark = pytest.mark.gpu
HID, HEADS, KV, D, VOCAB, BLOCK = 256, 8, 2, 64, 1003, 16
WL = MoEWorkload("step", T=0, H=HID, E=8, K=2, I=256, renorm=True, act_dtype=torch.bfloat16, seed=3)


class Step:
    def __init__(self, dev):
        self.dev = dev
        g = torch.Generator(device=dev).manual_seed(0)
        rnd = lambda *s, m=1.0: (torch.randn(*s, generator=g, device=dev) * m).bfloat16()  # noqa: E731
        self.w_qkv, self.b_qkv, self.w_o = rnd((HEADS + 2 * KV) * D, HID, m=0.06), rnd((HEADS + 2 * KV) * D, m=0.1), rnd(HID, HEADS * D, m=0.04)
        self.w_head, self.qn, self.kn, self.norm = rnd(VOCAB, HID, m=0.1), 1 + rnd(D, m=0.1), 1 + rnd(D, m=0.1), 1 + rnd(HID, m=0.1)
        inp = LayerInputs(WL, dev)
        self.gate = inp.gate_weight()
        self.bank, _ = helpers.build_bank(WL, dev, inp, keep=())
        self.table = self.bank.table()
        self.inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        seqs = {}
        block = iter(torch.randperm(40, generator=torch.Generator().manual_seed(1)).tolist())
        for s, (cached, drafts) in enumerate([(33, 4), (5, 0), (17, 2), (16, 3)]):
            n = cached + drafts
            seqs[s] = odsd.SequenceSlots(BLOCK, [next(block) for _ in range(-(-n // BLOCK))], n, cached)
        self.ctx = odsd.build_verify_context(seqs, [0, 1, 2, 3], dev)
        self.lens = self.ctx["verify_query_lens"].tolist()
        self.positions = torch.cat([torch.arange(st.draft_start_num_tokens - 1, st.num_tokens) for st in seqs.values()]).to(dev)
        T = sum(self.lens)
        self.kc, self.vc = rnd(40 * BLOCK, KV * D), rnd(40 * BLOCK, KV * D)
        self.hidden = rnd(T, HID)
        self.drafts = torch.randint(0, VOCAB, (T - 4,), generator=g, device=dev)
        self.draft_logits = rnd(T - 4, VOCAB, m=2.0).float()
        self.draft_logits.scatter_(1, self.drafts[:, None], 1.0)
        self.accept_u, self.sample_u = torch.rand(T - 4, generator=g, device=dev), torch.rand(4, generator=g, device=dev)

    def run(self):
        o = {}
        o["x"] = ops.rmsnorm(self.hidden, self.norm)
        o["qkv"] = ops.linear(o["x"], self.w_qkv, self.b_qkv)
        o["q0"], o["k0"], o["v0"] = (t.unflatten(1, (-1, D)) for t in o["qkv"].split([HEADS * D, KV * D, KV * D], 1))
        o["q"] = odsd.rotary_store_kvcache(o["q0"], o["k0"], o["v0"], self.positions, self.inv, self.kc, self.vc, self.ctx["slot_mapping"],
                                           self.ctx["verify_q_indices"], q_weight=self.qn, k_weight=self.kn)
        o["attn"] = odsd.paged_attention(o["q"], self.kc, self.vc, self.ctx, KV, BLOCK)
        o["h"] = ops.linear(o["attn"].flatten(1), self.w_o, residual=self.hidden)
        o["moe"] = ops.moe_forward(ops.rmsnorm(o["h"], self.norm), self.gate, self.table, WL.K, WL.I, renorm=True).out_f32
        o["last"] = (o["h"].float() + o["moe"]).bfloat16()
        o["logits"] = ops.linear(o["last"], self.w_head, out_dtype=torch.float32)
        r = odsd.verify_drafts(o["logits"], self.drafts, self.ctx, self.accept_u, self.sample_u, draft_logits=self.draft_logits, temperature=0.9)
        o["tokens"], o["accepted"], o["probs"] = r.tokens, r.num_accepted, r.accept_probs
        return o


def f64(t):
    return t.double().cpu().numpy()


def test_step_operator_by_operator(dev):
    s = Step(dev)
    old_k, old_v = s.kc.clone(), s.vc.clone()
    o = s.run()
    e = 2.0 ** -8                                            # half a step of bf16
    want, size, _ = orc.linear(f64(o["x"]), f64(s.w_qkv), f64(s.b_qkv))
    assert (np.abs(f64(o["qkv"]) - want) <= e * np.abs(want) + 64 * 2.0 ** -23 * size).all()
    pos, inv = f64(s.positions), f64(s.inv)
    for got, src, w in ((o["q"], o["q0"], s.qn), (None, o["k0"], s.kn)):
        want, size = orc.rotary(f64(src), pos, inv, weight=f64(w))
        if got is None:                                      # the keys: where the context says, and nowhere else
            rows, slots = s.ctx["verify_q_indices"].tolist(), s.ctx["slot_mapping"].tolist()
            want, size = want[rows].reshape(len(rows), -1), size[rows].reshape(len(rows), -1)
            got = s.kc[slots]
            old_k[slots], old_v[slots] = s.kc[slots], o["v0"].flatten(1)[rows]
            assert torch.equal(s.kc, old_k) and torch.equal(s.vc, old_v)
        assert (np.abs(f64(got) - want) <= e * np.abs(want) + 2.0 ** -19 * size).all()
    want, size, _ = orc.linear(f64(o["attn"].flatten(1)), f64(s.w_o), residual=f64(s.hidden))
    assert (np.abs(f64(o["h"]) - want) <= e * np.abs(want) + 64 * 2.0 ** -23 * (size + np.abs(f64(s.hidden)))).all()
    want, size, _ = orc.linear(f64(o["last"]), f64(s.w_head))
    assert (np.abs(f64(o["logits"]) - want) <= 32 * 2.0 ** -23 * size).all()
    tokens, accepted, probs = orc.verify(f64(o["logits"]), f64(s.drafts), s.lens, f64(s.accept_u), f64(s.sample_u), f64(s.draft_logits), np.float32(0.9))
    assert o["tokens"].tolist() == tokens.tolist() and o["accepted"].tolist() == accepted.tolist()
    assert np.allclose(f64(o["probs"]), probs, rtol=2.0 ** -23, atol=1e-40)


def test_step_captured_and_on_another_stream(dev):
    s = Step(dev)
    names = ("qkv", "q", "h", "logits", "tokens", "accepted", "probs")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = s.run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        again = s.run()
        torch.cuda.synchronize()
        for n in names:
            assert torch.equal(out[n], again[n]), (i, n)
            assert i or torch.equal(first[n], again[n]), n
        s.hidden.normal_()
        s.accept_u.uniform_()
