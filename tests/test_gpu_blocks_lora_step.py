"""One layer's attention part of a batched step, as a server with adapters and
long contexts runs it: q|k|v projection + adapters, RoPE + append, key ranges,
block selection, attention over the lists, O projection onto the residual +
adapters. Each stage is held to the 64-bit form of what the stage before wrote;
then the whole is captured and replayed along the sequences."""
import numpy as np
import pytest
import torch

import block_ref as ref
from pkg import layerops

pytestmark = pytest.mark.gpu

D, HK, HQ, H = 128, 2, 8, 256
NQ, NK = HQ * D, HK * D
L = None


def setup_module(module):
    global L
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L = layerops()
    torch.cuda.init()
    L.use_stream()


def f64(t):
    torch.cuda.synchronize()
    return t.float().cpu().numpy().astype(np.float64)


class Step:
    def __init__(self, pos, block=32, top_k=4, bits=8, seed=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std)  # noqa: E731
        self.rows, self.block, self.top_k, self.bits = len(pos), block, top_k, bits
        need = [(p + 80) // block + 1 for p in pos]  # room to go on
        self.stride = block * sum(need)
        order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
        rows = (order[:, None] * block + torch.arange(block, device="cuda", dtype=torch.int32)).reshape(-1)
        at = np.cumsum([0] + need) * block
        self.tables = [rows[at[i]:at[i + 1]].contiguous() for i in range(self.rows)]
        self.row_pt = torch.tensor([t.data_ptr() for t in self.tables], dtype=torch.int64, device="cuda")
        self.pos = torch.tensor(pos, dtype=torch.int32, device="cuda")
        self.slot = torch.stack([t[p] for t, p in zip(self.tables, pos)])
        self.cos, self.sin = L.rope_tables(1e4, D, max(pos) + 80)
        self.arena = L.KvArena(bits, HK, self.stride)
        self.ranges = L.KvRanges(HK, self.stride, block)
        # the contexts so far, appended and ranged by the same entry points
        for t, p in zip(self.tables, pos):
            if p:
                kv = rnd(p, 2 * NK).to(torch.bfloat16)
                L.rope_append(self.arena, None, kv[:, :NK], kv[:, NK:], self.cos, self.sin, d_pt=t)
                L.kv_ranges(self.arena, self.ranges, p, d_pt=t)
        fp8 = lambda n, k: rnd(n, k, std=8).to(torch.float8_e4m3fn)  # noqa: E731
        self.wqkv, self.wo = fp8(NQ + 2 * NK, H), fp8(H, NQ)
        self.s_qkv, self.s_o = (0.03, 0.01, 0.01), 0.004
        lora = lambda parts, n, k: ((rnd(4, parts, 16, k) / k ** 0.5).to(torch.bfloat16),  # noqa: E731
                                    rnd(4, n, 16, std=0.1).to(torch.bfloat16))
        self.lq, self.lo = lora(3, NQ + 2 * NK, H), lora(1, H, NQ)
        self.alpha = 0.5 + torch.rand(4, generator=g, device="cuda")
        self.adapter = torch.tensor([r % 5 - 1 for r in range(self.rows)], dtype=torch.int32, device="cuda")
        self.x = rnd(self.rows, H).to(torch.bfloat16)
        self.hidden = rnd(self.rows, H).to(torch.bfloat16)
        self.hidden0 = self.hidden.clone()
        n = self.rows
        z = lambda name, *a: torch.zeros(max(16, L.call_size(name, *a)), dtype=torch.uint8, device="cuda")  # noqa: E731
        self.w_lora = z("granite4_lora_work_bytes", n, NQ + 2 * NK, max(H, NQ), 16, NQ, NQ + NK)
        self.w_sel = z("granite4_block_select_work_bytes", n, HK, self.stride, block)
        self.w_att = z("granite4_attn_blocks_scratch_bytes", HQ, n, top_k, block)
        self.qkv = torch.empty((n, NQ + 2 * NK), dtype=torch.bfloat16, device="cuda")
        self.plain_qkv = torch.empty_like(self.qkv)
        self.q_rot = torch.empty((n, NQ), dtype=torch.bfloat16, device="cuda")
        self.sel = torch.empty((n, HK, top_k), dtype=torch.int32, device="cuda")
        self.out = torch.empty_like(self.q_rot)
        self.mid = torch.empty_like(self.hidden)

    def run(self):
        segs, where = (NQ, NQ + NK), dict(row_pos=self.pos, row_pt=self.row_pt)
        L.prefill_gemm(self.x, self.wqkv.view(torch.uint8), scales=self.s_qkv, segs=segs, out=self.plain_qkv)
        L.lora_add(self.x, *self.lq, self.alpha, self.adapter, base=self.plain_qkv, segs=segs,
                   out=self.qkv, work=self.w_lora)
        L.rope_append(self.arena, self.qkv[:, :NQ], self.qkv[:, NQ:NQ + NK], self.qkv[:, NQ + NK:],
                      self.cos, self.sin, pos_rows=self.pos, arena_rows=self.slot, k_round_bf16=True,
                      q_rot=self.q_rot)
        L.kv_ranges(self.arena, self.ranges, self.rows, **where)
        L.block_select(self.q_rot, self.ranges, self.top_k, work=self.w_sel, sel=self.sel, **where)
        L.attn_blocks(self.q_rot, self.arena, self.sel, self.block, 1 / 16, scratch=self.w_att,
                      out=self.out, **where)
        L.prefill_gemm(self.out, self.wo.view(torch.uint8), L.GEMM_RESIDUAL, (self.s_o,) * 3,
                       out=self.mid, residual=self.hidden0, resid_scale=0.22)
        L.lora_add(self.out, *self.lo, self.alpha, self.adapter, base=self.mid, mult=0.22,
                   out=self.hidden, work=self.w_lora)

    def outputs(self):
        return [self.qkv, self.arena.k, self.arena.v, self.ranges.codes, self.ranges.scale, self.sel,
                self.out, self.hidden]


def lora_ok(x, ab, s, base, segs, mult, got):
    want, tol = ref.lora(f64(x), f64(ab[0]), f64(ab[1]), s.alpha.cpu().numpy().astype(np.float64),
                         s.adapter.cpu().numpy(), f64(base), segs, np.float64(np.float32(mult)))
    d = np.abs(f64(got) - want)
    assert (d <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("pos", [[0], [31], [130, 5, 95, 0, 318, 64, 63]])
def test_a_layers_step(pos):
    s = Step(pos)
    s.run()
    torch.cuda.synchronize()
    big = 2**31 - 1
    lora_ok(s.x, s.lq, s, s.plain_qkv, (NQ, NQ + NK), 1.0, s.qkv)
    # what the pool holds now, as values
    kc = s.arena.k.view(torch.int8).cpu().numpy().astype(np.float32)
    vc = s.arena.v.view(torch.int8).cpu().numpy().astype(np.float32)
    kval = (kc * s.arena.k_scale.cpu().numpy()).astype(np.float64)
    vval = (vc * s.arena.v_scale.cpu().numpy()).astype(np.float64)
    rc, rs = s.ranges.codes.cpu().numpy(), s.ranges.scale.cpu().numpy()
    tables = [t.cpu().numpy() for t in s.tables]
    wc, ws = np.zeros_like(rc, np.int64), np.zeros_like(rs)
    for t, p in zip(tables, pos):
        wc, ws = ref.ranges(kval, s.block, t, s.stride, range((p + 1) // s.block), wc, ws)
    np.testing.assert_array_equal(rc, wc)
    np.testing.assert_array_equal(rs, ws)
    sel = s.sel.cpu().numpy()
    for r, p in enumerate(pos):
        q = f64(s.q_rot)[r].reshape(HQ, D).astype(np.float32)
        np.testing.assert_array_equal(sel[r], ref.select(q, rc, rs, s.block, p, tables[r], s.stride,
                                                         s.top_k, 1, 2))
        want, tol = ref.attend(q, kval, vval, s.block, p, tables[r], s.stride, sel[r], 1 / 16)
        assert (np.abs(f64(s.out)[r].reshape(HQ, D) - want) <= tol).all()
    lora_ok(s.out, s.lo, s, s.mid, (big, big), 0.22, s.hidden)


def test_steps_in_a_graph():
    """The step captured once and replayed while the sessions go on (with eager work and
    waits between): every output, the pool and the ranges included, as the eager calls'."""
    pos = [30, 5, 95, 0, 190]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        L.use_stream(stream)
        a, b = Step(pos), Step(pos)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            b.run()
        for i in range(40):
            for s in (a, b):
                s.pos.copy_(torch.tensor([p + i for p in pos], dtype=torch.int32))
                s.slot.copy_(torch.stack([t[p + i] for t, p in zip(s.tables, pos)]))
                s.x.copy_(torch.roll(a.x if s is b else s.x, 1 if s is a else 0, 1))
                s.adapter.copy_(torch.roll(a.adapter, 1) if s is a else a.adapter)
            a.run()
            graph.replay()
            if i % 7 == 0:
                torch.cuda.synchronize()
            for x, y in zip(a.outputs(), b.outputs()):
                assert torch.equal(x, y), i
        torch.cuda.synchronize()
    L.use_stream()
