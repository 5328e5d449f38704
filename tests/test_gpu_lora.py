"""granite4_lora_add on the GPU against the float64 form in block_ref.lora, whose
bound counts the kernel's roundings (a bf16 result adds 2^-8 of itself)."""
import numpy as np
import pytest
import torch

import block_ref as ref
from pkg import layerops

pytestmark = pytest.mark.gpu

L = None


def setup_module(module):
    global L
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    L = layerops()
    torch.cuda.init()
    L.use_stream()


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


class Case:
    def __init__(self, M, N, K, rank, count, segs=None, fp8=False, f32=False, seed=0, pad=8):
        rng = self.rng = np.random.default_rng(seed + M + N + K + rank)
        self.M, self.N, self.K, self.rank, self.count = M, N, K, rank, count
        self.segs, self.fp8, self.f32 = segs or (2**31 - 1, 2**31 - 1), fp8, f32
        self.parts = 1 + sum(s < N for s in self.segs)
        self.pad = pad
        ldx = self.ldx = K + 2 * pad
        x = rng.standard_normal((M, ldx)).astype(np.float32)
        if fp8:
            self.xs = np.float32(0.0173)
            t = torch.from_numpy(x / self.xs * np.float32(0.2)).clamp(-448, 448).to(torch.float8_e4m3fn)
            self.x = t.view(torch.uint8).numpy()
            self.xv = (t.float().numpy()[:, :K].astype(np.float64) * np.float64(self.xs))
        else:
            self.x = ref.bf16(x)
            self.xv = ref.f32(self.x)[:, :K].astype(np.float64)
        self.A = ref.bf16((rng.standard_normal((count, self.parts, rank, K)) / np.sqrt(K)).astype(np.float32))
        self.B = ref.bf16((rng.standard_normal((count, N, rank)) * 0.1).astype(np.float32))
        self.alpha = (0.5 + rng.random(count)).astype(np.float32)
        self.ldb, self.ldy = N + 8, N + 16
        b = rng.standard_normal((M, self.ldb)).astype(np.float32)
        self.base = b if f32 else ref.bf16(b)
        self.adapter = rng.integers(-1, count, M).astype(np.int32)

    def run(self, mult=1.0, base=True, in_place=False, stream=None):
        t = torch.float32 if self.f32 else torch.int16
        d_base = dev(self.base)
        y = d_base if in_place else torch.full((self.M + 1, self.ldy), 77, dtype=t, device="cuda")
        ldy = self.ldb if in_place else self.ldy
        n = L.call_size("granite4_lora_work_bytes", self.M, self.N, self.K, self.rank, *self.segs)
        work = torch.full((n + 16,), 255, dtype=torch.uint8, device="cuda")  # NaN, were it read first
        work[:2048] = 0  # where calls count
        L.call("granite4_lora_add", int(self.f32), dev(self.x), 8 if self.fp8 else 16, self.ldx,
               dev(np.array([self.xs])) if self.fp8 else None, dev(self.A), dev(self.B),
               dev(self.alpha), self.count, self.rank, dev(self.adapter), self.M, self.N, self.K,
               *self.segs, d_base if base else None, self.ldb if base else 0, mult, y, ldy, work)
        got = host(y)
        assert (host(work)[n:] == 255).all() and (host(work)[:2048] == 0).all()
        if in_place:
            keep = self.base if self.f32 else self.base.view(np.int16)
            np.testing.assert_array_equal(got[:, self.N:], keep[:, self.N:])
        else:
            assert (got[self.M] == 77).all() and (got[:, self.N:] == 77).all()
        got = got[:self.M, :self.N]
        return got if self.f32 else got.view(np.uint16)

    def check(self, got, mult=1.0, base=True):
        b = (self.base if self.f32 else ref.f32(self.base))[:, :self.N].astype(np.float64)
        # the product mult * alpha is one f32 rounding, in the bound's last term
        want, tol = ref.lora(self.xv, ref.f32(self.A).astype(np.float64),
                             ref.f32(self.B).astype(np.float64), self.alpha.astype(np.float64),
                             self.adapter, b if base else 0 * b, self.segs, np.float64(np.float32(mult)))
        g = got if self.f32 else ref.f32(got)
        if not self.f32:
            tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want)
        d = np.abs(g.astype(np.float64) - want)
        assert (d <= tol).all(), (d / tol).max()
        none = (self.adapter < 0) | (self.adapter >= self.count)
        np.testing.assert_array_equal(got[none], self.base[none][:, :self.N] if base else 0 * got[none])
        print(f"  at most {(d / tol).max():.3f} of the bound", flush=True)


SHAPES = [
    # M, N, K, rank, adapters, segs
    (1, 64, 64, 8, 1, None),
    (1, 384, 256, 16, 3, (256, 320)),
    (5, 200, 448, 24, 2, (64, 128)),
    (16, 512, 512, 32, 20, (256, 512)),
    (17, 328, 192, 48, 4, None),
    (33, 136, 1024, 128, 5, (64, 128)),
    (64, 72, 128, 64, 7, (64, 72)),
    (65, 264, 640, 16, 2, (128, 256)),
    (130, 1000, 320, 40, 3, None),
    (300, 264, 1088, 72, 2, (64, 192)),
    (517, 8, 64, 16, 1, None),
]


@pytest.mark.parametrize("M,N,K,rank,count,segs", SHAPES)
@pytest.mark.parametrize("fp8,f32", [(False, False), (False, True), (True, False), (True, True)])
def test_lora(M, N, K, rank, count, segs, fp8, f32):
    c = Case(M, N, K, rank, count, segs, fp8, f32)
    c.check(c.run(0.22), 0.22)


@pytest.mark.parametrize("M,K,rank", [(4113, 1600, 40), (4100, 64, 64), (4230, 320, 16), (300, 1088, 72), (150, 640, 24)])
@pytest.mark.parametrize("fp8", [False, True])
def test_lora_of_sessions_in_runs(M, K, rank, fp8):
    """Rows of a few sessions one after another, as a chunk has them: borders inside
    and at the ends of 16- and 64-row tiles, runs of one row, rows without an adapter."""
    c = Case(M, 72, K, rank, 5, fp8=fp8)
    c.adapter[:] = -1
    at = [0, 16, 33, 34, 80, 128, 135, 144, M - 70, M - 64, M - 17, M - 1, M]
    for i, (lo, hi) in enumerate(zip(at, at[1:])):
        c.adapter[lo:hi] = (3 * i) % 7 - 1  # -1 .. 5: none, 0 .. 4, out of range
    c.check(c.run(0.5), 0.5)


@pytest.mark.parametrize("M", [3, 40, 270])
@pytest.mark.parametrize("f32", [False, True])
def test_lora_without_base_and_in_place(M, f32):
    c = Case(M, 192, 128, 16, 3, (64, 128), f32=f32)
    c.check(c.run(1.5, base=False), 1.5, base=False)
    want = c.run(1.5)
    np.testing.assert_array_equal(c.run(1.5, in_place=True), want)
    c.check(want, 1.5)


@pytest.mark.parametrize("M", [16, 64, 200])
def test_lora_row_order_and_batch_do_not_matter(M):
    """Every order of the adapters in a tile, no adapter at all, numbers out of range;
    a row's result among others equals the row's alone in this kernel form."""
    c = Case(M, 136, 256, 16, 16)
    for kind in ("runs", "all", "none", "out", "cycle"):
        c.adapter = {"runs": np.sort(c.adapter), "all": np.full(M, 3), "none": np.full(M, -1),
                     "out": np.where(np.arange(M) % 3 == 0, 16, np.where(np.arange(M) % 3 == 1, -2**31, 15)),
                     "cycle": np.arange(M) % 16}[kind].astype(np.int32)
        got = c.run()
        c.check(got)
    order = c.rng.permutation(M)
    c.x, c.xv, c.base, c.adapter = c.x[order], c.xv[order], c.base[order], c.adapter[order]
    np.testing.assert_array_equal(c.run(), got[order])


def test_lora_not_finite_stays_in_its_row():
    c = Case(20, 128, 128, 16, 3)
    c.adapter[:] = np.arange(20) % 3
    want = c.run()
    c.x[4, 7] = 0x7FC0
    c.x[9, 3] = 0x7F80
    c.A[2, 0, 5, 9] = 0x7FFF        # adapter 2 is broken: rows 2, 5, 8, ...
    got = c.run()
    bad = (np.arange(20) % 3 == 2) | (np.arange(20) == 4) | (np.arange(20) == 9)
    np.testing.assert_array_equal(got[~bad], want[~bad])
    assert not np.isfinite(ref.f32(got[bad])).any()


def test_lora_far_adapter():
    """An adapter whose A and B begin past 2^31 bytes."""
    K, N, rank, count = 4096, 25600, 128, 340
    A = torch.zeros((count, 1, rank, K), dtype=torch.bfloat16, device="cuda")
    B = torch.zeros((count, N, rank), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    A[-1].copy_(torch.randn((1, rank, K), generator=g, device="cuda") / 64)
    B[-1].copy_(torch.randn((N, rank), generator=g, device="cuda"))
    x = torch.randn((2, K), generator=g, device="cuda").to(torch.bfloat16)
    alpha = torch.ones(count, device="cuda")
    y = L.lora_add(x, A, B, alpha, torch.tensor([count - 1, 0], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    want = x[0].double().cpu() @ A[-1, 0].double().cpu().T @ B[-1].double().cpu().T
    # a bf16 result, an f32 sum of 4096 products and one of 256 under it
    scale = (x[0].abs().double().cpu() @ A[-1, 0].abs().double().cpu().T) @ B[-1].abs().double().cpu().T
    assert ((y[0].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * scale).all()
    assert (y[1] == 0).all()


def test_lora_in_a_graph_with_changing_rows():
    c = Case(16, 256, 256, 16, 6, (64, 128))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        L.use_stream(s)
        x, A, B, alpha, base = (dev(t) for t in (c.x, c.A, c.B, c.alpha, c.base))
        adapter = dev(c.adapter)
        work = torch.zeros(L.call_size("granite4_lora_work_bytes", 16, 256, 256, 16, 64, 128),
                           dtype=torch.uint8, device="cuda")
        y = torch.empty((16, 256), dtype=torch.int16, device="cuda")

        def step():
            L.call("granite4_lora_add", 0, x, 16, c.ldx, None, A, B, alpha, 6, 16, adapter, 16, 256,
                   256, 64, 128, base, c.ldb, 1.0, y, 256, work)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        for i in range(6):
            adapter.copy_(dev(np.roll(c.adapter, i)))
            x.copy_(dev(np.roll(c.x, i, 0)))
            step()
            want = y.clone()
            y.fill_(1)
            torch.cuda.synchronize()
            graph.replay()
            assert torch.equal(y, want), i
    L.use_stream()


@pytest.mark.parametrize("fp8", [False, True])
def test_lora_beside_its_projection(fp8):
    """q|k|v of 20 rows: the shared GEMM, then the adapters in place, against the
    float64 sum of both (the projection's bf16 rounding is one more step of 2^-8)."""
    M, K, N, segs = 20, 256, 640, (512, 576)
    c = Case(M, N, K, 16, 3, segs, fp8=fp8, pad=0)
    rng = c.rng
    W = torch.from_numpy(rng.standard_normal((N, K)).astype(np.float32) * 8).to(torch.float8_e4m3fn)
    wv, Wd = W.float().numpy().astype(np.float64), W.view(torch.uint8).cuda()
    sc = (0.01, 0.02, 0.005)
    if fp8:
        y = L.gemm_fp8(dev(c.x), float(c.xs), Wd, scales=sc, segs=segs)
    else:
        y = L.prefill_gemm(dev(c.x).view(torch.bfloat16), Wd, scales=sc, segs=segs)
    L.lora_add(dev(c.x) if fp8 else dev(c.x).view(torch.bfloat16), dev(c.A).view(torch.bfloat16),
               dev(c.B).view(torch.bfloat16), dev(c.alpha), dev(c.adapter), base=y, segs=segs,
               x_scale=dev(np.array([c.xs])) if fp8 else None, out=y)
    s = np.repeat(np.array(sc, np.float32).astype(np.float64), [512, 64, 64])
    p = (c.xv @ wv.T) * s
    want, tol = ref.lora(c.xv, ref.f32(c.A).astype(np.float64), ref.f32(c.B).astype(np.float64),
                         c.alpha.astype(np.float64), c.adapter, p, segs, 1.0)
    tol = tol + K * 2.0 ** -23 * (np.abs(c.xv) @ np.abs(wv.T)) * s + 2.0 ** -8 * (np.abs(p) + np.abs(want)) * (1 + 2.0 ** -7)
    d = np.abs(y.float().cpu().numpy().astype(np.float64) - want)
    assert (d <= tol).all(), (d / tol).max()
