"""Block-sparse attention on the GPU (granite4_kv_ranges, granite4_block_select,
granite4_attn_blocks) against the 64-bit forms in block_ref.py: ranges and lists
are equal, attention within the bound that block_ref.attend derives."""
import numpy as np
import pytest
import torch

import block_ref as ref
from pkg import layerops

pytestmark = pytest.mark.gpu

D = 128
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


class Pool:
    """A filled arena on the host and the device, with its ranges."""

    def __init__(self, bits, group, Hk, stride, block, seed):
        self.rng = np.random.default_rng(seed)
        self.bits, self.group, self.Hk, self.stride, self.block = bits, group, Hk, stride, block
        k, v, ks, vs, self.kval, self.vval = ref.pool(self.rng, bits, group, Hk, stride)
        self.k, self.v = dev(k), dev(v)
        self.ks, self.vs = (None, None) if ks is None else (dev(ks), dev(vs))
        n = stride // block
        self.rc = self.rng.integers(-127, 128, (Hk, n, 2, D)).astype(np.int8)
        self.rs = (self.rng.random((Hk, n)) + 0.5).astype(np.float32)
        self.drc, self.drs = dev(self.rc), dev(self.rs)

    def ranges(self, base, rows, pt=None, d_pos=None, row_pos=None, row_pt=None):
        L.call("granite4_kv_ranges", self.k, self.ks, self.bits, self.group, self.Hk, D,
               self.stride, self.block, base, rows, d_pos, pt, row_pos, row_pt, self.drc, self.drs)

    def select(self, q, base=0, pt=None, d_pos=None, row_pos=None, row_pt=None, top_k=4, sink=1,
               recent=1, max_len=0):
        rows = q.shape[0]
        work = torch.full((L.call_size("granite4_block_select_work_bytes", rows, self.Hk,
                                       max_len or self.stride, self.block),), 255,
                          dtype=torch.uint8, device="cuda")
        work = work if work.numel() else None
        sel = torch.full((rows + 1, self.Hk, top_k), -77, dtype=torch.int32, device="cuda")
        L.call("granite4_block_select", dev(q), rows, 4 * self.Hk, self.Hk, D, self.drc, self.drs,
               self.stride, self.block, base, d_pos, pt, row_pos, row_pt, max_len, top_k, sink,
               recent, work, sel)
        got = host(sel)
        assert (got[rows] == -77).all()  # nothing behind the last row
        return got[:rows]

    def attend(self, q, sel, scale, base=0, pt=None, d_pos=None, row_pos=None, row_pt=None):
        rows, top_k = q.shape[0], sel.shape[-1]
        n = L.call_size("granite4_attn_blocks_scratch_bytes", 4 * self.Hk, rows, top_k, self.block)
        # zeros where calls count, NaN where they put their sums
        head = 2048
        scratch = torch.full((n + 16,), 255, dtype=torch.uint8, device="cuda")
        scratch[:head if n else 0] = 0
        out = torch.full((rows + 1, 4 * self.Hk * D), 0x7FC1, dtype=torch.int16, device="cuda")
        L.call("granite4_attn_blocks", dev(q), rows, 4 * self.Hk, self.Hk, D, scale, self.k, self.v,
               self.ks, self.vs, self.bits, self.group, self.stride, base, d_pos, pt, row_pos,
               row_pt, dev(sel), top_k, self.block, scratch, out)
        got = host(out).view(np.uint16)
        assert (got[rows] == 0x7FC1).all() and (host(scratch)[n:] == 255).all()
        assert n == 0 or (host(scratch)[:head] == 0).all()
        return got[:rows].reshape(rows, 4 * self.Hk, D)

    def check(self, got, q, sel, pos, pts, scale):
        worst = 0.0
        for r in range(q.shape[0]):
            x = ref.f32(q[r]).reshape(4 * self.Hk, D)
            want, tol = ref.attend(x, self.kval, self.vval, self.block, pos[r], pts[r],
                                         self.stride, sel[r], scale)
            d = np.abs(ref.f32(got[r]).astype(np.float64) - want)
            part = d / np.maximum(tol, 1e-30)
            worst = max(worst, part.max())
            assert (d <= tol).all(), f"row {r}: {part.max():.2f} of the bound"
        print(f"  at most {worst:.3f} of the bound", flush=True)


def queries(rng, rows, Hk, std=4.0):
    return ref.bf16((std * rng.standard_normal((rows, 4 * Hk * D))).astype(np.float32))


def ptrs(tables):
    return torch.tensor([0 if t is None else t.data_ptr() for t in tables], dtype=torch.int64,
                        device="cuda")


FORMATS = [(16, 128), (8, 128), (8, 32), (4, 128), (4, 64), (5, 128), (5, 32)]


# ------------------------------------------------------------------- ranges
@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_ranges_chunk(bits, group, block):
    P = Pool(bits, group, 3, 8 * 128, block, 100 * bits + group + block)
    pt = ref.table(P.rng, 1024 // block, block)
    start, rows = block + 5, 4 * block + 3
    done = range(start // block, (start + rows) // block)
    assert len(done) == 4
    wc, ws = ref.ranges(P.kval, block, pt, P.stride, done, P.rc, P.rs)
    P.ranges(start, rows, dev(pt))
    np.testing.assert_array_equal(host(P.drs), ws)
    np.testing.assert_array_equal(host(P.drc), wc)
    P.ranges(0, block - 1, dev(pt))  # completes nothing
    np.testing.assert_array_equal(host(P.drc), wc)


@pytest.mark.parametrize("bits,group,block", [(16, 128, 64), (8, 64, 16), (5, 32, 128)])
def test_ranges_positions_on_the_device(bits, group, block):
    P = Pool(bits, group, 2, 1024, block, 7 + bits)
    pt = ref.table(P.rng, 1024 // block, block)
    pos = dev(np.array([2 * block - 9], np.int32))
    wc, ws = ref.ranges(P.kval, block, pt, P.stride, [1, 2], P.rc, P.rs)
    P.ranges(0, 2 * block - 7 + 9, dev(pt), d_pos=pos)  # up to 4 block - 7 (ends inside block 3)
    np.testing.assert_array_equal(host(P.drc), wc)
    np.testing.assert_array_equal(host(P.drs), ws)
    # rows of sequences of their own: only a row on its block's last position counts; no
    # table: row = position; positions off the arena change nothing
    where = np.array([4 * block - 1, 5 * block, 6 * block - 2, block - 1, -1, 1 << 30, 2**31 - 1], np.int32)
    t = dev(pt)
    wc, ws = ref.ranges(P.kval, block, pt, P.stride, [3], wc, ws)
    wc, ws = ref.ranges(P.kval, block, np.arange(1024), P.stride, [0], wc, ws)
    P.ranges(0, 7, row_pos=dev(where), row_pt=ptrs([t, t, t, None, t, None, None]))
    np.testing.assert_array_equal(host(P.drc), wc)
    np.testing.assert_array_equal(host(P.drs), ws)


def test_ranges_holes_zeros_nan():
    P = Pool(16, 128, 2, 512, 32, 3)
    pt = ref.table(P.rng, 16, 32)
    pt[32] = -1        # block 1 begins nowhere
    pt[64 + 7] = -1    # block 2 misses a key
    pt[64 + 8] = 512   # and one off the arena
    pt[96:128] += 1    # block 3 begins inside an arena block
    pt[96:128] %= 512
    k = P.kval.copy()
    k[:, pt[128:160]] = 0.0            # block 4: zeros
    k[0, pt[160 + 3], 5] = np.nan      # block 5: one NaN, passed over
    P.k = dev(ref.bf16(np.nan_to_num(k).astype(np.float32)))
    P.k[0, pt[160 + 3], 5] = 0x7FC0
    P.k = P.k.view(torch.uint8)
    wc, ws = ref.ranges(k, 32, pt, 512, range(8), P.rc, P.rs)
    P.ranges(0, 256, dev(pt))
    np.testing.assert_array_equal(host(P.drs), ws)
    np.testing.assert_array_equal(host(P.drc), wc)


# ---------------------------------------------------------------- selection
def lists(P, q, pos, pts, top_k, sink, recent):
    rc, rs = host(P.drc), host(P.drs)
    return np.stack([ref.select(ref.f32(q[r]).reshape(-1, D), rc, rs, P.block, pos[r], pts[r],
                                P.stride, top_k, sink, recent) for r in range(q.shape[0])])


@pytest.mark.parametrize("rows,block,top_k,sink,recent",
                         [(1, 64, 4, 1, 1), (1, 16, 33, 0, 1), (5, 16, 7, 2, 3), (18, 32, 1, 0, 1),
                          (70, 16, 200, 1, 2), (3, 128, 3, 0, 3)])
def test_select_chunk(rows, block, top_k, sink, recent):
    P = Pool(16, 128, 2, 4096, block, rows + block)
    pt = ref.table(P.rng, 4096 // block, block)
    q = queries(P.rng, rows, 2)
    start = 4096 - rows - 77
    got = P.select(q, start, dev(pt), top_k=top_k, sink=sink, recent=recent)
    want = lists(P, q, start + np.arange(rows), [pt] * rows, top_k, sink, recent)
    np.testing.assert_array_equal(got, want)
    # the same rows alone, and with the position on the device
    for r in (0, rows - 1):
        one = P.select(q[r:r + 1], 0, dev(pt), d_pos=dev(np.array([start + r], np.int32)),
                       top_k=top_k, sink=sink, recent=recent)
        np.testing.assert_array_equal(one, want[r:r + 1])
    # from the first position on: lists that grow
    got = P.select(q, 0, dev(pt), top_k=top_k, sink=sink, recent=recent)
    np.testing.assert_array_equal(got, lists(P, q, np.arange(rows), [pt] * rows, top_k, sink, recent))


@pytest.mark.parametrize("rows,stride", [(9, 1 << 15), (3, 1 << 17), (2, 20480)])
def test_select_rows_of_a_long_sequence(rows, stride):
    P = Pool(16, 128, 1, 16, 16, 8)
    P.stride = stride
    n = stride // 16
    P.rc = P.rng.integers(-127, 128, (1, n, 2, D)).astype(np.int8)
    P.rs = (P.rng.random((1, n)) + 0.5).astype(np.float32)
    P.drc, P.drs = dev(P.rc), dev(P.rs)
    pt = ref.table(P.rng, n, 16)
    q = queries(P.rng, rows, 1)
    for start in (stride - rows, stride // 2 - 3):
        got = P.select(q, start, dev(pt), top_k=70, sink=1, recent=2)
        np.testing.assert_array_equal(got, lists(P, q, start + np.arange(rows), [pt] * rows, 70, 1, 2))


def test_select_sessions_and_edges():
    P = Pool(16, 128, 3, 2048, 32, 11)
    a, b = ref.table(P.rng, 64, 32), ref.table(P.rng, 64, 32)
    b[5 * 32] = -1       # blocks off the arena are never listed
    b[7 * 32] = 2048
    b[9 * 32] += 16      # nor those that begin inside an arena block
    da, db = dev(a), dev(b)
    pos = np.array([0, 31, 32, 2047, 1500, -1, 700, 5 * 32 + 3, 1 << 30], np.int32)
    tabs = [a, b, a, a, b, a, np.arange(2048), b, a]
    q = queries(P.rng, len(pos), 3)
    got = P.select(q, row_pos=dev(pos), row_pt=ptrs([da, db, da, da, db, da, None, db, da]), top_k=9,
                   sink=2, recent=2)
    want = lists(P, q, np.minimum(pos, 2047), tabs, 9, 2, 2)
    np.testing.assert_array_equal(got, want)
    assert (got[5] == -1).all() and (got[7, :, 5:] == -1).all()
    # a shorter table: positions are taken up to max_len
    got = P.select(q, row_pos=dev(pos), row_pt=ptrs([da, db, da, da, db, da, None, db, da]), top_k=9,
                   sink=2, recent=2, max_len=1000)
    np.testing.assert_array_equal(got, lists(P, q, np.minimum(pos, 999), tabs, 9, 2, 2))


def test_select_ties_zero_and_not_finite():
    P = Pool(16, 128, 2, 2048, 16, 5)
    P.rc[:, 1::2] = P.rc[:, 0::2]   # pairs of equal blocks
    P.rs[:, 1::2] = P.rs[:, 0::2]
    P.rs[:, 40:50] = 0.0            # whole runs of score 0, from either sign
    P.rs[0, 60] = np.inf
    P.rs[1, 61] = np.nan
    P.drc, P.drs = dev(P.rc), dev(P.rs)
    q = queries(P.rng, 4, 2)
    q[1] = 0                        # every score 0: the lowest numbers
    q[2] = ref.bf16(np.full(8 * D, -2.0, np.float32))
    q[3, :D] = 0
    got = P.select(q, 2000, top_k=21, sink=0, recent=1)
    want = lists(P, q, 2000 + np.arange(4), [np.arange(2048)] * 4, 21, 0, 1)
    np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(got[1, 0, :20], np.arange(20))
    q[0, 3] = 0x7FC0                # a NaN in a query: a list all the same, in range and ascending
    got = P.select(q, 2000, top_k=21, sink=0, recent=1)
    assert (np.diff(got[0], axis=-1) > 0).all() and got[0].min() >= 0 and got[0].max() <= 125
    np.testing.assert_array_equal(got[1:], want[1:])


@pytest.mark.parametrize("stride,rows", [(1 << 18, 1100), (1 << 20, 300)])
def test_select_long_arena(stride, rows):
    """16384 keys a row, which one workgroup holds, and 65536: scores in memory,
    those of some of the rows at a time."""
    P = Pool(16, 128, 1, 16, 16, 6)
    P.stride = stride
    n = P.stride // 16
    P.rc = P.rng.integers(-127, 128, (1, n, 2, D)).astype(np.int8)
    P.rs = (P.rng.random((1, n)) + 0.5).astype(np.float32)
    P.drc, P.drs = dev(P.rc), dev(P.rs)
    size = L.call_size("granite4_block_select_work_bytes", rows, 1, P.stride, 16)
    assert size == 0 if n == 16384 else 0 < size < rows * n * 4
    q = queries(P.rng, rows, 1)
    got = P.select(q, 700, top_k=12, sink=1, recent=2)
    at = [0, 127, 255, 256, 259, rows - 1]
    want = lists(P, q[at], 700 + np.array(at), [np.arange(P.stride)] * len(at), 12, 1, 2)
    np.testing.assert_array_equal(got[at], want)
    # the longest context: every key of the arena
    got = P.select(q[:1], P.stride - 1, top_k=12, sink=1, recent=2)
    np.testing.assert_array_equal(got, lists(P, q[:1], [P.stride - 1], [np.arange(P.stride)], 12, 1, 2))


# ---------------------------------------------------------------- attention
def random_lists(rng, pos, Hk, top_k, block):
    sel = np.full((len(pos), Hk, top_k), -1, np.int32)
    for r, p in enumerate(pos):
        n = p // block + 1
        for h in range(Hk):
            k = min(n, top_k)
            pick = np.sort(rng.permutation(n)[:k])
            pick[-1] = n - 1
            sel[r, h, :k] = pick
    return sel


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("rows,block,top_k", [(1, 64, 5), (3, 16, 9), (19, 32, 3), (1, 128, 1)])
def test_attend_chunk(bits, group, rows, block, top_k):
    P = Pool(bits, group, 2, 2048, block, bits + group + rows)
    pt = ref.table(P.rng, 2048 // block, block)
    start = 2048 - rows - 45
    pos = start + np.arange(rows)
    q = queries(P.rng, rows, 2)
    sel = random_lists(P.rng, pos, 2, top_k, block)
    got = P.attend(q, sel, 1 / 16, start, dev(pt))
    P.check(got, q, sel, pos, [pt] * rows, 1 / 16)


@pytest.mark.parametrize("bits,group", [(16, 128), (8, 128), (5, 32)])
def test_attend_short_and_empty(bits, group):
    """From the first position on, lists without an entry, with entries behind the
    row, negative, repeated, and blocks whose keys have no arena row."""
    P = Pool(bits, group, 2, 1024, 32, 40 + bits)
    pt = ref.table(P.rng, 32, 32)
    pt[3 * 32:4 * 32] = -1
    pt[4 * 32 + 1] = 1024
    pos = np.array([0, 1, 33, 300, 300, 300, 300, 1000, -1, 500], np.int32)
    q = queries(P.rng, len(pos), 2)
    sel = np.full((len(pos), 2, 6), -1, np.int32)
    sel[0] = [0, -1, -1, -1, -1, -1]
    sel[1] = [0, 1, 2, 3, 4, 31]          # mostly behind the row
    sel[2] = [1, 0, -5, 1 << 30, 2**31 - 1, -2**31]
    sel[3, 0] = [3, 3, 3, -1, -1, -1]     # no key has a row; the other head lists nothing
    sel[4] = [3, 4, -1, 9, 9, 2]          # one counted twice, one partly mapped, any order
    sel[5, 1] = [-1, -1, -1, -1, -1, 5]
    sel[6] = [31, 30, 29, 28, 27, 26]     # all behind the row
    sel[7] = [31, 0, 15, 16, 30, 7]       # the row ends inside block 31
    sel[8] = [0, 1, 2, 3, 4, 5]           # a row at -1 sees nothing
    sel[9] = [15, 14, 13, 12, 11, 10]
    d = dev(pt)
    got = P.attend(q, sel, 0.125, row_pos=dev(pos), row_pt=ptrs([d] * 9 + [None]))
    P.check(got, q, sel, pos, [pt] * 9 + [np.arange(1024)], 0.125)
    for r, h in ((3, 0), (3, 1), (5, 0), (6, 0), (6, 1), (8, 0), (8, 1)):
        assert (got[r, 4 * h:4 * h + 4] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_attend_masked_garbage(bits):
    """Keys and values of a listed block behind the row's position are not looked
    at: NaN and infinities there change nothing."""
    P = Pool(bits, 128, 1, 256, 64, 50 + bits)
    q = queries(P.rng, 1, 1)
    sel = np.array([[[0, 2]]], np.int32)
    want = P.attend(q, sel, 0.25, 140)
    for t in (P.k, P.v) if bits == 16 else (P.ks, P.vs):
        x = t.view(torch.int16).view(1, 256, -1)
        x[:, 141:] = 0x7FC0 if bits == 16 else -1   # NaN (f32 0xffffffff)
        x[:, 200:210] = 0x7F80 if bits == 16 else 0x7F80
        x[:, 64:128] = 0x7FC0 if bits == 16 else -1  # block 1 is not listed
    np.testing.assert_array_equal(P.attend(q, sel, 0.25, 140), want)
    P.check(want, q, sel, [140], [np.arange(256)], 0.25)


@pytest.mark.parametrize("bits,group", [(16, 128), (8, 128), (5, 32)])
def test_attend_not_finite(bits, group):
    """A NaN in an attended value or query reaches exactly the outputs it should."""
    P = Pool(bits, group, 2, 256, 64, 60 + bits)
    q = queries(P.rng, 2, 2)
    q[1, 3 * D + 7] = 0x7FC0   # row 1, head 3
    sel = np.array([[[0, 1], [0, 1]]] * 2, np.int32)
    got = ref.f32(P.attend(q, sel, 0.25, 100))
    bad = np.isnan(got)
    assert bad[1, 3].all() and bad.sum() == D
    if bits == 16:
        P.v.view(torch.int16).view(2, 256, D)[1, 90, 5] = 0x7FC0
        bad = np.isnan(ref.f32(P.attend(q, sel, 0.25, 100)))
        assert bad[:, 4:, 5].all() and bad[1, 3].all() and bad.sum() == D + 8


@pytest.mark.parametrize("bits", [16, 4])
def test_attend_rows_of_two_launches(bits):
    """More rows than one launch has: each at its own position still."""
    rows, base, group = 65537 + 70, 40, 128
    P = Pool(bits, group, 1, 65536 + 256, 64, 80 + bits)
    pos = base + np.arange(rows)
    sel = np.stack([pos // 64, pos // 128 - 1], -1).astype(np.int32)[:, None]
    q = queries(P.rng, rows, 1)
    got = P.attend(q, sel, 0.125, base)
    at = np.array([0, 1, 100, 65534, 65535, 65536, 65537, rows - 2, rows - 1])
    P.check(got[at], q[at], sel[at], pos[at], [np.arange(P.stride)] * len(at), 0.125)


@pytest.mark.parametrize("rows,Hk,block,top_k", [(512, 2, 64, 5), (300, 8, 64, 9), (601, 8, 128, 3), (790, 8, 64, 70)])
@pytest.mark.parametrize("side", ["together", "apart"])
def test_attend_rows_together(rows, Hk, block, top_k, side):
    """bf16 rows of one sequence that share a wave (one to four of them): lists in any
    order, with entries behind the row, negative, repeated and shared with the next
    row; arena rows side by side or apart, some keys without one; the position on the
    device."""
    P = Pool(16, 128, Hk, 8192, block, rows + top_k)
    pt = ref.table(P.rng, 8192 // block, block) if side == "together" else P.rng.permutation(8192).astype(np.int32)
    pt[5 * block + 3] = -1
    pt[7 * block:8 * block] = 8192
    start = 4000
    pos = start + np.arange(rows)
    q = queries(P.rng, rows, Hk)
    sel = random_lists(P.rng, pos, Hk, top_k, block)
    at = np.r_[0:8, 130:142, rows - 9:rows]
    sel[at[0]] = -1
    sel[at[1], 0] = 8192 // block - 1             # behind the row, every entry
    sel[at[2]] = sel[at[2]][:, ::-1]              # descending, the -1 first
    sel[at[3], 1, 1:3] = sel[at[3], 1, 0]         # counted three times
    sel[at[4]:at[6], 0] = sel[at[4], 0]           # two rows alike
    sel[at[6], 0, :2] = [2**31 - 1, -2**31]
    sel[at[9]:at[9] + 4] = sel[at[9]]             # four rows alike
    sel[at[15], 0, 0] = 7                         # no key with a row
    sel[at[-1], 0] = np.where(np.arange(top_k) == top_k - 1, 5, -1)
    d_pos = dev(np.array([start], np.int32)) if side == "apart" else None
    got = P.attend(q, sel, 1 / 16, 0 if side == "apart" else start, dev(pt), d_pos)
    P.check(got[at], q[at], sel[at], pos[at], [pt] * len(at), 1 / 16)
    assert (got[at[0]] == 0).all() and (got[at[1], :4] == 0).all()


@pytest.mark.parametrize("bits,group", [(16, 128), (8, 128), (4, 32), (5, 64)])
@pytest.mark.parametrize("rows,block", [(254, 32), (511, 16)])
def test_attend_many_sequences(bits, group, rows, block):
    """A wave for each row: rows of sequences with tables of their own, their lists
    in any order."""
    P = Pool(bits, group, 8, 4096, block, rows + bits)
    pts = [ref.table(P.rng, 4096 // block, block) for _ in range(3)] + [np.arange(4096, dtype=np.int32)]
    pts[1][2 * block + 1] = -1
    pos = P.rng.integers(0, 4096, rows).astype(np.int32)
    pos[:4] = -1, 0, 4095, 5
    q = queries(P.rng, rows, 8)
    sel = random_lists(P.rng, np.maximum(pos, 0), 8, 7, block)
    sel[4] = sel[4][:, ::-1]
    sel[5, 2] = -1
    sel[6, 1, 3] = 4096 // block - 1
    d = [dev(t) for t in pts[:3]] + [None]
    got = P.attend(q, sel, 1 / 16, row_pos=dev(pos), row_pt=ptrs([d[r % 4] for r in range(rows)]))
    at = np.r_[0:12, rows - 6:rows]
    P.check(got[at], q[at], sel[at], pos[at], [pts[r % 4] for r in at], 1 / 16)
    assert (got[0] == 0).all() and (got[5, 8:12] == 0).all()


def test_attend_rows_together_garbage():
    """What a row does not list or see does not reach it from the rows beside it."""
    P = Pool(16, 128, 8, 2048, 64, 83)
    rows, start = 520, 1000
    pos = start + np.arange(rows)
    q = queries(P.rng, rows, 8)
    sel = random_lists(P.rng, pos, 8, 6, 64)
    want = P.attend(q, sel, 0.25, start)
    at = np.r_[0:6, 400:406, 514:520]
    P.check(want[at], q[at], sel[at], pos[at], [np.arange(2048)] * len(at), 0.25)
    for t in (P.k, P.v):  # NaN in block 3, infinity behind the last row
        x = t.view(torch.int16).view(8, 2048, D)
        x[:, 192:256] = 0x7FC0
        x[:, start + rows:] = 0x7F80
    listed = np.repeat((sel == 3).any(-1), 4, 1)
    assert listed.any() and not listed.all()
    got = P.attend(q, sel, 0.25, start)
    np.testing.assert_array_equal(got[~listed], want[~listed])
    # the last row sees its own key last
    q[9, 2 * D + 1] = 0x7FC0
    bad = np.isnan(ref.f32(P.attend(q, sel, 0.25, start)))
    clean = ~listed
    assert bad[9, 2].all() and bad[clean].sum() == (D if clean[9, 2] else 0)


def test_attend_large_logits():
    """Logits in the hundreds, of either sign: the running maximum holds."""
    P = Pool(16, 128, 2, 1024, 64, 71)
    pos = np.array([900, 1000], np.int32)
    q = queries(P.rng, 2, 2, std=40.0)
    sel = random_lists(P.rng, pos, 2, 9, 64)
    for scale in (1.0, -1.0):
        got = P.attend(q, sel, scale, row_pos=dev(pos), row_pt=ptrs([None, None]))
        assert np.isfinite(ref.f32(got)).all()
        P.check(got, q, sel, pos, [np.arange(1024)] * 2, scale)


@pytest.mark.parametrize("rows", [1, 6, 300])
def test_attend_every_split_is_the_same_answer(rows):
    """A row alone (its list over many workgroups), among a few and among many (one
    workgroup a row): each within the bound of the 64-bit result."""
    P = Pool(8, 128, 2, 4096, 64, 80)
    pos = 3000 + np.arange(rows)
    q = np.repeat(queries(P.rng, 1, 2), rows, 0)
    sel = np.repeat(random_lists(P.rng, [2999], 2, 40, 64), rows, 0)
    got = P.attend(q, sel, 1 / 16, 3000)
    some = [0, rows // 2, rows - 1]
    P.check(got[some], q[some], sel[some], pos[some], [np.arange(4096)] * 3, 1 / 16)


# ------------------------------------------------------------ whole sequence
@pytest.mark.parametrize("bits,group", [(16, 128), (8, 128), (5, 32)])
def test_lists_of_everything_give_dense_attention(bits, group):
    """With room for every block the three calls answer what the dense decode and
    prefill attention answer, which round their logits to bf16 as well: 2^-8 of
    a logit moves p by that much on either side."""
    P = Pool(bits, group, 8, 1024, 64, 90 + bits)
    pt = ref.table(P.rng, 16, 64)
    d, rows, start, scale = dev(pt), 5, 800, 1 / 128
    P.ranges(0, start + rows, d)
    q = queries(P.rng, rows, 8, std=8.0)
    sel = P.select(q, start, d, top_k=13, sink=1, recent=1)
    np.testing.assert_array_equal(sel[0, 0], np.arange(13))
    got = ref.f32(P.attend(q, sel, scale, start, d)).reshape(rows, -1)
    dense = torch.empty((rows, 32 * D), dtype=torch.int16, device="cuda")
    L.call("granite4_prefill_attn", dev(q), rows, 32, 8, D, scale, P.k, P.v, P.ks, P.vs, bits,
           group, P.stride, start, d, 0, dense)
    want = ref.f32(host(dense).view(np.uint16))
    lmax = np.abs(ref.f32(q)).reshape(rows, 32, D).sum(-1).max() * np.abs(P.kval).max() * scale
    vmax = np.abs(P.vval).max()
    assert np.abs(got - want).max() <= 2.0 ** -8 * vmax * (4 + 4 * lmax)
    assert np.sqrt(np.mean((got - want) ** 2)) <= 2.0 ** -7 * np.sqrt(np.mean(want ** 2)) * 2


def test_decode_steps_in_a_graph():
    """Append, ranges, selection and attention of one token, captured once with the
    position on the device and replayed along a sequence that crosses blocks, with
    eager work in between: every replay equals the eager calls."""
    Hk, block, stride, top_k = 2, 16, 256, 4
    rng = np.random.default_rng(1)
    pt = dev(ref.table(rng, stride // block, block))
    cos, sin = L.rope_tables(1e4, D, stride)
    steps = 40
    qs, ks, vs = (torch.from_numpy(rng.standard_normal((steps, n * D)).astype(np.float32)).cuda()
                  .to(torch.bfloat16) for n in (4 * Hk, Hk, Hk))

    def program(stream):
        arena = L.KvArena(8, Hk, stride)
        R = L.KvRanges(Hk, stride, block)
        pos = torch.full((1,), 100, dtype=torch.int32, device="cuda")
        q, k, v = (torch.empty_like(t[:1]) for t in (qs, ks, vs))
        q_rot = torch.empty_like(q)
        work = torch.empty(L.call_size("granite4_block_select_work_bytes", 1, Hk, stride, block),
                           dtype=torch.uint8, device="cuda")
        sel = torch.empty((1, Hk, top_k), dtype=torch.int32, device="cuda")
        scratch = torch.zeros(L.call_size("granite4_attn_blocks_scratch_bytes", 4 * Hk, 1, top_k, block),
                              dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)

        def step():
            L.call("granite4_rope_append_at_pos", q, k, v, cos, sin, stride, pos, pt, 4 * Hk, Hk, D,
                   8, 128, q_rot, arena.k, arena.v, arena.k_scale, arena.v_scale, stride)
            L.kv_ranges(arena, R, 1, d_pos=pos, d_pt=pt)
            L.block_select(q_rot, R, top_k, d_pos=pos, d_pt=pt, work=work, sel=sel)
            L.attn_blocks(q_rot, arena, sel, block, 1 / 16, d_pos=pos, d_pt=pt, scratch=scratch, out=out)

        def feed(i):
            pos.fill_(100 + i)
            q.copy_(qs[i:i + 1])
            k.copy_(ks[i:i + 1])
            v.copy_(vs[i:i + 1])
        return step, feed, (sel, out, R.codes, R.scale)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        L.use_stream(s)
        step, feed, eager = program(s)
        want = []
        for i in range(steps):
            feed(i)
            step()
            want.append([t.clone() for t in eager])
        step, feed, got = program(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        for i in range(steps):
            feed(i)
            graph.replay()
            if i % 5 == 0:
                torch.cuda.synchronize()
                torch.ones(1000, device="cuda").sum().item()
            for a, b in zip(got, want[i]):
                assert torch.equal(a, b), i
        torch.cuda.synchronize()
    L.use_stream()
