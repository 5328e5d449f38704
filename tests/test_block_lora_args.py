"""What granite4_kv_ranges, granite4_block_select, granite4_attn_blocks and
granite4_lora_add refuse: -1 before any launch, so no GPU is needed (device
pointers are only compared and never read)."""
import pytest

from pkg import layerops

L = layerops()
P16, P24 = 1 << 20, (1 << 20) + 8  # 16-byte aligned, and not

RANGES = dict(cache_k=P16, k_scale=P16, bits=8, group=128, Hk=8, d=128, stride=1024, block=64,
              base_pos=0, rows=64, d_pos=None, d_pt=None, row_pos=None, row_pt=None, ranges=P16,
              range_scale=P16)
SELECT = dict(q=P16, rows=4, Hq=32, Hk=8, d=128, ranges=P16, range_scale=P16, stride=1024, block=64,
              kv_base=0, d_pos=None, d_pt=None, row_pos=None, row_pt=None, max_len=0, top_k=8,
              sink=1, recent=2, work=P16, sel=P16)
BLOCKS = dict(q=P16, rows=4, Hq=32, Hk=8, d=128, scale=0.1, cache_k=P16, cache_v=P16, k_scale=P16,
              v_scale=P16, bits=8, group=128, stride=1024, kv_base=0, d_pos=None, d_pt=None,
              row_pos=None, row_pt=None, sel=P16, top_k=8, block=64, scratch=P16, out=P16)
LORA = dict(out=0, X=P16, x_bits=16, ldx=4096, d_x_scale=None, A=P16, B=P16, d_alpha=P16,
            adapters=4, rank=16, d_row_adapter=P16, M=5, N=6144, K=4096, seg1=4096, seg2=5120,
            base=P16, ldb=6144, mult=1.0, y=2 * P16, ldy=6144, work=P16)

BAD = [
    ("granite4_kv_ranges", RANGES, [
        dict(cache_k=None), dict(ranges=None), dict(range_scale=None), dict(k_scale=None),
        dict(bits=6), dict(group=16), dict(group=48), dict(d=64), dict(Hk=0), dict(block=48),
        dict(block=8), dict(block=256), dict(stride=1000), dict(stride=0), dict(rows=0),
        dict(rows=-1), dict(base_pos=-1), dict(base_pos=961), dict(base_pos=2**31 - 1),
        dict(row_pos=P16), dict(row_pt=P16), dict(cache_k=P24), dict(ranges=P24)]),
    ("granite4_block_select", SELECT, [
        dict(q=None), dict(ranges=None), dict(range_scale=None), dict(sel=None),
        dict(work=None, stride=1 << 20, block=16), dict(work=None, rows=65536, stride=1 << 17),
        dict(d=64), dict(Hk=0, Hq=0), dict(Hq=24), dict(block=24), dict(stride=1016),
        dict(max_len=-1), dict(max_len=1025), dict(max_len=3), dict(rows=0), dict(kv_base=1021),
        dict(kv_base=-1), dict(top_k=0), dict(sink=-1), dict(recent=0), dict(sink=7),
        dict(recent=9, sink=0), dict(recent=2**31 - 1), dict(sink=2**31 - 1), dict(row_pos=P16),
        dict(row_pt=P16), dict(q=P24), dict(ranges=P24), dict(work=P24)]),
    ("granite4_attn_blocks", BLOCKS, [
        dict(q=None), dict(cache_k=None), dict(cache_v=None), dict(sel=None), dict(out=None),
        dict(scratch=None), dict(k_scale=None), dict(v_scale=None), dict(bits=7), dict(group=96),
        dict(scale=float("nan")), dict(scale=float("inf")), dict(d=256), dict(Hq=8), dict(Hk=-1),
        dict(block=63), dict(stride=1025), dict(rows=0), dict(kv_base=1021), dict(top_k=0),
        dict(row_pos=P16), dict(row_pt=P16), dict(q=P24), dict(cache_k=P24), dict(cache_v=P24),
        dict(scratch=P24), dict(out=P16 + 2)]),
    ("granite4_lora_add", LORA, [
        dict(out=2), dict(out=-1), dict(X=None), dict(x_bits=4), dict(x_bits=8), dict(A=None),
        dict(B=None), dict(d_alpha=None), dict(adapters=0), dict(rank=0), dict(rank=12),
        dict(rank=136), dict(d_row_adapter=None), dict(M=0), dict(M=16 * 65535 + 1), dict(N=6140),
        dict(N=0), dict(K=4000), dict(K=0), dict(ldx=4088), dict(ldx=4100),
        dict(x_bits=8, d_x_scale=P16, ldx=4104), dict(seg1=0), dict(seg1=4000), dict(seg2=4096 - 64),
        dict(seg2=5000), dict(ldb=6136), dict(ldb=6148), dict(ldy=6136), dict(ldy=6145),
        dict(mult=float("nan")), dict(y=None), dict(work=None), dict(X=P24), dict(A=P24),
        dict(B=P24), dict(base=P24), dict(y=P24), dict(work=P24),
        dict(base=2 * P16, ldb=6152)]),
]


@pytest.mark.parametrize("name,good,change", [(n, g, c) for n, g, cs in BAD for c in cs],
                         ids=lambda v: v if isinstance(v, str) else "-".join(v) if len(v) < 4 else "")
def test_refused(name, good, change, capfd):
    assert set(change) <= set(good)
    assert len(good) == len(L._SIG[name])
    assert getattr(L.lib, name)(*{**good, **change}.values()) == -1
    assert f"{name}: invalid arguments" in capfd.readouterr().err
    with pytest.raises(L.Granite4Error):
        L.call(name, *{**good, **change}.values())


def test_a_call_that_completes_no_block_launches_nothing():
    assert L.lib.granite4_kv_ranges(*{**RANGES, "rows": 63}.values()) == 0
    assert L.lib.granite4_kv_ranges(*{**RANGES, "base_pos": 64, "rows": 1}.values()) == 0


def test_workspace_sizes():
    f = L.lib.granite4_block_select_work_bytes
    assert f(1, 8, 65536, 64) == f(65535, 8, 16384 * 16, 16) == 0  # kept on chip
    assert f(1, 8, 16384 * 16 + 1, 16) == 8 * (16384 + 64) * 4
    assert f(4, 8, 1 << 20, 16) == 4 * 8 * 65536 * 4
    assert f(100000, 8, 65536, 64) <= 64 << 20      # rows beyond are made in turns
    assert f(100000, 8, 65536, 64) > 60 << 20
    assert f(16, 64, 1 << 20, 16) == 16 * 64 * 65536 * 4  # but 16 rows at a time at least
    for bad in ((0, 8, 64, 16), (1, 0, 64, 16), (1, 8, 0, 16), (1, 8, 64, 0)):
        assert f(*bad) == 0
    f = L.lib.granite4_attn_blocks_scratch_bytes
    assert f(32, 4096, 32, 64) == 0
    assert f(32, 1, 32, 64) > 2048 and (f(32, 1, 32, 64) - 2048) % (32 * 130 * 4) == 0
    for bad in ((0, 1, 1, 16), (30, 1, 1, 16), (32, 0, 1, 16), (32, 1, 0, 16), (32, 1, 1, 0)):
        assert f(*bad) == 0
    f = L.lib.granite4_lora_work_bytes
    big = 2**31 - 1
    # counts, three bf16 terms of t (16-row tiles, 32 ranks), a sum of t for each share of K
    for k, shares in ((64, 1), (1024, 1), (2048, 2), (4096, 4), (12800, 8)):
        more = 4 * shares if shares > 1 else 0
        assert f(5, 6144, k, 16, 4096, 5120) == 2048 + 3 * (16 * 32 * 6 + 5 * 16 * more)
        assert f(5, 6144, k, 16, 4096, big) == 2048 + 2 * (16 * 32 * 6 + 5 * 16 * more)
    assert f(1 << 20, 6144, 4096, 128, big, big) == 2048 + (6 << 27)
    assert f(0, 64, 64, 16, big, big) == 0
