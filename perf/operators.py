"""What a server of many sessions over long contexts asks of this library beside
its dense attention and its shared projections, each in elementary torch
operations (`own` false) and through the library's entry points (`own` true):

  ranges   as the key cache is written, each completed block of positions gets
           the smallest and the largest value of every channel, in 8 bits
  select   for each query row and KV head, the blocks whose ranges promise the
           largest products with the row's queries
  blocks   attention of each row over the blocks listed for it
  lora     each row's own low-rank adapter, added to a shared projection

Sizes are those of the 8B configuration (hidden 4096, MLP 12800, 32 query and 8
KV heads of 128, positions up to 65536), over the ranges an engine meets.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

H, INTER, HQ, HK, D = 4096, 12800, 32, 8, 128
NQ, NK, G = HQ * D, HK * D, HQ // HK
MAX_POS = 65536
RESID, ATTN_SCALE = 0.22, 1.0 / 128
#: N, K, the columns where the second and third weight block of the projection begin
PROJ = {"qkv": (NQ + 2 * NK, H, NQ, NQ + NK), "o": (H, NQ, H, H),
        "gate_up": (2 * INTER, H, INTER, 2 * INTER), "down": (H, INTER, H, H)}
MODEST = 1 << 20  # rows x listed positions of the largest sparse attention


# --------------------------------------------------------------------- cases
def listed():
    return [
        # a short prompt's last chunk, its start inside a block, bf16 keys
        {"name": "ranges-500", "kind": "ranges", "rows": 500, "start": 77, "bits": 16,
         "group": 128, "block": 32},
        # a document's chunk in the smallest key format with group scales
        {"name": "ranges-8192", "kind": "ranges", "rows": 8192, "start": 4096, "bits": 5,
         "group": 32, "block": 64},
        # one user's token loop far into a document
        {"name": "select-token", "kind": "select", "sessions": 0, "rows": 1, "start": 30010,
         "block": 64, "top_k": 32, "sink": 1, "recent": 2},
        # a server's batched step, its sessions at positions of their own, small blocks
        {"name": "select-16", "kind": "select", "sessions": 16, "rows": 16, "start": 0,
         "block": 32, "top_k": 64, "sink": 1, "recent": 4},
        # a chunk at the end of a long document: every row its own blocks
        {"name": "select-1000", "kind": "select", "sessions": 0, "rows": 1000, "start": 57344,
         "block": 64, "top_k": 32, "sink": 1, "recent": 2},
        # the token loop's attention: 32 blocks of 64 out of some 470
        {"name": "blocks-token", "kind": "blocks", "sessions": 0, "rows": 1, "start": 30010,
         "bits": 8, "group": 128, "block": 64, "top_k": 32},
        # the batched step's, in the smallest cache format
        {"name": "blocks-16", "kind": "blocks", "sessions": 16, "rows": 16, "start": 0,
         "bits": 5, "group": 32, "block": 32, "top_k": 64},
        # the long document's chunk, bf16 cache
        {"name": "blocks-511", "kind": "blocks", "sessions": 0, "rows": 511, "start": 40000,
         "bits": 16, "group": 128, "block": 64, "top_k": 32},
        # one session's token through the adapter of its q|k|v projection
        {"name": "lora-token", "kind": "lora", "proj": "qkv", "rows": 1, "adapters": 8,
         "rank": 16, "fp8": False, "f32": False},
        # 16 sessions, nearly as many adapters, FP8 activations
        {"name": "lora-16", "kind": "lora", "proj": "gate_up", "rows": 16, "adapters": 24,
         "rank": 32, "fp8": True, "f32": False},
        # prompts of three sessions in one ragged chunk, the bf16 form's f32 gate|up
        {"name": "lora-1001", "kind": "lora", "proj": "gate_up", "rows": 1001, "adapters": 4,
         "rank": 16, "fp8": False, "f32": True},
        # the widest input at a full chunk
        {"name": "lora-8192", "kind": "lora", "proj": "down", "rows": 8192, "adapters": 4,
         "rank": 64, "fp8": False, "f32": False},
    ]


def _between(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _pool(rng):
    bits = rng.choice([16, 8, 8, 4, 5])
    return bits, 128 if bits == 16 else rng.choice([32, 64, 128, 128])


def draw(rng):
    kind = rng.choice(["ranges", "select", "blocks", "blocks", "lora", "lora"])
    block = rng.choice([16, 32, 64, 64, 128])
    if kind == "ranges":
        bits, group = _pool(rng)
        rows = _between(rng, 16, 8192)
        return {"kind": kind, "rows": rows, "start": rng.randint(0, rows // 2), "bits": bits,
                "group": group, "block": block}
    if kind in ("select", "blocks"):
        sessions = rng.choice([0, 0, rng.randint(2, 16)])
        rows = sessions or rng.choice([1, rng.randint(2, 16), _between(rng, 17, 1000)])
        start = 0 if sessions else _between(rng, 16, 57344)
        top_k = _between(rng, 4, 128)
        if kind == "select":
            if rows > 16:
                block = max(block, 64)
            return {"kind": kind, "sessions": sessions, "rows": rows, "start": start,
                    "block": block, "top_k": top_k, "sink": rng.randint(0, 2),
                    "recent": rng.randint(1, 2)}
        while rows * top_k * block > MODEST // 2:
            top_k = max(4, top_k // 2)
            block = max(16, block // 2)
        bits, group = _pool(rng)
        return {"kind": kind, "sessions": sessions, "rows": rows, "start": start, "bits": bits,
                "group": group, "block": block, "top_k": top_k}
    proj = rng.choice(["qkv", "o", "gate_up", "down"])
    rows = rng.choice([rng.randint(1, 16), _between(rng, 17, 1400 if proj == "gate_up" else 8000)])
    few = rows > 16
    return {"kind": kind, "proj": proj, "rows": rows,
            "adapters": rng.randint(1, 4) if few else rng.randint(1, 32),
            "rank": rng.choice([8, 16, 16, 32, 64] if few else [8, 16, 16, 32, 64, 128]),
            "fp8": proj != "o" and rng.random() < 0.4,
            "f32": proj == "gate_up" and rng.random() < 0.5}


# -------------------------------------------------------------------- inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * std

    def bf16(self, *shape, std=1.0):
        return self.normal(*shape, std=std).to(torch.bfloat16)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def hidden(self, rows, k):
        """Normalised rows: N(0, 1), 1 % of the channels 10 times larger."""
        x = self.normal(rows, k)
        x[:, torch.randperm(k, generator=self.g, device="cuda")[:k // 100]] *= 10
        return x


def _div(x, y):
    """The f32 quotient, correctly rounded (a 64-bit division rounded once more)."""
    return (x.double() / y.double()).float()


def _codes(x, s):
    """8-bit codes of x under the scale s: x / s rounded half away from zero; 0 where s is 0."""
    r = _div(x, torch.where(s == 0, 1.0, s))
    t = r.trunc()
    t = t + torch.where((r - t).abs() >= 0.5, r.sign(), 0.0)
    return torch.where(s == 0, 0.0, t.clamp(-127, 127))


def _pool_of(r, bits, group, stride):
    """One layer's filled pool: cache_k, cache_v (bytes) and their scales."""
    out = []
    for is_k in (True, False):
        x = r.normal(HK, stride, D)
        if is_k:  # keys have channels off zero
            x += r.normal(HK, 1, D)
        if bits == 16:
            out.append((x.to(torch.bfloat16).view(torch.uint8), None))
            continue
        qmax = 127 if bits == 8 else 15 if bits == 5 and is_k else 7
        xg = x.view(HK, stride, D // group, group)
        s = (xg.abs().amax(-1) / qmax).contiguous()
        c = torch.round(xg / s[..., None]).clamp_(-qmax, qmax).to(torch.int8).view(x.shape)
        del x, xg
        if bits == 8:
            out.append((c.view(torch.uint8), s))
            continue
        u = (c + (qmax + 1)).view(torch.uint8)
        rows = (u[..., 0::2] & 15) | ((u[..., 1::2] & 15) << 4)
        if qmax == 15:
            b = (u >> 4).view(HK, stride, 16, 8).to(torch.int32)
            b = b << torch.arange(8, device="cuda", dtype=torch.int32)
            rows = torch.cat([rows, b.sum(-1, dtype=torch.int32).to(torch.uint8)], -1)
        out.append((rows.contiguous(), s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _place(r, lengths, block):
    """Page tables of sequences of these lengths over one pool, the pages (of
    one or two blocks) in random order: tables [sequences][longest] (-1 past a
    sequence's end) and the pool's rows."""
    page = block * (1 + len(lengths) % 2)
    need = [(n + page - 1) // page for n in lengths]
    stride = sum(need) * page
    order = torch.randperm(sum(need), generator=r.g, device="cuda").to(torch.int32)
    rows = (order[:, None] * page + torch.arange(page, device="cuda", dtype=torch.int32)).reshape(-1)
    tables = torch.full((len(lengths), max(need) * page), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n * page] = rows[at:at + n * page]
        at += n * page
    return tables, stride


def prepare(case, seed):
    r = _Rand(seed)
    s = {"case": case}
    kind = case["kind"]
    if kind == "ranges":
        s["tables"], s["stride"] = _place(r, [case["start"] + case["rows"]], case["block"])
        s["k"], _, s["ks"], _ = _pool_of(r, case["bits"], case["group"], s["stride"])
        n = s["stride"] // case["block"]
        s["ranges"] = torch.zeros((HK, n, 2, D), dtype=torch.int8, device="cuda")
        s["rscale"] = torch.zeros((HK, n), dtype=torch.float32, device="cuda")
        return s
    if kind in ("select", "blocks"):
        rows, block = case["rows"], case["block"]
        if case["sessions"]:
            where = torch.rand(rows, generator=r.g, device="cuda")
            pos = torch.exp(where * math.log(65000 / 64) + math.log(64)).to(torch.int32)
            s["tables"], s["stride"] = _place(r, [p + 1 for p in pos.tolist()], block)
            width = 4 * s["tables"].shape[1]
            s["row_pos"] = pos
            s["row_pt"] = torch.arange(rows, device="cuda") * width + s["tables"].data_ptr()
        else:
            pos = case["start"] + torch.arange(rows, device="cuda", dtype=torch.int32)
            s["tables"], s["stride"] = _place(r, [case["start"] + rows], block)
        s["pos"] = pos
        s["q"] = r.bf16(rows, NQ, std=16)
        if kind == "select":
            # ranges as blocks of keys have them: channel means and spreads of their own
            n = s["stride"] // block
            mid = r.normal(HK, n, D, std=0.3) + r.normal(HK, 1, D)
            wide = (2.0 + r.normal(HK, n, D, std=0.4)).abs()
            lohi = torch.stack([mid - wide, mid + wide], 2)
            s["rscale"] = _div(lohi.abs().amax((2, 3)), torch.tensor(127.0, device="cuda"))
            s["ranges"] = _codes(lohi, s["rscale"][..., None, None]).to(torch.int8)
            return s
        s["k"], s["v"], s["ks"], s["vs"] = _pool_of(r, case["bits"], case["group"], s["stride"])
        # each row's list: random blocks up to its own, ascending, the last one always
        last = (pos // block).long()[:, None, None]
        n = int(last.max()) + 1
        key = torch.rand((rows, HK, n), generator=r.g, device="cuda")
        ids = torch.arange(n, device="cuda")
        key = torch.where(ids == last, 2.0, torch.where(ids < last, key, -1.0))
        top, at = key.topk(min(n, case["top_k"]), -1)
        at = torch.where(top < 0, n, at).sort(-1).values
        sel = torch.full((rows, HK, case["top_k"]), -1, dtype=torch.int32, device="cuda")
        sel[..., :at.shape[-1]] = torch.where(at == n, -1, at).to(torch.int32)
        s["sel"] = sel
        return s
    n, k, seg1, _ = PROJ[case["proj"]]
    rows, count, rank = case["rows"], case["adapters"], case["rank"]
    parts = {"qkv": 3, "gate_up": 2}.get(case["proj"], 1)
    x = r.hidden(rows, k)
    if case["fp8"]:
        s["xs"] = (x.abs().max() / 448).reshape(1)
        s["x"] = (x / s["xs"]).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s["x"] = x.to(torch.bfloat16)
    s["A"] = r.bf16(count, parts, rank, k, std=1 / math.sqrt(k))
    s["B"] = r.bf16(count, n, rank, std=0.05)
    s["alpha"] = 0.5 + 2 * torch.rand(count, generator=r.g, device="cuda")
    if rows <= 16:  # a row a session; some have no adapter
        s["adapter"] = r.ints(0, 8 * count + 7, rows) % (count + 1) - 1 if count > 1 else r.ints(0, 1, rows)
    else:  # runs of one session's rows
        ends = r.ints(0, rows, 2).sort().values
        which = r.ints(0, count, 3)
        at = torch.arange(rows, device="cuda")
        s["adapter"] = which[(at >= ends[0]).long() + (at >= ends[1]).long()]
    s["base"] = r.normal(rows, n) if case["f32"] else r.bf16(rows, n)
    s["mult"] = RESID if case["proj"] in ("o", "down") else 1.0
    return s


# ---------------------------------------------------------------- plain forms
def _values(rows, scale, bits, is_k, dtype=torch.float32):
    """The values of pool rows [..., row bytes] with scales [..., groups]."""
    if bits == 16:
        return rows.contiguous().view(torch.bfloat16).to(dtype)
    if bits == 8:
        c = rows.contiguous().view(torch.int8).to(dtype)
    else:
        n = rows[..., :D // 2]
        c = torch.stack([n & 15, n >> 4], -1).flatten(-2).to(torch.int32)
        if bits == 5 and is_k:
            p = rows[..., D // 2:, None].to(torch.int32)
            b = (p >> torch.arange(8, device=rows.device, dtype=torch.int32)) & 1
            c = c + (b << 4).flatten(-2) - 16
        else:
            c = c - 8
        c = c.to(dtype)
    return c * scale.to(dtype).repeat_interleave(D // scale.shape[-1], -1)


def _ranges(s):
    c = s["case"]
    block, end = c["block"], c["start"] + c["rows"]
    ids = torch.arange(c["start"] // block, end // block, device="cuda")
    at = s["tables"][0, (ids[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)].long()
    x = _values(s["k"][:, at], None if s["ks"] is None else s["ks"][:, at], c["bits"], True)
    x = x.view(HK, ids.numel(), block, D)
    lohi = torch.stack([x.amin(2), x.amax(2)], 2)
    scale = _div(lohi.abs().amax((2, 3)), torch.tensor(127.0, device="cuda"))
    to = at[::block] // block
    codes, scales = s["ranges"].clone(), s["rscale"].clone()
    codes[:, to] = _codes(lohi, scale[..., None, None]).to(torch.int8)
    scales[:, to] = scale
    return codes * scales[..., None, None]


def _select(s):
    c = s["case"]
    block, top_k, rows = c["block"], c["top_k"], c["rows"]
    n = (s["tables"].shape[1] + block - 1) // block
    ids = torch.arange(n, device="cuda")
    first = s["tables"][:, ids * block].long()  # [sequences][blocks]
    to = first.clamp(min=0) // block
    seqs = first.shape[0]
    lohi = s["ranges"][:, to].float()  # [HK][sequences][blocks][2][D]
    q = s["q"].float().view(seqs, rows // seqs, HK, G, D)
    sq = _div(q.abs().amax(-1, keepdim=True), torch.tensor(127.0, device="cuda"))
    qc = _codes(q, sq).permute(2, 0, 1, 3, 4).reshape(HK, seqs, -1, D)
    # whole numbers below 2^24: exact in any order
    dot = qc.clamp(min=0) @ lohi[..., 1, :].mT + qc.clamp(max=0) @ lohi[..., 0, :].mT
    dot = dot * s["rscale"][:, to][:, :, None, :]
    dot = dot * sq.permute(2, 0, 1, 3, 4).reshape(HK, seqs, -1, 1)
    score = dot.view(HK, rows, G, n).amax(2).permute(1, 0, 2)  # [rows][HK][blocks]
    have = (s["pos"].long() // block + 1)[:, None, None]
    usable = (first >= 0).expand(rows, n)[:, None, :] if seqs == 1 else (first >= 0)[:, None, :]
    kept = (ids < c["sink"]) | (ids >= have - c["recent"])
    score = torch.where(kept, math.inf, score)
    score = torch.where((ids < have) & usable, score, -math.inf)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    at = torch.where(best[..., :top_k] > -math.inf, at[..., :top_k], n).sort(-1).values
    sel = torch.full((rows, HK, top_k), -1, dtype=torch.int32, device="cuda")
    sel[..., :at.shape[-1]] = torch.where(at == n, -1, at).to(torch.int32)
    return sel


def _keys(s):
    """Each row's listed positions [rows][HK][slots], which of them it attends to, and their pool rows."""
    c = s["case"]
    sel = s["sel"].long()
    p = (sel[..., None] * c["block"] + torch.arange(c["block"], device="cuda")).flatten(2)
    ok = (sel >= 0).repeat_interleave(c["block"], -1) & (p <= s["pos"].long()[:, None, None])
    seq = torch.arange(c["rows"], device="cuda") if c["sessions"] else torch.zeros(c["rows"], dtype=torch.int64, device="cuda")
    at = s["tables"][seq[:, None, None], p.clamp(0, s["tables"].shape[1] - 1)].long()
    return ok, at.clamp(min=0)


def _blocks(s):
    c = s["case"]
    ok, at = _keys(s)
    head = torch.arange(HK, device="cuda")[None, :, None]
    k = _values(s["k"][head, at], None if s["ks"] is None else s["ks"][head, at], c["bits"], True)
    q = s["q"].float().view(c["rows"], HK, G, D)
    x = (q @ k.mT) * ATTN_SCALE
    x = torch.where(ok[:, :, None, :], x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    v = _values(s["v"][head, at], None if s["vs"] is None else s["vs"][head, at], c["bits"], False)
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.reshape(c["rows"], NQ).to(torch.bfloat16)


def _lora(s):
    c = s["case"]
    rows, count, rank = c["rows"], c["adapters"], c["rank"]
    n, k, seg1, seg2 = PROJ[c["proj"]]
    x = s["x"].view(torch.float8_e4m3fn).float() * s["xs"] if c["fp8"] else s["x"].float()
    parts = s["A"].shape[1]
    cut = [0, seg1, seg2, n][:parts] + [n]
    a = s["adapter"].long()
    alpha = torch.where(a < 0, 0.0, s["alpha"][a.clamp(min=0)])[:, None] * s["mult"]
    if rows <= 16:  # each row's own matrices
        A, B = s["A"][a.clamp(min=0)].float(), s["B"][a.clamp(min=0)].float()
        t = (A.view(rows, parts * rank, k) @ x[:, :, None]).view(rows, parts, rank, 1)
        y = torch.cat([(B[:, cut[i]:cut[i + 1]] @ t[:, i])[..., 0] for i in range(parts)], 1)
    else:  # few adapters: all of them, the others' columns cleared
        t = (x @ s["A"].float().view(-1, k).T).view(rows, count, parts, rank)
        t = torch.where((torch.arange(count, device="cuda") == a[:, None])[:, :, None, None], t, 0.0)
        y = torch.cat([t[:, :, i].reshape(rows, -1) @
                       s["B"][:, cut[i]:cut[i + 1]].float().transpose(1, 2).reshape(count * rank, -1)
                       for i in range(parts)], 1)
    y = s["base"].float() + alpha * y
    return y if c["f32"] else y.to(torch.bfloat16)


# -------------------------------------------------------- the library's calls
_L = None


def _layerops():
    global _L
    if _L is None:
        path = os.path.join(os.getcwd(), "granite-4-rtx-4070-ti-super_amd", "layerops.py")
        spec = importlib.util.spec_from_file_location("g4_layerops", path)
        _L = importlib.util.module_from_spec(spec)
        sys.modules["g4_layerops"] = _L
        spec.loader.exec_module(_L)
        _L.use_stream()
    return _L


def _work(s, size):
    """The workspace that a program keeps between its calls, made before its first."""
    if "work" not in s:
        s["work"] = torch.zeros(max(16, size()), dtype=torch.uint8, device="cuda")
    return s["work"]


def _call(s):
    L, c = _layerops(), s["case"]
    kind = c["kind"]
    if kind == "ranges":
        L.call("granite4_kv_ranges", s["k"], s["ks"], c["bits"], c["group"], HK, D, s["stride"],
               c["block"], c["start"], c["rows"], None, s["tables"], None, None, s["ranges"],
               s["rscale"])
        return s["ranges"] * s["rscale"][..., None, None]
    if kind in ("select", "blocks"):
        many = c["sessions"] > 0
        where = (0 if many else c["start"], None, None if many else s["tables"],
                 s["row_pos"] if many else None, s["row_pt"] if many else None)
        if kind == "select":
            length = s["tables"].shape[1]
            work = _work(s, lambda: L.call_size("granite4_block_select_work_bytes", c["rows"], HK,
                                                length, c["block"]))
            if "sel" not in s:
                s["sel"] = torch.empty((c["rows"], HK, c["top_k"]), dtype=torch.int32, device="cuda")
            L.call("granite4_block_select", s["q"], c["rows"], HQ, HK, D, s["ranges"], s["rscale"],
                   s["stride"], c["block"], *where, length, c["top_k"], c["sink"], c["recent"],
                   work, s["sel"])
            return s["sel"]
        work = _work(s, lambda: L.call_size("granite4_attn_blocks_scratch_bytes", HQ, c["rows"],
                                            c["top_k"], c["block"]))
        if "out" not in s:
            s["out"] = torch.empty_like(s["q"])
        L.call("granite4_attn_blocks", s["q"], c["rows"], HQ, HK, D, ATTN_SCALE, s["k"], s["v"],
               s["ks"], s["vs"], c["bits"], c["group"], s["stride"], *where, s["sel"], c["top_k"],
               c["block"], work, s["out"])
        return s["out"]
    n, k, seg1, seg2 = PROJ[c["proj"]]
    work = _work(s, lambda: L.call_size("granite4_lora_work_bytes", c["rows"], n, k, c["rank"],
                                        seg1, seg2))
    if "out" not in s:
        s["out"] = torch.empty_like(s["base"])
    L.call("granite4_lora_add", int(c["f32"]), s["x"], 8 if c["fp8"] else 16, k,
           s["xs"] if c["fp8"] else None, s["A"], s["B"], s["alpha"], c["adapters"], c["rank"],
           s["adapter"], c["rows"], n, k, seg1, seg2, s["base"], n, s["mult"], s["out"], n, work)
    return s["out"]


def run(state):
    if own:
        return _call(state)
    return {"ranges": _ranges, "select": _select, "blocks": _blocks, "lora": _lora}[state["case"]["kind"]](state)


# ----------------------------------------------------------------------- work
def _bytes_of(bits, group):
    """Bytes of a cached key and of a cached value with their scales."""
    kb, vb = {16: (256, 256), 8: (128, 128), 4: (64, 64), 5: (80, 64)}[bits]
    more = 0 if bits == 16 else 4 * (D // group)
    return kb + more, vb + more


def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "ranges":
        done = (case["start"] + rows) // case["block"] - case["start"] // case["block"]
        kb, _ = _bytes_of(case["bits"], case["group"])
        return {"bytes": done * HK * (case["block"] * kb + 2 * D + 4) + 4 * rows,
                "flops": 2 * done * case["block"] * NK}
    if kind in ("select", "blocks"):
        block, top_k = case["block"], case["top_k"]
        # sessions lie anywhere: the mean of their positions
        ctx = (65000 - 64) / math.log(65000 / 64) if case["sessions"] else case["start"] + rows / 2
        n = math.ceil(ctx / block)
        seqs = rows if case["sessions"] else 1
        if kind == "select":
            scored = max(0, n - case["sink"] - case["recent"])
            return {"bytes": seqs * scored * HK * (2 * D + 4) + rows * (2 * NQ + 4 * HK * top_k),
                    "flops": rows * HQ * scored * 2 * D}
        slots = min(n, top_k) * block
        kb, vb = _bytes_of(case["bits"], case["group"])
        keys = rows * slots if case["sessions"] else min(rows * slots, n * block)
        return {"bytes": keys * HK * (kb + vb) + rows * (4 * NQ + 4 * HK * top_k),
                "flops": rows * HQ * slots * 4 * D}
    n, k, _, _ = PROJ[case["proj"]]
    parts = {"qkv": 3, "gate_up": 2}.get(case["proj"], 1)
    rank, used = case["rank"], min(case["adapters"], rows if rows <= 16 else 3)
    each = 4 if case["f32"] else 2
    return {"bytes": rows * (k * (1 if case["fp8"] else 2) + 2 * n * each + 4) + used * 2 * rank * (parts * k + n),
            "flops": 2 * rows * rank * (parts * k + n)}


# ---------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    kind, rows = case["kind"], case["rows"]
    if kind == "ranges":
        block, out = case["block"], torch.zeros((HK, s["stride"] // case["block"], 2, D), dtype=torch.float64, device="cuda")
        x = _values(s["k"], s["ks"], case["bits"], True, torch.float64).float()  # a key's value is one f32 product
        for b in range(case["start"] // block, (case["start"] + rows) // block):
            at = s["tables"][0, b * block:(b + 1) * block].long()
            lo, hi = x[:, at].min(1).values, x[:, at].max(1).values
            scale = (torch.maximum(lo.abs(), hi.abs()).max(-1, keepdim=True).values.double() / 127).float().double()
            for i, y in enumerate((lo, hi)):
                z = (y.double() / scale).float().double()  # the code is the rounded quotient's
                out[:, int(at[0]) // block, i] = scale * torch.sign(z) * torch.floor(z.abs() + 0.5)
        return out
    if kind == "select":
        block, top_k = case["block"], case["top_k"]
        out = torch.full((rows, HK, top_k), -1, dtype=torch.int32)
        lohi, scale = s["ranges"].double(), s["rscale"]
        for r in range(rows):
            table = s["tables"][r if case["sessions"] else 0]
            have = int(s["pos"][r]) // block + 1
            if have <= top_k:
                out[r, :, :have] = torch.arange(have, dtype=torch.int32)
                continue
            to = (table[:have * block:block] // block).long()
            q = s["q"][r].double().view(HK, G, 1, D)
            sq = (q.abs().amax(-1, keepdim=True) / 127).float()
            z = (q / sq.double()).float().double()
            z = torch.sign(z) * torch.floor(z.abs() + 0.5)
            dot = torch.empty((HK, G, have), dtype=torch.float64, device="cuda")
            for h in range(HK):
                dot[h] = torch.maximum(z[h] * lohi[h, to, 0], z[h] * lohi[h, to, 1]).sum(-1)
            # the score is defined with two f32 roundings
            score = ((dot.float() * scale[:, to][:, None]) * sq[..., 0]).max(1).values.double()
            score[:, :case["sink"]] = math.inf
            score[:, have - case["recent"]:] = math.inf
            # by score, then by the lower index
            best = torch.argsort(-score, dim=-1, stable=True)[:, :top_k]
            out[r] = best.sort(-1).values.int().cpu()
        return out.cuda()
    if kind == "blocks":
        out = torch.empty((rows, HK, G, D), dtype=torch.float64, device="cuda")
        ids = torch.arange(case["block"], device="cuda")
        for r in range(rows):
            table = s["tables"][r if case["sessions"] else 0]
            for h in range(HK):
                p = (s["sel"][r, h].long()[:, None] * case["block"] + ids).reshape(-1)
                at = table[p[(p >= 0) & (p <= s["pos"][r])]].long()
                k = _values(s["k"][h, at], None if s["ks"] is None else s["ks"][h, at], case["bits"], True, torch.float64)
                v = _values(s["v"][h, at], None if s["vs"] is None else s["vs"][h, at], case["bits"], False, torch.float64)
                q = s["q"][r].double().view(HK, G, D)[h]
                out[r, h] = torch.softmax(q @ k.T * ATTN_SCALE, -1) @ v
        return out.view(rows, NQ)
    n, k, seg1, seg2 = PROJ[case["proj"]]
    x = s["x"].view(torch.float8_e4m3fn).double() * s["xs"].double() if case["fp8"] else s["x"].double()
    y = s["base"].double()
    for a in range(case["adapters"]):
        at = (s["adapter"] == a).nonzero()[:, 0]
        for i, (lo, hi) in enumerate(((0, seg1), (seg1, seg2), (seg2, n))):
            if at.numel() and lo < hi:
                d = x[at] @ s["A"][a, i].double().T @ s["B"][a, lo:hi].double().T
                y[at, lo:hi] += s["mult"] * s["alpha"][a].double() * d
    return y
