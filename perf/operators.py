"""Rotary positions, the latent cache written and read back, and attention for
trees of drafted tokens: the operators that surround an MLA layer's attention
when a server rotates, quantises, re-reads and verifies by itself.

Kinds of case:

* rope    apply_rotary: a step's q (the last 64 dims of a head, interleaved
          pairs), k_pe, and with `idx` the indexer's q and k (the first 64 of
          128 dims, half layout), or one tensor of odd sizes (`dim`, `rot`,
          `offset`; `pairs`: interleaved).
* cache   rope_concat_and_cache_mla of a step's tokens, then
          gather_latent_cache of their rows (`read` "new") or of the whole
          context up to them ("context").
* gather  gather_latent_cache of requests' contexts.
* tree    tree_attention: every request's drafted tokens over its paged context.

Sizes are those of the benchmark and tests (64 heads and a tensor-parallel
rank's 8-32, 512 + 64 latent dims, 128 + 64 query dims, 32 x 128 indexer, pages
of 64, contexts up to 184,320) and odd ones around them.

`own` false: plain torch in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
LAT, VAL, ROT, NOPE = 576, 512, 64, 128
SCALE = (NOPE + ROT) ** -0.5
BASE = 10000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one user's decode step at a far position: one launch, latency only
        dict(name="rope_decode_1", kind="rope", tokens=1, heads=64, idx=True, dtype="fp16",
             ctx=184320, scaling="yarn"),
        # a prefill chunk in the model's own type
        dict(name="rope_prefill_8192_bf16", kind="rope", tokens=8192, heads=64, idx=False,
             dtype="bf16", ctx=65536, scaling="yarn"),
        # odd sizes: 17 heads of 100 dims, 36 of them rotated from dim 13 on, fp32
        dict(name="rope_odd_fp32", kind="rope", tokens=1537, heads=17, idx=False, dtype="fp32",
             ctx=5000, scaling="linear", dim=100, rot=36, offset=13, pairs=False),
        # a full server's decode step, two tokens a request: write, and read the new rows
        dict(name="cache_decode_24x2", kind="cache", requests=24, tokens=2, ctx=30011, heads=64,
             kv="fp8", dtype="fp16", page=64, read="new", scaling="none"),
        # a prefill chunk behind its history: write 4096 tokens, read the 16k context back
        dict(name="cache_chunk_2x4096_bf16", kind="cache", requests=2, tokens=4096, ctx=16384,
             heads=64, kv="fp8", dtype="bf16", page=64, read="context", scaling="yarn"),
        # the context of four 32k requests for a dense chunk pass
        dict(name="gather_4x32k_fp8", kind="gather", requests=4, ctx=32768, ragged=False,
             kv="fp8", dtype="fp16", page=64, start=0),
        # short ragged prompts on small pages, fp16 rows read as bf16 from an odd start
        dict(name="gather_7_ragged_fp16", kind="gather", requests=7, ctx=5003, ragged=True,
             kv="fp16", dtype="bf16", page=16, start=37),
        # one user, four drafted tokens, short context: latency
        dict(name="tree_1x4_16h", kind="tree", requests=1, nodes=4, heads=16, ctx=500,
             kv="fp16", page=64, ragged=False),
        # an ordinary verification step
        dict(name="tree_8x8_64h_16k_fp8", kind="tree", requests=8, nodes=8, heads=64, ctx=16384,
             kv="fp8", page=64, ragged=False),
        # a tensor-parallel rank's 16 heads, one wide tree at the longest context
        dict(name="tree_1x64_16h_180k", kind="tree", requests=1, nodes=64, heads=16, ctx=184320,
             kv="fp16", page=64, ragged=False),
        # mixed requests: trees of 1 to 13 nodes, contexts from nothing to 20k, odd page size
        dict(name="tree_24_ragged_32h", kind="tree", requests=24, nodes=13, heads=32, ctx=20011,
             kv="fp16", page=48, ragged=True),
        # the largest: 16 requests, 40 nodes each, fp8 rows at 32k
        dict(name="tree_16x40_64h_32k_fp8", kind="tree", requests=16, nodes=40, heads=64,
             ctx=32768, kv="fp8", page=64, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rope", "cache", "gather", "tree", "tree", "tree"])
    kv = rng.choice(["fp8", "fp16"])
    page = rng.choice([64, 64, 16, 48, 128, 1])
    scaling = rng.choice(["none", "linear", "yarn"])
    if kind == "rope":
        if rng.random() < 0.3:
            rot = 2 * rng.randint(1, 64)
            offset = rng.randint(0, 40)
            return dict(kind=kind, tokens=_log(rng, 1, 4096), heads=rng.randint(1, 33), idx=False,
                        dtype=rng.choice(["fp16", "bf16", "fp32"]), ctx=_log(rng, 5000, 184320),
                        scaling=scaling, dim=rot + offset + rng.randint(0, 30), rot=rot,
                        offset=offset, pairs=rng.random() < 0.5)
        return dict(kind=kind, tokens=_log(rng, 1, 8192), heads=rng.choice([64, 32, 16, 8]),
                    idx=rng.random() < 0.5, dtype=rng.choice(["fp16", "bf16"]),
                    ctx=_log(rng, 8192, 184320), scaling=scaling)
    if kind == "cache":
        requests = _log(rng, 1, 48)
        tokens = _log(rng, 1, 8192 // requests)
        return dict(kind=kind, requests=requests, tokens=tokens,
                    ctx=tokens + _log(rng, 1, 32768 // requests), heads=rng.choice([64, 32, 16, 5]),
                    kv=kv, dtype="fp16" if kv == "fp16" else rng.choice(["fp16", "bf16"]),
                    page=page, read=rng.choice(["new", "context"]), scaling=scaling)
    if kind == "gather":
        requests = _log(rng, 1, 64)
        ctx = _log(rng, 1, 131072 // requests)
        return dict(kind=kind, requests=requests, ctx=ctx,
                    ragged=rng.random() < 0.6, kv=kv, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    page=page, start=rng.choice([0, 0, rng.randint(0, ctx - 1)]))
    heads = rng.choice([64, 64, 32, 16, 8, 20])
    requests, nodes = _log(rng, 1, 32), _log(rng, 1, 64)
    rows = requests * nodes * heads
    most = min(184320, 600000 // requests, 1300000000 // rows)
    return dict(kind=kind, requests=requests, nodes=nodes, heads=heads,
                ctx=_log(rng, min(100, most), most), kv=kv, page=page, ragged=rng.random() < 0.5)


def _lens(case):
    """Context length of each request (a property of the case): the ragged ones
    from ctx down to nothing."""
    n, ctx = case["requests"], case["ctx"]
    if not case.get("ragged"):
        return [ctx] * n
    return [ctx * (n - 1 - i) // max(n - 1, 1) for i in range(n)]


def _nodes(case):
    n, k = case["requests"], case["nodes"]
    return [1 + (5 * i + k - 1) % k for i in range(n)] if case.get("ragged") else [k] * n


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inv_freq(rot, scaling):
    """Angle per position of each pair, and the factor on cos and sin."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEV)
    f = BASE ** (-i / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":  # factor 40 over 4096 positions, 32 / 1 turns, magnitude 1 over all dims 0
        def turns(r):
            return rot * math.log(4096 / (r * 2 * math.pi)) / (2 * math.log(BASE))
        lo, hi = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64, device=DEV) - lo)
                / max(hi - lo, 0.001)).clamp(0, 1)
        return f / 40.0 * ramp + f * (1 - ramp), 0.1 * math.log(40.0) + 1.0
    return f, 1.0


def _table(rot, n, scaling):
    """[n, rot] fp32: the cosines of a position's pairs, then the sines."""
    f, m = _inv_freq(rot, scaling)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * f
    return (torch.cat([a.cos(), a.sin()], 1) * m).float()


def _quantise(lat):
    """fp8_ds_mla rows [n, 656] of latents [n, 576]: e4m3 per 128-dim tile, the
    four scales, the rope values as fp16."""
    n = lat.shape[0]
    t = lat[:, :VAL].float().view(n, 4, 128)
    s = (t.abs().amax(2) / 448.0).clamp_min(torch.finfo(torch.float32).tiny)
    q = (t / s[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(n, VAL)
    return torch.cat([q, s.view(torch.uint8).view(n, 16),
                      lat[:, VAL:].half().view(torch.uint8).view(n, 128)], 1)


def _cache(blocks, page, kv, g):
    n = blocks * page
    out = torch.empty(n, 656 if kv == "fp8" else LAT, device=DEV,
                      dtype=torch.uint8 if kv == "fp8" else torch.float16)
    for lo in range(0, n, 1 << 18):
        lat = torch.randn(min(n - lo, 1 << 18), LAT, generator=g, device=DEV)
        out[lo:lo + lat.shape[0]] = _quantise(lat) if kv == "fp8" else lat
    return out.view(blocks, page, -1)


def _paging(lens, page, g):
    """A random page order: block table [requests, blocks] and the pool's size."""
    most = max(1, max(-(-n // page) for n in lens))
    pool = sum(max(1, -(-n // page)) for n in lens) + 3
    perm = torch.randperm(pool, generator=g, device=DEV).int()
    bt, at = torch.full((len(lens), most), -1, dtype=torch.int32), 0
    order = perm.cpu()
    for r, n in enumerate(lens):
        k = max(1, -(-n // page))
        bt[r, :k] = order[at:at + k]
        at += k
    return bt.to(DEV), pool


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=DEV)


def _slots(bt, page, lens, counts):
    """Cache row of the last counts[r] positions of each request."""
    r = torch.repeat_interleave(torch.arange(len(lens), device=DEV),
                                torch.tensor(counts, device=DEV))
    off = _cu(counts).long()
    p = (torch.arange(int(off[-1]), device=DEV) - off[r]
         + torch.tensor([n - c for n, c in zip(lens, counts)], device=DEV)[r])
    return bt[r, p // page].long() * page + p % page, p


def prepare(case, seed):
    g = _gen(seed)
    k = case["kind"]
    if k == "rope":
        dt, T, H = DTYPES[case["dtype"]], case["tokens"], case["heads"]
        rot, off = case.get("rot", ROT), case.get("offset", NOPE)
        dim = case.get("dim", NOPE + ROT)
        x = [torch.randn(T, H, dim, generator=g, device=DEV).to(dt)]
        offs, inter = [off], [True]
        if "dim" not in case:
            x.append(torch.randn(T, ROT, generator=g, device=DEV).to(dt))
            offs, inter = [off, 0], [True, True]
        else:
            inter = [case["pairs"]]
        if case["idx"]:
            x += [torch.randn(T, 32, 128, generator=g, device=DEV).to(dt),
                  torch.randn(T, 128, generator=g, device=DEV).to(dt)]
            offs, inter = offs + [0, 0], inter + [False, False]
        pos = torch.randint(0, case["ctx"], (T,), generator=g, device=DEV)
        if T > 256:  # a chunk of one request
            pos = pos[0] % max(case["ctx"] - T, 1) + torch.arange(T, device=DEV)
        return dict(case=case, x=x, offs=offs, inter=inter, pos=pos,
                    table=_table(rot, max(case["ctx"], T), case["scaling"]))
    lens = _lens(case)
    if k == "tree":
        counts = _nodes(case)
        lens = [a + b for a, b in zip(lens, counts)]  # the drafted tokens are in the cache
    bt, pool = _paging(lens, case["page"], g)
    cache = _cache(pool, case["page"], case["kv"], g)
    s = dict(case=case, bt=bt, cache=cache, lens=lens)
    if k == "cache":
        T, H = case["requests"] * case["tokens"], case["heads"]
        dt = DTYPES[case["dtype"]]
        counts = [case["tokens"]] * case["requests"]
        s["slots"], s["pos"] = _slots(bt, case["page"], lens, counts)
        s["table"] = _table(ROT, case["ctx"], case["scaling"])
        s["q"] = torch.randn(T, H, NOPE + ROT, generator=g, device=DEV).to(dt)
        s["kv_c"] = torch.randn(T, VAL, generator=g, device=DEV).to(dt)
        s["k_pe"] = torch.randn(T, ROT, generator=g, device=DEV).to(dt)
        if dt is torch.bfloat16:  # the history's rope values are of that type too
            c = cache.view(-1, 656)[:, 528:]
            c.copy_(c.contiguous().view(torch.float16).to(dt).view(torch.uint8))
        first = [0 if case["read"] == "context" else n - case["tokens"] for n in lens]
    elif k == "gather":
        first = [min(case["start"], n) for n in lens]
    if k in ("cache", "gather"):
        n = [a - b for a, b in zip(lens, first)]
        s["first"] = torch.tensor(first, dtype=torch.int32, device=DEV)
        s["cu"], s["total"] = _cu(n), sum(n)
        return s
    rng = random.Random(seed)
    mask = []
    for r, n in enumerate(counts):
        anc = []
        for j in range(n):  # node j hangs on an earlier one, or on the context
            p = rng.randint(-1, j - 1)
            anc.append((anc[p] if p >= 0 else 0) | 1 << j)
        if r == len(counts) - 1 and case["ragged"]:
            anc[0] = 0  # sees no drafted token, and its context may be empty
        mask += [a - (1 << 64) if a >> 63 else a for a in anc]
    T = sum(counts)
    s.update(cu=_cu(counts), counts=counts, mask=torch.tensor(mask, device=DEV),
             seq=torch.tensor(lens, dtype=torch.int32, device=DEV),
             q=torch.randn(T, case["heads"], LAT, generator=g, device=DEV).half() * 0.5)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _rotate(x, pos, table, off, inter):
    rot = table.shape[1]
    cs = table[pos].view(pos.shape[0], *([1] * (x.dim() - 2)), rot)
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    y = x.float()
    z = y[..., off:off + rot]
    a, b = (z[..., 0::2], z[..., 1::2]) if inter else (z[..., :rot // 2], z[..., rot // 2:])
    u, v = a * c - b * s, b * c + a * s
    r = torch.stack([u, v], -1).flatten(-2) if inter else torch.cat([u, v], -1)
    return torch.cat([y[..., :off], r, y[..., off + rot:]], -1).to(x.dtype)


def _values(rows, pe):
    """Rows of either cache as fp32 values; `pe` the type of the rope values."""
    if rows.dtype != torch.uint8:
        return rows.float()
    n = rows.shape[0]
    v = rows[:, :VAL].contiguous().view(torch.float8_e4m3fn).float().view(n, 4, 128)
    v = v * rows[:, VAL:VAL + 16].contiguous().view(torch.float32)[:, :, None]
    return torch.cat([v.view(n, VAL), rows[:, VAL + 16:].contiguous().view(pe).float()], 1)


def _gathered(s, dt, pe):
    cu, page = s["cu"].long(), s["case"]["page"]
    t = torch.arange(s["total"], device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True)
    p = t - cu[r] + s["first"].long()[r]
    row = s["bt"][r, p // page].long() * page + p % page
    return _values(s["cache"].flatten(0, 1)[row], pe).to(dt)


def _write(s):
    kv, pe = s["kv_c"], _rotate(s["k_pe"], s["pos"], s["table"], 0, True)
    rows = s["cache"].view(-1, s["cache"].shape[-1])
    if rows.dtype == torch.uint8:
        n = kv.shape[0]
        t = kv.float().view(n, 4, 128)
        sc = (t.abs().amax(2) / 448.0).clamp_min(torch.finfo(torch.float32).tiny)
        q = (t / sc[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(n, VAL)
        rows[s["slots"]] = torch.cat([q, sc.view(torch.uint8).view(n, 16),
                                      pe.view(torch.uint8).view(n, 128)], 1)
    else:
        rows[s["slots"]] = torch.cat([kv, pe], 1)
    return _rotate(s["q"], s["pos"], s["table"], NOPE, True)


def _tree(s):
    """Every request padded to the longest: its tokens x heads against its keys.
    fp8 rows count as the fp16 values that reading them back gives."""
    H, page, R = s["q"].shape[1], s["case"]["page"], len(s["lens"])
    n, L = max(s["counts"]), max(s["lens"])
    cu, seq = s["cu"].long(), s["seq"].long()
    cnt = cu[1:] - cu[:-1]
    j = torch.arange(n, device=DEV)
    tok = (cu[:-1, None] + j).clamp(max=s["q"].shape[0] - 1)           # [R, n]
    p = torch.arange(L, device=DEV)
    row = (s["bt"].long()[:, p // page] * page + p % page).clamp_min(0)  # [R, L]
    K = _values(s["cache"].flatten(0, 1)[row.view(-1)], torch.float16).half().float()
    K = K.view(R, L, LAT)
    q = s["q"][tok].float().view(R, n * H, LAT)
    d = p - (seq - cnt)[:, None]                                        # [R, L] drafted index
    bit = (s["mask"][tok][:, :, None] >> d.clamp(0, 63)[:, None, :]) & 1
    see = (((d < 0)[:, None, :]) | (bit != 0)) & (p < seq[:, None])[:, None, :]  # [R, n, L]
    see = see[:, :, None, :].expand(R, n, H, L).reshape(R, n * H, L)
    S = torch.bmm(q, K.transpose(1, 2).contiguous()).mul_(SCALE).masked_fill_(~see, -math.inf)
    m = S.amax(2, keepdim=True).clamp_min(-1e30)
    P = S.sub_(m).exp_()
    l = P.sum(2, keepdim=True)
    o = torch.bmm(P, K[:, :, :VAL].contiguous()) / l.clamp_min(1e-30)
    live = (j < cnt[:, None]).view(-1)
    lse = (m + l.log()).view(R * n, H)[live]
    return o.view(R * n, H, VAL)[live].half(), lse


def run(state):
    s, c = state, state["case"]
    k = c["kind"]
    if own:
        from __graft_entry__ import load_package

        pkg = load_package()
        if k == "rope":
            return pkg.rope.apply_rotary(s["x"], s["pos"], s["table"], offsets=s["offs"],
                                         interleaved=s["inter"])
        if k == "tree":
            return pkg.mla_tree.tree_attention(s["q"], s["cache"], s["bt"], s["seq"], s["cu"],
                                               s["mask"], SCALE)
        dt = DTYPES[c["dtype"]]
        pe = dt if k == "cache" else torch.float16
        out = {}
        if k == "cache":
            out["q"] = pkg._cache_ops.rope_concat_and_cache_mla(
                s["pos"], s["table"], s["kv_c"], s["k_pe"], s["cache"], s["slots"],
                "fp8_ds_mla" if c["kv"] == "fp8" else "auto", q=s["q"], q_offset=NOPE)
        out["kv"] = pkg._cache_ops.gather_latent_cache(
            s["cache"], s["bt"], s["cu"], s["total"], starts=s["first"], dtype=dt, pe_dtype=pe)
        return out
    if k == "rope":
        if len(s["x"]) == 1:
            return [_rotate(s["x"][0], s["pos"], s["table"], s["offs"][0], s["inter"][0])]
        y = [_rotate(s["x"][0], s["pos"], s["table"], s["offs"][0], s["inter"][0]),
             _rotate(s["x"][1], s["pos"], s["table"], s["offs"][1], s["inter"][1])]
        if c["idx"]:
            y += [_rotate(s["x"][2], s["pos"], s["table"], s["offs"][2], s["inter"][2]),
                  _rotate(s["x"][3], s["pos"], s["table"], s["offs"][3], s["inter"][3])]
        return y
    if k == "tree":
        return _tree(s)
    dt = DTYPES[c["dtype"]]
    if k == "cache":
        q = _write(s)
        return {"q": q, "kv": _gathered(s, dt, dt)}
    return {"kv": _gathered(s, dt, torch.float16)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    k, kv = case["kind"], 656 if case.get("kv") == "fp8" else 1152
    if k == "rope":
        e, T, rot = torch.finfo(DTYPES[case["dtype"]]).bits // 8, case["tokens"], case.get("rot", ROT)
        n = T * case["heads"] * case.get("dim", NOPE + ROT)
        turned = T * case["heads"] * rot
        if "dim" not in case:
            n, turned = n + T * ROT, turned + T * ROT
        if case["idx"]:
            n, turned = n + T * 33 * 128, turned + T * 33 * ROT
        return dict(bytes=2 * e * n + T * (rot * 4 + 8), flops=3 * turned)
    lens = _lens(case)
    if k == "gather":
        n = sum(x - min(case["start"], x) for x in lens)
        return dict(bytes=n * (kv + LAT * torch.finfo(DTYPES[case["dtype"]]).bits // 8), flops=n * VAL)
    if k == "cache":
        T = case["requests"] * case["tokens"]
        n = sum(lens) if case["read"] == "context" else T
        move = T * (2 * 2 * case["heads"] * (NOPE + ROT) + 2 * LAT + kv + 4 * ROT + 16)
        return dict(bytes=move + n * (kv + 2 * LAT), flops=T * 3 * VAL + n * VAL)
    nodes = _nodes(case)
    rows = [a * case["heads"] for a in nodes]
    keys = [a + b for a, b in zip(lens, nodes)]
    io = sum(rows) * (2 * LAT + 2 * VAL + 4) + sum(keys) * kv
    return dict(bytes=io, flops=sum(a * b for a, b in zip(rows, keys)) * 2 * (LAT + VAL))


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _turn64(x, pos, rot, off, inter, scaling):
    f, m = _inv_freq(rot, scaling)
    ang = pos.double()[:, None] * f
    z = x.double()
    z = z[:, None] if z.dim() == 2 else z
    y = z.clone()
    for i in range(rot // 2):
        a, b = (off + 2 * i, off + 2 * i + 1) if inter else (off + i, off + rot // 2 + i)
        c, s = m * ang[:, i].cos()[:, None], m * ang[:, i].sin()[:, None]
        y[:, :, a], y[:, :, b] = z[:, :, a] * c - z[:, :, b] * s, z[:, :, b] * c + z[:, :, a] * s
    return y.view(x.shape)


def _row64(cache, page, bt, r, p, pe):
    rows = cache.flatten(0, 1)[bt[r].long()[p // page] * page + p % page]
    if cache.dtype != torch.uint8:
        return rows.double()
    b = rows[:, :VAL].long()
    e, f = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * torch.exp2(e.double() - 10))
    val = torch.where(b >= 128, -mag, mag)
    sc = rows[:, VAL:VAL + 16].contiguous().view(torch.float32).double()
    return torch.cat([val * sc.repeat_interleave(128, 1),
                      rows[:, VAL + 16:].contiguous().view(pe).double()], 1)


def exact(case, seed):
    s = prepare(case, seed)
    k, page = case["kind"], case.get("page")
    if k == "rope":
        return [_turn64(x, s["pos"], s["table"].shape[1], o, i, case["scaling"])
                for x, o, i in zip(s["x"], s["offs"], s["inter"])]
    if k == "tree":
        out, lses = [], []
        cu = s["cu"].tolist()
        for r, n in enumerate(s["lens"]):
            lo, hi = cu[r], cu[r + 1]
            K = _row64(s["cache"], page, s["bt"], r, torch.arange(n, device=DEV), torch.float16)
            K = K.half().double()
            q = s["q"][lo:hi].double()
            sc = torch.einsum("thd,kd->thk", q, K) * SCALE
            for j in range(hi - lo):
                m = int(s["mask"][lo + j])
                for i in range(hi - lo):
                    if not (m >> i) & 1:
                        sc[j, :, n - (hi - lo) + i] = -math.inf
            lse = torch.logsumexp(sc, 2)
            P = torch.exp(sc - lse[:, :, None]).nan_to_num(0.0)
            out.append(torch.einsum("thk,kd->thd", P, K[:, :VAL]))
            lses.append(lse)
        return torch.cat(out), torch.cat(lses)
    pe = DTYPES[case["dtype"]] if k == "cache" else torch.float16
    if k == "cache":  # the quantised rows' values are whole steps of their scale
        q = _turn64(s["q"], s["pos"], ROT, NOPE, True, case["scaling"])
        new = torch.cat([s["kv_c"].double(),
                         _turn64(s["k_pe"], s["pos"], ROT, 0, True, case["scaling"])], 1)
        if case["kv"] == "fp8":
            t = s["kv_c"].float().view(-1, 4, 128)
            sc = (t.abs().amax(2) / 448.0).double()[:, :, None]
            x = t.double() / sc
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
            new[:, :VAL] = (torch.round(x / step) * step * sc).view(-1, VAL)
    kv, lens, first = [], s["lens"], s["first"].tolist()
    for r, n in enumerate(lens):
        v = _row64(s["cache"], page, s["bt"], r, torch.arange(first[r], n, device=DEV), pe)
        if k == "cache":
            c = case["tokens"]
            v[v.shape[0] - c:] = new[r * c:(r + 1) * c]
        kv.append(v)
    out = {"kv": torch.cat(kv)}
    return {"q": q, **out} if k == "cache" else out
