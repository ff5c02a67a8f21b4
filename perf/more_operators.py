"""A decode step of many requests of one prompt: attention that reads the prompt's
cache rows once for all of them, the block tables and slot maps of the step, and the
projections with 4-bit weights.

Kinds of case:

* prefix    shared_prefix_attention: groups of requests whose first positions are the
            same cache rows; each request's own positions behind them, its last
            `nodes` a drafted tree (1: an ordinary decode step).
* tables    extend_tables of a step's tokens, the length that each group shares, then
            truncate_tables back (a step whose tokens are all rejected), so that the
            state is again what it was.
* expand    token_tables: a step's block-table rows and lengths token by token.
* linear    w4_linear of a layer's projections at decode batch sizes.
* weights   w4_quantize of a projection's weights and w4_dequant of the result.

Sizes are those of the benchmark and tests (64 heads and a tensor-parallel rank's
8-32, 512 + 64 latent dims, pages of 64, contexts up to 184,320, projections
6144 x 24576 and 2112 x 6144) and odd ones around them.

`own` false: plain torch in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
LAT, VAL = 576, 512
SCALE = 192 ** -0.5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # four answers to a short prompt on a tensor-parallel rank: latency
        dict(name="prefix_4_16h_500", kind="prefix", groups=1, requests=4, nodes=1, heads=16,
             shared=512, own_len=20, kv="fp16", page=64, ragged=False),
        # a server whose requests share a long system prompt, fp8 rows
        dict(name="prefix_32_64h_32k_fp8", kind="prefix", groups=1, requests=32, nodes=1, heads=64,
             shared=32768, own_len=500, kv="fp8", page=64, ragged=False),
        # few answers over the longest context, four drafted tokens each, 16 heads
        dict(name="prefix_8x4_16h_180k", kind="prefix", groups=1, requests=8, nodes=4, heads=16,
             shared=184320 - 64, own_len=60, kv="fp16", page=64, ragged=False),
        # several prompts at once, answers of mixed lengths, odd page size, a request alone
        dict(name="prefix_5_groups_ragged", kind="prefix", groups=5, requests=7, nodes=3, heads=20,
             shared=9000, own_len=3001, kv="fp16", page=48, ragged=True),
        # the largest: 128 answers of 64 heads over 32k
        dict(name="prefix_128_64h_32k", kind="prefix", groups=1, requests=128, nodes=1, heads=64,
             shared=32768, own_len=1000, kv="fp16", page=64, ragged=False),
        # a full server's decode step: 256 requests, one token each, eight prompts
        dict(name="tables_256x1", kind="tables", groups=8, requests=32, tokens=1, ctx=30011, page=64),
        # prefill chunks of eight requests
        dict(name="tables_8x4096", kind="tables", groups=2, requests=4, tokens=4096, ctx=16384,
             page=16),
        # per-token tables of a prefill chunk at the longest context
        dict(name="expand_2x2048_180k", kind="expand", requests=2, tokens=2048, ctx=184320, page=64),
        # one user's output projection
        dict(name="linear_1_6144x24576", kind="linear", m=1, n=6144, k=24576, group=128,
             dtype="fp16", zeros=True),
        # a small batch through the fused down projections
        dict(name="linear_5_2112x6144_bf16", kind="linear", m=5, n=2112, k=6144, group=64,
             dtype="bf16", zeros=True),
        # a full decode batch
        dict(name="linear_64_24576x6144", kind="linear", m=64, n=24576, k=6144, group=128,
             dtype="fp16", zeros=False),
        # weights quantised at load, and read back for prefill
        dict(name="weights_24576x6144", kind="weights", n=24576, k=6144, group=128, dtype="fp16",
             zeros=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "tables", "expand", "linear", "linear", "weights"])
    page = rng.choice([64, 64, 16, 48, 128, 1])
    if kind == "prefix":
        heads = rng.choice([64, 64, 32, 16, 8, 20])
        groups, nodes = rng.choice([1, 1, 1, 2, 5]), rng.choice([1, 1, 1, 2, 4, 9])
        requests = _log(rng, 1, 128 // groups)
        rows = groups * requests * nodes * heads
        most = min(184320, 400000 // groups, 250000000 // rows)
        shared = _log(rng, min(100, most), most)
        own_len = nodes + _log(rng, 1, max(1, min(4000, 1500000 // (groups * requests),
                                                  30000000 // rows)))
        return dict(kind=kind, groups=groups, requests=requests, nodes=nodes, heads=heads,
                    shared=shared, own_len=own_len, kv=rng.choice(["fp8", "fp16"]), page=page,
                    ragged=rng.random() < 0.5)
    if kind == "tables":
        groups, requests = _log(rng, 1, 16), _log(rng, 1, 64)
        tokens = _log(rng, 1, 32768 // (groups * requests))
        return dict(kind=kind, groups=groups, requests=requests, tokens=tokens,
                    ctx=_log(rng, 64, min(184320, 8000000 // (groups * requests))), page=page)
    if kind == "expand":
        requests = _log(rng, 1, 64)
        page = max(page, 16)
        ctx = _log(rng, 1000, 184320)
        tokens = _log(rng, 1, min(8192, 20000000 // (ctx // page + 1)) // requests + 1)
        return dict(kind=kind, requests=requests, tokens=tokens, ctx=max(ctx, tokens), page=page)
    n = _log(rng, 100, 24576)
    k = 8 * _log(rng, 16, min(3000, 6144 * 24576 // (8 * n)))
    more = dict(n=n, k=k, group=rng.choice([32, 64, 128, 128]), dtype=rng.choice(["fp16", "bf16"]),
                zeros=rng.random() < 0.7)
    if kind == "linear":
        return dict(kind=kind, m=_log(rng, 1, 64), **more)
    return dict(kind=kind, **more)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cu(counts):
    c = [0]
    for n in counts:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=DEV)


def _shape(case):
    """Requests of each group, the positions that it shares, own positions and drafted
    tokens of each request (properties of the case)."""
    G, n = case["groups"], case["requests"]
    if not case["ragged"]:
        R = G * n
        return [n] * G, [case["shared"]] * G, [case["own_len"]] * R, [case["nodes"]] * R
    # groups from `requests` down to a request alone, which shares nothing
    sizes = [max(1, n - (n - 1) * i // max(G - 1, 1)) for i in range(G)]
    shared = [case["shared"] * (G - i) // G if s > 1 or G == 1 else 0 for i, s in enumerate(sizes)]
    R = sum(sizes)
    nodes = [1 + (5 * r + case["nodes"] - 1) % case["nodes"] for r in range(R)]
    own_len = [max(k, case["own_len"] * (R - r) // R) for r, k in zip(range(R), nodes)]
    return sizes, shared, own_len, nodes


def _quantise(lat):
    """fp8_ds_mla rows [n, 656] of latents [n, 576]."""
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


def _prefix_state(case, seed, g):
    page = case["page"]
    sizes, shared, own_len, nodes = _shape(case)
    shared = [p // page * page for p in shared]  # whole pages are shared
    group = [s for s, n in enumerate(sizes) for _ in range(n)]
    lens = [shared[s] + n for s, n in zip(group, own_len)]
    width = max(-(-n // page) for n in lens)
    own_pages = [-(-n // page) for n in own_len]
    pool = sum(p // page for p in shared) + sum(own_pages) + 3
    order = torch.randperm(pool, generator=g, device=DEV).int().cpu()
    bt, at, first = torch.full((len(lens), width), -1, dtype=torch.int32), 0, []
    for p in shared:
        first.append(order[at:at + p // page])
        at += p // page
    for r, s in enumerate(group):
        k = shared[s] // page
        bt[r, :k] = first[s]
        bt[r, k:k + own_pages[r]] = order[at:at + own_pages[r]]
        at += own_pages[r]
    rng = random.Random(seed)
    mask = []
    for n in nodes:
        anc = []
        for j in range(n):  # node j hangs on an earlier one, or on the context
            p = rng.randint(-1, j - 1)
            anc.append((anc[p] if p >= 0 else 0) | 1 << j)
        mask += anc
    T = sum(nodes)
    return dict(case=case, sizes=sizes, shared=shared, lens=lens, nodes=nodes, group=group,
                bt=bt.to(DEV), cache=_cache(pool, page, case["kv"], g),
                seq=torch.tensor(lens, dtype=torch.int32, device=DEV), cu_shared=_cu(sizes),
                shared_lens=torch.tensor(shared, dtype=torch.int32, device=DEV),
                cu=_cu(nodes), mask=torch.tensor(mask, device=DEV),
                q=torch.randn(T, case["heads"], LAT, generator=g, device=DEV).half() * 0.5)


def _tables_state(case, g):
    page, G, n = case["page"], case["groups"], case["requests"]
    R, ctx, new = G * n, case["ctx"], case["tokens"]
    # contexts from ctx down to a third of it; the first half of the shortest is the prompt
    lens = [ctx - (2 * ctx // 3) * r // max(R - 1, 1) for r in range(R)]
    counts = [new if new > 1 or r % 7 else 0 for r in range(R)]  # an idle request here and there
    width = -(-(ctx + new) // page) + 1
    share = min(lens) // 2 // page
    held = [-(-x // page) for x in lens]
    pool = sum(held) + sum(-(-(x + c) // page) - h for x, c, h in zip(lens, counts, held)) + 5
    order = torch.randperm(pool, generator=g, device=DEV).int()
    pages = torch.arange(width, device=DEV)
    h = torch.tensor(held, device=DEV)
    start = _cu(held)[:-1].long()
    bt = order[(start[:, None] + pages).clamp(max=pool - 1)]
    lead = torch.arange(R, device=DEV) // n * n  # the group's first request
    bt = torch.where(pages < share, bt[lead], bt)
    bt = torch.where(pages < h[:, None], bt, -1).int().contiguous()
    free = torch.full((pool,), -1, dtype=torch.int32, device=DEV)
    left = order[sum(held):]
    free[:left.numel()] = left
    return dict(case=case, bt=bt, seq=torch.tensor(lens, dtype=torch.int32, device=DEV),
                new=torch.tensor(counts, dtype=torch.int32, device=DEV), free=free,
                count=torch.tensor([left.numel()], dtype=torch.int32, device=DEV),
                old=torch.tensor(lens, dtype=torch.int32, device=DEV),
                cu_shared=_cu([n] * G), total=sum(counts) + 3)  # a padded batch


def _weight(case, g):
    w = torch.randn(case["n"], case["k"], generator=g, device=DEV, dtype=torch.float32)
    return w.mul_(case["k"] ** -0.5).to(DTYPES[case["dtype"]])


def _package():
    from __graft_entry__ import load_package

    return load_package()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "prefix":
        return _prefix_state(case, seed, g)
    if kind == "tables":
        return _tables_state(case, g)
    if kind == "expand":
        R, n, page = case["requests"], case["tokens"], case["page"]
        lens = [case["ctx"] - (case["ctx"] - n) * r // (2 * R) for r in range(R)]
        width = -(-case["ctx"] // page)
        bt = torch.randint(0, 1 << 24, (R, width), generator=g, device=DEV).int()
        return dict(case=case, bt=bt, seq=torch.tensor(lens, dtype=torch.int32, device=DEV),
                    cu=_cu([n] * R), total=R * n + 1)
    if kind == "weights":
        return dict(case=case, w=_weight(case, g))
    n, k, gs, dt = case["n"], case["k"], case["group"], DTYPES[case["dtype"]]
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    kg = -(-k // gs)
    s = (torch.rand(n, kg, generator=g, device=DEV) + 0.5).mul_(0.2 * k ** -0.5).to(dt)
    z = torch.randint(4, 12, (n, kg), generator=g, device=DEV, dtype=torch.uint8) \
        if case["zeros"] else None
    state = dict(case=case, x=torch.randn(case["m"], k, generator=g, device=DEV).to(dt))
    if own:
        state["w"] = _package().w4.w4_pack(codes, s, z, gs)
    state.update(codes=codes, s=s, z=z)
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _values(rows):
    """Rows of either cache as the fp16 values that reading them back gives, in fp32."""
    if rows.dtype != torch.uint8:
        return rows.float()
    n = rows.shape[0]
    v = rows[:, :VAL].contiguous().view(torch.float8_e4m3fn).float().view(n, 4, 128)
    v = v * rows[:, VAL:VAL + 16].contiguous().view(torch.float32)[:, :, None]
    return torch.cat([v.view(n, VAL).half(), rows[:, VAL + 16:].contiguous().view(torch.float16)],
                     1).float()


def _prefix(s):
    """Each group's rows against the shared keys in one product, each request's rows
    against its own keys padded to the longest, and the two joined."""
    H, page, R = s["q"].shape[1], s["case"]["page"], len(s["lens"])
    cu, cu_s, rows = s["cu"].long(), s["cu_shared"].tolist(), s["cache"].flatten(0, 1)
    bt, seq, T = s["bt"].long(), s["seq"].long(), s["q"].shape[0]
    q = s["q"].float().view(T * H, LAT)
    m = torch.full((T * H, 1), -math.inf, device=DEV)
    l, o = torch.zeros(T * H, 1, device=DEV), torch.zeros(T * H, VAL, device=DEV)
    tok = s["cu"].tolist()
    for g, P in enumerate(s["shared"]):
        if P == 0:
            continue
        a, b = tok[cu_s[g]] * H, tok[cu_s[g + 1]] * H
        p = torch.arange(P, device=DEV)
        K = _values(rows[bt[cu_s[g]][p // page] * page + p % page])
        S = (q[a:b] @ K.t()).mul_(SCALE)
        m[a:b] = S.amax(1, keepdim=True)
        S = S.sub_(m[a:b]).exp_()
        l[a:b] = S.sum(1, keepdim=True)
        o[a:b] = S @ K[:, :VAL]
    n = max(s["nodes"])
    base = s["shared_lens"].long()[torch.tensor(s["group"], device=DEV)]
    L = max(x - s["shared"][g] for x, g in zip(s["lens"], s["group"]))
    cnt = cu[1:] - cu[:-1]
    j = torch.arange(n, device=DEV)
    at = (cu[:-1, None] + j).clamp(max=T - 1)                             # [R, n]
    p = base[:, None] + torch.arange(L, device=DEV)                       # [R, L]
    row = torch.gather(bt, 1, (p // page).clamp(max=bt.shape[1] - 1)) * page + p % page
    K = _values(rows[row.clamp(0, rows.shape[0] - 1).view(-1)]).view(R, L, LAT)
    d = p - (seq - cnt)[:, None]                                          # drafted index
    bit = (s["mask"][at][:, :, None] >> d.clamp(0, 63)[:, None, :]) & 1
    see = (((d < 0)[:, None, :]) | (bit != 0)) & (p < seq[:, None])[:, None, :]
    see = see[:, :, None, :].expand(R, n, H, L).reshape(R, n * H, L)
    qs = q.view(T, H, LAT)[at].view(R, n * H, LAT)
    S = torch.bmm(qs, K.transpose(1, 2).contiguous()).mul_(SCALE).masked_fill_(~see, -math.inf)
    live = (j < cnt[:, None]).view(-1)

    def real(x):  # [R, n * H, c] -> [T * H, c]
        return x.view(R * n, H, -1)[live].view(T * H, -1)

    m2 = torch.maximum(real(S.amax(2, keepdim=True)), m).clamp_min(-1e30)
    pad = torch.zeros(R * n, H, device=DEV)
    pad[live] = m2.view(T, H)
    S = S.sub_(pad.view(R, n * H, 1)).exp_()
    f = (m - m2).exp()
    l = l * f + real(S.sum(2, keepdim=True))
    o = o * f + real(torch.bmm(S, K[:, :, :VAL].contiguous()))
    lse = (m2 + l.log()).view(T, H)
    return (o / l.clamp_min(1e-30)).view(T, H, VAL).half(), lse


def _pages(n, page):
    return (n + page - 1) // page


def _tables(s):
    """Prefix sums over the requests, then every new page and token by its place."""
    page, bt, W, R = s["case"]["page"], s["bt"], s["bt"].shape[1], s["bt"].shape[0]
    seq, new, T = s["seq"].long(), s["new"].long(), s["total"]
    have, want = _pages(seq, page), _pages(seq + new, page)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    ok = (want <= W) & (cu[1:] <= T)
    need = torch.where(ok, want - have, 0)
    upto = need.cumsum(0)
    granted = ok & ((need == 0) | (upto <= s["count"]))
    taken = torch.where(granted, need, 0)
    k = torch.arange(W, device=DEV)
    fresh = (k >= have[:, None]) & (k < (have + taken)[:, None])
    place = s["count"].long() - 1 - (upto - need)[:, None] - (k - have[:, None])
    bt.copy_(torch.where(fresh, s["free"][place.clamp(0, s["free"].numel() - 1)], bt))
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=R - 1)
    live = (t < cu[-1]) & granted[r]
    pos = torch.where(live, seq[r] + t - cu[r], -1)
    slot = bt[r, (pos // page).clamp(0, W - 1)].long() * page + pos % page
    slot = torch.where(live, slot, -1)
    s["seq"].copy_(torch.where(granted, seq + new, seq))
    s["count"].sub_(taken.sum().int())
    after = bt.clone(), s["seq"].clone(), s["count"].clone()
    cs = s["cu_shared"].long()
    lead = cs[:-1][torch.searchsorted(cs[1:], torch.arange(R, device=DEV), right=True)]
    same = (bt == bt[lead]).int().cumprod(1).sum(1) * page
    common = torch.minimum(same, s["seq"].long()).view(cs.numel() - 1, -1).amin(1)
    # back to the old lengths
    seq2, old = s["seq"].long(), s["old"].long()
    keep, had = _pages(old, page), _pages(seq2, page)
    gone = (k >= keep[:, None]) & (k < had[:, None])
    rank = gone.view(-1).long().cumsum(0) - 1
    total = gone.sum()
    at = (s["count"].long() + total - 1 - rank)[gone.view(-1)]
    s["free"][at] = bt.view(-1)[gone.view(-1)]
    bt.masked_fill_(gone, -1)
    s["seq"].copy_(old)
    s["count"].add_(total.int())
    return dict(slots=slot.int(), positions=pos.int(), cu=cu.clamp(max=T).int(), granted=granted,
                tables=after[0], lens=after[1], left=after[2], common=common.int(),
                tables_back=bt, lens_back=s["seq"], free=s["free"], left_back=s["count"])


def _expand(s):
    cu, T, R = s["cu"].long(), s["total"], s["bt"].shape[0]
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True)
    live, r = r < R, r.clamp(max=R - 1)
    lens = s["seq"].long()[r] - (cu[r + 1] - cu[r]) + t - cu[r] + 1
    return torch.where(live[:, None], s["bt"][r], -1), torch.where(live, lens, 0).int()


def _spread(x, gs, k):
    """[n, groups] -> [n, k]: each group's value for its columns."""
    return x.repeat_interleave(gs, 1)[:, :k]


def _linear(s):
    c = s["case"]
    z = s["z"].float() if s["z"] is not None else torch.full_like(s["s"], 8, dtype=torch.float32)
    w = s["codes"].float().sub_(_spread(z, c["group"], c["k"])) \
        .mul_(_spread(s["s"].float(), c["group"], c["k"]))
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


def _quantised(w, gs, zeros):
    """Codes, scales and zero points; the scales in 64 bits up to their rounding, as a
    last bit of a scale moves codes."""
    n, k = w.shape
    kg = -(-k // gs)
    v = torch.nn.functional.pad(w.float(), (0, kg * gs - k)).view(n, kg, gs)
    lo, hi = v.amin(2).clamp(max=0).double(), v.amax(2).clamp(min=0).double()
    s = (hi - lo) / 15 if zeros else torch.maximum(hi / 7, -lo / 8)
    least = 2.0 ** -24 if w.dtype == torch.float16 else 2.0 ** -126
    s = s.float().to(w.dtype).float().clamp_min(least)
    z = torch.round(-lo.float() / s).clamp(0, 15) if zeros else torch.full_like(s, 8)
    c = (torch.round(v / s[:, :, None]) + z[:, :, None]).clamp(0, 15)
    return c, s, z


def _weights(s):
    c, w = s["case"], s["w"]
    code, sc, z = _quantised(w, c["group"], c["zeros"])
    v = ((code - z[:, :, None]) * sc[:, :, None]).view(c["n"], -1)[:, :c["k"]]
    return v.to(w.dtype).contiguous()


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return dict(prefix=_prefix, tables=_tables, expand=_expand, linear=_linear,
                    weights=_weights)[kind](s)
    pkg = _package()
    if kind == "prefix":
        more = {} if c["nodes"] == 1 else dict(cu_seqlens_q=s["cu"], tree_mask=s["mask"])
        return pkg.mla_prefix.shared_prefix_attention(
            s["q"], s["cache"], s["bt"], s["seq"], s["cu_shared"], s["shared_lens"], SCALE, **more)
    if kind == "tables":
        slots, pos, cu, granted = pkg.paging.extend_tables(
            s["bt"], s["seq"], s["new"], s["free"], s["count"], c["page"], s["total"])
        after = s["bt"].clone(), s["seq"].clone(), s["count"].clone()
        common = pkg.paging.shared_lengths(s["bt"], s["seq"], s["cu_shared"], c["page"])
        pkg.paging.truncate_tables(s["bt"], s["seq"], s["old"], s["free"], s["count"], c["page"])
        return dict(slots=slots, positions=pos, cu=cu, granted=granted, tables=after[0],
                    lens=after[1], left=after[2], common=common, tables_back=s["bt"],
                    lens_back=s["seq"], free=s["free"], left_back=s["count"])
    if kind == "expand":
        return pkg.paging.token_tables(s["bt"], s["seq"], s["cu"], s["total"])
    if kind == "linear":
        return pkg.w4.w4_linear(s["x"], s["w"])
    return pkg.w4.w4_dequant(pkg.w4.w4_quantize(s["w"], c["group"], symmetric=not c["zeros"]))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "prefix":
        kv, H = 656 if case["kv"] == "fp8" else 1152, case["heads"]
        sizes, shared, own_len, nodes = _shape(case)
        shared = [p // case["page"] * case["page"] for p in shared]
        group = [s for s, n in enumerate(sizes) for _ in range(n)]
        rows = [n * H for n in nodes]
        flops = sum(m * (shared[s] + n) for m, s, n in zip(rows, group, own_len)) * 2 * (LAT + VAL)
        return dict(bytes=sum(rows) * (2 * LAT + 2 * VAL + 4) + (sum(shared) + sum(own_len)) * kv,
                    flops=flops)
    if kind == "tables":
        R, page = case["groups"] * case["requests"], case["page"]
        T = R * case["tokens"]
        lens = [case["ctx"] - (2 * case["ctx"] // 3) * r // max(R - 1, 1) for r in range(R)]
        # lengths, slots, positions; the entries compared; the tables that are returned
        width = -(-(case["ctx"] + case["tokens"]) // page) + 1
        same = min(lens) // 2 // page
        return dict(bytes=R * 6 * 4 + T * 8 + R * same * 4 + R * width * 8, flops=T)
    if kind == "expand":
        T = case["requests"] * case["tokens"]
        width = -(-case["ctx"] // case["page"])
        return dict(bytes=(T + case["requests"]) * width * 4 + T * 4, flops=T)
    n, k = case["n"], case["k"]
    packed = n * k // 2 + n * -(-k // case["group"]) * (3 if case["zeros"] else 2)
    if kind == "linear":
        m = case["m"]
        return dict(bytes=packed + 2 * m * (n + k), flops=2 * m * n * k)
    return dict(bytes=4 * n * k + 2 * packed, flops=4 * n * k)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _row64(cache, page, entries, p):
    rows = cache.flatten(0, 1)[entries.long()[p // page] * page + p % page]
    if cache.dtype != torch.uint8:
        return rows.double()
    b = rows[:, :VAL].long()
    e, f = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * torch.exp2(e.double() - 10))
    val = torch.where(b >= 128, -mag, mag)
    sc = rows[:, VAL:VAL + 16].contiguous().view(torch.float32).double()
    v = val * sc.repeat_interleave(128, 1)
    return torch.cat([v, rows[:, VAL + 16:].contiguous().view(torch.float16).double()],
                     1).half().double()


def _exact_prefix(case, seed):
    s = prepare(case, seed)
    T, H = s["q"].shape[:2]
    if T * H * max(s["lens"]) > 3e8:  # a slice of the heads would not be the output
        return None
    out, lses, at = [], [], 0
    for r, n in enumerate(s["lens"]):
        k = s["nodes"][r]
        K = _row64(s["cache"], case["page"], s["bt"][r], torch.arange(n, device=DEV))
        sc = (s["q"][at:at + k].double().reshape(k * H, LAT) @ K.T * SCALE).view(k, H, n)
        for j in range(k):
            m = int(s["mask"][at + j])
            for i in range(k):
                if not (m >> i) & 1:
                    sc[j, :, n - k + i] = -math.inf
        lse = torch.logsumexp(sc, 2)
        P = torch.exp(sc - lse[:, :, None])
        out.append((P.view(k * H, n) @ K[:, :VAL]).view(k, H, VAL))
        lses.append(lse)
        at += k
    return torch.cat(out), torch.cat(lses)


def _exact_tables(case, seed):
    """Request by request, page by page, in whole numbers."""
    s, page = prepare(case, seed), case["page"]
    bt, seq, new = s["bt"].tolist(), s["seq"].tolist(), s["new"].tolist()
    free, count = s["free"].tolist(), int(s["count"])
    W, T = len(bt[0]), s["total"]
    slots, pos, cu, granted, out_of = [], [], [0], [], False
    old_bt = [list(x) for x in bt]
    wanted = 0
    for r, (n, k) in enumerate(zip(seq, new)):
        cu.append(cu[-1] + k)
        need = -(-(n + k) // page) - -(-n // page)
        fits = -(-(n + k) // page) <= W and cu[-1] <= T
        if fits:
            wanted += need
            out_of = wanted > int(s["count"])
        ok = fits and (need == 0 or not out_of)
        granted.append(ok)
        if ok:
            for i in range(-(-n // page), -(-(n + k) // page)):
                count -= 1
                bt[r][i] = free[count]
            seq[r] = n + k
        for i in range(k):
            pos.append(n + i if ok else -1)
            slots.append(bt[r][(n + i) // page] * page + (n + i) % page if ok else -1)
    pad = T - len(slots)
    common, at = [], 0
    for _ in range(case["groups"]):
        a = bt[at]
        least = min(seq[at:at + case["requests"]])
        for b in bt[at:at + case["requests"]]:
            same = next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), W)
            least = min(least, same * page)
        common.append(least)
        at += case["requests"]

    def t(x):
        return torch.tensor(x, dtype=torch.int32)
    # truncating gives every page back to its place
    return dict(slots=t(slots + [-1] * pad), positions=t(pos + [-1] * pad), cu=t(cu),
                granted=torch.tensor(granted), tables=t(bt), lens=t(seq), left=t([count]),
                common=t(common), tables_back=t(old_bt), lens_back=s["old"],
                free=t(free), left_back=s["count"])


def exact(case, seed):
    kind = case["kind"]
    if kind == "prefix":
        return _exact_prefix(case, seed)
    if kind == "tables":
        return _exact_tables(case, seed)
    s = prepare(case, seed)
    if kind == "expand":
        n, R = case["tokens"], case["requests"]
        rows = [s["bt"][r].expand(n, -1) for r in range(R)] + [torch.full_like(s["bt"][:1], -1)]
        lens = [x - n + 1 + i for x in s["seq"].tolist() for i in range(n)]
        return torch.cat(rows), torch.tensor(lens + [0], dtype=torch.int32)
    gs, k, n = case["group"], case["k"], case["n"]
    if kind == "linear":
        y = torch.zeros(case["m"], n, dtype=torch.float64, device=DEV)
        for j, lo in enumerate(range(0, k, gs)):
            c = s["codes"][:, lo:lo + gs].double()
            c -= s["z"][:, j:j + 1].double() if s["z"] is not None else 8.0
            y += s["x"][:, lo:lo + gs].double() @ c.T * s["s"][:, j].double()
        return y
    out = torch.empty(n, k, dtype=torch.float64, device=DEV)
    w, least = s["w"], 2.0 ** -24 if case["dtype"] == "fp16" else 2.0 ** -126
    for lo in range(0, k, gs):
        v = w[:, lo:lo + gs].double()
        a, b = v.amin(1).clamp(max=0), v.amax(1).clamp(min=0)
        sc = (b - a) / 15 if case["zeros"] else torch.maximum(b / 7, -a / 8)
        sc = sc.float().to(w.dtype).double().clamp_min(least)[:, None]
        z = torch.round(-a[:, None] / sc).clamp(0, 15) if case["zeros"] else 8.0
        out[:, lo:lo + gs] = (torch.clamp(torch.round(v / sc) + z, 0, 15) - z) * sc
    return out
