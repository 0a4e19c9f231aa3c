"""The operators of a batch that shares a long prefix, each in a plain form and as the package's calls.

  plan     block tables and slot maps from request lengths (plan_pages)
  append   rotary of the new tokens, keys and values written into their pages (append_pages)
  attend   attention over [shared prefix | the sequence's own pages] (shared_prefix_attention)

A case is a dict of sizes; `listed()` names twelve, `draw()` gives more of the same ranges. Lengths of the
sequences are a fixed ragged spread, dealt to the sequences by the seed, so every seed has outputs of one shape.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 500000.0


def listed():
    return [
        # one decode step of a batch: a token a sequence, a page now and then; latency is all that counts
        dict(name="plan_decode_64", op="plan", n_seq=64, page=16, ctx=2048, new=1, base=8192),
        # the suffixes of a batch go in at once: long ragged prompts into an empty pool
        dict(name="plan_prompts_256", op="plan", n_seq=256, page=64, ctx=0, new=1024, base=32768),
        # a decode step's tokens of one layer
        dict(name="append_decode_64", op="append", dtype="f16", n_seq=64, hq=32, hk=8, d=128, page=64, ctx=512, new=1,
             base=131072),
        # the questions of a batch, one layer
        dict(name="append_chunk_bf16", op="append", dtype="bf16", n_seq=32, hq=32, hk=8, d=128, page=64, ctx=100,
             new=512, base=32768),
        # the same in 32 bits, small heads and odd lengths
        dict(name="append_chunk_f32", op="append", dtype="f32", n_seq=7, hq=8, hk=2, d=64, page=16, ctx=33, new=301,
             base=4097),
        # a few users of a short prompt: launches and latency
        dict(name="attend_decode_4", op="attend", dtype="f16", n_seq=4, hq=32, hk=8, d=128, prefix=1000, page=16,
             ctx=300, new=1, mask=False),
        # an ordinary batch over an 8k document
        dict(name="attend_decode_32", op="attend", dtype="f16", n_seq=32, hq=32, hk=8, d=128, prefix=8192, page=64,
             ctx=512, new=1, mask=False),
        # long answers: the sequences' own pages weigh as much as the document
        dict(name="attend_decode_64_32k", op="attend", dtype="bf16", n_seq=64, hq=32, hk=8, d=128, prefix=32768,
             page=64, ctx=2048, new=1, mask=False),
        # the longest document
        dict(name="attend_decode_64_128k", op="attend", dtype="bf16", n_seq=64, hq=32, hk=8, d=128, prefix=131072,
             page=128, ctx=512, new=1, mask=False),
        # the questions of a batch read the document: many ragged query rows, causal among themselves
        dict(name="attend_chunk_8", op="attend", dtype="bf16", n_seq=8, hq=32, hk=8, d=128, prefix=16384, page=32,
             ctx=0, new=257, mask=False),
        # drafts of a few tokens are checked against a document of which some tokens were dropped; wide groups
        dict(name="attend_draft_24_d64", op="attend", dtype="f16", n_seq=24, hq=16, hk=2, d=64, prefix=5001, page=16,
             ctx=777, new=5, mask=True),
        # 32-bit layers
        dict(name="attend_decode_8_f32", op="attend", dtype="f32", n_seq=8, hq=8, hk=2, d=128, prefix=4097, page=16,
             ctx=200, new=1, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (8, 2, 128), (16, 2, 128), (4, 4, 64), (16, 2, 64), (8, 1, 64), (12, 6, 128)]


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        n_seq = _log(rng, 1, 512)
        return dict(op=op, n_seq=n_seq, page=page, ctx=rng.choice([0, _log(rng, 1, 4096)]),
                    new=rng.choice([1, _log(rng, 2, max(2, min(2048, 131072 // n_seq)))]), base=_log(rng, 1, 131072))
    hq, hk, d = rng.choice(HEADS)
    dtype = rng.choice(["f32", "f16", "bf16", "f16", "bf16"])
    if op == "append":
        n_seq = _log(rng, 1, 128)
        return dict(op=op, dtype=dtype, n_seq=n_seq, hq=hq, hk=hk, d=d, page=page, ctx=rng.choice([0, _log(rng, 1, 512)]),
                    new=rng.choice([1, _log(rng, 2, max(2, min(512, 8192 // n_seq)))]), base=_log(rng, 1, 131072))
    n_seq = _log(rng, 1, 64)
    new = rng.choice([1, 1, _log(rng, 2, max(2, min(256, 1024 // n_seq)))])
    most = 64 * 131072 // 4 if dtype == "f32" else 64 * 131072
    prefix = _log(rng, 1, min(131072, most // (n_seq * new)))
    return dict(op=op, dtype=dtype, n_seq=n_seq, hq=hq, hk=hk, d=d, prefix=prefix, page=page,
                ctx=rng.choice([0, _log(rng, 1, 1024)]), new=new, mask=rng.random() < 0.25)


def _spread(most, n, least):
    """n ragged lengths between `least` and `most`, the last one `most`; the same for every seed."""
    if most <= least:
        return np.full(n, most, np.int64)
    f = (np.arange(1, n + 1) * 0.6180339887498949) % 1.0
    v = least + np.floor(f * (most - least + 1)).astype(np.int64)
    v[-1] = most
    return v


def _lengths(case):
    """(tokens in the pages before the call, new tokens) of every sequence, undealt."""
    return _spread(case["ctx"], case["n_seq"], 0), _spread(case["new"], case["n_seq"], 1)


def _blocks(n, page):
    return -(-n // page)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    r = np.random.RandomState(int(seed) % (1 << 32))
    ctx, new = _lengths(case)
    ctx, new = r.permutation(ctx), r.permutation(new)
    B, ps, total = case["n_seq"], case["page"], int(new.sum())
    max_blocks = _blocks(case["ctx"] + case["new"], ps)
    n_pages = int((_blocks(ctx, ps) + _blocks(new, ps)).sum()) + 5  # a pool nearly used up, however the lengths are dealt
    order = r.permutation(n_pages).astype(np.int32)
    # pages held before the call come from the front of `order`, the rest is the free stack
    table = np.full((B, max_blocks), -1, np.int32)
    at = 0
    for b in range(B):
        n = _blocks(int(ctx[b]), ps)
        table[b, :n] = order[at:at + n]
        at += n
    free = np.zeros(n_pages, np.int32)
    n_free = n_pages - at
    free[:n_free] = order[at:]

    def dev(x, t):
        return torch.from_numpy(np.ascontiguousarray(x)).to(device="cuda", dtype=t)

    s = dict(case=dict(case), total=total, page=ps)
    if case["op"] == "plan":
        s.update(lens=dev(ctx, torch.int32), new_lens=dev(new, torch.int32), table=dev(table, torch.int32),
                 free=dev(free, torch.int32), n_free=torch.full((1,), n_free, dtype=torch.int32, device="cuda"),
                 base=case["base"],
                 out=dict(cu_new=torch.empty(B + 1, dtype=torch.int32, device="cuda"),
                          slots=torch.empty(total, dtype=torch.int64, device="cuda"),
                          seq_ids=torch.empty(total, dtype=torch.int32, device="cuda"),
                          positions=torch.empty(total, dtype=torch.int64, device="cuda"),
                          lens=torch.empty(B, dtype=torch.int32, device="cuda"),
                          n_free=torch.empty(1, dtype=torch.int32, device="cuda"),
                          status=torch.zeros(1, dtype=torch.int32, device="cuda")))
        return s
    # the step's pages are planned: the new tokens' blocks come off the stack
    for b in range(B):
        for j in range(_blocks(int(ctx[b]), ps), _blocks(int(ctx[b] + new[b]), ps)):
            n_free -= 1
            table[b, j] = free[n_free]
    cu = np.concatenate([[0], np.cumsum(new)])
    t, hq, hk, d = TYPES[case["dtype"]], case["hq"], case["hk"], case["d"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(t)

    s.update(k_pages=normal(n_pages, hk, ps, d), v_pages=normal(n_pages, hk, ps, d))
    if case["op"] == "append":
        seq = np.repeat(np.arange(B), new)
        p = ctx[seq] + np.arange(total) - cu[seq]
        s.update(q=normal(total, hq, d), k=normal(total, hk, d), v=normal(total, hk, d),
                 slots=dev(table[seq, p // ps].astype(np.int64) * ps + p % ps, torch.int64),
                 positions=dev(case["base"] + p, torch.int64),
                 inv_freq=dev(1.0 / THETA ** (np.arange(0, d, 2) / d), torch.float32))
        return s
    P = case["prefix"]
    # the prefix as a model's projection leaves it: (tokens, heads, d), seen as (heads, tokens, d)
    s.update(q=normal(total, hq, d), prefix_k=normal(P, hk, d).transpose(0, 1), prefix_v=normal(P, hk, d).transpose(0, 1),
             table=dev(table, torch.int32), lens=dev(ctx + new, torch.int32), cu_new=dev(cu, torch.int32),
             scaling=1.0 / math.sqrt(d),
             mask=(torch.rand(P, generator=g, device="cuda") < 0.85).to(torch.uint8) if case["mask"] else None)
    return s


# ---------------------------------------------------------------------------- plain forms
def _plan_plain(s):
    lens, new, table, o = s["lens"].long(), s["new_lens"].long(), s["table"], s["out"]
    ps, total, dev = s["page"], s["total"], lens.device
    have = (lens + ps - 1) // ps
    need = (lens + new + ps - 1) // ps - have
    first = torch.cumsum(need, 0) - need
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(new, 0)])
    n_free = s["n_free"].long()
    fits = (need.sum() <= n_free) & (have + need <= table.shape[1]).all() & (cu[-1] <= total)
    new = torch.where(fits, new, 0)
    need = torch.where(fits, need, 0)
    cu = torch.where(fits, cu, 0)
    j = torch.arange(table.shape[1], device=dev)[None]
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None])
    at = (n_free - 1 - first[:, None] - (j - have[:, None])).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at], table))
    t = torch.arange(total, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = seq < lens.numel()
    b = seq.clamp(max=lens.numel() - 1)
    p = torch.where(live, lens[b] + t - cu[b], 0)
    slot = table[b, p // ps].long() * ps + p % ps
    return dict(cu_new=cu.int(), slots=torch.where(live, slot, -1), seq_ids=torch.where(live, b, -1).int(),
                positions=torch.where(live, s["base"] + p, -1), lens=(lens + new).int(),
                n_free=(n_free - need.sum()).int(), table=table)


def _rotate(x, cos, sin):
    x = x.float()
    h = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def _append_plain(s):
    # the angle of a far position needs more than 32 bits
    a = s["positions"].double()[:, None] * s["inv_freq"].double()[None]
    a = torch.cat([a, a], -1)[:, None]
    cos, sin = torch.cos(a).float(), torch.sin(a).float()
    page, row = s["slots"] // s["page"], s["slots"] % s["page"]
    s["k_pages"][page, :, row] = _rotate(s["k"], cos, sin).to(s["k"].dtype)
    s["v_pages"][page, :, row] = s["v"]
    return dict(q=_rotate(s["q"], cos, sin).to(s["q"].dtype), k_pages=s["k_pages"], v_pages=s["v_pages"])


def _attend_plain(s):
    c, q, dev = s["case"], s["q"].float(), s["q"].device
    B, N, hk, ps = c["n_seq"], c["new"], c["hk"], s["page"]
    T, hq, d = q.shape
    cu, lens = s["cu_new"].long(), s["lens"].long()
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    i = t - cu[seq]
    # queries of sequence b in row b of a padded block, heads grouped by the key head they read
    qb = torch.zeros((B, N, hk, hq // hk, d), device=dev)
    qb[seq, i] = q.view(T, hk, hq // hk, d) * s["scaling"]
    qb = qb.permute(0, 2, 1, 3, 4).reshape(B, hk, N * (hq // hk), d)
    # prefix: one product per key head for the whole batch
    pk, pv = s["prefix_k"].float(), s["prefix_v"].float()
    P = pk.shape[1]
    qa = qb.transpose(0, 1).reshape(hk, -1, d)
    sp = (qa @ pk.transpose(1, 2)).view(hk, B, -1, P)
    if s["mask"] is not None:
        sp = sp.masked_fill(s["mask"][None, None, None] == 0, -math.inf)
    # the sequences' own pages, gathered; token j is seen by query i where j <= len - new + i
    own_k = s["k_pages"][s["table"].long().clamp(min=0)].float().transpose(1, 2).reshape(B, hk, -1, d)
    own_v = s["v_pages"][s["table"].long().clamp(min=0)].float().transpose(1, 2).reshape(B, hk, -1, d)
    L = own_k.shape[2]
    ss = (qb @ own_k.transpose(2, 3)).view(B, hk, N, -1, L)
    last = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(N, device=dev)[None]
    ss = ss.masked_fill(torch.arange(L, device=dev) > last[:, None, :, None, None], -math.inf)
    ss = ss.reshape(B, hk, -1, L).transpose(0, 1)
    m = torch.maximum(sp.amax(-1), ss.amax(-1)).clamp(min=-1e30)[..., None]
    sp, ss = torch.exp(sp - m), torch.exp(ss - m)
    o = (sp.reshape(hk, -1, P) @ pv).view(hk, B, -1, d) + ss @ own_v.transpose(0, 1)
    o = o / (sp.sum(-1) + ss.sum(-1))[..., None].clamp(min=1e-30)
    o = o.view(hk, B, N, hq // hk, d).permute(1, 2, 0, 3, 4)
    return o[seq, i].reshape(T, hq, d).to(s["q"].dtype)


# ---------------------------------------------------------------------------- the package's calls
def _own(s):
    import hotcold_kv_cache_b200 as hc
    op = s["case"]["op"]
    if op == "plan":
        p = hc.plan_pages(s["lens"], s["new_lens"], s["table"], s["free"], s["n_free"], s["page"], s["total"],
                          base_pos=s["base"], out=hc.PagePlan(**s["out"]))
        return dict(cu_new=p.cu_new, slots=p.slots, seq_ids=p.seq_ids, positions=p.positions, lens=p.lens,
                    n_free=p.n_free, table=s["table"])
    if op == "append":
        q = hc.append_pages(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["k_pages"], s["v_pages"],
                            inv_freq=s["inv_freq"])
        return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])
    return hc.shared_prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["k_pages"], s["v_pages"], s["table"],
                                      s["lens"], s["cu_new"], s["scaling"], prefix_mask=s["mask"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan_plain, "append": _append_plain, "attend": _attend_plain}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------- the work, and 64-bit values
def work(case):
    ctx, new = _lengths(case)
    T = int(new.sum())
    if case["op"] == "plan":
        fresh = int((_blocks(ctx + new, case["page"]) - _blocks(ctx, case["page"])).sum())
        return {"bytes": 16 * case["n_seq"] + 20 * T + 8 * fresh, "flops": 0}
    es, hq, hk, d = SIZE[case["dtype"]], case["hq"], case["hk"], case["d"]
    if case["op"] == "append":
        return {"bytes": 2 * T * (hq + 2 * hk) * d * es + 16 * T, "flops": 3 * T * (hq + hk) * d}
    # the deal of lengths to sequences moves this by little: the mean over deals
    seen = float(np.mean(ctx)) * T + float((new * (new + 1) / 2).sum())
    keys = case["prefix"] + int(ctx.sum()) + T
    return {"bytes": keys * hk * d * 2 * es + 2 * T * hq * d * es, "flops": 4 * hq * d * (T * case["prefix"] + seen)}


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers: equal or not
    s = prepare(case, seed)
    if case["op"] == "append":
        d = case["d"]
        w = s["inv_freq"].to(torch.float64)
        ang = torch.outer(s["positions"].to(torch.float64), w)
        z = torch.polar(torch.ones_like(ang), ang)[:, None, :]

        def turn(x):
            x = x.to(torch.float64)
            y = torch.complex(x[..., :d // 2], x[..., d // 2:]) * z
            return torch.cat([y.real, y.imag], -1)

        kp, vp = s["k_pages"].to(torch.float64), s["v_pages"].to(torch.float64)
        ps = case["page"]
        flat_k = kp.transpose(1, 2).reshape(-1, case["hk"], d)
        flat_v = vp.transpose(1, 2).reshape(-1, case["hk"], d)
        flat_k.index_copy_(0, s["slots"], turn(s["k"]))
        flat_v.index_copy_(0, s["slots"], s["v"].to(torch.float64))
        back = (kp.shape[0], ps, case["hk"], d)
        return dict(q=turn(s["q"]), k_pages=flat_k.view(back).transpose(1, 2), v_pages=flat_v.view(back).transpose(1, 2))
    hq, hk = case["hq"], case["hk"]
    G = hq // hk
    q = s["q"].to(torch.float64)
    out = torch.zeros_like(q)
    cu, lens, table = s["cu_new"].tolist(), s["lens"].tolist(), s["table"].tolist()
    keep = None if s["mask"] is None else s["mask"].bool()
    step = max(1, (1 << 28) // max(1, case["prefix"]) // G)
    for h in range(hk):
        pk, pv = s["prefix_k"][h].to(torch.float64), s["prefix_v"][h].to(torch.float64)
        if keep is not None:
            pk, pv = pk[keep], pv[keep]
        for b in range(case["n_seq"]):
            n, length = cu[b + 1] - cu[b], lens[b]
            pages = table[b][:-(-length // case["page"])]
            sk = s["k_pages"][pages, h].reshape(-1, case["d"])[:length].to(torch.float64)
            sv = s["v_pages"][pages, h].reshape(-1, case["d"])[:length].to(torch.float64)
            for i0 in range(0, n, step):
                i1 = min(n, i0 + step)
                x = q[cu[b] + i0:cu[b] + i1, h * G:(h + 1) * G]
                a = torch.einsum("igd,pd->igp", x, torch.cat([pk, sk])) * s["scaling"]
                hidden = torch.arange(length, device=q.device)[None] > torch.arange(length - n + i0, length - n + i1,
                                                                                    device=q.device)[:, None]
                a[:, :, pk.shape[0]:].masked_fill_(hidden[:, None], -math.inf)
                out[cu[b] + i0:cu[b] + i1, h * G:(h + 1) * G] = torch.einsum(
                    "igp,pd->igd", torch.softmax(a, -1), torch.cat([pv, sv]))
    return out
