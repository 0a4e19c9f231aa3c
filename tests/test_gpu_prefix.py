"""The shared-prefix batch operators on the GPU against their plain 64-bit forms: plan_pages, release_pages,
append_pages, shared_prefix_attention, alone and as a run of steps."""

import math

import numpy as np
import pytest
import torch

import prefix_ref as R
from hotcold_kv_cache_b200 import _lib

pytestmark = pytest.mark.gpu

CAPACITY, INDEX = _lib.HC_DEV_CAPACITY, _lib.HC_DEV_INDEX
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(x, t):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device="cuda", dtype=t)


def spare_out(n_seq, n_tokens):
    import hotcold_kv_cache_b200 as hc
    i32, i64 = torch.int32, torch.int64
    z = dict(device="cuda")
    return hc.PagePlan(torch.full((n_seq + 1,), -7, dtype=i32, **z), torch.full((n_tokens,), -7, dtype=i64, **z),
                       torch.full((n_tokens,), -7, dtype=i32, **z), torch.full((n_tokens,), -7, dtype=i64, **z),
                       torch.full((n_seq,), -7, dtype=i32, **z), torch.full((1,), -7, dtype=i32, **z),
                       torch.zeros(1, dtype=i32, **z))


def make_table(rng, ctx, ps, max_blocks, extra):
    """(table, free stack, n_free) of sequences that hold ctx tokens, pages in random order."""
    held = [-(-int(c) // ps) for c in ctx]
    n_pages = sum(held) + extra
    order = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(ctx), max_blocks), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    free = np.full(n_pages, -1, np.int32)
    free[:n_pages - at] = order[at:]
    return table, free, n_pages - at


# ------------------------------------------------------------------------------------------------ plan and release
@pytest.mark.parametrize("n_seq,ps,ctx,new,pad", [
    (1, 16, 0, 1, 0), (1, 16, 15, 2, 3), (1, 256, 256, 1, 0), (3, 16, 40, 0, 2), (64, 16, 2048, 1, 0),
    (5, 32, 0, 70, 1), (33, 64, 500, 300, 0), (513, 128, 700, 3, 100), (4096, 16, 30, 2, 5), (7, 16, 0, 9000, 11)])
@pytest.mark.parametrize("commit", [False, True])
def test_plan(n_seq, ps, ctx, new, pad, commit):
    import hotcold_kv_cache_b200 as hc
    rng = np.random.default_rng(n_seq * 1000 + ps + new)
    c, a = rng.integers(0, ctx + 1, n_seq), rng.integers(0, new + 1, n_seq)
    c[0], a[0] = ctx, new
    max_blocks = -(-(ctx + new) // ps) or 1
    fresh = int(sum(-(-int(x + y) // ps) - -(-int(x) // ps) for x, y in zip(c, a)))
    table, free, n_free = make_table(rng, c, ps, max_blocks, fresh + 1)
    total = int(a.sum()) + pad
    want = R.plan(c, a, table, free, n_free, ps, total, 8192)
    g = dict(lens=dev(c, torch.int32), table=dev(table, torch.int32), n_free=dev([n_free], torch.int32))
    out = None if commit else spare_out(n_seq, total)
    p = hc.plan_pages(g["lens"], dev(a, torch.int32), g["table"], dev(free, torch.int32), g["n_free"], ps, total,
                      base_pos=8192, out=out)
    for name in ("cu_new", "slots", "seq_ids", "positions", "lens"):
        assert np.array_equal(getattr(p, name).cpu().numpy(), want[name]), name
    assert int(p.n_free) == want["n_free"] and int(p.status) == 0
    assert np.array_equal(g["table"].cpu().numpy(), want["table"])
    if commit:
        assert p.lens is g["lens"] and p.n_free is g["n_free"]
    else:
        assert np.array_equal(g["lens"].cpu().numpy(), c) and int(g["n_free"]) == n_free


@pytest.mark.parametrize("n_seq,new", [(3, 5), (300, 400)])
def test_plan_over_its_own_inputs(n_seq, new):
    """The lengths after the step may go where the new lengths came from, for one CTA's step and for many."""
    import hotcold_kv_cache_b200 as hc
    rng = np.random.default_rng(n_seq)
    c, a = rng.integers(0, 50, n_seq), rng.integers(0, new + 1, n_seq)
    table, free, n_free = make_table(rng, c, 16, 40, 30 * n_seq)
    want = R.plan(c, a, table, free, n_free, 16, int(a.sum()), 0)
    add = dev(a, torch.int32)
    out = spare_out(n_seq, int(a.sum()))._replace(lens=add)
    nf = dev([n_free], torch.int32)
    p = hc.plan_pages(dev(c, torch.int32), add, dev(table, torch.int32), dev(free, torch.int32), nf, 16, int(a.sum()), out=out)
    for name in ("cu_new", "slots", "seq_ids", "positions", "lens"):
        assert np.array_equal(getattr(p, name).cpu().numpy(), want[name]), name
    assert int(p.n_free) == want["n_free"] and int(nf) == n_free and int(p.status) == 0


@pytest.mark.parametrize("what,bit", [("pages", CAPACITY), ("rows", CAPACITY), ("table", CAPACITY),
                                      ("negative_new", INDEX), ("negative_len", INDEX), ("long_len", INDEX),
                                      ("n_free", INDEX)])
def test_plan_refuses_the_whole_step(what, bit):
    import hotcold_kv_cache_b200 as hc
    rng = np.random.default_rng(3)
    ps, c, a = 16, np.array([5, 0, 33]), np.array([20, 3, 17])
    table, free, n_free = make_table(rng, c, ps, 4, 6)
    total = 40
    if what == "pages":
        n_free = 2
    if what == "rows":
        total = 39
    if what == "table":
        a[2] = 32
        total = 80
    if what == "negative_new":
        a[1] = -1
    if what == "negative_len":
        c[1] = -1
    if what == "long_len":
        c[1] = 65
    if what == "n_free":
        n_free = 1000
    lens, tb, nf = dev(c, torch.int32), dev(table, torch.int32), dev([n_free], torch.int32)
    p = hc.plan_pages(lens, dev(a, torch.int32), tb, dev(free, torch.int32), nf, ps, total)
    assert int(p.status) == bit
    assert np.array_equal(lens.cpu().numpy(), c) and int(nf) == n_free and np.array_equal(tb.cpu().numpy(), table)
    assert (p.cu_new == 0).all() and (p.slots == -1).all() and (p.seq_ids == -1).all() and (p.positions == -1).all()


def test_release_takes_a_step_back_and_frees():
    import hotcold_kv_cache_b200 as hc
    rng = np.random.default_rng(4)
    ps, c, a = 32, rng.integers(0, 200, 50), rng.integers(0, 100, 50)
    table, free, n_free = make_table(rng, c, ps, 10, 300)
    lens, tb, fr, nf = (dev(x, torch.int32) for x in (c, table, free, [n_free]))
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    hc.plan_pages(lens, dev(a, torch.int32), tb, fr, nf, ps, int(a.sum()))
    hc.release_pages(lens, dev(c, torch.int32), tb, fr, nf, ps, status=st)
    assert np.array_equal(lens.cpu().numpy(), c) and int(nf) == n_free
    assert np.array_equal(fr.cpu().numpy()[:n_free], free[:n_free])
    keep = np.minimum(c, 33)
    hc.release_pages(lens, dev(keep, torch.int32), tb, fr, nf, ps, status=st)
    back = sum(-(-int(x) // ps) - -(-int(y) // ps) for x, y in zip(c, keep))
    assert int(nf) == n_free + back and np.array_equal(lens.cpu().numpy(), keep) and int(st) == 0
    held = [tb.cpu().numpy()[b, :-(-int(k) // ps)] for b, k in enumerate(keep)]
    every = np.concatenate(held + [fr.cpu().numpy()[:int(nf)]])
    assert np.array_equal(np.sort(every), np.arange(len(free)))  # every page once
    before = [x.clone() for x in (lens, tb, fr, nf)]
    hc.release_pages(lens, dev(keep + 1, torch.int32), tb, fr, nf, ps, status=st)
    assert int(st) == INDEX and all(torch.equal(x, y) for x, y in zip(before, (lens, tb, fr, nf)))
    st.zero_()
    nf.fill_(len(free))
    hc.release_pages(lens, torch.zeros_like(lens), tb, fr, nf, ps, status=st)
    assert int(st) == CAPACITY and np.array_equal(lens.cpu().numpy(), keep)


# ------------------------------------------------------------------------------------------------ append
def norm(g, t, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(t)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,Hq,Hk,D,ps,layout", [(1, 32, 8, 128, 64, "plain"), (37, 8, 2, 64, 16, "heads_first"),
                                                 (129, 4, 4, 128, 256, "odd"), (1000, 8, 1, 64, 32, "plain")])
def test_append(dt, T, Hq, Hk, D, ps, layout):
    import hotcold_kv_cache_b200 as hc
    g = torch.Generator(device="cuda").manual_seed(T + D)
    t = DT[dt]
    n_pages = -(-T // ps) + 3

    def make(H):
        if layout == "heads_first":
            return norm(g, t, H, T, D).transpose(0, 1)
        if layout == "odd":  # rows that do not start on 16 bytes
            return norm(g, t, T, H, D + 1)[..., 1:]
        return norm(g, t, T, H, D)

    q, k, v = make(Hq), make(Hk), make(Hk)
    kp, vp = norm(g, t, n_pages, Hk, ps, D), norm(g, t, n_pages, Hk, ps, D)
    slots = torch.randperm(n_pages * ps, generator=g, device="cuda")[:T]
    pos = torch.randint(0, 200000, (T,), generator=g, device="cuda")
    pos[0] = 131071
    skip = torch.zeros(T, dtype=torch.bool, device="cuda")
    if T > 5:
        skip[3] = skip[-1] = True
    slots = torch.where(skip, -1, slots)
    inv = torch.tensor(1.0 / 500000.0 ** (np.arange(0, D, 2) / D), dtype=torch.float32, device="cuda")
    want_k, want_v = kp.double(), vp.double()
    live = ~skip
    rows = slots[live]
    want_k[rows // ps, :, rows % ps] = R.rotate(k, pos, inv, 0.75)[live]
    want_v[rows // ps, :, rows % ps] = v.double()[live]
    want_q = R.rotate(q, pos, inv, 0.75)
    q_out = torch.full((T, Hq, D), 7.0, dtype=t, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = hc.append_pages(q, k, v, slots, pos, kp, vp, inv_freq=inv, rope_scaling=0.75, q_out=q_out, status=st)
    assert r is q_out and int(st) == 0
    # |x'| <= 0.75 (|a| + |b|): sincosf (2 ulp) and the angle's last rounding to 32 bits (2^-24 pi, absolute), two
    # products and a sum, scaling: 8 roundings of 2^-24 of at most 2 max|x|; then one rounding to the type
    u = torch.finfo(t).eps / 2
    m = max(float(q.abs().max()), float(k.abs().max()))
    tol = 16 * 2.0 ** -24 * m
    assert ((r.double() - want_q)[live].abs() <= u * want_q[live].abs() + tol).all()
    assert ((kp.double() - want_k).abs() <= u * want_k.abs() + tol).all()
    assert torch.equal(vp.double(), want_v)
    assert (r[skip] == 7.0).all()


def test_append_without_rotary_and_bad_slots():
    import hotcold_kv_cache_b200 as hc
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = norm(g, torch.float16, 4, 2, 64), norm(g, torch.float16, 4, 2, 64), norm(g, torch.float16, 4, 4, 64)
    kp, vp = torch.zeros(3, 2, 16, 64, dtype=torch.float16, device="cuda"), torch.zeros(3, 2, 16, 64,
                                                                                       dtype=torch.float16, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.tensor([47, 48, -5, 0], device="cuda")
    assert hc.append_pages(q, k, v, slots, None, kp, vp, status=st) is q
    assert int(st) == INDEX
    assert torch.equal(kp[2, :, 15], k[0]) and torch.equal(vp[0, :, 0], v[3])
    kp[2, :, 15] = 0
    kp[0, :, 0] = 0
    assert not kp.any()
    assert hc.append_pages(None, k[:0], v[:0], slots[:0], None, kp, vp) is None


# ------------------------------------------------------------------------------------------------ attention
def state(seed, dt, Hq, Hk, D, P, ps, ctx, new, pad=0, mask=None, layout="tokens", fill=None):
    """Inputs of an attention whose sequences hold ctx tokens and add `new`; pages in random order, the rest of the
    pool, the page tails and masked prefix rows NaN."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DT[dt]
    ctx, new = np.asarray(ctx), np.asarray(new)
    B, T = len(ctx), int(np.sum(new))
    lens = ctx + new
    max_blocks = max(1, int(max(-(-int(x) // ps) for x in lens)) + 1)
    table, _, _ = make_table(rng, lens, ps, max_blocks, 3)
    n_pages = int(sum(-(-int(x) // ps) for x in lens)) + 3
    kp, vp = (torch.full((n_pages, Hk, ps, D), math.nan, dtype=t, device="cuda") for _ in range(2))
    for b in range(B):
        for j in range(-(-int(lens[b]) // ps)):
            n = min(ps, int(lens[b]) - j * ps)
            kp[int(table[b, j]), :, :n] = norm(g, t, Hk, n, D)
            vp[int(table[b, j]), :, :n] = norm(g, t, Hk, n, D)
    pk = pv = m = None
    if P:
        if layout == "tokens":
            pk, pv = norm(g, t, P, Hk, D).transpose(0, 1), norm(g, t, P, Hk, D).transpose(0, 1)
        else:
            pk, pv = norm(g, t, Hk, P, D), norm(g, t, Hk, P, D)
        if mask is not None:
            m = torch.rand(P, generator=g, device="cuda") < mask
            pk[:, ~m] = math.nan
            pv[:, ~m] = math.inf
    q = norm(g, t, T + pad, Hq, D)
    cu = np.concatenate([[0], np.cumsum(new)])
    return dict(q=q, prefix_k=pk, prefix_v=pv, k_pages=kp, v_pages=vp, block_table=dev(table, torch.int32),
                lens=dev(lens, torch.int32), cu_new=dev(cu, torch.int32), scaling=1.0 / math.sqrt(D), prefix_mask=m)


def check(s, dt, got, lse, T):
    """Every row of a sequence within the derived tolerance, finite, with its log-sum."""
    q = s["q"][:T]
    ref, rl, A, S = R.attend(q, s["prefix_k"], s["prefix_v"], s["k_pages"], s["v_pages"], s["block_table"], s["lens"],
                             s["cu_new"], s["scaling"], s["prefix_mask"])
    D = q.shape[2]
    n = (s["prefix_k"].shape[1] if s["prefix_k"] is not None else 0) + int(s["lens"].max())
    tol = R.attend_tolerance(DT[dt], D, max(n, 1), ref, A, S)
    err = (got[:T].double() - ref).abs()
    assert torch.isfinite(got[:T]).all()
    worst = (err / tol).max()
    assert worst <= 1, f"off by {float(worst):.2f} of the tolerance"
    empty = torch.isinf(rl)
    assert torch.equal(torch.isinf(lse[:T]), empty)
    # the log-sum: a score's error, 2^-20 for the exponentials and the logarithm, and the 32-bit sum's
    lt = D * 2.0 ** -22 * S + 2.0 ** -20 + 2.0 ** -22 * rl.abs() + 8 * math.sqrt(max(n, 1)) * 2.0 ** -24
    assert ((lse[:T].double() - rl).abs()[~empty] <= lt[~empty]).all()


CASES = [
    # Hq, Hk, D, P, page, ctx, new
    (4, 4, 64, 0, 16, [0], [1]),                       # one token alone
    (8, 8, 128, 1, 16, [0], [1]),
    (8, 2, 128, 63, 16, [1], [1]),
    (8, 2, 128, 129, 32, [15, 16, 17, 0], [1, 1, 1, 1]),
    (32, 8, 128, 1000, 16, [300, 0, 77, 128], [1, 1, 1, 1]),
    (16, 2, 64, 300, 64, [5, 0, 700], [1, 0, 3]),      # an idle sequence, a draft
    (8, 1, 64, 257, 16, [0, 130, 3], [70, 1, 5]),      # ragged chunk beside decode steps
    (4, 2, 128, 0, 128, [0, 0, 200], [300, 17, 129]),  # no prefix: causal prompts
    (32, 8, 128, 640, 64, [0] * 33, [1] * 33),         # more rows than one tile of 128
    (32, 8, 128, 1500, 64, list(range(70)), [1] * 70),  # more than one row tile
    (8, 2, 64, 2049, 256, [255, 256, 257], [1, 2, 1]),
    (8, 8, 128, 128, 16, [10] * 5, [0, 0, 0, 0, 1]),
    # a full row tile over many key tiles, then pages of one and of several key tiles in turn
    (32, 8, 128, 9000, 64, [(b * 397) % 900 if b % 3 else b for b in range(64)], [1] * 64),
    (16, 2, 64, 4100, 16, [(b * 211) % 600 if b % 4 else 0 for b in range(40)], [1 + b % 3 for b in range(40)]),
    # tall causal row tiles, and behind them many pieces in a row that only one of two streams takes part in
    (32, 8, 128, 40, 32, [0] * 16, [70, 20, 20, 20, 25, 3, 20, 20, 20, 100, 20, 31, 1, 20, 20, 65]),
    (32, 8, 128, 3000, 16, [0] * 40, [97] + [20 + b % 12 for b in range(18)] + [1, 130] + [20] * 18 + [257]),
]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("masked", [False, True])
def test_attention(dt, case, masked):
    import hotcold_kv_cache_b200 as hc
    Hq, Hk, D, P, ps, ctx, new = CASES[case]
    if masked and P == 0:
        pytest.skip("no prefix to mask")
    s = state(100 + case, dt, Hq, Hk, D, P, ps, ctx, new, pad=2, mask=0.7 if masked else None,
              layout="tokens" if case % 2 else "heads")
    T = int(np.sum(new))
    out = torch.full((T + 2, Hq, D), 7.0, dtype=DT[dt], device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    got, lse = hc.shared_prefix_attention(**s, out=out, return_lse=True, status=st)
    assert got is out and (out[T:] == 7.0).all() and int(st) == 0
    check(s, dt, got, lse, T)
    again = hc.shared_prefix_attention(**s, out=torch.zeros_like(out))
    assert torch.equal(again[:T], got[:T])  # the same sums in the same order


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_rows_that_attend_nothing_are_zero(dt):
    import hotcold_kv_cache_b200 as hc
    s = state(5, dt, 8, 2, 128, 200, 16, [0, 40, 0], [1, 1, 2], mask=0.0)
    s["lens"] = dev([0, 41, 1], torch.int32)  # sequence 0 sees no own key; of sequence 2 only the last token does
    got, lse = hc.shared_prefix_attention(**s, return_lse=True)
    check(s, dt, got, lse, 4)
    assert not got[0].any() and not got[2].any() and torch.isinf(lse[[0, 2]]).all()
    assert got[1].abs().max() > 0 and got[3].abs().max() > 0


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_tokens_that_are_not_finite(dt, bad):
    """A token whose value or key is not finite reaches the rows that attend it, and no row before it."""
    import hotcold_kv_cache_b200 as hc
    s = state(6, dt, 8, 2, 128, 100, 16, [20, 7], [40, 3])
    clean = hc.shared_prefix_attention(**s)
    p = 20 + 25  # place of the 26th new token of sequence 0
    page = int(s["block_table"][0, p // 16])
    s["v_pages"][page, 1, p % 16, 9] = bad
    got = hc.shared_prefix_attention(**s)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[25:40, 4:8, 9] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert (torch.isnan(got[hit]) if math.isnan(bad) else got[hit] == bad).all()
    s["k_pages"][page, 0, p % 16, 3] = math.nan
    got = hc.shared_prefix_attention(**s)
    rows = torch.zeros_like(got, dtype=torch.bool)
    rows[25:40, 0:4] = True
    assert torch.isnan(got[rows]).all() and torch.equal(got[~hit & ~rows], clean[~hit & ~rows])


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_bad_tables_are_reported(dt):
    """Table entries outside the pool read as zero keys and values; lengths behind the table are cut."""
    import hotcold_kv_cache_b200 as hc
    s = state(7, dt, 8, 2, 64, 50, 16, [30, 30], [1, 1])
    good = hc.shared_prefix_attention(**s)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    t = s["block_table"]
    for entry in (-1, 1 << 30, s["k_pages"].shape[0]):
        old = int(t[0, 0])
        t[0, 0] = entry
        st.zero_()
        got = hc.shared_prefix_attention(**s, status=st)
        assert int(st) == INDEX and torch.equal(got[1], good[1]) and torch.isfinite(got).all()
        t[0, 0] = old
    s["lens"][0] = 1 << 30
    t[0, :] = t[0, 0]
    st.zero_()
    got = hc.shared_prefix_attention(**s, status=st)
    assert int(st) == INDEX and torch.equal(got[1], good[1])


def test_offsets_past_32_bits():
    import hotcold_kv_cache_b200 as hc
    n_pages = 40000  # 40000 * 2 * 256 * 128 = 2.6e9 elements a pool
    kp, vp = (torch.empty(n_pages, 2, 256, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(8)
    table = dev([[39999, 5], [33000, 39998]], torch.int32)
    lens, cu = dev([300, 256], torch.int32), dev([0, 1, 2], torch.int32)
    for p in (39999, 5, 33000, 39998):
        kp[p], vp[p] = norm(g, torch.float16, 2, 256, 128), norm(g, torch.float16, 2, 256, 128)
    k, v = norm(g, torch.float16, 1, 2, 128), norm(g, torch.float16, 1, 2, 128)
    hc.append_pages(None, k, v, dev([39999 * 256 + 255], torch.int64), None, kp, vp)
    assert torch.equal(kp[39999, :, 255], k[0]) and torch.equal(vp[39999, :, 255], v[0])
    s = dict(q=norm(g, torch.float16, 2, 8, 128), prefix_k=None, prefix_v=None, k_pages=kp, v_pages=vp,
             block_table=table, lens=lens, cu_new=cu, scaling=0.09, prefix_mask=None)
    got, lse = hc.shared_prefix_attention(**s, return_lse=True)
    check(s, "f16", got, lse, 2)


@pytest.mark.parametrize("scale", [1.0, 30.0])
def test_sharp_scores(scale):
    """Scores far apart: running maxima that keep rising, rows of one token's weight."""
    import hotcold_kv_cache_b200 as hc
    s = state(9, "f16", 8, 2, 128, 1024, 16, [100, 3], [1, 9])
    ramp = torch.linspace(0.05, 1.0, 1024, device="cuda")[None, :, None]
    s["prefix_k"].copy_((s["q"][0, 0].float() * ramp + 0.01 * s["prefix_k"].float()).half())
    s["scaling"] = scale / math.sqrt(128)
    got, lse = hc.shared_prefix_attention(**s, return_lse=True)
    check(s, "f16", got, lse, 10)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("Hq,Hk,D,T", [(8, 2, 128, 1), (8, 2, 128, 10), (16, 2, 64, 13), (32, 4, 64, 608)])
def test_sink_before_a_long_prefix(dt, Hq, Hk, D, T):
    """One key of a probability near 1 and 100 thousand others near 2^-26 each, which together are 0.15 % of the weight and
    all of the result, since the first key's value is 0."""
    import hotcold_kv_cache_b200 as hc
    P = 100000
    s = state(14, dt, Hq, Hk, D, P, 16, [0], [T], layout="heads")
    s["q"].zero_()
    s["q"][..., 0] = 1
    s["scaling"] = math.log(2)  # a score is 2's exponent
    s["prefix_k"][..., 0] = (-26 + 0.125 * s["prefix_k"][..., 0].float()).to(DT[dt])
    s["k_pages"][..., 0] = -26
    for v in (s["prefix_v"], s["v_pages"]):
        v.copy_((1 + 0.25 * v.float()).to(DT[dt]))
    s["prefix_k"][:, 0, 0] = 0
    s["prefix_v"][:, 0] = 0
    got, lse = hc.shared_prefix_attention(**s, return_lse=True)
    ref, rl, A, S = R.attend(s["q"], s["prefix_k"], s["prefix_v"], s["k_pages"], s["v_pages"], s["block_table"], s["lens"],
                             s["cu_new"], s["scaling"])
    assert 1e-3 < float(ref.mean()) < 2e-3
    # f16 holds a probability 2^11 times larger; what is below its normal numbers is off by up to 2^-25, and each of the
    # P + T probabilities so by 2^-36 of the largest
    lost = (P + T) * 2.0 ** -36 * float(s["prefix_v"].abs().max()) if dt == "f16" else 0.0
    tol = R.attend_tolerance(DT[dt], D, P + T, ref, A, S) + lost
    worst = ((got.double() - ref).abs() / tol).max()
    assert worst <= 1, f"off by {float(worst):.2f} of the tolerance"
    assert ((lse.double() - rl).abs() <= D * 2.0 ** -22 * S + 2.0 ** -20 + 2.0 ** -22 * rl.abs() +
            8 * math.sqrt(P + T) * 2.0 ** -24).all()


def relaid(x, how, fill=math.nan):
    """x (heads, tokens, D) with the same values in another layout, the memory around it not finite."""
    H, N, D = x.shape
    if how == "slice":  # tokens in the middle of a longer buffer, between heads of another use
        big = torch.full((H + 2, N + 24, D), fill, dtype=x.dtype, device=x.device)
        view = big[1:H + 1, 16:16 + N]
    elif how == "fused":  # heads of a fused projection's rows
        big = torch.full((N, H + 3, D), fill, dtype=x.dtype, device=x.device)
        view = big[:, 2:2 + H].transpose(0, 1)
    elif how == "wide":  # rows of D inside longer ones
        big = torch.full((H, N, D + 32), fill, dtype=x.dtype, device=x.device)
        view = big[..., 16:16 + D]
    view.copy_(x)
    return view


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lay_q,lay_k,lay_v", [("fused", "slice", "slice"), ("slice", "fused", "slice"), ("wide", "wide", "fused"),
                                               ("fused", "slice", "fused")])
@pytest.mark.parametrize("case", [3, 5, 13, 14])
def test_attention_reads_strided_inputs_in_place(dt, lay_q, lay_k, lay_v, case):
    """Queries as slices of a fused projection, prefixes as slices of longer buffers, keys and values laid out differently:
    the bits of the contiguous call."""
    import hotcold_kv_cache_b200 as hc
    Hq, Hk, D, P, ps, ctx, new = CASES[case]
    s = state(200 + case, dt, Hq, Hk, D, P, ps, ctx, new, mask=0.8 if case == 3 else None, layout="heads")
    want, lse = hc.shared_prefix_attention(**s, return_lse=True)
    check(s, dt, want, lse, int(np.sum(new)))
    t = dict(s, q=relaid(s["q"].transpose(0, 1), lay_q).transpose(0, 1), prefix_k=relaid(s["prefix_k"], lay_k),
             prefix_v=relaid(s["prefix_v"], lay_v))
    assert not t["q"].is_contiguous() and not t["prefix_k"].is_contiguous()
    assert torch.equal(hc.shared_prefix_attention(**t), want)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("Hk,P", [(1, 1), (1, 2), (1, 300), (4, 1)])
def test_strides_of_single_heads_and_tokens_say_nothing(dt, T, Hk, P):
    import hotcold_kv_cache_b200 as hc
    D = 128
    s = state(15, dt, 2 * Hk, Hk, D, P, 16, [20], [T], layout="heads")
    want, lse = hc.shared_prefix_attention(**s, return_lse=True)
    check(s, dt, want, lse, T)
    t = dict(s)
    for name, x in (("prefix_k", s["prefix_k"]), ("prefix_v", s["prefix_v"])):
        t[name] = x.as_strided(x.shape, (3 if Hk == 1 else x.stride(0), 5 if P == 1 else x.stride(1), 1))
    if T == 1:
        t["q"] = s["q"].as_strided(s["q"].shape, (7, D, 1))
    assert torch.equal(hc.shared_prefix_attention(**t), want)
    odd = torch.zeros(T, 2 * Hk, D + 1, dtype=DT[dt], device="cuda")[..., 1:]  # rows that do not start on 16 bytes: copied
    odd.copy_(s["q"])
    assert torch.equal(hc.shared_prefix_attention(**dict(s, q=odd)), want)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_rows_of_no_sequence_are_left_alone(dt):
    """The sequences' rows may start behind the first and end before the last."""
    import hotcold_kv_cache_b200 as hc
    s = state(16, dt, 8, 2, 128, 200, 16, [30, 0, 9], [1, 5, 40], pad=3)
    want, lse = hc.shared_prefix_attention(**s, return_lse=True)
    check(s, dt, want, lse, 46)
    s["q"] = torch.cat([torch.full_like(s["q"][:7], math.nan), s["q"]])
    s["cu_new"] = s["cu_new"] + 7
    out = torch.full_like(s["q"], 7.0)
    hc.shared_prefix_attention(**s, out=out)
    lo, hi = out[:7], out[53:]
    assert (lo == 7.0).all() and (hi == 7.0).all()
    # row tiles fall elsewhere: sums in another order
    shifted = dict(s, q=s["q"][7:], cu_new=s["cu_new"] - 7)
    check(shifted, dt, out[7:], lse, 46)


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_another_stream_and_a_captured_graph(dt):
    import hotcold_kv_cache_b200 as hc
    a = state(10, dt, 8, 2, 128, 500, 16, [10, 90, 40], [1, 1, 1])
    b = state(11, dt, 8, 2, 128, 500, 16, [80, 20, 10], [1, 1, 1])
    want_a, want_b = hc.shared_prefix_attention(**a), hc.shared_prefix_attention(**b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hc.shared_prefix_attention(**a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want_a)
    # two captured graphs, replayed at the same time on two streams
    graphs, outs = [], []
    for s in (a, b):
        out = torch.zeros_like(want_a)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            for _ in range(5):
                hc.shared_prefix_attention(**s, out=out)
        graphs.append(gr)
        outs.append(out)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want_a) and torch.equal(outs[1], want_b)
    a["q"].copy_(b["q"])  # a replay reads the inputs anew
    graphs[0].replay()
    assert not torch.equal(outs[0], want_a) and torch.equal(outs[0], hc.shared_prefix_attention(**a))


# ------------------------------------------------------------------------------------------------ a run of steps
@pytest.mark.parametrize("dt,Hq,Hk,D,ps", [("f32", 4, 2, 64, 16), ("f16", 8, 2, 128, 32), ("bf16", 8, 1, 128, 16)])
def test_steps_together(dt, Hq, Hk, D, ps):
    """Questions of ragged lengths, decode steps, a draft that is thrown away, a request that ends and one that
    takes its place: every step's attention equals dense causal attention over all tokens so far."""
    import hotcold_kv_cache_b200 as hc
    t, B, P = DT[dt], 3, 333
    g = torch.Generator(device="cuda").manual_seed(12)
    inv = torch.tensor(1.0 / 500000.0 ** (np.arange(0, D, 2) / D), dtype=torch.float32, device="cuda")
    pk, pv = norm(g, t, Hk, P, D), norm(g, t, Hk, P, D)
    n_pages, max_blocks = 30, 12
    kp, vp = (torch.full((n_pages, Hk, ps, D), math.nan, dtype=t, device="cuda") for _ in range(2))
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    table = torch.full((B, max_blocks), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(n_pages, dtype=torch.int32, device="cuda")
    nf = torch.full((1,), n_pages, dtype=torch.int32, device="cuda")
    dense = [(torch.zeros(0, Hk, D, dtype=t, device="cuda"),) * 2 for _ in range(B)]

    def step(new, keep=True):
        T = int(sum(new))
        q, k, v = norm(g, t, T + 1, Hq, D), norm(g, t, T + 1, Hk, D), norm(g, t, T + 1, Hk, D)  # one row of padding
        out = None if keep else spare_out(B, T + 1)
        p = hc.plan_pages(lens, dev(new, torch.int32), table, free, nf, ps, T + 1, base_pos=P, out=out)
        qr = hc.append_pages(q, k, v, p.slots, p.positions, kp, vp, inv_freq=inv)
        got, lse = hc.shared_prefix_attention(qr, pk, pv, kp, vp, table, p.lens, p.cu_new, 1 / math.sqrt(D),
                                              return_lse=True)
        assert int(p.status) == 0
        at = 0
        pages, now = [], []
        for b in range(B):  # the tokens so far, dense: rotated here, then held as the model dtype
            ks = R.rotate(k[at:at + new[b]], p.positions[at:at + new[b]], inv).to(t)
            now.append((torch.cat([dense[b][0], ks]), torch.cat([dense[b][1], v[at:at + new[b]]])))
            at += new[b]
        L = max(x.shape[0] for x, _ in now)
        for side in (0, 1):  # one page per sequence, as large as the longest
            pages.append(torch.stack([torch.cat([x[side], x[side].new_zeros(L - x[side].shape[0], Hk, D)])
                                      for x in now]).transpose(1, 2))
        s = dict(q=qr, prefix_k=pk, prefix_v=pv, k_pages=pages[0], v_pages=pages[1],
                 block_table=torch.arange(B, device="cuda", dtype=torch.int32)[:, None], lens=p.lens,
                 cu_new=p.cu_new, scaling=1 / math.sqrt(D), prefix_mask=None)
        # the page rows are the device's rotation, the dense ones the 64-bit one rounded: 1 ulp apart at most
        kk = torch.cat([kp[table[b, : -(-int(p.lens[b]) // ps)].long()].transpose(1, 2).reshape(-1, Hk, D)[:int(p.lens[b])]
                        for b in range(B)]).double()
        dd = torch.cat([x for x, _ in now]).double()
        assert ((kk - dd).abs() <= torch.finfo(t).eps * dd.abs() + 1e-5).all()
        # compare on the keys as stored
        at = 0
        for b in range(B):
            n = int(p.lens[b])
            pages[0][b, :, :n] = kk[at:at + n].to(t).transpose(0, 1)
            at += n
        check(s, dt, got, lse, T)
        if keep:
            dense[:] = now

    step([40, 7, 0])
    for _ in range(5):
        step([1, 1, 1])
    step([4, 4, 0], keep=False)  # a draft that is not taken
    step([1, 1, 1])
    hc.release_pages(lens, dev([int(lens[0]), 0, int(lens[2])], torch.int32), table, free, nf, ps)
    dense[1] = (torch.zeros(0, Hk, D, dtype=t, device="cuda"),) * 2
    step([1, 60, 1])
    for _ in range(ps + 1):
        step([1, 1, 1])


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    import hotcold_kv_cache_b200 as hc
    s = state(13, "f16", 8, 2, 128, 64, 16, [3], [2])

    def bad(err, **kw):
        with pytest.raises(err):
            hc.shared_prefix_attention(**{**s, **kw})

    bad(ValueError, q=s["q"].cpu())
    bad(ValueError, q=s["q"][0])
    bad(ValueError, lens=s["lens"].cpu())
    bad(TypeError, lens=s["lens"].long())
    bad(ValueError, cu_new=s["cu_new"][:1])
    bad(TypeError, k_pages=s["k_pages"].float())
    bad(ValueError, v_pages=s["v_pages"][:1])
    bad(ValueError, prefix_v=None)
    bad(ValueError, prefix_k=s["prefix_k"].float())
    bad(ValueError, prefix_k=s["prefix_k"].transpose(1, 2).contiguous().transpose(1, 2))
    bad(ValueError, prefix_mask=torch.ones(63, dtype=torch.bool, device="cuda"))
    bad(TypeError, prefix_mask=torch.ones(64, device="cuda"))
    bad(RuntimeError, scaling=0.0)
    bad(RuntimeError, scaling=-1.0)
    bad(RuntimeError, scaling=math.inf)
    bad(TypeError, q=s["q"].double())
    bad(RuntimeError, q=s["q"][:, :6])             # 3 query heads a key head
    bad(ValueError, out=torch.empty(1, 8, 128, dtype=torch.float16, device="cuda"))
    shifted = torch.empty(2 * 64 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 64, 128)
    bad(RuntimeError, prefix_k=shifted)            # a prefix that does not start on 16 bytes
    pools = [torch.zeros(4, 2, 24, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    bad(RuntimeError, k_pages=pools[0], v_pages=pools[1])  # 24 tokens a page
    got = hc.shared_prefix_attention(**{**s, "q": s["q"][:0]})
    assert got.shape == (0, 8, 128)
    with pytest.raises(ValueError):
        hc.plan_pages(s["lens"], s["lens"], s["block_table"], s["lens"], s["lens"], 16, -1)
    with pytest.raises(RuntimeError):
        hc.plan_pages(s["lens"], s["lens"], s["block_table"], s["lens"], s["lens"].clone(), 12, 4)
    k = torch.zeros(1, 2, 128, dtype=torch.float16, device="cuda")
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        hc.append_pages(k, k, k, z.int(), z, s["k_pages"], s["v_pages"])
    with pytest.raises(ValueError):
        hc.append_pages(k, k, k, z, z, s["k_pages"], s["v_pages"], q_out=k)


@pytest.mark.parametrize("base,ok", [(-1, False), (1 << 31, False), ((1 << 31) - 1, True)])
def test_base_position_bounds(base, ok):
    """Positions are 64 bits, their base 32: the last one that fits is taken, the next refused."""
    import hotcold_kv_cache_b200 as hc
    args = (dev([3], torch.int32), dev([2], torch.int32), dev([[0]], torch.int32), dev([0], torch.int32),
            dev([0], torch.int32), 16, 2)
    if not ok:
        with pytest.raises(ValueError, match="base_pos"):
            hc.plan_pages(*args, base_pos=base)
        assert args[0].tolist() == [3]
        return
    p = hc.plan_pages(*args, base_pos=base)
    assert p.positions.tolist() == [base + 3, base + 4] and p.slots.tolist() == [3, 4] and int(p.status) == 0
