"""Plain 64-bit forms of the shared-prefix batch operators, for the tests."""

import math

import numpy as np
import torch


def plan(lens, new, table, free, n_free, ps, n_tokens, base):
    """plan_pages on host lists; returns a dict, or None where the step does not fit."""
    n_seq, max_blocks = table.shape
    have = [-(-int(x) // ps) for x in lens]
    need = [-(-(int(x) + int(y)) // ps) - h for x, y, h in zip(lens, new, have)]
    if sum(need) > n_free or int(np.sum(new)) > n_tokens or any(h + n > max_blocks for h, n in zip(have, need)):
        return None
    table, top = table.copy(), n_free
    for b in range(n_seq):
        for i in range(need[b]):
            top -= 1
            table[b, have[b] + i] = free[top]
    slots, seq, pos = (np.full(n_tokens, -1, np.int64) for _ in range(3))
    t = 0
    for b in range(n_seq):
        for i in range(int(new[b])):
            p = int(lens[b]) + i
            slots[t] = int(table[b, p // ps]) * ps + p % ps
            seq[t], pos[t] = b, base + p
            t += 1
    return dict(cu_new=np.concatenate([[0], np.cumsum(new)]), slots=slots, seq_ids=seq, positions=pos,
                lens=np.asarray(lens) + np.asarray(new), n_free=top, table=table)


def rotate(x, positions, inv_freq, scaling=1.0):
    """Rotary of x (T,H,D) at positions (T), in 64 bits."""
    a = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (torch.cos(a) * scaling)[:, None], (torch.sin(a) * scaling)[:, None]
    h = x.shape[-1] // 2
    x = x.double()
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def attend(q, pk, pv, k_pages, v_pages, table, lens, cu, scaling, mask=None):
    """(out, lse, A, S): the attention, its log-sum, A = sum_j p_j |v_j| and S = max_j scale sum_d |q_d k_jd| per row,
    64 bits, by loops over sequences and heads. Rows of no sequence are NaN."""
    T, Hq, D = q.shape
    Hk, ps = k_pages.shape[1], k_pages.shape[2]
    G = Hq // Hk
    q = q.double()
    out, A = torch.full_like(q, math.nan), torch.full_like(q, math.nan)
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64, device=q.device)
    S = torch.full((T, Hq), math.nan, dtype=torch.float64, device=q.device)
    lens, cu, table = lens.tolist(), cu.tolist(), table.tolist()
    for b in range(len(lens)):
        n, ln = cu[b + 1] - cu[b], lens[b]
        for h in range(Hk):
            pages = table[b][: -(-ln // ps)]
            ks = [k_pages[pages, h].reshape(-1, D)[:ln].double()]
            vs = [v_pages[pages, h].reshape(-1, D)[:ln].double()]
            if pk is not None:
                keep = slice(None) if mask is None else mask.bool()
                ks.insert(0, pk[h][keep].double())
                vs.insert(0, pv[h][keep].double())
            P = ks[0].shape[0] if pk is not None else 0
            k, v = torch.cat(ks), torch.cat(vs)
            for i in range(n):
                end = P + max(0, ln - n + i + 1)
                x = q[cu[b] + i, h * G:(h + 1) * G]
                rows = slice(h * G, (h + 1) * G)
                if end == 0:
                    out[cu[b] + i, rows] = 0
                    A[cu[b] + i, rows] = 0
                    S[cu[b] + i, rows] = 0
                    lse[cu[b] + i, rows] = -math.inf
                    continue
                s = x @ k[:end].T * scaling
                p = torch.softmax(s, -1)
                out[cu[b] + i, rows] = p @ v[:end]
                A[cu[b] + i, rows] = p @ v[:end].abs()
                S[cu[b] + i, rows] = (x.abs() @ k[:end].abs().T * scaling).amax(-1)
                lse[cu[b] + i, rows] = torch.logsumexp(s, -1)
    return out, lse, A, S


def attend_tolerance(dtype, D, n_keys, ref, A, S):
    """How far an output may be off, element by element.
    A score is a sum of D products in 32 bits (the tensor cores keep at least 22 bits of the running sum): off by at
    most delta = D 2^-22 S, a probability by the factor e^(+-delta) over the sum's own e^(+-delta), so 2 delta A; the
    2^x instruction adds 2^-21 to both. For 16-bit types a probability is rounded (u A) and the result is rounded
    (u |ref|). Sums over n keys in 32 bits: a random walk of n steps, 8 sigma: 8 sqrt(n) 2^-24 A."""
    u = torch.finfo(dtype).eps / 2
    delta = D * 2.0 ** -22 * S[..., None] + 2.0 ** -21
    probs = u * A if dtype != torch.float32 else 0.0
    return u * ref.abs() + probs + 2 * delta * A + 8 * math.sqrt(n_keys) * 2.0 ** -24 * A + 1e-30
