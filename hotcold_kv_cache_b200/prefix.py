"""A batch of sequences behind one shared prefix: its page tables, its append and its attention.

One long document, many requests: the prefix's keys and values are stored once and read once per step
for the whole batch, and each sequence keeps only its own tokens, in pages. `plan_pages` turns request
lengths into block tables and slot maps on the GPU, `append_pages` rotates a step's queries and keys and
writes keys and values into their pages, `shared_prefix_attention` attends over [prefix | own pages],
`release_pages` gives pages back. They stand beside `triton_evict_attention_forward`, the decode
attention over dense keys of one sequence each. The reference has no counterpart.

All work on the current stream of the tensors' device without host synchronisation, so a step can be
captured as a CUDA graph; nothing is kept between calls. There is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


class PagePlan(NamedTuple):
    """What plan_pages writes: cu_new (n_seq + 1) int32, the first row of each sequence; per row t slots
    int64, seq_ids int32 and positions int64, -1 behind the last token; lens (n_seq) int32 and n_free (1)
    int32 after the step; status (1) int32, into which HC_DEV_* bits are OR-ed."""
    cu_new: torch.Tensor
    slots: torch.Tensor
    seq_ids: torch.Tensor
    positions: torch.Tensor
    lens: torch.Tensor
    n_free: torch.Tensor
    status: torch.Tensor


_FN: dict = {}
_SCRATCH_BYTES: dict = {}
_I32, _I64 = torch.int32, torch.int64
_CODE = {torch.float32: _lib.HC_F32, torch.float16: _lib.HC_F16, torch.bfloat16: _lib.HC_BF16}


def _dtype_code(dtype) -> int:
    code = _CODE.get(dtype)
    return _lib.dtype_code(dtype) if code is None else code  # raises


def _call(name: str, device, *args):
    """Launch on the current stream of `device` (made current when it is not)."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _lib.stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream_of(device))
    if rc != 0:
        raise RuntimeError(f"{name} failed (code {rc}): {_lib.load().hc_last_error().decode(errors='replace')}")


def _check(name: str, t: torch.Tensor, dtype, shape, device):
    """A contiguous CUDA tensor of this dtype, shape and device."""
    if t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous():
        return
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _vector(name: str, t: torch.Tensor, dtype, n: int, dev):
    """A contiguous CUDA tensor of n values of this dtype on device `dev` (a torch.device)."""
    if t.dtype is dtype and t.numel() == n and t.get_device() == dev.index and t.is_contiguous():
        return
    _check(name, t, dtype, (n,), dev)


def _cuda(name: str, t: torch.Tensor):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: there is no CPU path")
    return t.device


def plan_pages(lens, new_lens, block_table, free_pages, n_free, page_size: int, n_tokens: int, base_pos: int = 0,
               out: Optional[PagePlan] = None) -> PagePlan:
    """Block tables and slot maps of a step that adds new_lens[b] >= 0 tokens to sequence b.

    lens, new_lens (n_seq) int32, block_table (n_seq, max_blocks) int32, free_pages (n_pages) int32 with
    n_free (1) int32 of them free, all on one GPU. Fresh pages come off the top of the stack in the order
    of (sequence, block) into block_table. n_tokens is the number of rows of the step's tensors (at least
    the sum of new_lens; rows behind the last token get -1), base_pos the position of a sequence's first
    token (the prefix length). Without `out` the step is committed: lens and n_free are updated in place
    and returned in the plan. With `out`, the plan goes into its tensors; out.lens and out.n_free may be
    lens and n_free themselves (commit; out.lens may be new_lens too) or others (the step may be thrown away: the next plan
    starts from the same state); bits are OR-ed into out.status, which is not cleared. When the tokens do not fit n_tokens, the free pages or the tables, nothing is
    changed, the plan has no tokens and status gets HC_DEV_CAPACITY; a length out of range likewise with
    HC_DEV_INDEX."""
    dev = _cuda("lens", lens)
    n_seq, max_blocks = block_table.shape
    i32, i64 = _I32, _I64
    n_tokens = int(n_tokens)
    n_pages = free_pages.numel()
    _vector("lens", lens, i32, n_seq, dev)
    _vector("new_lens", new_lens, i32, n_seq, dev)
    _vector("block_table", block_table, i32, n_seq * max_blocks, dev)
    _vector("free_pages", free_pages, i32, n_pages, dev)
    _vector("n_free", n_free, i32, 1, dev)
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, not {n_tokens}")
    if not 0 <= base_pos < 1 << 31:
        raise ValueError(f"base_pos must be a 32-bit position, not {base_pos}")
    if out is None:
        out = PagePlan(torch.empty(n_seq + 1, dtype=i32, device=dev), torch.empty(n_tokens, dtype=i64, device=dev),
                       torch.empty(n_tokens, dtype=i32, device=dev), torch.empty(n_tokens, dtype=i64, device=dev),
                       lens, n_free, torch.zeros(1, dtype=i32, device=dev))
    else:
        _vector("out.cu_new", out.cu_new, i32, n_seq + 1, dev)
        _vector("out.slots", out.slots, i64, n_tokens, dev)
        _vector("out.seq_ids", out.seq_ids, i32, n_tokens, dev)
        _vector("out.positions", out.positions, i64, n_tokens, dev)
        _vector("out.lens", out.lens, i32, n_seq, dev)
        _vector("out.n_free", out.n_free, i32, 1, dev)
        _vector("out.status", out.status, i32, 1, dev)
    _call("hc_plan_pages", dev, lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(),
          n_free.data_ptr(), n_seq, int(page_size), max_blocks, n_pages, n_tokens, int(base_pos),
          out.lens.data_ptr(), out.n_free.data_ptr(), out.cu_new.data_ptr(), out.slots.data_ptr(),
          out.seq_ids.data_ptr(), out.positions.data_ptr(), out.status.data_ptr())
    return out


def release_pages(lens, keep_lens, block_table, free_pages, n_free, page_size: int, status=None) -> None:
    """Sequence b keeps its first keep_lens[b] <= lens[b] tokens (0 frees it): lens becomes keep_lens and
    the pages behind them go back on the stack, in the reverse of the order plan_pages takes them. When a
    keep_lens is out of range or the stack would overflow nothing changes and status (1) int32, when
    given, gets HC_DEV_INDEX or HC_DEV_CAPACITY."""
    dev = _cuda("lens", lens)
    n_seq, max_blocks = block_table.shape
    i32 = _I32
    _check("lens", lens, i32, (n_seq,), dev)
    _check("keep_lens", keep_lens, i32, (n_seq,), dev)
    _check("block_table", block_table, i32, (n_seq, max_blocks), dev)
    _check("free_pages", free_pages, i32, (free_pages.numel(),), dev)
    _check("n_free", n_free, i32, (1,), dev)
    if status is not None:
        _check("status", status, i32, (1,), dev)
    _call("hc_release_pages", dev, lens.data_ptr(), keep_lens.data_ptr(), block_table.data_ptr(),
          free_pages.data_ptr(), n_free.data_ptr(), n_seq, int(page_size), max_blocks, free_pages.numel(),
          _lib.ptr(status))


def _rows16(t: torch.Tensor):
    """`t` (rows, heads, D), or a contiguous copy, with 16-byte aligned rows of unit stride; its address and
    strides over rows and heads."""
    s0, s1, s2 = t.stride()
    p = t.data_ptr()
    if s2 != 1 or (p | (s0 | s1) * t.element_size()) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        (s0, s1, _), p = t.stride(), t.data_ptr()
    return t, p, s0, s1


def _pools(k_pages, v_pages, Hk: int, D: int, dtype, dev):
    n_pages, _, page_size, _ = k_pages.shape
    _check("k_pages", k_pages, dtype, (n_pages, Hk, page_size, D), dev)
    _check("v_pages", v_pages, dtype, (n_pages, Hk, page_size, D), dev)
    return n_pages, page_size


def append_pages(q, k, v, slots, positions, k_pages, v_pages, inv_freq=None, rope_scaling: float = 1.0, q_out=None,
                 status=None):
    """Rotate a step's queries and keys and write its keys and values into their pages.

    q (T,Hq,D) or None, k and v (T,Hk,D), any strides over tokens and heads; slots, positions (T) int64 as
    plan_pages writes them; k_pages, v_pages (n_pages,Hk,page_size,D) contiguous. The rotary angle of pair
    (i, i + D/2) is positions[t] * inv_freq[i] (inv_freq (D/2) float32), cos and sin times rope_scaling,
    rounded once; without inv_freq q and k are taken as rotated and q is returned as it is. Returns the
    rotated queries (q_out when given, (T,Hq,D) contiguous). Tokens with slot -1 are skipped and their
    rows of q_out left alone; another slot outside the pool sets HC_DEV_INDEX in status (1) int32. Of two
    tokens with the same slot either one's keys and values stay, in parts too: plan_pages never makes any."""
    dev = _cuda("k", k)
    T, Hk, D = k.shape
    dtype = k.dtype
    code = _dtype_code(dtype)
    n_pages, page_size = _pools(k_pages, v_pages, Hk, D, dtype, dev)
    if v.shape != k.shape or v.dtype is not dtype or v.device != dev:
        raise ValueError("k and v must share shape, dtype and device")
    _vector("slots", slots, _I64, T, dev)
    k, kp, k_st, k_sh = _rows16(k)
    v, vp, v_st, v_sh = _rows16(v)
    Hq, qp, q_st, q_sh, qo, pp, wp = Hk, None, 0, 0, None, None, None
    if inv_freq is not None:
        _vector("positions", positions, _I64, T, dev)
        _vector("inv_freq", inv_freq, torch.float32, D // 2, dev)
        pp, wp = positions.data_ptr(), inv_freq.data_ptr()
        if q is not None:
            if q.dim() != 3 or q.shape[0] != T or q.shape[2] != D or q.dtype is not dtype or q.device != dev:
                raise ValueError(f"q must be ({T}, Hq, {D}) of k's dtype and device")
            Hq = q.shape[1]
            q, qp, q_st, q_sh = _rows16(q)
            if q_out is None:
                q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, Hq, D))
            else:
                _check("q_out", q_out, dtype, (T, Hq, D), dev)
            qo = q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without inv_freq: the queries are not rotated")
    else:
        q_out = q
    if status is not None:
        _vector("status", status, _I32, 1, dev)
    _call("hc_append_pages", dev, qp, q_st, q_sh, kp, k_st, k_sh, vp, v_st, v_sh, qo, slots.data_ptr(), pp,
          k_pages.data_ptr(), v_pages.data_ptr(), wp, rope_scaling, T, Hq, Hk, D, page_size, n_pages, code,
          _lib.ptr(status))
    return q_out


def shared_prefix_attention(q, prefix_k, prefix_v, k_pages, v_pages, block_table, lens, cu_new, scaling: float,
                            prefix_mask=None, out=None, return_lse: bool = False, status=None):
    """Attention of a step's queries over [shared prefix | the sequence's own pages].

    q (T,Hq,D) post-RoPE, any strides over tokens and heads, row t of the sequence b with cu_new[b] <= t <
    cu_new[b + 1] (cu_new (n_seq + 1) int32); prefix_k, prefix_v (Hk,P,D) or None (no prefix), any
    16-byte aligned strides over heads and tokens; k_pages, v_pages (n_pages,Hk,page_size,D);
    block_table (n_seq, max_blocks) and lens (n_seq) int32, lens counting the step's tokens. Token i of
    sequence b's n_b attends the prefix keys where prefix_mask (P) bool or uint8 is set (None: all) and
    its own keys j <= lens[b] - n_b + i. Returns out (T,Hq,D), contiguous, and with return_lse the
    natural-log sum of exponentials (T,Hq) float32 too. A row that attends nothing is 0 (lse -inf); rows
    of no sequence (before cu_new[0], from cu_new[n_seq] on) are left as they were. A table entry outside
    the pool reads as zero keys and values, a length outside the table is cut, and both set HC_DEV_INDEX in
    status (1) int32, when given. HC_DEV_TIMEOUT there means that a wait inside the kernel ran out and the
    results are worthless. Without status nothing tells of either."""
    dev = _cuda("q", q)
    if q.dim() != 3:
        raise ValueError(f"q must be (T, Hq, D), not {tuple(q.shape)}")
    T, Hq, D = q.shape
    dtype = q.dtype
    code = _dtype_code(dtype)
    Hk = k_pages.shape[1]
    n_pages, page_size = _pools(k_pages, v_pages, Hk, D, dtype, dev)
    n_seq, max_blocks = block_table.shape
    i32 = _I32
    _vector("block_table", block_table, i32, n_seq * max_blocks, dev)
    _vector("lens", lens, i32, n_seq, dev)
    _vector("cu_new", cu_new, i32, n_seq + 1, dev)
    P, pk, pv, ks0, ks1, vs0, vs1 = 0, None, None, 0, 0, 0, 0
    if prefix_k is not None:
        P = prefix_k.shape[1]
        shape = (Hk, P, D)
        if prefix_k.shape != shape or prefix_k.dtype is not dtype or prefix_k.device != dev:
            raise ValueError(f"prefix_k must be {shape} of q's dtype and device")
        if prefix_v is None or prefix_v.shape != shape or prefix_v.dtype is not dtype or prefix_v.device != dev:
            raise ValueError(f"prefix_v must be {shape} of q's dtype and device")
        pk, pv = prefix_k.data_ptr(), prefix_v.data_ptr()
        ks0, ks1, ks2 = prefix_k.stride()
        vs0, vs1, vs2 = prefix_v.stride()
        if ks2 != 1 or vs2 != 1:
            raise ValueError("prefix_k and prefix_v must have unit stride over head_dim")
    if prefix_mask is not None:
        if prefix_mask.dtype is torch.bool:
            prefix_mask = prefix_mask.view(torch.uint8)
        _vector("prefix_mask", prefix_mask, torch.uint8, P, dev)
    q, qp, q_st, q_sh = _rows16(q)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, Hq, D))
    else:
        _check("out", out, dtype, (T, Hq, D), dev)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if status is not None:
        _vector("status", status, i32, 1, dev)
    if T > 0:
        key = (dev.index, code, T, n_seq, Hq, Hk, D, P)
        nbytes = _SCRATCH_BYTES.get(key)
        if nbytes is None:
            with torch.cuda.device(dev):  # the work is divided among this device's multiprocessors
                nbytes = _lib.size("hc_shared_prefix_attention_scratch_bytes", code, T, n_seq, Hq, Hk, D, P)
            if len(_SCRATCH_BYTES) < 4096:
                _SCRATCH_BYTES[key] = nbytes
        # this call's own: two streams, or two captured graphs, never share it
        es = 4 if code == _lib.HC_F32 else 2
        scratch = q.new_empty(nbytes // es + 8)
        _call("hc_shared_prefix_attention", dev, qp, q_st, q_sh, pk, ks0, ks1, pv, vs0, vs1, _lib.ptr(prefix_mask),
              k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(), lens.data_ptr(), cu_new.data_ptr(),
              out.data_ptr(), _lib.ptr(lse), _lib.ptr(status), T, n_seq, Hq, Hk, D, P, page_size, max_blocks, n_pages,
              code, scaling, scratch.data_ptr(), scratch.numel() * es)
    return (out, lse) if return_lse else out
