"""A transformers cache for a batch of sequences behind one shared prefix.

    cache = build_shared_prefix_cache(model)
    model(document_ids, past_key_values=cache)          # (1, P): the prefix, run once
    cache.begin(n_seq=16, max_new_tokens=512)            # sixteen requests behind it
    model(question_ids, past_key_values=cache)          # (16, T); cache.next_lens([...]) first where they are ragged
    model(next_ids, past_key_values=cache)              # (16, 1), and so on

It needs install_monkeypatch(): the patched LlamaAttention.forward hands layers of this cache to
`shared_prefix_forward`. The prefix's keys and values exist once; the sequences' own tokens are in pages
(plan_pages, append_pages) and every step reads the prefix once for the whole batch
(shared_prefix_attention). Nothing is compressed or evicted: it is the exact counterpart of
build_hotcold_cache for many short requests on one long document. The reference has no counterpart.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F
from transformers.cache_utils import Cache, CacheLayerMixin

from .prefix import PagePlan, append_pages, plan_pages, release_pages, shared_prefix_attention


# What the kernels take (include/hotcold_b200.h); checked here before a step moves lengths and pages.
MAX_SEQ, MAX_ROWS, MAX_PREFIX, MAX_OWN, MAX_POOL_ROWS = 4096, 65536, 1 << 24, 1 << 30, (1 << 31) - 1


def check_heads(Hq: int, Hk: int, D: int, dtype):
    if D not in (64, 128):
        raise ValueError(f"a shared-prefix cache takes a head_dim of 64 or 128, not {D}")
    if Hq not in (Hk, 2 * Hk, 4 * Hk, 8 * Hk):
        raise ValueError(f"a shared-prefix cache takes 1, 2, 4 or 8 query heads a key head, not {Hq} over {Hk}")
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"a shared-prefix cache takes float32, float16 or bfloat16, not {dtype}")


class SharedPrefixLayer(CacheLayerMixin):
    """One layer: the prefix's post-RoPE keys and values (Hk, P, D) and the pages of the sequences' own."""
    is_compileable = False

    def __init__(self, owner: "SharedPrefixCache", layer_idx: int):
        super().__init__()
        self.owner, self.layer_idx = owner, layer_idx
        self.prefix_k: Optional[torch.Tensor] = None
        self.prefix_v: Optional[torch.Tensor] = None
        self.k_pages: Optional[torch.Tensor] = None
        self.v_pages: Optional[torch.Tensor] = None
        self.is_initialized = False

    @property
    def keys(self):
        return self.prefix_k

    @keys.setter
    def keys(self, _):
        pass

    @property
    def values(self):
        return self.prefix_v

    @values.setter
    def values(self, _):
        pass

    def lazy_initialization(self, key_states, value_states=None):
        self.is_initialized = True

    def update(self, *args, **kwargs):
        raise RuntimeError("a shared-prefix cache is read by the patched attention: call install_monkeypatch() first")

    def get_mask_sizes(self, cache_position) -> Tuple[int, int]:
        q = cache_position if isinstance(cache_position, int) else int(cache_position.shape[0])
        return int(self.get_seq_length() + q), 0

    def get_seq_length(self) -> int:
        """Prefix tokens plus the longest sequence's own."""
        return self.owner.prefix_len + max(self.owner.host_lens, default=0)

    def get_max_cache_shape(self) -> int:
        return -1


class SharedPrefixCache(Cache):
    """`rotary`: a rotary module whose inv_freq and attention_scaling take the place of the two given here. They are
    read in begin() and at every step, since a module whose frequencies follow the length replaces them in a forward."""

    def __init__(self, n_layers: int, inv_freq: torch.Tensor, rope_scaling: float = 1.0, page_size: int = 64, rotary=None):
        if page_size < 16 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 256, not {page_size}")
        super().__init__(layers=[SharedPrefixLayer(self, i) for i in range(n_layers)])
        self.inv_freq, self.rope_scaling, self.page_size, self.rotary = inv_freq, float(rope_scaling), int(page_size), rotary
        self.prefix_len = 0
        self.prefix_mask: Optional[torch.Tensor] = None
        self.prefix_hidden = False  # the prefix's forward had a mask that hides some of its tokens
        self.n_seq = 0  # 0 until begin()
        self.host_lens: List[int] = []  # own tokens of each sequence, as the device's lens
        self.plan: Optional[PagePlan] = None
        self._next: Optional[List[int]] = None
        self._rows: Optional[torch.Tensor] = None

    # ------------------------------------------------------------------ setup
    def set_prefix(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor):
        """Post-RoPE keys and values (Hk, P, D) of the prefix in one layer; read in place, not copied, where
        their rows are 16-byte aligned."""
        layer = self.layers[layer_idx]
        if layer.prefix_k is not None:
            raise RuntimeError("the prefix is set: it goes through the model in one forward, before begin()")
        if k.shape != v.shape or k.dim() != 3:
            raise ValueError("prefix keys and values must share a shape (Hk, P, D)")

        def rows(x):
            per = 16 // x.element_size()
            ok = x.stride(2) == 1 and x.stride(0) % per == 0 and x.stride(1) % per == 0 and x.data_ptr() % 16 == 0
            return x if ok and x.stride(0) > 0 and x.stride(1) > 0 else x.contiguous()

        layer.prefix_k, layer.prefix_v = rows(k.detach()), rows(v.detach())
        layer.is_initialized = True
        self.prefix_len = int(k.shape[1])

    def begin(self, n_seq: int, max_new_tokens: int, pool_tokens: Optional[int] = None,
              prefix_mask: Optional[torch.Tensor] = None):
        """n_seq empty sequences behind the prefix, each with at most max_new_tokens own tokens; the pages of
        all hold pool_tokens (default: enough for every sequence's most). prefix_mask (P) bool leaves prefix
        tokens out; a prefix that was padded needs it."""
        first = self.layers[0]
        if first.prefix_k is None:
            raise RuntimeError("begin() comes after the prefix's forward")
        if self.prefix_hidden and prefix_mask is None:
            raise ValueError("the prefix's attention mask hid some of its tokens: begin(prefix_mask=) says which stay hidden")
        if n_seq < 1 or max_new_tokens < 1:
            raise ValueError("begin() needs at least one sequence and one new token")
        dev, (Hk, P, D) = first.prefix_k.device, first.prefix_k.shape
        for layer in self.layers:
            if layer.prefix_k is None:
                raise RuntimeError("begin() comes after the prefix's forward")
            if any(x.shape != first.prefix_k.shape or x.dtype is not first.prefix_k.dtype or x.device != dev
                   for x in (layer.prefix_k, layer.prefix_v)):
                raise ValueError("the prefix's keys and values must share shape, dtype and device over all layers")
        check_heads(Hk, Hk, D, first.prefix_k.dtype)
        ps = self.page_size
        max_blocks = -(-int(max_new_tokens) // ps)
        most = int(n_seq) * max_blocks
        n_pages = most if pool_tokens is None else max(1, min(most, -(-int(pool_tokens) // ps)))
        if n_seq > MAX_SEQ or P > MAX_PREFIX or max_blocks * ps > MAX_OWN or n_pages * Hk * ps > MAX_POOL_ROWS:
            raise ValueError(f"a shared-prefix cache takes up to {MAX_SEQ} sequences, a prefix of {MAX_PREFIX} tokens, {MAX_OWN} "
                             f"own tokens a sequence and 2^31 - 1 rows of a head a pool; asked for {n_seq}, {P}, "
                             f"{max_blocks * ps} and {n_pages * Hk * ps}")
        freq = self.inv_freq if self.rotary is None else self.rotary.inv_freq
        if freq.numel() * 2 != D:
            raise ValueError(f"{freq.numel()} rotary frequencies do not turn a whole head of {D}")
        if prefix_mask is not None:
            if prefix_mask.dtype.is_floating_point:
                raise TypeError(f"prefix_mask must be bool or whole numbers (0 leaves a token out), not {prefix_mask.dtype}")
            if prefix_mask.numel() != P:
                raise ValueError(f"prefix_mask has {prefix_mask.numel()} values for a prefix of {P} tokens")
            prefix_mask = (prefix_mask.reshape(P) != 0).to(device=dev, dtype=torch.uint8)
        self.n_seq, self.max_blocks, self.n_pages = int(n_seq), max_blocks, n_pages
        z = dict(dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.n_seq, **z)
        self.block_table = torch.full((self.n_seq, self.max_blocks), -1, **z)
        self.free_pages = torch.arange(self.n_pages, **z)
        self.n_free = torch.full((1,), self.n_pages, **z)
        self.status = torch.zeros(1, **z)
        self.prefix_mask = prefix_mask
        self._read_rotary(dev)
        for layer in self.layers:
            layer.k_pages = torch.empty((self.n_pages, Hk, ps, D), dtype=layer.prefix_k.dtype, device=dev)
            layer.v_pages = torch.empty_like(layer.k_pages)
        self.host_lens = [0] * self.n_seq
        self._next = self.plan = None

    def _read_rotary(self, dev):
        """The frequencies and the factor on cos and sin that this forward's positions were turned by."""
        if self.rotary is not None:
            self.inv_freq, self.rope_scaling = self.rotary.inv_freq, float(getattr(self.rotary, "attention_scaling", 1.0))
        self.inv_freq = self.inv_freq.detach().to(device=dev, dtype=torch.float32).contiguous()

    # ------------------------------------------------------------------ steps
    def next_lens(self, lens: Sequence[int]):
        """How many of the next forward's tokens of each row are real (the row's first ones; the rest is
        padding, whose outputs mean nothing). Without it all are."""
        self._begun("next_lens")
        lens = [int(x) for x in lens]
        if len(lens) != self.n_seq or min(lens) < 0:
            raise ValueError(f"next_lens needs {self.n_seq} lengths, none negative")
        self._next = lens

    def refresh_lens(self):
        """Read the sequences' lengths back from the device (synchronises): replays of a captured step advance
        them there only, and the checks of later steps and release() go by the host's."""
        self._begun("refresh_lens")
        self.host_lens = self.lens.tolist()

    def _begun(self, name: str):
        if self.n_seq == 0:
            raise RuntimeError(f"{name} comes after begin()")

    def _pages(self, lens) -> int:
        return sum(-(-x // self.page_size) for x in lens)

    def start_step(self, batch: int, tokens: int):
        """Page plan of a forward of (batch, tokens), shared by its layers."""
        self._begun("a step")
        if batch != self.n_seq:
            raise ValueError(f"the batch has {batch} rows, the cache {self.n_seq} sequences")
        if batch * tokens > MAX_ROWS:
            raise ValueError(f"a step takes up to {MAX_ROWS} rows, padding included, not {batch} x {tokens}: send it in parts")
        new = self._next if self._next is not None else [tokens] * self.n_seq
        if max(new) > tokens:
            raise ValueError(f"next_lens names {max(new)} tokens of a row of {tokens}")
        after = [a + b for a, b in zip(self.host_lens, new)]
        if max(after) > self.max_blocks * self.page_size or self._pages(after) > self.n_pages:
            raise RuntimeError(f"the pages do not hold this step: {self._pages(after)} of {self.n_pages} pages, longest "
                               f"sequence {max(after)} of {self.max_blocks * self.page_size} tokens")
        dev = self.lens.device
        self._read_rotary(dev)
        n = batch * tokens
        uniform = min(new) == tokens
        add = torch.full((self.n_seq,), tokens, dtype=torch.int32, device=dev) if uniform else \
            torch.tensor(new, dtype=torch.int32, device=dev)
        # committed in place; the status is the cache's own, which keeps the bits of every step, replayed ones too
        i32, i64 = dict(dtype=torch.int32, device=dev), dict(dtype=torch.int64, device=dev)
        p = self.plan = plan_pages(self.lens, add, self.block_table, self.free_pages, self.n_free, self.page_size, n,
                                   base_pos=self.prefix_len,
                                   out=PagePlan(torch.empty(self.n_seq + 1, **i32), torch.empty(n, **i64), torch.empty(n, **i32),
                                                torch.empty(n, **i64), self.lens, self.n_free, self.status))
        # packed row t comes from row seq * tokens + its place in the sequence; row n stands for none
        self._rows = None
        if not uniform:
            seq = p.seq_ids.long()
            place = torch.arange(n, device=dev) - p.cu_new[seq.clamp(min=0)]
            self._rows = torch.where(seq >= 0, seq * tokens + place, n)
        self.host_lens, self._next = after, None

    def attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float) -> torch.Tensor:
        """The layer's step after start_step: q (B*T,Hq,D), k and v (B*T,Hk,D) pre-RoPE; returns (B*T,Hq,D)."""
        layer, p, rows = self.layers[layer_idx], self.plan, self._rows
        n = q.shape[0]
        if rows is not None:
            at = rows.clamp(max=n - 1)
            q, k, v = q.index_select(0, at), k.index_select(0, at), v.index_select(0, at)
        q = append_pages(q, k, v, p.slots, p.positions, layer.k_pages, layer.v_pages, inv_freq=self.inv_freq,
                         rope_scaling=self.rope_scaling, status=self.status)
        # a step that the plan refuses on the device has no tokens: its rows stay 0 (ragged steps: `back` below)
        out = q.new_zeros(q.shape) if rows is None else None
        out = shared_prefix_attention(q, layer.prefix_k, layer.prefix_v, layer.k_pages, layer.v_pages, self.block_table,
                                      p.lens, p.cu_new, scaling, prefix_mask=self.prefix_mask, out=out, status=self.status)
        if rows is None:
            return out
        back = torch.zeros((n + 1,) + out.shape[1:], dtype=out.dtype, device=out.device)
        back.index_copy_(0, rows, out)  # the padding rows all land in the last one
        return back[:n]

    def release(self, keep_lens: Sequence[int]):
        """Sequence b keeps its first keep_lens[b] own tokens (0 frees it for another request)."""
        self._begun("release")
        keep = [int(x) for x in keep_lens]
        if len(keep) != self.n_seq or any(x < 0 or x > n for x, n in zip(keep, self.host_lens)):
            raise ValueError(f"release keeps {keep} of {self.host_lens} tokens")
        release_pages(self.lens, torch.tensor(keep, dtype=torch.int32, device=self.lens.device), self.block_table,
                      self.free_pages, self.n_free, self.page_size, status=self.status)
        self.host_lens = keep

    def device_status(self) -> int:
        """OR of the HC_DEV_* bits of the steps since begin(), replays included (synchronises). HC_DEV_CAPACITY: a step
        did not fit the pages and left everything as it was, with outputs of 0. HC_DEV_TIMEOUT: a step's outputs are
        worthless."""
        return 0 if self.n_seq == 0 else int(self.status)

    # ------------------------------------------------------------------ what transformers may ask of a cache
    # Its own versions work on dense keys and values of a layer, here the prefix of all sequences.
    def _refuse(self, name: str):
        raise NotImplementedError(f"a shared-prefix cache has no {name}: sequences are cut or freed with release(), "
                                  "another document takes another cache")

    def reset(self):
        self._refuse("reset")

    def crop(self, max_length):
        self._refuse("crop")

    def reorder_cache(self, beam_idx):
        self._refuse("reorder_cache (beam search)")

    def batch_repeat_interleave(self, repeats):
        self._refuse("batch_repeat_interleave")

    def batch_select_indices(self, indices):
        self._refuse("batch_select_indices")


def build_shared_prefix_cache(model, page_size: int = 64) -> SharedPrefixCache:
    """A SharedPrefixCache for a Llama model: its layer count and rotary module."""
    rot = model.model.rotary_emb
    return SharedPrefixCache(int(model.config.num_hidden_layers), rot.inv_freq, page_size=page_size, rotary=rot)


def hides_keys(mask) -> bool:
    """Whether an attention mask hides a key: a (B, 1, T, keys) one, bool or additive, from a sequence's last row, which
    a causal mask alone shows everything; a (B, keys) one, as flash attention is given, anywhere. Of another kind it
    cannot tell and says yes. Synchronises; under capture, where that cannot be, it says no to the kinds it knows."""
    if mask is None:
        return False
    if not isinstance(mask, torch.Tensor) or mask.dim() not in (2, 4):
        return True
    if mask.is_cuda and torch.cuda.is_current_stream_capturing():
        return False
    if mask.dim() == 2:  # 1 or True: there
        return not bool((mask != 0).all())
    last = mask[:, :, -1]
    return not bool((last if mask.dtype is torch.bool else last == 0).all())


def moved(position_ids: Optional[torch.Tensor], tokens: int) -> bool:
    """Whether a forward's positions are others than 0 to tokens - 1. Synchronises; under capture it says no."""
    if position_ids is None or (position_ids.is_cuda and torch.cuda.is_current_stream_capturing()):
        return False
    return not torch.equal(position_ids.reshape(-1), torch.arange(tokens, dtype=position_ids.dtype, device=position_ids.device))


def shared_prefix_forward(attn, hidden_states, position_embeddings, attention_mask, cache: SharedPrefixCache,
                          position_ids: Optional[torch.Tensor] = None):
    """LlamaAttention.forward over a SharedPrefixCache: before begin() the prefix's forward (transformers' RoPE and
    stock causal attention, as the patched prompt forward; at positions 0 to P - 1, since own tokens go on from P),
    after it the batch's step, whose positions and mask are the cache's own: padding comes from next_lens(). A mask
    that hides keys from a step of several tokens is refused where next_lens() says nothing."""
    from transformers.models.llama import modeling_llama
    b, t, _ = hidden_states.shape
    li, d = int(attn.layer_idx), int(attn.head_dim)
    q = attn.q_proj(hidden_states).view(b, t, -1, d)
    k = attn.k_proj(hidden_states).view(b, t, -1, d)
    v = attn.v_proj(hidden_states).view(b, t, -1, d)
    if cache.n_seq == 0:
        check_heads(q.shape[2], k.shape[2], d, k.dtype)
        if b != 1:
            raise ValueError("the prefix goes through the model as one sequence; begin() then opens the batch")
        if li == 0 and cache.layers[0].prefix_k is None and moved(position_ids, t):
            raise ValueError("the prefix sits at positions 0 to P - 1: own tokens go on from P")
        qt, kt, vt = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
        cos, sin = position_embeddings
        if attention_mask is not None and not (isinstance(attention_mask, torch.Tensor) and attention_mask.dim() == 4):
            if hides_keys(attention_mask):
                raise ValueError("the prefix's attention mask hides keys or is of a kind that is not read: hand the document in "
                                 "without padding")
            attention_mask = None  # a (1, P) mask of ones says nothing that is not causal
        qt, kt = modeling_llama.apply_rotary_pos_emb(qt, kt, cos, sin)
        cache.set_prefix(li, kt[0], vt[0])
        if li == 0:
            cache.prefix_hidden = hides_keys(attention_mask)
        rep = qt.shape[1] // kt.shape[1]
        kr, vr = (modeling_llama.repeat_kv(kt, rep), modeling_llama.repeat_kv(vt, rep)) if rep > 1 else (kt, vt)
        out = F.scaled_dot_product_attention(qt, kr, vr, attn_mask=attention_mask, dropout_p=0.0,
                                             is_causal=attention_mask is None and t > 1)
        return attn.o_proj(out.transpose(1, 2).reshape(b, t, -1)), None
    if li == 0:
        if t > 1 and cache._next is None and hides_keys(attention_mask):
            raise ValueError("the attention mask hides keys of a step: name its padding with next_lens(), and the prefix's "
                             "with begin(prefix_mask=); a shared-prefix cache does not read the mask")
        pre = cache.layers[0].prefix_k
        if k.dtype is not pre.dtype or k.device != pre.device:
            raise ValueError(f"a step of {k.dtype} on {k.device} behind a prefix of {pre.dtype} on {pre.device}")
        cache.start_step(b, t)
    out = cache.attend(li, q.reshape(b * t, -1, d), k.reshape(b * t, -1, d), v.reshape(b * t, -1, d), float(attn.scaling))
    return attn.o_proj(out.reshape(b, t, -1)), None
