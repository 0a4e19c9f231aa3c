"""CPU checks of the shared-prefix batch operators: refusals that reach no GPU, and the plain plan itself."""

import ctypes

import numpy as np
import pytest
import torch

import prefix_ref as R
from hotcold_kv_cache_b200 import _lib


def test_cpu_tensors_are_refused():
    import hotcold_kv_cache_b200 as hc
    i = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 64)
    pool = torch.zeros(1, 2, 16, 64)
    with pytest.raises(ValueError, match="CUDA"):
        hc.plan_pages(i, i, i[None], i, i, 16, 1)
    with pytest.raises(ValueError, match="CUDA"):
        hc.release_pages(i, i, i[None], i, i, 16)
    with pytest.raises(ValueError, match="CUDA"):
        hc.append_pages(q, q, q, i.long(), i.long(), pool, pool)
    with pytest.raises(ValueError, match="CUDA"):
        hc.shared_prefix_attention(q, None, None, pool, pool, i[None], i, torch.zeros(2, dtype=torch.int32), 0.1)


def attend_args(**kw):
    a = dict(q=4096, q_st=1024, q_sh=128, pk=4096, pk_sh=128, pk_st=1024, pv=4096, pv_sh=128, pv_st=1024, mask=None,
             kp=4096, vp=4096, table=4096, lens=4096, cu=4096, out=4096, lse=None, status=None, T=1, n_seq=1, Hq=8, Hk=2,
             D=128, P=16, page=16, blocks=1, pages=1, dtype=1, scale=0.1, scratch=None, nbytes=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(D=96), b"head_dim"), (dict(Hq=7), b"multiple"), (dict(Hq=6), b"group"), (dict(dtype=5), b"dtype"),
    (dict(n_seq=0), b"n_seq"), (dict(n_seq=5000), b"n_seq"), (dict(T=65537), b"query tokens"), (dict(T=-1), b"query tokens"),
    (dict(P=-1), b"prefix"), (dict(page=24), b"page_size"), (dict(page=8), b"page_size"), (dict(page=512), b"page_size"),
    (dict(blocks=0), b"max_blocks"), (dict(blocks=1 << 28), b"max_blocks"), (dict(pages=0), b"n_pages"),
    (dict(q=None), b"NULL"), (dict(pk=None), b"prefix"), (dict(scale=0.0), b"scaling"), (dict(scale=float("nan")), b"scaling"),
    (dict(q=4098), b"aligned"), (dict(T=2, q_st=1001), b"aligned"), (dict(pv_st=1001), b"aligned"), (dict(kp=4104), b"aligned"),
    (dict(), b"scratch")])
def test_attention_refusals_launch_nothing(kw, word):
    lib = _lib.load()
    assert lib.hc_shared_prefix_attention(*attend_args(**kw)) != 0
    assert word in lib.hc_last_error()


def test_plan_and_append_refusals_launch_nothing():
    lib = _lib.load()
    p = [4096] * 5
    o = [4096] * 6 + [None, None]
    for sizes, word in (((0, 16, 1, 1, 1, 0), b"n_seq"), ((4097, 16, 1, 1, 1, 0), b"n_seq"), ((1, 17, 1, 1, 1, 0), b"page_size"),
                        ((1, 16, 1, 1, -1, 0), b"n_tokens")):
        assert lib.hc_plan_pages(*p, *sizes, *o) != 0 and word in lib.hc_last_error()
    assert lib.hc_plan_pages(None, *p[1:], 1, 16, 1, 1, 1, 0, *o) != 0 and b"NULL" in lib.hc_last_error()
    assert lib.hc_release_pages(*p, 1, 20, 1, 1, None, None) != 0 and b"page_size" in lib.hc_last_error()

    def append(T=1, Hq=8, D=128, page=16, inv=4096, k=4096, st=1024, q=4096):
        return lib.hc_append_pages(q, st, 128, k, st, 128, 4096, st, 128, 4096, 4096, 4096, 4096, 4096, inv, 1.0, T, Hq, 2,
                                   D, page, 1, 1, None, None)

    assert append(T=0) == 0  # nothing to do, nothing launched
    for kw, word in ((dict(T=-1), b"n_tokens"), (dict(D=80), b"head_dim"), (dict(page=4), b"page_size"),
                     (dict(k=4100), b"aligned"), (dict(st=1023), b"aligned"), (dict(k=None), b"NULL"), (dict(q=None), b"q_out")):
        assert append(**kw) != 0 and word in lib.hc_last_error()


def test_scratch_grows_with_the_rows():
    n = [_lib.size("hc_shared_prefix_attention_scratch_bytes", 1, T, 64, 32, 8, 128, 8192) for T in (0, 1, 64, 4096)]
    assert n[0] == 0 and 0 < n[1] < n[2] < n[3] < 1 << 30
    assert _lib.size("hc_shared_prefix_attention_scratch_bytes", 1, 1, 1, 6, 2, 128, 0) == 0


def test_plain_plan():
    table = np.full((2, 3), -1, np.int32)
    table[0, 0] = 4
    r = R.plan([15, 0], [2, 16], table, np.array([0, 1, 2, 3]), 4, 16, 19, 100)
    assert r["slots"].tolist() == [79, 48] + list(range(32, 48)) + [-1]
    assert r["positions"][:2].tolist() == [115, 116] and r["n_free"] == 2
    assert r["table"].tolist() == [[4, 3, -1], [2, -1, -1]]
    assert R.plan([15, 0], [2, 16], table, np.array([0]), 1, 16, 18, 0) is None


def cpu_cache(n_layers=2):
    from hotcold_kv_cache_b200.prefix_cache import SharedPrefixCache
    cache, k = SharedPrefixCache(n_layers, torch.ones(32)), torch.randn(2, 8, 64)
    for i in range(n_layers):
        cache.set_prefix(i, k.clone(), k.clone())
    return cache, k


def test_cache_refuses_what_it_cannot_do():
    """Beam reordering, cropping and resetting would touch the prefix or leave the pages as they were."""
    cache, k = cpu_cache()
    one = torch.tensor([0])
    for name, args in [("reset", ()), ("crop", (3,)), ("reorder_cache", (one,)), ("batch_repeat_interleave", (2,)),
                       ("batch_select_indices", (one,))]:
        with pytest.raises(NotImplementedError, match=name):
            getattr(cache, name)(*args)
    assert all(torch.equal(x.prefix_k, k) and torch.equal(x.prefix_v, k) for x in cache.layers)


def test_cache_before_begin():
    cache, _ = cpu_cache()
    for call in (lambda: cache.release([]), lambda: cache.next_lens([]), lambda: cache.start_step(1, 1)):
        with pytest.raises(RuntimeError, match="begin"):
            call()
    assert cache.device_status() == 0


def test_cache_keeps_no_autograd_graph():
    from hotcold_kv_cache_b200.prefix_cache import SharedPrefixCache
    cache, k = SharedPrefixCache(1, torch.ones(32)), torch.randn(2, 8, 64, requires_grad=True)
    cache.set_prefix(0, k * 2, k * 3)
    assert not cache.layers[0].prefix_k.requires_grad and not cache.layers[0].prefix_v.requires_grad


@pytest.mark.parametrize("hidden", [None, (0, 0), (1, 5), (1, 6)])
@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.bfloat16])
def test_hidden_keys_of_a_mask(dtype, hidden):
    """A causal mask of 3 tokens behind 4 hides nothing; one padded on the left or the right does."""
    from hotcold_kv_cache_b200.prefix_cache import hides_keys
    see = torch.ones(3, 7, dtype=torch.bool).tril(4).expand(2, 1, 3, 7).clone()
    if hidden is not None:
        see[hidden[0], :, :, hidden[1]] = False
    mask = see if dtype is torch.bool else torch.zeros(see.shape, dtype=dtype).masked_fill(~see, torch.finfo(dtype).min)
    assert hides_keys(mask) is (hidden is not None)
    assert not hides_keys(None)


def cpu_model(rope=None, **kw):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    more = {} if rope is None else dict(rope_parameters=rope)
    return LlamaForCausalLM(LlamaConfig(vocab_size=50, hidden_size=128, intermediate_size=64, num_hidden_layers=2,
                                        num_attention_heads=2, num_key_value_heads=1, head_dim=64,
                                        max_position_embeddings=64, **more), **kw).eval()


@pytest.fixture
def patched():
    import hotcold_kv_cache_b200 as hc
    hc.install_monkeypatch(enable_debug=False)
    yield hc
    hc.uninstall_monkeypatch()


ROPES = [dict(rope_type="dynamic", factor=2.0, rope_theta=10000.0),
         dict(rope_type="longrope", rope_theta=10000.0, factor=4.0, short_factor=[1.0] * 32, long_factor=[2.0] * 32,
              original_max_position_embeddings=64),
         dict(rope_type="default", rope_theta=10000.0)]


@pytest.mark.parametrize("rope", ROPES, ids=lambda r: r["rope_type"])
def test_frequencies_are_the_model_s_own_now(patched, rope):
    """A rotary module may replace its frequencies in the forward that passes its length: begin() and every step take
    those of that forward, not those of the day the cache was built."""
    model = cpu_model(rope)
    rot = model.model.rotary_emb
    with torch.no_grad():
        cache = patched.build_shared_prefix_cache(model, page_size=16)
        built = rot.inv_freq.clone()
        model(input_ids=torch.randint(0, 50, (1, 200)), past_key_values=cache)
        assert torch.equal(rot.inv_freq, built) is (rope["rope_type"] == "default")
        cache.begin(2, 512)
        assert torch.equal(cache.inv_freq, rot.inv_freq) and cache.rope_scaling == rot.attention_scaling
        x = torch.zeros(1, 1, 128)
        rot(x, torch.arange(700)[None])  # as the forward of a step that gets as far
        rot.attention_scaling = 0.5
        with pytest.raises(ValueError, match="CUDA"):  # the step itself needs a GPU
            cache.start_step(2, 3)
        assert torch.equal(cache.inv_freq, rot.inv_freq) and cache.rope_scaling == 0.5


@pytest.mark.parametrize("dtype", [torch.bool, torch.int64, torch.float32])
def test_hidden_keys_of_a_flat_mask(dtype):
    """A (B, keys) mask, as flash attention is given, hides where it is 0; of a kind not known nothing can be told."""
    from hotcold_kv_cache_b200.prefix_cache import hides_keys
    mask = torch.ones(2, 26).to(dtype)
    assert not hides_keys(mask)
    mask[1, 24:] = 0
    assert hides_keys(mask)
    assert hides_keys(mask[None]) and hides_keys(object())


@pytest.mark.parametrize("kind", ["sdpa", "eager", "flash_attention_2"])
@pytest.mark.parametrize("side", ["left", "right"])
def test_padded_batch_is_refused_whatever_the_attention(patched, kind, side):
    """The padding mask reaches the layers in the form of the model's attention implementation: each is refused."""
    model = cpu_model()
    model.config._attn_implementation = kind
    with torch.no_grad():
        cache = patched.build_shared_prefix_cache(model, page_size=16)
        model(input_ids=torch.randint(0, 50, (1, 20)), past_key_values=cache)
        cache.begin(2, 64)
        mask = torch.ones(2, 26, dtype=torch.long)
        mask[1, 24:] = 0
        if side == "left":
            mask[1] = mask[1].flip(0)
        with pytest.raises(ValueError, match="next_lens"):
            model(input_ids=torch.randint(0, 50, (2, 6)), attention_mask=mask, past_key_values=cache)
        assert cache.host_lens == [0, 0] and cache.plan is None


@pytest.mark.parametrize("kind", ["sdpa", "flash_attention_2"])
def test_prefix_s_forward_under_either_mask(patched, kind):
    """The prefix's forward is causal whatever form its mask has; a padded document is refused where its mask is flat."""
    ids = torch.randint(0, 50, (1, 20))
    model = cpu_model()
    with torch.no_grad():
        want = model(input_ids=ids, use_cache=False).logits
        model.config._attn_implementation = kind
        for mask in (None, torch.ones(1, 20, dtype=torch.long)):
            cache = patched.build_shared_prefix_cache(model, page_size=16)
            got = model(input_ids=ids, attention_mask=mask, past_key_values=cache).logits
            assert (got - want).abs().max() <= 1e-5 * want.abs().max()
        if kind == "flash_attention_2":
            mask[0, 17:] = 0
            cache = patched.build_shared_prefix_cache(model, page_size=16)
            with pytest.raises(ValueError, match="padding"):
                model(input_ids=ids, attention_mask=mask, past_key_values=cache)
            assert cache.layers[0].prefix_k is None


@pytest.mark.parametrize("padded", [False, True])
def test_padded_prefix_needs_a_prefix_mask(patched, padded):
    """Tokens that were hidden in the prefix's forward would be seen by every step after it."""
    model, ids = cpu_model(), torch.randint(0, 50, (1, 20))
    mask = torch.ones(1, 20, dtype=torch.long)
    if padded:
        mask[0, :3] = 0
    with torch.no_grad():
        cache = patched.build_shared_prefix_cache(model, page_size=16)
        model(input_ids=ids, attention_mask=mask, past_key_values=cache)
        if padded:
            with pytest.raises(ValueError, match="prefix_mask"):
                cache.begin(2, 64)
            assert cache.n_seq == 0
            cache.begin(2, 64, prefix_mask=mask[0].bool())
            assert cache.prefix_mask.tolist() == mask[0].tolist()
        else:
            cache.begin(2, 64)
        assert cache.n_seq == 2


def test_prefix_mask_is_checked_before_any_step():
    cache, _ = cpu_cache()
    for bad in (torch.ones(5, dtype=torch.bool), torch.ones(2, 8, dtype=torch.bool), torch.ones(0, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="prefix of 8 tokens"):
            cache.begin(2, 16, prefix_mask=bad)
    with pytest.raises(TypeError, match="prefix_mask"):  # an additive mask's 0 means the opposite
        cache.begin(2, 16, prefix_mask=torch.zeros(8))
    assert cache.n_seq == 0
    for mask in (torch.tensor([1, 0, 256, 1, 1, 1, 1, 1]), torch.tensor([[True, False] + [True] * 6])):
        cache.begin(2, 16, prefix_mask=mask)
        assert cache.prefix_mask.dtype is torch.uint8 and cache.prefix_mask.tolist() == [1, 0, 1, 1, 1, 1, 1, 1]


def test_limits_are_checked_before_a_step_moves_anything():
    """What the kernels refuse is refused before lengths and pages move: rows with padding, sequences, pools, heads."""
    from hotcold_kv_cache_b200.prefix_cache import SharedPrefixCache
    cache, _ = cpu_cache()
    cache.begin(256, 512)
    cache.next_lens([300] + [1] * 255)
    with pytest.raises(ValueError, match="65536"):
        cache.start_step(256, 300)
    assert cache.host_lens == [0] * 256 and not cache.lens.any() and int(cache.n_free) == cache.n_pages
    assert (cache.block_table == -1).all() and cache.plan is None
    cache, _ = cpu_cache()
    for n_seq, new in ((4097, 16), (2, (1 << 30) + 1), (4096, 1 << 20)):
        with pytest.raises(ValueError, match="up to"):
            cache.begin(n_seq, new)
        assert cache.n_seq == 0 and cache.layers[0].k_pages is None
    cache.begin(4096, 16, pool_tokens=64)
    for D, dtype, freq, err in ((96, torch.float32, 48, ValueError), (64, torch.float64, 32, TypeError),
                                (64, torch.float32, 16, ValueError)):
        cache, k = SharedPrefixCache(1, torch.ones(freq)), torch.zeros(2, 8, D, dtype=dtype)
        cache.set_prefix(0, k, k)
        with pytest.raises(err):
            cache.begin(2, 16)
        assert cache.n_seq == 0
    cache = SharedPrefixCache(2, torch.ones(32))
    cache.set_prefix(0, torch.zeros(2, 8, 64), torch.zeros(2, 8, 64))
    with pytest.raises(RuntimeError, match="begin"):  # the second layer has none
        cache.begin(2, 16)
    cache.set_prefix(1, torch.zeros(2, 9, 64), torch.zeros(2, 9, 64))
    with pytest.raises(ValueError, match="all layers"):
        cache.begin(2, 16)
    assert cache.n_seq == 0


def test_model_s_heads_and_types_are_checked(patched):
    """A group of 3 query heads is refused in the prefix's forward, a step of another type before it moves anything."""
    from transformers import LlamaConfig, LlamaForCausalLM
    ids = torch.randint(0, 50, (1, 20))
    with torch.no_grad():
        odd = LlamaForCausalLM(LlamaConfig(vocab_size=50, hidden_size=192, intermediate_size=64, num_hidden_layers=1,
                                           num_attention_heads=3, num_key_value_heads=1, head_dim=64)).eval()
        cache = patched.build_shared_prefix_cache(odd, page_size=16)
        with pytest.raises(ValueError, match="query heads"):
            odd(input_ids=ids, past_key_values=cache)
        assert cache.layers[0].prefix_k is None
        model = cpu_model()
        cache = patched.build_shared_prefix_cache(model, page_size=16)
        model(input_ids=ids, past_key_values=cache)
        cache.begin(1, 64)
        with pytest.raises(ValueError, match="behind a prefix"):
            model.to(torch.bfloat16)(input_ids=ids, past_key_values=cache)
        assert cache.host_lens == [0] and cache.plan is None


def test_prefix_sits_at_the_first_positions(patched):
    """Own tokens go on from the prefix's length, so a prefix at other positions is refused."""
    model, ids = cpu_model(), torch.randint(0, 50, (1, 20))
    at = torch.arange(20)[None]
    padded = (torch.tensor([[0] * 3 + [1] * 17]).cumsum(1) - 1).clamp(min=0)  # as for three tokens of padding on the left
    with torch.no_grad():
        for bad in (at + 5, padded):
            cache = patched.build_shared_prefix_cache(model, page_size=16)
            with pytest.raises(ValueError, match="positions 0 to"):
                model(input_ids=ids, position_ids=bad, past_key_values=cache)
            assert cache.layers[0].prefix_k is None
        for good in (at, at.int(), None):
            cache = patched.build_shared_prefix_cache(model, page_size=16)
            model(input_ids=ids, position_ids=good, past_key_values=cache)
            assert cache.prefix_len == 20
