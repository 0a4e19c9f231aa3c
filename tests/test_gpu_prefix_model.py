"""The shared-prefix cache through the patched Llama forward: every request's logits equal those of the stock model on
[prefix + its own tokens] alone."""

import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(vocab_size=500, hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=8,
           num_key_value_heads=2, head_dim=64, rope_theta=500000.0, max_position_embeddings=4096)


def setup(dtype):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(3)
    model = LlamaForCausalLM(LlamaConfig(**CFG)).eval().to(device="cuda", dtype=dtype)
    g = torch.Generator().manual_seed(4)
    ids = lambda *s: torch.randint(0, CFG["vocab_size"], s, generator=g).cuda()  # noqa: E731
    return model, ids


def stock(model, prefix, own):
    """Logits of the own tokens in one stock forward over [prefix | own]."""
    out = model(input_ids=torch.cat([prefix, own], 1), use_cache=False)
    return out.logits[0, prefix.shape[1]:].float()


# a 3-layer model in fp32: sums of up to 1024 terms in other orders, 1e-4 of logits of order 1; in 16 bits each of the 3
# layers rounds its activations (2^-8 in bf16) in two places on other paths: 16 roundings, 2^-4, and 2^-7 for fp16
TOL = {torch.float32: 1e-4, torch.float16: 2.0 ** -7, torch.bfloat16: 2.0 ** -4}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_requests_behind_a_document(dtype):
    import hotcold_kv_cache_b200 as hc
    model, ids = setup(dtype)
    prefix, B = ids(1, 700), 3
    q = ids(B, 40)
    lens = [40, 7, 23]
    steps = [ids(B, 1) for _ in range(4)]
    hc.install_monkeypatch(enable_debug=False)
    try:
        with torch.inference_mode():
            cache = hc.build_shared_prefix_cache(model, page_size=16)
            first = model(input_ids=prefix, past_key_values=cache, use_cache=True).logits[0].float()
            cache.begin(B, max_new_tokens=64)
            cache.next_lens(lens)
            got = [[x] for x in model(input_ids=q, past_key_values=cache, use_cache=True).logits.float()]
            got = [[x[0][:n]] for x, n in zip(got, lens)]
            for s in steps:
                o = model(input_ids=s, past_key_values=cache, use_cache=True).logits.float()
                for b in range(B):
                    got[b].append(o[b])
            assert cache.device_status() == 0 and cache.host_lens == [44, 11, 27]
            assert cache.lens.tolist() == cache.host_lens and cache.get_seq_length() == 744
            # request 1 ends; another question takes its place
            cache.release([44, 0, 27])
            q2 = ids(1, 9)
            pad = torch.zeros(B, 9, dtype=torch.long, device="cuda")
            pad[1] = q2
            cache.next_lens([0, 9, 0])
            late = model(input_ids=pad, past_key_values=cache, use_cache=True).logits[1].float()
            assert cache.device_status() == 0
    finally:
        hc.uninstall_monkeypatch()
    with torch.inference_mode():
        tol = TOL[dtype]
        ref = model(input_ids=prefix, use_cache=False).logits[0].float()
        assert (first - ref).abs().max() <= tol * ref.abs().max()
        for b in range(B):
            own = torch.cat([q[b:b + 1, :lens[b]]] + [s[b:b + 1] for s in steps], 1)
            ref = stock(model, prefix, own)
            assert (torch.cat(got[b]) - ref).abs().max() <= tol * ref.abs().max()
        ref = stock(model, prefix, q2)
        assert (late - ref).abs().max() <= tol * ref.abs().max()


def test_decode_step_as_a_graph():
    """A uniform decode step captured once and replayed: the tables advance on the device."""
    import hotcold_kv_cache_b200 as hc
    model, ids = setup(torch.float16)
    prefix, B = ids(1, 300), 4
    q = ids(B, 5)
    steps = [ids(B, 1) for _ in range(4)]

    def run(graph):
        out = []
        cache = hc.build_shared_prefix_cache(model, page_size=16)
        model(input_ids=prefix, past_key_values=cache, use_cache=True)
        cache.begin(B, max_new_tokens=64)
        model(input_ids=q, past_key_values=cache, use_cache=True)
        if not graph:
            for s in steps:
                out.append(model(input_ids=s, past_key_values=cache, use_cache=True).logits.clone())
        else:
            tok = steps[0].clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # warm up, then take the step back
                model(input_ids=tok, past_key_values=cache, use_cache=True)
                cache.release([5] * B)
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                logits = model(input_ids=tok, past_key_values=cache, use_cache=True).logits
            for s in steps:
                tok.copy_(s)
                g.replay()
                out.append(logits.clone())
            assert cache.lens.tolist() == [9] * B
        assert cache.device_status() == 0
        return torch.stack(out).float()

    hc.install_monkeypatch(enable_debug=False)
    try:
        with torch.inference_mode():
            assert torch.equal(run(True), run(False))
    finally:
        hc.uninstall_monkeypatch()


def test_refusals():
    import hotcold_kv_cache_b200 as hc
    model, ids = setup(torch.float16)
    hc.install_monkeypatch(enable_debug=False)
    try:
        with torch.inference_mode():
            cache = hc.build_shared_prefix_cache(model, page_size=16)
            with pytest.raises(RuntimeError):
                cache.begin(2, 10)
            with pytest.raises(ValueError):
                model(input_ids=ids(2, 10), past_key_values=cache, use_cache=True)
            model(input_ids=ids(1, 10), past_key_values=cache, use_cache=True)
            with pytest.raises(RuntimeError):
                model(input_ids=ids(1, 10), past_key_values=cache, use_cache=True)
            with pytest.raises(ValueError):
                cache.begin(0, 10)
            cache.begin(2, 16)
            with pytest.raises(ValueError):
                model(input_ids=ids(3, 1), past_key_values=cache, use_cache=True)
            with pytest.raises(ValueError):
                cache.next_lens([1])
            cache.next_lens([3, 1])
            with pytest.raises(ValueError):
                model(input_ids=ids(2, 2), past_key_values=cache, use_cache=True)
            cache.next_lens([16, 1])
            model(input_ids=ids(2, 16), past_key_values=cache, use_cache=True)
            with pytest.raises(RuntimeError):
                model(input_ids=ids(2, 1), past_key_values=cache, use_cache=True)  # the first sequence is full
            with pytest.raises(ValueError):
                cache.release([17, 1])
    finally:
        hc.uninstall_monkeypatch()
    with pytest.raises(ValueError):
        hc.build_shared_prefix_cache(model, page_size=24)


def test_padding_comes_from_next_lens():
    """A padded batch's attention mask is refused, or the step is told its padding and the mask is not needed."""
    import hotcold_kv_cache_b200 as hc
    model, ids = setup(torch.float16)
    prefix, q = ids(1, 40), ids(2, 6)
    full = torch.ones(2, 46, dtype=torch.long, device="cuda")
    padded = full.clone()
    padded[1, 44:] = 0
    hc.install_monkeypatch(enable_debug=False)
    try:
        with torch.inference_mode():
            def begun():
                cache = hc.build_shared_prefix_cache(model, page_size=16)
                model(input_ids=prefix, past_key_values=cache, use_cache=True)
                cache.begin(2, max_new_tokens=16)
                return cache

            cache = begun()
            with pytest.raises(ValueError, match="next_lens"):
                model(input_ids=q, attention_mask=padded, past_key_values=cache, use_cache=True)
            assert cache.host_lens == [0, 0] and cache.lens.tolist() == [0, 0]
            a = model(input_ids=q, attention_mask=full, past_key_values=cache, use_cache=True).logits
            cache = begun()
            assert torch.equal(a, model(input_ids=q, past_key_values=cache, use_cache=True).logits)
            cache = begun()
            cache.next_lens([6, 4])
            b = model(input_ids=q, attention_mask=padded, past_key_values=cache, use_cache=True).logits
            cache = begun()
            cache.next_lens([6, 4])
            c = model(input_ids=q, past_key_values=cache, use_cache=True).logits
            assert torch.equal(b[0], c[0]) and torch.equal(b[1, :4], c[1, :4]) and cache.device_status() == 0
    finally:
        hc.uninstall_monkeypatch()


def test_lengths_after_replays():
    """Replays advance the lengths on the device; refresh_lens brings the host's up, and steps go on from there."""
    import hotcold_kv_cache_b200 as hc
    model, ids = setup(torch.float16)
    prefix, q, steps = ids(1, 40), ids(2, 5), [ids(2, 1) for _ in range(3)]
    hc.install_monkeypatch(enable_debug=False)
    try:
        with torch.inference_mode():
            def run(graph):
                cache = hc.build_shared_prefix_cache(model, page_size=16)
                model(input_ids=prefix, past_key_values=cache, use_cache=True)
                cache.begin(2, max_new_tokens=16)
                model(input_ids=q, past_key_values=cache, use_cache=True)
                tok = steps[0].clone()
                if graph:
                    side = torch.cuda.Stream()
                    side.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.stream(side):
                        model(input_ids=tok, past_key_values=cache, use_cache=True)
                        cache.release([5, 5])
                    torch.cuda.current_stream().wait_stream(side)
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g):
                        model(input_ids=tok, past_key_values=cache, use_cache=True)
                    for s in steps[:2]:
                        tok.copy_(s)
                        g.replay()
                    cache.refresh_lens()
                else:
                    for s in steps[:2]:
                        model(input_ids=s, past_key_values=cache, use_cache=True)
                assert cache.host_lens == [7, 7] and cache.get_seq_length() == 47
                cache.release([7, 6])
                out = model(input_ids=steps[2], past_key_values=cache, use_cache=True).logits
                assert cache.host_lens == cache.lens.tolist() == [8, 7] and cache.device_status() == 0
                return out
            assert torch.equal(run(True), run(False))
    finally:
        hc.uninstall_monkeypatch()


@pytest.mark.parametrize("kind", ["dynamic", "longrope"])
def test_rotary_that_follows_the_length(kind):
    """Frequencies that move with the length: the steps turn by the frequencies of their own forward, as the stock model
    does with a cache of the whole batch."""
    import hotcold_kv_cache_b200 as hc
    from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM
    rope = dict(rope_type="dynamic", factor=4.0, rope_theta=500000.0) if kind == "dynamic" else \
        dict(rope_type="longrope", rope_theta=500000.0, factor=8.0, short_factor=[1.0] * 32,
             long_factor=[1.0 + 0.1 * i for i in range(32)], original_max_position_embeddings=128)
    cfg = {k: v for k, v in CFG.items() if k != "rope_theta"}
    cfg["max_position_embeddings"] = 128

    def fresh():  # the module keeps what a forward made of its frequencies
        torch.manual_seed(5)
        return LlamaForCausalLM(LlamaConfig(**cfg, rope_parameters=rope)).eval().cuda()

    g = torch.Generator().manual_seed(6)
    ids = lambda *s: torch.randint(0, CFG["vocab_size"], s, generator=g).cuda()  # noqa: E731
    prefix, B = ids(1, 300), 2
    steps = [ids(B, 9), ids(B, 1), ids(B, 70), ids(B, 1)]

    def run(model, cache, first, begin):
        model(input_ids=first, past_key_values=cache, use_cache=True)
        if begin:
            cache.begin(B, max_new_tokens=128)
        return torch.cat([model(input_ids=s, past_key_values=cache, use_cache=True).logits for s in steps], 1)

    with torch.inference_mode():
        model = fresh()
        before = model.model.rotary_emb.inv_freq.clone()
        ref = run(model, DynamicCache(), prefix.expand(B, -1), False)
        assert not torch.equal(model.model.rotary_emb.inv_freq, before)
        model = fresh()
        hc.install_monkeypatch(enable_debug=False)
        try:
            cache = hc.build_shared_prefix_cache(model, page_size=16)
            got = run(model, cache, prefix, True)
            assert cache.device_status() == 0
        finally:
            hc.uninstall_monkeypatch()
    assert (got - ref).abs().max() <= TOL[torch.float32] * ref.abs().max()


def test_replays_past_the_pages_are_reported():
    """A captured step replayed until the pages are full: the refused replays leave the tables alone and outputs of 0, and
    their bit outlasts the steps behind them."""
    import hotcold_kv_cache_b200 as hc
    from hotcold_kv_cache_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float32).half()  # noqa: E731
    cache = hc.SharedPrefixCache(1, torch.ones(32), page_size=16)
    cache.set_prefix(0, rnd(2, 50, 64), rnd(2, 50, 64))
    cache.begin(3, 32)
    q, k, v = rnd(3, 8, 64), rnd(3, 2, 64), rnd(3, 2, 64)

    def step():
        cache.start_step(3, 1)
        return cache.attend(0, q, k, v, 0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(31):
        graph.replay()
        assert bool((out != 0).any(-1).all())
    assert cache.lens.tolist() == [32] * 3 and cache.device_status() == 0
    pages = cache.layers[0].k_pages.clone()
    for _ in range(2):
        graph.replay()
    assert not out.any() and cache.lens.tolist() == [32] * 3 and int(cache.n_free) == 0
    assert torch.equal(cache.layers[0].k_pages, pages)
    cache.refresh_lens()
    cache.release([3, 0, 32])
    with pytest.raises(RuntimeError):
        step()  # the third sequence is full
    cache.release([3, 0, 31])
    assert bool((step() != 0).any(-1).all()) and cache.lens.tolist() == [4, 1, 32]
    assert cache.device_status() == _lib.HC_DEV_CAPACITY
    cache.begin(3, 32)
    assert cache.device_status() == 0
