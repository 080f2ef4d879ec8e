"""Generation as it is used: append -> attention -> sampling through the layer and the stack, against the same model without a
cache."""
import pytest
import torch

from multimodal_amd import harness

pytestmark = pytest.mark.gpu

# Both sides round to bf16 at every stage (a rounding is off by at most 2^-8 of the value).  They differ in the rotation (three
# roundings against one), the probabilities, the order of the sums and what follows from those: query, key, probability, context,
# dense, adapters and the residual sums, some 13 roundings of values no larger than the row's largest.
LAYER_TOL = 16 * 2.0 ** -8


def build(name, seed=1, **over):
    from multimodal_amd import mpu
    mpu.destroy_model_parallel()
    mpu.initialize_model_parallel(1)
    mpu.model_parallel_cuda_manual_seed(seed)
    torch.manual_seed(seed)
    cfg = dict(harness.CONFIGS[name], **over)
    stack = harness.MagmaStack(cfg).eval()
    with torch.no_grad():  # adapters that do something
        for n, p in stack.named_parameters():
            if "adapter" in n:
                p.normal_(0.0, 0.05)
    return cfg, stack


@pytest.mark.parametrize("name", ["tiny_magma", "tiny_1_3B", "tiny"])
@pytest.mark.parametrize("chunks", [[70], [1] * 9, [33, 1, 1, 20, 1], [64, 64]])
def test_layer_over_the_cache_equals_the_layer(name, chunks):
    from multimodal_amd.kv_cache import PagedKVCache, PagedPast
    cfg, stack = build(name)
    layer, h, s = stack.layers[1], cfg["hidden_size"], sum(chunks)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(s, 2, h, generator=g).bfloat16().cuda()
    with torch.no_grad():
        want = layer(x, stack.attention_mask(s, x.device))
        heads = cfg["num_attention_heads"]
        cache = PagedKVCache(1, heads, h // heads, 40, page_size=16)
        seqs = [cache.add(s), cache.add(s)]
        done, got = 0, []
        for n in chunks:
            step = cache.step(seqs, [n, n], [done + n] * 2)
            rows = x[done:done + n].transpose(0, 1).reshape(2 * n, 1, h)  # packed: sequence 0's rows, then sequence 1's
            y = layer(rows, None, layer_past=PagedPast(cache.layers[0], step, s))
            got.append(y.view(2, n, h).transpose(0, 1))
            done += n
        got = torch.cat(got)
    err = (got.float() - want.float()).abs().max() / want.float().abs().max()
    assert err <= LAYER_TOL, f"{err}"


def full_logits(stack, seq, enc=None):
    """Logits of every position of one sequence, without a cache."""
    with torch.no_grad():
        pre = stack.image_prefix(enc).view(1, -1, stack.word_embeddings.weight.size(1)) if enc is not None else None
        p = 0 if pre is None else pre.size(1)
        from multimodal_amd import ops
        tok = torch.cat((seq, torch.zeros(p, dtype=torch.int64))).view(1, -1).cuda()
        x = ops.embed_prefix(stack.word_embeddings.weight, tok, pre)
        mask = stack.attention_mask(x.size(0), x.device)
        for layer in stack.layers:
            x = layer(x, mask)
        logits, _ = stack.final_linear(stack.final_norm(x))
        return logits[:, 0].float().cpu(), p


@pytest.mark.parametrize("name", ["tiny_magma", "tiny_1_3B"])
@pytest.mark.parametrize("image", [False, True])
def test_greedy_tokens_are_the_largest_logits_of_the_model_without_a_cache(name, image):
    """Every token generated has, given the tokens before it, a logit within the two sides' rounding of the largest."""
    cfg, stack = build(name)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (7, 1, 30)]
    enc = torch.randn(3, 1, cfg["encoder_out_dim"], generator=g).bfloat16().cuda() if image else None
    out = stack.generate(prompts, enc_out=enc, maximum_tokens=20)
    for i, (p, o) in enumerate(zip(prompts, out)):
        assert o.shape == (20,)
        logits, pl = full_logits(stack, torch.cat((p, o)), None if enc is None else enc[i:i + 1])
        first = pl + len(p) - 1
        for t in range(20):
            row = logits[first + t]
            # two layers' difference, then the head: hidden rows of unit variance within LAYER_TOL a layer
            assert row[o[t]] >= row.max() - 2 * LAYER_TOL * row.abs().max(), (i, t)


def test_generation_is_the_same_eagerly_replayed_and_for_any_paging():
    cfg, stack = build("tiny_magma")
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (5, 17, 2, 40)]
    enc = torch.randn(4, 1, cfg["encoder_out_dim"], generator=g).bfloat16().cuda()
    run = lambda **kw: stack.generate(prompts, enc_out=enc, maximum_tokens=25, temperature=0.9, top_k=50, top_p=0.95, min_p=0.001,
                                      vocab_size=1000, generator=torch.Generator("cuda").manual_seed(9), **kw)
    ref = run(graph=False)
    assert all(int(o.max()) < 1000 and int(o.min()) >= 0 for o in ref)
    for kw in (dict(graph=True), dict(graph=True), dict(graph=False, page_size=24), dict(graph=True, page_size=64)):
        got = run(**kw)
        assert all(torch.equal(a, b) for a, b in zip(got, ref)), kw
    # per-row parameters
    t = torch.tensor([0.0, 0.9, 0.9, 0.0], device="cuda")
    got = stack.generate(prompts, enc_out=enc, maximum_tokens=25, temperature=t, top_k=50, top_p=0.95, min_p=0.001, vocab_size=1000,
                         generator=torch.Generator("cuda").manual_seed(9))
    assert torch.equal(got[1], ref[1]) and torch.equal(got[2], ref[2])


def test_end_of_text_and_the_pages_come_back():
    from multimodal_amd.generation import make_cache
    cfg, stack = build("tiny")
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (3, 9)]
    free = stack.generate(prompts, maximum_tokens=40)
    eos = int(free[0][5])
    cut = stack.generate(prompts, maximum_tokens=40, eos_token_id=eos)
    for f, c in zip(free, cut):
        n = int((f == eos).nonzero()[0]) + 1 if bool((f == eos).any()) else 40
        assert torch.equal(c, f[:n])
    cache = make_cache(stack, 2, 64)
    pages = cache.free_pages
    a = stack.generate(prompts, maximum_tokens=10, cache=cache)
    b = stack.generate(prompts, maximum_tokens=10, cache=cache)
    assert cache.free_pages == pages and all(torch.equal(x, y) and torch.equal(x, f[:10]) for x, y, f in zip(a, b, free))
    with pytest.raises(RuntimeError, match="pages needed"):
        stack.generate(prompts, maximum_tokens=500, cache=cache)
    assert cache.free_pages == pages
    assert [len(x) for x in stack.generate(prompts, maximum_tokens=1)] == [1, 1]
    assert [len(x) for x in stack.generate([], maximum_tokens=5)] == []


def test_refusals_of_the_layer():
    from multimodal_amd.kv_cache import PagedKVCache, PagedPast
    cfg, stack = build("tiny")
    layer, h = stack.layers[0], cfg["hidden_size"]
    cache = PagedKVCache(1, 4, 64, 8)
    step = cache.step([cache.add(10)], [10], [10])
    past = PagedPast(cache.layers[0], step, 10)
    x = torch.zeros(10, 1, h, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="no backward"):
        layer(x, None, layer_past=past)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="attention_mask=None"):
            layer(x, stack.attention_mask(10, x.device), layer_past=past)
        with pytest.raises(RuntimeError, match="packed rows"):
            layer(x.view(5, 2, h), None, layer_past=past)
        with pytest.raises(NotImplementedError, match="PagedPast"):
            layer(x, None, layer_past=torch.zeros(2, 3, device="cuda"))
    stack.train()
    with pytest.raises(RuntimeError, match="eval"):
        stack.generate([[1, 2]], maximum_tokens=3)


def test_arguments_of_generate():
    """Prompts may live on the GPU; a cache of another depth and a vocabulary the head does not have are refused; a sequence whose
    logits hold a NaN ends with -1, the others go on."""
    from multimodal_amd.kv_cache import PagedKVCache
    cfg, stack = build("tiny")
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (3, 9)]
    ref = stack.generate(prompts, maximum_tokens=10)
    got = stack.generate([p.cuda() for p in prompts], maximum_tokens=10)
    assert all(torch.equal(x, y) for x, y in zip(ref, got))
    heads = cfg["num_attention_heads"]
    for layers in (len(stack.layers) - 1, len(stack.layers) + 1):
        cache = PagedKVCache(layers, heads, cfg["hidden_size"] // heads, 40)
        with pytest.raises(RuntimeError, match="layers"):
            stack.generate(prompts, maximum_tokens=4, cache=cache)
        assert cache.free_pages == 40
    for v in (-1, 0, stack.word_embeddings.weight.size(0) + 1):
        with pytest.raises(RuntimeError, match="vocab_size"):
            stack.generate(prompts, maximum_tokens=4, vocab_size=v)
    unused = next(t for t in range(1000) if all(t not in o.tolist() + p.tolist() for o, p in zip(ref, prompts)))
    with torch.no_grad():
        stack.word_embeddings.weight[unused] = float("nan")
    got = stack.generate([prompts[0], torch.cat((prompts[1], torch.tensor([unused])))], maximum_tokens=10)
    assert torch.equal(got[0], ref[0]) and got[1].tolist() == [-1]


def test_generation_on_another_stream():
    cfg, stack = build("tiny_magma")
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (5, 17)]
    ref = stack.generate(prompts, maximum_tokens=12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = stack.generate(prompts, maximum_tokens=12)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_generation_between_replays_of_a_captured_layer():
    """A captured forward keeps its rotary tables while generation of other lengths runs and memory is handed out anew."""
    cfg, stack = build("tiny_magma")
    layer, s = stack.layers[0], 96
    g = torch.Generator().manual_seed(4)
    x = torch.randn(s, 2, cfg["hidden_size"], generator=g).bfloat16().cuda()
    mask = stack.attention_mask(s, x.device)
    with torch.no_grad():
        layer(x, mask)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x, mask)
    graph.replay()
    want = y.clone()
    for n in (1, 30, 150):
        stack.generate([torch.randint(0, 1000, (n,), generator=g)], maximum_tokens=6)
        held = [torch.full((1 << k,), 3.0, device="cuda", dtype=torch.bfloat16) for k in range(6, 16) for _ in range(4)]
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), n
        del held


@pytest.mark.parametrize("h,heads,part", [(256, 4, 0.25), (256, 2, 1.0), (512, 8, 0.25)])
def test_attention_over_the_cache_rotates_places_and_scales(h, heads, part):
    """The layer's attention against the definition by hand, on scores that spread by several units: two sequences that grow by chunks
    and single tokens of their own.  Roundings are independent, so the difference over all elements stays within 2 of the spreads
    that the harness bounds; the CPU test shows that mistakes of the wiring do not."""
    import generation_harness as G
    import layer_harness as LH
    from multimodal_amd import mpu
    from multimodal_amd.kv_cache import PagedKVCache, PagedPast
    mpu.destroy_model_parallel()
    mpu.initialize_model_parallel(1)
    p, d = G.layer_params(h, heads), int(h // heads * part)
    layer = LH.build_hip_layer(LH.make_neox_args(h, heads, torch.bfloat16, part, True, True), p, "cuda").eval()
    layer.attention.rotary_emb.to(torch.bfloat16)
    lens = (119, 60)
    x = [torch.randn(n, h, generator=torch.Generator().manual_seed(i + 1)).bfloat16() for i, n in enumerate(lens)]
    cache = PagedKVCache(1, heads, h // heads, 40, page_size=16)
    seqs = [cache.add(n) for n in lens]
    done, got = [0, 0], [[], []]
    with torch.no_grad():
        for new in [(70, 1), (1, 33), (0, 1), (20, 0), (1, 1), (1, 1), (26, 23)]:
            rows = torch.cat([x[i][done[i]:done[i] + n] for i, n in enumerate(new)]).cuda()
            done = [a + n for a, n in zip(done, new)]
            past = PagedPast(cache.layers[0], cache.step(seqs, list(new), done), 130)
            y = layer.attention(rows[:, None], None, layer_past=past)[0][:, 0].double().cpu()
            for i, part_ in enumerate(y.split(list(new))):
                got[i].append(part_)
    assert done == list(lens)
    for i in range(2):
        want, spread = G.attention_by_hand(p, heads, d, x[i])
        diff = torch.cat(got[i]) - want
        assert diff.norm() <= 2 * spread.norm(), float(diff.norm() / spread.norm())


def test_generated_logits_are_those_of_the_oracle(monkeypatch):
    """Every step's logits against the fp32 oracle's over the whole sequence, on sharp attention: within twice what the oracle's own
    bf16 evaluation is off, and a rounding.  The replayed run draws the same tokens."""
    import generation_harness as G
    import golden_params
    from multimodal_amd import generation
    cfg, stack = build("tiny")
    assert (cfg["padded_vocab_size"], cfg["hidden_size"], cfg["num_attention_heads"], cfg["num_layers"], cfg["rotary_pct"]) == tuple(G.MODEL.values())
    p = G.model_params()
    names = {"word_embeddings.weight": "emb", "final_norm.weight": "fln.w", "final_norm.bias": "fln.b", "final_linear.weight": "head"}
    names.update({f"layers.{i}.{k}": f"l{i}.{k}" for i in range(cfg["num_layers"]) for k in golden_params.PARAM_ORDER})
    with torch.no_grad():
        own = dict(stack.named_parameters())
        for mine, theirs in names.items():
            own[mine].copy_(p[theirs])
    prompts = [torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(n)) for n in (7, 1, 30)]
    seen, head = [], generation._head
    monkeypatch.setattr(generation, "_head", lambda *a: seen.append(head(*a)) or seen[-1])
    out = stack.generate(prompts, maximum_tokens=20, graph=False)
    assert len(seen) == 20
    for i, (t, o) in enumerate(zip(prompts, out)):
        got = torch.stack([s[i] for s in seen]).float().cpu()
        tokens = torch.cat((t, o[:-1]))
        want = G.model_logits(p, tokens, torch.float32)[-20:]
        bound = 2 * G.off(G.model_logits(p, tokens, torch.bfloat16)[-20:], want) + G.U
        assert G.off(got, want) <= bound, (i, G.off(got, want), bound)
        assert torch.equal(got.argmax(1), o)
    monkeypatch.undo()
    assert all(torch.equal(a, b) for a, b in zip(out, stack.generate(prompts, maximum_tokens=20)))


def test_generation_under_inference_mode():
    """With an ordinary stack, and with one made there, whose tensors count no versions: the same tokens."""
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (5, 17)]
    _, stack = build("tiny")
    ref = stack.generate(prompts, maximum_tokens=12)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(stack.generate(prompts, maximum_tokens=12), ref))
        _, own = build("tiny")
        assert all(torch.equal(a, b) for a, b in zip(own.generate(prompts, maximum_tokens=12), ref))
    assert all(torch.equal(a, b) for a, b in zip(own.generate(prompts, maximum_tokens=12), ref))


def test_a_stack_is_copied_after_it_has_generated_and_run():
    import copy
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (5, 17)]
    cfg, stack = build("tiny")
    ref = stack.generate(prompts, maximum_tokens=8)
    with torch.no_grad():
        stack.layers[0](torch.zeros(8, 2, cfg["hidden_size"], dtype=torch.bfloat16, device="cuda"), stack.attention_mask(8, "cuda"))
    twin = copy.deepcopy(stack)
    with torch.no_grad():
        for layer in stack.layers:  # the copy's frequencies and tables are its own
            layer.attention.rotary_emb.inv_freq.zero_()
    assert all(torch.equal(a, b) for a, b in zip(twin.generate(prompts, maximum_tokens=8), ref))
