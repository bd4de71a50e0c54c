"""The operators of a server together: a stack with norms of q and k heads,
half-layout rotation of a part of each head and adapters, over cache pages
that are reserved, forked, freed and compacted between its steps."""

import numpy as np
import pytest
import torch

from mk import gqa_ops, kv_page_ops, lora_ops, rope_ops
from mk import llama_layer_ops as ll
from mk import llama_stack_ops as ls
from mk.lora_ops import LoraAdapters
from mk.paged_kv_ops import make_identity_block_table
from mk.rope_ops import build_scaled_rope_tables
from tests._data import assert_close

pytestmark = pytest.mark.gpu

CFG = ll.LlamaLikeConfig(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2,
                         head_dim=64, num_hidden_layers=2, max_position_embeddings=256, vocab_size=512).validate()
ROTARY = 32


def _weights(dev, bits=4, dtype=torch.float16):
    w = ls.create_random_quantized_llama_stack_weights(CFG, bits=bits, dtype=dtype, seed=3, device=dev)
    g = torch.Generator(device=dev).manual_seed(4)

    def lora(n, k):
        a = torch.randn(3, 8, k, generator=g, device=dev) / k ** 0.5
        b = torch.randn(3, n, 8, generator=g, device=dev) * 0.1
        return LoraAdapters(a.to(dtype), b.to(dtype), torch.tensor([0.5, 1.0, 2.0], device=dev))

    for layer in w.layers:
        layer.q_norm_weight, layer.k_norm_weight = (
            (1 + 0.2 * torch.randn(CFG.head_dim, generator=g, device=dev)).to(dtype) for _ in range(2))
        layer.rope_layout = "half"
        layer.qkv_lora, layer.o_lora = lora(CFG.qkv_output_dim(), CFG.hidden_size), lora(CFG.hidden_size, CFG.hidden_size)
    return w


def _tables(dev):
    return build_scaled_rope_tables(CFG.max_position_embeddings, ROTARY, device=dev,
                                    scaling={"type": "yarn", "factor": 4, "original_max_position": 64})


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layout", ["paged", "contiguous"])
def test_layer_against_reference_backend(dev, bits, dtype, layout):
    torch.manual_seed(bits)
    w = _weights(dev, bits, dtype).layers[0]
    cos, sin = _tables(dev)
    B, S = 5, 48
    cache = ll.init_llama_layer_cache(CFG, B, S, cache_layout=layout, dtype=dtype, device=dev)
    for t in cache[:2]:
        t.copy_(torch.randn(t.shape, device=dev))
    x = torch.randn(B, 1, CFG.hidden_size, device=dev).to(dtype)
    pos = torch.tensor([0, 47, 16, 15, 30], dtype=torch.int32, device=dev)
    ids = torch.tensor([2, -1, 0, 1, 2], dtype=torch.int32, device=dev)
    kw = dict(cache_layout=layout, adapter_ids=ids)
    ref, ref_cache = ll.reference_llama_layer_decode_step(x, w, cache, cos, sin, pos, CFG, **kw)
    got, got_cache = ll.llama_layer_decode_step(x, w, tuple(t.clone() for t in cache), cos, sin, pos, CFG, **kw)
    # the bound of the layer's other test against its reference path; bf16 rounds 8 times as coarsely
    scale = 1 if dtype == torch.float16 else 8
    assert_close(got, ref.float().cpu().numpy(), what="layer", rtol=1e-2 * scale, atol=1e-3 * scale)
    for a, b in zip(got_cache[:2], ref_cache[:2]):
        assert_close(a, b.float().cpu().numpy(), what="cache", rtol=1e-2 * scale, atol=1e-3 * scale)
    plain, _ = ll.llama_layer_decode_step(x, w, tuple(t.clone() for t in cache), cos, sin, pos, CFG,
                                          cache_layout=layout)
    none, _ = ll.llama_layer_decode_step(x, w, tuple(t.clone() for t in cache), cos, sin, pos, CFG,
                                         cache_layout=layout, adapter_ids=torch.full_like(ids, -1))
    assert torch.equal(plain, none) and not torch.equal(got, plain) and torch.equal(got[1], plain[1])


def _own_pages(caches, table, lengths, P, blocks):
    """Every row's history in pages of its own, under an identity table."""
    B = table.shape[0]
    own = make_identity_block_table(B, blocks * P, P, device=table.device)
    out = []
    for K, V, _ in caches:
        pair = []
        for t in (K, V):
            rows = t[table.clamp(min=0).long()].reshape(B * blocks, *t.shape[1:])
            pair.append(rows.clone())
        out.append((*pair, own))
    return out


def test_forked_decode_steps(dev):
    """Two prompts written through their reserved pages; then steps whose rows fork, end and are compacted: each gives
    bit by bit what the same step gives on pages that nobody shares."""
    torch.manual_seed(0)
    rng = np.random.default_rng(0)
    w, (cos, sin) = _weights(dev), _tables(dev)
    P, blocks, NP, L = 8, 8, 40, CFG.num_hidden_layers
    Hq, Hkv, D = CFG.num_attention_heads, CFG.num_key_value_heads, CFG.head_dim
    pages = [torch.randn(NP, P, Hkv, D, device=dev).half() for _ in range(2 * L)]
    table = torch.full((2, blocks), -1, dtype=torch.int32, device=dev)
    refs = torch.zeros(NP, dtype=torch.int32, device=dev)
    prompt = [21, 9]
    table, lengths, refs, ready = kv_page_ops.fork_kv_sequences(pages, table, [0, 0], refs, [0, 1], reserve=max(prompt))
    assert all(ready.tolist())
    seq = torch.tensor([0] * prompt[0] + [1] * prompt[1], dtype=torch.int32, device=dev)
    pos = torch.tensor(list(range(prompt[0])) + list(range(prompt[1])), dtype=torch.int32, device=dev)
    for i, layer in enumerate(w.layers):
        qkv = torch.randn(sum(prompt), CFG.qkv_output_dim(), device=dev).half()
        gqa_ops.paged_qk_norm_rope_update(qkv, pages[2 * i], pages[2 * i + 1], table, cos, sin, pos,
                                          num_attention_heads=Hq, num_key_value_heads=Hkv, head_dim=D,
                                          q_weight=layer.q_norm_weight, k_weight=layer.k_norm_weight, sequences=seq,
                                          layout="half", rotary_dim=ROTARY)
    lengths = torch.tensor(prompt, dtype=torch.int32, device=dev)
    for step in range(12):
        alive = [b for b in range(table.shape[0]) if int(lengths[b]) > 0]
        parents = torch.tensor([int(rng.choice(alive)) for _ in range(5)], dtype=torch.int32, device=dev)
        table, lengths, refs, ready = kv_page_ops.fork_kv_sequences(pages, table, lengths, refs, parents)
        assert all(ready.tolist())
        if step % 3 == 2:
            table, refs, _, live = kv_page_ops.compact_kv_pages(pages, table, refs)
            assert (refs[int(live):] == 0).all()
        ids = torch.from_numpy(rng.integers(-1, 3, size=5)).to(torch.int32).to(dev)
        x = torch.randn(5, 1, CFG.hidden_size, device=dev).half()
        shared = [(pages[2 * i], pages[2 * i + 1], table) for i in range(L)]
        own = _own_pages(shared, table, lengths, P, blocks)
        outs = []
        for caches in (shared, own):
            cache = ls.LlamaStackCache(caches, "paged", blocks * P, P)
            outs.append(ls.llama_stack_decode_step(x, w, cache, cos, sin, lengths, CFG, adapter_ids=ids)[0])
        assert torch.equal(outs[0], outs[1]) and outs[0].isfinite().all(), step
        for (K, V, _), (Ko, Vo, to) in zip(shared, own):  # the new token, where each table says
            for b in range(5):
                j, o = int(lengths[b]) // P, int(lengths[b]) % P
                assert torch.equal(K[table[b, j], o], Ko[to[b, j], o]) and torch.equal(V[table[b, j], o], Vo[to[b, j], o])
        lengths = lengths + 1


def test_decode_graph_with_adapters(dev):
    """The captured step of such a stack, adapters changed between replays, against eager steps."""
    w, (cos, sin) = _weights(dev), _tables(dev)
    B, S = 4, 64
    caches = [ls.LlamaStackCache([ll.init_llama_layer_cache(CFG, B, S, cache_layout="paged", device=dev)
                                  for _ in range(CFG.num_hidden_layers)], "paged", S, 16) for _ in range(2)]
    tokens = torch.tensor([3, 5, 7, 11], device=dev)
    pos = torch.zeros(B, dtype=torch.int32, device=dev)
    ids = torch.tensor([0, 1, 2, -1], dtype=torch.int32, device=dev)
    graph = ls.DecodeGraph(w, caches[0], cos, sin, CFG, tokens, pos, adapter_ids=ids)
    got, want = [graph.first_tokens.clone()], []
    order = [ids.clone()]
    for i in range(6):
        ids.copy_(torch.roll(ids, 1))
        order.append(ids.clone())
        got.append(graph.step().clone())
    t, p = tokens, pos.clone()
    for step_ids in order:
        x = ls.embed_token_ids(t, w.embedding)
        logits, _, caches[1] = ls.llama_stack_decode_step(x, w, caches[1], cos, sin, p, CFG, float_logits=False,
                                                          adapter_ids=step_ids)
        t, p = ls.greedy_sample(logits), p + 1
        want.append(t)
    assert torch.equal(torch.stack(got), torch.stack(want))
    for a, b in zip(caches[0].layer_caches, caches[1].layer_caches):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_block_refusals(dev):
    w, (cos, sin) = _weights(dev), _tables(dev)
    cache = ll.init_llama_layer_cache(CFG, 1, 16, cache_layout="paged", device=dev)
    x = torch.zeros(1, 1, CFG.hidden_size, device=dev).half()
    layer = w.layers[0]
    layer.k_norm_weight = None
    with pytest.raises(ValueError, match="q_norm_weight and k_norm_weight"):
        ll.llama_layer_decode_step(x, layer, cache, cos, sin, 0, CFG, cache_layout="paged")
    from mk.quantized_decode_block_ops import paged_quantized_decode_block

    with pytest.raises(ValueError, match="need adapter_ids"):
        paged_quantized_decode_block(x, layer.qkv_w, layer.qkv_scales, layer.o_w, layer.o_scales, *cache, cos, sin, 0,
                                     H=4, num_key_value_heads=2, head_dim=64, qkv_lora=layer.qkv_lora)


def test_numbers_past_32_bits(dev, monkeypatch):
    """Unread int64 ids and positions that do not fit 32 bits are outside of every range, as they were."""
    monkeypatch.setenv("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
    far = 2 ** 32
    ids = lambda *v: torch.tensor(v, device=dev)  # noqa: E731
    x = torch.randn(3, 1, 4, 16, device=dev).half()
    cos, sin = torch.ones(8, 8, device=dev), torch.zeros(8, 8, device=dev)
    y = rope_ops.apply_rope(x, cos, sin, positions=ids(1, far + 1, -far))
    assert torch.equal(y[0], x[0]) and not y[1:].any()
    K, V = torch.zeros(2, 4, 4, 1, 16, device=dev).half()
    kw = dict(num_attention_heads=2, num_key_value_heads=1, head_dim=16)
    q, _, _ = gqa_ops.paged_qk_norm_rope_update(x, K, V, ids([0, far], [far + 1, 3], [2, 2]), cos, sin,
                                                ids(1, 2, far), **kw)
    assert q[:2].any() and not q[2].any() and K.any(-1).sum() == 1 and V[0, 1].any()
    q, _, _ = gqa_ops.paged_qk_norm_rope_update(x, K, V, ids([3, 3], [3, 3], [3, 3]), cos, sin, ids(1, 2, 3),
                                                sequences=ids(far, -far, far + 2), **kw)
    assert not q.any() and not K[3].any()
    pages = torch.arange(4, device=dev).half()[:, None].expand(4, 8).contiguous()
    kv_page_ops.copy_kv_pages([pages], ids(0, far + 1, 2), ids(3, 1, far))
    assert pages[:, 0].tolist() == [0, 1, 2, 0]
    table, lengths, refs, _ = kv_page_ops.fork_kv_sequences([], ids([0, far]), ids(far), ids(1, 0, 0),
                                                            ids(0, far, -far), reserve=0, page_size=2)
    assert table.tolist() == [[0, -1], [-1, -1], [-1, -1]]
    assert lengths.tolist() == [4, 0, 0] and refs.tolist() == [1, 0, 0]
    base = torch.randn(2, 8, device=dev).half()
    a, b = torch.ones(1, 2, 4, device=dev).half(), torch.ones(1, 8, 2, device=dev).half()
    out = lora_ops.lora_add(torch.ones(2, 4, device=dev).half(), base, a, b, ids(far, 0))
    assert torch.equal(out[0], base[0]) and (out[1] != base[1]).all()


@pytest.mark.parametrize("W", [2, 5])
@pytest.mark.parametrize("layout", ["paged", "contiguous"])
def test_verify_step_with_adapters(dev, W, layout):
    """One pass over W draft rows of three sequences, each with its adapter, against W staged steps; the bound of the
    plain stack's own test."""
    from mk.speculative_verify_ops import llama_stack_verify_step, parallel_verify_tokens

    torch.manual_seed(W)
    w, (cos, sin) = _weights(dev), _tables(dev)
    B, S = 3, 64
    first = [ll.init_llama_layer_cache(CFG, B, S, cache_layout=layout, device=dev) for _ in range(CFG.num_hidden_layers)]
    for c in first:
        for t in c[:2]:
            t.copy_(torch.randn(t.shape, device=dev))
    caches = [ls.LlamaStackCache([tuple(t.clone() for t in c) for c in first], layout, S, 16) for _ in range(2)]
    x = torch.randn(B, W, CFG.hidden_size, device=dev).half()
    pos = torch.tensor([0, 30, S - W], dtype=torch.int32, device=dev)
    ids = torch.tensor([2, -1, 0], device=dev)
    logits, _, caches[0] = llama_stack_verify_step(x, w, caches[0], cos, sin, pos, CFG, adapter_ids=ids)
    staged = []
    for i in range(W):
        lg, _, caches[1] = ls.llama_stack_decode_step(x[:, i:i + 1], w, caches[1], cos, sin, pos + i, CFG, adapter_ids=ids)
        staged.append(lg[:, 0])
    staged = torch.stack(staged, 1).float()
    rms = float(staged.square().mean().sqrt())
    assert_close(logits.float().cpu().numpy() / rms, staged.cpu().numpy() / rms, atol=8 * 2.0 ** -11, what="verify")
    # k and v are sums over 256 activations, and the passes' matvec kernels (for 3 and for 3 W rows) may round each to
    # a neighbour, 2^-10 of it: a sum moves by up to 2^-10 sum |w a| = 2^-10 (2 / pi) sqrt(256) of its rms (products
    # of normal values); a norm weight multiplies that, 1.8 at most.  (1e-3 flat, as for values of a single rounding,
    # was below that: 4e-3 came.)
    moves = 2.0 ** -10 * (2 / np.pi) * 16 * 1.8
    for a, b in zip(caches[0].layer_caches, caches[1].layer_caches):
        for s, t in zip(a[:2], b[:2]):
            t = t.float().cpu().numpy()
            assert_close(s, t, rtol=0, atol=moves * float(np.sqrt((t ** 2).mean())), what="cache")
    with pytest.raises(ValueError, match="adapter_ids must have shape"):
        llama_stack_verify_step(x, w, caches[0], cos, sin, pos, CFG, adapter_ids=ids[:2])
    one = ls.LlamaStackCache([tuple(t[:1] for t in c) if layout == "contiguous" else (*c[:2], c[2][:1]) for c in first],
                             layout, S, 16)
    kw = dict(context_token_ids=[1], proposed_token_ids=[3] * W, model_config=CFG, stack_weights=w, stack_cache=one,
              cos=cos, sin=sin, position=9)
    with_a, without = (parallel_verify_tokens(**kw, adapter_id=i).logits[0] for i in (1, None))
    assert not torch.equal(with_a, without)


def test_decode_loop_with_adapters(dev):
    w, (cos, sin) = _weights(dev), _tables(dev)
    x = torch.randn(2, 3, CFG.hidden_size, device=dev).half()
    ids = torch.tensor([1, -1], dtype=torch.int32, device=dev)

    def cache():
        return ls.LlamaStackCache([ll.init_llama_layer_cache(CFG, 2, 16, cache_layout="contiguous", device=dev)
                                   for _ in range(CFG.num_hidden_layers)], "contiguous", 16, 16)

    got, _ = ls.llama_stack_decode_loop(x, w, cache(), cos, sin, CFG, adapter_ids=ids)
    plain, _ = ls.llama_stack_decode_loop(x, w, cache(), cos, sin, CFG)
    assert not torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    want, run = [], cache()
    for t in range(3):
        lg, _, run = ls.llama_stack_decode_step(x[:, t:t + 1], w, run, cos, sin, t, CFG, adapter_ids=ids)
        want.append(lg)
    assert torch.equal(got, torch.cat(want, 1))


def test_two_streams_at_once(dev):
    """Calls of two streams that run side by side share no workspace: each gives what it gives alone."""
    g = torch.Generator(device=dev).manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev).half()  # noqa: E731
    work = []
    for k in range(2):
        x, base, a, b = rand(300, 512), rand(300, 1024), rand(20, 16, 512), rand(20, 1024, 16)
        ids = torch.randint(-1, 20, (300,), generator=g, device=dev, dtype=torch.int32)
        table = torch.randperm(9000, generator=g, device=dev)[:1200].reshape(300, 4).int()
        lengths = torch.randint(1, 13, (300,), generator=g, device=dev, dtype=torch.int32)
        parents = torch.randint(-1, 300, (300,), generator=g, device=dev, dtype=torch.int32)
        refs = kv_page_ops.count_page_refs(table, 10000)
        pages = [rand(10000, 4, 8)]
        work.append((x, base, a, b, ids, table, lengths, parents, refs, pages))

    def run(x, base, a, b, ids, table, lengths, parents, refs, pages):
        pool = [t.clone() for t in pages]
        out = lora_ops.lora_add(x, base, a, b, ids)
        new = kv_page_ops.fork_kv_sequences(pool, table, lengths, refs, parents)
        packed = kv_page_ops.compact_kv_pages(pool, new[0], new[2])
        return [out, *new, *packed, *pool]

    want = [run(*w) for w in work]
    streams = [torch.cuda.Stream(dev) for _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(*work[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for one in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(one, want[k]))


def test_two_graphs_of_one_pool(dev):
    """Two captured steps that share a memory pool, replayed in turn, several times, with eager work between."""
    g = torch.Generator(device=dev).manual_seed(6)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev).half()  # noqa: E731
    x, base, a, b = rand(300, 256), rand(300, 512), rand(9, 16, 256), rand(9, 512, 16)
    ids = torch.randint(-1, 9, (300,), generator=g, device=dev, dtype=torch.int32)
    few = torch.randint(-1, 9, (40,), generator=g, device=dev, dtype=torch.int32)
    side, pool = torch.cuda.Stream(dev), torch.cuda.graph_pool_handle()
    side.wait_stream(torch.cuda.current_stream(dev))
    calls = [lambda: lora_ops.lora_add(x, base, a, b, ids), lambda: lora_ops.lora_add(x[:40], base[:40], a, b, few)]
    with torch.cuda.stream(side):
        for call in calls:
            call()
    side.synchronize()
    graphs, outs = [], []
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=side):
            outs.append(call())
        graphs.append(graph)
    for i in range(4):
        x.copy_(rand(300, 256))
        want = [call() for call in calls]
        torch.cuda.synchronize()
        for graph, out, w in zip(graphs, outs, want):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w), i


def test_far_pages(dev):
    """Pages past 2^31 values of an array: written, copied, forked and compacted."""
    NP, P, Hkv, D = 140000, 16, 8, 128
    K, V = (torch.zeros(NP, P, Hkv, D, dtype=torch.float16, device=dev) for _ in range(2))
    cos, sin = build_scaled_rope_tables(64, D, device=dev)
    table = torch.tensor([[NP - 1, NP - 2]], dtype=torch.int32, device=dev)
    qkv = torch.randn(1, 32 * D, device=dev).half()
    kw = dict(num_attention_heads=16, num_key_value_heads=Hkv, head_dim=D)
    gqa_ops.paged_qk_norm_rope_update(qkv, K, V, table, cos, sin, torch.tensor([5], device=dev), **kw)
    small = [torch.zeros(2, P, Hkv, D, dtype=torch.float16, device=dev) for _ in range(2)]
    gqa_ops.paged_qk_norm_rope_update(qkv, *small, torch.tensor([[0, 1]], dtype=torch.int32, device=dev), cos, sin,
                                      torch.tensor([5], device=dev), **kw)
    assert torch.equal(K[NP - 1], small[0][0]) and torch.equal(V[NP - 1], small[1][0]) and V[NP - 1, 5].any()
    kv_page_ops.copy_kv_pages([K, V], [NP - 1, NP - 1], [3, NP - 5])
    assert torch.equal(K[3], small[0][0]) and torch.equal(V[NP - 5], small[1][0])
    refs = torch.ones(NP, dtype=torch.int32, device=dev)
    refs[NP - 7] = 0
    new, _, refs, ready = kv_page_ops.fork_kv_sequences([K, V], table, [6], refs, [0, 0])
    assert new[:, 0].tolist() == [NP - 1, NP - 7] and all(ready.tolist()) and torch.equal(K[NP - 7], small[0][0])
    refs.zero_()
    refs[new[:, 0].long()] = 1
    new, refs, _, live = kv_page_ops.compact_kv_pages([K, V], new, refs)
    assert new[:, 0].tolist() == [1, 0] and int(live) == 2 and int(refs.sum()) == 2
    assert all(torch.equal(t[i], s[0]) for t, s in ((K, small[0]), (V, small[1])) for i in range(2))


def test_positions_of_every_form(dev):
    """A stack of layers with head norms takes positions in the forms that plain layers take."""
    w, (cos, sin) = _weights(dev), _tables(dev)
    B, S, p = 5, 64, 37
    torch.manual_seed(2)
    x = torch.randn(B, 1, CFG.hidden_size, device=dev).half()
    first = [tuple(torch.randn_like(t) if t.is_floating_point() else t
                   for t in ll.init_llama_layer_cache(CFG, B, S, cache_layout="paged", device=dev))
             for _ in range(CFG.num_hidden_layers)]
    outs = []
    for position in (p, torch.tensor([p] * B, dtype=torch.int32, device=dev), torch.tensor(p, device=dev),
                     torch.tensor(p, dtype=torch.int32, device=dev), torch.tensor(p), [p] * B, torch.tensor([p] * B),
                     torch.full((B, 2), p, dtype=torch.int32, device=dev)[:, 1]):
        cache = ls.LlamaStackCache([tuple(t.clone() for t in c) for c in first], "paged", S, 16)
        logits, hidden, cache = ls.llama_stack_decode_step(x, w, cache, cos, sin, position, CFG)
        step, layer_cache = ll.llama_layer_decode_step(x, w.layers[0], tuple(t.clone() for t in first[0]), cos, sin,
                                                       position, CFG, cache_layout="paged")
        outs.append([logits, hidden, *(t for c in cache.layer_caches for t in c), step, *layer_cache])
    for out in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))


def _plain_weights(dev, adapted, bits=4, dtype=torch.float16):
    """Layers as an ordinary stack has them -- interleaved rotation of whole heads, no head norms -- with adapters beside
    qkv and o, or one of them; and their tables."""
    w = _weights(dev, bits, dtype)
    for layer in w.layers:
        layer.q_norm_weight = layer.k_norm_weight = None
        layer.rope_layout = "interleaved"
        if "qkv" not in adapted:
            layer.qkv_lora = None
        if "o" not in adapted:
            layer.o_lora = None
    return w, ll.build_rope_tables(CFG, device=dev)


ADAPTED = [("qkv", "o"), ("qkv",), ("o",)]


def _filled(dev, B, S, layout="paged", dtype=torch.float16):
    first = [ll.init_llama_layer_cache(CFG, B, S, cache_layout=layout, dtype=dtype, device=dev)
             for _ in range(CFG.num_hidden_layers)]
    for c in first:
        for t in c[:2]:
            t.copy_(torch.randn(t.shape, device=dev))
    return first


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("adapted", ADAPTED)
def test_plain_layer_with_adapters_against_reference_backend(dev, adapted, bits, dtype):
    torch.manual_seed(bits)
    w, (cos, sin) = _plain_weights(dev, adapted, bits, dtype)
    w, (cache, _) = w.layers[0], _filled(dev, 5, 48, dtype=dtype)
    x = torch.randn(5, 1, CFG.hidden_size, device=dev).to(dtype)
    pos = torch.tensor([0, 47, 16, 15, 30], dtype=torch.int32, device=dev)
    ids = torch.tensor([2, -1, 0, 1, 2], dtype=torch.int32, device=dev)
    kw = dict(cache_layout="paged", adapter_ids=ids)
    ref, ref_cache = ll.reference_llama_layer_decode_step(x, w, cache, cos, sin, pos, CFG, **kw)
    got, got_cache = ll.llama_layer_decode_step(x, w, tuple(t.clone() for t in cache), cos, sin, pos, CFG, **kw)
    # the bound of the layer's other tests against its reference path; bf16 rounds 8 times as coarsely
    scale = 1 if dtype == torch.float16 else 8
    assert_close(got, ref.float().cpu().numpy(), what="layer", rtol=1e-2 * scale, atol=1e-3 * scale)
    for a, b in zip(got_cache[:2], ref_cache[:2]):
        assert_close(a, b.float().cpu().numpy(), what="cache", rtol=1e-2 * scale, atol=1e-3 * scale)
    none, _ = ll.llama_layer_decode_step(x, w, tuple(t.clone() for t in cache), cos, sin, pos, CFG, cache_layout="paged",
                                         adapter_ids=torch.full_like(ids, -1))
    assert not torch.equal(got[ids >= 0], none[ids >= 0]) and torch.equal(got[1], none[1])


@pytest.mark.parametrize("W", [2, 5])
@pytest.mark.parametrize("layout", ["paged", "contiguous"])
@pytest.mark.parametrize("adapted", ADAPTED)
def test_plain_verify_step_with_adapters(dev, adapted, layout, W, monkeypatch):
    """W draft rows of an ordinary stack with adapters: one read of a sequence's pages a layer, and what W staged steps
    give (bounds as in test_verify_step_with_adapters, without its norm weights' 1.8)."""
    from mk import _lib
    from mk.speculative_verify_ops import llama_stack_verify_step

    torch.manual_seed(W)
    w, (cos, sin) = _plain_weights(dev, adapted)
    B, S = 3, 64
    first = _filled(dev, B, S, layout)
    caches = [ls.LlamaStackCache([tuple(t.clone() for t in c) for c in first], layout, S, 16) for _ in range(2)]
    x = torch.randn(B, W, CFG.hidden_size, device=dev).half()
    pos = torch.tensor([0, 30, S - W], dtype=torch.int32, device=dev)
    ids = torch.tensor([2, -1, 0], device=dev)
    names, launch = [], _lib.launch
    monkeypatch.setattr(_lib, "launch", lambda name, *a: (names.append(name), launch(name, *a))[1])
    logits, _, caches[0] = llama_stack_verify_step(x, w, caches[0], cos, sin, pos, CFG, adapter_ids=ids)
    assert names.count("mk_paged_verify_attention") == CFG.num_hidden_layers
    assert "mk_paged_decode_attention" not in names
    monkeypatch.undo()
    staged = []
    for i in range(W):
        lg, _, caches[1] = ls.llama_stack_decode_step(x[:, i:i + 1], w, caches[1], cos, sin, pos + i, CFG, adapter_ids=ids)
        staged.append(lg[:, 0])
    staged = torch.stack(staged, 1).float()
    rms = float(staged.square().mean().sqrt())
    assert_close(logits.float().cpu().numpy() / rms, staged.cpu().numpy() / rms, atol=8 * 2.0 ** -11, what="verify")
    moves = 2.0 ** -10 * (2 / np.pi) * 16
    for a, b in zip(caches[0].layer_caches, caches[1].layer_caches):
        for s, t in zip(a[:2], b[:2]):
            t = t.float().cpu().numpy()
            assert_close(s, t, rtol=0, atol=moves * float(np.sqrt((t ** 2).mean())), what="cache")


@pytest.mark.parametrize("adapted", ADAPTED)
def test_plain_loop_and_graph_with_adapters(dev, adapted):
    """The loop against its steps, and the captured step, adapters changed between replays, against eager steps."""
    w, (cos, sin) = _plain_weights(dev, adapted)
    B, S = 4, 64
    x = torch.randn(B, 3, CFG.hidden_size, device=dev).half()
    ids = torch.tensor([0, 1, 2, -1], dtype=torch.int32, device=dev)
    caches = [ls.LlamaStackCache([ll.init_llama_layer_cache(CFG, B, S, cache_layout="paged", device=dev)
                                  for _ in range(CFG.num_hidden_layers)], "paged", S, 16) for _ in range(4)]
    got, _ = ls.llama_stack_decode_loop(x, w, caches[0], cos, sin, CFG, cache_layout="paged", adapter_ids=ids)
    want, run = [], caches[1]
    for t in range(3):
        lg, _, run = ls.llama_stack_decode_step(x[:, t:t + 1], w, run, cos, sin, t, CFG, adapter_ids=ids)
        want.append(lg)
    assert torch.equal(got, torch.cat(want, 1))
    tokens, pos = torch.tensor([3, 5, 7, 11], device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    graph = ls.DecodeGraph(w, caches[2], cos, sin, CFG, tokens, pos, adapter_ids=ids)
    got, order = [graph.first_tokens.clone()], [ids.clone()]
    for _ in range(6):
        ids.copy_(torch.roll(ids, 1))
        order.append(ids.clone())
        got.append(graph.step().clone())
    want, run, t, p = [], caches[3], tokens, pos.clone()
    for step_ids in order:
        h = ls.embed_token_ids(t, w.embedding)
        logits, _, run = ls.llama_stack_decode_step(h, w, run, cos, sin, p, CFG, float_logits=False, adapter_ids=step_ids)
        t, p = ls.greedy_sample(logits), p + 1
        want.append(t)
    assert torch.equal(torch.stack(got), torch.stack(want))
    for a, b in zip(caches[2].layer_caches, run.layer_caches):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_layer_with_part_rotation(dev):
    """An ordinary layer whose ``rotary_dim`` is part of a head, against its reference backend; without the field,
    narrower tables are refused before anything is launched."""
    w, (cos, sin) = _plain_weights(dev, ("qkv", "o"))
    w, part = w.layers[0], build_scaled_rope_tables(CFG.max_position_embeddings, ROTARY, device=dev)
    cache = _filled(dev, 5, 48)[0]
    x = torch.randn(5, 1, CFG.hidden_size, device=dev).half()
    pos = torch.tensor([0, 47, 16, 15, 30], dtype=torch.int32, device=dev)
    for ids in (None, torch.tensor([2, -1, 0, 1, 2], dtype=torch.int32, device=dev)):
        kw = dict(cache_layout="paged", adapter_ids=ids)
        with pytest.raises(ValueError, match="cos and sin must be"):
            ll.llama_layer_decode_step(x, w, cache, *part, pos, CFG, **kw)
        w.rotary_dim = ROTARY
        with pytest.raises(ValueError, match="cos and sin must be"):
            ll.llama_layer_decode_step(x, w, cache, cos, sin, pos, CFG, **kw)
        ref, ref_cache = ll.reference_llama_layer_decode_step(x, w, cache, *part, pos, CFG, **kw)
        got, got_cache = ll.llama_layer_decode_step(x, w, tuple(t.clone() for t in cache), *part, pos, CFG, **kw)
        assert_close(got, ref.float().cpu().numpy(), what="layer")
        for a, b in zip(got_cache[:2], ref_cache[:2]):
            assert_close(a, b.float().cpu().numpy(), what="cache")
        w.rotary_dim = None


def test_graph_refuses_ids_that_it_cannot_read_anew(dev):
    """Adapter ids on the host, as a list or of another shape are refused before the capture begins; int64 ones are read
    anew by every replay."""
    w, (cos, sin) = _weights(dev), _tables(dev)
    tokens, pos = torch.tensor([3, 5], device=dev), torch.zeros(2, dtype=torch.int32, device=dev)

    def cache():
        return ls.LlamaStackCache([ll.init_llama_layer_cache(CFG, 2, 32, cache_layout="paged", device=dev)
                                   for _ in range(CFG.num_hidden_layers)], "paged", 32, 16)

    for ids in ([0, 1], torch.tensor([0, 1]), torch.tensor([0], device=dev), torch.tensor([0.0, 1.0], device=dev)):
        with pytest.raises(ValueError, match="adapter_ids must be"):
            ls.DecodeGraph(w, cache(), cos, sin, CFG, tokens, pos, adapter_ids=ids)
    runs = []
    for dtype in (torch.int32, torch.int64):
        ids = torch.tensor([0, -1], dtype=dtype, device=dev)
        graph = ls.DecodeGraph(w, cache(), cos, sin, CFG, tokens, pos, adapter_ids=ids)
        out = [graph.first_tokens.clone(), graph.step().clone()]
        ids.copy_(torch.tensor([2, 1]))
        runs.append(torch.stack(out + [graph.step().clone() for _ in range(4)]))
    assert torch.equal(*runs)


@pytest.mark.parametrize("kind", ["plain", "norms", "norms at -1"])
def test_steps_with_ended_rows(dev, kind):
    """Rows that a fork has ended (parent -1) stay in the batch at position 0, without pages: nothing is written or read
    for them, their outputs are finite, and the other rows give what they give without them, bit by bit the same whatever
    the ended rows hold.  Layers with head norms take them at position -1 too; ordinary ones refuse that, as the reference does."""
    torch.manual_seed(1)
    w, tables = _plain_weights(dev, ("qkv", "o")) if kind == "plain" else (_weights(dev), _tables(dev))
    P, blocks, NP, L, D = 8, 4, 30, CFG.num_hidden_layers, CFG.head_dim
    pages = [torch.randn(NP, P, CFG.num_key_value_heads, D, device=dev).half() for _ in range(2 * L)]
    table = torch.full((4, blocks), -1, dtype=torch.int32, device=dev)
    table[:, :3] = torch.randperm(NP, device=dev)[:12].reshape(4, 3).int()
    lengths = torch.tensor([21, 9, 17, 24], dtype=torch.int32, device=dev)
    refs = kv_page_ops.count_page_refs(table, NP)
    parents = torch.tensor([2, -1, 0, 2, -1], dtype=torch.int32, device=dev)
    table, lengths, refs, ready = kv_page_ops.fork_kv_sequences(pages, table, lengths, refs, parents)
    live = parents >= 0
    assert all(ready.tolist()) and (table[~live] == -1).all() and not lengths[~live].any()
    x = torch.randn(5, 1, CFG.hidden_size, device=dev).half()
    ids = torch.tensor([0, 1, -1, 2, 0], dtype=torch.int32, device=dev)

    def step(rows, position):
        pool = [t.clone() for t in pages]
        cache = ls.LlamaStackCache([(pool[2 * i], pool[2 * i + 1], table[rows].contiguous()) for i in range(L)], "paged",
                                   blocks * P, P)
        logits, hidden, _ = ls.llama_stack_decode_step(x[rows], w, cache, *tables, position, CFG, adapter_ids=ids[rows])
        return logits, hidden, pool

    position = torch.where(live, lengths, -1) if kind == "norms at -1" else lengths
    all_rows = torch.ones_like(live)
    logits, hidden, pool = step(all_rows, position)
    assert logits.isfinite().all()
    # (a step of fewer rows may take other matvec kernels)
    want_logits, want_hidden, want_pool = step(live, lengths[live])
    for got, want in ((logits[live], want_logits), (hidden[live], want_hidden)):
        assert_close(got.float().cpu().numpy(), want.float().cpu().numpy(), what="live rows")
    written = torch.zeros(NP, P, dtype=torch.bool, device=dev)
    for b in live.nonzero().flatten().tolist():
        written[table[b, int(lengths[b]) // P], int(lengths[b]) % P] = True
    for a, before, b in zip(pool, pages, want_pool):
        assert torch.equal(a[~written], before[~written]) and torch.equal(b[~written], before[~written])
        assert_close(a[written].float().cpu().numpy(), b[written].float().cpu().numpy(), what="new tokens")
    x[~live] = torch.randn_like(x[~live]) * 3
    again = step(all_rows, position)
    assert torch.equal(again[0][live], logits[live]) and all(torch.equal(a, b) for a, b in zip(again[2], pool))
    if kind == "plain":
        with pytest.raises(ValueError, match="positions must be in"):
            step(all_rows, torch.where(live, lengths, -1))
