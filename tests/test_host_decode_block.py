"""Host (CPU tensor) side of the decode-block callers from a packed qkv row:
``paged_decode_block_from_qkv`` (ops/decode_block_ops.py:174-257) and
``gqa_decode_block_from_qkv`` (ops/gqa_ops.py:345-444).  Their 'reference'
backends against the oracle's composition, the MHA/GQA routing, and the
validation messages the reference raises.  No GPU."""

import numpy as np
import pytest
import torch

import mk.decode_block_ops as dbo
import mk.gqa_ops as gqa
from oracle import paged as op
from tests._data import assert_close


def _f16(a):
    return a.astype(np.float16).astype(np.float32)


def _case(seed, B, H, D, P, mb):
    rng = np.random.default_rng(seed)
    NP = B * mb
    Kp = rng.standard_normal((NP, P, H, D)).astype(np.float16)
    Vp = rng.standard_normal((NP, P, H, D)).astype(np.float16)
    bt = rng.permutation(NP).astype(np.int32).reshape(B, mb)
    pos = rng.integers(0, mb * P, size=B)
    return rng, Kp, Vp, bt, pos


@pytest.mark.parametrize("layout", ["packed", "explicit"])
@pytest.mark.parametrize("int_pos", [False, True])
def test_reference_paged_block_mha_matches_oracle(layout, int_pos):
    B, H, D, P, mb = 3, 4, 16, 4, 3
    rng, Kp, Vp, bt, pos = _case(11, B, H, D, P, mb)
    if int_pos:
        pos[:] = 5
    qkv = rng.standard_normal((B, 1, 3 * H * D)).astype(np.float16)
    cos, sin = op.rope_tables(mb * P, D, 10000.0)
    t = torch.from_numpy
    q_in = t(qkv) if layout == "packed" else t(qkv).reshape(B, 1, 3, H, D)
    kw = dict(H=H, D=D) if layout == "packed" else {}
    position = 5 if int_pos else t(pos)
    out, K1, V1 = dbo.paged_decode_block_from_qkv(q_in, t(Kp), t(Vp), t(bt), t(cos), t(sin), position,
                                                  backend="reference", **kw)
    q, k, v = op.qkv_split_rope(qkv[:, 0], cos, sin, pos, H, H, D)
    rK, rV = op.paged_kv_update(Kp, Vp, k, v, bt, pos)
    assert np.array_equal(K1.numpy(), rK) and np.array_equal(V1.numpy(), rV)
    ref = op.paged_attention(q.astype(np.float32), rK, rV, bt, pos + 1)
    assert_close(out[:, 0], ref, what="reference paged block", extra=1e-3)
    assert tuple(out.shape) == (B, 1, H, D) and out.dtype == torch.float16


def test_reference_paged_block_routes_gqa():
    B, Hq, Hkv, D, P, mb = 2, 8, 2, 16, 4, 3
    rng, Kp, Vp, bt, pos = _case(12, B, Hkv, D, P, mb)
    qkv = rng.standard_normal((B, 1, (Hq + 2 * Hkv) * D)).astype(np.float16)
    cos, sin = op.rope_tables(mb * P, D, 500000.0)
    t = torch.from_numpy
    out, K1, _ = dbo.paged_decode_block_from_qkv(t(qkv), t(Kp), t(Vp), t(bt), t(cos), t(sin), t(pos), H=Hq,
                                                 backend="reference")
    q, k, v = op.qkv_split_rope(qkv[:, 0], cos, sin, pos, Hq, Hkv, D)
    rK, rV = op.paged_kv_update(Kp, Vp, k, v, bt, pos)
    assert np.array_equal(K1.numpy(), rK)
    assert_close(out[:, 0], op.paged_attention(q.astype(np.float32), rK, rV, bt, pos + 1), what="gqa route",
                 extra=1e-3)


def test_reference_contiguous_gqa_block_matches_oracle():
    B, Hq, Hkv, D, S = 2, 8, 2, 16, 24
    rng = np.random.default_rng(13)
    K = rng.standard_normal((B, S, Hkv, D)).astype(np.float16)
    V = rng.standard_normal((B, S, Hkv, D)).astype(np.float16)
    qkv = rng.standard_normal((B, 1, (Hq + 2 * Hkv) * D)).astype(np.float16)
    cos, sin = op.rope_tables(S, D, 500000.0)
    pos = np.array([0, 23])
    t = torch.from_numpy
    for fn in (gqa.reference_gqa_decode_block_from_qkv,
               lambda *a, **k: gqa.gqa_decode_block_from_qkv(*a, backend="reference", **k)):
        Kt, Vt = t(K.copy()), t(V.copy())
        out, K1, V1 = fn(t(qkv), Kt, Vt, t(cos), t(sin), t(pos), num_attention_heads=Hq, num_key_value_heads=Hkv,
                         head_dim=D)
        assert np.array_equal(Kt.numpy(), K)  # functional: the inputs stay
        q, k, v = op.qkv_split_rope(qkv[:, 0], cos, sin, pos, Hq, Hkv, D)
        rK, rV = op.contiguous_update(K, V, k, v, pos)
        assert np.array_equal(K1.numpy(), rK) and np.array_equal(V1.numpy(), rV)
        assert_close(out[:, 0], op.contiguous_attention(q.astype(np.float32), rK, rV, pos + 1),
                     what="contiguous gqa block", extra=1e-3)


def test_paged_block_validation_messages():
    t = torch.zeros
    K = t(6, 4, 2, 16, dtype=torch.float16)
    bt = torch.zeros(2, 3, dtype=torch.int32)
    cos = sin = t(12, 8)
    qkv = t(2, 1, 3 * 2 * 16, dtype=torch.float16)
    with pytest.raises(ValueError, match="K_pages and V_pages must be matching"):
        dbo.paged_decode_block_from_qkv(qkv, K, K[:, :2], bt, cos, sin, 0, H=2, D=16)
    with pytest.raises(ValueError, match="block_table must be"):
        dbo.paged_decode_block_from_qkv(qkv, K, K, bt[0], cos, sin, 0, H=2, D=16)
    with pytest.raises(ValueError, match="H and D are required"):
        dbo.paged_decode_block_from_qkv(qkv, K, K, bt, cos, sin, 0)
    with pytest.raises(ValueError, match="3\\*H\\*D"):
        dbo.paged_decode_block_from_qkv(qkv[..., :-16], K, K, bt, cos, sin, 0, H=2, D=16)
    with pytest.raises(TypeError, match="qkv dtype"):
        dbo.paged_decode_block_from_qkv(qkv.float(), K, K, bt, cos, sin, 0, H=2, D=16)
    # the reference's split step takes only these names; its attention step rejects the GQA ones
    with pytest.raises(ValueError, match="'reference', 'metal', 'auto'"):
        dbo.paged_decode_block_from_qkv(qkv, K, K, bt, cos, sin, 0, H=2, D=16, backend="metal_threadgroup")
    with pytest.raises(ValueError, match="metal_d128"):
        dbo.paged_decode_block_from_qkv(qkv, K, K, bt, cos, sin, 0, H=2, D=16, backend="metal_gqa")
    with pytest.raises(ValueError, match="must normalize to"):
        dbo.paged_decode_block_from_qkv(t(2, 1, 3, 2, 8, dtype=torch.float16), K, K, bt, cos, sin, 0)
    with pytest.raises(ValueError, match="metal_gqa_threadgroup"):  # GQA route, unknown backend
        dbo.paged_decode_block_from_qkv(qkv, K, K, bt, cos, sin, 0, H=4, D=16, backend="bogus")


def test_contiguous_gqa_block_validation_messages():
    K = torch.zeros(2, 8, 2, 16, dtype=torch.float16)
    qkv = torch.zeros(2, 1, 8 * 16, dtype=torch.float16)
    cos = sin = torch.zeros(8, 8)
    kw = dict(num_attention_heads=4, num_key_value_heads=2, head_dim=16)
    with pytest.raises(ValueError, match="metal_gqa_threadgroup"):
        gqa.gqa_decode_block_from_qkv(qkv, K, K, cos, sin, 0, backend="metal_d64", **kw)
    with pytest.raises(ValueError, match="divisible"):
        gqa.gqa_decode_block_from_qkv(qkv, K, K, cos, sin, 0, num_attention_heads=3, num_key_value_heads=2,
                                      head_dim=16)
    with pytest.raises(ValueError, match="matching"):
        gqa.gqa_decode_block_from_qkv(qkv, K, K[:1], cos, sin, 0, **kw)
    with pytest.raises(ValueError, match="cache batch/head/head_dim"):
        gqa.gqa_decode_block_from_qkv(qkv[:1], K, K, cos, sin, 0, **kw)


def test_adapters_refuse_gradients_beside_kernels():
    """With adapters the kernels' backends take no input that records a gradient: the result would have the adapters'
    part of it alone.  The reference backends are tensor ops throughout and give all of it."""
    from mk.lora_ops import LoraAdapters
    from mk.quantized_decode_block_ops import paged_quantized_decode_block

    g = torch.Generator().manual_seed(3)
    B, H, Hkv, D, K, P = 2, 2, 1, 16, 32, 4
    N = (H + 2 * Hkv) * D
    w = lambda n, k: torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)  # noqa: E731
    sc = lambda n, k: (0.02 * torch.rand(n, k // 32, generator=g)).half()  # noqa: E731
    rand = lambda *s: torch.randn(*s, generator=g).half()  # noqa: E731
    cos, sin = (torch.randn(12, D // 2, generator=g) for _ in range(2))
    lora = lambda n, k: LoraAdapters(rand(1, 4, k) / 4, rand(1, n, 4) / 4, torch.ones(1))  # noqa: E731
    x, qkv_lora, out_lora = rand(B, 1, K), lora(N, K), lora(K, H * D)
    args = (w(N, K), sc(N, K), w(K, H * D), sc(K, H * D), rand(6, P, Hkv, D), rand(6, P, Hkv, D),
            torch.arange(6, dtype=torch.int32).reshape(2, 3), cos, sin, torch.tensor([5, 2]))
    kw = dict(H=H, num_key_value_heads=Hkv, head_dim=D, qkv_lora=qkv_lora, out_lora=out_lora,
              adapter_ids=torch.tensor([0, -1], dtype=torch.int32))
    leaves = [x, qkv_lora.a, qkv_lora.b, qkv_lora.scales, out_lora.a, out_lora.b, out_lora.scales]
    for leaf in leaves:
        leaf.requires_grad_()
        for backends in ({}, dict(matvec_backend="reference"), dict(block_backend="reference")):
            with pytest.raises(RuntimeError, match="record no gradient"):
                paged_quantized_decode_block(x, *args, **kw, **backends)
        with torch.no_grad(), pytest.raises(ValueError, match="ROCm device"):
            paged_quantized_decode_block(x, *args, **kw)
        leaf.requires_grad_(False)
    for leaf in leaves:
        leaf.requires_grad_()
    y, _, _ = paged_quantized_decode_block(x, *args, **kw, matvec_backend="reference", block_backend="reference")
    y.float().sum().backward()
    assert all(leaf.grad.abs().sum() > 0 for leaf in leaves)
    assert (x.grad[1] != 0).any()  # the row without an adapter: through the projections and the attention


def test_tables_of_another_width_are_refused():
    """The page writes' kernels read D/2 angles a row: tables of another width, or of two shapes, never reach them."""
    import mk.paged_quantized_kv_ops as pq
    from mk.quantized_decode_block_ops import rmsnorm_qkv_rope_paged_update

    B, Hq, Hkv, D, P, K = 2, 2, 1, 32, 4, 32
    N = (Hq + 2 * Hkv) * D
    Kp, Vp = torch.zeros(2, 6, P, Hkv, D).half()
    bt, pos = torch.arange(6, dtype=torch.int32).reshape(2, 3), torch.tensor([5, 2])
    kw = dict(num_attention_heads=Hq, num_key_value_heads=Hkv, head_dim=D)
    cache = pq.quantize_kv_pages(Kp, Vp, bt, torch.tensor([6, 3]), pq.PagedQuantizedKVConfig(page_size=P))
    w, sc = torch.zeros(N, K // 2, dtype=torch.uint8), torch.ones(N, K // 32).half()
    qkv = torch.zeros(B, 1, N).half()
    calls = [lambda c, s: gqa.paged_gqa_decode_block_from_qkv(qkv, Kp, Vp, bt, c, s, pos, **kw),
             lambda c, s: rmsnorm_qkv_rope_paged_update(torch.zeros(B, K).half(), torch.ones(K).half(), w, sc, None, Kp,
                                                        Vp, bt, c, s, pos, **kw),
             lambda c, s: pq.paged_quantized_kv_update_from_qkv(qkv, cache, c, s, pos, **kw)]
    cos = torch.ones(12, D // 2)
    for call in calls:
        for c, s in ((cos[:, :8], cos[:, :8]), (cos, cos[:, :8]), (cos, cos[:5]), (torch.ones(12, D), torch.ones(12, D)),
                     (cos[0], cos[0])):
            with pytest.raises(ValueError, match="cos and sin must be"):
                call(c, s)
        with pytest.raises(ValueError, match="ROCm device"):
            call(cos, cos)


def test_layer_tables_say_no_more_than_its_weights():
    """An ordinary layer takes tables of whole heads only; part of a head turns where ``rotary_dim`` says so, or where
    head norms or the half layout leave it to the tables."""
    from mk import llama_layer_ops as ll

    cfg = ll.LlamaLikeConfig(hidden_size=64, intermediate_size=128, num_attention_heads=2, num_key_value_heads=1,
                             head_dim=32, num_hidden_layers=1, max_position_embeddings=16, vocab_size=64).validate()
    g = torch.Generator().manual_seed(1)
    linears = {}
    for name, n, k in (("qkv", 128, 64), ("o", 64, 64), ("gate", 128, 64), ("up", 128, 64), ("down", 64, 128)):
        linears[name + "_w"] = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
        linears[name + "_scales"] = (0.02 * (1 + torch.rand(n, k // 32, generator=g))).half()
        linears[name + "_zeros"] = torch.full((n, k // 32), 8.0).half()
    w = ll.LlamaLayerKernelWeights(input_layernorm_weight=torch.ones(64).half(),
                                   post_attention_layernorm_weight=torch.ones(64).half(), **linears)
    cos, sin = ll.build_rope_tables(cfg)
    part = cos[:, :8].contiguous(), sin[:, :8].contiguous()
    cache = ll.init_llama_layer_cache(cfg, 2, 16, cache_layout="contiguous", device="cpu")
    x = torch.randn(2, 1, 64, generator=torch.Generator().manual_seed(0)).half()
    ends = torch.ones(16, 8), torch.zeros(16, 8)  # angles of pairs 8 .. 15: they stay

    def step(tables):
        return ll.reference_llama_layer_decode_step(x, w, cache, *tables, 3, cfg, cache_layout="contiguous")

    whole, _ = step((cos, sin))
    for c, s in (part, (torch.cat([cos, cos], 1), torch.cat([sin, sin], 1))):
        with pytest.raises(ValueError):
            step((c, s))
        with pytest.raises(ValueError):
            ll.llama_layer_decode_step(x, w, cache, c, s, 3, cfg, cache_layout="contiguous")
    w.rotary_dim = 16
    got, (K, _) = step(part)
    with pytest.raises(ValueError, match="cos and sin must be"):
        step((cos, sin))
    w.rotary_dim = 32
    assert torch.equal(step((cos, sin))[0], whole)
    with pytest.raises(ValueError):
        step(part)
    w.rotary_dim = None
    want, (Kw, _) = step((torch.cat([part[0], ends[0]], 1), torch.cat([part[1], ends[1]], 1)))
    assert torch.equal(got, want) and torch.equal(K, Kw) and not torch.equal(got, whole)
    w.rope_layout = "half"
    half, _ = step(part)
    w.rotary_dim = 16
    assert torch.equal(step(part)[0], half)
