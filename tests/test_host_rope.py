"""Rotary positions and the q/k norm + rotation + page write on the host: the
tensor-op paths against the 64-bit oracle, the scaled tables, and what is
refused."""

import math

import numpy as np
import pytest
import torch

import mk.gqa_ops as gqa
import mk.rope_ops as rope
from oracle import serving as sv

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of each type


def near(got, want, size, dtype, terms, what):
    """|got - want| <= one rounding of the value + ``terms`` fp32 roundings of what it is a sum of (2^-24 each) and
    half of the smallest fp16 step."""
    got = got.double().cpu().numpy()
    lim = U[dtype] * np.abs(want) + 1.01 * terms * 2.0 ** -24 * size + 2.0 ** -25
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - want).max()))


def rope_size(x, rd, layout):
    x = np.abs(np.asarray(x, np.float64))
    a, b = sv.rope_pairs(rd, layout)
    size = x.copy()
    size[..., a] = size[..., b] = x[..., a] + x[..., b]
    return size


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rd", [16, 10, 2])
def test_reference_rope_layouts(layout, rd):
    torch.manual_seed(rd)
    x = torch.randn(3, 5, 2, 16).to(torch.float16)
    cos, sin = rope.build_scaled_rope_tables(20, rd)
    pos = torch.tensor([[3, 4, 5, 6, 7], [15, 16, 17, 18, 19], [0, -1, 2, -1, -1]], dtype=torch.int32)
    got = rope.reference_apply_rope(x, cos, sin, positions=pos, layout=layout, rotary_dim=rd)
    want = sv.rope(x.numpy(), cos.numpy(), sin.numpy(), pos.numpy(), layout)
    near(got, want, rope_size(x, rd, layout), torch.float16, 4, "each")
    first = rope.apply_rope(x, cos, sin, positions=torch.tensor([3, 15, -1]), layout=layout, rotary_dim=rd,
                            backend="reference")
    pos[2] = -1
    near(first, sv.rope(x.numpy(), cos.numpy(), sin.numpy(), pos.numpy(), layout), rope_size(x, rd, layout),
         torch.float16, 4, "first")


def test_reference_rope_as_before():
    """The reference's own call: interleaved, whole heads, one offset."""
    torch.manual_seed(0)
    x = torch.randn(2, 4, 3, 8).to(torch.bfloat16)
    cos, sin = rope.build_rope_tables(9, 8)
    got = rope.reference_apply_rope(x, cos, sin, 5)
    xe, xo, c, s = x[..., 0::2].float(), x[..., 1::2].float(), cos[5:9].view(1, 4, 1, 4), sin[5:9].view(1, 4, 1, 4)
    want = torch.stack([xe * c - xo * s, xe * s + xo * c], -1).reshape(x.shape).to(x.dtype)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="cos/sin last dim must be D/2=4, got 2"):
        rope.reference_apply_rope(x, cos[:, :2], sin[:, :2])


def test_rope_gradient_through_tensor_ops():
    x = torch.randn(1, 3, 2, 8, dtype=torch.float16, requires_grad=True)
    cos, sin = rope.build_rope_tables(4, 8)
    y = rope.apply_rope(x, cos, sin, layout="half", backend="metal")  # needs more than values: tensor ops, on any device
    y.float().square().sum().backward()
    # a rotation keeps the length: the gradient of |y|^2 is 2x, to three fp16 roundings (y, its gradient, x's) and fp32's
    size = rope_size(x.detach(), 8, "half")
    assert (np.abs(x.grad.double().numpy() - 2 * x.detach().double().numpy()) <= 8 * 2.0 ** -11 * size + 2.0 ** -22).all()


def test_scaled_tables():
    base_c, base_s = rope.build_scaled_rope_tables(64, 8, 500000.0)
    inv = 500000.0 ** (-np.arange(4) / 4)
    angles = np.arange(64)[:, None] * inv
    assert np.abs(base_c.numpy() - np.cos(angles)).max() <= 2.0 ** -24 and base_s.dtype == torch.float32
    # linear: position 4p of the scaled table is position p of the plain one
    c, s = rope.build_scaled_rope_tables(253, 8, 500000.0, scaling={"type": "linear", "factor": 4})
    assert (c[::4] - base_c).abs().max() <= 2.0 ** -23 and (s[::4] - base_s).abs().max() <= 2.0 ** -23
    # ntk: the fastest pair as before, the slowest slowed by the factor
    c, _ = rope.build_scaled_rope_tables(253, 8, 500000.0, scaling={"type": "ntk", "factor": 4})
    assert torch.equal(c[:64, 0], base_c[:, 0]) and (c[::4, 3] - base_c[:, 3]).abs().max() <= 2.0 ** -23
    # llama3: few turns over the original length: slowed; many: as before
    sc = {"type": "llama3", "factor": 8, "low_freq_factor": 1, "high_freq_factor": 4, "original_max_position": 8192}
    c, _ = rope.build_scaled_rope_tables(505, 8, 500000.0, scaling=sc)
    assert torch.equal(c[:64, 0], base_c[:, 0]) and (c[::8, 3] - base_c[:, 3]).abs().max() <= 2.0 ** -23
    # yarn: the same at both ends, times its attention factor
    sc = {"type": "yarn", "factor": 4, "original_max_position": 4096}
    c, s = rope.build_scaled_rope_tables(253, 8, 500000.0, scaling=sc)
    gain = 0.1 * math.log(4) + 1
    assert (c[:64, 0] / gain - base_c[:, 0]).abs().max() <= 2.0 ** -22
    assert (s[::4, 3] / gain - base_s[:, 3]).abs().max() <= 2.0 ** -22
    c, _ = rope.build_scaled_rope_tables(4, 8, scaling=dict(sc, attention_factor=1.0))
    assert c[0].tolist() == [1.0] * 4
    for bad in ({"type": "nope"}, {"type": "linear"}, {"type": "linear", "factor": 0.5}, {"type": "yarn", "factor": 2},
                dict(type="llama3", factor=8, low_freq_factor=4, high_freq_factor=1, original_max_position=8192)):
        with pytest.raises(ValueError):
            rope.build_scaled_rope_tables(4, 8, scaling=bad)
    with pytest.raises(ValueError):
        rope.build_scaled_rope_tables(4, 7)
    with pytest.raises(ValueError):
        rope.build_scaled_rope_tables(0, 8)


def test_rope_refusals():
    x = torch.zeros(2, 3, 4, 16, dtype=torch.float16)
    cos, sin = rope.build_rope_tables(10, 16)
    for kw, exc in ((dict(layout="neox"), ValueError), (dict(rotary_dim=7), ValueError),
                    (dict(rotary_dim=18), ValueError), (dict(rotary_dim=8), ValueError),
                    (dict(position_offset=8), ValueError), (dict(position_offset=-1), ValueError),
                    (dict(positions=torch.tensor([0, 8])), ValueError),
                    (dict(positions=torch.tensor([0, -2])), ValueError),
                    (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError),
                    (dict(positions=torch.zeros(2)), TypeError),
                    (dict(positions=torch.tensor([0, 1]), position_offset=1), ValueError),
                    (dict(backend="cuda"), ValueError)):
        with pytest.raises(exc):
            rope.apply_rope(x, cos, sin, **{"backend": "reference", **kw})
    with pytest.raises(TypeError):
        rope.apply_rope(x.float(), cos, sin, backend="reference")
    with pytest.raises(ValueError, match="ROCm device"):
        rope.apply_rope(x, cos, sin)


def qk_case(seed, T, B, Hq, Hkv, D, rd, P, mb, dtype, norm=True, ragged=False):
    g = torch.Generator().manual_seed(seed)
    NP = B * mb + 2
    c = dict(num_attention_heads=Hq, num_key_value_heads=Hkv, head_dim=D, rotary_dim=rd)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    K, V = (torch.randn(NP, P, Hkv, D, generator=g).to(dtype) for _ in range(2))
    bt = torch.randperm(NP, generator=g)[:B * mb].reshape(B, mb).to(torch.int32)
    cos, sin = rope.build_scaled_rope_tables(mb * P, rd, 500000.0)
    if ragged:
        where = torch.randperm(B * mb * P, generator=g)[:T]  # distinct places, in any order
        seq, pos = (where // (mb * P)).to(torch.int32), (where % (mb * P)).to(torch.int32)
        pos[T // 2] = -1
        c["sequences"] = seq
    else:
        pos = torch.randint(0, mb * P, (T,), generator=g, dtype=torch.int32)
        if T > 2:
            pos[1] = -1
    if norm:
        c["q_weight"], c["k_weight"] = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    return qkv, K, V, bt, cos, sin, pos, c


def check_qk(got, case, dtype, layout, eps=1e-6):
    qkv, K, V, bt, cos, sin, pos, c = case
    Hq, Hkv, D, P = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"], K.shape[1]
    f = lambda t: None if t is None else t.double().numpy()  # noqa: E731
    q, k, v, size = sv.qk_norm_rope(f(qkv), cos.numpy(), sin.numpy(), pos.tolist(), Hq, Hkv, D, f(c.get("q_weight")),
                                    f(c.get("k_weight")), eps, layout)
    # the sum of squares has D roundings, its root halves them; eight more for the root, the weights and the rotation
    terms = D / 2 + 8 if "q_weight" in c else 4
    near(got[0][:, 0], q, size[:, :Hq], dtype, terms, "q")
    wantK, wantV = K.clone(), V.clone()
    limit = torch.zeros(K.shape, dtype=torch.float64)
    seq = c.get("sequences")
    for t in range(len(pos)):
        p, b = int(pos[t]), t if seq is None else int(seq[t])
        page = int(bt[b, p // P]) if 0 <= p < bt.shape[1] * P else -1
        if 0 <= p < len(cos) and 0 <= page < len(K):
            wantK[page, p % P], wantV[page, p % P] = torch.from_numpy(k[t]).to(dtype), qkv[t].reshape(-1, D)[Hq + Hkv:]
            limit[page, p % P] = torch.from_numpy(U[dtype] * np.abs(k[t]) * 2
                                                  + terms * 2.0 ** -24 * size[t, Hq:] + 2.0 ** -24)
    # a k value is one rounding off, and so is the rounded oracle; everything else in the pages is as it was
    assert ((got[1].cpu().double() - wantK.double()).abs() <= limit).all()
    assert torch.equal(got[2].cpu(), wantV)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_reference_qk_norm_rope(layout, ragged, norm):
    T, B = (9, 3) if ragged else (4, 4)
    case = qk_case(5, T, B, 6, 2, 16, 12, 4, 5, torch.float16, norm, ragged)
    qkv, K, V, bt, cos, sin, pos, c = case
    before = K.clone()
    got = gqa.paged_qk_norm_rope_update(qkv, K, V, bt, cos, sin, pos, layout=layout, backend="reference", **c)
    check_qk(got, case, torch.float16, layout)
    assert torch.equal(K, before) and got[0].shape == (T, 1, 6, 16)


def test_reference_qk_as_the_decode_block():
    """Without norms, interleaved over whole heads: what paged_gqa_decode_block_from_qkv writes."""
    qkv, K, V, bt, cos, sin, pos, c = qk_case(6, 2, 2, 4, 2, 16, 16, 4, 3, torch.float16, False)
    _, K1, V1 = gqa.paged_gqa_decode_block_from_qkv(qkv[:, None], K, V, bt, cos, sin, pos, num_attention_heads=4,
                                                    num_key_value_heads=2, head_dim=16, backend="reference")
    _, K2, V2 = gqa.paged_qk_norm_rope_update(qkv.reshape(2, 1, 8, 16), K, V, bt, cos, sin, pos, backend="reference", **c)
    assert torch.equal(K1, K2) and torch.equal(V1, V2)


def test_qk_refusals():
    qkv, K, V, bt, cos, sin, pos, c = qk_case(7, 3, 3, 4, 2, 16, 8, 4, 3, torch.float16)
    ok = dict(qkv=qkv, K_pages=K, V_pages=V, block_table=bt, cos=cos, sin=sin, position=pos, backend="reference", **c)
    gqa.paged_qk_norm_rope_update(**ok)
    w = c["q_weight"]
    bad = [dict(qkv=qkv[:, :-1]), dict(num_attention_heads=3), dict(layout="x"), dict(rotary_dim=6), dict(rotary_dim=20),
           dict(K_pages=K[..., :8]), dict(V_pages=V[:-1]), dict(cos=cos[:, :2]), dict(sin=sin[:-1]),
           dict(q_weight=None), dict(q_weight=w[:-1]), dict(position=pos[:-1]), dict(position=12), dict(position=-2),
           dict(position=pos.float()), dict(block_table=bt[:2]), dict(block_table=bt[0]), dict(backend="x"),
           dict(sequences=torch.tensor([0, 1])), dict(sequences=torch.tensor([0, 1, 3])),
           dict(sequences=torch.tensor([0, -1, 1])),
           dict(sequences=torch.tensor([1, 1, 2]), position=torch.tensor([5, 5, 5]))]
    for kw in bad:
        with pytest.raises(ValueError):
            gqa.paged_qk_norm_rope_update(**{**ok, **kw})
    for kw in (dict(qkv=qkv.float()), dict(K_pages=K.float(), V_pages=V.float()), dict(V_pages=V.bfloat16()),
               dict(q_weight=w.double(), k_weight=w.double()), dict(q_weight=w.float())):
        with pytest.raises(TypeError):
            gqa.paged_qk_norm_rope_update(**{**ok, **kw})
    with pytest.raises(RuntimeError, match="records no gradient"):
        gqa.paged_qk_norm_rope_update(**{**ok, "backend": "auto", "qkv": qkv.clone().requires_grad_()})
    with pytest.raises(ValueError, match="ROCm device"):
        gqa.paged_qk_norm_rope_update(**{**ok, "backend": "auto"})


@pytest.mark.parametrize("T,ragged", [(65536, False), (2 ** 24, True)])
def test_qk_row_limits(T, ragged):
    z = lambda *shape: torch.zeros(1, dtype=torch.float16).expand(*shape)  # noqa: E731
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="at most"):
        gqa.paged_qk_norm_rope_update(z(T, 6), z(1, 1, 1, 2).contiguous(), z(1, 1, 1, 2).contiguous(),
                                      one.expand(1 if ragged else T, 1), torch.ones(1, 1), torch.ones(1, 1),
                                      one.expand(T), sequences=one.expand(T) if ragged else None,
                                      num_attention_heads=1, num_key_value_heads=1, head_dim=2)


@pytest.mark.parametrize("name", ["qkv", "K_pages", "V_pages", "cos", "sin", "q_weight", "k_weight"])
def test_qk_records_no_gradient_of_any_input(name):
    """Every floating input that records a gradient is refused, not only the rows and the norm weights."""
    qkv, K, V, bt, cos, sin, pos, c = qk_case(7, 3, 3, 4, 2, 16, 8, 4, 3, torch.float16)
    ok = dict(qkv=qkv, K_pages=K, V_pages=V, block_table=bt, cos=cos, sin=sin, position=pos, **c)
    ok[name] = ok[name].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="records no gradient"):
        gqa.paged_qk_norm_rope_update(**ok)
    with torch.no_grad(), pytest.raises(ValueError, match="ROCm device"):
        gqa.paged_qk_norm_rope_update(**ok)


def test_qk_one_position_for_all_rows():
    """An int, a number of numpy's and a tensor without dimensions are one position for every row."""
    qkv, K, V, bt, cos, sin, _, c = qk_case(8, 3, 3, 4, 2, 16, 8, 4, 3, torch.float16)
    outs = [gqa.paged_qk_norm_rope_update(qkv, K, V, bt, cos, sin, position, backend="reference", **c)
            for position in ([5, 5, 5], 5, np.int64(5), torch.tensor(5), torch.tensor(5, dtype=torch.int32))]
    for out in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))
    for bad in (torch.tensor(12), torch.tensor(-2), torch.tensor(1.0), torch.tensor([5]), [5]):
        with pytest.raises(ValueError, match="position must be"):
            gqa.paged_qk_norm_rope_update(qkv, K, V, bt, cos, sin, bad, backend="reference", **c)


def test_rope_of_padding_alone():
    """A batch whose sequences are all padding is zeros, also where they are longer than the tables."""
    cos, sin = rope.build_rope_tables(4, 8)
    x = torch.ones(2, 9, 1, 8).half()
    for pos in (torch.tensor([-1, -1]), torch.full((2, 9), -1)):
        assert not rope.apply_rope(x, cos, sin, positions=pos, backend="reference").any()
    for pos in (torch.tensor([-1, 0]), torch.tensor([-1, -2]), torch.full((2, 9), 4)):
        with pytest.raises(ValueError, match="positions must be in"):
            rope.apply_rope(x, cos, sin, positions=pos, backend="reference")


def test_scaled_tables_between_the_ends():
    """The pairs on the ramps of llama3 and yarn, worked out by hand from their definitions.

    llama3, theta 10000, d 8, factor 8, 1 to 4 turns over 128 positions: pair 1 (0.1 a position) turns 12.8 / 2 pi =
    2.0371833 times, so 1.0371833 / 3 = 0.34572776 of its frequency stays and the rest is divided by 8: 0.1 (0.34572776 +
    0.65427224 / 8 = 0.08178403) = 0.042751179.  Pair 0 (20.4 turns) stays, pairs 2 and 3 (0.2 and 0.02) are divided.

    yarn, theta 10000, d 16, factor 4, 4096 positions: the pairs of 32 turns and of one are 16 ln(4096 / 64 pi) / (2 ln
    10000) = 2.62 and 16 ln(4096 / 2 pi) / (2 ln 10000) = 5.63, outwards 2 and 6; pair i in between keeps 1 - 0.75 (i - 2)
    / 4 of 10000^(-i / 8), and cos and sin are multiplied by 0.1 ln 4 + 1."""
    cases = [(8, {"type": "llama3", "factor": 8, "low_freq_factor": 1, "high_freq_factor": 4,
                  "original_max_position": 128}, [1.0, 0.042751179, 0.00125, 0.000125], 1.0),
             (16, {"type": "yarn", "factor": 4, "original_max_position": 4096},
              [1.0, 0.31622777, 0.1, 0.031622777 * 0.8125, 0.01 * 0.625, 0.0031622777 * 0.4375, 0.00025,
               0.00031622777 / 4], 1.13862944)]
    for d, scaling, inv, gain in cases:
        c, s = rope.build_scaled_rope_tables(41, d, 10000.0, scaling=scaling)
        for p in (1, 7, 40):
            angles = p * np.array(inv)
            # eight digits of a frequency, and the table's rounding
            lim = 40 * 2e-8 * np.maximum(np.array(inv), 1e-3) * gain + 2.0 ** -24 * gain
            assert (np.abs(c[p].numpy() - gain * np.cos(angles)) <= lim).all(), (scaling, p)
            assert (np.abs(s[p].numpy() - gain * np.sin(angles)) <= lim).all(), (scaling, p)


def test_qk_refuses_tangents():
    """A forward-mode tangent would be lost by the kernel as a gradient would."""
    import torch.autograd.forward_ad as fwad

    qkv, K, V, bt, cos, sin, pos, c = qk_case(7, 3, 3, 4, 2, 16, 8, 4, 3, torch.float16)
    with fwad.dual_level():
        for name in ("qkv", "cos", "q_weight"):
            ok = dict(qkv=qkv, K_pages=K, V_pages=V, block_table=bt, cos=cos, sin=sin, position=pos, **c)
            ok[name] = fwad.make_dual(ok[name], torch.ones_like(ok[name]))
            with torch.no_grad(), pytest.raises(RuntimeError, match="records no gradient"):
                gqa.paged_qk_norm_rope_update(**ok)
        with pytest.raises(ValueError, match="ROCm device"):
            gqa.paged_qk_norm_rope_update(qkv, K, V, bt, cos, sin, pos, **c)
