"""mk_apply_rope and mk_qk_norm_rope_paged_update against the 64-bit oracle:
both layouts, parts of heads, strides and alignments of both kernels, empty
rows, other streams and graph replays."""

import numpy as np
import pytest
import torch

import mk.gqa_ops as gqa
import mk.rope_ops as rope
from oracle import serving as sv
from tests.test_host_rope import check_qk, near, qk_case, rope_size

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def check_rope(x, cos, sin, pos, layout, rd, got):
    want = sv.rope(x.double().cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), pos, layout)
    near(got, want, rope_size(x.double().cpu().numpy(), rd, layout), x.dtype, 4, (tuple(x.shape), rd, layout))
    assert got.is_contiguous() and got.dtype == x.dtype


# (B, S, H, D, rotary_dim): units of 16 values; one unit; parts of a head in and outside of whole units; odd halves
SHAPES = [(1, 1, 32, 128, 128), (2, 7, 3, 64, 32), (1, 5, 2, 16, 16), (3, 2, 5, 80, 80), (2, 3, 2, 256, 96),
          (2, 3, 2, 64, 24), (1, 4, 3, 20, 20), (2, 2, 2, 6, 2), (1, 3, 1, 7, 4), (1, 300, 9, 128, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,S,H,D,rd", SHAPES)
def test_apply_rope(dev, B, S, H, D, rd, layout, dtype):
    g = torch.Generator().manual_seed(B * 1000 + S * 100 + D + rd)
    x = torch.randn(B, S, H, D, generator=g).to(dtype).to(dev)
    cos, sin = rope.build_scaled_rope_tables(S + 40, rd, 500000.0, device=dev)
    each = torch.randint(-1, S + 40, (B, S), generator=g, dtype=torch.int32)
    got = rope.apply_rope(x, cos, sin, positions=each.to(dev), layout=layout, rotary_dim=rd)
    check_rope(x, cos, sin, each.numpy(), layout, rd, got)
    first = torch.randint(0, 41, (B,), generator=g, dtype=torch.int32)
    first[-1] = 40 if B == 1 else -1
    pos = np.where(first.numpy()[:, None] < 0, -1, first.numpy()[:, None] + np.arange(S))
    check_rope(x, cos, sin, pos, layout, rd,
               rope.apply_rope(x, cos, sin, positions=first.to(dev), layout=layout, rotary_dim=rd))
    pos = np.broadcast_to(40 + np.arange(S), (B, S))
    check_rope(x, cos, sin, pos, layout, rd, rope.apply_rope(x, cos, sin, 40, layout=layout, rotary_dim=rd))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_apply_rope_strides(dev, layout):
    """Views: heads of a packed row, an odd offset (no 16-byte addresses), a transposed cache, an expanded one, a
    strided last dimension; tables off a 16-byte boundary, in fp16 and on the host."""
    g = torch.Generator().manual_seed(3)
    cos, sin = rope.build_scaled_rope_tables(30, 32, device=dev)
    pos = np.broadcast_to(4 + np.arange(5), (2, 5))
    packed = torch.randn(2, 5, 9, 64, generator=g).half().to(dev)
    flat = torch.randn(2 * 5 * 3 * 64 + 1, generator=g).half().to(dev)
    views = [packed[:, :, 2:6], flat[1:].view(2, 5, 3, 64), packed.transpose(1, 2)[:, 1:6].transpose(1, 2)[:, :, :5],
             packed[:1].expand(2, 5, 9, 64), packed[:, :, :1].expand(2, 5, 4, 64),
             torch.randn(2, 5, 64, 3, generator=g).half().to(dev).transpose(2, 3), packed[..., ::2][..., :32].contiguous()]
    for x in views:
        rd = min(32, x.shape[3])
        got = rope.apply_rope(x, cos, sin, 4, layout=layout, rotary_dim=rd)
        check_rope(x, cos, sin, pos, layout, rd, got)
    x = views[0]
    want = rope.apply_rope(x, cos, sin, 4, layout=layout, rotary_dim=32)
    off = [torch.empty(30 * 16 + 1, device=dev)[1:].view(30, 16) for _ in range(2)]
    off[0].copy_(cos), off[1].copy_(sin)
    near(rope.apply_rope(x, *off, 4, layout=layout, rotary_dim=32), want.double().cpu().numpy(),
         rope_size(x.double().cpu().numpy(), 32, layout), torch.float16, 4, "tables off a boundary")
    assert torch.equal(rope.apply_rope(x, cos.cpu(), sin.cpu(), 4, layout=layout, rotary_dim=32), want)
    check_rope(x, cos.half().float(), sin.half().float(), pos, layout, 32,
               rope.apply_rope(x, cos.half(), sin.half(), 4, layout=layout, rotary_dim=32))
    for shape in ((0, 5, 3, 64), (2, 0, 3, 64), (2, 5, 0, 64)):
        empty = rope.apply_rope(torch.empty(shape, dtype=torch.float16, device=dev), cos, sin, rotary_dim=32)
        assert tuple(empty.shape) == shape


def test_apply_rope_values_past_the_rotation(dev):
    """Infinities, NaNs and the smallest values of the copied part come back bit by bit; a NaN stays in its pair."""
    x = torch.randn(1, 2, 2, 64, device=dev).half()
    x[..., 40], x[..., 41], x[..., 42], x[0, 0, 0, 3] = float("inf"), float("nan"), 6e-8, float("nan")
    cos, sin = rope.build_scaled_rope_tables(4, 32, device=dev)
    for layout, partner in (("half", 19), ("interleaved", 2)):
        y = rope.apply_rope(x, cos, sin, 1, layout=layout, rotary_dim=32)
        assert torch.equal(y[..., 32:].view(torch.int16), x[..., 32:].view(torch.int16))
        assert y[..., :32].isnan().nonzero().tolist() == sorted([[0, 0, 0, 3], [0, 0, 0, partner]])


def test_rope_unread_positions(dev, monkeypatch):
    """Where the host does not read positions back, rows outside of the tables come back zero."""
    monkeypatch.setenv("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
    x = torch.randn(2, 3, 2, 32, device=dev).half()
    cos, sin = rope.build_scaled_rope_tables(6, 32, device=dev)
    big = torch.tensor([[0, 6, 5], [2 ** 31 - 1, -2 ** 31, 3]], dtype=torch.int32)
    got = rope.apply_rope(x, cos, sin, positions=big.to(dev))
    check_rope(x, cos, sin, np.array([[0, -1, 5], [-1, -1, 3]]), "interleaved", 32, got)
    got = rope.apply_rope(x, cos, sin, positions=torch.tensor([5, 2 ** 31 - 1], dtype=torch.int32, device=dev))
    check_rope(x, cos, sin, np.array([[5, -1, -1], [-1, -1, -1]]), "interleaved", 32, got)


# (T, B, Hq, Hkv, D, rotary_dim, P, blocks): lanes of a head 1 .. 64; heads not in whole workgroups; sizes off 16
QK = [(1, 1, 32, 8, 128, 128, 16, 4), (3, 3, 8, 1, 64, 32, 4, 5), (5, 5, 7, 7, 16, 16, 3, 4), (2, 2, 6, 2, 80, 80, 16, 2),
      (4, 4, 4, 2, 256, 64, 8, 3), (2, 2, 3, 1, 1024, 1024, 2, 2), (2, 2, 2, 1, 1040, 16, 2, 2), (3, 3, 4, 2, 20, 20, 4, 3),
      (3, 3, 4, 2, 64, 24, 4, 3), (33, 33, 4, 4, 64, 64, 1, 6)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("shape", QK)
def test_qk_decode(dev, shape, norm, layout, dtype):
    case = qk_case(sum(shape), *shape, dtype, norm)
    qkv, K, V, bt, cos, sin, pos, c = case
    d = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    Kd, Vd = K.to(dev), V.to(dev)
    got = gqa.paged_qk_norm_rope_update(d(qkv), Kd, Vd, d(bt), d(cos), d(sin), d(pos), layout=layout,
                                        **{k: d(v) for k, v in c.items()})
    assert got[1] is Kd and got[2] is Vd and got[0].shape == (shape[0], 1, shape[2], shape[4])
    check_qk(got, case, dtype, layout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(9, 3, 6, 2, 16, 16, 4, 5), (70, 4, 8, 2, 128, 64, 16, 2), (40, 2, 4, 1, 20, 12, 5, 6),
                                   (1, 2, 4, 4, 64, 64, 8, 2)])
def test_qk_prompt_rows(dev, shape, dtype):
    case = qk_case(sum(shape), *shape, dtype, True, True)
    qkv, K, V, bt, cos, sin, pos, c = case
    d = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    kw = {k: d(v) for k, v in c.items()}
    check_qk(gqa.paged_qk_norm_rope_update(d(qkv), d(K), d(V), d(bt), d(cos), d(sin), d(pos), layout="half", **kw),
             case, dtype, "half")
    # rows of a wider fused projection, at a stride
    wide = torch.zeros(len(qkv), qkv.shape[1] + 24, dtype=dtype, device=dev)
    wide[:, 8:-16] = qkv.to(dev)
    check_qk(gqa.paged_qk_norm_rope_update(wide[:, 8:-16], d(K), d(V), d(bt), d(cos), d(sin), d(pos), layout="half",
                                           **kw), case, dtype, "half")
    # norm weights in fp32, position and sequences in int64 and on the host
    kw["q_weight"], kw["k_weight"] = kw["q_weight"].float(), kw["k_weight"].float()
    kw["sequences"] = c["sequences"].long()
    check_qk(gqa.paged_qk_norm_rope_update(d(qkv), d(K), d(V), d(bt), d(cos), d(sin), pos.long(), layout="half", **kw),
             case, dtype, "half")


def test_qk_same_slot_and_bad_pages(dev, monkeypatch):
    """The later of two decode rows of one slot wins; page ids outside of the pages and positions past the table are
    not written; empty rows leave q zero."""
    monkeypatch.setenv("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
    T, P = 300, 4
    case = qk_case(11, T, T, 2, 1, 32, 32, P, 3, torch.float16)
    qkv, K, V, bt, cos, sin, pos, c = case
    bt[5], bt[250], bt[251] = bt[299], bt[17], bt[17]
    pos[5] = pos[299]
    pos[17], pos[250], pos[251] = 7, 7, 7
    bt[20, :], bt[21, :], pos[22], pos[23] = -7, 2 ** 30, 12, 2 ** 31 - 1
    d = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    got = gqa.paged_qk_norm_rope_update(d(qkv), d(K), d(V), d(bt), d(cos), d(sin), d(pos), layout="half",
                                        **{k: d(v) for k, v in c.items()})
    check_qk(got, case, torch.float16, "half")
    seq = torch.arange(T, dtype=torch.int32)
    seq[30], seq[31], pos[250], pos[251], pos[5] = -1, T, -1, -1, -1
    case[-1]["sequences"] = seq
    got = gqa.paged_qk_norm_rope_update(d(qkv), d(K), d(V), d(bt), d(cos), d(sin), d(pos), layout="half",
                                        **{k: d(v) for k, v in case[-1].items()})
    for t in (30, 31):
        assert (got[0][t] == 0).all()
        pos[t] = -1
    check_qk(got, case, torch.float16, "half")


def test_qk_contiguous_cache_and_empty(dev):
    from mk import _contig

    qkv, K, V, bt, cos, sin, pos, c = qk_case(12, 3, 3, 4, 2, 64, 64, 16, 2, torch.bfloat16)
    d = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    cache = [torch.randn(3, 32, 2, 64, device=dev).bfloat16() for _ in range(2)]
    pages = [_contig.as_pages(t, 16) for t in cache]
    before = [t.clone().cpu() for t in pages]
    table = _contig.identity_table(3, 32, 16, dev)
    kw = {k: d(v) for k, v in c.items()}
    got = gqa.paged_qk_norm_rope_update(d(qkv), *pages, table, d(cos), d(sin), d(pos), **kw)
    check_qk(got, (qkv, *before, table.cpu(), cos, sin, pos, c), torch.bfloat16, "interleaved")
    none = gqa.paged_qk_norm_rope_update(d(qkv)[:0], *pages, table[:0], d(cos), d(sin), d(pos)[:0], **kw)
    assert none[0].shape == (0, 1, 4, 64)


def test_qk_stream_and_graph(dev):
    """On a side stream, and captured: every replay against the eager call, with eager work between the replays."""
    qkv, K, V, bt, cos, sin, pos, c = (t.to(dev) if isinstance(t, torch.Tensor) else t for t in qk_case(
        13, 8, 8, 8, 2, 128, 128, 16, 4, torch.float16))
    c = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    x = torch.randn(8, 1, 8, 128, device=dev).half()

    def step(K, V):
        q, _, _ = gqa.paged_qk_norm_rope_update(qkv, K, V, bt, cos, sin, pos, layout="half", **c)
        return q, rope.apply_rope(q + x, cos, sin, positions=pos, layout="half")

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    Kg, Vg = K.clone(), V.clone()
    with torch.cuda.stream(side):
        eager = step(Kg.clone(), Vg.clone())
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(Kg, Vg)
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, device=dev))
        pos.copy_(torch.randint(-1, 64, (8,), device=dev))
        Ke, Ve = Kg.clone(), Vg.clone()
        eager = step(Ke, Ve)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*eager, Ke, Ve), (*out, Kg, Vg))), i


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_every_size(dev, layout):
    """Every part of heads of 2 .. 40 values and some larger ones, from addresses of 2 bytes: pieces that overlap, regions
    of fewer values than a piece, heads that begin anywhere; the norms' sums count every value once."""
    g = torch.Generator().manual_seed(21)
    for D in [*range(2, 41), 90, 120, 250]:
        flat = torch.randn(6 * 3 * D + 1, generator=g).half().to(dev)
        x = flat[1:].view(2, 3, 3, D)
        for rd in sorted({2, D // 4 * 2, *range(2, min(D, 40) + 1, 4 if D % 4 else 2), D // 2 * 2} - {0}):
            cos, sin = (torch.randn(9, rd // 2, generator=g).to(dev) for _ in range(2))
            got = rope.apply_rope(x, cos, sin, 2, layout=layout, rotary_dim=rd)
            check_rope(x, cos, sin, np.broadcast_to(2 + np.arange(3), (2, 3)), layout, rd, got)
            if D % 2:
                continue  # (heads with a cache are even)
            case = qk_case(D + rd, 2, 2, 2, 1, D, rd, 2, 3, torch.float16, True)
            qkv, K, V, bt, c, s, pos, kw = case
            wide = torch.zeros(2, 4 * D + 1, dtype=torch.float16, device=dev)
            wide[:, 1:] = qkv.to(dev)
            out = gqa.paged_qk_norm_rope_update(
                wide[:, 1:], K.to(dev), V.to(dev), bt.to(dev), c.to(dev), s.to(dev), pos.to(dev), layout=layout,
                **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
            check_qk(out, case, torch.float16, layout)


@pytest.mark.parametrize("B,S,H", [(3, 2 ** 30 - 5, 2), (1, 2 ** 30 + 9, 4)])
def test_rope_long(dev, B, S, H):
    """More units of work than a launch numbers: sequences, and parts of one, in launches of their own.  Only rows of
    position 0 .. 9 are inside of the tables, which are asked for at both sides of each seam."""
    g = torch.Generator().manual_seed(B)
    x = torch.randn(1, 1, H, 2, generator=g).half().to(dev).expand(B, S, H, 2)
    cos, sin = torch.randn(10, 1, generator=g).to(dev), torch.randn(10, 1, generator=g).to(dev)
    for at in ([0, 2 ** 29 - 6, S - 10] if B == 1 else [0, S - 10]):
        pos = torch.full((B, S), -1, dtype=torch.int32, device=dev)
        pos[:, at:at + 10] = torch.arange(10, dtype=torch.int32, device=dev)
        got = rope.apply_rope(x, cos, sin, positions=pos, rotary_dim=2)
        check_rope(x[:, :10].contiguous(), cos, sin, np.broadcast_to(np.arange(10), (B, 10)), "interleaved", 2,
                   got[:, at:at + 10].contiguous())
        live = sum(int((row != 0).any(-1).any(-1).sum()) for part in got.split(2 ** 26, 1) for row in part)
        assert live == 10 * B
        del got, pos


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_qk_rows_past_the_tables(dev, layout, monkeypatch):
    """Tables shorter than the block table's reach: a row past them is empty, and keeps no earlier row of the slot that it
    would have had from writing; among the live rows of a slot the later one still wins."""
    monkeypatch.setenv("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
    T, P = 300, 4
    qkv, K, V, bt, cos, sin, pos, c = qk_case(31, T, T, 2, 1, 32, 32, P, 3, torch.float16)
    cos, sin = cos[:9], sin[:9]  # positions 9, 10 and 11 of the table's twelve are past them
    pos[2::3] = 8 + pos[2::3] % 4
    bt[7, 2] = bt[100, 2] = bt[7, 1]  # page of positions 4 .. 7 and 8 .. 11 of row 7, and of row 100
    bt[299, 1] = bt[40, 0]
    pos[7], pos[100] = 5, 9  # row 100 would write slot 1 of the page, row 7 does
    pos[40], pos[299] = 2, 6  # both live: row 299's
    bt[200, 2], bt[201, 2], bt[202, 0] = bt[199, 0], bt[199, 0], bt[199, 0]
    pos[199], pos[200], pos[201], pos[202] = 1, 9, 9, -1  # empty rows of two kinds behind a live one
    case = qkv, K, V, bt, cos, sin, pos, c
    d = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    got = gqa.paged_qk_norm_rope_update(d(qkv), d(K), d(V), d(bt), d(cos), d(sin), d(pos), layout=layout,
                                        **{k: d(v) for k, v in c.items()})
    check_qk(got, case, torch.float16, layout)
    want = gqa.reference_paged_qk_norm_rope_update(d(qkv), d(K), d(V), d(bt), d(cos), d(sin), d(pos), layout=layout,
                                                   **{k: d(v) for k, v in c.items()})
    assert torch.equal(got[2], want[2])  # v is copied
    for t in (7, 199):
        assert torch.equal(got[2][bt[t, pos[t] // P].long(), pos[t] % P].cpu(), qkv[t].reshape(-1, 32)[3:])
