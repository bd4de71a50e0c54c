"""mk_lora_add against the 64-bit oracle: ranks, widths and row counts at tile
edges, mixed and sorted adapters, strides, values that are not numbers."""

import pytest
import torch

import mk.lora_ops as lo
from mk.mlp_block_ops import quantized_linear
from tests._data import quant_weight, to_dev
from tests.test_host_lora import check_linear_gradients, check_lora, lora_case, quantized_case

import numpy as np

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]

# (M, N, K, R, adapters)
SHAPES = [(1, 64, 64, 16, 1), (1, 6144, 4096, 16, 4), (2, 1, 1, 1, 1), (3, 100, 72, 8, 2), (16, 64, 32, 16, 3),
          (17, 65, 33, 17, 2), (5, 40, 30, 4, 3), (33, 130, 264, 32, 9), (20, 48, 520, 33, 20), (64, 256, 96, 64, 4),
          (7, 200, 1000, 128, 2), (65, 72, 2056, 48, 1), (130, 1024, 136, 100, 5), (300, 96, 512, 16, 2),
          (31, 8, 4100, 2, 3), (48, 4096, 8, 127, 2), (70, 328, 1504, 64, 7), (64, 40, 64, 8, 80), (2000, 72, 96, 8, 300),
          (200, 16, 24, 3, 4096), (1100, 300, 520, 128, 2),
          (1, 520, 4096, 32, 2), (1, 1030, 520, 20, 3), (1, 513, 1100, 7, 2), (1, 64, 14336, 16, 2), (1, 4096, 8, 128, 3)]


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_lora_add(dev, shape, dtype):
    case = lora_case(sum(shape), *shape, dtype)
    x, base, a, b, ids, s = on(dev, *case)
    before = base.clone()
    check_lora(lo.lora_add(x, base, a, b, ids, scales=s), *case)
    assert torch.equal(base, before)
    check_lora(lo.lora_add(x, base, a, b, ids), *case[:5], None)
    order = torch.argsort(case[4], stable=True)  # prompts one after another
    sorted_case = (case[0], case[1], *case[2:4], case[4][order], case[5])
    check_lora(lo.lora_add(x, base, a, b, sorted_case[4].to(dev), scales=s), *sorted_case)
    assert lo.lora_add(x, base, a, b, ids, scales=s, out=base) is base  # in place
    check_lora(base, *case)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dev, dtype):
    """Rows of wider tensors, bases off a 16-byte boundary, 3-D rows, an adapter of every sequence."""
    M, N, K, R, NA = 24, 80, 136, 16, 3
    case = lora_case(7, M, N, K, R, NA, dtype)
    x, base, a, b, ids, s = on(dev, *case)

    def rows(t, pad, off):
        wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=dtype, device=dev)
        view = wide[:, off:off + t.shape[1]]
        view.copy_(t)
        return view

    for pad, off in ((8, 8), (8, 0), (3, 1), (16, 2)):
        out = rows(torch.zeros_like(base), pad, off)
        check_lora(lo.lora_add(rows(x, pad, off), rows(base, pad, off), a, b, ids, scales=s, out=out), *case)
        same = rows(base, pad, off)
        check_lora(lo.lora_add(rows(x, 0, 0), same, a, b, ids, scales=s, out=same), *case)
    for t in (1, 3):  # adapters off a boundary
        flat_a, flat_b = (torch.empty(v.numel() + t, dtype=dtype, device=dev)[t:].view(v.shape) for v in (a, b))
        flat_a.copy_(a), flat_b.copy_(b)
        check_lora(lo.lora_add(x, base, flat_a, flat_b, ids, scales=s), *case)
    check_lora(lo.lora_add(x, base, a.transpose(1, 2).contiguous().transpose(1, 2), b, ids, scales=s), *case)
    x3, base3 = x.reshape(6, 4, K), base.reshape(6, 4, N)
    per = torch.tensor([2, 0, -1, 1, 1, 0], dtype=torch.int32)
    got = lo.lora_add(x3, base3, a, b, per, scales=s)
    check_lora(got.reshape(M, N), *case[:4], per.repeat_interleave(4), case[5])
    turned = x3.transpose(0, 1).contiguous().transpose(0, 1)  # rows not at one stride
    assert torch.equal(lo.lora_add(turned, base3.transpose(0, 1).contiguous().transpose(0, 1), a, b, per, scales=s), got)
    for i in (-1, 2):  # a single row, with and without an adapter
        args = x[:1], base[:1], a, b, torch.tensor([i], dtype=torch.int32, device=dev)
        check_lora(lo.lora_add(*args, scales=s), case[0][:1], case[1][:1], case[2], case[3], torch.tensor([i]), case[5])
    out = torch.zeros_like(base3).transpose(0, 1).contiguous().transpose(0, 1)
    assert lo.lora_add(x3, base3, a, b, per, scales=s, out=out) is out and torch.equal(out, got)
    assert lo.lora_add(x[:0], base[:0], a, b, ids[:0]).shape == (0, N)
    assert torch.equal(lo.lora_add(x, base, a[:0], b[:0], ids * 0 - 1), base)


def test_overlaps_refused(dev):
    x, base, a, b, ids, s = on(dev, *lora_case(8, 4, 16, 16, 4, 2, torch.float16))
    both = torch.zeros(4, 40, dtype=torch.float16, device=dev)
    for out, kw in ((x, {}), (both[:, 1:17], {"base": both[:, 0:16]}), (both[:, :16], {"x": both[:, 8:24]})):
        with pytest.raises(ValueError, match="share no memory"):
            lo.lora_add(**{**dict(x=x, base=base, lora_a=a, lora_b=b, adapter_ids=ids, out=out), **kw})
    with pytest.raises(ValueError):
        lo.lora_add(x, base, a, b, ids, out=base[:3])
    with pytest.raises(ValueError):
        lo.lora_add(x, base, a, b, ids.clone().fill_(2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [20, 100])
def test_values_stay_in_their_rows(dev, dtype, M, monkeypatch):
    """A row or an adapter of infinities and NaNs changes no row that has neither; ids outside of the adapters add
    nothing where the host does not look; large values of fp16 stay finite in between."""
    monkeypatch.setenv("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
    x, base, a, b, ids, s = lora_case(9, M, 72, 160, 16, 5, dtype)
    ids[3], ids[9], ids[10] = 5, 2 ** 31 - 1, -2 ** 31
    clean = lo.lora_add(*on(dev, x, base, a, b, ids), scales=s.to(dev))
    check_lora(clean, x, base, a, b, ids, s)
    ids[5], ids[6] = 0, 1
    clean = lo.lora_add(*on(dev, x, base, a, b, ids), scales=s.to(dev)).cpu()
    x[5, 7], x[6, 3] = float("nan"), float("inf")
    a[4, 1, 2], b[3, 5, 1] = float("inf"), float("nan")
    got = lo.lora_add(*on(dev, x, base, a, b, ids), scales=s.to(dev)).cpu()
    rows = torch.ones(M, dtype=torch.bool)
    rows[5] = rows[6] = False
    rows[(ids == 4) | (ids == 3)] = False
    assert torch.equal(got[rows], clean[rows])
    assert got[5].isnan().all() and not got[6].isfinite().any()
    assert got[ids == 3][:, 5].isnan().all() and torch.equal(got[ids == 3][:, :5], clean[ids == 3][:, :5])
    # A x past fp16 (2^18), small B: the result is finite and right
    x, base, a, b, ids, s = lora_case(10, M, 40, 64, 8, 2, dtype, none=0.0)
    x, a, b = torch.full_like(x, 64.0), torch.full_like(a, 64.0), b * 2.0 ** -14
    a[:, 1::2] *= 2.0 ** -24  # and ranks that are small beside them
    check_lora(lo.lora_add(*on(dev, x, base, a, b, ids), scales=s.to(dev)), x, base, a, b, ids, s)


def test_quantized_lora_linear(dev):
    """The shared projection and its adapters: what the two calls give."""
    rng = np.random.default_rng(0)
    K, N, g = 256, 192, 64
    for bits in (4, 8):
        _, w, sc, z = quant_weight(rng, N, K, g, bits)
        w, sc, z = to_dev(w, dev), to_dev(sc, dev, torch.float16), to_dev(z, dev, torch.float16)
        x, _, a, b, ids, s = on(dev, *lora_case(bits, 9, N, K, 16, 3, torch.float16))
        x = x[:, None]
        y = quantized_linear(x, w, sc, z, bits=bits, group_size=g)
        got = lo.quantized_lora_linear(x, w, sc, z, a, b, ids, lora_scales=s, bits=bits, group_size=g)
        assert got.shape == (9, 1, N) and torch.equal(got, lo.lora_add(x, y, a, b, ids, scales=s))
        check_lora(got[:, 0], x[:, 0], y[:, 0], a, b, ids, s)


def test_stream_and_graph(dev):
    """On a side stream, and two captured calls on one: every replay against the eager calls, with eager work between."""
    cases = [lora_case(20 + i, 12, 96, 256, 16, 3, torch.bfloat16) for i in range(2)]
    given = [on(dev, *c) for c in cases]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        warm = lo.lora_add(*given[0][:5], scales=given[0][5])
    side.synchronize()
    check_lora(warm, *cases[0])
    graphs, outs = [], []
    for c in given:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(lo.lora_add(*c[:5], scales=c[5]))
    for i in range(4):
        for c in given:
            c[0].copy_(torch.randn(c[0].shape, device=dev))
            c[4].copy_(torch.randint(-1, 3, c[4].shape, device=dev))
        eager = [lo.lora_add(*c[:5], scales=c[5]) for c in given]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, outs)), i


@pytest.mark.parametrize("M", [1, 5, 70])
@pytest.mark.parametrize("R", [3, 12, 20, 40, 100])
def test_infinity_in_a_row(dev, R, M):
    """With positive adapters an infinity in a row gives infinities, whatever lies between the ranks and whole tiles."""
    g = torch.Generator().manual_seed(R)
    x, base = torch.rand(M, 40, generator=g).half(), torch.rand(M, 72, generator=g).half()
    a, b = 0.1 + torch.rand(2, R, 40, generator=g).half(), 0.1 + torch.rand(2, 72, R, generator=g).half()
    x[M // 2, 5] = float("inf")
    got = lo.lora_add(*on(dev, x, base, a, b, torch.zeros(M, dtype=torch.int32))).cpu()
    assert (got[M // 2] == float("inf")).all()
    assert got[[m for m in range(M) if m != M // 2]].isfinite().all()


@pytest.mark.parametrize("M", [1, 5, 70])
def test_infinity_beside_large_sums(dev, M):
    """An infinity of one rank leaves the others, above fp16's range, finite."""
    x, base = torch.full((M, 40), 64.0).half(), torch.zeros(M, 64).half()
    a, b = torch.full((1, 4, 40), 100.0).half(), torch.full((1, 64, 4), 2.0 ** -10).half()
    a[0, 2, 7], b[0, 32:, 2] = float("inf"), 2.0 ** -5
    got = lo.lora_add(*on(dev, x, base, a, b, torch.zeros(M, dtype=torch.int32))).cpu()
    assert (got == float("inf")).all()


@pytest.mark.parametrize("M,N", [(1, 517), (1, 2), (40, 3), (64, 255), (64, 1030), (200, 93), (700, 1026)])
def test_rows_without_an_adapter(dev, M, N):
    """Most rows have none: copied bit by bit, from and to strided rows at any address, in place left alone."""
    g = torch.Generator().manual_seed(M + N)
    x, base = torch.randn(M, 24, generator=g).half().to(dev), torch.randn(M, N + 3, generator=g).half().to(dev)[:, 1:N + 1]
    base[0, 0] = float("nan")
    a, b = torch.randn(2, 4, 24, generator=g).half().to(dev), torch.randn(2, N, 4, generator=g).half().to(dev)
    ids = torch.where(torch.rand(M, generator=g) < 0.9, -1, torch.randint(0, 2, (M,), generator=g)).to(torch.int32)
    ids[0] = -1
    out = torch.full((M, N + 2), 7.0, device=dev).half()
    got = lo.lora_add(x, base, a, b, ids.to(dev), out=out[:, :N])
    none = (ids < 0).to(dev)
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(got[none]), bits(base[none])) and (out[:, N:] == 7).all()
    if (~none).any():
        keep = [t[~none].cpu() for t in (x, base)]
        check_lora(got[~none], *keep, a.cpu(), b.cpu(), ids[ids >= 0], None)
    before = base.clone()
    assert lo.lora_add(x, base, a, b, ids.to(dev), out=base) is base
    assert torch.equal(bits(base[none]), bits(before[none]))


@pytest.mark.parametrize("M", [63, 64, 65, 128, 129, 192, 255, 256, 257])
@pytest.mark.parametrize("adapters", [1, 2, 70, 300])
def test_groups(dev, M, adapters):
    """Every number of adapters in a batch, each of one row to all of them, in any order."""
    g = torch.Generator().manual_seed(M + adapters)
    x, base, a, b, _, s = lora_case(M, M, 40, 16, 8, adapters, torch.float16)
    few = torch.randint(-1, adapters, (3,), generator=g)
    for ids in (torch.randint(-1, adapters, (M,), generator=g), few[torch.randint(0, 3, (M,), generator=g)],
                torch.full((M,), adapters - 1), torch.full((M,), -1), torch.arange(M) % adapters,
                torch.where(torch.arange(M) == M - 1, 0, -1), torch.arange(M).flip(0) // 67 % (adapters + 1) - 1):
        ids = ids.to(torch.int32)
        check_lora(lo.lora_add(*on(dev, x, base, a, b, ids), scales=s.to(dev)), x, base, a, b, ids, s)


def test_many_adapters_of_many_rows(dev):
    case = lora_case(9, 600, 16, 24, 3, 4096, torch.bfloat16)
    x, base, a, b, ids, s = on(dev, *case)
    check_lora(lo.lora_add(x, base, a, b, ids, scales=s), *case)


@pytest.mark.parametrize("M,N,R", [(4100, 16390, 72), (9000, 8191, 128), (5000, 4100, 8)])
def test_many_rows(dev, M, N, R):
    """Prompts of thousands of rows: some of them against the oracle, rows without an adapter in between."""
    g = torch.Generator(device=dev).manual_seed(M)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()  # noqa: E731
    x, base, a, b = rand(M, 40), rand(M, N), rand(3, R, 40), (rand(3, N, R) / 8)
    ids = torch.arange(M, device=dev) // 700 % 4 - 1
    got = lo.lora_add(x, base, a, b, ids)
    some = torch.randperm(M, generator=g, device=dev)[:40]
    some = torch.cat([some, torch.tensor([0, 1, M - 2, M - 1], device=dev)])
    check_lora(got[some], *(t.cpu() for t in (x[some], base[some], a, b, ids[some])), None)
    assert torch.equal(got[ids < 0], base[ids < 0])


@pytest.mark.parametrize("M,K,R,adapters", [(20, 2048, 16, 2), (64, 1500, 40, 3), (200, 2048, 16, 4), (333, 2048, 16, 5),
                                            (1500, 1024, 64, 7), (3000, 4096, 8, 40), (700, 515, 128, 3)])
def test_results_do_not_depend_on_places(dev, M, K, R, adapters):
    """The same call again, and its rows in another order, bit by bit: groups of every number of rows."""
    x, base, a, b, ids = on(dev, *lora_case(M + R, M, 96, K, R, adapters, torch.bfloat16)[:5])
    base = base.zero_()  # (what a row adds is not rounded away)
    want = lo.lora_add(x, base, a, b, ids)
    for k in range(6):
        assert torch.equal(lo.lora_add(x, base, a, b, ids), want)
        p = torch.randperm(M, generator=torch.Generator().manual_seed(k)).to(dev)
        assert torch.equal(lo.lora_add(x[p], base, a, b, ids[p]), want[p])


def test_far_adapters_and_rows(dev):
    """Adapters and rows past 2^31 values of their arrays."""
    N, R, K, M, NA = 8192, 128, 256, 66000, 2100
    g = torch.Generator().manual_seed(1)
    a, b = torch.zeros(NA, R, K, dtype=torch.float16, device=dev), torch.zeros(NA, N, R, dtype=torch.float16, device=dev)
    a[-1], b[-1] = torch.randn(R, K, generator=g).half().to(dev), torch.randn(N, R, generator=g).half().to(dev)
    wide = torch.zeros(M, 33000, dtype=torch.float16, device=dev)
    x, base = wide[:, :K], wide[:, 1024:1024 + N]
    rows = torch.tensor([0, 1, M - 2, M - 1], device=dev)
    x[rows] = torch.randn(4, K, generator=g).half().to(dev)
    base[rows] = torch.randn(4, N, generator=g).half().to(dev)
    ids = torch.full((M,), -1, dtype=torch.int32, device=dev)
    ids[rows] = NA - 1
    own = [x[rows].cpu(), base[rows].cpu(), a[-1:].cpu(), b[-1:].cpu(), torch.zeros(4, dtype=torch.int32), None]
    for take in (slice(None), slice(M - 2, M)):  # listed groups; two rows
        got = lo.lora_add(x[take], base[take], a, b, ids[take])
        which = rows if take == slice(None) else torch.tensor([0, 1], device=dev)
        want = own if take == slice(None) else [own[0][2:], own[1][2:], *own[2:4], own[4][2:], None]
        check_lora(got[which], *want)
    assert lo.lora_add(x, base, a, b, ids, out=base) is base
    check_lora(base[rows], *own)
    assert not base[2:M - 2].any()


@pytest.mark.parametrize("bits", [4, 8])
def test_quantized_lora_linear_gradients(dev, bits):
    """x's gradient has both parts; where only the adapters record one, the shared product stays on its kernel and the
    adapters' gradients are those of the same formula."""
    *tensors, W = quantized_case(10 + bits, 40, 64, 128, 8, 3, bits, 32, dev)
    x, w, sc, z, a, b, ids, s = tensors
    g = torch.randn(40, 64, generator=torch.Generator().manual_seed(bits)).half().to(dev)
    kw = dict(lora_scales=s, bits=bits, group_size=32)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    lo.quantized_lora_linear(leaves[0], w, sc, z, *leaves[1:], ids, **kw).backward(g)
    check_linear_gradients([t.grad for t in leaves], x, a, b, ids, s, W, g)
    own = [t.clone().requires_grad_() for t in (a, b)]
    y = lo.quantized_lora_linear(x, w, sc, z, *own, ids, **kw)
    y.backward(g)
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(own, leaves[1:]))
    shared = quantized_linear(x, w, sc, z, bits=bits, group_size=32)
    assert torch.equal(y, lo.lora_add(x, shared, a, b, ids, scales=s, backend="reference"))
