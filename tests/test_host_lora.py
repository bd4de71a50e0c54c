"""Low-rank adapters on the host: the tensor-op path against the 64-bit oracle
and against differences, and what is refused."""

import numpy as np
import pytest
import torch

import mk.lora_ops as lo
from oracle import serving as sv

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of each type
# A x is kept as the sum of two values of the type where it goes through the matrix cores
TWO = {torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -16}


def lora_case(seed, M, N, K, R, NA, dtype, none=0.2, scales=True):
    g = torch.Generator().manual_seed(seed)
    x, base = torch.randn(M, K, generator=g).to(dtype), torch.randn(M, N, generator=g).to(dtype)
    a = (torch.randn(NA, R, K, generator=g) / K ** 0.5).to(dtype)
    b = (torch.randn(NA, N, R, generator=g) / R ** 0.5).to(dtype)
    ids = torch.randint(0, NA, (M,), generator=g, dtype=torch.int32)
    ids[torch.rand(M, generator=g) < none] = -1
    return x, base, a, b, ids, 0.5 + torch.rand(NA, generator=g) if scales else None


def check_lora(got, x, base, a, b, ids, scales):
    """One rounding of the result, and K + R + 4 fp32 roundings and those of A x of what it is a sum of; over all
    values their root mean square is that of one rounding, with a sixteenth for the sums."""
    f = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    want, size = sv.lora(f(x), f(base), f(a), f(b), ids.tolist(), f(scales))
    dtype, K, R = x.dtype, x.shape[-1], a.shape[1]
    err = np.abs(got.double().cpu().numpy() - want)
    lim = U[dtype] * np.abs(want) + size * ((K + R + 4) * 2.0 ** -24 + TWO[dtype]) * 1.01 + 2.0 ** -25
    assert (err <= lim).all(), (int((err > lim).sum()), float(err.max()))
    if err.size:
        assert np.sqrt((err ** 2).mean()) <= U[dtype] * np.sqrt((want ** 2).mean()) * 1.0625 + 2.0 ** -25
    none = ~((ids >= 0) & (ids < len(a))).cpu()
    assert torch.equal(got.cpu()[none], base.cpu()[none])


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("shape", [(5, 12, 20, 4, 3), (1, 1, 1, 1, 1), (9, 33, 17, 8, 2)])
def test_reference_lora(shape, dtype):
    case = lora_case(sum(shape), *shape, dtype)
    check_lora(lo.lora_add(*case[:5], scales=case[5], backend="reference"), *case)
    check_lora(lo.lora_add(*case[:5], backend="reference"), *case[:5], None)


def test_ids_of_sequences_and_rows():
    x, base, a, b, ids, s = lora_case(3, 6, 8, 16, 4, 3, torch.float16)
    x3, base3 = x.reshape(2, 3, 16), base.reshape(2, 3, 8)
    flat = lo.lora_add(x, base, a, b, ids, scales=s, backend="reference")
    for form in (ids, ids.reshape(2, 3), ids.long(), ids.tolist()):
        assert torch.equal(lo.lora_add(x3, base3, a, b, form, scales=s, backend="reference").reshape(6, 8), flat)
    per = lo.lora_add(x3, base3, a, b, [2, -1], scales=s, backend="reference")
    assert torch.equal(per.reshape(6, 8), lo.lora_add(x, base, a, b, [2] * 3 + [-1] * 3, scales=s, backend="reference"))
    out = torch.empty_like(base)
    assert lo.lora_add(x, base, a, b, ids, scales=s, out=out, backend="reference") is out and torch.equal(out, flat)
    assert torch.equal(lo.lora_add(x, base, a[:0], b[:0], [-1] * 6, backend="reference"), base)
    assert lo.lora_add(x[:0], base[:0], a, b, [], backend="reference").shape == (0, 8)


def test_gradients_against_formula_and_differences():
    """What needs a gradient takes the tensor ops, on any backend; the gradients against their formulas and against
    differences of the result (which is linear in x, so that they are exact but for its roundings)."""
    x, base, a, b, ids, s = lora_case(4, 5, 6, 7, 3, 2, torch.float16)
    leaves = [t.clone().requires_grad_() for t in (x, base, a, b)]
    g = torch.randn(5, 6).half()
    lo.lora_add(*leaves, ids, scales=s).backward(g)
    for i in range(2):
        rows = ids == i
        gi, xi = g[rows].double(), x[rows].double()
        da = s[i].double() * (b[i].double().t() @ gi.t()) @ xi
        db = s[i].double() * gi.t() @ (xi @ a[i].double().t())
        for got, want in ((leaves[2].grad[i], da), (leaves[3].grad[i], db)):
            assert (got.double() - want).abs().max() <= 4 * 2.0 ** -11 * (want.abs().max() + 1)
    assert torch.equal(leaves[1].grad, g) and (leaves[0].grad[ids < 0] == 0).all()
    step = torch.randn(5, 7).half()
    y0, y1 = (lo.lora_add(x + k * step, base, a, b, ids, scales=s, backend="reference").double() for k in (0, 1))
    moved = ((x + step).double() - x.double())  # what the sum's own rounding leaves of the step
    slope = (leaves[0].grad.double() * moved).sum()
    size = (leaves[0].grad.double().abs() * moved.abs()).sum() + (g.double().abs() * (y0.abs() + y1.abs())).sum()
    assert abs(((y1 - y0) * g.double()).sum() - slope) <= 4 * 2.0 ** -11 * size


def test_refusals():
    x, base, a, b, ids, s = lora_case(5, 4, 6, 8, 2, 3, torch.float16)
    ok = dict(x=x, base=base, lora_a=a, lora_b=b, adapter_ids=ids, scales=s, backend="reference")
    lo.lora_add(**ok)
    for kw in (dict(x=x[:, :7]), dict(base=base[:3]), dict(base=base[None]), dict(lora_a=a[0]), dict(lora_b=b[:2]),
               dict(lora_b=b[:, :5]), dict(lora_a=a[:, :1]), dict(adapter_ids=ids[:3]), dict(adapter_ids=[0, 1, 2, 3]),
               dict(adapter_ids=[0, 1, 2, -2]), dict(scales=s[:2]), dict(backend="triton"),
               dict(lora_a=torch.zeros(4097, 2, 8).half(), lora_b=torch.zeros(4097, 6, 2).half(), scales=None),
               dict(lora_a=a[:, :0], lora_b=b[:, :, :0]), dict(x=x[:, :0], lora_a=a[:, :, :0]),
               dict(lora_a=torch.zeros(1, 129, 8).half(), lora_b=torch.zeros(1, 6, 129).half())):
        with pytest.raises(ValueError):
            lo.lora_add(**{**ok, **kw})
    for kw in (dict(x=x.float(), base=base.float(), lora_a=a.float(), lora_b=b.float()), dict(base=base.bfloat16()),
               dict(lora_a=a.bfloat16()), dict(adapter_ids=ids.float())):
        with pytest.raises(TypeError):
            lo.lora_add(**{**ok, **kw})
    with pytest.raises(ValueError, match="ROCm device"):
        lo.lora_add(**{**ok, "backend": "auto"})


def test_limits():
    """More rows or outputs than a call takes are refused before anything is read."""
    z = lambda *shape: torch.zeros(1, dtype=torch.float16).expand(*shape)  # noqa: E731
    for M, N in ((lo.MAX_ROWS + 1, 1), (1, lo.MAX_OUTPUTS + 1)):
        with pytest.raises(ValueError, match="at most"):
            lo.lora_add(z(M, 1), z(M, N), z(1, 1, 1), z(1, N, 1), torch.zeros(M, dtype=torch.int32))


def test_apart():
    wide = torch.zeros(6, 20)
    part = lambda r0, r1, c0, c1: wide[r0:r1, c0:c1]  # noqa: E731
    apart = [(part(0, 6, 0, 5), part(0, 6, 5, 20)), (part(0, 6, 10, 20), part(0, 6, 0, 10)),
             (part(0, 2, 0, 20), part(2, 6, 0, 20)), (part(1, 6, 3, 6), part(0, 5, 7, 19)),
             (part(0, 6, 0, 5), torch.zeros(6, 20))]
    over = [(part(0, 6, 0, 6), part(0, 6, 5, 20)), (part(0, 6, 10, 20), part(1, 5, 8, 11)), (wide, wide),
            (part(0, 6, 0, 20), part(0, 6, 3, 4)), (wide.view(3, 40)[:, :5], part(0, 6, 7, 9)),
            (wide.view(-1)[18:].as_strided((5, 4), (20, 1)), part(0, 6, 0, 3))]
    assert all(lo._apart(a, b) and lo._apart(b, a) for a, b in apart)
    assert not any(lo._apart(a, b) or lo._apart(b, a) for a, b in over)


def quantized_case(seed, M, N, K, R, NA, bits, group, device="cpu"):
    """(x, packed w, scales, zeros, adapters, ids, lora scales, W as the product takes it)"""
    from mk.quant_ops import reference_dequant_q4, reference_dequant_q8

    g = torch.Generator().manual_seed(seed)
    x, _, a, b, ids, s = lora_case(seed, M, N, K, R, NA, torch.float16)
    ids[M // 2] = -1
    w = torch.randint(0, 256, (N, K // 2 if bits == 4 else K), generator=g, dtype=torch.uint8)
    sc = (0.02 * (0.5 + torch.rand(N, K // group, generator=g))).half()
    z = torch.randint(3, 12, (N, K // group), generator=g).half()
    W = (reference_dequant_q4 if bits == 4 else reference_dequant_q8)(w, sc, z, group_size=group, out_dtype=torch.float16)
    return [t.to(device) for t in (x, w, sc, z, a, b, ids, s, W)]


def check_linear_gradients(got, x, a, b, ids, s, W, g):
    """Gradients (x, a, b) of <g, x W^T + s_i B_i A_i x>: fp32 sums, each part rounded to fp16 on its way into x's."""
    x, a, b, s, W, g = (t.double().cpu() for t in (x, a, b, s, W, g))
    dx, size = g @ W, g.abs() @ W.abs()
    for m, i in enumerate(ids.tolist()):
        if i < 0:
            continue
        dx[m] += s[i] * (g[m] @ b[i]) @ a[i]
        size[m] += s[i] * (g[m].abs() @ b[i].abs()) @ a[i].abs()
    assert ((got[0].double().cpu() - dx).abs() <= 4 * 2.0 ** -11 * size).all()
    assert (got[0][ids < 0] != 0).any()  # a row without an adapter has the shared product's part
    for i in range(len(a)):
        rows = (ids == i).cpu()
        da, db = s[i] * (b[i].t() @ g[rows].t()) @ x[rows], s[i] * g[rows].t() @ (x[rows] @ a[i].t())
        sa, sb = (s[i] * (b[i].abs().t() @ g[rows].abs().t()) @ x[rows].abs(),
                  s[i] * g[rows].abs().t() @ (x[rows].abs() @ a[i].abs().t()))
        for t, want, mag in ((got[1][i], da, sa), (got[2][i], db, sb)):
            assert ((t.double().cpu() - want).abs() <= 2 * 2.0 ** -11 * mag + 2.0 ** -25).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("backend", ["auto", "reference"])
def test_quantized_lora_linear_gradients(bits, backend):
    """The gradient of x has the shared product's part as well as the adapters', on every backend."""
    x, w, sc, z, a, b, ids, s, W = quantized_case(bits, 9, 12, 16, 3, 2, bits, 8)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    g = torch.randn(9, 12, generator=torch.Generator().manual_seed(1)).half()
    kw = dict(lora_scales=s, bits=bits, group_size=8, backend=backend)
    y = lo.quantized_lora_linear(leaves[0], w, sc, z, *leaves[1:], ids, **kw)
    y.backward(g)
    check_linear_gradients([t.grad for t in leaves], x, a, b, ids, s, W, g)
    with torch.no_grad():
        assert torch.equal(y, lo.quantized_lora_linear(x, w, sc, z, a, b, ids, **{**kw, "backend": "reference"}))
    # against differences: linear in x, so exact but for the roundings of both results and of the gradient
    step = torch.randn(9, 16, generator=torch.Generator().manual_seed(2)).half()
    y0, y1 = (lo.quantized_lora_linear(t, w, sc, z, a, b, ids, **{**kw, "backend": "reference"}).double()
              for t in (x, x + step))
    moved = (x + step).double() - x.double()
    slope = (leaves[0].grad.double() * moved).sum()
    size = (leaves[0].grad.double().abs() * moved.abs()).sum() + (g.double().abs() * (y0.abs() + y1.abs())).sum()
    assert abs(((y1 - y0) * g.double()).sum() - slope) <= 4 * 2.0 ** -11 * size
    # a gradient of the quantization's scales, and a forward-mode tangent
    sc_leaf = sc.clone().requires_grad_()
    lo.quantized_lora_linear(x, w, sc_leaf, z, a, b, ids, **kw).sum().backward()
    assert sc_leaf.grad.abs().sum() > 0
    _, tangent = torch.func.jvp(lambda t: lo.quantized_lora_linear(t, w, sc, z, a, b, ids, **kw).float(), (x,), (step,))
    want = step.double() @ W.double().t()
    for m, i in enumerate(ids.tolist()):
        if i >= 0:
            want[m] += s[i].double() * (step[m].double() @ a[i].double().t()) @ b[i].double().t()
    assert (tangent.double() - want).abs().max() <= 8 * 2.0 ** -11 * want.abs().max()
    with pytest.raises(ValueError, match="backend must be one of"):
        lo.quantized_lora_linear(leaves[0], w, sc, z, a, b, ids, **{**kw, "backend": "x"})


@pytest.mark.parametrize("grad", [False, True])
def test_out_of_another_shape_or_type(grad):
    """The tensor ops take no ``out`` that the kernels would refuse: nothing is broadcast or cast into it."""
    x, base, a, b, ids, s = lora_case(6, 4, 6, 8, 2, 3, torch.float16)
    kw = dict(backend="auto") if grad else dict(backend="reference")
    a.requires_grad_(grad)
    for out in (torch.zeros(2, 4, 6).half(), torch.zeros(4, 6), torch.zeros(4, 6).bfloat16(), torch.zeros(24).half()):
        with pytest.raises(ValueError, match="out must match base"):
            lo.lora_add(x, base, a, b, ids, scales=s, out=out, **kw)
        assert not out.any()
    out = torch.zeros(4, 6).half()
    assert lo.lora_add(x, base, a, b, ids, scales=s, out=out, **kw) is out
    assert torch.equal(out, lo.lora_add(x, base, a, b, ids, scales=s, backend="reference"))


def test_gradients_beside_rows_that_are_not_finite():
    """What stands in a padding row or in another adapter's rows touches no gradient of an adapter or a finite row."""
    x, base, a, b, ids, s = lora_case(7, 8, 6, 10, 3, 3, torch.float16)
    ids = torch.tensor([0, 1, -1, 0, 2, 1, -1, 0], dtype=torch.int32)
    g = torch.randn(8, 6, generator=torch.Generator().manual_seed(3)).half()
    clean = [t.clone().requires_grad_() for t in (x, base, a, b, s)]
    lo.lora_add(*clean[:4], ids, scales=clean[4]).backward(g)
    x[2], x[6, 3], x[4, 1] = float("nan"), float("inf"), float("-inf")  # two padding rows, the row of adapter 2
    leaves = [t.clone().requires_grad_() for t in (x, base, a, b, s)]
    y = lo.lora_add(*leaves[:4], ids, scales=leaves[4])
    y.backward(g)
    fine = ids != 2
    assert torch.equal(y[ids < 0], base[ids < 0])
    assert torch.equal(leaves[0].grad[fine], clean[0].grad[fine]) and (leaves[0].grad[ids < 0] == 0).all()
    for k in (2, 3):
        assert torch.equal(leaves[k].grad[:2], clean[k].grad[:2])
    assert torch.equal(leaves[4].grad[:2], clean[4].grad[:2])
    a[2, 1, 4] = float("inf")  # an adapter that no finite row has
    leaves = [t.clone().requires_grad_() for t in (x, base, a, b, s)]
    lo.lora_add(*leaves[:4], torch.where(ids == 2, -1, ids), scales=leaves[4]).backward(g)
    assert all((leaves[k].grad[2] == 0).all() for k in (2, 3, 4)) and leaves[0].grad.isfinite().all()
