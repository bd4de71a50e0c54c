"""Low-rank adapters of many requests beside a shared projection: row m of a
batch adds s_i B_i (A_i x[m]) for its own adapter i to what the shared weight
gave.  The reference has no counterpart.

Adapters lie stacked: ``lora_a`` [ADAPTERS, R, K] and ``lora_b`` [ADAPTERS, N,
R] in the activations' dtype (an adapter of lower rank is filled up with
zeros), ``scales`` fp32 [ADAPTERS] (None: 1).
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any

import torch

from . import _lib
from ._common import ACT_DTYPES, as_dense, ci_safe_mode_enabled, narrow_i32, values_only
from .kv_cache_ops import host_checks_enabled
from .mlp_block_ops import quantized_linear
from .quant_ops import _MATVEC_BACKENDS_MSG

MAX_RANK, MAX_ADAPTERS = 128, 4096
MAX_ROWS, MAX_OUTPUTS = 2 ** 20 - 1, 2 ** 24 - 1


@dataclass
class LoraAdapters:
    """The adapters beside one projection [N, K]: a [ADAPTERS, R, K], b
    [ADAPTERS, N, R], scales fp32 [ADAPTERS] or None."""

    a: Any
    b: Any
    scales: Any | None = None


def _check_out(out, base):
    if out is not None and (out.shape != base.shape or out.dtype != base.dtype or out.device != base.device):
        raise ValueError(f"out must match base {tuple(base.shape)} {base.dtype} on {base.device}, got "
                         f"{tuple(out.shape)} {out.dtype} on {out.device}")


def _validate(x, base, lora_a, lora_b, adapter_ids, scales):
    """(M, N, K, R, adapters, ids [M])"""
    *rows, K = x.shape or (0,)
    *same, N = base.shape or (0,)
    if rows != same or not x.shape or not base.shape:
        raise ValueError(f"x and base must be [...,K] and [...,N] of the same rows, got {tuple(x.shape)}, "
                         f"{tuple(base.shape)}")
    a_shape = lora_a.shape
    if len(a_shape) != 3 or lora_b.ndim != 3:
        raise ValueError(f"lora_a and lora_b must be [ADAPTERS,R,K] and [ADAPTERS,N,R], got {tuple(lora_a.shape)}, "
                         f"{tuple(lora_b.shape)}")
    adapters, R, _ = a_shape
    if a_shape[2] != K or lora_b.shape != (adapters, N, R):
        raise ValueError(f"lora_a and lora_b must be [ADAPTERS,R,{K}] and [ADAPTERS,{N},R], got {tuple(lora_a.shape)}, "
                         f"{tuple(lora_b.shape)}")
    if K < 1 or not 1 <= R <= MAX_RANK or adapters > MAX_ADAPTERS:
        raise ValueError(f"K must be positive, R in [1, {MAX_RANK}] and ADAPTERS at most {MAX_ADAPTERS}, got K={K}, "
                         f"R={R}, ADAPTERS={adapters}")
    dtype = x.dtype
    if dtype not in ACT_DTYPES:
        raise TypeError(f"x dtype must be float16 or bfloat16, got {x.dtype}")
    if base.dtype != dtype or lora_a.dtype != dtype or lora_b.dtype != dtype:
        raise TypeError(f"base, lora_a and lora_b must carry x's dtype {dtype}, got {base.dtype}, {lora_a.dtype}, "
                        f"{lora_b.dtype}")
    if scales is not None and scales.shape != (adapters,):
        raise ValueError(f"scales must have shape {(adapters,)}, got {tuple(scales.shape)}")
    M = math.prod(rows)
    if not isinstance(adapter_ids, torch.Tensor):
        adapter_ids = torch.as_tensor(adapter_ids, dtype=torch.int32)
    if adapter_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"adapter_ids must be int32 or int64, got {adapter_ids.dtype}")
    shape = adapter_ids.shape
    ids = adapter_ids
    if shape == (M,):
        pass
    elif shape == tuple(rows):
        ids = ids.reshape(M)
    elif len(rows) == 2 and shape == (rows[0],):
        ids = ids[:, None].expand(rows).reshape(M)
    else:
        raise ValueError(f"adapter_ids must have shape {tuple(rows)}, {(M,)} or one a sequence, got "
                         f"{tuple(adapter_ids.shape)}")
    if M and host_checks_enabled(ids):
        lo, hi = int(ids.min()), int(ids.max())
        if lo < -1 or hi >= adapters:
            raise ValueError(f"adapter_ids must be in [-1, {adapters}), got {lo} to {hi}")
    return M, N, K, R, adapters, narrow_i32(ids, x.device)


def reference_lora_add(x, base, lora_a, lora_b, adapter_ids, *, scales=None):
    """``lora_add`` with tensor ops, an adapter at a time."""
    M, N, K, R, adapters, ids = _validate(x, base, lora_a, lora_b, adapter_ids, scales)
    x2, out = x.reshape(M, K).float(), base.reshape(M, N).float()
    for i in range(adapters):
        # other rows are zeros in both products: what is not finite in them would reach this adapter's gradients as 0 * inf
        own = (ids == i)[:, None]
        t = torch.where(own, torch.where(own, x2, 0.0) @ lora_a[i].float().t(), 0.0)
        d = t @ lora_b[i].float().t()
        if scales is not None:
            d = d * scales[i].float()
        out = torch.where(own, out + d, out)
    return out.to(base.dtype).reshape(base.shape)


def _rows(t, width):
    """(t as rows of ``width`` dense values at one stride, that stride); None where it is not."""
    if t.is_contiguous():
        return t, width
    if t.ndim == 2 and t.stride(1) == 1 and t.stride(0) >= width:
        return t, t.stride(0)
    return None, 0


def _apart(a, b):
    """Whether two tensors (of one dtype) share no memory: their spans do not overlap, or they are different columns."""
    def span(t):
        n = sum((s - 1) * k for s, k in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (n + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    if a.ndim != 2 or b.ndim != 2 or a.stride() != b.stride() or a.stride(1) != 1:
        return False
    # columns of the same rows
    row, off = a.stride(0) * a.element_size(), b0 - a0
    return off % row >= a.shape[1] * a.element_size() and off % row + b.shape[1] * b.element_size() <= row


def lora_add(x, base, lora_a, lora_b, adapter_ids, *, scales=None, out=None, backend: str = "auto"):
    """base + s_i B_i (A_i x) for each row's adapter i = adapter_ids[row]: x
    [...,K], base [...,N] of the same rows (fp16 / bf16), ``adapter_ids`` int32
    of the rows' shape, flat, or one for each sequence of [B,S,...] rows; -1 is
    a row without an adapter.  Both products are summed in fp32 and the result
    is rounded once.  ``out``: a tensor to write, ``base`` itself among them
    (the rows may be strided; no other overlap).  At most 2^20 - 1 rows and
    2^24 - 1 outputs.  An infinity in lora_b may come back as a NaN of its
    outputs; one in x, base or lora_a is what the formula makes of it.
    In fp16 a value of A x below 2^-38 of the largest of its row counts as zero.

    ids are checked on the host unless that is off (``host_checks_enabled``);
    then one outside [0, ADAPTERS) is a row without an adapter.  Backend
    "reference", and inputs that need more than their values (a gradient, a
    function transform, tracing), take the tensor ops."""
    backend_name = backend.lower()
    if backend_name not in ("auto", "reference", "metal"):
        raise ValueError("backend must be one of 'reference', 'metal', 'auto'")
    _check_out(out, base)
    tensors = (x, base, lora_a, lora_b) if scales is None else (x, base, lora_a, lora_b, scales)
    if backend_name == "reference" or ci_safe_mode_enabled() or not values_only(*tensors):
        y = reference_lora_add(x, base, lora_a, lora_b, adapter_ids, scales=scales)
        return y if out is None else out.copy_(y)
    M, N, K, R, adapters, ids = _validate(x, base, lora_a, lora_b, adapter_ids, scales)
    if M > MAX_ROWS or N > MAX_OUTPUTS:
        raise ValueError(f"at most {MAX_ROWS} rows and {MAX_OUTPUTS} outputs, got {M}, {N}")
    dev = _lib.require_device(x, base, lora_a, lora_b, scales)
    x2, x_stride = _rows(x, K)
    if x2 is None:
        x2, x_stride = x.contiguous(), K
    b2, base_stride = _rows(base, N)
    if b2 is None:
        b2, base_stride = base.contiguous(), N
    target = out
    if out is None:
        target, out_stride = torch.empty(base.shape, dtype=base.dtype, device=dev), N
    else:
        same = out.data_ptr() == base.data_ptr() and out.stride() == base.stride()
        if not (same or _apart(out, base)) or not _apart(out, x):
            raise ValueError("out may be base itself, and share no memory with it or x otherwise")
        target, out_stride = _rows(out, N)
        if target is None:
            target, out_stride = torch.empty(base.shape, dtype=base.dtype, device=dev), N
    if not adapters:
        target.copy_(base)
    elif M and N:
        a, b = lora_a.contiguous(), lora_b.contiguous()
        scales = as_dense(scales, torch.float32)
        size = _lib.load().mk_lora_workspace_bytes(M, N, K, R, adapters)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.launch("mk_lora_add", dev, x2.data_ptr(), x_stride, b2.data_ptr(), base_stride, a.data_ptr(),
                    b.data_ptr(), ids.data_ptr(), _lib.ptr(scales), target.data_ptr(), out_stride, M, N, K, R,
                    adapters, _lib.dtype_code(x.dtype), _lib.ptr(ws), size)
    if out is not None and target is not out:
        out.copy_(target)
        return out
    return target


def quantized_lora_linear(x, w, scales, zeros, lora_a, lora_b, adapter_ids, *, lora_scales=None, bits=4, group_size=32,
                          backend: str = "auto"):
    """``quantized_linear`` with every row's adapter added to its result, in place:
    the shared product in the activation dtype, then ``lora_add``.  Where x, scales
    or zeros need more than their values (a gradient, a function transform,
    tracing) the shared product takes the tensor ops too, so that a gradient has
    both parts; where only the adapters do, it stays on its kernel."""
    if backend.lower() not in ("reference", "metal", "metal_parallel", "metal_tiled", "auto"):
        raise ValueError(_MATVEC_BACKENDS_MSG)
    if not values_only(*(t for t in (x, scales, zeros) if t is not None)):
        backend = "reference"
    y = quantized_linear(x, w, scales, zeros, bits=bits, group_size=group_size, backend=backend)
    reference = backend.lower() == "reference"
    adapters = (lora_a, lora_b) if lora_scales is None else (lora_a, lora_b, lora_scales)
    return lora_add(x, y, lora_a, lora_b, adapter_ids, scales=lora_scales,
                    out=None if reference or not values_only(*adapters) else y,
                    backend="reference" if reference else "auto")
