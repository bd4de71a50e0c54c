"""Rotary positions -- drop-in for ops/rope_ops.py (interleaved layout over
whole heads, ops/rope_ops.py:61-75, and the table builder of
models/llama_config.py:107-124), with the half layout, rotation of the first
part of each head, positions of every sequence or token, and frequencies
scaled for long contexts beside them.

Layouts: ``"interleaved"`` turns the pairs (2i, 2i+1) of the first
``rotary_dim`` values of a head, ``"half"`` the pairs (i, i + rotary_dim/2);
pair i of a token at position p by the angle of ``cos[p, i]``, ``sin[p, i]``.
Values past ``rotary_dim`` are copied.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._common import ci_safe_mode_enabled, narrow_i32, values_only
from .kv_cache_ops import host_checks_enabled

_LAYOUTS = {"interleaved": 0, "half": 1}


def _layout_code(layout: str) -> int:
    code = _LAYOUTS.get(layout)
    if code is None:
        raise ValueError(f"layout must be one of 'interleaved', 'half', got {layout!r}")
    return code


def _rotary_dim(rotary_dim, D: int) -> int:
    if rotary_dim is None:
        return D
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > D:
        raise ValueError(f"rotary_dim must be even and in [2, {D}], got {rotary_dim}")
    return int(rotary_dim)


def _rotate(x, c, s, layout: str):
    """x [..., D] in fp32 turned by c, s [..., rotary_dim / 2]."""
    h = c.shape[-1]
    rest = x[..., 2 * h:]
    if layout == "half":
        a, b = x[..., :h], x[..., h:2 * h]
        return torch.cat([a * c - b * s, a * s + b * c, rest], dim=-1)
    a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
    y = torch.stack([a * c - b * s, a * s + b * c], dim=-1)
    return torch.cat([y.flatten(-2), rest], dim=-1)


def _validate_inputs(x, cos, sin, position_offset: int, rotary_dim=None, *, any_rows: bool = False):
    """ops/rope_ops.py:25-58.  ``any_rows``: the rows needed are the
    positions' matter, not the offset's."""
    shape, table = x.shape, cos.shape
    if len(shape) != 4:
        raise ValueError(f"x must be 4-D [B,S,H,D], got {tuple(x.shape)}")
    if table != sin.shape or len(table) != 2:
        if cos.ndim != 2 or sin.ndim != 2:
            raise ValueError(f"cos and sin must be 2-D [S_total, D/2], got {tuple(cos.shape)}, {tuple(sin.shape)}")
        raise ValueError(f"cos and sin must have identical shapes, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    B, S, H, D = shape
    if D % 2 != 0 and rotary_dim is None:
        raise ValueError(f"RoPE requires even D, got D={D}")
    if rotary_dim is not None:
        rd = _rotary_dim(rotary_dim, D)
        if table[1] != rd // 2:
            raise ValueError(f"cos/sin last dim must be rotary_dim/2={rd // 2}, got {table[1]}")
    elif table[1] != D // 2:
        raise ValueError(f"cos/sin last dim must be D/2={D // 2}, got {table[1]}")
    if position_offset < 0:
        raise ValueError("position_offset must be non-negative")
    if not any_rows and position_offset + S > table[0]:
        raise ValueError(
            f"position_offset + S must fit in cos/sin rows, got offset={position_offset}, S={S}, rows={table[0]}"
        )
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"x dtype must be float16 or bfloat16, got {x.dtype}")
    return B, S, H, D, table[0]


def _validate_positions(positions, B: int, S: int, rows: int, device):
    """int32 tensor [B] (a sequence's first position; -1: all of it is padding)
    or [B, S] (a row's position; -1: padding) on ``device``, checked against
    the table's rows where the host may read it."""
    if not isinstance(positions, torch.Tensor):
        positions = torch.as_tensor(positions, dtype=torch.int32)
    dtype, shape = positions.dtype, positions.shape
    if dtype != torch.int32 and dtype != torch.int64:
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if shape != (B,) and shape != (B, S):
        raise ValueError(f"positions must have shape [B]={(B,)} or [B,S]={(B, S)}, got {tuple(positions.shape)}")
    if positions.numel() and host_checks_enabled(positions):
        lo, hi = int(positions.min()), int(positions.max())
        hi += S if positions.ndim == 1 and hi >= 0 else 1  # (a padding sequence has no further rows)
        if lo < -1 or hi > rows:
            raise ValueError(f"positions must be in [-1, {rows}) with S={S}, got {lo} to {hi - 1}")
    return narrow_i32(positions, device)


def reference_apply_rope(x, cos, sin, position_offset: int = 0, *, positions=None, layout: str = "interleaved",
                         rotary_dim=None):
    """ops/rope_ops.py:61-75: pairs (2i, 2i+1) rotate by the angle of row
    position_offset + s; fp32 math, result in x's dtype.  The tables may sit
    on the host: the rows used move to x's device.  ``positions``, ``layout``
    and ``rotary_dim`` as in ``apply_rope``."""
    if positions is None:
        _, S, _, D, _ = _validate_inputs(x, cos, sin, position_offset, rotary_dim)
        c = cos[position_offset:position_offset + S].to(device=x.device, dtype=torch.float32).reshape(1, S, 1, -1)
        s = sin[position_offset:position_offset + S].to(device=x.device, dtype=torch.float32).reshape(1, S, 1, -1)
    else:
        if position_offset != 0:
            raise ValueError("give position_offset or positions, not both")
        B, S, _, D, rows = _validate_inputs(x, cos, sin, 0, rotary_dim, any_rows=True)
        pos = _validate_positions(positions, B, S, rows, cos.device).long()
        if pos.ndim == 1:
            pos = torch.where(pos[:, None] < 0, -1, pos[:, None] + torch.arange(S, device=pos.device))
        live = (pos >= 0) & (pos < rows)
        at = torch.where(live, pos, 0)
        c = cos[at].to(device=x.device, dtype=torch.float32)[:, :, None]
        s = sin[at].to(device=x.device, dtype=torch.float32)[:, :, None]
    _layout_code(layout)
    if positions is None and layout == "interleaved" and 2 * c.shape[-1] == D:
        xe = x[..., 0::2].to(torch.float32)
        xo = x[..., 1::2].to(torch.float32)
        ye = xe * c - xo * s
        yo = xe * s + xo * c
        return torch.stack([ye, yo], dim=-1).reshape(x.shape).to(x.dtype)
    y = _rotate(x.to(torch.float32), c, s, layout)
    if positions is not None:
        y = torch.where(live.to(x.device)[:, :, None, None], y, 0.0)
    return y.to(x.dtype)


def apply_rope(x, cos, sin, position_offset: int = 0, *, positions=None, layout: str = "interleaved", rotary_dim=None,
               backend: str = "auto"):
    """Rotary positions of x [B,S,H,D] (fp16 / bf16, any strides) -> a dense
    tensor of its shape: row s of sequence b turns by position_offset + s, or
    by ``positions`` (int32, on x's device; not with an offset): [B] holds
    each sequence's first position, [B,S] every row's.  A position of -1 marks
    padding, whose rows come back zero.  cos, sin [rows, rotary_dim / 2]
    (fp32; ``build_rope_tables``, ``build_scaled_rope_tables``).

    Positions on the device are read back to be checked against the tables'
    rows as ``normalize_positions`` does; where that is off (graph capture,
    MK_SKIP_DEVICE_RANGE_CHECKS=1) a row outside of them comes back zero.
    Backend "reference", and inputs that need more than their values (a
    gradient, a function transform, tracing), take the tensor ops."""
    if positions is not None and position_offset != 0:
        raise ValueError("give position_offset or positions, not both")
    code = _layout_code(layout)
    backend_name = backend.lower()
    if backend_name not in ("auto", "reference", "metal"):
        raise ValueError("backend must be one of 'reference', 'metal', 'auto'")
    if backend_name == "reference" or ci_safe_mode_enabled() or not values_only(x, cos, sin):
        return reference_apply_rope(x, cos, sin, position_offset, positions=positions, layout=layout,
                                    rotary_dim=rotary_dim)
    B, S, H, D, rows = _validate_inputs(x, cos, sin, position_offset, rotary_dim, any_rows=positions is not None)
    dev = _lib.require_device(x)
    pos, per_token = None, 0
    if positions is not None:
        pos = _validate_positions(positions, B, S, rows, dev)
        per_token = pos.ndim - 1
    c, s = _tables(cos, dev), _tables(sin, dev)
    sb, ss, sh, sd = x.stride()
    if sd != 1 and D != 1:
        x = x.contiguous()
        sb, ss, sh, sd = x.stride()
    y = torch.empty((B, S, H, D), dtype=x.dtype, device=dev)
    if B == 0 or S == 0 or H == 0:
        return y
    _lib.launch("mk_apply_rope", dev, x.data_ptr(), c.data_ptr(), s.data_ptr(), _lib.ptr(pos), y.data_ptr(), B, S, H, D,
                sb, ss, sh, rotary_dim or D, position_offset, per_token, rows, code, _lib.dtype_code(x.dtype))
    return y


def _tables(t, dev):
    if t.dtype == torch.float32 and t.device == dev and t.is_contiguous():
        return t
    return t.to(device=dev, dtype=torch.float32).contiguous()


def build_rope_tables(seq_len: int, head_dim: int, theta: float = 10000.0, *, device=None):
    """models/llama_config.py:107-124: inv_freq = theta^(-arange(0,D,2)/D),
    returns fp32 cos/sin of shape [seq_len, D/2]."""
    if seq_len <= 0:
        raise ValueError(f"seq_len must be positive, got {seq_len}")
    if head_dim % 2 != 0:
        raise ValueError(f"head_dim must be even for RoPE, got {head_dim}")
    positions = torch.arange(seq_len, dtype=torch.float32, device=device)
    inv_freq = 1.0 / (float(theta) ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / float(head_dim)))
    freqs = positions.reshape(seq_len, 1) * inv_freq.reshape(1, head_dim // 2)
    return torch.cos(freqs), torch.sin(freqs)


def build_scaled_rope_tables(seq_len: int, rotary_dim: int, theta: float = 10000.0, *, scaling=None, device=None):
    """fp32 cos/sin [seq_len, rotary_dim / 2] with frequencies scaled for
    contexts longer than those a model was trained on.  ``scaling`` is a dict:

    {"type": "linear", "factor"}: positions divided by the factor.
    {"type": "ntk", "factor"}: theta * factor^(d / (d - 2)), which leaves the
        fastest pair alone and slows the slowest one by the factor.
    {"type": "llama3", "factor", "low_freq_factor", "high_freq_factor",
        "original_max_position"}: with n = original_max_position / wavelength,
        pairs of n > high_freq_factor stay, those of n < low_freq_factor are
        slowed by the factor, linear in n between.
    {"type": "yarn", "factor", "original_max_position"; "beta_fast" 32,
        "beta_slow" 1, "attention_factor" 0.1 ln(factor) + 1}: linear between
        the pairs that turn beta_fast and beta_slow times over the original
        length (rounded outwards); the attention factor multiplies the tables.

    Angles are formed in 64 bits and rounded once: at position 131072 an fp32
    product is off by up to 2^-6 radians.  Runs once, where weights are
    loaded."""
    if seq_len <= 0:
        raise ValueError(f"seq_len must be positive, got {seq_len}")
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    scaling = dict(scaling or {})
    kind = scaling.get("type")
    if kind not in (None, "linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"scaling type must be one of 'linear', 'ntk', 'llama3', 'yarn', got {kind!r}")
    needed = {None: (), "linear": ("factor",), "ntk": ("factor",),
              "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position"),
              "yarn": ("factor", "original_max_position")}[kind]
    missing = [k for k in needed if k not in scaling]
    if missing:
        raise ValueError(f"scaling of type {kind!r} needs {missing}")
    factor = float(scaling.get("factor", 1.0))
    if factor < 1.0:
        raise ValueError(f"scaling factor must be at least 1, got {factor}")
    d, theta, gain = rotary_dim, float(theta), 1.0
    if kind == "ntk" and d > 2:
        theta *= factor ** (d / (d - 2))
    i = torch.arange(d // 2, dtype=torch.float64, device=device)
    inv = theta ** (-2.0 * i / d)
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not 0 < low < high:
            raise ValueError(f"low_freq_factor must be positive and below high_freq_factor, got {low}, {high}")
        turns = float(scaling["original_max_position"]) * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / factor)
    elif kind == "yarn":
        length = float(scaling["original_max_position"])

        def pair_of(turns):  # the (fractional) pair that turns so often over the original length
            return d * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))

        first = max(0, math.floor(pair_of(float(scaling.get("beta_fast", 32.0)))))
        last = min(d - 1, math.ceil(pair_of(float(scaling.get("beta_slow", 1.0)))))
        slow = ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1.0 - slow + slow / factor)
        gain = scaling.get("attention_factor")
        gain = 0.1 * math.log(factor) + 1.0 if gain is None else float(gain)
    angles = torch.arange(seq_len, dtype=torch.float64, device=device)[:, None] * inv
    return (torch.cos(angles) * gain).float(), (torch.sin(angles) * gain).float()
