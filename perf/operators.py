"""Operators of a server that decodes many requests at once, as measured cases.

Sizes are those of a Llama-3-8B decoder (hidden 4096, intermediate 14336, 32
query and 8 key/value heads of 128, a fused qkv projection of 6144 rows, pages
of 16 positions), which the benchmark and the tests use, and others of the
same kind in ``draw``.  A case is a dict of plain values; its ``kind`` names
the entry point it goes through:

  rope     rope_ops.apply_rope                    (rotary positions: both layouts, part of the head)
  qk       gqa_ops.paged_qk_norm_rope_update      (norms of q and k heads, rotation, write to the pages)
  copy     kv_page_ops.copy_kv_pages              (pages of every layer from place to place)
  fork     kv_page_ops.fork_kv_sequences          (rows continue others: beams, samples, rows that end)
  compact  kv_page_ops.compact_kv_pages           (live pages to the front of the pool)
  lora     lora_ops.lora_add                      (low-rank adapters of many requests)

``own`` false computes them with elementary tensor operations in fp32, rounded
once.  A serving loop checks its positions once, on the host, where it makes
them; it runs with MK_SKIP_DEVICE_RANGE_CHECKS=1, so that a call does not read
them back from the device.
"""

import math
import os
import sys

os.environ.setdefault("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
sys.path.insert(0, os.path.join(os.getcwd(), "mlx-metal-kernels_amd"))

import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    heads = {"hq": 32, "hkv": 8, "d": 128, "page": 16}
    return [
        # the smallest call: the query heads of a single decoding sequence
        {"name": "rope_half_b1", "kind": "rope", "batch": 1, "seq": 1, "h": 32, "d": 128, "rotary": 128,
         "layout": "half", "rows": 8192, "pad": False, "dtype": "float16"},
        # four prompts of odd length, half of each head turned, far positions of a long context
        {"name": "rope_part_prompt", "kind": "rope", "batch": 4, "seq": 2047, "h": 32, "d": 128, "rotary": 64,
         "layout": "interleaved", "rows": 131072, "pad": False, "dtype": "bfloat16"},
        # one decoding sequence between its qkv projection and its attention
        {"name": "qk_decode_b1", "kind": "qk", **heads, "tokens": 1, "seqs": 1, "ctx": 2048, "norm": True,
         "rotary": 128, "layout": "half", "dtype": "float16"},
        # a full decode batch, some of its rows empty
        {"name": "qk_decode_b32", "kind": "qk", **heads, "tokens": 32, "seqs": 32, "ctx": 8192, "norm": True,
         "rotary": 128, "layout": "half", "dtype": "bfloat16"},
        # the rows of seven prompts of different lengths, an odd number of them
        {"name": "qk_prompts_8191", "kind": "qk", **heads, "tokens": 8191, "seqs": 7, "ctx": 8192, "norm": True,
         "rotary": 128, "layout": "half", "dtype": "bfloat16"},
        # a prompt's pages duplicated in an 8-bit cache: codes and scales of 16 layers
        {"name": "copy_q8_509", "kind": "copy", "layers": 16, "hkv": 8, "d": 128, "page": 16, "pages": 1280,
         "moved": 509, "quantized": True, "dtype": "float16"},
        # four beams of one short request, two layers: latency
        {"name": "fork_beams4", "kind": "fork", "layers": 2, "hkv": 8, "d": 128, "page": 16, "prompts": 1, "beams": 4,
         "ctx": 100, "spare": 8, "reserve": 1, "dtype": "float16"},
        # eight beams of each of four requests over the whole stack
        {"name": "fork_beams32", "kind": "fork", "layers": 32, "hkv": 8, "d": 128, "page": 16, "prompts": 4,
         "beams": 8, "ctx": 2048, "spare": 64, "reserve": 1, "dtype": "bfloat16"},
        # the pool of a whole stack after half of its sequences have ended
        {"name": "compact_half", "kind": "compact", "layers": 32, "hkv": 8, "d": 128, "page": 16, "seqs": 11,
         "ctx": 1000, "gone": 5, "dtype": "float16"},
        # one decoding sequence with an adapter of rank 16 beside its qkv projection
        {"name": "lora_qkv_m1", "kind": "lora", "rows": 1, "k": 4096, "n": 6144, "rank": 16, "adapters": 4,
         "mixed": True, "dtype": "float16"},
        # a full decode batch over eight adapters, some rows without one
        {"name": "lora_qkv_m32", "kind": "lora", "rows": 32, "k": 4096, "n": 6144, "rank": 16, "adapters": 8,
         "mixed": True, "dtype": "bfloat16"},
        # prompts of five requests through the gate projection, each with its adapter of rank 64
        {"name": "lora_gate_4093", "kind": "lora", "rows": 4093, "k": 4096, "n": 14336, "rank": 64, "adapters": 5,
         "mixed": False, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["rope", "qk", "qk", "copy", "fork", "compact", "lora", "lora"])
    c = {"kind": kind, "dtype": rng.choice(["float16", "bfloat16"])}
    d = rng.choice([64, 80, 128, 128, 256])
    if kind in ("rope", "qk"):
        c.update(d=d, rotary=rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]),
                 layout=rng.choice(["half", "interleaved"]))
    if kind == "rope":
        h = rng.choice([1, 2, 4, 8, 16, 32])
        batch = _log(rng, 1, 16)
        seq = _log(rng, 1, max(1, min(4096, 4 * 2047 * 32 * 128 // (batch * h * d))))
        return {**c, "batch": batch, "seq": seq, "h": h, "rows": seq + _log(rng, 1, 131072 - seq),
                "pad": rng.random() < 0.3}
    if kind == "lora":
        c.update(k=_log(rng, 64, 14336), n=_log(rng, 64, 14336), rank=rng.choice([1, 4, 8, 16, 16, 32, 33, 64, 128]),
                 adapters=_log(rng, 1, 16), mixed=rng.random() < 0.5)
        if rng.random() < 0.8:  # widths are whole 8s but now and then
            c.update(k=8 * max(1, c["k"] // 8), n=8 * max(1, c["n"] // 8))
        most = min(4093 * 32768 // (c["k"] + 2 * c["n"]), 4093 * 320 // (c["adapters"] * c["rank"]))
        return {**c, "rows": _log(rng, 1, max(1, min(4093, most)))}
    hkv = rng.choice([1, 2, 4, 8])
    c.update(hkv=hkv, page=rng.choice([8, 16, 16, 32, 64]))
    if kind == "qk":
        c.update(hq=hkv * rng.choice([1, 4, 4, 7, 8]), norm=rng.random() < 0.7)
        if rng.random() < 0.5:
            n = _log(rng, 1, 256)
            return {**c, "tokens": n, "seqs": n, "ctx": _log(rng, 16, min(8192, 262144 // n))}
        seqs = _log(rng, 1, 16)
        most = min(8191, 8191 * 6144 // ((c["hq"] + 2 * hkv) * d))
        tokens = _log(rng, 2 * seqs, max(2 * seqs, most))
        return {**c, "tokens": tokens, "seqs": seqs, "ctx": tokens + _log(rng, 1, 4096)}
    c.update(layers=_log(rng, 1, 32), d=rng.choice([64, 128]))
    at_most = 32 * 704 * 16 * 8 * 128 // (c["layers"] * c["page"] * hkv * c["d"])  # pages: the largest listed pool
    if kind == "copy":
        pages = _log(rng, 8, max(8, min(4096, at_most)))
        return {**c, "pages": pages, "moved": _log(rng, 1, pages // 2), "quantized": rng.random() < 0.4}
    if kind == "fork":
        prompts, beams = _log(rng, 1, 16), _log(rng, 1, 8)
        ctx = _log(rng, 1, max(1, min(2048, c["page"] * at_most // (prompts * (1 + beams)))))
        return {**c, "prompts": prompts, "beams": beams, "ctx": ctx, "spare": _log(rng, 1, 64),
                "reserve": rng.choice([0, 1, 1, 1, 5, 40])}
    seqs = _log(rng, 2, 64)
    return {**c, "seqs": seqs, "ctx": _log(rng, 1, max(1, min(2048, c["page"] * at_most // seqs - c["page"]))),
            "gone": rng.randint(1, seqs - 1)}


# ----------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 17)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _randint(gen, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=gen, device=DEV, dtype=torch.int32)


def _perm(gen, n):
    return torch.randperm(n, generator=gen, device=DEV).to(torch.int32)


def _angles(rows, rotary, base=500000.0):
    """cos and sin [rows, rotary / 2]: the angles in 64 bits, rounded once."""
    inv = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    f = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cos(f).float(), torch.sin(f).float()


def _pool(gen, c, pages, dtype):
    """K and V pages of every layer: [2 * layers, pages, page, hkv, d]."""
    shape = (2 * c["layers"], pages, c["page"], c["hkv"], c["d"])
    small = torch.randn((2 * c["layers"], 1, *shape[2:]), generator=gen, device=DEV, dtype=torch.float32)
    per_page = torch.randn((1, pages, 1, 1, shape[4]), generator=gen, device=DEV, dtype=torch.float32)
    return small.to(dtype) + per_page.to(dtype)


def prepare(case, seed):
    c, gen = case, _gen(seed)
    dtype = DTYPES[c["dtype"]]
    kind = c["kind"]
    if kind == "rope":
        cos, sin = _angles(c["rows"], c["rotary"])
        B, S = c["batch"], c["seq"]
        start = _randint(gen, 0, c["rows"] - S + 1, (B,))
        positions = start
        if c["pad"]:  # rows behind a sequence's end
            s = torch.arange(S, dtype=torch.int32, device=DEV)
            length = _randint(gen, 0, S + 1, (B, 1))
            positions = torch.where(s < length, start[:, None] + s, -1).to(torch.int32)
        return {"case": c, "x": _randn(gen, (B, S, c["h"], c["d"]), dtype), "cos": cos, "sin": sin,
                "positions": positions}
    if kind == "qk":
        T, n, P = c["tokens"], c["seqs"], c["page"]
        blocks = -(-c["ctx"] // P)
        cos, sin = _angles(c["ctx"], c["rotary"])
        pages = n * blocks + 3 if T == n else T // P + 2 * n + 3  # three that no sequence has, at least
        if T == n:  # one new token a sequence; an eighth of a larger batch's rows are empty
            table = _perm(gen, pages)[:n * blocks].reshape(n, blocks)
            positions = _randint(gen, c["ctx"] // 2, c["ctx"], (T,))
            if T > 8:
                positions[1::8] = -1
            sequences = None
        else:  # prompts one after another, behind what each holds already
            cut = 1 + torch.randperm(T - 1, generator=gen, device=DEV)[:n - 1].sort().values
            cut = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), T)])
            t = torch.arange(T, device=DEV)
            owner = torch.searchsorted(cut, t, right=True) - 1
            first = _randint(gen, 0, c["ctx"] - T + 1, (n,)).long()
            positions = (first[owner] + t - cut[owner]).to(torch.int32)
            sequences = owner.to(torch.int32)
            end = (first + cut[1:] - cut[:-1])[:, None]
            j = torch.arange(blocks, device=DEV)
            written = (j >= (first // P)[:, None]) & (j * P < end)  # the blocks that the rows fall into
            number = torch.cumsum(written.reshape(-1), 0) - 1
            table = torch.where(written, _perm(gen, pages)[number.reshape(n, blocks).clamp(min=0)], -1).to(torch.int32)
        shape = (pages, P, c["hkv"], c["d"])
        w = [(1.0 + 0.2 * torch.randn(c["d"], generator=gen, device=DEV)).to(dtype) for _ in range(2)]
        return {"case": c, "qkv": _randn(gen, (T, (c["hq"] + 2 * c["hkv"]) * c["d"]), dtype), "cos": cos, "sin": sin,
                "q_weight": w[0] if c["norm"] else None, "k_weight": w[1] if c["norm"] else None,
                "K": _randn(gen, shape, dtype), "V": _randn(gen, shape, dtype), "table": table,
                "positions": positions, "sequences": sequences}
    if kind == "copy":
        ids = _perm(gen, c["pages"])
        src, dst = ids[:c["moved"]].contiguous(), ids[c["moved"]:2 * c["moved"]].contiguous()
        if not c["quantized"]:
            pools = [_pool(gen, c, c["pages"], dtype)]
        else:
            shape = (2 * c["layers"], c["pages"], c["page"], c["hkv"])
            pools = [torch.randint(0, 256, (*shape, c["d"]), generator=gen, device=DEV, dtype=torch.uint8),
                     _randn(gen, (*shape, c["d"] // 64), torch.float16)]
        return {"case": c, "pools": pools, "pages": [t for p in pools for t in p.unbind(0)], "src": src, "dst": dst}
    if kind == "fork":
        n, beams, P = c["prompts"], c["beams"], c["page"]
        B, blocks = n * beams, -(-(c["ctx"] + 2 * c["reserve"] + 1) // P)
        prompt = _randint(gen, 0, c["ctx"] + 1, (n, 1)).expand(n, beams).reshape(B)  # positions that beams share
        lengths = torch.minimum(prompt + _randint(gen, 0, 2 + c["ctx"] // 32, (1,)), prompt.new_tensor(c["ctx"]))
        shared = (prompt // P)[:, None]
        used = (-(-lengths // P))[:, None]
        j = torch.arange(blocks, dtype=torch.int32, device=DEV)
        row = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
        first = row // beams * beams  # the row whose page a shared block is
        slot = torch.where(j < shared, first, row) * blocks + j
        own_slot = (j < used) & ((j >= shared) | (row == first))
        number = torch.cumsum(own_slot.reshape(-1), 0) - 1
        pages = n * (c["ctx"] // P) + B * (c["ctx"] // 32 // P + 2) + c["spare"]
        ids = _perm(gen, pages)
        table = torch.where(j < used, ids[number[slot.long()].clamp(min=0)], -1).to(torch.int32)
        refs = torch.bincount(table[table >= 0].long(), minlength=pages).to(torch.int32)
        # so many pages are free; the others are held by somebody else (a cache of prefixes)
        refs[ids[number[-1] + 1 + c["spare"]:].long()] = 1
        # beams continue any beam of their prompt; now and then one has ended
        parents = first[:, 0] + _randint(gen, 0, beams, (B,))
        parents = torch.where(torch.rand(B, generator=gen, device=DEV) < 0.05, -1, parents).to(torch.int32)
        pool = _pool(gen, c, pages, dtype)
        return {"case": c, "pools": [pool], "pages": list(pool.unbind(0)), "table": table,
                "lengths": lengths.to(torch.int32), "refs": refs, "parents": parents}
    if kind == "compact":
        n, P = c["seqs"], c["page"]
        blocks = -(-c["ctx"] // P)
        length = _randint(gen, c["ctx"] // 2, c["ctx"] + 1, (n, 1))
        used = -(-length // P)
        j = torch.arange(blocks, dtype=torch.int32, device=DEV)
        number = torch.cumsum((j < used).reshape(-1), 0) - 1
        ids = _perm(gen, n * blocks)
        table = torch.where(j < used, ids[number.reshape(n, blocks).clamp(min=0)], -1).to(torch.int32)
        table[_perm(gen, n)[:c["gone"]].long()] = -1
        refs = torch.bincount(table[table >= 0].long(), minlength=n * blocks).to(torch.int32)
        pool = _pool(gen, c, n * blocks, dtype)
        return {"case": c, "pools": [pool], "pages": list(pool.unbind(0)), "table": table, "refs": refs}
    M, K, N, R, NA = c["rows"], c["k"], c["n"], c["rank"], c["adapters"]
    if c["mixed"]:  # decoding rows: each its own adapter, one in eight or so none
        ids = _randint(gen, 0, NA, (M,))
        ids = torch.where(torch.rand(M, generator=gen, device=DEV) < (0.12 if M > 1 else 0.0), -1, ids)
    else:  # prompts one after another
        ids = _randint(gen, 0, NA, (M,)).sort().values
    return {"case": c, "x": _randn(gen, (M, K), dtype), "base": _randn(gen, (M, N), dtype),
            "a": (_randn(gen, (NA, R, K), torch.float32) / math.sqrt(K)).to(dtype),
            "b": (_randn(gen, (NA, N, R), torch.float32) * 0.5 / math.sqrt(R)).to(dtype),
            "scales": 0.5 + torch.rand(NA, generator=gen, device=DEV), "ids": ids.to(torch.int32)}


# ----------------------------------------------------------------- one pass


def _bits(s):
    """The pools as whole numbers: pages are moved bit by bit."""
    return [p if p.dtype == torch.uint8 else p.view(torch.int16) for p in s["pools"]]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from mk import gqa_ops, kv_page_ops, lora_ops, rope_ops

        if kind == "rope":
            return rope_ops.apply_rope(s["x"], s["cos"], s["sin"], positions=s["positions"], layout=c["layout"],
                                       rotary_dim=c["rotary"])
        if kind == "qk":
            q, K, V = gqa_ops.paged_qk_norm_rope_update(
                s["qkv"], s["K"], s["V"], s["table"], s["cos"], s["sin"], s["positions"],
                num_attention_heads=c["hq"], num_key_value_heads=c["hkv"], head_dim=c["d"], q_weight=s["q_weight"],
                k_weight=s["k_weight"], sequences=s["sequences"], eps=1e-6, layout=c["layout"],
                rotary_dim=c["rotary"])
            return {"q": q.reshape(c["tokens"], c["hq"], c["d"]), "K": K, "V": V}
        if kind == "copy":
            kv_page_ops.copy_kv_pages(s["pages"], s["src"], s["dst"])
            return _bits(s)
        if kind == "fork":
            table, lengths, refs, ready = kv_page_ops.fork_kv_sequences(
                s["pages"], s["table"], s["lengths"], s["refs"], s["parents"], reserve=c["reserve"])
            return {"table": table, "lengths": lengths, "refs": refs, "ready": ready, "pool": _bits(s)[0]}
        if kind == "compact":
            table, refs, page_map, live = kv_page_ops.compact_kv_pages(s["pages"], s["table"], s["refs"])
            return {"table": table, "refs": refs, "map": page_map, "live": live, "pool": _bits(s)[0]}
        return lora_ops.lora_add(s["x"], s["base"], s["a"], s["b"], s["ids"], scales=s["scales"])
    plain = {"rope": _plain_rope, "qk": _plain_qk, "copy": _plain_copy, "fork": _plain_fork,
             "compact": _plain_compact, "lora": _plain_lora}
    return plain[kind](s, c)


def _turn(x, c, s, layout, rotary):
    """x [..., heads, d] in fp32, c and s [..., 1, rotary / 2]."""
    h = rotary // 2
    if layout == "half":
        a, b = x[..., :h], x[..., h:rotary]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., rotary:]], dim=-1)
    a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    y = torch.stack([a * c - b * s, a * s + b * c], dim=-1)
    return torch.cat([y.flatten(-2), x[..., rotary:]], dim=-1)


def _plain_rope(s, c):
    x = s["x"]
    pos = s["positions"].long()
    if pos.ndim == 1:
        pos = pos[:, None] + torch.arange(c["seq"], device=DEV)
    at = pos.clamp(min=0)
    y = _turn(x.float(), s["cos"][at][:, :, None], s["sin"][at][:, :, None], c["layout"], c["rotary"])
    if c["pad"]:
        y = torch.where((pos >= 0)[:, :, None, None], y, 0.0)
    return y.to(x.dtype)


def _plain_qk(s, c):
    T, hq, hkv, d, P = c["tokens"], c["hq"], c["hkv"], c["d"], c["page"]
    x = s["qkv"].reshape(T, hq + 2 * hkv, d)
    pos = s["positions"].long()
    at = pos.clamp(min=0)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    qk = x[:, :hq + hkv].float()
    if c["norm"]:
        w = torch.cat([s["q_weight"].float().expand(hq, d), s["k_weight"].float().expand(hkv, d)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-6) * w
    qk = _turn(qk, cos, sin, c["layout"], c["rotary"]).to(x.dtype)
    live = pos >= 0  # row 0 always is: empty rows write what it writes
    owner = torch.arange(T, device=DEV) if s["sequences"] is None else s["sequences"].long()
    owner, at = torch.where(live, owner, owner[0]), torch.where(live, pos, pos[0])
    row = torch.where(live, torch.arange(T, device=DEV), 0)
    page = s["table"][owner, at // P].long()
    s["K"][page, at % P] = qk[row, hq:]
    s["V"][page, at % P] = x[row, hq + hkv:]
    return {"q": torch.where(live[:, None, None], qk[:, :hq], 0.0).to(x.dtype), "K": s["K"], "V": s["V"]}


def _move(pool, src, dst):
    pool[:, dst] = pool[:, src]


def _plain_copy(s, c):
    src, dst = s["src"].long(), s["dst"].long()
    _move(s["pools"][0], src, dst)
    if c["quantized"]:
        _move(s["pools"][1], src, dst)
    return _bits(s)


def _plain_fork(s, c):
    table, lengths, refs, parents = s["table"], s["lengths"].long(), s["refs"], s["parents"].long()
    P, n = c["page"], c["reserve"]
    B, blocks = table.shape
    j, b = torch.arange(blocks, device=DEV), torch.arange(B, device=DEV)
    live, p = parents >= 0, parents.clamp(min=0)
    L = torch.where(live, lengths[p], 0)
    nb = (L + P - 1) // P
    kept = torch.where(j < nb[:, None], table[p].long(), -1)
    drop = table.reshape(-1).long()
    refs = refs.index_add(0, drop.clamp(min=0), -(drop >= 0).to(torch.int32))
    keep = kept.reshape(-1)
    refs = refs.index_add(0, keep.clamp(min=0), (keep >= 0).to(torch.int32))
    new_lengths = L.to(torch.int32)
    if n == 0:
        return {"table": kept.to(torch.int32), "lengths": new_lengths, "refs": refs, "ready": torch.ones_like(live),
                "pool": _bits(s)[0]}
    # a partly filled last page stays with the longest of its rows (the first of those), if nobody else holds it
    part = L % P != 0
    last = torch.where(part, kept.gather(1, (nb - 1).clamp(min=0)[:, None])[:, 0], -1)
    same = (last[:, None] == last) & part & part[:, None]
    key = L % P * B + (B - 1 - b)
    mine = (torch.where(same, key, -1).amax(1) == key) & (refs[last.clamp(min=0)] == same.sum(1))
    copy = part & ~mine
    fits = L + n <= blocks * P
    need = torch.where(live & fits, copy + (L + n + P - 1) // P - nb, 0)
    off = need.cumsum(0) - need
    free = refs == 0
    rank = torch.cumsum(free, 0)
    pages = refs.shape[0]
    ids = torch.zeros(pages + 1, dtype=torch.int64, device=DEV)
    ids = ids.scatter(0, torch.where(free, rank - 1, pages), torch.arange(pages, device=DEV))
    ready = ~live | (fits & (off + need <= rank[-1]))
    k = j - nb[:, None] + copy[:, None].long()
    take = (k >= 0) & (k < need[:, None]) & ready[:, None]
    got = ids[(off[:, None] + k).clamp(0, pages)]
    new_table = torch.where(take, got, kept)
    refs = refs.index_add(0, torch.where(take, got, 0).reshape(-1), take.reshape(-1).to(torch.int32))
    moves = copy & ready & live & (need > 0)
    refs = refs.index_add(0, last.clamp(min=0), -moves.to(torch.int32))
    # rows that copy nothing do as the first that does; no row: page 0 onto itself
    one = moves.to(torch.int32).argmax().reshape(1)
    dst = ids[off.clamp(max=pages)]
    src0, dst0 = torch.where(moves[one], last[one], 0), torch.where(moves[one], dst[one], 0)
    _move(s["pools"][0], torch.where(moves, last, src0), torch.where(moves, dst, dst0))
    return {"table": new_table.to(torch.int32), "lengths": new_lengths, "refs": refs, "ready": ready,
            "pool": _bits(s)[0]}


def _plain_compact(s, c):
    table, refs = s["table"].long(), s["refs"]
    pages = refs.shape[0]
    ids = torch.arange(pages, device=DEV)
    held = refs > 0
    n = held.sum()
    src, dst = torch.nonzero(held & (ids >= n))[:, 0], torch.nonzero(~held & (ids < n))[:, 0]
    page_map = torch.where(held, ids, -1).index_put((src,), dst)
    new_refs = torch.zeros_like(refs).index_put((page_map[held],), refs[held])
    new_table = torch.where(table >= 0, page_map[table.clamp(min=0)], -1)
    _move(s["pools"][0], src, dst)
    return {"table": new_table.to(torch.int32), "refs": new_refs, "map": page_map.to(torch.int32),
            "live": n.to(torch.int32).reshape(1), "pool": _bits(s)[0]}


def _plain_lora(s, c):
    M, R, NA = c["rows"], c["rank"], c["adapters"]
    t = s["x"].float() @ s["a"].reshape(NA * R, -1).float().t()
    pick = (s["ids"][:, None] == torch.arange(NA, device=DEV)) * s["scales"]
    t = (t.reshape(M, NA, R) * pick[:, :, None]).reshape(M, NA * R)
    b = s["b"].float().permute(1, 0, 2).reshape(c["n"], NA * R)
    return (s["base"].float() + t @ b.t()).to(s["base"].dtype)


# ----------------------------------------------------------------- what a pass cannot do without


def work(case):
    c, e = case, 2
    kind = c["kind"]
    if kind == "rope":
        n = c["batch"] * c["seq"]
        return {"bytes": n * (2 * c["h"] * c["d"] * e + 4 * c["rotary"]), "flops": 3 * n * c["h"] * c["rotary"]}
    if kind == "qk":
        heads = c["hq"] + c["hkv"]
        row = 2 * (heads + c["hkv"]) * c["d"] * e + 4 * c["rotary"]
        return {"bytes": c["tokens"] * row, "flops": c["tokens"] * heads * (3 * c["rotary"] + 4 * c["d"] * c["norm"])}
    if kind == "lora":
        use = min(c["rows"], c["adapters"])
        return {"bytes": e * (c["rows"] * (c["k"] + 2 * c["n"]) + use * c["rank"] * (c["k"] + c["n"])),
                "flops": 2 * c["rows"] * c["rank"] * (c["k"] + c["n"])}
    page = 2 * c["layers"] * c["page"] * c["hkv"] * c["d"] * e
    if kind == "copy":
        if c["quantized"]:
            page = page // 2 + 2 * c["layers"] * c["page"] * c["hkv"] * (c["d"] // 64) * 2
        return {"bytes": 2 * c["moved"] * page, "flops": 0}
    if kind == "fork":  # about half of the rows have a parent that another row has too, at an odd place of a page
        B = c["prompts"] * c["beams"]
        blocks = -(-(c["ctx"] + 2 * c["reserve"] + 1) // c["page"])
        moved = 0.35 * B * (c["beams"] > 1) * (c["reserve"] > 0)
        return {"bytes": 8 * B * blocks + 2 * moved * page, "flops": 0}
    pages = 0.75 * c["seqs"] * c["ctx"] / c["page"]
    kept = 1 - c["gone"] / c["seqs"]
    return {"bytes": 8 * pages + 2 * pages * kept * (1 - kept) * page, "flops": 0}


# ----------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """The operators that compute numbers, from their definitions in 64 bits; moved pages have none."""
    c = case
    if c["kind"] in ("copy", "fork", "compact"):
        return None
    s = prepare(case, seed)
    if c["kind"] == "lora":
        x, out = s["x"].double(), s["base"].double()
        for i in range(c["adapters"]):
            rows = torch.nonzero(s["ids"] == i)[:, 0]
            inner = torch.mm(x[rows], s["a"][i].double().t().contiguous())
            out[rows] += s["scales"][i].double() * torch.mm(inner, s["b"][i].double().t().contiguous())
        return out
    h = c["rotary"] // 2
    first = torch.arange(h, device=DEV) * (2 if c["layout"] == "interleaved" else 1)
    second = first + (1 if c["layout"] == "interleaved" else h)

    def rotate(x, pos):  # x [rows, heads, d], pos [rows] >= 0: the complex product
        z = torch.complex(x[..., first], x[..., second])
        z = z * torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if c["kind"] == "rope":
        B, S = c["batch"], c["seq"]
        pos = s["positions"].long().reshape(B, -1)
        pos = (pos if c["pad"] else pos + torch.arange(S, device=DEV)).reshape(-1)
        x = s["x"].double().reshape(B * S, c["h"], c["d"])
        out = torch.zeros_like(x)
        rows = torch.nonzero(pos >= 0)[:, 0]
        out[rows] = rotate(x[rows], pos[rows])
        return out.reshape(s["x"].shape)
    hq, hkv, P = c["hq"], c["hkv"], c["page"]
    rows = torch.nonzero(s["positions"] >= 0)[:, 0]
    pos = s["positions"][rows].long()
    x = s["qkv"].double().reshape(c["tokens"], hq + 2 * hkv, c["d"])[rows]
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q = s["q_weight"].double() * q / torch.sqrt(q.square().mean(-1, keepdim=True) + 1e-6)
        k = s["k_weight"].double() * k / torch.sqrt(k.square().mean(-1, keepdim=True) + 1e-6)
    out = torch.zeros((c["tokens"], hq, c["d"]), dtype=torch.float64, device=DEV)
    out[rows] = rotate(q, pos)
    owner = rows if s["sequences"] is None else s["sequences"][rows].long()
    page = s["table"][owner, pos // P].long()
    K, V = s["K"].double(), s["V"].double()
    K[page, pos % P] = rotate(k, pos)
    V[page, pos % P] = v
    return {"q": out, "K": K, "V": V}
