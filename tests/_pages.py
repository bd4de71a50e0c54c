"""Cache pools, block tables and counts for the tests of the page operators."""

import numpy as np
import torch

from oracle import serving as sv


def pool(rng, NP, P, spec):
    """Page arrays of random bits: spec = [(shape after [NP, P], dtype)]."""
    out = []
    for shape, dtype in spec:
        n = torch.empty((), dtype=dtype).element_size()
        raw = rng.integers(0, 256, size=(NP, P, *shape, n), dtype=np.uint8)
        out.append(torch.from_numpy(raw).view(dtype).reshape(NP, P, *shape))
    return out


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


def moved(pages, moves):
    """Copies of the arrays with the moves made (all sources read first)."""
    out = []
    for t in pages:
        u = t.clone()
        for a, b in moves:
            u[b] = t[a]
        out.append(u)
    return out


def random_state(rng, B, blocks, P, NP, others=0.1):
    """(table, lengths, refs): rows that share prefixes with earlier rows, pages in random order, some held by others
    or free.  A row's last partly filled page may be shared too."""
    ids = list(rng.permutation(NP))
    refs = np.zeros(NP, np.int64)
    table = np.full((B, blocks), -1, np.int64)
    lengths = np.zeros(B, np.int64)
    for b in range(B):
        share = int(rng.integers(0, b)) if b and rng.random() < 0.6 else -1
        L = int(rng.integers(0, blocks * P + 1))
        if share >= 0:  # behind a whole number of the other's pages, or all of it as a lazy fork leaves it
            if rng.random() < 0.4:
                L, keep = int(lengths[share]), blocks
            else:
                keep = int(rng.integers(0, blocks + 1))
        for j in range(-(-L // P)):
            if share >= 0 and j < keep and (j + 1) * P <= lengths[share] or (share >= 0 and keep == blocks
                                                                            and L == lengths[share]):
                table[b, j] = table[share, j]
            elif ids and refs.sum() >= 0:
                table[b, j] = ids.pop()
            else:
                L = j * P
                break
        L = min(L, int((table[b] >= 0).sum()) * P)
        lengths[b] = L
        table[b, -(-L // P):] = -1
        # now and then a page reserved behind the row's positions
        j = -(-L // P)
        if j < blocks and ids and rng.random() < 0.3:
            table[b, j] = ids.pop()
    for p in table.reshape(-1):
        if p >= 0:
            refs[p] += 1
    extra = rng.random(NP) < others
    refs[extra] += 1
    return table, lengths, refs


def check_fork(got, pages_after, pages_before, table, lengths, refs, parents, P, reserve):
    want_t, want_l, want_r, ready, moves = sv.fork(table, lengths, refs, parents, P, reserve, len(refs))
    g = [t.cpu().numpy() for t in got]
    assert np.array_equal(g[0], want_t), (g[0], want_t)
    assert np.array_equal(g[1], want_l) and np.array_equal(g[2], want_r) and np.array_equal(g[3], ready)
    for a, b in zip(pages_after, moved(pages_before, moves)):
        assert torch.equal(bits(a), bits(b))
    return moves


class Histories:
    """Sequences as their own lists of tokens, beside a pool that is forked, appended to and compacted: what a row
    reads through its table has to be its list."""

    def __init__(self, ops, dev, seed, P, blocks, NP, n):
        self.ops, self.dev, self.P = ops, dev, P
        self.rng = np.random.default_rng(seed)
        self.pages = [torch.full((NP, P, 2), -1, dtype=torch.int32, device=dev),
                      torch.full((NP, P, 3), -1, dtype=torch.float16, device=dev)]
        self.table = torch.full((n, blocks), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(n, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(NP, dtype=torch.int32, device=dev)
        self.rows = [[] for _ in range(n)]
        self.token = 0

    def fork(self, parents, reserve, **kw):
        self.table, self.lengths, self.refs, ready = self.ops.fork_kv_sequences(
            self.pages, self.table, self.lengths, self.refs, parents, reserve=reserve, **kw)
        self.rows = [list(self.rows[p]) if p >= 0 else None for p in parents]
        return ready.tolist()

    def append(self, ready, count):
        table, lengths = self.table.cpu().numpy(), self.lengths.cpu().numpy().copy()
        for b, row in enumerate(self.rows):
            if row is None or not ready[b]:
                continue
            for _ in range(count):
                L = int(lengths[b])
                page = int(table[b, L // self.P])
                assert page >= 0
                self.pages[0][page, L % self.P] = self.token
                self.pages[1][page, L % self.P] = self.token % 2048
                row.append(self.token)
                lengths[b] += 1
                self.token += 1
        self.lengths = torch.from_numpy(lengths).to(self.dev)

    def check(self):
        table, lengths, refs = (t.cpu().numpy() for t in (self.table, self.lengths, self.refs))
        a, b = (t.cpu().numpy() for t in self.pages)
        for r, row in enumerate(self.rows):
            assert lengths[r] == len(row or [])
            for i, token in enumerate(row or []):
                page = table[r, i // self.P]
                assert (a[page, i % self.P] == token).all() and (b[page, i % self.P] == token % 2048).all(), (r, i)
        counts = np.zeros_like(refs)
        for p in table.reshape(-1):
            if p >= 0:
                counts[p] += 1
        assert np.array_equal(counts, refs)

    def compact(self, **kw):
        self.table, self.refs, _, live = self.ops.compact_kv_pages(self.pages, self.table, self.refs, **kw)
        n = int(live)
        assert (self.refs[:n] > 0).all() and (self.refs[n:] == 0).all()


def run_histories(ops, dev, seed, P, blocks, NP, n, steps, **kw):
    h = Histories(ops, dev, seed, P, blocks, NP, n)
    waited = 0
    for _ in range(steps):
        rows = [r for r, row in enumerate(h.rows) if row is not None]
        parents = [int(h.rng.choice(rows)) if rows and h.rng.random() < 0.5 else (r if r < len(h.rows) and
                   h.rows[r] is not None and h.rng.random() < 0.9 else -1) for r in range(n)]
        if not rows:
            h.rows, parents = [[] for _ in range(n)], list(range(n))
        reserve = int(h.rng.integers(0, 4))
        ready = h.fork(parents, reserve, **kw)
        h.check()
        waited += sum(not r for r in ready)
        h.append([r and reserve for r in ready], reserve)
        h.check()
        if h.rng.random() < 0.3:
            h.compact(**kw)
            h.check()
    return waited
