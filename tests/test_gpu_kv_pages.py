"""mk_copy_kv_pages, mk_fork_kv_sequences and mk_compact_kv_pages against the
oracle and against sequences kept as lists: bit by bit, whatever the arrays
hold."""

import numpy as np
import pytest
import torch

import mk.kv_page_ops as kp
from oracle import serving as sv
from tests._pages import bits, check_fork, moved, pool, random_state, run_histories

pytestmark = pytest.mark.gpu

# whole 16-byte pages of several sizes, and pages of odd bytes
SPECS = [[((2, 16), torch.float16), ((2, 16), torch.bfloat16)], [((3, 5), torch.uint8), ((3,), torch.float16)],
         [((8, 128), torch.float16), ((8, 64), torch.uint8), ((8, 2), torch.float16)]]


def t32(a, dev):
    return torch.from_numpy(np.asarray(a)).to(torch.int32).to(dev)


@pytest.mark.parametrize("reserve", [0, 1, 9])
@pytest.mark.parametrize("seed", range(10))
def test_fork(dev, seed, reserve):
    rng = np.random.default_rng(100 + seed)
    P, blocks, B = int(rng.integers(1, 17)), int(rng.integers(1, 9)), int(rng.integers(1, 40))
    NP, n = int(rng.integers(B, 3 * B + 10)), int(rng.integers(1, 70))
    table, lengths, refs = random_state(rng, B, blocks, P, NP)
    parents = rng.integers(-1, B, size=n)
    pages = [t.to(dev) for t in pool(rng, NP, P, SPECS[seed % 3])]
    before = [t.clone() for t in pages]
    given = [t32(a, dev) for a in (table, lengths, refs, parents)]
    copies = [t.clone() for t in given]
    got = kp.fork_kv_sequences(pages, *given, reserve=reserve)
    check_fork(got, pages, before, table, lengths, refs, parents, P, reserve)
    assert all(torch.equal(a, b) for a, b in zip(given, copies))


@pytest.mark.parametrize("n,B,blocks,P,NP,reserve", [(4096, 700, 3, 2, 30000, 1), (1025, 1025, 5, 4, 9000, 7),
                                                     (3, 2, 700, 16, 20000, 5000), (300, 1, 2, 1, 400, 1),
                                                     (0, 3, 4, 4, 40, 1), (1500, 4, 3, 8, 8193, 3)])
def test_fork_large(dev, n, B, blocks, P, NP, reserve):
    """Several rows a thread, several turns of the search for free pages, rows that need many pages, none at all."""
    rng = np.random.default_rng(n)
    table, lengths, refs = random_state(rng, B, blocks, P, NP, 0.6)
    parents = rng.integers(-1, B, size=n)
    pages = [t.to(dev) for t in pool(rng, NP, P, [((2,), torch.float16)])]
    before = [t.clone() for t in pages]
    got = kp.fork_kv_sequences(pages, *(t32(a, dev) for a in (table, lengths, refs, parents)), reserve=reserve)
    check_fork(got, pages, before, table, lengths, refs, parents, P, reserve)


@pytest.mark.parametrize("seed", range(8))
def test_compact(dev, seed):
    rng = np.random.default_rng(seed)
    P, NP = 2, [1, 2, 30, 257, 8192, 8200, 20000, 64][seed]
    B = max(1, NP // 8)
    table, _, refs = random_state(rng, B, 6, P, NP, 0.0)
    table[rng.random(B) < 0.5] = -1
    refs = np.bincount(table[table >= 0], minlength=NP) + (rng.random(NP) < (0.1 if seed < 7 else 1.0))
    pages = [t.to(dev) for t in pool(rng, NP, P, SPECS[seed % 3])]
    before = [t.clone() for t in pages]
    got = kp.compact_kv_pages(pages, t32(table, dev), t32(refs, dev))
    want = sv.compact(table, refs)
    assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got[:3], want[:3])) and got[3].tolist() == [want[3]]
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, moved(before, want[4])))


@pytest.mark.parametrize("NP,held,entries", [(16384, 8192, 60), (16384, 16384, 0), (24576, 0, 9), (16385, 1, 20000),
                                             (70000, 40001, 300000), (50, 30, 16385), (8193, 8192, 5),
                                             (8192, 8191, 16384)])
def test_compact_large(dev, NP, held, entries):
    """Live counts at and beside the edges of a workgroup's pages, in any order; tables of more entries than pages."""
    rng = np.random.default_rng(NP + held)
    refs = np.zeros(NP, np.int64)
    refs[rng.permutation(NP)[:held]] = rng.integers(1, 5, size=held)
    table = rng.integers(-1, NP, size=(1, entries)) if entries else np.full((1, 1), -1)
    counts = np.bincount(table[table >= 0], minlength=NP)
    refs = np.where(refs > 0, refs + counts, 0)
    table = np.where((table >= 0) & (refs[table] > 0), table, -1)
    pages = [t.to(dev) for t in pool(rng, NP, 1, [((3,), torch.float16)])]
    before = [t.clone() for t in pages]
    got = kp.compact_kv_pages(pages, t32(table, dev), t32(refs, dev))
    want = sv.compact(table, refs)
    assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got[:3], want[:3])) and got[3].tolist() == [want[3]]
    src, dst = (torch.tensor([m[k] for m in want[4]], dtype=torch.long, device=dev) for k in (0, 1))
    before[0][dst] = before[0][src]
    assert torch.equal(bits(pages[0]), bits(before[0]))


@pytest.mark.parametrize("n", [256, 257, 700])
def test_fork_shared_last_pages(dev, n):
    """Many rows on few last pages of different fill, the free pages behind thousands that are held."""
    rng = np.random.default_rng(n)
    P, blocks, NP, B = 8, 4, 30000, 24
    table = rng.permutation(20000)[:B * blocks].reshape(B, blocks)
    table[B // 2:] = table[:B // 2]  # pairs of rows that share all of their pages, up to different positions
    lengths = rng.integers(2 * P + 1, 3 * P, size=B)
    table[:, 3] = -1
    refs = np.bincount(table[table >= 0], minlength=NP)
    refs[rng.random(NP) < 0.5] += 1
    refs[:26000] = np.maximum(refs[:26000], 1)
    parents = rng.integers(-1, B, size=n)
    pages = [t.to(dev) for t in pool(rng, NP, P, [((2,), torch.float16)])]
    before = [t.clone() for t in pages]
    got = kp.fork_kv_sequences(pages, *(t32(a, dev) for a in (table, lengths, refs, parents)), reserve=9)
    assert check_fork(got, pages, before, table, lengths, refs, parents, P, 9)


@pytest.mark.parametrize("spec", SPECS)
def test_copy(dev, spec):
    rng = np.random.default_rng(3)
    NP = 90
    pages = [t.to(dev) for t in pool(rng, NP, 16, spec)]
    before = [t.clone() for t in pages]
    ids = rng.permutation(NP)
    src, dst = np.concatenate([ids[:30], ids[:10]]), ids[40:80]  # a page may be the source of several copies
    assert kp.copy_kv_pages(pages, t32(src, dev), dst.tolist()) is pages
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, moved(before, list(zip(src, dst)))))
    kp.copy_kv_pages(pages, [], [])
    # more arrays than one launch takes
    many = [torch.full((4, 2, 8), i, dtype=torch.float32, device=dev) + torch.arange(4, device=dev).view(4, 1, 1) * 1000
            for i in range(259)]
    kp.copy_kv_pages(many, [1, 3], [2, 0])
    for i, t in enumerate(many):
        assert t[:, 0, 0].tolist() == [3000.0 + i, 1000.0 + i, 1000.0 + i, 3000.0 + i]


def test_unread_entries(dev, monkeypatch):
    """Where the host does not look, entries outside of the pages and parents outside of the table are empty ones."""
    monkeypatch.setenv("MK_SKIP_DEVICE_RANGE_CHECKS", "1")
    rng = np.random.default_rng(4)
    P, NP = 4, 12
    pages = [t.to(dev) for t in pool(rng, NP, P, SPECS[0])]
    before = [t.clone() for t in pages]
    kp.copy_kv_pages(pages, t32([0, -1, 12, 3, 2 ** 31 - 1, 5], dev), t32([7, 1, 2, -5, 4, 12], dev))
    before = moved(before, [(0, 7)])
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, before))
    table = np.array([[1, 2, -9], [12, 3, 4], [2 ** 31 - 1, 5, -1], [6, 2, 0]])
    lengths, parents = np.array([7, 2 ** 31 - 1, 6, -4]), np.array([0, 0, 1, 2, 4, 2 ** 31 - 1, -2 ** 31, 3, 2])
    refs = kp.count_page_refs(torch.from_numpy(table), NP).numpy()
    got = kp.fork_kv_sequences(pages, *(t32(a, dev) for a in (table, lengths, refs, parents)), reserve=2)
    check_fork(got, pages, before, table, lengths, refs, parents, P, 2)
    before = [t.clone() for t in pages]
    got = kp.compact_kv_pages(pages, t32(table, dev), t32(refs, dev))
    want = sv.compact(table, refs)
    assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got[:3], want[:3]))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, moved(before, want[4])))


@pytest.mark.parametrize("P,blocks,NP", [(4, 6, 30), (1, 9, 25), (16, 3, 60), (3, 5, 8)])
def test_histories(dev, P, blocks, NP):
    run_histories(kp, dev, P, P, blocks, NP, 6, 25)


def test_tables_alone(dev):
    table, lengths = torch.tensor([[0, 1]], dtype=torch.int32, device=dev), [5]
    refs = kp.count_page_refs(table, 4)
    t, L, r, ready = kp.fork_kv_sequences([], table, lengths, refs, [0, 0], page_size=4)
    assert t.tolist() == [[0, 1], [0, 2]] and L.tolist() == [5, 5] and r.tolist() == [2, 1, 1, 0] and all(ready.tolist())
    assert kp.compact_kv_pages([], t, torch.flip(r, [0]).contiguous() * 0 + r)[3].tolist() == [3]


def test_stream_and_graph(dev):
    """A beam step captured: every replay against the oracle, with eager work between the replays."""
    rng = np.random.default_rng(8)
    B, blocks, P, NP = 8, 6, 4, 90
    pages = [t.to(dev) for t in pool(rng, NP, P, SPECS[0])]
    states = [random_state(rng, B, blocks, P, NP) + (rng.integers(-1, B, size=B),) for _ in range(4)]
    given = [t32(a, dev) for a in states[0]]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graph = torch.cuda.CUDAGraph()
    scratch = [t.clone() for t in pages]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        check_fork(kp.fork_kv_sequences(scratch, *given), scratch, pages, *states[0], P, 1)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = kp.fork_kv_sequences(pages, *given)
        new = kp.compact_kv_pages(pages, got[0], got[2])
    for state in states[1:]:
        for t, a in zip(given, state):
            t.copy_(t32(a, dev))
        before = [t.clone() for t in pages]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        table, lengths, refs, ready, moves = sv.fork(*state, P, 1, NP)
        assert np.array_equal(got[0].cpu().numpy(), table) and np.array_equal(got[3].cpu().numpy(), ready)
        want = sv.compact(table, refs)
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(new[:3], want[:3]))
        after = moved(moved(before, moves), want[4])
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, after))


@pytest.mark.parametrize("NP", [40, 9000])
def test_all_rows_end_without_a_workspace(dev, NP):
    """The C entry point with no new rows: the old rows' pages are freed, and no workspace is needed or touched."""
    from mk import _lib

    table = torch.tensor([[3, 7, -1], [3, 9, 2]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([6, 11], dtype=torch.int32, device=dev)
    refs = kp.count_page_refs(table, NP)
    refs[5] = 2
    page = torch.arange(NP * 4, device=dev).half().reshape(NP, 4)
    before = page.clone()
    for ints in (0, 3):  # none; one that is left alone
        new_refs, guard = torch.full_like(refs, -7), torch.full((3,), -7, dtype=torch.int32, device=dev)
        at, size = kp._addresses([page], NP)
        _lib.launch("mk_fork_kv_sequences", dev, at.buffer_info()[0], size.buffer_info()[0], 1, table.data_ptr(),
                    lengths.data_ptr(), refs.data_ptr(), None, None, None, new_refs.data_ptr(), None,
                    guard.data_ptr() if ints else None, ints, 2, 0, 3, 4, NP, 5)
        torch.cuda.synchronize()
        want = torch.zeros_like(refs)
        want[5] = 2
        assert torch.equal(new_refs, want) and (guard == -7).all() and torch.equal(page, before)
