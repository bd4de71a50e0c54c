"""Page operators on the host: the tensor-op paths against the oracle and
against sequences kept as lists, and what is refused."""

import numpy as np
import pytest
import torch

import mk.kv_page_ops as kp
from oracle import serving as sv
from tests._pages import bits, check_fork, moved, pool, random_state, run_histories

SPEC = [((2, 3), torch.float16), ((5,), torch.uint8)]


def t32(a):
    return torch.from_numpy(np.asarray(a)).to(torch.int32)


@pytest.mark.parametrize("reserve", [0, 1, 5])
@pytest.mark.parametrize("seed", range(6))
def test_reference_fork(seed, reserve):
    rng = np.random.default_rng(seed)
    P, blocks, B, NP = int(rng.integers(1, 6)), 4, 5, 20
    table, lengths, refs = random_state(rng, B, blocks, P, NP)
    parents = rng.integers(-1, B, size=7)
    pages = pool(rng, NP, P, SPEC)
    before = [t.clone() for t in pages]
    got = kp.fork_kv_sequences(pages, t32(table), t32(lengths), t32(refs), t32(parents), reserve=reserve,
                               backend="reference")
    check_fork(got, pages, before, table, lengths, refs, parents, P, reserve)


@pytest.mark.parametrize("seed", range(6))
def test_reference_compact(seed):
    rng = np.random.default_rng(seed)
    P, NP = 3, 17
    table, _, refs = random_state(rng, 4, 4, P, NP)
    table[rng.integers(0, 4)] = -1
    refs = np.bincount(table[table >= 0], minlength=NP) + (rng.random(NP) < 0.1)
    pages = pool(rng, NP, P, SPEC)
    before = [t.clone() for t in pages]
    got = kp.compact_kv_pages(pages, t32(table), t32(refs), backend="reference")
    want = sv.compact(table, refs)
    assert all(np.array_equal(g.numpy(), w) for g, w in zip(got[:3], want[:3])) and int(got[3]) == want[3]
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, moved(before, want[4])))


def test_reference_copy():
    rng = np.random.default_rng(0)
    pages = pool(rng, 9, 2, SPEC)
    before = [t.clone() for t in pages]
    assert kp.copy_kv_pages(pages, [1, 1, 8], torch.tensor([0, 3, 4]), backend="reference") is pages
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(pages, moved(before, [(1, 0), (1, 3), (8, 4)])))


@pytest.mark.parametrize("P,blocks,NP", [(4, 6, 30), (1, 9, 25), (5, 3, 60), (3, 5, 8)])
def test_reference_histories(P, blocks, NP):
    waited = run_histories(kp, torch.device("cpu"), P, P, blocks, NP, 6, 25, backend="reference")
    assert (waited > 0) == (NP < 60 or P * blocks < 40)  # pages or table rows run out, and nothing is lost


def test_rows_that_need_nothing_are_ready():
    """Behind a row whose pages did not suffice, one that needs none is ready, and a full row is not."""
    table, lengths = t32([[0, -1], [1, -1], [2, 3]]), t32([4, 2, 8])
    refs = kp.count_page_refs(table, 4)
    for parents, ready in (([0, 1, 2], [False, True, False]), ([1, 1, 2], [True, True, False])):
        args = table, lengths, refs, t32(parents)
        got = kp.fork_kv_sequences([], *args, reserve=1, page_size=4, backend="reference")
        want = sv.fork(*(a.numpy() for a in args), 4, 1, 4)
        assert got[3].tolist() == ready == want[3].tolist()
        assert np.array_equal(got[0].numpy(), want[0]) and np.array_equal(got[2].numpy(), want[2])


def test_count_page_refs():
    counts = kp.count_page_refs(torch.tensor([[0, 2, -1], [2, 7, 2]]), 4)
    assert counts.tolist() == [1, 0, 3, 0] and counts.dtype == torch.int32


def test_refusals():
    rng = np.random.default_rng(1)
    pages = pool(rng, 8, 4, SPEC)
    table, lengths = t32([[0, 1, -1], [2, -1, -1]]), t32([6, 3])
    refs = kp.count_page_refs(table, 8)
    ok = dict(pages=pages, block_table=table, lengths=lengths, ref_counts=refs, parents=[0, 1], backend="reference")
    kp.fork_kv_sequences(**ok)
    for kw in (dict(parents=[2]), dict(parents=[-2]), dict(parents=[[0]]), dict(parents=[0] * 4097), dict(lengths=t32([13, 0])),
               dict(lengths=t32([-1, 0])), dict(lengths=lengths[:1]), dict(reserve=-1), dict(ref_counts=refs - 1),
               dict(ref_counts=refs[:0]), dict(ref_counts=refs[:7]), dict(block_table=table[0]),
               dict(block_table=t32([[0, 8, -1], [2, -1, -1]])), dict(block_table=table[:, :0]), dict(pages=[]),
               dict(pages=pages + [pages[0][:7]]), dict(pages=[pages[0], pages[1][:, :2]]), dict(pages=[pages[0][:, :, 0, 0].t()]),
               dict(page_size=3), dict(pages=[], page_size=0), dict(pages=[pages[0].transpose(2, 3)]), dict(backend="x"),
               dict(pages=[pages[0][:, 0, 0, 0]])):
        with pytest.raises(ValueError):
            kp.fork_kv_sequences(**{**ok, **kw})
    for kw in (dict(block_table=table.float()), dict(ref_counts=refs.double()), dict(lengths=lengths.float()),
               dict(parents=torch.zeros(2))):
        with pytest.raises(TypeError):
            kp.fork_kv_sequences(**{**ok, **kw})
    with pytest.raises(ValueError, match="31 bits"):
        kp.fork_kv_sequences([], table, lengths, refs, [0], page_size=2 ** 30)
    for kw in (dict(src=[0], dst=[8]), dict(src=[-1], dst=[0]), dict(src=[0, 1], dst=[2, 2]), dict(src=[0, 1], dst=[1, 2]),
               dict(src=[0], dst=[0]), dict(src=[0, 1], dst=[2]), dict(src=[[0]], dst=[[1]])):
        with pytest.raises(ValueError):
            kp.copy_kv_pages(pages, kw["src"], kw["dst"], backend="reference")
    with pytest.raises(ValueError):
        kp.copy_kv_pages([], [0], [1])
    with pytest.raises(TypeError):
        kp.copy_kv_pages(pages, torch.zeros(1), [1])
    with pytest.raises(ValueError):
        kp.compact_kv_pages(pages, table, refs - 1, backend="reference")
    for fn in (lambda: kp.copy_kv_pages(pages, [0], [1]), lambda: kp.compact_kv_pages(pages, table, refs),
               lambda: kp.fork_kv_sequences(**{**ok, "backend": "auto"})):
        with pytest.raises(ValueError, match="ROCm device"):
            fn()
