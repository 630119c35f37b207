"""Which lists of strided tensors share memory (clip_grads_ refuses them), against a count of every byte."""
import random

import pytest
import torch

from instancerefer_amd import optim


def by_counting(tensors):
    """(a tensor meets itself, two tensors meet), from a count of how often each element of the base is reached"""
    base, itself, both = None, False, False
    for t in tensors:
        seen = torch.zeros(t.untyped_storage().nbytes() // t.element_size(), dtype=torch.int64)
        where = torch.full(tuple(t.shape), t.storage_offset())
        for d, (n, st) in enumerate(zip(t.shape, t.stride())):
            where = where + (torch.arange(n) * st).view([-1] + [1] * (t.dim() - d - 1))
        seen.index_add_(0, where.reshape(-1), torch.ones(t.numel(), dtype=torch.int64))
        itself |= bool((seen > 1).any())
        base = seen.clamp(max=1) if base is None else base + seen.clamp(max=1)
    return itself, base is not None and bool((base > 1).any())


def decided(tensors):
    try:
        optim._refuse_shared(tensors)
    except ValueError:
        return "itself"
    except RuntimeError:
        return "shared"
    return "apart"


def expect(tensors):
    itself, both = by_counting(tensors)
    return "itself" if itself else "shared" if both else "apart"


BASE = torch.zeros(40, 30)
LISTS = {
    "columns": lambda b: [b[:, :5], b[:, 5:8], b[:, 8:]], "columns that meet": lambda b: [b[:, :5], b[:, 4:8]], "a base and its piece": lambda b: [b, b[:, 3:4]],
    "the same twice": lambda b: [b[:, 1:4], b[:, 1:4]], "every other row": lambda b: [b[::2], b[1::2]], "rows that meet": lambda b: [b[::2], b[::3]],
    "every other column": lambda b: [b[:, ::2], b[:, 1::2]], "a column and a row": lambda b: [b[:, 2], b[3]], "a column and a row beside it": lambda b: [b[4:, 2], b[3]],
    "in a gap": lambda b: [b[:, :5], b.view(-1)[35:60]], "not in a gap": lambda b: [b[:, :5], b.view(-1)[33:36]],
    "windows": lambda b: [b.view(-1).unfold(0, 8, 4)], "interleaved by itself": lambda b: [b.view(-1).as_strided((3, 2), (2, 3))],
    "meets itself": lambda b: [b.view(-1).as_strided((4, 2), (2, 4))], "three axes": lambda b: [b.view(4, 10, 30)[:, 2:5, 3:9], b.view(4, 10, 30)[:, 2:5, 9:], b.view(4, 10, 30)[:, 5:]],
    "three axes that meet": lambda b: [b.view(4, 10, 30)[:, 2:5, 3:9], b.view(4, 10, 30)[1:, 4:6]], "rows over the border": lambda b: [b.view(-1).as_strided((4, 10), (30, 1), 25), b[:, 6:20]],
    "rows over the border that meet": lambda b: [b.view(-1).as_strided((4, 10), (30, 1), 25), b[:, :6]], "nothing": lambda b: [b[:0], b[:, 1:3], b[5:, 4:4]],
    "one value": lambda b: [b[3:4, 4:5], b[:, 3:4], b[:3, 4]],
}


@pytest.mark.parametrize("name", sorted(LISTS))
def test_lists(name):
    ts = LISTS[name](BASE)
    assert decided(ts) == expect(ts)


def test_many_random_pieces():
    rng = random.Random(4)
    kinds = set()
    for _ in range(600):
        flat, ts = torch.zeros(rng.choice([60, 200])), []
        for _ in range(rng.randrange(1, 4)):
            dims = rng.randrange(1, 4)
            shape, stride = [rng.randrange(1, 5) for _ in range(dims)], [rng.randrange(1, 12) for _ in range(dims)]
            need = 1 + sum((n - 1) * s for n, s in zip(shape, stride))
            if need <= flat.numel():
                ts.append(flat.as_strided(shape, stride, rng.randrange(flat.numel() - need + 1)))
        want = expect(ts)
        assert decided(ts) == want, [(t.shape, t.stride(), t.storage_offset()) for t in ts]
        kinds.add(want)
    assert kinds == {"itself", "shared", "apart"}


def test_tensors_of_different_types_over_one_storage():
    b = torch.zeros(40, 30)
    half = b.view(torch.float16)                                          # (40, 60) over the same bytes
    assert decided([b[:, :5], half[:, 9:12]]) == "shared" and decided([b[:, :5], half[:, 10:12]]) == "apart"


def test_many_columns_of_one_base_are_quick():
    b = torch.zeros(2000, 3000)
    assert decided([b[:, i:i + 2] for i in range(0, 3000, 3)]) == "apart"
    assert decided([b[:, i:i + 2] for i in range(0, 3000, 3)] + [b[1999:, 7:9]]) == "shared"
    assert decided([b[:, ::2], b[:, 1::2]]) == "apart" and decided([b[::2, ::2], b[1::2, ::2], b[:, 1::2]]) == "apart"
