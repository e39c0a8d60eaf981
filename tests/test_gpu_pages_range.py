"""Releases of as many pages as ids reach (qvx_kv_free)."""
from __future__ import annotations

import pytest

import qorvix_amd as qvx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_pages", [2 ** 31 - 1, 2 ** 31 - 8191, 2 ** 31 - 8192, 2 ** 31 - 8193])
def test_ids_next_to_2_31(cuda, n_pages):
    """Pages of the last range of ids, which ends where 32 bits do, return with those of the first one, in the order of their ids."""
    torch = cuda
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    extra = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    table = ints([[n_pages - 1, 5, n_pages - 8000], [n_pages - 2, 5, -1]])
    extra[5] = 1
    free, taken, lens = ints([7, 7, 7, 7, 9]), ints([4, 0]), ints([40, 20])
    qvx.kv_free_t(ints([0]), table, lens, extra, free, taken)
    assert taken.tolist() == [2, 0] and free.tolist() == [7, 7, n_pages - 8000, n_pages - 1, 9] and not bool(extra.any())
    assert lens.tolist() == [0, 20] and table.tolist() == [[-1] * 3, [n_pages - 2, 5, -1]]
    qvx.kv_free_t(ints([1]), table, lens, extra, free, taken)
    assert taken.tolist() == [0, 0] and free.tolist() == [5, n_pages - 2, n_pages - 8000, n_pages - 1, 9] and not bool(extra.any())
