"""Where the paged cache's values lie, and how its attention cuts the work, walked on the CPU."""
import ctypes

import numpy as np
import pytest

import native_build

I32 = np.ctypeslib.ndpointer(dtype=np.int32)


@pytest.fixture(scope="module")
def lib():
    L = native_build.load("kv_plan", False)
    L.kv_walk.argtypes = [ctypes.c_int] * 4 + [ctypes.c_longlong] + [ctypes.c_int] * 2 + [I32, I32, ctypes.c_void_p,
                                                                                          ctypes.c_longlong] + [ctypes.c_int] * 5 + \
        [I32, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]
    return L


@pytest.mark.parametrize("fmt", [0, 1, 5])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_every_value_has_a_place_of_its_own(lib, fmt, hd):
    assert lib.kv_places(fmt, hd) == 0


def walk(lib, page, rows, lens, group, kv_heads, window, grid, cols=8, table=None, begin="sums", total=None, n_pages=None, width=None):
    width = width or max(1, max(-(-n // page) for n in lens))
    n_pages = n_pages or len(lens) * width
    if table is None:
        table = np.random.default_rng(0).permutation(len(lens) * width)
    table = np.ascontiguousarray(table, dtype=np.int32)
    total = total if total is not None else sum(rows)
    b = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32) if isinstance(begin, str) else begin
    tokens = max(16, max(lens))
    visits = np.zeros((max(total, 1), kv_heads, group, tokens), dtype=np.int32)
    bad_rows, bad_pages = ctypes.c_int(), ctypes.c_int()
    rc = lib.kv_walk(1, kv_heads, 128, page, n_pages, len(lens), width, table, np.asarray(lens, dtype=np.int32),
                     None if b is None else b.ctypes.data, total, group, window, cols, grid, tokens, visits, bad_rows, bad_pages)
    assert rc == 0, rc
    return visits, bad_rows.value, bad_pages.value


@pytest.mark.parametrize("rows,lens", [([1] * 5, [1, 16, 17, 700, 33]), ([3, 0, 9], [3, 50, 1200]), ([40], [40]), ([5, 2], [0, 1]),
                                       ([1], [5000]), ([0, 0], [3, 0])])
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (8, 2), (7, 1), (24, 1)])
@pytest.mark.parametrize("window", [0, 1, 37])
@pytest.mark.parametrize("grid", [1, 7, 592])
@pytest.mark.parametrize("cols", [8, 16])
def test_every_pair_is_visited_once(lib, rows, lens, group, kv_heads, window, grid, cols):
    visits, bad_rows, bad_pages = walk(lib, 32, rows, lens, group, kv_heads, window, grid, cols)
    assert bad_rows == bad_pages == 0
    at = 0
    for r, n in zip(rows, lens):
        for i in range(r):
            pos = n - r + i
            want = np.zeros(visits.shape[-1], dtype=np.int32)
            if pos >= 0:
                want[(max(0, pos - window + 1) if window else 0):pos + 1] = 1
            assert (visits[at + i] == want).all()
        at += r


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30])
@pytest.mark.parametrize("rows,lens", [([8], [3]), ([40], [20]), ([10, 1, 5], [5, 90, 0]), ([3], [3])])
@pytest.mark.parametrize("cols", [8, 16])
def test_a_window_wider_than_any_sequence_is_none(lib, rows, lens, window, cols):
    """Rows in front of the first token have negative positions, from which such a window cannot be taken in 32 bits."""
    visits, bad_rows, bad_pages = walk(lib, 16, rows, lens, 2, 1, window, 7, cols)
    without, _, _ = walk(lib, 16, rows, lens, 2, 1, 0, 7, cols)
    assert bad_rows == bad_pages == 0 and without.sum() > 0
    np.testing.assert_array_equal(visits, without)


def test_one_row_per_sequence_without_an_array(lib):
    visits, _, _ = walk(lib, 16, [1, 1, 1], [4, 90, 1], 4, 2, 0, 444, begin=None)
    assert visits.sum() == (4 + 90 + 1) * 8


@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1])
def test_pages_outside_the_pool_are_not_looked_up(lib, page):
    table = np.array([[0, page, 2], [3, 4, 5]], dtype=np.int32)
    visits, bad_rows, bad_pages = walk(lib, 16, [1, 1], [48, 48], 2, 1, 0, 8, table=table, n_pages=6)
    assert bad_rows == 0 and bad_pages == 1
    assert visits[0, 0, 0].sum() == 32 and visits[1, 0, 0].sum() == 48


@pytest.mark.parametrize("lens,begin", [([49, 40], [0, 1, 2]), ([-1, 40], [0, 1, 2]), ([40, 40], [0, -5, 2]), ([40, 40], [0, 9, 2]),
                                        ([40, 40], [-3, 1, 2]), ([2 ** 31 - 1, -2 ** 31], [0, 1, 2])])
def test_rows_and_lengths_that_cannot_be_right_are_left_out(lib, lens, begin):
    width, tokens = 3, 64
    visits = np.zeros((2, 1, 2, tokens), dtype=np.int32)
    bad_rows, bad_pages = ctypes.c_int(), ctypes.c_int()
    rc = lib.kv_walk(1, 1, 128, 16, 6, 2, width, np.arange(6, dtype=np.int32), np.array(lens, dtype=np.int32),
                     np.array(begin, dtype=np.int32).ctypes.data, 2, 2, 0, 8, 444, tokens, visits, bad_rows, bad_pages)
    assert rc == 0 and bad_rows.value >= 1 and bad_pages.value == 0
    assert visits.max() <= 1 and visits[:, :, :, 40:].sum() == 0
