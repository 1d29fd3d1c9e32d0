"""The arrays that MoeContext.lora_set takes, without a GPU: a stand-in for the library reads what the addresses that it is given hold,
as phx_lora_set does, and arrays of another type or size never reach it."""
import ctypes as C

import numpy as np
import pytest

ROWS, COLS, RANK = 24, 16, 4


class Library:
    """phx_lora_create hands out handle 7; phx_lora_set copies rank x COLS and ROWS x rank 16-bit values from its addresses, behind
    the allocations that a program makes meanwhile."""

    def __init__(self):
        self.set, self.freed = [], []

    def phx_lora_create(self, h, type_, n_slot, max_rank, rows, cols, out):
        out._obj.value = 7
        return 0

    def phx_lora_set(self, h, handle, slot, rank, a, b, scale):
        between = [np.full(n, 0x7E7E, np.uint16) for n in (RANK * COLS, ROWS * RANK) for _ in range(8)]
        read = lambda at, n: None if at is None else np.frombuffer(C.string_at(at, 2 * n), np.uint16).copy()  # noqa: E731
        self.set.append((rank, read(a, rank * COLS), read(b, ROWS * rank)))
        del between
        return 0

    def phx_lora_free(self, h, handle):
        self.freed.append(handle)


@pytest.fixture
def host(pkg):
    c = pkg.MoeContext.__new__(pkg.MoeContext)
    c.lib, c.h = Library(), 1
    return c


def matrices(type_):
    rng = np.random.default_rng(type_)
    if type_ == 1:
        return rng.standard_normal((RANK, COLS)).astype(np.float16), rng.standard_normal((ROWS, RANK)).astype(np.float16)
    return rng.integers(0, 1 << 16, (RANK, COLS)).astype(np.uint16), rng.integers(0, 1 << 16, (ROWS, RANK)).astype(np.uint16)


@pytest.mark.parametrize("type_", [1, 30])
def test_views_arrive_as_they_are(host, type_):
    """A and B as whole arrays, transposed views, every second column of a wider array, and one row after another backwards."""
    a, b = matrices(type_)
    wide_a, wide_b = np.repeat(a, 2, 1), np.repeat(b, 2, 1)
    h = host.lora_create(type_, 2, RANK, ROWS, COLS)
    forms = [(a, b), (np.ascontiguousarray(a.T).T, np.ascontiguousarray(b.T).T), (wide_a[:, ::2], wide_b[:, 1::2]),
             (np.ascontiguousarray(a[::-1])[::-1], np.ascontiguousarray(b[::-1])[::-1]), (a.ravel(), b.ravel())]
    for fa, fb in forms:
        host.lora_set(h, 1, RANK, fa, fb, 0.5)
        rank, got_a, got_b = host.lib.set[-1]
        np.testing.assert_array_equal(got_a, a.ravel().view(np.uint16))
        np.testing.assert_array_equal(got_b, b.ravel().view(np.uint16))


@pytest.mark.parametrize("type_", [1, 30])
def test_other_types_and_sizes_are_refused(host, pkg, type_):
    a, b = matrices(type_)
    h = host.lora_create(type_, 2, RANK, ROWS, COLS)
    other = np.uint16 if type_ == 1 else np.float16
    for bad in ((a.astype(np.float32), b), (a, b.astype(np.float32)), (a.astype(np.float64), b), (a.view(other), b), (a, b.view(other)),
                (a, b.view(np.int16)), (a[:-1], b), (a, b[:-1]), (a, b[:, :-1]), (a.ravel()[1:], b), (a, b.ravel()[1:]), (a.T, b), (a, b.T),
                (np.vstack([a, a]), b), (a[:0], b)):
        with pytest.raises(pkg.ArgumentError):
            host.lora_set(h, 0, RANK, *bad)
    with pytest.raises(pkg.ArgumentError):
        host.lora_set(h, 0, RANK - 1, a, b)
    with pytest.raises(pkg.ArgumentError):
        host.lora_set(h + 1, 0, RANK, a, b)
    assert not host.lib.set


def test_addresses_and_empty_slots(host, pkg):
    """Addresses go through as they are, beside an array too; rank 0 reads neither; a freed handle's arrays are refused."""
    a, b = matrices(1)
    h = host.lora_create(1, 2, RANK, ROWS, COLS)
    host.lora_set(h, 0, RANK, a.ctypes.data, b.ctypes.data)
    host.lora_set(h, 0, RANK, a.ctypes.data, np.ascontiguousarray(b.T).T)
    for rank, got_a, got_b in host.lib.set:
        np.testing.assert_array_equal(got_a, a.ravel().view(np.uint16))
        np.testing.assert_array_equal(got_b, b.ravel().view(np.uint16))
    host.lora_set(h, 0, 0, a, None)
    host.lora_set(h, 0, 0, None, None)
    assert [s[1:] for s in host.lib.set[2:]] == [(None, None)] * 2
    host.lora_free(h)
    with pytest.raises(pkg.ArgumentError):
        host.lora_set(h, 0, RANK, a, b)
