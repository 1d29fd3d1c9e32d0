"""The host-array forms of the products (MoeContext.MatMul, MatMulK, MatMulI8, ExpertsI8), without a GPU: a stand-in for the
library records its calls, and what these forms refuse never reaches a product."""
import numpy as np
import pytest

I8, F32 = np.int8, np.float32


class Calls:
    """Every entry point returns PHX_OK and is recorded; phx_weight_shape answers for `shapes`."""

    def __init__(self, shapes):
        self.shapes, self.made = shapes, []

    def __getattr__(self, name):
        def call(*args):
            self.made.append(name)
            if name == "phx_weight_shape":
                if args[0] not in self.shapes:
                    return -1
                for p, v in zip(args[1:], self.shapes[args[0]]):
                    p._obj.value = v
            if name == "phx_moe_last_error":
                return b""
            return 0
        return call


@pytest.fixture
def host(pkg):
    """A context over the stand-in; handles 1: 64 x 256 plain, 2: 4 x 128 x 256 paired, 3: 4 x 256 x 64."""
    c = pkg.MoeContext.__new__(pkg.MoeContext)
    c.lib, c.h = Calls({1: (1, 64, 256), 2: (4, 128, 256), 3: (4, 256, 64)}), 1
    return c


def product(host, name, rows, cols, T=2, handle=1):
    xq = np.zeros((T, cols), I8)
    if name == "MatMul":
        return host.MatMul(handle, rows, cols, xq, np.zeros((T, cols // 32), np.uint16))
    if name == "MatMulK":
        return host.MatMulK(handle, rows, cols, xq, np.zeros((T, cols // 256), F32))
    return host.MatMulI8(handle, rows, cols, xq, np.zeros(T, F32))


PRODUCTS = {"MatMul": "phx_matmul", "MatMulK": "phx_matmul_k", "MatMulI8": "phx_matmul_i8"}


@pytest.mark.parametrize("name", list(PRODUCTS))
def test_products_go_by_the_handles_sizes(host, pkg, name):
    for rows, cols in ((63, 256), (65, 256), (64, 512), (256, 64 * 4)):
        with pytest.raises(pkg.ArgumentError):
            product(host, name, rows, cols)
    with pytest.raises(pkg.ArgumentError):
        product(host, name, 64, 256, handle=None)
    assert PRODUCTS[name] not in host.lib.made
    product(host, name, 64, 256)
    assert PRODUCTS[name] in host.lib.made


def experts(host, d, T=3, k=2):
    return host.ExpertsI8(2, 3, 1, np.zeros((T, d), I8), np.zeros(T, F32), np.zeros((T, k), np.int32), np.zeros((T, k), F32))


def test_experts_go_by_the_handles_sizes(host, pkg):
    for d in (224, 288, 512):
        with pytest.raises(pkg.ArgumentError):
            experts(host, d)
    assert "phx_experts_i8" not in host.lib.made
    assert experts(host, 256).shape == (3, 256)
    assert "phx_experts_i8" in host.lib.made


@pytest.mark.parametrize("bad", [np.full((3, 256), 200, np.uint8), np.full((3, 256), -129, np.int64), np.full((3, 256), 0.5),
                                 np.full((3, 256), 128.0, F32), np.full((3, 256), np.nan, F32)])
def test_quants_that_int8_does_not_hold(host, pkg, bad):
    ids, w = np.zeros((3, 2), np.int32), np.zeros((3, 2), F32)
    with pytest.raises(pkg.ArgumentError):
        host.MatMulI8(1, 64, 256, bad, np.zeros(3, F32))
    with pytest.raises(pkg.ArgumentError):
        host.ExpertsI8(2, 3, 1, bad, np.zeros(3, F32), ids, w)
    with pytest.raises(pkg.ArgumentError):
        host.weight_upload_i8(1, 3, 256, bad, np.zeros(3, F32))
    assert not {"phx_matmul_i8", "phx_experts_i8", "phx_weight_upload_i8"} & set(host.lib.made)


def test_ids_that_int32_does_not_hold(host, pkg):
    """An id past 32 bits is no expert; cut to 32 bits it would be expert 0."""
    xq, xd, w = np.zeros((3, 256), I8), np.zeros(3, F32), np.zeros((3, 2), F32)
    for bad in (np.full((3, 2), 1 << 32), np.full((3, 2), 0xFFFFFFFF, np.uint32), np.full((3, 2), 0.5)):
        with pytest.raises(pkg.ArgumentError):
            host.ExpertsI8(2, 3, 1, xq, xd, bad, w)
    assert "phx_experts_i8" not in host.lib.made
    host.ExpertsI8(2, 3, 1, np.full((3, 256), 127.0), xd, np.full((3, 2), -1, np.int64), w)  # these they hold
    assert "phx_experts_i8" in host.lib.made
