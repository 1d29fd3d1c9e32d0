"""The rules that choose a kernel for a product with fp16 or bf16 matrices, asked on the CPU: what its tables of measurements say on
both sides of each border."""
import pytest

import half_rules as rules


@pytest.mark.parametrize("n,n_mat,rows,paired,want", [
    (96, 64, 4096, False, 16), (192, 64, 4096, False, 32), (384, 64, 4096, False, 32), (385, 64, 4096, False, 128),
    (768, 128, 1408, True, 32), (769, 128, 1408, True, 128), (64, 1, 4096, False, 16), (65, 1, 4096, False, 32), (256, 1, 4096, False, 32),
    (512, 1, 4096, False, 128), (2048, 1, 4096, False, 128), (8192, 1, 8192, False, 256), (16412, 32, 2816, False, 256),
    (16384, 128, 1408, True, 128), (8192, 2, 4096, True, 256), (1 << 20, 1, 32, False, 32)])
def test_capacity(n, n_mat, rows, paired, want):
    assert rules.capacity(n, n_mat, rows, paired) == want


@pytest.mark.parametrize("n,n_mat,rows,want", [(192, 128, 2816, 16), (16384, 128, 2816, 96), (16384, 32, 2816, 96), (700, 3, 64, 32)])
def test_capacity_of_two_terms(n, n_mat, rows, want):
    assert rules.capacity(n, n_mat, rows, x_terms=2) == want


@pytest.mark.parametrize("n,n_mat,rows,cols,want", [(96, 64, 4096, 1408, True), (512, 128, 1408, 2816, True), (1120, 128, 1408, 2816, True),
                                                    (192, 32, 1024, 1024, False), (12, 1, 16384, 4096, True), (24, 1, 16384, 4096, False)])
def test_weights_past_the_caches(n, n_mat, rows, cols, want):
    assert rules.once(n, n_mat, rows, cols, rows == 1408) == want
