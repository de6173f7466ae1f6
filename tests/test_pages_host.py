"""The paged cache's C entries without a GPU: sizes, and calls that are refused
before anything is launched."""
import ctypes

import pytest

from conftest import load_pkg


@pytest.fixture(scope="module")
def lib():
    pkg = load_pkg()
    pkg.build()
    return pkg.load_library()


@pytest.mark.parametrize("layers,n_pages,page,KH,want", [
    (1, 1, 16, 1, 2 * 16 * 512), (10, 4096, 64, 2, 10 * 2 * 4096 * 64 * 2 * 512), (1, 3, 48, 3, 2 * 3 * 48 * 3 * 512),
    (1, 1 << 20, 1024, 1, 2 * (1 << 20) * 1024 * 512),
    (0, 1, 16, 1, 0), (1, 0, 16, 1, 0), (1, 1, 8, 1, 0), (1, 1, 24, 1, 0), (1, 1, 2048, 1, 0), (1, 1, 16, 0, 0),
    (1, (1 << 20) + 1, 16, 1, 0), (1, 1 << 20, 1024, 2, 0), (1000, 1, 16, 1, 0)])
def test_pool_sizes(lib, layers, n_pages, page, KH, want):
    assert lib.coli_cuda_pages_bytes(layers, n_pages, page, KH, 256) == want
    assert lib.coli_cuda_pages_bytes(layers, n_pages, page, KH, 128) == 0


def test_calls_before_init_are_refused(lib):
    if lib.coli_cuda_available():
        pytest.skip("the backend is up")
    h = ctypes.c_void_p()
    assert lib.coli_cuda_pages_create(ctypes.byref(h), 1, 4, 16, 2, 256, None) == 0
    assert b"not ready" in lib.coli_cuda_last_error() and not h.value
    assert lib.coli_cuda_pages_copy_dev(None, 1, None, None) == 0
    assert lib.coli_cuda_pages_fork_dev(None, 1, None, None, None, None, None, 2, 1) == 0
    assert lib.coli_cuda_pages_compact_dev(None, 1, None, None, 1, None, None) == 0
    assert lib.coli_cuda_gqa_decode_pages_dev(None, 0, 1, None, None, None, None, None, 1, None, 16, 2, 256, 64, 1e-6, 1e7, 1) == 0
    assert lib.coli_cuda_gqa_prefill_pages_dev(None, 0, 1, 1, None, None, None, None, None, None, 1, None, 16, 2, 256, 64, 1e-6,
                                               1e7, 1) == 0
    assert lib.coli_cuda_pages_device_ptr(None, 0, None, None) == 0
    assert lib.coli_cuda_pages_norm_weight(None, 0, None, None, 256) == 0
    assert lib.coli_cuda_pages_workspace_bytes(None) == 0
    assert lib.coli_cuda_pages_set_workspace(None, None, 0) == 0
    lib.coli_cuda_pages_free(None)
