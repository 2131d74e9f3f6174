"""A workspace for max_m rows of max_k covers every smaller batch (no GPU)."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from talechime_b200 import _lib, build

    build.build()
    return _lib.lib()


@pytest.mark.parametrize("k", [32, 256, 1024, 2048, 2080, 4096, 6144, 8192, 16384])
def test_workspaces_grow_with_the_rows(lib, k):
    """The kernels that serve up to 32 rows take turns, and the next may need less: 12 rows of 6144
    86 KB where 11 need 2.5 MB."""
    sizes = [lib.q8lin_workspace_bytes(m, k) for m in list(range(1, 80)) + [127, 128, 129, 1000, 4096]]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("m", [1, 2, 4, 5, 8, 11, 12, 16, 17, 32, 33, 100, 1000])
def test_workspaces_grow_with_the_width(lib, m):
    sizes = [lib.q8lin_workspace_bytes(m, k) for k in range(32, 12289, 32)]
    assert sizes == sorted(sizes)
