"""Which kernel a grouped forward product of few rows takes (without a GPU: the
rule for 148 SMs)."""
import pytest


# rows, groups, summed values, output columns: the streaming kernel (16) up to 80 MiB of weights in use
@pytest.mark.parametrize("rows,groups,K,N,tile", [
    (1, 8, 1024, 1024, 16), (2, 8, 4096, 4096, 16), (16, 8, 512, 512, 16), (2, 8, 8192, 2048, 16), (1, 1, 8192, 4096, 16),
    (3, 8, 8192, 2048, 32), (2, 8, 16384, 4096, 32), (8, 8, 16384, 1024, 32), (2, 8, 4096, 16384, 32), (17, 8, 512, 512, 32)])
def test_few_rows(rows, groups, K, N, tile):
    import tempname_dcu_b200.ops.grouped  # noqa: F401
    from tempname_dcu_b200.ops import native
    assert native.lib().tdb_grouped_pick_tile(0, rows, groups, K, N) == tile
