"""The tiles that 8-bit products take, without a GPU: what tlm_gemm_mx8_plan answers."""
import pytest

from test_mx8_oracle import plan

# gated products of few rows and more than 32768 columns, some whole rounds of 256 x 256 tiles and a rest: (M, N, K)
WIDE_COLUMNS = [(1, 33024, 512), (16, 33024, 4096), (1, 40960, 4096), (32, 40960, 256), (16, 53248, 16384), (32, 53248, 16384),
                (1, 65568, 8192), (32, 65568, 8192)]


@pytest.mark.parametrize("M,N,K", WIDE_COLUMNS)
def test_few_rows_of_many_columns_are_whole(M, N, K):
    """Up to 32 rows are summed in fp32, by tiles of 16 or 32 rows: no part of them goes to 256 x 256 tiles."""
    for split in (True, False):
        rows, cols, ns, first_rows, first_cols = plan(M, N, K, True, split)
        assert rows in (16, 32) and cols in (64, 128) and ns == 1
        assert (first_rows, first_cols) == (M, N)
