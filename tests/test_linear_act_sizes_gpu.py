"""Plans of the dense layer's backward pass at the largest sizes it counts (host arithmetic: nothing is launched)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [1, 64, 256])
def test_column_sums_of_the_most_rows(N):
    """db of so many rows is added up from sums of their blocks: as many as at a smaller number of rows."""
    from strata_b200 import _lib
    from strata_b200.ops import _MOST
    need = lambda M: _lib.load().strata_linear_act_backward_workspace_bytes(M, N, 8, 0, 1, 1, 1, 1, 0, 0, 1)
    assert need(2 ** 30) >= 2 * 4 * N
    for M in (2145700000, _MOST - 1, _MOST):
        # (a few blocks more or less, as rows come in whole ones)
        assert 0.99 * need(2 ** 30) - 256 <= need(M) <= 1.01 * need(2 ** 30) + 256
