"""The queries of the layers' products' workspaces go by sizes and alignment: operands that are not at hand yet count as aligned ones."""
import pytest

import rocwmma_amd as R

AT = 0x100000


@pytest.mark.parametrize("rows,n,k,groups", [(1500, 1496, 1500, 1), (1003, 1001, 1499, 1), (3000, 700, 1003, 4), (1500, 1496, 1504, 1), (100, 512, 8192, 1)])
def test_before_there_are_operands(rows, n, k, groups):
    kw = dict(groups=groups, offsets=AT if groups > 1 else None)
    need = R.linear_workspace_bytes(R.linear_args(R.BF16, R.BF16, rows, n, k, AT, AT, AT, **kw))
    assert R.linear_workspace_bytes(R.linear_args(R.BF16, R.BF16, rows, n, k, None, None, None, **kw)) == need
    if k % 8:
        assert need >= 2 * k * (rows + groups * n)  # both operands laid out evenly
    need = R.linear_backward_workspace_bytes(R.linear_backward_args(R.BF16, R.BF16, rows, n, k, AT, AT, AT, dx=AT, dw=AT, **kw))
    assert R.linear_backward_workspace_bytes(R.linear_backward_args(R.BF16, R.BF16, rows, n, k, None, None, None, dx=AT, dw=AT, **kw)) == need
