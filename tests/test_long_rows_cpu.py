"""Layer norm of rows past 2^27 columns, on the CPU behind launch_stub.cpp: the
grids cover all columns within the runtime's limit on a launch (its threads
fit 32 bits), whose refusal ended such calls."""
import pytest

from test_launches_cpu import _child, stub  # noqa: F401

BODY = """
n = %d
need = L.qgemm_layer_norm_backward_workspace_bytes(1, n)
assert need == 2048 + 8 * n
stub.stub_reset(0)
st = L.qgemm_layer_norm_backward(far(0), n, far(1), n, 1, 1, n, far(2), far(3), None, 0, far(4), n, far(5), far(6), P(far(7)),
                                 need, None)
assert st == 0, st
got = launches()
dx, cols, sums = got[0], got[1], got[2:]
assert dx[1:5] == (1, 1, 1, 1024)
assert n <= cols[1] * 256 < n + 256 and cols[2] == 1, cols
assert 2 * n <= sum(s[1] for s in sums) * 64 < 2 * n + 64 and all(s[1] * s[4] < 1 << 32 for s in sums), sums
assert len({s[5] for s in sums}) == 1
print("ok")
"""


@pytest.mark.parametrize("n", [40000, 2 ** 27, 2 ** 27 + 1, 2 ** 30 + 8, 2 ** 31 - 300, 2 ** 31 - 1])
def test_backward_launches(stub, n):  # noqa: F811
    assert _child(stub, BODY % n) == ["ok"]
