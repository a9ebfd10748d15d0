"""The policy operators at the edges of what they allow: calls that the other tests do not make, each against 64-bit
formulas, against the same work done another way, or refused."""
import pytest

from test_policy_gpu import TYPES, check_norm, norm_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("m", [1, 3, 33, 65])
@pytest.mark.parametrize("c", [24, 200, 1500])
def test_norm_without_eps(t, gate, eps, m, c):
    """eps = 0 (and one that 32 bits round to 0) for rows that are not zero: threads behind the last row, of which every
    width class has some at these row counts, add nothing to the sums over the rows."""
    check_norm(*norm_case(m, c, t, gate), 0.5, eps, f"{m}x{c} {gate} eps={eps}")
