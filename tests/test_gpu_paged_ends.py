"""Pages at the ends of what they take: the smallest caps."""
import pytest

from test_gpu_paged import TYPES, B, Case, check_attention, dev, run_attention  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news", [[1, 3, 1], [40, 3, 70]])
@pytest.mark.parametrize("cap", [2.0 ** -149, 1e-40, 2.0 ** -126, 1e-30, 2.0 ** -41, 2.0 ** -40, 1e-6])
def test_the_smallest_caps(B, dev, dtype, news, cap):
    """Every position weighs the same to the last place, whatever its score is (below 0, above, 0 itself).  The bounds of tests/test_gpu_paged.py: a cap may
    be taken for one of up to 2^-40, which moves a score by 2^-39 at most, less than the 4 u that they have for an exponential."""
    c = Case(dtype, 4, 2, 64, 16, [120, 60, 90], news, seed=12)
    c.qkv[1] = 0                                 # (a query of zeros: its scores are 0)
    check_attention(c, *run_attention(B, dev, c, 0.125, cap), 0.125, cap)
