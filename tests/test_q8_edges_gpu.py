"""Rows and products in eight bits at the ends of what the calls allow, against the restatement of tests/q8_reference.py."""
import pytest

import test_q8_gpu as q8
from test_q8_gpu import dev  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- rows that are longer than shared memory

# rows and residual of f32, more rows than there are threads for at once: from dim 28168 on the two rows are longer than the shared memory that a ring has
@pytest.mark.parametrize("rows, dim, w_f32, outputs, place", [(297, 28160, False, "q", "residual"), (297, 28168, True, "qy", "residual"), (300, 32768, False, "q", "x"), (300, 32761, True, "qy", ""),
                                                              (301, 30001, False, "y", "nothing")])
def test_norms_of_the_longest_rows(t0, rt, dev, rows, dim, w_f32, outputs, place):  # noqa: F811
    q8.test_rmsnorm(t0, rt, dev, rows, dim, True, "f32", w_f32, outputs, place)
