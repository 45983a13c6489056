"""The gradient clip where its tensors fill the kernels' tables of 48 and 768, with the bounds of
test_gpu_clip.py."""

import math

import pytest

from oracle import step_oracle as O
from tests.test_gpu_clip import BF16, F32, check, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("n", [47, 48, 49, 767, 768, 769, 1536, 1537, 1700])
def test_tables_that_are_just_full_and_just_over(n, norm_type):
    g = tensors([(i * 37) % 211 + 1 for i in range(n)], [F32, BF16], 1)
    if norm_type == math.inf:  # the largest is in the last tensor, then in the first
        g[-1][0] = 50.0
        check([t.clone() for t in g], 0.3, norm_type)
        g[0][0] = -60.0
    want = O.grad_norm(g, norm_type)
    check([t.clone() for t in g], 0.2 * want, norm_type)
    check([t.clone() for t in g], 0.2 * want, norm_type, out=[t.clone() for t in g])


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("n", [48, 768])
def test_empty_tensors_after_and_between(n, norm_type):
    """A second table may have nothing to take."""
    full = [(i * 37) % 211 + 1 for i in range(n)]
    for sizes in (full + [0] * 900, [0] * 900 + full, [s for f in full for s in (0, f)], [0] * 1000):
        g = tensors(sizes, [F32, BF16], 1)
        check(g, 0.2 * O.grad_norm(g, norm_type) + 1.0, norm_type)


@pytest.mark.parametrize("at", [0, 768, 1699])
def test_a_nan_in_any_table_reaches_the_norm(at):
    import spark_gpt_b200 as b200
    for norm_type in (2.0, math.inf):
        g = tensors([5] * 1700, [F32, BF16], 1)
        g[at][2] = math.nan
        before = [t.clone() for t in g]
        assert math.isnan(float(b200.clip_grads(g, 0.1, norm_type=norm_type)))
        assert all((a.nan_to_num(7.0) == b.nan_to_num(7.0)).all() for a, b in zip(g, before))
