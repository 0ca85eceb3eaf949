"""Plans of so many requests that their rows pass the shared memory that a launch has by itself."""

from __future__ import annotations

import pytest

from test_paged_gpu import plan_problem, run_plan, status_word

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [3071, 3072, 5000, 8192])
def test_plan_of_thousands_of_requests(cuda_dev, requests):
    ctx, new, held, free, tables, tokens = plan_problem(requests, requests, 3, 40, 16)
    status = status_word(cuda_dev)
    got = run_plan(cuda_dev, ctx, new, held, free, 0, tables, 16, tokens, status)
    assert got == O.plan(ctx, new, held, free, 0, tables, 16, tokens)
    assert status.item() == 0
