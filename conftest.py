"""Tests that hold a wrong value run on, and are expected to fail.

``test_topk_divergence`` compares with ``head_loss_oracle.topk_divergence``, whose gradient ``q - p`` takes it that listed
and rest masses sum to one.  Where their sum S is another number, its loss, sum p (log p - log q), has the derivative
``S q - p``: for the one column of the first case below the loss does not depend on ``h`` (q is 1 whatever ``h`` is), and the
oracle's gradient is 0.0118 g w.  In the four cases S is 0.988 to 1.011 and the difference is above the tolerance.
``test_lifted_normalisers`` has the same inputs against the derivative, which is itself tested against differences.
"""

import pytest

WRONG_VALUES = {f"tests/test_head_loss_gpu.py::test_topk_divergence[True-False-False-dtype2-512-{shape}]"
                for shape in ("1-8-1-1", "3-72-40-40", "256-64-600-512", "257-64-512-512")}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid in WRONG_VALUES:
            item.add_marker(pytest.mark.xfail(reason="q - p in place of S q - p where the masses sum to S", strict=True))
