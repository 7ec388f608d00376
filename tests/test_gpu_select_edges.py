"""Selected pages at the edge of what the entries take, against the references of
test_gpu_select.py."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_select import INF, TYPES, check_select, make_table, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [8, 24, 40, 64, 80, 96, 136, 192, 248])
@pytest.mark.parametrize("bad", [INF, -INF])
def test_infinite_queries(ofh, dt, D, bad):
    """An infinity in one of q's columns, the last among them, ranks pages by the sign
    of that column's bound, also where a row does not fill the words of its lanes."""
    lengths = [700, 333]
    table, total = make_table(D, lengths, 16)
    for column in (D - 1, 0):
        k = randn(1, (total, 2, 16, D), dt)
        sign = torch.from_numpy(np.random.default_rng(D).choice([-1.0, 1.0], (total, 2, 1))).to(TYPES[dt])
        k[..., column] = (k[..., column].abs() + 0.25) * sign
        for H in (2, 6):
            q = randn(2, (2, H, 2, D), dt)
            q[:, ::3, :, column] = bad  # (the first head of each key-value head)
            for scale in (1.0, -1.0):
                check_select(ofh, dt, lengths, H, 2, 2, D, 16, 9, k=k, q=q, table=table, scale=scale, attend=False)
