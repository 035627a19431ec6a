"""sh_sample_f32 at temperatures near fp32's ends, against its definition in 64 bits
(as in test_gpu_sample.py)."""
import numpy as np
import pytest

import test_gpu_sample as sampling

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1000, 3000, 40000])
@pytest.mark.parametrize("temperature", [2.0 ** -149, 1e-41, 2e-39, 4e-39, 8e-39, 1.2e-38, 2e-38])
def test_temperatures_below_the_normal_range(ctx, n, temperature):
    # logits whose weights at such a temperature differ, and a row of ordinary ones (temperatures below
    # 8.5e-39 take log2(e) / temperature past fp32's range: with a threshold that did not know of it, of 3,000
    # such logits with top-p 0.5 a row gathered 28 of the 54 tokens it had counted at 4e-39, 1 of 8 at 1e-41)
    rng = np.random.default_rng(n)
    rows = 16
    x = -rng.uniform(0, 40 * max(temperature, 1e-39), (rows, n)).astype(np.float32)
    x[5] = rng.normal(0, 2, n)
    x[6, n // 2:] = -1
    k = np.resize([0, 5, 0, 700, 0, 0, 40, 2500], rows)
    p = np.resize([1.0, 1.0, 0.5, 0.9, 0.99, 0.7, 0.8, 1.0, 0.05], rows)
    sampling.check(ctx, x, np.full(rows, temperature), k, p, np.resize([0, 0, 0.1], rows), rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("n", [1000, 40000])
@pytest.mark.parametrize("temperature", [1e36, 3e38])
def test_temperatures_near_the_largest(ctx, n, temperature):
    rng = np.random.default_rng(n + 1)
    rows = 8
    x = rng.uniform(-3.4e38, 3.4e38, (rows, n)).astype(np.float32)
    x[3] = rng.normal(0, 2, n)
    sampling.check(ctx, x, np.full(rows, temperature), [0, 9, 0, 300, 3000, 0, 0, 2], [1, 1, 0.6, 0.9, 0.5, 0.99, 0.01, 1],
                   None, rng.random(rows).astype(np.float32))
