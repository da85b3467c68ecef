"""Sampling at temperatures for which a histogram bin's logits are less than fp32's smallest normal number apart."""

import numpy as np
import pytest

from test_gpu_sampling import agree, dev, draw  # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1e-40, 1e-38, 1.3e-37, 1.4e-37, 1e-36])
@pytest.mark.parametrize("n", [200, 300, 5000, 40000])
def test_tiny_temperatures(dev, n, temperature):
    print(f"sample n={n} temperature={temperature}", flush=True)
    rng = np.random.default_rng(n)
    t = np.float32(temperature)
    f = dict(top_k=np.tile([0, 20, 230, 700, 0, 1500], 4).astype(np.int32),
             top_p=np.repeat([1.0, 0.9, 0.5, 0.999], 6).astype(np.float32),
             min_p=np.tile([0, 0, 0.01, 0, 0.05, 0], 4).astype(np.float32))
    rows = len(f["top_k"])
    u = rng.random(rows).astype(np.float32)
    for highest in (0.0, 1.0, 1000.0):  # the maximum, in temperatures: 0, or of the others' size
        l = (2.5 * rng.standard_normal((rows, n)) * np.float64(t)).astype(np.float32)
        l += np.float32(highest * np.float64(t)) - l.max(axis=1, keepdims=True)
        token, lp, err = draw(dev, l, u, temperature=np.full(rows, t), **f)
        assert err == 0
        agree(token, lp, l, u, temperature=np.full(rows, t), **f)
