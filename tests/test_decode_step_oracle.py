"""The decode-step oracle against definitions worked out by hand and plain probability arithmetic (no device)."""

import math

import numpy as np
import pytest

import decode_step_oracle as dso


def test_to_bf16_rounds_to_nearest_even():
    x = np.array([1.0, 1.00390625, 1.01171875, -1.00390626, 3.0e38, np.inf, np.nan], np.float32)
    _, v = dso.to_bf16(x)
    # fp32 steps at 1 are 2^-23: the fourth literal is -(1 + 2^-8) in fp32, half a bfloat16 step, a tie to the even 1.
    assert v[0] == 1.0 and v[1] == 1.0 and v[2] == np.float32(1.015625) and v[3] == np.float32(-1.0)
    assert np.isinf(v[5]) and np.isnan(v[6])


@pytest.mark.parametrize("u, want", [(0.0, 0), (0.124, 0), (0.125, 1), (0.5, 4), (0.874, 6), (0.875, 7), (0.99, 7)])
def test_equal_logits_split_evenly(u, want):
    assert dso.sample(np.zeros(8), u=u) == (want, pytest.approx(-math.log(8)))


def test_filters_keep_prefixes():
    l = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    drawn = lambda **f: {dso.sample(l, u=u, **f)[0] for u in np.linspace(0, 0.999, 200)}  # noqa: E731
    assert drawn() == {0, 1, 2, 3}
    assert drawn(top_k=2) == {1, 3}
    assert drawn(top_p=0.65) == {1, 3} and drawn(top_p=0.75) == {1, 2, 3} and drawn(top_p=0.05) == {1}
    assert drawn(min_p=0.45) == {1, 2, 3} and drawn(min_p=0.6) == {1, 3} and drawn(min_p=1.0) == {1}
    assert drawn(top_k=2, top_p=0.5) == {1}  # 0.4 of 0.7 is more than half
    assert drawn(temperature=0.0) == {1}
    # ties go to the lower id
    assert dso.sample(np.zeros(5), top_k=1, u=0.9)[0] == 0
    assert {dso.sample(np.zeros(5), top_k=2, u=u)[0] for u in (0.0, 0.49, 0.51, 0.99)} == {0, 1}


def test_shares_follow_the_softmax():
    rng = np.random.default_rng(3)
    l = rng.standard_normal(50).astype(np.float32) * 2
    n = 20000
    got = np.bincount([dso.sample(l, temperature=0.7, u=(i + 0.5) / n)[0] for i in range(n)], minlength=50) / n
    p = np.exp((l - l.max()) / 0.7)
    assert np.abs(got - p / p.sum()).max() <= 1.0 / n + 1e-9


def test_lora_of_no_adapter_is_the_layer():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 64)).astype(np.float32)
    q, a = dso.quantize_rows(x)
    w = rng.integers(-127, 128, size=(5, 64)).astype(np.int8)
    mult, bias = np.full(5, 100, np.float32), np.ones(5, np.float32)
    la, lb = rng.standard_normal((1, 8, 64)), rng.standard_normal((1, 5, 8))
    y, _ = dso.lora(x, q, a, w, mult, bias, la, lb, [2.0], [3], [-1, 0, -1])
    plain = (q.astype(float) @ w.astype(float).T) / (a[:, None].astype(float) * 100) + 1
    assert np.allclose(y[[0, 2]], plain[[0, 2]], rtol=1e-12)
    assert np.allclose(y[1] - plain[1], 2 * lb[0, :, :3] @ (la[0, :3] @ x[1].astype(float)))
