"""CPU: the dropout tests' Philox against the oracle's, and what the dropout entry points refuse on the host."""
import math

import numpy as np
import pytest

import drop_ref


def test_philox_of_the_reference(oracle):
    rng = np.random.default_rng(1)
    for _ in range(20):
        ctr, key = rng.integers(0, 1 << 32, 4, dtype=np.uint64), rng.integers(0, 1 << 32, 2, dtype=np.uint64)
        got = drop_ref.philox([ctr[i:i + 1] for i in range(4)], int(key[0]), int(key[1]))
        assert [int(w[0]) for w in got] == oracle.philox4x32_10(ctr.tolist(), key.tolist()).tolist()


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9])
def test_share_of_kept_elements(p):
    """n draws of probability 1 - p: within 6 standard deviations of the mean."""
    n = 1 << 20
    kept = int(drop_ref.keep(n, p, 7, 3, 0).sum())
    assert abs(kept - n * (1 - p)) <= 6 * math.sqrt(n * p * (1 - p)) + 1e-6 * n


def calls(lib):
    p = [1 << 20 | 256 * i for i in range(10)]
    return {"dropout_forward": lambda *a, q=p: lib.ugk_dropout_forward(*q[:2], 8, *a),
            "dropout_backward": lambda *a, q=p: lib.ugk_dropout_backward(*q[:2], 8, *a),
            "dropout_residual_forward": lambda *a, q=p: lib.ugk_dropout_residual_forward(*q[:3], 8, *a),
            "dropout_residual_backward": lambda *a, q=p: lib.ugk_dropout_residual_backward(*q[:3], 8, *a),
            "dropout_residual_layernorm_forward":
                lambda *a, q=p: lib.ugk_dropout_residual_layernorm_forward(*q[:8], 2, 3, 4, *a),
            "layernorm_dropout_residual_backward":
                lambda *a, q=p: lib.ugk_layernorm_dropout_residual_backward(*q[:10], 2, 3, 4, *a)}


@pytest.mark.parametrize("name", ["dropout_forward", "dropout_backward", "dropout_residual_forward", "dropout_residual_backward",
                                  "dropout_residual_layernorm_forward", "layernorm_dropout_residual_backward"])
def test_refused_on_the_host(name):
    import ugk
    lib, call = ugk.lib, calls(ugk.lib)[name]
    for bad in (1.0, -0.1, 1.5, math.nan, math.inf):
        assert call(bad, 1, 1, 0) == 1 and b"p must be" in lib.ugk_last_error()
    assert call(0.5, 1, 1, -1) == 1 and b"site" in lib.ugk_last_error()
    assert call(0.5, 1, 1, 0, q=[None] * 10) == 1 and b"NULL" in lib.ugk_last_error()


def test_layernorm_pairs_refused_on_the_host():
    import ugk
    lib, p = ugk.lib, [1 << 20 | 256 * i for i in range(10)]
    assert lib.ugk_dropout_residual_layernorm_forward(*p[:8], 2, 3, 0, 0.1, 1, 1, 0) == 1
    assert lib.ugk_dropout_residual_layernorm_forward(*p[:8], -2, 3, 4, 0.1, 1, 1, 0) == 1
    assert lib.ugk_layernorm_dropout_residual_backward(p[0], p[1], p[2], p[0], *p[4:], 2, 3, 4, 0.1, 1, 1, 0) == 1
    assert b"distinct" in lib.ugk_last_error()
    assert lib.ugk_dropout_forward(None, None, 0, 0.1, 1, 1, 0) == 0
    assert lib.ugk_dropout_residual_layernorm_forward(*[None] * 8, 0, 3, 4, 0.1, 1, 1, 0) == 0
    assert lib.ugk_layernorm_dropout_residual_backward(*[None] * 10, 2, 3, 0, 0.1, 1, 1, 0) == 0
    assert lib.ugk_last_error() == b""
