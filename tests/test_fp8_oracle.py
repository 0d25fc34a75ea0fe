"""The oracle of the 8-bit floats and the experts against values written by hand, and its gradients against
differences."""
import numpy as np
import pytest

import fp8_oracle as fp8


def test_grid_of_the_format():
    assert fp8.GRID[1] == 2.0**-9 and fp8.GRID[8] == 2.0**-6 and fp8.GRID[0x38] == 1 and fp8.GRID[0x7e] == 448
    assert (np.diff(fp8.GRID) > 0).all()


@pytest.mark.parametrize("x, code", [(0, 0), (1, 0x38), (-1, 0xB8), (448, 0x7E), (1.0625, 0x38), (1.1875, 0x3A),
                                     (2.0**-10, 0), (3 * 2.0**-10, 2), (17, 0x58), (-19, 0xDA), (0.2, 0x25)])
def test_codes(x, code):
    assert fp8.encode(np.array([float(x)]))[0] == code


def test_scales():
    x = np.zeros((6, 130))
    x[0, 5], x[1, 5], x[2, 5], x[3, 129], x[4, 0] = 448, 449, 1, -1.75, 2.0**-140
    Q, S = fp8.pack(x)
    assert S.shape == (2, 6) and Q.shape == (6, 256)
    assert S[0, 0] == 1 and S[0, 1] == 2 and S[0, 2] == 2.0**-8 and S[1, 3] == 2.0**-8 and S[0, 4] == S[0, 5] == 2.0**-126
    Q, S = fp8.pack(x, 128)
    assert S.shape == (2, 1) and S[0, 0] == 2 and S[1, 0] == 2.0**-8
    assert fp8.values(Q, S, 6, 130, 128)[0, 5] == 448


def test_route_by_hand():
    l = np.log([[1.0, 2, 4, 8], [8, 8, 1, 1], [1, 1, 1, 1]])
    l[1, 3] = -np.inf
    idx, w = fp8.route(l, None, 2, "softmax", scale=3)
    assert idx.tolist() == [[3, 2], [0, 1], [0, 1]] and np.allclose(w, [[2, 1], [1.5, 1.5], [1.5, 1.5]])
    idx, w = fp8.route(l, None, 2, "softmax", renormalize=False)
    assert np.allclose(w[0], [8 / 15, 4 / 15]) and np.allclose(w[1], [8 / 17, 8 / 17])
    # groups {0, 1} and {2, 3}: the second of the first token is better, the first of the second one
    assert fp8.route(l, None, 2, "sigmoid", 2, 1, 2)[0].tolist() == [[3, 2], [0, 1], [0, 1]]
    # the bias takes part in the choice alone
    idx, w = fp8.route(l, np.array([10.0, 0, 0, 0]), 1, "sigmoid", renormalize=False)
    assert idx.tolist() == [[0], [0], [0]] and np.allclose(w[0], 0.5)
    # nothing to choose
    idx, w = fp8.route(np.full((1, 4), -np.inf), None, 2, "softmax")
    assert idx.tolist() == [[-1, -1]] and not w.any()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient_against_differences(scoring, renormalize):
    rng = np.random.default_rng(1)
    T, E, k, h = 3, 6, 3, 1e-6
    l, dw = rng.standard_normal((T, E)), rng.standard_normal((T, k))
    idx = np.array([[0, 3, 5], [2, -1, 1], [4, 4, 0]])  # no expert, and one twice
    got = fp8.route_grad(l, idx, dw, scoring, renormalize, 2.5)
    for t in range(T):
        for e in range(E):
            d = np.zeros((T, E))
            d[t, e] = h
            f = [(dw * fp8.weights(l + s * d, idx, scoring, renormalize, 2.5)).sum() for s in (1, -1)]
            assert abs(got[t, e] - (f[0] - f[1]) / (2 * h)) < 1e-7  # h^2 of a third derivative, and 2^-52 / h


def test_swiglu_gradient_against_differences():
    rng = np.random.default_rng(2)
    GU, dH, h = rng.standard_normal((2, 8)), rng.standard_normal((2, 4)), 1e-6
    got = fp8.swiglu_grad(GU, dH)
    for i in np.ndindex(GU.shape):
        d = np.zeros(GU.shape)
        d[i] = h
        diff = (dH * (fp8.swiglu(GU + d) - fp8.swiglu(GU - d))).sum() / (2 * h)
        assert abs(got[i] - diff) < 1e-7


def test_order_by_hand():
    o = fp8.order(np.array([[2, 0], [2, -1], [0, 5], [2, 2]]), 3)
    assert o["start"].tolist() == [0, 128, 128, 256] and o["count"].tolist() == [2, 0, 4]
    assert o["slot"].tolist() == [[128, 0], [129, -1], [1, -1], [130, 131]]
    assert o["pair"][:2].tolist() == [1, 4] and (o["pair"][2:128] == -1).all() and o["pair"][128:132].tolist() == [0, 2, 6, 7]
    assert o["expert"].tolist() == [0, 2, -1] and o["rows"] == 384
