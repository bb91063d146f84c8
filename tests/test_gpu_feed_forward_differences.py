"""Gradients of the feed-forward block against central differences along the gradient itself, where the difference is as
large as a step of its size can make it."""

import math

import pytest
import torch

from tests.test_gpu_feed_forward import ACTS, NAMES, _F, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n,width,hidden", [(40, 64, 96), (300, 40, 50), (20, 48, 2000)])
def test_gradient_along_itself(n, width, hidden, act):
    """The direction v is the gradient scaled to elements of order one, so that the quotient is |g| |v|. With steps of 2^-8
    (float64, these sizes) the next term of the expansion is up to 3.2e-5 of it, and roundings of y by 1e-6 of its size come
    to 4e-6."""
    (x, w_in, w_out), grad = _inputs(n, width, hidden, torch.float32, seed=1)
    args = (act, 1.0, width ** -0.5, hidden ** -0.5)
    got = _run(x, w_in, w_out, *args, grad)
    e = 2.0 ** -8
    for k, name in enumerate(NAMES[1:]):
        v = got[name] * (math.sqrt(got[name].numel()) / got[name].norm())
        sides = []
        for s in (e, -e):
            t = [x, w_in, w_out]
            t[k] = t[k] + s * v
            sides.append((_F().gated_feed_forward(*t, *args).double() * grad).sum())
        quotient, want = float(sides[0] - sides[1]) / (2 * e), float((got[name].double() * v).sum())
        assert want > 0 and abs(quotient / want - 1) <= 2.0 ** -13, (name, quotient, want)
