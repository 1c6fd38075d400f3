"""GPU: the token operators at the edges of what they take -- torch's default type, layouts with long strides, values near the type's largest."""
import math

import pytest
import torch

from tests import token_ref as R
from tests.conftest import rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rn(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=F32) * scale).to(dtype)


@pytest.mark.parametrize("default", [BF16, torch.float64])
def test_results_do_not_depend_on_the_default_type(default):
    """The same bits under any torch default type: statistics and parameter gradients are fp32 buffers whatever it is."""
    from pdae_amd import tokens
    x, dy, w, b = (t.to(DEV) for t in (rn(1, 37, 72, dtype=BF16), rn(2, 37, 72, dtype=BF16), rn(3, 72), rn(4, 72)))
    q, k, v, g = (rn(5 + i, 2, 50, 2, 32, dtype=BF16).to(DEV) for i in range(4))

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b, q, k, v)]
        y = tokens.layer_norm(*leaves[:3])
        o = tokens.attention(*leaves[3:], causal=True)
        torch.autograd.backward([y, o], [dy, g])
        return [y.detach(), o.detach()] + [t.grad for t in leaves]
    want = run()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = run()
    finally:
        torch.set_default_dtype(before)
    for a, c in zip(want, got):
        assert a.dtype == c.dtype and torch.equal(a, c)
