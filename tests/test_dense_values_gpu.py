"""Dense attention: what single entries of K, of weights and of output gradients do to a result, kernel by kernel (algo 2: tensor
cores, 1: 32 bits).

With u = eps / 2 of the type of the tensors (half a step) and w = 2^-24 as in the other tests of this operator.
"""
import math

import pytest
import torch

from sparseattention_b200.ops.dense import dense_attention_forward

pytestmark = pytest.mark.gpu



def normal(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("algo", [1, 2])
def test_one_nan_key_shows_wherever_it_lies(D, dtype, algo):
    """Every place of a tile that is computed in a way of its own: pairs of keys in turn, both members, both halves, and the tail."""
    q, k, v = (normal(1, n, 1, D, dtype=dtype, seed=n) for n in (130, 300, 300))
    for key in (*range(8), *range(64, 72), 127, 128, 131, 255, 256, 299):
        bad = k.clone()
        bad[0, key] = math.nan
        out, _, lse = dense_attention_forward(q, bad, v, scale=D ** -0.5, algo=algo)
        assert out.isnan().all() and lse.isnan().all(), key


@pytest.mark.parametrize("algo", [1, 2])
def test_infinite_scores(algo):
    """Finite bfloat16 rows whose product passes the largest 32-bit number.  An infinite score makes its row NaN, as inf - inf does
    in the definition; minus infinity is a weight of zero."""
    q, k, v = (normal(1, n, 1, 64, dtype=torch.bfloat16, seed=n) for n in (130, 300, 300))
    q[..., 0], k[..., 0] = 0.0, 0.0
    q[0, 17, 0, 0] = 3e38
    for key in (*range(8), 65, 70, 130, 298):
        for sign in (1.0, -1.0):
            one = k.clone()
            one[0, key, 0, 0] = sign * 3e38
            out, _, lse = dense_attention_forward(q, one, v, scale=0.125, algo=algo)
            s = 0.125 * q[0, :, 0].double() @ k[0, :, 0].double().T
            if sign < 0:
                s[17, key] = -math.inf
            want = torch.softmax(s, -1) @ v[0, :, 0].double()
            rest = torch.arange(130, device="cuda") != 17 if sign > 0 else slice(None)
            # weights and result rounded once each, and the rest of the arithmetic (a dot product of 64, exponentials) below 2^-15
            near = torch.softmax(s, -1) @ v[0, :, 0].double().abs() * (2.0 ** -8 + 2.0 ** -15) + want.abs() * 2.0 ** -8
            assert ((out[0, :, 0].double() - want).abs() <= near)[rest].all(), (key, sign)
            assert lse[0, rest, 0].isfinite().all()
            if sign > 0:
                assert out[0, 17].isnan().all() and not lse[0, 17].isfinite().any(), key
