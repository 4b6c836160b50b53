"""GELU of a dense layer where the normal distribution is small: values and slopes keep their relative precision.

The layer copies inputs (its weight holds one 1 per row), so ``z`` is the input itself.  With ``u`` = 2^-24 the kernels' Phi(z) is
off by at most 1e-5 (bf16) or 9 u (f32) of itself below 0 and by 2e-7 (bf16) or 3 u (f32) above, where Phi is at least a half; the
hardware's exponential and reciprocal are within 2 u each.  The product with ``z`` and the sum of a slope add 2 u, the output's
rounding 2^-8 (bf16) or ``u`` of it.  So: 2^-16 + 2^-8 (1 + 2^-16) for bf16, 16 u for f32, of the value; for a slope
Phi + z phi the first part is of Phi + |z| phi.  Below 1e-36 numbers may be flushed to zero.
"""
import math

import pytest
import torch

U = 2.0 ** -24


def _inputs(M, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(M + K)
    return (torch.rand(M, K, device="cuda", generator=g) * 20.5 - 12.5).to(dtype)


def _copies(N, K, dtype):
    w = torch.zeros(N, K, device="cuda", dtype=dtype)
    w[torch.arange(N), torch.arange(N) % K] = 1
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(16, 64, 64), (100, 128, 72), (40, 1024, 16), (2300, 264, 4100)])
def test_values(dtype, M, K, N):
    """Few rows, 64- and 128-tiles, a split contraction, 256-tiles."""
    from mitune.ops.linear import linear
    x = _inputs(M, K, dtype)
    y = linear(x, _copies(N, K, dtype), activation="gelu")
    z = x.double()[:, torch.arange(N, device="cuda") % K]
    want = 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    bound = (16 * U if dtype == torch.float32 else 2.0 ** -16 + 2.0 ** -8 * (1 + 2.0 ** -16)) * want.abs() + 1e-36
    assert ((y.double() - want).abs() / bound).max().item() <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(16, 64, 64), (100, 128, 72), (3000, 512, 512)])
def test_slopes(dtype, M, K, N):
    from mitune.ops.linear import linear
    x = _inputs(M, K, dtype).requires_grad_()
    dx, = torch.autograd.grad(linear(x, _copies(N, K, dtype), activation="gelu").sum(), x)
    z = x.detach().double()[:, :N]
    cdf, pdf = 0.5 * torch.special.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    want, size = cdf + z * pdf, cdf + z.abs() * pdf
    bound = 16 * U * size if dtype == torch.float32 else 2.0 ** -16 * (1 + 2.0 ** -8) * size + 2.0 ** -8 * want.abs()
    assert ((dx[:, :N].double() - want).abs() / (bound + 1e-36)).max().item() <= 1
    assert not dx[:, N:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_and_nan(dtype):
    """As the formula has them: gelu(inf) = inf, gelu(-inf) = -inf * 0 is not a number."""
    from mitune.ops.linear import linear
    x = torch.tensor([[float("inf")], [float("-inf")], [float("nan")], [1e30], [-1e30], [0.0], [-0.0]], device="cuda", dtype=dtype)
    y = linear(x, torch.ones(1, 1, device="cuda", dtype=dtype), activation="gelu").flatten().tolist()
    assert y[0] == math.inf and math.isnan(y[1]) and math.isnan(y[2]) and y[4] == 0 and y[5] == 0 and y[6] == 0
    assert y[3] == x[3].item()
