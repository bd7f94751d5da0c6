"""GPU: quantr_logprobs_dev at small temperatures, with barred tokens, against
64-bit sums; formulas and tolerances are test_logprobs_gpu.py's."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_logprobs_gpu import BF16, DTYPE, F16, F32, check, logits, run, tokens  # noqa: E402


def near(rows, V, type_, temperature, base, seed=0):
    """Logits a few temperatures apart, around `base`."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, V, generator=g, device="cuda", dtype=torch.float64) * 2 * temperature + base
    return x.to(DTYPE[type_])


@pytest.mark.parametrize("V", [40, 5000, 40003])
@pytest.mark.parametrize("temperature,base", [(1e-2, 30.0), (1e-3, 10.0), (1e-4, -7.0), (2e-5, 1.0), (1e-6, 0.5)])
def test_large_logits_over_small_temperatures(qr_gpu, temperature, base, V):
    """Thousands of temperatures from 0, a few of them apart: the weights go by
    the differences, which the large quotients do not blur."""
    x = near(4, V, F32, temperature, base, seed=V)
    t = tokens(4, V)
    check(run(qr_gpu, x, 5, t, temperature), x, 5, t, temperature)


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("temperature", [1e-30, 1e-12, 1e-9, 5e-9, 3e-8])
def test_temperatures_that_leave_one_token(qr_gpu, type_, temperature):
    x = logits(4, 5000, type_, seed=7)
    t = tokens(4, 5000)
    check(run(qr_gpu, x, 5, t, temperature), x, 5, t, temperature)


@pytest.mark.parametrize("V", [1, 40, 5000, 40003])
@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("temperature,top", [(1e-30, 3.0), (1e-9, 3.0), (4e-9, 3.0), (1e-7, 3.0), (1e-9, 1e-3), (1e-30, 0.0)])
def test_barred_tokens_at_small_temperatures(qr_gpu, type_, temperature, top, V):
    """A barred token has weight 0, however small the temperature: the entropy
    is that of the others, not a NaN."""
    x = logits(4, V, type_, seed=V, sigma=top / 3)
    x[:, 1::2] = -math.inf
    x[1, 1::2] = torch.finfo(x.dtype).min
    x[2] = -math.inf
    x[3, V // 2:] = -math.inf
    x[3, 0] = 0.0
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    check(run(qr_gpu, x, 5, t, temperature), x, 5, t, temperature)


@pytest.mark.parametrize("V", [40, 5000, 40003])
def test_ragged_rows_at_small_temperatures(qr_gpu, V):
    """Rows that do not fill their threads' loads, whose missing places count
    as barred: the same."""
    x = near(4, V, F32, 1e-30, 1e-24, seed=V)
    t = tokens(4, V)
    check(run(qr_gpu, x, 5, t, 1e-30), x, 5, t, 1e-30)
