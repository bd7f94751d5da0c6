"""GPU: what the cache's attention keeps of small weights and small query
elements, for every type of queries, against the 64-bit definition.

Tolerances.  A weight is off by up to 2^-24 of its page's largest and the score
arithmetic by a relative 2^-18 of the weight (ex2 2^-21, scores below 2^5 formed
with four fp32 roundings), so n tokens of |v| <= v_max beside a dominant one
whose value is 0 cost at most v_max (n 2^-24 + 2^-18 sum of their weights).  A
query element is off by half a step, at most 2^-23 of the row's largest: over hd
independent terms 6 sigma = 6 sqrt(hd) step / sqrt(12) rms(k).  The result is
rounded once to its type (half an ulp: 2^-24, 2^-11 or 2^-8 of it)."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_kv8_gpu import BF16, DTYPE, F16, F32, Cache, attend, want_attend  # noqa: E402

HALF_ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("P", [32, 64, 128])
@pytest.mark.parametrize("bits", [8.0, 14.0, 16.5, 17.05, 19.0, 22.0])
def test_weights_beside_a_dominant_token(qr_gpu, type_, P, bits):
    """One token of a page has nearly all of the weight and a value of 0 (an
    attention sink); each of the others has 2^-bits of its weight, and they are
    what the output is made of."""
    c = Cache(qr_gpu, [P], 1, 64, P, seed=P)
    page = int(c.table[0, 0])
    c.k.zero_()
    c.k[page, 0, 0, 9, 0] = 127
    c.ks.fill_(bits * math.log(2) / 127 / 0.125)
    c.v.abs_()
    c.v[page, 0, 0, 9] = 0
    q = torch.zeros(1, 1, 64, device="cuda", dtype=DTYPE[type_])
    q[..., 0] = 1.0
    out, lse = attend(qr_gpu, c, q, [1])
    want, want_lse = want_attend(c, q, [1])
    v_max = 127 * float(c.vs.max())
    tol = v_max * (P - 1) * (2.0 ** -24 + 2.0 ** -18 * 2.0 ** -bits) + HALF_ULP[type_] * want.abs()
    assert float(want.abs().max()) > 0
    assert bool(((out.double() - want).abs() <= tol).all())
    assert float((lse.double() - want_lse).abs().max()) <= (P - 1) * 2.0 ** -24 + 2.0 ** -20


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("large", [8.0, 256.0, 2048.0])
def test_queries_with_one_large_element(qr_gpu, type_, large):
    """The large element meets keys of 0 in its place: the scores are made of the
    small ones."""
    hd, lens = 64, [500]
    c = Cache(qr_gpu, lens, 1, hd, 64, seed=11)
    c.k[..., 5] = 0
    g = torch.Generator(device="cuda")
    g.manual_seed(12)
    q = torch.randn(1, 4, hd, generator=g, device="cuda").to(DTYPE[type_])
    q[..., 5] = large
    out, lse = attend(qr_gpu, c, q, [1])
    want, want_lse = want_attend(c, q, [1])
    k_rms = 32 * float(c.ks.max())
    dx = 6 * hd ** -0.5 * math.sqrt(hd) * large * 2.0 ** -23 / math.sqrt(12) * k_rms
    dx += 2.0 ** -22 * hd ** -0.5 * 6 * math.sqrt(hd) * 4 * k_rms  # scores of elements below 4, formed in fp32
    e = dx + 2.0 ** -20 + c.P * 2.0 ** -24
    v_max = 127 * float(c.vs.max())
    assert float((out.double() - want).abs().max()) <= 2 * e * v_max + HALF_ULP[type_] * float(want.abs().max())
    assert float((lse.double() - want_lse).abs().max()) <= e + 2.0 ** -20
