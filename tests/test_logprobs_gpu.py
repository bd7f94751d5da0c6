"""GPU: quantr_logprobs_dev against 64-bit sums and a stable sort.

Tolerances: y = x/temperature is formed with one rounding, weights 2^d are good
to 2^-21 plus the rounding of d (|d| <= 200 counts only while the weight does,
|d| < 40), sums to a few ulp.  So lse and log probabilities are within
2^-21 + 4 ulp of the largest |y|, and the entropy, a quotient of two such sums,
within (1 + entropy) 2^-17."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = 0, 1, 30
DTYPE = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}


def run(qr, x, k, token=None, temperature=1.0, vocab=None, stream=0):
    rows, V = x.shape[0], vocab or x.shape[1]
    type_ = {v: t for t, v in DTYPE.items()}[x.dtype]
    f = lambda *s: torch.full(s, 77.0, device="cuda")  # noqa: E731
    o = {"logprob": f(rows), "entropy": f(rows), "lse": f(rows), "top": f(rows, k),
         "ids": torch.full((rows, k), 77, dtype=torch.int32, device="cuda")}
    token = torch.zeros(rows, dtype=torch.int32, device="cuda") if token is None else token
    torch.cuda.synchronize()
    qr.logprobs_dev(x.data_ptr(), x.stride(0), type_, rows, V, token.data_ptr(), o["logprob"].data_ptr(),
                    o["entropy"].data_ptr(), k, o["ids"].data_ptr(), o["top"].data_ptr(), None, 0,
                    temperature=temperature, lse=o["lse"].data_ptr(), stream=stream)
    torch.cuda.synchronize()
    assert qr.device_status() == 0
    return o


def check(o, x, k, token, temperature=1.0):
    raw = x.double().cpu()
    y = raw / float(np.float32(temperature))
    V = y.shape[1]
    lse = torch.logsumexp(y, 1)
    p = torch.softmax(y, 1)
    ent = -(p * torch.where(p > 0, y - lse[:, None], 0.0)).sum(1)
    none = torch.isneginf(lse)
    ent[none] = 0.0
    big = y.abs().nan_to_num(0, 0, 0).amax(1)
    tol = 2.0 ** -21 + 4 * 2.0 ** -23 * big
    got = {n: v.double().cpu() for n, v in o.items()}
    assert torch.equal(torch.isneginf(got["lse"]), none)
    assert bool(((got["lse"] - lse).abs() <= tol)[~none].all())
    assert bool(((got["entropy"] - ent).abs() <= (1 + ent) * 2.0 ** -17).all())
    token = token.cpu().long()
    has = (token >= 0) & (token < V)
    lp = torch.where(has, y[torch.arange(len(y)), token.clamp(0, V - 1)] - lse, 0.0)
    lp[none & has] = -math.inf
    low = torch.isneginf(lp)
    assert torch.equal(torch.isneginf(got["logprob"]), low)
    assert bool(((got["logprob"] - lp).abs() <= 2 * tol)[has & ~low].all())
    assert bool((got["logprob"][token == -1] == 0).all())
    assert bool(torch.isnan(got["logprob"][~has & (token != -1)]).all())
    # Alternatives: by value, then by id.
    order = np.lexsort((np.arange(V)[None].repeat(len(y), 0), -raw.numpy()), axis=1)[:, :k]
    ids = o["ids"].cpu().numpy()
    for r in range(len(y)):
        w = [int(i) for i in order[r] if raw[r, i] > -math.inf]
        w += [-1] * (k - len(w))
        assert ids[r].tolist() == w, r
        for i, t in zip(w, got["top"][r].tolist()):
            assert t == -math.inf if i < 0 else abs(t - float(y[r, i] - lse[r])) <= 2 * float(tol[r])


def logits(rows, V, type_, seed=0, ld=None, sigma=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = (torch.randn(rows, ld or V, generator=g, device="cuda") * sigma).to(DTYPE[type_])
    return x[:, :V]


def tokens(rows, V, seed=0):
    t = torch.from_numpy(np.random.default_rng(seed).integers(0, V, rows).astype(np.int32))
    if rows > 2:
        t[1], t[2] = -1, V + 3
    return t.cuda()


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V,ld,k", [
    (1, 1, 1, 1), (1, 2, 2, 5), (3, 7, 7, 7), (2, 33, 40, 64), (4, 255, 255, 3), (3, 500, 501, 64), (5, 1000, 1003, 20),
    (2, 1800, 1800, 64), (3, 4096, 4097, 8), (2, 8191, 8191, 32), (1, 32000, 32000, 5), (40, 12345, 12350, 2),
    (300, 2049, 2051, 4), (1, 151936, 151936, 20), (700, 300, 300, 1), (2, 700001, 700001, 11),
])
def test_logprobs(qr_gpu, type_, rows, V, ld, k):
    x = logits(rows, V, type_, seed=V, ld=ld)
    t = tokens(rows, V)
    check(run(qr_gpu, x, k, t), x, k, t)


@pytest.mark.parametrize("temperature", [0.01, 0.7, 2.0, 1000.0, 1e30])
@pytest.mark.parametrize("type_", [F32, F16])
def test_temperature(qr_gpu, type_, temperature):
    x = logits(5, 5000, type_)
    x[:, 100:200] = -math.inf
    t = tokens(5, 5000)
    check(run(qr_gpu, x, 9, t, temperature), x, 9, t, temperature)


@pytest.mark.parametrize("type_", [F32, F16, BF16])
def test_ties_go_to_the_lower_id(qr_gpu, type_):
    """Few different values, so that hundreds tie at the threshold, in short and
    in split rows; and rows of one value."""
    for V in (600, 5001, 33000):
        x = (logits(4, V, type_, seed=V) / 3).round().clamp(-2, 2)
        x[3] = 1.5
        x[2, ::2] = -0.0
        x[2, 1::2] = 0.0  # equal
        t = tokens(4, V)
        check(run(qr_gpu, x, 64, t), x, 64, t)


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("V", [1000, 40000])
def test_masked_tokens(qr_gpu, type_, V):
    """Bans by -inf and by the type's lowest value; all but a few banned; all."""
    lowest = torch.finfo(DTYPE[type_]).min
    x = logits(8, V, type_)
    x[0, 1:] = -math.inf
    x[1, 10:] = lowest
    x[2, :] = -math.inf
    x[3, :] = lowest
    x[4, ::2] = -math.inf
    x[5, : V - 3] = -math.inf
    x[6, 5:] = lowest
    x[6, 0] = -math.inf
    t = torch.tensor([0, 5, 1, 2, 0, V - 1, 1, 3], dtype=torch.int32, device="cuda")
    if type_ != F16:
        # The lowest values' sums do not fit an fp32 lse to an ulp: only their
        # alternatives and their weights' shape are looked at.
        o = run(qr_gpu, x[3:4], 5, t[3:4])
        assert o["ids"].tolist() == [[0, 1, 2, 3, 4]]
        assert abs(float(o["entropy"][0]) - math.log(V)) < 1e-3
        assert float(o["lse"][0]) == lowest
        keep = [0, 1, 2, 4, 5, 6, 7]
        x, t = x[keep], t[keep]
    check(run(qr_gpu, x, 20, t), x, 20, t)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_not_finite(qr_gpu, bad):
    """NaN or +inf makes its row NaN; the others, and its own alternatives'
    order, stay."""
    x = logits(3, 9000, F32)
    clean = run(qr_gpu, x, 6, tokens(3, 9000))
    x[1, 4321] = bad
    o = run(qr_gpu, x, 6, tokens(3, 9000))
    for n in ("lse", "entropy"):
        assert bool(torch.isnan(o[n][1]))
        assert torch.equal(o[n][[0, 2]], clean[n][[0, 2]])
    assert bool(torch.isnan(o["top"][1]).all())
    want = clean["ids"][1].tolist()
    assert o["ids"][1].tolist() == (want if math.isnan(bad) else [4321] + want[:5])


def test_sorted_rows(qr_gpu):
    """Rows that rise, fall, or hold their largest values in one thread's
    places, where a threshold from samples is far off."""
    V = 50000
    up = torch.linspace(-30, 0, V, device="cuda")
    x = torch.stack([up, up.flip(0), up.clone(), torch.zeros(V, device="cuda")])
    x[2, 4::1024] += 100
    x[3, 0:40000:4] = torch.rand(10000, device="cuda")
    t = tokens(4, V)
    check(run(qr_gpu, x, 64, t), x, 64, t)


def test_optional_outputs_and_streams(qr_gpu):
    x = logits(4, 3000, F32)
    want = run(qr_gpu, x, 3)
    s = torch.cuda.Stream()
    got = run(qr_gpu, x, 3, stream=s.cuda_stream)
    assert all(torch.equal(got[n], want[n]) for n in want)
    ids = torch.empty(4, 3, dtype=torch.int32, device="cuda")
    qr_gpu.logprobs_dev(x.data_ptr(), 3000, F32, 4, 3000, None, None, None, 3, ids.data_ptr(), None, None, 0)
    lse = torch.empty(4, device="cuda")
    qr_gpu.logprobs_dev(x.data_ptr(), 3000, F32, 4, 3000, None, None, None, 0, None, None, None, 0, lse=lse.data_ptr())
    qr_gpu.logprobs_dev(x.data_ptr(), 3000, F32, 0, 3000, None, None, None, 0, None, None, None, 0, lse=lse.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(ids, want["ids"]) and torch.equal(lse, want["lse"])


def test_rows_past_32_bits(qr_gpu):
    """Logits whose offsets pass 2^32 bytes and 2^31 elements."""
    rows, V = 15000, 151936
    x = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda")
    x[-2:] = logits(2, V, BF16)
    t = tokens(2, V)
    o = {n: torch.empty(rows, device="cuda") for n in ("logprob", "entropy", "lse")}
    full = torch.zeros(rows, dtype=torch.int32, device="cuda")
    full[-2:] = t
    ids = torch.empty(rows, 3, dtype=torch.int32, device="cuda")
    top = torch.empty(rows, 3, device="cuda")
    x[:-2] = 0
    qr_gpu.logprobs_dev(x.data_ptr(), V, BF16, rows, V, full.data_ptr(), o["logprob"].data_ptr(),
                        o["entropy"].data_ptr(), 3, ids.data_ptr(), top.data_ptr(), None, 0, lse=o["lse"].data_ptr())
    torch.cuda.synchronize()
    o = {n: v[-2:] for n, v in o.items()}
    check({**o, "ids": ids[-2:], "top": top[-2:]}, x[-2:], 3, t)
