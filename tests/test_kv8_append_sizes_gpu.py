"""GPU: appending any number of rows to a page, at every head dim, page size and
element type, bit for bit against include/quantr_cuda.h's formulas in fp32."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_kv8_gpu import BF16, DTYPE, F16, F32, Cache  # noqa: E402


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("P", [32, 64, 128])
@pytest.mark.parametrize("hd", range(16, 129, 16))
def test_append_every_row_count(qr_gpu, type_, P, hd):
    """1 to P rows begin a page: its scale, every element's code, and nothing
    behind them."""
    KV = 2
    c = Cache(qr_gpu, [P], KV, hd, P, seed=hd)
    page = int(c.table[0, 0])
    g = torch.Generator(device="cuda")
    g.manual_seed(P + hd)
    x = torch.randn(2, P, KV, hd, generator=g, device="cuda").to(DTYPE[type_])
    # The last row holds the largest magnitudes, so that the scale shows if any
    # of it is left out.
    grow = 1.0 + torch.arange(P, device="cuda")[None, :, None, None] / 4
    x = (x.float() * grow).to(DTYPE[type_])
    wrong = []
    for rows in range(1, P + 1):
        c.lens.fill_(rows)
        c.k.fill_(99), c.v.fill_(99)
        b = qr_gpu.Kv8Batch(None, None, 1, rows)
        qr_gpu.kv8_append_dev(x[0].data_ptr(), KV * hd, x[1].data_ptr(), KV * hd, type_, c.pool, c.tables, b, 0)
        for new, codes, scales in ((x[0], c.k, c.ks), (x[1], c.v, c.vs)):
            f = new[:rows].float()
            # (Tensor by tensor: a division by a Python number is a product here.)
            top = f.abs().amax((0, 2))
            s = (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126)
            inv = torch.ones_like(s) / s
            want = torch.full((KV, P, hd), 99, dtype=torch.int8, device="cuda")
            want[:, :rows] = (f * inv[:, None]).round().clamp(-127, 127).to(torch.int8).transpose(0, 1)
            if not (torch.equal(scales[page, 0], s) and torch.equal(codes[page, 0], want)):
                wrong.append(rows)
                break
    assert wrong == []
    assert qr_gpu.device_status() == 0
