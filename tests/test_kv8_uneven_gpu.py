"""GPU: attention over the 8-bit cache where long sequences lie among short ones,
so that neighbouring row tiles are each shared by more than 32 CTAs, call after
call on one workspace.  Formulas and tolerances are test_kv8_gpu.py's.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_kv8_gpu import BF16, ERR_PAGES, F32, Cache, attend, check, query, want_attend  # noqa: E402

SHAPES = [
    # KV, G, lens: on 296 CTAs the last group of one row tile is one CTA, which
    # is also the first of the next row tile
    (4, 1, [65600, 1000]),
    (4, 1, [131072, 64000]),
    (4, 8, [100000] + [2000] * 21),
    (4, 8, [131072] + [2000] * 29),
    (8, 2, [100000] + [2000] * 5),
    # and others around them
    (2, 4, [70000, 1, 129, 0, 3000]),
    (1, 1, [40000, 150000]),
]


@pytest.mark.parametrize("type_", [F32, BF16])
def test_uneven_long_contexts_on_one_workspace(qr_gpu, type_):
    """Every output is written and right, the counters are zero after every call
    (attend() looks), and the bits stay the same from call to call."""
    ws = torch.zeros(1 << 23, dtype=torch.uint8, device="cuda")
    made = []
    for i, (KV, G, lens) in enumerate(SHAPES):
        c = Cache(qr_gpu, lens, KV, 64, 64, seed=40 + i)
        q = query(len(lens), KV * G, 64, type_, seed=50 + i)
        made.append((c, q, [1] * len(lens)))
    first = []
    for c, q, rows in made:
        got = attend(qr_gpu, c, q, rows, ws=ws)
        check(c, q, got, want_attend(c, q, rows))
        first.append(got)
    for _ in range(20):
        for (c, q, rows), want in zip(made, first):
            got = attend(qr_gpu, c, q, rows, ws=ws)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert qr_gpu.device_status() == 0


@pytest.mark.parametrize("window", [5, 1000, 2 ** 31 - 2, 2 ** 31 - 1])
def test_windows_of_any_size(qr_gpu, window):
    """A window past every length hides nothing, rows before position 0 or not."""
    c = Cache(qr_gpu, [3, 300, 1, 0], 2, 64, 64, seed=8)
    rows = [6, 2, 40, 3]
    q = query(sum(rows), 4, 64, F32)
    check(c, q, attend(qr_gpu, c, q, rows, window=window), want_attend(c, q, rows, window=window))


@pytest.mark.parametrize("length", [-1, -70, -2 ** 31 + 1, -2 ** 31])
def test_lengths_below_zero_are_empty(qr_gpu, length):
    """A length below 0 is an empty sequence to every call, and is reported."""
    c = Cache(qr_gpu, [100, 70], 2, 32, 32, seed=9)
    keys, used = c.k.clone(), c.table[1].clone()
    c.lens[0] = length
    q = query(5, 4, 32, F32)
    out, lse = attend(qr_gpu, c, q, [3, 2])
    assert bool((out[:3] == 0).all()) and bool(torch.isneginf(lse[:3]).all()) and bool(torch.isfinite(lse[3:]).all())
    assert qr_gpu.device_status() == ERR_PAGES
    b = qr_gpu.Kv8Batch(None, None, 2, 3)
    rows = torch.full((2, 6, 2, 32), 7.0, device="cuda")
    qr_gpu.kv8_read_dev(rows[0].data_ptr(), 64, rows[1].data_ptr(), 64, F32, c.pool, c.tables, b, 0)
    torch.cuda.synchronize()
    assert bool((rows[:, :3] == 0).all()) and bool((rows[:, 3:] != 7).all())
    assert qr_gpu.device_status() == ERR_PAGES
    qr_gpu.kv8_append_dev(rows[0].data_ptr(), 64, rows[1].data_ptr(), 64, F32, c.pool, c.tables, b, 0)
    torch.cuda.synchronize()
    others = [p for p in range(c.k.shape[0]) if p not in used.tolist()]
    assert torch.equal(c.k[others], keys[others])
    assert qr_gpu.device_status() == ERR_PAGES
