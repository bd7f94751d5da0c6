"""GPU: the 8-bit paged KV cache (quantr_kv8_append_dev / _read_dev / _attend_dev)
against plain 64-bit restatements of include/quantr_cuda.h's formulas.

Appending and reading are compared bit for bit with an fp32 restatement (every
step has one rounding), and with the bound that doubling scales gives.
Attention's tolerance is derived from what its fixed-point digits keep, below.
"""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = 0, 1, 30
DTYPE = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
ERR_PAGES = 11


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """A pool with codes and scales everywhere, and tables whose pages lie
    anywhere in it."""

    def __init__(self, qr, lens, KV, hd, P, seed=0, layers=1, spare=3, max_pages=None, n_pages=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        need = [-(-n // P) for n in lens]
        n_pages = n_pages or sum(need) + spare
        self.lens_l, self.P, self.KV, self.hd = list(lens), P, KV, hd
        shape = (n_pages, layers, KV, P, hd)
        self.k, self.v = ((torch.randn(shape, generator=g, device="cuda") * 30).round().clamp(-127, 127).to(torch.int8)
                          for _ in range(2))
        self.ks, self.vs = (torch.rand(shape[:3], generator=g, device="cuda") * 0.03 + 0.01 for _ in range(2))
        max_pages = max_pages or max(need + [1]) + 1
        perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max_pages), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        self.refs[perm[:at].long()] = 1
        self.lens = i32(lens)
        self.bind(qr)

    def bind(self, qr):
        self.pool = qr.Kv8Pool.of(self.k, self.v, self.ks, self.vs)
        self.tables = qr.Kv8Tables.of(self.table, self.lens, self.refs)


def batch_of(qr, rows, slots=None):
    """Ragged batch with rows[b] rows each; keeps its tensors alive."""
    start = i32(np.concatenate([[0], np.cumsum(rows)]).tolist())
    slot = None if slots is None else i32(slots)
    b = qr.Kv8Batch(None if slot is None else slot.data_ptr(), start.data_ptr(), len(rows), max(rows + [0]))
    b.keep = (start, slot)
    return b


def attend(qr, c, q, rows, slots=None, window=0, layer=0, scale=None, max_len=None, stream=0, ldq=None, ws=None):
    total, H, hd = q.shape
    b = batch_of(qr, rows, slots)
    type_ = {v: k for k, v in DTYPE.items()}[q.dtype]
    out = torch.full((total, H, hd), 77.0, dtype=q.dtype, device="cuda")
    lse = torch.full((total, H), 77.0, device="cuda")
    n = qr.kv8_attend_workspace_bytes(c.pool, b, H, max_len or max(c.lens_l + [1]))
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda") if ws is None else ws
    torch.cuda.synchronize()
    qr.kv8_attend_dev(out.data_ptr(), H * hd, q.data_ptr(), ldq or q.stride(0), type_, H, c.pool, c.tables, b, layer,
                      hd ** -0.5 if scale is None else scale, max_len or max(c.lens_l + [1]), ws.data_ptr(), ws.numel(),
                      window=window, lse=lse.data_ptr(), stream=stream)
    torch.cuda.synchronize()
    assert int(ws[:4096].view(torch.int32).abs().sum()) == 0  # the counters are zero again
    return out, lse


def want_attend(c, q, rows, slots=None, window=0, layer=0, scale=None):
    """The definition in 64 bits, one row and head at a time."""
    total, H, hd = q.shape
    G = H // c.KV
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(total, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((total, H), -math.inf, dtype=torch.float64, device="cuda")
    table, lens, n_pages = c.table.tolist(), c.lens.tolist(), c.k.shape[0]
    r = 0
    for b, n in enumerate(rows):
        slot = b if slots is None else slots[b]
        ok = 0 <= slot < len(lens)
        ln = lens[slot] if ok else 0
        pages = table[slot][:-(-ln // c.P)] if ok else []
        there = torch.tensor([0 <= p < n_pages for p in pages], device="cuda").repeat_interleave(c.P)[:ln]
        idx = torch.tensor([p if 0 <= p < n_pages else 0 for p in pages], dtype=torch.long, device="cuda")
        for h in range(c.KV):
            if ln > 0:
                k = (c.k[idx, layer, h].double() * c.ks[idx, layer, h].double()[:, None, None]).view(-1, hd)[:ln]
                v = (c.v[idx, layer, h].double() * c.vs[idx, layer, h].double()[:, None, None]).view(-1, hd)[:ln]
            for i in range(n):
                pos = ln - n + i
                t = torch.arange(max(ln, 0), device="cuda")
                seen = (t <= pos) & (t > pos - window if window else t >= 0)
                if ln > 0:
                    seen &= there
                if ln <= 0 or not bool(seen.any()):
                    continue
                x = q[r + i, h * G:(h + 1) * G].double() @ k[seen].T * scale
                lse[r + i, h * G:(h + 1) * G] = torch.logsumexp(x, 1)
                out[r + i, h * G:(h + 1) * G] = torch.softmax(x, 1) @ v[seen]
        r += n
    return out, lse


def tolerances(c, q, scale=None):
    """Absolute bounds of out and lse.

    A query element is off by half a digit step, at most 2^-23 (fp32) or 2^-15
    (16-bit) of the row's largest; over a dot product of hd independent terms
    that is 6 sigma = 6 sqrt(hd) * step/sqrt(12) * rms(k).  Forming the score
    rounds it 4 times.  ex2 is good to 2^-21.  A weight is rounded to 2^-24
    (2^-17) of its page's largest, so P of them cost at most P times that.  A
    relative error e of the weights moves their mean of v by at most 2 e max|v|."""
    hd = q.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    qmax = float(q.float().abs().nan_to_num(0, 0, 0).max())
    k_rms = 32 * float(c.ks.nan_to_num(0).max())
    digit, weight = (2.0 ** -23, 2.0 ** -24) if q.dtype == torch.float32 else (2.0 ** -14, 2.0 ** -17)
    x_max = scale * qmax * math.sqrt(hd) * k_rms * 6
    dx = 6 * scale * math.sqrt(hd) * qmax * digit / math.sqrt(12) * k_rms + x_max * 2.0 ** -22
    e = dx + 2.0 ** -20 + c.P * weight
    v_max = 127 * float(c.vs.nan_to_num(0).max())
    rounding = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[q.dtype]
    return v_max * (2 * e + rounding), dx + 2.0 ** -20 + c.P * 2.0 ** -24 + 40 * 2.0 ** -22


def check(c, q, got, want, scale=None):
    tol_o, tol_l = tolerances(c, q, scale)
    out, lse = got
    w_out, w_lse = want
    empty = torch.isinf(w_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    assert bool((out[empty] == 0).all())
    assert float((out.double() - w_out).abs().max()) <= tol_o
    assert float((lse.double() - w_lse)[~empty].abs().max() if bool((~empty).any()) else 0.0) <= tol_l


def query(total, H, hd, type_, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(total, H, hd, generator=g, device="cuda").to(DTYPE[type_])


# ----------------------------------------------------------------- attend --

CASES = [
    # type, H, KV, hd, P, lens, rows, window
    (F32, 1, 1, 128, 128, [1], [1], 0),
    (F32, 32, 4, 64, 64, [513], [1], 0),
    (F32, 32, 4, 128, 64, [0, 1, 63, 64, 65, 127, 128, 129, 1000], [1] * 9, 0),
    (BF16, 14, 2, 64, 32, [31, 32, 33, 700], [1, 5, 33, 64], 0),
    (F16, 14, 2, 64, 32, [300, 301], [17, 2], 40),
    (F32, 16, 16, 128, 64, [200, 390], [5, 3], 100),
    (BF16, 12, 1, 80, 128, [257, 5], [2, 1], 0),
    (F16, 3, 3, 96, 64, [129, 640], [4, 9], 0),
    (F32, 8, 8, 112, 32, [77], [1], 1),
    (F32, 8, 2, 16, 64, [190, 3], [3, 3], 0),
    (BF16, 24, 2, 48, 64, [555], [7], 333),
    (F16, 40, 2, 128, 128, [2100, 17], [1, 1], 0),
    (F32, 6, 2, 32, 32, [5, 4], [9, 4], 0),  # rows before position 0
    (BF16, 64, 1, 128, 64, [1500] * 3, [1, 2, 3], 0),
]


@pytest.mark.parametrize("type_,H,KV,hd,P,lens,rows,window", CASES)
def test_attend(qr_gpu, type_, H, KV, hd, P, lens, rows, window):
    c = Cache(qr_gpu, lens, KV, hd, P, seed=hd + P)
    q = query(sum(rows), H, hd, type_)
    check(c, q, attend(qr_gpu, c, q, rows, window=window), want_attend(c, q, rows, window=window))
    assert qr_gpu.device_status() == 0


@pytest.mark.parametrize("B,H,KV,n", [(300, 4, 2, 260), (7, 8, 4, 3000), (1, 1, 1, 20000), (140, 2, 2, 700)])
def test_attend_splits(qr_gpu, B, H, KV, n):
    """More row tiles than CTAs, long rows shared by many CTAs, and both with
    ragged lengths: every way of sharing the work out."""
    lens = [1 + (b * 7919 + n // 2) % n for b in range(B)]
    lens[0] = n
    c = Cache(qr_gpu, lens, KV, 64, 64, seed=3)
    q = query(B, H, 64, F32)
    got = attend(qr_gpu, c, q, [1] * B)
    check(c, q, got, want_attend(c, q, [1] * B))
    again = attend(qr_gpu, c, q, [1] * B)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])  # whoever joins, the bits are the same


def test_attend_layers_slots_strides(qr_gpu):
    """A middle layer, slots in another order, queries with gaps that leave
    their rows unaligned."""
    c = Cache(qr_gpu, [100, 40, 300], 2, 64, 32, layers=3)
    big = torch.randn(8, 4 * 64 + 3, device="cuda")
    q = torch.as_strided(big, (6, 4, 64), (big.stride(0), 64, 1), 1)
    slots, rows = [2, 0], [4, 2]
    got = attend(qr_gpu, c, q, rows, slots=slots, layer=1, ldq=big.stride(0))
    check(c, q, got, want_attend(c, q, rows, slots=slots, layer=1))


def test_attend_uniform_rows(qr_gpu):
    """start = NULL: max_rows rows each."""
    c = Cache(qr_gpu, [90, 200], 2, 64, 64)
    q = query(6, 4, 64, F16)
    b = qr_gpu.Kv8Batch(None, None, 2, 3)
    out = torch.empty_like(q)
    ws = torch.zeros(qr_gpu.kv8_attend_workspace_bytes(c.pool, b, 4, 200), dtype=torch.uint8, device="cuda")
    qr_gpu.kv8_attend_dev(out.data_ptr(), 256, q.data_ptr(), 256, F16, 4, c.pool, c.tables, b, 0, 0.125, 200,
                          ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    want, _ = want_attend(c, q, [3, 3])
    assert float((out.double() - want).abs().max()) <= tolerances(c, q)[0]


def test_attend_missing_pages_and_slots(qr_gpu):
    """Pages that are -1 or outside the pool are masked, a slot that does not
    exist is an empty sequence, and both are reported."""
    c = Cache(qr_gpu, [400, 200, 64], 2, 64, 64)
    c.table[0, 2] = -1
    c.table[0, 4] = 10 ** 6
    c.table[2, 0] = -5  # nothing left of this one
    q = query(4, 4, 64, F32)
    rows, slots = [1, 1, 1, 1], [0, 1, 2, 9]
    got = attend(qr_gpu, c, q, rows, slots=slots)
    check(c, q, got, want_attend(c, q, rows, slots=slots))
    assert bool((got[0][2:] == 0).all()) and bool(torch.isneginf(got[1][2:]).all())
    assert qr_gpu.device_status() == ERR_PAGES
    assert qr_gpu.device_status() == 0


def test_attend_nan_stays_where_it_is(qr_gpu):
    """NaN scales of pages that no row sees change nothing; of one that is seen,
    they make that head NaN; a query with an infinity makes its row NaN."""
    c = Cache(qr_gpu, [200, 200], 2, 64, 32, spare=5)
    q = query(2, 4, 64, F32)
    clean = attend(qr_gpu, c, q, [1, 1], window=50)
    used = set(c.table.flatten().tolist())
    for p in set(range(c.k.shape[0])) - used:
        c.ks[p], c.vs[p] = math.nan, math.nan
    outside = c.table[0, 1]  # tokens 32..63: before the window
    c.ks[outside], c.vs[outside] = math.nan, math.nan
    got = attend(qr_gpu, c, q, [1, 1], window=50)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    c.ks[c.table[0, 6], 0, 1] = math.nan
    got = attend(qr_gpu, c, q, [1, 1], window=50)
    assert bool(torch.isnan(got[0][0, 2:]).all()) and bool(torch.isnan(got[1][0, 2:]).all())
    assert torch.equal(got[0][0, :2], clean[0][0, :2]) and torch.equal(got[0][1], clean[0][1])
    q[1, 3, 5] = math.inf
    got = attend(qr_gpu, c, q, [1, 1], window=50)
    assert bool(torch.isnan(got[0][1, 3]).all()) and torch.equal(got[0][1, :3], clean[0][1, :3])


def test_attend_stale_codes_behind_the_end(qr_gpu):
    """What lies in a page behind the sequence's end is not seen."""
    c = Cache(qr_gpu, [70], 1, 64, 64)
    q = query(1, 2, 64, BF16)
    clean = attend(qr_gpu, c, q, [1])
    c.k[c.table[0, 1].long(), 0, 0, 6:] = 127
    c.v[c.table[0, 1].long(), 0, 0, 6:] = -127
    got = attend(qr_gpu, c, q, [1])
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("gap", [10.0, 17.0, 60.0])
def test_attend_one_token_above_all(qr_gpu, gap):
    """One token's score lies `gap` above 4095 equal ones: the small weights
    keep their share, whichever page the large one is in."""
    c = Cache(qr_gpu, [4096], 1, 64, 64)
    c.k.zero_()
    c.ks.fill_(gap / 127 / 0.125)
    c.k[c.table[0, 5].long(), 0, 0, 9, 0] = 127
    q = torch.zeros(1, 1, 64, device="cuda")
    q[..., 0] = 1.0
    check(c, q, attend(qr_gpu, c, q, [1]), want_attend(c, q, [1]))


def test_attend_zero_and_tiny_queries(qr_gpu):
    c = Cache(qr_gpu, [130], 1, 64, 64)
    for x in (0.0, 1e-38, 1e-20):
        q = torch.full((1, 2, 64), x, device="cuda")
        check(c, q, attend(qr_gpu, c, q, [1]), want_attend(c, q, [1]))


def test_attend_wide_scales(qr_gpu):
    """Neighbouring pages whose scales of v differ by 2^30."""
    c = Cache(qr_gpu, [256], 1, 64, 32)
    c.vs[c.table[0, ::2].long()] *= 2.0 ** -30
    q = query(1, 2, 64, F32)
    out, _ = attend(qr_gpu, c, q, [1])
    want, _ = want_attend(c, q, [1])
    assert float((out.double() - want).abs().max()) <= tolerances(c, q)[0]


def test_attend_offsets_past_32_bits(qr_gpu):
    """Pages at the end of a pool of more than 4 GB."""
    KV, P, hd, n_pages = 8, 128, 128, 36000  # 4.7 GB of keys
    c = Cache(qr_gpu, [300], KV, hd, P, n_pages=4, max_pages=4)
    k, v = (torch.zeros(n_pages, 1, KV, P, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(n_pages, 1, KV, device="cuda") * 0.02 for _ in range(2))
    pages = [n_pages - 1, 17, n_pages - 3]
    for i, p in enumerate(pages):
        old = int(c.table[0, i])
        k[p], v[p], ks[p], vs[p] = c.k[old], c.v[old], c.ks[old], c.vs[old]
    small = want_attend(c, query(1, 8, hd, F32), [1])
    c.k, c.v, c.ks, c.vs = k, v, ks, vs
    c.table[0, :3] = i32(pages)
    c.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    c.bind(qr_gpu)
    q = query(1, 8, hd, F32)
    check(c, q, attend(qr_gpu, c, q, [1]), small)
    # Appending there, and reading it back.
    c.lens.fill_(301)
    new = torch.randn(1, KV, hd, device="cuda")
    b = batch_of(qr_gpu, [1])
    qr_gpu.kv8_append_dev(new.data_ptr(), KV * hd, new.data_ptr(), KV * hd, F32, c.pool, c.tables, b, 0)
    back = torch.empty(2, 1, KV, hd, device="cuda")
    qr_gpu.kv8_read_dev(back[0].data_ptr(), KV * hd, back[1].data_ptr(), KV * hd, F32, c.pool, c.tables, b, 0)
    torch.cuda.synchronize()
    step = ks[pages[2], 0, :, None]
    assert bool(((back - new).abs() <= step * 1.001).all())


def test_attend_streams_and_graphs(qr_gpu):
    """Another stream than the default one, and a captured call replayed."""
    c = Cache(qr_gpu, [2000, 100], 2, 64, 64)
    q = query(2, 8, 64, F32)
    want = attend(qr_gpu, c, q, [1, 1])
    s = torch.cuda.Stream()
    got = attend(qr_gpu, c, q, [1, 1], stream=s.cuda_stream)
    assert torch.equal(got[0], want[0])
    b = batch_of(qr_gpu, [1, 1])
    out = torch.zeros_like(q)
    ws = torch.zeros(qr_gpu.kv8_attend_workspace_bytes(c.pool, b, 8, 2000), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        for _ in range(3):
            qr_gpu.kv8_attend_dev(out.data_ptr(), 512, q.data_ptr(), 512, F32, 8, c.pool, c.tables, b, 0, 0.125, 2000,
                                  ws.data_ptr(), ws.numel(), stream=s.cuda_stream)
        g.capture_end()
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])


# ----------------------------------------------------------- append, read --

def append_restated(codes, scales, table, lens, rows, new, P):
    """Page by page in fp32, as the header says (numpy arrays, changed in
    place).  codes (pages, KV, P, hd), scales (pages, KV)."""
    f = np.float32
    r = 0
    for b, n in enumerate(rows):
        first = lens[b] - n
        for at in range(max(first, 0) // P, -(-lens[b] // P) if lens[b] > 0 else 0):
            lo, hi = max(at * P, first, 0), min(at * P + P, lens[b])
            page, had = table[b][at], lo - at * P
            x = new[r + lo - first:r + hi - first].transpose(1, 0, 2)  # KV, rows, hd
            for h in range(x.shape[0]):
                top = np.abs(x[h]).max()
                if not np.isfinite(x[h]).all() or (had and not np.isfinite(scales[page, h])):
                    scales[page, h] = np.nan
                    codes[page, h, had:had + hi - lo] = 0
                    continue
                if not had:
                    s = max(f(top) / f(127), f(2.0 ** -126))
                else:
                    s, j = scales[page, h], 0
                    room = f(s * f(127))
                    while top > room * f(2) ** j:
                        j += 1
                    s = f(s * f(2) ** j)
                    if j:
                        codes[page, h, :had] = np.rint(codes[page, h, :had].astype(f) * f(2.0 ** -j))
                inv = f(1) / f(s)
                codes[page, h, had:had + hi - lo] = np.clip(np.rint(x[h] * inv), -127, 127)
                scales[page, h] = s
        r += n


def do_append(qr, c, k, v, rows, layer=0, slots=None):
    type_ = {x: y for y, x in DTYPE.items()}[k.dtype]
    b = batch_of(qr, rows, slots)
    qr.kv8_append_dev(k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), type_, c.pool, c.tables, b, layer)
    torch.cuda.synchronize()


@pytest.mark.parametrize("type_,KV,hd,P,lens,rows", [
    (F32, 1, 128, 128, [1], [1]),
    (F32, 4, 128, 64, [640, 65, 64, 1, 100], [1, 1, 1, 1, 1]),
    (BF16, 4, 128, 64, [300, 129, 64], [300, 40, 64]),
    (F16, 2, 80, 32, [97, 33, 5], [70, 33, 2]),
    (F32, 3, 16, 128, [400, 130], [399, 5]),
    (F32, 2, 112, 128, [128, 1], [7, 1]),
    (BF16, 1, 48, 32, [7, 3], [7, 9]),  # rows before position 0
])
def test_append_bit_exact(qr_gpu, type_, KV, hd, P, lens, rows):
    c = Cache(qr_gpu, lens, KV, hd, P, seed=5)
    c.ks *= 0.05
    c.vs *= 0.4  # some pages' scales grow, some do not
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    k, v = ((torch.randn(sum(rows), KV, hd, generator=g, device="cuda") * 2).to(DTYPE[type_]) for _ in range(2))
    want = []
    for codes, scales, new in ((c.k, c.ks, k), (c.v, c.vs, v)):
        w = codes[:, 0].cpu().numpy().copy(), scales[:, 0].cpu().numpy().copy()
        append_restated(*w, c.table.tolist(), lens, rows, new.float().cpu().numpy(), P)
        want.append(w)
    do_append(qr_gpu, c, k, v, rows)
    assert qr_gpu.device_status() == 0
    for codes, scales, w in ((c.k, c.ks, want[0]), (c.v, c.vs, want[1])):
        assert np.array_equal(scales[:, 0].cpu().numpy().view(np.uint32), w[1].view(np.uint32))
        assert np.array_equal(codes[:, 0].cpu().numpy(), w[0])


@pytest.mark.parametrize("P", [32, 128])
@pytest.mark.parametrize("growth", [1.0, 1.1, 3.0])
def test_append_one_by_one_stays_within_a_step(qr_gpu, P, growth):
    """Rows of growing size, one at a time: no value is further than one step of
    its page's final scale from what was written."""
    KV, hd, n = 2, 32, P + 5
    c = Cache(qr_gpu, [n], KV, hd, P)
    x = torch.randn(n, KV, hd, device="cuda") * (growth ** torch.arange(n, device="cuda"))[:, None, None].clamp(max=1e30)
    for i in range(n):
        c.lens.fill_(i + 1)
        do_append(qr_gpu, c, x[i:i + 1], -x[i:i + 1], [1])
    back = torch.empty(2, n, KV, hd, device="cuda")
    b = batch_of(qr_gpu, [n])
    qr_gpu.kv8_read_dev(back[0].data_ptr(), KV * hd, back[1].data_ptr(), KV * hd, F32, c.pool, c.tables, b, 0)
    torch.cuda.synchronize()
    page = c.table[0, torch.arange(n, device="cuda") // P].long()
    for got, want, scales in ((back[0], x, c.ks), (back[1], -x, c.vs)):
        step = scales[page, 0][..., None]
        assert bool(((got - want).abs() <= step * 1.0001).all())
        # Doubling leaves at least half of the codes' range in use.
        top = torch.stack([want[i * P:(i + 1) * P].abs().amax((0, 2)) for i in range(2)])
        assert bool((top / scales[c.table[0, :2].long(), 0] >= 127 / 2 * 0.999).all())


def test_append_not_finite(qr_gpu):
    """A page with an infinity or NaN among its rows has a NaN scale in that
    head, until it is begun anew; others do not notice."""
    c = Cache(qr_gpu, [10], 2, 32, 32)
    x = torch.randn(10, 2, 32, device="cuda")
    x[4, 1, 7] = math.inf
    do_append(qr_gpu, c, x, torch.nan_to_num(x), [10])
    page = c.table[0, 0].long()
    assert bool(torch.isnan(c.ks[page, 0, 1])) and bool(torch.isfinite(c.ks[page, 0, 0]))
    assert bool(torch.isfinite(c.vs[page]).all())
    assert bool((c.k[page, 0, 1, :10] == 0).all())
    c.lens.fill_(11)
    do_append(qr_gpu, c, torch.ones(1, 2, 32, device="cuda"), torch.ones(1, 2, 32, device="cuda"), [1])
    assert bool(torch.isnan(c.ks[page, 0, 1]))
    c.lens.fill_(10)
    do_append(qr_gpu, c, torch.ones(10, 2, 32, device="cuda"), torch.ones(10, 2, 32, device="cuda"), [10])
    assert bool(torch.isfinite(c.ks[page]).all())


def test_append_zeros_and_denormals(qr_gpu):
    c = Cache(qr_gpu, [32, 32], 1, 32, 32)
    x = torch.zeros(64, 1, 32, device="cuda")
    x[32:] = 1e-44
    do_append(qr_gpu, c, x, x, [32, 32])
    back = torch.full((64, 1, 32), 5.0, device="cuda")
    b = batch_of(qr_gpu, [32, 32])
    qr_gpu.kv8_read_dev(back.data_ptr(), 32, back.data_ptr(), 32, F32, c.pool, c.tables, b, 0)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(c.ks[c.table[:, 0].long()]).all()) and bool((c.ks[c.table[:, 0].long()] > 0).all())
    assert float(back.abs().max()) <= 2.0 ** -126


def test_append_missing_page_is_skipped(qr_gpu):
    c = Cache(qr_gpu, [70, 70], 1, 32, 32)
    c.table[0, 1] = -1
    before = c.k.clone()
    x = torch.randn(140, 1, 32, device="cuda")
    do_append(qr_gpu, c, x, x, [70, 70])
    assert qr_gpu.device_status() == ERR_PAGES
    mine = set(c.table[0, [0, 2]].tolist()) | set(c.table[1, :3].tolist())
    for p in set(range(c.k.shape[0])) - mine:
        assert torch.equal(c.k[p], before[p])
    assert not torch.equal(c.k[c.table[0, 2].long()], before[c.table[0, 2].long()])


@pytest.mark.parametrize("type_", [F32, F16, BF16])
def test_read_types_strides_and_rows_before_the_start(qr_gpu, type_):
    c = Cache(qr_gpu, [5, 100], 3, 48, 32, layers=2)
    rows, ld = [8, 90], 3 * 48 + 5
    buf = torch.full((2, 98 * ld + 1), 9.0, dtype=DTYPE[type_], device="cuda")
    b = batch_of(qr_gpu, rows)
    es = buf.element_size()
    qr_gpu.kv8_read_dev(buf[0].data_ptr() + es, ld, buf[1].data_ptr() + es, ld, type_, c.pool, c.tables, b, 1)
    torch.cuda.synchronize()
    for got, codes, scales in ((buf[0], c.k, c.ks), (buf[1], c.v, c.vs)):
        got = got[1:].view(98, ld)
        assert bool((got[:, 144:] == 9.0).all())
        want = torch.zeros(98, 3, 48, device="cuda")
        for r, (s, pos) in enumerate([(0, i - 3) for i in range(8)] + [(1, 10 + i) for i in range(90)]):
            if pos >= 0:
                p = c.table[s, pos // 32].long()
                want[r] = codes[p, 1, :, pos % 32].float() * scales[p, 1][:, None]
        assert torch.equal(got[:, :144].reshape(98, 3, 48), want.to(DTYPE[type_]))


def test_append_strided_rows(qr_gpu):
    """Rows that are unaligned slices of a wider array (a fused QKV output)."""
    c = Cache(qr_gpu, [40], 2, 32, 32)
    wide = torch.randn(40, 201, device="cuda")
    k, v = (torch.as_strided(wide, (40, 2, 32), (201, 32, 1), off) for off in (65, 129))
    w = [(x[:, 0].cpu().numpy().copy(), y[:, 0].cpu().numpy().copy()) for x, y in ((c.k, c.ks), (c.v, c.vs))]
    for (codes, scales), new in zip(w, (k, v)):
        append_restated(codes, scales, c.table.tolist(), [40], [40], new.cpu().numpy(), 32)
    do_append(qr_gpu, c, k, v, [40])
    assert np.array_equal(c.k[:, 0].cpu().numpy(), w[0][0]) and np.array_equal(c.v[:, 0].cpu().numpy(), w[1][0])


def test_empty_batches_do_nothing(qr_gpu):
    c = Cache(qr_gpu, [40], 2, 32, 32)
    before = c.k.clone()
    b = qr_gpu.Kv8Batch(None, None, 0, 4)
    n = ctypes.c_void_p(256)
    qr_gpu.kv8_append_dev(None, 0, None, 0, F32, c.pool, c.tables, b, 0)
    qr_gpu.kv8_read_dev(None, 0, None, 0, F32, c.pool, c.tables, b, 0)
    qr_gpu.kv8_attend_dev(None, 0, None, 0, F32, 2, c.pool, c.tables, b, 0, 1.0, 40, n, 0)
    torch.cuda.synchronize()
    assert torch.equal(c.k, before)
