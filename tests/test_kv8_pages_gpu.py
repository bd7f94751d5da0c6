"""GPU: the page operators of the 8-bit KV cache (quantr_kv8_select_dev,
_extend_dev, _compact_dev, _copy_pages_dev) against a sequential restatement:
whole numbers, equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

ERR_PAGES = 11


class State:
    """Tables and pool on the device, and the same in plain Python."""

    def __init__(self, qr, slots, max_pages, n_pages, P=32, L=2, KV=3, hd=16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.qr, self.P = qr, P
        self.k, self.v = (torch.randint(-128, 128, (n_pages, L, KV, P, hd), generator=g, device="cuda",
                                        dtype=torch.int8) for _ in range(2))
        self.ks, self.vs = (torch.rand(n_pages, L, KV, generator=g, device="cuda") for _ in range(2))
        self.pool = qr.Kv8Pool.of(self.k, self.v, self.ks, self.vs)
        self.dev = [self.new_tables(slots, max_pages, n_pages) for _ in range(2)]
        self.table = [[-1] * max_pages for _ in range(slots)]
        self.lens, self.refs = [0] * slots, [0] * n_pages
        self.content = self.snapshot()
        self.ws = torch.zeros(qr.kv8_pages_workspace_bytes(self.pool, self.dev[0][0]), dtype=torch.uint8, device="cuda")

    def new_tables(self, slots, max_pages, n_pages):
        t = (torch.full((slots, max_pages), -1, dtype=torch.int32, device="cuda"),
             torch.zeros(slots, dtype=torch.int32, device="cuda"),
             torch.zeros(n_pages, dtype=torch.int32, device="cuda"))
        return (self.qr.Kv8Tables.of(*t),) + t

    def snapshot(self):
        return [x.cpu().numpy().copy() for x in (self.k, self.v, self.ks, self.vs)]

    def move(self, dst, src):
        for x in self.content:
            x[dst] = x[src]

    # each operator: on the device, then restated
    def select(self, pick):
        f = torch.tensor(pick, dtype=torch.int32, device="cuda")
        self.qr.kv8_select_dev(self.dev[1][0], self.dev[0][0], f.data_ptr(), self.pool)
        torch.cuda.synchronize()
        self.dev.reverse()
        blank = [-1] * len(self.table[0])
        pick = [p if 0 <= p < len(self.table) else -1 for p in pick]
        lens = [self.lens[p] if p >= 0 else 0 for p in pick]
        self.table = [list(self.table[p]) if p >= 0 else list(blank) for p in pick]
        self.lens = lens
        self.refs = [0] * len(self.refs)
        for row in self.table:
            for p in row:
                if p >= 0:
                    self.refs[p] += 1

    def extend(self, n_new=None, slot=None, B=None):
        B = B if B is not None else len(slot if slot is not None else n_new)
        t = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (slot, n_new)]
        grown = torch.full((B,), 7, dtype=torch.int32, device="cuda")
        self.qr.kv8_extend_dev(self.pool, self.dev[0][0], *[x if x is None else x.data_ptr() for x in t], B,
                               self.ws.data_ptr(), self.ws.numel(), grown=grown.data_ptr())
        torch.cuda.synchronize()
        want, P = [], self.P
        free = [p for p, r in enumerate(self.refs) if r == 0]
        moves = []
        out = False  # the pages ran out: for those after it that need one, too
        for b in range(B):
            s, n = b if slot is None else slot[b], 1 if n_new is None else n_new[b]
            if not 0 <= s < len(self.table) or n < 0 or self.lens[s] + n > len(self.table[0]) * P:
                want.append(0)
                continue
            ln = self.lens[s]
            tail = self.table[s][ln // P] if n and ln % P else -1
            copy = tail >= 0 and self.refs[tail] > 1
            more = -(-(ln + n) // P) - -(-ln // P)
            need = more + copy
            if need and (out or need > len(free)):
                out = True
                want.append(0)
                # its turn still passes for those that share its last page
                continue
            if copy:
                page = free.pop(0)
                moves.append((page, tail))
                self.refs[tail] -= 1
                self.refs[page] = 1
                self.table[s][ln // P] = page
            for i in range(more):
                page = free.pop(0)
                self.refs[page] = 1
                self.table[s][-(-ln // P) + i] = page
            self.lens[s] = ln + n
            want.append(1)
        for dst, src in moves:
            self.move(dst, src)
        assert grown.tolist() == want
        return want

    def compact(self, outputs=True):
        N = len(self.refs)
        m = torch.full((N,), 5, dtype=torch.int32, device="cuda")
        live = torch.full((1,), 5, dtype=torch.int32, device="cuda")
        self.qr.kv8_compact_dev(self.pool, self.dev[0][0], m.data_ptr() if outputs else None,
                                live.data_ptr() if outputs else None, self.ws.data_ptr(), self.ws.numel())
        torch.cuda.synchronize()
        n = sum(r > 0 for r in self.refs)
        to = [p if r else -1 for p, r in enumerate(self.refs)]
        holes = [p for p in range(n) if not self.refs[p]]
        for dst, src in zip(holes, [p for p in range(n, N) if self.refs[p]]):
            to[src] = dst
            self.move(dst, src)
            self.refs[dst], self.refs[src] = self.refs[src], 0
        self.table = [[to[p] if p >= 0 else -1 for p in row] for row in self.table]
        if outputs:
            assert live.tolist() == [n] and m.tolist() == to
        assert all(r > 0 for r in self.refs[:n]) and not any(self.refs[n:])

    def same(self):
        _, table, lens, refs = self.dev[0]
        assert table.tolist() == self.table
        assert lens.tolist() == self.lens
        assert refs.tolist() == self.refs
        for x, y in zip(self.snapshot(), self.content):
            assert np.array_equal(x, y)


def test_fork_extend_free(qr_gpu):
    """A prompt, forked; every fork writes into a last page of its own; losers
    are freed."""
    s = State(qr_gpu, 5, 8, 40)
    s.extend([70], slot=[0])
    s.same()
    s.select([0] * 5)
    s.same()
    assert max(s.refs) == 5
    s.extend(B=5)
    s.same()
    assert len({row[2] for row in s.table}) == 5  # 70 tokens: the third page was shared
    s.select([3, -1, 3, -1, 0])
    s.extend([1, 1, 1], slot=[2, 0, 4])  # the pair's order is the batch's
    s.same()
    s.select([-1] * 5)
    s.same()
    assert not any(s.refs)
    assert qr_gpu.device_status() == 0


def test_extend_at_page_ends(qr_gpu):
    """No copy at a page's end, none for a sole owner, several pages at once,
    and nothing for no new tokens."""
    s = State(qr_gpu, 4, 6, 30)
    s.extend([64, 31, 0, 33])
    s.select([0, 1, 0, 1])
    s.extend([1, 1, 1, 1])
    s.same()
    s.extend([100, 0, 3, 64])
    s.same()
    assert qr_gpu.device_status() == 0


def test_extend_runs_out_of_pages(qr_gpu):
    """Who comes too late stays as it was; who needs no page still grows."""
    s = State(qr_gpu, 5, 8, 7)
    assert s.extend([60, 40, 70, 5, 1]) == [1, 1, 1, 0, 0]
    assert qr_gpu.device_status() == ERR_PAGES
    s.same()
    assert s.extend([4, 30, 2, 1, 2]) == [1, 0, 1, 0, 0]
    qr_gpu.device_status()
    s.same()


def test_extend_table_too_short_and_bad_slots(qr_gpu):
    s = State(qr_gpu, 3, 2, 20)
    assert s.extend([65, 64, 1]) == [0, 1, 1]
    assert qr_gpu.device_status() == ERR_PAGES
    s.same()
    assert s.extend([1, 1, -3], slot=[9, 2, 0]) == [0, 1, 0]
    assert qr_gpu.device_status() == ERR_PAGES
    s.same()


def test_select_bad_slots_and_empty(qr_gpu):
    s = State(qr_gpu, 3, 4, 12)
    s.select([-1, -1, -1])
    s.same()
    s.extend([10, 40, 100])
    s.select([2, 7, 1])
    assert qr_gpu.device_status() == ERR_PAGES
    s.same()


def test_select_leaves_its_source(qr_gpu):
    s = State(qr_gpu, 4, 4, 16)
    s.extend([10, 40, 100, 1])
    before = [x.clone() for x in s.dev[0][1:]]
    s.select([1, 1, 1, 1])
    assert all(torch.equal(x, y) for x, y in zip(s.dev[1][1:], before))
    s.same()


@pytest.mark.parametrize("n_pages,slots,max_pages", [(1, 1, 1), (50, 6, 8), (1025, 20, 40), (9000, 60, 100)])
def test_compact(qr_gpu, n_pages, slots, max_pages):
    rng = np.random.default_rng(n_pages)
    s = State(qr_gpu, slots, max_pages, n_pages, L=1, KV=1)
    for _ in range(3):
        s.extend([int(x) for x in rng.integers(0, min(max_pages * 32, n_pages * 32 // slots) // 3 + 1, slots)])
        s.select([int(x) if rng.random() < 0.7 else -1 for x in rng.permutation(slots)])
        s.compact()
        s.same()
    s.compact(outputs=False)  # nothing moves
    s.same()
    qr_gpu.device_status()


@pytest.mark.parametrize("seed", range(4))
def test_random_steps(qr_gpu, seed):
    """Forks, growth, ends and compactions in random order, with pools that run
    out now and then, odd numbers of scales per page."""
    rng = np.random.default_rng(seed)
    s = State(qr_gpu, 9, 7, 45, P=[32, 64, 128, 32][seed], L=1 + seed, KV=[1, 3, 1, 5][seed], hd=[16, 80, 48, 128][seed],
              seed=seed)
    for step in range(25):
        what = rng.integers(0, 10)
        if what < 5:
            n = [int(x) for x in rng.integers(0, s.P + 3, 9)]
            order = [int(x) for x in rng.permutation(9)]
            s.extend(n, slot=order)
        elif what < 8:
            s.select([int(x) for x in rng.integers(-1, 9, 9)])
        else:
            s.compact()
        s.same()
    qr_gpu.device_status()


def test_copy_pages(qr_gpu):
    s = State(qr_gpu, 1, 1, 30, P=64, L=5, KV=1, hd=112)
    dst, src = [3, 9, 29, 0], [4, 4, 1, 28]
    t = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (dst, src)]
    qr_gpu.kv8_copy_pages_dev(s.pool, t[0].data_ptr(), t[1].data_ptr(), 4)
    torch.cuda.synchronize()
    for a, b in zip(dst, src):
        s.move(a, b)
    s.same()
    bad = torch.tensor([2, -1, 30], dtype=torch.int32, device="cuda")
    ok = torch.tensor([1, 5, 6], dtype=torch.int32, device="cuda")
    qr_gpu.kv8_copy_pages_dev(s.pool, bad.data_ptr(), ok.data_ptr(), 3)
    assert qr_gpu.device_status() == ERR_PAGES
    s.move(2, 1)
    s.same()


def test_select_on_another_stream_and_in_a_graph(qr_gpu):
    s = State(qr_gpu, 3, 4, 12)
    s.extend([10, 40, 100])
    want = State(qr_gpu, 3, 4, 12)
    pick = torch.tensor([2, 0, 2], dtype=torch.int32, device="cuda")
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g.capture_begin()
        qr_gpu.kv8_select_dev(s.dev[1][0], s.dev[0][0], pick.data_ptr(), s.pool, stream=st.cuda_stream)
        g.capture_end()
        g.replay()
        g.replay()
    torch.cuda.synchronize()
    got = [x.tolist() for x in s.dev[1][1:]]
    s.select([2, 0, 2])
    assert got == [s.table, s.lens, s.refs]
    del want
