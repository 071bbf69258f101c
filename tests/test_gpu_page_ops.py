"""Page operations on the device against the page-by-page oracle
(oracle/page_pool.py): tables, reference counts and every layer's contents
are equal, bit for bit; a refused call changes nothing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.page_pool import Pool, Refused

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda_device):
    from pagelora_b200 import kernels

    return kernels


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64).reshape(-1), dtype=torch.int32, device="cuda")


class Pair:
    """The same pool on the device and in the oracle."""

    def __init__(self, seed, *, rows=7, pages=60, cap=9, ps=16, layers=3, token=(2, 64), dtype=torch.bfloat16, lens=()):
        self.rng = np.random.default_rng(seed)
        shape = (layers, pages, 2, ps) + token
        raw = torch.as_tensor(self.rng.integers(0, 256, size=shape + (torch.empty(0, dtype=dtype).element_size(),),
                                                dtype=np.uint8))
        self.pool = raw.cuda().view(dtype).view(shape)
        self.refcount = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.table = torch.full((rows, cap), -7, dtype=torch.int32, device="cuda")
        self.num = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.last = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        perm = self.rng.permutation(pages)
        at, rows_h, last_h, count = 0, [], [], np.zeros(pages, np.int64)
        for r in range(rows):
            n = lens[r] if r < len(lens) else 0
            k = -(-n // ps)
            pg = [int(p) for p in perm[at:at + k]]
            at += k
            rows_h.append(pg)
            last_h.append(n - (k - 1) * ps if k else 0)
            count[pg] = 1
            if k:
                self.table[r, :k] = _i32(pg)
        self.num.copy_(_i32([len(x) for x in rows_h]))
        self.last.copy_(_i32(last_h))
        self.refcount.copy_(_i32(count))
        self.ref = Pool(self.bytes(), count.tolist(), rows_h, last_h, cap)
        self.tables = (self.refcount, self.table, self.num, self.last)

    def bytes(self):
        p = self.pool
        return p.reshape(p.shape[:4] + (-1,)).contiguous().view(torch.uint8).cpu().numpy().copy()

    def check(self, status=0):
        torch.cuda.synchronize()
        assert int(self.status.item()) == status
        self.status.zero_()
        assert self.refcount.tolist() == self.ref.refcount
        assert self.num.tolist() == [len(r) for r in self.ref.rows]
        assert self.last.tolist() == self.ref.last
        for r, row in enumerate(self.ref.rows):
            assert self.table[r, : len(row)].tolist() == row, r
        assert (self.bytes() == self.ref.data).all()

    def reserve(self, K, counts, want=0, **kw):
        total = int(sum(counts))
        sp, so, pos = (torch.full((total,), -1, dtype=torch.int32, device="cuda") for _ in range(3))
        rows, cap = self.table.shape
        indptr, indices = _i32([0] * (rows + 1)), _i32([0] * (rows * cap))
        before = [self.ref.length(r) for r in range(rows)]
        K.page_reserve(*self.tables, _i32(np.cumsum([0] + list(counts))), self.ref.ps, slot_page=sp, slot_offset=so,
                       positions=pos, out_indptr=indptr, out_indices=indices, status=self.status, **kw)
        try:
            slots = self.ref.reserve(counts)
        except Refused:
            slots = None
        self.check(want)
        if slots is None:
            return
        assert list(zip(sp.tolist(), so.tolist())) == slots
        assert pos.tolist() == [b + i for b, n in zip(before, counts) for i in range(n)]
        flat = sum(self.ref.rows, [])
        assert indptr.tolist() == np.cumsum([0] + [len(r) for r in self.ref.rows]).tolist()
        assert indices[: len(flat)].tolist() == flat

    def write(self, slots_seed):
        """New contents in every used slot that one row alone holds (as a decode step would append)."""

        noise = np.random.default_rng(slots_seed)
        flat = self.pool.reshape(self.pool.shape[:4] + (-1,)).view(torch.uint8)
        for row, last in zip(self.ref.rows, self.ref.last):
            if row and self.ref.refcount[row[-1]] == 1:
                x = noise.integers(0, 256, size=(flat.shape[0], 2, flat.shape[4]), dtype=np.uint8)
                self.ref.data[:, row[-1], :, last - 1] = x
                flat[:, row[-1], :, last - 1] = torch.as_tensor(x).cuda()

    def fork(self, K, src, dst, want=0):
        K.page_fork(self.pool, *self.tables, _i32(src), _i32(dst), status=self.status)
        try:
            self.ref.fork(src, dst)
        except Refused:
            pass
        self.check(want)

    def release(self, K, rows, want=0):
        K.page_release(*self.tables, _i32(rows), status=self.status)
        self.ref.release(rows)
        self.check(want)

    def compact(self, K, keep_from, keep, want=0):
        width = max([len(k) for k in keep] + [1])
        m = np.full((len(keep), width + 2), -1)
        for r, k in enumerate(keep):
            m[r, : len(k)] = k
        kt = torch.tensor(m, dtype=torch.int32, device="cuda")[:, :width]
        K.cache_compact(self.pool, *self.tables, _i32(keep_from), kt, _i32([len(k) for k in keep]), status=self.status)
        try:
            self.ref.compact(keep_from, keep)
        except Refused:
            pass
        self.check(want)


KINDS = [dict(), dict(ps=32, token=(1, 64), cap=6), dict(ps=5, token=(3, 8), cap=25), dict(dtype=torch.float32),
         dict(dtype=torch.float8_e4m3fn, token=(2, 16)), dict(ps=128, pages=25, cap=4), dict(ps=1, pages=300, cap=100)]


@pytest.mark.parametrize("kind", range(len(KINDS)))
@pytest.mark.parametrize("seed", range(3))
def test_sequences(K, kind, seed):
    """Random steps of a branching decode; the state is compared after each."""

    s = Pair(seed, lens=[20, 1, 0, 33, 16], **KINDS[kind])
    rng, ref = s.rng, s.ref
    for step in range(14):
        rows = len(ref.rows)
        kind_ = rng.integers(0, 4)
        if kind_ == 0:
            room = sum(-(-(ref.length(r) + 5) // ref.ps) for r in range(rows)) < len(ref.refcount) // 2
            if room and max(ref.length(r) + 5 for r in range(rows)) <= ref.cap * ref.ps:
                s.reserve(K, [int(x) for x in rng.integers(0, 6, rows) * (rng.random(rows) < 0.7)])
            else:
                s.release(K, [int(rng.integers(rows))])
        elif kind_ == 1:
            empty = [r for r in range(rows) if not ref.rows[r]]
            full = [r for r in range(rows) if ref.rows[r]]
            if empty and full:
                n = int(rng.integers(1, len(empty) + 1))
                s.fork(K, [int(x) for x in rng.choice(full, n)], [int(x) for x in rng.permutation(empty)[:n]])
        elif kind_ == 2:
            s.release(K, [int(x) for x in rng.permutation(rows)[: rng.integers(0, 3)]])
        else:
            kf = [int(rng.integers(0, ref.length(r) + 1)) for r in range(rows)]
            keep = [[t for t in range(kf[r], ref.length(r)) if rng.random() < rng.choice([0.0, 0.5, 1.0])] for r in range(rows)]
            s.compact(K, kf, keep)
        s.write(step)
        s.check()


def test_compact_kinds(K):
    """Nothing kept, all kept, a cut in place, a cut inside a shared page, one moved token, an empty row."""

    s = Pair(5, rows=8, pages=80, lens=[40, 40, 40, 48, 40, 0])
    s.fork(K, [3], [6])  # rows 3 and 6 share three full pages
    s.compact(K, [0, 40, 21, 20, 8, 0, 48, 0], [[], [], [], [], [30], [], [], []])
    assert s.ref.length(3) == 20 and s.ref.rows[3][0] == s.ref.rows[6][0] and s.ref.rows[3][1] != s.ref.rows[6][1]


def test_rows_and_pools_of_size(K):
    """Thousands of rows, a pool that spans many warps' ranges, long rows."""

    s = Pair(7, rows=4096, pages=30000, cap=7, ps=2, layers=1, token=(1, 8),
             lens=[int(x) for x in np.random.default_rng(1).integers(0, 9, 4096)])
    s.reserve(K, [int(x) for x in np.random.default_rng(2).integers(0, 4, 4096)])
    live = [r for r in range(4096) if s.ref.rows[r]]
    s.release(K, live[::2])
    s.fork(K, live[1::2][:900], live[::2][:900])
    rng = np.random.default_rng(3)
    s.compact(K, [0] * 4096, [[t for t in range(s.ref.length(r)) if rng.random() < 0.6] for r in range(4096)])
    t = Pair(8, rows=3, pages=900, cap=300, ps=16, layers=2, token=(1, 8), lens=[4001, 17, 2000])
    t.compact(K, [4, 17, 0], [[x for x in range(4, 4001) if rng.random() < 0.5], [], list(range(1000, 2000))])


def test_refusals_change_nothing(K):
    from pagelora_b200 import _capi

    s = Pair(3, rows=5, pages=9, cap=4, lens=[40, 16, 30, 0, 0])
    s.reserve(K, [30, 30, 0, 0, 40], want=_capi.PL_ERR_ROW_CAPACITY)
    s.reserve(K, [20, 30, 0, 0, 40], want=_capi.PL_ERR_POOL_EXHAUSTED)
    s.reserve(K, [40, 0, 0, 0, 0], want=_capi.PL_ERR_ROW_CAPACITY)
    s.fork(K, [0, 1], [3, 3], want=_capi.PL_ERR_INVALID_ARGUMENT)
    s.fork(K, [0], [1], want=_capi.PL_ERR_INVALID_ARGUMENT)
    s.fork(K, [3, 0], [4, 3], want=_capi.PL_ERR_INVALID_ARGUMENT)
    s.fork(K, [0], [9], want=_capi.PL_ERR_INVALID_ARGUMENT)
    s.compact(K, [0, 0, 0, 0, 0], [list(range(41)), [], [], [], []], want=_capi.PL_ERR_INVALID_ARGUMENT)
    s.fork(K, [1, 1], [3, 4])  # row 1's page is full: shared, nothing allocated
    s.ref.rows[3], s.ref.last[3] = list(s.ref.rows[3]), 7  # a partial last page with other owners
    s.last[3] = 7
    s.reserve(K, [0, 0, 0, 1, 0], want=_capi.PL_ERR_PAGE_SHARED)
    # slots counted wrongly
    one = _i32([0])
    K.page_reserve(*s.tables, _i32([0, 1, 1, 1, 1, 2]), 16, slot_page=one, slot_offset=one, status=s.status)
    s.check(_capi.PL_ERR_INVALID_ARGUMENT)
    # released twice
    s.release(K, [1])
    s.refcount[s.ref.rows[0][0]] = 0
    K.page_release(*s.tables, _i32([0]), status=s.status)
    torch.cuda.synchronize()
    assert int(s.status.item()) == _capi.PL_ERR_REFCOUNT and int(s.refcount.min()) == 0
    s.status.zero_()
    K.page_release(*s.tables, _i32([77]), status=s.status)
    assert int(s.status.item()) == _capi.PL_ERR_INVALID_ARGUMENT


def test_host_refusals(K):
    s = Pair(3)
    with pytest.raises(TypeError):
        K.page_release(s.refcount.long(), s.table, s.num, s.last, _i32([0]))
    with pytest.raises(ValueError):
        K.page_release(s.refcount, s.table[:, :3], s.num, s.last, _i32([0]))
    with pytest.raises(ValueError):
        K.page_fork(s.pool[:, :5], *s.tables, _i32([0]), _i32([1]))
    with pytest.raises(ValueError):
        K.page_fork(s.pool, *s.tables, _i32([0, 1]), _i32([2, 3, 4]))
    with pytest.raises(RuntimeError, match="unsupported"):
        K.page_fork(s.pool.view(3, 60, 2, 16, 128)[..., :3].contiguous(), *s.tables, _i32([0]), _i32([1]))
    with pytest.raises(RuntimeError, match="workspace"):
        K.page_fork(s.pool, *s.tables, _i32([0]), _i32([1]), workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA"):
        K.page_release(s.refcount.cpu(), s.table, s.num, s.last, _i32([0]))


def test_layer_stride_and_long_offsets(K):
    """Layers apart from one another, and slots whose byte offset passes 2^32."""

    ps, unit = 16, (8, 128)
    pages = (1 << 32) // (2 * ps * 8 * 128 * 2) + 8
    both = torch.zeros(2, 2, pages, 2, ps, *unit, dtype=torch.bfloat16, device="cuda")
    pool = both[:, 1]
    count = torch.ones(pages, dtype=torch.int32, device="cuda")
    table = _i32([pages - 3, pages - 1, 0, 0]).view(2, 2)
    num, last = _i32([2, 0]), _i32([5, 0])
    count[pages - 2] = 0
    pool[:, pages - 1, :, :5] = torch.randn(2, 2, 5, *unit, device="cuda").to(torch.bfloat16)
    K.page_fork(pool, count, table, num, last, _i32([0]), _i32([1]))
    assert table.tolist() == [[pages - 3, pages - 1], [pages - 3, pages - 2]]
    assert torch.equal(pool[:, pages - 2], pool[:, pages - 1]) and int(count[pages - 3]) == 2
    assert not both[:, 0].any()
