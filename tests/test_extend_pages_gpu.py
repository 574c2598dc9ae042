"""GPU: the tables of a step (extend_pages) and giving pages back (trim_pages) against a sequential
model of them."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

pytestmark = pytest.mark.gpu
GONE = _lib.PAGE_TRIMMED


class Model:
    """Tables, lengths and counts on the host, changed as the operators say."""

    def __init__(self, slots, width, page, pages, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.page, self.pages, self.width = page, pages, width
        self.tables = torch.full((slots, width), -1, dtype=torch.int32)
        self.seq = torch.zeros(slots, dtype=torch.int32)
        self.refs = torch.zeros(pages, dtype=torch.int32)
        self.error = 0

    def fill(self, slot, n):
        free = (self.refs == 0).nonzero().flatten()
        for j in range(-(-n // self.page)):
            p = int(free[torch.randint(0, len(free), (), generator=self.g)])
            free = free[free != p]
            self.tables[slot, j], self.refs[p] = p, 1
        self.seq[slot] = n

    def drop(self, p):
        if p >= self.pages or self.refs[p] <= 0:
            self.error |= _lib.DEVERR_BAD_PAGE
        else:
            self.refs[p] -= 1

    def extend(self, slots, new, lens, tokens):
        P, n = self.page, len(slots)
        start = [None] * n
        for k, (s, m) in enumerate(zip(slots, new)):
            if not 0 <= s < len(self.seq) or s in slots[:k]:
                self.error |= _lib.DEVERR_BAD_SLOT
                continue
            have = int(self.seq[s])
            at = have if lens is None else lens[k]
            if m < 0 or at < 0 or at > have:
                self.error |= _lib.DEVERR_SEQ_LEN
            elif at + m > self.width * P:
                self.error |= _lib.DEVERR_CAPACITY
            else:
                pg = int(self.tables[s, at // P]) if m and at % P else None
                if pg is not None and (not 0 <= pg < self.pages or self.refs[pg] != 1):
                    self.error |= _lib.DEVERR_BAD_PAGE
                else:
                    start[k] = at
        for k, s in enumerate(slots):
            if start[k] is not None:
                for j in range(-(-start[k] // P), min(self.width, -(-int(self.seq[s]) // P))):
                    if self.tables[s, j] >= 0:
                        self.drop(int(self.tables[s, j]))
                    self.tables[s, j] = -1
        free = (self.refs == 0).nonzero().flatten().tolist()
        t = q = 0
        out = dict(slot=[], pos=[], cu=[0], lens=[], tables=[])
        for k, (s, m) in enumerate(zip(slots, new)):
            ok = start[k] is not None
            if ok:
                need = -(-(start[k] + m) // P) - -(-start[k] // P)
                t += m
                q += need
                self.seq[s] = start[k]
                if (m and t > tokens) or (need and q > len(free)):
                    self.error |= _lib.DEVERR_CAPACITY
                    ok = False
            if not ok:
                out["cu"].append(out["cu"][-1])
                out["lens"].append(0)
                out["tables"].append(torch.full((self.width,), -1, dtype=torch.int32))
                continue
            first = -(-start[k] // P)
            for i in range(need):
                self.tables[s, first + i] = free[q - need + i]
                self.refs[free[q - need + i]] = 1
            self.seq[s] = start[k] + m
            for p in range(start[k], start[k] + m):
                out["slot"].append(int(self.tables[s, p // P]) * P + p % P)
                out["pos"].append(p)
            out["cu"].append(out["cu"][-1] + m)
            out["lens"].append(start[k] + m)
            out["tables"].append(self.tables[s].clone())
        pad = tokens - len(out["slot"])
        return (torch.tensor(out["slot"] + [-1] * pad, dtype=torch.int64), torch.tensor(out["pos"] + [0] * pad, dtype=torch.int32),
                torch.tensor(out["cu"], dtype=torch.int32), torch.tensor(out["lens"], dtype=torch.int32),
                torch.stack(out["tables"]) if n else torch.zeros(0, self.width, dtype=torch.int32))

    def trim(self, slots, window, sinks):
        P = self.page
        for s in slots:
            if not 0 <= s < len(self.seq):
                self.error |= _lib.DEVERR_BAD_SLOT
                continue
            n = int(self.seq[s])
            for j in range(self.width):
                p = int(self.tables[s, j])
                behind = window and j * P >= sinks and (j + 1) * P <= n - window + 1
                if p >= 0 and (behind or j * P >= n):
                    self.drop(p)
                    self.tables[s, j] = GONE if behind else -1

    def cuda(self):
        return self.tables.cuda(), self.seq.cuda(), self.refs.cuda()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def step(m, dev, slots, new, lens, tokens, page=None):
    """One call on the device copies `dev` and on the model: everything equal."""
    tables, seq, refs = dev
    m.error = 0
    want = m.extend(slots, new, lens, tokens)
    got = rt.extend_pages(tables, seq, ints(slots), ints(new), refs, m.page, tokens, lens=None if lens is None else ints(lens))
    assert rt.device_errors() == m.error
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
    same(m, dev)
    return got


def same(m, dev):
    for a, b in zip(dev, (m.tables, m.seq, m.refs)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("page,lens,new,pages,pad", [
    (64, [0], [1], 1, 0), (64, [63, 64, 65], [1, 1, 1], 20, 5), (16, [0, 5, 16, 31, 100], [40, 0, 16, 1, 7], 60, 0),
    (1, [3, 0], [5, 2], 11, 1), (48, [47, 48, 1000], [1, 100, 500], 60, 3), (16, [7] * 300, [3, 0, 20] * 100, 3000, 0),
    (64, [100] * 1500, [1, 30, 70] * 500, 6000, 17), (128, [5000], [9000], 200, 0), (16, [0] * 40, [500] * 40, 20000, 9),
])
def test_a_step_matches_the_model(page, lens, new, pages, pad):
    n = len(lens)
    width = max(-(-(a + b) // page) for a, b in zip(lens, new)) + 2
    m = Model(n + 3, width, page, pages, seed=pages)
    order = torch.randperm(n + 3, generator=m.g)[:n].tolist()
    for s, a in zip(order, lens):
        m.fill(s, a)
    dev = m.cuda()
    step(m, dev, order, new, None, sum(new) + pad)
    assert m.error == 0
    # a second step: half of the first one's tokens are taken back
    back = [a + b - b // 2 for a, b in zip(lens, new)]
    step(m, dev, order, [1] * n, back, n + pad)
    rt.free_pages(dev[0], dev[1], ints(order), dev[2])
    assert rt.device_errors() == 0 and not dev[2].any() and bool((dev[0] == -1).all())


@pytest.mark.parametrize("n", [1000, 2500])
def test_many_requests_and_slots(n):
    """More slots, and more requests, than the chip's own memory holds, some of them twice."""
    m = Model(5000, 4, 16, 8000, seed=n)
    order = torch.randperm(5000, generator=m.g)[:n].tolist()
    order[7], order[n - 1] = order[3], order[400]
    new = torch.randint(0, 40, (n,), generator=m.g).tolist()
    dev = m.cuda()
    step(m, dev, order, new, None, sum(new))
    assert m.error == _lib.DEVERR_BAD_SLOT
    back = [a - a // 3 for a in new]
    step(m, dev, order, [1] * n, back, n)
    assert m.error == _lib.DEVERR_BAD_SLOT


def test_every_request_that_is_skipped():
    m = Model(12, 8, 16, 40, seed=2)
    for s, n in enumerate([20, 33, 16, 0, 40, 100, 5, 50]):
        m.fill(s, n)
    m.refs[m.tables[1, 2]] = 2                     # the page that slot 1's next token falls into is shared
    m.tables[4, 2] = -1                            # that of slot 4 is missing, of slot 7 out of range
    m.tables[7, 3] = 40
    slots = [0, 0, 1, 2, -1, 12, 3, 4, 5, 6, 7]
    new = [4, 1, 1, -1, 1, 1, 3, 2, 29, 0, 1]      # (slot 5: past the table)
    dev = m.cuda()
    step(m, dev, slots, new, None, 50)
    assert m.error == _lib.DEVERR_BAD_SLOT | _lib.DEVERR_SEQ_LEN | _lib.DEVERR_BAD_PAGE | _lib.DEVERR_CAPACITY
    # lens above the length, below zero; a page that is cut back into is checked like any other
    step(m, dev, [0, 2, 1], [1, 1, 1], [25, -1, 32], 9)
    assert m.error == _lib.DEVERR_SEQ_LEN


@pytest.mark.parametrize("tokens,pages", [(20, 30), (100, 9), (0, 30), (33, 12)])
def test_what_there_is_goes_to_the_first(tokens, pages):
    """Too few rows or free pages: in order, and a request that needs neither still counts."""
    m = Model(8, 10, 16, pages, seed=5)
    for s, n in enumerate([20, 16, 3, 30]):
        m.fill(s, n)
    dev = m.cuda()
    step(m, dev, [3, 1, 0, 2, 5, 6], [10, 20, 1, 2, 0, 16], [25, 16, 20, 1, 0, 0], tokens)
    assert m.error == _lib.DEVERR_CAPACITY


def test_no_requests_and_no_tokens():
    m = Model(3, 4, 16, 6)
    m.fill(1, 20)
    dev = m.cuda()
    step(m, dev, [], [], None, 5)
    step(m, dev, [], [], None, 0)
    step(m, dev, [1, 2], [0, 0], None, 0)
    step(m, dev, [1, 2], [0, 0], None, 3)
    assert m.error == 0
    rt.trim_pages(dev[0], dev[1], ints([]), dev[2], 16, window=3)
    same(m, dev)


@pytest.mark.parametrize("page,window,sinks", [(16, 1, 0), (16, 40, 4), (16, 40, 17), (64, 128, 64), (1, 3, 2), (16, 10 ** 12, 3), (16, 0, 0)])
def test_trim(page, window, sinks):
    m = Model(7, 12, page, 90, seed=page + sinks)
    for s, n in enumerate([0, 1, page, 5 * page + 1, 12 * page, 7 * page - 1]):
        m.fill(s, n)
    m.seq[4] = 9 * page + 3 if page > 3 else 9     # shortened: its pages past the end go back too
    slots = [0, 3, 5, 4, 1, 2, 3, 6]
    dev = m.cuda()
    for _ in range(2):                             # (the second call finds nothing)
        m.trim(slots, window, sinks)
        rt.trim_pages(dev[0], dev[1], ints(slots), dev[2], page, window=window, sinks=sinks)
        assert rt.device_errors() == m.error == 0
        same(m, dev)


def test_trim_bad_ids():
    m = Model(4, 6, 16, 12, seed=4)
    m.fill(0, 90)
    m.fill(1, 70)
    m.tables[0, 1] = 12                            # out of range
    m.refs[m.tables[1, 1]] = 0                     # has no reference left
    dev = m.cuda()
    m.trim([0, 1, -1, 4], 20, 0)
    rt.trim_pages(dev[0], dev[1], ints([0, 1, -1, 4]), dev[2], 16, window=20)
    assert rt.device_errors() == m.error == _lib.DEVERR_BAD_SLOT | _lib.DEVERR_BAD_PAGE
    same(m, dev)


def test_a_windowed_sequence_is_forked_compacted_and_freed():
    """Trimmed entries stay trimmed in a fork and a compaction, and free_pages passes over them."""
    m = Model(4, 12, 16, 30, seed=6)
    m.fill(0, 150)
    m.fill(1, 20)
    dev = m.cuda()
    tables, seq, refs = dev
    cache = torch.randint(0, 256, (30, 16, 8), dtype=torch.uint8, device="cuda")
    rt.trim_pages(tables, seq, ints([0]), refs, 16, window=40, sinks=4)
    gone = tables[0] == GONE
    assert gone.tolist() == [False] + [True] * 5 + [False] * 6      # pages 1 .. 5: tokens 16 .. 95 of 111
    rows = lambda s: [cache[int(p)].clone() for p in tables[s] if int(p) >= 0]  # noqa: E731
    before = rows(0)
    rt.fork_pages([cache], tables, seq, ints([0]), ints([2]), refs)
    assert rt.device_errors() == 0
    assert torch.equal(tables[2] == GONE, gone) and int(seq[2]) == 150
    rt.free_pages(tables, seq, ints([1]), refs)
    live = rt.compact_pages([cache], tables, refs)
    assert rt.device_errors() == 0
    assert int(live) == int((refs > 0).sum()) and bool((refs[: int(live)] > 0).all())
    assert torch.equal(tables[0] == GONE, gone) and torch.equal(tables[2] == GONE, gone)
    after = rows(0)
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    for a, b in zip(rows(2)[:-1], after[:-1]):
        assert torch.equal(a, b)
    e = rt.extend_pages(tables, seq, ints([0, 2]), ints([11, 11]), refs, 16, 22)
    assert rt.device_errors() == 0 and len(set(e.slot_mapping.tolist())) == 22
    rt.free_pages(tables, seq, ints([0, 2]), refs)
    assert rt.device_errors() == 0 and not refs.any() and bool((tables == -1).all())


def test_strided_tables_large_pools_and_other_streams():
    m = Model(70, 40, 16, 100001, seed=8)
    m.refs[:97000] = 1                             # the free pages lie far into the pool, which is not a multiple of 16
    for s in range(70):
        m.fill(s, 8 * s)
    m.refs[torch.randperm(97000, generator=m.g)[:50]] = 0
    wide = torch.full((70, 50), 7, dtype=torch.int32, device="cuda")
    wide[:, 5:45] = m.tables.cuda()
    offset = torch.zeros(100002, dtype=torch.int32, device="cuda")
    offset[1:] = m.refs.cuda()                     # counts that no 16-byte load can take
    dev = (wide[:, 5:45], m.seq.cuda(), offset[1:])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    slots = torch.randperm(70, generator=m.g).tolist()
    new = [int(v) for v in torch.randint(0, 30, (70,), generator=m.g)]
    with torch.cuda.stream(s):
        step(m, dev, slots, new, None, sum(new) + 3)
    s.synchronize()
    assert m.error == 0 and bool((wide[:, :5] == 7).all()) and bool((wide[:, 45:] == 7).all())


def test_a_graph_follows_the_lengths_on_the_device():
    m = Model(6, 20, 16, 50, seed=9)
    for s, n in enumerate([5, 16, 40, 0, 90, 31]):
        m.fill(s, n)
    dev = m.cuda()
    start = [t.clone() for t in dev]
    slots, new, lens = ints([4, 1, 2]), ints([1, 1, 1]), ints([90, 16, 40])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rt.extend_pages(*dev[:2], slots, new, dev[2], 16, 40, lens=lens)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            e = rt.extend_pages(*dev[:2], slots, new, dev[2], 16, 40, lens=lens)
            rt.trim_pages(*dev[:2], slots, dev[2], 16, window=20, sinks=2)
        rt.extend_pages(torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), ints([0, 0, 0]), ints([0]), ints([9]),
                        torch.zeros(9000, dtype=torch.int32, device="cuda"), 16, 10)      # grows the stream's buffer
        for rows in (([4, 1, 2], [1, 1, 1], [90, 16, 40]), ([0, 3, 5], [7, 33, 0], [3, 0, 31]), ([2, 2, 1], [20, 1, 9], [35, 35, 2])):
            model = Model(6, 20, 16, 50)
            model.tables, model.seq, model.refs = m.tables.clone(), m.seq.clone(), m.refs.clone()
            for t, t0 in zip(dev, start):
                t.copy_(t0)
            for t, v in zip((slots, new, lens), rows):
                t.copy_(torch.tensor(v, dtype=torch.int32))
            graph.replay()
            s.synchronize()
            want = model.extend(*rows, 40)
            for a, b in zip(e, want):
                assert torch.equal(a.cpu(), b)
            model.trim(rows[0], 20, 2)
            assert rt.device_errors() == model.error
            same(model, dev)


BASE = dict(block_tables=lambda: torch.full((4, 3), -1, dtype=torch.int32, device="cuda"), seq_lens=lambda: ints([0] * 4),
            slots=lambda: ints([0, 1]), ref_counts=lambda: ints([0] * 9), page_size=16)
EXTEND = BASE | dict(new_lens=lambda: ints([1, 2]), num_tokens=4)


@pytest.mark.parametrize("call,args,change,error,word", [
    (rt.extend_pages, EXTEND, dict(block_tables=torch.full((4, 3), -1, dtype=torch.int32)), ValueError, "CUDA"),
    (rt.extend_pages, EXTEND, dict(seq_lens=lambda: ints([0] * 3)), ValueError, "one entry per row"),
    (rt.extend_pages, EXTEND, dict(seq_lens=lambda: ints([0] * 4).long()), TypeError, "seq_lens must be int32"),
    (rt.extend_pages, EXTEND, dict(slots=torch.tensor([0, 1], dtype=torch.int32)), ValueError, "slots must be a CUDA"),
    (rt.extend_pages, EXTEND, dict(new_lens=lambda: ints([1])), ValueError, "one entry per slot"),
    (rt.extend_pages, EXTEND, dict(new_lens=lambda: ints([1, 1, 1, 1])[::2]), ValueError, "contiguous"),
    (rt.extend_pages, EXTEND, dict(lens=lambda: ints([1, 2, 3])), ValueError, "one entry per slot"),
    (rt.extend_pages, EXTEND, dict(lens=lambda: ints([1, 2]).float()), TypeError, "lens must be int32"),
    (rt.extend_pages, EXTEND, dict(num_tokens=-1), ValueError, "num_tokens"),
    (rt.extend_pages, EXTEND, dict(page_size=0), RuntimeError, "page_size"),
    (rt.extend_pages, EXTEND, dict(page_size=1 << 30), RuntimeError, "2\\^31"),
    (rt.extend_pages, EXTEND, dict(block_tables=lambda: torch.full((4, 6), -1, dtype=torch.int32, device="cuda")[:, ::2]), ValueError, "contiguous"),
    (rt.extend_pages, EXTEND, dict(ref_counts=lambda: ints([])), RuntimeError, "null|num_pages"),
    (rt.trim_pages, BASE, dict(seq_lens=lambda: ints([0] * 5)), ValueError, "one entry per row"),
    (rt.trim_pages, BASE, dict(window=-1), ValueError, "window"),
    (rt.trim_pages, BASE, dict(sinks=4), ValueError, "window"),
    (rt.trim_pages, BASE, dict(page_size=0), RuntimeError, "page_size"),
    (rt.trim_pages, BASE, dict(slots=lambda: ints([0]).long()), TypeError, "slots must be int32"),
])
def test_refusals(call, args, change, error, word):
    with pytest.raises(error, match=word):
        call(**{k: v() if callable(v) else v for k, v in (args | change).items()})
    assert rt.device_errors() == 0
