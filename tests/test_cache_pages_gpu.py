"""GPU: freeing, forking, copying and compacting pages against a sequential model of them."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

pytestmark = pytest.mark.gpu


def make(pages, page, lens, slots, width, seed, widths=(288, 128, 72)):
    g = torch.Generator().manual_seed(seed)
    caches = [torch.randint(0, 256, (pages, page, w), generator=g, dtype=torch.uint8).cuda() for w in widths]
    perm = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((slots, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    seq = torch.zeros(slots, dtype=torch.int32)
    for s, n in enumerate(lens):
        seq[s] = n
        for j in range(-(-n // page)):
            tables[s, j] = perm.pop()
            refs[tables[s, j]] = 1
    return caches, tables, refs, seq


def model_fork(caches, tables, refs, seq, src, dst, page):
    """In place on host copies; parents are read as they were before the call."""
    t0, s0 = tables.clone(), seq.clone()
    free = [p for p in range(refs.numel()) if refs[p] == 0]
    done = set()
    for s, d in zip(src, dst):
        if not (0 <= s < len(s0) and 0 <= d < len(s0)) or s0[d] != 0 or d in done or s == d:
            continue
        n = int(s0[s])
        full, rest = divmod(n, page)
        if rest and int(t0[s, full]) >= 0 and not free:
            continue
        done.add(d)
        row = torch.full((tables.shape[1],), -1, dtype=torch.int32)
        for j in range(full):
            row[j] = t0[s, j]
            if row[j] >= 0:
                refs[row[j]] += 1
        if rest and int(t0[s, full]) >= 0:
            p = free.pop(0)
            row[full] = p
            refs[p] += 1
            for c in caches:
                c[p, :rest] = c[int(t0[s, full]), :rest]
        tables[d], seq[d] = row, n


def same(caches, host, *pairs):
    for c, h in zip(caches, host):
        assert torch.equal(c.cpu(), h)
    for a, b in pairs:
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("page,lens,children,pages", [(64, [200, 64, 1, 130], 9, 40), (16, [1000], 70, 200),
                                                      (1, [5, 3], 4, 20), (4, [7] * 30, 2000, 3000),
                                                      (16, [0, 17], 3, 17000)])
def test_fork_then_free(page, lens, children, pages):
    P = len(lens)
    width = max(1, max(-(-n // page) for n in lens)) + 2
    caches, tables, refs, seq = make(pages, page, lens, P + children, width, page + children)
    g = torch.Generator().manual_seed(1)
    src = torch.randint(0, P, (children,), generator=g, dtype=torch.int32)
    dst = (P + torch.randperm(children, generator=g)).int()
    dt, dr, ds = tables.cuda(), refs.cuda(), seq.cuda()
    host = [c.cpu() for c in caches]
    t, r, s = tables.clone(), refs.clone(), seq.clone()
    model_fork(host, t, r, s, src.tolist(), dst.tolist(), page)
    rt.fork_pages(caches, dt, ds, src.cuda(), dst.cuda(), dr)
    assert rt.device_errors() == 0
    same(caches, host, (dt, t), (dr, r), (ds, s))
    rt.free_pages(dt, ds, dst.cuda(), dr)
    assert rt.device_errors() == 0
    same(caches, host, (dt, tables), (dr, refs), (ds, seq))


def test_fork_refuses_on_the_device():
    page = 16
    caches, tables, refs, seq = make(8, page, [40, 33], 8, 4, 3)       # 6 pages used, 2 free
    tables[1, 0] = -1                                                   # a missing full page
    src = [0, 0, 9, 0, 1, 0, 0, 4]
    dst = [2, 2, 3, 1, 4, 0, 5, 6]
    dt, dr, ds = tables.cuda(), refs.cuda(), seq.cuda()
    host = [c.cpu() for c in caches]
    t, r, s = tables.clone(), refs.clone(), seq.clone()
    model_fork(host, t, r, s, src, dst, page)
    rt.fork_pages(caches, dt, ds, torch.tensor(src, dtype=torch.int32).cuda(), torch.tensor(dst, dtype=torch.int32).cuda(), dr)
    # twice named, bad, occupied and own slots; a missing page; no page left for the fork into 5
    assert rt.device_errors() == _lib.DEVERR_BAD_SLOT | _lib.DEVERR_BAD_PAGE | _lib.DEVERR_CAPACITY
    same(caches, host, (dt, t), (dr, r), (ds, s))


def test_free_twice_and_bad_ids():
    caches, tables, refs, seq = make(12, 16, [40, 33], 3, 4, 4)
    tables[1, 1] = 12
    refs[tables[1, 0]] = 0                                              # has no reference left
    dt, dr, ds = tables.cuda(), refs.cuda(), seq.cuda()
    rt.free_pages(dt, ds, torch.tensor([0, 0, 1, 7, -1], dtype=torch.int32).cuda(), dr)
    assert rt.device_errors() == _lib.DEVERR_BAD_SLOT | _lib.DEVERR_BAD_PAGE
    want = refs.clone()
    want[tables[0, :3].long()] = 0
    want[tables[1, 2]] = 0
    assert torch.equal(dr.cpu(), want) and bool((dt == -1).all()) and not ds.any()


@pytest.mark.parametrize("widths", [(288, 128, 72), (72,), (7, 288)])
def test_copy_pages(widths):
    caches, _, _, _ = make(30, 2, [], 1, 1, 7, widths)
    src = torch.tensor([3, 4, -1, 29, 5, 30, 8], dtype=torch.int32)
    dst = torch.tensor([10, 11, 12, 0, -1, 13, 31], dtype=torch.int32)
    host = [c.cpu() for c in caches]
    for s, d in [(3, 10), (4, 11), (29, 0)]:
        for h in host:
            h[d] = h[s]
    rt.copy_pages(caches, src.cuda(), dst.cuda())
    assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
    same(caches, host)
    rt.copy_pages(caches, src[:0].cuda(), dst[:0].cuda())


@pytest.mark.parametrize("pages,live,seed", [(1, 1, 0), (7, 0, 1), (50, 50, 2), (1025, 300, 3), (5000, 4100, 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(pages, live, seed, in_place):
    page, width = 4, 6
    g = torch.Generator().manual_seed(seed)
    caches = [torch.randint(0, 256, (pages, page, w), generator=g, dtype=torch.uint8).cuda() for w in (288, 8)]
    used = torch.randperm(pages, generator=g)[:live]
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[used] = torch.randint(1, 4, (live,), generator=g, dtype=torch.int32)
    slots = 40
    wide = torch.full((slots, width + 3), -7, dtype=torch.int32)
    tables = wide[:, :width]
    tables[:] = used[torch.randint(0, max(live, 1), (slots, width), generator=g)] if live else -1
    tables[3, 2:] = -1
    dead = [p for p in range(pages) if refs[p] == 0][:1]
    if dead:
        tables[5, 0] = dead[0]
    tables[6, 1] = pages
    order = sorted(used.tolist())
    holes, movers = [p for p in range(live) if refs[p] == 0], [p for p in order if p >= live]
    remap = {p: p for p in order} | dict(zip(movers, holes))
    host = [c.cpu() for c in caches]
    r = refs.clone()
    for a, b in zip(movers, holes):
        for h in host:
            h[b] = h[a]
        r[b], r[a] = refs[a], 0
    t = tables.clone().apply_(lambda p: remap.get(p, -1))
    dw, dr = wide.cuda(), refs.cuda()
    dt = dw[:, :width]
    out_t, out_r = (dt, dr) if in_place else (torch.full_like(dt, 9), torch.full_like(dr, 9))
    n = rt.compact_pages(caches, dt, dr, out_tables=out_t, out_ref_counts=out_r)
    assert int(n) == live
    assert rt.device_errors() == _lib.DEVERR_BAD_PAGE
    same(caches, host, (out_t, t), (out_r, r))
    assert bool((dw[:, width:] == -7).all())
    if not in_place:
        same([], [], (dt, tables), (dr, refs))


def test_compact_far_pages():
    """Page addresses past 2^32 bytes."""
    pages, page = 250000, 64
    cache = torch.empty(pages, page, 288, dtype=torch.uint8, device="cuda")
    cache[-1] = 7
    cache[-5] = 9
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[-1] = refs[-5] = 2
    tables = torch.tensor([[pages - 1, pages - 5, -1]], dtype=torch.int32, device="cuda")
    assert int(rt.compact_pages([cache], tables, refs)) == 2
    assert tables.tolist() == [[1, 0, -1]] and refs[:3].tolist() == [2, 2, 0]
    assert bool((cache[0] == 9).all()) and bool((cache[1] == 7).all())
    assert rt.device_errors() == 0
