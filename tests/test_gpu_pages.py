"""Page tables of the paged cache on the GPU against entry-by-entry loops: every table, count and map exactly."""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import F8, gpu, raw
from gpu_util import note
from oracle import cache_ops as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


def state(rng, B, cols, P, page, fill=0.7, share=0.0, ragged=True):
    """A table over distinct pages (some shared), its counts, and the rows' lengths."""
    tbl = np.full((B, cols), -1, np.int32)
    ids, at = rng.permutation(P).astype(np.int32), 0
    lens = np.zeros(B, np.int32)
    for b in range(B):
        n = int(rng.integers(0, cols * page + 1)) if ragged else cols * page
        n = min(n, max(0, int(P * fill) - at) * page)
        lens[b] = n
        k = -(-n // page)
        tbl[b, :k] = ids[at:at + k]
        at += k
        if b and k and rng.random() < share and lens[b - 1] >= page:
            s = min(k, lens[b - 1] // page)
            tbl[b, :s] = tbl[b - 1, :s]
    ref = np.bincount(tbl[tbl >= 0], minlength=P).astype(np.int32)
    return tbl, ref, lens


def pools(rng, P, page, H=2, D=64):
    kc = rng.integers(-128, 128, (P, page, H, D), dtype=np.int8)
    return [kc, (kc + 1).view(np.uint8), rng.standard_normal((P, max(page // 16, 1), H)).astype(np.float32),
            rng.standard_normal((P, 3)).astype(np.float32)]


def equal(name, got, want):
    got = raw(got)
    assert np.array_equal(got, want), f"{name}: {np.argwhere(got != want)[:4].tolist()}"


SIZES = [(1, 1, 1, 16), (3, 5, 20, 16), (32, 70, 1500, 16), (7, 1030, 5000, 64), (1030, 3, 2500, 32),
         (2, 20, 70000, 16)]  # more rows than a workgroup has threads, more columns, a pool of several scans


@pytest.mark.parametrize("B,cols,P,page", SIZES)
@pytest.mark.parametrize("room", [0.3, 0.95])
def test_reserve_and_free(B, cols, P, page, room):
    rng = np.random.default_rng(B + cols)
    tbl, ref, lens = state(rng, B, cols, P, page, fill=room, share=0.5)
    if B > 2:
        tbl[1, 0], tbl[2, cols - 1] = P, 2 ** 31 - 1  # no pages
    ref = np.bincount(tbl[(tbl >= 0) & (tbl < P)], minlength=P).astype(np.int32)
    want = (lens + rng.integers(-page, 3 * page, B)).astype(np.int32)
    want[0] = 2 ** 31 - 1  # past the table: clamped
    note(f"pages reserve B={B} cols={cols} P={P}")
    tt, tr, tw = gpu(tbl, ref, want)
    short = K.paged_kv_reserve(tt, tr, tw, page)
    torch.cuda.synchronize()
    t2, r2, s2 = C.reserve(tbl, ref, want, page)
    equal("table", tt, t2), equal("ref", tr, r2), equal("shortage", short, np.asarray([s2], np.int32))
    again = K.paged_kv_reserve(tt, tr, tw, page)  # nothing more to give but what was short
    torch.cuda.synchronize()
    equal("table", tt, t2), equal("ref", tr, r2), equal("shortage", again, np.asarray([s2], np.int32))
    keep = (lens - rng.integers(0, 2 * page + 1, B)).astype(np.int32)
    keep[-1] = -2 ** 31
    K.paged_kv_free(tt, tr, gpu(keep)[0], page)
    torch.cuda.synchronize()
    t3, r3 = C.free(t2, r2, keep, page)
    equal("table", tt, t3), equal("ref", tr, r3)


def test_more_rows_wants_and_moves_than_stay_on_the_chip():
    """5000 rows, 15000 wants at once and as many moves; then rows that grow by a page each in a wide table."""
    rng = np.random.default_rng(5)
    B, cols, P, page = 5000, 3, 60000, 16
    tbl, ref = np.full((B, cols), -1, np.int32), np.zeros(P, np.int32)
    ref[rng.permutation(P)[:P // 2]] = 1  # held elsewhere
    lens = np.full(B, cols * page, np.int32)
    lens[::7] = rng.integers(-5, cols * page, lens[::7].shape)
    note("pages many rows and moves")
    tt, tr = gpu(tbl, ref)
    short = K.paged_kv_reserve(tt, tr, gpu(lens)[0], page)
    t2, r2, s2 = C.reserve(tbl, ref, lens, page)
    torch.cuda.synchronize()
    equal("table", tt, t2), equal("ref", tr, r2), equal("shortage", short, np.asarray([s2], np.int32))
    perm = rng.permutation(P).astype(np.int32)  # the same pages, spread over the pool
    t3, r3 = perm[t2] * (t2 >= 0) - (t2 < 0), np.zeros(P, np.int32)
    t3 = t3.astype(np.int32)
    r3[t3[t3 >= 0]] = 1
    tt, tr = gpu(t3, r3)
    got = K.paged_kv_compact(tt, tr, [])
    t4, r4, m4, _ = C.compact(t3, r3)
    torch.cuda.synchronize()
    assert (m4 != np.arange(P)).sum() > 8192
    equal("table", tt, t4), equal("ref", tr, r4), equal("map", got, m4)
    wide, ref = np.full((70, 1024), -1, np.int32), np.zeros(900, np.int32)
    tt, tr = gpu(wide, ref)
    for n in (1, 17, 100, 161):
        lens = np.full(70, n, np.int32)
        lens[3], lens[69] = 0, n + 16
        short = K.paged_kv_reserve(tt, tr, gpu(lens)[0], page)
        wide, ref, s2 = C.reserve(wide, ref, lens, page)
        torch.cuda.synchronize()
        equal("table", tt, wide), equal("ref", tr, ref), equal("shortage", short, np.asarray([s2], np.int32))


@pytest.mark.parametrize("B,cols,P,page,extra", [(1, 1, 4, 16, 4), (4, 6, 60, 16, 40), (32, 40, 1500, 16, 64),
                                                 (9, 1030, 5000, 16, 9), (300, 4, 1500, 48, 20), (6, 5, 33, 16, 2)])
def test_fork(B, cols, P, page, extra):
    rng = np.random.default_rng(B * 3 + cols)
    tbl, ref, lens = state(rng, B, cols, P - extra, page, fill=1.0, share=0.3)
    ref = np.concatenate([ref, np.zeros(extra, np.int32)])
    parent = rng.integers(0, max(B // 3, 1), B).astype(np.int32)
    if B > 3:
        parent[1], parent[2] = -1, B
        ref[int(tbl[tbl >= 0][0])] += 1  # held elsewhere too
    caches = pools(rng, P, page)
    note(f"pages fork B={B} cols={cols} P={P}")
    tt, tr, tl, tp, *tc = gpu(tbl, ref, lens, parent, *caches)
    short = K.paged_kv_fork(tt, tr, tl, tp, tc, page)
    torch.cuda.synchronize()
    t2, r2, l2, s2, copies = C.fork(tbl, ref, lens, parent, page)
    equal("table", tt, t2), equal("ref", tr, r2), equal("lens", tl, l2)
    equal("shortage", short, np.asarray([s2], np.int32))
    for i, c in enumerate(caches):
        want = c.copy()
        for a, b in copies:
            want[b] = c[a]
        equal(f"cache {i}", tc[i], want)


def test_fork_reuses_pages_it_releases():
    """A full pool: the dropped row's pages hold the copies."""
    page, P = 16, 6
    tbl = np.asarray([[0, 1, -1], [2, 3, -1], [4, 5, -1]], np.int32)
    ref, lens, parent = np.ones(P, np.int32), np.asarray([20, 30, 32], np.int32), np.asarray([0, 0, 0], np.int32)
    rng = np.random.default_rng(0)
    caches = pools(rng, P, page)
    note("pages fork full pool")
    tt, tr, tl, tp, *tc = gpu(tbl, ref, lens, parent, *caches)
    short = K.paged_kv_fork(tt, tr, tl, tp, tc, page)
    torch.cuda.synchronize()
    equal("table", tt, np.asarray([[0, 1, -1], [0, 2, -1], [0, 3, -1]], np.int32))
    equal("ref", tr, np.asarray([3, 1, 1, 1, 0, 0], np.int32))
    assert int(short) == 0 and np.array_equal(raw(tc[0])[2], caches[0][1]) and np.array_equal(raw(tc[0])[3], caches[0][1])


@pytest.mark.parametrize("B,cols,P,page", SIZES)
@pytest.mark.parametrize("fill", [0.0, 0.4, 1.0])
def test_compact(B, cols, P, page, fill):
    if P > 10000:
        page = 1  # any page size serves a pool; small pages keep it small
    rng = np.random.default_rng(B + P)
    tbl, ref, _ = state(rng, B, cols, P, page, fill=fill, share=0.4, ragged=fill < 1)
    if B > 2:
        tbl[1, 0] = -5
        ref = np.bincount(tbl[tbl >= 0], minlength=P).astype(np.int32)
    if P > 100 and fill > 0:
        ref[P - 7] += 2  # held by no row of this table
    caches = pools(rng, P, page)
    note(f"pages compact B={B} cols={cols} P={P} fill={fill}")
    tt, tr, *tc = gpu(tbl, ref, *caches)
    to = K.paged_kv_compact(tt, tr, tc)
    torch.cuda.synchronize()
    t2, r2, m2, moves = C.compact(tbl, ref)
    equal("table", tt, t2), equal("ref", tr, r2), equal("map", to, m2)
    src, dst = (np.asarray([m[i] for m in moves], np.int64) for i in (0, 1))
    for i, c in enumerate(caches):
        want = c.copy()
        want[dst] = c[src]
        equal(f"cache {i}", tc[i], want)


def test_copy_layers_and_odd_pages():
    """Seventy page tensors of different sizes and alignments, one of them a layer of a larger pool."""
    rng = np.random.default_rng(7)
    P = 40
    plain = [rng.integers(0, 255, (P, 1 + 37 * i), dtype=np.int64).astype(np.int8) for i in range(68)]
    plain.append(rng.standard_normal((P, 9000)).astype(np.float32))  # more than one chunk
    pool = rng.integers(-128, 128, (P, 2, 16, 64), dtype=np.int64).astype(np.int8)
    src = rng.permutation(P)[:20].astype(np.int32)
    left = np.setdiff1d(np.arange(P), src).astype(np.int32)
    dst = rng.permutation(left)[:20].astype(np.int32)
    src[3], dst[5] = -1, P  # left out
    note("pages copy")
    tp = gpu(pool)[0]
    tc = gpu(*plain) + [tp[:, 1]]
    K.paged_kv_copy(*gpu(src, dst), tc)
    torch.cuda.synchronize()
    ok = [i for i in range(20) if i not in (3, 5)]
    for i, c in enumerate(plain):
        want = c.copy()
        want[dst[ok]] = c[src[ok]]
        equal(f"tensor {i}", tc[i], want)
    want = pool.copy()
    want[dst[ok], 1] = pool[src[ok], 1]
    equal("layer", tp, want)


def test_graph_replays_and_a_second_stream():
    """A step's reserve and free, and a fork, captured and replayed, each replay against the loops; then the same on
    a stream with a workspace of its own."""
    from specq.workspace import Workspace
    rng = np.random.default_rng(11)
    B, cols, P, page = 6, 12, 200, 16
    tbl, ref, lens = state(rng, B, cols, P, page, fill=0.4)
    caches = pools(rng, P, page)
    tt, tr, tl, *tc = gpu(tbl, ref, lens, *caches)
    want, keep, parent = (torch.zeros(B, dtype=torch.int32, device=DEV) for _ in range(3))
    short = torch.zeros(2, dtype=torch.int32, device=DEV)
    ws = Workspace(DEV)

    def step(**kw):
        K.paged_kv_reserve(tt, tr, want, page, shortage=short[:1], **kw)
        K.paged_kv_free(tt, tr, keep, page)
        K.paged_kv_fork(tt, tr, tl, parent, tc, page, shortage=short[1:], **kw)
    note("pages graph")
    parent.copy_(torch.arange(B, dtype=torch.int32))
    want.copy_(tl), keep.copy_(tl)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    st = torch.cuda.Stream()
    t, r, n = raw(tt).copy(), raw(tr).copy(), lens
    for i in range(6):
        w = (n + rng.integers(0, 40, B)).astype(np.int32)
        w = np.minimum(w, cols * page)
        k = np.minimum(w, n + rng.integers(0, 10, B)).astype(np.int32)
        p = rng.integers(-1, B, B).astype(np.int32)
        for x, y in ((want, w), (keep, k), (parent, p), (tl, k)):
            x.copy_(gpu(y)[0])
        torch.cuda.synchronize()
        if i % 2 == 0:
            g.replay()
        else:
            with torch.cuda.stream(st):
                step(workspace=ws)
        torch.cuda.synchronize()
        t, r, s0 = C.reserve(t, r, w, page)
        t, r = C.free(t, r, k, page)
        t, r, n, s1, copies = C.fork(t, r, k, p, page)
        for j, c in enumerate(caches):
            c2 = c.copy()
            for a, b in copies:
                c2[b] = c[a]
            caches[j] = c2
            equal(f"cache {j}", tc[j], c2)
        equal("table", tt, t), equal("ref", tr, r), equal("lens", tl, n), equal("shortage", short, np.asarray([s0, s1], np.int32))


def test_refusals():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    tbl, ref, v = i32(3, 4), i32(10), i32(3)
    cache = torch.zeros((10, 16, 2, 64), dtype=torch.int8, device=DEV)
    note("pages refusals")
    for f, args in [(K.paged_kv_reserve, (tbl.long(), ref, v, 16)), (K.paged_kv_reserve, (tbl, ref.long(), v, 16)),
                    (K.paged_kv_reserve, (tbl, ref, v[:2], 16)), (K.paged_kv_reserve, (tbl, ref, v, 0)),
                    (K.paged_kv_reserve, (tbl.t(), ref, i32(4), 16)), (K.paged_kv_reserve, (tbl[:, :0], ref, v, 16)),
                    (K.paged_kv_reserve, (i32(1, 4).expand(3, 4), ref, v, 16)), (K.paged_kv_reserve, (tbl, ref[:0], v, 16)),
                    (K.paged_kv_free, (tbl, ref, v.cpu(), 16)), (K.paged_kv_free, (tbl.cpu(), ref, v, 16)),
                    (K.paged_kv_fork, (tbl, ref, v, v[:1], [cache], 16)), (K.paged_kv_fork, (tbl, ref, v, v, [cache[:9]], 16)),
                    (K.paged_kv_fork, (tbl, ref, v, v, [cache.transpose(1, 2)], 16)), (K.paged_kv_fork, (tbl, ref, v, v, [cache.cpu()], 16)),
                    (K.paged_kv_compact, (tbl, ref, [cache[:, :0]])), (K.paged_kv_copy, (v, v[:2], [cache])),
                    (K.paged_kv_copy, (v.long(), v, [cache])), (K.paged_kv_copy, (v, v, []))]:
        with pytest.raises(RuntimeError):
            f(*args)
    with pytest.raises(RuntimeError):
        K.paged_kv_reserve(tbl, ref, v, 16, shortage=i32(1).long())
    with pytest.raises(RuntimeError):
        K.paged_kv_compact(tbl, ref, [cache], page_map=i32(9))
    K.paged_kv_copy(v[:0], v[:0], [cache])
    assert cache.view(torch.uint8).view(F8).shape == cache.shape


def test_outputs_on_another_device_are_refused():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    tbl, ref, v = i32(3, 4), i32(10), i32(3)
    note("pages outputs elsewhere")
    for call in (lambda: K.paged_kv_reserve(tbl, ref, v, 16, shortage=i32(1).cpu()),
                 lambda: K.paged_kv_fork(tbl, ref, v, v.clone(), [], 16, shortage=i32(1).cpu()),
                 lambda: K.paged_kv_compact(tbl, ref, [], page_map=i32(10).cpu())):
        with pytest.raises(RuntimeError, match="cpu"):
            call()


WIDTHS = {  # bytes of a page: chunks of 16384 in full and in part, next to pages of a scale or two
    "16 bytes": (40 * 1024 + 16, 16384, 16),
    "one scale": (32 * 1024, 4 * 16384 + 48, 4),
    "two scales": (20 * 1024, 8),
    "odd": (16384 + 36, 37, 1),
}


@pytest.mark.parametrize("what", list(WIDTHS))
def test_page_copies_at_every_access_width(what):
    """Fork, compact and copy of pages that take several workgroups each, at 16, 4 and 1 bytes an access."""
    rng = np.random.default_rng(len(what))
    B, cols, page, P = 8, 6, 16, 60
    make = lambda: [rng.integers(-128, 128, (P, n), dtype=np.int64).astype(np.int8) for n in WIDTHS[what]]  # noqa: E731

    def held(caches, tensors, moves, step):
        for i, (c, t) in enumerate(zip(caches, tensors)):
            want = c.copy()
            for a, b in moves:
                want[b] = c[a]
            equal(f"{step} {i}", t, want)

    tbl, ref, lens = state(rng, B, cols, P - 12, page, fill=1.0)
    ref = np.concatenate([ref, np.zeros(12, np.int32)])
    lens[0] += lens[0] % page == 0  # a last page to copy
    tbl[0, (lens[0] - 1) // page] = P - 1
    ref = np.bincount(tbl[tbl >= 0], minlength=P).astype(np.int32)
    parent = np.zeros(B, np.int32)
    caches = make()
    note(f"pages widths {what}")
    tt, tr, tl, tp, *tc = gpu(tbl, ref, lens, parent, *caches)
    K.paged_kv_fork(tt, tr, tl, tp, tc, page)
    torch.cuda.synchronize()
    *_, copies = C.fork(tbl, ref, lens, parent, page)
    assert len(copies) == B - 1
    held(caches, tc, copies, "fork")

    tbl, ref, _ = state(rng, B, cols, P, page, fill=0.5)
    caches = make()
    tt, tr, *tc = gpu(tbl, ref, *caches)
    K.paged_kv_compact(tt, tr, tc)
    torch.cuda.synchronize()
    *_, moves = C.compact(tbl, ref)
    assert len(moves) > 4
    held(caches, tc, moves, "compact")

    caches = make()
    src, dst = np.split(rng.permutation(P).astype(np.int32), 2)
    tc = gpu(*caches)
    K.paged_kv_copy(*gpu(src, dst), tc)
    torch.cuda.synchronize()
    held(caches, tc, list(zip(src, dst)), "copy")
