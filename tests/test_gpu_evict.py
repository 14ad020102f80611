"""Eviction from a paged cache on the GPU: everything it moves, keeps and leaves, exactly."""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import gpu
from gpu_util import note
from oracle import batch_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(rng, ctx, HK, D, PAGE, weights="spread", spare=3):
    pages = [max(0, -(-c // PAGE)) for c in ctx]
    P, C = sum(pages) + spare, max(max(pages), 1) + 1
    bt = np.full((len(ctx), C), -1, np.int32)
    perm, at = rng.permutation(P).astype(np.int32), 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[at:at + n]
        at += n
    caches = [rng.integers(-128, 128, (P, PAGE, HK, D), dtype=np.int8) for _ in "kv"]
    caches += [rng.uniform(0, 1, (P, PAGE, HK)).astype(np.float16) for _ in "kv"]
    shape = (len(ctx), HK, C * PAGE)
    w = {"spread": lambda: np.exp(2 * rng.standard_normal(shape)), "few": lambda: rng.integers(0, 3, shape),
         "zero": lambda: np.zeros(shape), "signed": lambda: rng.standard_normal(shape)}[weights]().astype(np.float32)
    return bt, np.asarray(ctx, np.int32), w, caches


def run_check(case, budget, recent, sinks, limit=None, ref=None, what=""):
    bt, ctx, w, caches = case
    PAGE = caches[0].shape[1]
    tb, tc, tw = gpu(bt, ctx, w)
    tcs = gpu(*caches)
    kept = K.paged_kv_evict(tb, tc, tw, tcs, PAGE, budget, recent, sinks, limit, None if ref is None else gpu(ref)[0])
    torch.cuda.synchronize()
    k, c, w2, cs = O.evict(bt, ctx, w, caches, budget, recent, sinks, budget if limit is None else limit, ref)
    assert np.array_equal(kept.cpu().numpy(), k), f"{what}: kept"
    assert np.array_equal(tc.cpu().numpy(), c), f"{what}: ctx_len"
    assert np.array_equal(tw.cpu().numpy().view(np.int32), w2.view(np.int32)), f"{what}: weights"
    for i, (got, want) in enumerate(zip(tcs, cs)):
        assert np.array_equal(got.cpu().numpy().view(np.uint8), want.view(np.uint8)), f"{what}: cache {i}"
    assert torch.equal(tb, gpu(bt)[0])
    return kept


@pytest.mark.parametrize("weights", ["spread", "few", "zero", "signed"])
@pytest.mark.parametrize("ctx,HK,D,PAGE,budget,recent,sinks", [
    ([2], 1, 64, 16, 1, 0, 0),                       # the smallest
    ([2], 1, 64, 16, 1, 1, 0),
    ([300, 77, 150], 8, 128, 16, 100, 30, 4),        # one that stays
    ([513, 512, 511], 2, 64, 48, 512, 0, 0),         # one token to drop, none, none
    ([1000], 4, 128, 128, 64, 60, 4),                # nothing to choose
    ([5000, 4097], 2, 64, 16, 1000, 100, 0),         # a chunk of positions and a little more
    ([9000], 1, 64, 32, 4500, 7, 1),                 # more than the registers hold
    ([64, 0, 1], 3, 16, 8, 63, 5, 50),               # rows of three heads, pages of 8
    ([40000, 9000, 100], 1, 16, 64, 8200, 300, 5),   # a table of more tokens than one workgroup selects from
    ([33000, 32768], 2, 16, 16, 32767, 4097, 0),
    ([300000], 1, 16, 128, 70000, 64, 4),            # slices of more than one chunk
])
def test_exact(ctx, HK, D, PAGE, budget, recent, sinks, weights):
    rng = np.random.default_rng(sum(ctx) + budget)
    note(f"evict ctx={ctx} HK={HK} D={D} PAGE={PAGE} budget={budget} recent={recent} sinks={sinks} weights={weights}")
    run_check(make(rng, ctx, HK, D, PAGE, weights), budget, recent, sinks, what="evict")


def test_special_weights():
    """NaN counts as -infinity, -0 as 0; infinities; ties go to the lower position."""
    rng = np.random.default_rng(1)
    case = make(rng, [400, 300], 2, 64, 16, "few")
    w = case[2]
    w[0, 0, ::3], w[0, 0, 1::7], w[0, 1, ::2], w[0, 1, 1::5] = np.nan, -np.inf, np.inf, -0.0
    w[1, 0], w[1, 1, ::2] = np.nan, -np.inf
    for budget in (1, 99, 250, 299):
        note(f"evict special budget={budget}")
        run_check(case, budget, 0, 0, what=f"budget {budget}")


def test_long_rows_special_weights_and_pages():
    """The slices of a long row: ties across them, NaN, a page that is none or shared in one of them."""
    rng = np.random.default_rng(11)
    case = make(rng, [50000, 36000, 45000], 1, 16, 64, "few")
    bt, ctx, w, caches = case
    P = len(caches[0])
    w[0, 0, ::3], w[0, 0, 1::7], w[0, 0, 2::1001] = np.nan, -np.inf, np.inf
    ref = np.bincount(bt[bt >= 0], minlength=P).astype(np.int32)
    ref[bt[1, 400]] = 2
    for budget in (1, 3000, 20000, 35999):
        note(f"evict long special budget={budget}")
        run_check(case, budget, 0, 0, ref=ref, what=f"budget {budget}")
    bt[2, 700] = -1
    note("evict long bad page")
    run_check(case, 30000, 5000, 3, limit=40000, what="bad page")


def test_limit_shared_and_bad_pages():
    """Rows up to the limit stay, and those with a page that is shared, or that is none."""
    rng = np.random.default_rng(2)
    case = make(rng, [300, 200, 150, 260, 260], 2, 64, 16)
    bt, ctx, w, caches = case
    P = len(caches[0])
    bt[4, 3] = bt[3, 3]  # rows 3 and 4 share a page
    ref = np.bincount(bt[bt >= 0], minlength=P).astype(np.int32)
    note("evict limit, shared")
    run_check(case, 100, 10, 2, limit=200, ref=ref, what="limit")
    for bad in (-1, P, 2 ** 31 - 1, -2 ** 31):
        worse = (bt.copy(), ctx, w, caches)
        worse[0][0, 18] = bad
        note(f"evict bad page {bad}")
        run_check(worse, 100, 10, 2, limit=150, ref=ref, what=f"bad page {bad}")
    # A page behind the tokens is not looked at, and a context past the table counts as the table's length.
    bt[0, 19] = -5
    ctx[1] = 10 ** 6
    bt[1, 13:] = -1
    note("evict long context")
    run_check(case, 100, 10, 2, limit=150, ref=ref, what="long")


@pytest.mark.parametrize("dtype,inner", [(torch.float16, (80,)), (torch.uint8, (3,)), (torch.float32, ()), (torch.int16, (5,)),
                                         (torch.uint8, (1,)), (torch.float16, (256,)), (torch.float8_e4m3fn, (2, 8)),
                                         (torch.float32, (513,))])
def test_cache_types_and_views(dtype, inner):
    """Rows of any size and type, one tensor of them in another order of dimensions."""
    rng = np.random.default_rng(3)
    bt, ctx, w, _ = make(rng, [200, 260], 2, 16, 16)
    P = int(bt.max()) + 1
    size = torch.empty(0, dtype=dtype).element_size() * int(np.prod(inner))
    raw = rng.integers(0, 256, (P, 16, 2, size), dtype=np.uint8)
    tb, tc, tw = gpu(bt, ctx, w)
    plain = gpu(raw)[0].view(torch.uint8)
    one = plain.clone().view(dtype).view(P, 16, 2, *inner)
    two = torch.empty((16, 2, P, size), dtype=torch.uint8, device=DEV).permute(2, 0, 1, 3)
    two.copy_(plain)
    note(f"evict rows {dtype} {inner}")
    kept = K.paged_kv_evict(tb, tc, tw, [one, two], 16, 120, 20)
    torch.cuda.synchronize()
    k, _, _, (want,) = O.evict(bt, ctx, w, [raw], 120, 20, 0, 120)
    assert np.array_equal(kept.cpu().numpy(), k)
    assert np.array_equal(one.contiguous().view(torch.uint8).cpu().numpy().reshape(raw.shape), want)
    assert np.array_equal(two.cpu().numpy(), want)


def test_weights_off_a_border_and_given_kept():
    rng = np.random.default_rng(4)
    bt, ctx, w, caches = make(rng, [5000], 2, 64, 16)
    tb, tc, tw = gpu(bt, ctx, w)
    wide = torch.zeros((1, 2, w.shape[2] + 5), device=DEV)
    wide[:, :, 1:1 + w.shape[2]] = tw
    out = torch.full((1, 2, 77), 9, dtype=torch.int32, device=DEV)
    note("evict unaligned weights")
    got = K.paged_kv_evict(tb, tc, wide[:, :, 1:], gpu(*caches), 16, 77, 5, kept=out)
    torch.cuda.synchronize()
    k, _, w2, _ = O.evict(bt, ctx, w, caches, 77, 5, 0, 77)
    assert got is out and np.array_equal(out.cpu().numpy(), k)
    assert np.array_equal(wide[:, :, 1:1 + w.shape[2]].cpu().numpy(), w2) and bool((wide[:, :, 0] == 0).all())


def test_more_pages_than_lds_holds():
    """Pages of one token: the table is read from memory."""
    rng = np.random.default_rng(5)
    note("evict pages of one token")
    run_check(make(rng, [9000], 1, 16, 1), 8900, 10, 0, what="tiny pages")


def test_graph_replays():
    """A captured call, replayed on sequences that have grown again, and on ones that have not."""
    rng = np.random.default_rng(6)
    case = make(rng, [300, 222, 60], 2, 128, 16)
    bt, ctx, w, caches = case
    tb, tc, tw = gpu(bt, ctx, w)
    tcs = gpu(*caches)
    kept = torch.empty((3, 2, 90), dtype=torch.int32, device=DEV)
    call = lambda: K.paged_kv_evict(tb, tc, tw, tcs, 16, 90, 20, 1, kept=kept)  # noqa: E731
    note("evict graph")
    start = [x.clone() for x in (tc, tw, *tcs)]
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ([300, 222, 60], [91, 90, 89], [0, 300, 1], [300, 222, 60]):
        for x, s in zip((tc, tw, *tcs), start):
            x.copy_(s)
        tc.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        g.replay()  # nothing is left to do
        torch.cuda.synchronize()
        k, c, w2, cs = O.evict(bt, np.asarray(lens, np.int32), w, caches, 90, 20, 1, 90)
        assert np.array_equal(tc.cpu().numpy(), c) and np.array_equal(tw.cpu().numpy(), w2)
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(tcs, cs))


def test_large_pool():
    """Rows past 2^31 bytes of a pool."""
    rng = np.random.default_rng(7)
    bt, ctx, w, caches = make(rng, [500], 8, 128, 64)
    P = (1 << 31) // (64 * 8 * 128) + 20
    big = torch.zeros((P, 64, 8, 128), dtype=torch.int8, device=DEV)
    big[-len(caches[0]):] = gpu(caches[0])[0]
    far = bt.copy()
    far[far >= 0] += P - len(caches[0])
    tb, tc, tw = gpu(far, ctx, w)
    note("evict large pool")
    K.paged_kv_evict(tb, tc, tw, [big], 64, 200, 20)
    torch.cuda.synchronize()
    _, _, _, (want, *_) = O.evict(bt, ctx, w, caches, 200, 20, 0, 200)
    assert np.array_equal(big[-len(want):].cpu().numpy(), want)


def test_refusals():
    rng = np.random.default_rng(8)
    bt, ctx, w, caches = make(rng, [40, 30], 2, 64, 16)
    tb, tc, tw = gpu(bt, ctx, w)
    tcs = gpu(*caches)
    before = [x.clone() for x in (tc, tw, *tcs)]
    note("evict refusals")
    good = dict(block_tbl=tb, ctx_len=tc, weights=tw, caches=tcs, PAGE=16, budget=10)
    k = tcs[0]
    for kw in [dict(block_tbl=tb.long()), dict(block_tbl=tb.t()), dict(block_tbl=tb[:0]), dict(ctx_len=tc[:1]),
               dict(ctx_len=tc.long()), dict(weights=tw.double()), dict(weights=tw[:, :, :-1]), dict(weights=tw[:, :1]),
               dict(weights=tw[:1]), dict(weights=tw[:1].expand(2, -1, -1)), dict(weights=tw[0]), dict(weights=tw.cpu()),
               dict(caches=[]), dict(caches=[k[:, :8]]), dict(caches=[k, k]), dict(caches=[k[:, :, :1]]), dict(caches=[k[..., ::2]]),
               dict(caches=[k[:1].expand(len(k), -1, -1, -1)]), dict(caches=[k.clone() for _ in range(17)]),
               dict(caches=[k, tcs[1][1:]]), dict(caches=[k.cpu()]), dict(PAGE=8), dict(PAGE=0), dict(budget=0), dict(recent=11),
               dict(recent=6, sinks=5), dict(recent=-1), dict(sinks=-1), dict(limit=9), dict(ref=tc), dict(ref=tw[0, 0]),
               dict(kept=torch.empty((2, 2, 9), dtype=torch.int32, device=DEV)),
               dict(kept=torch.empty((2, 2, 10), dtype=torch.int64, device=DEV)),
               dict(caches=[torch.zeros((len(k), 16, 2, 4097), dtype=torch.int8, device=DEV)])]:
        with pytest.raises(RuntimeError):
            K.paged_kv_evict(**dict(good, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((tc, tw, *tcs), before))


@pytest.mark.parametrize("weights", ["spread", "few", "zero", "signed"])
@pytest.mark.parametrize("ctx,budget,recent,sinks", [
    ([20000], 9000, 100, 4),           # more than one group of chunks
    ([16385, 32000], 16384, 1, 0),     # the first group and a token; nearly two groups
    ([32768], 30000, 29000, 5),
])
def test_tables_of_several_groups_in_one_workgroup(ctx, budget, recent, sinks, weights):
    """Tables of 16385 to 32768 tokens: more than a workgroup keeps in registers, less than is cut into slices."""
    rng = np.random.default_rng(budget)
    note(f"evict groups ctx={ctx} budget={budget} weights={weights}")
    case = make(rng, ctx, 1, 16, 64, weights)
    bt = case[0][:, :512]  # 32768 tokens at most
    run_check((np.ascontiguousarray(bt), case[1], np.ascontiguousarray(case[2][:, :, :bt.shape[1] * 64]), case[3]), budget, recent, sinks,
              what="groups")


def test_long_rows_of_many_heads():
    """A table of more than 32768 tokens with more rows than leave half of the CUs idle: one workgroup a row."""
    rng = np.random.default_rng(40)
    HK, PAGE, L, budget = 129, 64, 33500, 7001
    C = -(-L // PAGE)
    bt = rng.permutation(C).astype(np.int32)[None]
    w = rng.integers(0, 5000, (1, HK, C * PAGE)).astype(np.float32)
    cache = rng.integers(0, 1 << 31, (C, PAGE, HK)).astype(np.int32)
    tb, tc, tw, tk = gpu(bt, np.asarray([L], np.int32), w, cache)
    note("evict many heads")
    kept = K.paged_kv_evict(tb, tc, tw, [tk], PAGE, budget, 50, 3)
    torch.cuda.synchronize()
    key = w[0, :, :L].copy()
    key[:, :3] = key[:, L - 50:] = np.inf
    want = np.sort(np.argsort(-key, axis=1, kind="stable")[:, :budget], axis=1)
    assert np.array_equal(kept.cpu().numpy()[0], want) and tc.item() == budget
    rows = cache[bt[0]].reshape(C * PAGE, HK)
    got = tk.cpu().numpy()[bt[0]].reshape(C * PAGE, HK)
    assert np.array_equal(got[:budget], np.take_along_axis(rows, want.T, 0)) and np.array_equal(got[budget:], rows[budget:])
    assert np.array_equal(tw.cpu().numpy()[0, :, :budget], np.take_along_axis(w[0], want, 1))
    assert np.array_equal(tw.cpu().numpy()[0, :, budget:], w[0, :, budget:])
