"""Gathered attention weights on the GPU against float64.

Tolerance: a score is a sum of D exact products, accumulated in fp32 (at most D roundings), times its scale, times
sm_scale log2 e (three more): off by at most e = (D + 4) 2^-24 A, A the sum of its terms' sizes, in units of ln, and so is
the row's log-sum; the exponent's subtraction and the log-sum's own rounding add 2^-23 of values up to A + ln(tokens), the
exponentials and the logarithm 2^-22 each, and the row's sum, in pieces of at most 64 and their joins, 2^-17.  A
probability is so within p (2 e + 2 * 2^-23 (A + 12) + 2^-16) and the sum over the rows, with the weight there was, adds
2^-20 of itself (at most 16 additions in a row of lanes' order for the rows here).  2^-126 is the smallest power exp2
gives.
"""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import gpu
from gpu_util import note
from oracle import batch_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(rng, ctx, QL, H, HK, D, PAGE, f32, cols=None):
    pages = [max(0, -(-c // PAGE)) for c in ctx]
    P, C = sum(pages) + 3, cols or max(max(pages), 1) + 1
    bt = np.full((len(ctx), C), -1, np.int32)
    perm, at = rng.permutation(P).astype(np.int32), 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[at:at + n]
        at += n
    kc = rng.integers(-127, 128, (P, PAGE, HK, D), dtype=np.int8)
    ks = (rng.uniform(0.5, 1.5, (P, PAGE, HK)) / 64).astype(np.float32 if f32 else np.float16)
    q = rng.standard_normal((len(ctx), QL, H, D)).astype(np.float16)
    w = rng.uniform(0, 2, (len(ctx), HK, C * PAGE)).astype(np.float32)
    return q, kc, ks, bt, np.asarray(ctx, np.int32), w


def check(got, case, q_lens, sm, what):
    q, kc, ks, bt, ctx, w = case
    ref, spread = O.attn_weights(q, kc, ks, bt, ctx, w, q_lens, sm)
    D = q.shape[-1]
    fresh = np.zeros(w.shape, bool)
    gained = ref.copy()
    for b, ql in enumerate(q_lens):
        L = min(max(int(ctx[b]), 0), bt.shape[1] * kc.shape[1])
        fresh[b, :, max(L - ql, 0):L] = ql > 0
    gained -= np.where(fresh, 0, w.astype(np.float64))
    tol = spread * (2 * (D + 4) * 2.0 ** -24 + 2 * 2.0 ** -23) + gained * (2 * 12 * 2.0 ** -23 + 2.0 ** -16) + \
        2.0 ** -20 * ref + 2.0 ** -126
    g = got.double().cpu().numpy()
    err = np.abs(g - ref)
    assert np.isfinite(g).all(), f"{what}: not finite"
    assert (err <= tol).all(), f"{what}: worst {err.max():.3e} at {np.unravel_index((err - tol).argmax(), err.shape)}"
    for b in range(len(ctx)):  # what lies behind a sequence stays, bit for bit
        L = min(max(int(ctx[b]), 0), bt.shape[1] * kc.shape[1]) if b < len(q_lens) and q_lens[b] else 0
        assert np.array_equal(got[b, :, L:].cpu().numpy(), w[b, :, L:]), f"{what}: behind sequence {b}"


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("ctx,QL,H,HK,D,PAGE", [
    ([1], 1, 1, 1, 64, 16),                       # one token that sees itself
    ([300, 77], 1, 32, 8, 128, 16),
    ([513, 9, 256, 257], 9, 8, 2, 128, 32),       # tiles that end at, before and behind a border
    ([2000], 4, 16, 4, 64, 48),                   # 16 rows: the most that are stored
    ([700, 40], 5, 8, 2, 64, 64),                 # 20 rows: computed again
    ([5000], 3, 8, 1, 128, 128),                  # 24 rows of one head, 20 tiles
    ([400, 90], 90, 8, 2, 128, 16),               # a prompt chunk of 23 row blocks; a whole prompt
    ([600], 600, 2, 1, 64, 16),                   # more row blocks than are joined at a time
    ([900, 620], 610, 4, 1, 128, 64),             # rows of several segments, for one sequence nearly a prompt
    ([1100], 1100, 8, 1, 64, 16),                 # and of several pairs of launches
    ([333, 1000], 150, 8, 2, 64, 16),             # ... whose first seen ones lie anywhere among them
    ([291, 180, 777], 177, 12, 4, 128, 48),
    ([0, 3, 20], 7, 4, 4, 128, 16),               # an empty sequence, one of fewer tokens than are new
])
def test_matches_float64(ctx, QL, H, HK, D, PAGE, f32):
    rng = np.random.default_rng(sum(ctx) + QL)
    case = make(rng, ctx, QL, H, HK, D, PAGE, f32)
    note(f"attn_weights ctx={ctx} QL={QL} H={H}/{HK} D={D} PAGE={PAGE} f32={f32}")
    t = gpu(*case)
    got = K.paged_attention_weights(*t)
    torch.cuda.synchronize()
    assert got is t[5]
    check(got, case, [QL] * len(ctx), D ** -0.5, "weights")
    # Twice the same: the sums have one order.
    again = gpu(case[5])[0]
    K.paged_attention_weights(*t[:5], again)
    torch.cuda.synchronize()
    assert torch.equal(got, again)


@pytest.mark.parametrize("QL,G", [(3, 2), (9, 4)])
def test_accepted_drafts_bad_pages_and_long_contexts(QL, G):
    """q_lens of none, some and all drafts (and past q_len); table ids outside the pool; a context past the table."""
    rng = np.random.default_rng(5)
    HK, D, PAGE = 2, 128, 16
    ctx = [300, 280, 200, 33]
    case = make(rng, ctx, QL, G * HK, HK, D, PAGE, False)
    q, kc, ks, bt, cl, w = case
    bt[0, [0, 5, 18]] = -1, 2 ** 31 - 1, len(kc)
    bt[3, :] = -7  # a sequence on no page at all
    case[4][1] = bt.shape[1] * PAGE + 1000  # its table's length counts
    bt[1, 18:] = bt[1, 0]
    lens = np.asarray([2, QL, 0, QL + 5], np.int32)
    note(f"attn_weights q_lens QL={QL} G={G}")
    t = gpu(*case)
    K.paged_attention_weights(*t, q_lens=gpu(lens)[0], sm_scale=0.05)
    torch.cuda.synchronize()
    check(t[5], case, [2, QL, 0, QL], 0.05, "q_lens")


def test_masked_places_do_not_count():
    """NaN scales of tokens past the context on pages in use, and infinite ones, reach nothing."""
    rng = np.random.default_rng(6)
    for QL in (1, 9):
        case = make(rng, [40, 100], QL, 8, 2, 64, 32, True)
        q, kc, ks, bt, cl, w = case
        for b, n in enumerate(cl):
            page, at = bt[b, n // 32], n % 32
            ks[page, at:] = np.nan
            ks[page, at + 1:] = np.inf
        note(f"attn_weights masked QL={QL}")
        t = gpu(*case)
        K.paged_attention_weights(*t)
        torch.cuda.synchronize()
        ks[~np.isfinite(ks)] = 0
        check(t[5], case, [QL, QL], 64 ** -0.5, "masked")


def test_large_scores():
    """Scores of hundreds: one token takes a row's weight, others underflow."""
    rng = np.random.default_rng(7)
    case = make(rng, [500, 300], 2, 4, 2, 128, 16, True)
    case = (case[0] * np.float16(20), *case[1:])
    note("attn_weights large scores")
    t = gpu(*case)
    K.paged_attention_weights(*t)
    torch.cuda.synchronize()
    check(t[5], case, [2, 2], 128 ** -0.5, "large")


def test_views_and_alignment():
    """q out of a fused projection, a cache with heads ahead of tokens, weights off a 16-byte border and of more tokens
    than the table holds."""
    rng = np.random.default_rng(8)
    B, QL, H, HK, D, PAGE = 2, 3, 8, 2, 128, 16
    case = make(rng, [200, 331], QL, H, HK, D, PAGE, False)
    q, kc, ks, bt, cl, w = case
    note("attn_weights views")
    tq, tk, ts, tb, tc, tw = gpu(*case)
    fused = torch.zeros((B, QL, H + 2 * HK, D), dtype=torch.float16, device=DEV)
    fused[:, :, :H] = tq
    k2 = torch.empty((len(kc), HK, PAGE, D), dtype=torch.int8, device=DEV).transpose(1, 2)
    k2.copy_(tk)
    s2 = torch.empty((len(kc), HK, PAGE), dtype=torch.float16, device=DEV).transpose(1, 2)
    s2.copy_(ts)
    wide = torch.zeros((B, HK, w.shape[2] + 7), device=DEV)
    w2 = wide[:, :, 3:3 + w.shape[2]]
    w2.copy_(tw)
    K.paged_attention_weights(fused[:, :, :H], k2, s2, tb, tc, w2)
    K.paged_attention_weights(tq, tk, ts, tb, tc, tw)
    torch.cuda.synchronize()
    assert torch.equal(w2, tw)
    assert bool((wide[:, :, :3] == 0).all()) and bool((wide[:, :, 3 + w.shape[2]:] == 0).all())
    check(tw, case, [QL] * B, D ** -0.5, "views")


def test_cache_past_32_bit_offsets():
    """A pool of more than 2^31 bytes: pages at its end."""
    HK, D, PAGE = 8, 128, 64
    P = (1 << 31) // (PAGE * HK * D) + 40
    rng = np.random.default_rng(9)
    case = make(rng, [150], 2, 8, HK, D, PAGE, True)
    q, kc, ks, bt, cl, w = case
    note("attn_weights large pool")
    big = torch.zeros((P, PAGE, HK, D), dtype=torch.int8, device=DEV)
    bigs = torch.zeros((P, PAGE, HK), device=DEV)
    far = bt.copy()
    far[far >= 0] += P - len(kc)
    big[-len(kc):], bigs[-len(kc):] = gpu(kc)[0], gpu(ks)[0]
    tq, tb, tc, tw = gpu(q, far, cl, w)
    K.paged_attention_weights(tq, big, bigs, tb, tc, tw)
    torch.cuda.synchronize()
    check(tw, case, [2], D ** -0.5, "far")


def test_plan_graph_equals_eager_and_leaves_the_rest():
    """One graph over (4, 9) replays every active size with the eager call's bits: from few rows, whose scores an eager
    call stores, to many.  Eager work of the same workspace runs between the replays."""
    rng = np.random.default_rng(10)
    B, QL, H, HK, D, PAGE = 4, 9, 16, 4, 128, 16
    case = make(rng, [700, 31, 300, 64], QL, H, HK, D, PAGE, False)
    tq, tk, ts, tb, tc, tw = gpu(*case)
    plan = torch.tensor([B, QL], dtype=torch.int32, device=DEV)
    work = tw.clone()
    call = lambda: K.paged_attention_weights(tq, tk, ts, tb, tc, work, plan=plan)  # noqa: E731
    note("attn_weights plan graph")
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for n, ql in ((4, 9), (1, 1), (3, 4), (2, 5), (0, 4), (4, 0), (4, 9)):
        plan.copy_(torch.tensor([n, ql], dtype=torch.int32))
        work.copy_(tw)
        g.replay()
        want = tw.clone()
        K.paged_attention_weights(tq, tk, ts, tb, tc, want, q_len=ql, n_seqs=n)
        torch.cuda.synchronize()
        assert torch.equal(work, want), f"plan {n} {ql}"
        assert torch.equal(work[n:], tw[n:])
        check(want, case, [ql if b < n else 0 for b in range(B)], D ** -0.5, f"{n} {ql}")


def test_two_streams_with_a_workspace_each():
    from specq.workspace import Workspace
    rng = np.random.default_rng(11)
    cases = [make(rng, [900, 33], 2, 8, 2, 64, 16, True), make(rng, [100, 1300], 9, 8, 2, 64, 16, True)]
    note("attn_weights streams")
    ts = [gpu(*c) for c in cases]
    torch.cuda.synchronize()
    streams, spaces = [torch.cuda.Stream() for _ in cases], [Workspace("cuda") for _ in cases]
    want = [t[5].clone() for t in ts]
    for _ in range(3):
        for t, s, ws in zip(ts, streams, spaces):
            with torch.cuda.stream(s):
                K.paged_attention_weights(*t, workspace=ws)
    torch.cuda.synchronize()
    for t, w in zip(ts, want):
        for _ in range(3):
            K.paged_attention_weights(*t[:5], w)
    torch.cuda.synchronize()
    assert all(torch.equal(t[5], w) for t, w in zip(ts, want))


def test_shared_pages_gather_for_each_row():
    """Rows that share pages (a fork) have weights of their own."""
    rng = np.random.default_rng(12)
    case = make(rng, [200, 200], 1, 4, 2, 64, 16, False)
    case[3][1] = case[3][0]
    note("attn_weights shared pages")
    t = gpu(*case)
    K.paged_attention_weights(*t)
    torch.cuda.synchronize()
    check(t[5], case, [1, 1], 64 ** -0.5, "shared")


def test_empty_and_refusals():
    rng = np.random.default_rng(13)
    case = make(rng, [40, 30], 2, 4, 2, 64, 16, False)
    t = gpu(*case)
    q, kc, ks, bt, cl, w = t
    before = w.clone()
    note("attn_weights refusals")
    K.paged_attention_weights(*t, q_len=0)
    K.paged_attention_weights(*t, n_seqs=0)
    K.paged_attention_weights(q[:0], kc, ks, bt[:0], cl[:0], w[:0])
    torch.cuda.synchronize()
    assert torch.equal(w, before)
    bad = lambda i, x: [x if j == i else y for j, y in enumerate(t)]  # noqa: E731
    for args, kw in [(bad(0, q.float()), {}), (bad(0, q[..., :32]), {}), (bad(0, q[:, :, :3]), {}), (bad(0, q[0]), {}),
                     (bad(1, kc.half()), {}), (bad(1, kc[:, :, :, ::2]), {}), (bad(2, ks[:, :, :1]), {}), (bad(2, ks.double()), {}),
                     (bad(3, bt.long()), {}), (bad(3, bt[:1]), {}), (bad(3, bt.t()), {}), (bad(4, cl.long()), {}),
                     (bad(4, cl[:1]), {}), (bad(5, w.half()), {}), (bad(5, w[:, :, :-1]), {}), (bad(5, w[:, :1]), {}),
                     (bad(5, w[:1]), {}), (bad(5, w[:1].expand(2, -1, -1)), {}), (bad(5, w[:, :1].expand(-1, 2, -1)), {}),
                     (bad(5, w.cpu()), {}), (t, dict(q_len=3)), (t, dict(n_seqs=3)), (t, dict(q_lens=cl[:1])),
                     (t, dict(q_lens=cl.long())), (t, dict(plan=cl.long())), (t, dict(plan=cl[:1]))]:
        with pytest.raises(RuntimeError):
            K.paged_attention_weights(*args, **kw)
    assert torch.equal(w, before)


@pytest.mark.parametrize("QL,G,ctx", [(4, 4, 700), (9, 4, 700), (300, 2, 700), (700, 2, 700)])
def test_a_nan_row_shares_nothing_out_to_tokens_it_does_not_see(QL, G, ctx):
    """16, 36, 600 and 1400 rows: stored scores, scores formed twice, in one pass of the queries and in segments."""
    rng = np.random.default_rng(23)
    q, kc, ks, bt, cl, w = make(rng, [ctx], QL, 2 * G, 2, 64, 16, True)
    bad, i = q.copy(), QL // 2 - 1
    bad[0, i, 1] = np.nan  # a head of the first group
    got = [K.paged_attention_weights(*gpu(x, kc, ks, bt, cl, w)).cpu().numpy() for x in (q, bad)]
    sees = ctx - QL + i + 1
    assert np.isnan(got[1][0, 0, :sees]).sum() == sees
    assert (got[1][0, 0, sees:] != got[0][0, 0, sees:]).sum() == 0
    assert (got[1][0, 1] != got[0][0, 1]).sum() == 0


@pytest.mark.parametrize("QL,H,HK,D", [(150, 8, 1, 128), (300, 8, 1, 64), (40, 8, 2, 128), (700, 4, 2, 128),
                                       (1100, 8, 1, 64), (68, 8, 1, 128)])
def test_the_table_size_does_not_change_a_bit(QL, H, HK, D):
    """A table of many more columns, and a plan-mode call of more tokens and sequences, split the rows otherwise."""
    rng = np.random.default_rng(QL)
    q, kc, ks, bt, cl, w = make(rng, [QL + 200, QL], QL, H, HK, D, 16, False)
    note(f"attn_weights table size QL={QL}")
    want = K.paged_attention_weights(*gpu(q, kc, ks, bt, cl, w))
    wide = np.full((5, 9000), -1, np.int32)
    wide[:2, :bt.shape[1]] = bt
    more = np.zeros((5, HK, 9000 * 16), np.float32)
    more[:2, :, :w.shape[2]] = w
    got = K.paged_attention_weights(*gpu(q, kc, ks, wide[:2], cl, more[:2]))
    assert torch.equal(got[:, :, :w.shape[2]], want) and not got[:, :, w.shape[2]:].any()
    q5, cl5 = np.zeros((5, QL + 500, H, D), np.float16), np.zeros(5, np.int32)
    q5[:2, :QL], cl5[:2] = q, cl
    plan = torch.tensor([2, QL], dtype=torch.int32, device=DEV)
    got = K.paged_attention_weights(*gpu(q5, kc, ks, wide, cl5, more), plan=plan)
    assert torch.equal(got[:2, :, :w.shape[2]], want) and not got[2:].any()


@pytest.mark.parametrize("QL,G", [(1, 4), (3, 5), (9, 8), (40, 3)])
def test_rows_add_up_to_one_whatever_their_scores(QL, G):
    """Scores of some 16000 that differ by a few: 4 rows (stored), 15, 72 and 120.  A score is rounded, but alike in the row's sum
    and in its probabilities, so a row adds up to 1: within the exponentials (2^-23 each) of both passes and of four joins, at
    most 60 additions of the row's sum (2^-24 each) and 40 over the rows, and the reciprocal, in all (6 * 2 + 101) 2^-24 < 2^-17."""
    rng = np.random.default_rng(QL)
    HK, D, PAGE, ctx = 8, 64, 16, [3000, 700]
    q, kc, ks, bt, cl, w = make(rng, ctx, QL, HK * G, HK, D, PAGE, True)
    kc[..., :32], ks[:] = 127, 1.0
    q[..., :32], q[..., 32:] = 8, 0.01 * q[..., 32:]
    w[:] = 0
    note(f"attn_weights sums QL={QL} G={G}")
    got = K.paged_attention_weights(*gpu(q, kc, ks, bt, cl, w), sm_scale=0.5)
    torch.cuda.synchronize()
    got = got.double().cpu().numpy()
    for b, n in enumerate(ctx):
        total = got[b, :, :n].sum(-1) / (QL * G)
        assert (got[b, :, :n] > 0).sum() > HK * 100  # the rows are spread out
        assert (np.abs(total - 1) < 2.0 ** -17).all(), f"sequence {b}: off by {np.abs(total - 1).max():.2e}"


@pytest.mark.parametrize("QL,G,PAGE", [(1, 4, 64), (3, 8, 16)])
def test_batches_whose_workgroups_walk_several_tiles(QL, G, PAGE):
    """17 sequences of 8 heads, tables of 12 tiles: two blocks of eight sequences and one more, three tiles a workgroup; stored
    scores and a tile's worth of rows formed twice."""
    rng = np.random.default_rng(31)
    ctx = [3000, 1, 255, 256, 257, 512, 513, 2999, 0, 768, 1025, 2048, 1537, 100, 2900, 1793, 2305]
    case = make(rng, ctx, QL, 8 * G, 8, 64, PAGE, False)
    lens = np.asarray([QL] * 7 + [0] + [QL] * 9, np.int32)
    case[3][4, 0] = case[3][11, 2048 // PAGE - 1] = -1
    note(f"attn_weights many tiles QL={QL} G={G}")
    t = gpu(*case)
    K.paged_attention_weights(*t, q_lens=gpu(lens)[0])
    torch.cuda.synchronize()
    check(t[5], case, lens.tolist(), 64 ** -0.5, "tiles")
    # A sequence by itself, a tile a workgroup, has the same bits.
    for b in (0, 4, 11, 14):
        one = gpu(case[0][b:b + 1], case[1], case[2], case[3][b:b + 1], case[4][b:b + 1], case[5][b:b + 1])
        K.paged_attention_weights(*one)
        torch.cuda.synchronize()
        assert torch.equal(one[5][0], t[5][b])


@pytest.mark.parametrize("QL,G", [(40, 4), (180, 4), (600, 4)])
def test_many_rows_of_some_drafts_bad_pages_and_masked_scales(QL, G):
    """160, 720 and 2400 rows: q_lens of none, one, one segment's worth, and all; pages that are none on and off the rows'
    diagonal; a context past its table; NaN and infinite scales behind the contexts."""
    rng = np.random.default_rng(QL)
    HK, D, PAGE = 2, 64, 16
    ctx = [QL + 300, QL + 35, QL + 1, 700, QL // 2]
    case = make(rng, ctx, QL, G * HK, HK, D, PAGE, True)
    q, kc, ks, bt, cl, w = case
    lens = [QL, min(QL, 1024 // G), 0, 1, QL]  # the last has more new tokens than it is long
    for b, n in enumerate(ctx):
        if n % PAGE:
            ks[bt[b, n // PAGE], n % PAGE:] = np.nan
            ks[bt[b, n // PAGE], n % PAGE + 1:] = np.inf
    bt[0, [0, 7, 300 // PAGE + 1, (300 + QL // 2) // PAGE]] = -1, 2 ** 31 - 1, len(kc), -9
    cl[3] = bt.shape[1] * PAGE + 50  # its table's length counts
    bt[3, 40:] = -1
    note(f"attn_weights many rows QL={QL}")
    t = gpu(*case)
    K.paged_attention_weights(*t, q_lens=gpu(np.asarray(lens, np.int32))[0], sm_scale=0.1)
    torch.cuda.synchronize()
    ks[~np.isfinite(ks)] = 0
    check(t[5], case, lens, 0.1, "many rows")
    # In plan mode, with room for more tokens and sequences, the same bits.
    more = np.zeros((7, QL + 70, *q.shape[2:]), np.float16)
    more[:5, :QL] = q
    pad = lambda a, v: np.concatenate((a, np.full((2, *a.shape[1:]), v, a.dtype)))  # noqa: E731
    plan = torch.tensor([5, QL], dtype=torch.int32, device=DEV)
    p = gpu(more, kc, ks, pad(bt, 0), pad(cl, 90), pad(w, 1.5))
    K.paged_attention_weights(*p, q_lens=gpu(np.asarray([*lens, 3, 3], np.int32))[0], sm_scale=0.1, plan=plan)
    torch.cuda.synchronize()
    assert torch.equal(p[5][:5], t[5]) and bool((p[5][5:] == 1.5).all())


@pytest.mark.parametrize("B,QL,G,ctx", [
    (7, 4, 4, [900, 3, 2000, 0, 300, 1, 1200]),          # stored: 64 MiB of scores a sequence
    (150, 8, 8, [700, 5, 300]),                          # 64 rows: 2 MiB of statistics a sequence
    (9, 260, 4, [600, 260, 1500, 300, 0, 100, 333]),     # 1040 rows, 32 MiB a sequence and segment
])
def test_batches_that_are_taken_in_turns(B, QL, G, ctx):
    """Tables of 131072 columns' tokens: not all sequences' scores, statistics and sums find room at once."""
    rng = np.random.default_rng(B)
    HK, D, PAGE, wide = 8, 64, 16, 8192
    ctx = (ctx * B)[:B]
    q, kc, ks, bt, cl, w = make(rng, ctx, QL, HK * G, HK, D, PAGE, False)
    tq, tk, ts, tb, tc, tw = gpu(q, kc, ks, bt, cl, w)
    lens = gpu(rng.integers(0, QL + 1, B).astype(np.int32))[0]
    cols, T = bt.shape[1], w.shape[2]
    wbt = torch.full((B, wide), -1, dtype=torch.int32, device=DEV)
    wbt[:, :cols] = tb
    note(f"attn_weights turns B={B} QL={QL}")
    for plan in (None, (B, QL), (B - 1, QL - 1), (1, QL)):
        ww = torch.zeros((B, HK, wide * PAGE), device=DEV)
        ww[:, :, :T] = tw
        want = tw.clone()
        if plan is None:
            K.paged_attention_weights(tq, tk, ts, wbt, tc, ww, q_lens=lens)
            K.paged_attention_weights(tq, tk, ts, tb, tc, want, q_lens=lens)
        else:
            K.paged_attention_weights(tq, tk, ts, wbt, tc, ww, plan=torch.tensor(plan, dtype=torch.int32, device=DEV))
            K.paged_attention_weights(tq, tk, ts, tb, tc, want, n_seqs=plan[0], q_len=plan[1])
        torch.cuda.synchronize()
        assert torch.equal(ww[:, :, :T], want), f"plan {plan}"
        assert not ww[:, :, T:].any()


@pytest.mark.parametrize("QL,G", [(1, 2), (9, 2), (40, 2)])
def test_more_items_than_workgroups(QL, G):
    """300 sequences of 8 heads: workgroups come back for more, up to the longest sequence.  In parts, the same bits."""
    rng = np.random.default_rng(77)
    B, HK, D, PAGE = 300, 8, 64, 16
    ctx = rng.integers(0, 300, B)
    ctx[[3, 120, 121, 299]] = 1900, 1300, 1800, 2000
    case = make(rng, ctx.tolist(), QL, G * HK, HK, D, PAGE, False)
    lens = rng.integers(0, QL + 1, B).astype(np.int32)
    lens[[3, 299]] = QL
    note(f"attn_weights many items QL={QL}")
    tq, tk, ts, tb, tc, tw = gpu(*case)
    tl = gpu(lens)[0]
    parts = tw.clone()
    K.paged_attention_weights(tq, tk, ts, tb, tc, tw, q_lens=tl)
    for b in range(0, B, 20):
        at = slice(b, b + 20)
        K.paged_attention_weights(tq[at], tk, ts, tb[at], tc[at], parts[at], q_lens=tl[at])
    torch.cuda.synchronize()
    assert torch.equal(tw, parts)
    for at in (slice(0, 8), slice(118, 124), slice(295, 300)):
        check(tw[at], (case[0][at], case[1], case[2], case[3][at], case[4][at], case[5][at]), lens[at].tolist(), D ** -0.5, f"{at}")


@pytest.mark.parametrize("QL", [1, 9, 40])
def test_scores_that_are_infinite(QL):
    """A scale of infinity: tokens of score -inf get nothing from a row, one of +inf makes NaN of what the row sees."""
    rng = np.random.default_rng(51)
    q, kc, ks, bt, cl, w = make(rng, [200], QL, 4, 2, 64, 16, True)
    q, w = np.abs(q) + np.float16(0.25), np.zeros_like(w)
    page, slot = bt[0, 3], 5  # token 53, seen by every row
    kc[page, slot, 0], kc[page, slot, 1], ks[page, slot] = -1, 1, np.inf
    note(f"attn_weights infinite QL={QL}")
    got = K.paged_attention_weights(*gpu(q, kc, ks, bt, cl, w)).cpu().numpy()[0]
    assert got[0, 53] == 0 and np.isfinite(got[0]).all()
    assert abs(got[0, :200].astype(np.float64).sum() - 2 * QL) < 2.0 ** -16 * 2 * QL
    first = 200 - QL + 1  # what the first new token sees
    assert np.isnan(got[1, :first]).all() and not got[:, 200:].any()
