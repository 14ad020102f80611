"""Attention over a block-scaled paged cache on the GPU against float64.

Tolerance, with u = 2^-11 (half a step of fp16): the output is rounded once (u |ref|); every probability
times its V scale is rounded once (u * sum p |v|); scores are summed in fp32 over D terms, which moves a
probability by at most D 2^-24 of the largest sum |q k|, plus a few fp32 steps of the exponent and the
exponential (2^-21), counted twice for numerator and denominator; and fp32 sums (2^-20).  2^-24 covers
subnormal outputs.
"""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import F8, gpu, make_cache, raw
from gpu_util import note
from oracle import cache_ops as C

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -11


def check(out, ref, q_len, n_seqs, D, what):
    exact, spread, big = ref
    got = out.float().cpu().numpy().astype(np.float64)[:n_seqs, :q_len]
    exact, spread = exact[:n_seqs, :q_len], spread[:n_seqs, :q_len]
    eps = 2 * (D * 2.0 ** -24 * big + 2.0 ** -21) + 2.0 ** -20
    bad = ~(np.abs(got - exact) <= U * np.abs(exact) + (U + eps) * spread + 2.0 ** -24)
    assert not bad.any(), f"{what}: {bad.sum()} off, worst {np.abs(got - exact)[bad].max():.3e}"


def queries(rng, B, QL, H, D):
    return rng.standard_normal((B, QL, H, D)).astype(np.float16)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("ctx,q_len,H,H_KV,D,PAGE,SB", [
    ([1], 1, 1, 1, 64, 16, 16),                         # one token
    ([17, 16, 15], 1, 4, 4, 128, 16, 16),               # no head groups, pages just reached and just missed
    ([300, 41, 9, 130], 9, 32, 8, 128, 16, 16),         # verification: 36 rows
    ([700, 33, 5], 5, 16, 2, 64, 32, 16),               # groups of 8, two blocks to a page
    ([513, 64], 3, 12, 3, 128, 48, 48),                 # groups of 4, pages of three sub-tiles
    ([1000, 128, 127], 2, 8, 1, 128, 128, 64),          # one K/V head
    ([2, 0, 1, 700], 4, 8, 2, 64, 64, 32),              # fewer tokens than queries, and none at all
    ([90], 40, 6, 2, 128, 16, 16),                      # more rows than one program holds
])
def test_matches_float64(ctx, q_len, H, H_KV, D, PAGE, SB, fmt):
    rng = np.random.default_rng(len(ctx) * 1000 + q_len + D)
    cache = make_cache(rng, ctx, H_KV, D, PAGE, SB, fmt)
    q = queries(rng, len(ctx), q_len, H, D)
    ref = C.attention_block(q, *cache, q_len, fmt)
    note(f"block attn {fmt} ctx={ctx} q_len={q_len} H={H}/{H_KV} D={D} PAGE={PAGE} SB={SB}")
    out, ck = K.paged_attention_block_scaled(*gpu(q, *cache), q_len)
    torch.cuda.synchronize()
    check(out, ref, q_len, len(ctx), D, "default")
    assert ck.n_regs > 0 and ("true>" if fmt == "fp8" else "false>") in ck.name
    for b, n in enumerate(ctx):  # rows that see nothing
        assert bool((out[b, :max(0, q_len - n)] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_long_context_many_splits(fmt):
    rng = np.random.default_rng(5)
    ctx, q_len, H, H_KV, D = [20011, 9000], 2, 8, 2, 128
    cache = make_cache(rng, ctx, H_KV, D, 64, 32, fmt)
    q = queries(rng, 2, q_len, H, D)
    ref = C.attention_block(q, *cache, q_len, fmt)
    note(f"block attn long {fmt}")
    t = gpu(q, *cache)
    out, _ = K.paged_attention_block_scaled(*t, q_len)
    one, _ = K.paged_attention_block_scaled(*t, q_len, QPP=1)
    torch.cuda.synchronize()
    check(out, ref, q_len, 2, D, "long")
    assert torch.equal(out, one)


@pytest.mark.parametrize("q_len,QPPs", [(9, (1, 4, 9, 16)), (16, (5, 8, 16))])
def test_programs_agree_bit_for_bit(q_len, QPPs):
    rng = np.random.default_rng(q_len)
    ctx = [900, 77, 30]
    cache = make_cache(rng, ctx, 8, 128, 16, 16, "fp8")
    t = gpu(queries(rng, 3, q_len, 32, 128), *cache)
    note(f"block attn QPP {QPPs}")
    outs = [K.paged_attention_block_scaled(*t, q_len, QPP=n)[0] for n in QPPs]
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_scales_of_any_size(fmt):
    """V scales from 2^-30 to 2^8 in one split, K scales that make one block dominate, and zero scales."""
    rng = np.random.default_rng(8)
    ctx, q_len, H, H_KV, D = [600, 600, 96], 3, 4, 2, 64
    kc, vc, ks, vs, bt, cl = make_cache(rng, ctx, H_KV, D, 16, 16, fmt)
    vs[:] = np.exp2(rng.integers(-30, 9, vs.shape)).astype(np.float32) * rng.uniform(1, 2, vs.shape).astype(np.float32)
    vs[bt[1, :38]] = np.float32(2.0 ** -30)    # a whole sequence of tiny scales
    vs[bt[2, 2]] = 0
    ks[bt[0, 7]] *= 4
    vs[vs > 140] = 140                         # 448 * 140 and 127 * 140 stay inside fp16
    q = queries(rng, 3, q_len, H, D)
    ref = C.attention_block(q, kc, vc, ks, vs, bt, cl, q_len, fmt)
    note(f"block attn scales {fmt}")
    out, _ = K.paged_attention_block_scaled(*gpu(q, kc, vc, ks, vs, bt, cl), q_len)
    torch.cuda.synchronize()
    check(out, ref, q_len, 3, D, "scales")


def test_pages_outside_the_pool_are_masked():
    rng = np.random.default_rng(9)
    ctx, q_len = [400, 200, 48], 3
    kc, vc, ks, vs, bt, cl = make_cache(rng, ctx, 2, 128, 16, 16, "fp8")
    for b, c, bad in ((0, 3, kc.shape[0]), (0, 20, -1), (0, 24, 2 ** 31 - 1), (1, 12, -7)):
        bt[b, c] = bad
    bt[2, :] = -1  # a row with no page at all
    q = queries(rng, 3, q_len, 8, 128)
    ref = C.attention_block(q, kc, vc, ks, vs, bt, cl, q_len, "fp8")
    note("block attn bad pages")
    out, _ = K.paged_attention_block_scaled(*gpu(q, kc, vc, ks, vs, bt, cl), q_len)
    torch.cuda.synchronize()
    check(out, ref, q_len, 3, 128, "bad pages")
    assert bool((out[2] == 0).all())


@pytest.mark.parametrize("H,H_KV,q_len", [(8, 2, 4), (32, 8, 9), (16, 2, 8)])
def test_what_is_masked_does_not_reach_a_row(H, H_KV, q_len):
    """NaN codes and infinite or NaN scales behind the context, on pages no row names, and in tokens that some
    rows see and others do not."""
    rng = np.random.default_rng(q_len)
    D, PAGE, SB = 128, 32, 16
    ctx = [150, 39]
    kc, vc, ks, vs, bt, cl = make_cache(rng, ctx, H_KV, D, PAGE, SB, "fp8")
    q = queries(rng, 2, q_len, H, D)
    clean = C.attention_block(q, kc, vc, ks, vs, bt, cl, q_len, "fp8")
    for b, n in enumerate(ctx):  # slots behind the context, and the blocks that hold none of its tokens
        pg, at = bt[b, n // PAGE], n % PAGE
        kc[pg, at:], vc[pg, at:] = 0x7F, 0xFF
        blk = -(-at // SB)
        ks[pg, blk:], vs[pg, blk:] = np.inf, np.nan
    named = set(bt[bt >= 0].tolist())
    for pg in set(range(len(kc))) - named:
        kc[pg], vc[pg], ks[pg], vs[pg] = 0x7F, 0x7F, np.nan, np.inf
    note(f"block attn masked NaN H={H} q_len={q_len}")
    out, _ = K.paged_attention_block_scaled(*gpu(q, kc, vc, ks, vs, bt, cl), q_len)
    torch.cuda.synchronize()
    check(out, clean, q_len, 2, D, "behind the context")
    # The last token's V holds a NaN at one place, its K is clean: the last row has a NaN there and nowhere else.
    n, hd = ctx[0], 1
    pg, at = bt[0, (n - 1) // PAGE], (n - 1) % PAGE
    vc[pg, at, hd, 37] = 0x7F
    out, _ = K.paged_attention_block_scaled(*gpu(q, kc, vc, ks, vs, bt, cl), q_len)
    torch.cuda.synchronize()
    got = out.float().cpu().numpy()
    G = H // H_KV
    expect = np.zeros(got.shape, bool)
    expect[0, q_len - 1, hd * G:(hd + 1) * G, 37] = True
    assert np.array_equal(np.isnan(got), expect)
    keep = torch.from_numpy(np.where(expect, 0, got))
    check(keep, (np.where(expect, 0, clean[0]), clean[1], clean[2]), q_len, 2, D, "a NaN some rows see")
    # A NaN K code: every row that sees the token is NaN, the others are as before.
    vc[pg, at, hd, 37] = 0
    kc[pg, at, hd, 5] = 0x7F
    out, _ = K.paged_attention_block_scaled(*gpu(q, kc, vc, ks, vs, bt, cl), q_len)
    torch.cuda.synchronize()
    got = np.isnan(out.float().cpu().numpy())
    expect[:] = False
    expect[0, q_len - 1, hd * G:(hd + 1) * G] = True
    assert np.array_equal(got, expect)


def test_queries_infinite_or_nan_stay_in_their_row():
    rng = np.random.default_rng(3)
    cache = make_cache(rng, [200], 2, 64, 16, 16, "int8")
    q = queries(rng, 1, 3, 8, 64)
    ref = C.attention_block(q, *cache, 3, "int8")
    q[0, 1, 2, 5] = np.nan
    note("block attn NaN query")
    out, _ = K.paged_attention_block_scaled(*gpu(q, *cache), 3)
    torch.cuda.synchronize()
    got = out.float().cpu().numpy()
    assert np.isnan(got[0, 1, 2]).all()
    got[0, 1, 2] = ref[0][0, 1, 2]
    check(torch.from_numpy(got), ref, 3, 1, 64, "other rows")


def test_strides_and_views():
    """q inside a fused projection, caches as one layer of a [pages, layers, ...] pool, a wider table, an output view."""
    rng = np.random.default_rng(4)
    B, ql, H, HK, D, PAGE, SB = 2, 5, 8, 2, 128, 32, 16
    kc, vc, ks, vs, bt, cl = make_cache(rng, [333, 60], HK, D, PAGE, SB, "int8")
    q = queries(rng, B, ql, H, D)
    ref = C.attention_block(q, kc, vc, ks, vs, bt, cl, ql, "int8")
    tq, tk, tv, tks, tvs, tbt, tcl = gpu(q, kc, vc, ks, vs, bt, cl)
    fused = torch.zeros((B, ql, H + 2 * HK, D), dtype=torch.float16, device=DEV)
    fused[:, :, :H] = tq
    pool = lambda t: torch.stack([torch.full_like(t, 7), t], 1)[:, 1]  # noqa: E731
    wide = torch.full((B, bt.shape[1] + 9), -1, dtype=torch.int32, device=DEV)
    wide[:, :bt.shape[1]] = tbt
    big = torch.full((B, ql + 1, H + 1, D), 9.0, dtype=torch.float16, device=DEV)
    note("block attn strides")
    K.paged_attention_block_scaled(fused[:, :, :H], pool(tk), pool(tv), pool(tks), pool(tvs), wide[:, :bt.shape[1]],
                                   tcl, ql, out=big[:, :ql, :H])
    torch.cuda.synchronize()
    check(big[:, :ql, :H], ref, ql, B, D, "strided")
    assert bool((big[:, ql:] == 9).all()) and bool((big[:, :, H:] == 9).all())


def test_cache_past_32_bit_offsets():
    """A pool of 5 GiB a tensor whose table names its first and last pages."""
    rng = np.random.default_rng(6)
    HK, D, PAGE, SB, P = 8, 128, 64, 32, 81920
    ctx, ql, H = [500], 2, 16
    kc, vc, ks, vs, bt, cl = make_cache(rng, ctx, HK, D, PAGE, SB, "int8", spare=0)
    n = len(kc)
    ids = np.concatenate([np.arange(n // 2), np.arange(P - (n - n // 2), P)]).astype(np.int32)
    q = queries(rng, 1, ql, H, D)
    ref = C.attention_block(q, kc, vc, ks, vs, bt, cl, ql, "int8")
    note("block attn 5 GiB pool")
    tq, tk, tv, tks, tvs, tbt, tcl, tid = gpu(q, kc, vc, ks, vs, bt, cl, ids)
    pool = [torch.zeros((P, *t.shape[1:]), dtype=t.dtype, device=DEV) for t in (tk, tv, tks, tvs)]
    for p, t in zip(pool, (tk, tv, tks, tvs)):
        p[tid.long()] = t
    table = torch.where(tbt >= 0, tid[tbt.clamp(min=0).long()], -1)
    out, _ = K.paged_attention_block_scaled(tq, *pool, table, tcl, ql)
    torch.cuda.synchronize()
    check(out, ref, ql, 1, D, "far pages")


def test_plan_mode_equals_eager_and_leaves_the_rest():
    rng = np.random.default_rng(12)
    BM, QM, H, HK, D = 5, 9, 32, 8, 128
    ctx = [300, 41, 129, 16, 777]
    cache = gpu(*make_cache(rng, ctx, HK, D, 16, 16, "fp8"))
    q = gpu(queries(rng, BM, QM, H, D))[0]
    plan = torch.zeros(8, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    call = lambda: K.paged_attention_block_scaled(q, *cache, plan=plan[1:], out=out)  # noqa: E731
    plan[1], plan[2] = BM, QM
    note("block attn plan graph")
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for n, ql in ((5, 9), (1, 3), (3, 1), (0, 4), (4, 0), (2, 9), (5, 5)):
        plan[1], plan[2] = n, ql
        out.fill_(7)
        g.replay()
        eager = torch.full_like(q, 7)
        if n and ql:
            K.paged_attention_block_scaled(q[:n], *cache[:4], cache[4][:n], cache[5][:n], ql, out=eager[:n])
        torch.cuda.synchronize()
        assert torch.equal(out, eager), (n, ql)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("ctx,q_len,QM,H,H_KV,D", [
    ([5000, 63], 1, 4, 40, 8, 128),      # merged by a launch: one row block, captured for two
    ([5000, 5000], 1, 8, 8, 2, 128),     # ... for two
    ([3000, 2000], 3, 16, 32, 8, 64),    # ... for four
    ([4096, 300], 9, 20, 32, 8, 128),    # three of four, two programs
    ([5000, 2100], 1, 1, 16, 16, 128),   # eight splits an eager call merges in place and the graph does not
    ([4100, 1000], 2, 5, 16, 16, 64),
])
def test_plan_mode_of_many_splits(ctx, q_len, QM, H, H_KV, D, fmt):
    rng = np.random.default_rng(sum(ctx) + QM)
    cache = make_cache(rng, ctx, H_KV, D, 64, 64, fmt)
    q = queries(rng, len(ctx), q_len, H, D)
    ref = C.attention_block(q, *cache, q_len, fmt)
    q, *cache = gpu(q, *cache)
    eager = K.paged_attention_block_scaled(q, *cache, q_len)[0]
    note(f"block attn plan of many splits {fmt} ctx={ctx} q_len={q_len} QM={QM}")
    grid = torch.full((len(ctx), QM, H, D), 3, dtype=torch.float16, device=DEV)
    grid[:, :q_len] = q
    out = torch.full_like(grid, 7)
    plan = torch.tensor([len(ctx), q_len], dtype=torch.int32, device=DEV)
    K.paged_attention_block_scaled(grid, *cache, plan=plan, out=out)
    torch.cuda.synchronize()
    check(out, ref, q_len, len(ctx), D, "plan")
    assert torch.equal(out[:, :q_len], eager) and bool((out[:, q_len:] == 7).all())
    plan[0] = 1
    K.paged_attention_block_scaled(grid, *cache, plan=plan, out=out)
    one = K.paged_attention_block_scaled(q[:1], *cache[:4], cache[4][:1], cache[5][:1], q_len)[0]
    assert torch.equal(out[:1, :q_len], one) and torch.equal(out[1:, :q_len], eager[1:])


def test_more_programs_than_counters():
    """1100 sequences of 64 heads: 70400 programs, two splits each; a few of them long, on the same pages."""
    rng = np.random.default_rng(8)
    B, H, D, PAGE = 1100, 64, 64, 16
    kc, vc, ks, vs, row, _ = make_cache(rng, [9000], H, D, PAGE, 16, "int8", spare=0)
    ctx = np.full(B, 20, np.int32)
    ctx[[0, 700, 1099]] = 9000, 8193, 8500
    bt = np.full((B, 1024), -1, np.int32)  # 16384 tokens
    bt[:, :row.shape[1]] = row
    q = queries(rng, B, 1, H, D)
    note("block attn more programs than counters")
    out = K.paged_attention_block_scaled(*gpu(q, kc, vc, ks, vs, bt, ctx), 1)[0]
    torch.cuda.synchronize()
    some = [0, 1, 350, 700, 1098, 1099]
    ref = C.attention_block(q[some], kc, vc, ks, vs, bt[some], ctx[some], 1, "int8")
    check(out[some], ref, 1, len(some), D, "many programs")


def test_workspace_is_what_the_splits_in_flight_need():
    from specq import _lib
    size = lambda B, ql, plan, cols=256: _lib.lib().specq_paged_attn_block_workspace_size(  # noqa: E731
        B, 32, 8, ql, max(1, min(ql, 16)), 128, cols, 16, plan)
    assert size(64, 2048, 0) == 0  # prompt chunks that fill the GPU are not split
    for B, ql, cols in ((1, 1, 64), (8, 9, 256), (32, 256, 8192), (64, 2048, 1024)):
        graph = size(B, ql, 1, cols)
        assert graph <= 256 * 1024 + 256 + 2 * 16 * max(256, B * 8) * max(1, ql // 16) * 64 * 130 * 4
        for b in {1, B // 2 or 1, B}:
            for q in {1, ql // 2 or 1, ql}:
                if min(q, 16) == min(ql, 16):
                    assert size(b, q, 0, cols) <= graph, (B, ql, cols, b, q)


def test_streams_with_their_own_workspaces():
    from specq.workspace import Workspace
    rng = np.random.default_rng(14)
    sets = []
    for i in range(2):
        ctx = [6000 + i, 300]
        cache = make_cache(rng, ctx, 2, 128, 16, 16, "int8")
        q = queries(rng, 2, 3, 8, 128)
        sets.append((gpu(q, *cache), C.attention_block(q, *cache, 3, "int8"), torch.cuda.Stream(), Workspace(DEV)))
    note("block attn two streams")
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(3):
        for i, (t, _, st, ws) in enumerate(sets):
            with torch.cuda.stream(st):
                outs[i].append(K.paged_attention_block_scaled(*t, 3, workspace=ws)[0])
    torch.cuda.synchronize()
    for i, (_, ref, _, _) in enumerate(sets):
        for o in outs[i]:
            check(o, ref, 3, 2, 128, f"stream {i}")


def test_lengths_out_of_range():
    """Negative contexts see nothing, ones past the table end with it; the splits' counters are back at zero."""
    rng = np.random.default_rng(15)
    H, HK, D, ql = 8, 2, 128, 5
    kc, vc, ks, vs, bt, _ = make_cache(rng, [2048, 2048, 700, 2048, 1], HK, D, 16, 16, "int8")
    bt = bt[:, :128]  # 2048 tokens
    q = queries(rng, 5, ql, H, D)
    note("block attn lengths out of range")
    for given, counted in (([-2 ** 31, 2048, -3, 2 ** 31 - 1, 4], [0, 2048, 0, 2048, 4]),
                           ([2048, -2 ** 31 + 7, 700, 2050, -1], [2048, 0, 700, 2048, 0])):
        cache = (kc, vc, ks, vs, bt)
        ref = C.attention_block(q, *cache, np.asarray(counted, np.int32), ql, "int8")
        out = K.paged_attention_block_scaled(*gpu(q, *cache, np.asarray(given, np.int32)), ql)[0]
        torch.cuda.synchronize()
        check(out, ref, ql, 5, D, given)


@pytest.mark.parametrize("D,fmt", [(64, "int8"), (64, "fp8"), (128, "int8"), (128, "fp8")])
def test_even_programs_of_many_tokens(D, fmt):
    """More tokens than a program holds, with every number of row blocks, masked chunks first and last."""
    rng = np.random.default_rng(D)
    for q_len, ctx in ((17, [900, 17, 3]), (33, [515, 40, 33]), (49, [300, 1024, 60])):
        cache = make_cache(rng, ctx, 2, D, 16, 16, fmt)
        q = queries(rng, len(ctx), q_len, 8, D)
        note(f"block attn even programs {fmt} D={D} q_len={q_len}")
        t = gpu(q, *cache)
        out = K.paged_attention_block_scaled(*t, q_len)[0]
        check(out, C.attention_block(q, *cache, q_len, fmt), q_len, len(ctx), D, q_len)
        for QPP in (1, 8, 12, 16):
            assert torch.equal(out, K.paged_attention_block_scaled(*t, q_len, QPP=QPP)[0]), (q_len, QPP)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("q_len,ctx,H,H_KV,D,PAGE,SB", [
    (1030, [1030], 8, 2, 128, 16, 16),           # a whole prompt: no token before it, programs of 64 rows
    (515, [1500, 515, 600], 6, 2, 128, 48, 16),  # ... of 63 rows, behind cached tokens and without
    (700, [4000, 20], 4, 4, 64, 64, 32),         # one sequence shorter than its new tokens: its first rows are empty
])
def test_whole_prompts(q_len, ctx, H, H_KV, D, PAGE, SB, fmt):
    rng = np.random.default_rng(q_len + D)
    cache = make_cache(rng, ctx, H_KV, D, PAGE, SB, fmt)
    q = queries(rng, len(ctx), q_len, H, D)
    note(f"block attn whole prompts {fmt} q_len={q_len} ctx={ctx}")
    t = gpu(q, *cache)
    out = K.paged_attention_block_scaled(*t, q_len)[0]
    torch.cuda.synchronize()
    check(out, C.attention_block(q, *cache, q_len, fmt), q_len, len(ctx), D, q_len)
    plan = torch.tensor([len(ctx), q_len], dtype=torch.int32, device=DEV)
    assert torch.equal(out, K.paged_attention_block_scaled(*t, plan=plan)[0])


def test_refusals():
    rng = np.random.default_rng(1)
    q, kc, vc, ks, vs, bt, cl = gpu(queries(rng, 2, 4, 8, 128), *make_cache(rng, [40, 20], 2, 128, 32, 16, "int8"))
    f = K.paged_attention_block_scaled
    note("block attn refusals")
    bad = [
        (q.float(), kc, vc, ks, vs, bt, cl), (q, kc.view(torch.uint8), vc, ks, vs, bt, cl),
        (q, kc, vc.view(F8), ks, vs, bt, cl), (q, kc, vc, ks.half(), vs.half(), bt, cl),
        (q, kc, vc, ks[:, :, :1], vs[:, :, :1], bt, cl), (q, kc, vc, ks[:-1], vs[:-1], bt, cl),
        (q, kc, vc, ks.repeat(1, 2, 1), vs.repeat(1, 2, 1), bt, cl),  # blocks of 8 tokens
        (q, kc, vc, ks, vs, bt.long(), cl), (q, kc, vc, ks, vs, bt[:1], cl), (q, kc, vc, ks, vs, bt, cl[:1]),
        (q[:, :, :7], kc, vc, ks, vs, bt, cl), (q, kc[..., :64], vc[..., :64], ks, vs, bt, cl),
        (q, kc, vc, ks, vs, bt, cl.cpu()), (q.cpu(), kc, vc, ks, vs, bt, cl),
    ]
    for args in bad:
        with pytest.raises(RuntimeError):
            f(*args, 4)
    for kw in (dict(q_len=5), dict(q_len=-1), dict(n_seqs=3), dict(QPP=0), dict(QPP=17), dict(out=q[:1]),
               dict(plan=torch.zeros(1, dtype=torch.int32, device=DEV))):
        with pytest.raises(RuntimeError):
            f(q, kc, vc, ks, vs, bt, cl, **kw)
    q96 = torch.zeros((2, 4, 8, 96), dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="head_dim"):
        f(q96, kc[..., :96].contiguous(), vc[..., :96].contiguous(), ks, vs, bt, cl)
    assert np.array_equal(raw(f(q, kc, vc, ks, vs, bt, cl, 0)[0]), np.zeros((2, 4, 8, 128), np.float16))
