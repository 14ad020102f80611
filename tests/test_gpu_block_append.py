"""Append to a block-scaled paged cache on the GPU against the format's definition, bit for bit, and the values
it stands for against the inputs in 64 bits (half a step of the code, and fp32 rounding of the quotient)."""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import gpu, make_cache, raw
from gpu_util import note
from oracle import cache_ops as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


def new_kv(rng, B, QL, H, D, size=2.0):
    return [(rng.standard_normal((B, QL, H, D)) * size).astype(np.float16) for _ in "kv"]


def same(got, ref, fmt, what):
    for name, g, r in zip(("kc", "vc", "ks", "vs"), got, ref):
        g = raw(g)
        if name in ("kc", "vc") and fmt == "fp8":  # +0 and -0 are one value
            g, r = (np.where(a == 128, 0, a) for a in (g, r))
        bad = np.argwhere(g.view(np.int32 if g.dtype == np.float32 else g.dtype) !=
                          r.view(np.int32 if r.dtype == np.float32 else r.dtype))
        assert len(bad) == 0, f"{what}: {name} differs at {len(bad)} places, first {tuple(bad[0])}"


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("ctx,q_len,H,D,PAGE,SB", [
    ([1], 1, 1, 64, 16, 16),
    ([17, 16, 300, 33], 1, 8, 128, 16, 16),        # a block's first slot, its last, and between
    ([300, 41, 9, 130], 9, 8, 128, 16, 16),
    ([64, 65, 100], 20, 3, 256, 48, 48),
    ([700, 128, 129], 100, 2, 128, 128, 32),       # several blocks at once
    ([260, 77], 70, 2, 64, 128, 128),              # one block a page
    ([600, 512], 500, 1, 256, 512, 512),           # blocks too large for registers
    ([3, 0, 5, 40], 5, 2, 64, 32, 16),             # fewer tokens in all than new ones: the first are skipped
])
def test_bit_exact(ctx, q_len, H, D, PAGE, SB, fmt):
    rng = np.random.default_rng(q_len * 7 + D)
    cache = make_cache(rng, ctx, H, D, PAGE, SB, fmt, lo=0.2, hi=3.0)
    k, v = new_kv(rng, len(ctx), q_len, H, D)
    ref = C.append_block(k, v, *cache, q_len, fmt)
    note(f"block append {fmt} ctx={ctx} q_len={q_len} D={D} PAGE={PAGE} SB={SB}")
    t = gpu(k, v, *cache)
    K.paged_kv_append_block_scaled(*t, q_len)
    torch.cuda.synchronize()
    same(t[2:6], ref, fmt, "append")
    # The new tokens' values, in 64 bits: half a step of the code's grid.
    bt, sb = cache[4], SB
    for x, cd, sc in ((k, raw(t[2]), raw(t[4])), (v, raw(t[3]), raw(t[5]))):
        for b, n in enumerate(ctx):
            for i in range(max(0, q_len - n), q_len):
                pos = n - q_len + i
                pg, at = bt[b, pos // PAGE], pos % PAGE
                s = sc[pg, at // sb].astype(np.float64)[:, None]
                got, want = C.decode(cd[pg, at], fmt) * s, x[b, i].astype(np.float64)
                half = s / 2 if fmt == "int8" else np.maximum(np.abs(want) * 2.0 ** -4, s * 2.0 ** -10)
                assert (np.abs(got - want) <= half * (1 + 2.0 ** -15)).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_token_by_token_scale_grows(fmt):
    """Forty appends of one token each, larger and larger: every step requantises the block so far."""
    rng = np.random.default_rng(2)
    H, D, PAGE, SB = 2, 128, 32, 32
    cache = make_cache(rng, [40], H, D, PAGE, SB, fmt)
    ref, t = cache[:4], gpu(*cache)
    note(f"block append growing {fmt}")
    for n in range(1, 41):
        k, v = new_kv(rng, 1, 1, H, D, size=0.1 * n)
        cl = np.asarray([n], np.int32)
        ref = C.append_block(k, v, *ref, cache[4], cl, 1, fmt)
        K.paged_kv_append_block_scaled(*gpu(k, v), *t[:5], *gpu(cl), 1)
    torch.cuda.synchronize()
    same(t[:4], ref, fmt, "growing")


def test_rolled_back_tokens_are_written_over():
    """Drafts are appended, three of nine kept, nine more appended behind them."""
    rng = np.random.default_rng(3)
    cache = make_cache(rng, [60, 33], 4, 64, 16, 16, "int8")
    ref, t = cache[:4], gpu(*cache)
    note("block append roll back")
    for ctx in ([40, 20], [34, 14], [43, 23]):
        k, v = new_kv(rng, 2, 9, 4, 64)
        cl = np.asarray(ctx, np.int32)
        ref = C.append_block(k, v, *ref, cache[4], cl, 9, "int8")
        K.paged_kv_append_block_scaled(*gpu(k, v), *t[:5], *gpu(cl), 9)
    torch.cuda.synchronize()
    same(t[:4], ref, "int8", "roll back")


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_infinities_and_nan(fmt):
    rng = np.random.default_rng(4)
    cache = make_cache(rng, [20], 2, 64, 16, 16, fmt)
    k, v = new_kv(rng, 1, 6, 2, 64)
    k[0, 1, 0, 3], k[0, 1, 0, 4], v[0, 5, 1, 0], v[0, 2] = np.inf, np.nan, -np.inf, np.nan
    ref = C.append_block(k, v, *cache, 6, fmt)
    note(f"block append inf/nan {fmt}")
    t = gpu(k, v, *cache)
    K.paged_kv_append_block_scaled(*t, 6)
    torch.cuda.synchronize()
    same(t[2:6], ref, fmt, "inf")
    assert all(np.isfinite(raw(x)).all() for x in t[4:6])


def test_pages_outside_the_pool_and_table_are_skipped():
    rng = np.random.default_rng(5)
    kc, vc, ks, vs, bt, cl = make_cache(rng, [50, 60, 70], 2, 128, 16, 16, "fp8")
    bt[0, 2], bt[1, 3] = -1, len(kc)
    cl[2] = 16 * bt.shape[1] + 4  # tokens past the table
    k, v = new_kv(rng, 3, 30, 2, 128)
    ref = C.append_block(k, v, kc, vc, ks, vs, bt, cl, 30, "fp8")
    note("block append bad pages")
    t = gpu(k, v, kc, vc, ks, vs, bt, cl)
    K.paged_kv_append_block_scaled(*t, 30)
    torch.cuda.synchronize()
    same(t[2:6], ref, "fp8", "bad pages")
    for far in (2 ** 31 - 1, -2 ** 31):  # nothing to write, nothing read out of range
        K.paged_kv_append_block_scaled(*t[:7], torch.full((3,), far, dtype=torch.int32, device=DEV), 30)
    torch.cuda.synchronize()
    same(t[2:6], ref, "fp8", "far lengths")


def test_views_and_plan_graph():
    """K and V inside a fused projection, one layer of a pool, and a captured plan-mode call replayed."""
    rng = np.random.default_rng(6)
    B, QL, H, D, PAGE, SB = 4, 9, 2, 128, 32, 16
    full = [300, 41, 129, 77]
    cache = make_cache(rng, full, H, D, PAGE, SB, "int8")
    k, v = new_kv(rng, B, QL, H, D)
    tk, tv = gpu(k, v)
    fused = torch.cat([torch.zeros_like(tk), tk, tv], 2)
    kn, vn = fused[:, :, H:2 * H], fused[:, :, 2 * H:]
    start = gpu(*cache[:4])
    pools = [torch.stack([x, torch.full_like(x, 3)], 1) for x in start]
    t = [p[:, 0] for p in pools]
    bt, cl = gpu(cache[4], cache[5])
    plan = torch.tensor([B, QL], dtype=torch.int32, device=DEV)
    note("block append plan graph")
    K.paged_kv_append_block_scaled(kn, vn, *t, bt, cl, plan=plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.paged_kv_append_block_scaled(kn, vn, *t, bt, cl, plan=plan)
    for n, ql in ((4, 9), (2, 4), (1, 1), (0, 5), (3, 0)):
        for x, s in zip(t, start):
            x.copy_(s)
        ctx = np.asarray([c - (QL - ql) for c in full], np.int32)
        cl.copy_(gpu(ctx)[0])
        plan.copy_(torch.tensor([n, ql], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        same(t, C.append_block(k, v, *cache[:4], cache[4], ctx, ql, "int8", n_seqs=n), "int8", f"plan {n} {ql}")
    assert all(bool((p[:, 1] == 3).all()) for p in pools)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_every_small_and_negative_zero(fmt):
    """Zeros of both signs, subnormals, and every value next to them, below amax from one subnormal to the largest."""
    bits = np.concatenate([np.arange(0, 1024), np.arange(1024, 0x7C00, 37)]).astype(np.uint16)
    bits = np.concatenate([bits, bits | 0x8000])
    rows = -(-len(bits) // 64)
    x = np.zeros(rows * 64, np.uint16)
    x[:len(bits)] = bits
    x = np.random.default_rng(3).permutation(x).view(np.float16).reshape(rows, 64)
    for top in (0.0, 6e-8, 6e-5, 0.37, 65504.0):
        new = np.where(np.abs(x) <= np.float16(top), x, np.copysign(np.float16(0), x))
        new = np.stack([new, -new])[:, None, :, None, :]
        pages = -(-rows // 16)
        kc, vc, ks, vs, bt, ctx = make_cache(np.random.default_rng(1), [rows], 1, 64, 16, 16, fmt)
        note(f"block append zeros {fmt} {top}")
        t = gpu(new[0], new[1], kc, vc, ks, vs, bt, ctx)
        K.paged_kv_append_block_scaled(*t, rows)
        torch.cuda.synchronize()
        want = C.append_block(new[0], new[1], kc, vc, ks, vs, bt, ctx, rows, fmt)
        assert (bt[0] >= 0).sum() == pages
        for got, w in zip(t[2:6], want):
            assert np.array_equal(raw(got), w), top


def test_nan_codes_of_earlier_tokens_stay_nan():
    """A NaN among a block's earlier e4m3 codes is NaN over the grown scale too, whatever its sign; its neighbours are
    requantised as ever, and where the scale stays the codes do."""
    rng = np.random.default_rng(22)
    for size, D, SB in ((40.0, 128, 16), (1e-3, 128, 16), (40.0, 256, 512)):  # grows, stays; a block read twice
        ctx, ql = [SB - 3, 2 * SB - 1], 4
        kc, vc, ks, vs, bt, cl = make_cache(rng, ctx, 2, D, SB, SB, "fp8")
        kc[:, ::5, 0, 3], kc[:, 1::7, 1, 60], vc[:, ::3, :, 9] = 0x7F, 0xFF, 0x7F
        k, v = new_kv(rng, 2, ql, 2, D, size=size)
        ref = C.append_block(k, v, kc, vc, ks, vs, bt, cl, ql, "fp8")
        note(f"block append NaN codes size={size} SB={SB}")
        t = gpu(k, v, kc, vc, ks, vs, bt, cl)
        K.paged_kv_append_block_scaled(*t, ql)
        torch.cuda.synchronize()
        for got, want in zip(t[2:4], ref[:2]):
            assert np.array_equal(C.decode(raw(got), "fp8"), C.decode(want, "fp8"), equal_nan=True)
        assert all(np.array_equal(raw(a), b) for a, b in zip(t[4:6], ref[2:]))
        assert (np.isnan(C.decode(ref[0], "fp8")) == np.isnan(C.decode(kc, "fp8")))[bt[0, 0], :SB - 3 - ql].all()


def test_negative_lengths_write_nothing():
    rng = np.random.default_rng(21)
    kc, vc, ks, vs, bt, _ = make_cache(rng, [64, 64, 64], 2, 64, 16, 16, "int8")
    new = rng.standard_normal((2, 3, 4, 2, 64)).astype(np.float16)
    t = gpu(kc, vc, ks, vs, bt)
    note("block append negative lengths")
    K.paged_kv_append_block_scaled(*gpu(new[0], new[1]), *t, *gpu(np.asarray([-2 ** 31, -1, 0], np.int32)), 4)
    torch.cuda.synchronize()
    for got, was in zip(t, (kc, vc, ks, vs)):
        assert np.array_equal(raw(got), was)


def test_refusals():
    rng = np.random.default_rng(1)
    k, v, kc, vc, ks, vs, bt, cl = gpu(*new_kv(rng, 2, 4, 2, 128), *make_cache(rng, [40, 20], 2, 128, 32, 16, "int8"))
    f = K.paged_kv_append_block_scaled
    note("block append refusals")
    for args in [(k.float(), v.float(), kc, vc, ks, vs, bt, cl), (k, v[:, :3], kc, vc, ks, vs, bt, cl),
                 (k, v, kc.view(torch.uint8), vc, ks, vs, bt, cl), (k, v, kc, vc, ks.double(), vs.double(), bt, cl),
                 (k, v, kc, vc, ks.repeat(1, 2, 1), vs.repeat(1, 2, 1), bt, cl), (k, v, kc, vc, ks, vs, bt[:1], cl),
                 (k, v, kc, vc, ks, vs, bt, cl[:1]), (k[..., :64], v[..., :64], kc, vc, ks, vs, bt, cl),
                 (k, v, kc, vc, ks, vs, bt, cl.cpu())]:
        with pytest.raises(RuntimeError):
            f(*args, 4)
    for kw in (dict(q_len=5), dict(n_seqs=-1), dict(n_seqs=3)):
        with pytest.raises(RuntimeError):
            f(k, v, kc, vc, ks, vs, bt, cl, **kw)
    f(k, v, kc, vc, ks, vs, bt, cl, 0)
    f(k, v, kc, vc, ks, vs, bt, cl, 4, n_seqs=0)
    torch.cuda.synchronize()
