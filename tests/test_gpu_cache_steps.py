"""The steps of a verification loop over a block-scaled cache run together, as a serving loop would: reserve pages,
turn q and k, append, attend, roll back to the accepted tokens; then fork the sequences, go on with the samples,
and compact the pool.  Every step is held to the plain implementations fed with what the device held before it."""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import F8, gpu, raw
from gpu_util import note
from oracle import cache_ops as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_a_serving_loop(fmt):
    rng = np.random.default_rng(21)
    B, H, HK, D, PAGE, SB, P, cols = 4, 8, 2, 128, 32, 16, 64, 12
    dt = torch.int8 if fmt == "int8" else F8
    kc, vc = (torch.zeros((P, PAGE, HK, D), dtype=torch.uint8, device=DEV).view(dt) for _ in "kv")
    ks, vs = (torch.zeros((P, PAGE // SB, HK), device=DEV) for _ in "kv")
    tbl = torch.full((B, cols), -1, dtype=torch.int32, device=DEV)
    ref = torch.zeros(P, dtype=torch.int32, device=DEV)
    f, m = K.rotary_inv_freq(64, scaling="yarn", factor=4.0, device=DEV)
    ctx = np.zeros(B, np.int32)
    t_np, r_np = raw(tbl).copy(), raw(ref).copy()
    note(f"serving loop {fmt}")

    def step(ql, accept):
        nonlocal ctx, t_np, r_np
        ctx = (ctx + ql).astype(np.int32)
        cl = gpu(ctx)[0]
        new = gpu(rng.standard_normal((B, ql, H + 2 * HK, D)).astype(np.float16))[0]
        q, k, v = new[:, :, :H], new[:, :, H:H + HK], new[:, :, H + HK:]
        q0, k0, v0 = (raw(x).copy() for x in (q, k, v))
        before = [raw(x).copy() for x in (kc, vc, ks, vs)]
        short = K.paged_kv_reserve(tbl, ref, cl, PAGE)
        K.rotary_embed(q, k, f, cl, mscale=m, q_out=q, k_out=k)
        K.paged_kv_append_block_scaled(k, v, kc, vc, ks, vs, tbl, cl)
        out, _ = K.paged_attention_block_scaled(q, kc, vc, ks, vs, tbl, cl)
        torch.cuda.synchronize()
        t_np, r_np, s = C.reserve(t_np, r_np, ctx, PAGE)
        assert int(short) == s == 0 and np.array_equal(raw(tbl), t_np) and np.array_equal(raw(ref), r_np)
        pos = ctx[:, None] - ql + np.arange(ql)[None]
        for got, x in ((q, q0), (k, k0)):
            want = C.rotary(x, f.cpu().numpy(), pos, False, m)
            assert np.abs(raw(got) - want).max() <= 2.0 ** -11 * np.abs(want).max() + 1e-5
        assert np.array_equal(raw(v), v0)
        want = C.append_block(raw(k), raw(v), *before, t_np, ctx, ql, fmt)
        for a, b in zip((kc, vc), want[:2]):
            assert np.array_equal(C.decode(raw(a), fmt), C.decode(b, fmt), equal_nan=True)
        for a, b in zip((ks, vs), want[2:]):
            assert np.array_equal(raw(a), b)
        attend(q, out, ql)
        ctx = (ctx - ql + np.asarray(accept)).astype(np.int32)
        K.paged_kv_free(tbl, ref, gpu(ctx)[0], PAGE)
        t_np, r_np = C.free(t_np, r_np, ctx, PAGE)
        torch.cuda.synchronize()
        assert np.array_equal(raw(tbl), t_np) and np.array_equal(raw(ref), r_np)

    def attend(q, out, ql):
        exact, spread, big = C.attention_block(raw(q), *(raw(x) for x in (kc, vc, ks, vs)), t_np, ctx, ql, fmt)
        tol = 2.0 ** -11 * np.abs(exact) + (2.0 ** -11 + 2 * D * 2.0 ** -24 * big + 2.0 ** -19) * spread + 2.0 ** -24
        assert (np.abs(out.double().cpu().numpy() - exact) <= tol).all()

    step(70, [70, 45, 33, 64])
    for _ in range(3):
        step(9, rng.integers(1, 10, B))
    # Rows 1 and 3 become samples of rows 0 and 2.
    lens, parent = gpu(ctx.copy(), np.asarray([0, 0, 2, 2], np.int32))
    K.paged_kv_fork(tbl, ref, lens, parent, [kc, vc, ks, vs], PAGE)
    t_np, r_np, ctx, s, _ = C.fork(t_np, r_np, ctx, raw(parent), PAGE)
    torch.cuda.synchronize()
    assert s == 0 and np.array_equal(raw(tbl), t_np) and np.array_equal(raw(ref), r_np) and np.array_equal(raw(lens), ctx)
    for _ in range(2):
        step(5, rng.integers(1, 6, B))  # the samples differ from here: their last pages are their own
    # Row 0 leaves; the pool is compacted; what the others see does not change.
    q = gpu(rng.standard_normal((B, 1, H, D)).astype(np.float16))[0]
    keep = ctx.copy()
    keep[0] = 0
    K.paged_kv_free(tbl, ref, gpu(keep)[0], PAGE)
    ctx = keep
    one = K.paged_attention_block_scaled(q, kc, vc, ks, vs, tbl, gpu(ctx)[0])[0]
    K.paged_kv_compact(tbl, ref, [kc, vc, ks, vs])
    two = K.paged_attention_block_scaled(q, kc, vc, ks, vs, tbl, gpu(ctx)[0])[0]
    torch.cuda.synchronize()
    assert torch.equal(one, two) and bool((one[0] == 0).all())
    n = int((ref > 0).sum())
    assert bool((ref[:n] > 0).all()) and int(tbl.max()) == n - 1
    t_np, r_np = raw(tbl).copy(), raw(ref).copy()
    step(3, [1, 2, 3, 1])
