"""Head norms with rotary positions on the GPU against float64.

Tolerance for a pair (a, b) of normalised values turned with factor m: one rounding to fp16 (2^-11 of the result, 2^-25
below its normal range); the sine and cosine within 4e-7 and three fp32 operations (2^-22), as for rotary_embed; and the
normalised values within 2^-19: the squares' sum takes at most 16 additions in a lane and 6 between lanes (22 * 2^-24,
halved by the root), the mean, eps, the root and two products add at most 6 * 2^-24: 17 * 2^-24 < 2^-19.
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


def rand16(rng, *shape, size=1.0):
    return (size * rng.standard_normal(shape)).astype(np.float16)


def check(got, x, weight, eps, inv_freq, pos, interleaved, m, what):
    ref = O.qk_norm_rotary(x, weight, eps, inv_freq, pos, interleaved, m)
    a = np.abs(O.qk_norm(x, weight, eps))
    R = 2 * len(inv_freq)
    size = a.copy()
    i0, i1 = (np.arange(0, R, 2), np.arange(1, R, 2)) if interleaved else (np.arange(R // 2), np.arange(R // 2, R))
    size[..., i0] = size[..., i1] = m * (a[..., i0] + a[..., i1])
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + size * (4e-7 + 2.0 ** -22 + 2.0 ** -19)
    assert (err <= tol).all(), f"{what}: worst {err.max():.3e} at {np.unravel_index((err - tol).argmax(), err.shape)}"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,QL,H,H_KV,D,R,wtype", [
    (1, 1, 32, 8, 128, 128, "f16"),
    (3, 17, 12, 3, 80, 20, "f16"),        # pairs that no vector holds whole
    (2, 700, 4, 1, 64, 32, "f32"),        # more than 1024 tokens: a wave each
    (5, 9, 8, 8, 96, 96, "heads"),        # a row of weights for each head
    (2, 3, 5, 2, 192, 64, "none"),
    (1, 2, 1, 1, 2, 2, "f32"),            # the smallest head
    (2, 2, 3, 1, 510, 6, "heads"),        # rows that are not 16-byte aligned
    (1, 5, 2, 2, 512, 512, "f16"),        # the largest head
    (2, 2, 3, 2, 512, 16, "f32"),         # ... hardly turned: 63 units of 64 lanes
    (1, 3, 9, 4, 256, 128, "f16"),
    (1, 2, 2, 1, 400, 390, "none"),       # more items than lanes in the unaligned form
    (1, 4, 3, 1, 16, 16, "f16"),          # a lane or two for a row
])
def test_matches_float64(B, QL, H, H_KV, D, R, wtype, interleaved):
    rng = np.random.default_rng(B * 100 + QL + D)
    q, k = rand16(rng, B, QL, H, D, size=3.0), rand16(rng, B, QL, H_KV, D, size=0.2)
    q[0, 0, 0] = 0  # a row of zeros
    k[-1, -1, -1] = np.where(np.arange(D) % 2, 65504, -65504)  # the largest values
    make = lambda h: {"none": None, "heads": rng.uniform(0.5, 1.5, (h, D)).astype(np.float16),  # noqa: E731
                      "f32": rng.uniform(-1.5, 1.5, D).astype(np.float32),
                      "f16": rng.uniform(0.5, 1.5, D).astype(np.float16)}[wtype]
    wq, wk = make(H), make(H_KV)
    f, _ = K.rotary_inv_freq(R, device="cpu")
    ctx = rng.integers(QL, 100000 + QL, B).astype(np.int32)
    pos = ctx[:, None] - QL + np.arange(QL)[None]
    note(f"qk_norm B={B} QL={QL} H={H}/{H_KV} D={D} R={R} weights={wtype} interleaved={interleaved}")
    tq, tk, tc = gpu(q, k, ctx)
    tw = [None if w is None else gpu(w)[0] for w in (wq, wk)]
    kw = dict(interleaved=interleaved, mscale=1.25, eps=1e-5)
    qo, ko = K.qk_norm_rotary(tq, tk, *tw, f.to(DEV), tc, **kw)
    torch.cuda.synchronize()
    check(qo, q, wq, 1e-5, f.numpy(), pos, interleaved, 1.25, "q")
    check(ko, k, wk, 1e-5, f.numpy(), pos, interleaved, 1.25, "k")
    assert torch.equal(tq, gpu(q)[0]) and torch.equal(tk, gpu(k)[0])
    K.qk_norm_rotary(tq, tk, *tw, f.to(DEV), tc, q_out=tq, k_out=tk, **kw)
    torch.cuda.synchronize()
    assert torch.equal(tq, qo) and torch.equal(tk, ko), "in place"


def test_positions_views_and_q_alone():
    """q and k as parts of one projection, turned in place at explicit positions: V and the tokens past q_len stay.  Rows
    off a 16-byte border and weights off one take the element-wise form; q alone is as q beside k."""
    rng = np.random.default_rng(2)
    B, QL, H, HK, D, R = 3, 6, 8, 2, 128, 64
    fused = rand16(rng, B, QL, H + 2 * HK, D)
    f = K.rotary_inv_freq(R, device="cpu")[0]
    pos = rng.integers(-50, 5000, (B, QL + 2)).astype(np.int32)
    wq, wk = rng.uniform(0.5, 1.5, (2, D)).astype(np.float16)
    t, tp, tq, tk = gpu(fused, pos, wq, wk)
    note("qk_norm views")
    alone, none = K.qk_norm_rotary(t[:, :, :H], None, tq, None, f.to(DEV), positions=tp, q_len=4)
    assert none is None
    q, k = t[:, :, :H], t[:, :, H:H + HK]
    K.qk_norm_rotary(q, k, tq, tk, f.to(DEV), positions=tp, q_len=4, q_out=q, k_out=k)
    torch.cuda.synchronize()
    check(q[:, :4], fused[:, :4, :H], wq, 1e-6, f.numpy(), pos[:, :4], False, 1.0, "q")
    check(k[:, :4], fused[:, :4, H:H + HK], wk, 1e-6, f.numpy(), pos[:, :4], False, 1.0, "k")
    assert torch.equal(alone[:, :4], q[:, :4])
    got = t.cpu().numpy()
    assert np.array_equal(got[:, :, H + HK:], fused[:, :, H + HK:]) and np.array_equal(got[:, 4:], fused[:, 4:])
    x = gpu(fused[:, :, :H])[0]
    odd = torch.zeros(x.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(x.shape)
    odd.copy_(x)
    w_odd = torch.zeros(D + 1, dtype=torch.float16, device=DEV)[1:]
    w_odd.copy_(tq)
    for xs, ws in ((odd, tq), (x, w_odd)):
        got, _ = K.qk_norm_rotary(xs, None, ws, None, f.to(DEV), positions=tp)
        torch.cuda.synchronize()
        check(got, fused[:, :, :H], wq, 1e-6, f.numpy(), pos[:, :QL], False, 1.0, "unaligned")


def test_rows_without_a_norm():
    """eps = 0: a row of zeros is NaN, as 0 / 0 is; NaN and infinity stay in their rows."""
    f, _ = K.rotary_inv_freq(64, device=DEV)
    q = torch.ones((1, 4, 2, 64), dtype=torch.float16, device=DEV)
    q[0, 0, 0] = 0
    q[0, 1, 1, 5] = float("nan")
    q[0, 2, 0, 63] = float("inf")
    c = torch.full((1,), 9, dtype=torch.int32, device=DEV)
    note("qk_norm eps 0")
    got, _ = K.qk_norm_rotary(q, None, None, None, f, c, eps=0.0)
    torch.cuda.synchronize()
    bad = torch.isnan(got).any(-1)[0].cpu()
    want = torch.zeros((4, 2), dtype=torch.bool)
    want[0, 0] = want[1, 1] = want[2, 0] = True
    assert torch.equal(bad, want)


def test_plan_graph_streams_and_inactive_tokens():
    rng = np.random.default_rng(3)
    B, QL, H, HK, D = 4, 9, 8, 2, 128
    q, k = rand16(rng, B, QL, H, D), rand16(rng, B, QL, HK, D)
    wq, wk = rng.uniform(0.5, 1.5, (2, D)).astype(np.float16)
    f, _ = K.rotary_inv_freq(D, device=DEV)
    ctx = np.asarray([40, 9, 1000, 77], np.int32)
    tq, tk, tc, twq, twk = gpu(q, k, ctx, wq, wk)
    plan = torch.tensor([B, QL], dtype=torch.int32, device=DEV)
    qo, ko = torch.empty_like(tq), torch.empty_like(tk)
    call = lambda: K.qk_norm_rotary(tq, tk, twq, twk, f, tc, plan=plan, q_out=qo, k_out=ko)  # noqa: E731
    note("qk_norm plan graph")
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for n, ql in ((4, 9), (1, 2), (3, 1), (0, 4), (4, 0)):
        plan.copy_(torch.tensor([n, ql], dtype=torch.int32))
        qo.fill_(7), ko.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        if n and ql:
            pos = ctx[:n, None] - ql + np.arange(ql)[None]
            check(qo[:n, :ql], q[:n, :ql], wq, 1e-6, f.cpu().numpy(), pos, False, 1.0, f"plan {n} {ql}")
            check(ko[:n, :ql], k[:n, :ql], wk, 1e-6, f.cpu().numpy(), pos, False, 1.0, f"plan {n} {ql}")
        assert bool((qo[n:] == 7).all()) and bool((qo[:, ql:] == 7).all()) and bool((ko[:, ql:] == 7).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = K.qk_norm_rotary(tq, tk, twq, twk, f, tc)
    s.synchronize()
    check(got, q, wq, 1e-6, f.cpu().numpy(), ctx[:, None] - QL + np.arange(QL)[None], False, 1.0, "stream")


def test_empty_and_refusals():
    f, _ = K.rotary_inv_freq(64, device=DEV)
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=DEV)
    c = torch.full((2,), 9, dtype=torch.int32, device=DEV)
    w = torch.ones(64, dtype=torch.float16, device=DEV)
    note("qk_norm refusals")
    K.qk_norm_rotary(q, None, w, None, f, c, q_len=0)
    K.qk_norm_rotary(q[:0], q[:0], w, w, f, c)
    torch.cuda.synchronize()
    wide = K.rotary_inv_freq(66, device=DEV)[0]
    ok = (q, None, w, None, f, c)
    for args, kw in [((q.float(), None, w, None, f, c), {}), ((q, q[:1], w, w, f, c), {}), ((q, None, w, None, wide, c), {}),
                     ((q, None, w, None, f[:0], c), {}), ((q, None, w, None, f), {}), ((q, None, w, None, f, c[:1]), {}),
                     ((q, None, w[:32], None, f, c), {}), ((q, None, w.double(), None, f, c), {}),
                     ((q, None, w.cpu(), None, f, c), {}), ((q, None, w.expand(3, 64), None, f, c), {}),
                     ((q, None, w, w, f, c), {}), ((q, q, w, w.float(), f, c), {}),
                     ((q, None, w.view(64, 1).expand(64, 64)[:4], None, f, c), {}),
                     ((q, None, torch.ones(128, dtype=torch.float16, device=DEV)[::2], None, f, c), {}),
                     (ok, dict(q_len=4)), (ok, dict(n_seqs=3)), (ok, dict(q_out=q[:1])), (ok, dict(k_out=q)),
                     (ok, dict(eps=-1.0)), (ok, dict(eps=float("nan"))), (ok, dict(eps=float("inf")))]:
        with pytest.raises(RuntimeError):
            K.qk_norm_rotary(*args, **kw)
    big = torch.zeros((1, 1, 1, 514), dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="512"):
        K.qk_norm_rotary(big, None, None, None, f, c)
    # One row of weights for all heads may be an expanded one.
    K.qk_norm_rotary(q, None, w.expand(4, 64), None, f, c)
    torch.cuda.synchronize()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,per_head", [(80, 20, False), (90, 90, True)])
def test_prompts_of_unaligned_heads(D, R, per_head, interleaved):
    """More than 1024 tokens of heads that the vector form does not take: four waves a token."""
    rng = np.random.default_rng(D)
    B, QL, H, HK = 3, 401, 5, 2
    q, k = rand16(rng, B, QL, H, D, size=3.0), rand16(rng, B, QL, HK, D, size=0.2)
    wq, wk = (rng.uniform(0.5, 1.5, (h, D) if per_head else D).astype(np.float16) for h in (H, HK))
    f, _ = K.rotary_inv_freq(R, device="cpu")
    ctx = rng.integers(QL, 100000, B).astype(np.int32)
    pos = ctx[:, None] - QL + np.arange(QL)[None]
    note(f"qk_norm unaligned prompt D={D} R={R} interleaved={interleaved}")
    tq, tk, twq, twk, tc = gpu(q, k, wq, wk, ctx)
    qo, ko = K.qk_norm_rotary(tq, tk, twq, twk, f.to(DEV), tc, interleaved=interleaved)
    torch.cuda.synchronize()
    check(qo, q, wq, 1e-6, f.numpy(), pos, interleaved, 1.0, "q")
    check(ko, k, wk, 1e-6, f.numpy(), pos, interleaved, 1.0, "k")
