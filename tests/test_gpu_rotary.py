"""Rotary positions on the GPU against float64.

Tolerance for a pair (a, b) turned with factor m: one rounding to fp16 (2^-11 of the result, 2^-25 below
its normal range), the sine and cosine within 4e-7 (the fraction of a turn is rounded to 2^-25, 1.9e-7
radians, and the hardware functions are within 1.3e-7 of the exact ones over a turn, measured), and three
fp32 operations (2^-22): |err| <= 2^-11 |ref| + 2^-25 + m (|a| + |b|) (4e-7 + 2^-22).
"""
import math

import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import gpu
from gpu_util import note
from oracle import cache_ops as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand16(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def check(got, x, inv_freq, pos, interleaved, m, what):
    ref = C.rotary(x, inv_freq, pos, interleaved, m)
    R = 2 * len(inv_freq)
    size = np.zeros(x.shape)
    a = np.abs(x.astype(np.float64))
    i0, i1 = (np.arange(0, R, 2), np.arange(1, R, 2)) if interleaved else (np.arange(R // 2), np.arange(R // 2, R))
    size[..., i0] = size[..., i1] = a[..., i0] + a[..., i1]
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + m * size * (4e-7 + 2.0 ** -22)
    assert (err <= tol).all(), f"{what}: worst {err.max():.3e}"
    assert np.array_equal(got.cpu().numpy()[..., R:], x[..., R:]), f"{what}: copied dimensions"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,QL,H,H_KV,D,R,far", [
    (1, 1, 32, 8, 128, 128, 8192),
    (3, 17, 12, 3, 80, 20, 1000003),       # pairs that no vector holds whole
    (2, 700, 4, 1, 64, 32, 100000),        # more than 1024 tokens: a wave each
    (5, 9, 8, 8, 96, 96, 2 ** 20),
    (2, 3, 5, 2, 192, 64, 3000),           # a third of the head
    (1, 2, 1, 1, 2, 2, 50),                # the smallest head
    (2, 2, 3, 1, 511 - 1, 6, 50),          # rows that are not 16-byte aligned
    (1, 5, 2, 2, 512, 512, 2 ** 30),       # the largest head, positions past 2^24
    (1, 2, 2, 1, 400, 390, 700),           # more items than threads in the unaligned form
])
def test_matches_float64(B, QL, H, H_KV, D, R, far, interleaved):
    rng = np.random.default_rng(B * 100 + QL + D)
    q, k = rand16(rng, B, QL, H, D), rand16(rng, B, QL, H_KV, D)
    f, _ = K.rotary_inv_freq(R, device="cpu")
    ctx = rng.integers(QL, far + QL, B).astype(np.int32)
    pos = ctx[:, None] - QL + np.arange(QL)[None]
    note(f"rotary B={B} QL={QL} H={H}/{H_KV} D={D} R={R} interleaved={interleaved}")
    tq, tk, tc = gpu(q, k, ctx)
    qo, ko = K.rotary_embed(tq, tk, f.to(DEV), tc, interleaved=interleaved, mscale=1.25)
    torch.cuda.synchronize()
    check(qo, q, f.numpy(), pos, interleaved, 1.25, "q")
    check(ko, k, f.numpy(), pos, interleaved, 1.25, "k")
    assert torch.equal(tq, gpu(q)[0]) and torch.equal(tk, gpu(k)[0])
    K.rotary_embed(tq, tk, f.to(DEV), tc, interleaved=interleaved, mscale=1.25, q_out=tq, k_out=tk)
    torch.cuda.synchronize()
    assert torch.equal(tq, qo) and torch.equal(tk, ko), "in place"


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_fp32_frequencies_and_views(interleaved):
    """Explicit positions (negative ones too), fp32 frequencies, q and k as parts of one projection, turned in place:
    the V part and the tokens past q_len stay."""
    rng = np.random.default_rng(2)
    B, QL, H, HK, D, R = 3, 6, 8, 2, 128, 64
    fused = rand16(rng, B, QL, H + 2 * HK, D)
    f = K.rotary_inv_freq(R, device="cpu")[0].float()
    pos = rng.integers(-50, 5000, (B, QL + 2)).astype(np.int32)
    t, tp = gpu(fused, pos)
    note(f"rotary views interleaved={interleaved}")
    q, k = t[:, :, :H], t[:, :, H:H + HK]
    K.rotary_embed(q, k, f.to(DEV), positions=tp, q_len=4, interleaved=interleaved, q_out=q, k_out=k)
    torch.cuda.synchronize()
    check(q[:, :4], fused[:, :4, :H], f.double().numpy(), pos[:, :4], interleaved, 1.0, "q")
    check(k[:, :4], fused[:, :4, H:H + HK], f.double().numpy(), pos[:, :4], interleaved, 1.0, "k")
    got = t.cpu().numpy()
    assert np.array_equal(got[:, :, H + HK:], fused[:, :, H + HK:]) and np.array_equal(got[:, 4:], fused[:, 4:])
    # Rows that start off a 16-byte border take the element-wise form, with the same results to rounding.
    odd = torch.zeros(B * QL * H * D + 1, dtype=torch.float16, device=DEV)[1:].view(B, QL, H, D)
    odd.copy_(gpu(fused[:, :, :H])[0])
    qo, none = K.rotary_embed(odd, None, f.to(DEV), positions=tp, interleaved=interleaved)
    torch.cuda.synchronize()
    assert none is None
    check(qo, fused[:, :, :H], f.double().numpy(), pos[:, :QL], interleaved, 1.0, "unaligned")


def test_plan_graph_and_inactive_tokens():
    rng = np.random.default_rng(3)
    B, QL, H, HK, D = 4, 9, 8, 2, 128
    q, k = rand16(rng, B, QL, H, D), rand16(rng, B, QL, HK, D)
    f, _ = K.rotary_inv_freq(D, device=DEV)
    ctx = np.asarray([40, 9, 1000, 77], np.int32)
    tq, tk, tc = gpu(q, k, ctx)
    plan = torch.tensor([B, QL], dtype=torch.int32, device=DEV)
    qo, ko = torch.empty_like(tq), torch.empty_like(tk)
    call = lambda: K.rotary_embed(tq, tk, f, tc, plan=plan, q_out=qo, k_out=ko)  # noqa: E731
    note("rotary plan graph")
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
            check(qo[:n, :ql], q[:n, :ql], f.cpu().numpy(), pos, False, 1.0, f"plan {n} {ql}")
            check(ko[:n, :ql], k[:n, :ql], f.cpu().numpy(), pos, False, 1.0, f"plan {n} {ql}")
        assert bool((qo[n:] == 7).all()) and bool((qo[:, ql:] == 7).all()) and bool((ko[:, ql:] == 7).all())


def test_empty_and_refusals():
    f, _ = K.rotary_inv_freq(64, device=DEV)
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=DEV)
    c = torch.full((2,), 9, dtype=torch.int32, device=DEV)
    note("rotary refusals")
    K.rotary_embed(q, None, f, c, q_len=0)
    K.rotary_embed(q[:0], q[:0], f, c)
    torch.cuda.synchronize()
    wide = K.rotary_inv_freq(66, device=DEV)[0]
    for args, kw in [((q.float(), None, f, c), {}), ((q, q[:1], f, c), {}), ((q, None, wide, c), {}),
                     ((q, None, f[:0], c), {}), ((q, None, f.half(), c), {}), ((q, None, f), {}),
                     ((q, None, f, c[:1]), {}), ((q, None, f, c.long()), {}), ((q, None, f.cpu(), c), {}),
                     ((q.cpu(), None, f, c), {}), ((q, None, f, c), dict(q_len=4)), ((q, None, f, c), dict(n_seqs=3)),
                     ((q, None, f, c), dict(q_out=q[:1])), ((q, None, f, c), dict(k_out=q)),
                     ((q.transpose(2, 3), None, f[:2], c), {}),
                     ((q, None, f), dict(positions=c)), ((q, None, f), dict(positions=torch.zeros((2, 2), dtype=torch.int32, device=DEV)))]:
        with pytest.raises(RuntimeError):
            K.rotary_embed(*args, **kw)
    big = torch.zeros((1, 1, 1, 514), dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="512"):
        K.rotary_embed(big, None, f, c)
    assert math.isfinite(float(K.rotary_embed(q, None, f, c)[0].sum()))
