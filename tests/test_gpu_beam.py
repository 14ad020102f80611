"""Beam selection and reordering on the GPU.

Selected tokens and parents are the float64 oracle's exactly; each case asserts that the oracle's neighbouring scores of
different beams lie further apart than the kernel can be off.  That is: a segment's sum of exponentials in fp32 (at most
64 additions in a lane and 6 between lanes, 70 * 2^-24, and 2^-22 for the exponentials with their argument's rounding
on values that matter) makes a log-sum off by less than GAP = 2^-17; everything behind it is fp64.  Scores are rounded to
fp32 once: within GAP + 2^-24 |score|.
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
GAP = 2.0 ** -17


def check(got, logits, scores, n, finished=None, eos=None, ties=False, what=""):
    score, token, parent = (t.cpu().numpy() for t in got)
    want, wt, wp, behind = O.beam_select(logits, scores, n, finished, eos)
    row = np.concatenate((want, behind[:, None]), 1)
    for b in range(len(row)):
        for i in range(n):
            other = wp[b, i] != wp[b, i + 1] if i + 1 < n else True
            d = row[b, i] - row[b, i + 1] if np.isfinite(row[b, i + 1]) else np.inf
            assert ties or d > 2 * GAP or not other or i + 1 == n and d == 0, f"{what}: the case itself is too close at {b}, {i}: {d}"
    assert np.array_equal(token, wt), f"{what}: tokens {token} {wt}"
    assert np.array_equal(parent, wp), f"{what}: parents"
    none = wt < 0
    assert np.isneginf(score[none]).all()
    err = np.abs(score.astype(np.float64) - want)[~none]
    assert (err <= GAP + 2.0 ** -24 * np.abs(want[~none])).all(), f"{what}: scores off {err.max()}"


def make(rng, B, W, V, f32, size=3.0):
    x = (size * rng.standard_normal((B, W, V))).astype(np.float32 if f32 else np.float16)
    return x, -rng.uniform(0, 10, (B, W)).astype(np.float32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("B,W,V,n", [
    (1, 1, 1, 1),            # one token
    (1, 1, 1, 5),            # fewer candidates than wanted
    (2, 3, 7, 21),           # all of them
    (1, 4, 32000, 4),
    (3, 5, 1003, 10),        # rows off 16-byte borders
    (2, 2, 50257, 64),       # as many as are supported
    (1, 64, 513, 64),        # as many beams
    (4, 8, 2048, 16),
    (2, 16, 20000, 32),
])
def test_matches_float64(B, W, V, n, f32):
    rng = np.random.default_rng(V + n)
    x, s = make(rng, B, W, V, f32)
    note(f"beam B={B} W={W} V={V} n={n} f32={f32}")
    got = K.beam_select(*gpu(x, s), n)
    torch.cuda.synchronize()
    check(got, x, s, n, what="beam")


@pytest.mark.parametrize("f32", [False, True])
def test_large_batch(f32):
    """Eight vectors a lane: enough rows to fill the GPU."""
    rng = np.random.default_rng(1)
    x, s = make(rng, 12, 8, 60001, f32)
    note(f"beam large f32={f32}")
    got = K.beam_select(*gpu(x, s), 16)
    torch.cuda.synchronize()
    check(got, x, s, 16, what="large")


@pytest.mark.parametrize("n", [1, 40, 64])
def test_many_parts_and_scores_in_place(n):
    """64 beams of more parts than threads read ahead; with n = W the new scores may replace the old ones."""
    rng = np.random.default_rng(11)
    x, s = make(rng, 2, 64, 40001, True)
    note(f"beam parts n={n}")
    tx, ts = gpu(x, s)
    out = (ts if n == 64 else torch.empty((2, n), device=DEV), *(torch.empty((2, n), dtype=torch.int32, device=DEV) for _ in "tp"))
    got = K.beam_select(tx, ts, n, out=out)
    torch.cuda.synchronize()
    assert got[0].data_ptr() == out[0].data_ptr()
    check(got, x, s, n, what="parts")


def test_finished_beams_and_missing_ones():
    """A finished beam goes on with eos alone; a beam of score -inf has nothing; banned tokens are none."""
    rng = np.random.default_rng(2)
    B, W, V = 5, 4, 5000
    x, s = make(rng, B, W, V, False)
    done = rng.uniform(size=(B, W)) < 0.4
    s[0, 1:] = -np.inf     # the first step: one beam
    done[1] = True         # all finished
    s[1, 2] = -np.inf
    x[2] = -np.inf         # nothing but three tokens
    x[2, 1, [7, 4000, 30]] = 1.0, 2.0, 0.5
    done[2] = False
    done[3], x[3, :, ::2] = False, -np.inf
    note("beam finished")
    tx, ts, td = gpu(x, s, done)
    before = tx.clone()
    for n in (4, 8):
        got = K.beam_select(tx, ts, n, td, 4999)
        torch.cuda.synchronize()
        check(got, x, s, n, done, 4999, what=f"n={n}")
    assert torch.equal(tx, before)


def test_ties_go_to_the_lower_beam_and_token():
    """Equal rows, equal beams, constant rows of any length: lists that overflow."""
    rng = np.random.default_rng(3)
    note("beam ties")
    for V, W, n in ((100, 2, 7), (5000, 3, 16), (40000, 4, 64), (70, 64, 64)):
        for kind in ("constant", "equal beams", "few values", "two"):
            row = {"constant": np.zeros(V), "equal beams": rng.standard_normal(V), "few values": rng.integers(0, 4, V),
                   "two": np.where(np.arange(V) == V - 1, 1, 0)}[kind].astype(np.float16)
            x = np.broadcast_to(row, (2, W, V)).copy()
            s = np.full((2, W), -1.5, np.float32)
            got = K.beam_select(*gpu(x, s), n)
            torch.cuda.synchronize()
            check(got, x, s, n, ties=True, what=f"{kind} V={V} W={W} n={n}")


def test_rows_that_are_not_numbers():
    """A row with NaN or +inf has no candidates; the others are as ever."""
    rng = np.random.default_rng(4)
    x, s = make(rng, 2, 4, 9001, True)
    x[0, 1, 77], x[0, 2, 9000], x[1, 0] = np.nan, np.inf, -np.inf
    s[1, 3] = np.nan
    note("beam nan")
    got = K.beam_select(*gpu(x, s), 8)
    torch.cuda.synchronize()
    s2 = s.copy()
    s2[1, 3] = -np.inf
    check(got, x, s2, 8, what="nan")


def test_extreme_logits():
    rng = np.random.default_rng(5)
    x, s = make(rng, 1, 3, 4000, False)
    x[0, 0, 5], x[0, 1, 9], x[0, 2] = 65504, -65504, x[0, 2] - np.float16(300)
    note("beam extreme")
    got = K.beam_select(*gpu(x, s), 6)
    torch.cuda.synchronize()
    check(got, x, s, 6, what="extreme")


def test_views_given_outputs_graph_and_streams():
    from specq.workspace import Workspace
    rng = np.random.default_rng(6)
    B, W, V, n = 2, 3, 3001, 6
    x, s = make(rng, B, W, V, False)
    tx, ts = gpu(x, s)
    wide = torch.zeros((B, W + 1, V + 2), dtype=torch.float16, device=DEV)
    wide[:, 1:, 1:-1] = tx
    out = (torch.empty((B, n), device=DEV), *(torch.empty((B, n), dtype=torch.int32, device=DEV) for _ in "tp"))
    note("beam graph")
    got = K.beam_select(wide[:, 1:, 1:-1], ts, n, out=out)
    torch.cuda.synchronize()
    assert all(a is b for a, b in zip(got, out))
    check(got, x, s, n, what="views")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.beam_select(tx, ts, n, out=out)
    for seed in range(3):
        x2, s2 = make(np.random.default_rng(100 + seed), B, W, V, False)
        tx.copy_(gpu(x2)[0]), ts.copy_(gpu(s2)[0])
        g.replay()
        other = K.beam_select(tx, ts, n)
        torch.cuda.synchronize()
        check(out, x2, s2, n, what="replay")
        assert all(torch.equal(a, b) for a, b in zip(out, other))
    streams, spaces = [torch.cuda.Stream() for _ in range(2)], [Workspace("cuda") for _ in range(2)]
    torch.cuda.synchronize()
    both = []
    for st, ws in zip(streams, spaces):
        with torch.cuda.stream(st):
            both.append(K.beam_select(tx, ts, n, workspace=ws))
    torch.cuda.synchronize()
    for o in both:
        assert all(torch.equal(a, b) for a, b in zip(out, o))


def test_select_refusals():
    x = torch.zeros((2, 3, 50), dtype=torch.float16, device=DEV)
    s = torch.zeros((2, 3), device=DEV)
    d = torch.zeros((2, 3), dtype=torch.bool, device=DEV)
    note("beam refusals")
    assert [t.shape for t in K.beam_select(x[:0], s[:0])] == [(0, 3)] * 3
    outs = K.beam_select(x, s, 3, None, 4)  # a token to end with, and no beam that has
    for args, kw in [((x.bfloat16(), s), {}), ((x[0], s), {}), ((x[..., ::2], s), {}), ((x, s[:1]), {}), ((x, s.half()), {}),
                     ((x, s, 0), {}), ((x, s, 65), {}), ((x, s, 3, d), {}), ((x, s, 3, d, 50), {}),
                     ((x, s, 3, d, -1), {}), ((x, s, 3, d.int(), 4), {}), ((x, s, 3, d[:1], 4), {}), ((x.cpu(), s), {}),
                     ((x, s.cpu()), {}), ((x[:, :0], s[:, :0]), {}), ((x[..., :0], s), {}), ((x, s, 4), dict(out=outs)),
                     ((x, s), dict(out=outs[:2])), ((x, s), dict(out=(outs[0], outs[1].long(), outs[2]))),
                     ((torch.zeros((1, 65, 9), device=DEV), torch.zeros((1, 65), device=DEV), 3), {})]:
        with pytest.raises(RuntimeError):
            K.beam_select(*args, **kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 13, 32])
def test_reorder_is_exact(W):
    """States of any type, size and alignment; parents that repeat, stay, cross and lie outside their group."""
    rng = np.random.default_rng(W)
    for B in (1, 3):
        rows = B * W
        parents = (rng.integers(0, W, rows) + np.repeat(np.arange(B) * W, W)).astype(np.int32)
        parents[rng.uniform(size=rows) < 0.2] = -1
        if B > 1:
            parents[0], parents[-1] = W, 2 ** 31 - 1
        states = [rng.integers(0, 1000, (rows, 77)).astype(np.int32), rng.standard_normal((rows, 4096)).astype(np.float16),
                  rng.uniform(size=(rows, 3, 5, 7)).astype(np.float32), rng.integers(0, 2, rows).astype(bool),
                  rng.integers(0, 255, (rows, 13)).astype(np.uint8), rng.standard_normal((rows, 20000)).astype(np.float32),
                  rng.standard_normal(rows), rng.integers(0, 9, (rows, 0)).astype(np.int64)]
        ts = [torch.from_numpy(s).to(DEV) for s in states]
        strided = torch.zeros((rows, 600), dtype=torch.int32, device=DEV)
        strided[:, 100:177] = ts[0]
        note(f"reorder W={W} B={B}")
        K.beam_reorder([*ts, strided[:, 100:177]], gpu(parents)[0], W)
        torch.cuda.synchronize()
        want = O.reorder([*states, states[0]], parents, W)
        for i, (a, b) in enumerate(zip([*ts, strided[:, 100:177]], want)):
            assert np.array_equal(a.cpu().numpy(), b), f"state {i}"
        assert bool((strided[:, :100] == 0).all()) and bool((strided[:, 177:] == 0).all())


def test_reorder_many_states_large_rows_and_graph():
    """More states than one launch takes; rows of 5 MB; a graph replayed with other parents."""
    rng = np.random.default_rng(9)
    W, rows = 4, 8
    states = [rng.integers(0, 100, (rows, 3)).astype(np.int32) for _ in range(70)]
    states.append(rng.integers(0, 1 << 30, (rows, 5 << 18)).astype(np.int32))
    ts = gpu(*states)
    parents = torch.zeros(rows, dtype=torch.int32, device=DEV)
    note("reorder many")
    parents.copy_(torch.arange(rows, dtype=torch.int32))
    K.beam_reorder(ts, parents, W)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.beam_reorder(ts, parents, W)
    for _ in range(3):
        p = (rng.integers(0, W, rows) + np.repeat([0, W], W)).astype(np.int32)
        parents.copy_(torch.from_numpy(p))
        g.replay()
        torch.cuda.synchronize()
        states = O.reorder(states, p, W)
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(ts, states))


def test_reorder_refusals():
    p = torch.zeros(4, dtype=torch.int32, device=DEV)
    x = torch.arange(12, device=DEV, dtype=torch.int32).view(4, 3)
    before = x.clone()
    note("reorder refusals")
    K.beam_reorder([], p, 2)
    K.beam_reorder([x[:0]], p[:0], 2)
    for states, parents, group in [([x[:3]], p, 2), ([x], p, 3), ([x], p, 0), ([x], p.long(), 2), ([x], p.view(2, 2), 2),
                                   ([x.cpu()], p, 2), ([x, x], p, 2), ([x[:1].expand(4, 3)], p, 2), ([x.t()], p[:3], 3),
                                   ([torch.zeros((66, 2), device=DEV)], torch.zeros(66, dtype=torch.int32, device=DEV), 33),
                                   ([x], torch.zeros(8, dtype=torch.int32, device=DEV)[::2], 2)]:
        with pytest.raises(RuntimeError):
            K.beam_reorder(states, parents, group)
    torch.cuda.synchronize()
    assert torch.equal(x, before)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V", [1001, 128257])
def test_beams_closer_than_an_fp32_step_of_their_scores(V, f32):
    """The best candidates of two different rows, some 2^-28 apart at scores of -1 to -20, whose fp32 steps are 2^-24 and more.

    Every row's log-sum is off by less than 2^-33.9 (exponentials within 2^-34 of themselves, sums in fp64), and what is behind it
    is fp64 of values below 2^7, within 2^-44: candidates further apart than 2^-32 are ordered as the formula has them.  The
    second beam's score is chosen so that the difference is no more than half of its fp32 step (below 2^-26) and a little."""
    rng = np.random.default_rng(V)
    B = 48
    x, _ = make(rng, B, 2, V, f32, 2.0)
    lse = lambda r: r.max() + np.log(np.exp(r - r.max()).sum())  # noqa: E731
    best = np.array([[r.max() - lse(r) for r in b.astype(np.float64)] for b in x])
    s = np.zeros((B, 2), np.float32)
    s[:, 0] = rng.uniform(0.001, 0.25, B)
    # Beam 1's score, within +-0.25 of 0, makes up what its best candidate lacks against beam 0's; rows too far apart are moved.
    for b in range(B):
        d = best[b, 0] + s[b, 0].astype(np.float64) - best[b, 1]
        s[b, 1] = d
        if abs(d) > 0.25:  # all of a row's logits but its largest shifted until the largest are alike
            at = x[b, 1].argmax()
            lo, hi = np.float64(-20.0), np.float64(20.0)
            for _ in range(60):
                mid = (lo + hi) / 2
                r = x[b, 1].astype(np.float64) + mid
                r[at] = x[b, 1, at]
                lo, hi = (mid, hi) if r[at] - lse(r) > best[b, 0] else (lo, mid)
            top = x[b, 1, at]
            x[b, 1] = np.minimum((x[b, 1].astype(np.float64) + lo).astype(x.dtype), top)
            x[b, 1, at] = top
            r = x[b, 1].astype(np.float64)
            s[b, 1] = best[b, 0] + s[b, 0].astype(np.float64) - (r.max() - lse(r))
    want, token, parent, _ = O.beam_select(x, s, 2)
    apart = want[:, 0] - want[:, 1]
    note(f"beam close V={V} f32={f32}")
    got = K.beam_select(*gpu(x, s), 2)
    torch.cuda.synchronize()
    sure = (apart > 2.0 ** -32) & (parent[:, 0] != parent[:, 1])
    assert sure.sum() > B // 2 and (apart[sure] < 2.0 ** -24).sum() > B // 2  # the case is what it says
    assert np.array_equal(got[2].cpu().numpy()[sure], parent[sure])
    assert np.array_equal(got[1].cpu().numpy()[sure], token[sure])
    err = np.abs(got[0].cpu().numpy().astype(np.float64) - want)
    assert (err <= 2.0 ** -32 + 2.0 ** -24 * np.abs(want)).all()


def test_lowest_values_as_masks():
    """Beams that are not there and banned tokens by fp32's lowest value, not by -inf: either alone is a candidate, the last of
    all; both together have no fp32 score, and are none.  Next to the lowest value the logits' differences are below half a step
    of fp64 (2^74), so that a beam of that score has its tokens tie, in their order."""
    low = np.finfo(np.float32).min
    x = np.full((2, 2, 300), low, np.float32)
    x[:, :, [3, 200]] = 1.0, 2.0
    s = np.array([[-1, low], [low, low]], np.float32)
    note("beam lowest values")
    score, token, parent = (t.cpu().numpy() for t in K.beam_select(*gpu(x, s), 6))
    assert token.tolist() == [[200, 3, 0, 1, 2, 4], [3, 200, 3, 200, -1, -1]]
    assert parent.tolist() == [[0] * 6, [2, 2, 3, 3, -1, -1]]
    assert (score[0, 2:] == low).all() and np.isneginf(score[1, 4:]).all() and np.isfinite(score[1, :4]).all()


@pytest.mark.parametrize("size", [1e6, 1e15, 1e20, 1e38])
def test_logits_of_any_size(size):
    """A row's sum is relative to its largest logit, whatever that is: rows of 10^6 to 10^38, constant ones among them, and of
    fp32's lowest value throughout."""
    rng = np.random.default_rng(12)
    x = (size * rng.uniform(-1, 1, (3, 4, 3000))).astype(np.float32)
    x[0, 1], x[0, 2], x[1, 0] = size, -size, np.finfo(np.float32).min
    x[1, 1, 5:90] = x[1, 1].max()
    s = np.array([[-1, -2, -3, -4], [-0.5, -8, -9, -10], [-1, -1, -1, -1]], np.float32)
    note(f"beam size {size}")
    got = K.beam_select(*gpu(x, s), 12)
    torch.cuda.synchronize()
    check(got, x, s, 12, ties=True, what=f"size {size}")
