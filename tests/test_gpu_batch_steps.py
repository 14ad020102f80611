"""Beam search and drafts with eviction over the paged int8 cache, run as a serving loop would: norms and positions, append,
attention, gathered weights; selection, reordering and fork of the beams; acceptance, eviction and release of pages.  Every
step is held to the plain implementations fed with what the device held before it."""
import numpy as np
import pytest
import torch

import kernels as K
from block_cache_util import gpu, raw
from gpu_util import note
from oracle import batch_ops as O
from oracle import cache_ops as C
from oracle import oracle as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, HK, D, PAGE = 8, 2, 64, 16


class Loop:
    """A batch of rows over a pool of pages, and the oracle's view of its tables."""

    def __init__(self, rng, rows, pages, cols):
        self.rng, self.rows = rng, rows
        self.kc, self.vc = (torch.zeros((pages, PAGE, HK, D), dtype=torch.int8, device=DEV) for _ in "kv")
        self.ks, self.vs = (torch.zeros((pages, PAGE, HK), device=DEV) for _ in "kv")
        self.caches = [self.kc, self.vc, self.ks, self.vs]
        self.tbl = torch.full((rows, cols), -1, dtype=torch.int32, device=DEV)
        self.ref = torch.zeros(pages, dtype=torch.int32, device=DEV)
        self.weights = torch.zeros((rows, HK, cols * PAGE), device=DEV)
        self.t, self.r = raw(self.tbl).copy(), raw(self.ref).copy()
        self.freq, _ = K.rotary_inv_freq(D, device=DEV)
        self.wq, self.wk = gpu(*rng.uniform(0.5, 1.5, (2, D)).astype(np.float16))
        self.ctx, self.pos = np.zeros(rows, np.int32), np.zeros(rows, np.int32)  # tokens held, and seen

    def tables(self):
        torch.cuda.synchronize()
        assert np.array_equal(raw(self.tbl), self.t) and np.array_equal(raw(self.ref), self.r)

    def step(self, ql, accept=None):
        """`ql` new tokens a row, of which accept[b] stay; returns the attention's output."""
        accept = np.full(self.rows, ql, np.int32) if accept is None else np.asarray(accept, np.int32)
        positions = (self.pos[:, None] + np.arange(ql)[None]).astype(np.int32)
        self.ctx = (self.ctx + ql).astype(np.int32)
        new = gpu(self.rng.standard_normal((self.rows, ql, H + 2 * HK, D)).astype(np.float16))[0]
        q, k, v = new[:, :, :H], new[:, :, H:H + HK], new[:, :, H + HK:]
        q0, k0 = raw(q).copy(), raw(k).copy()
        cl, before = gpu(self.ctx)[0], [raw(x).copy() for x in self.caches]
        short = K.paged_kv_reserve(self.tbl, self.ref, cl, PAGE)
        K.qk_norm_rotary(q, k, self.wq, self.wk, self.freq, positions=gpu(positions)[0], q_out=q, k_out=k)
        K.paged_kv_append(k, v, *self.caches, self.tbl, cl)
        out, _ = K.paged_attention(q, *self.caches, self.tbl, cl, ql, QPP=min(ql, 16))
        self.t, self.r, s = C.reserve(self.t, self.r, self.ctx, PAGE)
        self.tables()
        assert int(short) == s == 0
        for got, x, w in ((q, q0, self.wq), (k, k0, self.wk)):
            want = O.qk_norm_rotary(x, raw(w), 1e-6, self.freq.cpu().numpy(), positions, False, 1.0)
            assert np.abs(raw(got) - want).max() <= 2.0 ** -11 * np.abs(want).max() + 1e-4
        want = R.paged_kv_append(raw(k), raw(v), *before, self.t, self.ctx, ql)
        for a, b in zip(self.caches, want):
            assert np.array_equal(raw(a), np.asarray(b))
        attn, mag = R.paged_attention(raw(q), *want, self.t, self.ctx, ql, magnitude=True)
        assert (np.abs(raw(out) - attn) <= 2.0 ** -9 * mag + 2.0 ** -10 * np.abs(attn) + 2.0 ** -14).all()
        # What was accepted stays, and gathers.
        self.ctx = (self.ctx - ql + accept).astype(np.int32)
        self.pos = (self.pos + accept).astype(np.int32)
        cl, had = gpu(self.ctx)[0], raw(self.weights).copy()
        K.paged_kv_free(self.tbl, self.ref, cl, PAGE)
        K.paged_attention_weights(q, self.kc, self.ks, self.tbl, cl, self.weights, q_lens=gpu(accept)[0])
        self.t, self.r = C.free(self.t, self.r, self.ctx, PAGE)
        self.tables()
        want, _ = O.attn_weights(raw(q), raw(self.kc), raw(self.ks), self.t, self.ctx, had, accept, D ** -0.5)
        assert np.abs(raw(self.weights) - want).max() <= 1e-4 * max(1.0, want.max())
        return out

    def evict(self, budget, recent, sinks, limit):
        cl = gpu(self.ctx)[0]
        had = [raw(x).copy() for x in self.caches]
        kept, ctx, w, caches = O.evict(self.t, self.ctx, raw(self.weights).copy(), had, budget, recent, sinks, limit, self.r)
        got = K.paged_kv_evict(self.tbl, cl, self.weights, self.caches, PAGE, budget, recent, sinks, limit, self.ref)
        K.paged_kv_free(self.tbl, self.ref, cl, PAGE)
        self.t, self.r = C.free(self.t, self.r, ctx, PAGE)
        self.tables()
        assert np.array_equal(raw(got), kept) and np.array_equal(raw(cl), ctx) and np.array_equal(raw(self.weights), w)
        assert all(np.array_equal(raw(a), b) for a, b in zip(self.caches, caches))
        cut = int((ctx != self.ctx).sum())
        self.ctx = ctx
        return cut


def test_beam_search():
    """Two sequences of three beams: a prompt, then steps that end some beams; at the end the best beam alone is cut back."""
    rng = np.random.default_rng(31)
    B, W, V, eos, T = 2, 3, 1009, 5, 16
    loop = Loop(rng, B * W, 80, 8)
    proj = gpu((rng.standard_normal((H * D, V)) / 8).astype(np.float32))[0]
    history = torch.zeros((B * W, T), dtype=torch.int32, device=DEV)
    done = torch.zeros((B, W), dtype=torch.bool, device=DEV)
    scores = torch.full((B, W), float("-inf"), device=DEV)
    scores[:, 0] = 0  # one beam at the start
    note("beam search loop")
    # One prompt a sequence: the first row's; the others become its copies at the first fork.
    out = loop.step(37)
    for i in range(5):
        logits = (out[:, -1].reshape(B * W, -1).float() @ proj).view(B, W, V)
        if i == 2:
            logits[:, 1, eos] += 40  # a beam that ends
        s0, d0, h0, w0, p0 = raw(scores).copy(), raw(done).copy(), raw(history).copy(), raw(loop.weights).copy(), loop.pos.copy()
        scores, token, parent = K.beam_select(logits, scores, W, done, eos)
        pos = gpu(loop.pos)[0]
        K.beam_reorder([history, loop.weights, pos, done.view(-1)], parent.view(-1), W)
        lens = gpu(loop.ctx)[0]
        short = K.paged_kv_fork(loop.tbl, loop.ref, lens, parent.view(-1), loop.caches, PAGE)
        want, wt, wp, _ = O.beam_select(raw(logits), s0, W, d0, eos)
        torch.cuda.synchronize()
        assert np.array_equal(raw(token), wt) and np.array_equal(raw(parent), wp) and (wt >= 0).all()
        assert np.abs(raw(scores) - want).max() <= 1e-4
        for got, was in ((history, h0), (loop.weights, w0), (pos, p0), (done.view(-1), d0.reshape(-1))):
            assert np.array_equal(raw(got), O.reorder([was], wp.reshape(-1), W)[0])
        loop.t, loop.r, loop.ctx, s, _ = C.fork(loop.t, loop.r, loop.ctx, wp.reshape(-1), PAGE)
        loop.tables()
        assert int(short) == s == 0 and np.array_equal(raw(lens), loop.ctx)
        loop.pos = raw(pos).copy()
        history[:, i] = token.view(-1)
        done |= token == eos
        assert bool(done.any()) == (i >= 2)
        assert loop.evict(20, 4, 1, 30) == 0, "rows that share pages stay"
        out = loop.step(1)
    # The best beam of each sequence stays; its pages are its own now.
    keep = np.where(np.arange(B * W) % W == 0, loop.ctx, 0).astype(np.int32)
    K.paged_kv_free(loop.tbl, loop.ref, gpu(keep)[0], PAGE)
    loop.t, loop.r = C.free(loop.t, loop.r, keep, PAGE)
    loop.ctx = keep
    loop.tables()
    assert loop.evict(20, 4, 1, 30) == B
    loop.step(2)


def test_drafts_with_eviction():
    """Drafts of which some are accepted, the cache cut back to 48 tokens whenever it holds more than 70."""
    rng = np.random.default_rng(32)
    loop = Loop(rng, 3, 40, 8)
    note("drafts with eviction")
    loop.step(60, [60, 33, 47])
    cut = 0
    for _ in range(8):
        loop.step(9, rng.integers(1, 10, 3))
        cut += loop.evict(48, 12, 2, 70)
    assert cut >= 3 and (loop.ctx <= 70).all() and (loop.pos > loop.ctx).any()
