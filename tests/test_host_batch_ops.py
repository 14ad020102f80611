"""CPU tier of the head norms, gathered weights, eviction and beam entry points: refusals ahead of any launch, and the plain
implementations' own properties."""
import os
import re

import numpy as np
import pytest
import torch

from oracle import batch_ops as O

# Pointers are fake: every call below must fail validation (or have nothing to do), so nothing is launched.


def _fail(name, args, code, **change):
    from specq import _lib
    a = dict(args)
    a.update(change)
    rc = getattr(_lib.lib(), name)(*a.values())
    assert rc == code, (name, change, rc, _lib.lib().specq_last_error())


NORM = dict(q=16, a=1024, b=512, c=64, k=16, d=256, e=128, f=64, qo=16, g=1024, h=512, i=64, ko=16, j=256, l=128, m=64,
            wq=16, s_wq=0, wk=16, s_wk=0, w32=0, eps=1e-6, freq=16, f64=1, ms=1.0, ctx=16, pos=0, s_pb=0, B=2, n_seqs=2,
            q_len=2, ql=2, H=8, HK=2, D=64, R=64, il=0, plan=0, stream=0)
WEIGHTS = dict(q=16, s_qb=9 * 4096, s_qt=4096, s_qh=128, kc=16, s_kp=16 * 1024, s_ko=1024, s_kh=128, ks=16, s_sp=128, s_so=8,
               s_sh=1, f32=1, bt=16, s_bt=64, max_pages=64, n_pages=100, ctx=16, q_lens=0, w=16, s_wb=8 * 1024, s_wh=1024,
               B=2, n_seqs=2, q_len=9, ql=9, H=32, HK=8, D=128, PAGE=16, sm=0.088, plan=0, ws=0, wsb=0, stream=0)


def test_norm_refusals(built_lib):
    f = lambda code, **kw: _fail("specq_qk_norm_rotary", NORM, code, **kw)  # noqa: E731
    for name in ("q", "qo", "freq", "k", "ko", "ctx"):
        f(-22, **{name: 0})
    f(-22, R=0), f(-22, R=3), f(-22, R=66), f(-22, H=0), f(-22, D=0), f(-95, D=514, R=64), f(-22, n_seqs=3), f(-22, q_len=3)
    f(-22, eps=-1.0), f(-22, eps=float("nan")), f(-22, eps=float("inf")), f(-22, B=1 << 16, ql=1 << 16)
    for k in ("g", "h", "i", "j", "l", "m"):
        f(-95, **{k: 0}), f(-95, **{k: 56})
    f(-95, h=64), f(-95, h=448), f(-95, g=512), f(-95, l=64), f(-95, j=128)  # (1, 0) and (0, 1) are, or share, one row
    f(0, B=0, n_seqs=0), f(0, ql=0, q_len=0)


def test_weights_refusals(built_lib):
    f = lambda code, **kw: _fail("specq_paged_attn_weights", WEIGHTS, code, **kw)  # noqa: E731
    for name in ("q", "kc", "ks", "bt", "ctx", "w"):
        f(-22, **{name: 0})
    f(-95, D=96), f(-95, D=256), f(-95, PAGE=24), f(-95, PAGE=8), f(-22, H=30), f(-22, HK=0), f(-22, n_seqs=3), f(-22, q_len=10)
    f(-22, max_pages=0), f(-22, n_pages=0), f(-22, max_pages=65), f(-95, max_pages=1 << 27, s_bt=1 << 27), f(-95, q=24), f(-95, s_qh=100)
    f(-95, kc=24), f(-95, s_kp=1000), f(-22, ks=18), f(-22, w=18), f(-95, s_wh=1023), f(-95, s_wb=0), f(-95, s_wh=0)
    f(-95, B=1 << 14, n_seqs=0), f(-95, ql=1 << 21, q_len=0), f(-28)
    f(-95, s_wb=1024, s_wh=1024), f(-95, s_wb=1024, s_wh=2047), f(-28, s_wb=1024, s_wh=2048)  # (1, 0) and (0, 1) are one row
    f(-95, H=8 * 4096)
    f(0, B=0, n_seqs=0), f(0, ql=0, q_len=0)


def test_weights_workspace_covers_what_a_call_asks_for(built_lib):
    from specq import _lib
    size = _lib.lib().specq_paged_attn_weights_workspace_size
    need = size(2, 32, 8, 9, 64, 16)
    # 1024 rows at a time, or more where that stays below 64 MiB.
    assert size(32, 32, 8, 4096, 2048, 16) == size(32, 32, 8, 256, 2048, 16)
    assert size(2, 32, 8, 256, 64, 16) < size(2, 32, 8, 4096, 64, 16) < size(2, 32, 8, 256, 64, 16) + (64 << 20)
    # 36 rows: statistics of each of four tiles and a sum a row; a fake workspace a byte too small is refused.
    assert need >= 2 * 8 * 36 * (4 * 8 + 4)
    _fail("specq_paged_attn_weights", WEIGHTS, -28, ws=4096, wsb=need - 1)
    assert size(2, 32, 8, 4, 64, 16) >= 2 * 8 * 16 * (1024 * 4 + 4 * 8 + 4)  # 16 rows: their scores as well
    assert size(0, 32, 8, 1, 64, 16) == size(2, 30, 8, 1, 64, 16) == size(2, 32, 8, 1, 64, 0) == 0


@pytest.mark.parametrize("B,H,HK,ql,tokens", [
    (32, 32, 8, 1, 131072), (32, 64, 8, 2, 131072), (256, 32, 8, 1, 131072), (256, 32, 8, 9, 131072), (64, 32, 8, 4096, 131072),
    (8192, 64, 8, 2, 32768), (1, 64, 8, 2, 524288), (3, 8, 8, 1, 1 << 22), (2, 8, 1, 2048, 1 << 20)])
def test_weights_workspace_has_a_bound(built_lib, B, H, HK, ql, tokens):
    """Wide tables: some sequences at a time, whatever the batch.  What one sequence needs with 1024 rows lies within it here."""
    from specq import _lib
    assert _lib.lib().specq_paged_attn_weights_workspace_size(B, H, HK, ql, tokens // 16, 16) <= (256 << 20) + (256 << 10) + 4096


def _evict(n=1, base=(4096,), sp=(16 * 1024,), so=(1024,), sh=(128,), rb=(128,), **kw):
    keep = [np.asarray(v, np.int64) for v in (base, sp, so, sh, rb)]
    a = dict(bt=16, s_bt=64, B=2, C=64, ref=0, P=100, ctx=16, w=16, s_wb=8 * 1024, s_wh=1024, HK=8, PAGE=16, n=n,
             base=keep[0].ctypes.data, sp=keep[1].ctypes.data, so=keep[2].ctypes.data, sh=keep[3].ctypes.data,
             rb=keep[4].ctypes.data, budget=100, recent=10, sinks=4, limit=100, kept=16, ws=0, wsb=0, stream=0)
    a.update(kw)
    return keep, a


def test_evict_refusals(built_lib):
    def f(code, **kw):
        keep, a = _evict(**kw)
        _fail("specq_kv_evict", a, code)
        del keep

    for name in ("bt", "ctx", "w", "kept"):
        f(-22, **{name: 0})
    f(-22, B=0), f(-22, HK=0), f(-22, C=0), f(-22, P=0), f(-22, PAGE=0), f(-22, C=65), f(-95, C=1 << 27, s_bt=1 << 27)
    f(-22, budget=0), f(-22, recent=-1), f(-22, sinks=-1), f(-22, recent=97), f(-22, recent=2 ** 31 - 1, sinks=2 ** 31 - 1), f(-22, limit=99)
    f(-95, budget=(1 << 30) + 1, limit=2 ** 31 - 1)
    f(-95, s_wb=1024, s_wh=1024), f(-95, sp=(15 * 1024 + 128,)), f(-95, so=(512,)), f(-28, so=(128,), sh=(2048,))
    f(-95, w=18), f(-95, s_wb=0), f(-95, s_wh=1023), f(-95, n=17), f(-95, n=-1)
    f(-22, base=(0,)), f(-22, rb=(0,)), f(-22, rb=(4097,)), f(-95, sp=(0,)), f(-95, so=(127,)), f(-95, sh=(64,))
    two = dict(n=2, sp=(16384, 16384), so=(1024, 1024), sh=(128, 128), rb=(128, 128))
    f(-22, base=(4096, 4096), **two)
    f(-28), f(-28, ws=4096, wsb=1000)
    f(-28, base=(4096, 1 << 20), **two)


def test_rows_far_apart_and_overlapping(built_lib):
    """Strides whose extents pass 64 bits do not hide rows that overlap."""
    f = lambda code, **kw: _fail("specq_paged_attn_weights", WEIGHTS, code, B=9, n_seqs=9, H=36, HK=9, **kw)  # noqa: E731
    f(-95, s_wb=1 << 62, s_wh=1 << 62)  # one stride for both: eight steps of it are 2^65
    f(-95, s_wb=-(1 << 62), s_wh=1 << 62), f(-95, s_wb=-(1 << 63), s_wh=-(1 << 63))
    f(-28, s_wb=9 * 1024, s_wh=-1024)   # apart; no workspace


def test_evict_refuses_what_a_launch_does_not_take_before_the_first(built_lib):
    """A selection of 2^32 threads and more, and a move of them behind a selection that could have run."""
    for kw in (dict(B=1 << 19), dict(B=1 << 17, sp=(16 * 8 * 4096,), so=(8 * 4096,), sh=(4096,), rb=(4096,))):
        keep, a = _evict(**kw, ws=4096, wsb=1 << 40)
        _fail("specq_kv_evict", a, -95)
        del keep


def test_beam_refusals(built_lib):
    base = dict(x=16, f32=0, s_lb=4 * 1000, s_lw=1000, scores=16, s_sb=4, done=0, s_fb=4, eos=0, os=16, ot=16, op=16, B=2, W=4,
                V=1000, n=4, ws=0, wsb=0, stream=0)
    f = lambda code, **kw: _fail("specq_beam_select", base, code, **kw)  # noqa: E731
    for name in ("x", "scores", "os", "ot", "op"):
        f(-22, **{name: 0})
    f(-22, W=0), f(-22, V=0), f(-22, n=0), f(-95, W=65), f(-95, n=65), f(-95, V=(1 << 28) + 1), f(-95, B=1 << 30)
    f(-22, done=16, eos=-1), f(-22, done=16, eos=1000), f(-22, x=17), f(-22, f32=1, x=18), f(-22, scores=18)
    f(-28), f(-28, ws=4096, wsb=200000)
    f(0, B=0)
    keep = [np.asarray(v, np.int64) for v in ((4096, 8192), (128, 128), (128, 128))]
    states = dict(parents=16, rows=8, group=4, n=2, base=keep[0].ctypes.data, stride=keep[1].ctypes.data,
                  bytes=keep[2].ctypes.data, stream=0)
    g = lambda code, **kw: _fail("specq_beam_reorder", states, code, **kw)  # noqa: E731
    g(-22, parents=0), g(-22, rows=-4), g(-22, rows=7), g(-22, group=0), g(-95, rows=33, group=33), g(-22, n=-1), g(-22, base=0)
    g(0, rows=0), g(0, group=1), g(0, n=0)
    for i, v in ((0, (4096, 0)), (0, (4096, 16)), (0, (4096, 4096)), (1, (128, 64)), (2, (128, 0)), (1, (-128, 128))):
        bad = np.asarray(v, np.int64)
        g(-22, **{("base", "stride", "bytes")[i]: bad.ctypes.data})
    wide = np.full(2, 1 << 50, np.int64)
    g(-95, stride=wide.ctypes.data, bytes=wide.ctypes.data)


def test_launches_past_their_size(built_lib):
    """More threads than a launch takes are refused ahead of it."""
    _fail("specq_qk_norm_rotary", NORM, -95, B=1 << 13, ql=1 << 13, n_seqs=0, q_len=0, R=20, f=0, i=64, h=512, m=64)
    keep = [np.asarray([v], np.int64) for v in (4096, 1 << 36, 1 << 36)]
    _fail("specq_beam_reorder", dict(parents=16, rows=1 << 7, group=2, n=1, base=keep[0].ctypes.data, stride=keep[1].ctypes.data,
                                     bytes=keep[2].ctypes.data, stream=0), -95)


def test_reorder_refuses_before_its_first_launch(built_lib):
    """Of more states than a launch takes the last is too large: refused for that, not by the first launch."""
    n = 65
    base, stride = np.arange(4096, 4096 + 4096 * n, 4096, dtype=np.int64), np.full(n, 1 << 50, np.int64)
    size = np.full(n, 128, np.int64)
    size[-1] = 1 << 45
    _fail("specq_beam_reorder", dict(parents=16, rows=4, group=2, n=n, base=base.ctypes.data, stride=stride.ctypes.data,
                                     bytes=size.ctypes.data, stream=0), -95)


def test_sizes_past_their_types(built_lib):
    from specq import _lib
    for name, args, word in (("specq_qk_norm_rotary", NORM, "B"), ("specq_paged_attn_weights", WEIGHTS, "ql")):
        with pytest.raises(RuntimeError, match="out of its type"):
            _lib.packed(name)(*dict(args, **{word: 1 << 33}).values())


def test_kernels_keep_to_their_registers(built_lib):
    """The compiler's report beside the library: none of these kernels spills."""
    report = os.path.join(os.path.dirname(built_lib), "libspecq.resources.txt")
    if not os.path.exists(report):
        pytest.skip("library without its report")
    ours = re.compile(r"qk_norm_(vec|any)_kernel|aw_\w+_kernel|evict_\w+_kernel|beam_(part|join|reorder)_kernel")
    scratch, name = {}, ""
    for line in open(report):
        if m := re.search(r"Function Name: (\S+)", line):
            name = m.group(1)
        elif (m := re.search(r"ScratchSize \[bytes/lane\]: (\d+)", line)) and ours.search(name):
            scratch[name] = int(m.group(1))
    assert len(scratch) >= 12 + 21 + 5 + 9
    assert not any(scratch.values()), scratch


def test_python_entry_points_want_gpu_tensors():
    import kernels as K
    z, f = torch.zeros((1, 1, 2, 64), dtype=torch.float16), torch.zeros((1, 2, 64))
    i = torch.zeros(1, dtype=torch.int32)
    for fn, args in [(K.qk_norm_rotary, (z, z, None, None, torch.ones(32), i)), (K.paged_attention_weights, (z, z, z, i, i, f)),
                     (K.paged_kv_evict, (i[None], i, f, [z], 16, 4)), (K.beam_select, (f, f[0])), (K.beam_reorder, ([f], i, 1))]:
        with pytest.raises(RuntimeError, match="GPU only"):
            fn(*args)


def test_every_tensor_is_held_to_one_gpu(monkeypatch):
    """Nothing is launched: whatever a call would hand to a kernel has been through the check of its device."""
    import kernels as K
    held, calls = [], []
    monkeypatch.setattr(K, "_gpu_of", lambda who, *ts: held.extend(t.data_ptr() for t in ts if t is not None) or 0)
    monkeypatch.setattr(K, "_call_on", lambda dev, name, *args: calls.append((name, args)))
    monkeypatch.setattr(K, "_workspace", lambda ws, dev: type("W", (), {"ensure": staticmethod(lambda n: (0, 0))}))
    monkeypatch.setattr(K, "_beam_workspace", lambda *a: 0)
    monkeypatch.setattr(K, "_evict_workspace", lambda *a: 0)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, k, w = torch.zeros((2, 3, 8, 64)).half(), torch.zeros((2, 3, 2, 64)).half(), torch.ones(64)
    qo, ko, wk, freq, ctx, pos, plan = q.clone(), k.clone(), w.clone(), torch.ones(32), i32(2), i32(2, 3), i32(2)
    kc, ks, tbl, gathered = torch.zeros((5, 16, 2, 64), dtype=torch.int8), torch.zeros((5, 16, 2)), i32(2, 4), torch.zeros((2, 2, 64))
    lens, ref, kept = i32(2), i32(5), i32(2, 2, 8)
    logits, scores, done = torch.zeros((2, 3, 9)), torch.zeros((2, 3)), torch.zeros((2, 3), dtype=torch.bool)
    out = (torch.zeros((2, 3)), i32(2, 3), i32(2, 3))
    a, b, parents = torch.zeros((6, 2)), torch.zeros((6, 3)), i32(6)
    for call, given in [
            (lambda: K.qk_norm_rotary(q, k, w, wk, freq, ctx, plan=plan, q_out=qo, k_out=ko), (q, k, w, wk, freq, ctx, plan, qo, ko)),
            (lambda: K.qk_norm_rotary(q, k, w, wk, freq, positions=pos), (q, k, w, wk, freq, pos)),
            (lambda: K.paged_attention_weights(q, kc, ks, tbl, ctx, gathered, q_lens=lens, plan=plan),
             (q, kc, ks, tbl, ctx, gathered, lens, plan)),
            (lambda: K.paged_kv_evict(tbl, ctx, gathered, [kc, ks], 16, 8, ref=ref, kept=kept), (tbl, ctx, gathered, kc, ks, ref, kept)),
            (lambda: K.beam_select(logits, scores, 3, done, 1, out=out), (logits, scores, done, *out)),
            (lambda: K.beam_reorder([a, b], parents, 3), (a, b, parents))]:
        held.clear()
        call()
        assert {t.data_ptr() for t in given} <= set(held), calls[-1][0]
    assert len(calls) == 6


def test_a_workspace_on_another_device_is_refused(monkeypatch):
    import kernels as K
    from specq.workspace import Workspace
    calls = []
    monkeypatch.setattr(K, "_gpu_of", lambda who, *ts: 0)
    monkeypatch.setattr(K, "_call_on", lambda dev, name, *args: calls.append(name))
    monkeypatch.setattr(K, "_beam_workspace", lambda *a: 1 << 20)
    monkeypatch.setattr(K, "_evict_workspace", lambda *a: 1 << 20)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, kc, ks = torch.zeros((2, 3, 8, 64)).half(), torch.zeros((5, 16, 2, 64), dtype=torch.int8), torch.zeros((5, 16, 2))
    for call in (lambda: K.paged_attention_weights(q, kc, ks, i32(2, 4), i32(2), torch.zeros((2, 2, 64)), workspace=Workspace("cuda:1")),
                 lambda: K.paged_kv_evict(i32(2, 4), i32(2), torch.zeros((2, 2, 64)), [kc], 16, 8, workspace=Workspace("cpu")),
                 lambda: K.beam_select(torch.zeros((2, 3, 9)), torch.zeros((2, 3)), workspace=Workspace("cuda:1"))):
        with pytest.raises(RuntimeError, match="workspace"):
            call()
    assert not calls


def test_plain_weights_are_probabilities():
    """Each row that sees a token gives 1 in all."""
    rng = np.random.default_rng(0)
    q = rng.standard_normal((2, 3, 4, 64)).astype(np.float16)
    kc, ks = rng.integers(-127, 128, (6, 16, 2, 64), dtype=np.int8), np.full((6, 16, 2), 0.01, np.float32)
    bt = np.array([[3, 1, -1], [5, -1, 9]], np.int32)
    w, _ = O.attn_weights(q, kc, ks, bt, np.array([30, 2]), np.zeros((2, 2, 48)), [3, 3], 0.1)
    assert np.allclose(w[0].sum(-1), 3 * 2) and np.allclose(w[1].sum(-1), 2 * 2)  # the second's first row sees nothing
    assert (w[0, :, 30:] == 0).all() and (w[1, :, 2:] == 0).all()


def test_plain_eviction_known_answer():
    bt, ctx, w = np.array([[1, 0]], np.int32), np.array([6], np.int32), np.array([[[5, 1, 9, 2, 9, 0, 7, 7]]], np.float32)
    cache = np.arange(8).reshape(2, 4, 1)  # position t lies in page 1 - t // 4
    kept, ctx, w, (c,) = O.evict(bt, ctx, w, [cache], 3, 1, 0, 3)
    assert kept.tolist() == [[[2, 4, 5]]] and ctx.tolist() == [3]
    assert c[1, :, 0].tolist() == [6, 0, 1, 7] and w[0, 0].tolist() == [9, 9, 0, 2, 9, 0, 7, 7]


def test_plain_beams_known_answer():
    x = np.log(np.array([[[0.5, 0.25, 0.25], [0.1, 0.8, 0.1]]]))
    score, token, parent, behind = O.beam_select(x, np.log(np.array([[0.5, 0.5]])), 3)
    assert token.tolist() == [[1, 0, 1]] and parent.tolist() == [[1, 0, 0]]
    assert np.allclose(np.exp(score), [[0.4, 0.25, 0.125]]) and np.allclose(np.exp(behind), 0.125)
    _, token, parent, _ = O.beam_select(x, np.log(np.array([[0.5, 0.5]])), 5, np.array([[True, False]]), 2)
    assert token.tolist() == [[2, 1, 0, 2, -1]] and parent.tolist() == [[0, 1, 1, 1, -1]]
    assert [a.tolist() for a in O.reorder([np.arange(4)], [1, -1, 2, 0], 2)] == [[1, 1, 2, 3]]
