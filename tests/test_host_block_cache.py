"""CPU tier of the block-scaled cache, rotary and page-table entry points: refusals ahead of any launch, the rotary
frequencies, and the plain implementations' own properties."""
import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

from oracle import cache_ops as C

# Pointers are fake: every call below must fail validation (or have nothing to do), so nothing is launched.


def _fail(name, args, code, **change):
    from specq import _lib
    a = dict(args)
    a.update(change)
    rc = getattr(_lib.lib(), name)(*a.values())
    assert rc == code, (name, change, rc, _lib.lib().specq_last_error())


ATTN = dict(q=16, s_qb=9 * 4096, s_qt=4096, s_qh=128, kc=16, vc=16, f8=1, s_kp=16 * 1024, s_ko=1024, s_kh=128, ks=16, vs=16,
            s_sp=8, s_sb=8, s_sh=1, block=16, bt=16, s_bt=64, max_pages=64, n_pages=100, ctx=16, out=16, s_ob=9 * 4096,
            s_ot=4096, s_oh=128, B=2, n_seqs=2, q_len=9, ql=9, H=32, HK=8, D=128, PAGE=16, QPP=9, sm=0.088, plan=0, ws=0,
            wsb=0, stream=0)


def test_attention_refusals(built_lib):
    f = lambda code, **kw: _fail("specq_paged_attn_block", ATTN, code, **kw)  # noqa: E731
    for name in ("q", "kc", "vc", "ks", "vs", "bt", "ctx", "out"):
        f(-22, **{name: 0})
    f(-95, D=96), f(-95, block=8), f(-95, block=0), f(-95, block=32), f(-95, block=-16), f(-95, PAGE=24, block=24)
    f(-95, PAGE=40, block=8), f(-95, QPP=17), f(-22, QPP=0), f(-22, H=30), f(-22, n_seqs=3), f(-22, q_len=10)
    f(-22, max_pages=0), f(-22, n_pages=0), f(-95, max_pages=1 << 20), f(-95, q=24), f(-95, kc=24), f(-95, s_kp=1000)
    f(-95, out=8), f(-22, ks=18), f(-95, s_ko=1 << 27), f(-28, max_pages=1024)
    f(0, B=0, n_seqs=0)


APPEND = dict(k=16, v=16, s_nb=9 * 1024, s_nt=1024, s_nh=128, kc=16, vc=16, f8=0, s_kp=16 * 1024, s_ko=1024, s_kh=128, ks=16,
              vs=16, s_sp=16, s_sb=8, s_sh=1, block=16, bt=16, s_bt=64, max_pages=64, n_pages=100, ctx=16, B=2, n_seqs=2,
              q_len=9, ql=9, HK=8, D=128, PAGE=32, plan=0, stream=0)
ROTARY = dict(q=16, a=1024, b=512, c=64, k=16, d=256, e=128, f=64, qo=16, g=1024, h=512, i=64, ko=16, j=256, l=128, m=64,
              freq=16, f64=1, ms=1.0, ctx=16, pos=0, s_pb=0, B=2, n_seqs=2, q_len=2, ql=2, H=8, HK=2, D=64, R=64, il=0,
              plan=0, stream=0)


def test_outputs_that_name_a_place_twice_are_refused(built_lib):
    """Expanded tensors (a stride of 0) and rows closer than they are long: workgroups would write over one another.  A
    dimension of one entry may have any stride."""
    none = dict(n_seqs=0)  # what is not refused has nothing to do
    for k in ("g", "h", "i", "j", "l", "m"):
        _fail("specq_rotary", ROTARY, -95, **{k: 0}), _fail("specq_rotary", ROTARY, -95, **{k: 56})
    for k in ("s_ob", "s_ot", "s_oh"):
        _fail("specq_paged_attn_block", ATTN, -95, **{k: 0}), _fail("specq_paged_attn_block", ATTN, -95, **{k: 64})
    _fail("specq_paged_attn_block", ATTN, 0, q_len=1, ql=1, QPP=1, s_ot=0, **none)
    for k in ("s_kp", "s_ko", "s_kh", "s_sp", "s_sb", "s_sh"):
        _fail("specq_kv_append_block", APPEND, -95, **{k: 0})
        if k[2] == "k":
            _fail("specq_kv_append_block", APPEND, -95, **{k: 64})
    _fail("specq_kv_append_block", APPEND, 0, s_sb=0, block=32, **none)
    _fail("specq_kv_append_block", APPEND, 0, s_sp=0, s_kp=0, n_pages=1, **none)
    _fail("specq_kv_append_block", APPEND, 0, s_sh=0, s_kh=0, HK=1, **none)


def test_append_refusals(built_lib):
    base = dict(k=16, v=16, s_nb=9 * 1024, s_nt=1024, s_nh=128, kc=16, vc=16, f8=0, s_kp=16 * 1024, s_ko=1024, s_kh=128, ks=16,
                vs=16, s_sp=8, s_sb=8, s_sh=1, block=16, bt=16, s_bt=64, max_pages=64, n_pages=100, ctx=16, B=2, n_seqs=2,
                q_len=9, ql=9, HK=8, D=128, PAGE=16, plan=0, stream=0)
    f = lambda code, **kw: _fail("specq_kv_append_block", base, code, **kw)  # noqa: E731
    for name in ("k", "v", "kc", "vc", "ks", "vs", "bt", "ctx"):
        f(-22, **{name: 0})
    f(-95, D=96), f(-95, block=8), f(-95, block=32), f(-95, k=24), f(-95, s_nt=1001), f(-95, kc=20), f(-95, s_kh=100)
    f(-95, ks=18), f(-22, n_seqs=3), f(-22, q_len=10), f(-22, HK=0), f(-22, n_pages=0)
    f(-95, max_pages=1 << 28, s_bt=1 << 28)
    f(0, B=0, n_seqs=0), f(0, q_len=0)


def test_rotary_refusals(built_lib):
    base = dict(q=16, a=512, b=512, c=64, k=16, d=128, e=128, f=64, qo=16, g=512, h=512, i=64, ko=16, j=128, l=128, m=64,
                freq=16, f64=1, ms=1.0, ctx=16, pos=0, s_pb=0, B=2, n_seqs=2, q_len=1, ql=1, H=8, HK=2, D=64, R=64, il=0,
                plan=0, stream=0)
    f = lambda code, **kw: _fail("specq_rotary", base, code, **kw)  # noqa: E731
    f(-22, q=0), f(-22, qo=0), f(-22, k=0), f(-22, ko=0), f(-22, freq=0), f(-22, ctx=0), f(-22, R=0), f(-22, R=7)
    f(-22, R=66), f(-95, D=514), f(-22, n_seqs=3), f(-22, q_len=2), f(-22, H=0), f(0, B=0, n_seqs=0), f(0, q_len=0, ql=0)
    f(-22, B=1 << 20, ql=1 << 12, q_len=1)


def test_pages_refusals(built_lib):
    t = dict(bt=16, s_bt=8, B=4, C=8, ref=16, P=100)
    ws = dict(ws=16, wsb=1 << 30, stream=0)
    arr = lambda ct, *v: (ct * len(v))(*v)  # noqa: E731
    tensors = dict(n=1, base=arr(ctypes.c_void_p, 16), stride=arr(ctypes.c_int64, 64), bytes=arr(ctypes.c_int64, 64))
    calls = {
        "specq_kv_pages_reserve": dict(t, lens=16, PAGE=16, short=16, **ws),
        "specq_kv_pages_free": dict(t, keep=16, PAGE=16, stream=0),
        "specq_kv_pages_fork": dict(t, lens=16, parent=16, PAGE=16, **tensors, short=16, **ws),
        "specq_kv_pages_compact": dict(t, map=16, **tensors, **ws),
    }
    for name, base in calls.items():
        for k in ("bt", "ref", "lens", "keep", "parent", "short", "map"):
            if k in base:
                _fail(name, base, -22, **{k: 0})
        _fail(name, base, -22, B=0), _fail(name, base, -22, C=0), _fail(name, base, -22, P=0), _fail(name, base, -22, s_bt=7)
        _fail(name, base, -95, P=2 ** 31 - 1)
        if "PAGE" in base:
            _fail(name, base, -22, PAGE=0), _fail(name, base, -95, PAGE=1 << 30)
        if "wsb" in base:
            _fail(name, base, -28, wsb=1 << 18), _fail(name, base, -28, ws=0)
        if "n" in base:
            _fail(name, base, -22, n=-1), _fail(name, base, -22, base=None)
            _fail(name, base, -22, base=arr(ctypes.c_void_p, None)), _fail(name, base, -22, stride=arr(ctypes.c_int64, 60))
            _fail(name, base, -22, bytes=arr(ctypes.c_int64, 0))
    copy = dict(src=16, dst=16, n=3, P=10, m=1, base=tensors["base"], stride=tensors["stride"], bytes=tensors["bytes"], stream=0)
    f = lambda code, **kw: _fail("specq_kv_pages_copy", copy, code, **kw)  # noqa: E731
    f(-22, src=0), f(-22, dst=0), f(-22, n=-1), f(-22, P=0), f(-22, m=-1), f(0, n=0), f(0, m=0)
    from specq import _lib
    size = _lib.lib().specq_kv_pages_workspace_size
    assert size(0, 1, 1) == 0 and size(4, 8, 100) >= 256 * 1024 + 4 * (4 * 8 + 3 * 4 + 3 * 100)


def test_sizes_past_their_types(built_lib):
    _fail("specq_paged_attn_block", ATTN, -95, s_ko=112), _fail("specq_paged_attn_block", ATTN, -95, QPP=1 << 30)
    free = dict(bt=16, s_bt=1 << 31, B=4, C=(1 << 30) + 1, ref=16, P=100, keep=16, PAGE=1, stream=0)
    _fail("specq_kv_pages_free", free, -95)
    from specq import _lib
    words = list(ATTN.values())
    with pytest.raises(RuntimeError, match="range"):
        _lib.packed("specq_paged_attn_block")(*[w if k != "n_pages" else 2 ** 32 + 100 for k, w in zip(ATTN, words)])
    with pytest.raises(RuntimeError, match="arguments"):
        _lib.check(_lib.lib().specq_call_packed(b"specq_rotary", b"\0" * 64, 8), "specq_rotary")
    with pytest.raises(RuntimeError, match="no entry point"):
        _lib.check(_lib.lib().specq_call_packed(b"specq_version", b"\0" * 8, 1), "specq_version")


def test_kernels_keep_to_their_registers(built_lib):
    """The compiler's report beside the library: bytes of scratch a lane, for all kernels of these operators.  The e4m3
    programs of 64 rows at head dim 128 spill."""
    report = os.path.join(os.path.dirname(built_lib), "libspecq.resources.txt")
    if not os.path.exists(report):
        pytest.skip("library without its report")
    ours = re.compile(r"attn_block_(plan_)?kernel|attn_merge_kernel|rotary_(vec|any)_kernel|kv_append_block_kernel|pages_\w+_kernel")
    scratch, name = {}, ""
    for line in open(report):
        if m := re.search(r"Function Name: (\S+)", line):
            name = m.group(1)
        elif (m := re.search(r"ScratchSize \[bytes/lane\]: (\d+)", line)) and ours.search(name):
            scratch[name] = int(m.group(1))
    assert len(scratch) >= 28 + 2 + 4 + 10 + 6
    most = {"attn_block_kernelILi128ELi4ELb1E": 96, "attn_block_plan_kernelILi128ELi4ELb1E": 108}
    for name, n in scratch.items():
        assert n <= max([v for k, v in most.items() if k in name], default=0), (name, n)


def test_reserve_refuses_more_entries_than_it_counts(built_lib):
    """Wants are counted in 32 bits: a table of 2^32 entries that all want a page would count them past it, and take
    places before the list of free pages."""
    base = dict(bt=16, s_bt=1 << 20, B=4096, C=1 << 20, ref=16, P=100, lens=16, PAGE=1, short=16, ws=16, wsb=1 << 20, stream=0)
    for B, C in ((4096, 1 << 20), (2048, 1 << 20), (1 << 30, 2), ((1 << 31) - 1, 1 << 5)):
        _fail("specq_kv_pages_reserve", base, -95, B=B, C=C)
    _fail("specq_kv_pages_reserve", base, -28, B=2047)  # 2^31 - 2^20 entries are counted


def test_python_entry_points_want_gpu_tensors():
    import kernels as K
    z = torch.zeros((1, 1, 2, 64), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    for f, args in [(K.rotary_embed, (z, z, torch.ones(32), i)), (K.paged_kv_reserve, (i[None], i, i, 16)),
                    (K.paged_attention_block_scaled, (z, z, z, z, z, i, i)), (K.paged_kv_copy, (i, i, [z])),
                    (K.paged_kv_append_block_scaled, (z, z, z, z, z, z, i, i))]:
        with pytest.raises(RuntimeError, match="GPU only"):
            f(*args)
    with pytest.raises(RuntimeError):
        K.paged_kv_copy(i, i, [])


def test_every_tensor_is_held_to_one_gpu(monkeypatch):
    """Nothing is launched: whatever a call would hand to a kernel has been through the check of its device."""
    import kernels as K
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    tbl, ref, lens, parent, short, where = i32(3, 4), i32(10), i32(3), i32(3), i32(1), i32(10)
    held, calls = [], []
    monkeypatch.setattr(K, "_gpu_of", lambda who, *ts: held.extend(t.data_ptr() for t in ts if t is not None) or 0)
    monkeypatch.setattr(K, "_call_on", lambda dev, name, *args: calls.append(name))
    monkeypatch.setattr(K, "_pages_workspace", lambda *a: (0, 0))
    for call, given in [(lambda: K.paged_kv_reserve(tbl, ref, lens, 16, shortage=short), (tbl, ref, lens, short)),
                        (lambda: K.paged_kv_free(tbl, ref, lens, 16), (tbl, ref, lens)),
                        (lambda: K.paged_kv_fork(tbl, ref, lens, parent, [], 16, shortage=short), (tbl, ref, lens, parent, short)),
                        (lambda: K.paged_kv_compact(tbl, ref, [], page_map=where), (tbl, ref, where))]:
        held.clear()
        call()
        assert {t.data_ptr() for t in given} <= set(held), calls[-1]
    assert len(calls) == 4


def test_a_workspace_on_another_device_is_refused(monkeypatch):
    """On the host memory's, or another GPU's: nothing is launched with its address."""
    import kernels as K
    from specq.workspace import Workspace
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    tbl, ref, lens = i32(3, 200), i32(10), i32(3)
    q = torch.zeros((3, 1, 8, 64), dtype=torch.float16)
    kc, ks = torch.zeros((10, 16, 8, 64), dtype=torch.int8), torch.zeros((10, 1, 8))
    calls = []
    monkeypatch.setattr(K, "_gpu_of", lambda who, *ts: 0)
    monkeypatch.setattr(K, "_call_on", lambda dev, name, *args: calls.append(name))
    monkeypatch.setattr(K, "_block_attn_info", lambda *a: None)
    monkeypatch.setattr(K, "_block_attn_workspace", lambda *a: 1 << 20)
    far = Workspace("cuda:1")
    far._buf = torch.zeros(1 << 22, dtype=torch.uint8)  # stands for memory of that GPU
    for ws in (Workspace("cpu"), far):
        for call in (lambda: K.paged_kv_reserve(tbl, ref, lens, 16, workspace=ws),
                     lambda: K.paged_kv_fork(tbl, ref, lens, lens.clone(), [], 16, workspace=ws),
                     lambda: K.paged_kv_compact(tbl, ref, [], workspace=ws),
                     lambda: K.paged_attention_block_scaled(q, kc, kc, ks, ks, tbl, lens, workspace=ws)):
            with pytest.raises(RuntimeError, match="workspace"):
                call()
    assert not calls


@pytest.mark.parametrize("dim", [2, 20, 64, 128])
def test_rotary_frequencies(dim):
    import kernels as K
    f, m = K.rotary_inv_freq(dim, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    assert np.allclose(f.numpy(), [10000.0 ** (-2 * j / dim) for j in range(dim // 2)], rtol=1e-14, atol=0)
    assert np.allclose(K.rotary_inv_freq(dim, scaling="linear", factor=4, device="cpu")[0].numpy(), f.numpy() / 4, rtol=1e-14)
    w, _ = K.rotary_inv_freq(dim, scaling="wavelength", factor=8.0, original_len=8192, device="cpu")
    for a, b in zip(w.tolist(), f.tolist()):
        turns = 8192 * b / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / 3))
        assert math.isclose(a, b * keep + b / 8 * (1 - keep), rel_tol=1e-13)
    y, my = K.rotary_inv_freq(dim, scaling="yarn", factor=8.0, original_len=8192, device="cpu")
    assert math.isclose(my, 0.1 * math.log(8) + 1) and math.isclose(float(y[0]), float(f[0]), rel_tol=1e-13) or dim <= 4
    assert bool((y <= f * (1 + 1e-12)).all()) and bool((y >= f / 8 * (1 - 1e-12)).all())
    if dim > 2:
        n, _ = K.rotary_inv_freq(dim, scaling="ntk", factor=4.0, device="cpu")
        assert math.isclose(float(n[-1]), float(f[-1]) / 4, rel_tol=1e-12) and float(n[0]) == 1.0


@pytest.mark.parametrize("dim,base,length,factor", [
    (128, 10000.0, 4096, 8.0), (128, 500000.0, 131072, 4.0), (64, 1000000.0, 32768, 4.0), (20, 10000.0, 8192, 8.0),
    # The ramp ends past the last pair: that pair still turns more than beta_slow times.
    (8, 10000.0, 8192, 8.0), (6, 10000.0, 8192, 8.0), (4, 10000.0, 8192, 8.0), (64, 10000.0, 65536, 8.0),
    (128, 10000.0, 131072, 8.0), (128, 10000.0, 1 << 20, 40.0),
    (2, 10000.0, 100000, 8.0),  # ... and would end past dim - 1, where it is cut
])
def test_yarn_frequencies_are_the_closed_form(dim, base, length, factor):
    """Every pair: the ramp runs from the pair that turns 32 times in `length` tokens, rounded down, to the one that
    turns once, rounded up, within [0, dim - 1]; it may end past the last pair, dim / 2 - 1.  fp64 on both sides, some ten
    operations of half an ulp each: 1e-13 covers them."""
    import kernels as K
    pair = lambda turns: dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
    y, m = K.rotary_inv_freq(dim, base=base, scaling="yarn", factor=factor, original_len=length, device="cpu")
    assert m == 0.1 * math.log(factor) + 1.0 and len(y) == dim // 2
    for j in range(dim // 2):
        f = base ** (-2.0 * j / dim)
        ramp = min(1.0, max(0.0, (j - lo) / (hi - lo if hi > lo else 1e-3)))
        assert math.isclose(float(y[j]), f * (1 - ramp) + f / factor * ramp, rel_tol=1e-13), j
        if length * f / (2 * math.pi) > 1 and dim > 2:  # turns more than beta_slow times: not divided in full
            assert float(y[j]) > f / factor * (1 + 1e-9), j


def test_rotary_frequency_refusals():
    import kernels as K
    for kw in (dict(dim=0), dict(dim=3), dict(dim=64, scaling="cubic"), dict(dim=64, base=1.0), dict(dim=64, factor=0.0),
               dict(dim=2, scaling="ntk"), dict(dim=64, scaling="wavelength", high_freq_factor=1.0)):
        with pytest.raises(RuntimeError):
            K.rotary_inv_freq(device="cpu", **kw)


def test_refusals_are_runtime_errors(monkeypatch):
    """No query heads; yarn's numbers of turns that have no logarithm or no order."""
    import kernels as K
    monkeypatch.setattr(K, "_gpu_of", lambda who, *ts: 0)
    monkeypatch.setattr(K, "_call_on", lambda dev, name, *args: None)
    q, kc, ks = torch.zeros((1, 1, 0, 64), dtype=torch.float16), torch.zeros((2, 16, 2, 64), dtype=torch.int8), torch.zeros((2, 1, 2))
    with pytest.raises(RuntimeError, match="does not fit"):
        K.paged_attention_block_scaled(q, kc, kc, ks, ks, torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    for kw in (dict(beta_slow=0.0), dict(beta_slow=-1.0), dict(beta_fast=0.0), dict(beta_fast=1.0, beta_slow=2.0)):
        with pytest.raises(RuntimeError, match="beta"):
            K.rotary_inv_freq(64, scaling="yarn", factor=4.0, device="cpu", **kw)


def test_e4m3_codes_are_torchs():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(t, C.E4M3.astype(np.float32), equal_nan=True)
    x = np.concatenate([np.random.default_rng(0).standard_normal(20000) * 80, C.E4M3[:126] / 2 + C.E4M3[1:127] / 2])
    x = np.clip(x, -448, 448).astype(np.float32)
    assert np.array_equal(torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), C.encode(x.astype(np.float64), "fp8"))


def test_plain_codes_of_nan():
    assert np.isnan(C.decode(C.encode(np.asarray([np.nan, -np.nan, 1.0]), "fp8"), "fp8")).tolist() == [True, True, False]


def test_plain_append_holds_half_a_step():
    rng = np.random.default_rng(1)
    kc, ks = np.zeros((3, 32, 1, 8), np.int8), np.zeros((3, 2, 1), np.float32)
    bt = np.asarray([[2, 0]], np.int32)
    out = (kc, kc, ks, ks)
    for n in range(1, 40):
        k = (rng.standard_normal((1, 1, 1, 8)) * n).astype(np.float16)
        out = C.append_block(k, -k, *out, bt, np.asarray([n], np.int32), 1, "int8")
        got = out[0][bt[0, (n - 1) // 32], (n - 1) % 32, 0] * out[2][bt[0, (n - 1) // 32], (n - 1) % 32 // 16, 0]
        assert (np.abs(got - k[0, 0, 0]) <= out[2][bt[0, (n - 1) // 32], (n - 1) % 32 // 16, 0] * 0.5001).all()
    assert np.array_equal(out[0], -out[1]) and np.array_equal(out[2], out[3])
