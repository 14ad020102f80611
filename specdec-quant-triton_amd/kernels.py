"""Quantized speculative-decoding verification kernels for MI355X (gfx950).

Drop-in counterpart of the reference's kernels.py: the same public names, signatures,
defaults and return values, so correctness and benchmark scripts written against the
reference run unchanged (`from kernels import *`).  The kernels themselves are hand-written
HIP for gfx950 in csrc/, reached through the C ABI of libspecq.so (include/specq.h):

  w8a8_matmul      INT8 x INT8 -> INT32 MFMA GEMM, per-token x per-channel scale epilogue
                   (reference kernels.py:27-55, 71-86)
  w4a16_matmul     packed-INT4 (group scales) x FP16 GEMM, dequantised once per weight
                   element and fed to FP16 MFMA (reference kernels.py:94-135, 150-166)
  paged_attention  INT8 paged-KV verification attention, GQA x (k+1) rows packed per
                   program, QPP=1 (decode style) or QPP=q_len (fused)
                   (reference kernels.py:178-236, 239-262)

and the steps either side of them on the device: paged_kv_append (the new tokens' K/V
quantised into the cache pages, the q8 of kernels.py:280-284), silu_mul /
silu_mul_quant_int8 / quantize_act_int8_gpu (kernels.py:58-62 on the device), and
w4a8_matmul (INT4 weights on the INT8 MFMA path, the reference's REPORT.md:156
recommendation; no reference kernel).  Without a reference counterpart: rotary_embed (positions
of q and k), paged_kv_append_block_scaled and paged_attention_block_scaled (an int8 or e4m3
cache with one scale for each block of tokens and head), the cache's page tables,
paged_kv_reserve / _free / _fork / _compact / _copy, qk_norm_rotary (norms of q and k for each head with
their positions), paged_attention_weights and paged_kv_evict (the attention weight that cached tokens
gather, and eviction by it), and beam search, beam_select and beam_reorder.

Every launcher takes `plan` (an int32 device tensor read by the kernel at run time) and a
fixed grid size, so a single captured graph replays every (B, k) (reference kernels.py:14-17).
Launches go to torch's current stream and never synchronise or allocate (except the
optional output allocation and the first growth of the shared workspace).

The host-side helpers (quantizers, INT4 packer, paged-KV generator, dense attention
reference) restate the reference formulas in torch and run on any device.

Differences a caller may notice:
  * BLOCK_K and num_stages are accepted and ignored (the MFMA K step and register
    pipelining are fixed per kernel).  BLOCK_M=None (or 0) picks the tile from the measured
    M staircase; BLOCK_N defaults to None (the channel width and split-K are then picked
    from M, N and K by a cost model fitted to measured latencies; the reference's default
    is 64).  Every tile choice gives bit-identical results.  W8A8 BLOCK_M
    is at most 304; BLOCK_N is 16/32/64/128 channels per workgroup (larger values are taken as
    128); W4A16 BLOCK_N is 64 or 128.
  * w8a8_matmul also accepts a PackedWeightInt8 (pack_weight_int8), the weight pre-packed
    once into MFMA fragments, with bit-identical results.
  * `ck` is a KernelInfo with n_regs / n_spills / metadata.shared like Triton's compiled
    kernel, plus the resolved tile configuration.
  * w4a16_matmul also accepts the int32 "8 nibbles per word along K" packing and a
    PackedWeightInt4 (pack_weight_int4), bit-identical to the int32 packing; its fp32
    summation order depends only on (N, K), split_k and whether the weight is the reference
    uint8 packing (whose bytes pair k with k + K/2), so every W4A16 tile choice is
    bit-identical too.
    W4A16 BLOCK_M is at most 256 (tiles deeper than 144 rows run as equal chunks of at most
    144 rows); its LDS-staged kernels run 8 waves whatever num_warps says.
"""
from __future__ import annotations

import array
import ctypes
import functools
import math
import os
import sys

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
if _HERE not in sys.path:
    sys.path.insert(0, _HERE)

from specq import _lib  # noqa: E402
from specq import workspace as _ws  # noqa: E402

__all__ = [
    "w8a8_matmul", "w4a16_matmul", "paged_attention",
    "quantize_act_int8", "quantize_weight_int8", "quantize_weight_int4",
    "make_paged_kv", "paged_attention_ref",
    "silu_mul", "quantize_act_int8_gpu", "silu_mul_quant_int8", "paged_kv_append",
    "pack_int4_i32", "KernelInfo", "PackedWeightInt8", "pack_weight_int8", "PackedWeightInt4", "pack_weight_int4",
    "w4a8_matmul", "quantize_weight_int4_channel", "PackedWeightW4A8", "pack_weight_w4a8",
    "w8a8_matmul_grouped", "w4a16_matmul_grouped", "set_weight_pack_cache", "clear_weight_pack_cache",
    "rotary_embed", "rotary_inv_freq", "paged_kv_append_block_scaled", "paged_attention_block_scaled",
    "paged_kv_reserve", "paged_kv_free", "paged_kv_fork", "paged_kv_compact", "paged_kv_copy",
    "qk_norm_rotary", "paged_attention_weights", "paged_kv_evict", "beam_select", "beam_reorder",
]


# ----------------------------------------------------------------------------------------
# Kernel bookkeeping: the reference's `ck` object and the JIT-cache stand-ins read by
# correctness.py:18-24 (n_compiled).
# ----------------------------------------------------------------------------------------
class _Meta:
    def __init__(self, shared: int):
        self.shared = shared

    def __getitem__(self, key):
        return getattr(self, key)


class KernelInfo:
    """Resource usage of the kernel a call launched (lazy: queried on first access)."""

    def __init__(self, kind: int, variant: int, m_grid: int, N: int, K: int, block_m: int, block_n: int,
                 num_warps: int, split_k: int):
        # The kernel also depends on the library options (kernel-family overrides), so the
        # cache key carries them and a first-time query happens now, under the options the
        # call ran with.
        self._key = (kind, variant, m_grid, N, K, block_m, block_n, num_warps, split_k)
        try:
            self._attrs, self._err = _attrs_cached(self._key, _lib.options_key()), None
        except RuntimeError as e:  # reported when the attributes are read
            self._attrs, self._err = None, e

    def _get(self):
        if self._err is not None:
            raise self._err
        return self._attrs

    @property
    def name(self) -> str:
        return self._get().name.decode()

    @property
    def n_regs(self) -> int:
        return self._get().num_regs

    @property
    def n_spills(self) -> int:
        return self._get().scratch_bytes // 4

    @property
    def metadata(self) -> _Meta:
        return _Meta(self._get().lds_bytes)

    @property
    def config(self) -> dict:
        """The tiles the call ran.  Given back as arguments they name the same kernel, except those of a
        many-row kernel (block_n up to 256): these run a streaming kernel, with the same results."""
        a = self._get()
        return dict(block_m=a.block_m, block_n=a.block_n, num_warps=a.num_warps, split_k=a.split_k,
                    threads=a.threads, grid=a.grid)

    def __repr__(self):
        return f"KernelInfo({self.name}, regs={self.n_regs}, spills={self.n_spills}, lds={self.metadata.shared})"


_ATTRS: dict = {}


def _attrs_cached(key, options):
    a = _ATTRS.get((key, options))
    if a is None:
        a = _ATTRS[(key, options)] = _lib.kernel_attrs(*key)
    return a


class _KernelRegistry:
    """Stand-in for a Triton JITFunction's cache: counts the distinct binaries launched."""

    def __init__(self, name: str):
        self.__name__ = name
        self.device_caches: dict = {}

    def _note(self, device_index: int, key) -> None:
        self.device_caches.setdefault(device_index, (set(),))[0].add(key)

    @property
    def cache(self) -> dict:
        return {d: v[0] for d, v in self.device_caches.items()}


_w8a8_kernel = _KernelRegistry("_w8a8_kernel")
_w4a16_kernel = _KernelRegistry("_w4a16_kernel")
_paged_attn_kernel = _KernelRegistry("_paged_attn_kernel")


def _stream_ptr(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _require_gpu(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.device.type != "cuda":
            raise RuntimeError(f"specq kernels run on the GPU only; got a {t.device} tensor")


def _rowmajor(t: torch.Tensor) -> torch.Tensor:
    """2-D view with a unit inner stride (copies only when the inner stride is not 1)."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _check_out(out: torch.Tensor, M: int, N: int, who: str) -> None:
    """The kernels write rows < M and columns < N of out: it must hold at least that."""
    if out.dim() != 2 or out.shape[0] < M or out.shape[1] < N:
        raise RuntimeError(f"{who}: out {tuple(out.shape)} is smaller than [M, N] = [{M}, {N}]")


def _check_w4_scales(sc: torch.Tensor, N: int, K: int, group: int, who: str) -> None:
    """W4A16 scales are fp16 [N, K/group]; a smaller tensor would be read past its end."""
    if group <= 0 or K % group:
        raise RuntimeError(f"{who}: K={K} is not a multiple of group={group}")
    if sc.dim() != 2 or tuple(sc.shape) != (N, K // group):
        raise RuntimeError(f"{who}: scales {tuple(sc.shape)} must be [N, K/group] = [{N}, {K // group}]")


def _plan_ptr(plan) -> int:
    if plan is None:
        return 0
    if plan.dtype != torch.int32 or plan.device.type != "cuda":
        raise RuntimeError("plan must be an int32 device tensor")
    return plan.data_ptr()


# ----------------------------------------------------------------------------------------
# W8A8
# ----------------------------------------------------------------------------------------
def _w8a8_block_n(block_n) -> int:
    if not block_n:
        return 0
    return 16 if block_n <= 16 else (32 if block_n <= 32 else (64 if block_n <= 64 else 128))


class PackedWeightInt8:
    """An int8 weight [N, K] pre-packed once into MFMA fragments for w8a8_matmul.

    Fragments are stored K-step-major: fragment (64-byte K step s, 16-row tile t) is the 1 KB
    at (s * ceil(N/16) + t) KB holding, for lane l and byte b, w[16t + l%16][64s + 16*(l/16) + b]
    (zero-padded), so every load is 1 KB contiguous and the workgroups running at one time
    read one compact window.  Results are bit-identical to passing the row-major weight.
    """

    def __init__(self, w_q: torch.Tensor):
        _require_gpu(w_q)
        if w_q.dtype != torch.int8 or w_q.dim() != 2:
            raise RuntimeError("PackedWeightInt8 expects an int8 [N, K] weight")
        w_q = _rowmajor(w_q)
        self.N, self.K = w_q.shape
        self.shape = (self.N, self.K)
        self.device = w_q.device
        nbytes = _lib.lib().specq_w8a8_packed_bytes(self.N, self.K)
        self.data = torch.empty(nbytes, dtype=torch.int8, device=w_q.device)
        _lib.call("specq_w8a8_pack_weight", w_q.data_ptr(), w_q.stride(0), self.N, self.K, self.data.data_ptr(),
                  _stream_ptr(w_q))


def pack_weight_int8(w_q):
    """Pack an int8 [N, K] weight for w8a8_matmul (see PackedWeightInt8)."""
    return PackedWeightInt8(w_q)


class _WeightPackCache:
    """Row-major int8 weights packed once, for callers that pass the reference's w_q layout.

    w8a8_matmul and w8a8_matmul_grouped given a row-major int8 weight (as the reference's
    scripts pass it, bench_graphs.py:55-64, correctness.py:36) look it up here and run the
    packed-fragment kernels on its PackedWeightInt8: the results are bit-identical (the INT32
    sums do not depend on the weight layout), and the packed layout streams each weight as 1 KB
    contiguous fragments where the row-major one reads half cache lines.  An entry is keyed on
    the weight's storage, offset, shape and strides and remembers the storage's version counter,
    so an in-place update of the weight (through it or any view of it) repacks it on the next
    call; the entry holds the source storage, so its memory cannot be reused under the key while
    cached.  A miss inside graph capture does not pack (that would allocate): the call runs the
    row-major kernel, with the same results.  Entries beyond the byte budget are evicted least
    recently used first.  Controls: set_weight_pack_cache(enabled, budget_bytes),
    clear_weight_pack_cache(); the environment variable SPECQ_PACK_CACHE=0 starts it disabled.
    """

    def __init__(self):
        import collections
        import threading
        self.enabled = os.environ.get("SPECQ_PACK_CACHE", "1") != "0"
        self.budget = 64 << 30
        self.bytes = 0
        self._d = collections.OrderedDict()
        self._lock = threading.Lock()

    @staticmethod
    def _key(w: torch.Tensor):
        return (w.device.index, w.untyped_storage().data_ptr(), w.storage_offset(), tuple(w.shape), tuple(w.stride()))

    def lookup(self, w: torch.Tensor):
        """The PackedWeightInt8 of w (packing it now on a miss), or None (disabled, or a miss
        during graph capture)."""
        if not self.enabled or w.dtype != torch.int8 or w.dim() != 2 or w.stride(-1) != 1:
            return None
        key = self._key(w)
        with self._lock:
            e = self._d.get(key)
            if e is not None:
                if e[1] == w._version:
                    self._d.move_to_end(key)
                    return e[0]
                del self._d[key]
                self.bytes -= e[0].data.numel()
        if torch.cuda.is_current_stream_capturing():
            return None
        packed = PackedWeightInt8(w)
        with self._lock:
            old = self._d.pop(key, None)
            if old is not None:
                self.bytes -= old[0].data.numel()
            self._d[key] = (packed, w._version, w.untyped_storage())
            self.bytes += packed.data.numel()
            while self.bytes > self.budget and len(self._d) > 1:
                _, (pw, _, _) = self._d.popitem(last=False)
                self.bytes -= pw.data.numel()
        return packed

    def clear(self):
        with self._lock:
            self._d.clear()
            self.bytes = 0


_pack_cache = _WeightPackCache()


def set_weight_pack_cache(enabled: bool = True, budget_bytes: int | None = None) -> None:
    """Turn the transparent packing of row-major W8A8 weights on or off, and set its byte budget."""
    _pack_cache.enabled = bool(enabled)
    if budget_bytes is not None:
        _pack_cache.budget = int(budget_bytes)
    if not enabled:
        _pack_cache.clear()


def clear_weight_pack_cache() -> None:
    """Drop every packed copy the transparent cache holds (their memory returns to torch)."""
    _pack_cache.clear()


def _aligned16(a_q: torch.Tensor, K: int) -> bool:
    """The packed-fragment kernels read 16-byte pieces of the activation rows."""
    return a_q.data_ptr() % 16 == 0 and (a_q.stride(0) % 16 == 0 or a_q.shape[0] <= 1) and K % 16 == 0


def w8a8_matmul(a_q, sa, w_q, sw, out=None, BLOCK_M=16, BLOCK_N=None, BLOCK_K=128,
                num_warps=4, num_stages=3, plan=None, grid_m_max=None, split_k=0, workspace=None,
                plan_tiles=None):
    """C[M, N] = fp16((int32(a_q @ w_q.T) * sa[:, None]) * sw[None, :]).  Returns (out, ck).

    a_q int8 [M, K]; w_q int8 [N, K] (or a PackedWeightInt8); sa fp32 [M]; sw fp32 [N].
    With `plan`, M is read from plan[0] on the device and the grid covers grid_m_max rows
    (reference kernels.py:71-86).  Plan-mode calls with an automatic BLOCK_M use tiles of at
    most 80 rows, so a small active M leaves the later chunks idle; plan_tiles="grid" instead
    runs the tiles an eager call of grid_m_max rows would pick (for plan graphs whose active M
    stays close to the grid, e.g. one graph per shape bucket).  The INT32 sums are exact, so
    every tile gives the same result.
    """
    packed = isinstance(w_q, PackedWeightInt8)
    _require_gpu(a_q, sa, sw)
    if not packed:
        _require_gpu(w_q)
    if a_q.dtype != torch.int8 or (not packed and w_q.dtype != torch.int8):
        raise RuntimeError("w8a8_matmul expects int8 activations and weights")
    M, K = a_q.shape
    N = w_q.shape[0]
    if w_q.shape[1] != K:
        raise RuntimeError(f"w8a8_matmul: K mismatch {tuple(a_q.shape)} vs {tuple(w_q.shape)}")
    a_q = _rowmajor(a_q)
    if not packed:
        w_q = _rowmajor(w_q)
        if _aligned16(a_q, K):
            pw = _pack_cache.lookup(w_q)
            if pw is not None:
                w_q, packed = pw, True
    sa = sa.float().contiguous()
    sw = sw.float().contiguous()
    if sa.numel() < M or sw.numel() != N:
        raise RuntimeError(f"w8a8_matmul: scales sa {tuple(sa.shape)} / sw {tuple(sw.shape)} do not cover M={M} / N={N}")
    if out is None:
        out = torch.empty((M, N), device=a_q.device, dtype=torch.float16)
    if out.dtype != torch.float16 or out.stride(-1) != 1:
        raise RuntimeError("w8a8_matmul: out must be fp16 with unit inner stride")
    _check_out(out, M, N, "w8a8_matmul")
    m_grid = int(grid_m_max) if grid_m_max is not None else M
    bm = int(BLOCK_M) if BLOCK_M else 0  # 0: the library picks the tile (cost model over M, N, K)
    bn = _w8a8_block_n(BLOCK_N)
    nw = int(num_warps) if num_warps else 4
    if plan is not None and plan_tiles is not None:
        if plan_tiles != "grid":
            raise RuntimeError(f"w8a8_matmul: plan_tiles={plan_tiles!r} (None or 'grid')")
        if not bm:
            cfg = KernelInfo(0, (1 if packed else 0) | 32, m_grid, N, K, 0, bn, nw, split_k).config
            bm, bn, split_k = cfg["block_m"], cfg["block_n"], cfg["split_k"]
    ws = workspace.on(a_q.get_device()) if workspace is not None else _ws.shared(a_q.device)
    if packed:
        need = _lib.lib().specq_w8a8_packed_workspace_size(m_grid, N, K, bm, bn, nw, split_k)
        wptr, wbytes = ws.ensure(need)
        _lib.call("specq_w8a8_packed", a_q.data_ptr(), a_q.stride(0), w_q.data.data_ptr(),
                  sa.data_ptr(), sw.data_ptr(), out.data_ptr(), out.stride(0),
                  M, N, K, int(grid_m_max or 0), _plan_ptr(plan), bm, bn, nw, split_k,
                  wptr, wbytes, _stream_ptr(a_q))
    else:
        need = _lib.lib().specq_w8a8_workspace_size(m_grid, N, K, bm, bn, nw, split_k)
        wptr, wbytes = ws.ensure(need)
        _lib.call("specq_w8a8", a_q.data_ptr(), a_q.stride(0), w_q.data_ptr(), w_q.stride(0),
                  sa.data_ptr(), sw.data_ptr(), out.data_ptr(), out.stride(0),
                  M, N, K, int(grid_m_max or 0), _plan_ptr(plan), bm, bn, nw, split_k,
                  wptr, wbytes, _stream_ptr(a_q))
    _w8a8_kernel._note(a_q.device.index or 0, (bm, bn, nw))
    return out, KernelInfo(0, (1 if packed else 0) | (16 if plan is not None else 0), m_grid, N, K, bm, bn, nw, split_k)


def w8a8_matmul_grouped(a_q, sa, weights, outs=None, BLOCK_M=16, BLOCK_N=None, num_warps=4, plan=None,
                        grid_m_max=None, split_k=0, workspace=None, plan_tiles=None):
    """Up to four W8A8 GEMMs that share one activation (q, k and v; gate and up) in one launch.

    outs[g] = fp16((int32(a_q @ W_g.T) * sa[:, None]) * sw_g[None, :]) for weights[g] = (W_g, sw_g),
    bit-identical to one w8a8_matmul (or w4a8_matmul) call per GEMM.  The W_g are all int8 [N_g, K]
    tensors, all PackedWeightInt8 or all PackedWeightW4A8.  The launch uses the tiles of one GEMM
    of width sum(N_g), as the reference's fused qkv / gate_up weights do (bench_matmul.py:16),
    while the weights and outputs stay separate.  Other arguments as w8a8_matmul.  Returns
    (outs, ck).
    """
    n = len(weights)
    if not 1 <= n <= 4:
        raise RuntimeError(f"w8a8_matmul_grouped: {n} GEMMs (1..4 supported)")
    ws_ = [w for w, _ in weights]
    if all(isinstance(w, PackedWeightInt8) for w in ws_):
        layout = 1
    elif all(isinstance(w, PackedWeightW4A8) for w in ws_):
        layout = 2
    elif all(isinstance(w, torch.Tensor) and w.dtype == torch.int8 for w in ws_):
        layout = 0
    else:
        raise RuntimeError("w8a8_matmul_grouped: weights must all be int8 tensors, all PackedWeightInt8 "
                           "or all PackedWeightW4A8")
    _require_gpu(a_q, sa, *(sw for _, sw in weights))
    if layout == 0:
        _require_gpu(*ws_)
        ws_ = [_rowmajor(w) for w in ws_]
    if a_q.dtype != torch.int8:
        raise RuntimeError("w8a8_matmul_grouped expects int8 activations")
    M, K = a_q.shape
    Ns = [int(w.shape[0]) if layout == 0 else int(w.N) for w in ws_]
    for w in ws_:
        if (w.shape[1] if layout == 0 else w.K) != K:
            raise RuntimeError(f"w8a8_matmul_grouped: K mismatch {tuple(a_q.shape)} vs {tuple(w.shape)}")
    a_q = _rowmajor(a_q)
    if layout == 0 and _aligned16(a_q, K):
        pws = [_pack_cache.lookup(w) for w in ws_]
        if all(pw is not None for pw in pws):
            ws_, layout = pws, 1
    sa = sa.float().contiguous()
    sws = [sw.float().contiguous() for _, sw in weights]
    for sw, N in zip(sws, Ns):
        if sw.numel() != N:
            raise RuntimeError(f"w8a8_matmul_grouped: channel scale of {sw.numel()} entries for N={N}")
    if outs is None:
        outs = [torch.empty((M, N), device=a_q.device, dtype=torch.float16) for N in Ns]
    if len(outs) != n:
        raise RuntimeError("w8a8_matmul_grouped: one output per GEMM")
    for o, N in zip(outs, Ns):
        if o.dtype != torch.float16 or o.stride(-1) != 1 or tuple(o.shape) != (M, N):
            raise RuntimeError(f"w8a8_matmul_grouped: outputs must be fp16 [M, N] with unit inner stride, got "
                               f"{tuple(o.shape)} for N={N}")
    m_grid = int(grid_m_max) if grid_m_max is not None else M
    N_total = sum(Ns)
    bm = int(BLOCK_M) if BLOCK_M else 0
    bn = _w8a8_block_n(BLOCK_N)
    nw = int(num_warps) if num_warps else 4
    if plan is not None and plan_tiles is not None:
        if plan_tiles != "grid":
            raise RuntimeError(f"w8a8_matmul_grouped: plan_tiles={plan_tiles!r} (None or 'grid')")
        if not bm:
            cfg = KernelInfo(0, layout | 32, m_grid, N_total, K, 0, bn, nw, split_k).config
            bm, bn, split_k = cfg["block_m"], cfg["block_n"], cfg["split_k"]
    arr = lambda ct, vals: (ct * n)(*vals)  # noqa: E731
    n_arr = arr(ctypes.c_int, Ns)
    w_arr = arr(ctypes.c_void_p, [w.data_ptr() if layout == 0 else w.data.data_ptr() for w in ws_])
    ldw_arr = arr(ctypes.c_int64, [w.stride(0) if layout == 0 else 0 for w in ws_])
    sw_arr = arr(ctypes.c_void_p, [sw.data_ptr() for sw in sws])
    c_arr = arr(ctypes.c_void_p, [o.data_ptr() for o in outs])
    ldc_arr = arr(ctypes.c_int64, [o.stride(0) for o in outs])
    ws = workspace.on(a_q.get_device()) if workspace is not None else _ws.shared(a_q.device)
    need = _lib.lib().specq_w8a8_grouped_workspace_size(layout, m_grid, n, n_arr, K, bm, bn, nw, split_k)
    wptr, wbytes = ws.ensure(need)
    _lib.call("specq_w8a8_grouped", layout, a_q.data_ptr(), a_q.stride(0), sa.data_ptr(), n, w_arr, ldw_arr, sw_arr,
              c_arr, ldc_arr, n_arr, M, K, int(grid_m_max or 0), _plan_ptr(plan), bm, bn, nw, split_k,
              wptr, wbytes, _stream_ptr(a_q))
    _w8a8_kernel._note(a_q.device.index or 0, (bm, bn, nw, "grouped", layout))
    return outs, KernelInfo(0, layout | (16 if plan is not None else 0), m_grid, N_total, K, bm, bn, nw, split_k)


def quantize_act_int8(x):
    """Dynamic per-token symmetric INT8 quantisation (reference kernels.py:58-62)."""
    s = x.abs().amax(dim=-1).float().clamp(min=1e-8) / 127.0
    q = torch.round(x.float() / s[:, None]).clamp(-127, 127).to(torch.int8)
    return q, s


def quantize_weight_int8(w):
    """Per-output-channel symmetric INT8 quantisation (reference kernels.py:65-68)."""
    s = w.abs().amax(dim=-1).float().clamp(min=1e-8) / 127.0
    q = torch.round(w.float() / s[:, None]).clamp(-127, 127).to(torch.int8)
    return q, s


# ----------------------------------------------------------------------------------------
# W4A16
# ----------------------------------------------------------------------------------------
def quantize_weight_int4(w, group=128):
    """Group-wise symmetric INT4 (reference kernels.py:138-147).

    Returns (packed uint8 [N, K/2], scales fp16 [N, K/group], dequantised fp16 [N, K]).
    Byte j of a packed row holds k = j (low nibble) and k = j + K/2 (high nibble), each as
    q + 8 with q in [-8, 7].
    """
    N, K = w.shape
    assert K % 2 == 0 and (K // 2) % group == 0
    wg = w.float().reshape(N, K // group, group)
    sc = wg.abs().amax(-1).clamp(min=1e-8) / 7.0
    q = torch.round(wg / sc[..., None]).clamp(-8, 7).reshape(N, K).to(torch.int16) + 8
    half = K // 2
    packed = (q[:, :half] | (q[:, half:] << 4)).to(torch.uint8).contiguous()
    deq = ((q - 8).float().reshape(N, K // group, group) * sc[..., None]).reshape(N, K)
    return packed, sc.to(torch.float16).contiguous(), deq.to(torch.float16)


def pack_int4_i32(q_unsigned):
    """Pack unsigned nibbles [N, K] (values 0..15) as int32 [N, K/8]: nibble i of word j = k 8j+i."""
    N, K = q_unsigned.shape
    assert K % 8 == 0
    v = q_unsigned.to(torch.int64).reshape(N, K // 8, 8)
    shifts = torch.arange(0, 32, 4, device=v.device, dtype=torch.int64)
    word = (v << shifts).sum(-1)
    word = torch.where(word >= 2 ** 31, word - 2 ** 32, word)
    return word.to(torch.int32).contiguous()


class PackedWeightInt4:
    """A W4A16 weight (uint8 [N, K/2] reference packing or int32 [N, K/8]) re-packed once into
    MFMA fragments for w4a16_matmul.

    Fragment (128-wide K block b, 16-row tile t) is the 1 KB at (b * ceil(N/16) + t) KB; lane
    l's 16 bytes hold row 16t + l%16 at k = 128b + 32*(l/16) + 8u + j as word u, nibble j at
    bits 4p..4p+3 with p = j/2 for even j and 4 + j/2 for odd j (each pair of weights then
    becomes two fp16 with one AND-OR).  Every weight load is 1 KB contiguous.  The
    group scales are not repacked.  Results are bit-identical to passing the int32 packing of
    the same weight (the reference uint8 packing sums K in another order, so it agrees to
    fp32 rounding).
    """

    def __init__(self, wp: torch.Tensor):
        _require_gpu(wp)
        if wp.dim() != 2 or wp.dtype not in (torch.uint8, torch.int32):
            raise RuntimeError("PackedWeightInt4 expects uint8 [N, K/2] or int32 [N, K/8] packed weights")
        wp = _rowmajor(wp)
        layout = 0 if wp.dtype == torch.uint8 else 1
        self.N = wp.shape[0]
        self.K = wp.shape[1] * (2 if layout == 0 else 8)
        self.shape = (self.N, self.K)
        self.device = wp.device
        nbytes = _lib.lib().specq_w4a16_packed_bytes(self.N, self.K)
        if nbytes == 0:
            raise RuntimeError(f"PackedWeightInt4: K={self.K} must be a multiple of 128")
        self.data = torch.empty(nbytes, dtype=torch.uint8, device=wp.device)
        _lib.call("specq_w4a16_pack_weight", wp.data_ptr(), wp.stride(0), layout, self.N, self.K,
                  self.data.data_ptr(), _stream_ptr(wp))


def pack_weight_int4(wp):
    """Pack a W4A16 weight for w4a16_matmul (see PackedWeightInt4)."""
    return PackedWeightInt4(wp)


def w4a16_matmul(a, wp, sc, group=128, out=None, BLOCK_M=16, BLOCK_N=None, BLOCK_K=64,
                 num_warps=4, num_stages=3, plan=None, grid_m_max=None, split_k=0, workspace=None):
    """C[M, N] = fp16(a @ dequant(wp, sc).T) (reference kernels.py:150-166).  Returns (out, ck).

    a fp16 [M, K].  wp is uint8 [N, K/2] (reference packing), int32 [N, K/8] (8 nibbles per
    word along K) or a PackedWeightInt4.  sc fp16 [N, K/group].
    """
    _require_gpu(a, sc)
    assert BLOCK_K <= group and group % BLOCK_K == 0
    M, K = a.shape
    N = wp.shape[0]
    if isinstance(wp, PackedWeightInt4):
        layout = 2
        if wp.K != K:
            raise RuntimeError(f"w4a16_matmul: packed weight K={wp.K} does not match K={K}")
    elif wp.dtype == torch.uint8:
        layout = 0
        if wp.shape[1] * 2 != K:
            raise RuntimeError(f"w4a16_matmul: packed uint8 weights {tuple(wp.shape)} do not match K={K}")
    elif wp.dtype == torch.int32:
        layout = 1
        if wp.shape[1] * 8 != K:
            raise RuntimeError(f"w4a16_matmul: packed int32 weights {tuple(wp.shape)} do not match K={K}")
    else:
        raise RuntimeError("w4a16_matmul: wp must be uint8 [N, K/2], int32 [N, K/8] or a PackedWeightInt4")
    if a.dtype != torch.float16 or sc.dtype != torch.float16:
        raise RuntimeError("w4a16_matmul expects fp16 activations and fp16 scales")
    _check_w4_scales(sc, N, K, int(group), "w4a16_matmul")
    a, sc = _rowmajor(a), _rowmajor(sc)
    if layout == 2:
        w_ptr, w_ld = wp.data.data_ptr(), 0
    else:
        _require_gpu(wp)
        wp = _rowmajor(wp)
        w_ptr, w_ld = wp.data_ptr(), wp.stride(0)
    if a.data_ptr() % 16 or a.stride(0) % 8:
        a = a.contiguous() if a.data_ptr() % 16 == 0 else a.clone()
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=torch.float16)
    if out.dtype != torch.float16 or out.stride(-1) != 1:
        raise RuntimeError("w4a16_matmul: out must be fp16 with unit inner stride")
    _check_out(out, M, N, "w4a16_matmul")
    m_grid = int(grid_m_max) if grid_m_max is not None else M
    bm = int(BLOCK_M) if BLOCK_M else 0
    bn = 0 if not BLOCK_N else (64 if BLOCK_N <= 64 else 128)
    ws = workspace.on(a.get_device()) if workspace is not None else _ws.shared(a.device)
    need = _lib.lib().specq_w4a16_workspace_size(m_grid, N, K, bm, bn, 4, split_k)
    wptr, wbytes = ws.ensure(need)
    _lib.call("specq_w4a16", a.data_ptr(), a.stride(0), w_ptr, w_ld, layout,
              sc.data_ptr(), sc.stride(0), out.data_ptr(), out.stride(0),
              M, N, K, int(group), int(grid_m_max or 0), _plan_ptr(plan), bm, bn, 4, split_k,
              wptr, wbytes, _stream_ptr(a))
    _w4a16_kernel._note(a.device.index or 0, (bm, bn, layout))
    return out, KernelInfo(1, layout | (16 if plan is not None else 0), m_grid, N, K, bm, bn, 4, split_k)


def w4a16_matmul_grouped(a, weights, group=128, outs=None, BLOCK_M=None, BLOCK_N=None, num_warps=4, plan=None,
                         grid_m_max=None, split_k=0, workspace=None):
    """Up to four W4A16 GEMMs that share one fp16 activation (q, k and v; gate and up) in one launch.

    outs[g] = fp16(a @ dequant(wp_g, sc_g).T) for weights[g] = (wp_g, sc_g), bit-identical to one
    w4a16_matmul call per GEMM with the same split_k.  The wp_g are all PackedWeightInt4, all int32
    [N_g, K/8] or all uint8 [N_g, K/2].  The launch uses the tiles of one GEMM of width sum(N_g), as
    the reference's fused qkv / gate_up weights do (bench_matmul.py:16), while the weights and
    outputs stay separate; members whose automatic split counts differ run as one launch each.
    Other arguments as w4a16_matmul.  Returns (outs, ck).
    """
    n = len(weights)
    if not 1 <= n <= 4:
        raise RuntimeError(f"w4a16_matmul_grouped: {n} GEMMs (1..4 supported)")
    wps = [w for w, _ in weights]
    if all(isinstance(w, PackedWeightInt4) for w in wps):
        layout = 2
    elif all(isinstance(w, torch.Tensor) and w.dtype == torch.int32 for w in wps):
        layout = 1
    elif all(isinstance(w, torch.Tensor) and w.dtype == torch.uint8 for w in wps):
        layout = 0
    else:
        raise RuntimeError("w4a16_matmul_grouped: weights must all be PackedWeightInt4, all int32 [N, K/8] "
                           "or all uint8 [N, K/2]")
    scs = [sc for _, sc in weights]
    _require_gpu(a, *scs)
    if a.dtype != torch.float16 or any(sc.dtype != torch.float16 for sc in scs):
        raise RuntimeError("w4a16_matmul_grouped expects fp16 activations and fp16 scales")
    assert BLOCK_N is None or BLOCK_N in (64, 128)
    M, K = a.shape
    if layout == 2:
        Ns = [w.N for w in wps]
        if any(w.K != K for w in wps):
            raise RuntimeError(f"w4a16_matmul_grouped: packed weight K does not match K={K}")
        w_ptrs, w_lds = [w.data.data_ptr() for w in wps], [0] * n
    else:
        _require_gpu(*wps)
        wps = [_rowmajor(w) for w in wps]
        per = 2 if layout == 0 else 8
        Ns = [int(w.shape[0]) for w in wps]
        if any(w.shape[1] * per != K for w in wps):
            raise RuntimeError(f"w4a16_matmul_grouped: packed weights do not match K={K}")
        w_ptrs, w_lds = [w.data_ptr() for w in wps], [w.stride(0) for w in wps]
    for sc, N in zip(scs, Ns):
        _check_w4_scales(sc, N, K, int(group), "w4a16_matmul_grouped")
    a = _rowmajor(a)
    scs = [_rowmajor(sc) for sc in scs]
    if a.data_ptr() % 16 or a.stride(0) % 8:
        a = a.contiguous() if a.data_ptr() % 16 == 0 else a.clone()
    if outs is None:
        outs = [torch.empty((M, N), device=a.device, dtype=torch.float16) for N in Ns]
    if len(outs) != n:
        raise RuntimeError("w4a16_matmul_grouped: one output per GEMM")
    for o, N in zip(outs, Ns):
        if o.dtype != torch.float16 or o.stride(-1) != 1 or tuple(o.shape) != (M, N):
            raise RuntimeError(f"w4a16_matmul_grouped: outputs must be fp16 [M, N] with unit inner stride, got "
                               f"{tuple(o.shape)} for N={N}")
    m_grid = int(grid_m_max) if grid_m_max is not None else M
    bm = int(BLOCK_M) if BLOCK_M else 0
    bn = 0 if not BLOCK_N else int(BLOCK_N)
    arr = lambda ct, vals: (ct * n)(*vals)  # noqa: E731
    n_arr = arr(ctypes.c_int, Ns)
    ws = workspace.on(a.get_device()) if workspace is not None else _ws.shared(a.device)
    need = _lib.lib().specq_w4a16_grouped_workspace_size(m_grid, n, n_arr, K, bm, bn, 4, split_k)
    wptr, wbytes = ws.ensure(need)
    _lib.call("specq_w4a16_grouped", a.data_ptr(), a.stride(0), n, arr(ctypes.c_void_p, w_ptrs),
              arr(ctypes.c_int64, w_lds), layout, arr(ctypes.c_void_p, [sc.data_ptr() for sc in scs]),
              arr(ctypes.c_int64, [sc.stride(0) for sc in scs]), arr(ctypes.c_void_p, [o.data_ptr() for o in outs]),
              arr(ctypes.c_int64, [o.stride(0) for o in outs]), n_arr, M, K, int(group), int(grid_m_max or 0),
              _plan_ptr(plan), bm, bn, 4, split_k, wptr, wbytes, _stream_ptr(a))
    _w4a16_kernel._note(a.device.index or 0, (bm, bn, "grouped", layout))
    # The launch runs the members' common split count: report the tiles of that launch.
    sk = w4a16_group_split(Ns, K, split_k) if n > 1 else split_k
    return outs, KernelInfo(1, layout | (16 if plan is not None else 0), m_grid, sum(Ns), K, bm, bn, 4,
                            sk if sk > 0 else split_k)


def w4a16_group_split(Ns, K: int, split_k: int = 0) -> int:
    """The split count a grouped W4A16 launch of members of widths Ns runs, or 0 when their
    counts differ (the members then run as one launch each)."""
    arr = (ctypes.c_int * len(Ns))(*[int(n) for n in Ns])
    return int(_lib.lib().specq_w4a16_grouped_split(len(Ns), arr, int(K), int(split_k)))


# ----------------------------------------------------------------------------------------
# Paged verification attention
# ----------------------------------------------------------------------------------------
def paged_attention(q, kc, vc, ks, vs, block_tbl, ctx_len, q_len, QPP=None, BLOCK_N=64,
                    num_warps=4, num_stages=2, plan=None, n_seqs=None, out=None, workspace=None):
    """Verification attention over an INT8 paged KV cache (reference kernels.py:239-262).

    q fp16 [B, QLMAX, H, D]; kc/vc int8 [pages, PAGE, H_KV, D]; ks/vs fp16 or fp32
    [pages, PAGE, H_KV]; block_tbl int32 [B, max_pages]; ctx_len int32 [B] (includes the
    q_len query tokens; block-table ids outside [0, pages) mask their page's tokens).  QPP
    query tokens per program (default q_len = fused).  With
    `plan`, (n_seqs, q_len) = plan[0:2] on the device and the grid covers (B, QLMAX).
    Returns (out, ck).
    """
    _require_gpu(q, kc, vc, ks, vs, block_tbl, ctx_len)
    B, QLMAX, H, D = q.shape
    PAGE, H_KV = kc.shape[1], kc.shape[2]
    if QPP is None:
        QPP = q_len
    if out is None:
        out = torch.zeros_like(q)
    n_seqs = B if n_seqs is None else n_seqs
    if q.dtype != torch.float16 or out.dtype != torch.float16:
        raise RuntimeError("paged_attention expects fp16 q and out")
    if kc.dtype != torch.int8 or vc.dtype != torch.int8:
        raise RuntimeError("paged_attention expects an int8 KV cache")
    if kc.stride() != vc.stride() or ks.stride() != vs.stride() or ks.dtype != vs.dtype:
        raise RuntimeError("paged_attention: K and V (and their scales) must share layout and dtype")
    if ks.dtype not in (torch.float16, torch.float32):
        raise RuntimeError("paged_attention: scales must be fp16 or fp32")
    if q.stride(3) != 1 or out.stride(3) != 1 or kc.stride(3) != 1:
        raise RuntimeError("paged_attention: head_dim must be contiguous")
    if block_tbl.dtype != torch.int32 or ctx_len.dtype != torch.int32:
        raise RuntimeError("paged_attention: block_tbl and ctx_len must be int32")
    if out.shape != q.shape:
        raise RuntimeError(f"paged_attention: out {tuple(out.shape)} must have q's shape {tuple(q.shape)}")
    if kc.shape != vc.shape or kc.shape[3] != D or H % H_KV != 0:
        raise RuntimeError(f"paged_attention: cache {tuple(kc.shape)} does not fit q {tuple(q.shape)}")
    if tuple(ks.shape) != tuple(kc.shape[:3]) or ks.shape != vs.shape:
        raise RuntimeError(f"paged_attention: scales {tuple(ks.shape)} must be [pages, PAGE, H_KV]")
    if int(QPP) < 1:
        raise RuntimeError(f"paged_attention: QPP={QPP} must be at least 1")
    if plan is None and not (0 <= int(n_seqs) <= B and 0 <= int(q_len) <= QLMAX):
        raise RuntimeError(f"paged_attention: need 0 <= n_seqs <= {B} and 0 <= q_len <= {QLMAX}")
    block_tbl = _rowmajor(block_tbl)
    ctx_len = ctx_len.contiguous()
    B_grid = B if plan is not None else int(n_seqs)
    if block_tbl.dim() != 2 or block_tbl.shape[0] < B_grid or ctx_len.numel() < B_grid:
        raise RuntimeError("paged_attention: block_tbl and ctx_len must cover every sequence of the grid")
    G = H // H_KV
    max_pages = block_tbl.shape[1]
    ws = workspace.on(q.get_device()) if workspace is not None else _ws.shared(q.device)
    need = _lib.lib().specq_paged_attn_workspace_size(B_grid, H, H_KV, QLMAX, int(QPP), max_pages, PAGE)
    wptr, wbytes = ws.ensure(need)
    _lib.call("specq_paged_attn",
              q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
              kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2),
              ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), ks.stride(2),
              1 if ks.dtype == torch.float32 else 0,
              block_tbl.data_ptr(), block_tbl.stride(0), max_pages, min(kc.shape[0], 2**31 - 1), ctx_len.data_ptr(),
              out.data_ptr(), out.stride(0), out.stride(1), out.stride(2),
              B_grid, int(n_seqs), int(q_len), QLMAX, H, H_KV, D, PAGE, int(QPP),
              1.0 / math.sqrt(D), _plan_ptr(plan), wptr, wbytes, _stream_ptr(q))
    rows = int(QPP) * G
    _paged_attn_kernel._note(q.device.index or 0, (D, (rows + 15) // 16, str(ks.dtype)))
    return out, KernelInfo(2, D | (1 << 16 if ks.dtype == torch.float32 else 0), 0, 0, 0, rows, 0, 4, 0)


def make_paged_kv(B, ctx_len, H_KV, D, PAGE=16, device="cuda", seed=0):
    """Random INT8 KV cache with a shuffled page table (reference kernels.py:265-286).

    Same generator calls in the same order as the reference, so a given seed yields the
    same cache.  Returns (kc, vc, ks, vs, block_tbl, ctx_len) with fp16 scales.
    """
    g = torch.Generator(device="cpu").manual_seed(seed)
    pages_per_seq = [(int(l) + PAGE - 1) // PAGE for l in ctx_len]
    total = sum(pages_per_seq)
    perm = torch.randperm(total, generator=g)
    bt = torch.zeros((B, max(pages_per_seq)), dtype=torch.int32)
    start = 0
    for b, n in enumerate(pages_per_seq):
        bt[b, :n] = perm[start:start + n].to(torch.int32)
        start += n
    kf = torch.randn((total, PAGE, H_KV, D), generator=g).half()
    vf = torch.randn((total, PAGE, H_KV, D), generator=g).half()

    def q8(x):
        s = x.float().abs().amax(-1).clamp(min=1e-8) / 127.0
        return torch.round(x.float() / s[..., None]).clamp(-127, 127).to(torch.int8), s.half()

    kc, ks = q8(kf)
    vc, vs = q8(vf)
    dev = lambda t: t.to(device).contiguous()  # noqa: E731
    return dev(kc), dev(vc), dev(ks), dev(vs), dev(bt), torch.tensor(list(ctx_len), dtype=torch.int32, device=device)


def paged_attention_ref(q, kc, vc, ks, vs, block_tbl, ctx_len, q_len):
    """Dense fp32 verification attention (reference kernels.py:289-309), any device."""
    B, _, H, D = q.shape
    PAGE, H_KV = kc.shape[1], kc.shape[2]
    G = H // H_KV
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    for b in range(B):
        L = int(ctx_len[b])
        pos = torch.arange(L, device=q.device)
        page = block_tbl[b, pos // PAGE].long()
        slot = pos % PAGE
        k = (kc[page, slot].float() * ks[page, slot].float()[..., None]).repeat_interleave(G, dim=1)
        v = (vc[page, slot].float() * vs[page, slot].float()[..., None]).repeat_interleave(G, dim=1)
        qq = q[b, :q_len].float()
        s = torch.einsum("qhd,khd->hqk", qq, k) / math.sqrt(D)
        qpos = L - q_len + torch.arange(q_len, device=q.device)
        s = s.masked_fill(pos[None, None, :] > qpos[None, :, None], float("-inf"))
        out[b, :q_len] = torch.einsum("hqk,khd->qhd", s.softmax(-1), v)
    return out.half()


# ----------------------------------------------------------------------------------------
# Device-side steps of a verification layer (no reference counterpart on the device)
# ----------------------------------------------------------------------------------------
def silu_mul(gate, up, out=None, plan=None, grid_m_max=None):
    """h = fp16(silu(gate) * up) on the GPU; gate/up fp16 [M, N]."""
    _require_gpu(gate, up)
    M, N = gate.shape
    gate, up = _rowmajor(gate), _rowmajor(up)
    if out is None:
        out = torch.empty((M, N), device=gate.device, dtype=torch.float16)
    _lib.call("specq_silu_mul", gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0),
              out.data_ptr(), out.stride(0), M, N, int(grid_m_max or 0), _plan_ptr(plan), _stream_ptr(gate))
    return out


def quantize_act_int8_gpu(x, q=None, s=None, plan=None, grid_m_max=None):
    """quantize_act_int8 on the GPU (bit-identical to the torch formula); x fp16 [M, K]."""
    _require_gpu(x)
    M, K = x.shape
    x = _rowmajor(x)
    q = torch.empty((M, K), device=x.device, dtype=torch.int8) if q is None else q
    s = torch.empty((M,), device=x.device, dtype=torch.float32) if s is None else s
    _lib.call("specq_quantize_act_int8", x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), s.data_ptr(),
              M, K, int(grid_m_max or 0), _plan_ptr(plan), _stream_ptr(x))
    return q, s


def silu_mul_quant_int8(gate, up, q=None, s=None, plan=None, grid_m_max=None):
    """quantize_act_int8(silu_mul(gate, up)) fused on the GPU; returns (int8 [M, N], fp32 [M])."""
    _require_gpu(gate, up)
    M, N = gate.shape
    gate, up = _rowmajor(gate), _rowmajor(up)
    q = torch.empty((M, N), device=gate.device, dtype=torch.int8) if q is None else q
    s = torch.empty((M,), device=gate.device, dtype=torch.float32) if s is None else s
    _lib.call("specq_silu_mul_quant_int8", gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0),
              q.data_ptr(), q.stride(0), s.data_ptr(), M, N, int(grid_m_max or 0), _plan_ptr(plan),
              _stream_ptr(gate))
    return q, s


# ----------------------------------------------------------------------------------------
# Paged INT8 KV-cache append (the device-side counterpart of make_paged_kv's q8)
# ----------------------------------------------------------------------------------------
def paged_kv_append(k_new, v_new, kc, vc, ks, vs, block_tbl, ctx_len, q_len=None, plan=None, n_seqs=None):
    """Quantise the new tokens' K/V into the paged INT8 cache, in place (kernels.py:280-284).

    k_new, v_new fp16 [B, QLMAX, H_KV, D] (the q_len tokens being verified); kc/vc int8
    [pages, PAGE, H_KV, D]; ks/vs fp16 or fp32 [pages, PAGE, H_KV]; block_tbl int32
    [B, max_pages]; ctx_len int32 [B], already counting the new tokens, so token i of
    sequence b goes to position ctx_len[b] - q_len + i.  Each (token, head) row gets
    s = max(amax, 1e-8) / 127 and q = clamp(rne(x / s), -127, 127), exactly as the
    reference quantises its cache.  With `plan`, (n_seqs, q_len) = plan[0:2] on the device
    and the grid covers (B, QLMAX).  Slots of inactive sequences and tokens are not written.
    """
    _require_gpu(k_new, v_new, kc, vc, ks, vs, block_tbl, ctx_len)
    B, QLMAX, H_KV, D = k_new.shape
    if v_new.shape != k_new.shape:
        raise RuntimeError("paged_kv_append: k_new and v_new must have the same shape")
    if k_new.dtype != torch.float16 or v_new.dtype != torch.float16:
        raise RuntimeError("paged_kv_append expects fp16 k_new and v_new")
    if kc.dtype != torch.int8 or vc.dtype != torch.int8 or kc.shape != vc.shape:
        raise RuntimeError("paged_kv_append expects int8 K/V caches of one shape")
    if kc.shape[2] != H_KV or kc.shape[3] != D:
        raise RuntimeError(f"paged_kv_append: cache {tuple(kc.shape)} does not match new K/V {tuple(k_new.shape)}")
    if kc.stride() != vc.stride() or ks.stride() != vs.stride() or ks.dtype != vs.dtype:
        raise RuntimeError("paged_kv_append: K and V (and their scales) must share layout and dtype")
    if ks.dtype not in (torch.float16, torch.float32):
        raise RuntimeError("paged_kv_append: scales must be fp16 or fp32")
    if block_tbl.dtype != torch.int32 or ctx_len.dtype != torch.int32:
        raise RuntimeError("paged_kv_append: block_tbl and ctx_len must be int32")
    if kc.stride(3) != 1:
        raise RuntimeError("paged_kv_append: head_dim of the cache must be contiguous")
    if k_new.stride() != v_new.stride() or k_new.stride(3) != 1:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    block_tbl = _rowmajor(block_tbl)
    ctx_len = ctx_len.contiguous()
    q_len = QLMAX if q_len is None else int(q_len)
    n_seqs = B if n_seqs is None else int(n_seqs)
    if not (0 <= n_seqs <= B and 0 <= q_len <= QLMAX):
        raise RuntimeError(f"paged_kv_append: need 0 <= n_seqs <= {B} and 0 <= q_len <= {QLMAX}")
    B_grid = B if plan is not None else n_seqs
    ql_grid = QLMAX if plan is not None else q_len
    if block_tbl.dim() != 2 or block_tbl.shape[0] < B_grid or ctx_len.numel() < B_grid:
        raise RuntimeError("paged_kv_append: block_tbl and ctx_len must cover every sequence of the grid")
    _lib.call("specq_kv_append_int8",
              k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_new.stride(1), k_new.stride(2),
              kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2),
              ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), ks.stride(2),
              1 if ks.dtype == torch.float32 else 0,
              block_tbl.data_ptr(), block_tbl.stride(0), block_tbl.shape[1], kc.shape[0], ctx_len.data_ptr(),
              B_grid, n_seqs, q_len, ql_grid, H_KV, D, kc.shape[1], _plan_ptr(plan), _stream_ptr(k_new))


# ----------------------------------------------------------------------------------------
# W4A8: INT4 weights on the INT8 MFMA path, per-channel scale in the W8A8 epilogue
# ----------------------------------------------------------------------------------------
def quantize_weight_int4_channel(w):
    """Per-channel symmetric INT4 weight for w4a8_matmul: (packed uint8 [N, K/2], scale fp32 [N]).

    The reference quantiser with one group per row (kernels.py:138-147 at group = K) and the
    scale kept in fp32: sc = max(amax_row, 1e-8) / 7, q = clamp(round(w / sc), -8, 7) + 8,
    packed as the reference packs (byte j = q[:, j] | q[:, j + K/2] << 4).
    """
    N, K = w.shape
    if K % 2:
        raise RuntimeError("quantize_weight_int4_channel: K must be even")
    wf = w.float()
    sc = wf.abs().amax(-1).clamp(min=1e-8) / 7.0
    q = (torch.round(wf / sc[:, None]).clamp(-8, 7) + 8).to(torch.uint8)
    half = K // 2
    return (q[:, :half] | (q[:, half:] << 4)).contiguous(), sc


class PackedWeightW4A8:
    """An INT4 weight packed once into the W4A8 kernel's 512-byte MFMA fragments.

    Source: the reference uint8 packing [N, K/2] (byte j holds k = j and k = j + K/2) or the
    int32 packing [N, K/8] (nibble i of word j holds k = 8j + i), nibbles with offset 8.
    Fragment (64-wide K step s, 16-row tile t) is the 512 bytes at (s * ceil(N/16) + t) * 512.
    """

    def __init__(self, wq: torch.Tensor, K: int = None):
        _require_gpu(wq)
        if wq.dim() != 2 or wq.dtype not in (torch.uint8, torch.int32):
            raise RuntimeError("PackedWeightW4A8 expects a uint8 [N, K/2] or int32 [N, K/8] INT4 weight")
        wq = _rowmajor(wq)
        layout = 0 if wq.dtype == torch.uint8 else 1
        self.N = wq.shape[0]
        self.K = int(K) if K is not None else wq.shape[1] * (2 if layout == 0 else 8)
        self.shape = (self.N, self.K)
        self.device = wq.device
        nbytes = _lib.lib().specq_w4a8_packed_bytes(self.N, self.K)
        self.data = torch.empty(nbytes, dtype=torch.int8, device=wq.device)
        _lib.call("specq_w4a8_pack_weight", wq.data_ptr(), wq.stride(0), layout, self.N, self.K,
                  self.data.data_ptr(), _stream_ptr(wq))


def pack_weight_w4a8(wq, K: int = None):
    """Pack an INT4 weight (uint8 [N, K/2] or int32 [N, K/8]) for w4a8_matmul."""
    return PackedWeightW4A8(wq, K)


def w4a8_matmul(a_q, sa, wq, sw, out=None, BLOCK_M=16, BLOCK_N=None, BLOCK_K=128, num_warps=4,
                num_stages=3, plan=None, grid_m_max=None, split_k=0, workspace=None):
    """C[M, N] = fp16((int32(a_q @ (q - 8).T) * sa[:, None]) * sw[None, :]).  Returns (out, ck).

    a_q int8 [M, K] with per-token scale sa fp32 [M] (quantize_act_int8); wq a
    PackedWeightW4A8, or an INT4 weight in the reference uint8 / int32 packing (packed here on
    every call; pack once at load time instead); sw fp32 [N] per-channel scale
    (quantize_weight_int4_channel).  Arguments otherwise as w8a8_matmul; results are
    bit-identical to w8a8_matmul on the unpacked INT4 weight.
    """
    if not isinstance(wq, PackedWeightW4A8):
        wq = PackedWeightW4A8(wq, a_q.shape[1])
    _require_gpu(a_q, sa, sw)
    if a_q.dtype != torch.int8:
        raise RuntimeError("w4a8_matmul expects int8 activations")
    M, K = a_q.shape
    N = wq.N
    if wq.K != K:
        raise RuntimeError(f"w4a8_matmul: K mismatch {tuple(a_q.shape)} vs {wq.shape}")
    a_q = _rowmajor(a_q)
    sa = sa.float().contiguous()
    sw = sw.float().contiguous()
    if out is None:
        out = torch.empty((M, N), device=a_q.device, dtype=torch.float16)
    if out.dtype != torch.float16 or out.stride(-1) != 1:
        raise RuntimeError("w4a8_matmul: out must be fp16 with unit inner stride")
    m_grid = int(grid_m_max) if grid_m_max is not None else M
    bm = int(BLOCK_M) if BLOCK_M else 0  # 0: the library picks the tile (cost model over M, N, K)
    bn = _w8a8_block_n(BLOCK_N)
    nw = int(num_warps) if num_warps else 4
    ws = workspace.on(a_q.get_device()) if workspace is not None else _ws.shared(a_q.device)
    need = _lib.lib().specq_w4a8_packed_workspace_size(m_grid, N, K, bm, bn, nw, split_k)
    wptr, wbytes = ws.ensure(need)
    _lib.call("specq_w4a8_packed", a_q.data_ptr(), a_q.stride(0), wq.data.data_ptr(),
              sa.data_ptr(), sw.data_ptr(), out.data_ptr(), out.stride(0),
              M, N, K, int(grid_m_max or 0), _plan_ptr(plan), bm, bn, nw, split_k,
              wptr, wbytes, _stream_ptr(a_q))
    _w8a8_kernel._note(a_q.device.index or 0, (bm, bn, nw, "w4a8"))
    return out, KernelInfo(0, 2 | (16 if plan is not None else 0), m_grid, N, K, bm, bn, nw, split_k)


# ----------------------------------------------------------------------------------------
# Rotary positions, and the paged cache with block scales (no reference counterpart)
# ----------------------------------------------------------------------------------------
def _gpu_of(who: str, *ts) -> int:
    """The index of the GPU that holds all tensors (None left out)."""
    dev = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise RuntimeError(f"{who}: tensors on {ts[0].device} and {t.device}")
    if dev < 0 or ts[0].device.type != "cuda":
        raise RuntimeError(f"specq kernels run on the GPU only; got a {ts[0].device} tensor")
    return dev


def _call_on(dev: int, name: str, *args) -> None:
    """Call an entry point on GPU `dev`'s current stream (its last argument), with that GPU the current one, so
    that the launch and the CU count are its own."""
    if dev == torch._C._cuda_getDevice():
        _lib.packed(name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            _lib.packed(name)(*args, torch._C._cuda_getCurrentRawStream(dev))


def _workspace(workspace, dev: int):
    return _ws.shared_cuda(dev) if workspace is None else workspace.on(dev)


def _plan_of(plan, need: int, who: str) -> int:
    if plan is None:
        return 0
    if plan.dtype != torch.int32 or plan.numel() < need or plan.stride(-1) != 1:
        raise RuntimeError(f"{who}: plan must be an int32 device tensor of at least {need} entries")
    return plan.data_ptr()


def _token_grid(who: str, B: int, QL: int, q_len, n_seqs, plan):
    """(sequences and tokens of the grid, n_seqs, q_len) of a call on [B, QL, ...] tensors."""
    q_len = QL if q_len is None else int(q_len)
    n_seqs = B if n_seqs is None else int(n_seqs)
    if not (0 <= n_seqs <= B and 0 <= q_len <= QL):
        raise RuntimeError(f"{who}: need 0 <= n_seqs <= {B} and 0 <= q_len <= {QL}")
    return (B, QL, n_seqs, q_len) if plan is not None else (n_seqs, q_len, n_seqs, q_len)


def _int32_vec(who: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] < n or (t.stride(0) != 1 and t.shape[0] > 1):
        raise RuntimeError(f"{who}: {name} must be a contiguous int32 vector of at least {n} entries")


def rotary_inv_freq(dim: int, base: float = 10000.0, scaling=None, factor: float = 1.0, original_len: int = 8192,
                    low_freq_factor: float = 1.0, high_freq_factor: float = 4.0, beta_fast: float = 32.0,
                    beta_slow: float = 1.0, device="cuda"):
    """(inv_freq fp64 [dim / 2], mscale) for rotary_embed: f_j = base^(-2j / dim), stretched for long contexts.

    scaling: None; "linear" (f / factor); "ntk" (base * factor^(dim / (dim - 2))); "wavelength" (waves longer
    than original_len / low_freq_factor divided by factor, those shorter than original_len / high_freq_factor
    kept, a blend between); "yarn" (f / factor for pairs that turn less than beta_slow times in original_len
    tokens, f for those above beta_fast, a ramp over the pair's index between, which may end past the last pair;
    mscale 0.1 ln(factor) + 1).
    """
    dim = int(dim)
    if dim < 2 or dim % 2:
        raise RuntimeError(f"rotary_inv_freq: dim={dim} must be even and at least 2")
    if not (base > 1 and factor > 0 and original_len > 0):
        raise RuntimeError("rotary_inv_freq: need base > 1, factor > 0 and original_len > 0")
    if scaling == "ntk":
        if dim == 2:
            raise RuntimeError("rotary_inv_freq: \"ntk\" needs dim > 2")
        base = base * factor ** (dim / (dim - 2))
    f = torch.tensor([base ** (-2.0 * j / dim) for j in range(dim // 2)], dtype=torch.float64)
    mscale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "wavelength":
        if not high_freq_factor > low_freq_factor:
            raise RuntimeError("rotary_inv_freq: high_freq_factor must exceed low_freq_factor")
        turns = original_len * f / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    elif scaling == "yarn":
        if not beta_fast >= beta_slow > 0:
            raise RuntimeError("rotary_inv_freq: need beta_fast >= beta_slow > 0")
        index = lambda turns: dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        # Cut at dim - 1, not at the last pair: where that pair still turns more than beta_slow times, the ramp ends past it.
        lo, hi = max(math.floor(index(beta_fast)), 0), min(math.ceil(index(beta_slow)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mscale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise RuntimeError(f"rotary_inv_freq: unknown scaling {scaling!r}")
    return f.to(device), mscale


def _rotary_out(who: str, x, shape, strides, D: int, out):
    """Checks an input of rotary_embed and its output, made where omitted; returns the output and its strides."""
    if x.dtype != torch.float16 or (D > 1 and strides[3] != 1):
        raise RuntimeError(f"{who}: inputs must be fp16 with contiguous head_dim")
    if out is None:
        out = torch.empty_like(x)
    elif out.dtype != torch.float16 or out.shape != shape:
        raise RuntimeError(f"{who}: inputs and outputs must be fp16 of one shape")
    so = out.stride()
    if D > 1 and so[3] != 1:
        raise RuntimeError(f"{who}: head_dim must be contiguous")
    return out, so


def rotary_embed(q, k, inv_freq, ctx_len=None, q_len=None, positions=None, interleaved=False, mscale=1.0, plan=None,
                 n_seqs=None, q_out=None, k_out=None, _norm=None):
    """Rotary positions of the new tokens' q and k; returns (q_out, k_out).

    q fp16 [B, QL, H, D], k fp16 [B, QL, H_KV, D] or None; inv_freq fp32 or fp64 [R / 2], R <= D <= 512
    (rotary_inv_freq).  Pair j of the first R dimensions -- (j, j + R/2), or (2j, 2j + 1) with
    interleaved -- is turned by pos * inv_freq[j] and scaled by mscale; the other dimensions are copied.
    Token i of sequence b is at ctx_len[b] - q_len + i (ctx_len counts the new tokens, as the K/V append
    and the attention have it), or at positions[b, i] (int32 [B, QL]).  Angles are formed in fp64.
    Outputs may be the inputs (in place); they must not overlap them otherwise.  With `plan`,
    (n_seqs, q_len) = plan[0:2] on the device and the grid covers (B, QL).  Tokens that are not active
    are not written (an omitted output holds anything there).
    """
    # _norm: qk_norm_rotary's (q_weight, k_weight, eps).  One body, since a function between it and the callers costs a step 4 %.
    if _norm is None:
        who = "rotary_embed"
        dev = _gpu_of(who, q, k, inv_freq, ctx_len, positions, plan, q_out, k_out)
    else:
        who = "qk_norm_rotary"
        q_weight, k_weight, eps = _norm
        dev = _gpu_of(who, q, k, q_weight, k_weight, inv_freq, ctx_len, positions, plan, q_out, k_out)
    shape, qs = q.shape, q.stride()
    if len(shape) != 4:
        raise RuntimeError(f"{who}: q [B, QL, H, D] expected")
    B, QL, H, D = shape
    q_out, qo = _rotary_out(who, q, shape, qs, D, q_out)
    if k is not None:
        shape, ks = k.shape, k.stride()
        if len(shape) != 4 or shape[0] != B or shape[1] != QL or shape[3] != D:
            raise RuntimeError(f"{who}: k [B, QL, H_KV, D] expected")
        H_KV = shape[2]
        k_out, ko = _rotary_out(who, k, shape, ks, D, k_out)
    elif k_out is not None:
        raise RuntimeError(f"{who}: k_out without k")
    else:
        H_KV, ks, ko = 0, (0, 0, 0), (0, 0, 0)
    if inv_freq.dtype not in (torch.float32, torch.float64) or inv_freq.dim() != 1 or \
            (inv_freq.stride(0) != 1 and inv_freq.shape[0] > 1):
        raise RuntimeError(f"{who}: inv_freq must be a contiguous fp32 or fp64 vector")
    Bg, Qg, n_seqs, q_len = _token_grid(who, B, QL, q_len, n_seqs, plan)
    s_pb = 0
    if positions is not None:
        if positions.dtype != torch.int32 or positions.dim() != 2 or positions.shape[0] < Bg or \
                positions.shape[1] < Qg or (positions.stride(1) != 1 and positions.shape[1] > 1):
            raise RuntimeError(f"{who}: positions must be int32 [B, QL] with unit inner stride")
        s_pb = positions.stride(0)
    elif ctx_len is not None:
        _int32_vec(who, "ctx_len", ctx_len, Bg)
    else:
        raise RuntimeError(f"{who}: ctx_len or positions must be given")
    if _norm is not None:
        if k is None and k_weight is not None:
            raise RuntimeError(f"{who}: k_weight without k")
        s_wq = _norm_weights(who, "q_weight", q_weight, H, D)
        s_wk = _norm_weights(who, "k_weight", k_weight, H_KV, D)
        w = q_weight if q_weight is not None else k_weight
        if k_weight is not None and w.dtype != k_weight.dtype:
            raise RuntimeError(f"{who}: q_weight and k_weight must be of one type")
    if Bg == 0 or Qg == 0:
        return q_out, k_out
    R = 2 * inv_freq.shape[0]
    if _norm is None:
        _call_on(dev, "specq_rotary", q.data_ptr(), qs[0], qs[1], qs[2], _ptr(k), ks[0], ks[1], ks[2],
                 q_out.data_ptr(), qo[0], qo[1], qo[2], _ptr(k_out), ko[0], ko[1], ko[2],
                 inv_freq.data_ptr(), inv_freq.dtype == torch.float64, mscale,
                 _ptr(ctx_len), _ptr(positions), s_pb, Bg, n_seqs, q_len, Qg, H, H_KV, D, R,
                 bool(interleaved), _plan_of(plan, 2, who))
    else:
        _call_on(dev, "specq_qk_norm_rotary", q.data_ptr(), qs[0], qs[1], qs[2], _ptr(k), ks[0], ks[1], ks[2],
                 q_out.data_ptr(), qo[0], qo[1], qo[2], _ptr(k_out), ko[0], ko[1], ko[2],
                 _ptr(q_weight), s_wq, _ptr(k_weight), s_wk, w is not None and w.dtype == torch.float32, eps,
                 inv_freq.data_ptr(), inv_freq.dtype == torch.float64, mscale,
                 _ptr(ctx_len), _ptr(positions), s_pb, Bg, n_seqs, q_len, Qg, H, H_KV, D, R,
                 bool(interleaved), _plan_of(plan, 2, who))
    return q_out, k_out


def _norm_weights(who: str, name: str, w, heads: int, D: int) -> int:
    """Checks norm weights [D] or [heads, D]; returns the elements from head to head."""
    if w is None:
        return 0
    if w.dtype not in (torch.float16, torch.float32) or w.dim() not in (1, 2) or w.shape[-1] != D or \
            (w.stride(-1) != 1 and D > 1) or (w.dim() == 2 and w.shape[0] != heads):
        raise RuntimeError(f"{who}: {name} must be fp16 or fp32 [{D}] or [{heads}, {D}] with unit inner stride")
    return w.stride(0) if w.dim() == 2 else 0


def qk_norm_rotary(q, k, q_weight, k_weight, inv_freq, ctx_len=None, q_len=None, positions=None, interleaved=False,
                   mscale=1.0, eps=1e-6, plan=None, n_seqs=None, q_out=None, k_out=None):
    """Norms of the new tokens' q and k for each head, and their rotary positions, in one pass; returns (q_out, k_out).

    A head's row x becomes y = x / sqrt(mean(x^2) + eps) * weight, whose first dimensions are then turned as
    rotary_embed turns them: fp32, rounded once.  q_weight, k_weight fp16 or fp32, both of one type, [D], or a row for
    each head ([H, D], [H_KV, D]), or None (no weights; k_weight is None where k is).  Everything else as rotary_embed.
    """
    return rotary_embed(q, k, inv_freq, ctx_len, q_len, positions, interleaved, mscale, plan, n_seqs, q_out, k_out,
                        (q_weight, k_weight, eps))


def _block_cache(who: str, kc, vc, ks, vs, block_tbl, ctx_len, seqs: int, H_KV: int, D: int):
    """Checks a block-scaled cache for `seqs` sequences; returns (e4m3 codes, tokens per block, strides of the codes
    and of the scales)."""
    kind = kc.dtype
    if kind != vc.dtype or kind not in (torch.int8, torch.float8_e4m3fn):
        raise RuntimeError(f"{who} expects int8 or float8_e4m3fn K/V caches of one type")
    shape, cs = kc.shape, kc.stride()
    if len(shape) != 4 or shape != vc.shape or cs != vc.stride() or cs[3] != 1:
        raise RuntimeError(f"{who}: K/V caches must share a layout [pages, PAGE, H_KV, D] with contiguous head_dim")
    P, PAGE, heads, dim = shape
    if heads != H_KV or dim != D:
        raise RuntimeError(f"{who}: cache {tuple(shape)} does not fit {H_KV} K/V heads of {D}")
    shape, ss = ks.shape, ks.stride()
    if ks.dtype != torch.float32 or vs.dtype != torch.float32 or len(shape) != 3 or shape != vs.shape or ss != vs.stride():
        raise RuntimeError(f"{who}: scales must be fp32 [pages, blocks, H_KV] of one layout")
    NB = shape[1]
    if shape[0] != P or shape[2] != H_KV or NB < 1 or PAGE % NB or (PAGE // NB) % 16:
        raise RuntimeError(f"{who}: scales {tuple(shape)} must be [{P}, blocks, {H_KV}] with blocks of a multiple "
                           f"of 16 of the page's {PAGE} tokens")
    if block_tbl.dtype != torch.int32 or block_tbl.dim() != 2 or block_tbl.shape[0] < seqs or \
            (block_tbl.stride(1) != 1 and block_tbl.shape[1] > 1):
        raise RuntimeError(f"{who}: block_tbl must be int32 [B, max_pages] with unit inner stride for {seqs} sequences")
    _int32_vec(who, "ctx_len", ctx_len, seqs)
    return kind == torch.float8_e4m3fn, PAGE // NB, cs, ss


def paged_kv_append_block_scaled(k_new, v_new, kc, vc, ks, vs, block_tbl, ctx_len, q_len=None, plan=None, n_seqs=None):
    """Quantise the new tokens' K/V into a paged cache with block scales, in place.

    k_new, v_new fp16 [B, QLMAX, H_KV, D], D 64, 128 or 256; kc/vc int8 or float8_e4m3fn [pages, PAGE,
    H_KV, D]; ks/vs fp32 [pages, PAGE / SB, H_KV], one scale for each block of SB tokens (a multiple of
    16) and head; block_tbl int32 [B, max_pages]; ctx_len int32 [B], counting the new tokens.  A block
    that new tokens reach gets s' = max(amax, 1e-8) / Q (Q = 127 or 448) over them, or its present
    scale where that is larger and the block holds earlier tokens of the sequence; the new codes are
    rne(x / s'), and where the scale grows the earlier codes become rne(c * s / s') (NaN stays NaN).  New
    infinities count as +-65504, new NaN as 0.  Present scales are finite and not negative.  Tokens at
    positions below zero, past the table or on a page outside the pool are skipped, every other slot keeps
    what it holds.  A page that the call writes must be named by one entry of the table only (paged_kv_fork
    sees to that, unless a row is cut back into a page it shares).  D = 256 is for other readers:
    paged_attention_block_scaled takes 64 and 128.  With `plan`, (n_seqs, q_len) = plan[0:2] on the device
    and the grid covers (B, QLMAX).
    """
    who = "paged_kv_append_block_scaled"
    dev = _gpu_of(who, k_new, v_new, kc, vc, ks, vs, block_tbl, ctx_len, plan)
    if k_new.dim() != 4 or v_new.shape != k_new.shape:
        raise RuntimeError(f"{who}: k_new and v_new must have one shape [B, QLMAX, H_KV, D]")
    if k_new.dtype != torch.float16 or v_new.dtype != torch.float16:
        raise RuntimeError(f"{who} expects fp16 k_new and v_new")
    B, QL, H_KV, D = k_new.shape
    Bg, Qg, n_seqs, q_len = _token_grid(who, B, QL, q_len, n_seqs, plan)
    f8, sb, cs, ss = _block_cache(who, kc, vc, ks, vs, block_tbl, ctx_len, Bg, H_KV, D)
    if k_new.stride() != v_new.stride() or k_new.stride(3) != 1:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if Bg == 0 or Qg == 0:
        return
    kn = k_new.stride()
    _call_on(dev, "specq_kv_append_block", k_new.data_ptr(), v_new.data_ptr(), kn[0], kn[1], kn[2],
             kc.data_ptr(), vc.data_ptr(), f8, cs[0], cs[1], cs[2],
             ks.data_ptr(), vs.data_ptr(), ss[0], ss[1], ss[2], sb,
             block_tbl.data_ptr(), block_tbl.stride(0), block_tbl.shape[1], min(kc.shape[0], 2**31 - 1),
             ctx_len.data_ptr(), Bg, n_seqs, q_len, Qg, H_KV, D, kc.shape[1], _plan_of(plan, 2, who))


@functools.lru_cache(maxsize=4096)
def _block_attn_workspace(Bg, H, H_KV, Qg, QPP, D, max_pages, PAGE, plan, dev, options) -> int:
    """Bytes a call needs: a function of its sizes, the GPU's CU count and the library options."""
    with torch.cuda.device(dev):
        return _lib.lib().specq_paged_attn_block_workspace_size(Bg, H, H_KV, Qg, QPP, D, max_pages, PAGE, plan)


@functools.lru_cache(maxsize=None)
def _block_attn_info(D, f8, rows, dev) -> KernelInfo:
    with torch.cuda.device(dev):
        return KernelInfo(2, D | (1 << 18 if f8 else 1 << 17), 0, 0, 0, rows, 0, 4, 0)


def paged_attention_block_scaled(q, kc, vc, ks, vs, block_tbl, ctx_len, q_len=None, QPP=None, plan=None, n_seqs=None,
                                 out=None, sm_scale=None, workspace=None):
    """Verification attention over a paged cache with block scales.  Returns (out, ck).

    q fp16 [B, QLMAX, H, D], D 64 or 128; kc/vc int8 or float8_e4m3fn [pages, PAGE, H_KV, D]; ks/vs fp32
    [pages, PAGE / SB, H_KV] (paged_kv_append_block_scaled); block_tbl int32 [B, max_pages]; ctx_len
    int32 [B], counting the q_len new tokens, which are each sequence's last ones and see one another
    causally; a context longer than the table counts as the table's length.  Block-table ids outside
    [0, pages) mask their page's tokens; a row that sees no token gives 0.  QPP query tokens run in one
    program, at most 64 rows of H / H_KV heads each (default: as few programs as that takes, of even
    size); every QPP gives the same bits.  sm_scale defaults to D^-1/2.  With `plan`, (n_seqs, q_len) =
    plan[0:2] on the device and the grid covers (B, QLMAX); rows that are not active are not written (an
    omitted `out` is zero there).  Calls that may run at the same time on several streams need a workspace
    each.
    """
    who = "paged_attention_block_scaled"
    dev = _gpu_of(who, q, kc, vc, ks, vs, block_tbl, ctx_len, plan, out)
    if q.dim() != 4 or q.dtype != torch.float16 or q.stride(3) != 1:
        raise RuntimeError(f"{who} expects fp16 q [B, QLMAX, H, D] with contiguous head_dim")
    B, QL, H, D = q.shape
    if H < 1 or kc.dim() != 4 or kc.shape[2] < 1 or H % kc.shape[2]:
        raise RuntimeError(f"{who}: cache {tuple(kc.shape)} does not fit q {tuple(q.shape)}")
    H_KV = kc.shape[2]
    G = H // H_KV
    Bg, Qg, n_seqs, q_len = _token_grid(who, B, QL, q_len, n_seqs, plan)
    f8, sb, cs, ss = _block_cache(who, kc, vc, ks, vs, block_tbl, ctx_len, Bg, H_KV, D)
    if QPP is None:
        n = -(-Qg // max(1, 64 // G))  # programs
        QPP = max(1, -(-Qg // max(1, n)))
    elif int(QPP) < 1:
        raise RuntimeError(f"{who}: QPP={QPP} must be at least 1")
    if out is None:
        out = torch.empty_like(q) if plan is None and n_seqs == B and q_len == QL else torch.zeros_like(q)
    elif out.dtype != torch.float16 or out.shape != q.shape or out.stride(3) != 1:
        raise RuntimeError(f"{who}: out must be fp16 of q's shape {tuple(q.shape)} with contiguous head_dim")
    PAGE, max_pages = kc.shape[1], block_tbl.shape[1]
    qs, os_ = q.stride(), out.stride()
    QPP = int(QPP)
    ck = _block_attn_info(D, f8, QPP * G, dev)
    if Bg == 0 or Qg == 0:
        return out, ck
    need = _block_attn_workspace(Bg, H, H_KV, Qg, QPP, D, max_pages, PAGE, plan is not None, dev, _lib.options_key())
    wptr, wbytes = _workspace(workspace, dev).ensure(need)
    _call_on(dev, "specq_paged_attn_block", q.data_ptr(), qs[0], qs[1], qs[2],
             kc.data_ptr(), vc.data_ptr(), f8, cs[0], cs[1], cs[2],
             ks.data_ptr(), vs.data_ptr(), ss[0], ss[1], ss[2], sb,
             block_tbl.data_ptr(), block_tbl.stride(0), max_pages, min(kc.shape[0], 2**31 - 1),
             ctx_len.data_ptr(), out.data_ptr(), os_[0], os_[1], os_[2],
             Bg, n_seqs, q_len, Qg, H, H_KV, D, PAGE, QPP,
             D ** -0.5 if sm_scale is None else sm_scale, _plan_of(plan, 2, who), wptr, wbytes)
    _paged_attn_kernel._note(dev, (D, (QPP * G + 15) // 16, kc.dtype))
    return out, ck


# ----------------------------------------------------------------------------------------
# Page tables of the paged caches
# ----------------------------------------------------------------------------------------
def _page_state(who: str, block_tbl, ref, *vecs, out=None):
    """Checks the table, the counts and per-row vectors (name, tensor), and that `out`, where given, is on their GPU;
    returns (GPU, B, C, P)."""
    dev = _gpu_of(who, block_tbl, ref, *(t for _, t in vecs), out)
    if block_tbl.dtype != torch.int32 or block_tbl.dim() != 2 or block_tbl.shape[0] < 1 or block_tbl.shape[1] < 1 or \
            (block_tbl.stride(1) != 1 and block_tbl.shape[1] > 1):
        raise RuntimeError(f"{who}: block_tbl must be int32 [B, max_pages] with unit inner stride")
    if block_tbl.shape[0] > 1 and block_tbl.stride(0) < block_tbl.shape[1]:
        raise RuntimeError(f"{who}: block_tbl rows overlap")
    _int32_vec(who, "ref", ref, 1)
    B, C = block_tbl.shape
    for name, t in vecs:
        _int32_vec(who, name, t, B)
    return dev, B, C, ref.shape[0]


def _page_tensors(who: str, caches, pages: int, dev: int):
    """The page tensors of a pool: (their number, [bases, page strides, page bytes] as one array)."""
    base, stride, nbytes = [], [], []
    for t in caches:
        if t.get_device() != dev:
            raise RuntimeError(f"{who}: a cache on {t.device}, the table on GPU {dev}")
        if t.dim() < 1 or t.shape[0] != pages or t.numel() == 0:
            raise RuntimeError(f"{who}: a cache {tuple(t.shape)} must have {pages} pages")
        if not t.is_contiguous() and not t[0].is_contiguous():
            raise RuntimeError(f"{who}: the pages of a cache must be contiguous")
        size = t.element_size()
        n = t.numel() // pages * size
        nbytes.append(n)
        stride.append(t.stride(0) * size if pages > 1 else n)
        base.append(t.data_ptr())
    return len(base), array.array("q", base + stride + nbytes)


def _page_tensor_args(n: int, words) -> tuple:
    at = words.buffer_info()[0]
    return n, at, at + 8 * n, at + 16 * n


def _pages_workspace(workspace, dev: int, B: int, C: int, P: int):
    need = _lib.lib().specq_kv_pages_workspace_size(B, C, P)
    return _workspace(workspace, dev).ensure(need)


def paged_kv_reserve(block_tbl, ref, lens, PAGE, shortage=None, workspace=None):
    """Give the rows of a block table the pages that lens[b] tokens need, in place.

    block_tbl int32 [B, max_pages]; ref int32 [pages], how often the tables name each page (<= 0: free);
    lens int32 [B].  Entries of a row's first ceil(lens / PAGE) columns that name no page (an id outside
    [0, pages)) get the lowest free page, in the table's order; ref of a page given becomes 1.  Where the
    free pages run out, entries get -1.  Returns shortage, int32 [1]: how many pages are missing (a row has no
    more than its max_pages columns, whatever lens says).  Calls that may run beside other calls on another
    stream need a workspace of their own, here as in paged_kv_fork and paged_kv_compact.
    """
    who = "paged_kv_reserve"
    dev, B, C, P = _page_state(who, block_tbl, ref, ("lens", lens), out=shortage)
    shortage = torch.empty(1, dtype=torch.int32, device=ref.device) if shortage is None else shortage
    _int32_vec(who, "shortage", shortage, 1)
    wptr, wbytes = _pages_workspace(workspace, dev, B, C, P)
    _call_on(dev, "specq_kv_pages_reserve", block_tbl.data_ptr(), block_tbl.stride(0) if B > 1 else C, B, C,
             ref.data_ptr(), P, lens.data_ptr(), int(PAGE), shortage.data_ptr(), wptr, wbytes)
    return shortage


def paged_kv_free(block_tbl, ref, keep, PAGE):
    """Let go of the pages past each row's first keep[b] tokens (0: the whole row), in place.

    Entries past a row's first ceil(keep / PAGE) columns become -1, and ref of each page they named
    falls by one; a page that no table names any more (ref 0) is free.  A row that keep cuts back into a page it
    shares with another (paged_kv_fork) must not be appended to before it has a page of its own there.
    """
    who = "paged_kv_free"
    dev, B, C, P = _page_state(who, block_tbl, ref, ("keep", keep))
    _call_on(dev, "specq_kv_pages_free", block_tbl.data_ptr(), block_tbl.stride(0) if B > 1 else C, B, C,
             ref.data_ptr(), P, keep.data_ptr(), int(PAGE))


def paged_kv_fork(block_tbl, ref, lens, parent, caches, PAGE, shortage=None, workspace=None):
    """Make row b a copy of row parent[b], in place: several samples of a prompt, a beam's survivors.

    lens int32 [B], tokens each row holds, becomes lens[parent]; parent int32 [B], an id outside [0, B)
    empties the row.  Rows share their parent's full pages.  Of the rows with one parent the lowest
    keeps its partly filled last page, the others get a free page each (lowest first, in the order of the
    rows) with a copy of it, in every tensor of `caches` ([pages, ...], each page contiguous; K, V and
    scales of any number of layers).  ref follows; pages that no row names any more are free, and may be
    given out by this very call.  Where the free pages run out a row's last entry is -1.  A row's pages
    past its tokens are let go of.  Returns shortage, int32 [1]: how many pages are missing.
    """
    who = "paged_kv_fork"
    dev, B, C, P = _page_state(who, block_tbl, ref, ("lens", lens), ("parent", parent), out=shortage)
    n, words = _page_tensors(who, caches, P, dev)
    shortage = torch.empty(1, dtype=torch.int32, device=ref.device) if shortage is None else shortage
    _int32_vec(who, "shortage", shortage, 1)
    wptr, wbytes = _pages_workspace(workspace, dev, B, C, P)
    _call_on(dev, "specq_kv_pages_fork", block_tbl.data_ptr(), block_tbl.stride(0) if B > 1 else C, B, C,
             ref.data_ptr(), P, lens.data_ptr(), parent.data_ptr(), int(PAGE), *_page_tensor_args(n, words),
             shortage.data_ptr(), wptr, wbytes)
    return shortage


def paged_kv_compact(block_tbl, ref, caches, page_map=None, workspace=None):
    """Move the pages in use below their own number, in place; returns page_map.

    With n pages in use (ref > 0), the i-th of them at or past n moves to the i-th free page below n:
    its contents in every tensor of `caches`, its count, and its entries of block_tbl.  page_map int32
    [pages] holds every page's id afterwards, for other holders of ids.
    """
    who = "paged_kv_compact"
    dev, B, C, P = _page_state(who, block_tbl, ref, out=page_map)
    n, words = _page_tensors(who, caches, P, dev)
    page_map = torch.empty(P, dtype=torch.int32, device=ref.device) if page_map is None else page_map
    _int32_vec(who, "page_map", page_map, P)
    wptr, wbytes = _pages_workspace(workspace, dev, B, C, P)
    _call_on(dev, "specq_kv_pages_compact", block_tbl.data_ptr(), block_tbl.stride(0) if B > 1 else C, B, C,
             ref.data_ptr(), P, page_map.data_ptr(), *_page_tensor_args(n, words), wptr, wbytes)
    return page_map


def paged_kv_copy(src, dst, caches):
    """Copy pages src[i] to dst[i] (int32 vectors) in every tensor of `caches` ([pages, ...]), in place.

    The destinations must be distinct, and none of them a source.  Pairs with an id outside [0, pages)
    are left out.
    """
    who = "paged_kv_copy"
    if len(caches) == 0 or caches[0].dim() < 1:
        raise RuntimeError(f"{who}: no caches of [pages, ...]")
    dev = _gpu_of(who, src, dst)
    n, P = src.numel(), caches[0].shape[0]
    _int32_vec(who, "src", src, n)
    _int32_vec(who, "dst", dst, n)
    if dst.numel() != n:
        raise RuntimeError(f"{who}: {n} sources and {dst.numel()} destinations")
    m, words = _page_tensors(who, caches, P, dev)
    _call_on(dev, "specq_kv_pages_copy", src.data_ptr(), dst.data_ptr(), n, min(P, 2**31 - 1),
             *_page_tensor_args(m, words))


# ----------------------------------------------------------------------------------------
# Eviction by gathered attention weight
# ----------------------------------------------------------------------------------------
def _gathered(who: str, weights, B: int, H_KV: int, tokens: int):
    """Checks gathered weights of at least B sequences; returns their strides."""
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[0] < B or weights.shape[1] != H_KV or \
            weights.shape[2] < tokens or (weights.stride(2) != 1 and weights.shape[2] > 1):
        raise RuntimeError(f"{who}: weights must be fp32 [{B}, {H_KV}, >= {tokens}] with unit inner stride")
    return weights.stride(0), weights.stride(1)


@functools.lru_cache(maxsize=4096)
def _weights_workspace(B, H, H_KV, QL, max_pages, PAGE) -> int:
    """Bytes a call needs: a function of its sizes."""
    return _lib.lib().specq_paged_attn_weights_workspace_size(B, H, H_KV, QL, max_pages, PAGE)


def paged_attention_weights(q, kc, ks, block_tbl, ctx_len, weights, q_len=None, q_lens=None, plan=None, n_seqs=None,
                            sm_scale=None, workspace=None):
    """Add to `weights` the attention weight that the new tokens' queries give each cached token, in place; returns it.

    q fp16 [B, QLMAX, H, D], D 64 or 128; kc int8 [pages, PAGE, H_KV, D], ks fp16 or fp32 [pages, PAGE, H_KV],
    block_tbl int32 [B, max_pages], ctx_len int32 [B] as paged_attention takes them (ctx_len counts the q_len new
    tokens); weights fp32 [B, H_KV, T], T at least max_pages * PAGE.  For a token t of sequence b the softmax
    probabilities p_t of paged_attention's scores are summed over the new tokens and the query heads of KV head h:
    weights[b, h, t] grows by that sum, or becomes it where t is one of the new tokens; positions past the sequence stay.
    q_lens int32 [B]: how many of the q_len tokens sequence b really has (accepted drafts), counted by ctx_len; 0
    leaves its weights as they are.  Block-table ids outside [0, pages) mask their page's tokens, a context longer
    than the table counts as the table's length.  sm_scale defaults to D^-1/2.  A score of -infinity gives its token
    nothing, one of NaN or +infinity makes NaN of its row's share.  With `plan`, (n_seqs, q_len) = plan[0:2] on the device and the grid covers (B, QLMAX).  Calls that may
    run at the same time on several streams need a workspace each.
    """
    who = "paged_attention_weights"
    dev = _gpu_of(who, q, kc, ks, block_tbl, ctx_len, weights, q_lens, plan)
    if q.dim() != 4 or q.dtype != torch.float16 or q.stride(3) != 1:
        raise RuntimeError(f"{who} expects fp16 q [B, QLMAX, H, D] with contiguous head_dim")
    B, QL, H, D = q.shape
    shape, cs = kc.shape, kc.stride()
    if kc.dtype != torch.int8 or len(shape) != 4 or cs[3] != 1:
        raise RuntimeError(f"{who} expects an int8 K cache [pages, PAGE, H_KV, D] with contiguous head_dim")
    P, PAGE, H_KV = shape[0], shape[1], shape[2]
    if shape[3] != D or H_KV < 1 or H % H_KV:
        raise RuntimeError(f"{who}: cache {tuple(shape)} does not fit q {tuple(q.shape)}")
    if ks.dtype not in (torch.float16, torch.float32) or ks.shape != shape[:3]:
        raise RuntimeError(f"{who}: scales must be fp16 or fp32 [{P}, {PAGE}, {H_KV}]")
    Bg, Qg, n_seqs, q_len = _token_grid(who, B, QL, q_len, n_seqs, plan)
    if block_tbl.dtype != torch.int32 or block_tbl.dim() != 2 or block_tbl.shape[0] < Bg or \
            (block_tbl.stride(1) != 1 and block_tbl.shape[1] > 1):
        raise RuntimeError(f"{who}: block_tbl must be int32 [B, max_pages] with unit inner stride for {Bg} sequences")
    _int32_vec(who, "ctx_len", ctx_len, Bg)
    if q_lens is not None:
        _int32_vec(who, "q_lens", q_lens, Bg)
    max_pages = block_tbl.shape[1]
    s_wb, s_wh = _gathered(who, weights, Bg, H_KV, max_pages * PAGE)
    if Bg == 0 or Qg == 0:
        return weights
    wptr, wbytes = _workspace(workspace, dev).ensure(_weights_workspace(Bg, H, H_KV, Qg, max_pages, PAGE))
    qs, ss = q.stride(), ks.stride()
    _call_on(dev, "specq_paged_attn_weights", q.data_ptr(), qs[0], qs[1], qs[2], kc.data_ptr(), cs[0], cs[1], cs[2],
             ks.data_ptr(), ss[0], ss[1], ss[2], ks.dtype == torch.float32,
             block_tbl.data_ptr(), block_tbl.stride(0) if block_tbl.shape[0] > 1 else max_pages, max_pages,
             min(P, 2**31 - 1), ctx_len.data_ptr(), _ptr(q_lens), weights.data_ptr(), s_wb, s_wh,
             Bg, n_seqs, q_len, Qg, H, H_KV, D, PAGE, D ** -0.5 if sm_scale is None else sm_scale,
             _plan_of(plan, 2, who), wptr, wbytes)
    return weights


@functools.lru_cache(maxsize=4096)
def _evict_workspace(B, H_KV, max_pages, PAGE, dev) -> int:
    """Bytes a call needs: a function of its sizes and the GPU's CU count."""
    with torch.cuda.device(dev):
        return _lib.lib().specq_kv_evict_workspace_size(B, H_KV, max_pages, PAGE)


def _cache_rows(who: str, t, pages: int, PAGE: int, H_KV: int):
    """(base, strides from page to page, token to token and head to head, bytes of a row) of a cache [pages, PAGE, H_KV, ...]."""
    shape, st, size = t.shape, t.stride(), t.element_size()
    if len(shape) < 3 or shape[0] != pages or shape[1] != PAGE or shape[2] != H_KV or 0 in shape:
        raise RuntimeError(f"{who}: a cache {tuple(shape)} must be [{pages}, {PAGE}, {H_KV}, ...]")
    n = 1
    for d in range(len(shape) - 1, 2, -1):
        if st[d] != n and shape[d] != 1:
            raise RuntimeError(f"{who}: the rows of a cache must be contiguous")
        n *= shape[d]
    return t.data_ptr(), st[0] * size, st[1] * size, st[2] * size, n * size


def paged_kv_evict(block_tbl, ctx_len, weights, caches, PAGE, budget, recent=0, sinks=0, limit=None, ref=None, kept=None,
                   workspace=None):
    """Cut sequences of more than `limit` tokens (default: budget) back to `budget`, in place; returns kept.

    block_tbl int32 [B, max_pages]; ctx_len int32 [B]; weights fp32 [B, H_KV, >= max_pages * PAGE]
    (paged_attention_weights); caches at most 16 tensors [pages, PAGE, H_KV, ...] of any type, the rest of each
    contiguous (K, V and their scales with a scale for each token; a cache with block scales cannot give single tokens
    up).  For each K/V head stay the first `sinks` tokens, the last `recent` and, of the others, those of greatest weight,
    ties to the lower position; NaN counts as -infinity.  They move together in the order they have: token j comes from
    position kept[b, h, j], in every tensor and in weights, and ctx_len[b] becomes budget.  What lies behind it is left
    as it was; paged_kv_free(block_tbl, ref, ctx_len, PAGE) lets go of its pages.  A sequence stays as it is (kept[j] = j,
    -1 past its tokens) where it is not longer than limit, where one of its table entries names no page and, with the
    page counts `ref` given, where another row names one of its pages too.  Without `ref` the caller answers for
    that: a page must be named by one entry of the table only.  Keys keep the positions they were turned by, so the
    new tokens' positions go on from the uncut length (rotary_embed's `positions`).  Layers that share ctx_len and the table
    but not their caches and weights have a call each, all but the last with a copy of ctx_len.  kept int32
    [B, H_KV, budget].
    """
    who = "paged_kv_evict"
    dev = _gpu_of(who, block_tbl, ctx_len, weights, ref, kept, *caches)
    if block_tbl.dtype != torch.int32 or block_tbl.dim() != 2 or block_tbl.shape[0] < 1 or block_tbl.shape[1] < 1 or \
            (block_tbl.stride(1) != 1 and block_tbl.shape[1] > 1):
        raise RuntimeError(f"{who}: block_tbl must be int32 [B, max_pages] with unit inner stride")
    B, C = block_tbl.shape
    _int32_vec(who, "ctx_len", ctx_len, B)
    PAGE, budget = int(PAGE), int(budget)
    limit = budget if limit is None else int(limit)
    if PAGE < 1 or budget < 1:
        raise RuntimeError(f"{who}: PAGE={PAGE} and budget={budget} must be at least 1")
    if weights.dim() != 3 or weights.shape[1] < 1:
        raise RuntimeError(f"{who}: weights must be fp32 [B, H_KV, T]")
    H_KV = weights.shape[1]
    s_wb, s_wh = _gathered(who, weights, B, H_KV, C * PAGE)
    if len(caches) == 0:
        raise RuntimeError(f"{who}: no caches of [pages, PAGE, H_KV, ...]")
    P = caches[0].shape[0] if caches[0].dim() else 0
    rows = [_cache_rows(who, t, P, PAGE, H_KV) for t in caches]
    if ref is not None:
        _int32_vec(who, "ref", ref, P)
    if kept is None:
        kept = torch.empty((B, H_KV, budget), dtype=torch.int32, device=ctx_len.device)
    elif kept.dtype != torch.int32 or kept.shape != (B, H_KV, budget) or not kept.is_contiguous():
        raise RuntimeError(f"{who}: kept must be contiguous int32 [{B}, {H_KV}, {budget}]")
    words = array.array("q", [v for col in zip(*rows) for v in col])
    at, n = words.buffer_info()[0], len(caches)
    wptr, wbytes = _workspace(workspace, dev).ensure(_evict_workspace(B, H_KV, C, PAGE, dev))
    _call_on(dev, "specq_kv_evict", block_tbl.data_ptr(), block_tbl.stride(0) if B > 1 else C, B, C, _ptr(ref),
             min(P, 2**31 - 1), ctx_len.data_ptr(), weights.data_ptr(), s_wb, s_wh, H_KV, PAGE,
             n, at, at + 8 * n, at + 16 * n, at + 24 * n, at + 32 * n, budget, int(recent), int(sinks), limit,
             kept.data_ptr(), wptr, wbytes)
    return kept


# ----------------------------------------------------------------------------------------
# Beam search
# ----------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _beam_workspace(B, W, V, fp32, dev) -> int:
    """Bytes a call needs: a function of its sizes and the GPU's CU count."""
    with torch.cuda.device(dev):
        return _lib.lib().specq_beam_select_workspace_size(B, W, V, fp32)


def beam_select(logits, scores, n=None, finished=None, eos=None, out=None, workspace=None):
    """The best n continuations of each sequence's beams; returns (scores fp32, tokens int32, parents int32), [B, n] each.

    logits fp16 or fp32 [B, W, V]; scores fp32 [B, W], the beams' log-probabilities so far (-inf: no beam).  A
    continuation by token v has scores[b, w] + logits[b, w, v] - log(sum(exp(logits[b, w]))); a beam with
    finished[b, w] (bool) has one, token `eos`, with the score it has.  Best first, formed and compared in fp64 (a row's
    log-sum is within 2^-33), ties to the lower beam, then the lower token; n defaults to W, and both are at most 64.  parents holds rows b * W + w, as
    paged_kv_fork and beam_reorder take them.  Continuations of score -inf in fp32 or NaN (logits of -inf; every one of a row
    that holds NaN or +inf) are none; where there are fewer than n the rest has score -inf, token and parent -1.  `out` may hold
    `scores` itself where n is W.
    Calls that may run at the same time on several streams need a workspace each.
    """
    who = "beam_select"
    dev = _gpu_of(who, logits, scores, finished, *(out if out is not None else ()))
    if logits.dtype not in (torch.float16, torch.float32) or logits.dim() != 3 or \
            (logits.stride(2) != 1 and logits.shape[2] > 1):
        raise RuntimeError(f"{who}: logits must be fp16 or fp32 [B, W, V] with unit inner stride")
    B, W, V = logits.shape
    if scores.dtype != torch.float32 or scores.shape != (B, W) or (scores.stride(1) != 1 and W > 1):
        raise RuntimeError(f"{who}: scores must be fp32 [{B}, {W}] with unit inner stride")
    if finished is not None and eos is None:
        raise RuntimeError(f"{who}: finished beams go on with eos, which is not given")
    if finished is not None and (finished.dtype != torch.bool or finished.shape != (B, W) or
                                 (finished.stride(1) != 1 and W > 1)):
        raise RuntimeError(f"{who}: finished must be bool [{B}, {W}] with unit inner stride")
    n = W if n is None else int(n)
    if n < 1 or W < 1 or V < 1:
        raise RuntimeError(f"{who}: {n} of {W} beams over {V} tokens")
    if out is None:
        out = (torch.empty((B, n), dtype=torch.float32, device=logits.device),
               *(torch.empty((B, n), dtype=torch.int32, device=logits.device) for _ in "tp"))
    elif len(out) != 3 or any(t.shape != (B, n) or not t.is_contiguous() for t in out) or \
            [t.dtype for t in out] != [torch.float32, torch.int32, torch.int32]:
        raise RuntimeError(f"{who}: out must be contiguous (fp32, int32, int32) of [{B}, {n}]")
    if B == 0:
        return tuple(out)
    fp32 = logits.dtype == torch.float32
    wptr, wbytes = _workspace(workspace, dev).ensure(_beam_workspace(B, W, V, fp32, dev))
    _call_on(dev, "specq_beam_select", logits.data_ptr(), fp32, logits.stride(0), logits.stride(1),
             scores.data_ptr(), scores.stride(0), _ptr(finished), finished.stride(0) if finished is not None else 0,
             int(eos) if finished is not None else 0, *(t.data_ptr() for t in out), B, W, V, n, wptr, wbytes)
    return tuple(out)


def beam_reorder(states, parents, group):
    """Make row r of every state its row parents[r], in place, within groups of `group` rows (a sequence's beams).

    states: tensors [rows, ...] of any type, each row contiguous (token histories, gathered weights, hidden states, a
    dense cache), no two of them over the same memory; parents int32 [rows] (beam_select's, flattened), group at most 32.  A parent
    outside the row's group (-1) leaves the row as it is.  A paged cache follows by paged_kv_fork.
    """
    who = "beam_reorder"
    dev = _gpu_of(who, parents, *states)
    rows, group = parents.shape[0] if parents.dim() == 1 else -1, int(group)
    _int32_vec(who, "parents", parents, 0)
    if group < 1 or rows % group:
        raise RuntimeError(f"{who}: {rows} rows are no groups of {group}")
    base, stride, nbytes = [], [], []
    for t in states:
        if t.dim() < 1 or t.shape[0] != rows:
            raise RuntimeError(f"{who}: a state {tuple(t.shape)} must have {rows} rows")
        if t.numel() == 0:
            continue
        if not t.is_contiguous() and not t[0].is_contiguous():
            raise RuntimeError(f"{who}: the rows of a state must be contiguous")
        size = t.element_size()
        base.append(t.data_ptr())
        stride.append(t.stride(0) * size)
        nbytes.append(t.numel() // rows * size)
    if not base:
        return
    words = array.array("q", base + stride + nbytes)
    _call_on(dev, "specq_beam_reorder", parents.data_ptr(), rows, group, *_page_tensor_args(len(base), words))
