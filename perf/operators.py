"""The steps around a paged 8-bit K/V cache with block scales, as cases that can be measured.

A case is a dict of plain values; `listed()` holds the fixed ones, `draw(rng)` gives more of the
same ranges.  Four operators, as a verification step runs them:

  rope    rotary positions of the new tokens' q and k (half or interleaved pairs, all or part of
          the head, frequencies stretched for long contexts)
  append  the new tokens' K/V quantised into cache pages that hold one scale for each block of
          tokens and head; a block whose scale grows has its earlier tokens requantised
  attn    attention of the new tokens over that cache
  pages   the cache's page tables: reserve and free (a step's traffic), fork (several samples of
          one prompt), compact (a batch's turnover)

Where `own` is false, run() computes them from elementary torch operations; where it is true,
with the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
F8 = torch.float8_e4m3fn
QMAX = {"int8": 127.0, "fp8": 448.0}
_framework = None


def _K():
    """The framework's kernels module (own calls only)."""
    global _framework
    if _framework is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "specdec-quant-triton_amd"))
        import kernels
        _framework = kernels
    return _framework


# ----------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------
def listed():
    return [
        # The smallest call: one token's q and k of one sequence, between the projection and the append.
        dict(name="rope_decode", op="rope", B=1, q_len=1, H=32, H_KV=8, D=128, R=128, pairs="half", scaling="none",
             far=8192),
        # Odd sizes: a head of 80 of which 20 dimensions rotate in interleaved pairs, far positions.
        dict(name="rope_partial_far", op="rope", B=3, q_len=17, H=12, H_KV=3, D=80, R=20, pairs="interleaved",
             scaling="yarn", far=1000003),
        # Two prompts of 4096 tokens, frequencies stretched by wavelength for long contexts.
        dict(name="rope_prefill", op="rope", B=2, q_len=4096, H=32, H_KV=8, D=128, R=128, pairs="half",
             scaling="wavelength", far=32768),
        # 8 drafts and a token for 8 sequences appended: most blocks hold earlier tokens.
        dict(name="append_verify_int8", op="append", B=8, q_len=9, ctx=300, H_KV=8, D=128, PAGE=16, SB=16, fmt="int8"),
        # Two prompts' tokens appended at once, blocks of half a page.
        dict(name="append_prefill_fp8", op="append", B=2, q_len=2048, ctx=2100, H_KV=8, D=128, PAGE=64, SB=32,
             fmt="fp8"),
        # Verification of 8 drafts for 8 sequences, context 4096.
        dict(name="attn_verify_fp8", op="attn", B=8, q_len=9, ctx=4096, ragged=False, H=32, H_KV=8, D=128, PAGE=16,
             SB=16, fmt="fp8"),
        # Plain decoding of a full batch whose sequences have all lengths up to 8192.
        dict(name="attn_decode_int8", op="attn", B=32, q_len=1, ctx=8192, ragged=True, H=32, H_KV=8, D=128, PAGE=64,
             SB=64, fmt="int8"),
        # One sequence with a very long context, 4 drafts, narrow heads in groups of 8.
        dict(name="attn_long_fp8", op="attn", B=1, q_len=5, ctx=131072, ragged=False, H=16, H_KV=2, D=64, PAGE=32,
             SB=16, fmt="fp8"),
        # Chunked prefill of two prompts: 256 new tokens each behind up to 3840 cached ones.
        dict(name="attn_chunk_int8", op="attn", B=2, q_len=256, ctx=4096, ragged=True, H=32, H_KV=8, D=128, PAGE=16,
             SB=16, fmt="int8"),
        # A verification step's page traffic: pages for 9 new tokens each, then those of the rejected ones freed.
        dict(name="pages_step", op="pages", kind="step", B=32, ctx=4096, q_len=9, H_KV=8, D=128, PAGE=16, SB=16),
        # Four samples of each of 8 prompts: full pages are shared, the last page is copied.
        dict(name="pages_fork", op="pages", kind="fork", B=32, group=4, ctx=2000, H_KV=8, D=128, PAGE=64, SB=64),
        # A batch's turnover, in two halves: sequences leave, the pool is compacted, new ones enter.
        dict(name="pages_turnover", op="pages", kind="turnover", B=16, ctx=4096, H_KV=8, D=128, PAGE=16, SB=16),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _blocks(rng):
    """Page and block sizes: whole 16s, the block a divisor of the page."""
    page = rng.choice((16, 16, 32, 48, 64, 128))
    return page, rng.choice([s for s in range(16, page + 1, 16) if page % s == 0])


def draw(rng):
    op = rng.choice(("rope", "append", "attn", "attn", "pages"))
    h_kv = rng.choice((1, 2, 4, 8))
    page, sb = _blocks(rng)
    if op == "rope":
        D = rng.choice((64, 80, 96, 128, 192, 256))
        R = D if rng.random() < 0.5 else 2 * rng.randrange(1, D // 2 + 1)
        B, H = _log(rng, 1, 32), h_kv * rng.choice((1, 2, 3, 4, 8))
        q_len = max(1, min(_log(rng, 1, 4096), (1 << 25) // (B * (H + h_kv) * D)))
        return dict(op=op, B=B, q_len=q_len, H=H, H_KV=h_kv, D=D, R=R, pairs=rng.choice(("half", "interleaved")),
                    scaling=rng.choice(("none", "linear", "yarn", "wavelength")), far=_log(rng, 4096, 2000000))
    if op == "append":
        D, B = rng.choice((64, 128, 128, 256)), _log(rng, 1, 32)
        q_len = max(1, min(_log(rng, 1, 2048), (1 << 22) // (B * h_kv * D)))
        return dict(op=op, B=B, q_len=q_len, ctx=q_len + _log(rng, 1, 300), H_KV=h_kv, D=D, PAGE=page, SB=sb,
                    fmt=rng.choice(("int8", "fp8")))
    if op == "attn":
        G, D, fmt = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128)), rng.choice(("int8", "fp8"))
        chunk = rng.random() < 0.25
        q_len = _log(rng, 16, 256) if chunk else rng.randrange(1, 10)
        B = rng.randrange(1, 3) if chunk else _log(rng, 1, 32)
        ctx = _log(rng, max(q_len, 64), 4096 if chunk else 131072 // max(B, 2))
        return dict(op=op, B=B, q_len=q_len, ctx=ctx, ragged=rng.random() < 0.7, H=h_kv * G, H_KV=h_kv, D=D, PAGE=page,
                    SB=sb, fmt=fmt)
    kind = rng.choice(("step", "fork", "turnover"))
    c = dict(op=op, kind=kind, ctx=_log(rng, 64, 4096), H_KV=h_kv, D=rng.choice((64, 128)), PAGE=page, SB=sb)
    if kind == "step":
        return dict(c, B=_log(rng, 1, 64), q_len=rng.randrange(1, 10))
    if kind == "fork":
        group = rng.randrange(2, 9)
        return dict(c, B=group * rng.randrange(1, 9), group=group)
    return dict(c, B=2 * rng.randrange(1, 9))


# ----------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 29)
        self.cpu = torch.Generator().manual_seed(1000003 * int(seed) + 31)

    def normal(self, *shape):
        return torch.randn(shape, device=DEV, generator=self.g)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, device=DEV, generator=self.g) * (hi - lo) + lo

    def lens(self, n, lo, hi):
        return torch.randint(lo, hi + 1, (n,), generator=self.cpu).tolist()

    def perm(self, n):
        return torch.randperm(n, device=DEV, generator=self.g).to(torch.int32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _frequencies(R, scaling):
    """(fp64 [R/2] frequencies in radians a token, the factor on cos and sin): base 10000, trained on 8192
    tokens, stretched 8-fold."""
    base, factor, trained = 10000.0, 8.0, 8192.0
    f = [base ** (-2.0 * j / R) for j in range(R // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "wavelength":  # long waves stretched, short ones kept, a blend between
        lo, hi = 1.0, 4.0
        mix = [min(1.0, max(0.0, (trained * x / (2 * math.pi) - lo) / (hi - lo))) for x in f]
        f = [x * m + x / factor * (1 - m) for x, m in zip(f, mix)]
    elif scaling == "yarn":  # a ramp over the pair's index between two numbers of turns
        at = lambda turns: R * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), R // 2 - 1)
        ramp = [min(1.0, max(0.0, (j - lo) / max(hi - lo, 1e-3))) for j in range(R // 2)]
        f = [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)]
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _codes(gen, fmt, shape):
    """Codes of normal values quantised against the largest of a block (some 3.3 deviations)."""
    x = gen.normal(*shape).mul_(QMAX[fmt] / 3.5).clamp_(-QMAX[fmt], QMAX[fmt])
    return x.round_().to(torch.int8) if fmt == "int8" else x.to(F8)


def _cache(gen, c, fmt, pages):
    nb = c["PAGE"] // c["SB"]
    kv = [_codes(gen, fmt, (pages, c["PAGE"], c["H_KV"], c["D"])) for _ in "kv"]
    return kv + [gen.uniform(0.8, 1.2, pages, nb, c["H_KV"]) * (3.5 / QMAX[fmt]) for _ in "kv"]


def _table(gen, rows, pool, cols):
    """A block table of `rows` page counts over a shuffled pool; -1 where a row holds no page."""
    ids = gen.perm(pool)
    tbl = torch.full((len(rows), cols), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(rows):
        tbl[b, :n] = ids[at:at + n]
        at += n
    return tbl


def _refs(tbl, pool):
    return torch.bincount(tbl[tbl >= 0].long(), minlength=pool).to(torch.int32)


def prepare(case, seed):
    c, gen, op = case, _Gen(seed), case["op"]
    up = lambda n: -(-n // c["PAGE"])  # noqa: E731
    s = {"c": c}
    if op == "rope":
        f, s["mscale"] = _frequencies(c["R"], c["scaling"])
        s["inv_freq"] = torch.tensor(f, dtype=torch.float64, device=DEV)
        s["q"] = gen.normal(c["B"], c["q_len"], c["H"], c["D"]).half()
        s["k"] = gen.normal(c["B"], c["q_len"], c["H_KV"], c["D"]).half()
        s["ctx"] = _i32(gen.lens(c["B"], min(c["q_len"], c["far"]), max(c["far"], c["q_len"])))
    elif op == "append":
        lens = gen.lens(c["B"], c["q_len"], c["ctx"])
        pool = c["B"] * up(c["ctx"]) + 2
        s["kv"] = _cache(gen, c, c["fmt"], pool)
        s["tbl"], s["ctx"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"])), _i32(lens)
        s["new"] = [gen.normal(c["B"], c["q_len"], c["H_KV"], c["D"]).half() for _ in "kv"]
        if c["fmt"] == "int8":
            s["values"] = [torch.empty(x.shape, dtype=torch.float16, device=DEV) for x in s["kv"][:2]]
    elif op == "attn":
        lens = gen.lens(c["B"], max(c["q_len"], c["ctx"] // 8), c["ctx"]) if c["ragged"] else [c["ctx"]] * c["B"]
        lens[0] = c["ctx"]
        pool = sum(up(n) for n in lens) + 2
        s["kv"] = _cache(gen, c, c["fmt"], pool)
        s["tbl"], s["ctx"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"])), _i32(lens)
        s["q"] = gen.normal(c["B"], c["q_len"], c["H"], c["D"]).half()
    elif c["kind"] == "step":
        lens = gen.lens(c["B"], max(1, c["ctx"] // 8), c["ctx"])
        pool = c["B"] * (up(c["ctx"] + c["q_len"]) + 1)
        s["tbl"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"] + c["q_len"]))
        s["ref"], s["want"] = _refs(s["tbl"], pool), _i32([n + c["q_len"] for n in lens])
        taken = gen.lens(c["B"], 1, c["q_len"])
        s["keep"] = _i32([n + t for n, t in zip(lens, taken)])
    elif c["kind"] == "fork":
        lead = gen.lens(c["B"] // c["group"], max(1, c["ctx"] // 8), c["ctx"])
        lens = [n if i == 0 else 0 for n in lead for i in range(c["group"])]
        pool = len(lead) * up(c["ctx"]) + 2 * c["B"]
        s["kv"] = _cache(gen, c, "fp8", pool)
        s["tbl"], s["lens"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"])), _i32(lens)
        s["ref"] = _refs(s["tbl"], pool)
        s["parent"] = _i32([b // c["group"] * c["group"] for b in range(c["B"])])
    else:
        lens = gen.lens(c["B"], max(1, c["ctx"] // 8), c["ctx"])
        pool = c["B"] * up(c["ctx"]) + 8
        s["kv"] = _cache(gen, c, "fp8", pool)
        s["tbl"], s["want"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"])), _i32(lens)
        s["ref"] = _refs(s["tbl"], pool)
        s["leave"] = [_i32([0 if b % 2 == k else n for b, n in enumerate(lens)]) for k in (0, 1)]
    return s


# ----------------------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------------------
def _rope(x, cos, sin, pairs):
    R = 2 * cos.shape[-1]
    y = x.float()
    rot = y[..., :R]
    a, b = (rot[..., :R // 2], rot[..., R // 2:]) if pairs == "half" else (rot[..., 0::2], rot[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    rot = torch.cat((u, v), -1) if pairs == "half" else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((rot, y[..., R:]), -1).half()


def _plain_rope(s):
    c = s["c"]
    pos = s["ctx"][:, None].double() - c["q_len"] + torch.arange(c["q_len"], device=DEV)
    ang = pos[..., None] * s["inv_freq"]
    cos, sin = (f(ang)[:, :, None].mul(s["mscale"]).float() for f in (torch.cos, torch.sin))
    return _rope(s["q"], cos, sin, c["pairs"]), _rope(s["k"], cos, sin, c["pairs"])


def _to_codes(x, fmt):
    m = QMAX[fmt]
    return x.round().clamp(-m, m).to(torch.int8) if fmt == "int8" else x.clamp(-m, m).float().to(F8)


def _plain_append(s):
    """Whole blocks at a time: each block that new tokens reach is read, requantised and written back."""
    c, ql, SB, PAGE = s["c"], s["c"]["q_len"], s["c"]["SB"], s["c"]["PAGE"]
    pos0 = s["ctx"].long() - ql
    first, last = pos0 // SB, (pos0 + ql - 1) // SB
    j = torch.arange((ql + SB - 1) // SB + 1, device=DEV)
    blk = torch.minimum(first[:, None] + j, last[:, None])  # a block past the last repeats it
    page = s["tbl"].long().gather(1, blk * SB // PAGE)
    sub = blk % (PAGE // SB)
    at = blk[..., None] * SB + torch.arange(SB, device=DEV)  # positions [B, blocks, SB]
    tok = at - pos0[:, None, None]
    new, old = ((tok >= 0) & (tok < ql))[..., None, None], (tok < 0)[..., None, None]
    row = torch.arange(c["B"], device=DEV)[:, None, None]
    for x, codes, scale in ((s["new"][0], s["kv"][0], s["kv"][2]), (s["new"][1], s["kv"][1], s["kv"][3])):
        view = codes.view(torch.uint8).view(codes.shape[0], -1, SB, *codes.shape[2:])
        was = view[page, sub]
        q0, s0 = was.view(codes.dtype).float(), scale[page, sub]  # [B, blocks, SB, H, D], [B, blocks, H]
        xn = x[row, tok.clamp(0, ql - 1)].float()
        amax = torch.where(new, xn, 0.0).abs().amax((2, 4))
        sn = (amax.clamp(min=1e-8).double() / QMAX[c["fmt"]]).float()
        sn = torch.where(old.any((2, 4)), torch.maximum(sn, s0), sn)
        div = sn.double()[:, :, None, :, None]
        got = torch.where(new, xn.double(), (q0 * s0[:, :, None, :, None]).double()) / div
        got = _to_codes(got.float(), c["fmt"]).view(torch.uint8)
        grew = (sn > s0)[:, :, None, :, None]
        view[page, sub] = torch.where(new | (old & grew), got, was)
        scale[page, sub] = sn


def _plain_attn(s):
    c, q = s["c"], s["q"]
    B, ql, H, D = q.shape
    hk, nb = c["H_KV"], c["PAGE"] // c["SB"]
    tbl = s["tbl"].long().clamp(min=0)

    def dense(codes, scale):  # [B, H_KV, T, D]
        x = codes.view(torch.uint8)[tbl].view(codes.dtype).float().view(B, -1, nb, c["SB"], hk, D)
        return (x * scale[tbl][:, :, :, None, :, None]).view(B, -1, hk, D).transpose(1, 2).contiguous()

    k, v = dense(s["kv"][0], s["kv"][2]), dense(s["kv"][1], s["kv"][3])
    T = k.shape[2]
    qg = q.float().view(B, ql, hk, H // hk, D).permute(0, 2, 1, 3, 4).reshape(B, hk, -1, D)
    sc = torch.matmul(qg, k.transpose(2, 3).contiguous()).view(B, hk, ql, H // hk, T) * (1.0 / math.sqrt(D))
    end = s["ctx"].long()[:, None] - ql + torch.arange(ql, device=DEV)
    hidden = (torch.arange(T, device=DEV) > end[..., None])[:, None, :, None]  # [B, 1, ql, 1, T]
    sc = sc.masked_fill(hidden, float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p.view(B, hk, -1, T), v).view(B, hk, ql, H // hk, D) / p.sum(-1)[..., None]
    return o.permute(0, 2, 1, 3, 4).reshape(B, ql, H, D).half()


def _held(lens, page):
    """Whether a row of `lens` tokens holds column c."""
    return lambda cols: cols < ((lens.long().clamp(min=0) + page - 1) // page)[:, None]


def _count(ref, ids, mask, by):
    ref.scatter_add_(0, ids.clamp(min=0).long().flatten(), (mask.int() * by).flatten())


def _take(tbl, ref, need):
    """Gives the entries that need one the lowest free pages, in the table's order; how many are short."""
    free = (ref <= 0)
    order = torch.argsort((~free).to(torch.uint8), stable=True).to(torch.int32)
    n = free.sum()
    rank = need.flatten().cumsum(0).view(need.shape) - 1
    got = torch.where(rank < n, order[rank.clamp(0, ref.numel() - 1)], -1)
    tbl.copy_(torch.where(need, got, tbl))
    _count(ref, got, need & (got >= 0), 1)
    return (need.sum() - n).clamp(min=0).to(torch.int32).view(1)


def _plain_reserve(tbl, ref, lens, page):
    cols = torch.arange(tbl.shape[1], device=DEV)
    return _take(tbl, ref, _held(lens, page)(cols) & ((tbl < 0) | (tbl >= ref.numel())))


def _plain_free(tbl, ref, keep, page):
    gone = ~_held(keep, page)(torch.arange(tbl.shape[1], device=DEV))
    _count(ref, tbl, gone & (tbl >= 0), -1)
    tbl.masked_fill_(gone, -1)


def _plain_fork(tbl, ref, lens, parent, caches, page):
    B, C = tbl.shape
    row, cols = torch.arange(B, device=DEV), torch.arange(C, device=DEV)
    p = parent.long()
    n = lens[p]
    src = tbl[p]
    full = cols < (n // page).long()[:, None]
    part = (cols == (n // page).long()[:, None]) & (n % page > 0)[:, None]
    keeps = torch.full((B,), B, device=DEV).scatter_reduce(0, p, row, "amin")[p] == row
    new = torch.where((full | (part & keeps[:, None])) & (src >= 0), src, -1)
    _count(ref, tbl, tbl >= 0, -1)
    _count(ref, new, new >= 0, 1)
    need = part & ~keeps[:, None] & (src >= 0)
    tbl.copy_(new)
    short = _take(tbl, ref, need)
    done = need & (tbl >= 0)
    at, to = src[done].long(), tbl[done].long()
    for t in caches:
        b = t.view(torch.uint8).view(t.shape[0], -1)
        b[to] = b[at]
    lens.copy_(n)
    return short


def _plain_compact(tbl, ref, caches):
    used = ref > 0
    n, ids = used.sum(), torch.arange(ref.numel(), device=DEV)
    moves = used & (ids >= n)
    holes = torch.argsort(used.to(torch.uint8), stable=True)
    to = torch.where(moves, holes[(moves.cumsum(0) - 1).clamp(min=0)], ids)
    at = moves.nonzero().flatten()
    for t in caches:
        b = t.view(torch.uint8).view(t.shape[0], -1)
        b[to[at]] = b[at]
    ref[to[at]] = ref[at]
    ref[at] = 0
    tbl.copy_(torch.where(tbl >= 0, to[tbl.clamp(min=0).long()].to(torch.int32), tbl))
    return to.to(torch.int32)


# ----------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------
def _values(s):
    """What the 8-bit cache stands for: e4m3 codes are numbers, int8 codes are multiplied by their scales."""
    c, (kc, vc, ks, vs) = s["c"], s["kv"]
    if c["fmt"] == "int8":
        shape = (kc.shape[0], -1, c["SB"], *kc.shape[2:])
        for x, scale, out in ((kc, ks, s["values"][0]), (vc, vs, s["values"][1])):
            torch.mul(x.view(shape), scale[:, :, None, :, None], out=out.view(shape))
        kc, vc = s["values"]
    return {"k": kc, "v": vc, "ks": ks, "vs": vs}


def _run_rope(s):
    c = s["c"]
    if own:
        return _K().rotary_embed(s["q"], s["k"], s["inv_freq"], s["ctx"], c["q_len"],
                                 interleaved=c["pairs"] == "interleaved", mscale=s["mscale"])
    return _plain_rope(s)


def _run_append(s):
    if own:
        _K().paged_kv_append_block_scaled(*s["new"], *s["kv"], s["tbl"], s["ctx"], s["c"]["q_len"])
    else:
        _plain_append(s)
    return _values(s)


def _run_attn(s):
    if own:
        return _K().paged_attention_block_scaled(s["q"], *s["kv"], s["tbl"], s["ctx"], s["c"]["q_len"])[0]
    return _plain_attn(s)


def _reserve(s):
    f = _K().paged_kv_reserve if own else _plain_reserve
    return f(s["tbl"], s["ref"], s["want"], s["c"]["PAGE"])


def _free(s, keep):
    f = _K().paged_kv_free if own else _plain_free
    f(s["tbl"], s["ref"], keep, s["c"]["PAGE"])


def _run_pages(s):
    c = s["c"]
    if c["kind"] == "step":
        short = _reserve(s)
        _free(s, s["keep"])
        return {"tbl": s["tbl"], "ref": s["ref"], "short": short}
    if c["kind"] == "fork":
        f = _K().paged_kv_fork if own else _plain_fork
        short = f(s["tbl"], s["ref"], s["lens"], s["parent"], s["kv"], c["PAGE"])
        return {"tbl": s["tbl"], "ref": s["ref"], "lens": s["lens"], "short": short, "kv": s["kv"]}
    moved = []
    for leave in s["leave"]:
        _free(s, leave)
        moved.append((_K().paged_kv_compact if own else _plain_compact)(s["tbl"], s["ref"], s["kv"]))
        moved.append(_reserve(s))
    return {"tbl": s["tbl"], "ref": s["ref"], "moved": moved, "kv": s["kv"]}


def run(state):
    return {"rope": _run_rope, "append": _run_append, "attn": _run_attn, "pages": _run_pages}[state["c"]["op"]](state)


# ----------------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    up = lambda n: -(-n // c["PAGE"])  # noqa: E731
    if op == "rope":
        tok, heads = c["B"] * c["q_len"], c["H"] + c["H_KV"]
        return {"bytes": tok * heads * c["D"] * 4 + 4 * c["R"], "flops": 3 * tok * heads * c["R"]}
    if op == "append":
        # The new tokens read, their codes and their blocks' scales written; what the pass hands back as
        # values (int8) is read and written too.
        n, width = c["B"] * c["q_len"], c["H_KV"] * c["D"]
        pool = c["B"] * up(c["ctx"]) + 2
        back = 6 * pool * c["PAGE"] * width if c["fmt"] == "int8" else 0
        return {"bytes": n * width * 6 + 8 * c["H_KV"] * (n // c["SB"] + c["B"]) + back, "flops": 6 * n * width}
    if op == "attn":
        lens = _Gen(0).lens(c["B"], max(c["q_len"], c["ctx"] // 8), c["ctx"]) if c["ragged"] else [c["ctx"]] * c["B"]
        lens[0] = c["ctx"]
        ql, kv = c["q_len"], c["H_KV"] * 2 * c["D"]
        b = sum(n * kv + up(n) * (4 + 8 * c["H_KV"] * (c["PAGE"] // c["SB"])) for n in lens)
        f = sum(4 * c["H"] * c["D"] * (ql * (n - ql) + ql * (ql + 1) // 2) for n in lens)
        return {"bytes": b + 4 * c["B"] * ql * c["H"] * c["D"], "flops": f}
    page = 2 * c["H_KV"] * (c["PAGE"] * c["D"] + 4 * (c["PAGE"] // c["SB"]))  # bytes of a page, K and V and scales
    if c["kind"] == "step":  # the tables and counts are read, and what changes in them written
        lens = _Gen(0).lens(c["B"], max(1, c["ctx"] // 8), c["ctx"])
        return {"bytes": 8 * sum(up(n) for n in lens) + 12 * c["B"], "flops": 0}
    if c["kind"] == "fork":  # a last page copied for each sample but the first, rows of the table written
        lead = _Gen(0).lens(c["B"] // c["group"], max(1, c["ctx"] // 8), c["ctx"])
        rows = sum(up(n) for n in lead)
        return {"bytes": 4 * rows * (1 + c["group"]) + 8 * rows + 2 * page * (c["B"] - len(lead)), "flops": 0}
    lens = _Gen(0).lens(c["B"], max(1, c["ctx"] // 8), c["ctx"])
    half = [sum(up(n) for n in lens[k::2]) for k in (0, 1)]
    # Once the halves take turns, each compaction moves as many pages as the smaller half has.
    return {"bytes": 4 * page * min(half) + 2 * 8 * sum(half), "flops": 0}


# ----------------------------------------------------------------------------------------
# The same in 64 bits, sequence by sequence
# ----------------------------------------------------------------------------------------
def _exact_rope(s):
    c, out = s["c"], []
    w = torch.arange(c["q_len"], dtype=torch.float64, device=DEV)
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        for b, n in enumerate(s["ctx"].tolist()):
            for j in range(c["R"] // 2):
                i0, i1 = (j, j + c["R"] // 2) if c["pairs"] == "half" else (2 * j, 2 * j + 1)
                z = torch.polar(torch.full_like(w, s["mscale"]), (w + (n - c["q_len"])) * s["inv_freq"][j])[:, None]
                r = torch.complex(x[b, :, :, i0].double(), x[b, :, :, i1].double()) * z
                y[b, :, :, i0], y[b, :, :, i1] = r.real, r.imag
        out.append(y)
    return tuple(out)


def _exact_append(s):
    c, got = s["c"], []
    SB, PAGE, ql, m = c["SB"], c["PAGE"], c["q_len"], QMAX[c["fmt"]]
    for x, codes, scale in zip(s["new"], s["kv"][:2], s["kv"][2:]):
        val, sc = codes.double(), scale.double()
        for b, n in enumerate(s["ctx"].tolist()):
            at = n - ql
            while at < n:
                lo, hi = at // SB * SB, min(at // SB * SB + SB, n)
                pg, off, blk = int(s["tbl"][b, lo // PAGE]), lo % PAGE, lo % PAGE // SB
                new = x[b, at - n + ql:hi - n + ql].double()  # [tokens, H, D]
                was = sc[pg, blk].clone()
                now = (new.abs().amax((0, 2)).clamp(min=1e-8) / m).float().double()
                if at > lo:
                    now = torch.maximum(now, was)
                    old = val[pg, off:off + at - lo] * was[:, None] / now[:, None]
                    val[pg, off:off + at - lo] = _exact_codes(old, c["fmt"])
                val[pg, off + at - lo:off + hi - lo] = _exact_codes(new / now[:, None], c["fmt"])
                sc[pg, blk] = now
                at = hi
        got.append((val, sc))
    (k, ks), (v, vs) = got
    if c["fmt"] == "int8":
        k, v = (a * z.repeat_interleave(SB, 1)[..., None] for a, z in got)
    return {"k": k, "v": v, "ks": ks, "vs": vs}


def _exact_codes(x, fmt):
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    # e4m3: 3 bits behind the leading one, down to steps of 2^-9.
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_attn(s):
    c, q = s["c"], s["q"].double()
    B, ql, H, D = q.shape
    G, SB = H // c["H_KV"], c["SB"]
    out = torch.zeros_like(q)
    for b, n in enumerate(s["ctx"].tolist()):
        t = torch.arange(n, device=DEV)
        pg, sl = s["tbl"][b, t // c["PAGE"]].long(), t % c["PAGE"]
        seen = t[None] <= (n - ql + torch.arange(ql, device=DEV))[:, None]
        for h in range(c["H_KV"]):
            kc, vc = (x.view(torch.uint8)[pg, sl, h].view(x.dtype).double() for x in s["kv"][:2])
            k, v = (x * z[pg, sl // SB, h].double()[:, None] for x, z in ((kc, s["kv"][2]), (vc, s["kv"][3])))
            qq = q[b, :, h * G:(h + 1) * G].reshape(-1, D)
            w = (qq @ k.t() / math.sqrt(D)).view(ql, G, n).masked_fill(~seen[:, None], -math.inf).softmax(-1)
            out[b, :, h * G:(h + 1) * G] = (w.view(-1, n) @ v).view(ql, G, D)
    return out


def exact(case, seed):
    if case["op"] == "pages":  # whole numbers and copies
        return None
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn}[case["op"]](s)
