"""What a serving loop does to its batch around the paged cache, as cases that can be measured.

A case is a dict of plain values; `listed()` holds the fixed ones, `draw(rng)` gives more of the
same ranges.  Five operators:

  norm     every head of the new tokens' q and k normalised (root mean square, weights) and turned by its
           rotary position in the same pass
  weights  the attention weight that the new tokens' queries give each cached token, added to what it has
           gathered so far
  evict    of each sequence past its budget, the tokens of least gathered weight dropped for each K/V head, the
           others moved together in the cache pages
  beam     beam search's selection over beams and vocabulary from the model's logits
  reorder  the rows of a beam batch's states (token histories, gathered weights, a draft model's dense K/V) put
           in the order of the selected beams

Where `own` is false, run() computes them from elementary torch operations; where it is true,
with the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
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
        dict(name="norm_decode", op="norm", B=1, q_len=1, H=32, H_KV=8, D=128, R=128, pairs="half", far=8192),
        # Odd sizes: a head of 80 of which 20 dimensions turn in interleaved pairs, 17 tokens of 3 sequences.
        dict(name="norm_partial", op="norm", B=3, q_len=17, H=12, H_KV=3, D=80, R=20, pairs="interleaved", far=1000003),
        # Two prompts of 4096 tokens.
        dict(name="norm_prefill", op="norm", B=2, q_len=4096, H=32, H_KV=8, D=128, R=128, pairs="half", far=32768),
        # Plain decoding of a full batch whose sequences have all lengths up to 8192.
        dict(name="weights_decode", op="weights", B=32, q_len=1, ctx=8192, ragged=True, H=32, H_KV=8, D=128, PAGE=64,
             scales="fp32"),
        # Verification of 8 drafts for 8 sequences, context 4096.
        dict(name="weights_verify", op="weights", B=8, q_len=9, ctx=4096, ragged=False, H=32, H_KV=8, D=128, PAGE=16,
             scales="fp16"),
        # Chunked prefill of two prompts: 256 new tokens each behind up to 3840 cached ones.
        dict(name="weights_chunk", op="weights", B=2, q_len=256, ctx=4096, ragged=True, H=32, H_KV=8, D=128, PAGE=16,
             scales="fp16"),
        # A batch whose longer sequences are cut back to 2048 tokens, 256 of them the last ones.
        dict(name="evict_batch", op="evict", B=8, ctx=4096, H_KV=8, D=128, PAGE=16, budget=2048, recent=256, sinks=4,
             scales="fp16"),
        # One sequence with a very long prompt, narrow heads, an odd budget.
        dict(name="evict_long", op="evict", B=1, ctx=65536, H_KV=2, D=64, PAGE=32, budget=8191, recent=1000, sinks=4,
             scales="fp32"),
        # One prompt's four beams, a vocabulary of 32000.
        dict(name="beam_one", op="beam", B=1, W=4, n=4, V=32000, dtype="fp16", done=False),
        # A batch of 16 with 8 beams each, twice as many candidates as beams, some beams finished, an odd vocabulary.
        dict(name="beam_batch", op="beam", B=16, W=8, n=16, V=128257, dtype="fp32", done=True),
        # Four beams' histories, last hidden rows and gathered weights.
        dict(name="reorder_one", op="reorder", B=1, W=4, T=500, hidden=4096, H_KV=8, draft=0),
        # 16 x 8 beams, with a draft model's dense K/V (two heads of 64 for 512 tokens) beside them.
        dict(name="reorder_batch", op="reorder", B=16, W=8, T=4096, hidden=4096, H_KV=8, draft=512),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("norm", "weights", "evict", "beam", "reorder"))
    h_kv, page = rng.choice((1, 2, 4, 8)), rng.choice((16, 16, 32, 48, 64, 128))
    scales = rng.choice(("fp16", "fp32"))
    if op == "norm":
        D = rng.choice((64, 80, 96, 128, 192, 256))
        R = D if rng.random() < 0.5 else 2 * rng.randrange(1, D // 2 + 1)
        B, H = _log(rng, 1, 32), h_kv * rng.choice((1, 2, 3, 4, 8))
        q_len = max(1, min(_log(rng, 1, 4096), (1 << 25) // (B * (H + h_kv) * D)))
        return dict(op=op, B=B, q_len=q_len, H=H, H_KV=h_kv, D=D, R=R, pairs=rng.choice(("half", "interleaved")),
                    far=_log(rng, 4096, 2000000))
    if op == "weights":
        G, D = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128))
        chunk = rng.random() < 0.25
        q_len = _log(rng, 16, 256) if chunk else rng.randrange(1, 10)
        B = rng.randrange(1, 3) if chunk else _log(rng, 1, 32)
        ctx = _log(rng, max(q_len, 64), 4096 if chunk else 131072 // max(B, 2))
        return dict(op=op, B=B, q_len=q_len, ctx=ctx, ragged=rng.random() < 0.7, H=h_kv * G, H_KV=h_kv, D=D, PAGE=page,
                    scales=scales)
    if op == "evict":
        B, D = _log(rng, 1, 16), rng.choice((64, 128))
        ctx = _log(rng, 64, min(65536, (1 << 25) // (B * h_kv * D)))
        budget = max(2, int(ctx * rng.uniform(0.05, 0.95)))
        recent = int(budget * rng.uniform(0.0, 0.6))
        return dict(op=op, B=B, ctx=ctx, H_KV=h_kv, D=D, PAGE=page, budget=budget, recent=recent,
                    sinks=rng.randrange(0, min(5, budget - recent)), scales=scales)
    if op == "beam":
        B, W = _log(rng, 1, 16), rng.randrange(1, 17)
        V = _log(rng, 1000, min(131072, (1 << 24) // (B * W)))
        return dict(op=op, B=B, W=W, n=W * rng.choice((1, 2)), V=V, dtype=rng.choice(("fp16", "fp32")),
                    done=rng.random() < 0.5)
    B, W = _log(rng, 1, 16), rng.randrange(2, 17)
    return dict(op=op, B=B, W=W, T=_log(rng, 16, (1 << 19) // (B * W)), hidden=8 * rng.randrange(16, 513), H_KV=h_kv,
                draft=rng.choice((0, _log(rng, 1, (1 << 16) // (B * W)))))


# ----------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 37)
        self.cpu = torch.Generator().manual_seed(1000003 * int(seed) + 41)

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


def _table(gen, rows, pool, cols):
    """A block table of `rows` page counts over a shuffled pool; -1 where a row holds no page."""
    ids = gen.perm(pool)
    tbl = torch.full((len(rows), cols), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(rows):
        tbl[b, :n] = ids[at:at + n]
        at += n
    return tbl


def _codes(gen, *shape):
    """int8 codes of normal values quantised against the largest of a row (some 2.8 deviations)."""
    return gen.normal(*shape).mul_(127 / 2.8).clamp_(-127, 127).round_().to(torch.int8)


def _scales(gen, c, *shape):
    s = gen.uniform(0.8, 1.2, *shape) * (2.8 / 127)
    return s.half() if c["scales"] == "fp16" else s


def _ragged(gen, c, lo):
    lens = gen.lens(c["B"], max(lo, c["ctx"] // 8), c["ctx"]) if c.get("ragged", True) else [c["ctx"]] * c["B"]
    lens[0] = c["ctx"]
    return lens


def _parents(gen, c):
    """Which beam each of a group's rows goes on from: some survive several times, some not at all."""
    out = []
    for b in range(c["B"]):
        out += [b * c["W"] + p for p in sorted(gen.lens(c["W"], 0, c["W"] - 1))]
    return out


def prepare(case, seed):
    c, gen, op = case, _Gen(seed), case["op"]
    up = lambda n: -(-n // c["PAGE"])  # noqa: E731
    s = {"c": c}
    if op == "norm":
        s["inv_freq"] = torch.tensor([10000.0 ** (-2.0 * j / c["R"]) for j in range(c["R"] // 2)], dtype=torch.float64,
                                     device=DEV)
        s["q"] = gen.normal(c["B"], c["q_len"], c["H"], c["D"]).mul_(3.0).half()
        s["k"] = gen.normal(c["B"], c["q_len"], c["H_KV"], c["D"]).mul_(2.0).half()
        s["wq"], s["wk"] = (gen.uniform(0.5, 1.5, c["D"]).half() for _ in "qk")
        s["ctx"] = _i32(gen.lens(c["B"], min(c["q_len"], c["far"]), max(c["far"], c["q_len"])))
    elif op == "weights":
        lens = _ragged(gen, c, c["q_len"])
        pool = sum(up(n) for n in lens) + 2
        s["kc"], s["ks"] = _codes(gen, pool, c["PAGE"], c["H_KV"], c["D"]), _scales(gen, c, pool, c["PAGE"], c["H_KV"])
        s["tbl"], s["ctx"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"])), _i32(lens)
        s["q"] = gen.normal(c["B"], c["q_len"], c["H"], c["D"]).half()
        s["w"] = gen.uniform(0.0, 2.0, c["B"], c["H_KV"], up(c["ctx"]) * c["PAGE"])
    elif op == "evict":
        lens = _ragged(gen, c, 1)
        pool = c["B"] * up(c["ctx"]) + 2
        s["kv"] = [_codes(gen, pool, c["PAGE"], c["H_KV"], c["D"]) for _ in "kv"]
        s["kv"] += [_scales(gen, c, pool, c["PAGE"], c["H_KV"]) for _ in "kv"]
        s["tbl"], s["ctx0"] = _table(gen, [up(n) for n in lens], pool, up(c["ctx"])), _i32(lens)
        # Gathered weights: most tokens get little, a few much.
        s["w0"] = gen.normal(c["B"], c["H_KV"], up(c["ctx"]) * c["PAGE"]).mul_(2.0).exp_()
        s["ctx"], s["w"] = s["ctx0"].clone(), s["w0"].clone()
        s["values"] = [torch.empty(x.shape, dtype=torch.float32, device=DEV) for x in s["kv"][:2]]
    elif op == "beam":
        dt = torch.float16 if c["dtype"] == "fp16" else torch.float32
        # Some rows sure of themselves, some not; a few tokens banned.
        x = gen.normal(c["B"], c["W"], c["V"]).mul_(gen.uniform(1.0, 4.0, c["B"], c["W"], 1))
        x.masked_fill_(gen.uniform(0.0, 1.0, 1, 1, c["V"]) < 0.01, -math.inf)
        s["logits"] = x.to(dt)
        s["scores"] = -gen.uniform(0.0, 20.0, c["B"], c["W"])
        s["eos"] = c["V"] // 2
        s["done"] = gen.uniform(0.0, 1.0, c["B"], c["W"]) < 0.25 if c["done"] else None
    else:
        rows = c["B"] * c["W"]
        s["states"] = [torch.randint(0, 1 << 15, (rows, c["T"]), device=DEV, generator=gen.g, dtype=torch.int32),
                       gen.normal(rows, c["hidden"]).half(), gen.uniform(0.0, 2.0, rows, c["H_KV"], c["T"])]
        if c["draft"]:
            s["states"].append(gen.normal(rows, 2, 2, c["draft"], 64).half())
        s["parents"] = _i32(_parents(gen, c))
    return s


# ----------------------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------------------
def _norm_turn(x, w, cos, sin, pairs):
    R = 2 * cos.shape[-1]
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    rot = y[..., :R]
    a, b = (rot[..., :R // 2], rot[..., R // 2:]) if pairs == "half" else (rot[..., 0::2], rot[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    rot = torch.cat((u, v), -1) if pairs == "half" else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((rot, y[..., R:]), -1).half()


def _plain_norm(s):
    c = s["c"]
    pos = s["ctx"][:, None].double() - c["q_len"] + torch.arange(c["q_len"], device=DEV)
    ang = pos[..., None] * s["inv_freq"]
    cos, sin = (f(ang)[:, :, None].float() for f in (torch.cos, torch.sin))
    return _norm_turn(s["q"], s["wq"], cos, sin, c["pairs"]), _norm_turn(s["k"], s["wk"], cos, sin, c["pairs"])


def _plain_weights(s):
    c, q = s["c"], s["q"]
    B, ql, H, D = q.shape
    hk = c["H_KV"]
    tbl = s["tbl"].long().clamp(min=0)
    k = (s["kc"][tbl].float() * s["ks"][tbl].float()[..., None]).view(B, -1, hk, D).transpose(1, 2).contiguous()
    T = k.shape[2]
    qg = q.float().view(B, ql, hk, H // hk, D).permute(0, 2, 1, 3, 4).reshape(B, hk, -1, D)
    sc = torch.matmul(qg, k.transpose(2, 3).contiguous()).view(B, hk, ql, H // hk, T) * (1.0 / math.sqrt(D))
    end = s["ctx"].long()[:, None] - ql + torch.arange(ql, device=DEV)
    t = torch.arange(T, device=DEV)
    hidden = (t > end[..., None])[:, None, :, None]  # [B, 1, ql, 1, T]
    sc = sc.masked_fill(hidden, float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    got = (p / p.sum(-1, keepdim=True)).sum((2, 3))  # [B, hk, T]
    at, n = t[None, None], s["ctx"].long()[:, None, None]
    # A new token starts from nothing; what lies behind a sequence stays.
    s["w"].copy_(torch.where(at >= n, s["w"], torch.where(at >= n - ql, got, s["w"] + got)))
    return s["w"]


def _plain_evict(tbl, ctx, w, caches, page, budget, recent, sinks):
    B, H, T = w.shape
    n, t, j = ctx.long()[:, None, None], torch.arange(T, device=DEV), torch.arange(budget, device=DEV)
    key = w.masked_fill((t < sinks) | (t >= n - recent), math.inf).masked_fill(t >= n, -math.inf)
    best = torch.argsort(key, dim=-1, descending=True, stable=True)[..., :budget].sort(-1).values
    over = n > budget
    kept = torch.where(over, best, torch.where(j < n, j, -1).expand(B, H, budget))
    b, h, to = (over & (kept != j)).nonzero(as_tuple=True)
    src = kept[b, h, to]
    from_page, to_page = tbl[b, src // page].long(), tbl[b, to // page].long()
    for x in caches:
        x[to_page, to % page, h] = x[from_page, src % page, h]
    w[b, h, to] = w[b, h, src]
    ctx.copy_(torch.where(ctx > budget, budget, ctx))
    return kept.to(torch.int32)


def _plain_beam(logits, scores, n, done, eos):
    B, W, V = logits.shape
    x = logits.double()  # candidates next to the border differ by little
    m = x.amax(-1, keepdim=True)
    x = x - (m + (x - m).exp().sum(-1, keepdim=True).log()) + scores.double()[..., None]
    if done is not None:
        only = torch.arange(V, device=DEV) == eos
        x = torch.where(done[..., None], torch.where(only, scores.double()[..., None], -math.inf), x)
    x = x.view(B, -1)
    row = torch.arange(B, device=DEV)
    best, at = [], []
    for _ in range(n):  # the first of the largest, and the next without it
        i = x.argmax(-1)
        best.append(x[row, i])
        at.append(i)
        x[row, i] = -math.inf
    best, at = torch.stack(best, 1), torch.stack(at, 1)
    none = best == -math.inf
    token = (at % V).masked_fill(none, -1).to(torch.int32)
    parent = (at // V + row[:, None] * W).masked_fill(none, -1).to(torch.int32)
    return best.float(), token, parent


def _plain_reorder(states, parents):
    p = parents.long()
    p = torch.where(p < 0, torch.arange(p.numel(), device=DEV), p)
    for x in states:
        x.copy_(x[p])


# ----------------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------------
def _run_norm(s):
    c = s["c"]
    if own:
        return _K().qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["inv_freq"], s["ctx"],
                                   interleaved=c["pairs"] == "interleaved", eps=1e-6)
    return _plain_norm(s)


def _run_weights(s):
    if own:
        return _K().paged_attention_weights(s["q"], s["kc"], s["ks"], s["tbl"], s["ctx"], s["w"])
    return _plain_weights(s)


def _run_evict(s):
    c, (kc, vc, ks, vs) = s["c"], s["kv"]
    # The sequences have grown again since the last pass.
    s["ctx"].copy_(s["ctx0"])
    s["w"].copy_(s["w0"])
    f = _K().paged_kv_evict if own else _plain_evict
    kept = f(s["tbl"], s["ctx"], s["w"], s["kv"], c["PAGE"], c["budget"], c["recent"], c["sinks"])
    for x, scale, out in ((kc, ks, s["values"][0]), (vc, vs, s["values"][1])):  # what the codes stand for
        torch.mul(x, scale.float()[..., None], out=out)
    return {"kept": kept, "ctx": s["ctx"], "w": s["w"], "k": s["values"][0], "v": s["values"][1], "ks": ks, "vs": vs}


def _run_beam(s):
    f = _K().beam_select if own else _plain_beam
    return f(s["logits"], s["scores"], s["c"]["n"], s["done"], s["eos"])


def _run_reorder(s):
    if own:
        _K().beam_reorder(s["states"], s["parents"], s["c"]["W"])
    else:
        _plain_reorder(s["states"], s["parents"])
    return s["states"]


def run(state):
    return {"norm": _run_norm, "weights": _run_weights, "evict": _run_evict, "beam": _run_beam,
            "reorder": _run_reorder}[state["c"]["op"]](state)


# ----------------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    up = lambda n: -(-n // c["PAGE"])  # noqa: E731
    if op == "norm":
        tok, heads = c["B"] * c["q_len"], c["H"] + c["H_KV"]
        return {"bytes": tok * heads * c["D"] * 4 + 4 * (c["R"] + c["D"]),
                "flops": tok * heads * (4 * c["D"] + 3 * c["R"])}
    if op == "weights":
        lens, ql, size = _ragged(_Gen(0), c, c["q_len"]), c["q_len"], 2 if c["scales"] == "fp16" else 4
        # Keys, their scales and the queries read, gathered weights read and written.
        b = sum(n * c["H_KV"] * (c["D"] + size + 8) + 4 * up(n) for n in lens) + 2 * c["B"] * ql * c["H"] * c["D"]
        return {"bytes": b, "flops": sum(2 * c["H"] * c["D"] * (ql * (n - ql) + ql * (ql + 1) // 2) for n in lens)}
    if op == "evict":
        lens, size = _ragged(_Gen(0), c, 1), 2 if c["scales"] == "fp16" else 4
        over, pool = [n for n in lens if n > c["budget"]], c["B"] * up(c["ctx"]) + 2
        # Gathered weights read; the tokens that stay read and written with their weights and positions; what the pass
        # hands back as values read and written.
        move = len(over) * c["budget"] * (2 * (2 * c["D"] + 2 * size + 4) + 4)
        back = 2 * pool * c["PAGE"] * (5 * c["D"] + size)
        return {"bytes": c["H_KV"] * (4 * sum(over) + move + back), "flops": 0}
    if op == "beam":
        n = c["B"] * c["W"] * c["V"]
        return {"bytes": n * (2 if c["dtype"] == "fp16" else 4) + 12 * c["B"] * c["n"] + 4 * c["B"] * c["W"], "flops": 4 * n}
    parents = _parents(_Gen(0), c)
    moved = [p for r, p in enumerate(parents) if p != r]
    row = 4 * c["T"] * (1 + c["H_KV"]) + 2 * c["hidden"] + 2 * 2 * 2 * c["draft"] * 64
    return {"bytes": row * (len(moved) + len(set(moved))) + 4 * len(parents), "flops": 0}


# ----------------------------------------------------------------------------------------
# The same in 64 bits, sequence by sequence
# ----------------------------------------------------------------------------------------
def _exact_norm(s):
    c, out = s["c"], []
    w = torch.arange(c["q_len"], dtype=torch.float64, device=DEV)
    for x, g in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c["D"] + 1e-6) * g.double()
        y = x.clone()
        for b, n in enumerate(s["ctx"].tolist()):
            for j in range(c["R"] // 2):
                i0, i1 = (j, j + c["R"] // 2) if c["pairs"] == "half" else (2 * j, 2 * j + 1)
                z = torch.polar(torch.ones_like(w), (w + (n - c["q_len"])) * s["inv_freq"][j])[:, None]
                r = torch.complex(x[b, :, :, i0], x[b, :, :, i1]) * z
                y[b, :, :, i0], y[b, :, :, i1] = r.real, r.imag
        out.append(y)
    return tuple(out)


def _exact_weights(s):
    c, q, w = s["c"], s["q"].double(), s["w"].double()
    B, ql, H, D = q.shape
    G = H // c["H_KV"]
    for b, n in enumerate(s["ctx"].tolist()):
        t = torch.arange(n, device=DEV)
        pg, sl = s["tbl"][b, t // c["PAGE"]].long(), t % c["PAGE"]
        seen = t[None] <= (n - ql + torch.arange(ql, device=DEV))[:, None]
        for h in range(c["H_KV"]):
            k = s["kc"][pg, sl, h].double() * s["ks"][pg, sl, h].double()[:, None]
            x = (q[b, :, h * G:(h + 1) * G].reshape(-1, D) @ k.t() / math.sqrt(D)).view(ql, G, n)
            p = x.masked_fill(~seen[:, None], -math.inf).softmax(-1).sum((0, 1))
            w[b, h, n - ql:n] = 0
            w[b, h, :n] += p
    return w


def _exact_evict(s):
    c, (kc, vc, ks, vs) = s["c"], s["kv"]
    size, page, w = c["budget"], c["PAGE"], s["w0"].double()
    val = [(x.double() * z.double()[..., None], z.double()) for x, z in ((kc, ks), (vc, vs))]
    kept = torch.full((c["B"], c["H_KV"], size), -1, dtype=torch.int32, device=DEV)
    ctx = s["ctx0"].tolist()
    for b, n in enumerate(ctx):
        if n <= size:
            kept[b, :, :n] = torch.arange(n, device=DEV)
            continue
        ctx[b] = size
        to = torch.arange(size, device=DEV)
        for h in range(c["H_KV"]):
            mid = w[b, h, c["sinks"]:n - c["recent"]]
            take = size - c["sinks"] - c["recent"]
            least = mid.sort(descending=True).values[take - 1] if take else math.inf
            above, ties = (mid > least).nonzero().flatten(), (mid == least).nonzero().flatten()
            chosen = torch.cat((above, ties[:take - above.numel()])).sort().values + c["sinks"]
            src = torch.cat((to[:c["sinks"]], chosen, torch.arange(n - c["recent"], n, device=DEV)))
            kept[b, h] = src
            w[b, h, :size] = w[b, h, src]
            sp, dp = s["tbl"][b, src // page].long(), s["tbl"][b, to // page].long()
            for x, z in val:
                x[dp, to % page, h] = x[sp, src % page, h]
                z[dp, to % page, h] = z[sp, src % page, h]
    (k, ks), (v, vs) = val
    return {"kept": kept, "ctx": _i32(ctx), "w": w, "k": k, "v": v, "ks": ks, "vs": vs}


def _exact_beam(s):
    c, out = s["c"], []
    for b in range(c["B"]):
        rows = []
        for w in range(c["W"]):
            x, at = s["logits"][b, w].double(), float(s["scores"][b, w])
            if c["done"] and bool(s["done"][b, w]):
                rows.append([(-at, w, s["eos"])])
                continue
            p = torch.log_softmax(x, -1) + at
            least = p.topk(c["n"]).values[-1]
            rows.append([(-float(p[v]), w, v) for v in (p >= least).nonzero().flatten().tolist() if p[v] > -math.inf])
        best = sorted(sum(rows, []))[:c["n"]]
        out.append(best + [(math.inf, -1 - b * c["W"], -1)] * (c["n"] - len(best)))
    return (torch.tensor([[-x for x, _, _ in r] for r in out], dtype=torch.float64, device=DEV),
            _i32([[v for _, _, v in r] for r in out]),
            _i32([[b * c["W"] + w for _, w, _ in r] for b, r in enumerate(out)]))


def _exact_reorder(s):
    rows = s["parents"].tolist()
    return [torch.stack([x[r] for r in rows]).to(torch.float64 if x.is_floating_point() else x.dtype) for x in s["states"]]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "weights": _exact_weights, "evict": _exact_evict, "beam": _exact_beam,
            "reorder": _exact_reorder}[case["op"]](s)
