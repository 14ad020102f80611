"""Random block-scaled paged caches for the tests: numpy codes, scales and tables, and their GPU tensors."""
import numpy as np
import torch

F8 = torch.float8_e4m3fn


def codes(rng, fmt, shape):
    if fmt == "int8":
        return rng.integers(-127, 128, shape, dtype=np.int8)
    c = rng.integers(0, 256, shape, dtype=np.uint8)
    c[(c & 127) == 127] -= 1  # no NaN
    return c


def make_cache(rng, ctx, H_KV, D, PAGE, SB, fmt, spare=3, lo=0.5, hi=1.5):
    """(kc, vc, ks, vs, bt, ctx): values of size about 1; table entries past a row's pages are -1."""
    pages = [-(-c // PAGE) if c > 0 else 0 for c in ctx]
    P, C = sum(pages) + spare, max(max(pages), 1) + 1
    bt = np.full((len(ctx), C), -1, np.int32)
    perm, at = rng.permutation(P).astype(np.int32), 0
    for b, n in enumerate(pages):
        bt[b, :n] = perm[at:at + n]
        at += n
    unit = 1 / 64 if fmt == "int8" else 1 / 64
    kc, vc = codes(rng, fmt, (P, PAGE, H_KV, D)), codes(rng, fmt, (P, PAGE, H_KV, D))
    ks, vs = ((rng.uniform(lo, hi, (P, PAGE // SB, H_KV)) * unit).astype(np.float32) for _ in "kv")
    return kc, vc, ks, vs, bt, np.asarray(ctx, np.int32)


def gpu(*arrays, dev="cuda"):
    """numpy arrays as GPU tensors; uint8 arrays are e4m3 bytes."""
    out = []
    for a in arrays:
        t = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        out.append(t.view(F8) if t.dtype == torch.uint8 else t)
    return out


def raw(t):
    """A GPU tensor's values, e4m3 as bytes."""
    return (t.view(torch.uint8) if t.dtype == F8 else t).cpu().numpy()
