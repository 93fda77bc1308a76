"""Plain forms of the paged 8-bit cache in 64 bits, written as loops over rows, pages and tokens."""
import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


def e4m3(x):
    """float64 array on the e4m3 grid: ties to even, exponents down to -6, NaN for infinities and NaN."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(all="ignore"):
        _, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
        step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
        return np.where(np.isfinite(x), np.rint(x / step) * step, np.nan)


def scale_of(values):
    fin = np.abs(values[np.isfinite(values)])
    top = fin.max() if fin.size else 0.0
    s = 2.0 ** -64
    if top > 0:
        m, e = math.frexp(top / 448.0)
        s = max(s, math.ldexp(1.0, e - (m == 0.5)))
    return s


def write(codes, scales, x, segments):
    """codes [pages, P, H, D], scales [pages, H] float64 arrays, changed in place."""
    for page, off, tok, n in segments:
        if n == 0:
            continue
        for h in range(x.shape[1]):
            rows = x[tok:tok + n, h]
            s = scale_of(rows)
            if off:
                s = max(s, scales[page, h])
                codes[page, :off, h] = e4m3(codes[page, :off, h] * (scales[page, h] / s))
            codes[page, off:off + n, h] = e4m3(rows / s)
            scales[page, h] = s


def plan(old, new, table, free, head, P, T):
    """Lists in, a dict of lists out; `table` (list of lists) is changed in place.  For steps that fit."""
    out = dict(cu=[0], positions=[], slots=[], lens=[], segments=[])
    for b, (o, n) in enumerate(zip(old, new)):
        for i in range(-(-o // P), -(-(o + n) // P)):
            table[b][i] = free[head]
            head += 1
        at = o
        while at < o + n:
            m = min(P - at % P, o + n - at)
            out["segments"].append([table[b][at // P], at % P, out["cu"][-1] + at - o, m])
            at += m
        for p in range(o, o + n):
            out["positions"].append(p)
            out["slots"].append(table[b][p // P] * P + p % P)
        out["cu"].append(out["cu"][-1] + n)
        out["lens"].append(o + n)
    spare = T - len(out["slots"])
    out["positions"] += [-1] * spare
    out["slots"] += [-1] * spare
    out["segments"] += [[0, 0, 0, 0]] * (min(T, T // P + 2 * len(old)) - len(out["segments"]))
    out["head"] = [head]
    return out


def decode(q, k, v, ks, vs, table, lens, scale, score=None, keep=None):
    """q [B, Sq, Hq, D]; codes and scales as the cache holds them.  float64 [B, Sq, Hq, DV]; zeros for a row without a kept key.
    `score(s, b, h)` and `keep(b, h, q_idx, kv_idx)` work on tensors over the keys."""
    q, kd, vd, ks, vs = q.double().cpu(), k.double().cpu(), v.double().cpu(), ks.double().cpu(), vs.double().cpu()
    B, Sq, Hq, _ = q.shape
    P, Hkv, DV = k.shape[1], k.shape[2], v.shape[3]
    out = torch.zeros(B, Sq, Hq, DV, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        pages = [int(x) for x in table[b][:-(-n // P)]]
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk = (kd[pages, :, g] * ks[pages, g][:, None, None]).reshape(-1, kd.shape[3])[:n]
            vv = (vd[pages, :, g] * vs[pages, g][:, None, None]).reshape(-1, DV)[:n]
            for i in range(Sq):
                s = (q[b, i, h] * kk).sum(-1) * scale
                if score is not None:
                    s = score(s, b, h)
                if keep is not None:
                    s = torch.where(keep(b, h, i, torch.arange(n)), s, -math.inf)
                if not torch.isinf(s).all() or (s > 0).any():
                    out[b, i, h] = torch.softmax(s, -1) @ vv
    return out
