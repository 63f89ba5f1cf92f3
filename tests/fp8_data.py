"""FP8 block-scale references for the tests: 64-bit restatements of the operators,
from the formulas, on the CPU."""
import numpy as np
import torch

BLOCK = 128
FMT = {"e4m3": 1, "e5m2": 2}
QMAX = {"e4m3": 448.0, "e5m2": 57344.0}
TYPE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def up(n, m=BLOCK):
    return -(-n // m)


def nearest8(x, fmt):
    """Nearest 8-bit value (ties to even) of a float64 array within range."""
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    _, ex = np.frexp(x)
    ulp = np.ldexp(1.0, np.maximum(ex - 1, low) - mant)
    return np.round(x / ulp) * ulp


def quant_rows(x, fmt):
    """float64 [M, K] -> (8-bit values, scales) per 1 x 128."""
    m, k = x.shape
    q, s = np.zeros_like(x), np.ones((m, up(k)))
    for b in range(up(k)):
        blk = x[:, b * BLOCK:(b + 1) * BLOCK]
        amax = np.abs(blk).max(axis=1)
        s[:, b] = np.where(amax > 0, amax / QMAX[fmt], 1.0)
        q[:, b * BLOCK:(b + 1) * BLOCK] = nearest8(blk * QMAX[fmt] / np.where(amax > 0, amax, 1.0)[:, None], fmt)
    return q, s


def dequant(q, s, rows_per):
    n, k = q.shape
    return q * s[np.arange(n) // rows_per][:, np.arange(k) // BLOCK]


def to_fp8(v, fmt):
    """float array of representable values -> uint8 codes."""
    return torch.from_numpy(np.asarray(v, np.float32)).to(TYPE[fmt]).view(torch.uint8)


def from_fp8(codes, fmt):
    return codes.cpu().view(TYPE[fmt]).to(torch.float64).numpy()


def random_operand(rng, rows, k, fmt, row_block):
    """(uint8 codes, fp32 scales, float64 values) of a block-scaled matrix."""
    v = nearest8(rng.standard_normal((rows, k)) * QMAX[fmt] / 8, fmt)
    v = np.clip(v, -QMAX[fmt], QMAX[fmt])
    s = np.exp(rng.uniform(-6, 2, (up(rows, row_block), up(k)))).astype(np.float32)
    return to_fp8(v, fmt), torch.from_numpy(s), dequant(v, s.astype(np.float64), row_block)


def gate(z, bias, k, sigmoid, groups, top_groups, group_top, renorm, scale):
    """(ids, weights) in float64, one token after the other."""
    z = np.asarray(z, np.float64)
    t, e = z.shape
    size = e // groups
    ids, w = np.zeros((t, k), np.int32), np.zeros((t, k))
    for r in range(t):
        masked = ~(z[r] > -np.inf)
        zr = np.where(masked, -np.inf, z[r])
        with np.errstate(over="ignore", invalid="ignore"):
            if sigmoid:
                s = 1.0 / (1.0 + np.exp(-zr))
            else:
                m = zr.max()
                x = np.where(zr == m, 1.0, np.exp(zr - m))
                x = np.where(masked, 0.0, x)
                s = x / x.sum() if x.sum() > 0 else x
            v = s + (0.0 if bias is None else np.asarray(bias, np.float64))
        v = np.where(masked | np.isnan(v), -np.inf, v)
        order = zr if bias is None else v   # without a bias by the logits, also where 64 bits saturate
        if groups > 1:
            one = min(group_top, size) == 1
            per = np.sort((order if one else v).reshape(groups, size), axis=1)[:, ::-1]
            worth = per[:, :min(group_top, size)].sum(axis=1)
            stay = np.argsort(-worth, kind="stable")[:top_groups]
            inside = np.isin(np.arange(e) // size, stay)
        else:
            inside = np.ones(e, bool)
        cand = np.nonzero(inside)[0]
        pick = cand[np.argsort(-order[cand], kind="stable")[:k]]
        ids[r] = pick
        with np.errstate(over="ignore", invalid="ignore"):
            if renorm and not masked[pick].all():
                zc = zr[pick]
                m = zc.max()
                x = np.where(zc == m, 1.0, np.exp(zc - m))   # scores over e^m: none is lost to underflow
                if sigmoid:
                    x = s[pick] if m > 0 else x / (1.0 + np.exp(zc))
                x = np.where(masked[pick], 0.0, x)
                w[r] = x / x.sum()
            elif not renorm:
                w[r] = np.where(masked[pick], 0.0, s[pick])
    return ids, w * scale
