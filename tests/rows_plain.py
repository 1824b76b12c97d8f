"""The row cache's operators in plain numpy, in 64 bits: what tests/test_gpu_rows.py and tests/test_rows_cpu.py hold the engine to."""
import numpy as np

from redisearch_amd import rows as R
from redisearch_amd import vecsim as V

F32, F16, BF16 = V.VecSimType_FLOAT32, V.VecSimType_FLOAT16, V.VecSimType_BFLOAT16
EPS = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}      # half a step, relative
LEAST = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}  # half of the smallest step
LARGEST = {F32: float(np.finfo(np.float32).max), F16: 65504.0, BF16: float(np.float32(3.38953139e38))}
SMALLEST = 2.0 ** -100


def padded(dim):
    return -(-dim // 32) * 32


def row_bytes(vtype, dim, fmt):
    if fmt == R.NATIVE:
        return padded(dim) * (4 if vtype == F32 else 2)
    return padded(dim) // (2 if fmt == R.INT4 else 1)


def row_scales(dim, fmt, block):
    return 0 if fmt == R.NATIVE else -(-dim // (block or dim))


def e4m3_values():
    v = [f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10) for e in range(16) for f in range(8)]
    v[127] = np.nan
    return np.array(v + [-x for x in v])


def e4m3_code(y):
    """codes of fp64 values of magnitude <= 448"""
    table = e4m3_values()[:127]
    a = np.abs(y)
    k = np.clip(np.searchsorted(table, a, side="right") - 1, 0, 125)
    below, above = a - table[k], table[k + 1] - a
    k = np.where((above < below) | ((above == below) & (k % 2 == 1)), k + 1, k)
    return (k | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def quantise(x, fmt, block):
    """(packed codes [n, row bytes] uint8, scales [n, blocks] fp32) of rows given as fp64"""
    n, dim = x.shape
    block = block or dim
    nb = -(-dim // block)
    codes = np.zeros((n, padded(dim)), np.uint8)
    scales = np.zeros((n, nb), np.float32)
    for b in range(nb):
        part = x[:, b * block:(b + 1) * block]
        with np.errstate(invalid="ignore"):
            a = np.abs(part).max(1)
        bad = ~np.isfinite(part).all(1)
        live = ~bad & (np.where(bad, 0, a) >= SMALLEST)
        a = np.where(live, a, 1.0)
        if fmt == R.E4M3:
            m, e = np.frexp(a)
            s = np.ldexp(1.0, e - 9 + (m > 0.875))
        else:
            s = (a / (127 if fmt == R.INT8 else 7)).astype(np.float32).astype(np.float64)
        y = np.where(live[:, None], np.where(np.isfinite(part), part, 0) / s[:, None], 0.0)
        c = e4m3_code(y) if fmt == R.E4M3 else np.rint(y).astype(np.int64).astype(np.uint8)
        codes[:, b * block:b * block + part.shape[1]] = np.where(live[:, None], c, 0)
        scales[:, b] = np.where(bad, np.nan, np.where(live, s, 0.0))
    if fmt == R.INT4:
        codes = (codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)
    return codes, scales


def dequantise(codes, scales, dim, fmt, block):
    """fp64 rows"""
    if fmt == R.INT4:
        v = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).astype(np.int64)
        v = np.where(v > 7, v - 16, v).astype(np.float64)
    elif fmt == R.INT8:
        v = codes.view(np.int8).astype(np.float64)
    else:
        v = e4m3_values()[codes]
    return v[:, :dim] * np.repeat(scales.astype(np.float64), block or dim, axis=1)[:, :dim]


def adjust(rules, scores, out, counts):
    """rules: a dict of the ScoreRules fields as arrays.  Returns (fp64 result, bound of its rounding in fp32)."""
    distance = rules.get("form", R.PRODUCT) == R.DISTANCE
    out, slack = out.astype(np.float64), np.zeros(out.shape)
    nq, nc = scores.shape

    def span(name, m, total):
        lo, hi = (min(max(int(v), 0), total) for v in rules[name + "_offsets"][m:m + 2])
        return lo, hi

    with np.errstate(all="ignore"):
        for m in range(nq):
            row = scores[m].astype(np.float64)
            n = nc if counts is None else min(max(int(counts[m]), 0), nc)
            value, size = row.copy(), np.zeros(nc)
            shown, boost = {}, {}
            if "seen_offsets" in rules:
                lo, hi = span("seen", m, len(rules["seen_ids"]))
                for c in rules["seen_ids"][lo:hi]:
                    shown[int(c)] = shown.get(int(c), 0) + 1
            if "bias_offsets" in rules:
                lo, hi = span("bias", m, len(rules["bias_ids"]))
                boost = {int(c): float(v) for c, v in zip(rules["bias_ids"][lo:hi], rules["bias_values"][lo:hi])}
            for c in set(shown) | set(boost):
                if not 0 <= c < nc:
                    continue
                s = row[c]
                p = 1 - s if distance else s
                size[c] = abs(s) + abs(p) + (1 if distance else 0)
                if c in shown:
                    rep = float(rules["repetition"][m]) if "repetition" in rules else 1.0
                    p = p / rep if p > 0 else p * rep
                    size[c] = (size[c]) * max(rep, 1 / rep)
                    off = shown[c] * (float(rules["frequency"][m]) if "frequency" in rules else 0.0) + (float(rules["presence"][m]) if "presence" in rules else 0.0)
                    p -= off
                    size[c] += abs(off) + abs(p)
                if c in boost:
                    p += boost[c]
                    size[c] += abs(boost[c]) + abs(p)
                value[c] = 1 - p if distance else p
            if rules.get("mask") is not None:
                which = int(rules["mask_rows"][m]) if "mask_rows" in rules else m
                if 0 <= which < len(rules["mask"]):
                    bits = np.unpackbits(rules["mask"][which].view(np.uint8), bitorder="little")[:nc]
                    value = np.where(bits == 1, value, np.inf if distance else -np.inf)
                    size = np.where(bits == 1, size, 0)
            out[m, :n] = value[:n]
            slack[m, :n] = size[:n] * 6 * 2.0 ** -24      # at most six roundings, each of a number no larger than size
    return out, slack
