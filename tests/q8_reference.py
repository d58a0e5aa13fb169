"""Plain 64-bit implementations of the operators on an 8-bit paged cache and of the block table operators, in numpy
loops, straight from the definitions; and the error bound the decode kernels are held to."""

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def e4m3_values():
    """The value of every e4m3 code: sign, 4 bits of exponent (bias 7), 3 of mantissa; 0x7f and 0xff are NaN."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


E4M3 = e4m3_values()
_POS = E4M3[:127]                                   # 0 .. 448, increasing, index = code


def decode_codes(codes, store):
    """Values of uint8 codes."""
    return codes.view(np.int8).astype(np.float64) if store == "int8" else E4M3[codes]


def nearest_codes(x, store):
    """uint8 codes nearest to float64 values, ties to the even code, beyond the largest: the largest."""
    x = np.asarray(x, np.float64)
    if store == "int8":
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(x), 448.0)
    hi = np.searchsorted(_POS, a)                   # first code >= a
    hi = np.minimum(hi, 126)
    lo = np.maximum(hi - 1, 0)
    mid = (_POS[lo] + _POS[hi]) / 2
    up = (a > mid) | ((a == mid) & (hi % 2 == 0)) | (a == _POS[hi])
    c = np.where(up, hi, lo).astype(np.uint8)
    return np.where(np.signbit(x), c | 128, c).astype(np.uint8)


def append(codes, scales, which, x, slots, page, store):
    """In place on uint8 codes [Nb, Hkv, P, D] and float32 scales [Nb, Hkv, 2]; x float64-convertible [N, Hkv, D]."""
    x = np.asarray(x, np.float64)
    i, n = 0, len(slots)
    while i < n:
        if slots[i] < 0 or slots[i] >= codes.shape[0] * page:
            i += 1
            continue
        blk, off = divmod(int(slots[i]), page)
        j = i + 1
        while j < n and slots[j] == slots[i] + (j - i) and off + (j - i) < page:
            j += 1
        for h in range(codes.shape[1]):
            old = scales[blk, h, which] if off else np.float32(0)
            rows = x[i:j, h]
            if not np.isfinite(rows).all() or np.isnan(old):
                new = np.float32(np.nan)
            else:
                new = np.maximum(old, np.float32(np.abs(rows).max()) / np.float32(TOP[store]))
            scales[blk, h, which] = new
            fine = np.isfinite(new) and new > 0
            if fine and off and new != old:
                held = decode_codes(codes[blk, h, :off], store)
                codes[blk, h, :off] = nearest_codes(held * np.float64(old) / np.float64(new), store)
            codes[blk, h, off:off + j - i] = nearest_codes(rows / np.float64(new), store) if fine else 0
        i = j


def values(codes, scales, which, store):
    return decode_codes(codes, store) * scales[..., which].astype(np.float64)[..., None, None]


def decode(q, k_codes, v_codes, scales, table, lens, store, weight_step):
    """(out, bound), float64 [B, Hq, D]: `bound` is what a kernel's float32 result may be off by before it is rounded
    to the type of q (decode_bound)."""
    q = np.asarray(q, np.float64)
    batch, hq, dim = q.shape
    hkv, page = k_codes.shape[1], k_codes.shape[2]
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for b in range(batch):
        n = int(lens[b])
        if n == 0:
            continue
        ids = table[b, : -(-n // page)]
        for h in range(hq):
            kv = h // (hq // hkv)
            k = values(k_codes[ids, kv], scales[ids, kv], 0, store).reshape(-1, dim)[:n]
            v = values(v_codes[ids, kv], scales[ids, kv], 1, store).reshape(-1, dim)[:n]
            vs = np.abs(np.repeat(scales[ids, kv, 1].astype(np.float64), page)[:n])
            s = k @ q[b, h] / np.sqrt(dim)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h] = p @ v
            size = (np.abs(k) @ np.abs(q[b, h]) / np.sqrt(dim)).max()
            bound[b, h] = decode_bound(p, v, size, (p * vs).max(), TOP[store], weight_step)
    return out, bound


def decode_bound(p, v, size, unit, top, weight_step):
    """Bound on the error of one head's float32 result.

    A score is a sum of D exact products of half-precision operands, q being its row times a power of two in one half, or
    two: two leave out 2^-22 of the row's largest element, each of the at most 16 tensor-core steps drops at most 2^-22
    of the running sum of magnitudes, and the factors (scale, 1/sqrt(D), log2 e) are off by a few 2^-24: together below
    2^-18 of sum |q k| / sqrt(D) (`size`, natural log units). exp2 adds 2^-21. So every weight is off by at most
    d = 2^-18 size + 2^-20, relative, in the numerator and in the sum below it.
    For the product with V a weight is rounded to half precision (`weight_step`: half a step, 2^-11, or 2^-21 where it
    goes in two halves), and a small one loses up to 2^-25 of the accumulator's unit, at most twice the largest
    weight * V scale (`unit`), times a code of at most `top`. Each of the at most n / 16 + 16 steps drops at most 2^-22 of
    the running sum of magnitudes."""
    a = p @ np.abs(v)
    d = 2.0 ** -18 * size + 2.0 ** -20
    n = len(p)
    return a * (2 * d + weight_step + (n / 16 + 16) * 2.0 ** -22) + n * 2.0 ** -24 * unit * top


def extend(table, lens, new, free, count, page, max_tokens):
    """table in place; returns slots, starts, lens, count."""
    lens, new = [max(int(x), 0) for x in lens], [max(int(x), 0) for x in new]
    batch, width = table.shape
    slots = np.full(max_tokens, -1, np.int32)
    starts = np.zeros(batch + 1, np.int64)
    out = list(lens)
    asked, taken = 0, 0
    for b in range(batch):
        starts[b + 1] = starts[b] + new[b]
        if lens[b] + new[b] > width * page or starts[b + 1] > max_tokens:
            continue
        held = -(-lens[b] // page)
        ask = -(-(lens[b] + new[b]) // page) - held
        asked += ask
        if ask and asked > count:
            continue
        for j in range(ask):
            table[b, held + j] = free[count - 1 - taken - j]
        taken += ask
        for j in range(new[b]):
            pos = lens[b] + j
            slots[starts[b] + j] = table[b, pos // page] * page + pos % page
        out[b] = lens[b] + new[b]
    return slots, np.minimum(starts, 2 ** 31 - 1).astype(np.int32), np.array(out, np.int32), count - taken


def trim(table, lens, keep, free, count, page):
    """free in place; returns lens, count."""
    out = []
    for b in range(table.shape[0]):
        n = max(int(lens[b]), 0)
        k = min(max(int(keep[b]), 0), n)
        for j in range(-(-k // page), -(-n // page)):
            if count < len(free):
                free[count] = table[b, j]
                count += 1
        out.append(k)
    return np.array(out, np.int32), count
