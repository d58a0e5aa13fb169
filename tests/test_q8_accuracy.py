"""Accuracy of the 8-bit decode attention, held to what float32 arithmetic gives whatever the type of q: weights and
queries of every size, V scales of every size. The 64-bit results are those of q8_reference.py; the bound is this
file's own (bound_of)."""

import numpy as np
import pytest
import torch

import q8_reference as ref
import test_q8_cache as q8

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}        # the result is rounded once: half a step


def bound_of(q, k_codes, v_codes, scales, table, lens, store):
    """(out, bound), float64 [B, Hq, D]: what the float32 result may be off by before it is rounded to the type of q.

    As in q8_reference.decode_bound a score is off by at most 2^-18 of sum |q k| / sqrt(D) (natural log units) and its
    exponential by 2^-20 more; both the numerator and the sum below it have that error. Queries go to the tensor cores
    as halves of a row scaled into [2^14, 2^15), where what is left out is at most half a step of the smallest one, 2^-25:
    2^-39 of the row's largest element (2^-38 here). For the product with V a weight goes in two halves, the remainder's
    rounding being 2^-21 of the weight or less, and is scaled likewise: a small one loses at most 2^-39 (2^-38 here) of
    the largest weight * V scale. A warp adds up at most one tensor-core step per 32 rows (generic kernel: 4 float32
    additions with a sixteenth of the error each), each off by at most 2^-22 of the running sum of magnitudes, and the
    partial results of up to 32 warps or ranges; so does the sum of the weights, hence 2^-21."""
    batch, hq, dim = q.shape
    hkv, page = k_codes.shape[1], k_codes.shape[2]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        n = int(lens[b])
        if n == 0:
            continue
        ids = table[b, : -(-n // page)]
        for h in range(hq):
            kv = h // (hq // hkv)
            k = ref.values(k_codes[ids, kv], scales[ids, kv], 0, store).reshape(-1, dim)[:n]
            v = ref.values(v_codes[ids, kv], scales[ids, kv], 1, store).reshape(-1, dim)[:n]
            vs = np.abs(np.repeat(scales[ids, kv, 1].astype(np.float64), page)[:n])
            s = k @ q[b, h] / np.sqrt(dim)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h] = p @ v
            size = (np.abs(k) @ np.abs(q[b, h])).max() / np.sqrt(dim)
            left = 2.0 ** -38 * np.abs(q[b, h]).max() * np.abs(k).sum(1).max() / np.sqrt(dim)
            d = 2.0 ** -18 * size + 2.0 ** -20 + left
            bound[b, h] = (p @ np.abs(v)) * (2 * d + 2.0 ** -21 + (n / 32 + 32) * 2.0 ** -21) + n * 2.0 ** -38 * (p * vs).max() * ref.TOP[store]
    return out, bound


def check(q, k, v, scales, table, lens, store, name):
    got = q8.ft().attention_decode_paged_q8(q.cuda(), q8.pool(k, store), q8.pool(v, store), q8.on_gpu(scales), q8.on_gpu(table),
                                            q8.on_gpu(np.asarray(lens, np.int32)))
    want, bound = bound_of(q.double().numpy(), k, v, scales, table, lens, store)
    # Numbers below the smallest normal one (2^-14 in float16) have a fixed step, and rounding to it is off by half of that.
    # The float32 result before it may be subnormal too, and so may be every row's weight (at most 1) * V scale, whose
    # rounding, up to 2^-150, meets a code.
    small = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2 + 2.0 ** -149 + max(lens) * 2.0 ** -150 * ref.TOP[store]
    tol = bound + (np.abs(want) + bound) * HALF[name] + small
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max() / np.abs(want).max()))
    return got


# ---- weights ---------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("store", list(q8.STORES))
@pytest.mark.parametrize("name", list(q8.DTYPES))
@pytest.mark.parametrize("hq,hkv,dim,page", [(8, 2, 128, 16), (5, 1, 128, 16), (16, 2, 128, 16), (7, 1, 64, 32), (16, 1, 128, 64), (24, 1, 96, 16),
                                             (13, 1, 80, 16), (8, 1, 192, 16), (12, 1, 256, 32), (8, 1, 112, 16), (6, 1, 64, 12)])
def test_weights_of_any_number_of_heads(hq, hkv, dim, page, name, store):
    """Few rows, small scores: what is left of the error is the rounding of the weights."""
    rng = np.random.default_rng(hq * dim + page)
    lens = [2, 17, 40, 64, 100]
    k, v, scales, table = q8.make_cache(rng, lens, hkv, dim, page, store)
    q = q8.rounded(0.1 * rng.standard_normal((len(lens), hq, dim)), name)
    check(q, k, v, scales, table, lens, store, name)


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(q8.STORES))
@pytest.mark.parametrize("gap", [9.0, 12.3, 15.0, 17.5, 20.0])
@pytest.mark.parametrize("name,hq,dim,page", [("f32", 4, 128, 16), ("f32", 8, 64, 64), ("f32", 3, 256, 16), ("bf16", 16, 128, 16), ("f16", 8, 80, 16),
                                              ("f16", 4, 128, 12)])
def test_one_row_far_above_thousands(name, hq, dim, page, gap, store):
    """One row whose own V is zero takes nearly all the weight; the result is what thousands of rows, `gap` natural log
    units below it, add up to. Their V share a sign, so nothing cancels and the bound is relative to the result."""
    rng = np.random.default_rng(int(gap * 10) + dim)
    lens = [6007, 2500]
    k, v, scales, table = q8.make_cache(rng, lens, 1, dim, page, store, spread=0.0)
    full = 100.0 if store == "int8" else 104.0
    k[:] = ref.nearest_codes(rng.integers(-2, 3, k.shape), store)
    v[:] = ref.nearest_codes(rng.integers(64, 112, v.shape), store)
    for b, at in enumerate((3333, 0)):
        k[table[b, at // page], 0, at % page] = ref.nearest_codes(np.full(dim, full), store)
        v[table[b, at // page], 0, at % page] = 0
    scales[..., 0] = gap / (full * np.sqrt(dim))
    q = q8.rounded(np.ones((2, hq, dim)), name)
    check(q, k, v, scales, table, lens, store, name)


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(q8.STORES))
@pytest.mark.parametrize("name,hq,dim,page", [("f32", 4, 128, 16), ("f32", 8, 64, 64), ("bf16", 8, 128, 16), ("bf16", 2, 256, 16), ("f16", 16, 80, 16),
                                              ("bf16", 4, 64, 12)])
def test_queries_far_below_the_largest_of_their_row(name, hq, dim, page, store):
    """One element of a query row is far larger than all others and meets codes that are zero: the scores are the others'."""
    rng = np.random.default_rng(dim + hq)
    lens = [90, 33, 5]
    k, v, scales, table = q8.make_cache(rng, lens, 1, dim, page, store)
    k[..., 7] = 0
    least = 2.0 ** -10 if name == "f16" else 1.0
    q = rng.standard_normal((3, hq, dim)) * least * 0.1
    q[..., 7] = least * 2.0 ** (18 if name != "f16" else 25)
    scales[..., 0] /= least
    check(q8.rounded(q, name), k, v, scales, table, lens, store, name)


# ---- V scales --------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("store", list(q8.STORES))
@pytest.mark.parametrize("name,hq,dim,page", [("f32", 4, 128, 16), ("f32", 8, 64, 64), ("bf16", 8, 128, 16), ("f32", 2, 256, 32), ("f32", 4, 64, 12)])
@pytest.mark.parametrize("power", [-130, -120, -90, -75, 76, 90, 115])
def test_v_scales_of_any_size_behind_blocks_of_zeros(power, name, hq, dim, page, store):
    """Blocks of zeros (scale 0) first, then V scales that do not differ much but are all very small (subnormal ones among
    them) or very large: what a block of zeros is taken for must not limit the others."""
    rng = np.random.default_rng(dim + 200 + power)
    lens = [page * 20 + 3, page * 4, page * 3 + 1, page * 9]
    k, v, scales, table = q8.make_cache(rng, lens, 1, dim, page, store)
    scales[..., 1] = (scales[..., 1].astype(np.float64) * 2.0 ** power).astype(np.float32)
    scales[table[0, :8], :, 1] = 0
    scales[table[0, 10], :, 1] = 0
    scales[table[1, :1], :, 1] = 0
    scales[table[2, 1:], :, 1] = 0
    q = q8.rounded(rng.standard_normal((4, hq, dim)), name)
    check(q, k, v, scales, table, lens, store, name)


def rows_of_one_score(scores, v_powers, dim, store, rng):
    """A sequence of blocks of 16 rows whose scores (log2 units, for q = 1) and V scales (powers of two; None: zero) are
    given for each block."""
    n = len(scores)
    k = ref.nearest_codes(np.ones((n, 1, 16, dim)), store)
    v = ref.nearest_codes(rng.integers(64, 112, (n, 1, 16, dim)), store)
    scales = np.zeros((n, 1, 2), np.float32)
    scales[:, 0, 0] = np.asarray(scores) * np.log(2.0) / np.sqrt(dim)
    scales[:, 0, 1] = [0.0 if e is None else 2.0 ** e for e in v_powers]
    return k, v, scales, np.arange(n, dtype=np.int32)[None]


# (scores, V scales) block by block; a tile has four blocks, and tiles 0 and 4 meet the same warps
FAR = [
    # what one warp adds up with its V scales counted from the largest, and another from the smallest
    ([-100, -7, -100, -100, -100, 0, -100, -100], [60, 0, 0, 0, 0, 60, 0, 0]),
    ([-100, 0, -100, -100, -100, -7, -100, -100], [0, 60, 0, 0, 60, 0, 0, 0]),
    # zeros first, then a scale far above the first that is not zero
    ([-7, -100] + [-100] * 14 + [0, -100], [None, 0] + [0] * 14 + [60, 0]),
    # and the other way round
    ([-100, -100] + [-100] * 14 + [0, -7], [0, 0] + [0] * 14 + [60, None]),
    # zeros far above everything else, and as far below
    ([0, -20, -25, 0, -20, -30, -22, -21], [None, 0, 0, None, 0, 0, 0, 0]),
    ([-90, 0, 0, -90, -1, -2, -3, -4], [None, 0, 0, None, 0, 0, 0, 0]),
    # 2^60 between the scales, every order
    ([0, 50, 60, 58, 3, 0, 0, 61] * 3, [60, 10, 0, 1, 58, 60, 59, 0] * 3),
    ([60, 61, 59, 0, 0, 0, 55, 50] * 3, [0, 0, 1, 60, 60, 58, 5, 10] * 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(q8.STORES))
@pytest.mark.parametrize("hq,dim", [(4, 128), (8, 64), (3, 256), (16, 96)])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_v_scales_and_scores_far_apart(case, hq, dim, store):
    """V scales that differ by 2^60, blocks of zeros, and scores that make up for it or do not: no weight that counts for the
    sum of the weights is lost, in whichever warp it is met first."""
    rng = np.random.default_rng(case)
    k, v, scales, table = rows_of_one_score(*FAR[case], dim, store, rng)
    lens = [16 * len(FAR[case][0])]
    check(torch.ones((1, hq, dim)), k, v, scales, table, lens, store, "f32")
    # the same blocks many times over: units that are cut, and folded by the merge
    table = np.repeat(table, 40, axis=0).reshape(1, -1)
    check(torch.ones((1, hq, dim)), k, v, scales, table, [16 * table.shape[1]], store, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(q8.STORES))
@pytest.mark.parametrize("hq,dim", [(4, 128), (8, 64), (3, 256), (16, 96)])
@pytest.mark.parametrize("spread", [61, 66, 75, 90, 120, 150])
def test_v_scales_beyond_the_range_that_is_promised(spread, hq, dim, store):
    """V scales further apart than 2^60, smallest and largest first, with scores that do not make up for it: the large ones
    decide, and the weights of the others count below the line."""
    rng = np.random.default_rng(spread)
    for order in (1, -1):
        powers = np.concatenate([np.linspace(-spread / 2, spread / 2, 12).round(), [-spread // 2, 0, spread // 2, None]])[::order]
        scores = rng.uniform(-4, 4, len(powers)).round(2)
        k, v, scales, table = rows_of_one_score(scores, [None if e is None else int(e) for e in powers], dim, store, rng)
        for n in (1, 40):
            wide = np.repeat(table, n, axis=0).reshape(1, -1)
            check(torch.ones((1, hq, dim)), k, v, scales, wide, [16 * wide.shape[1]], store, "f32")
