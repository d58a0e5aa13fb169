"""The serving operators around an 8-bit paged KV cache, as they are measured.

Four operators of one decode step: ``block_table_extend`` (blocks and slot map for the tokens of the step),
``kv_append_paged_q8`` (the tokens' keys and values into the 8-bit cache), ``attention_decode_paged_q8`` (attention
over it) and ``block_table_trim`` (blocks of finished or shortened sequences back to the free stack).

``run`` computes them in elementary torch operations, or through the package where ``own`` is true. Lengths are the
same for every seed up to their order, so that the work of a case is known from the case alone.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
STORES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token for each of the 256 sequences of the serving mix (log-uniform lengths up to 32768)
        dict(name="extend_step_b256", op="extend", batch=256, lo=1024, hi=32767, spread="log", new_lo=1, new_hi=1,
             page=16, refuse=False),
        # 64 ragged prompts arriving at once in an empty cache
        dict(name="extend_prompts_b64", op="extend", batch=64, lo=0, hi=0, spread="lin", new_lo=128, new_hi=8192,
             page=16, refuse=False),
        # every sixteenth sequence of the serving mix has finished
        dict(name="trim_finished_b256", op="trim", batch=256, lo=1024, hi=32768, spread="log", finished=16, back=0,
             page=16),
        # rejected draft tokens are cut off 2048 short sequences, half of which have finished
        dict(name="trim_drafts_b2048", op="trim", batch=2048, lo=1, hi=1024, spread="log", finished=2, back=8, page=16),
        # a decode step of 32 sequences around 4096 tokens: the smallest append, all latency
        dict(name="append_step_b32", op="append", batch=32, lo=3500, hi=4600, spread="lin", new_lo=1, new_hi=1,
             kv_heads=8, dim=128, page=16, dtype="bfloat16", store="int8", pad=0),
        # a decode step of 256 sequences, larger blocks, some padded tokens behind it
        dict(name="append_step_b256", op="append", batch=256, lo=64, hi=1023, spread="log", new_lo=1, new_hi=1,
             kv_heads=8, dim=128, page=64, dtype="bfloat16", store="e4m3", pad=13),
        # the next chunk of a few prompts, beginning and ending inside blocks; float32 values, small heads
        dict(name="append_chunk_f32", op="append", batch=5, lo=3, hi=771, spread="lin", new_lo=97, new_hi=411,
             kv_heads=8, dim=64, page=32, dtype="float32", store="e4m3", pad=0),
        # 64 whole prompts of up to 8192 tokens
        dict(name="append_prompts_b64", op="append", batch=64, lo=0, hi=0, spread="lin", new_lo=128, new_hi=8192,
             kv_heads=8, dim=128, page=16, dtype="float16", store="int8", pad=0),
        # one sequence, a head of its own for every query head: the smallest decode, all latency
        dict(name="decode_b1_f32", op="decode", batch=1, q_heads=8, kv_heads=8, dim=64, lo=512, hi=512, spread="lin",
             page=16, dtype="float32", store="int8", empty=0),
        # 32 sequences of 4096 tokens, four query heads on each kv head
        dict(name="decode_b32_4096", op="decode", batch=32, q_heads=32, kv_heads=8, dim=128, lo=4096, hi=4096,
             spread="lin", page=16, dtype="bfloat16", store="int8", empty=0),
        # 64 ragged sequences of 128 to 8192 tokens
        dict(name="decode_b64_ragged", op="decode", batch=64, q_heads=32, kv_heads=8, dim=128, lo=128, hi=8192,
             spread="lin", page=16, dtype="float16", store="e4m3", empty=0),
        # long contexts, eight query heads on each kv head
        dict(name="decode_b4_131072", op="decode", batch=4, q_heads=64, kv_heads=8, dim=128, lo=131072, hi=131072,
             spread="lin", page=16, dtype="bfloat16", store="e4m3", empty=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["extend", "trim", "append", "append", "decode", "decode", "decode"])
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "extend":
        batch, hi = _log(rng, 1, 1024), _log(rng, 1, 16384)
        new_hi = rng.choice([1, _log(rng, 1, 2048)])
        return dict(op=op, batch=batch, lo=rng.randint(0, hi), hi=hi, spread=rng.choice(["log", "lin"]),
                    new_lo=rng.randint(0, 1), new_hi=min(new_hi, max(1, 400000 // batch)), page=page,
                    refuse=rng.random() < 0.25)
    if op == "trim":
        hi = _log(rng, 1, 16384)
        return dict(op=op, batch=_log(rng, 1, 2048), lo=rng.randint(0, hi), hi=hi, spread=rng.choice(["log", "lin"]),
                    finished=rng.choice([1, 2, 7, 16]), back=rng.choice([0, 3, 8]), page=page)
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 128, 256])
    kinds = dict(dtype=rng.choice(list(DTYPES)), store=rng.choice(list(STORES)))
    spread = rng.choice(["log", "lin"])
    if op == "append":
        batch = _log(rng, 1, 256)
        tokens = 150_000_000 // (kv_heads * dim * batch)         # new and cached tokens of a sequence at most
        hi = min(_log(rng, 1, 8192), tokens)
        new_hi = rng.choice([1, min(_log(rng, 1, 4096), tokens)])
        return dict(op=op, batch=batch, lo=rng.randint(0, hi), hi=hi, spread=spread, new_lo=rng.randint(0, 1),
                    new_hi=new_hi, kv_heads=kv_heads, dim=dim, page=page, pad=rng.choice([0, 0, 5]), **kinds)
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    batch = _log(rng, 1, 256)
    hi = min(_log(rng, 1, 131072), 400_000_000 // (kv_heads * dim * batch))
    return dict(op=op, batch=batch, q_heads=group * kv_heads, kv_heads=kv_heads, dim=dim, lo=rng.randint(1, hi), hi=hi,
                spread=spread, page=page, empty=rng.choice([0, 0, 5]), **kinds)


def _spread(n, lo, hi, how):
    """n whole numbers over [lo, hi], at even steps of their value or of its logarithm."""
    at = (np.arange(n) + 0.5) / n
    if how == "log":
        x = np.exp(np.log(max(lo, 1)) + at * (np.log(hi + 1) - np.log(max(lo, 1)))) if hi >= 1 else np.zeros(n)
    else:
        x = lo + at * (hi + 1 - lo)
    return np.clip(np.floor(x), lo, hi).astype(np.int64)


def _lengths(case):
    """(tokens in the cache, tokens of this call) of each sequence, before the seed's order."""
    n = case["batch"]
    lens = _spread(n, case["lo"], case["hi"], case["spread"])
    if case["op"] == "decode" and case["empty"] and n > 1:
        lens[:: case["empty"]] = 0
    if case["op"] in ("extend", "append"):
        new = _spread(n, case["new_lo"], case["new_hi"], "lin")
        if not new.any():
            new[0] = 1
        return lens, new
    if case["op"] == "trim":
        keep = np.maximum(lens - np.arange(n) % (case["back"] + 1), 0)
        keep[:: case["finished"]] = 0
        return lens, keep
    return lens, np.zeros(n, np.int64)


def _pages(tokens, page):
    return -(-tokens // page)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _codes(shape, store, g):
    """What a block of a cache holds: normal values over the block's largest, rounded to the storage type."""
    made = []
    for first in range(0, shape[0], 2048):
        x = torch.randn((min(2048, shape[0] - first),) + tuple(shape[1:]), device="cuda", generator=g)
        x.mul_(TOP[store] / x.abs().amax(dim=(2, 3), keepdim=True).clamp_min(1e-6))
        made.append(x.round().to(torch.int8) if store == "int8" else x.to(torch.float8_e4m3fn))
    return torch.cat(made)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = rng.permutation(case["batch"])
    lens, second = (x[order] for x in _lengths(case))
    page, n = case["page"], case["batch"]
    gpu = lambda x, dt=torch.int32: torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dt)  # noqa: E731
    end = lens + second if case["op"] in ("extend", "append") else lens
    held, need = _pages(lens, page), _pages(end, page)
    width = max(1, int(need.max()))
    blocks = int(need.sum()) + 1 + int(need.sum()) // 16
    perm = rng.permutation(blocks).astype(np.int32)
    table = np.zeros((n, width), np.int32)
    filled = need if case["op"] in ("append", "decode") else held
    row = np.repeat(np.arange(n), filled)
    col = np.arange(int(filled.sum())) - np.repeat(np.cumsum(filled) - filled, filled)
    table[row, col] = perm[: len(row)]
    s = dict(op=case["op"], page=page, table=gpu(table), lens=gpu(lens))
    if case["op"] in ("extend", "trim"):
        free = np.full(blocks, -1, np.int32)
        left = perm[len(row):]
        if case["op"] == "extend" and case["refuse"]:            # fewer free blocks than the step asks for
            left = left[: int((need - held).sum()) * 2 // 3]
        free[: len(left)] = left
        s.update(free=gpu(free), free_count=gpu(np.array([len(left)])))
        if case["op"] == "extend":
            s.update(new_lens=gpu(second), max_tokens=int(second.sum()) + 3)
        else:
            s.update(keep=gpu(second))
        return s
    heads, dim, store, dtype = case["kv_heads"], case["dim"], case["store"], DTYPES[case["dtype"]]
    scales = 2.0 ** (torch.rand((blocks, heads, 2), device="cuda", generator=g) * 2 - 1) * (3.5 / TOP[store])
    s.update(store=store, k_pool=_codes((blocks, heads, page, dim), store, g),
             v_pool=_codes((blocks, heads, page, dim), store, g), kv_scales=scales)
    if case["op"] == "decode":
        s["q"] = torch.randn((n, case["q_heads"], dim), device="cuda", generator=g).to(dtype)
        return s
    row = np.repeat(np.arange(n), second)
    pos = lens[row] + np.arange(len(row)) - np.repeat(np.cumsum(second) - second, second)
    slots = table[row, pos // page].astype(np.int64) * page + pos % page
    slots = np.concatenate([slots, np.full(case["pad"], -1)])
    for name in ("k_new", "v_new"):
        s[name] = torch.randn((len(slots), heads, dim), device="cuda", generator=g).to(dtype)
    s["slots"] = gpu(slots)
    return s


# ---- the operators in elementary operations --------------------------------------------------------------------

def _extend_plain(s):
    table, page, free, limit = s["table"], s["page"], s["free"], s["max_tokens"]
    lens, new, count = s["lens"].long(), s["new_lens"].long(), s["free_count"].long()
    n, width = table.shape
    held = (lens + page - 1) // page
    end = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(end[:1]), end])
    fits = (lens + new <= width * page) & (end <= limit)
    ask = torch.where(fits, (lens + new + page - 1) // page - held, 0)
    upto = torch.cumsum(ask, 0)
    granted = fits & ((ask == 0) | (upto <= count))
    got = torch.where(granted, ask, 0)
    col = torch.arange(width, device=table.device)
    fresh = (col >= held[:, None]) & (col < (held + got)[:, None])
    pick = count - 1 - ((upto - ask - held)[:, None] + col)
    table.copy_(torch.where(fresh, free[pick.clamp(0, free.shape[0] - 1)], table))
    token = torch.arange(limit, device=table.device)
    seq = torch.searchsorted(end, token, right=True).clamp(max=n - 1)
    pos = lens[seq] + token - starts[seq]
    live = (token < end[-1]) & granted[seq]
    block = table[seq, (pos // page).clamp(0, width - 1)].long()
    slots = torch.where(live, block * page + pos % page, -1)
    total = torch.where(granted, lens + new, lens)
    return dict(block_table=table, slots=slots.int(), starts=starts.int(), lens=total.int(),
                free_count=(count - got.sum()).int())


def _trim_plain(s):
    table, page, free = s["table"], s["page"], s["free"]
    lens, count = s["lens"].long(), s["free_count"].long()
    keep = torch.minimum(s["keep"].long(), lens)
    held, left = (lens + page - 1) // page, (keep + page - 1) // page
    gone = held - left
    upto = torch.cumsum(gone, 0)
    col = torch.arange(table.shape[1], device=table.device)
    out = (col >= left[:, None]) & (col < held[:, None])
    at = torch.where(out, count + (upto - gone - left)[:, None] + col, free.shape[0])
    wide = torch.cat([free, free[:1]])
    wide.scatter_(0, at.reshape(-1), table.reshape(-1))
    free.copy_(wide[:-1])
    return dict(free_blocks=free, lens=keep.int(), free_count=(count + upto[-1]).int())


def _rounded(x, store):
    """float64 values to the nearest codes of the storage type, ties to even."""
    top = TOP[store]
    if store == "int8":
        return torch.round(x).clamp(-top, top).to(torch.int8)
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-top, top).float().to(torch.float8_e4m3fn)


def _append_one(pool, scales, which, x, slots, page, store):
    live = slots >= 0
    x, slots = x[live].double(), slots[live].long()
    blocks, of = torch.unique(slots // page, return_inverse=True)
    row = slots % page
    heads = pool.shape[1]
    first = torch.full_like(blocks, page).scatter_reduce(0, of, row, "amin")
    top = torch.zeros((len(blocks), heads), dtype=torch.float64, device=x.device)
    top = top.scatter_reduce(0, of[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    old = torch.where(first[:, None] > 0, scales[blocks, :, which], 0.0)
    scale = torch.maximum(old, (top / torch.full_like(top, TOP[store])).float())
    by = torch.where(scale > 0, scale, 1.0).double()
    held = pool[blocks]
    again = _rounded(held.double() * old.double()[:, :, None, None] / by[:, :, None, None], store)
    kept = (torch.arange(page, device=x.device) < first[:, None])[:, None, :, None]
    # (8-bit floats have no where(): their bytes are chosen)
    pool[blocks] = torch.where(kept, again.view(torch.int8), held.view(torch.int8)).view(pool.dtype)
    head = torch.arange(heads, device=x.device)
    pool[(slots // page)[:, None], head, row[:, None]] = _rounded(x / by[of][:, :, None], store)
    scales[blocks, :, which] = scale


def _append_plain(s):
    for_one = (s["slots"], s["page"], s["store"])
    _append_one(s["k_pool"], s["kv_scales"], 0, s["k_new"], *for_one)
    _append_one(s["v_pool"], s["kv_scales"], 1, s["v_new"], *for_one)
    return dict(k_pool=s["k_pool"], v_pool=s["v_pool"], kv_scales=s["kv_scales"])


def _values(pool, scale, table):
    """The rows a block table names, as float32 [B, Hkv, tokens, D]."""
    rows = pool[table].float() * scale[table][..., None, None]
    n, width, heads, page, dim = rows.shape
    return rows.transpose(1, 2).reshape(n, heads, width * page, dim)


def _decode_plain(s):
    table, scales, q = s["table"].long(), s["kv_scales"], s["q"]
    n, q_heads, dim = q.shape
    k = _values(s["k_pool"], scales[..., 0], table)
    grouped = q.float().reshape(n, k.shape[1], -1, dim)
    score = grouped @ k.transpose(2, 3) / math.sqrt(dim)
    dead = (torch.arange(k.shape[2], device=q.device) >= s["lens"][:, None])[:, None, None, :]
    del k
    score = score.masked_fill(dead, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = weight @ _values(s["v_pool"], scales[..., 1], table) / torch.where(total > 0, total, 1.0)
    return dict(out=out.reshape(n, q_heads, dim).to(q.dtype))


def run(state):
    s = state
    if own:
        import fusedtok_b200 as ft
        if s["op"] == "extend":
            step = ft.block_table_extend(s["table"], s["lens"], s["new_lens"], s["free"], s["free_count"], s["page"],
                                         s["max_tokens"])
            return dict(block_table=s["table"], slots=step.slots, starts=step.starts, lens=step.lens,
                        free_count=step.free_count)
        if s["op"] == "trim":
            lens, count = ft.block_table_trim(s["table"], s["lens"], s["keep"], s["free"], s["free_count"], s["page"])
            return dict(free_blocks=s["free"], lens=lens, free_count=count)
        if s["op"] == "append":
            ft.kv_append_paged_q8(s["k_pool"], s["v_pool"], s["kv_scales"], s["k_new"], s["v_new"], s["slots"])
            return dict(k_pool=s["k_pool"], v_pool=s["v_pool"], kv_scales=s["kv_scales"])
        return dict(out=ft.attention_decode_paged_q8(s["q"], s["k_pool"], s["v_pool"], s["kv_scales"], s["table"],
                                                     s["lens"]))
    return {"extend": _extend_plain, "trim": _trim_plain, "append": _append_plain, "decode": _decode_plain}[s["op"]](s)


# ---- work ------------------------------------------------------------------------------------------------------

def work(case):
    lens, second = _lengths(case)
    page, n = case["page"], case["batch"]
    if case["op"] == "extend":
        tokens = int(second.sum())
        fresh = int((_pages(lens + second, page) - _pages(lens, page)).sum())
        # lengths in and out, starts, free blocks read and written into the table, the slot map
        return {"bytes": 4 * (4 * n + 2 * fresh + tokens), "flops": 0}
    if case["op"] == "trim":
        gone = int((_pages(lens, page) - _pages(second, page)).sum())
        return {"bytes": 4 * (3 * n + 2 * gone), "flops": 0}
    heads, dim = case["kv_heads"], case["dim"]
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "append":
        tokens = int(second.sum())
        touched = int((_pages(lens + second, page) - lens // page)[second > 0].sum())
        return {"bytes": 2 * tokens * heads * dim * (size + 1) + 16 * touched * heads + 4 * tokens, "flops": 0}
    tokens, blocks = int(lens.sum()), int(_pages(lens, page).sum())
    return {"bytes": 2 * tokens * heads * dim + 8 * blocks * heads + 4 * blocks + 4 * n + 2 * n * case["q_heads"] * dim * size,
            "flops": 4 * tokens * case["q_heads"] * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def _near(x, store):
    """The code nearest to each float64 value: for 8-bit floats by the spacing 2^(e - 3) of the binade, e >= -6."""
    if store == "int8":
        return torch.round(x).clamp(-127, 127)
    size = x.abs()
    e = torch.floor(torch.log2(size.clamp_min(2.0 ** -9)))
    e = torch.where(2.0 ** (e + 1) <= size, e + 1, torch.where(2.0 ** e > size, e - 1, e)).clamp_min(-6)
    gap = 2.0 ** (e - 3)
    return (torch.round(x / gap) * gap).clamp(-448, 448)


def exact(case, seed):
    if case["op"] in ("extend", "trim"):
        return None                                     # whole numbers only
    s = prepare(case, seed)
    page, store = case["page"], case["store"]
    if case["op"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["q_heads"] // case["kv_heads"]
        for b, length in enumerate(s["lens"].tolist()):
            if not length:
                continue
            ids = s["table"][b, : _pages(length, page)].long()
            for h in range(case["kv_heads"]):
                k, v = (s[name][ids, h].to(torch.float32).double() * s["kv_scales"][ids, h, which].double()[:, None, None]
                        for which, name in enumerate(("k_pool", "v_pool")))
                k, v = (x.reshape(-1, case["dim"])[:length] for x in (k, v))
                mine = slice(h * group, (h + 1) * group)
                p = torch.softmax(s["q"][b, mine].double() @ k.T * case["dim"] ** -0.5, dim=-1)
                out[b, mine] = p @ v
        return dict(out=out)
    slots = s["slots"].long()
    live = slots >= 0
    at = slots[live]
    block, row = at // page, at % page
    pools, scales = [], s["kv_scales"].double()
    blocks = scales.shape[0]
    begin = torch.full((blocks,), page, device="cuda").index_reduce_(0, block, row, "amin")
    new = torch.zeros((blocks, page), dtype=torch.bool, device="cuda").index_put_((block, row), torch.ones_like(at, dtype=torch.bool))
    touched = new.any(1)
    for which, name in enumerate(("k_pool", "v_pool")):
        x = s[name[0] + "_new"][live]
        code = s[name].float()
        for h in range(case["kv_heads"]):
            held = torch.where(begin > 0, scales[:, h, which], 0)
            big = torch.zeros(blocks, dtype=torch.float64, device="cuda").index_reduce_(0, block, x[:, h].double().abs().amax(-1), "amax")
            most = torch.maximum(held, (big / TOP[store]).float().double())
            most = torch.where(touched, most, scales[:, h, which])
            was = code[:, h].double() * held[:, None, None]
            was[block, row] = x[:, h].double()
            # rows before the call's first one are rounded again, rows behind its last one stay
            change = touched[:, None] & (new | (torch.arange(page, device="cuda") < begin[:, None]))
            got = _near(was / torch.where(most > 0, most, 1.0)[:, None, None], store)
            code[:, h] = torch.where(change[:, :, None], got, code[:, h].double()).float()
            scales[:, h, which] = most
        pools.append(code.double() if store == "e4m3" else None)
    return dict(k_pool=pools[0], v_pool=pools[1], kv_scales=scales)
