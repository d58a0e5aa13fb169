"""The paged cache held in 8 bits and its block tables: refusals on the CPU, results on the GPU against plain 64-bit
implementations (q8_reference.py)."""

import numpy as np
import pytest
import torch

import q8_reference as ref

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {"f32": 2.0 ** -21, "bf16": 2.0 ** -11, "f16": 2.0 ** -11}       # rounding of a weight on its way to the tensor cores
STORES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def ft():
    import fusedtok_b200
    return fusedtok_b200


def on_gpu(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(dtype) if dtype else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def pool(codes, store):
    """uint8 codes as a CUDA pool of the code type."""
    return torch.from_numpy(codes).cuda().view(STORES[store])


def codes_of(t):
    return t.view(torch.uint8).cpu().numpy()


def random_codes(rng, shape, store):
    if store == "int8":
        return rng.integers(-127, 128, shape).astype(np.int8).view(np.uint8)
    return ref.nearest_codes(rng.standard_normal(shape) * 120, store)


def make_cache(rng, lens, hkv, dim, page, store, spare=3, spread=3.0):
    """Pools, scales and a table of distinct blocks in random order; scales differ by up to 2^spread between blocks."""
    need = [-(-n // page) for n in lens]
    blocks = sum(need) + spare
    perm = rng.permutation(blocks).astype(np.int32)
    width = max(1, max(need, default=1)) + 1
    table = np.zeros((len(lens), width), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    k, v = (random_codes(rng, (blocks, hkv, page, dim), store) for _ in range(2))
    unit = 1.7 / ref.TOP[store]
    scales = (unit * 2.0 ** rng.uniform(-spread / 2, spread / 2, (blocks, hkv, 2))).astype(np.float32)
    return k, v, scales, table


def rounded(x, name):
    """float64 values in the storage type, as a tensor."""
    return torch.from_numpy(np.asarray(x, np.float32)).to(DTYPES[name])


def check_decode(q, k, v, scales, table, lens, store, name, **kw):
    got = ft().attention_decode_paged_q8(q.cuda(), pool(k, store), pool(v, store), on_gpu(scales), on_gpu(table),
                                         None if lens is None else on_gpu(np.asarray(lens, np.int32)), **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    full = [table.shape[1] * k.shape[2]] * len(q) if lens is None else lens
    want, bound = ref.decode(q.double().numpy(), k, v, scales, table, full, store, STEP[name])
    # the result is rounded once to its type: half a step
    tol = bound + (np.abs(want) + bound) * torch.finfo(q.dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), (float((err / np.maximum(tol, 1e-300)).max()), float(err.max()))
    return got


# ---- refusals (no GPU) -----------------------------------------------------------------------------------------

def test_host_tensors_are_refused():
    k = torch.zeros((4, 2, 16, 64), dtype=torch.int8)
    scales = torch.zeros((4, 2, 2))
    with pytest.raises(TypeError):
        ft().attention_decode_paged_q8(torch.zeros((1, 4, 64)), k, k, scales, torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(TypeError):
        ft().kv_append_paged_q8(k, k, scales, torch.zeros((1, 2, 64)), torch.zeros((1, 2, 64)), [0])
    i = torch.zeros((1,), dtype=torch.int32)
    with pytest.raises(TypeError):
        ft().block_table_extend(i[None], i, i, i, i, 16, 4)
    with pytest.raises(TypeError):
        ft().block_table_trim(i[None], i, i, i, i, 16)


def test_launchers_refuse_before_touching_the_gpu():
    from fusedtok_b200 import _fusedtok as lib
    good = dict(dtype=1, store=0, q=64, k_pool=64, v_pool=64, kv_scales=64, table=64, lens=64, out=64, workspace=0,
                workspace_bytes=0, batch=1, hq=8, hkv=2, page=16, tbl_width=4, num_blocks=8, dim=64)
    for change in (dict(dtype=3), dict(store=2), dict(batch=-1), dict(hq=7), dict(hkv=0), dict(dim=66), dict(dim=516),
                   dict(page=0), dict(tbl_width=-1), dict(page=1 << 20, tbl_width=1 << 20), dict(num_blocks=-1), dict(q=0),
                   dict(out=0), dict(k_pool=0), dict(kv_scales=0), dict(table=0), dict(q=66), dict(out=68), dict(k_pool=66),
                   dict(kv_scales=68)):
        with pytest.raises(ValueError):
            lib.attention_decode_paged_q8_launch(**{**good, **change})
    lib.attention_decode_paged_q8_launch(**{**good, "batch": 0})
    good = dict(dtype=1, store=0, k_new=64, v_new=64, slots=64, k_pool=64, v_pool=1 << 20, kv_scales=64, tokens=1, hkv=2, dim=64,
                page=16, num_blocks=8)
    for change in (dict(dtype=-1), dict(store=5), dict(tokens=-1), dict(hkv=0), dict(dim=2), dict(dim=1024), dict(page=0),
                   dict(num_blocks=1 << 28), dict(k_new=0), dict(slots=0), dict(kv_scales=0), dict(k_new=68), dict(v_pool=65),
                   dict(v_pool=64), dict(v_pool=64 + 8 * 2 * 16 * 64 - 4)):
        with pytest.raises(ValueError):
            lib.kv_append_paged_q8_launch(**{**good, **change})
    lib.kv_append_paged_q8_launch(**{**good, "tokens": 0})
    good = dict(table=64, lens=64, new_lens=64, free_blocks=64, free_count=64, slots=64, starts=64, lens_out=64,
                free_count_out=64, batch=2, tbl_width=4, page=16, free_capacity=8, max_tokens=4)
    for change in (dict(batch=-1), dict(batch=8193), dict(page=0), dict(page=1 << 20, tbl_width=1 << 20), dict(max_tokens=-1),
                   dict(table=0), dict(lens=0), dict(free_blocks=0), dict(slots=0), dict(free_count_out=0)):
        with pytest.raises(ValueError):
            lib.block_table_extend_launch(**{**good, **change})
    good = dict(table=64, lens=64, keep_lens=64, free_blocks=64, free_count=64, lens_out=64, free_count_out=64, batch=2,
                tbl_width=4, page=16, free_capacity=8)
    for change in (dict(batch=8193), dict(page=-3), dict(free_capacity=-1), dict(keep_lens=0), dict(lens_out=0)):
        with pytest.raises(ValueError):
            lib.block_table_trim_launch(**{**good, **change})


def test_append_refuses_blocks_beyond_32_bits():
    from fusedtok_b200 import _fusedtok as lib
    good = dict(dtype=1, store=0, k_new=64, v_new=64, slots=64, k_pool=64, v_pool=1 << 45, kv_scales=64, tokens=1, hkv=1, dim=64,
                page=1 << 25, num_blocks=1)
    with pytest.raises(ValueError, match="below 2\\^31 bytes"):
        lib.kv_append_paged_q8_launch(**good)


def test_module_of_another_torch_is_left_alone(monkeypatch):
    """The module for plain calls binds to the torch it was built for; under another one every call takes the wrappers' way."""
    f = ft()
    if f._tensors is None:
        pytest.skip("not built")
    assert f._tensors.torch_version == torch.__version__.split("+")[0]
    import importlib.util
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    spec = importlib.util.spec_from_file_location("fusedtok_b200", f.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    assert again._tensors is None
    assert again._decode_q8_native(1, 2, 3, 4, 5, 6) is None


def test_workspace_of_a_refused_shape():
    from fusedtok_b200 import _fusedtok as lib
    with pytest.raises(ValueError):
        lib.attention_decode_paged_q8_workspace(0, 1, 5, 2, 16, 4, 64)
    assert lib.attention_decode_paged_q8_workspace(0, 0, 4, 2, 16, 4, 64) == 0


def test_host_slots_are_checked():
    check = ft()._host_slots
    assert check([3, -7, 17, 18], 4, 2, 16).tolist() == [3, -1, 17, 18]
    assert check([14, 15, 16, 17], 4, 2, 16).tolist() == [14, 15, 16, 17]       # two blocks, one run in each
    for bad in ([32], [1, 2, 4], [2, 1], [5, 5], [0, 16, 1], [0, -1, 1]):
        with pytest.raises(ValueError):
            check(bad, len(bad), 2, 16)
    with pytest.raises(ValueError):
        check([1, 2], 3, 2, 16)
    with pytest.raises(TypeError):
        check([0.5], 1, 2, 16)


def test_reference_rounding():
    """The oracle's own rounding, against the definition: no code is nearer, and ties go to the even one."""
    rng = np.random.default_rng(0)
    for store in STORES:
        every = np.unique(ref.decode_codes(np.arange(256, dtype=np.uint8), store))
        every = every[np.isfinite(every) & (np.abs(every) <= ref.TOP[store])]
        x = np.concatenate([rng.uniform(-130, 130, 2000), rng.standard_normal(2000) * 0.01, (every[1:] + every[:-1]) / 2, every])
        got = ref.decode_codes(ref.nearest_codes(x, store), store)
        best = np.abs(every[None] - x[:, None]).min(1)
        capped = np.abs(x) > ref.TOP[store]
        assert (np.abs(got - x)[~capped] == best[~capped]).all()
        ties = ref.nearest_codes((every[1:] + every[:-1]) / 2, store)
        assert (ties % 2 == 0).all()


# ---- decode ----------------------------------------------------------------------------------------------------

SHAPES = [
    # B, Hq, Hkv, D, P, lens
    (1, 8, 8, 64, 16, [512]),
    (1, 1, 1, 128, 16, [1]),
    (2, 4, 1, 128, 16, [1, 4097]),
    (3, 8, 2, 128, 16, [0, 63, 65]),
    (4, 40, 8, 128, 16, [100, 0, 1000, 17]),           # five heads a group
    (2, 16, 2, 128, 32, [777, 64]),
    (2, 32, 2, 128, 64, [300, 129]),                   # sixteen
    (2, 48, 2, 64, 128, [300, 1]),                     # twenty-four: several units per kv head
    (3, 6, 2, 256, 16, [515, 16, 15]),
    (2, 12, 1, 256, 64, [130, 2049]),
    (2, 6, 2, 80, 16, [211, 48]),
    (2, 14, 2, 96, 32, [95, 640]),
    (1, 8, 1, 192, 128, [383]),
    (5, 4, 4, 64, 1024, [5, 1025, 0, 2048, 1023]),     # blocks of many tiles
    # other kernels' ground: small, odd and unaligned blocks and head dims
    (2, 6, 3, 4, 16, [33, 7]),
    (2, 8, 2, 20, 5, [33, 7]),
    (3, 5, 1, 128, 8, [90, 0, 1]),
    (2, 4, 2, 128, 1, [70, 3]),
    (2, 9, 3, 64, 24, [500, 49]),
    (1, 4, 2, 512, 16, [300]),
    (2, 2, 1, 260, 48, [100, 999]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
def test_decode(shape, name, store):
    b, hq, hkv, d, page, lens = shape
    rng = np.random.default_rng(b * 1000 + hq * 31 + hkv * 7 + d + page)
    k, v, scales, table = make_cache(rng, lens, hkv, d, page, store)
    q = rounded(rng.standard_normal((b, hq, d)), name)
    got = check_decode(q, k, v, scales, table, lens, store, name)
    for i, n in enumerate(lens):
        if n == 0:
            assert not got[i].any()
    if b and all(lens):
        check_decode(q, k, v, scales, table[:, : min(-(-n // page) for n in lens)], None, store, name)


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
@pytest.mark.parametrize("page,dim", [(16, 128), (64, 64), (12, 96)])
def test_decode_large_batch(page, dim, store):
    """More sequences than the schedule's table holds, and than there are SMs, many of them empty."""
    rng = np.random.default_rng(5)
    for batch in (300, 2100):
        lens = rng.integers(0, 40, batch) * (rng.random(batch) < 0.7)
        k, v, scales, table = make_cache(rng, lens.tolist(), 1, dim, page, store)
        q = rounded(rng.standard_normal((batch, 3, dim)), "f16")
        check_decode(q, k, v, scales, table, lens.tolist(), store, "f16")


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,dim,page,lens", [(16, 1, 128, 16, [6007]), (13, 1, 128, 16, [2500, 0, 700]), (8, 1, 256, 32, [4001]),
                                                  (24, 1, 96, 16, [3000]), (6, 2, 112, 16, [2300]), (9, 1, 512, 16, [1500, 40])])
def test_decode_few_units_of_many_heads(hq, hkv, dim, page, lens):
    """Units cut into many ranges (more than 32, or not) whose merge several blocks share; last chunks of a group with fewer heads."""
    rng = np.random.default_rng(hq * dim)
    k, v, scales, table = make_cache(rng, lens, hkv, dim, page, "e4m3")
    check_decode(rounded(rng.standard_normal((len(lens), hq, dim)), "f16"), k, v, scales, table, lens, "e4m3", "f16")


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(16, 128), (64, 64), (12, 96), (32, 256)])
def test_decode_ignores_what_is_behind_the_end(page, dim):
    """NaN codes, infinite and NaN scales and out-of-range table entries behind the last token change nothing."""
    rng = np.random.default_rng(6)
    lens = [page * 2 + 5, 0, 1, page * 5, 70]
    k, v, scales, table = make_cache(rng, lens, 2, dim, page, "e4m3")
    q = rounded(rng.standard_normal((5, 8, dim)), "f32")
    args = lambda: (q.cuda(), pool(k, "e4m3"), pool(v, "e4m3"), on_gpu(scales), on_gpu(table), on_gpu(np.array(lens, np.int32)))  # noqa: E731
    clean = ft().attention_decode_paged_q8(*args())
    used = np.zeros(len(k), bool)
    for b, n in enumerate(lens):
        blocks = -(-n // page)
        used[table[b, :blocks]] = True
        if n % page:
            k[table[b, blocks - 1], :, n % page:] = 0x7f
            v[table[b, blocks - 1], :, n % page:] = 0xff
        table[b, blocks:] = rng.choice([-1, 2 ** 30, -2 ** 31, len(k)], table.shape[1] - blocks)
    k[~used], v[~used] = 0x7f, 0x7f
    scales[~used] = [np.nan, np.inf]
    dirty = ft().attention_decode_paged_q8(*args())
    assert torch.equal(clean, dirty) and torch.isfinite(dirty).all()


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 12)])
def test_decode_scales_of_any_size(dim, page, store):
    """Scales that differ by many powers of two between the blocks of a sequence, zero among them, and queries from tiny
    to large: the weights are rounded relative to the largest contribution, not to the largest weight."""
    rng = np.random.default_rng(7)
    lens = [page * 9 + 3, page * 30]
    k, v, scales, table = make_cache(rng, lens, 2, dim, page, store)
    scales[..., 1] *= 2.0 ** rng.integers(-25, 26, scales[..., 1].shape)
    scales[::5, 0, 1] = 0
    scales[1::7, 1, 0] = 0
    q = rng.standard_normal((2, 8, dim))
    q[0, 0] *= 1e-30
    q[1, 3] *= 40
    q[1, 5] = 0
    for name in ("f32", "bf16"):
        check_decode(rounded(q, name), k, v, scales, table, lens, store, name)


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 64)])
@pytest.mark.parametrize("big", [2.0 ** 40, 2.0 ** -40])
def test_decode_blocks_of_zeros(dim, page, store, big):
    """Blocks of zeros (scale 0) at the head of a sequence and all over it, among blocks of very large or very small values."""
    rng = np.random.default_rng(17)
    lens = [page * 20 + 3, page * 3, page * 2 + 1]
    k, v, scales, table = make_cache(rng, lens, 2, dim, page, store)
    scales[..., 1] *= np.float32(big)
    scales[table[0, :8], :, 1] = 0
    scales[table[1, :3], :, 1] = 0
    scales[table[2, 1:], 0, 1] = 0
    q = rounded(rng.standard_normal((3, 8, dim)), "f32")
    got = check_decode(q, k, v, scales, table, lens, store, "f32")
    assert not got[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 12)])
def test_decode_nan_stays_in_its_heads(dim, page):
    rng = np.random.default_rng(8)
    lens = [400, 333, 90]
    k, v, scales, table = make_cache(rng, lens, 2, dim, page, "int8")
    q = rounded(rng.standard_normal((3, 8, dim)), "bf16")
    clean = check_decode(q, k, v, scales, table, lens, "int8", "bf16")
    q[0, 2, 5] = float("nan")
    q[1, 7, 0] = float("inf")
    scales[table[2, 1], 0, 1] = np.nan
    scales[table[1, 0], 1, 0] = np.nan
    got = ft().attention_decode_paged_q8(q.cuda(), pool(k, "int8"), pool(v, "int8"), on_gpu(scales), on_gpu(table),
                                         on_gpu(np.array(lens, np.int32)))
    bad = torch.zeros((3, 8), dtype=torch.bool)
    bad[0, 2] = bad[1, 4:] = bad[2, :4] = True
    assert torch.isnan(got.cpu()).all(-1).equal(bad)
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])


@pytest.mark.gpu
def test_decode_no_rows_and_no_sequences():
    rng = np.random.default_rng(9)
    k, v, scales, table = make_cache(rng, [16], 2, 64, 16, "int8")
    q = torch.ones((1, 4, 64), device="cuda")
    a = (pool(k, "int8"), pool(v, "int8"), on_gpu(scales))
    assert not ft().attention_decode_paged_q8(q, *a, on_gpu(table[:, :0])).any()
    assert not ft().attention_decode_paged_q8(q, *a, on_gpu(table), on_gpu(np.array([0], np.int32))).any()
    assert ft().attention_decode_paged_q8(q[:0], *a, on_gpu(table[:0])).shape == (0, 4, 64)


@pytest.mark.gpu
def test_decode_refusals():
    rng = np.random.default_rng(10)
    k, v, scales, table = make_cache(rng, [64, 64], 2, 64, 16, "int8")
    q, kp, vp, s, t = torch.zeros((2, 4, 64), device="cuda"), pool(k, "int8"), pool(v, "int8"), on_gpu(scales), on_gpu(table)
    run = ft().attention_decode_paged_q8
    run(q, kp, vp, s, t)
    for bad in ((q.double(), kp, vp, s, t), (q, kp.float(), vp, s, t), (q, kp, vp.view(torch.float8_e4m3fn), s, t),
                (q, kp, vp, s.half(), t), (q, kp.cpu(), vp, s, t), (q, kp, vp, s, t, [0.5, 1.0]),
                (q, kp, vp, s, t, torch.ones(2, device="cuda")), (q, kp, vp, s, t.bool())):
        with pytest.raises(TypeError):
            run(*bad)
    for bad in ((q[:, :3], kp, vp, s, t), (q[..., :60].contiguous(), kp, vp, s, t), (q, kp, vp[:-1], s, t), (q, kp, vp, s[:-1], t),
                (q, kp[0], vp[0], s, t), (q, kp, vp, s, t[:1]), (q, kp, vp, s, t, [1, 2, 3]), (q, kp, vp, s, t, [999, 0]),
                (q, kp, vp, s, t.cpu() + 99), (q.transpose(0, 1), kp, vp, s, t), (q, kp, vp, s.transpose(0, 1).contiguous().transpose(0, 1), t)):
        with pytest.raises(ValueError):
            run(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [4, 8])
def test_decode_unaligned_pools(shift):
    """Pools that begin 4 or 8 bytes behind a 16-byte boundary run on the generic kernel; odd addresses are refused."""
    rng = np.random.default_rng(11)
    lens = [100, 37]
    k, v, scales, table = make_cache(rng, lens, 2, 128, 16, "int8")
    q = rounded(rng.standard_normal((2, 8, 128)), "bf16")

    def moved(codes, by):
        room = torch.zeros(codes.size + 64, dtype=torch.int8, device="cuda")
        view = room[by:by + codes.size].view(codes.shape)
        view.copy_(pool(codes, "int8"))
        return view
    want, bound = ref.decode(q.double().numpy(), k, v, scales, table, lens, "int8", STEP["bf16"])
    got = ft().attention_decode_paged_q8(q.cuda(), moved(k, shift), moved(v, shift), on_gpu(scales), on_gpu(table),
                                         on_gpu(np.array(lens, np.int32)))
    tol = bound + (np.abs(want) + bound) * 2.0 ** -8
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    with pytest.raises(ValueError):
        ft().attention_decode_paged_q8(q.cuda(), moved(k, 2), moved(v, 2), on_gpu(scales), on_gpu(table))


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(16, 128), (20, 128)])
def test_decode_blocks_far_into_a_large_pool(page, dim):
    """Blocks behind 2^32 bytes of pool."""
    rng = np.random.default_rng(12)
    hkv = 8
    blocks = (5 << 30) // (hkv * page * dim)
    k, v, scales, table = make_cache(rng, [page * 6 + 1, 40], hkv, dim, page, "int8", spare=0)
    n = len(k)
    where = np.sort(rng.choice(np.arange(blocks - 4 * n, blocks), n, replace=False))
    kp = torch.zeros((blocks, hkv, page, dim), dtype=torch.int8, device="cuda")
    vp, s = torch.zeros_like(kp), torch.zeros((blocks, hkv, 2), device="cuda")
    for i, w in enumerate(where):
        kp[w], vp[w], s[w] = pool(k[i], "int8"), pool(v[i], "int8"), on_gpu(scales[i])
    far = where[table].astype(np.int32)
    q = rounded(rng.standard_normal((2, 32, dim)), "f16")
    lens = np.array([page * 6 + 1, 40], np.int32)
    near = ft().attention_decode_paged_q8(q.cuda(), pool(k, "int8"), pool(v, "int8"), on_gpu(scales), on_gpu(table), on_gpu(lens))
    got = ft().attention_decode_paged_q8(q.cuda(), kp, vp, s, on_gpu(far), on_gpu(lens))
    assert torch.equal(near, got)
    new = rounded(rng.standard_normal((1, hkv, dim)), "bf16").cuda()
    slot = int(far[0, 6]) * page + 1
    ft().kv_append_paged_q8(kp, vp, s, new, new, torch.tensor([slot], dtype=torch.int64, device="cuda"))
    want_k, want_s = k[table[0, 6]][None].copy(), scales[table[0, 6]][None].copy()
    ref.append(want_k, want_s, 0, new.double().cpu().numpy(), [1], page, "int8")
    assert (codes_of(kp[far[0, 6]].contiguous()) == want_k[0]).all()


# ---- append ----------------------------------------------------------------------------------------------------

def slots_of(table, lens, new, page):
    return np.array([table[b, (lens[b] + j) // page] * page + (lens[b] + j) % page
                     for b in range(len(lens)) for j in range(new[b])], np.int64)


def check_append(k, v, scales, k_new, v_new, slots, page, store, as_host=False):
    kp, vp, s = pool(k.copy(), store), pool(v.copy(), store), on_gpu(scales.copy())
    where = slots if as_host else on_gpu(np.asarray(slots, np.int32))
    assert ft().kv_append_paged_q8(kp, vp, s, k_new.cuda(), v_new.cuda(), where) is None
    k, v, scales = k.copy(), v.copy(), scales.copy()
    ref.append(k, scales, 0, k_new.double().numpy(), slots, page, store)
    ref.append(v, scales, 1, v_new.double().numpy(), slots, page, store)
    got = s.cpu().numpy()
    assert ((got == scales) | (np.isnan(got) & np.isnan(scales))).all()
    assert (codes_of(kp) == k).all(), (codes_of(kp) != k).mean()
    assert (codes_of(vp) == v).all(), (codes_of(vp) != v).mean()
    return kp, vp, s


APPENDS = [
    # Hkv, D, P, lens, new
    (8, 128, 16, [5, 16, 0, 31, 100], [1, 1, 1, 1, 1]),
    (8, 128, 64, [5, 64, 0, 31, 100], [1, 1, 1, 1, 1]),
    (2, 64, 16, [0, 3, 15], [50, 13, 40]),
    (1, 128, 16, [0], [1]),
    (2, 256, 128, [100, 7], [300, 5]),
    (4, 80, 32, [9, 0, 33], [0, 70, 1]),
    (3, 4, 16, [9, 0], [20, 3]),
    (2, 20, 5, [9, 0], [20, 3]),
    (2, 12, 1, [2, 0], [3, 2]),
    (1, 512, 48, [40, 1], [60, 47]),
    (1, 128, 1024, [900, 0], [300, 1500]),
    (8, 64, 16, [7, 0, 130], [2000, 3000, 1500]),      # several runs per CTA
]


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "x".join(map(str, c[:3])) + "-" + str(sum(c[4])))
def test_append(case, name, store):
    """Codes and scales bit for bit."""
    hkv, dim, page, lens, new = case
    rng = np.random.default_rng(hkv * 100 + dim + page)
    k, v, scales, table = make_cache(rng, [a + b for a, b in zip(lens, new)], hkv, dim, page, store)
    slots = slots_of(table, lens, new, page)
    # rows from far below to far above what the blocks hold, so that some raise the scale and some do not
    x = rng.standard_normal((2, len(slots), hkv, dim)) * 2.0 ** rng.integers(-6, 4, (2, len(slots), hkv, 1))
    check_append(k, v, scales, rounded(x[0], name), rounded(x[1], name), slots, page, store)


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
@pytest.mark.parametrize("name", list(DTYPES))
def test_append_values_on_borders(name, store):
    """Values whose quotient lies exactly between two codes, and one unit in the last place to either side; scales from the
    smallest subnormal to large ones; zeros."""
    rng = np.random.default_rng(3)
    page, dim = 16, 128
    every = np.unique(np.abs(ref.decode_codes(np.arange(256, dtype=np.uint8), store)))
    every = every[np.isfinite(every) & (every <= ref.TOP[store])]
    ties = (every[1:] + every[:-1]) / 2
    tiny = [2.0 ** -149, 2.0 ** -140, 2.0 ** -126, 2.0 ** -110] if name != "f16" else [2.0 ** -24, 2.0 ** -14]
    rows = []
    for unit in [1.0, 2.0 ** -3, 2.0 ** 4, 0.7, 1.1, 3.3] + tiny:
        for _ in range(2):
            x = rng.choice(np.concatenate([ties, every]), dim) * unit * rng.choice([-1, 1], dim)
            x = np.asarray(rounded(x, name).double())
            move = np.asarray(rounded(x * (1 + torch.finfo(DTYPES[name]).eps * rng.integers(-1, 2, dim)), name).double())
            move[0] = ref.TOP[store] * unit
            rows.append(move)
    rows.append(np.zeros(dim))
    n = len(rows)
    x = rounded(np.array(rows)[:, None, :], name)
    k = random_codes(rng, (n, 1, page, dim), store)
    scales = np.full((n, 1, 2), 0.01, np.float32)
    check_append(k, k, scales, x, x.flip(0), np.arange(n) * page, page, store)
    # the same behind rows that the blocks hold already: codes are rounded again, from scales of every size
    scales[:, 0, 0] = 2.0 ** rng.uniform(-140, 3, n)
    scales[:, 0, 1] = 2.0 ** rng.integers(-8, 4, n)
    scales[3] = 0
    check_append(k, k, scales, x, x.flip(0), np.arange(n) * page + 7, page, store)


@pytest.mark.gpu
@pytest.mark.parametrize("store", list(STORES))
def test_append_what_is_not_finite(store):
    rng = np.random.default_rng(4)
    k, v, scales, table = make_cache(rng, [40] * 4, 2, 64, 16, store)
    lens, new = [5, 16, 0, 20], [1, 1, 18, 3]
    slots = slots_of(table, lens, new, 16)
    x = rng.standard_normal((len(slots), 2, 64))
    x[0, 1, 3] = np.nan
    x[1, 0, 63] = np.inf
    x[17, 0, 0] = -np.inf
    x = rounded(x, "f32")
    scales[table[3, 1], 1, 1] = np.nan                 # a block that is NaN already stays so ...
    kp, vp, s = check_append(k, v, scales, x, x.flip(1), slots, 16, store)
    # ... and its sequence reads NaN in the heads of that kv head, and only there
    out = ft().attention_decode_paged_q8(torch.ones((4, 2, 64), device="cuda"), kp, vp, s, on_gpu(table),
                                         on_gpu(np.array([a + b for a, b in zip(lens, new)], np.int32)))
    bad = np.isnan(s.cpu().numpy())
    for b in range(4):
        held = table[b, : -(-(lens[b] + new[b]) // 16)]
        for h in range(2):
            assert torch.isnan(out[b, h]).all().item() == bad[held, h].any()
            assert torch.isnan(out[b, h]).any().item() == bad[held, h].any()
    # begun again at offset 0, a block is clean
    again = rounded(rng.standard_normal((1, 2, 64)), "f32").cuda()
    ft().kv_append_paged_q8(kp, vp, s, again, again, [int(table[0, 0]) * 16])
    assert torch.isfinite(s[table[0, 0]]).all()


@pytest.mark.gpu
def test_append_passes_over_and_leaves():
    """Negative and out-of-range device slots are passed over; nothing but the run's rows, the rows before them in their
    block and the scales is written; host slots do the same."""
    rng = np.random.default_rng(5)
    k, v, scales, table = make_cache(rng, [64, 64], 2, 128, 16, "e4m3")
    slots = np.array([-1, table[0, 0] * 16 + 3, table[0, 0] * 16 + 4, -5, len(k) * 16, 2 ** 31 - 1, table[1, 2] * 16 + 15])
    x = rounded(rng.standard_normal((len(slots), 2, 128)) * 20, "bf16")
    check_append(k, v, scales, x, x.flip(0), slots, 16, "e4m3")
    slots[4:6] = -1
    check_append(k, v, scales, x, x.flip(0), slots, 16, "e4m3", as_host=True)
    kp, s = pool(k.copy(), "e4m3"), on_gpu(scales)
    ft().kv_append_paged_q8(kp, kp.clone(), s, x[:0].cuda(), x[:0].cuda(), [])
    assert (codes_of(kp) == k).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(DTYPES))
def test_append_unaligned(name):
    rng = np.random.default_rng(6)
    k, v, scales, table = make_cache(rng, [40], 2, 128, 16, "int8")
    slots = slots_of(table, [3], [30], 16)
    x = rounded(rng.standard_normal((30, 2, 128)), name)
    room = torch.zeros(x.numel() + 4, dtype=x.dtype, device="cuda")
    view = room[4:].view(x.shape)
    view.copy_(x)
    kp, vp, s = pool(k.copy(), "int8"), pool(v.copy(), "int8"), on_gpu(scales.copy())
    ft().kv_append_paged_q8(kp, vp, s, view, view, on_gpu(slots))
    kq, vq, t = pool(k.copy(), "int8"), pool(v.copy(), "int8"), on_gpu(scales.copy())
    ft().kv_append_paged_q8(kq, vq, t, x.cuda(), x.cuda(), on_gpu(slots))
    assert torch.equal(kp, kq) and torch.equal(vp, vq) and torch.equal(s, t)
    odd = torch.zeros(x.numel() + 4, dtype=x.dtype, device="cuda")[1:-3].view(x.shape)
    with pytest.raises(ValueError):
        ft().kv_append_paged_q8(kp, vp, s, odd, odd, on_gpu(slots))


@pytest.mark.gpu
def test_append_refusals():
    kp = torch.zeros((4, 2, 16, 64), dtype=torch.int8, device="cuda")
    vp = kp.clone()
    s, x = torch.zeros((4, 2, 2), device="cuda"), torch.zeros((3, 2, 64), device="cuda")
    run = ft().kv_append_paged_q8
    run(kp, kp.clone(), s, x, x, [0, 1, 2])
    for bad in ((kp, vp, s, x.cpu(), x, [0, 1, 2]), (kp, vp, s, x, x.half(), [0, 1, 2]), (kp, vp, s, x.double(), x.double(), [0, 1, 2]),
                (kp.short(), vp.short(), s, x, x, [0, 1, 2]), (kp, vp, s, x, x, [0.0, 1.0, 2.0]),
                (kp, vp, s, x, x, torch.zeros(3, device="cuda"))):
        with pytest.raises(TypeError):
            run(*bad)
    for bad in ((kp, kp, s, x, x, [0, 1, 2]), (kp, vp, s, x, x[:2], [0, 1, 2]), (kp, vp, s, x[:, :1].contiguous(), x[:, :1].contiguous(), [0, 1, 2]),
                (kp, vp, s, x, x, [0, 1]), (kp, vp, s, x, x, [0, 1, 64]), (kp, vp, s, x, x, [0, 1, 1]),
                (kp, vp, s[:2], x, x, [0, 1, 2]), (kp, vp[..., :32].contiguous(), s, x, x, [0, 1, 2]),
                (kp, vp, s, x.transpose(0, 1), x, [0, 1, 2])):
        with pytest.raises(ValueError):
            run(*bad)


# ---- block tables ----------------------------------------------------------------------------------------------

def run_extend(table, lens, new, free, count, page, limit):
    t, f = on_gpu(table.copy()), on_gpu(free.copy())
    step = ft().block_table_extend(t, on_gpu(np.asarray(lens, np.int32)), on_gpu(np.asarray(new, np.int32)), f,
                                   on_gpu(np.array([count], np.int32)), page, limit)
    want = table.copy()
    slots, starts, left, rest = ref.extend(want, lens, new, free, count, page, limit)
    assert (t.cpu().numpy() == want).all()
    assert (f.cpu().numpy() == free).all()
    assert (step.slots.cpu().numpy() == slots).all()
    assert (step.starts.cpu().numpy() == starts).all()
    assert (step.lens.cpu().numpy() == left).all()
    assert step.free_count.cpu().tolist() == [rest]
    return t, step


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 16, 24, 128])
@pytest.mark.parametrize("batch", [0, 1, 7, 255, 257, 3000])
def test_extend(batch, page):
    rng = np.random.default_rng(batch + page)
    for kind in ("step", "prompts", "short of blocks", "short of tokens", "odd"):
        lens = rng.integers(0, 200, batch)
        new = np.ones(batch, np.int64) if kind == "step" else rng.integers(0, 4 if batch > 1000 else 150, batch)
        if kind == "odd":
            lens[rng.random(batch) < 0.3] *= -1
            new[rng.random(batch) < 0.3] *= -1
        width = max(1, int((-(-(np.maximum(lens, 0) + np.maximum(new, 0)) // page)).max(initial=1)))
        if kind == "odd":
            width = max(1, width * 3 // 4)              # some sequences outgrow their row
        ask = int((-(-(np.maximum(lens, 0) + np.maximum(new, 0)) // page) - -(-np.maximum(lens, 0) // page)).sum())
        total = int(np.maximum(new, 0).sum())
        capacity = ask + batch * width + 5
        free = rng.permutation(capacity).astype(np.int32)
        table = rng.integers(0, capacity, (batch, width)).astype(np.int32)
        count = ask * 2 // 3 if kind == "short of blocks" else ask + 2
        limit = total * 2 // 3 if kind == "short of tokens" else total + (5 if kind == "odd" else 0)
        run_extend(table, lens, new, free, count, page, limit)


@pytest.mark.gpu
def test_extend_many_tokens_and_sequences():
    rng = np.random.default_rng(1)
    lens, new = rng.integers(0, 100, 8192), rng.integers(0, 30, 8192)
    table = np.zeros((8192, 9), np.int32)
    free = rng.permutation(40000).astype(np.int32)
    run_extend(table, lens, new, free, 40000, 16, int(new.sum()) + 3)
    run_extend(np.zeros((2, 8192), np.int32), [0, 5], [100001, 29999], free, 40000, 16, 130001)
    # counts whose sum passes 32 bits
    run_extend(np.zeros((3, 4), np.int32), [0, 3, 2 ** 31 - 1], [5, 2 ** 31 - 1, 2 ** 31 - 1], free, 40000, 16, 50)


def run_trim(table, lens, keep, free, count, page):
    t, f = on_gpu(table.copy()), on_gpu(free.copy())
    left, rest = ft().block_table_trim(t, on_gpu(np.asarray(lens, np.int32)), on_gpu(np.asarray(keep, np.int32)), f,
                                       on_gpu(np.array([count], np.int32)), page)
    want = free.copy()
    lens_out, total = ref.trim(table, lens, keep, want, count, page)
    assert (t.cpu().numpy() == table).all()
    assert (f.cpu().numpy() == want).all()
    assert (left.cpu().numpy() == lens_out).all()
    assert rest.cpu().tolist() == [total]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("batch", [0, 1, 9, 300, 8192])
def test_trim(batch, page):
    rng = np.random.default_rng(batch * 3 + page)
    lens = rng.integers(0, 120, batch)
    width = max(1, -(-120 // page))
    table = rng.permutation(max(1, batch * width)).astype(np.int32)[: batch * width].reshape(batch, width)
    capacity = batch * width + 7
    free = np.full(capacity, -9, np.int32)
    run_trim(table, lens, np.where(rng.random(batch) < 0.4, 0, lens), free, 3, page)
    run_trim(table, lens, lens - rng.integers(-3, 40, batch), free, 7, page)
    run_trim(table, lens, np.zeros(batch, np.int64), free[: capacity // 2].copy(), 2, page)      # a stack that cannot hold them


@pytest.mark.gpu
def test_block_table_page_beyond_32_bits():
    i = torch.zeros((2,), dtype=torch.int32, device="cuda")
    for page in (2 ** 31, 2 ** 32 + 16):                    # (the second is 16 to 32 bits)
        with pytest.raises(ValueError):
            ft().block_table_extend(i.view(2, 1), i, i, i, i[:1], page, 8)
        with pytest.raises(ValueError):
            ft().block_table_trim(i.view(2, 1), i, i, i, i[:1], page)


@pytest.mark.gpu
def test_block_table_refusals():
    i = torch.zeros((4,), dtype=torch.int32, device="cuda")
    t, one = i.view(2, 2), i[:1]
    good = (t, i[:2], i[:2], i, one, 16, 8)
    ft().block_table_extend(*good)
    for at, bad in ((0, t.long()), (1, i[:2].float()), (3, i.cpu()), (4, one.long())):
        with pytest.raises(TypeError):
            ft().block_table_extend(*good[:at], bad, *good[at + 1:])
    for at, bad in ((0, i), (0, t.t()), (1, i[:3]), (2, i), (3, t), (4, i[:2]), (5, 0), (5, 1.5), (6, -1), (6, 2 ** 31)):
        with pytest.raises(ValueError):
            ft().block_table_extend(*good[:at], bad, *good[at + 1:])
    many = torch.zeros((8193,), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ft().block_table_extend(many[:, None].contiguous(), many, many, i, one, 16, 8)
    with pytest.raises(ValueError):
        ft().block_table_trim(t, i[:2], i[:3], i, one, 16)
    with pytest.raises(TypeError):
        ft().block_table_trim(t, i[:2], i[:2], i.long(), one, 16)


# ---- together --------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [28, 8])
@pytest.mark.parametrize("store,name,hq,hkv,dim,page", [("int8", "bf16", 8, 2, 128, 16), ("e4m3", "f32", 5, 1, 64, 32),
                                                        ("e4m3", "f16", 4, 4, 96, 12)])
def test_serving_loop(store, name, hq, hkv, dim, page, blocks):
    """Prompts arrive, sequences decode, draft tokens are cut off, sequences finish and others take their blocks: the four
    operators together against a model of the same loop on the host."""
    rng = np.random.default_rng(dim)
    batch, width = 6, 10
    table, lens = np.zeros((batch, width), np.int32), np.zeros(batch, np.int64)
    free, count = rng.permutation(blocks).astype(np.int32), blocks
    k, v = (np.zeros((blocks, hkv, page, dim), np.uint8) for _ in range(2))
    scales = np.zeros((blocks, hkv, 2), np.float32)
    g = dict(table=on_gpu(table.copy()), lens=on_gpu(lens.astype(np.int32)), free=on_gpu(free.copy()),
             count=on_gpu(np.array([count], np.int32)), k=pool(k.copy(), store), v=pool(v.copy(), store), s=on_gpu(scales.copy()))
    refused = 0
    for step in range(12):
        new = np.ones(batch, np.int64)
        if step % 3 == 0:
            new = np.where(lens == 0, rng.integers(1, 4 * page, batch), rng.integers(0, 5, batch))
        limit = int(new.sum()) + 2
        plan = ft().block_table_extend(g["table"], g["lens"], on_gpu(new.astype(np.int32)), g["free"], g["count"], page, limit)
        slots, _, left, count = ref.extend(table, lens, new, free, count, page, limit)
        refused += int((left < lens + new).sum())
        lens = left.astype(np.int64)
        x = rounded(rng.standard_normal((2, limit, hkv, dim)) * 2.0 ** rng.integers(-3, 3), name)
        ft().kv_append_paged_q8(g["k"], g["v"], g["s"], x[0].cuda(), x[1].cuda(), plan.slots)
        ref.append(k, scales, 0, x[0].double().numpy(), slots, page, store)
        ref.append(v, scales, 1, x[1].double().numpy(), slots, page, store)
        q = rounded(rng.standard_normal((batch, hq, dim)), name)
        out = ft().attention_decode_paged_q8(q.cuda(), g["k"], g["v"], g["s"], g["table"], plan.lens)
        want, bound = ref.decode(q.double().numpy(), k, v, scales, table, lens, store, STEP[name])
        tol = bound + (np.abs(want) + bound) * torch.finfo(q.dtype).eps / 2
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all(), step
        keep = np.maximum(lens - rng.integers(0, 3, batch), 0) if step % 4 == 2 else lens.copy()
        if step % 3 == 2:
            keep[rng.integers(0, batch)] = 0
        g["lens"], g["count"] = ft().block_table_trim(g["table"], plan.lens, on_gpu(keep.astype(np.int32)), g["free"], plan.free_count, page)
        left, count = ref.trim(table, lens, keep, free, count, page)
        lens = left.astype(np.int64)
        assert (g["table"].cpu().numpy() == table).all() and (g["free"].cpu().numpy() == free).all()
        assert (g["lens"].cpu().numpy() == lens).all() and g["count"].item() == count
        assert (g["s"].cpu().numpy() == scales).all()
        assert (codes_of(g["k"]) == k).all() and (codes_of(g["v"]) == v).all()
    assert refused or blocks > 8                        # the small pool cannot hold six prompts


def _decode_step(state):
    """What a decode loop captures: one token for every sequence, all state on the GPU."""
    plan = ft().block_table_extend(state["table"], state["lens"], state["ones"], state["free"], state["count"], state["page"], len(state["ones"]))
    ft().kv_append_paged_q8(state["k"], state["v"], state["s"], state["x"], state["x"], plan.slots)
    out = ft().attention_decode_paged_q8(state["q"], state["k"], state["v"], state["s"], state["table"], plan.lens)
    state["lens"].copy_(plan.lens)
    state["count"].copy_(plan.free_count)
    return out


def _step_state(seed, page=16, dim=128, batch=5):
    rng = np.random.default_rng(seed)
    lens = rng.integers(1, 300, batch)
    k, v, scales, table = make_cache(rng, lens.tolist(), 2, dim, page, "int8", spare=40)
    used = {int(x) for b, n in enumerate(lens) for x in table[b, : -(-n // page)]}
    free = np.array([i for i in range(len(k)) if i not in used], np.int32)
    return dict(page=page, table=on_gpu(np.concatenate([table, np.zeros((batch, 8), np.int32)], 1)), lens=on_gpu(lens.astype(np.int32)),
                ones=torch.ones(batch, dtype=torch.int32, device="cuda"), free=on_gpu(free),
                count=on_gpu(np.array([len(free)], np.int32)), k=pool(k, "int8"), v=pool(v, "int8"), s=on_gpu(scales),
                x=on_gpu(rng.standard_normal((batch, 2, dim)), torch.bfloat16), q=on_gpu(rng.standard_normal((batch, 8, dim)), torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(16, 128), (12, 64)])
def test_captured_steps_on_two_streams(page, dim):
    """Two captured decode loops, replayed at the same time on two streams while a third runs eagerly: each gives what it
    gives alone, bit for bit."""
    states, alone = [_step_state(s, page, dim) for s in range(3)], [_step_state(s, page, dim) for s in range(3)]
    want = [[_decode_step(a).clone() for _ in range(6)] for a in alone]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s in states[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_decode_step(s))
        graphs.append(g)
    torch.cuda.synchronize()
    got = [[], [], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
                got[i].append(outs[i].clone())
        got[2].append(_decode_step(states[2]))
    torch.cuda.synchronize()
    for i in range(3):
        for a, b in zip(want[i], got[i]):
            assert torch.equal(a, b)
        for key in ("k", "v", "s", "table", "lens", "count"):
            assert torch.equal(states[i][key].view(torch.uint8), alone[i][key].view(torch.uint8)), key
    from fusedtok_b200 import _fusedtok
    assert _fusedtok.attention_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(16, 128), (12, 64)])
def test_plain_calls_and_the_careful_way_agree(page, dim, monkeypatch):
    """The module that takes plain calls straight to the library is there, takes them, and does what the wrappers do; what it
    does not take reaches them."""
    f = ft()
    assert f._tensors is not None
    native, careful = _step_state(21, page, dim), _step_state(21, page, dim)
    a = [_decode_step(native).clone() for _ in range(4)]
    names = ("_decode_q8_native", "_append_q8_native", "_extend_native", "_trim_native")
    taken = []
    for n in names:
        monkeypatch.setattr(f, n, lambda *x, n=n, real=getattr(f, n): taken.append((n, real(*x) is not None)))
    b = []
    for _ in range(4):
        plan = f.block_table_extend(careful["table"], careful["lens"], careful["ones"], careful["free"], careful["count"], page, 5)
        f.kv_append_paged_q8(careful["k"], careful["v"], careful["s"], careful["x"], careful["x"], plan.slots)
        b.append(f.attention_decode_paged_q8(careful["q"], careful["k"], careful["v"], careful["s"], careful["table"], plan.lens))
        assert type(plan) is f.BlockTableStep and plan.starts.tolist() == [0, 1, 2, 3, 4, 5]
        careful["lens"], careful["count"] = plan.lens, plan.free_count
    assert taken == [(n, True) for n in ("_extend_native", "_append_q8_native", "_decode_q8_native")] * 4
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    for key in ("k", "v", "s", "table", "lens", "count"):
        assert torch.equal(native[key].view(torch.uint8), careful[key].view(torch.uint8)), key
    monkeypatch.undo()
    keep = native["lens"] // 2
    one, two = native["free"].clone(), native["free"].clone()
    cut = f.block_table_trim(native["table"], native["lens"], keep, one, native["count"], page)
    monkeypatch.setattr(f, "_trim_native", lambda *x: None)
    again = f.block_table_trim(native["table"], native["lens"], keep, two, native["count"], page)
    assert all(torch.equal(x, y) for x, y in zip(cut, again)) and torch.equal(one, two)


@pytest.mark.gpu
def test_same_bits_every_call():
    rng = np.random.default_rng(2)
    lens = [3000, 17, 900]
    k, v, scales, table = make_cache(rng, lens, 2, 128, 16, "e4m3")
    args = (rounded(rng.standard_normal((3, 16, 128)), "bf16").cuda(), pool(k, "e4m3"), pool(v, "e4m3"), on_gpu(scales), on_gpu(table),
            on_gpu(np.array(lens, np.int32)))
    first = ft().attention_decode_paged_q8(*args)
    for _ in range(20):
        assert torch.equal(first, ft().attention_decode_paged_q8(*args))


@pytest.mark.gpu
def test_index_tensors_of_other_types():
    """int64 tables, lengths and slots (PyTorch's default) give what int32 ones give; a slot beyond 32 bits is passed over,
    not wrapped into the pool; host arrays and strided index tensors too."""
    rng = np.random.default_rng(13)
    lens = [100, 37]
    k, v, scales, table = make_cache(rng, lens, 2, 64, 16, "int8")
    q = rounded(rng.standard_normal((2, 4, 64)), "bf16").cuda()
    a = (pool(k, "int8"), pool(v, "int8"), on_gpu(scales))
    want = ft().attention_decode_paged_q8(q, *a, on_gpu(table), on_gpu(np.array(lens, np.int32)))
    wide = on_gpu(np.repeat(table, 2, axis=1).astype(np.int64))[:, ::2]
    for t in (on_gpu(table.astype(np.int64)), wide, table, torch.from_numpy(table)):
        for n in (on_gpu(np.array(lens)), lens, np.array(lens, np.int16)):
            assert torch.equal(want, ft().attention_decode_paged_q8(q, *a, t, n))
    x = rounded(rng.standard_normal((4, 2, 64)), "f16").cuda()
    slots = np.array([2 ** 32 + 3, table[0, 1] * 16 + 2, -2 ** 33, 2 ** 31 - 1])
    kq, vq, s = (t.clone() for t in a)
    ft().kv_append_paged_q8(kq, vq, s, x, x, on_gpu(slots))
    ref.append(k, scales, 0, x.double().cpu().numpy(), [-1, slots[1], -1, -1], 16, "int8")
    assert (codes_of(kq) == k).all() and (s.cpu().numpy()[..., 0] == scales[..., 0]).all()


@pytest.mark.gpu
def test_every_code():
    """All 256 codes are read as what they stand for (int8 -128 among them, which an append never writes)."""
    for store in STORES:
        codes = np.arange(256, dtype=np.uint8)
        codes = codes[np.isfinite(ref.decode_codes(codes, store))]
        for dim, page in ((64, 16), (128, 16), (20, 7)):
            n = -(-len(codes) // dim) * dim
            rows = np.resize(codes, n).reshape(-1, dim)
            for row in rows:
                pools = np.zeros((1, 1, page, dim), np.uint8)
                pools[0, 0, 0] = row
                scales = np.array([[[0.0, 0.37]]], np.float32)
                out = ft().attention_decode_paged_q8(torch.ones((1, 1, dim), device="cuda"), pool(pools, store), pool(pools, store),
                                                     on_gpu(scales), [[0]], [1])
                want = ref.decode_codes(row, store) * np.float64(np.float32(0.37))
                # one weight of exactly 1 in two halves, codes exact: the scale's product and its factors, a few half steps
                assert (np.abs(out.double().cpu().numpy()[0, 0] - want) <= np.abs(want) * 2.0 ** -21).all()


_SELF_CHECKING = """
import sys, numpy as np, torch
sys.path.insert(0, %r); sys.path.insert(0, %r)
import test_q8_cache as t
from fusedtok_b200 import _fusedtok
for shape in t.SHAPES:
    b, hq, hkv, d, page, lens = shape
    rng = np.random.default_rng(1)
    k, v, scales, table = t.make_cache(rng, lens, hkv, d, page, "e4m3")
    q = t.rounded(rng.standard_normal((b, hq, d)), "bf16")
    t.check_decode(q, k, v, scales, table, lens, "e4m3", "bf16")
    assert _fusedtok.attention_device_status() == 0, shape
    table[0, 0] = len(k) + 3 if hq %% 2 else -1       # outside the pool: reported, read as block 0
    t.ft().attention_decode_paged_q8(q.cuda(), t.pool(k, "e4m3"), t.pool(v, "e4m3"), t.on_gpu(scales), t.on_gpu(table),
                                     t.on_gpu(np.array(lens, np.int32)))
    assert _fusedtok.attention_device_status() == (8 if lens[0] else 0), shape
    assert _fusedtok.attention_device_status() == 0
print("self-checked")
"""


@pytest.mark.gpu
def test_self_checking_build():
    """The build that compares every computed row and slot with what the launch owns (see test_bounds_build_gpu.py)."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    variant = os.path.join(os.path.dirname(here), "fusedtok_b200", "libfusedtok_b200_bounds.so")
    if not os.path.exists(variant):
        pytest.skip("self-checking variant of the library not built")
    done = subprocess.run([sys.executable, "-c", _SELF_CHECKING % (os.path.dirname(here), here)], capture_output=True, text=True,
                          timeout=600, env=dict(os.environ, FUSEDTOK_B200_LIB=variant))
    assert done.returncode == 0 and "self-checked" in done.stdout, done.stdout + done.stderr


_FIRST_CALLS_CAPTURED = """
import sys, numpy as np, torch
sys.path.insert(0, %r); sys.path.insert(0, %r)
import test_q8_cache as t
state, alone = t._step_state(5, %d, %d), t._step_state(5, %d, %d)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = t._decode_step(state)                   # the first calls of the library in this process
got = []
for _ in range(3):
    g.replay()
    got.append(out.clone())
torch.cuda.synchronize()
for x in got:
    assert torch.equal(x, t._decode_step(alone))
for key in ("k", "v", "s", "table", "lens", "count"):
    assert torch.equal(state[key].view(torch.uint8), alone[key].view(torch.uint8)), key
print("captured first")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(16, 128), (12, 64)])
def test_first_calls_of_a_process_are_captured(page, dim):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = _FIRST_CALLS_CAPTURED % (os.path.dirname(here), here, page, dim, page, dim)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stdout + done.stderr


@pytest.mark.gpu
def test_calls_on_two_streams_and_threads():
    """Calls that overlap on different streams, issued from different threads, share nothing."""
    import threading
    rng = np.random.default_rng(14)
    cases = []
    for i in range(3):
        lens = [4000 - 700 * i, 17, 900]
        k, v, scales, table = make_cache(rng, lens, 2, 128, 16, "e4m3")
        cases.append((rounded(rng.standard_normal((3, 8, 128)), "bf16").cuda(), pool(k, "e4m3"), pool(v, "e4m3"), on_gpu(scales),
                      on_gpu(table), on_gpu(np.array(lens, np.int32))))
    want = [ft().attention_decode_paged_q8(*c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [ft().attention_decode_paged_q8(*cases[i]) for _ in range(50)]
        stream.synchronize()
        bad.extend(i for o in outs if not torch.equal(o, want[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
