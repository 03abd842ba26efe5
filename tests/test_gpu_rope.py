"""GPU: head norms, rotation and the cache write vs the formula in 64 bits."""
import pytest
import torch

from ocelotl_b200.errors import KernelError, UnsupportedError
from tests.decode_cases import rope_reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_errors(backend):
    backend.take_device_errors()
    yield
    assert backend.take_device_errors() == (0, 0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# One value: norm (sum of D squares in a tree of at most 5 + 8 levels, mean, rsqrt of 2
# units, two products: under 8 units of 2^-24 together with the root's halving), the
# turn (cos and sin good to 4 units of the largest, two products, one sum: 8 units).
UNITS = 16 * 2.0 ** -24


def check(backend, rows, heads, kv, dim, dtype, rot=None, base=10000.0, interleaved=False, norm=True, page=16, positions=None,
          eps=1e-6, seed=1, factors=None, far=5000, layout="hnd"):
    g = torch.Generator("cuda").manual_seed(seed)
    rot = dim if rot is None else rot
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, device="cuda", generator=g) * 2
    pos = positions if positions is not None else torch.randint(0, far, (rows,), device="cuda", generator=g).to(torch.int32)
    pages_a_seq = max(int(pos.max()), 0) // page + 1
    pages = rows + 1
    table = torch.full((rows, pages_a_seq), -1, dtype=torch.int32, device="cuda")
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:rows].to(torch.int32).cuda()
    table[torch.arange(rows, device="cuda"), (pos // page).clamp(min=0).long()] = perm  # only the rows' own pages exist
    shape = (pages, kv, page, dim) if layout == "hnd" else (pages, page, kv, dim)
    k, v = (torch.full(shape, 0.25, dtype=dtype, device="cuda") for _ in range(2))
    if layout == "nhd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    qn, kn = ((1 + 0.1 * torch.randn(dim, device="cuda", generator=g)) for _ in range(2)) if norm else (None, None)
    rope = backend.rope_table(rot, base, factors=factors, interleaved=interleaved) if rot else None
    out = torch.full((rows, heads, dim), float("nan"), device="cuda")
    got = backend.qk_norm_rope(qkv, backend.kv_cache_view(k, v), pos, table, rope, q_norm=qn, k_norm=kn, eps=eps, out=out)
    backend.synchronize()
    assert got is out
    (q, qs), (kk, ks), (vv, vs) = rope_reference(qkv, heads, kv, dim, pos.clamp(min=0), rot, base, interleaved, qn, kn, eps,
                                                 factors)
    live = pos >= 0
    assert ((got.double() - q).abs()[live] <= UNITS * qs[live]).all()
    assert (got[~live] == 0).all()
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    where = perm.long(), pos.long() % page
    for name, t, want, size in (("k", k, kk, ks), ("v", v, vv, vs)):
        cached = t[where[0], :, where[1]].double()
        room = half * want.abs() * (1 + half) + UNITS * size * (name == "k") * (1 + half) + tiny
        assert ((cached - want).abs()[live] <= room[live]).all(), name
        t[where[0][live], :, where[1][live]] = 0.25
        assert (t == 0.25).all(), name  # nothing else was written
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_dims_pairs_and_types(backend, dim, interleaved, dtype):
    for norm in (False, True):
        check(backend, 5, 8, 2, dim, dtype, interleaved=interleaved, norm=norm, seed=dim)


@pytest.mark.parametrize("rows", [1, 2, 37, 300])
@pytest.mark.parametrize("heads,kv", [(32, 8), (28, 4), (1, 1), (9, 3), (20, 1)])
def test_rows_and_heads(backend, rows, heads, kv):
    check(backend, rows, heads, kv, 128, torch.bfloat16, seed=rows)


@pytest.mark.parametrize("rot", [0, 8, 40, 64, 120, 128])
def test_partial_rotation(backend, rot):
    for interleaved in (False, True):
        check(backend, 7, 4, 2, 128, torch.bfloat16, rot=rot, interleaved=interleaved, seed=rot)


@pytest.mark.parametrize("base", [1.0, 0.5, 10000.0, 1000000.0, 5e8])
def test_far_positions(backend, base):
    pos = i32([0, 1, 131071, 1048575, 30_000_001])
    check(backend, 5, 4, 1, 128, torch.bfloat16, base=base, positions=pos, page=65536)


def test_factors(backend):
    f = [1.0 + 0.25 * i for i in range(64)]
    check(backend, 9, 4, 2, 128, torch.bfloat16, factors=f)
    check(backend, 9, 4, 2, 128, torch.bfloat16, factors=[0.125] * 64)


@pytest.mark.parametrize("page", [1, 7, 24, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages_and_layouts(backend, page, layout):
    check(backend, 11, 4, 2, 128, torch.float16, page=page, layout=layout, far=300)


def test_padding_rows(backend):
    check(backend, 6, 4, 2, 128, torch.bfloat16, positions=i32([5, -1, 17, -1, -3, 0]))
    check(backend, 3, 4, 2, 128, torch.bfloat16, positions=i32([-1, -1, -1]), eps=0.0)


def test_rounding_to_the_cache(backend):
    """v is copied, so its cache value is torch's own rounding, specials included."""
    vals = torch.tensor([0.0, -0.0, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, 65519.0, 65520.0, 1e-8, 3e38, float("inf"),
                         -float("inf"), float("nan"), 2.0 ** -24, 6e-8, 1.0 + 2.0 ** -11, 1.0 + 3 * 2.0 ** -11, -5.0],
                        device="cuda")
    qkv = vals.repeat(3 * 64 // 16).view(1, -1).contiguous()
    table = i32([[0]])
    for dtype in (torch.bfloat16, torch.float16):
        cache = backend.kv_cache(1, 16, 1, 64, dtype)
        backend.qk_norm_rope(qkv, cache, i32([3]), table, None)
        backend.synchronize()
        want = qkv[0, :64].to(dtype)
        for t in (cache.k, cache.v):
            assert torch.equal(torch.nan_to_num(t[0, 0, 3], nan=77.0), torch.nan_to_num(want, nan=77.0))
            assert torch.equal(torch.signbit(t[0, 0, 3][:2]), torch.signbit(want[:2]))


def test_rows_of_few_sequences(backend):
    dim, heads, kv, page = 128, 4, 2, 16
    cache = backend.kv_cache(20, page, kv, dim)
    table = i32([[3, 1, 4], [5, 9, 2]])
    seqs, pos = i32([1, 0, 1, 1, 0]), i32([0, 40, 1, 47, 41])
    qkv = torch.randn(5, (heads + 2 * kv) * dim, device="cuda")
    backend.qk_norm_rope(qkv, cache, pos, table, backend.rope_table(dim, 10000.0), seqs=seqs)
    backend.synchronize()
    _, (k, _), (v, _) = rope_reference(qkv, heads, kv, dim, pos, dim, 10000.0, False, None, None, 0)
    for r in range(5):
        pg = int(table[seqs[r].long(), pos[r].long() // page])
        assert (cache.k[pg, :, int(pos[r]) % page].double() - k[r]).abs().max() <= 2.0 ** -8 * k[r].abs().max()
        assert torch.equal(cache.v[pg, :, int(pos[r]) % page], v[r].to(torch.bfloat16))
    assert int((cache.v != 0).any(-1).any(1).sum()) == 5


def test_strided_rows(backend):
    wide = torch.randn(3, 8 * 64 + 64, device="cuda")
    cache = backend.kv_cache(4, 16, 2, 64)
    a = backend.qk_norm_rope(wide[:, :8 * 64], cache, i32([1, 2, 3]), i32([[0], [1], [2]]), backend.rope_table(64, 1e4))
    ka = cache.k.clone()
    b = backend.qk_norm_rope(wide[:, :8 * 64].contiguous(), cache, i32([1, 2, 3]), i32([[0], [1], [2]]),
                             backend.rope_table(64, 1e4))
    backend.synchronize()
    assert torch.equal(a, b) and torch.equal(ka, cache.k)


def test_cache_offsets_past_32_bits(backend):
    pages, kv, page, dim = 36000, 8, 64, 128  # 2.36e9 elements
    k = torch.empty(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    cache = backend.kv_cache_view(k, torch.empty_like(k))
    qkv = torch.randn(1, 24 * dim, device="cuda")
    backend.qk_norm_rope(qkv, cache, i32([63]), i32([[pages - 1]]), None)
    backend.synchronize()
    assert torch.equal(cache.k[-1, :, 63], qkv[0, 8 * dim:16 * dim].view(8, dim).to(torch.bfloat16))
    assert torch.equal(cache.v[-1, :, 63], qkv[0, 16 * dim:].view(8, dim).to(torch.bfloat16))


def test_places_out_of_range_cache_nothing(backend):
    cache = backend.kv_cache(4, 16, 2, 64)
    qkv = torch.randn(5, 8 * 64, device="cuda")
    table = i32([[0, -1], [4, 2], [1, 3]])
    pos, seqs = i32([16, 0, 32, 5, 7]), i32([0, 1, 2, 3, -1])  # page -1, page 4, past the table, no sequence, no sequence
    q = backend.qk_norm_rope(qkv, cache, pos, table, backend.rope_table(64, 1e4), seqs=seqs)
    backend.synchronize()
    assert backend.take_device_errors() == (5, 0)
    assert (cache.k == 0).all() and (cache.v == 0).all()
    (want, size), _, _ = rope_reference(qkv, 4, 2, 64, pos, 64, 1e4, False, None, None, 0)
    assert ((q.double() - want).abs() <= UNITS * size).all()


def test_captured_launch(backend):
    cache = backend.kv_cache(8, 16, 2, 64)
    qkv = torch.randn(2, 8 * 64, device="cuda")
    rope = backend.rope_table(64, 1e4)
    table, pos = i32([[0, 1], [2, 3]]), i32([0, 0])
    out = torch.empty(2, 4, 64, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            backend.use_current_stream()
            backend.qk_norm_rope(qkv, cache, pos, table, rope, out=out)
    finally:
        backend.set_stream(None)
    for p in ([3, 31], [16, 0]):
        pos.copy_(i32(p))
        qkv.normal_()
        graph.replay()
        torch.cuda.synchronize()
        (want, size), _, _ = rope_reference(qkv, 4, 2, 64, pos, 64, 1e4, False, None, None, 0)
        assert ((out.double() - want).abs() <= UNITS * size).all()


def test_refusals(backend):
    cache = backend.kv_cache(4, 16, 2, 64)
    qkv = torch.randn(2, 8 * 64, device="cuda")
    pos, table = i32([0, 1]), i32([[0], [1]])
    rope = backend.rope_table(64, 1e4)
    f = backend.qk_norm_rope
    with pytest.raises(KernelError):
        f(qkv.half(), cache, pos, table, rope)
    with pytest.raises(KernelError, match="width"):
        f(qkv[:, :500].contiguous(), cache, pos, table, rope)
    with pytest.raises(KernelError, match="multiple of n_kv_heads"):
        f(qkv[:, :7 * 64].contiguous(), cache, pos, table, rope)
    with pytest.raises(KernelError, match="rot_dim"):
        f(qkv, cache, pos, table, backend.rope_table(128, 1e4))
    with pytest.raises(KernelError, match="eps"):
        f(qkv, cache, pos, table, rope, eps=-1.0)
    with pytest.raises(KernelError, match="q_norm"):
        f(qkv, cache, pos, table, rope, q_norm=torch.ones(63, device="cuda"))
    with pytest.raises(KernelError, match="16-byte"):
        f(qkv, cache, pos, table, rope, q_norm=torch.ones(65, device="cuda")[1:])
    with pytest.raises(KernelError, match="overlaps"):
        f(qkv, cache, pos, table, rope, out=qkv.view(-1)[:2 * 4 * 64].view(2, 4, 64))
    for bad in (0, 12, 264):
        with pytest.raises(UnsupportedError):
            backend.rope_table(bad, 1e4)
    for base in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(KernelError):
            backend.rope_table(64, base)
    with pytest.raises(KernelError, match="factors"):
        backend.rope_table(64, 1e4, factors=[1.0] * 31)
    with pytest.raises(KernelError, match="factor"):
        backend.rope_table(64, 1e4, factors=[0.0] * 32)
