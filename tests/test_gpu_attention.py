"""GPU: attention of new tokens over the paged cache vs the formula in 64 bits."""
import pytest
import torch

from ocelotl_b200.errors import KernelError, UnsupportedError
from tests.decode_cases import attention_reference, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_errors(backend):
    backend.take_device_errors()
    yield
    assert backend.take_device_errors() == (0, 0)


def positions_of(lengths):
    return torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda")


def check(backend, lengths, kv_heads, group, dim, page, dtype, seed=1, layout="hnd", scale=None, fill=None, sharp=1.0):
    k, v, table = paged(lengths, page, kv_heads, dim, dtype, seed, layout, fill=fill)
    g = torch.Generator("cuda").manual_seed(seed + 1)
    q = torch.randn(len(lengths), kv_heads * group, dim, device="cuda", generator=g) * sharp
    pos = positions_of(lengths)
    out = torch.full_like(q, float("nan"))
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, scale=scale, out=out)
    backend.synchronize()
    assert got is out
    want, bound = attention_reference(q, k, v, pos, table, dim ** -0.5 if scale is None else scale)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), ((off / bound.clamp(min=1e-300)).max().item(), lengths)
    # and as a whole: f32 quality, far below one rounding of anything to 16 bits (2^-9)
    if want.norm() > 0:
        assert (off.norm() / want.norm()).item() < 2.0 ** -17
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_one_row(backend, dim, dtype):
    for n in (1, 2, 15, 16, 17, 63, 64, 65, 200):
        check(backend, [n], 2, 4, dim, 16, dtype, seed=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_ragged_batch_with_empty_rows(backend, dim, dtype):
    check(backend, [0, 1, 700, 64, 0, 129, 31, 5000, 0], 4, 7, dim, 16, dtype, seed=dim)


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (8, 1), (1, 8), (3, 5), (2, 9), (1, 20), (2, 16)])
def test_head_groups(backend, kv_heads, group):
    check(backend, [77, 300, 1], kv_heads, group, 128, 32, torch.bfloat16, seed=group)


@pytest.mark.parametrize("page", [1, 3, 7, 16, 24, 100, 256, 1000])
def test_page_sizes(backend, page):
    check(backend, [333, 47, 1025], 2, 4, 128, page, torch.bfloat16, seed=page)


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layouts(backend, layout, dtype):
    check(backend, [500, 33], 4, 4, 128, 16, dtype, layout=layout)


@pytest.mark.parametrize("n,kv_heads", [(9000, 8), (60001, 1), (30000, 2)])
def test_one_row_over_many_ctas(backend, n, kv_heads):
    check(backend, [n], kv_heads, 4, 128, 16, torch.bfloat16)
    check(backend, [n], kv_heads, 3, 64, 16, torch.float16)
    check(backend, [n], kv_heads, 8, 256, 64, torch.bfloat16)


def test_many_short_rows(backend):
    check(backend, [(i * 37) % 150 for i in range(400)], 2, 7, 64, 16, torch.float16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_many_items(backend, dim, dtype):
    """Enough rows and heads that every warp takes items of its own; some rows long, some empty."""
    lengths = [(i * 53) % 200 for i in range(240)]
    check(backend, lengths, 8, 3, dim, 16, dtype, seed=dim)
    if dim in (96, 128):
        check(backend, [0, 3000, 1] + lengths, 8, 6, dim, 24, dtype, seed=dim)


@pytest.mark.parametrize("scale,sharp", [(1e-6, 1.0), (1.0, 1.0), (0.0884, 8.0)])
def test_flat_and_peaked_weights(backend, scale, sharp):
    for dtype in (torch.bfloat16, torch.float16):
        check(backend, [400, 2000], 2, 4, 128, 16, dtype, scale=scale, sharp=sharp)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 3e4])
def test_slots_behind_a_sequence_do_not_count(backend, fill):
    for dtype in (torch.bfloat16, torch.float16):
        check(backend, [70, 1, 0, 333, 16], 2, 4, 128, 48, dtype, fill=fill)


def test_large_and_tiny_queries(backend):
    # f16 pieces are scaled per head: magnitudes far outside f16's range keep their precision
    k, v, table = paged([100, 100, 100], 16, 1, 128, torch.float16, 5)
    q = torch.randn(3, 2, 128, device="cuda") * torch.tensor([1e6, 1.0, 1e-9], device="cuda")[:, None, None]
    pos = positions_of([100] * 3)
    for scale in (1e-6, 1.0):
        got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, scale=scale)
        backend.synchronize()
        want, bound = attention_reference(q, k, v, pos, table, scale)
        assert ((got.double() - want).abs() <= bound).all()


def test_nan_in_a_seen_token_reaches_only_its_heads(backend):
    k, v, table = paged([90, 90], 16, 2, 128, torch.bfloat16, 5)
    k[table[0, 2].long(), 1, 3, 7] = float("nan")  # token 35 of sequence 0, k/v head 1
    q = torch.randn(2, 8, 128, device="cuda")
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), positions_of([90, 90]), table)
    backend.synchronize()
    assert torch.isnan(got[0, 4:]).all()
    assert torch.isfinite(got[0, :4]).all() and torch.isfinite(got[1]).all()


def test_several_rows_of_one_sequence_are_causal(backend):
    k, v, table = paged([40, 700, 9], 16, 2, 128, torch.bfloat16, 6)
    seqs = torch.tensor([1, 1, 1, 0, 2, 1, 0, 2], dtype=torch.int32, device="cuda")
    pos = torch.tensor([699, 698, 0, 39, 8, 64, -1, 3], dtype=torch.int32, device="cuda")
    q = torch.randn(8, 8, 128, device="cuda")
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs)
    backend.synchronize()
    want, bound = attention_reference(q, k, v, pos, table, 128 ** -0.5, seqs)
    assert ((got.double() - want).abs() <= bound).all()
    assert (got[6] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9])
def test_drafted_rows_and_prompts(backend, group, dim, dtype):
    """Runs of rows of one sequence, which are worked on together: drafted tokens, a prompt, padding between
    them, positions out of order; long enough to be split, and short."""
    lengths, rows = [900, 40, 3000, 7], []
    rows += [(0, 900 - 5 + i) for i in range(5)] + [(1, p) for p in range(40)] + [(1, -1)] * 3
    rows += [(2, p) for p in (2999, 2998, 0, 17, 31, 32, 1500)] + [(3, p) for p in (6, -1, 2)] + [(0, 64)]
    k, v, table = paged(lengths, 16, 2, dim, dtype, group)
    table = torch.nn.functional.pad(table, (0, 2000), value=-1)  # room for long sequences
    seqs, pos = (torch.tensor([r[i] for r in rows], dtype=torch.int32, device="cuda") for i in range(2))
    q = torch.randn(len(rows), 2 * group, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(dim))
    cache = backend.kv_cache_view(k, v)
    for n in (len(rows), 5, 2, 1):
        out = torch.full((n, 2 * group, dim), float("nan"), device="cuda")
        backend.paged_attention(q[:n], cache, pos[:n], table, seqs=seqs[:n], out=out)
        backend.synchronize()
        want, bound = attention_reference(q[:n], k, v, pos[:n], table, dim ** -0.5, seqs[:n])
        assert ((out.double() - want).abs() <= bound).all(), n


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [2, 4, 8])
def test_rows_of_a_sequence_do_not_see_later_tokens(backend, group, dim):
    """What a later row of the sequence sees, NaN and infinities too, does not reach an earlier one."""
    for dtype in (torch.bfloat16, torch.float16):
        k, v, table = paged([50], 16, 1, dim, dtype, 3)
        table = torch.nn.functional.pad(table, (0, 5000), value=-1)  # room for long sequences
        slot = table[0, 3].long(), 0, 0  # token 48
        seqs, pos = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor([46, 47, 48, 49], dtype=torch.int32, device="cuda")
        q = torch.randn(4, group, dim, device="cuda")
        want, bound = attention_reference(q, k, v, pos, table, dim ** -0.5, seqs)
        for t, bad in ((k, float("nan")), (v, float("nan")), (v, float("inf"))):
            old = t[slot].clone()
            t[slot] = bad
            got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs)
            backend.synchronize()
            t[slot] = old
            assert ((got[:2].double() - want[:2]).abs() <= bound[:2]).all()
            assert not torch.isfinite(got[2:]).any()


def test_drafted_rows_over_many_ctas(backend):
    for group, dim, dtype in ((8, 256, torch.bfloat16), (5, 128, torch.float16), (4, 128, torch.bfloat16), (1, 64, torch.float16)):
        k, v, table = paged([9000, 20000], 16, 2, dim, dtype, 3)
        pos = torch.tensor([8999 - 4 + i for i in range(5)] + [19999 - 4 + i for i in range(5)], dtype=torch.int32, device="cuda")
        seqs = torch.tensor([0] * 5 + [1] * 5, dtype=torch.int32, device="cuda")
        q = torch.randn(10, 2 * group, dim, device="cuda")
        got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs)
        backend.synchronize()
        want, bound = attention_reference(q, k, v, pos, table, dim ** -0.5, seqs)
        assert ((got.double() - want).abs() <= bound).all()


def test_many_items_of_several_rows(backend):
    """Enough prompts that a warp takes whole items."""
    for group, dim in ((4, 128), (2, 64), (4, 256)):
        n = 20
        lengths = [n] * 120
        k, v, table = paged(lengths, 16, 8, dim, torch.bfloat16, 3)
        pos = torch.arange(n, dtype=torch.int32, device="cuda").repeat(120)
        seqs = torch.arange(120, dtype=torch.int32, device="cuda").repeat_interleave(n)
        q = torch.randn(n * 120, 8 * group, dim, device="cuda")
        got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs)
        backend.synchronize()
        for s in (0, 7, 119):
            at = slice(s * n, (s + 1) * n)
            want, bound = attention_reference(q[at], k, v, pos[at], table, dim ** -0.5, seqs[at])
            assert ((got[at].double() - want).abs() <= bound).all()


def test_strided_queries_tables_and_neighbours(backend):
    k, v, table = paged([90, 200], 16, 2, 64, torch.bfloat16, 7)
    wide = torch.full((2, 40), 12345, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + table.shape[1]] = table
    qkv = torch.randn(2, (8 + 4) * 64, device="cuda")
    q = qkv[:, :8 * 64].view(2, 8, 64)
    pos = positions_of([90, 200])
    out = torch.full((4, 8, 64), 7.0, device="cuda")
    backend.paged_attention(q, backend.kv_cache_view(k, v), pos, wide[:, 5:5 + table.shape[1]], out=out[1:3])
    backend.synchronize()
    want, bound = attention_reference(q, k, v, pos, table, 64 ** -0.5)
    assert ((out[1:3].double() - want).abs() <= bound).all()
    assert (out[0] == 7).all() and (out[3] == 7).all()


def test_same_bits_again(backend):
    lengths = [5000, 3, 0, 1200, 64]
    a = check(backend, lengths, 4, 4, 128, 16, torch.bfloat16)
    b = check(backend, lengths, 4, 4, 128, 16, torch.bfloat16)
    assert torch.equal(a, b)


def test_cache_offsets_past_32_bits(backend):
    pages, kv, page, dim = 36000, 8, 64, 128  # 2.36e9 elements
    k = torch.empty(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 1, 2, pages - 2]], dtype=torch.int32, device="cuda")
    for p in table[0].tolist():
        k[p].normal_()
        v[p].normal_()
    q = torch.randn(1, 32, dim, device="cuda")
    pos = positions_of([3 * 64 - 5])
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table)
    backend.synchronize()
    want, bound = attention_reference(q, k, v, pos, table, dim ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()


def test_captured_launch_follows_the_positions(backend):
    k, v, table = paged([1500, 1500], 16, 2, 128, torch.bfloat16, 8)
    cache = backend.kv_cache_view(k, v)
    q = torch.randn(2, 8, 128, device="cuda")
    pos = positions_of([3, 1])
    out = torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            backend.use_current_stream()
            backend.paged_attention(q, cache, pos, table, out=out)
    finally:
        backend.set_stream(None)
    for lengths in ([3, 1], [1500, 0], [700, 1499], [64, 65]):
        pos.copy_(positions_of(lengths))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want, bound = attention_reference(q, k, v, pos, table, 128 ** -0.5)
        assert ((out.double() - want).abs() <= bound).all(), lengths
        # an eager call between replays shares the workspace
        eager = backend.paged_attention(q, cache, pos, table)
        torch.cuda.synchronize()
        assert torch.equal(eager, out)


def test_captured_launch_of_rows_of_a_sequence(backend):
    """Which rows belong together, and how long they are, is read on the device at every replay."""
    k, v, table = paged([1500, 1500], 16, 2, 128, torch.bfloat16, 8)
    table = torch.nn.functional.pad(table, (0, 2000), value=-1)
    cache = backend.kv_cache_view(k, v)
    q = torch.randn(6, 8, 128, device="cuda")
    pos, seqs = (torch.zeros(6, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            backend.use_current_stream()
            backend.paged_attention(q, cache, pos, table, seqs=seqs, out=out)
    finally:
        backend.set_stream(None)
    for of, at in (([0] * 6, [9, 10, 11, 12, 13, 14]), ([0, 1] * 3, [1499, 1499, 3, -1, 700, 701]),
                   ([1, 1, 1, 0, 0, 0], [1497, 1498, 1499, -1, -1, 0]), ([0, 0, 0, 0, 1, 1], [63, 64, 31, 32, 127, 128])):
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        seqs.copy_(torch.tensor(of, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want, bound = attention_reference(q, k, v, pos, table, 128 ** -0.5, seqs)
        assert ((out.double() - want).abs() <= bound).all(), (of, at)


def test_on_a_side_stream(backend):
    k, v, table = paged([900], 16, 2, 128, torch.bfloat16, 9)
    stream = torch.cuda.Stream()
    q0 = torch.randn(1, 8, 128, device="cuda")
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(stream):
            backend.use_current_stream()
            torch.cuda._sleep(20_000_000)
            q = q0 * 2
            got = backend.paged_attention(q, backend.kv_cache_view(k, v), positions_of([900]), table)
        stream.synchronize()
        # outputs of a call made under another current stream live on the backend's stream
        other = backend.paged_attention(q, backend.kv_cache_view(k, v), positions_of([900]), table)
        stream.synchronize()
    finally:
        backend.set_stream(None)
    assert torch.equal(got, other)
    want, bound = attention_reference(q, k, v, positions_of([900]), table, 128 ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()


def test_no_rows(backend):
    k, v, table = paged([10], 16, 2, 128, torch.bfloat16, 9)
    got = backend.paged_attention(torch.empty(0, 8, 128, device="cuda"), backend.kv_cache_view(k, v),
                                  torch.empty(0, dtype=torch.int32, device="cuda"), table)
    assert tuple(got.shape) == (0, 8, 128)


def test_places_out_of_range_are_counted_and_left_out(backend):
    k, v, table = paged([100, 100, 100, 100], 16, 2, 128, torch.bfloat16, 10)
    cache = backend.kv_cache_view(k, v)
    pos = positions_of([100, 100, 100, 100])
    q = torch.randn(4, 8, 128, device="cuda")
    bad = table.clone()
    bad[1, 2] = -7          # 16 tokens of row 1 have no page
    bad[2, :] = 1 << 30     # none of row 2's 100 has
    seqs = torch.tensor([0, 1, 2, 9], dtype=torch.int32, device="cuda")  # row 3 has no sequence
    got = backend.paged_attention(q, cache, pos, bad, seqs=seqs)
    backend.synchronize()
    assert backend.take_device_errors() == (16 + 100 + 1, 0)
    want, bound = attention_reference(q, k, v, pos, table, 128 ** -0.5)
    assert ((got[0].double() - want[0]).abs() <= bound[0]).all()
    assert (got[2] == 0).all() and (got[3] == 0).all()
    keep = [t for t in range(100) if not 32 <= t < 48]
    t = torch.tensor(keep, device="cuda")
    kk = k[table[1].long()[t // 16], :, t % 16].double().transpose(0, 1).repeat_interleave(4, 0)
    vv = v[table[1].long()[t // 16], :, t % 16].double().transpose(0, 1).repeat_interleave(4, 0)
    w = torch.softmax(torch.einsum("hd,htd->ht", q[1].double(), kk) * 128 ** -0.5, -1)
    assert (got[1].double() - torch.einsum("ht,htd->hd", w, vv)).abs().max() < 1e-5
    # a position past the block table: the tokens that it holds are used, and it is counted
    far = pos.clone()
    far[0] = 5000
    got = backend.paged_attention(q[:1], cache, far[:1], table)
    backend.synchronize()
    assert backend.take_device_errors() == (1, 0)
    full = torch.tensor([table.shape[1] * 16 - 1], dtype=torch.int32, device="cuda")
    same = backend.paged_attention(q[:1], cache, full, table)
    backend.synchronize()
    assert torch.equal(got, same)


def test_refusals(backend):
    k, v, table = paged([100, 100], 16, 2, 128, torch.bfloat16, 11)
    cache = backend.kv_cache_view(k, v)
    pos = positions_of([100, 100])
    q = torch.randn(2, 8, 128, device="cuda")
    f = backend.paged_attention
    with pytest.raises(KernelError):
        f(q.double(), cache, pos, table)
    with pytest.raises(KernelError):
        f(q.cpu(), cache, pos, table)
    with pytest.raises(KernelError):
        f(q[:, :, :64].contiguous(), cache, pos, table)
    with pytest.raises(KernelError, match="multiple of n_kv_heads"):
        f(q[:, :7].contiguous(), cache, pos, table)
    with pytest.raises(KernelError):
        f(q, cache, pos.long(), table)
    with pytest.raises(KernelError, match="positions"):
        f(q, cache, pos[:1], table)
    with pytest.raises(KernelError, match="exceed"):
        f(q, cache, pos, table[:1])
    with pytest.raises(KernelError, match="scale"):
        f(q, cache, pos, table, scale=0.0)
    with pytest.raises(KernelError, match="scale"):
        f(q, cache, pos, table, scale=float("nan"))
    with pytest.raises(KernelError, match="overlaps"):
        f(q, cache, pos, table, out=q)
    with pytest.raises(KernelError, match="16-byte"):
        f(torch.randn(2 * 8 * 128 + 1, device="cuda")[1:].view(2, 8, 128), cache, pos, table)
    with pytest.raises(UnsupportedError):
        backend.kv_cache_view(k.float(), v.float())
    with pytest.raises(UnsupportedError):
        backend.kv_cache(4, 16, 2, 80)
    with pytest.raises(KernelError):
        backend.kv_cache_view(k, v[:, :, :8])


# (k/v heads, query heads of each, head_dim, type, rows of each sequence, tokens): the layouts of the query heads
# (up to 4 of them, more, rows of a sequence together), one warp to an item, and items that several CTAs share.
LAYOUTS = [(2, 4, 128, torch.bfloat16, 1, 90), (2, 4, 64, torch.float16, 1, 90), (2, 7, 96, torch.bfloat16, 1, 90),
           (2, 8, 256, torch.float16, 1, 90), (2, 8, 256, torch.bfloat16, 1, 90), (2, 4, 128, torch.bfloat16, 4, 90),
           (2, 2, 64, torch.float16, 4, 90), (2, 1, 256, torch.bfloat16, 4, 90), (8, 3, 128, torch.bfloat16, 100, 30),
           (2, 4, 128, torch.bfloat16, 1, 20000), (2, 8, 128, torch.float16, 1, 20000), (2, 4, 128, torch.float16, 4, 20000)]


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("kv_heads,group,dim,dtype,rows,n", LAYOUTS)
def test_infinite_key_that_a_row_sees_makes_its_heads_nan(backend, kv_heads, group, dim, dtype, rows, n, bad):
    """Whatever the signs of the query: a score of minus infinity does not leave its token out silently."""
    k, v, table = paged([n, n], 16, kv_heads, dim, dtype, 3)
    if rows > 1:
        table = torch.nn.functional.pad(table, (0, 3000), value=-1)  # room for long sequences
    seqs = torch.arange(2, dtype=torch.int32, device="cuda").repeat_interleave(rows)
    pos = (n - rows + torch.arange(rows, dtype=torch.int32, device="cuda")).clamp(min=0).repeat(2)
    q = torch.randn(2 * rows, kv_heads * group, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    want, bound = attention_reference(q, k, v, pos, table, dim ** -0.5, seqs)
    at = n - 5  # a token that only later rows of sequence 0 see
    k[table[0, at // 16].long(), 1, at % 16, 9] = bad
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs if rows > 1 else None)
    backend.synchronize()
    hit = torch.zeros(2 * rows, kv_heads, group, dtype=torch.bool, device="cuda")
    hit[:rows, 1] = (pos[:rows] >= at)[:, None]
    hit = hit.view(2 * rows, kv_heads * group)
    assert torch.isnan(got[hit]).all()
    assert ((got.double() - want).abs() <= bound)[~hit].all()


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("kv_heads,group,dim,dtype,rows,n", LAYOUTS)
def test_infinite_value_that_a_row_sees_makes_its_element_nan(backend, kv_heads, group, dim, dtype, rows, n, bad):
    k, v, table = paged([n, n], 16, kv_heads, dim, dtype, 3)
    if rows > 1:
        table = torch.nn.functional.pad(table, (0, 3000), value=-1)  # room for long sequences
    seqs = torch.arange(2, dtype=torch.int32, device="cuda").repeat_interleave(rows)
    pos = (n - rows + torch.arange(rows, dtype=torch.int32, device="cuda")).clamp(min=0).repeat(2)
    q = torch.randn(2 * rows, kv_heads * group, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    want, bound = attention_reference(q, k, v, pos, table, dim ** -0.5, seqs)
    at = n - 5
    v[table[0, at // 16].long(), 1, at % 16, 9] = bad
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs if rows > 1 else None)
    backend.synchronize()
    hit = torch.zeros(2 * rows, kv_heads, group, dim, dtype=torch.bool, device="cuda")
    hit[:rows, 1, :, 9] = (pos[:rows] >= at)[:, None]
    hit = hit.view(got.shape)
    assert torch.isnan(got[hit]).all()
    assert ((got.double() - want).abs() <= bound)[~hit].all()
