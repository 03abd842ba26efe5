"""GPU: paged attention keeps f32 precision in every layout, by the norm of its error."""
import pytest
import torch

from tests.attention_precision import NORM, norm_error
from tests.decode_cases import attention_reference, paged

pytestmark = pytest.mark.gpu


def run(backend, lengths, kv_heads, group, dim, dtype, seqs=None, pos=None, room=0, check=None):
    """Error of the rows `check` (all) as a whole."""
    k, v, table = paged(lengths, 16, kv_heads, dim, dtype, dim + group)
    table = torch.nn.functional.pad(table, (0, room), value=-1)
    if pos is None:
        pos = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda")
    q = torch.randn(len(pos), kv_heads * group, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(group))
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs)
    backend.synchronize()
    at = slice(None) if check is None else check
    whose = torch.arange(len(pos), device="cuda") if seqs is None else seqs
    want, _ = attention_reference(q[at], k, v, pos[at], table, dim ** -0.5, whose[at])
    return norm_error(got[at], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 5, 8, 9])
def test_rows_by_themselves(backend, group, dim, dtype):
    assert run(backend, [200, 700, 1500, 3000, 333, 2048], 2, group, dim, dtype) < NORM


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 4, 8])
def test_rows_of_a_sequence(backend, group, dim, dtype):
    lengths = [900, 2500]
    seqs = torch.arange(2, dtype=torch.int32, device="cuda").repeat_interleave(9)
    pos = torch.cat([n - 9 + torch.arange(9, dtype=torch.int32, device="cuda") for n in lengths])
    assert run(backend, lengths, 2, group, dim, dtype, seqs, pos, room=3000) < NORM


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [3, 6])
def test_many_items(backend, group, dim, dtype):
    assert run(backend, [40 + i * 53 % 200 for i in range(240)], 8, group, dim, dtype) < NORM


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,dim", [(4, 128), (2, 64), (1, 96), (4, 256)])
def test_many_items_of_several_rows(backend, group, dim, dtype):
    seqs = torch.arange(120, dtype=torch.int32, device="cuda").repeat_interleave(20)
    pos = torch.arange(100, 120, dtype=torch.int32, device="cuda").repeat(120)
    assert run(backend, [120] * 120, 8, group, dim, dtype, seqs, pos, check=slice(600, 800)) < NORM


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,dim", [(4, 128), (8, 256), (2, 64)])
def test_one_row_over_many_ctas(backend, group, dim, dtype):
    assert run(backend, [4000], 1, group, dim, dtype) < NORM


@pytest.mark.parametrize("group,rows", [(4, 1), (8, 1), (2, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_infinite_query_makes_its_head_nan(backend, bad, dtype, group, rows):
    k, v, table = paged([300], 16, 2, 128, dtype, 3)
    table = torch.nn.functional.pad(table, (0, 5000), value=-1)
    pos, seqs = torch.arange(300 - rows, 300, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    q = torch.randn(rows, 2 * group, 128, device="cuda")
    want, bound = attention_reference(q, k, v, pos, table, 128 ** -0.5, seqs)
    q[0, 1, 77] = bad
    got = backend.paged_attention(q, backend.kv_cache_view(k, v), pos, table, seqs=seqs)
    backend.synchronize()
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = want[0, 1].float()
    assert ((got.double() - want).abs() <= bound + 1e-6 * want.abs()).all()
