"""CPU: the norm that the GPU tests of paged attention allow tells its precision from that with a piece lost."""
import pytest
import torch

from tests.attention_precision import NORM, attention_in_pieces, norm_error


@pytest.mark.parametrize("n", [200, 3000])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,all_pieces", [(torch.bfloat16, 3), (torch.float16, 2)])
def test_a_lost_piece_shows(dtype, all_pieces, dim, n):
    g = torch.Generator().manual_seed(dim + n)
    q = torch.randn(32, dim, generator=g)
    k, v = (torch.randn(n, dim, generator=g).to(dtype) for _ in range(2))
    want = torch.softmax(q.double() @ k.double().T * dim ** -0.5, -1) @ v.double()

    def off(q_pieces, p_pieces):
        return norm_error(attention_in_pieces(q, k, v, dim ** -0.5, dtype, q_pieces, p_pieces), want)

    assert off(all_pieces, all_pieces) < NORM / 3
    assert off(all_pieces - 1, all_pieces) > 1.25 * NORM  # q's last piece
    assert off(all_pieces, all_pieces - 1) > 1.25 * NORM  # that of the weights
