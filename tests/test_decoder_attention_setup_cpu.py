"""CPU: when a decoder sets up its attention, over a backend that only writes down its calls (no GPU)."""
import types

import pytest
import torch

from ocelotl_b200 import gguf
from ocelotl_b200.errors import InvalidRequestError, KernelError, UnsupportedError
from ocelotl_b200.model import QuantizedDecoderLinears
from tests.gguf_writer import write_gguf
from tests.model_files import decoder_tensors
from tests.test_attention_plan_cpu import META, f32


class HostBackend:
    torch_device = torch.device("cpu")

    def __init__(self):
        self.tables, self.refuse = [], False

    def upload_quant(self, *args):
        return types.SimpleNamespace(quant=types.SimpleNamespace(free=lambda: None))

    def pair_gated(self, gate, up):
        return types.SimpleNamespace()

    def rope_table(self, rot_dim, base, factors=None, interleaved=False):
        if self.refuse:
            raise KernelError("host", "rope_create: refused")
        self.tables.append((rot_dim, base, None if factors is None else list(factors), interleaved))
        return self.tables[-1]

    def qk_norm_rope(self, qkv, cache, positions, block_table, rope, q_norm=None, k_norm=None, eps=None, seqs=None, out=None):
        assert rope is self.tables[-1]
        return torch.zeros(qkv.shape[0], 4, 64) if q_norm is None else q_norm.repeat(qkv.shape[0], 4, 1)

    def paged_attention(self, q, cache, positions, block_table, scale=None, seqs=None, out=None):
        return q


def decoder(tmp_path, meta, backend):
    f = tmp_path / "m.gguf"
    write_gguf(f, decoder_tensors(n_layers=2) + [f32("blk.1.attn_q_norm.weight", 64), f32("blk.1.attn_k_norm.weight", 64)])
    m = gguf.inspect(f)
    m.metadata.update(meta)
    return f, QuantizedDecoderLinears(backend, m)


def test_attention_is_set_up_with_the_model(tmp_path):
    """Its first call makes no table, copies nothing and reads no file: it may be a captured one."""
    b = HostBackend()
    f, model = decoder(tmp_path, {**META, "qwen3.rope.scaling.factor": 2.0}, b)
    assert b.tables == [(64, 1e6, [2.0] * 32, False)]
    f.unlink()
    for i in range(2):
        a = model.attention(i, torch.zeros(3, 6 * 64), None, None, None)
        assert a.shape == (3, 4 * 64) and (a == i).all()  # layer 1 has head norms, of ones
    assert len(b.tables) == 1


@pytest.mark.parametrize("change,error", [
    ({"general.architecture": "other"}, UnsupportedError), ({"qwen3.attention.head_count": 3}, InvalidRequestError),
    ({"qwen3.rope.scaling.type": "yarn"}, UnsupportedError), ({"qwen3.attention.key_length": [64]}, Exception),
    ({"qwen3.rope.freq_base": "far"}, ValueError),
])
def test_linear_layers_serve_where_attention_does_not(tmp_path, change, error):
    """The model loads; what asks for attention says why there is none, each time."""
    _, model = decoder(tmp_path, {**META, **change}, HostBackend())
    assert len(model.layers) == 2
    for _ in range(2):
        with pytest.raises(error):
            model.attention(0, torch.zeros(1, 6 * 64), None, None, None)
        with pytest.raises(error):
            model.kv_caches(4)


def test_file_without_attention_metadata(tmp_path):
    _, model = decoder(tmp_path, {}, HostBackend())
    with pytest.raises(InvalidRequestError, match="general.architecture"):
        model.kv_caches(4)


def test_refused_table_is_tried_again(tmp_path):
    b = HostBackend()
    b.refuse = True
    _, model = decoder(tmp_path, META, b)
    with pytest.raises(KernelError, match="refused"):
        model.attention(0, torch.zeros(1, 6 * 64), None, None, None)
    b.refuse = False
    assert model.attention(0, torch.zeros(1, 6 * 64), None, None, None).shape == (1, 4 * 64)


def test_no_rows(tmp_path):
    _, model = decoder(tmp_path, META, HostBackend())
    assert model.attention(0, torch.zeros(0, 6 * 64), None, None, None).shape == (0, 4 * 64)
