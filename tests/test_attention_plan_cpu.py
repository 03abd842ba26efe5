"""CPU: what a GGUF file's metadata says about a decoder's attention (no GPU)."""
import numpy as np
import pytest

from ocelotl_b200 import gguf
from ocelotl_b200.errors import InvalidRequestError, UnsupportedError
from ocelotl_b200.model import attention_plan, plan
from tests.gguf_writer import write_gguf
from tests.model_files import decoder_tensors

META = {"general.architecture": "qwen3", "qwen3.attention.head_count": 4, "qwen3.attention.head_count_kv": 1,
        "qwen3.attention.layer_norm_rms_epsilon": 1e-5, "qwen3.rope.freq_base": 1e6}


def manifest(tmp_path, meta=None, extra=()):
    f = tmp_path / "m.gguf"
    write_gguf(f, decoder_tensors(n_layers=2) + list(extra))
    m = gguf.inspect(f)
    m.metadata.update(META if meta is None else meta)
    return m


def f32(name, n):
    return name, [n], 0, np.ones(n, np.float32).tobytes()


def test_heads_rotation_and_norms(tmp_path):
    m = manifest(tmp_path, extra=[f32("blk.1.attn_q_norm.weight", 64), f32("blk.1.attn_k_norm.weight", 64),
                                  f32("rope_freqs.weight", 32)])
    a = attention_plan(m, plan(m))
    assert (a.n_heads, a.n_kv_heads, a.head_dim, a.rot_dim) == (4, 1, 64, 64)
    assert a.scale == 0.125 and a.rope_base == 1e6 and a.eps == 1e-5 and a.rope_scale == 1.0 and not a.interleaved
    assert a.q_norm == [None, "blk.1.attn_q_norm.weight"] and a.k_norm == [None, "blk.1.attn_k_norm.weight"]
    assert a.rope_factors == "rope_freqs.weight"


def test_linear_scaling_and_pairs(tmp_path):
    meta = {k.replace("qwen3", "llama"): v for k, v in META.items()}
    meta.update({"general.architecture": "llama", "llama.rope.scaling.type": "linear", "llama.rope.scaling.factor": 4.0,
                 "llama.rope.dimension_count": 32})
    m = manifest(tmp_path, meta)
    a = attention_plan(m, plan(m))
    assert a.interleaved and a.rope_scale == 4.0 and a.rot_dim == 32 and a.q_norm == [None, None]


@pytest.mark.parametrize("change,error", [
    ({"general.architecture": "other"}, UnsupportedError), ({"qwen3.attention.head_count": None}, InvalidRequestError),
    ({"qwen3.attention.head_count": 3}, InvalidRequestError), ({"qwen3.attention.head_count_kv": [1, 1]}, UnsupportedError),
    ({"qwen3.attention.head_count_kv": 3}, InvalidRequestError), ({"qwen3.attention.value_length": 32}, UnsupportedError),
    ({"qwen3.attention.sliding_window": 512}, UnsupportedError), ({"qwen3.rope.scaling.type": "yarn"}, UnsupportedError),
    ({"qwen3.attention.layer_norm_rms_epsilon": None}, InvalidRequestError),
])
def test_what_is_not_served_is_named(tmp_path, change, error):
    meta = {**META, **change}
    m = manifest(tmp_path, {k: v for k, v in meta.items() if v is not None})
    p = plan(m)  # the linear layers stay available
    with pytest.raises(error):
        attention_plan(m, p)


def test_norms_of_another_shape(tmp_path):
    m = manifest(tmp_path, extra=[f32("blk.0.attn_q_norm.weight", 32)])
    with pytest.raises(InvalidRequestError, match="attn_q_norm"):
        attention_plan(m, plan(m))


def llama(**meta):
    return {**{k.replace("qwen3", "llama"): v for k, v in META.items()}, "general.architecture": "llama",
            **{"llama.rope." + k.replace("__", "."): v for k, v in meta.items()}}


@pytest.mark.parametrize("stated,scale", [
    ({"scaling__factor": 4.0}, 4.0), ({"scale_linear": 4.0}, 4.0), ({"scaling__type": "linear", "scale_linear": 2.5}, 2.5),
    ({"scaling__factor": 2.0, "scale_linear": 8.0}, 2.0), ({"scaling__factor": 8}, 8.0), ({"scaling__type": "linear"}, 1.0),
    ({"scaling__type": "none", "scaling__factor": 4.0, "scale_linear": 4.0}, 1.0), ({"scaling__factor": 1.0}, 1.0), ({}, 1.0),
])
def test_position_scaling_that_a_file_states(tmp_path, stated, scale):
    """A factor is linear scaling unless a type says otherwise; the older key counts where the newer is missing."""
    m = manifest(tmp_path, llama(**stated))
    assert attention_plan(m, plan(m)).rope_scale == scale


@pytest.mark.parametrize("stated,error", [
    ({"scaling__type": "linear", "scaling__factor": 0.0}, InvalidRequestError), ({"scaling__factor": 0.0}, InvalidRequestError),
    ({"scaling__factor": -2.0}, InvalidRequestError), ({"scale_linear": float("nan")}, InvalidRequestError),
    ({"scale_linear": float("inf")}, InvalidRequestError), ({"scaling__factor": "4"}, InvalidRequestError),
    ({"scaling__factor": [4.0]}, InvalidRequestError), ({"scaling__type": "yarn", "scaling__factor": 4.0}, UnsupportedError),
    ({"scaling__type": "yarn", "scale_linear": 4.0}, UnsupportedError),
])
def test_position_scaling_that_is_refused(tmp_path, stated, error):
    m = manifest(tmp_path, llama(**stated))
    with pytest.raises(error, match="scal"):
        attention_plan(m, plan(m))


@pytest.mark.parametrize("key,value", [("attention.causal", False), ("attention.clamp_kqv", 8.0), ("attention.max_alibi_bias", 8.0)])
def test_attention_of_another_kind_is_refused(tmp_path, key, value):
    m = manifest(tmp_path, {**META, "qwen3." + key: value})
    with pytest.raises(UnsupportedError, match=key):
        attention_plan(m, plan(m))
    m.metadata["qwen3." + key] = True if value is False else 0.0  # as good as absent
    assert attention_plan(m, plan(m)).n_heads == 4
