"""CPU: what the paged cache, the logit rules and the decode-step calls refuse before they reach the C ABI."""
import types

import pytest
import torch

from ocelotl_b200.backend import CudaKernelBackend
from ocelotl_b200.decode import LogitRules, PagedKvCache
from ocelotl_b200.errors import KernelError, UnsupportedError

CPU = torch.device("cpu")


def kv(pages=4, heads=2, page=16, dim=64, dtype=torch.bfloat16):
    return torch.zeros(pages, heads, page, dim, dtype=dtype), torch.zeros(pages, heads, page, dim, dtype=dtype)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_cache_description():
    c = PagedKvCache(*kv())
    assert (c.desc.n_pages, c.desc.page_size, c.desc.n_kv_heads, c.desc.head_dim) == (4, 16, 2, 64)
    assert (c.desc.page_stride, c.desc.head_stride, c.desc.token_stride) == (2 * 16 * 64, 16 * 64, 64) and c.desc.dtype == 30
    k, v = (t.transpose(1, 2) for t in kv(heads=16, page=2, dtype=torch.float16))  # tokens outside heads
    c = PagedKvCache(k, v)
    assert (c.desc.page_stride, c.desc.head_stride, c.desc.token_stride) == (16 * 2 * 64, 64, 2 * 64) and c.desc.dtype == 1
    k, v = kv(pages=1, heads=1, page=1)
    c = PagedKvCache(k.as_strided((1, 1, 1, 64), (0, 0, 0, 1)), v.as_strided((1, 1, 1, 64), (0, 0, 0, 1)))
    assert c.desc.page_stride == c.desc.head_stride == c.desc.token_stride == 64


def test_cache_refusals():
    k, v = kv()
    for bad in ((k[0], v[0]), (k, v[:2]), (k, v.half()), (k, v.transpose(1, 2)), (k[:0], v[:0]), (k[..., ::2], v[..., ::2])):
        with pytest.raises((KernelError, UnsupportedError)):
            PagedKvCache(*bad)
    for dim in (32, 80, 512):
        with pytest.raises(UnsupportedError, match="head_dim"):
            PagedKvCache(*kv(dim=dim))
    with pytest.raises(UnsupportedError, match="cache type"):
        PagedKvCache(*kv(dtype=torch.float32))


def test_rules_description():
    wide = torch.zeros(3, 20, dtype=torch.int32)
    r = LogitRules(CPU, history=wide[:, 2:12], history_lens=i32(1, 2, 3), repetition=torch.ones(3),
                   bias_ids=wide[:, 5:9], bias_values=torch.zeros(3, 20)[:, 1:5], allowed=wide[:, :7])
    assert r.rows == 3 and r.words == 7
    assert (r.desc.history_stride, r.desc.history_max, r.desc.bias_stride, r.desc.bias_count) == (20, 10, 20, 4)
    assert r.desc.allowed_stride == 20 and r.desc.prompt_lens_dev is None and r.desc.frequency_dev is None
    assert LogitRules(CPU).rows is None
    r = LogitRules(CPU, history=wide[:, :0], history_lens=i32(0, 0, 0), presence=torch.ones(3))
    assert r.desc.history_dev is None and r.desc.presence_dev is None


@pytest.mark.parametrize("parts", [
    dict(history=torch.zeros(2, 5, dtype=torch.int32)), dict(repetition=torch.ones(2)),
    dict(bias_ids=torch.zeros(2, 5, dtype=torch.int32)),
    dict(bias_ids=torch.zeros(2, 5, dtype=torch.int32), bias_values=torch.zeros(2, 4)),
    dict(bias_ids=torch.zeros(2, 9, dtype=torch.int32)[:, :5], bias_values=torch.zeros(2, 5)),
    dict(allowed=torch.zeros(2, 5, dtype=torch.int64)), dict(allowed=torch.zeros(5, dtype=torch.int32)),
    dict(allowed=torch.zeros(2, 10, dtype=torch.int32)[:, ::2]), dict(allowed=torch.zeros(1, 5, dtype=torch.int32).expand(3, 5)),
    dict(history=torch.zeros(2, 5, dtype=torch.int32), history_lens=i32(1, 2, 3)),
    dict(history=torch.zeros(2, 5, dtype=torch.int32), history_lens=i32(1, 2), presence=torch.ones(2).double()),
    dict(history=torch.zeros(2, 5, dtype=torch.int32), history_lens=i32(1, 2), presence=torch.ones(1).expand(2)),
])
def test_rules_refusals(parts):
    with pytest.raises(KernelError):
        LogitRules(CPU, **parts)


@pytest.fixture
def host_backend():
    """The Python side of the backend over a C ABI that only writes down its calls."""
    b = CudaKernelBackend.__new__(CudaKernelBackend)
    b.calls = []

    def entry(name):
        def call(*args):
            b.calls.append((name, args))
            return 0
        return call

    b._lib = types.SimpleNamespace(**{n: entry(n) for n in ("ocl_qk_norm_rope", "ocl_paged_attention", "ocl_logits_process")})
    b._ctx, b._stream, b.device_index, b.torch_device = None, 0, 0, CPU
    return b


def test_calls_pass_shapes_and_strides(host_backend):
    b = host_backend
    cache = PagedKvCache(*kv())
    table = torch.zeros(5, 9, dtype=torch.int32)[:, 1:4]
    out = torch.empty(3, 8, 64)
    assert b.qk_norm_rope(torch.zeros(3, 900)[:, :12 * 64], cache, i32(0, 1, 2), table, None, out=out) is out
    name, a = b.calls.pop()
    assert name == "ocl_qk_norm_rope" and a[2:5] == (900, 3, 8)
    q = torch.zeros(3, 12, 64)[:, :8]
    b.paged_attention(q, cache, i32(0, 1, 2), table, out=out)
    name, a = b.calls.pop()
    assert a[2:5] == (12 * 64, 3, 8) and a[7] == 0.125
    import struct
    assert struct.unpack("PPPNNN", a[6])[3:] == (5, 3, 9)
    x = torch.zeros(2, 40)[:, :33]
    b.process_logits(x, LogitRules(CPU), out=x)
    name, a = b.calls.pop()
    assert a[2:5] == (40, 2, 33) and a[1] == a[6] and a[7] == 40 and a[8] is None


def test_calls_refuse(host_backend):
    b = host_backend
    cache = PagedKvCache(*kv())
    table, pos = torch.zeros(2, 3, dtype=torch.int32), i32(0, 1)
    q, out = torch.zeros(2, 8, 64), torch.empty(2, 8, 64)
    for bad in (dict(q=q.half()), dict(q=q[0]), dict(q=q[..., ::2]), dict(q=torch.zeros(2, 8, 128)), dict(q=q.transpose(1, 2)),
                dict(pos=pos.long()), dict(pos=pos[:1]), dict(pos=pos[None]), dict(table=table[0]), dict(table=table.float()),
                dict(cache="no"), dict(seqs=i32(0)), dict(seqs=pos.long()), dict(out=out[:1]), dict(out=out.double())):
        with pytest.raises(KernelError):
            b.paged_attention(bad.get("q", q), bad.get("cache", cache), bad.get("pos", pos), bad.get("table", table),
                              seqs=bad.get("seqs"), out=bad.get("out", out))
    qkv = torch.zeros(2, 12 * 64)
    for bad in (dict(qkv=qkv[:, :700]), dict(qkv=qkv[:, :4 * 64]), dict(q_norm=torch.ones(32)), dict(k_norm=torch.ones(64).double()),
                dict(pos=pos[:1]), dict(out=out[:, :7])):
        with pytest.raises(KernelError):
            b.qk_norm_rope(bad.get("qkv", qkv), cache, bad.get("pos", pos), table, None, q_norm=bad.get("q_norm"),
                           k_norm=bad.get("k_norm"), out=bad.get("out", out))
    x, rules = torch.zeros(2, 40), LogitRules(CPU, allowed=torch.zeros(2, 2, dtype=torch.int32))
    for bad in (dict(x=x.half()), dict(x=torch.zeros(3, 40)), dict(x=torch.zeros(2, 65)), dict(out=torch.zeros(2, 39)),
                dict(ids=torch.zeros(3, dtype=torch.int32)), dict(ids=torch.zeros(2)), dict(rules=None)):
        with pytest.raises(KernelError):
            b.process_logits(bad.get("x", x), bad.get("rules", rules), out=bad.get("out", torch.zeros(2, 40)), ids=bad.get("ids"))
    assert not b.calls
