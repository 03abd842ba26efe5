"""GPU: a decoder's steps through QuantizedDecoderLinears: prompt rows, then one token at a
time, eagerly and as a captured graph, with the logit rules at the end."""
import numpy as np
import pytest
import torch

from tests.decode_cases import attention_reference, rope_reference
from tests.test_attention_plan_cpu import META

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE = 4, 1, 64, 16
PROMPTS = [[5, 17, 900, 3, 3, 41, 7, 7, 7, 12, 99, 250, 251, 252, 253, 254, 255, 256, 1], [8, 1, 1]]


def f32_tensor(name, values):
    return name, [len(values)], 0, np.asarray(values, np.float32).tobytes()


@pytest.fixture(scope="module", params=["qwen3", "llama"])
def model(request, backend, tmp_path_factory):
    from ocelotl_b200 import gguf
    from ocelotl_b200.model import QuantizedDecoderLinears
    from tests.gguf_writer import write_gguf
    from tests.model_files import decoder_tensors
    rng = np.random.default_rng(5)
    t = decoder_tensors(n_layers=2)
    if request.param == "qwen3":
        t += [f32_tensor(f"blk.{i}.attn_{s}_norm.weight", 1 + 0.2 * rng.standard_normal(DIM)) for i in range(2) for s in "qk"]
    else:
        t += [f32_tensor("rope_freqs.weight", 1 + rng.random(DIM // 2))]
    f = tmp_path_factory.mktemp("d") / "decoder.gguf"
    write_gguf(f, t)
    m = gguf.inspect(f)
    m.metadata.update({k.replace("qwen3", request.param): v for k, v in META.items()})
    m.metadata["general.architecture"] = request.param
    return QuantizedDecoderLinears(backend, m)


class Run:
    """The caller's side: caches, tables, histories, residual norms, and buffers that stay in place."""

    def __init__(self, model, dtype):
        self.m, b = model, model.backend
        self.caches = model.kv_caches(12, PAGE, dtype)
        self.table = torch.tensor([[7, 2, 9], [4, 0, 11]], dtype=torch.int32, device="cuda")
        self.history = torch.full((2, 64), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor([len(p) for p in PROMPTS], dtype=torch.int32, device="cuda")
        for r, p in enumerate(PROMPTS):
            self.history[r, :len(p)] = torch.tensor(p, dtype=torch.int32)
        mask = torch.full((2, (model.plan.vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
        mask[1] &= 0x55555555  # only even tokens for the second
        self.rules = b.logit_rules(
            history=self.history, history_lens=self.lens, prompt_lens=self.lens.clone(),
            repetition=torch.tensor([1.3, 1.0], device="cuda"), frequency=torch.tensor([0.2, 0.5], device="cuda"),
            presence=torch.tensor([0.1, 0.0], device="cuda"), allowed=mask,
            bias_ids=torch.tensor([[3, -1], [10, 12]], dtype=torch.int32, device="cuda"),
            bias_values=torch.tensor([[2.0, 0.0], [-50.0, 1.0]], device="cuda"))
        self.positions = self.lens - 1
        self.ids = torch.tensor([p[-1] for p in PROMPTS], dtype=torch.int32, device="cuda")
        self.last_logits = self.seen = None

    def norm(self, h):
        return (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5)).contiguous()

    def layers(self, h, rows, positions, seqs, watch=None):
        m, p = self.m, self.m.plan
        for i in range(len(p.layers)):
            qkv = torch.empty(rows, (HEADS + 2 * KV_HEADS) * DIM, device="cuda")
            m.qkv(i, self.norm(h), rows, qkv)
            a = m.attention(i, qkv, self.caches[i], positions, self.table, seqs=seqs)
            if watch:
                watch(i, qkv, a)
            o, act, mlp = (torch.empty(rows, n, device="cuda") for n in (p.hidden, p.intermediate, p.hidden))
            m.o(i, a, rows, o)
            h = h + o
            m.mlp(i, self.norm(h), rows, act, mlp)
            h = h + mlp
        return h

    def prefill(self, watch=None):
        """Every prompt token but the last of each sequence, in one pass; two padding rows at the end."""
        rows = [(t, s, i) for s, p in enumerate(PROMPTS) for i, t in enumerate(p[:-1])] + [(0, 0, -1)] * 2
        ids, seqs, pos = (torch.tensor([r[k] for r in rows], dtype=torch.int32, device="cuda") for k in range(3))
        self.layers(self.m.embed(ids), len(rows), pos, seqs, (lambda i, qkv, a: watch(i, qkv, a, pos, seqs)) if watch else None)

    def step(self, watch=None):
        pos = self.positions
        h = self.layers(self.m.embed(self.ids), 2, pos, None, (lambda i, qkv, a: watch(i, qkv, a, pos, None)) if watch else None)
        ids, self.last_logits = self.m.head_argmax(self.norm(h), 2, rules=self.rules)
        self.seen = self.history.clone(), self.lens.clone()
        self.ids.copy_(ids)
        self.history.scatter_(1, self.lens.long()[:, None], ids[:, None])
        self.lens.add_(1)
        self.positions.add_(1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_and_steps(backend, oracle, model, dtype):
    from ocelotl_b200.gguf import read_payload
    from tests.test_gpu_logits import reference
    backend.take_device_errors()
    run = Run(model, dtype)
    plan, _, qn, kn = model._attention_parts()
    factors = None if plan.rope_factors is None else \
        np.array(read_payload(model._manifest, plan.rope_factors)).view(np.float32).tolist()

    def watch(i, qkv, a, pos, seqs):
        torch.cuda.synchronize()
        (q, _), _, _ = rope_reference(qkv, HEADS, KV_HEADS, DIM, pos.clamp(min=0), DIM, 1e6, plan.interleaved, qn[i], kn[i], plan.eps,
                                      factors)
        want, bound = attention_reference(q, run.caches[i].k, run.caches[i].v, pos, run.table, plan.scale, seqs)
        # the kernel's own q is off by up to 16 units of 2^-24 of its pairs: as much again in each score
        k_max = run.caches[i].k.double().abs().max().item()
        more = 2 * 32 * 2.0 ** -24 * q.abs().sum(-1).amax().item() * k_max * plan.scale * run.caches[i].v.double().abs().max().item()
        assert ((a.view(want.shape).double() - want).abs() <= bound + more).all()

    run.prefill(watch)
    picks = []
    for _ in range(5):
        run.step(watch)
        torch.cuda.synchronize()
        hist, lens = (t.cpu().numpy() for t in run.seen)
        parts = {n: t.cpu().numpy() for n, t in run.rules.parts.items()}
        ruled = reference(run.last_logits.cpu().numpy(), **{**parts, "history": hist, "history_lens": lens})
        assert run.ids.tolist() == [oracle.greedy_sample_fast(r) for r in ruled]
        assert run.ids[1] % 2 == 0
        picks.append(run.ids.tolist())
    assert backend.take_device_errors() == (0, 0)

    # the same as a captured step, replayed: the same tokens
    other = Run(model, dtype)
    other.prefill()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            backend.use_current_stream()
            other.step()
    finally:
        backend.set_stream(None)
    got = []
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        got.append(other.ids.tolist())
    assert got == picks
    for a, b in zip(run.caches, other.caches):
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    assert backend.take_device_errors() == (0, 0)


def test_first_calls_of_a_context_may_be_captured():
    """Nothing is allocated or set up by a first call that a capture would refuse."""
    from ocelotl_b200 import CudaKernelBackend
    b = CudaKernelBackend(0)
    cache = b.kv_cache(4, 16, 1, 96, torch.float16)
    rope = b.rope_table(96, 1e4)
    qkv, pos = torch.randn(1, 5 * 96, device="cuda"), torch.tensor([0], dtype=torch.int32, device="cuda")
    table = torch.tensor([[2]], dtype=torch.int32, device="cuda")
    logits, ids = torch.randn(1, 777, device="cuda"), torch.full((1,), -1, dtype=torch.int32, device="cuda")
    rules = b.logit_rules()
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.use_current_stream()
        out = b.paged_attention(b.qk_norm_rope(qkv, cache, pos, table, rope), cache, pos, table)
        b.greedy_sample(logits, out=ids, rules=rules)
    b.set_stream(None)
    graph.replay()
    torch.cuda.synchronize()
    # one token: the softmax is 1 and the output is the value as cached
    v = qkv[0, 4 * 96:].half().float()
    assert (out[0] - v).abs().max() <= 2.0 ** -20 * v.abs().max()
    assert ids.item() == int(logits.argmax())


def test_two_contexts_on_two_streams(backend):
    """A context per stream: their calls may overlap on the GPU."""
    from ocelotl_b200 import CudaKernelBackend
    from tests.decode_cases import paged
    k, v, table = paged([20000], 16, 2, 128, torch.bfloat16, 3)
    q = torch.randn(1, 8, 128, device="cuda")
    pos = torch.tensor([19999], dtype=torch.int32, device="cuda")
    cache = backend.kv_cache_view(k, v)
    want = backend.paged_attention(q, cache, pos, table)
    torch.cuda.synchronize()
    streams, contexts, got = [torch.cuda.Stream() for _ in range(2)], [CudaKernelBackend(0) for _ in range(2)], []
    for _ in range(20):
        for s, b in zip(streams, contexts):
            with torch.cuda.stream(s):
                b.use_current_stream()
                got.append(b.paged_attention(q, cache, pos, table))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("busy", ["current", "kernels"])
def test_new_cache_is_zeroed_before_either_stream_writes(busy):
    """kv_cache's zeros precede the kernels' writes and the caller's, whichever stream is behind."""
    from ocelotl_b200 import CudaKernelBackend
    b, side = CudaKernelBackend(0), torch.cuda.Stream()
    qkv, pos = torch.ones(1, 3 * 64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    b.set_stream(side)
    b.qk_norm_rope(qkv, b.kv_cache(1, 16, 1, 64), pos, table, None)  # modules are loaded
    torch.cuda.synchronize()
    with torch.cuda.stream(side if busy == "kernels" else torch.cuda.current_stream()):
        torch.cuda._sleep(50_000_000)  # some 30 ms
    cache = b.kv_cache(1, 16, 1, 64)
    if busy == "kernels":
        cache.k.fill_(1.0)
        cache.v.fill_(1.0)
    else:
        b.qk_norm_rope(qkv, cache, pos, table, None)
    torch.cuda.synchronize()
    assert (cache.k[0, 0, 0] == 1).all() and (cache.v[0, 0, 0] == 1).all()


@pytest.mark.parametrize("stated", [{"llama.rope.scaling.factor": 4.0}, {"llama.rope.scale_linear": 4.0},
                                    {"llama.rope.scaling.type": "linear", "llama.rope.scaling.factor": 4.0}])
def test_step_of_a_file_with_scaled_positions(backend, tmp_path, stated):
    """A decode step at the angles that the file asks for, however it states them."""
    from ocelotl_b200 import gguf
    from ocelotl_b200.model import QuantizedDecoderLinears
    from tests.gguf_writer import write_gguf
    from tests.model_files import decoder_tensors
    from tests.test_gpu_rope import UNITS
    f = tmp_path / "scaled.gguf"
    write_gguf(f, decoder_tensors(n_layers=1))
    m = gguf.inspect(f)
    m.metadata.update({k.replace("qwen3", "llama"): v for k, v in META.items()} | {"general.architecture": "llama"} | stated)
    model = QuantizedDecoderLinears(backend, m)
    cache = model.kv_caches(40, PAGE)[0]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:39].to(torch.int32).cuda()[None]
    g = torch.Generator("cuda").manual_seed(2)
    qkv = torch.randn(600, (HEADS + 2 * KV_HEADS) * DIM, device="cuda", generator=g)
    pos, seqs = torch.arange(600, dtype=torch.int32, device="cuda"), torch.zeros(600, dtype=torch.int32, device="cuda")
    q = torch.empty(600, HEADS, DIM, device="cuda")
    model.attention(0, qkv[:599], cache, pos[:599], table, seqs=seqs[:599], q=q[:599])  # the prompt
    got = model.attention(0, qkv[599:], cache, pos[599:], table, q=q[599:])             # one token more
    backend.synchronize()
    (want_q, size), (want_k, k_size), _ = rope_reference(qkv, HEADS, KV_HEADS, DIM, pos, DIM, 1e6, True, None, None, 1e-5, [4.0] * (DIM // 2))
    assert ((q.double() - want_q).abs() <= UNITS * size).all()
    k = cache.k[table[0].long()[pos.long() // PAGE], :, pos.long() % PAGE].double()
    half = torch.finfo(torch.bfloat16).eps / 2
    assert ((k - want_k).abs() <= half * want_k.abs() * (1 + half) + UNITS * k_size * (1 + half) + 1e-38).all()
    want, bound = attention_reference(q[599:], cache.k, cache.v, pos[599:], table, DIM ** -0.5)
    assert ((got.view(want.shape).double() - want).abs() <= bound).all()


def test_first_attention_of_a_decoder_may_be_captured(backend, model):
    """Over the caller's own caches, with nothing called before."""
    from ocelotl_b200.model import QuantizedDecoderLinears
    from tests.test_gpu_rope import UNITS
    fresh = QuantizedDecoderLinears(backend, model._manifest)
    k, v = (torch.zeros(4, KV_HEADS, PAGE, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = backend.kv_cache_view(k, v)
    qkv = torch.randn(1, (HEADS + 2 * KV_HEADS) * DIM, device="cuda")
    pos, table = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([[2]], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            backend.use_current_stream()
            out = fresh.attention(1, qkv, cache, pos, table)
    finally:
        backend.set_stream(None)
    graph.replay()
    torch.cuda.synchronize()
    plan, _, qn, kn = fresh._attention_parts()
    _, (want, size), _ = rope_reference(qkv, HEADS, KV_HEADS, DIM, pos, DIM, 1e6, plan.interleaved, qn[1], kn[1], plan.eps)
    half = torch.finfo(torch.bfloat16).eps / 2
    assert ((k[2, :, 0].double() - want[0]).abs() <= half * want[0].abs() * (1 + half) + UNITS * size[0] * (1 + half) + 1e-38).all()
    # one token: the softmax is 1 and the output is the value as cached
    cached = qkv[0, 5 * DIM:].bfloat16().float()
    assert ((out.view(HEADS, DIM) - cached).abs() <= 2.0 ** -20 * cached.abs().max()).all()
