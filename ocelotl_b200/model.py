"""Quantized linear layers of a Llama / Qwen-style decoder, loaded from a GGUF file.

The reference's Qwen2.5 loader keeps every projection as a pre-transposed f32
matrix and runs it through `matmul` (crates/models/src/qwen/qwen2_5/weights.rs:
150-224: q/k/v with biases, o, gate/up/down per layer; embed_tokens; the head).
This module is the quantized path for the same layers: the GGUF tensors stay
quantized in HBM and run through the fused dequant-GEMV (`linear_d`), with

* q, k and v fused into one weight (their GGUF rows concatenated: rows are
  independent block runs, so concatenation is a byte concatenation) and their
  f32 biases concatenated -- one activation split and one launch per layer;
* gate and up interleaved into one pair for the fused gated MLP
  (`mlp_gated_silu`: silu(gate) * up, then down);
* the output head as a GEMV over the vocabulary followed by greedy argmax on
  the device (`greedy_sample`), with penalties, biases and a grammar mask where a
  request has them, the embedding as a Q8_0 row gather;
* between qkv and o, head norms, rotation and the paged cache write in one launch
  (`qk_norm_rope`) and the attention over the cache in another (`paged_attention`),
  set up from the file's metadata when the model is made.

Tensor names follow the GGUF convention for these models (token_embd.weight,
blk.N.attn_{q,k,v}.{weight,bias}, blk.N.attn_output.weight,
blk.N.ffn_{gate,up,down}.weight, output.weight; a missing head is tied to the
embedding table; blk.N.attn_{q,k}_norm.weight and rope_freqs.weight where a model
has them).  The norms of the residual stream are not part of this path; the caller
runs them between the calls.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import numpy as np

from .errors import InvalidRequestError, UnsupportedError
from .ggml import GgmlType
from .gguf import Manifest, TensorEntry, read_payload

QUANT_TYPES = (GgmlType.Q4_K, GgmlType.Q6_K, GgmlType.Q8_0)
F32 = 0


@dataclass
class LayerPlan:
    """Which GGUF tensors make up one decoder layer's linear projections."""
    index: int
    qkv: list[str]               # q, k, v weights fused in this order
    qkv_bias: list[str]          # their f32 biases (empty if none)
    qkv_rows: list[int]          # output rows of q, k, v
    o: str
    gate: str
    up: str
    down: str


@dataclass
class ModelPlan:
    hidden: int
    intermediate: int
    vocab: int
    embed: str
    head: str                    # == embed when the head is tied
    layers: list[LayerPlan] = field(default_factory=list)


def _need(m: Manifest, name: str) -> TensorEntry:
    try:
        return m.tensor(name)
    except InvalidRequestError:
        raise InvalidRequestError("tensor", f"GGUF file {m.path} has no tensor `{name}`") from None


def _quant(t: TensorEntry) -> None:
    if t.tensor_type not in QUANT_TYPES:
        raise UnsupportedError("quantized weight type", f"{t.name}: {t.tensor_type}",
                               ["Q4_K(12)", "Q6_K(14)", "Q8_0(8)"])


def plan(m: Manifest, n_layers: int | None = None) -> ModelPlan:
    """Map a GGUF manifest to the decoder's linear layers (host only, reads no payload)."""
    emb = _need(m, "token_embd.weight")
    hidden, vocab = emb.k, emb.n_rows
    names = {t.name for t in m.tensors}
    head = "output.weight" if "output.weight" in names else "token_embd.weight"
    count = 0
    while f"blk.{count}.attn_q.weight" in names:
        count += 1
    if n_layers is not None:
        if n_layers > count:
            raise InvalidRequestError("n_layers", f"requested {n_layers} layers, the file has {count}")
        count = n_layers
    out = None
    for i in range(count):
        p = f"blk.{i}."
        ws = [_need(m, p + f"attn_{s}.weight") for s in ("q", "k", "v")]
        for w in ws:
            _quant(w)
            if w.k != hidden:
                raise InvalidRequestError("tensor", f"`{w.name}` in_features {w.k} != hidden {hidden}")
        bias = [p + f"attn_{s}.bias" for s in ("q", "k", "v") if p + f"attn_{s}.bias" in names]
        if bias and len(bias) != 3:
            raise InvalidRequestError("tensor", f"layer {i}: q/k/v biases must be all present or all absent")
        for b in bias:
            if _need(m, b).tensor_type != F32:
                raise UnsupportedError("bias type", f"{b}: {_need(m, b).tensor_type}", ["F32(0)"])
        if len({w.tensor_type for w in ws}) != 1:  # fusion concatenates rows of one block format
            raise UnsupportedError("q/k/v of different quant types", str([int(w.tensor_type) for w in ws]),
                                   ["one type for q, k and v"])
        gate, up, down = (_need(m, p + f"ffn_{s}.weight") for s in ("gate", "up", "down"))
        for w in (gate, up, down):
            _quant(w)
        if gate.tensor_type != up.tensor_type or gate.n_rows != up.n_rows or gate.k != up.k:
            raise InvalidRequestError("tensor", f"layer {i}: ffn_gate and ffn_up differ in type or shape")
        if down.k != gate.n_rows or down.n_rows != hidden:
            raise InvalidRequestError("tensor", f"layer {i}: ffn_down is [{down.n_rows} x {down.k}], expected "
                                                f"[{hidden} x {gate.n_rows}]")
        o = _need(m, p + "attn_output.weight")
        _quant(o)
        lp = LayerPlan(i, [w.name for w in ws], bias, [w.n_rows for w in ws], o.name, gate.name, up.name,
                       down.name)
        if out is None:
            out = ModelPlan(hidden, gate.n_rows, vocab, emb.name, head)
        elif gate.n_rows != out.intermediate:
            raise InvalidRequestError("tensor", f"layer {i}: intermediate {gate.n_rows} != {out.intermediate}")
        out.layers.append(lp)
    if out is None:
        out = ModelPlan(hidden, 0, vocab, emb.name, head)
    _quant(_need(m, head))
    return out


@dataclass
class AttentionPlan:
    """What the metadata says about the attention of every layer."""
    n_heads: int
    n_kv_heads: int
    head_dim: int
    scale: float
    rot_dim: int
    rope_base: float
    rope_scale: float            # every frequency is divided by it (linear position scaling, 1 = none)
    rope_factors: str | None     # tensor of per-pair frequency divisors
    interleaved: bool            # pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)
    eps: float
    q_norm: list[str | None] = field(default_factory=list)
    k_norm: list[str | None] = field(default_factory=list)


# How an architecture's files pair the elements that a rotation turns together.
ROPE_INTERLEAVED = {"llama": True, "qwen2": False, "qwen3": False}


def _rope_scale(m: Manifest, arch: str) -> float:
    """Linear position scaling of a file: 1 where it states none.

    A factor without a type is linear; a type of "none" wins over a factor beside it.
    Older files have `rope.scale_linear` in place of `rope.scaling.factor`.
    """
    kind = m.metadata.get(f"{arch}.rope.scaling.type")
    if kind not in (None, "none", "linear"):
        raise UnsupportedError("rope scaling", str(kind), ["none", "linear"])
    if kind == "none":
        return 1.0
    for key in (f"{arch}.rope.scaling.factor", f"{arch}.rope.scale_linear"):
        if key in m.metadata:
            f = m.metadata[key]
            if isinstance(f, bool) or not isinstance(f, (int, float)) or not 0 < f < math.inf:
                raise InvalidRequestError("metadata", f"`{key}` must be a positive finite number, is {f!r}")
            return float(f)
    return 1.0


def attention_plan(m: Manifest, p: ModelPlan) -> AttentionPlan:
    """Head layout, rotation and head norms of a planned decoder (host only, reads no payload)."""
    def need(key):
        if key not in m.metadata:
            raise InvalidRequestError("metadata", f"GGUF file {m.path} has no `{key}`")
        return m.metadata[key]

    arch = need("general.architecture")
    if arch not in ROPE_INTERLEAVED:
        raise UnsupportedError("attention architecture", str(arch), sorted(ROPE_INTERLEAVED))
    heads = need(f"{arch}.attention.head_count")
    kv = m.metadata.get(f"{arch}.attention.head_count_kv", heads)
    if not isinstance(heads, int) or not isinstance(kv, int):
        raise UnsupportedError("heads per layer", f"{heads} / {kv}", ["one head count for all layers"])
    if heads <= 0 or kv <= 0 or heads % kv:
        raise InvalidRequestError("metadata", f"{heads} heads are not a multiple of {kv} key/value heads")
    dim = m.metadata.get(f"{arch}.attention.key_length", p.hidden // heads)
    if m.metadata.get(f"{arch}.attention.value_length", dim) != dim:
        raise UnsupportedError("attention value_length", str(m.metadata[f"{arch}.attention.value_length"]), [f"key_length={dim}"])
    for feature in ("attention.sliding_window", "attn_logit_softcapping", "attention.clamp_kqv", "attention.max_alibi_bias"):
        if m.metadata.get(f"{arch}.{feature}"):
            raise UnsupportedError(feature, str(m.metadata[f"{arch}.{feature}"]), ["none"])
    if not m.metadata.get(f"{arch}.attention.causal", True):
        raise UnsupportedError("attention.causal", "False", ["True"])
    rope_scale = _rope_scale(m, arch)
    for lp in p.layers:
        if lp.qkv_rows != [heads * dim, kv * dim, kv * dim]:
            raise InvalidRequestError("tensor", f"layer {lp.index}: q/k/v rows {lp.qkv_rows} are not {heads} + 2 * {kv} heads of {dim}")
    names = {t.name for t in m.tensors}

    def norms(s):
        out = []
        for lp in p.layers:
            name = f"blk.{lp.index}.attn_{s}_norm.weight"
            out.append(name if name in names else None)
            if name in names:
                t = m.tensor(name)
                if t.tensor_type != F32:
                    raise UnsupportedError("norm type", f"{name}: {t.tensor_type}", ["F32(0)"])
                if t.shape != [dim]:
                    raise InvalidRequestError("tensor", f"`{name}` has shape {t.shape}, expected [{dim}]")
        return out

    rot = m.metadata.get(f"{arch}.rope.dimension_count", dim)
    factors = "rope_freqs.weight" if "rope_freqs.weight" in names else None
    if factors and (m.tensor(factors).tensor_type != F32 or m.tensor(factors).shape != [rot // 2]):
        raise InvalidRequestError("tensor", f"`{factors}` is not {rot // 2} F32 values")
    return AttentionPlan(
        heads, kv, dim, float(m.metadata.get(f"{arch}.attention.scale", 0.0)) or dim ** -0.5, rot,
        float(m.metadata.get(f"{arch}.rope.freq_base", 10000.0)),
        rope_scale, factors,
        ROPE_INTERLEAVED[arch], float(need(f"{arch}.attention.layer_norm_rms_epsilon")), norms("q"), norms("k"))


def _f32(m: Manifest, name: str) -> np.ndarray:
    return np.frombuffer(bytes(read_payload(m, name)), dtype=np.float32)


def fused_qkv_payload(m: Manifest, lp: LayerPlan) -> tuple[int, np.ndarray, int]:
    """(type, concatenated GGUF rows of q, k, v, total rows)."""
    ts = [m.tensor(n) for n in lp.qkv]
    blob = np.concatenate([np.ascontiguousarray(read_payload(m, t.name)) for t in ts])
    return ts[0].tensor_type, blob, sum(t.n_rows for t in ts)


class QuantizedDecoderLinears:
    """Every linear layer of the decoder resident in HBM, quantized.

    Per layer: `qkv(x, rows, out)` -> [rows, q+k+v] (bias added),
    `attention(i, qkv, cache, ...)` -> [rows, q], `o(...)`, `mlp(x, rows, act, out)`
    (silu(gate)*up then down); plus `kv_caches(...)`, `embed(ids, out)` and
    `head_argmax(h, rows)` -> next token ids on the device.  x / out are contiguous
    f32 torch tensors on the backend's device.
    """

    def __init__(self, backend, manifest: Manifest, n_layers: int | None = None):
        import torch

        from .gguf import upload_quant_tensor
        self.backend = backend
        self.plan = plan(manifest, n_layers)
        self._manifest = manifest
        self._attention = None
        dev = backend.torch_device
        self.layers = []
        for lp in self.plan.layers:
            t, blob, rows = fused_qkv_payload(manifest, lp)
            qkv = backend.upload_quant(t, blob, rows, self.plan.hidden)
            bias = None
            if lp.qkv_bias:
                bias = torch.from_numpy(np.concatenate(
                    [np.frombuffer(bytes(read_payload(manifest, b)), dtype=np.float32) for b in lp.qkv_bias])).to(dev)
            gate = upload_quant_tensor(backend, manifest, lp.gate)
            up = upload_quant_tensor(backend, manifest, lp.up)
            pair = backend.pair_gated(gate, up)
            gate.quant.free()
            up.quant.free()
            self.layers.append({
                "qkv": qkv, "qkv_bias": bias, "qkv_rows": lp.qkv_rows,
                "o": upload_quant_tensor(backend, manifest, lp.o),
                "gate_up": pair,
                "down": upload_quant_tensor(backend, manifest, lp.down),
            })
        self.embed_table = upload_quant_tensor(backend, manifest, self.plan.embed)
        self.head_w = self.embed_table if self.plan.head == self.plan.embed else \
            upload_quant_tensor(backend, manifest, self.plan.head)
        # Made here, so that the first attention() copies and allocates nothing but its outputs and may
        # be a captured one.  A file whose metadata does not serve attention keeps its linear layers:
        # what asks for attention raises the reason then.
        try:
            self._attention_parts()
        except Exception:
            pass

    # -- per layer ----------------------------------------------------------
    def qkv(self, i: int, x, rows: int, out) -> None:
        L = self.layers[i]
        self.backend.linear_dev(L["qkv"], x, rows, out, bias=L["qkv_bias"])

    def _attention_parts(self):
        """(plan, rotation table, q norms, k norms), made with the model; raises why there are none."""
        if self._attention is None:
            import torch
            m, a = self._manifest, attention_plan(self._manifest, self.plan)
            factors = None
            if a.rope_factors or a.rope_scale != 1.0:
                factors = (_f32(m, a.rope_factors) if a.rope_factors else np.ones(a.rot_dim // 2, np.float32)) * a.rope_scale
            rope = self.backend.rope_table(a.rot_dim, a.rope_base, factors=factors, interleaved=a.interleaved)
            dev = self.backend.torch_device
            qn, kn = ([None if n is None else torch.from_numpy(_f32(m, n).copy()).to(dev) for n in names]
                      for names in (a.q_norm, a.k_norm))
            self._attention = (a, rope, qn, kn)
        return self._attention

    def kv_caches(self, n_pages: int, page_size: int = 16, dtype=None) -> list:
        """A paged key/value cache for every layer (bf16 unless told otherwise)."""
        import torch
        a = self._attention_parts()[0]
        return [self.backend.kv_cache(n_pages, page_size, a.n_kv_heads, a.head_dim, dtype or torch.bfloat16)
                for _ in self.layers]

    def attention(self, i: int, qkv, cache, positions, block_table, seqs=None, q=None, out=None):
        """Layer i between `qkv` and `o`: norms, rotation, cache write, attention -> f32 [rows, n_heads * head_dim].

        Row r of qkv is token positions[r] of sequence seqs[r] (r when None), as for
        qk_norm_rope; several rows of one sequence (a prompt) see each other causally.
        q, out: optional [rows, n_heads, head_dim] buffers.
        """
        a, rope, qn, kn = self._attention_parts()
        q = self.backend.qk_norm_rope(qkv, cache, positions, block_table, rope, q_norm=qn[i], k_norm=kn[i], eps=a.eps,
                                      seqs=seqs, out=q)
        o = self.backend.paged_attention(q, cache, positions, block_table, scale=a.scale, seqs=seqs, out=out)
        return o.view(o.shape[0], a.n_heads * a.head_dim)

    def o(self, i: int, x, rows: int, out) -> None:
        self.backend.linear_dev(self.layers[i]["o"], x, rows, out)

    def mlp(self, i: int, x, rows: int, act, out) -> None:
        L = self.layers[i]
        self.backend.mlp_gated_silu(x, rows, self.plan.hidden, self.plan.intermediate, L["gate_up"], None,
                                    L["down"], act, None, out)

    # -- model ends ---------------------------------------------------------
    def embed(self, ids, out=None):
        return self.backend.embed_rows(self.embed_table, ids, out)

    def head_argmax(self, h, rows: int, logits=None, ids=None, rules=None):
        """Greedy pick of the head's logits (under `rules`, see LogitRules, when given): (ids, the head's logits)."""
        import torch
        if logits is None:
            logits = torch.empty(rows, self.plan.vocab, device=self.backend.torch_device)
        self.backend.linear_dev(self.head_w, h, rows, logits)
        return self.backend.greedy_sample(logits, out=ids, rules=rules), logits
