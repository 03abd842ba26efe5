"""What a decode step holds between the linear layers: the paged key/value cache,
the rotation table and the rules on the logits.

The objects own (or view) torch memory of the backend's device and keep the C
descriptions of include/ocelotl_cuda.h; the calls on them are methods of
`CudaKernelBackend` (qk_norm_rope, paged_attention, process_logits,
greedy_sample).  Reference counterparts: PagedKvCacheLayout
(crates/core/src/lib.rs:578-665), rope and rmsnorm (crates/kernels/src/rope.rs,
rmsnorm.rs), sampling (crates/runtime/src/sampling.rs).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .errors import KernelError, UnsupportedError

KV_TYPES = {torch.float16: 1, torch.bfloat16: 30}  # GGUF tensor-type tags
HEAD_DIMS = (64, 96, 128, 256)


def _err(message: str) -> KernelError:
    return KernelError("cuda-sm100a", message)


def check_tensor(t, op: str, name: str, dtype: torch.dtype, device: torch.device, dims: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.dim() != dims \
            or not (t.is_contiguous() or t.shape[-1] <= 1 or t.stride(-1) == 1):
        raise _err(f"{op} {name} must be a {dims}-D {str(dtype)[6:]} tensor on {device} with a dense last dimension")


class PagedKvCache:
    """One layer's keys and values: `k`, `v` [n_pages, n_kv_heads, page_size, head_dim].

    Any strides with the elements of a head side by side, the same for k and v (a
    transposed [n_pages, page_size, n_kv_heads, head_dim] tensor is fine).
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor) or k.dim() != 4:
            raise _err("kv cache k and v must be 4-D tensors [n_pages, n_kv_heads, page_size, head_dim]")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            raise _err("kv cache k and v differ in shape, type, device or strides")
        if k.dtype not in KV_TYPES:
            raise UnsupportedError("cache type", str(k.dtype)[6:], ["float16", "bfloat16"])
        if k.shape[3] not in HEAD_DIMS:
            raise UnsupportedError("head_dim", str(k.shape[3]), [str(d) for d in HEAD_DIMS])
        if k.numel() == 0 or k.stride(3) != 1:
            raise _err("kv cache must not be empty and must hold the elements of a head side by side")
        self.k, self.v, self.device = k, v, k.device
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        # a dimension of size 1 has no stride of its own
        stride = [k.stride(i) if k.shape[i] > 1 else self.head_dim for i in range(3)]
        self.desc = _lib.KvCacheDesc(k.data_ptr(), v.data_ptr(), KV_TYPES[k.dtype], self.n_pages, self.page_size,
                                     self.n_kv_heads, self.head_dim, stride[0], stride[1], stride[2])
        self.ref = C.byref(self.desc)


class RopeTable:
    """Rotation steps of a position encoding on the backend's device (ocl_rope)."""

    def __init__(self, backend, handle: int, rot_dim: int):
        self._backend = backend
        self._handle = C.c_void_p(handle)
        self.rot_dim = rot_dim

    @property
    def handle(self) -> C.c_void_p:
        if not self._handle:
            raise _err("rope table used after free")
        return self._handle

    def free(self) -> None:
        if self._handle:
            self._backend._lib.ocl_rope_free(self._handle)
            self._handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class LogitRules:
    """Penalties, biases and the allowed-token mask of a batch of `rows` requests.

    history int32 [rows, n] with history_lens int32 [rows] (and prompt_lens: how
    many of them are the prompt); repetition, frequency, presence f32 [rows];
    bias_ids int32 / bias_values f32 [rows, m] (negative id = unused); allowed
    int32 [rows, words], token t is bit t % 32 of word t / 32.  Every part may be
    None.  The tensors are read at each call, so a program appends a token to
    `history` in place and adds 1 to `history_lens`.
    """

    def __init__(self, device: torch.device, history=None, history_lens=None, prompt_lens=None, repetition=None,
                 frequency=None, presence=None, bias_ids=None, bias_values=None, allowed=None):
        parts = {"history": (history, torch.int32, 2), "history_lens": (history_lens, torch.int32, 1),
                 "prompt_lens": (prompt_lens, torch.int32, 1), "repetition": (repetition, torch.float32, 1),
                 "frequency": (frequency, torch.float32, 1), "presence": (presence, torch.float32, 1),
                 "bias_ids": (bias_ids, torch.int32, 2), "bias_values": (bias_values, torch.float32, 2),
                 "allowed": (allowed, torch.int32, 2)}
        given = {n: t for n, (t, _, _) in parts.items() if t is not None}
        for n, t in given.items():
            check_tensor(t, "logit_rules", n, parts[n][1], device, parts[n][2])
        if (history is None) != (history_lens is None):
            raise _err("logit_rules history and history_lens go together")
        if history is None and any(t is not None for t in (prompt_lens, repetition, frequency, presence)):
            raise _err("logit_rules penalties need a history")
        if (bias_ids is None) != (bias_values is None):
            raise _err("logit_rules bias_ids and bias_values go together")
        if bias_ids is not None and (bias_ids.shape != bias_values.shape or
                                     (bias_ids.shape[0] > 1 and bias_ids.stride(0) != bias_values.stride(0))):
            raise _err("logit_rules bias_ids and bias_values differ in shape or strides")
        rows = {t.shape[0] for t in given.values()}
        if len(rows) > 1:
            raise _err(f"logit_rules parts differ in rows: { {n: t.shape[0] for n, t in given.items()} }")
        for n in ("history", "bias_ids", "allowed"):  # rows may not overlap a row's own length
            t = given.get(n)
            if t is not None and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
                raise _err(f"logit_rules {n} rows overlap")
        self.device = device
        self.rows = rows.pop() if rows else None  # None: no rule at all, any number of rows
        self.parts = given                        # keeps the tensors alive
        self.words = None if allowed is None else allowed.shape[1]
        # history, bias and mask widths of 0 count as absent
        if history is not None and history.shape[1] == 0:
            history = history_lens = prompt_lens = repetition = frequency = presence = None
        if bias_ids is not None and bias_ids.shape[1] == 0:
            bias_ids = bias_values = None

        def p(t):
            return None if t is None else t.data_ptr()

        def width(t):  # row stride; the row's own length where there is one row
            return 0 if t is None else (t.stride(0) if t.shape[0] > 1 else t.shape[1])

        def length(t):
            return 0 if t is None else t.shape[1]

        self.desc = _lib.LogitRulesDesc(p(history), width(history), length(history), p(history_lens), p(prompt_lens),
                                        p(repetition), p(frequency), p(presence), p(bias_ids), p(bias_values),
                                        width(bias_ids), length(bias_ids), p(allowed), width(allowed))
        self.ref = C.byref(self.desc)
