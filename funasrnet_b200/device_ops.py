"""Device-pointer operators of libfunasr_cuda.so (``fa_dev_*``) on torch CUDA tensors.

They enqueue work on a stream and return: no host copies, no allocation.  The
reference has no counterpart (it decodes one context at a time and picks
greedily, src/FunAsrNet/QwenDecoder.cs:161-326); a server that decodes many
contexts on one GPU calls them around its decode step:

* :meth:`DeviceOps.attention_packed` -- several prompts, or chunks of them, at once
* :meth:`DeviceOps.attention_shared` -- a batch whose sequences share a prompt prefix
* :meth:`DeviceOps.adjust_logits` -- penalties, hot-word biases and grammar masks, and the greedy pick

Arguments are tensors on the backend's device (torch itself is not imported:
anything with torch's ``data_ptr``, ``dtype``, ``shape``, ``stride`` and
``device`` serves).  A call returns True, or False when the library declines
the shape or alignment (outputs untouched); wrong arguments raise ``ValueError``
or ``FaError``.  ``stream`` is a CUDA stream handle such as
``torch.cuda.current_stream().cuda_stream`` (0 is the default stream); None
selects the backend's own stream.
"""
from __future__ import annotations

import math
import struct

from ._lib import FA_OK, FaError, check, lib
from .backend import CudaFloatBackend

_DTYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
_LEGACY_STREAM = 1  # cudaStreamLegacy: the default stream by name (NULL is the backend's own)

# The C structs of include/funasr_cuda.h; every field is naturally aligned.
_PACKED = struct.Struct("@8Pq8q2q6ifi")
_SHARED = struct.Struct("@9Pq14q2q5if")
_LOGITS = struct.Struct("@14P5q4i")


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class DeviceOps:
    """The ``fa_dev_*`` operators on one backend's device."""

    def __init__(self, backend: CudaFloatBackend):
        self.b = backend
        self._device = backend.device
        self._lib = lib()

    # ------------------------------------------------------------------ checks ----

    def _ptr(self, t, name: str, dtype: str | None = None, shape=None) -> int:
        """Address of a contiguous tensor of `dtype` and `shape` on the backend's device; None gives 0."""
        if t is None:
            return 0
        if dtype is not None and str(t.dtype) != dtype:
            raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
        if shape is not None and tuple(t.shape) != shape:
            raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: not contiguous")
        return self._on_device(t, name)

    def _on_device(self, t, name: str) -> int:
        d = t.device
        if d.type != "cuda" or d.index != self._device:
            raise ValueError(f"{name}: on {d}, not on the backend's device cuda:{self._device}")
        return t.data_ptr()

    def _rows(self, t, name: str, dtype, shape) -> tuple:
        """(address, strides but the innermost) of a strided tensor whose innermost dimension is contiguous."""
        if t.dtype != dtype:
            raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
        if tuple(t.shape) != shape:
            raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
        st = t.stride()
        if st[-1] != 1 and shape[-1] > 1:
            raise ValueError(f"{name}: the innermost dimension must be contiguous")
        return self._on_device(t, name), st[:-1]

    @staticmethod
    def _dtype(t, name: str) -> int:
        code = _DTYPES.get(str(t.dtype))
        if code is None:
            raise ValueError(f"{name}: {t.dtype} is not float32, float16 or bfloat16")
        return code

    def _workspace(self, t) -> tuple:
        if t is None:
            return 0, 0
        if not t.is_contiguous():
            raise ValueError("workspace: not contiguous")
        return self._on_device(t, "workspace"), t.numel() * t.element_size()

    def _call(self, fn, args: bytes, stream) -> bool:
        return check(fn(self.b.handle, args, _LEGACY_STREAM if stream == 0 else stream)) == FA_OK

    # --------------------------------------------------------------- attention ----

    def attention_packed_workspace(self, q, k, q_offsets) -> int:
        """Bytes of workspace for :meth:`attention_packed` on tensors of these shapes."""
        return int(self._lib.fa_dev_attention_packed_workspace(q.shape[0], k.shape[0], q_offsets.shape[0] - 1, q.shape[1],
                                                               k.shape[1], q.shape[2]))

    def attention_packed(self, q, k, v, q_offsets, k_offsets, out, *, causal: bool = True, scale: float | None = None,
                         lse=None, workspace=None, stream: int | None = None) -> bool:
        """Attention of packed sequences: q, out [tokens, heads, size]; k, v [keys, kv_heads, size].

        Sequence b owns queries ``q_offsets[b]:q_offsets[b+1]`` and keys
        ``k_offsets[b]:k_offsets[b+1]`` (int32).  Causal queries are the last
        positions of their sequence.  ``lse`` [tokens, heads] float32 receives
        the log of the sum of exponentials; ``scale`` defaults to size ** -0.5.
        """
        _need(len(q.shape) == 3 and len(k.shape) == 3, "q and k must have three dimensions")
        total_q, heads, size = q.shape
        total_k, kv_heads, _ = k.shape
        code, dtype = self._dtype(q, "q"), q.dtype
        _need(kv_heads > 0 and heads % kv_heads == 0, "heads must be a multiple of kv_heads")
        n = q_offsets.shape[0] - 1
        _need(n >= 0, "q_offsets: empty")
        kv_shape = (total_k, kv_heads, size)
        qp, qs = self._rows(q, "q", dtype, (total_q, heads, size))
        kp, ks = self._rows(k, "k", dtype, kv_shape)
        vp, vs = self._rows(v, "v", dtype, kv_shape)
        op, os_ = self._rows(out, "out", dtype, (total_q, heads, size))
        wp, wb = self._workspace(workspace)
        args = _PACKED.pack(qp, kp, vp, op, self._ptr(lse, "lse", "torch.float32", (total_q, heads)),
                            self._ptr(q_offsets, "q_offsets", "torch.int32", (n + 1,)),
                            self._ptr(k_offsets, "k_offsets", "torch.int32", (n + 1,)), wp, wb, *qs, *ks, *vs, *os_,
                            total_q, total_k, code, n, heads, kv_heads, size, 1 if causal else 0,
                            1.0 / math.sqrt(size) if scale is None else scale, 0)
        return self._call(self._lib.fa_dev_attention_packed, args, stream)

    def attention_shared_workspace(self, q, prefix_k, suffix_k) -> int:
        """Bytes of workspace for :meth:`attention_shared` on tensors of these shapes."""
        return int(self._lib.fa_dev_attention_shared_workspace(prefix_k.shape[0], suffix_k.shape[1], q.shape[0],
                                                               q.shape[1], prefix_k.shape[1], q.shape[2]))

    def attention_shared(self, q, prefix_k, prefix_v, suffix_k, suffix_v, suffix_lens, out, *,
                         scale: float | None = None, lse=None, workspace=None, stream: int | None = None) -> bool:
        """Attention of one query token per sequence over a shared prefix and the sequence's own keys.

        q, out [sequences, heads, size]; prefix_k, prefix_v [prefix, kv_heads,
        size]; suffix_k, suffix_v [sequences, capacity, kv_heads, size], of
        which sequence b uses the first ``suffix_lens[b]`` (int32) positions.
        """
        _need(len(q.shape) == 3 and len(prefix_k.shape) == 3 and len(suffix_k.shape) == 4,
              "q and prefix_k must have three dimensions, suffix_k four")
        n, heads, size = q.shape
        prefix, kv_heads, _ = prefix_k.shape
        cap = suffix_k.shape[1]
        code, dtype = self._dtype(q, "q"), q.dtype
        _need(kv_heads > 0 and heads % kv_heads == 0, "heads must be a multiple of kv_heads")
        qp, qs = self._rows(q, "q", dtype, (n, heads, size))
        pkp, pks = self._rows(prefix_k, "prefix_k", dtype, (prefix, kv_heads, size))
        pvp, pvs = self._rows(prefix_v, "prefix_v", dtype, (prefix, kv_heads, size))
        skp, sks = self._rows(suffix_k, "suffix_k", dtype, (n, cap, kv_heads, size))
        svp, svs = self._rows(suffix_v, "suffix_v", dtype, (n, cap, kv_heads, size))
        op, os_ = self._rows(out, "out", dtype, (n, heads, size))
        wp, wb = self._workspace(workspace)
        args = _SHARED.pack(qp, pkp, pvp, skp, svp, op, self._ptr(lse, "lse", "torch.float32", (n, heads)),
                            self._ptr(suffix_lens, "suffix_lens", "torch.int32", (n,)), wp, wb, *qs, *pks, *pvs, *sks,
                            *svs, *os_, prefix, cap, code, n, heads, kv_heads, size,
                            1.0 / math.sqrt(size) if scale is None else scale)
        return self._call(self._lib.fa_dev_attention_shared, args, stream)

    # ------------------------------------------------------------------ logits ----

    def adjust_logits(self, logits, out, tokens=None, *, history=None, history_offsets=None, prompt_lens=None,
                      repetition=None, presence=None, frequency=None, bias_tokens=None, bias_values=None,
                      bias_offsets=None, mask=None, mask_rows=None, stream: int | None = None) -> bool:
        """Penalties, biases and masks on ``logits`` [rows, vocab] into ``out``, and the greedy ``tokens`` [rows].

        Row r's history is ``history[history_offsets[r]:history_offsets[r+1]]``, of
        which the first ``prompt_lens[r]`` tokens are the prompt; ``repetition``,
        ``presence`` and ``frequency`` are float32 [rows].  Its biases are
        ``bias_tokens``/``bias_values`` between ``bias_offsets``.  ``mask`` [masks,
        ceil(vocab / 32)] holds one bit per allowed token (int32 words), and
        ``mask_rows[r]`` picks the row's mask (negative: none).  All optional.
        """
        _need(len(logits.shape) == 2, "logits must have two dimensions")
        rows, vocab = logits.shape
        code, dtype = self._dtype(logits, "logits"), logits.dtype
        lp, ls = self._rows(logits, "logits", dtype, (rows, vocab))
        op, os_ = self._rows(out, "out", dtype, (rows, vocab))
        one, more, i32, f32 = (rows,), (rows + 1,), "torch.int32", "torch.float32"
        _need((history is None) == (history_offsets is None), "history and history_offsets come together")
        _need((bias_tokens is None) == (bias_values is None) == (bias_offsets is None),
              "bias_tokens, bias_values and bias_offsets come together")
        history_total = 0 if history is None else history.numel()
        bias_total = 0 if bias_tokens is None else bias_tokens.numel()
        mp, ms, masks = 0, (0,), 0
        if mask is not None:
            _need(len(mask.shape) == 2, "mask must have two dimensions")
            masks = mask.shape[0]
            _need(str(mask.dtype) in ("torch.int32", "torch.uint32"), "mask: expected 32-bit words")
            mp, ms = self._rows(mask, "mask", mask.dtype, (masks, (vocab + 31) // 32))
        p = self._ptr
        args = _LOGITS.pack(lp, op, p(tokens, "tokens", i32, one), p(history, "history", i32),
                            p(history_offsets, "history_offsets", i32, more), p(prompt_lens, "prompt_lens", i32, one),
                            p(repetition, "repetition", f32, one), p(presence, "presence", f32, one),
                            p(frequency, "frequency", f32, one), p(bias_tokens, "bias_tokens", i32),
                            p(bias_values, "bias_values", f32, (bias_total,) if bias_tokens is not None else None),
                            p(bias_offsets, "bias_offsets", i32, more), mp, p(mask_rows, "mask_rows", i32, one), ls[0],
                            os_[0], ms[0], history_total, bias_total, code, rows, vocab, masks)
        return self._call(self._lib.fa_dev_adjust_logits, args, stream)

    def status(self) -> None:
        """Waits for the device; raises ``FaError`` (timeout) when a bounded device wait of these operators gave up."""
        check(self._lib.fa_dev_status(self.b.handle))


__all__ = ["DeviceOps", "FaError"]
