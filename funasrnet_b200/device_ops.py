"""Device-pointer operators of libfunasr_cuda.so (``fa_dev_*``) on torch CUDA tensors.

They enqueue work on a stream and return: no host copies, no allocation.  The
reference has no counterpart (it decodes one context at a time and picks
greedily, src/FunAsrNet/QwenDecoder.cs:161-326); a server that decodes many
contexts on one GPU calls them around its decode step:

* :meth:`DeviceOps.attention_packed` -- several prompts, or chunks of them, at once
* :meth:`DeviceOps.attention_shared` -- a batch whose sequences share a prompt prefix
* :meth:`DeviceOps.adjust_logits` -- penalties, hot-word biases and grammar masks, and the greedy pick

Arguments are torch tensors on the backend's device.  A call returns True, or
False when the library declines the shape or alignment (outputs untouched);
tensors that do not fit together raise ``ValueError``, what the library refuses
``FaError``.  There is no backward pass: tensors that require grad are refused where
grad mode is on, and a call raises the version of the tensors that it writes.

``stream`` is a CUDA stream handle such as
``torch.cuda.current_stream().cuda_stream`` (0 is the default stream); tensors of
another stream have to outlive the call's work (``Tensor.record_stream``).  Without
it a call runs on the backend's own stream, after what torch's current stream
holds and before what is enqueued there next; giving the stream saves the two
events of that, and keeps the backend's stream out of a capture while other threads
use it.  ``workspace`` is any contiguous tensor of at least the bytes that
the ``*_workspace`` method gives for the call's tensors, or the
``*_workspace_bound`` method for every call up to given sizes (a smaller batch can
need more than a larger one); calls that may overlap in time need one each.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import threading

import torch

from ._lib import FaError, check, lib
from .backend import CudaFloatBackend
from .build import binding_path

_lock = threading.Lock()
_binding = None


def _native():
    """The CPython binding, built next to the library (csrc/torch_binding.cpp)."""
    global _binding
    with _lock:
        if _binding is None:
            path = binding_path()
            if not path.exists():
                raise RuntimeError(f"{path} is missing: build it for this Python and torch with "
                                   "`python -m funasrnet_b200.build`")
            lib()  # the binding calls the same library
            spec = importlib.util.spec_from_file_location("funasrnet_b200._torch_ops", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            _binding = module
        return _binding


class DeviceOps:
    """The ``fa_dev_*`` operators on one backend's device."""

    def __init__(self, backend: CudaFloatBackend):
        self.b = backend
        self._device = backend.device
        self._native = _native()
        h = C.c_void_p()
        check(lib().fa_backend_stream(backend.handle, C.byref(h)))
        self._own = torch.cuda.ExternalStream(h.value, device=self._device)

    def _in_order(self, method, *args, **kw) -> bool:
        """The call on the backend's own stream, between the work of torch's current stream and what follows there."""
        self.b.handle  # raises when the backend is disposed, and its stream with it
        now = torch.cuda.current_stream(self._device)
        self._own.wait_stream(now)
        try:
            return method(*args, stream=self._own.cuda_stream, **kw)
        finally:
            now.wait_stream(self._own)

    # --------------------------------------------------------------- attention ----

    def attention_packed_workspace(self, q, k, q_offsets) -> int:
        """Bytes of workspace for :meth:`attention_packed` on tensors of these shapes."""
        return int(lib().fa_dev_attention_packed_workspace(q.shape[0], k.shape[0], q_offsets.shape[0] - 1, q.shape[1],
                                                           k.shape[1], q.shape[2]))

    @staticmethod
    def attention_packed_workspace_bound(tokens: int, keys: int, heads: int, kv_heads: int, size: int) -> int:
        """Bytes that are enough for every :meth:`attention_packed` of up to so many tokens and keys."""
        return int(lib().fa_dev_attention_packed_workspace_bound(tokens, keys, heads, kv_heads, size))

    def attention_packed(self, q, k, v, q_offsets, k_offsets, out, *, causal: bool = True, scale: float | None = None,
                         lse=None, workspace=None, stream: int | None = None) -> bool:
        """Attention of packed sequences: q, out [tokens, heads, size]; k, v [keys, kv_heads, size].

        Sequence b owns queries ``q_offsets[b]:q_offsets[b+1]`` and keys
        ``k_offsets[b]:k_offsets[b+1]`` (int32).  Causal queries are the last
        positions of their sequence.  ``lse`` [tokens, heads] float32 receives
        the log of the sum of exponentials; ``scale`` defaults to size ** -0.5.
        """
        if stream is None:
            return self._in_order(self.attention_packed, q, k, v, q_offsets, k_offsets, out, causal=causal, scale=scale,
                                  lse=lse, workspace=workspace)
        rc = self._native.attention_packed(self.b.handle.value, self._device, q, k, v, q_offsets, k_offsets, out, causal,
                                           scale, lse, workspace, stream)
        return rc == 0 or check(rc) == 0

    def attention_shared_workspace(self, q, prefix_k, suffix_k) -> int:
        """Bytes of workspace for :meth:`attention_shared` on tensors of these shapes."""
        return int(lib().fa_dev_attention_shared_workspace(prefix_k.shape[0], suffix_k.shape[1], q.shape[0], q.shape[1],
                                                           prefix_k.shape[1], q.shape[2]))

    @staticmethod
    def attention_shared_workspace_bound(prefix: int, capacity: int, sequences: int, heads: int, kv_heads: int,
                                         size: int) -> int:
        """Bytes that are enough for every :meth:`attention_shared` of up to this prefix, capacity and batch."""
        return int(lib().fa_dev_attention_shared_workspace_bound(prefix, capacity, sequences, heads, kv_heads, size))

    def attention_shared(self, q, prefix_k, prefix_v, suffix_k, suffix_v, suffix_lens, out, *,
                         scale: float | None = None, lse=None, workspace=None, stream: int | None = None) -> bool:
        """Attention of one query token per sequence over a shared prefix and the sequence's own keys.

        q, out [sequences, heads, size]; prefix_k, prefix_v [prefix, kv_heads,
        size]; suffix_k, suffix_v [sequences, capacity, kv_heads, size], of
        which sequence b uses the first ``suffix_lens[b]`` (int32) positions.
        """
        if stream is None:
            return self._in_order(self.attention_shared, q, prefix_k, prefix_v, suffix_k, suffix_v, suffix_lens, out,
                                  scale=scale, lse=lse, workspace=workspace)
        rc = self._native.attention_shared(self.b.handle.value, self._device, q, prefix_k, prefix_v, suffix_k, suffix_v,
                                           suffix_lens, out, scale, lse, workspace, stream)
        return rc == 0 or check(rc) == 0

    # ------------------------------------------------------------------ logits ----

    def adjust_logits(self, logits, out, tokens=None, *, history=None, history_offsets=None, prompt_lens=None,
                      repetition=None, presence=None, frequency=None, bias_tokens=None, bias_values=None,
                      bias_offsets=None, mask=None, mask_rows=None, stream: int | None = None) -> bool:
        """Penalties, biases and masks on ``logits`` [rows, vocab] into ``out``, and the greedy ``tokens`` [rows].

        Row r's history is ``history[history_offsets[r]:history_offsets[r+1]]``, of
        which the first ``prompt_lens[r]`` tokens are the prompt; ``repetition``,
        ``presence`` and ``frequency`` are float32 [rows].  Its biases are
        ``bias_tokens``/``bias_values`` between ``bias_offsets``.  ``mask`` [masks,
        ceil(vocab / 32)] holds one bit per allowed token (32-bit words), and
        ``mask_rows[r]`` picks the row's mask (negative: none).  All optional.
        """
        if stream is None:
            return self._in_order(self.adjust_logits, logits, out, tokens, history=history, history_offsets=history_offsets,
                                  prompt_lens=prompt_lens, repetition=repetition, presence=presence, frequency=frequency,
                                  bias_tokens=bias_tokens, bias_values=bias_values, bias_offsets=bias_offsets, mask=mask,
                                  mask_rows=mask_rows)
        rc = self._native.adjust_logits(self.b.handle.value, self._device, logits, out, tokens, history, history_offsets,
                                        prompt_lens, repetition, presence, frequency, bias_tokens, bias_values,
                                        bias_offsets, mask, mask_rows, stream)
        return rc == 0 or check(rc) == 0

    def status(self) -> None:
        """Waits for the device; raises ``FaError`` (timeout) when a bounded wait of a call on this backend gave up."""
        check(lib().fa_dev_status(self.b.handle))


__all__ = ["DeviceOps", "FaError"]
