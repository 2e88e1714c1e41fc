"""Verification of drafted tokens (speculative decoding) over the C ABI of include/et_speculative.h.

``DraftVerifier(vocab_size, max_sequences, max_drafts)`` holds the work buffers;
:meth:`DraftVerifier.verify` keeps as many of each sequence's drafts as the target model's
probabilities allow, from given random numbers, and draws the token behind them.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _capi
from .sampler import SamplerError, dtype_code


class DraftVerifier:
    """Work buffers for batches of at most ``max_sequences`` sequences with ``max_drafts`` drafts each
    on the current device (or ``device``); calls allocate nothing on the device but their outputs."""

    def __init__(self, vocab_size: int, max_sequences: int, max_drafts: int, device=None):
        self._h = C.c_void_p()
        L = _capi.lib()
        if device is None and not torch.cuda.is_available():
            st = L.ets_verifier_create(vocab_size, max_sequences, max_drafts, C.byref(self._h))
        else:
            with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
                self.device = torch.device("cuda", torch.cuda.current_device())
                st = L.ets_verifier_create(vocab_size, max_sequences, max_drafts, C.byref(self._h))
        if st != _capi.OK:
            raise SamplerError(st, L.ets_verifier_last_error(None).decode())
        self.vocab_size, self.max_sequences, self.max_drafts = vocab_size, max_sequences, max_drafts

    def close(self) -> None:
        if getattr(self, "_h", None) and self._h.value:
            _capi.lib().ets_verifier_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def verify(self, target_logits: torch.Tensor, draft_tokens: torch.Tensor, coins: torch.Tensor,
               draft_logits: torch.Tensor | None = None, draft_lengths: torch.Tensor | None = None, temperature=1.0,
               tokens_out: torch.Tensor | None = None, accepted_out: torch.Tensor | None = None):
        """``target_logits`` ``[S, K + 1, vocab]``, ``draft_tokens`` int32 ``[S, K]``, ``coins`` fp32
        ``[S, K + 1]`` uniforms in [0, 1) (one per draft, then the draw's), ``draft_logits``
        ``[S, K, vocab]`` of the same type or None (drafts that were looked up, not drawn),
        ``draft_lengths`` int32 ``[S]`` or None, ``temperature`` a float or fp32 ``[S]``; all on the
        verifier's device, any strides with a unit innermost one.

        Returns ``(tokens [S, K + 1], accepted [S])``, int32: the accepted drafts, the next token, then
        -1; asynchronously on the current stream.  Top-k and top-p are applied by masking both models'
        rows with -inf beforehand."""
        if target_logits.dim() != 3 or draft_tokens.dim() != 2 or coins.dim() != 2:
            raise SamplerError(_capi.INVALID_ARGUMENT, "verify wants target_logits [S, K + 1, vocab], draft_tokens [S, K], coins [S, K + 1]")
        S, positions, V = target_logits.shape
        K = positions - 1
        device = self.device
        if V != self.vocab_size:
            raise SamplerError(_capi.INVALID_ARGUMENT, "last dimension differs from vocab_size")
        if draft_tokens.shape != (S, K) or coins.shape != (S, positions):
            raise SamplerError(_capi.INVALID_ARGUMENT, "draft_tokens must be [S, K] and coins [S, K + 1]")
        code = dtype_code(target_logits)
        a = _capi.VerifyBatch()
        if draft_logits is not None:
            if draft_logits.shape != (S, K, V) or draft_logits.dtype != target_logits.dtype:
                raise SamplerError(_capi.INVALID_ARGUMENT, "draft_logits must be [S, K, vocab] of the target's type")
            if K:
                self._on_device(draft_logits, draft_logits.dtype, "draft_logits")
                a.draft_logits = draft_logits.data_ptr()
                a.draft_sequence_stride, a.draft_position_stride = draft_logits.stride(0), draft_logits.stride(1)
        self._on_device(target_logits, target_logits.dtype, "target_logits")
        self._on_device(draft_tokens, torch.int32, "draft_tokens")
        self._on_device(coins, torch.float32, "coins")
        if draft_lengths is not None:
            if draft_lengths.shape != (S,):
                raise SamplerError(_capi.INVALID_ARGUMENT, "draft_lengths must be [S]")
            self._on_device(draft_lengths, torch.int32, "draft_lengths")
            a.draft_lengths = draft_lengths.data_ptr()
        if isinstance(temperature, torch.Tensor):
            if temperature.shape != (S,):
                raise SamplerError(_capi.INVALID_ARGUMENT, "temperature must be a number or fp32 [S]")
            self._on_device(temperature, torch.float32, "temperature")
            a.temperatures = temperature.data_ptr()
        else:
            a.temperature = temperature
        if tokens_out is None:
            tokens_out = torch.empty((S, positions), dtype=torch.int32, device=device)
        else:
            if tokens_out.shape != (S, positions):
                raise SamplerError(_capi.INVALID_ARGUMENT, "tokens_out must be [S, K + 1]")
            self._on_device(tokens_out, torch.int32, "tokens_out")
        if accepted_out is None:
            accepted_out = torch.empty((S,), dtype=torch.int32, device=device)
        else:
            if accepted_out.shape != (S,):
                raise SamplerError(_capi.INVALID_ARGUMENT, "accepted_out must be [S]")
            self._on_device(accepted_out, torch.int32, "accepted_out")
        a.target_logits, a.dtype, a.sequences, a.drafts = target_logits.data_ptr(), code, S, K
        a.target_sequence_stride, a.target_position_stride = target_logits.stride(0), target_logits.stride(1)
        a.draft_tokens, a.draft_tokens_stride = draft_tokens.data_ptr(), draft_tokens.stride(0)
        a.coins, a.coins_stride = coins.data_ptr(), coins.stride(0)
        a.tokens, a.tokens_stride = tokens_out.data_ptr(), tokens_out.stride(0)
        a.accepted = accepted_out.data_ptr()
        st = _capi.lib().ets_verifier_verify(self._h, C.byref(a), torch.cuda.current_stream(device).cuda_stream)
        if st != _capi.OK:
            raise SamplerError(st, _capi.lib().ets_verifier_last_error(self._h).decode())
        return tokens_out, accepted_out

    def _on_device(self, t: torch.Tensor, dtype, name: str) -> None:
        if t.device != self.device or t.dtype != dtype or (t.stride(-1) != 1 and t.shape[-1] > 1):
            raise SamplerError(_capi.INVALID_ARGUMENT, f"{name} must be a {dtype} tensor on {self.device} with unit inner stride")
