"""From a step's logits to tokens (include/moe_spec.h): the logits of several tokens, their probabilities, and the
verification of drafted tokens against them, beside the greedy `stack.LmHead`. torch is used for device memory and
streams only."""
import torch

from . import _check, _lib
from .paged import _F32, _I32, _need, raw_stream


def check_logits(weight, T, logits):
    """Refuses logits that cannot take T rows of the head `weight`."""
    _need(logits.dtype == torch.float32 and logits.is_contiguous() and logits.numel() == T * weight.shape[0]
          and logits.device == weight.device, f"logits: expected contiguous float32 [{T}, {weight.shape[0]}]")


def lm_head_logits(weight, normed, logits, stream=None):
    """logits fp32 [T, V] = normed bf16 bits [T, H] . weight^T (bf16 bits [V, H]); the weight is read once for every
    four rows."""
    V, H = weight.shape
    T = normed.numel() // H
    dev = weight.device
    _need(weight.dtype == normed.dtype == torch.int16 and weight.is_contiguous() and normed.is_contiguous()
          and normed.numel() == T * H and normed.device == dev, "weight [V, H], normed [T, H]: contiguous bf16 bits")
    check_logits(weight, T, logits)
    s = raw_stream(weight.get_device(), stream)
    for t in range(0, T, 4):
        _check(_lib.moe_lm_head_logits(normed.data_ptr() + t * H * 2, weight.data_ptr(), V, H, min(4, T - t),
                                       logits.data_ptr() + t * V * 4, s), "moe_lm_head_logits")


def softmax_rows(logits, probs, temperature=None, stream=None):
    """probs = softmax(logits / temperature) over the last dimension, row by row: fp32 [R, V], rows any distance apart;
    temperature fp32 [R], 0 for a one-hot row at the largest logit. probs may be logits."""
    R, V = logits.shape
    dev = logits.get_device()
    ldx, unit_x = logits.stride()
    ldy, unit_y = probs.stride()
    if logits.dtype is not _F32 or probs.dtype is not _F32 or probs.shape != logits.shape or probs.get_device() != dev \
            or (V > 1 and (unit_x != 1 or unit_y != 1)) or dev < 0:
        raise ValueError("logits, probs: expected float32 [R, V] on one GPU, each row contiguous")
    t = None
    if temperature is not None:
        if temperature.dtype is not _F32 or temperature.numel() != R or not temperature.is_contiguous() \
                or temperature.get_device() != dev:
            raise ValueError(f"temperature: expected contiguous float32 ({R},)")
        t = temperature.data_ptr()
    if R < 2:
        ldx = ldy = V  # torch allows any distance between the rows of one
    rc = _lib.moe_softmax_rows(logits.data_ptr(), ldx, R, V, t, probs.data_ptr(), ldy, raw_stream(dev, stream))
    if rc:
        _check(rc, "moe_softmax_rows")


def _dense(t, dtype, n, dev):
    return t.dtype is dtype and t.numel() == n and t.is_contiguous() and t.get_device() == dev


class SpecVerifier:
    """Verification of up to K drafted tokens for up to max_B sequences over V tokens; owns the call's workspace. With
    K = 0 it draws one token a sequence (draft and drafted are None then)."""

    def __init__(self, max_B, K, V, device="cuda"):
        self.max_B, self.K, self.V = max_B, K, V
        n = _lib.moe_spec_workspace_bytes(max_B, V)
        if n == 0 or not 0 <= K <= 64:
            raise ValueError("unsupported sizes for the verification of drafts")
        self.ws = torch.zeros(n, dtype=torch.uint8, device=device)
        self.device, self._dev = self.ws.device, self.ws.get_device()
        self._ws = (self.ws.data_ptr(), n)
        torch.cuda.current_stream(self.device).synchronize()

    def verify(self, target, draft, drafted, u, tokens, accepted, n_drafted=None, stream=None):
        """target fp32 [B, K + 1, V] (rows may lie further apart), draft fp32 [B, K, V] or None, drafted int32 [B, K], u
        fp32 [B, K + 1] in [0, 1), n_drafted int32 [B] or None -> tokens int32 [B, K + 1] (-1 behind the drawn one),
        accepted int32 [B]."""
        B, K1, V = target.shape
        K, dev = self.K, self._dev
        if B > self.max_B or K1 != K + 1 or V != self.V:
            raise ValueError(f"target {tuple(target.shape)}: the verifier takes up to {self.max_B} x {K + 1} x {self.V}")
        ldp = self._rows(target, "target", B, K1)
        ldq, q = 0, None
        if draft is not None and K:
            ldq, q = self._rows(draft, "draft", B, K), draft.data_ptr()
        if not ((_dense(drafted, _I32, B * K, dev) if K else drafted is None) and _dense(u, _F32, B * K1, dev) and _dense(tokens, _I32, B * K1, dev)
                and _dense(accepted, _I32, B, dev)):
            raise ValueError(f"expected contiguous drafted int32 ({B}, {K}), u float32 ({B}, {K1}), tokens int32 "
                             f"({B}, {K1}) and accepted int32 ({B},) on {self.device}")
        n = None
        if n_drafted is not None:
            _need(_dense(n_drafted, _I32, B, dev), f"n_drafted: expected contiguous int32 ({B},) on {self.device}")
            n = n_drafted.data_ptr()
        rc = _lib.moe_spec_verify(target.data_ptr(), ldp, q, ldq, drafted.data_ptr() if K else None, n, u.data_ptr(), B, K, V,
                                  tokens.data_ptr(), accepted.data_ptr(), *self._ws, raw_stream(dev, stream))
        if rc:
            _check(rc, "moe_spec_verify")

    def _rows(self, t, what, B, rows):
        """The distance between the rows of t [B, rows, V], one for all of them (torch allows any between those of one)."""
        s0, s1, s2 = t.stride()
        ld = s1 if rows > 1 else (s0 if B > 1 else self.V)
        if t.dtype is not _F32 or t.shape != (B, rows, self.V) or t.get_device() != self._dev \
                or (s2 != 1 and self.V > 1) or ld < self.V or (B > 1 and s0 != rows * ld):
            raise ValueError(f"{what}: expected float32 [{B}, {rows}, {self.V}] on {self.device}, rows one distance apart")
        return ld
