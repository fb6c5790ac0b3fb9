"""From a step's logits to tokens (include/moe_spec.h): the logits of several tokens, their probabilities, and the
verification of drafted tokens against them, beside the greedy `stack.LmHead`. torch is used for device memory and
streams only."""
import torch

from . import _check, _lib
from .paged import _need, raw_stream


def lm_head_logits(weight, normed, logits, stream=None):
    """logits fp32 [T, V] = normed bf16 bits [T, H] . weight^T (bf16 bits [V, H]); the weight is read once for every
    four rows."""
    V, H = weight.shape
    T = normed.numel() // H
    dev = weight.device
    _need(weight.dtype == normed.dtype == torch.int16 and weight.is_contiguous() and normed.is_contiguous()
          and normed.numel() == T * H and normed.device == dev, "weight [V, H], normed [T, H]: contiguous bf16 bits")
    _need(logits.dtype == torch.float32 and logits.is_contiguous() and logits.numel() == T * V and logits.device == dev,
          f"logits: expected contiguous float32 [{T}, {V}]")
    s = raw_stream(dev, stream)
    for t in range(0, T, 4):
        _check(_lib.moe_lm_head_logits(normed.data_ptr() + t * H * 2, weight.data_ptr(), V, H, min(4, T - t),
                                       logits.data_ptr() + t * V * 4, s), "moe_lm_head_logits")


def softmax_rows(logits, probs, temperature=None, stream=None):
    """probs = softmax(logits / temperature) over the last dimension, row by row: fp32 [R, V], rows any distance apart;
    temperature fp32 [R], 0 for a one-hot row at the largest logit. probs may be logits."""
    R, V = logits.shape
    dev = logits.device
    _need(logits.dtype == probs.dtype == torch.float32 and probs.shape == logits.shape and probs.device == dev
          and (V == 1 or logits.stride(1) == probs.stride(1) == 1), "logits, probs: float32 [R, V] on one GPU, each row "
                                                                    "contiguous")
    _need(temperature is None or (temperature.dtype == torch.float32 and temperature.shape == (R,)
                                  and temperature.is_contiguous() and temperature.device == dev),
          f"temperature: expected contiguous float32 ({R},)")
    # the distance between rows means nothing for one row (torch allows any value there)
    ldx, ldy = (logits.stride(0), probs.stride(0)) if R > 1 else (V, V)
    _check(_lib.moe_softmax_rows(logits.data_ptr(), ldx, R, V, None if temperature is None else temperature.data_ptr(),
                                 probs.data_ptr(), ldy, raw_stream(dev, stream)), "moe_softmax_rows")


class SpecVerifier:
    """Verification of up to K drafted tokens for up to max_B sequences over V tokens; owns the call's workspace."""

    def __init__(self, max_B, K, V, device="cuda"):
        self.max_B, self.K, self.V = max_B, K, V
        n = _lib.moe_spec_workspace_bytes(max_B, V)
        if n == 0 or not 1 <= K <= 64:
            raise ValueError("unsupported sizes for the verification of drafts")
        self.ws = torch.zeros(n, dtype=torch.uint8, device=device)
        self.device = self.ws.device
        torch.cuda.current_stream(self.device).synchronize()

    def verify(self, target, draft, drafted, u, tokens, accepted, n_drafted=None, stream=None):
        """target fp32 [B, K + 1, V] (rows may lie further apart), draft fp32 [B, K, V] or None, drafted int32 [B, K], u
        fp32 [B, K + 1] in [0, 1), n_drafted int32 [B] or None -> tokens int32 [B, K + 1] (-1 behind the drawn one),
        accepted int32 [B]."""
        B, K1, V = target.shape
        K = K1 - 1
        _need(1 <= B <= self.max_B and K == self.K and V == self.V,
              f"target [{B}, {K1}, {V}]: the verifier takes up to {self.max_B} x {self.K + 1} x {self.V}")
        for n, t, rows in (("target", target, K1), ("draft", draft, K)):
            _need(t is None or (t.dtype == torch.float32 and t.shape == (B, rows, V) and t.device == self.device
                                and (V == 1 or t.stride(2) == 1) and t.stride(1) >= V
                                and (B == 1 or t.stride(0) == rows * t.stride(1))),
                  f"{n}: expected float32 [{B}, {rows}, {V}] on {self.device}, rows one distance apart")
        for n, t, shape, dt in (("drafted", drafted, (B, K), torch.int32), ("u", u, (B, K1), torch.float32),
                                ("tokens", tokens, (B, K1), torch.int32), ("accepted", accepted, (B,), torch.int32),
                                ("n_drafted", n_drafted, (B,), torch.int32)):
            _need((t is None and n == "n_drafted") or (t.dtype == dt and t.shape == shape and t.is_contiguous()
                                                       and t.device == self.device),
                  f"{n}: expected contiguous {dt} {shape} on {self.device}")
        _check(_lib.moe_spec_verify(
            target.data_ptr(), target.stride(1), None if draft is None else draft.data_ptr(),
            0 if draft is None else draft.stride(1), drafted.data_ptr(),
            None if n_drafted is None else n_drafted.data_ptr(), u.data_ptr(), B, K, V, tokens.data_ptr(),
            accepted.data_ptr(), self.ws.data_ptr(), self.ws.numel(), raw_stream(self.device, stream)),
            "moe_spec_verify")
