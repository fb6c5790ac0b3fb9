"""A paged key-value cache for batches of sequences, the attention over it, and a decode step built on them
(include/moe_paged.h).

`PagedCache` holds the pools, the page tables and the holders of each page as torch tensors and issues the page calls
(`resize`, `fork`, `compact`, `copy_pages`) and the attention calls (`append`, `attend`). `PagedAttnBlock` is
`stack.AttnBlock` for a batch over such a cache, `PagedDecodeStack` `stack.DecodeStack` for a batch with one or a few
new tokens a sequence. Lists, lengths and tables are device tensors, so a step can be captured into a CUDA graph once and
replayed while the sequences grow. torch is used for device memory and streams only.
"""
import ctypes

import torch

from . import MoeBlock, MoeError, MoePagedCache, _check, _lib, _ptr

KV_BF16, KV_E4M3 = 0, 1
ERR_TIMEOUT, ERR_PAGE_ID, ERR_SEQ_ID, ERR_NO_PAGES, ERR_SHARED = 1 << 3, 1 << 8, 1 << 9, 1 << 10, 1 << 11


_I16, _I32, _F32, _F64 = torch.int16, torch.int32, torch.float32, torch.float64


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def raw_stream(index, stream=None):
    """The handle of `stream`, or of the current stream of device `index`, which holds the tensors. The library launches
    on the current device, so that must be the same."""
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on cuda:{index}, but the current device is cuda:{torch.cuda.current_device()}")
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)


class PagedCache:
    """k, v: [layers, num_pages, Hkv, page, D], int16 (bf16 bits) or uint8 (e4m3 bits, with fp32 scales [layers, Hkv]);
    tables int32 [max_seqs, max_pages] (-1 where there is no page), refs int32 [num_pages] (holders of each page), lens
    int32 [max_seqs]. Lists of up to `max_batch` sequences, up to `max_new` new tokens each; Hq query heads.
    `PagedCache.empty` makes an empty one."""

    def __init__(self, k, v, tables, refs, lens, Hq, max_batch, max_new=1, k_scale=None, v_scale=None):
        _need(k.dim() == 5 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in (torch.int16, torch.uint8),
              "k, v: expected two equal [layers, pages, Hkv, page, D] tensors of int16 or uint8")
        self.layers, self.num_pages, self.Hkv, self.page, self.D = k.shape
        self.kv_type = KV_BF16 if k.dtype == torch.int16 else KV_E4M3
        _need(tables.dim() == 2, "tables: expected [max_seqs, max_pages]")
        self.max_seqs, self.max_pages = tables.shape
        want = {"tables": (tables, (self.max_seqs, self.max_pages)), "refs": (refs, (self.num_pages,)),
                "lens": (lens, (self.max_seqs,))}
        for n, (t, shape) in want.items():
            _need(tuple(t.shape) == shape and t.dtype == torch.int32, f"{n}: expected int32 {shape}")
        for n, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _need(t is None or (self.kv_type == KV_E4M3 and tuple(t.shape) == (self.layers, self.Hkv)
                                and t.dtype == torch.float32),
                  f"{n}: expected float32 {(self.layers, self.Hkv)}, and an e4m3 cache")
        for t in (k, v, tables, refs, lens, k_scale, v_scale):
            _need(t is None or (t.is_contiguous() and t.is_cuda and t.device == k.device),
                  "a cache's tensors are contiguous and on one GPU")
        self.k, self.v, self.tables, self.refs, self.lens = k, v, tables, refs, lens
        self.k_scale, self.v_scale = k_scale, v_scale
        self.device, self.Hq, self.max_batch, self.max_new = k.device, Hq, max_batch, max_new
        self._dev = k.get_device()
        self.c = MoePagedCache(*[None if t is None else t.data_ptr() for t in (k, v, tables, refs, lens, k_scale,
                                                                               v_scale)],
                               self.layers, self.num_pages, self.page, self.Hkv, self.D, self.kv_type, self.max_seqs,
                               self.max_pages)
        self._c = ctypes.byref(self.c)
        n = _lib.moe_paged_workspace_bytes(self._c, Hq, max_batch, max_new)
        if n == 0 or _lib.moe_paged_check(self._c) != 0:
            raise ValueError("unsupported paged cache (include/moe_paged.h lists what is supported)")
        self.ws = torch.zeros(n, dtype=torch.uint8, device=k.device)
        self._ws = (self.ws.data_ptr(), n)
        self._default_scale = self.D ** -0.5
        torch.cuda.current_stream(k.device).synchronize()  # the zeroing: the cache may be used from any stream

    @classmethod
    def empty(cls, layers, num_pages, page, Hkv, D, Hq, max_seqs, max_pages, max_batch, max_new=1, kv="bf16",
              k_scale=None, v_scale=None, device="cuda"):
        dev = torch.device(device)
        dt = {"bf16": torch.int16, "e4m3": torch.uint8}[kv]
        k, v = (torch.zeros(layers, num_pages, Hkv, page, D, dtype=dt, device=dev) for _ in range(2))
        return cls(k, v, torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=dev),
                   torch.zeros(num_pages, dtype=torch.int32, device=dev),
                   torch.zeros(max_seqs, dtype=torch.int32, device=dev), Hq, max_batch, max_new, k_scale, v_scale)

    # The calls below are a few microseconds of host time each, so their checks are written out rather than shared.
    def _list(self, t, what, n):
        if t.dtype is not _I32 or t.numel() != n or t.dim() != 1 or not t.is_contiguous() or t.get_device() != self._dev:
            raise ValueError(f"{what}: expected a contiguous int32 list of {n} on {self.device}")
        return t.data_ptr()

    def _rows(self, t, what, n):
        if t.dtype is not _I16 or t.numel() != n or not t.is_contiguous() or t.get_device() != self._dev:
            raise ValueError(f"{what}: expected {n} contiguous bf16 values (int16 bits) on {self.device}")
        return t.data_ptr()

    def _batch(self, seqs):
        B = seqs.numel()
        if B > self.max_batch:
            raise ValueError(f"a list of {B} sequences: max_batch is {self.max_batch}")
        return B

    def error_word(self, stream=None):
        """Reads and clears the workspace's error word (the ERR_ bits of this module)."""
        rc = _lib.moe_paged_workspace_error(*self._ws, raw_stream(self._dev, stream))
        if rc < 0:
            raise MoeError(f"moe_paged_workspace_error failed: cudaError {-rc}")
        return rc

    def resize(self, seqs, new_lens, stream=None):
        """Sets the listed sequences' lengths: pages are released, taken, or copied where a partly filled last page is
        shared."""
        n = self._batch(seqs)
        _check(_lib.moe_paged_resize(self._c, self._list(seqs, "seqs", n), self._list(new_lens, "new_lens", n), n,
                                     *self._ws, raw_stream(self._dev, stream)), "moe_paged_resize")

    def fork(self, src, dst, stream=None):
        """Makes each empty dst sequence share all pages of its src."""
        n = self._batch(src)
        _check(_lib.moe_paged_fork(self._c, self._list(src, "src", n), self._list(dst, "dst", n), n, *self._ws,
                                   raw_stream(self._dev, stream)), "moe_paged_fork")

    def compact(self, stream=None):
        """Moves the live pages to the lowest ids."""
        _check(_lib.moe_paged_compact(self._c, *self._ws, raw_stream(self._dev, stream)), "moe_paged_compact")

    def copy_pages(self, src, dst, stream=None):
        """Copies whole pages src[i] to dst[i] in every layer."""
        n = src.numel()
        _check(_lib.moe_paged_copy(self._c, self._list(src, "src", n), self._list(dst, "dst", n), n, *self._ws,
                                   raw_stream(self._dev, stream)), "moe_paged_copy")

    def append(self, layer, seqs, qkv, q_out, Tq=1, q_norm=None, k_norm=None, inv_freq=None, eps=1e-6, stream=None):
        """Norm, rotation and write of the new tokens' keys and values; q_out receives their queries."""
        B, D = self._batch(seqs), self.D
        T = B * Tq
        freq = pairs = 0
        if inv_freq is not None:
            pairs = inv_freq.numel()
            if inv_freq.dtype is not _F64 or not inv_freq.is_contiguous() or inv_freq.get_device() != self._dev:
                raise ValueError("inv_freq: expected a contiguous float64 list")
            freq = inv_freq.data_ptr()
        rc = _lib.moe_paged_append(
            self._c, layer, self._list(seqs, "seqs", B), B, Tq,
            self._rows(qkv, "qkv", T * (self.Hq + 2 * self.Hkv) * D), self.Hq,
            None if q_norm is None else self._rows(q_norm, "q_norm", D),
            None if k_norm is None else self._rows(k_norm, "k_norm", D), freq or None, 2 * pairs, eps,
            self._rows(q_out, "q_out", T * self.Hq * D), *self._ws, raw_stream(self._dev, stream))
        if rc:
            _check(rc, "moe_paged_append")

    def attend(self, layer, seqs, q, out, Tq=1, scale=None, stream=None):
        """Causal attention of the new tokens over their sequences' keys and values (scale: D^-1/2)."""
        B = self._batch(seqs)
        if Tq > self.max_new:
            raise ValueError(f"{Tq} new tokens a sequence: max_new is {self.max_new}")
        n = B * Tq * self.Hq * self.D
        rc = _lib.moe_paged_attend(self._c, layer, self._list(seqs, "seqs", B), B, Tq, self._rows(q, "q", n), self.Hq,
                                   self._default_scale if scale is None else scale, self._rows(out, "out", n),
                                   *self._ws, raw_stream(self._dev, stream))
        if rc:
            _check(rc, "moe_paged_attend")


def inv_frequencies(shape, device="cuda"):
    """theta^(-2 d / rope_dim), d < rope_dim / 2, in fp64: moe_paged_append's table for an AttnShape."""
    d = torch.arange(0, shape.rope_dim, 2, dtype=torch.float64)
    return (shape.theta ** (-d / shape.rope_dim)).to(device)


class PagedAttnBlock:
    """The attention branch of one layer for a batch over layer `index` of a paged cache. Blocks whose calls never overlap,
    as the layers of one step, may share a workspace: `ws`, another block's."""

    def __init__(self, layer, cache: PagedCache, index: int, inv_freq=None, ws=None):
        s = layer.shape
        _need(s.Hq == cache.Hq and s.Hkv == cache.Hkv and s.D == cache.D, "layer and cache differ in their heads")
        self.layer, self.cache, self.index = layer, cache, index
        self.inv_freq = inv_frequencies(s, cache.device) if inv_freq is None else inv_freq
        _need(self.inv_freq.dtype == torch.float64 and tuple(self.inv_freq.shape) == (s.rope_dim // 2,)
              and self.inv_freq.is_contiguous() and self.inv_freq.device == cache.device,
              f"inv_freq: expected contiguous float64 ({s.rope_dim // 2},)")
        n = _lib.moe_attn_paged_workspace_bytes(ctypes.byref(layer.c), cache._c, cache.max_batch, cache.max_new)
        if n == 0:
            raise ValueError("unsupported attention geometry")
        if ws is None:
            ws = torch.zeros(n, dtype=torch.uint8, device=cache.device)
            torch.cuda.current_stream(cache.device).synchronize()
        _need(ws.dtype == torch.uint8 and ws.numel() >= n and ws.is_contiguous() and ws.device == cache.device,
              f"ws: expected at least {n} contiguous bytes on {cache.device}")
        self.ws = ws

    def error_word(self, stream=None):
        rc = _lib.moe_paged_workspace_error(_ptr(self.ws), self.ws.numel(), raw_stream(self.cache._dev, stream))
        if rc < 0:
            raise MoeError(f"moe_paged_workspace_error failed: cudaError {-rc}")
        return rc

    def forward_rms(self, hidden, rms1, attn_out, seqs, Tq=1, stream=None):
        """AttnBlock.forward_rms for the batch: hidden fp32 [B Tq, H], attn_out bf16 bits [B Tq, H]; the sequences' lens
        already count the new tokens."""
        c, H = self.cache, self.layer.shape.H
        B = c._batch(seqs)
        _need(Tq <= c.max_new, f"{Tq} new tokens a sequence: max_new is {c.max_new}")
        if hidden.dtype is not _F32 or hidden.numel() != B * Tq * H or not hidden.is_contiguous() \
                or hidden.get_device() != c._dev:
            raise ValueError(f"hidden: expected contiguous float32 [{B * Tq}, {H}] on {c.device}")
        _check(_lib.moe_attn_paged_forward_rms(
            ctypes.byref(self.layer.c), c._rows(rms1, "rms1", H), hidden.data_ptr(), c._c, self.index,
            c._list(seqs, "seqs", B), B, Tq, self.inv_freq.data_ptr(), c._rows(attn_out, "attn_out", B * Tq * H),
            _ptr(self.ws), self.ws.numel(), raw_stream(c._dev, stream)), "moe_attn_paged_forward_rms")


class PagedDecodeStack:
    """The layers of a `stack.DecodeStack` over one paged cache: a step takes one or a few new tokens of each sequence
    of a batch. The weights are the given stack's; its contiguous caches are not used."""

    def __init__(self, stack, num_pages, page=64, max_seqs=64, max_pages=64, max_batch=8, max_new=1, kv="bf16",
                 k_scale=None, v_scale=None):
        a = stack.attn_shape
        self.stack = stack
        dev = stack.final_norm.device
        self.cache = PagedCache.empty(stack.L, num_pages, page, a.Hkv, a.D, a.Hq, max_seqs, max_pages, max_batch,
                                      max_new, kv, k_scale, v_scale, dev)
        f = inv_frequencies(a, dev)
        self.attn = []
        for i, b in enumerate(stack.attn):  # one after another in a step: one workspace for all
            self.attn.append(PagedAttnBlock(b.layer, self.cache, i, f, self.attn[0].ws if i else None))
        T = max_batch * max_new
        self.moe = [MoeBlock(b.layer, T) for b in stack.moe]
        self.normed = torch.zeros(T, a.H, dtype=torch.int16, device=dev)
        self.attn_out = torch.zeros(T, a.H, dtype=torch.int16, device=dev)
        torch.cuda.current_stream(dev).synchronize()  # the zeroing: steps may run on any stream

    def step(self, hidden, seqs, Tq=1, logits=None, stream=None):
        """One step for Tq new tokens of each listed sequence (-1: an unused slot): hidden fp32 [B Tq, H] is updated in
        place, and logits fp32 [B Tq, V] are written when given. The cache has been grown to the new lengths
        (cache.resize) beforehand."""
        from .spec import check_logits, lm_head_logits
        st, T = self.stack, seqs.numel() * Tq
        if logits is not None:  # refused before a layer has run
            check_logits(st.head.w, T, logits)
        for i in range(st.L):
            self.attn[i].forward_rms(hidden, st.rms1[i], self.attn_out[:T], seqs, Tq, stream)
            self.moe[i].forward(hidden, self.attn_out[:T], self.normed[:T],
                                next_rms1=st.final_norm if i + 1 == st.L else None, T=T, stream=stream)
        if logits is not None:
            lm_head_logits(st.head.w, self.normed[:T], logits, stream)

    def error_words(self, stream=None):
        """The cache's error word and the one that the attention blocks share, joined (read and cleared)."""
        e = self.cache.error_word(stream)
        for b in self.attn[:1]:
            e |= b.error_word(stream)
        return e
