"""CPU tests of the paged-cache and speculative-decoding entry points (include/moe_paged.h, include/moe_spec.h): what
they refuse before any launch, and how their workspaces are sized. No kernel is launched here."""
import ctypes

import pytest

BAD = 1  # cudaErrorInvalidValue
PTR = 1 << 20  # never dereferenced: every call below fails its checks first


def cache(**kw):
    import mvcc_b200 as m
    d = dict(k=PTR, v=PTR, tables=PTR, refs=PTR, lens=PTR, k_scale=None, v_scale=None, layers=2, num_pages=64, page=64,
             Hkv=2, D=256, kv_type=0, max_seqs=16, max_pages=32)
    d.update(kw)
    return m.MoePagedCache(*[d[n] for n, _ in m.MoePagedCache._fields_])


def lib():
    import mvcc_b200 as m
    return m._lib


@pytest.mark.parametrize("kw,ok", [
    ({}, True), ({"D": 128}, True), ({"D": 64}, True), ({"D": 64, "kv_type": 1}, False), ({"D": 128, "kv_type": 1}, True),
    ({"D": 96}, False), ({"kv_type": 2}, False), ({"page": 48}, True), ({"page": 8}, False), ({"page": 40}, False),
    ({"page": 2048}, False), ({"Hkv": 0}, False), ({"Hkv": 65}, False), ({"num_pages": 0}, False),
    ({"num_pages": (1 << 20) + 1}, False), ({"num_pages": 1 << 20}, True), ({"max_seqs": 0}, False),
    ({"max_seqs": 65537}, False), ({"max_pages": 0}, False), ({"max_pages": 1 << 24}, False), ({"layers": 0}, False),
    ({"k": None}, False), ({"v": PTR + 8}, False), ({"tables": None}, False), ({"refs": None}, False),
    ({"lens": None}, False),
])
def test_cache_check(kw, ok):
    assert (lib().moe_paged_check(ctypes.byref(cache(**kw))) == 0) == ok


def test_workspace_bytes():
    n = lib().moe_paged_workspace_bytes
    c = ctypes.byref(cache())
    assert n(c, 16, 8, 1) > 0 and n(c, 16, 8, 1) % 256 == 0
    assert n(c, 16, 8, 8) >= n(c, 16, 8, 2) >= n(c, 16, 8, 1)
    assert n(c, 16, 4096, 1) > 0 and n(c, 16, 8, 4096) == n(c, 16, 8, 8)  # long appends need nothing more
    assert n(c, 15, 8, 1) == 0 and n(c, 130, 8, 1) == 0 and n(c, 16, 0, 1) == 0 and n(c, 16, 4097, 1) == 0
    assert n(c, 16, 8, 0) == 0 and n(ctypes.byref(cache(D=100)), 16, 8, 1) == 0
    s = lib().moe_spec_workspace_bytes
    assert s(1, 151936) > 0 and s(64, 151936) > s(1, 151936)
    assert s(0, 10) == 0 and s(65536, 10) == 0 and s(1, 0) == 0 and s(1, 1 << 24) == 0


def test_workspace_holds_one_grid_of_partials():
    """Two parts a CTA, of 16 rows and their maxima and sums; heads of 256 run one CTA an SM, others two."""
    n = lib().moe_paged_workspace_bytes
    for D, ctas in ((256, 160), (128, 320), (64, 320)):
        assert n(ctypes.byref(cache(D=D)), 16, 8, 1) <= ctas * (2 * 16 * (D + 2) * 4 + 32) + 4096


def test_page_calls_refuse_before_launch():
    L, ws, big = lib(), ctypes.c_void_p(PTR), 1 << 40
    c = ctypes.byref(cache())
    bad = ctypes.byref(cache(page=8))
    for call in (L.moe_paged_resize, L.moe_paged_fork, L.moe_paged_copy):
        assert call(c, PTR, PTR, 4, None, big, None) == BAD          # no workspace
        assert call(c, PTR, PTR, 4, ws, 256, None) == BAD            # too small
        assert call(c, PTR, PTR, 4, PTR + 8, big, None) == BAD       # misaligned
        assert call(c, PTR, PTR, -1, ws, big, None) == BAD
        assert call(c, None, PTR, 4, ws, big, None) == BAD
        assert call(c, PTR, None, 4, ws, big, None) == BAD
        assert call(bad, PTR, PTR, 4, ws, big, None) == BAD
        assert call(None, PTR, PTR, 4, ws, big, None) == BAD
        assert call(c, None, None, 0, ws, big, None) == 0            # an empty list: nothing to do
    assert L.moe_paged_resize(c, PTR, PTR, 4097, ws, big, None) == BAD
    assert L.moe_paged_fork(c, PTR, PTR, 4097, ws, big, None) == BAD
    assert L.moe_paged_compact(c, ws, 256, None) == BAD and L.moe_paged_compact(bad, ws, big, None) == BAD


def test_attention_calls_refuse_before_launch():
    L, big = lib(), 1 << 40
    c = ctypes.byref(cache())

    def append(cc=c, layer=0, seqs=PTR, B=4, Tq=1, qkv=PTR, Hq=16, qn=PTR, kn=PTR, f=PTR, rope=64, q=PTR, ws=PTR, n=big):
        return L.moe_paged_append(cc, layer, seqs, B, Tq, qkv, Hq, qn, kn, f, rope, 1e-6, q, ws, n, None)

    def attend(cc=c, layer=0, seqs=PTR, B=4, Tq=1, q=PTR, Hq=16, out=PTR, ws=PTR, n=big):
        return L.moe_paged_attend(cc, layer, seqs, B, Tq, q, Hq, 0.0625, out, ws, n, None)

    for call in (append, attend):
        assert call(B=0) == 0
        for kw in ({"layer": 2}, {"layer": -1}, {"seqs": None}, {"B": -1}, {"B": 4097}, {"Tq": 0}, {"Hq": 15},
                   {"Hq": 0}, {"Hq": 130}, {"q": None}, {"q": PTR + 2}, {"ws": None}, {"ws": PTR + 4}, {"n": 256},
                   {"cc": None}, {"cc": ctypes.byref(cache(D=80))}):
            assert call(**kw) == BAD, kw
    for kw in ({"qn": None}, {"kn": None}, {"rope": 0}, {"f": None}, {"rope": 7}, {"rope": 258}, {"rope": -2},
               {"qkv": None}, {"qkv": PTR + 8}, {"B": 4096, "Tq": 1 << 12}):
        assert append(**kw) == BAD, kw
    for kw in ({"Tq": 9}, {"out": None}, {"out": PTR + 8}):
        assert attend(**kw) == BAD, kw
    # a batch whose key units could pass 32 bits
    assert attend(cc=ctypes.byref(cache(max_pages=1 << 23, Hkv=64)), Hq=64, B=2048) == BAD


def test_layer_call_refuses_before_launch():
    import mvcc_b200 as m
    L, big = lib(), 1 << 40
    w = m.MoeAttnWeights(PTR, None, PTR, PTR, PTR, 2048, 16, 2, 256, 64, 1e7, 1e-6)
    c = ctypes.byref(cache())
    n = L.moe_attn_paged_workspace_bytes
    assert n(ctypes.byref(w), c, 4, 2) > L.moe_paged_workspace_bytes(c, 16, 4, 2)
    assert n(ctypes.byref(w), c, 4, 9) == 0 and n(ctypes.byref(w), c, 0, 1) == 0
    assert n(ctypes.byref(w), ctypes.byref(cache(Hkv=4)), 4, 1) == 0 and n(ctypes.byref(w), ctypes.byref(cache(D=128)), 4,
                                                                         1) == 0

    def call(rms=PTR, h=PTR, cc=c, layer=0, seqs=PTR, B=4, Tq=1, f=PTR, out=PTR, ws=PTR, size=big):
        return L.moe_attn_paged_forward_rms(ctypes.byref(w), rms, h, cc, layer, seqs, B, Tq, f, out, ws, size, None)
    for kw in ({"rms": None}, {"h": None}, {"h": PTR + 4}, {"seqs": None}, {"B": 0}, {"Tq": 9}, {"f": None},
               {"out": None}, {"ws": None}, {"size": 256}, {"cc": ctypes.byref(cache(Hkv=4))},
               {"layer": -1}, {"layer": cache().layers}, {"cc": ctypes.byref(cache(k=None))}):
        assert call(**kw) == BAD, kw


@pytest.mark.parametrize("what", ["work", "q_norm", "k_norm"])
def test_layer_call_refuses_what_its_parts_would_before_any_launch(what):
    """A batch whose key units pass 32 bits (the attention's limit) and a misaligned norm (the append's): refused at once,
    not after the projections."""
    import mvcc_b200 as m
    L, big = lib(), 1 << 40
    w = m.MoeAttnWeights(PTR, None, PTR, PTR, PTR, 2048, 32, 32, 256, 64, 1e7, 1e-6)
    if what != "work":
        setattr(w, what, PTR + 8)
    cc = cache(Hkv=32, **({"max_pages": 1 << 13, "page": 64} if what == "work" else {}))
    m.reset_stats()
    assert L.moe_attn_paged_forward_rms(ctypes.byref(w), PTR, PTR, ctypes.byref(cc), 0, PTR, 4096, 1, PTR, PTR, PTR, big,
                                        None) == BAD
    assert m.stats()["launches"] == 0


def test_spec_calls_refuse_before_launch():
    L, big = lib(), 1 << 40

    def soft(x=PTR, ldx=100, R=4, V=100, y=PTR * 2, ldy=100):
        return L.moe_softmax_rows(x, ldx, R, V, None, y, ldy, None)
    assert soft(R=0) == 0
    for kw in ({"x": None}, {"y": None}, {"R": -1}, {"V": 0}, {"V": 1 << 24, "ldx": 1 << 24, "ldy": 1 << 24}, {"ldx": 99},
               {"ldy": 99}, {"y": PTR, "ldy": 101}):
        assert soft(**kw) == BAD, kw

    def verify(t=PTR, ldt=100, d=PTR, ldd=100, x=PTR, u=PTR, B=4, K=3, V=100, tok=PTR, acc=PTR, ws=PTR, n=big):
        return L.moe_spec_verify(t, ldt, d, ldd, x, None, u, B, K, V, tok, acc, ws, n, None)
    assert verify(B=0) == 0 and verify(K=0, d=None, x=None, tok=None) == BAD
    for kw in ({"t": None}, {"ldt": 99}, {"ldd": 99}, {"x": None}, {"u": None}, {"B": -1}, {"B": 65536}, {"K": -1},
               {"K": 65}, {"V": 0}, {"tok": None}, {"acc": None}, {"ws": None}, {"ws": PTR + 4}, {"n": 256}):
        assert verify(**kw) == BAD, kw
    for args in ((None, PTR, 100, 64, 1, PTR), (PTR, None, 100, 64, 1, PTR), (PTR, PTR, 0, 64, 1, PTR),
                 (PTR, PTR, 100, 60, 1, PTR), (PTR, PTR, 100, 64, 0, PTR), (PTR, PTR, 100, 64, 5, PTR),
                 (PTR, PTR, 100, 64, 1, None), (PTR + 8, PTR, 100, 64, 1, PTR), (PTR, PTR, 100, 8200, 1, PTR)):
        assert L.moe_lm_head_logits(*args, None) == BAD, args


def test_refused_calls_count_no_launch():
    import mvcc_b200 as m
    m.reset_stats()
    test_page_calls_refuse_before_launch()
    test_attention_calls_refuse_before_launch()
    test_spec_calls_refuse_before_launch()
    assert m.stats()["launches"] == 0


@pytest.mark.parametrize("argv", [["--draft", "2"], ["--batch", "2", "--draft", "8"], ["--batch", "-1"]])
def test_stack_command_refuses_its_arguments(argv):
    from mvcc_b200 import stack
    with pytest.raises(SystemExit):
        stack.main(argv)
