"""GPU tests of the step from logits to tokens (include/moe_spec.h): several tokens' logits, softmax rows, and the
verification of drafts, against 64-bit restatements."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def S():
    from mvcc_b200 import spec
    return spec


# ------------------------------------------------------------------ logits

@pytest.mark.parametrize("V,H,T", [(1000, 256, 1), (999, 2048, 4), (70, 8, 3), (5000, 8192, 7), (20000, 1024, 2)])
def test_lm_head_logits(V, H, T):
    g = torch.Generator(device="cuda").manual_seed(V)
    w = (0.05 * torch.randn(V, H, generator=g, device="cuda")).to(torch.bfloat16)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    out = torch.full((T, V), 7.0, device="cuda")
    S().lm_head_logits(w.view(torch.int16), x.view(torch.int16), out)
    want = x.double() @ w.double().T
    mag = x.double().abs() @ w.double().abs().T
    assert bool(((out.double() - want).abs() <= (H // 32 + 8) * F32 * mag + 1e-30).all())  # a lane's chain, then the tree
    if T == 1:  # the same numbers as the argmax head's
        from mvcc_b200 import stack as st
        l1, nxt = torch.zeros(V, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        st.LmHead(w.view(torch.int16)).argmax(x.view(torch.int16)[0], nxt, logits=l1)
        assert torch.equal(l1, out[0])


# ------------------------------------------------------------------ softmax

def softmax64(x, t):
    """[R, V] doubles, by the header's words; t doubles [R]."""
    out = torch.zeros_like(x)
    for i in range(x.shape[0]):
        v = torch.where(torch.isnan(x[i]), -math.inf, x[i])
        m = v.max()
        if m == -math.inf:
            continue
        if not t[i] > 0:
            out[i, int(torch.nonzero(v == m)[0, 0])] = 1.0
            continue
        e = torch.where(v == m, 1.0, torch.exp((v - m) / t[i]))
        out[i] = e / e.sum()
    return out


def near(got, x, t):
    """2^-20 (the exponential) plus a few roundings of its argument, relative; below fp32's normal range zero will do."""
    want = softmax64(x.double(), t.double())
    v = torch.where(torch.isfinite(x), x, 0.0).double()
    top = torch.where(torch.isfinite(x), x, -math.inf).amax(1, keepdim=True).double()
    arg = torch.where(torch.isfinite(x.double() - top), (v - top) / torch.where(t > 0, t, 1.0).double()[:, None], 0.0)
    arg = arg.abs().clamp(max=110)
    tol = want * (2.0 ** -20 + 8 * F32 * (1 + arg)) + 2.0 ** -120
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 7), (4, 151936), (9, 1001), (2, 20480), (2, 20484), (3, 40961),
                                 (2, 163840), (2, 163844), (1, 200001), (2, 262144), (1, 262145), (1, 600000), (70, 640)])
def test_softmax_rows(R, V):
    g = torch.Generator(device="cuda").manual_seed(R * V)
    x = 4 * torch.randn(R, V, generator=g, device="cuda")
    t = 0.3 + torch.rand(R, generator=g, device="cuda")
    t[1::3] = 0.0
    out = torch.full_like(x, 9.0)
    S().softmax_rows(x, out, temperature=t)
    near(out, x, t)
    S().softmax_rows(x, out)
    near(out, x, torch.ones_like(t))
    again = x.clone()
    S().softmax_rows(again, again)  # in place
    assert torch.equal(again, out)


@pytest.mark.parametrize("V", [37, 4096, 50001, 270000])
def test_softmax_of_masked_and_infinite_rows(V):
    x = torch.randn(9, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
    low = torch.finfo(torch.float32).min
    x[0] = -math.inf                        # nothing
    x[1], x[1, V // 2] = -math.inf, -3.0    # one left
    x[2, ::2] = low                         # masks of the type's lowest value
    x[3] = low                              # all of them: equal
    x[4, 5], x[4, V - 1] = math.inf, math.inf
    x[5] = math.nan
    x[6, 3], x[6, V // 3] = math.nan, -math.inf
    x[7] = 1.5                              # ties
    x[8, 7:] = -math.inf
    for t in (1.0, 0.0, -1.0, math.nan, 1e-3, 1e-40, 1e30):
        tt = torch.full((9,), t, device="cuda")
        out = torch.full_like(x, 9.0)
        S().softmax_rows(x, out, temperature=tt)
        if t == 1e-40:  # anything below the maximum is gone
            want = softmax64(x.double(), torch.full((9,), 1e-12, device="cuda").double())
            assert bool(((out.double() - want).abs() <= 2.0 ** -20 * want + 2.0 ** -120).all())
        else:
            near(out, x, tt)


@pytest.mark.parametrize("V", [1, 37, 4096, 50001, 151936, 270000])
def test_softmax_at_an_infinite_temperature_shares_equally(V):
    x = 9 * torch.randn(5, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
    x[1, ::3] = -math.inf
    x[2, V // 2] = math.nan
    x[3] = -math.inf
    x[4, V - 1] = math.inf
    out = torch.full_like(x, 9.0)
    S().softmax_rows(x, out, temperature=torch.full((5,), math.inf, device="cuda"))
    on = x > -math.inf  # False for a NaN
    on[4, :V - 1] = False
    want = on.double() / on.sum(1, keepdim=True).clamp(min=1).double()
    # the sum of up to V ones: its rounding, a chain's and a tree's, then the division's and the product's
    assert bool(((out.double() - want).abs() <= 2.0 ** -20 * want).all())


@pytest.mark.parametrize("R,V", [(64, 40961), (16, 151936), (2, 20484), (300, 163844), (3, 270000)])
def test_softmax_of_clusters_that_start_beside_other_work(R, V):
    """Rows shared by clusters of 2 to 8 CTAs, launched back to back on two streams beside a kernel that keeps the GPU's
    places busy, so that a cluster's CTAs start as room comes: the same bits every time."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = 3 * torch.randn(R, V, generator=g, device="cuda")
    want = torch.empty_like(x)
    S().softmax_rows(x, want)
    near(want, x, torch.ones(R, device="cuda"))
    busy = torch.randn(2048, 2048, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.full_like(x, 9.0) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(streams[2]):
            torch.mm(busy, busy)
        for out, s in zip(outs, streams):
            S().softmax_rows(x, out, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_softmax_keeps_what_lies_between_rows():
    x = torch.randn(6, 1000, device="cuda")
    y = torch.full((6, 1003), 5.0, device="cuda")
    S().softmax_rows(x[:, 1:777], y[:, 2:778])  # rows at odd places
    assert bool((y[:, :2] == 5).all()) and bool((y[:, 778:] == 5).all())
    near(y[:, 2:778].contiguous(), x[:, 1:777].contiguous(), torch.ones(6, device="cuda"))
    with pytest.raises(ValueError):
        S().softmax_rows(x.T, y[:, :6].T)
    with pytest.raises(ValueError):
        S().softmax_rows(x, y)
    with pytest.raises(ValueError):
        S().softmax_rows(x, torch.empty_like(x), temperature=torch.ones(5, device="cuda"))


# ------------------------------------------------------------------ verification

def verify64(p, q, x, u, n):
    """(tokens, accepted, gap) by the header's words, in numpy doubles. gap: how near, relative to the total, the drawn
    token's border is to the target: draws nearer than the sums' order can decide are left out of a comparison."""
    B, K1, V = p.shape
    K = K1 - 1
    clean = lambda a: np.where((a > 0) & np.isfinite(a), a, 0.0)  # noqa: E731
    p = clean(p)
    q = None if q is None else clean(q)
    tokens, acc, gap = np.full((B, K1), -1), np.zeros(B, int), np.ones(B)
    for b in range(B):
        m = K if n is None else min(max(int(n[b]), 0), K)
        a = 0
        while a < m:
            t = int(x[b, a])
            if not 0 <= t < V:
                break
            if not u[b, a] * (1.0 if q is None else q[b, a, t]) < p[b, a, t]:
                break
            tokens[b, a] = t
            a += 1
        w = p[b, a].copy()
        if a < m:
            if q is not None:
                w = np.maximum(w - q[b, a], 0)
            elif 0 <= x[b, a] < V:
                w[x[b, a]] = max(w[x[b, a]] - 1.0, 0)
        if not w.sum() > 0:
            w = p[b, a]
        acc[b] = a
        if not w.sum() > 0:
            continue
        run = np.cumsum(w)
        hit = np.flatnonzero((run > u[b, K] * run[-1]) & (w > 0))
        tokens[b, a] = hit[0] if len(hit) else np.flatnonzero(w > 0)[-1]
        gap[b] = np.abs(run - u[b, K] * run[-1]).min() / run[-1]
    return tokens, acc, gap


def run_verify(p, q, x, u, n=None, ver=None):
    B, K1, V = p.shape
    ver = ver or S().SpecVerifier(B, K1 - 1, V)
    tok = torch.full((B, K1), 55, dtype=torch.int32, device="cuda")
    acc = torch.full((B,), 55, dtype=torch.int32, device="cuda")
    ver.verify(p, q, x, u, tok, acc, n_drafted=n)
    return tok.cpu().numpy(), acc.cpu().numpy()


def compare(p, q, x, u, n=None, ver=None, least=0.9):
    tok, acc = run_verify(p, q, x, u, n, ver)
    d = lambda t: None if t is None else t.cpu().numpy().astype(np.float64)  # noqa: E731
    want, wacc, gap = verify64(d(p), d(q), x.cpu().numpy(), d(u), None if n is None else n.cpu().numpy())
    assert np.array_equal(acc, wacc)
    safe = gap > 1e-13  # V x 2^-53 and a margin
    assert safe.mean() >= least
    assert np.array_equal(tok[safe], want[safe])
    return tok, acc


def Draw(B, V):
    """A verifier that draws without drafts, called as one with drafts is."""
    ver = S().SpecVerifier(B, 0, V)
    verify = ver.verify
    ver.verify = lambda p, q, x, u, tok, acc, n_drafted=None: verify(p, None, None, u, tok, acc)
    return ver


def drafts(B, K, V, seed, noise=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 2 * torch.randn(B, K + 1, V, generator=g, device="cuda")
    p = torch.softmax(z, -1)
    y = z[:, :K] + noise * torch.randn(B, K, V, generator=g, device="cuda")
    q = torch.softmax(y, -1)
    x = (y - torch.log(-torch.log(torch.rand(B, K, V, generator=g, device="cuda").clamp(1e-30, 1 - 1e-7)))).argmax(-1)
    return p, q, x.int(), torch.rand(B, K + 1, generator=g, device="cuda")


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (2, 1, 2), (40, 3, 5), (33, 2, 4096), (9, 4, 4097), (64, 4, 8191),
                                   (5, 3, 151936), (3, 64, 300), (3, 33, 1000), (1, 2, 600001), (300, 1, 50)])
def test_verify_against_64_bits(B, K, V):
    p, q, x, u = drafts(B, K, V, seed=B + K + V)
    ver = S().SpecVerifier(B, K, V)
    _, a1 = compare(p, q, x, u, ver=ver)
    compare(p, None, x, u, ver=ver)
    g = torch.Generator(device="cuda").manual_seed(1)
    n = torch.randint(-1, K + 2, (B,), generator=g, device="cuda").int()
    compare(p, q, x, u, n=n, ver=ver)
    compare(p, None, x, u, n=n, ver=ver)
    assert np.array_equal(run_verify(p, q, x, u, ver=ver)[1], a1)  # the tickets came back to zero
    if B >= 30 and V > 100 and K > 1:
        assert len(set(a1.tolist())) > 1  # some rejected, some not


def test_verify_draws_by_the_residual_distribution():
    """Over many sequences the emitted first token follows the target's probabilities, whatever the draft's are."""
    V, B = 6, 60000
    p = torch.tensor([0.05, 0.3, 0.0, 0.4, 0.15, 0.1], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.2, 0.2, 0.1, 0.1], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.multinomial(q.expand(B, V), 1, generator=g).int()
    u = torch.rand(B, 2, generator=g, device="cuda")
    tok, _ = run_verify(p.expand(B, 2, V).contiguous(), q.expand(B, 1, V).contiguous(), x, u)
    got = np.bincount(tok[:, 0], minlength=V) / B
    sigma = np.sqrt(np.maximum(p.cpu().numpy() * (1 - p.cpu().numpy()), 0) / B)
    assert (np.abs(got - p.cpu().numpy()) <= 5 * sigma + 1e-12).all(), got


def test_verify_at_borders_and_with_bad_values():
    K, V = 2, 10000
    p = torch.zeros(10, K + 1, V, device="cuda")
    q = torch.zeros(10, K, V, device="cuda")
    x = torch.zeros(10, K, dtype=torch.int32, device="cuda")
    u = torch.full((10, K + 1), 0.5, device="cuda")
    p[:, :, 4000:4004] = 0.25
    q[:, :, 4000:4004] = 0.25
    x[:] = 4001
    u[0] = 0.0                          # accepted; the draw: the first token with weight
    u[1] = 1.0                          # out of range: u q < p fails, p = q leaves no residual: drawn from p, its last
    x[2, 0] = -1                        # no such token
    x[3, 1] = V
    x[4, 0] = 7                         # p and q zero there
    p[5, 0, 4001] = math.nan
    q[6, 0, 4001] = math.inf            # counts as zero: accepted
    p[7] = 0.0                          # nothing to draw from
    p[8, 0], p[8, 0, 9999] = 0.0, 1.0   # residual at the very end
    x[8, 0], q[8, 0], q[8, 0, 9998] = 9998, 0.0, 1.0
    p[9, :, 0], p[9, :, 4002], p[9, :, 4003] = -3.0, math.inf, math.nan
    tok, acc = compare(p, q, x, u, least=0.0)
    assert acc.tolist() == [2, 0, 0, 1, 0, 0, 2, 0, 0, 2]
    assert tok[0].tolist() == [4001, 4001, 4000] and tok[1].tolist() == [4003, -1, -1]
    assert tok[7].tolist() == [-1, -1, -1] and tok[8].tolist() == [9999, -1, -1]
    assert tok[2, 0] == 4002 and tok[3].tolist() == [4001, 4002, -1] and tok[4, 0] == 4002
    assert tok[5, 0] in (4000, 4002, 4003) and tok[9, 2] == 4001


@pytest.mark.parametrize("V", [8, 1001, 40000])
def test_verify_of_probabilities_below_the_normal_range(V):
    """Rows whose entries are all tiny, normal and subnormal ones together: weights and their sums as fp64 holds them."""
    B, K = 64, 1
    g = torch.Generator(device="cuda").manual_seed(V)
    p = torch.rand(B, K + 1, V, generator=g, device="cuda") * 2.0 ** -125  # a half of them below 2^-126
    q = torch.rand(B, K, V, generator=g, device="cuda") * 2.0 ** -125
    p[::4, :, ::2] = 0.0
    x = torch.randint(V, (B, K), generator=g, device="cuda").int()
    u = torch.rand(B, K + 1, generator=g, device="cuda")
    compare(p, q, x, u)
    compare(p, None, x, u)
    compare(p[:, :1].contiguous(), None, x[:, :0], u[:, :1].contiguous(), ver=Draw(B, V))


def test_verify_of_rows_apart_on_another_stream_and_in_a_graph():
    B, K, V = 6, 3, 5003
    p, q, x, u = drafts(B, K, V, seed=2)
    wide_p, wide_q = torch.full((B, K + 1, V + 5), 9.0, device="cuda"), torch.full((B, K, V + 9), 9.0, device="cuda")
    wide_p[..., :V], wide_q[..., :V] = p, q
    ver = S().SpecVerifier(8, K, V)  # a workspace for more
    tok, acc = run_verify(p, q, x, u, ver=ver)
    t2, a2 = run_verify(wide_p[..., :V], wide_q[..., :V], x, u, ver=ver)
    assert np.array_equal(tok, t2) and np.array_equal(acc, a2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    tt, aa = torch.zeros(B, K + 1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            ver.verify(p, q, x, u, tt, aa)
        for _ in range(3):
            u.copy_(torch.rand(B, K + 1, device="cuda"))
            graph.replay()
            s.synchronize()
            want, wacc, gap = verify64(p.double().cpu().numpy(), q.double().cpu().numpy(), x.cpu().numpy(),
                                       u.double().cpu().numpy(), None)
            assert np.array_equal(aa.cpu().numpy(), wacc) and np.array_equal(tt.cpu().numpy()[gap > 1e-13],
                                                                             want[gap > 1e-13])
    for bad in (lambda: ver.verify(p[:, :, ::2], q, x, u, tt, aa), lambda: ver.verify(p, q[:, :2], x, u, tt, aa),
                lambda: ver.verify(p, q, x.long(), u, tt, aa), lambda: ver.verify(p.cpu(), q, x, u, tt, aa),
                lambda: ver.verify(p.repeat(2, 1, 1), q, x, u, tt, aa), lambda: ver.verify(p, q, x, u, tt[:, :2], aa)):
        with pytest.raises(ValueError):
            bad()


def test_softmax_of_many_short_rows_and_two_streams_of_long_ones():
    g = torch.Generator(device="cuda").manual_seed(5)
    x = 3 * torch.randn(70000, 9, generator=g, device="cuda")
    out = torch.empty_like(x)
    S().softmax_rows(x, out)
    want = torch.softmax(x.double(), -1)
    assert float((out.double() - want).abs().max()) <= 2.0 ** -19
    a, b = torch.randn(40, 100000, generator=g, device="cuda"), torch.randn(30, 151936, generator=g, device="cuda")
    oa, ob = torch.empty_like(a), torch.empty_like(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        S().softmax_rows(a, oa, stream=s1)
        S().softmax_rows(b, ob, stream=s2)
    torch.cuda.synchronize()
    near(oa, a, torch.ones(40, device="cuda"))
    near(ob, b, torch.ones(30, device="cuda"))


def test_one_verifier_serves_batches_of_every_size_in_turn():
    K, V = 3, 4000
    ver = S().SpecVerifier(70, K, V)
    for B in (1, 70, 2, 33, 70, 1):
        p, q, x, u = drafts(B, K, V, seed=B)
        compare(p, q, x, u, ver=ver, least=0.0)


@pytest.mark.parametrize("B,V", [(1, 1), (7, 5), (64, 4096), (5, 151936)])
def test_a_token_is_drawn_without_drafts(B, V):
    """K = 0: one draw a sequence, by the running sum; at temperature 0 the likeliest token."""
    g = torch.Generator(device="cuda").manual_seed(B)
    z = 3 * torch.randn(B, V, generator=g, device="cuda")
    p, u = torch.empty_like(z), torch.rand(B, 1, generator=g, device="cuda")
    ver = S().SpecVerifier(B, 0, V)
    tok, acc = torch.zeros(B, 1, dtype=torch.int32, device="cuda"), torch.full((B,), 9, dtype=torch.int32, device="cuda")
    for t in (0.8, 0.0):
        S().softmax_rows(z, p, temperature=torch.full((B,), t, device="cuda"))
        ver.verify(p.view(B, 1, V), None, None, u, tok, acc)
        want, _, gap = verify64(p.view(B, 1, V).double().cpu().numpy(), None, None, u.double().cpu().numpy(), None)
        safe = gap > 1e-13 if t else np.ones(B, bool)
        assert np.array_equal(tok.cpu().numpy()[safe], want[safe]) and not bool(acc.any())
        if t == 0:
            assert tok[:, 0].tolist() == z.argmax(-1).tolist()


@pytest.mark.parametrize("B", [1, 5])
def test_one_row_a_sequence_may_lie_anywhere(B):
    """K = 0 over the first row of several, or over rows padded apart; K = 1 over one draft's row of several: torch gives a
    dimension of one any stride."""
    V = 1003
    g = torch.Generator(device="cuda").manual_seed(B)
    p = torch.softmax(2 * torch.randn(B, 4, V, generator=g, device="cuda"), -1)
    u = torch.rand(B, 1, generator=g, device="cuda")
    empty = torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    want = run_verify(p[:, :1].contiguous(), None, empty, u, ver=Draw(B, V))[0]
    padded = torch.full((B, V + 13), 9.0, device="cuda")
    padded[:, :V] = p[:, 0]
    for t in (p[:, :1], padded[:, None, :V], padded[:, :V].unsqueeze(1), p[:, 0].contiguous().view(B, 1, V)):
        assert np.array_equal(run_verify(t, None, empty, u, ver=Draw(B, V))[0], want)
    q = torch.softmax(2 * torch.randn(B, 3, V, generator=g, device="cuda"), -1)
    x, u2 = torch.randint(V, (B, 1), generator=g, device="cuda").int(), torch.rand(B, 2, generator=g, device="cuda")
    t = p[:, :2].contiguous()
    a, b = run_verify(t, q[:, :1].contiguous(), x, u2), run_verify(t, q[:, :1], x, u2)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    if B > 1:  # two rows of four: not one distance for all
        with pytest.raises(ValueError):
            run_verify(p[:, :2], None, x, u2)
