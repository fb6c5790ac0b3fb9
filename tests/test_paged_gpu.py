"""GPU tests of the paged cache (include/moe_paged.h): the page calls against a sequential model, the write of new keys
and values and the attention against 64-bit restatements, and a batch's step against the single-sequence stack."""
import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8  # half a step of bf16, relative
F32 = 2.0 ** -24


def P():
    from mvcc_b200 import paged
    return paged


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bits(x):
    return x.to(torch.bfloat16).view(torch.int16)


def vals(t):
    return t.view(torch.bfloat16).double()


# ------------------------------------------------------------------ pages

class Model:
    """The page calls one sequence after another, on the host."""

    def __init__(self, c):
        self.page = c.page
        self.tables, self.refs, self.lens = (t.cpu().numpy().copy() for t in (c.tables, c.refs, c.lens))
        self.k, self.v = c.k.cpu().numpy().copy(), c.v.cpu().numpy().copy()

    def held(self, n):
        return -(-n // self.page)

    def resize(self, seqs, new):
        old = (self.tables.copy(), self.refs.copy())
        for s, n in zip(seqs, new):
            for j in range(self.held(n), self.held(self.lens[s])):
                self.refs[self.tables[s, j]] -= 1
                self.tables[s, j] = -1
        copies = []
        free = None
        for s, n in zip(seqs, new):  # who copies is settled before any page is taken
            kept = min(self.lens[s], n)
            if kept % self.page:
                p = self.tables[s, kept // self.page]
                if self.refs[p] > 1:
                    self.refs[p] -= 1
                    copies.append((s, kept, p))
        free = [int(p) for p in np.flatnonzero(self.refs == 0)]
        take = iter(free)
        done = []
        try:
            for s, n in zip(seqs, new):
                for cs, kept, p in copies:
                    if cs == s:
                        d = next(take)
                        self.tables[s, kept // self.page] = d
                        self.refs[d] = 1
                        done.append((p, d, kept % self.page))
                for j in range(self.held(self.lens[s]), self.held(n)):
                    d = next(take)
                    self.tables[s, j] = d
                    self.refs[d] = 1
        except StopIteration:
            self.tables, self.refs = old
            return False
        for p, d, rows in done:
            for t in (self.k, self.v):
                t[:, d, :, :rows] = t[:, p, :, :rows]
        for s, n in zip(seqs, new):
            self.lens[s] = n
        return True

    def fork(self, src, dst):
        for s, d in zip(src, dst):
            self.tables[d] = self.tables[s]
            self.lens[d] = self.lens[s]
            for p in self.tables[s]:
                if p >= 0:
                    self.refs[p] += 1

    def compact(self):
        n = int((self.refs != 0).sum())
        holes = [p for p in range(n) if self.refs[p] == 0]
        high = [p for p in range(n, len(self.refs)) if self.refs[p] != 0]
        for d, p in zip(holes, high):
            for t in (self.k, self.v):
                t[:, d] = t[:, p]
            self.refs[d], self.refs[p] = self.refs[p], 0
            self.tables[self.tables == p] = d

    def same(self, c):
        torch.cuda.synchronize()
        for n in ("tables", "refs", "lens", "k", "v"):
            assert np.array_equal(getattr(c, n).cpu().numpy(), getattr(self, n)), n


def make(layers=2, pages=40, page=16, Hkv=2, D=64, max_seqs=12, max_pages=8, kv="bf16", seed=0, **kw):
    c = P().PagedCache.empty(layers, pages, page, Hkv, D, kw.pop("Hq", Hkv), max_seqs, max_pages,
                             kw.pop("max_batch", max_seqs), kw.pop("max_new", 1), kv, **kw)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (c.k, c.v):
        if kv == "bf16":
            t.copy_(bits(torch.randn(t.shape, generator=g, device="cuda")))
        else:
            t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 40).to(torch.float8_e4m3fn).view(torch.uint8))
    torch.cuda.synchronize()
    return c


@pytest.mark.parametrize("kw", [dict(), dict(page=48, D=128, layers=3), dict(kv="e4m3", D=128, Hkv=1),
                                dict(pages=9000, max_pages=700, max_seqs=40, layers=1, Hkv=1)])
@pytest.mark.parametrize("seed", [0, 1])
def test_page_calls_follow_the_sequential_model(kw, seed):
    c = make(seed=seed, **kw)
    m = Model(c)
    r = random.Random(seed)
    most = c.max_pages * c.page
    failed = 0
    for step in range(60):
        what = r.choice(("grow", "grow", "grow", "any", "fork", "free", "compact"))
        some = r.sample(range(c.max_seqs), r.randint(1, c.max_seqs))
        if what in ("grow", "any", "free"):
            new = [0 if what == "free" and r.random() < 0.7 else
                   (min(most, int(m.lens[s]) + r.randint(0, 2 * c.page)) if what == "grow" else r.randint(0, most))
                   for s in some]
            c.resize(i32(some), i32(new))
            ok = m.resize(some, new)
            assert c.error_word() == (0 if ok else P().ERR_NO_PAGES)
            failed += not ok
        elif what == "fork":
            dst = [s for s in some if m.lens[s] == 0]
            src = [s for s in range(c.max_seqs) if s not in dst]
            if not dst or not src:
                continue
            src = [r.choice(src) for _ in dst]
            c.fork(i32(src), i32(dst))
            m.fork(src, dst)
            assert c.error_word() == 0
        else:
            c.compact()
            m.compact()
            assert c.error_word() == 0
        m.same(c)
    assert failed > 0 or c.num_pages > 1000  # the run met a full pool


def test_resize_to_the_same_length_and_of_all_sequences_at_once():
    c = make(pages=300, max_seqs=2048, max_pages=2, layers=1, Hkv=1, max_batch=2048)
    m = Model(c)
    seqs = list(range(2048))
    new = [5 if s % 8 == 0 else 0 for s in seqs]
    c.resize(i32(seqs), i32(new))
    assert m.resize(seqs, new)
    m.same(c)
    src, dst = [0] * 1024, [s for s in seqs if s % 8][:1024]
    c.fork(i32(src), i32(dst))
    m.fork(src, dst)
    m.same(c)
    lst = [0] + dst[:20]
    c.resize(i32(lst), i32([int(m.lens[s]) for s in lst]))  # each gets a page of its own
    assert m.resize(lst, [int(m.lens[s]) for s in lst])
    m.same(c)
    c.resize(i32(seqs), i32([32] * 2048))
    assert not m.resize(seqs, [32] * 2048)
    assert c.error_word() == P().ERR_NO_PAGES
    m.same(c)
    c.resize(i32(seqs), i32([0] * 2048))
    assert m.resize(seqs, [0] * 2048)
    m.same(c)
    assert int(c.refs.abs().sum()) == 0


def test_page_calls_with_bad_lists_change_nothing():
    c = make()
    c.resize(i32([0, 1]), i32([40, 20]))
    m = Model(c)
    for seqs, new in (([0, 0], [1, 1]), ([12], [3]), ([-1], [3]), ([0], [-1]), ([0, 1], [5, 8 * 16 + 1])):
        c.resize(i32(seqs), i32(new))
        assert c.error_word() == P().ERR_SEQ_ID
        m.same(c)
    for src, dst in (([0], [1]), ([0, 0], [2, 2]), ([0], [0]), ([0, 2], [2, 3]), ([0], [12]), ([-1], [2]), ([99], [2])):
        c.fork(i32(src), i32(dst))
        assert c.error_word() == P().ERR_SEQ_ID
        m.same(c)
    c.copy_pages(i32([0, 99, 1, 2]), i32([10, 11, -1, 13]))
    assert c.error_word() == P().ERR_PAGE_ID
    for t in (m.k, m.v):
        t[:, 10], t[:, 13] = t[:, 0], t[:, 2]
    m.same(c)
    c.lens[3] = 10 ** 6  # a length that the table cannot hold
    c.resize(i32([3]), i32([1]))
    assert c.error_word() == P().ERR_SEQ_ID


def test_lists_on_the_wrong_type_or_place_are_refused():
    c = make()
    with pytest.raises(ValueError):
        c.resize(i32([0]).long(), i32([1]))
    with pytest.raises(ValueError):
        c.resize(torch.tensor([0], dtype=torch.int32), i32([1]))
    with pytest.raises(ValueError):
        c.resize(i32([0, 1]), i32([1]))
    with pytest.raises(ValueError):
        c.resize(i32([0, 0, 1, 1])[::2], i32([1, 1]))
    with pytest.raises(ValueError):
        c.resize(i32(list(range(13))), i32([0] * 13))  # more than max_batch
    with pytest.raises(ValueError):
        P().PagedCache(c.k, c.v, c.tables, c.refs[:-1], c.lens, 2, 4)
    with pytest.raises(ValueError):
        P().PagedCache(c.k, c.v, c.tables, c.refs, c.lens, 3, 4)  # Hq % Hkv
    with pytest.raises(ValueError):
        P().PagedCache(c.k, c.v, c.tables, c.refs, c.lens, 2, 4, k_scale=torch.ones(2, 2, device="cuda"))  # bf16


# ------------------------------------------------------------------ the write

def rotate64(x, w, pos, inv_freq, eps=1e-6):
    """[T, heads, D] doubles: norm and rotation, as the header states them."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    if inv_freq is None:
        return x
    h = inv_freq.numel()
    a = pos.double()[:, None] * inv_freq
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    return torch.cat([x[..., :h] * c - x[..., h:2 * h] * s, x[..., h:2 * h] * c + x[..., :h] * s, x[..., 2 * h:]], -1)


@pytest.mark.parametrize("D,page,Hq,Hkv,rope,Tq,norm", [
    (256, 64, 16, 2, 64, 1, True), (256, 16, 8, 8, 256, 3, True), (128, 48, 10, 2, 6, 37, True), (64, 32, 3, 1, 2, 5, True),
    (64, 16, 4, 4, 0, 1, True), (128, 64, 8, 1, 128, 130, False), (256, 32, 4, 2, 0, 2, False),
    # several tokens a CTA, and several rounds of them
    (128, 64, 4, 2, 128, 301, True), (256, 128, 2, 2, 64, 300, True), (64, 256, 2, 1, 6, 1001, True)])
def test_append_against_64_bits(D, page, Hq, Hkv, rope, Tq, norm):
    far = 200_000 // page
    c = make(layers=2, pages=60, page=page, Hkv=Hkv, D=D, max_seqs=6, max_pages=far, Hq=Hq, max_new=Tq)
    g = torch.Generator(device="cuda").manual_seed(3)
    # sequence 0 is new, 1 far into its cache, 2 shorter than the new tokens, 4 between; slot 3 is unused
    lens = [Tq, far * page - 5, max(0, Tq - 2), 0, page + Tq]
    seqs = [1, 0, 2, -1, 4]
    nxt = 0
    for s, n in enumerate(lens):
        for j in range(max(0, (n - Tq) // page), -(-n // page)):
            c.tables[s, j] = nxt
            c.refs[nxt] = 1
            nxt += 1
    c.lens[:5] = i32(lens)
    k0, v0 = c.k.clone(), c.v.clone()
    T = len(seqs) * Tq
    qkv = bits(torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda"))
    qn = bits(1 + 0.1 * torch.randn(D, generator=g, device="cuda")) if norm else None
    kn = bits(1 + 0.1 * torch.randn(D, generator=g, device="cuda")) if norm else None
    f = (1e7 ** (-torch.arange(0, rope, 2, dtype=torch.float64) / rope)).cuda() if rope else None
    q = torch.full((T, Hq * D), 77, dtype=torch.int16, device="cuda")
    c.append(1, i32(seqs), qkv, q, Tq=Tq, q_norm=qn, k_norm=kn, inv_freq=f)
    assert c.error_word() == 0
    x = vals(qkv).view(T, Hq + 2 * Hkv, D)
    pos = torch.tensor([lens[s] - Tq + t if s >= 0 else -1 for s in seqs for t in range(Tq)], device="cuda")
    live = torch.tensor([s >= 0 for s in seqs for t in range(Tq)], device="cuda") & (pos >= 0)
    qe = rotate64(x[:, :Hq], vals(qn) if norm else None, pos, f)
    ke = rotate64(x[:, Hq:Hq + Hkv], vals(kn) if norm else None, pos, f)
    ve = x[:, Hq + Hkv:]
    # one rounding to bf16; before it at most eight fp32 roundings of each of a pair's two terms (the mean, its root, two
    # products, sine or cosine at 2 ulp, the product, the sum)
    def near(got, want, scale):
        err = (got - want).abs()
        assert bool((err <= BF * want.abs() + 24 * F32 * scale + 1e-30).all()), float((err - BF * want.abs()).max())

    def pair(t):  # |x_d| + |x_e| of each rotated pair
        if f is None:
            return t.abs()
        h, a = f.numel(), t.abs()
        return torch.cat([a[..., :h] + a[..., h:2 * h], a[..., :h] + a[..., h:2 * h], a[..., 2 * h:]], -1)
    qs = pair(rotate64(x[:, :Hq], vals(qn) if norm else None, pos, None))
    ks = pair(rotate64(x[:, Hq:Hq + Hkv], vals(kn) if norm else None, pos, None))
    got = vals(q).view(T, Hq, D)
    near(got[live], qe[live], qs[live])
    assert bool((q.view(T, -1)[~live] == 77).all())
    kx, vx = k0.clone(), v0.clone()
    for i in torch.nonzero(live)[:, 0].tolist():
        s, p = seqs[i // Tq], int(pos[i])
        pid, off = int(c.tables[s, p // page]), p % page
        near(vals(c.k[1, pid, :, off]), ke[i], ks[i])
        kx[1, pid, :, off] = c.k[1, pid, :, off]
        vx[1, pid, :, off] = bits(ve[i])
    assert torch.equal(c.k, kx) and torch.equal(c.v, vx)  # nothing else is touched


def test_append_to_an_e4m3_cache_rounds_and_saturates():
    ks = torch.tensor([[0.5, 0.013]], device="cuda")
    vs = torch.tensor([[2.0, 0.0071]], device="cuda")
    c = make(layers=1, pages=8, page=16, Hkv=2, D=128, max_seqs=2, max_pages=4, kv="e4m3", Hq=2, max_new=9, k_scale=ks,
             v_scale=vs)
    c.resize(i32([0]), i32([20]))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = 3 * torch.randn(9, 6, 128, generator=g, device="cuda")
    x[2, 2, 5], x[3, 5, 7], x[4, 3, 0] = 1e4, -1e4, 3.0e38  # far beyond 448 scales
    x[5, 2] = 0
    qkv = bits(x).view(9, -1)
    q = torch.zeros(9, 256, dtype=torch.int16, device="cuda")
    c.append(0, i32([0]), qkv, q, Tq=9)
    assert c.error_word() == 0
    assert torch.equal(q.view(9, 2, 128), bits(x)[:, :2])
    xv = qkv.view(torch.bfloat16).float().view(9, 6, 128)
    want_k = (xv[:, 2:4] / ks.view(1, 2, 1)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    want_v = (xv[:, 4:6] / vs.view(1, 2, 1)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    for t in range(9):
        p = 11 + t
        pid = int(c.tables[0, p // 16])
        assert torch.equal(c.k[0, pid, :, p % 16], want_k[t]) and torch.equal(c.v[0, pid, :, p % 16], want_v[t])


@pytest.mark.parametrize("D,Hq,Hkv,rope,Tq", [(128, 6, 2, 64, 5), (128, 4, 1, 128, 700), (256, 16, 2, 64, 3), (256, 2, 2, 256, 301),
                                             (256, 3, 1, 6, 9), (128, 4, 4, 0, 2)])
def test_append_with_norm_and_rotation_to_an_e4m3_cache(D, Hq, Hkv, rope, Tq):
    """Normed and rotated keys, and values, in 64 bits against what is stored. Beside the tolerance of the bf16 cache's test:
    one more fp32 rounding (the division by the scale) and half a step of e4m3, 2^-4 of the value or 2^-10 scales, up to 448
    scales, where it saturates."""
    page, far = 32, 100_000 // 32
    g = torch.Generator(device="cuda").manual_seed(D + rope)
    ks = 0.002 + 0.01 * torch.rand(2, Hkv, generator=g, device="cuda")  # keys of up to 4.5 saturate in some heads
    vs = 0.002 + 0.01 * torch.rand(2, Hkv, generator=g, device="cuda")
    c = make(layers=2, pages=80, page=page, Hkv=Hkv, D=D, max_seqs=3, max_pages=far, kv="e4m3", Hq=Hq, max_batch=4, max_new=Tq,
             k_scale=ks, v_scale=vs)
    lens, seqs, nxt = [Tq, far * page - 5, max(0, Tq - 2)], [1, -1, 0, 2], 0
    for s, n in enumerate(lens):
        for j in range(max(0, (n - Tq) // page), -(-n // page)):
            c.tables[s, j], c.refs[nxt] = nxt, 1
            nxt += 1
    c.lens.copy_(i32(lens))
    T = len(seqs) * Tq
    qkv = bits(1.5 * torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda"))
    qn, kn = (bits(1 + 0.1 * torch.randn(D, generator=g, device="cuda")) for _ in range(2))
    f = (1e7 ** (-torch.arange(0, rope, 2, dtype=torch.float64) / rope)).cuda() if rope else None
    q = torch.full((T, Hq * D), 77, dtype=torch.int16, device="cuda")
    k0, v0 = c.k.clone(), c.v.clone()
    c.append(1, i32(seqs), qkv, q, Tq=Tq, q_norm=qn, k_norm=kn, inv_freq=f)
    assert c.error_word() == 0
    x = vals(qkv).view(T, Hq + 2 * Hkv, D)
    pos = torch.tensor([lens[s] - Tq + t if s >= 0 else -1 for s in seqs for t in range(Tq)], device="cuda")
    live = torch.nonzero(pos >= 0)[:, 0]
    sid = torch.tensor([max(s, 0) for s in seqs for t in range(Tq)], device="cuda")
    pid, off = c.tables[sid[live], pos[live] // page].long(), pos[live] % page
    qe, ke = rotate64(x[:, :Hq], vals(qn), pos, f)[live], rotate64(x[:, Hq:Hq + Hkv], vals(kn), pos, f)[live]

    def size(x, w):  # |x_d| + |x_e| of each rotated pair
        a = rotate64(x, vals(w), pos, None).abs()
        h = 0 if f is None else f.numel()
        both = a[..., :h] + a[..., h:2 * h]
        return torch.cat([both, both, a[..., 2 * h:]], -1)[live]
    assert bool(((vals(q).view(T, Hq, D)[live] - qe).abs() <= BF * qe.abs() + 24 * F32 * size(x[:, :Hq], qn) + 1e-30).all())
    for stored, want, slack, sc in ((c.k, ke, 25 * F32 * size(x[:, Hq:Hq + Hkv], kn), ks), (c.v, x[live, Hq + Hkv:], 0.0, vs)):
        sc = sc[1].double().view(1, Hkv, 1)
        got = stored[1, pid, :, off].view(torch.float8_e4m3fn).double() * sc
        want = torch.minimum(torch.maximum(want, -448 * sc), 448 * sc)
        tol = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * sc) + slack + F32 * want.abs()
        assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())
    k0[1, pid, :, off], v0[1, pid, :, off] = c.k[1, pid, :, off], c.v[1, pid, :, off]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)  # nothing else is touched


def test_append_skips_shared_and_bad_pages_and_bad_sequences():
    c = make(layers=1, pages=8, page=16, Hkv=2, D=64, max_seqs=4, max_pages=3, Hq=2)
    c.resize(i32([0, 1, 2]), i32([5, 6, 7]))
    c.fork(i32([0]), i32([3]))
    k0 = c.k.clone()
    qkv = bits(torch.ones(1, 6 * 64, device="cuda"))
    q = torch.zeros(1, 128, dtype=torch.int16, device="cuda")
    c.append(0, i32([3]), qkv, q)  # its page is sequence 0's too
    assert c.error_word() == P().ERR_SHARED and torch.equal(c.k, k0)
    for bad in (-1, 8, 2 ** 31 - 1):
        c.tables[1, 0] = bad
        c.append(0, i32([1]), qkv, q)
        assert c.error_word() == P().ERR_PAGE_ID and torch.equal(c.k, k0)
    for s in (4, -2, 2 ** 31 - 1):
        c.append(0, i32([s]), qkv, q)
        assert c.error_word() == P().ERR_SEQ_ID and torch.equal(c.k, k0)
    c.lens[2] = 49
    c.append(0, i32([2]), qkv, q)
    assert c.error_word() == P().ERR_SEQ_ID and torch.equal(c.k, k0)


# ------------------------------------------------------------------ attention

def attend64(c, layer, seqs, q, Tq, scale, kv):
    """(out, tolerance) [B Tq, Hq, D] in 64 bits. The tolerance, per value: the output's rounding (bf16); the weights'
    rounding to the products' type (bf16, or f16 over an e4m3 cache), which moves a weighted mean by at most that part of
    sum p |v| + |o|; the scores' fp32 sums ((D + 4) roundings of sum |q k| scale) and the exponential (2^-20), which move
    the weights relatively, the total likewise; fp32 sums of the products (n + 8 roundings, in 64 keys' pieces at least
    as exact as that)."""
    B, Hq, Hkv, D, page = len(seqs), c.Hq, c.Hkv, c.D, c.page
    q = vals(q).view(B, Tq, Hq, D)
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    wt = BF if kv == "bf16" else 2.0 ** -11
    for b, s in enumerate(seqs):
        n = int(c.lens[s]) if s >= 0 else 0
        for t in range(Tq):
            m = n - Tq + t + 1
            if m <= 0:
                continue
            ids = c.tables[s, :-(-m // page)].long()
            for h in range(Hkv):
                if kv == "bf16":
                    k, v = (vals(x[layer, ids, h]).reshape(-1, D)[:m] for x in (c.k, c.v))
                else:
                    k, v = (x[layer, ids, h].view(torch.float8_e4m3fn).double().reshape(-1, D)[:m] for x in (c.k, c.v))
                    if c.k_scale is not None:
                        k, v = k * c.k_scale[layer, h].double(), v * c.v_scale[layer, h].double()
                hs = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
                p = torch.softmax(q[b, t, hs] @ k.T * scale, -1)
                o = p @ v
                mag = p @ v.abs()
                ds = (D + 4) * F32 * (q[b, t, hs].abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True) + 2.0 ** -20
                out[b, t, hs] = o
                tol[b, t, hs] = BF * o.abs() + (wt + 2 * ds + 72 * F32) * (mag + o.abs()) + 1e-30
    return out.view(B * Tq, Hq * D), tol.view(B * Tq, Hq * D)


def filled(lens, Tq=1, Hq=2, seed=0, layers=1, **kw):
    """A cache whose sequences have these lengths, their pages in a scattered order."""
    page = kw.get("page", 16)
    need = sum(-(-n // page) for n in lens)
    c = make(layers=layers, pages=need + 3, max_seqs=len(lens), max_pages=max(1, max(-(-n // page) for n in lens)), Hq=Hq,
             max_new=Tq, seed=seed, **kw)
    order = torch.randperm(need + 3, generator=torch.Generator().manual_seed(seed)).int().tolist()
    for s, n in enumerate(lens):
        for j in range(-(-n // page)):
            p = order.pop()
            c.tables[s, j] = p
            c.refs[p] = 1
    c.lens.copy_(i32(lens))
    return c


def queries(c, B, Tq, seed=5, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return bits(std * torch.randn(B * Tq, c.Hq * c.D, generator=g, device="cuda"))


def check_attend(c, seqs, Tq, kv="bf16", layer=0, scale=None, q=None):
    q = queries(c, len(seqs), Tq) if q is None else q
    out = torch.full_like(q, 99)
    c.attend(layer, i32(seqs), q, out, Tq=Tq, scale=scale)
    assert c.error_word() == 0
    want, tol = attend64(c, layer, seqs, q, Tq, c.D ** -0.5 if scale is None else scale, kv)
    err = (vals(out) - want).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float((err / tol.clamp(min=1e-20)).max()))
    return out


SHAPES = [  # kv, D, page, Hq, Hkv, Tq
    ("bf16", 256, 64, 16, 2, 1), ("bf16", 256, 16, 8, 8, 1), ("bf16", 256, 48, 16, 2, 4), ("bf16", 256, 32, 16, 2, 8),
    ("bf16", 128, 64, 32, 8, 1), ("bf16", 128, 16, 5, 1, 5), ("bf16", 128, 48, 16, 1, 4), ("bf16", 64, 128, 8, 4, 1),
    ("bf16", 64, 16, 12, 1, 3), ("bf16", 64, 32, 128, 1, 2), ("e4m3", 256, 64, 16, 2, 1), ("e4m3", 256, 16, 14, 2, 7),
    ("e4m3", 128, 32, 32, 8, 4), ("e4m3", 128, 48, 3, 1, 1), ("e4m3", 128, 16, 64, 1, 2)]


@pytest.mark.parametrize("kv,D,page,Hq,Hkv,Tq", SHAPES)
def test_attention_of_a_ragged_batch_against_64_bits(kv, D, page, Hq, Hkv, Tq):
    lens = [1, 700, 0, page, page + 1, 2 * page - 1, Tq, max(0, Tq - 1), 63, 64, 65, 333]
    kw = {}
    if kv == "e4m3":
        kw = dict(k_scale=torch.linspace(0.02, 0.05, 2 * Hkv, device="cuda").view(2, Hkv),
                  v_scale=torch.linspace(0.05, 0.01, 2 * Hkv, device="cuda").view(2, Hkv))
    c = filled(lens, Tq=Tq, Hq=Hq, Hkv=Hkv, D=D, page=page, kv=kv, layers=2, max_batch=20, **kw)
    seqs = list(range(len(lens)))
    random.Random(2).shuffle(seqs)
    seqs.insert(3, -1)
    out = check_attend(c, seqs, Tq, kv, layer=1)
    rows = out.view(len(seqs), Tq, -1)
    for b, s in enumerate(seqs):
        n = lens[s] if s >= 0 else 0
        assert not bool(rows[b, :max(0, min(Tq, Tq - n))].any())


@pytest.mark.parametrize("kv,D,page,Hq,Hkv,Tq,n", [
    ("bf16", 256, 64, 16, 2, 1, 40001), ("bf16", 256, 64, 16, 2, 1, 1), ("bf16", 256, 64, 2, 2, 1, 17),
    ("bf16", 128, 32, 8, 1, 2, 9999), ("e4m3", 256, 128, 8, 1, 4, 20011), ("bf16", 64, 16, 4, 2, 1, 5000),
    ("e4m3", 128, 16, 8, 2, 1, 7777)])
def test_attention_of_one_sequence_split_over_its_length(kv, D, page, Hq, Hkv, Tq, n):
    c = filled([n], Tq=Tq, Hq=Hq, Hkv=Hkv, D=D, page=page, kv=kv,
               **({} if kv == "bf16" else {"k_scale": torch.full((1, Hkv), 0.025, device="cuda"),
                                           "v_scale": torch.full((1, Hkv), 0.025, device="cuda")}))
    a = check_attend(c, [0], Tq, kv)
    assert torch.equal(a, check_attend(c, [0], Tq, kv))  # the same bits again


@pytest.mark.parametrize("kv,D", [("bf16", 256), ("bf16", 64), ("e4m3", 128)])
def test_attention_ignores_what_lies_behind_a_sequence_and_ahead_of_a_token(kv, D):
    Tq, page, lens = 3, 32, [70, 3, 33, 2]
    c = filled(lens, Tq=Tq, Hq=4, Hkv=2, D=D, page=page, kv=kv)
    q = queries(c, len(lens), Tq)
    seqs = list(range(len(lens)))
    base = check_attend(c, seqs, Tq, kv, q=q)
    junk = [0x7FC0, 0x7F80, -0x80, 0x7F7F, -0x81] if kv == "bf16" else [0x7F, 0xFF, 0x7E, 0xFE]
    for s, n in enumerate(lens):  # NaN, infinities and the largest values behind the end, and in pages of no sequence
        for j, pid in enumerate(c.tables[s].tolist()):
            for r in range(page):
                if pid >= 0 and j * page + r >= n:
                    c.k[0, pid, :, r] = junk[r % len(junk)]
                    c.v[0, pid, :, r] = junk[(r + 1) % len(junk)]
    free = torch.nonzero(c.refs == 0)[:, 0]
    c.k[0, free], c.v[0, free] = junk[0], junk[0]
    out = torch.full_like(q, 99)
    c.attend(0, i32(seqs), q, out, Tq=Tq)
    assert torch.equal(out, base)
    # the last token's own key and value: its rows alone may see them
    for s, n in enumerate(lens):
        pid = int(c.tables[s, (n - 1) // page])
        c.k[0, pid, :, (n - 1) % page] = junk[0]
        c.v[0, pid, :, (n - 1) % page] = junk[0]
    c.attend(0, i32(seqs), q, out, Tq=Tq)
    o, w = out.view(len(lens), Tq, -1), base.view(len(lens), Tq, -1)
    assert torch.equal(o[:, :-1], w[:, :-1])
    assert bool(torch.isnan(vals(o[:, -1].contiguous())).all())


def test_attention_scores_of_any_size():
    """Scores of +-1e4 (one key takes all), equal scores, a scale of zero and a negative one."""
    c = filled([200, 57], Hq=4, Hkv=2, D=128, page=16)
    check_attend(c, [0, 1], 1, scale=0.0)
    check_attend(c, [1, 0], 1, scale=-0.05)
    check_attend(c, [0, 1], 1, q=queries(c, 2, 1, std=0.0))
    out = torch.zeros(2, 512, dtype=torch.int16, device="cuda")
    q = queries(c, 2, 1, std=3000.0)
    c.attend(0, i32([0, 1]), q, out)
    want, tol = attend64(c, 0, [0, 1], q, 1, 128 ** -0.5, "bf16")
    assert bool(((vals(out) - want).abs() <= tol).all()) and bool(torch.isfinite(vals(out)).all())
    f = filled([130], Hq=2, Hkv=1, D=256, page=64, kv="e4m3")
    for std in (1e-20, 1e-3, 1e20):  # queries far outside f16's range (unscaled e4m3 keys of about 40)
        q = queries(f, 1, 1, std=std)
        out = torch.zeros_like(q)
        f.attend(0, i32([0]), q, out, scale=1e-3 / std)
        want, tol = attend64(f, 0, [0], q, 1, 1e-3 / std, "e4m3")
        assert bool(((vals(out) - want).abs() <= tol).all())


@pytest.mark.parametrize("kv,D,Hq,Tq", [("bf16", 64, 4, 1), ("bf16", 256, 16, 1), ("bf16", 256, 16, 4), ("e4m3", 128, 8, 2)])
def test_attention_with_a_scale_that_is_no_number_is_no_number(kv, D, Hq, Tq):
    c = filled([130, 9, 0], Hq=Hq, Hkv=2, D=D, page=16, kv=kv, Tq=Tq)
    q = queries(c, 3, Tq)
    out = torch.zeros_like(q)
    c.attend(0, i32([0, 1, 2]), q, out, Tq=Tq, scale=math.nan)
    got = vals(out).view(3, Tq, -1)
    assert bool(torch.isnan(got[:2]).all()) and not bool(got[2].any())


@pytest.mark.parametrize("D,Hq,Tq", [(64, 4, 1), (128, 8, 2), (256, 4, 1), (256, 16, 4)])
def test_attention_of_values_near_the_largest_of_their_type(D, Hq, Tq):
    """Even scores, and one key late in the sequence a few powers of two above them whose value is 3e38: the mean is finite,
    and so is every sum of p v with p relative to the row's largest weight."""
    n, at, B = 600, 400, 400  # enough sequences that one warp meets a sequence's even keys before the high one
    for up in (1.0, 2.5, 3.5, 3.9, 4.5):
        c = filled([n] + [0] * (B - 1), Hq=Hq, Hkv=2, D=D, page=16, Tq=Tq)
        c.tables[1:] = c.tables[0]
        c.lens[:] = n
        pid = int(c.tables[0, at // 16])
        c.k.zero_()
        c.k.view(torch.bfloat16)[0, pid, :, at % 16, 0] = up / math.log2(math.e)
        c.v.view(torch.bfloat16)[0, pid, :, at % 16] = 3e38
        q = torch.zeros(B * Tq * Hq, D, device="cuda")
        q[:, 0] = 1.0
        q = bits(q).view(B * Tq, -1)
        out = torch.zeros_like(q)
        c.attend(0, i32(list(range(B))), q, out, Tq=Tq, scale=1.0)
        want, tol = attend64(c, 0, [0], q[:Tq], Tq, 1.0, "bf16")
        assert bool(((vals(out).view(B, Tq, -1) - want).abs() <= tol).all())


@pytest.mark.parametrize("D,Hq,Tq,n", [(64, 4, 1, 900), (128, 8, 2, 900), (256, 16, 1, 70_000), (256, 16, 4, 900)])
def test_attention_of_many_values_near_the_largest_of_their_type(D, Hq, Tq, n):
    """Rows whose keys all have values of 3e38: their sum is far beyond fp32, their mean is not. And values near the smallest,
    whose mean is off by no more than attend64 allows for any."""
    c = filled([n, 33], Hq=Hq, Hkv=2, D=D, page=16, Tq=Tq)
    q = queries(c, 2, Tq, std=0.5)
    for size in (3e38, -3e38, 1e-37):
        c.v.view(torch.bfloat16).fill_(size)
        out = check_attend(c, [0, 1], Tq, q=q)
        assert bool(torch.isfinite(vals(out)).all())


@pytest.mark.parametrize("D,Hq,Tq", [(64, 4, 1), (64, 16, 3), (128, 8, 1), (128, 32, 4), (256, 16, 1), (256, 16, 4), (256, 16, 8)])
def test_attention_keeps_more_of_a_weight_than_its_output_shows(D, Hq, Tq):
    """Rows of values that nearly cancel, where a weight of 8 bits would show: within the output's rounding (2^-8 of it) and
    2^-16 of sum p |v| for the weights' two bf16 parts, beside what attend64 allows for the scores and the sums in fp32."""
    lens = [9, 17, 24, 40, 57]
    c = filled(lens, Hq=Hq, Hkv=2, D=D, page=16, Tq=Tq)
    B, G = len(lens), Hq // 2
    q = queries(c, B, Tq, std=0.25)
    out = torch.zeros_like(q)
    c.attend(0, i32(list(range(B))), q, out, Tq=Tq)
    got, qq = vals(out).view(B, Tq, Hq, D), vals(q).view(B, Tq, Hq, D)
    for b, n in enumerate(lens):
        ids = c.tables[b, :-(-n // 16)].long()
        for t in range(Tq):
            m = n - Tq + t + 1
            for h in range(Hq):
                k, v = (vals(x[0, ids, h // G]).reshape(-1, D)[:m] for x in (c.k, c.v))
                p = torch.softmax(k @ qq[b, t, h] * D ** -0.5, 0)
                o, mag = p @ v, p @ v.abs()
                ds = (D + 4) * F32 * float((k.abs() @ qq[b, t, h].abs()).max()) * D ** -0.5 + 2.0 ** -20
                tol = BF * o.abs() + (2.0 ** -16 + 2 * ds + 72 * F32) * (mag + o.abs())
                assert bool(((got[b, t, h] - o).abs() <= tol).all()), (b, t, h)


@pytest.mark.parametrize("D,Hq,Tq", [(64, 4, 1), (64, 16, 3), (128, 8, 2), (256, 16, 1), (256, 16, 4), (256, 16, 8)])
def test_attention_of_infinite_values_that_a_row_sees(D, Hq, Tq):
    """A weight above zero times an infinity is that infinity, whatever the weight's bits (one key alone has a weight of a
    power of two); the columns beside it and the tokens that do not see it keep theirs."""
    lens = [1, 8, 40, 300]
    c = filled(lens, Hq=Hq, Hkv=2, D=D, page=16, Tq=Tq)
    v = c.v.view(torch.bfloat16)
    for b, n in enumerate(lens):
        first, last = int(c.tables[b, 0]), int(c.tables[b, (n - 1) // 16])
        v[0, first, :, 0, 2] = v[0, first, :, 0, 3] = -math.inf
        v[0, last, :, (n - 1) % 16, 1] = v[0, last, :, (n - 1) % 16, 3] = math.inf
    for std in (0.25, 0.0):
        q = queries(c, len(lens), Tq, std=std)
        out = torch.zeros_like(q)
        c.attend(0, i32(list(range(len(lens)))), q, out, Tq=Tq)
        want, tol = attend64(c, 0, list(range(len(lens))), q, Tq, D ** -0.5, "bf16")
        got, finite = vals(out), torch.isfinite(want)
        assert bool(((got - want).abs() <= tol)[finite].all())
        assert torch.equal(torch.nan_to_num(got[~finite], nan=5.0), torch.nan_to_num(want[~finite], nan=5.0))


@pytest.mark.parametrize("D,Hq,Tq", [(128, 4, 1), (128, 8, 3), (256, 4, 3), (256, 16, 8)])
def test_attention_over_8_bits_with_scores_too_small_to_tell(D, Hq, Tq):
    """A scale of zero with tiny queries, and queries of zero with tiny key scales: equal scores, so a row is the mean of
    the values that it sees, whatever the factors' product comes to in fp32."""
    c = filled([130, 9, 2, 33], Hq=Hq, Hkv=2, D=D, page=16, kv="e4m3", Tq=Tq,
               k_scale=torch.full((1, 2), 1e-9, device="cuda"), v_scale=torch.full((1, 2), 0.03, device="cuda"))
    for std, scale in ((0.0, None), (2.0 ** -30, 0.0), (2.0, 0.0), (2.0 ** -126, 1e-3)):
        check_attend(c, [2, 0, 3, 1], Tq, "e4m3", scale=scale, q=queries(c, 4, Tq, std=std))


@pytest.mark.parametrize("kv,D,Tq", [("bf16", 64, 1), ("bf16", 128, 4), ("bf16", 256, 1), ("e4m3", 128, 2), ("e4m3", 256, 3)])
def test_attention_of_scores_that_climb_and_fall(kv, D, Tq):
    """Scores that rise over 2000 keys by 50 powers of two, evenly, in steps, or falling: the running maximum moves in
    every tile, in a few, or never."""
    n, page = 2000, 16
    c = filled([n] * 3, Hq=4, Hkv=2, D=D, page=page, kv=kv, Tq=Tq)
    j = torch.arange(n, device="cuda")
    for s, ramp in enumerate((8.0 * j / n, 0.8 * (j // 200), 8.0 - 8.0 * j / n)):
        ids = c.tables[s, :n // page].long()
        at = ramp.view(-1, 1, page).expand(-1, 2, -1)
        k = c.k.view(torch.bfloat16 if kv == "bf16" else torch.float8_e4m3fn)
        k[0, ids, :, :, 0] = at.to(k.dtype)
    q = vals(queries(c, 3, Tq, std=0.5)).view(-1, D).float()
    q[:, 0] = 4.4 * D ** 0.5
    check_attend(c, [0, 1, 2], Tq, kv, q=bits(q.view(3 * Tq, -1)))


def test_attention_with_bad_pages_and_sequences_is_recorded_and_bounded():
    c = filled([100, 40], Hq=2, Hkv=2, D=64, page=16, max_batch=8)
    q = queries(c, 2, 1)
    out = torch.zeros_like(q)
    c.attend(0, i32([0, 1]), q, out)
    good = out.clone()
    keep = int(c.tables[0, 3])
    for bad in (-1, c.num_pages, 2 ** 31 - 1, -2 ** 31):
        c.tables[0, 3] = bad
        c.attend(0, i32([0, 1]), q, out)
        assert c.error_word() == P().ERR_PAGE_ID
        assert torch.equal(out[1], good[1]) and bool(torch.isfinite(vals(out)).all())
    c.tables[0, 3] = keep
    for bad in (2, -2, 2 ** 31 - 1):
        c.attend(0, i32([bad, 1]), q, out)
        assert c.error_word() == P().ERR_SEQ_ID
        assert torch.equal(out[1], good[1]) and not bool(out[0].any())
    c.lens[0] = 10 ** 9
    c.attend(0, i32([0, 1]), q, out)
    assert c.error_word() == P().ERR_SEQ_ID and torch.equal(out[1], good[1])
    c.lens[0] = 100
    c.attend(0, i32([0, 1]), q, out)
    assert c.error_word() == 0 and torch.equal(out, good)


def test_attention_of_shared_pages_and_a_large_batch():
    """Forked sequences read the same pages; a batch of 300 sequences of a few keys."""
    c = make(pages=400, page=16, Hkv=1, D=64, max_seqs=300, max_pages=4, Hq=4)
    c.resize(i32([0]), i32([45]))
    c.fork(i32([0] * 10), i32(list(range(1, 11))))
    out = check_attend(c, list(range(11)), 1, q=queries(c, 1, 1).repeat(11, 1))
    assert all(torch.equal(out[0], out[i]) for i in range(11))
    c.resize(i32(list(range(11, 300))), i32([1 + s % 17 for s in range(11, 300)]))
    assert c.error_word() == 0
    check_attend(c, list(range(300)), 1)


def test_attention_refuses_what_it_cannot_take():
    import mvcc_b200 as m
    c = filled([20], Tq=2, Hq=2, Hkv=2, D=64)
    q, out = queries(c, 1, 1), queries(c, 1, 1)
    for bad in (lambda: c.attend(0, i32([0]), q, out, Tq=3), lambda: c.attend(0, i32([0]), q[:, 1:], out),
                lambda: c.attend(0, i32([0]), q.float(), out), lambda: c.attend(0, i32([0, 0]), q, out),
                lambda: c.attend(0, i32([0]), q.cpu(), out)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(m.MoeError):
        c.attend(1, i32([0]), q, out)  # one layer
    with pytest.raises(m.MoeError):
        c.append(0, i32([0]), torch.cat([q, q, q], 1), q, inv_freq=torch.ones(33, dtype=torch.float64, device="cuda"))


# ------------------------------------------------------------------ together

def test_a_captured_step_follows_the_cache_as_it_grows():
    """append + attend captured once and replayed on another stream while sequences grow, fork and are compacted."""
    c = make(layers=1, pages=64, page=16, Hkv=2, D=128, max_seqs=4, max_pages=16, Hq=8, seed=4)
    seqs = i32([0, 1, -1, 3])
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = bits(torch.randn(4, 12 * 128, generator=g, device="cuda"))
    q = torch.zeros(4, 8 * 128, dtype=torch.int16, device="cuda")
    out = torch.zeros_like(q)
    f = (1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).cuda()
    lens = torch.tensor([15, 100, 3], dtype=torch.int32, device="cuda")
    who = i32([0, 1, 3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        c.resize(who, lens)
        c.append(0, seqs, qkv, q, inv_freq=f)
        c.attend(0, seqs, q, out)

    with torch.cuda.stream(s):
        step()
        lens += 1
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        for i in range(6):
            graph.replay()
            s.synchronize()
            assert c.error_word(s) == 0
            want, tol = attend64(c, 0, [0, 1, -1, 3], q, 1, 128 ** -0.5, "bf16")
            assert bool(((vals(out) - want).abs() <= tol).all())
            if i == 2:
                c.resize(i32([2]), i32([5]), stream=s)
                c.compact(stream=s)
            lens += 1
        s.synchronize()
    assert c.lens.tolist() == [21, 106, 5, 9]


def test_paged_layer_matches_the_contiguous_layer():
    """moe_attn_paged_forward_rms for one sequence against moe_attn_forward_rms on the same cache contents; both round
    the same values at the same places but for the angle (fp32 fast intrinsics there), so bf16 outputs agree within the
    bar of the contiguous layer's own tests."""
    from mvcc_b200 import stack as st
    from oracle import oracle as O
    for gate, T in ((False, 1), (True, 3)):
        a = st.AttnShape(gate=gate)
        layer = st.synth_attn_layer(a, seed=21)
        ctx, n = 512, 300
        g = torch.Generator(device="cuda").manual_seed(9)
        kc, vc = (bits(torch.randn(a.Hkv, ctx, a.D, generator=g, device="cuda")) for _ in range(2))
        c = make(layers=2, pages=24, page=64, Hkv=a.Hkv, D=a.D, max_seqs=3, max_pages=8, Hq=a.Hq, max_new=4)
        c.resize(i32([0, 1]), i32([70, n + T]))
        for p in range(n):
            pid = int(c.tables[1, p // 64])
            c.k[1, pid, :, p % 64] = kc[:, p]
            c.v[1, pid, :, p % 64] = vc[:, p]
        hidden = torch.randn(T, a.H, generator=g, device="cuda")
        rms = bits(1 + 0.1 * torch.randn(a.H, generator=g, device="cuda"))
        b0 = st.AttnBlock(layer, ctx, max_T=T, caches=(kc, vc))
        o0 = torch.zeros(T, a.H, dtype=torch.int16, device="cuda")
        b0.forward_rms(hidden, rms, o0, n)
        b1 = P().PagedAttnBlock(layer, c, 1)
        o1 = torch.zeros(T, a.H, dtype=torch.int16, device="cuda")
        b1.forward_rms(hidden, rms, o1, i32([1]), Tq=T)
        torch.cuda.synchronize()
        assert b1.error_word() == 0 and b0.error_word() == 0
        x, y = (vals(t).cpu().numpy() for t in (o1, o0))
        assert O.max_rel_err(x, y) < 1e-2
        for t in range(T):
            pid, off = int(c.tables[1, (n + t) // 64]), (n + t) % 64
            assert torch.equal(c.v[1, pid, :, off], vc[:, n + t])
            assert O.max_rel_err(vals(c.k[1, pid, :, off]).cpu().numpy(), vals(kc[:, n + t]).cpu().numpy()) < 1e-2


def small_stack(L=2, vocab=1000, seed=3):
    import mvcc_b200 as m
    from mvcc_b200 import stack as st
    return st.DecodeStack(L=L, ctx=64, vocab=vocab, attn=st.AttnShape(H=1024, Hq=8, Hkv=2),
                          moe=m.MoeShape(H=1024, E=32, TOPK=4, I=256, Is=256, G=64), seed=seed)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,Tq", [(5, 1), (3, 3), (16, 4), (64, 1)])
def test_paged_layer_of_more_rows_than_a_projection_takes_at_once(B, Tq, kv):
    """The layer for 5, 9 and 64 rows against its formula in 64 bits, rounded to bf16 where the layer stores bf16 (the first
    projection, the rotated queries, the attention's and the gate's output); its keys and values are those that it left in the
    cache. The bar is the contiguous layer's."""
    from mvcc_b200 import stack as st
    from oracle import oracle as O
    a = st.AttnShape(gate=True)
    layer = st.synth_attn_layer(a, seed=23)
    g = torch.Generator(device="cuda").manual_seed(B)
    kw = {} if kv == "bf16" else {n: 0.02 + 0.01 * torch.rand(2, a.Hkv, generator=g, device="cuda") for n in ("k_scale", "v_scale")}
    c = make(layers=2, pages=8 * B, page=32, Hkv=a.Hkv, D=a.D, max_seqs=B, max_pages=8, Hq=a.Hq, max_new=Tq, kv=kv, **kw)
    lens = [1 + (37 * b + 11) % 250 for b in range(B)]
    seqs = [(b + 1) % B for b in range(B)]
    c.resize(i32(list(range(B))), i32(lens))
    seqs[1] = -1
    hidden = torch.randn(B * Tq, a.H, generator=g, device="cuda")
    rms = bits(1 + 0.1 * torch.randn(a.H, generator=g, device="cuda"))
    blk = P().PagedAttnBlock(layer, c, 1)
    out = torch.full((B * Tq, a.H), 77, dtype=torch.int16, device="cuda")
    blk.forward_rms(hidden, rms, out, i32(seqs), Tq=Tq)
    torch.cuda.synchronize()
    assert blk.error_word() == 0
    h, w = hidden.double(), {n: vals(t) for n, t in layer.t.items()}
    x = h / torch.sqrt((h * h).mean(-1, keepdim=True) + a.eps) * vals(rms)
    qkv, z = vals(bits(x @ w["qkv"].T)), vals(bits(x @ w["gate"].T))
    pos = torch.tensor([(lens[s] if s >= 0 else 0) - Tq + t for s in seqs for t in range(Tq)], device="cuda")
    f = P().inv_frequencies(a)
    q = bits(rotate64(qkv[:, :a.Hq * a.D].view(-1, a.Hq, a.D), w["q_norm"], pos, f)).view(B * Tq, -1)
    o = vals(bits(attend64(c, 1, seqs, q, Tq, a.D ** -0.5, kv)[0]))
    want = vals(bits(o * torch.sigmoid(z))) @ w["o"].T
    assert O.max_rel_err(vals(out).cpu().numpy(), want.cpu().numpy()) < 1e-2
    for i in range(B * Tq):  # row by row, so that no row hides behind a larger one
        if pos[i] >= 0:
            assert O.max_rel_err(vals(out[i]).cpu().numpy(), want[i].cpu().numpy()) < 2e-2, i
    if kv == "bf16":
        for b, s in enumerate(seqs):
            for t in range(Tq):
                p = int(pos[b * Tq + t])
                if s >= 0 and p >= 0:
                    new = vals(c.v[1, int(c.tables[s, p // 32]), :, p % 32])
                    assert O.max_rel_err(new.cpu().numpy(), qkv[b * Tq + t].view(-1, a.D)[-a.Hkv:].cpu().numpy()) < 1e-2


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,Tq", [(3, 1), (3, 2), (6, 3)])
def test_a_captured_step_of_the_stack_is_replayed_as_the_sequences_grow(B, Tq, kv):
    """Growth and step captured once and replayed, against the same steps called one by one on a second cache."""
    st = small_stack()
    ones = {} if kv == "bf16" else {n: torch.full((st.L, 2), 0.03, device="cuda") for n in ("k_scale", "v_scale")}
    make_one = lambda: P().PagedDecodeStack(st, num_pages=40, page=16, max_seqs=B, max_pages=6, max_batch=B, max_new=Tq, kv=kv,
                                            **ones)
    one, two = make_one(), make_one()
    seqs, start = i32([-1 if b == 1 else b for b in range(B)]), i32([5 + 13 * b % 40 for b in range(B)])
    who = i32(list(range(B)))
    for ps in (one, two):
        ps.cache.resize(who, start)
    for n in ("k", "v"):
        t = getattr(one.cache, n)
        g = torch.Generator(device="cuda").manual_seed(ord(n))
        r = torch.randn(t.shape, generator=g, device="cuda")
        t.copy_(bits(r) if kv == "bf16" else (r * 30).to(torch.float8_e4m3fn).view(torch.uint8))
        getattr(two.cache, n).copy_(t)
    g = torch.Generator(device="cuda").manual_seed(B)
    inputs = [torch.randn(B * Tq, 1024, generator=g, device="cuda") for _ in range(4)]
    hidden, logits, lens = inputs[0].clone(), torch.zeros(B * Tq, st.V, device="cuda"), start + Tq
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one.step(hidden.clone(), seqs, Tq=Tq, logits=logits.clone())  # the first use of each kernel, at the old lengths
        one.cache.k.copy_(two.cache.k)
        one.cache.v.copy_(two.cache.v)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            one.cache.resize(who, lens)
            one.step(hidden, seqs, Tq=Tq, logits=logits)
        for i, x in enumerate(inputs):
            hidden.copy_(x)
            graph.replay()
            h2, l2 = x.clone(), torch.zeros_like(logits)
            two.cache.resize(who, lens)
            two.step(h2, seqs, Tq=Tq, logits=l2)
            lens += Tq
            s.synchronize()
            assert one.error_words(s) == 0 and two.error_words(s) == 0
            assert torch.equal(hidden, h2) and torch.equal(logits, l2) and bool(torch.isfinite(l2).all())
            for n in ("k", "v", "tables", "refs", "lens"):
                assert torch.equal(getattr(one.cache, n), getattr(two.cache, n)), n


def test_paged_stack_step_follows_the_single_sequence_stack():
    """Three decode steps of two sequences of a paged stack, one slot unused, against the contiguous stack's steps of
    each sequence alone: the same greedy tokens, or logits that agree where two tokens are near."""
    st = small_stack()
    ps = P().PagedDecodeStack(st, num_pages=12, page=16, max_seqs=4, max_pages=4, max_batch=3, max_new=2)
    V = st.V
    g = torch.Generator(device="cuda").manual_seed(8)
    start = [5, 17]
    ps.cache.resize(i32([2, 1]), i32(start))
    refs = []
    for who, n in zip((2, 1), start):
        caches = []
        for i in range(st.L):
            kc, vc = (bits(torch.randn(2, 64, 256, generator=g, device="cuda")) for _ in range(2))
            for p in range(n):
                pid = int(ps.cache.tables[who, p // 16])
                ps.cache.k[i, pid, :, p % 16], ps.cache.v[i, pid, :, p % 16] = kc[:, p], vc[:, p]
            caches.append((kc, vc))
        refs.append(caches)
    for step in range(3):
        h = torch.randn(3, 1024, generator=g, device="cuda")
        n = [s + step + 1 for s in start]
        ps.cache.resize(i32([2, 1]), i32(n))
        hp, logits = h.clone(), torch.zeros(3, V, device="cuda")
        ps.step(hp, i32([2, -1, 1]), logits=logits)
        torch.cuda.synchronize()
        assert ps.error_words() == 0
        for j, slot in ((0, 0), (1, 2)):
            for i in range(st.L):
                st.attn[i].kc.copy_(refs[j][i][0])
                st.attn[i].vc.copy_(refs[j][i][1])
            h1, l1 = h[slot:slot + 1].clone(), torch.zeros(V, device="cuda")
            st.step(h1, n[j] - 1, logits=l1)
            torch.cuda.synchronize()
            for i in range(st.L):
                refs[j][i][0].copy_(st.attn[i].kc)
                refs[j][i][1].copy_(st.attn[i].vc)
            err = float((logits[slot] - l1).abs().max() / l1.abs().max())
            assert err < 2e-2, err  # the bar of the contiguous stack's own test
            top = torch.topk(l1, 2).values
            if float(top[0] - top[1]) > 2 * float((logits[slot] - l1).abs().max()):
                assert int(logits[slot].argmax()) == int(st.next)


def test_the_layers_of_a_paged_stack_share_a_workspace_and_its_error_word():
    st = small_stack(L=3)
    ps = P().PagedDecodeStack(st, num_pages=12, page=16, max_seqs=4, max_pages=4, max_batch=3, max_new=2)
    assert len({b.ws.data_ptr() for b in ps.attn}) == 1
    seqs = i32([0, 1])
    ps.cache.resize(seqs, i32([20, 3]))
    ps.step(torch.randn(2, 1024, device="cuda"), seqs)
    assert ps.error_words() == 0
    keep = int(ps.cache.tables[0, 0])
    ps.cache.tables[0, 0] = -7
    ps.step(torch.randn(2, 1024, device="cuda"), seqs)
    assert ps.error_words() == P().ERR_PAGE_ID and ps.error_words() == 0
    ps.cache.tables[0, 0] = keep
    with pytest.raises(ValueError):
        P().PagedAttnBlock(st.attn[0].layer, ps.cache, 0, ws=ps.attn[0].ws[:256])
    with pytest.raises(ValueError):
        P().PagedAttnBlock(st.attn[0].layer, ps.cache, 0, ws=ps.attn[0].ws.view(torch.int32))


def test_a_paged_step_with_logits_that_do_not_fit_changes_nothing():
    st = small_stack()
    ps = P().PagedDecodeStack(st, num_pages=12, page=16, max_seqs=4, max_pages=4, max_batch=3, max_new=2)
    seqs = i32([0, 1])
    ps.cache.resize(seqs, i32([20, 3]))
    h = torch.randn(2, 1024, device="cuda")
    before, k = h.clone(), ps.cache.k.clone()
    for bad in (torch.zeros(3, st.V, device="cuda"), torch.zeros(2, st.V, device="cuda", dtype=torch.bfloat16),
                torch.zeros(2, st.V), torch.zeros(st.V, 2, device="cuda").T):
        with pytest.raises(ValueError):
            ps.step(h, seqs, logits=bad)
    assert torch.equal(h, before) and torch.equal(ps.cache.k, k)


def test_a_paged_stack_may_step_on_another_stream_at_once(monkeypatch):
    """Nothing that its making has launched is still on its way, slow as its zeroing may be."""
    st = small_stack()
    zeros = torch.zeros

    def slow_zeros(*a, **kw):
        torch.cuda._sleep(5000000)  # clocks
        return zeros(*a, **kw)
    monkeypatch.setattr(torch, "zeros", slow_zeros)
    ps = P().PagedDecodeStack(st, num_pages=64, page=16, max_seqs=64, max_pages=4, max_batch=64, max_new=8)
    assert torch.cuda.current_stream().query()
    monkeypatch.undo()
    seqs = i32(list(range(64)))
    ps.cache.resize(seqs, i32([16] * 64))
    h, torch_stream = torch.randn(64 * 8, 1024, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    want, got = h.clone(), h.clone()
    ps.step(want, seqs, Tq=8)
    first = ps.normed.clone()
    torch.cuda.synchronize()
    again = P().PagedDecodeStack(st, num_pages=64, page=16, max_seqs=64, max_pages=4, max_batch=64, max_new=8)
    for n in ("k", "v", "tables", "refs", "lens"):
        getattr(again.cache, n).copy_(getattr(ps.cache, n))
    torch.cuda.synchronize()
    again.step(got, seqs, Tq=8, stream=torch_stream)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(again.normed, first)


def test_drafts_are_verified_and_rolled_back():
    """A speculative step as it is used: grow by the drafts, step, logits, probabilities, verification, shrink to what
    was accepted; the cache then equals one that never saw the rejected tokens."""
    from mvcc_b200 import spec
    st = small_stack(L=1, vocab=500)
    K = 2
    ps = P().PagedDecodeStack(st, num_pages=20, page=16, max_seqs=2, max_pages=8, max_batch=2, max_new=K + 1)
    V, seqs = st.V, i32([0, 1])
    emb = torch.randn(V, 1024, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    lens = i32([14, 31])
    ps.cache.resize(seqs, lens)
    g = torch.Generator(device="cuda").manual_seed(4)
    ver = spec.SpecVerifier(2, K, V)
    probs = torch.zeros(2, K + 1, V, device="cuda")
    tokens, acc = torch.zeros(2, K + 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    seen = set()
    for step in range(8):
        last = torch.randint(V, (2, 1), generator=g, device="cuda")
        drafted = torch.randint(V, (2, K), generator=g, device="cuda").int()
        hidden = emb[torch.cat([last, drafted.long()], 1)].view(2 * (K + 1), -1).contiguous()
        grown = lens + K + 1
        ps.cache.resize(seqs, grown)
        logits = torch.zeros(2 * (K + 1), V, device="cuda")
        ps.step(hidden, seqs, Tq=K + 1, logits=logits)
        spec.softmax_rows(logits, probs.view(-1, V), temperature=torch.full((2 * (K + 1),), 0.7, device="cuda"))
        if step % 2:  # drafts that the target likes
            drafted = probs[:, :K].argmax(-1).int()
        ver.verify(probs, None, drafted, torch.rand(2, K + 1, generator=g, device="cuda") * (0.001 if step % 2 else 1),
                   tokens, acc)
        kept = lens + 1 + acc
        ps.cache.resize(seqs, kept)
        torch.cuda.synchronize()
        assert ps.error_words() == 0
        for b in range(2):
            a = int(acc[b])
            seen.add(a)
            assert tokens[b, :a].tolist() == drafted[b, :a].tolist() and 0 <= int(tokens[b, a]) < V
            assert tokens[b, a + 1:].tolist() == [-1] * (K - a)
            n = int(ps.cache.lens[b])
            row = ps.cache.tables[b].tolist()
            assert n == int(lens[b]) + 1 + a and all((p >= 0) == (j * 16 < n) for j, p in enumerate(row))
        lens = kept
    assert K in seen and 0 in seen
    assert int(ps.cache.refs.sum()) == sum(-(-int(n) // 16) for n in lens)


def test_the_stack_command_decodes_a_batch_with_and_without_drafts():
    from mvcc_b200 import stack
    st = small_stack(L=2, vocab=700)
    for new in (1, 3):
        got = list(stack.paged_steps(st, batch=3, length=130, new=new, steps=3))
        again = list(stack.paged_steps(st, batch=3, length=130, new=new, steps=3))
        assert len(got) == 3
        for (tok, acc), (tok2, acc2) in zip(got, again):
            assert torch.equal(tok, tok2) and torch.equal(acc, acc2)  # the same inputs give the same tokens
            for b in range(3):
                a = int(acc[b])
                assert 0 <= a < new and bool((tok[b, :a + 1] >= 0).all()) and bool((tok[b, a + 1:] == -1).all())
                assert int(tok[b].max()) < 700


# ------------------------------------------------------------------ several at once, far offsets, the largest lists

def test_two_caches_on_two_streams_at_once():
    """Calls of two caches (different heads, so different grids) overlap on two streams; each gives what it gives alone."""
    a = filled([3000, 17, 900], Tq=2, Hq=8, Hkv=2, D=256, page=32, seed=1)
    b = filled([5000, 1200, 64, 1], Hq=8, Hkv=4, D=128, page=16, seed=2)
    qa, qb = queries(a, 3, 2), queries(b, 4, 1)
    sa, sb = i32([0, 1, 2]), i32([3, 0, 2, 1])
    wa, wb = torch.zeros_like(qa), torch.zeros_like(qb)
    a.attend(0, sa, qa, wa, Tq=2)
    b.attend(0, sb, qb, wb)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs_a, outs_b = [torch.zeros_like(qa) for _ in range(30)], [torch.zeros_like(qb) for _ in range(30)]
    torch.cuda.synchronize()
    for x, y in zip(outs_a, outs_b):
        a.attend(0, sa, qa, x, Tq=2, stream=s1)
        b.attend(0, sb, qb, y, stream=s2)
    torch.cuda.synchronize()
    assert a.error_word() == 0 and b.error_word() == 0
    assert all(torch.equal(x, wa) for x in outs_a) and all(torch.equal(y, wb) for y in outs_b)


def test_two_graphs_of_one_stream_share_a_workspace():
    c = filled([700, 90, 33], Tq=4, Hq=16, Hkv=2, D=256, page=64)
    q1, q4 = queries(c, 3, 1), queries(c, 3, 4, seed=6)
    o1, o4 = torch.zeros_like(q1), torch.zeros_like(q4)
    seqs = i32([2, 0, 1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.attend(0, seqs, q1, o1)
        c.attend(0, seqs, q4, o4, Tq=4)
        s.synchronize()
        w1, w4 = o1.clone(), o4.clone()
        g1, g4 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1, stream=s):
            c.attend(0, seqs, q1, o1)
        with torch.cuda.graph(g4, stream=s):
            c.attend(0, seqs, q4, o4, Tq=4)
        for _ in range(5):
            o1.zero_()
            o4.zero_()
            g1.replay()
            g4.replay()
            g4.replay()
            g1.replay()
            s.synchronize()
            assert torch.equal(o1, w1) and torch.equal(o4, w4)
        assert c.error_word(s) == 0


def test_offsets_past_32_bits():
    """A layer of 2.6 GB pools: pages whose byte offsets pass 2^31 and, in the second layer, 2^32."""
    Hkv, D, page, pages = 2, 256, 64, 40000
    c = P().PagedCache.empty(2, pages, page, Hkv, D, 8, 3, 3, 4, 2)
    free = list(range(pages - 1, pages - 4, -1)) + [pages // 2, pages - 7]
    lens = [130, 65]
    for s, n in enumerate(lens):
        for j in range(-(-n // page)):
            p = free.pop(0)
            c.tables[s, j], c.refs[p] = p, 1
    c.lens[:2] = i32(lens)
    g = torch.Generator(device="cuda").manual_seed(0)
    for s, n in enumerate(lens):
        for p in c.tables[s][c.tables[s] >= 0].tolist():
            for t in (c.k, c.v):
                t[1, p] = bits(torch.randn(Hkv, page, D, generator=g, device="cuda"))
    qkv = bits(torch.randn(2, 12 * D, generator=g, device="cuda"))
    q = torch.zeros(2, 8 * D, dtype=torch.int16, device="cuda")
    c.append(1, i32([0, 1]), qkv, q)
    for s, n in enumerate(lens):
        pid = int(c.tables[s, (n - 1) // page])
        assert torch.equal(c.v[1, pid, :, (n - 1) % page], qkv[s].view(12, D)[10:])
    check_attend(c, [1, 0], 2, layer=1)
    src, dst = [int(c.tables[0, 0]), int(c.tables[1, 0])], [pages - 10, 3]
    want = c.k[:, src].clone()
    c.copy_pages(i32(src), i32(dst))
    assert torch.equal(c.k[:, dst], want)
    before = c.k[1, c.tables[0, :3].long()].clone()
    c.compact()
    assert c.error_word() == 0 and sorted(c.tables[:2].flatten().tolist()) == [-1, 0, 1, 2, 3, 4]
    assert torch.equal(c.k[1, c.tables[0, :3].long()], before)


@pytest.mark.parametrize("N,kv,D,Hq", [(2048, "bf16", 128, 2), (4096, "bf16", 128, 4), (4096, "bf16", 64, 2),
                                       (4096, "e4m3", 256, 2), (4096, "bf16", 256, 64)])
def test_a_batch_of_the_largest_size_over_one_shared_prompt(N, kv, D, Hq):
    """N slots of N sequences that share one prompt's pages, each with a token of its own."""
    c = make(layers=1, pages=N + 52, page=16, Hkv=1, D=D, max_seqs=N, max_pages=8, Hq=Hq, max_batch=N, kv=kv)
    c.resize(i32([0]), i32([100]))
    rest = list(range(1, N))
    c.fork(i32([0] * (N - 1)), i32(rest))
    allseq = i32(list(range(N)))
    c.resize(allseq, i32([101] * N))
    assert c.error_word() == 0 and c.refs.max() == N
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = bits(torch.randn(N, (Hq + 2) * D, device="cuda", generator=g))
    q, out = (torch.zeros(N, Hq * D, dtype=torch.int16, device="cuda") for _ in range(2))
    c.append(0, allseq, qkv, q)
    c.attend(0, allseq, q, out)
    assert c.error_word() == 0
    pick = [0, 1, 7, 1000, N - 1]
    want, tol = attend64(c, 0, pick, q[pick].contiguous(), 1, D ** -0.5, kv)
    assert bool(((vals(out[pick]) - want).abs() <= tol).all())


@pytest.mark.parametrize("kv,D,Hkv,G,Tq", [("bf16", 256, 1, 8, 8), ("e4m3", 256, 2, 16, 2), ("bf16", 64, 2, 1, 7),
                                          ("bf16", 128, 1, 128, 8), ("e4m3", 128, 4, 2, 8), ("bf16", 256, 2, 3, 1)])
def test_attention_of_random_batches(kv, D, Hkv, G, Tq):
    r = random.Random(D + G)
    for seed in range(4):
        lens = [max(0, int(r.expovariate(1 / 150))) if r.random() < 0.9 else r.randint(500, 2500)
                for _ in range(r.randint(1, 14))]
        kw = {} if kv == "bf16" else dict(k_scale=torch.full((1, Hkv), 0.02, device="cuda"),
                                          v_scale=torch.full((1, Hkv), 0.03, device="cuda"))
        c = filled(lens, Tq=Tq, Hq=G * Hkv, Hkv=Hkv, D=D, page=r.choice((16, 32, 48, 64, 128, 1024)), kv=kv, seed=seed,
                   max_batch=20, **kw)
        seqs = list(range(len(lens))) + [-1] * r.randint(0, 2)
        r.shuffle(seqs)
        check_attend(c, seqs, Tq, kv)
