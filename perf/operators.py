"""The paged-cache and speculative-decoding operators as they are measured: their cases, inputs, plain forms in elementary
torch operations and definitions in 64 bits.

A case names one pass: attention over a paged cache (`attend`), the write of new keys and values into it (`append`), the
fork of sequences and their first growth (`fork`), the compaction of a cache (`compact`), the verification of drafted
tokens (`verify`), and the step from logits to probabilities (`softmax`). bf16 values travel as their bits (int16), as
everywhere in this package; e4m3 caches as uint8."""
import math

import torch

own = False

OPS = ("attend", "append", "fork", "compact", "verify", "softmax")


# ------------------------------------------------------------------ cases

def _attend(name, B, length, Tq=1, Hq=16, Hkv=2, D=256, page=64, kv="bf16", ragged=True):
    return {"name": name, "op": "attend", "B": B, "len": length, "Tq": Tq, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "kv": kv, "ragged": ragged}


def _append(name, B, Tq, length, Hq=16, Hkv=2, D=256, page=64, rope=64):
    return {"name": name, "op": "append", "B": B, "Tq": Tq, "len": length, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "rope": rope}


def _fork(name, parents, children, length, layers, Hkv=2, D=256, page=64):
    return {"name": name, "op": "fork", "parents": parents, "children": children, "len": length, "layers": layers,
            "Hkv": Hkv, "D": D, "page": page}


def _compact(name, pages, layers, live, Hkv=2, D=256, page=64):
    return {"name": name, "op": "compact", "pages": pages, "layers": layers, "live": live, "Hkv": Hkv, "D": D,
            "page": page}


def _verify(name, B, K, V):
    return {"name": name, "op": "verify", "B": B, "K": K, "V": V}


def _softmax(name, R, V):
    return {"name": name, "op": "softmax", "R": R, "V": V}


def listed():
    return [
        # one user's chat a thousand tokens in: latency is all there is
        _attend("attend_one_short", B=1, length=1001, ragged=False),
        # one user's long document: the split over the length alone fills the card
        _attend("attend_one_long", B=1, length=131071, ragged=False),
        # a serving batch in mid-flight: every sequence has another length, some slots are empty
        _attend("attend_batch", B=48, length=8192, page=32),
        # the same service with an 8-bit cache, four drafted tokens a sequence, heads of 128
        _attend("attend_draft_e4m3", B=24, length=16000, Tq=4, Hq=32, Hkv=8, D=128, page=16, kv="e4m3"),
        # one decode step of a batch writes its keys and values
        _append("append_step", B=64, Tq=1, length=4097),
        # prompts in their middle: chunks of new tokens at far positions
        _append("append_prompt", B=3, Tq=1365, length=100003),
        # sampling several answers to each of a few prompts: fork them, then give every child room for a token
        _fork("fork_answers", parents=4, children=32, length=2087, layers=10),
        # after a day's service: the live pages are scattered over the pool
        _compact("compact_pool", pages=3001, layers=4, live=0.4),
        # one user's drafts
        _verify("verify_one", B=1, K=3, V=151936),
        # a batch's drafts
        _verify("verify_batch", B=64, K=4, V=151936),
        # one user's drafts once more: the rows of logits behind their probabilities
        _softmax("softmax_one", R=4, V=151936),
        # a batch's logits turned into probabilities, each row at its user's temperature
        _softmax("softmax_batch", R=192, V=151936),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(OPS)
    if op == "attend":
        while True:
            kv = rng.choice(("bf16", "e4m3"))
            D = rng.choice((128, 256) if kv == "e4m3" else (64, 128, 256))
            Hkv = rng.choice((1, 2, 4, 8))
            c = dict(_attend("", B=_log_int(rng, 1, 128), length=_log_int(rng, 1, 131071), Tq=rng.choice((1, 1, 1, 2, 4, 7)),
                             Hq=Hkv * rng.choice((1, 2, 4, 5, 8)), Hkv=Hkv, D=D, page=rng.choice((16, 32, 48, 64, 128)),
                             kv=kv, ragged=rng.random() < 0.8))
            if work(c)["bytes"] <= 6e8 and c["B"] * c["len"] * Hkv * D <= 4e8:
                break
    elif op == "append":
        Hkv = rng.choice((1, 2, 4, 8))
        D = rng.choice((64, 128, 256))
        Tq = _log_int(rng, 1, 2048)
        c = _append("", B=_log_int(rng, 1, max(1, 4096 // Tq)), Tq=Tq, length=Tq + _log_int(rng, 1, 120000),
                    Hq=Hkv * rng.choice((1, 2, 4, 8)), Hkv=Hkv, D=D, page=rng.choice((16, 32, 48, 64, 128)),
                    rope=rng.choice((0, 32, 64, D // 2, D)))
    elif op == "fork":
        c = _fork("", parents=_log_int(rng, 1, 8), children=_log_int(rng, 1, 96), length=_log_int(rng, 1, 4000),
                  layers=_log_int(rng, 1, 10), Hkv=rng.choice((1, 2, 4)), D=rng.choice((64, 128, 256)),
                  page=rng.choice((16, 32, 48, 64)))
    elif op == "compact":
        c = _compact("", pages=_log_int(rng, 40, 3001), layers=rng.choice((1, 2, 3, 4)), live=round(rng.uniform(0.05, 0.95), 2),
                     Hkv=rng.choice((1, 2)), D=rng.choice((64, 128, 256)), page=rng.choice((16, 32, 48, 64)))
    elif op == "verify":
        c = _verify("", B=_log_int(rng, 1, 64), K=rng.randint(1, 7), V=_log_int(rng, 1000, 200000))
    else:
        V = _log_int(rng, 1000, 200000)
        c = _softmax("", R=max(1, min(_log_int(rng, 1, 512), int(2.9e7 / V))), V=V)
    del c["name"]
    return c


def _lens(c):
    """The sequences' lengths: fixed by the case, so that its work is. Ragged batches spread over (0, len], and from eight
    sequences on hold a new one of one token and an empty one."""
    B, n = c["B"], c["len"]
    if not c.get("ragged"):
        return [n] * B
    got = [n] + [max(1, int(n * (((b + 1) * 0.6180339887498949) % 1.0))) for b in range(1, B)]
    if B >= 8:
        got[1], got[2] = 1, 0
    return got


def _slot(c):
    """The place in the batch that a captured step of a fixed size leaves unused, or none."""
    return 5 if c.get("ragged") and c["B"] >= 8 else -1


def _filled(n, page):
    return (n + page - 1) // page


def work(c):
    op = c["op"]
    if op == "attend":
        es = 1 if c["kv"] == "e4m3" else 2
        keys = sum(n for b, n in enumerate(_lens(c)) if b != _slot(c))
        rows = c["B"] * c["Tq"] * c["Hq"] * c["D"]
        return {"bytes": 2 * keys * c["Hkv"] * c["D"] * es + 4 * rows, "flops": 4 * keys * c["Hq"] * c["D"] * c["Tq"]}
    if op == "append":
        n, hq, hkv, D = c["B"] * c["Tq"], c["Hq"], c["Hkv"], c["D"]
        return {"bytes": 2 * n * D * ((hq + 2 * hkv) + (hq + 2 * hkv)), "flops": 6 * n * (hq + hkv) * D}
    if op == "fork":
        rest = c["len"] % c["page"]
        row = c["Hkv"] * c["D"] * 2
        return {"bytes": 2 * 2 * c["children"] * c["layers"] * rest * row + 8 * c["children"] * _filled(c["len"], c["page"]),
                "flops": 0}
    if op == "compact":
        n = c["pages"]
        moved = n * c["live"] * (1 - c["live"])  # live pages that lie behind the first n_live, on average
        return {"bytes": 2 * 2 * moved * c["layers"] * c["Hkv"] * c["page"] * c["D"] * 2 + 16 * n, "flops": 0}
    if op == "verify":
        return {"bytes": 8 * c["B"] * c["V"], "flops": 4 * c["B"] * c["V"]}
    return {"bytes": 8 * c["R"] * c["V"], "flops": 4 * c["R"] * c["V"]}


# ------------------------------------------------------------------ inputs

def _normal16(g, *shape, std=1.0, mean=0.0):
    return (mean + std * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16).view(torch.int16)


def _pool(g, c, layers, pages, kv):
    shape = (layers, pages, c["Hkv"], c["page"], c["D"])
    if kv == "bf16":
        return _normal16(g, *shape), _normal16(g, *shape)
    return tuple(torch.randn(*shape, generator=g, device="cuda").mul_(40.0).to(torch.float8_e4m3fn).view(torch.uint8)
                 for _ in range(2))


def _tables(lens, page, pages, seed, spare=0):
    """Every sequence's pages, scattered over the pool: [seqs][max_pages] with -1 behind the last, and the holders."""
    r = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=r).to(torch.int32)
    wide = max(1, max(_filled(n, page) for n in lens)) + spare
    tables = torch.full((len(lens), wide), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        k = _filled(n, page)
        tables[b, :k] = order[at:at + k]
        at += k
    refs[order[:at].long()] = 1
    return tables, refs


def _handle(c, s):
    from mvcc_b200.paged import PagedCache
    return PagedCache(s["k"], s["v"], s["tables"], s["refs"], s["lens"], Hq=c.get("Hq", c["Hkv"]),
                      max_batch=max(c.get("B", 1), c.get("children", 1)), max_new=c.get("Tq", 1),
                      k_scale=s.get("k_scale"), v_scale=s.get("v_scale"))


def prepare(case, seed):
    c, op = case, case["op"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if op in ("attend", "append"):
        lens = _lens(c) if op == "attend" else [max(c["Tq"], c["len"] - 17 * b) for b in range(c["B"])]
        # an appending batch keeps only the pages that its new tokens fall into: what was there before is not read
        if op == "attend":
            pages = sum(_filled(n, c["page"]) for n in lens) + 3
            tables, refs = _tables(lens, c["page"], pages, seed)
        else:
            first = [(n - c["Tq"]) // c["page"] for n in lens]
            held = [_filled(n, c["page"]) - f for n, f in zip(lens, first)]
            pages = sum(held) + 3
            some, refs = _tables([h * c["page"] for h in held], c["page"], pages, seed)
            tables = torch.full((c["B"], max(_filled(n, c["page"]) for n in lens)), -1, dtype=torch.int32)
            for b in range(c["B"]):
                tables[b, first[b]:first[b] + held[b]] = some[b, :held[b]]
        s["k"], s["v"] = _pool(g, c, 1, pages, c.get("kv", "bf16"))
        s["tables"], s["refs"] = tables.cuda(), refs.cuda()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        seqs = list(range(c["B"]))
        if op == "attend" and _slot(c) >= 0:
            seqs[_slot(c)] = -1
        s["seqs"] = torch.tensor(seqs, dtype=torch.int32, device="cuda")
        if c.get("kv") == "e4m3":
            s["k_scale"] = 0.02 + 0.01 * torch.rand(1, c["Hkv"], generator=g, device="cuda")
            s["v_scale"] = 0.02 + 0.01 * torch.rand(1, c["Hkv"], generator=g, device="cuda")
        n, D = c["B"] * c["Tq"], c["D"]
        if op == "attend":
            s["q"] = _normal16(g, n, c["Hq"] * D, std=2.0)  # sharper than even: a few keys carry a row
            s["out"] = torch.zeros(n, c["Hq"] * D, dtype=torch.int16, device="cuda")
        else:
            s["qkv"] = _normal16(g, n, (c["Hq"] + 2 * c["Hkv"]) * D, std=0.9)
            s["q_norm"], s["k_norm"] = _normal16(g, D, std=0.1, mean=1.0), _normal16(g, D, std=0.1, mean=1.0)
            s["q"] = torch.zeros(n, c["Hq"] * D, dtype=torch.int16, device="cuda")
            r = c["rope"]
            s["inv_freq"] = (1.0e7 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)).cuda() if r else None
    elif op in ("fork", "compact"):
        if op == "fork":
            p, n = c["parents"], c["children"]
            lens = [c["len"]] * p + [0] * n
            pages = p * _filled(c["len"], c["page"]) + n + 5
            tables, refs = _tables(lens, c["page"], pages, seed, spare=1)
            s["src"] = torch.tensor([i % p for i in range(n)], dtype=torch.int32, device="cuda")
            s["dst"] = torch.arange(p, p + n, dtype=torch.int32, device="cuda")
            s["none"] = torch.zeros(n, dtype=torch.int32, device="cuda")
            s["grown"] = torch.full((n,), c["len"] + 1, dtype=torch.int32, device="cuda")
        else:
            pages = c["pages"]
            live = max(1, min(pages, round(pages * c["live"])))
            each = max(1, live // 29)
            lens = [each * c["page"]] * (live // each) + ([live % each * c["page"]] if live % each else [])
            tables, refs = _tables(lens, c["page"], pages, seed)
        s["k"], s["v"] = _pool(g, c, c["layers"], pages, "bf16")
        # one buffer for the state, so that a pass can put it back in one copy
        rows, wide = tables.shape
        state = torch.cat([tables.reshape(-1), refs, torch.tensor(lens, dtype=torch.int32)]).cuda()
        s["state"], s["kept"] = state, state.clone()
        s["tables"] = state[:rows * wide].view(rows, wide)
        s["refs"] = state[rows * wide:rows * wide + pages]
        s["lens"] = state[rows * wide + pages:]
    elif op == "verify":
        B, K, V = c["B"], c["K"], c["V"]
        z = 2.5 * torch.randn(B, K + 1, V, generator=g, device="cuda")
        s["target"] = torch.softmax(z, -1)
        y = z[:, :K] + 0.8 * torch.randn(B, K, V, generator=g, device="cuda")
        s["draft"] = torch.softmax(y, -1)
        del z
        y -= torch.log(-torch.log(torch.rand(B, K, V, generator=g, device="cuda").clamp_(1e-30, 1 - 1e-7)))
        s["drafted"] = y.argmax(-1).to(torch.int32)  # drawn from the draft's own probabilities
        del y
        s["u"] = torch.rand(B, K + 1, generator=g, device="cuda")
        s["tokens"] = torch.zeros(B, K + 1, dtype=torch.int32, device="cuda")
        s["accepted"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    else:
        R, V = c["R"], c["V"]
        s["logits"] = 3.0 * torch.randn(R, V, generator=g, device="cuda")
        t = 0.5 + torch.rand(R, generator=g, device="cuda")
        t[3::7] = 0.0  # greedy users
        s["temperature"] = t
        s["probs"] = torch.empty(R, V, device="cuda")
    if own:
        if op == "verify":
            from mvcc_b200.spec import SpecVerifier
            s["handle"] = SpecVerifier(c["B"], c["K"], c["V"], device=s["u"].device)
        elif op != "softmax":
            s["handle"] = _handle(c, s)
    return s


# ------------------------------------------------------------------ one pass

def _values(t):
    return t.view(torch.bfloat16)


def run(s):
    c, op = s["case"], s["case"]["op"]
    if own:
        h = s.get("handle")
        if op == "attend":
            h.attend(0, s["seqs"], s["q"], s["out"], Tq=c["Tq"])
        elif op == "append":
            h.append(0, s["seqs"], s["qkv"], s["q"], Tq=c["Tq"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                     inv_freq=s["inv_freq"])
        elif op == "fork":
            h.resize(s["dst"], s["none"])
            h.fork(s["src"], s["dst"])
            h.resize(s["dst"], s["grown"])
        elif op == "compact":
            s["state"].copy_(s["kept"])
            h.compact()
        elif op == "verify":
            h.verify(s["target"], s["draft"], s["drafted"], s["u"], s["tokens"], s["accepted"])
        else:
            from mvcc_b200.spec import softmax_rows
            softmax_rows(s["logits"], s["probs"], temperature=s["temperature"])
    elif op == "attend":
        _plain_attend(s)
    elif op == "append":
        _plain_append(s)
    elif op == "fork":
        _plain_resize(s, s["dst"], s["none"])
        _plain_fork(s, s["src"], s["dst"])
        _plain_resize(s, s["dst"], s["grown"])
    elif op == "compact":
        s["state"].copy_(s["kept"])
        _plain_compact(s)
    elif op == "verify":
        _plain_verify(s)
    else:
        _plain_softmax(s)
    if op == "attend":
        return _values(s["out"])
    if op == "append":
        return {"q": _values(s["q"]), "k": _values(s["k"]), "v": _values(s["v"])}
    if op in ("fork", "compact"):
        return {"tables": s["tables"], "refs": s["refs"], "lens": s["lens"], "k": _values(s["k"]), "v": _values(s["v"])}
    if op == "verify":
        return {"tokens": s["tokens"], "accepted": s["accepted"]}
    return s["probs"]


# ------------------------------------------------------------------ plain forms

def _stored(t, scale):
    """A cache's values in 32 bits: [..., Hkv, page, D]."""
    if scale is None:
        return t.view(torch.bfloat16).float()
    return t.view(torch.float8_e4m3fn).float() * scale.view(-1, 1, 1)


def _plain_attend(s):
    c = s["case"]
    B, Tq, Hq, Hkv, D, page = (c[n] for n in ("B", "Tq", "Hq", "Hkv", "D", "page"))
    G = Hq // Hkv
    there = s["seqs"] >= 0
    row = s["seqs"].clamp(min=0).long()
    n = torch.where(there, s["lens"][row], 0)
    ids = s["tables"][row].clamp(min=0).long()
    P = ids.shape[1]

    def keys(pool, scale):  # [B, Hkv, P page, D]
        return _stored(pool[0][ids], scale).permute(0, 2, 1, 3, 4).reshape(B, Hkv, P * page, D)

    at = torch.arange(P * page, device=n.device)
    q = s["q"].view(torch.bfloat16).float().view(B, Tq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Tq * G, D)
    z = torch.matmul(q, keys(s["k"], s.get("k_scale")).transpose(-1, -2)) * (1.0 / math.sqrt(D))
    last = n[:, None] - Tq + torch.arange(Tq, device=n.device)  # the position of each new token
    seen = (at <= last[:, :, None]).repeat_interleave(G, 1)[:, None]  # [B, 1, Tq G, keys]
    z = torch.where(seen, z, -math.inf)
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isinf(m), 0.0, m))
    total = e.sum(-1, keepdim=True)
    v = torch.where((at < n[:, None])[:, None, :, None], keys(s["v"], s.get("v_scale")), 0.0)
    o = torch.matmul(e, v) / torch.where(total == 0, 1.0, total)
    o = o.view(B, Hkv, Tq, G, D).permute(0, 2, 1, 3, 4).reshape(B * Tq, Hq * D)
    s["out"].copy_(o.to(torch.bfloat16).view(torch.int16))


def _plain_append(s):
    c = s["case"]
    B, Tq, Hq, Hkv, D, page, r = (c[n] for n in ("B", "Tq", "Hq", "Hkv", "D", "page", "rope"))
    pos = (s["lens"][s["seqs"].long()][:, None] - Tq + torch.arange(Tq, device="cuda")).long()  # [B, Tq]
    x = s["qkv"].view(torch.bfloat16).float().view(B * Tq, Hq + 2 * Hkv, D)

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.view(torch.bfloat16).float()
        if not r:
            return x
        angle = pos.reshape(-1, 1).double() * s["inv_freq"]
        cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)

    s["q"].copy_(turned(x[:, :Hq], s["q_norm"]).to(torch.bfloat16).view(torch.int16).view(B * Tq, Hq * D))
    ids = torch.gather(s["tables"][s["seqs"].long()], 1, pos // page).reshape(-1).long()
    off = (pos % page).reshape(-1)
    s["k"][0][ids, :, off] = turned(x[:, Hq:Hq + Hkv], s["k_norm"]).to(torch.bfloat16).view(torch.int16)
    s["v"][0][ids, :, off] = s["qkv"].view(B * Tq, Hq + 2 * Hkv, D)[:, Hq + Hkv:]


def _plain_resize(s, seqs, new):
    c, page = s["case"], s["case"]["page"]
    tables, refs, lens = s["tables"], s["refs"], s["lens"]
    seqs = seqs.long()
    rows, old = tables[seqs], lens[seqs]
    held, want = (old + page - 1) // page, (new + page - 1) // page
    col = torch.arange(tables.shape[1], device=rows.device)
    # the pages behind the new end go
    gone = (col >= want[:, None]) & (col < held[:, None])
    refs.scatter_add_(0, torch.where(gone, rows, 0).reshape(-1).long(), -gone.reshape(-1).int())
    rows = torch.where(gone, -1, rows)
    # a partly filled last page that others hold too is copied: all its holders here but the last one, if no other has it
    kept = torch.minimum(old, new)
    part = kept % page != 0
    at = (kept // page).long().clamp(max=tables.shape[1] - 1)
    last = torch.gather(rows, 1, at[:, None])[:, 0]
    same = (last[:, None] == last) & part[:, None] & part
    before = torch.tril(same, -1).sum(1)
    copied = part & (before < refs[last.clamp(min=0).long()] - 1)
    # the lowest free pages, in the order of the list, the copy before the growth
    need = copied.int() + (want - held).clamp(min=0)
    start = torch.cumsum(need, 0) - need
    free = torch.argsort((refs != 0).to(torch.int8), stable=True).int()
    target = free[start.clamp(max=free.numel() - 1).long()]
    grown = (col >= held[:, None]) & (col < want[:, None])
    which = (start + copied)[:, None] + (col - held[:, None])
    rows = torch.where(grown, free[which.clamp(0, free.numel() - 1).long()], rows)
    rows = torch.where((col == at[:, None]) & copied[:, None], target[:, None], rows)
    refs.scatter_add_(0, torch.where(copied, last, 0).long(), -copied.int())
    refs.scatter_add_(0, torch.where(grown, rows, 0).reshape(-1).long(), grown.reshape(-1).int())
    refs.scatter_add_(0, torch.where(copied, target, 0).long(), copied.int())
    tables[seqs], lens[seqs] = rows, new
    i = torch.nonzero(copied)[:, 0]
    a, b = last[i].long(), target[i].long()
    fill = (torch.arange(page, device=rows.device) < (kept[i] % page)[:, None])[None, :, None, :, None]
    for_k, for_v = (torch.where(fill, t[:, a], t[:, b]) for t in (s["k"], s["v"]))
    s["k"][:, b], s["v"][:, b] = for_k, for_v


def _plain_fork(s, src, dst):
    tables, refs, lens = s["tables"], s["refs"], s["lens"]
    rows = tables[src.long()]
    tables[dst.long()], lens[dst.long()] = rows, lens[src.long()]
    refs.scatter_add_(0, rows.clamp(min=0).reshape(-1).long(), (rows >= 0).reshape(-1).int())


def _plain_compact(s):
    tables, refs = s["tables"], s["refs"]
    live = refs > 0
    n = int(live.sum())
    holes, high = torch.nonzero(~live[:n])[:, 0], torch.nonzero(live[n:])[:, 0] + n
    to = torch.arange(refs.numel(), device=refs.device, dtype=torch.int32)
    to[high] = holes.int()
    tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()], tables))
    refs[holes] = refs[high]
    refs[high] = 0
    s["k"][:, holes], s["v"][:, holes] = s["k"][:, high], s["v"][:, high]


def _plain_verify(s):
    p, q, x, u = s["target"], s["draft"], s["drafted"].long(), s["u"].double()
    B, K = x.shape
    px = torch.gather(p[:, :K], 2, x[:, :, None])[:, :, 0].double()
    qx = torch.gather(q, 2, x[:, :, None])[:, :, 0].double()
    n = torch.cumprod((u[:, :K] * qx < px).int(), 1).sum(1)
    b = torch.arange(B, device=p.device)
    pa = p[b, n].double()
    w = torch.where((n < K)[:, None], (pa - q[b, n.clamp(max=K - 1)].double()).clamp(min=0), pa)
    w = torch.where((w.sum(1) > 0)[:, None], w, pa)
    run = torch.cumsum(w, 1)
    token = (run <= u[:, K:] * run[:, -1:]).sum(1)
    at = torch.arange(K + 1, device=p.device)
    drafted = torch.cat([s["drafted"], s["drafted"][:, :1]], 1)
    s["tokens"].copy_(torch.where(at < n[:, None], drafted, torch.where(at == n[:, None], token[:, None], -1)))
    s["accepted"].copy_(n)


def _plain_softmax(s):
    x, t = s["logits"], s["temperature"][:, None]
    m = x.amax(1, keepdim=True)
    e = torch.exp((x - m) / torch.where(t > 0, t, 1.0))
    best = torch.arange(x.shape[1], device=x.device) == x.argmax(1, keepdim=True)
    s["probs"].copy_(torch.where(t > 0, e / e.sum(1, keepdim=True), best.float()))


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    if op == "attend":
        B, Tq, Hq, Hkv, D, page = (c[n] for n in ("B", "Tq", "Hq", "Hkv", "D", "page"))
        q = s["q"].view(torch.bfloat16).double().view(B, Tq, Hq, D)
        out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device="cuda")
        kinds = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
        for b, i in enumerate(s["seqs"].tolist()):
            n = int(s["lens"][i]) if i >= 0 else 0
            if n == 0:
                continue
            ids = s["tables"][i, :_filled(n, page)].long()
            for h in range(Hkv):
                k, v = (s[name][0, ids, h].view(kinds[c["kv"]]).double().view(-1, D)[:n] for name in ("k", "v"))
                if c["kv"] == "e4m3":
                    k, v = k * s["k_scale"][0, h].double(), v * s["v_scale"][0, h].double()
                heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                for t in range(max(0, Tq - n), Tq):
                    end = n - Tq + t + 1
                    z = q[b, t, heads] @ k[:end].T / math.sqrt(D)
                    out[b, t, heads] = torch.softmax(z, -1) @ v[:end]
        return out.view(B * Tq, Hq * D)
    if op == "append":
        B, Tq, Hq, Hkv, D, page, r = (c[n] for n in ("B", "Tq", "Hq", "Hkv", "D", "page", "rope"))
        x = s["qkv"].view(torch.bfloat16).double().view(B, Tq, Hq + 2 * Hkv, D)
        w = torch.cat([s["q_norm"].view(torch.bfloat16).double().expand(Hq, D),
                       s["k_norm"].view(torch.bfloat16).double().expand(Hkv, D)])
        y = x[:, :, :Hq + Hkv]
        y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + 1e-6) * w
        pos = s["lens"].double().view(B, 1) - Tq + torch.arange(Tq, device="cuda")
        if r:
            turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), pos[..., None] * s["inv_freq"])
            z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * turn[:, :, None]
            y = torch.cat([z.real, z.imag, y[..., r:]], -1)
        k, v = (s[n].view(torch.bfloat16).double() for n in ("k", "v"))
        for b in range(B):
            ids = s["tables"][b].long()[(pos[b].long() // page)]
            off = pos[b].long() % page
            k[0, ids, :, off] = y[b, :, Hq:]
            v[0, ids, :, off] = x[b, :, Hq + Hkv:]
        return {"q": y[:, :, :Hq].reshape(B * Tq, Hq * D), "k": k, "v": v}
    if op in ("fork", "compact"):
        page = c["page"]
        tables, refs, lens = (s[n].cpu() for n in ("tables", "refs", "lens"))
        k, v = s["k"].clone(), s["v"].clone()
        if op == "fork":
            for i, d in enumerate(s["dst"].tolist()):  # share, one child after another
                a = int(s["src"][i])
                tables[d], lens[d] = tables[a], lens[a]
                refs[tables[a][tables[a] >= 0].long()] += 1
            for d in s["dst"].tolist():
                n = int(lens[d])
                free = iter(torch.nonzero(refs == 0)[:, 0].tolist())
                if n % page:
                    p, t = int(tables[d, n // page]), next(free)
                    refs[p] -= 1
                    tables[d, n // page] = t
                    k[:, t, :, :n % page], v[:, t, :, :n % page] = k[:, p, :, :n % page], v[:, p, :, :n % page]
                else:
                    t = next(free)
                    tables[d, n // page] = t
                refs[t] = 1
                lens[d] = n + 1
        else:
            n = int((refs > 0).sum())
            to = 0
            moved = {}
            for p in range(n, refs.numel()):
                if refs[p] > 0:
                    while refs[to] > 0:
                        to += 1
                    refs[to], refs[p], moved[p] = refs[p].clone(), 0, to
            a, b = (torch.tensor(list(z), dtype=torch.long, device="cuda") for z in (moved.keys(), moved.values()))
            k[:, b], v[:, b] = k[:, a], v[:, a]
            tables = torch.tensor([[moved.get(p, p) for p in row] for row in tables.tolist()], dtype=torch.int32)
        return {"tables": tables, "refs": refs, "lens": lens, "k": _values(k).double(), "v": _values(v).double()}
    if op == "verify":
        B, K = c["B"], c["K"]
        p, q, x, u = s["target"].double(), s["draft"].double(), s["drafted"].tolist(), s["u"].double()
        tokens, accepted = torch.full((B, K + 1), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        for b in range(B):
            a = 0
            while a < K and float(u[b, a]) * float(q[b, a, x[b][a]]) < float(p[b, a, x[b][a]]):
                tokens[b, a] = x[b][a]
                a += 1
            w = torch.relu(p[b, a] - q[b, a]) if a < K else p[b, a]
            run_ = torch.cumsum(w, 0)
            tokens[b, a] = int(torch.searchsorted(run_, u[b, K] * run_[-1], right=True))
            accepted[b] = a
        return {"tokens": tokens, "accepted": accepted}
    x, t = s["logits"].double(), s["temperature"].double()
    out = torch.zeros_like(x)
    for i, f in enumerate(t.tolist()):
        if f > 0:
            out[i] = torch.softmax(x[i] / f, 0)
        else:
            out[i, int(x[i].argmax())] = 1.0
    return out
