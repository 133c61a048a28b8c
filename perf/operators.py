"""Cases of the batched decoder's cache operators, with their plain forms.

Four operators work on one paged key/value cache (``wisp_b200.paged``):

* ``rope``      rotary positions on q and k, with k and v appended to the cache's pages;
* ``attention`` causal attention over the pages, with a sliding window and a few first
  tokens (sinks) that stay visible, for prompts, chunks and single tokens;
* ``prefix``    the same attention for sequences that share a long prefix, whose pages
  are read once for all of a group;
* ``pages``     pages copied inside the pool of all layers (fork and compaction).

A case's lengths follow from the case alone; the values, the page order and the page
moves follow from the seed.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------ cases
def _attention(name, op="attention", **kw):
    case = {"name": name, "op": op, "seqs": 1, "empty": 0, "q_min": 1, "q_max": 1, "kv_min": 1,
            "kv_max": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "f16",
            "cache": "f16", "page": 16, "window": 0, "sinks": 0, "groups": 0, "prefix": 0}
    case.update(kw)
    return case


def _rope(name, **kw):
    case = {"name": name, "op": "rope", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 1,
            "kv_max": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "f16",
            "cache": "f16", "page": 16, "rot": 128, "off": 0, "interleaved": False,
            "theta": 1e6, "stretch": 1.0}
    case.update(kw)
    return case


def _pages(name, **kw):
    case = {"name": name, "op": "pages", "layers": 32, "pool": 256, "moves": 4, "page": 16,
            "kv_heads": 8, "dim": 128, "cache": "f16"}
    case.update(kw)
    return case


def listed():
    return [
        # one token of a single chat at 1024 positions, in the decoder's own 32-bit rows
        _attention("attn-one", dtype="f32", kv_min=1024, kv_max=1024),
        # a decode batch of 16 ragged chats, two slots of the fixed-size batch unused
        _attention("attn-batch", seqs=16, empty=2, kv_min=1, kv_max=4096),
        # 64 long chats that keep a window of 4096 and four first tokens
        _attention("attn-window", seqs=64, kv_min=8192, kv_max=32768, dtype="bf16",
                   cache="bf16", page=64, window=4096, sinks=4),
        # four drafted tokens of each of four very long documents verified at once
        _attention("attn-verify", seqs=4, q_min=4, q_max=4, kv_min=65536, kv_max=131072,
                   heads=64, page=64),
        # one prompt of 8192 tokens
        _attention("attn-prompt", q_min=8192, q_max=8192, kv_min=8192, kv_max=8192, page=64),
        # ragged prompt chunks behind what is cached already, window and sinks, 64-wide heads
        _attention("attn-chunks", seqs=5, q_min=1, q_max=3001, kv_min=3001, kv_max=9001,
                   heads=16, kv_heads=16, dim=64, dtype="bf16", cache="bf16", page=32,
                   window=1024, sinks=16),
        # eight answers to one question
        _attention("prefix-few", op="prefix", seqs=8, groups=1, prefix=2048, kv_min=1,
                   kv_max=128),
        # 64 chats in two groups, each behind its own long shared document
        _attention("prefix-many", op="prefix", seqs=64, groups=2, prefix=32768, kv_min=32,
                   kv_max=1032, dtype="bf16", cache="bf16", page=64),
        # the rows of one decode step of 16 chats, 32-bit projections into a 16-bit cache
        _rope("rope-step", seqs=16, kv_min=1, kv_max=32768, dtype="f32"),
        # the rows of three ragged prompts, some 10,000 tokens: interleaved pairs, half of the
        # head, frequencies stretched for a long context
        _rope("rope-prompt", seqs=3, q_min=1000, q_max=4461, kv_min=4461, kv_max=131072,
              dtype="bf16", cache="bf16", page=64, rot=64, interleaved=True, stretch=8.0),
        # the last pages of four forked chats
        _pages("pages-fork"),
        # a pool of 2048 pages compacted
        _pages("pages-compact", pool=2048, moves=512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "few", "prompt", "prefix", "rope", "pages"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (8, 2), (16, 1), (24, 8), (12, 4)])
    dim = rng.choice([64, 128, 128, 128, 96])
    cache = rng.choice(["f16", "bf16"])
    dtype = rng.choice([cache, cache, "f32"])
    page = rng.choice([16, 32, 48, 64, 128])
    common = dict(heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, cache=cache, page=page)
    if rng.random() < 0.4 and kind in ("decode", "few", "prompt"):
        common.update(window=_log(rng, 100, 5000), sinks=rng.choice([0, 1, 4, 50]))
    if kind in ("decode", "few"):
        seqs = _log(rng, 1, 64)
        kv = _log(rng, 16, min(131072, int(5e8) // (seqs * kv_heads * dim)))
        q = 1 if kind == "decode" else min(kv, rng.randint(2, 9))
        return _drop(_attention("", seqs=seqs, empty=rng.randint(0, seqs // 4), q_min=q, q_max=q,
                                kv_min=max(q, kv // rng.randint(1, 9)), kv_max=kv, **common))
    if kind == "prompt":
        seqs = rng.randint(1, 6)
        most = 8192 * 4096 // max(4096, heads * dim)
        q = _log(rng, 16, most // seqs)
        kv = q + rng.choice([0, _log(rng, 1, (most - q) // 3 + 1)])
        return _drop(_attention("", seqs=seqs, q_min=rng.randint(1, q), q_max=q, kv_min=q,
                                kv_max=kv, **common))
    if kind == "prefix":
        groups = rng.randint(1, 3)
        seqs = max(groups, _log(rng, 2, 64))
        prefix = _log(rng, 64, 32768)
        return _drop(_attention("", op="prefix", seqs=seqs, groups=groups, prefix=prefix,
                                kv_min=rng.randint(1, 40), kv_max=rng.randint(41, 900),
                                **common))
    if kind == "rope":
        seqs = _log(rng, 1, 64)
        q = _log(rng, 1, 8192 // seqs)
        kv = _log(rng, q, 131072) if seqs < 9 else _log(rng, q, 16384)
        return _drop(_rope("", seqs=seqs, q_min=rng.randint(1, q), q_max=q, kv_min=q, kv_max=kv,
                           rot=rng.choice([dim, dim // 2, 32]), off=rng.choice([0, dim // 2])
                           if dim > 64 else 0, interleaved=rng.random() < 0.5,
                           stretch=rng.choice([1.0, 4.0, 16.0]), **common))
    case = _pages("", layers=rng.choice([1, 4, 32]), page=rng.choice([16, 16, 48, 8]),
                  kv_heads=rng.choice([1, 2, 8]), dim=rng.choice([64, 96, 128]), cache=cache)
    one = 2 * case["layers"] * case["page"] * case["kv_heads"] * case["dim"]
    case["pool"] = _log(rng, 8, min(2048, (1 << 31) // one))
    case["moves"] = _log(rng, 1, case["pool"] // 4)
    return _drop(case)


def _drop(case):
    if case["op"] == "rope" and case["off"] + case["rot"] > case["dim"]:
        case["off"] = case["dim"] - case["rot"]
    del case["name"]
    return case


# ------------------------------------------------------------------------ lengths
def _lengths(case):
    """(tokens, cached positions) of each sequence: spread over the case's range, which counts
    from the end of the prefix where there is one."""
    n, live = case["seqs"], case["seqs"] - case.get("empty", 0)
    q, kv = [], []
    for i in range(live):
        f, g = (i * 0.6180339887) % 1.0, (i * 0.7548776662) % 1.0
        f, g = (1.0, 1.0) if i == 0 else (f, g)
        kv.append(case["kv_min"] + round(f * (case["kv_max"] - case["kv_min"])))
        q.append(min(kv[-1], case["q_min"] + round(g * (case["q_max"] - case["q_min"]))))
    if case.get("groups"):
        starts, before = _group_starts(case), _prefixes(case)
        kv = [a + before[sum(s >= b for b in starts[1:])] for s, a in enumerate(kv)]
    q += [case["q_min"]] * (n - live)  # an unused slot: tokens, but nothing cached
    kv += [0] * (n - live)
    return q, kv


def _group_starts(case):
    n, g = case["seqs"], case["groups"]
    return [i * n // g for i in range(g + 1)]


def _prefixes(case):
    """The groups' prefix lengths: the first has the case's, the next ones less."""
    return [max(1, case["prefix"] * (case["groups"] - i) // case["groups"])
            for i in range(case["groups"])]


def _frequencies(case):
    """Rotary frequencies of each pair, 64-bit; with a stretch s the slow ones are divided by s
    and the ones between blended (fewer than 1 and more than 32 turns in 4096 positions)."""
    r = case["rot"]
    f = case["theta"] ** (-2.0 * torch.arange(r // 2, dtype=torch.float64) / r)
    s = case["stretch"]
    if s != 1.0:
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
    return f, 1.0 if s == 1.0 else 0.1 * math.log(s) + 1.0


# ------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    cdt = DTYPES[case["cache"]]

    def randn(*shape, dtype):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    if case["op"] == "pages":
        shape = (case["layers"], case["pool"], case["page"], case["kv_heads"], case["dim"])
        order = torch.randperm(case["pool"], generator=torch.Generator().manual_seed(int(seed)))
        order, m = order.tolist(), case["moves"]
        return {"case": case, "k": randn(*shape, dtype=cdt), "v": randn(*shape, dtype=cdt),
                "src": order[:m], "dst": order[m:2 * m]}
    q_len, kv_len = _lengths(case)
    page, nh, nkv, hd = case["page"], case["heads"], case["kv_heads"], case["dim"]
    T = sum(q_len)
    pages_of = [-(-n // page) for n in kv_len]
    shared = [0] * len(kv_len)
    if case["op"] == "prefix":  # a prefix ends where it ends: only its whole pages are shared
        for i, p in enumerate(_prefixes(case)):
            for s in range(_group_starts(case)[i], _group_starts(case)[i + 1]):
                shared[s] = p // page
    n_shared = 0
    if case["op"] == "prefix":
        n_shared = sum(p // page for p in _prefixes(case))
    n_pages = n_shared + sum(a - b for a, b in zip(pages_of, shared)) + 3
    perm = torch.randperm(n_pages, generator=g, device=dev, dtype=torch.int32)
    table = torch.zeros(len(kv_len), max(1, max(pages_of)), dtype=torch.int32, device=dev)
    at, group_at = n_shared, 0
    if case["op"] == "prefix":
        starts = _group_starts(case)
        for i, p in enumerate(_prefixes(case)):
            n = p // page
            table[starts[i]:starts[i + 1], :n] = perm[group_at:group_at + n]
            group_at += n
    for s, n in enumerate(pages_of):
        fresh = n - shared[s]
        table[s, shared[s]:n] = perm[at:at + fresh]
        at += fresh
    k, v = (randn(n_pages, page, nkv, hd, dtype=cdt) for _ in range(2))
    starts = torch.tensor([0] + q_len).cumsum(0).to(dev, torch.int32)
    st = {"case": case, "k": k, "v": v, "table": table, "q_start": starts,
          "kv_len": torch.tensor(kv_len, dtype=torch.int32, device=dev),
          "max_q": max(q_len), "max_kv": max(kv_len)}
    if case["op"] == "rope":
        rows = randn(T, (nh + 2 * nkv) * hd, dtype=DTYPES[case["dtype"]])  # the fused projection
        st["rows"] = [rows[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in
                      ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv))]
        freq, st["gain"] = _frequencies(case)
        st["freq"] = freq.to(dev)
    else:
        st["q"] = randn(T, nh, hd, dtype=DTYPES[case["dtype"]])
        if case["op"] == "prefix":
            # what lies past the shared whole pages belongs to each sequence
            lens = [p // page * page for p in _prefixes(case)]
            st["groups"] = torch.tensor(_group_starts(case), dtype=torch.int32, device=dev)
            st["prefix"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    return st


# ------------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    if own:
        return _own(st, op)
    if op == "rope":
        return _plain_rope(st)
    if op == "pages":
        return _plain_pages(st)
    return _plain_attention(st)


def _own(st, op):
    from wisp_b200 import paged
    case = st["case"]
    if op == "pages":
        paged.copy_pages(st["k"], st["v"], st["src"], st["dst"])
        return {"k": st["k"], "v": st["v"]}
    batch = paged.TokenBatch(st["q_start"], st["kv_len"], st["table"], st["max_q"])
    if op == "rope":
        q, k, v = st["rows"]
        out = paged.rope_append(q, k, v, st["k"], st["v"], batch, st["freq"],
                                offset=case["off"], interleaved=case["interleaved"],
                                gain=st["gain"])
        return {"q": out, "k": st["k"], "v": st["v"]}
    if op == "prefix":
        out, lse = paged.prefix_attention(st["q"], st["k"], st["v"], batch, st["groups"],
                                          st["prefix"], window=case["window"],
                                          sinks=case["sinks"], return_lse=True)
    else:
        out, lse = paged.attention(st["q"], st["k"], st["v"], batch, window=case["window"],
                                   sinks=case["sinks"], return_lse=True)
    return {"out": out, "lse": lse}


def _token_places(st):
    """For each token: its sequence and its position in the sequence's cache."""
    T = st["rows"][0].shape[0] if "rows" in st else st["q"].shape[0]
    q_start, kv_len = st["q_start"].long(), st["kv_len"].long()
    t = torch.arange(T, device=q_start.device)
    seq = torch.searchsorted(q_start, t, right=True) - 1
    return seq, kv_len[seq] - (q_start[seq + 1] - t)


def _plain_rope(st):
    case = st["case"]
    seq, pos = _token_places(st)
    ang = pos.double()[:, None] * st["freq"]
    c, s = (ang.cos() * st["gain"]).float()[:, None], (ang.sin() * st["gain"]).float()[:, None]
    lo, r = case["off"], case["rot"]

    def rotated(x):
        y = x.float()
        w = y[..., lo:lo + r]
        if case["interleaved"]:
            a, b = w[..., 0::2], w[..., 1::2]
            w = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
        else:
            a, b = w[..., :r // 2], w[..., r // 2:]
            w = torch.cat((a * c - b * s, b * c + a * s), -1)
        return torch.cat((y[..., :lo], w, y[..., lo + r:]), -1)

    q, k, v = st["rows"]
    page = st["table"].long()[seq, pos // case["page"]]
    st["k"][page, pos % case["page"]] = rotated(k).to(st["k"].dtype)
    st["v"][page, pos % case["page"]] = v.to(st["v"].dtype)
    return {"q": rotated(q).to(q.dtype), "k": st["k"], "v": st["v"]}


def _plain_attention(st):
    case, dev = st["case"], st["q"].device
    nh, nkv, hd, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    B, Q, N, G = case["seqs"], st["max_q"], max(1, st["max_kv"]), nh // nkv
    seq, pos = _token_places(st)
    row = torch.arange(len(seq), device=dev) - st["q_start"].long()[seq]
    q = torch.zeros(B, Q, nkv, G, hd, device=dev)
    q[seq, row] = st["q"].float().view(-1, nkv, G, hd)
    at = torch.full((B, Q), -1, device=dev)
    at[seq, row] = pos
    j = torch.arange(N, device=dev)
    pages = st["table"].long()[:, j // page]
    k = st["k"][pages, j % page].permute(0, 2, 3, 1).float()  # [B, nkv, hd, N]
    v = st["v"][pages, j % page].permute(0, 2, 1, 3).float()  # [B, nkv, N, hd]
    s = q.permute(0, 2, 3, 1, 4).reshape(B, nkv, G * Q, hd) @ k
    del k
    s = s.view(B, nkv, G, Q, N).mul_(hd ** -0.5)
    p = at[:, :, None]
    seen = (j <= p) & (j < st["kv_len"][:, None, None])
    if case["window"]:
        seen &= (p - j < case["window"]) | (j < case["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m.isinf(), torch.zeros_like(m), m)
    s = s.sub_(m).exp_()
    l = s.sum(-1, keepdim=True)
    o = (s.view(B, nkv, G * Q, N) @ v).view(B, nkv, G, Q, hd)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    lse = (m + l.log()).squeeze(-1)
    out = o.permute(0, 3, 1, 2, 4)[seq, row].reshape(-1, nh, hd)
    return {"out": out.to(st["q"].dtype), "lse": lse.permute(0, 3, 1, 2)[seq, row].reshape(-1, nh)}


def _plain_pages(st):
    src, dst = (torch.tensor(st[n], device=st["k"].device) for n in ("src", "dst"))
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]
    return {"k": st["k"], "v": st["v"]}


# ------------------------------------------------------------------------ costs
def _visible(case, q, kv):
    """(visible pairs of one head, positions that some token sees) of one sequence."""
    w, sinks, pairs = case["window"], case["sinks"], 0
    for i in range(q):
        p = kv - q + i  # sees j <= p: the window's and the sinks before it
        if p >= 0:
            pairs += p + 1 if not w else min(p + 1, w) + min(sinks, max(0, p + 1 - w))
    first = max(0, kv - q)
    low = max(0, first - w + 1) if w else 0
    return pairs, (kv - low) + min(sinks, low) if kv else 0


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    c = size[case["cache"]]
    if case["op"] == "pages":
        one = case["layers"] * case["page"] * case["kv_heads"] * case["dim"] * c
        return {"bytes": 4 * case["moves"] * one, "flops": 0}
    q_len, kv_len = _lengths(case)
    T, d, nh, nkv, hd = sum(q_len), size[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        rows = T * hd * ((2 * nh + 2 * nkv) * d + 2 * nkv * c)
        return {"bytes": rows + case["rot"] * 4, "flops": 3 * T * (nh + nkv) * case["rot"]}
    pairs = keys = 0
    for q, kv in zip(q_len, kv_len):
        a, b = _visible(case, q, kv)
        pairs, keys = pairs + a, keys + b
    if case["op"] == "prefix" and not case["window"]:
        starts = _group_starts(case)
        for i, p in enumerate(_prefixes(case)):
            keys -= (starts[i + 1] - starts[i] - 1) * (p // case["page"] * case["page"])
    return {"bytes": T * nh * (2 * hd * d + 4) + 2 * keys * nkv * hd * c,
            "flops": 4 * hd * nh * pairs}


# ------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "pages":
        for n in ("k", "v"):
            kept = [st[n][:, a].clone() for a in st["src"]]
            for b, x in zip(st["dst"], kept):
                st[n][:, b] = x
        return {"k": st["k"], "v": st["v"]}
    q_len, kv_len = _lengths(case)
    page, hd, G = case["page"], case["dim"], case["heads"] // case["kv_heads"]
    if case["op"] == "rope":
        q, k, v = (x.double() for x in st["rows"])
        freq, gain = _frequencies(case)
        at, half = 0, case["rot"] // 2
        first, step, gap = (0, 2, 1) if case["interleaved"] else (0, 1, half)
        one = torch.arange(half, device=q.device) * step + case["off"] + first
        kp, vp = st["k"].double(), st["v"].double()
        for s, (n, kv) in enumerate(zip(q_len, kv_len)):
            p = torch.arange(kv - n, kv, device=q.device)
            turn = torch.polar(torch.full((n, half), gain, dtype=torch.float64, device=q.device),
                               p.double()[:, None] * freq.to(q.device))[:, None]
            for x in (q, k):
                z = torch.complex(x[at:at + n][..., one], x[at:at + n][..., one + gap]) * turn
                x[at:at + n, :, one], x[at:at + n, :, one + gap] = z.real, z.imag
            where = st["table"][s, p // page].long()
            kp[where, p % page], vp[where, p % page] = k[at:at + n], v[at:at + n]
            at += n
        return {"q": q, "k": kp, "v": vp}
    out = torch.zeros(sum(q_len), case["heads"], hd, dtype=torch.float64, device=st["q"].device)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device=out.device)
    at = 0
    for s, (n, kv) in enumerate(zip(q_len, kv_len)):
        if kv:
            pages = st["table"][s, :-(-kv // page)].long()
            i = torch.arange(kv - n, kv, device=out.device)[:, None]
            j = torch.arange(kv, device=out.device)[None]
            hidden = j > i
            if case["window"]:
                hidden |= (i - j >= case["window"]) & (j >= case["sinks"])
            for h in range(case["kv_heads"]):
                k = st["k"][pages][:, :, h].reshape(-1, hd)[:kv].double()
                v = st["v"][pages][:, :, h].reshape(-1, hd)[:kv].double()
                for a in range(h * G, h * G + G):
                    x = (st["q"][at:at + n, a].double() @ k.T / math.sqrt(hd)).masked_fill(
                        hidden, -math.inf)
                    z = torch.logsumexp(x, 1)
                    out[at:at + n, a] = torch.exp(x - z[:, None]) @ v
                    lse[at:at + n, a] = z
        at += n
    return {"out": out, "lse": lse}
