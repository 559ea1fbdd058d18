"""Serving from a 4-bit key/value cache, as cases whose time can be measured: block tables, norm and rotation of queries and keys,
writing to the cache and reading from it, attention over it.

``own = False`` computes each in elementary torch operations; ``own = True`` calls the framework.  The cache's storage (one uint8
record per page and kv head) is the framework's, and :func:`_parts` says what lies where.
"""
import math
import random

import torch

own = False


def _case(name, op, **kw):
    c = {"name": name, "op": op}
    c.update(kw)
    return c


def listed():
    return [
        # page bookkeeping of one decoding step, and of a step that takes in many prompts at once
        _case("tables_step", "tables", B=48, before=6000, new=1, page=64),
        _case("tables_prompts", "tables", B=700, before=500, new=1000, page=16),
        # norm and rotation: a decoding step; an image model's layout without norms, adjacent channels paired; a video transformer
        _case("rope_step", "rope", B=1, N=48, Hq=32, Hkv=8, D=128, rot=128, norm=True, adjacent=False, layout="NHD"),
        _case("rope_image", "rope", B=4, N=4096, Hq=32, Hkv=32, D=64, rot=32, norm=False, adjacent=True, layout="HND"),
        _case("rope_video", "rope", B=1, N=32760, Hq=40, Hkv=40, D=128, rot=128, norm=True, adjacent=True, layout="NHD"),
        # new tokens into the cache and their values back: a decoding step straight from the projections; many prompts' k and v
        _case("cache_step", "cache", N=48, Hq=32, Hkv=8, D=128, page=64, fused=True),
        _case("cache_prompts", "cache", N=20011, Hq=32, Hkv=8, D=128, page=64, fused=False),
        # attention over the cache: one short conversation; a serving batch; few very long contexts; some drafted tokens per
        # sequence; chunks of prompts behind cached prefixes
        _case("decode_one", "attend", B=1, Hq=32, Hkv=8, D=128, q=1, kv=1000, page=64, lse=False),
        _case("decode_batch", "attend", B=32, Hq=32, Hkv=8, D=128, q=1, kv=8192, page=64, lse=False),
        _case("decode_long", "attend", B=2, Hq=32, Hkv=8, D=128, q=1, kv=131072, page=128, lse=True),
        _case("drafts", "attend", B=16, Hq=32, Hkv=8, D=64, q=5, kv=4096, page=16, lse=False),
        _case("prompt_chunks", "attend", B=2, Hq=32, Hkv=8, D=128, q=2048, kv=16384, page=64, lse=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["tables", "rope", "rope", "cache", "cache", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 64, 128])
    D = rng.choice([128, 128, 64])
    Hkv = rng.choice([1, 4, 8, 8, 16])
    Hq = Hkv * rng.choice([1, 2, 4, 4, 7, 8])
    if op == "tables":
        c = dict(B=_log_uniform(rng, 1, 1024), before=_log_uniform(rng, 1, 8192), new=_log_uniform(rng, 1, 1024), page=page)
        c["new"] = min(c["new"], max(1, 350000 // c["B"]))
        return _drawn(op, **c)
    if op == "rope":
        N = _log_uniform(rng, 1, 32768)
        return _drawn(op, B=1 if N > 4096 else rng.choice([1, 2, 4]), N=N, Hq=Hq if Hq <= 40 else 32, Hkv=Hkv if Hq <= 40 else 8, D=rng.choice([64, 96, 128, 128]),
                      rot=rng.choice([32, 64, 64]), norm=rng.random() < 0.7, adjacent=rng.random() < 0.5, layout=rng.choice(["NHD", "HND"]))
    if op == "cache":
        return _drawn(op, N=_log_uniform(rng, 1, 20000 * 8 // max(8, Hkv)), Hq=min(Hq, 64), Hkv=Hkv if Hq <= 64 else 8, D=D, page=page, fused=rng.random() < 0.5)
    q = rng.choice([1, 1, 1, _log_uniform(rng, 2, 16), _log_uniform(rng, 17, 2048)])
    Hq, Hkv = (Hq, Hkv) if Hq <= 64 else (32, 8)
    kv = max(q, _log_uniform(rng, 128, 131072 if q == 1 else 16384))
    B = _log_uniform(rng, 1, max(1, min(64, (262144 if q == 1 else 32768) * 8 // (max(Hkv, 8) * kv))))
    if q > 16:
        B = max(1, min(B, 2 ** 31 // (q * kv * Hq)))
    return _drawn(op, B=B, Hq=Hq, Hkv=Hkv, D=D, q=q, kv=kv, page=page, lse=rng.random() < 0.3)


def _drawn(op, **kw):
    return {"op": op, **kw}


# ------------------------------------------------------------------------------------------------ the cache's storage
def _record_bytes(D):
    return 18 * D                                       # of 16 tokens: 8 D + D bytes of keys, as many of values


def _parts(rec, D):
    """Records of 16 tokens [..., 18 D] -> key codes [..., 16, D/2], key scales [..., 16, D/16], and those of the values."""
    lead, nb = rec.shape[:-1], D // 16
    n = len(lead)
    keep = list(range(n))
    kc = rec[..., :8 * D].reshape(*lead, 16, D // 2)
    ks = rec[..., 8 * D:9 * D].reshape(*lead, 8, 4, 2, nb // 4).permute(*keep, n + 2, n, n + 1, n + 3).reshape(*lead, 16, nb)
    vc = rec[..., 9 * D:17 * D].reshape(*lead, 2, 8, 4, 2, D // 16).permute(*keep, n, n + 2, n + 3, n + 1, n + 4).reshape(*lead, 16, D // 2)
    vs = rec[..., 17 * D:].reshape(*lead, nb, 4, 2, 2).permute(*keep, n + 2, n + 1, n + 3, n).reshape(*lead, 16, nb)
    return kc, ks, vc, vs


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x):
    """fp32 [..., D] -> codes uint8 [..., D/2] (two to a byte, the even channel low) and E4M3 scale bytes [..., D/16]."""
    b = x.reshape(*x.shape[:-1], -1, 16)
    s = (b.abs().amax(-1) / 6).clamp(max=448.0).to(torch.float8_e4m3fn)
    sf = s.float()[..., None]
    y = torch.where(sf > 0, b / sf, torch.zeros_like(b))
    a = y.abs()
    c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)) + 8 * (y < 0).to(torch.uint8)
    c = c.reshape(*x.shape)
    return c[..., 0::2] + 16 * c[..., 1::2], s.view(torch.uint8)


def _values(codes, scales, dtype=torch.float32):
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=dtype, device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[pair.int()]
    s = scales.contiguous().view(torch.float8_e4m3fn).to(dtype)
    return (x.unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2)


def _write(data, slots, k, v, page, offset):
    """k, v bf16 [T, H, D] to their slots."""
    T, H, D = k.shape
    R = _record_bytes(D)
    k = (k.float() - offset.float()).to(torch.bfloat16).float()
    at = _parts(torch.arange(R, device=k.device), D)
    group = (slots // page)[:, None] * (H * page // 16) + torch.arange(H, device=k.device) * (page // 16) + (slots % page // 16)[:, None]
    flat = data.view(-1)
    for w, o in zip(_quantise(k) + _quantise(v.float()), at):
        flat[group[..., None] * R + o[slots % 16][:, None]] = w


def _read(data, slots, D, page, offset):
    H = data.shape[1]
    rec = data.view(data.shape[0], H, page // 16, _record_bytes(D))[slots // page, :, slots % page // 16]
    row = (slots % 16)[:, None, None, None]
    kc, ks, vc, vs = (p.gather(2, row.expand(-1, H, 1, p.shape[-1]))[:, :, 0] for p in _parts(rec, D))
    return (_values(kc, ks) + offset.float()).to(torch.bfloat16), _values(vc, vs).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(B, longest, seed):
    """Ragged lengths, the longest one first, the others spread over a factor of four."""
    rng = random.Random(B * 1000003 + longest * 7 + seed)
    return [longest] + [_log_uniform(rng, max(1, longest // 4), longest) for _ in range(B - 1)]


def _int(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _q_lengths(case):
    return _lengths(case["B"], case["q"], 2) if case["q"] > 16 else [case["q"]] * case["B"]


def _kv_lengths(case):
    return [max(a, b) for a, b in zip(_lengths(case["B"], case["kv"], 1), _q_lengths(case))]


def _starts(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def perm(n):
        return torch.randperm(n, generator=g, device="cuda")

    op, st = case["op"], {"case": case}
    if op == "tables":
        B, page = case["B"], case["page"]
        # the same requests in another order for another seed, so that there are as many tokens
        rng = random.Random(B * 1000003 + case["new"])
        new = [1] * B if case["new"] == 1 else [_log_uniform(rng, 1, case["new"]) for _ in range(B)]
        rng = random.Random(seed)
        rng.shuffle(new)
        before = [rng.randint(0, case["before"]) for _ in range(B)]
        cols = -(-(case["before"] + case["new"]) // page)
        have = [-(-n // page) for n in before]
        ids = perm(sum(have) + B * (2 + case["new"] // page)).to(torch.int32)
        table = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(cols, device="cuda")[None, :] < _int(have)[:, None]
        table[held] = ids[:sum(have)]
        st.update(before=_int(before), new=_int(new), table=table, free=ids[sum(have):].contiguous(), tokens=sum(new))
        return st
    if op in ("rope", "cache"):
        D, Hq, Hkv, N = case["D"], case["Hq"], case["Hkv"], case["N"]
        B, rot = case.get("B", 1), case.get("rot", case["D"])
        # projections: q, k and v side by side in one row, as a fused projection leaves them
        qkv = normal(B, N, Hq + 2 * Hkv, D)
        qkv[:, :, Hq:Hq + Hkv] += 2.0 * normal(1, 1, Hkv, D)
        qkv = qkv.to(torch.bfloat16)
        if case.get("layout", "NHD") == "HND":
            q, k, v = (t.transpose(1, 2).contiguous() for t in (qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]))
        else:
            q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
        st.update(q=q, k=k, v=v)
        places = 4096 if N <= 4096 else 32768
        angle = torch.arange(places, device="cuda", dtype=torch.float64)[:, None] * torch.pow(10000.0, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        st.update(cos=angle.cos().float(), sin=angle.sin().float(),
                  positions=torch.randint(places, (B, N), generator=g, device="cuda", dtype=torch.int32),
                  qw=(1 + 0.2 * normal(D)).to(torch.bfloat16), kw=(1 + 0.2 * normal(D)).to(torch.bfloat16))
        if op == "cache":
            pages = -(-N // case["page"]) + 3
            st.update(data=torch.randint(256, (pages, Hkv, case["page"] // 16 * _record_bytes(D)), generator=g, device="cuda", dtype=torch.uint8),
                      slots=perm(pages * case["page"])[:N].contiguous() if N <= 64 else
                      (perm(pages)[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).flatten()[:N].contiguous(),
                      offset=normal(Hkv, D).to(torch.bfloat16))
            st["q"], st["k"], st["v"], st["positions"] = q[0], k[0], v[0], st["positions"][0]
        return st
    B, Hq, Hkv, D, page = (case[n] for n in ("B", "Hq", "Hkv", "D", "page"))
    ql, kl = _q_lengths(case), _kv_lengths(case)
    pages = [-(-n // page) for n in kl]
    total, G = sum(pages), page // 16
    data = torch.empty(total + 2, Hkv, G, _record_bytes(D), device="cuda", dtype=torch.uint8)
    for p in range(0, total + 2, max(1, 65536 // page)):
        part = data[p:p + max(1, 65536 // page)]
        for w, to in zip(_quantise(normal(part.shape[0], Hkv, G, 16, D).to(torch.bfloat16).float()) +
                         _quantise(normal(part.shape[0], Hkv, G, 16, D).to(torch.bfloat16).float()),
                         _parts(torch.arange(_record_bytes(D), device="cuda"), D)):
            part[..., to.flatten()] = w.flatten(-2)
    table = torch.full((B, max(pages)), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(max(pages), device="cuda")[None, :] < _int(pages)[:, None]] = perm(total + 2)[:total].to(torch.int32)
    st.update(data=data.view(total + 2, Hkv, G * _record_bytes(D)), table=table, kv_lens=_int(kl), cu=_int(_starts(ql)),
              q=normal(sum(ql), Hq, D).to(torch.bfloat16), offset=normal(Hkv, D).to(torch.bfloat16), max_q=max(ql), max_k=max(kl))
    return st


# ------------------------------------------------------------------------------------------------ the plain forms
def _tables_plain(st):
    page, table, T, dev = st["case"]["page"], st["table"], st["tokens"], st["table"].device
    before, new, free = st["before"].long(), st["new"].long(), st["free"]
    after = before + new
    have = (before + page - 1) // page
    need = (after + page - 1) // page - have
    off = need.cumsum(0) - need
    j = torch.arange(table.shape[1], device=dev)[None, :] - have[:, None]
    idx = off[:, None] + j
    entry = torch.where(idx < free.numel(), free[idx.clamp(0, free.numel() - 1)], torch.full_like(table, -1))
    table.copy_(torch.where((j >= 0) & (j < need[:, None]), entry, table))
    cu = torch.cat((new.new_zeros(1), new.cumsum(0)))
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=dev), new, output_size=T)
    position = before[seq] + torch.arange(T, device=dev) - cu[seq]
    held = table[seq, (position // page).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where((held >= 0) & (position // page < table.shape[1]), held * page + position % page, torch.full_like(held, -1))
    return {"table": table, "kv_lens": after.int(), "cu": cu.int(), "positions": position.int(), "slots": slots, "pages": need.sum().int()[None]}


def _norm_rope(x, w, cos, sin, rot, adjacent, dtype=torch.float32):
    x = x.to(dtype)
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.to(dtype)
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if adjacent else (r[..., :rot // 2], r[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((ra, rb), -1).flatten(-2) if adjacent else torch.cat((ra, rb), -1)
    return torch.cat((r, x[..., rot:]), -1).to(torch.bfloat16 if dtype == torch.float32 else dtype)


def _rope_plain(st, dtype=torch.float32):
    case = st["case"]
    heads = 1 if case.get("layout") == "HND" else -2
    cos, sin = (st[n][st["positions"].long()].to(dtype).unsqueeze(heads) for n in ("cos", "sin"))
    norm, rot = case.get("norm", True), case.get("rot", case["D"])
    return tuple(_norm_rope(st[n], st[w] if norm else None, cos, sin, rot, case.get("adjacent", False), dtype) for n, w in (("q", "qw"), ("k", "kw")))


def _attend_plain(st):
    case, q = st["case"], st["q"]
    B, Hq, Hkv, D, page = (case[n] for n in ("B", "Hq", "Hkv", "D", "page"))
    scale, dev = D ** -0.5, q.device
    rec = st["data"].view(-1, Hkv, page // 16, _record_bytes(D))[st["table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3)
    kc, ks, vc, vs = (p.flatten(2, 3) for p in _parts(rec, D))
    k, v = _values(kc, ks), _values(vc, vs)                                    # [B, Hkv, keys, D]
    cu, kv = st["cu"].long(), st["kv_lens"].long()
    ql = cu[1:] - cu[:-1]
    t = torch.arange(st["max_q"], device=dev)
    rows = (cu[:-1, None] + t).clamp(max=q.shape[0] - 1)
    x = q[rows].float().unflatten(2, (Hkv, Hq // Hkv)).permute(0, 2, 1, 3, 4).flatten(2, 3)         # [B, Hkv, tokens x group, D]
    s = torch.matmul(x * scale, k.transpose(2, 3)).unflatten(2, (st["max_q"], -1))
    seen = (kv - ql)[:, None] + t + 1                                          # keys that a token sees
    s.masked_fill_(torch.arange(k.shape[2], device=dev) >= seen[:, None, :, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(m))
    total = p.sum(-1, keepdim=True)
    o = (torch.matmul(p.flatten(2, 3), v).unflatten(2, (st["max_q"], -1)) / total).permute(0, 2, 1, 3, 4).flatten(2, 3)
    lse = (m + total.log())[..., 0].permute(0, 2, 1, 3).flatten(2, 3)          # [B, tokens, Hq]
    use = t < ql[:, None]
    lse = lse + scale * (q[rows].float() * st["offset"].float().repeat_interleave(Hq // Hkv, 0)).sum(-1)
    out = o[use].to(torch.bfloat16)
    return (out, lse[use]) if case["lse"] else out


def run(state):
    st, case = state, state["case"]
    op = case["op"]
    if own:
        import sageattention_b200 as sa
        if op == "tables":
            r = sa.build_block_tables(st["before"], st["new"], st["table"], st["free"], case["page"], num_tokens=st["tokens"])
            return {"table": st["table"], "kv_lens": r.kv_lens, "cu": r.cu_seqlens_q, "positions": r.positions, "slots": r.slots, "pages": r.pages_taken}
        if op == "rope":
            return sa.qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], st["positions"], q_weight=st["qw"] if case["norm"] else None,
                                   k_weight=st["kw"] if case["norm"] else None, adjacent_pairs=case["adjacent"], tensor_layout=case["layout"])
        cache = sa.FP4KVCache(st["data"], head_dim=case["D"], page_size=case["page"], k_offset=st["offset"])
        if op == "cache" and case["fused"]:
            q = sa.qk_norm_rope_append(st["q"], st["k"], st["v"], cache, st["slots"], st["cos"], st["sin"], st["positions"], q_weight=st["qw"], k_weight=st["kw"])
            return (q,) + cache.read(st["slots"])
        if op == "cache":
            cache.append(st["k"], st["v"], st["slots"])
            return cache.read(st["slots"])
        return sa.sageattn_kvcache(st["q"], cache, st["table"], st["kv_lens"], st["cu"], max_seqlen_q=st["max_q"], max_seqlen_k=st["max_k"], return_lse=case["lse"])
    if op == "tables":
        return _tables_plain(st)
    if op == "rope":
        return _rope_plain(st)
    if op == "cache":
        q, k = _rope_plain(st) if case["fused"] else (None, st["k"])
        _write(st["data"], st["slots"], k, st["v"], case["page"], st["offset"])
        kv = _read(st["data"], st["slots"], case["D"], case["page"], st["offset"])
        return (q,) + kv if case["fused"] else kv
    return _attend_plain(st)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "tables":
        B, mean = case["B"], 1 if case["new"] == 1 else (case["new"] - 1) / math.log(case["new"])
        return {"bytes": B * (4 * 4.0 + 8 * mean / case["page"]) + 12.0 * B * mean, "flops": 0.0}
    if op in ("rope", "cache"):
        rows, D, Hq, Hkv = case.get("B", 1) * case["N"], case["D"], case["Hq"], case["Hkv"]
        if op == "rope":
            return {"bytes": rows * (8.0 * D * (Hq + Hkv) / 2 + 4 * case["rot"] + 4), "flops": 0.0}
        stored = 9 * D / 8.0 * Hkv
        own_part = rows * (4.0 * D * Hq + 4 * D + 4) if case["fused"] else 0.0
        return {"bytes": own_part + rows * (4.0 * D * Hkv + stored + 8 + stored + 8 + 4.0 * D * Hkv), "flops": 0.0}
    ql, kl = _q_lengths(case), _kv_lengths(case)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(ql, kl))
    return {"bytes": sum(kl) * Hkv * 9 * D / 8.0 + sum(ql) * Hq * (4.0 * D + (4 if case["lse"] else 0)), "flops": 4.0 * Hq * D * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def _nearest(x, grid):
    """The value of an ascending grid (from 0) that is nearest to each |x|, the even place on a tie, with x's sign."""
    a = x.abs()
    i = torch.searchsorted(grid, a).clamp(1, len(grid) - 1)
    lo, hi = grid[i - 1], grid[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    return torch.where(up, hi, lo) * torch.where(x < 0, -1.0, 1.0).to(x.dtype)


def _exact_round(x):
    """What a block of 16 of x (64 bits) stands for in the cache."""
    b = x.unflatten(-1, (-1, 16))
    e4m3 = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                        dtype=torch.float64, device=x.device)
    e2m1 = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    s = _nearest(b.abs().amax(-1, keepdim=True) / 6, e4m3)
    return (_nearest(torch.where(s > 0, b / s.clamp(min=1e-300), torch.zeros_like(b)), e2m1) * s).flatten(-2)


def exact(case, seed):
    op = case["op"]
    if op == "tables":
        return None
    st = prepare(case, seed)
    if op == "rope":
        places = st["positions"].long().unsqueeze(1 if case["layout"] == "HND" else 2)
        half, D = case["rot"] // 2, case["D"]
        # a rotation is a product of complex numbers
        turn = torch.complex(st["cos"].double()[places], st["sin"].double()[places])
        out = []
        for n in ("q", "k"):
            x = st[n].double()
            if case["norm"]:
                x = x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * st[n + "w"].double()
            pairs = x[..., :2 * half].unflatten(-1, (half, 2)) if case["adjacent"] else x[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            out.append(torch.cat((z.flatten(-2) if case["adjacent"] else z.transpose(-1, -2).flatten(-2), x[..., 2 * half:]), -1))
        return tuple(out)
    if op == "cache":
        q, k, v = (st[n].double() for n in ("q", "k", "v"))
        if case["fused"]:
            turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"].long()][:, None]
            half, both = case["D"] // 2, []
            for x, w in ((q, st["qw"]), (k, st["kw"])):
                x = x / ((x * x).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
                z = torch.complex(x[..., :half], x[..., half:]) * turn
                both.append(torch.cat((z.real, z.imag), -1))
            q, k = both[0], both[1].to(torch.bfloat16).double()
        off = st["offset"].double()
        kh = _exact_round((k - off).to(torch.bfloat16).double()) + off
        vh = _exact_round(v)
        return (q, kh, vh) if case["fused"] else (kh, vh)
    B, Hq, Hkv, D, page = (case[n] for n in ("B", "Hq", "Hkv", "D", "page"))
    ql, kl, g = _q_lengths(case), _kv_lengths(case), Hq // Hkv
    cu = _starts(ql)
    if sum(a * b for a, b in zip(ql, kl)) * Hq * D > 2 ** 43:
        return None
    outs, lses = [], []
    for i in range(B):
        rec = st["data"][st["table"][i, :-(-kl[i] // page)].long()].view(-1, Hkv, page // 16, 18 * D)
        rec = rec.permute(1, 0, 2, 3).reshape(Hkv, -1, 18 * D)
        oh, lh = [], []
        for h in range(Hkv):
            kc, ks, vc, vs = (p.reshape(-1, p.shape[-1])[:kl[i]] for p in _parts(rec[h], D))
            k, v = _values(kc, ks, torch.float64), _values(vc, vs, torch.float64)
            x = st["q"][cu[i]:cu[i + 1], h * g:(h + 1) * g].double()
            s = torch.einsum("tgd,kd->gtk", x, k) * D ** -0.5
            late = torch.arange(kl[i], device="cuda")[None, :] > torch.arange(kl[i] - ql[i], kl[i], device="cuda")[:, None]
            s.masked_fill_(late, float("-inf"))
            l = torch.logsumexp(s, -1)
            oh.append(torch.einsum("gtk,kd->tgd", torch.exp(s - l[..., None]), v))
            lh.append(l.T + D ** -0.5 * torch.einsum("tgd,d->tg", x, st["offset"][h].double()))
        outs.append(torch.cat(oh, 1))
        lses.append(torch.cat(lh, 1))
    return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)
