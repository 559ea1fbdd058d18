"""Serving from the 4-bit cache against the restatement in 64 bits (``_kv_reference``), whose bounds on the errors are derived there.
Every kernel's inputs lie in pages in a shuffled order, in a cache full of arbitrary bytes, NaN scales among them."""
import random

import numpy as np
import pytest
import torch

import sageattention_b200 as sa
from tests import _kv_reference as R

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, generator=g).to(BF)


# ------------------------------------------------------------------------------------------------ block tables
def tables_reference(before, new, table, free, page, n):
    table, pos, slots, kv, cu, taken = [list(r) for r in table], [0] * n, [-1] * n, [], [0], 0
    at = 0
    for i, (b, a) in enumerate(zip(before, new)):
        for j in range(-(-b // page), -(-(b + a) // page)):
            if j < len(table[i]):
                table[i][j] = free[taken] if taken < len(free) else -1
            taken += 1
        for t in range(a):
            if at < n:
                p = b + t
                col = p // page
                pos[at] = p
                slots[at] = table[i][col] * page + p % page if col < len(table[i]) and table[i][col] >= 0 else -1
            at += 1
        kv.append(b + a)
        cu.append(at)
    return table, kv, cu, pos, slots, taken


def run_tables(before, new, table, free, page, n):
    i32 = dict(dtype=torch.int32, device=DEV)
    t = torch.tensor(table, **i32)
    r = sa.build_block_tables(torch.tensor(before, **i32), torch.tensor(new, **i32), t, torch.tensor(free, **i32), page, n)
    return t, r


@pytest.mark.parametrize("B,longest,new,page,spare,cols,pad", [
    (1, 0, 1, 16, 0, 1, 0), (1, 16, 1, 16, 0, 2, 0), (1, 15, 1, 16, 0, 1, 3), (3, 100, 0, 32, 0, 5, 2), (257, 300, 40, 16, 5, 25, 0), (700, 500, 200, 64, 0, 11, 100),
    (5, 200, 100, 16, -4, 20, 0), (5, 200, 100, 16, 3, 12, 0), (1, 10, 5000, 128, 1, 60, 1), (3000, 50, 3, 32, 0, 2, 0), (16384, 20, 2, 16, 0, 2, 5)])
def test_block_tables(B, longest, new, page, spare, cols, pad):
    rng = random.Random(B + longest)
    before = [rng.choice([0, longest, rng.randint(0, longest)]) for _ in range(B)]
    fresh = [rng.choice([0, 1, new, rng.randint(0, new)]) for _ in range(B)]
    need = sum(-(-(b + a) // page) + b // -page for b, a in zip(before, fresh))
    ids = list(range(B * cols + need + 10))
    rng.shuffle(ids)
    table = [[ids.pop() if j < -(-b // page) else -7 for j in range(cols)] for b in before]
    free = ids[:max(0, need + spare)]
    n = sum(fresh) + pad
    t, r = run_tables(before, fresh, table, free, page, n)
    want = tables_reference(before, fresh, table, free, page, n)
    assert t.tolist() == want[0]
    assert r.kv_lens.tolist() == want[1] and r.cu_seqlens_q.tolist() == want[2]
    assert r.positions.tolist() == want[3] and r.slots.tolist() == want[4] and r.pages_taken.tolist() == [want[5]]


def test_block_tables_row_stride_fewer_tokens_and_negative_lengths():
    wide = torch.full((2, 9), 5, dtype=torch.int32, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    r = sa.build_block_tables(torch.tensor([16, -3], **i32), torch.tensor([2, 17], **i32), wide[:, :4], torch.tensor([8, 9, 10], **i32), 16, 4)
    assert wide.tolist() == [[5, 8, 5, 5, 5, 5, 5, 5, 5], [9, 10, 5, 5, 5, 5, 5, 5, 5]]        # a negative length counts as none
    assert r.positions.tolist() == [16, 17, 0, 1] and r.slots.tolist() == [128, 129, 144, 145] and r.cu_seqlens_q.tolist() == [0, 2, 19]


# ------------------------------------------------------------------------------------------------ norm and rotation
def rope_reference(x, w, cos, sin, pos, eps, adjacent):
    """x [tokens, heads, D] -> (y, bound): fp32 arithmetic of under 40 rounded steps on the two products of a channel, then bf16."""
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    mag = x.abs()
    y = x.clone()
    if cos is not None:
        half = cos.shape[1]
        i = torch.arange(half)
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        m = x[..., a].abs() + x[..., b].abs()
        mag[..., a] = mag[..., b] = m
    return y, 2.0 ** -8 * y.abs() * 1.01 + 40 * 2.0 ** -24 * mag


def angles(places, rot, g):
    a = torch.rand(places, rot // 2, generator=g) * 6.3
    return a.cos(), a.sin()


@pytest.mark.parametrize("B,N,Hq,Hkv,D,rot,norm,adjacent,layout,pos", [
    (1, 1, 1, 1, 128, 128, True, False, "NHD", "given"), (1, 5, 32, 8, 128, 128, True, False, "NHD", "given64"), (2, 33, 9, 3, 64, 64, True, True, "HND", "given"),
    (3, 17, 5, 5, 96, 96, True, False, "NHD", "none"), (1, 40, 3, 1, 72, 72, True, False, "NHD", "given"), (2, 7, 17, 16, 80, 40, False, False, "HND", "given"),
    (1, 9, 2, 2, 8, 8, True, False, "NHD", "given"), (1, 9, 40, 4, 120, 120, False, True, "NHD", "given"), (1, 300, 7, 2, 128, 0, True, False, "NHD", "none"),
    (1, 6, 8, 1, 64, 8, True, False, "NHD", "given"), (2, 20, 4, 2, 128, 64, True, True, "NHD", "none")])
def test_norm_rope(B, N, Hq, Hkv, D, rot, norm, adjacent, layout, pos):
    g = gen(N + D + rot)
    # a slice of a fused projection: rows further apart than they are long
    x = normal(g, B, N, Hq + Hkv + 1, D) * 3
    q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv]
    places = 50 if pos != "none" else N
    cos, sin = angles(places, rot, g) if rot else (None, None)
    p = torch.randint(places, (B, N), generator=g, dtype=torch.int64 if pos == "given64" else torch.int32)
    if pos == "none":
        p = torch.arange(N).expand(B, N)
    qw, kw = (1 + 0.3 * normal(g, D), normal(g, D)) if norm else (None, None)
    xd = x.to(DEV)
    qd, kd = xd[:, :, :Hq], xd[:, :, Hq:Hq + Hkv]
    if layout == "HND":
        qd, kd = qd.transpose(1, 2), kd.transpose(1, 2)
    up = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got = sa.qk_norm_rope(qd, kd, up(cos), up(sin), up(p) if pos != "none" else None, up(qw), up(kw), eps=1e-5, adjacent_pairs=adjacent, tensor_layout=layout)
    for y, t, w in zip(got, (q, k), (qw, kw)):
        y = (y.transpose(1, 2) if layout == "HND" else y).cpu().double()
        for b in range(B):
            want, tol = rope_reference(t[b], w, cos, sin, p[b].long() if rot else None, 1e-5, adjacent)
            assert ((y[b] - want).abs() <= tol).all()
    # in place gives the same bits, and 3-D the same as a batch of one
    same = [t.clone() for t in got]
    res = sa.qk_norm_rope(qd, kd, up(cos), up(sin), up(p) if pos != "none" else None, up(qw), up(kw), eps=1e-5, adjacent_pairs=adjacent, tensor_layout=layout,
                          out=(qd, kd))
    assert res[0] is qd and torch.equal(qd, same[0]) and torch.equal(kd, same[1])
    if B == 1 and layout == "NHD":
        xd = x.to(DEV)
        a = sa.qk_norm_rope(xd[0, :, :Hq], xd[0, :, Hq:Hq + Hkv], up(cos), up(sin), up(p[0].contiguous()) if pos != "none" else None, up(qw), up(kw), eps=1e-5,
                            adjacent_pairs=adjacent)
        assert torch.equal(a[0], same[0][0]) and torch.equal(a[1], same[1][0])


def test_norm_rope_positions_outside_the_table_and_no_tokens():
    g = gen(1)
    q, k = normal(g, 4, 2, 64).to(DEV), normal(g, 4, 1, 64).to(DEV)
    cos, sin = (t.to(DEV) for t in angles(3, 32, g))
    y, _ = sa.qk_norm_rope(q, k, cos, sin, torch.tensor([0, 3, -1, 2], device=DEV))
    assert y[1:3, :, :32].isnan().all() and torch.equal(y[1:3, :, 32:], q[1:3, :, 32:]) and y[[0, 3]].isfinite().all()
    y, z = sa.qk_norm_rope(q[:0], k[:0], cos, sin)
    assert y.shape == (0, 2, 64) and z.shape == (0, 1, 64)


# ------------------------------------------------------------------------------------------------ into the cache and back
def odd_blocks(x, g):
    """Rows whose blocks meet the quantiser's borders: zeros, the largest and smallest numbers, ties between codes and between scales."""
    x = x.clone()
    flat = x.view(-1, 16) if x.shape[-1] % 16 == 0 else None
    if flat is not None and len(flat) >= 8:
        flat[0] = 0
        flat[1] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6]) * 7      # scale 7: reciprocal rounded
        flat[2] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6]) * 13
        flat[3] = 3e38
        flat[4] = 1e-30
        flat[5] *= 2.0 ** -9
        flat[6, 0] = 6 * 17 * 2.0 ** -3                        # a scale between two of E4M3
        flat[7] = 6 * 2.0 ** -10
    return x


@pytest.mark.parametrize("T,H,D,page,offset", [(1, 1, 128, 64, False), (1, 8, 128, 16, True), (37, 3, 64, 16, True), (130, 9, 64, 128, False), (200, 8, 128, 32, True),
                                               (50, 2, 96, 64, True), (50, 1, 72, 16, False), (33, 17, 8, 32, True)])
def test_append_and_read(T, H, D, page, offset):
    g = gen(T + D)
    x = odd_blocks(normal(g, T, 2 * H, D) * 2, g)
    k, v = x[:, :H], x[:, H:]
    off = normal(g, H, D) if offset else None
    pages = -(-T // page) + 2
    data = torch.randint(256, (pages, H, sa.FP4KVCache.page_bytes(D, page)), generator=g, dtype=torch.uint8)
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[T // 2:T // 2 + 1] = -1
    if T > 10:
        slots[3], slots[7] = pages * page, 2 ** 40
    want = data.numpy().copy()
    R.write(want, page, slots, k, v, off)
    xd = x.to(DEV)
    cache = sa.FP4KVCache(data.to(DEV), D, page, None if off is None else off.to(DEV))
    cache.append(xd[:, :H], xd[:, H:], slots.to(DEV))
    assert np.array_equal(cache.data.cpu().numpy(), want)      # and nothing else has changed
    kk, vv = R.values(want, D, page)
    rk, rv = (t.cpu() for t in cache.read(slots.to(DEV)))
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            a, b = kk[s // page, :, s % page], vv[s // page, :, s % page]
            if off is not None:
                # one rounding to bf16 of a sum that fp32 holds but for 2^-24 of its larger part
                tol = 2.0 ** -8 * np.abs(a + off.double().numpy()) + 2.0 ** -23 * np.abs(a)
                assert (np.abs(rk[i].double().numpy() - (a + off.double().numpy())) <= tol).all()
            else:
                assert np.array_equal(rk[i].double().numpy(), a)
            assert np.array_equal(rv[i].double().numpy(), b)
        else:
            assert not rk[i].any() and not rv[i].any()


def test_append_of_infinities_and_nan_stays_in_its_block():
    g = gen(5)
    k, v = normal(g, 4, 2, 64), normal(g, 4, 2, 64)
    k[1, 0, 3], v[2, 1, 17], v[3, 0, 40], k[0, 1, 16:32] = float("inf"), float("-inf"), float("nan"), float("nan")
    cache = sa.FP4KVCache.empty(1, 2, 64, 16)
    cache.append(k.to(DEV), v.to(DEV), torch.arange(4, device=DEV))
    rk, rv = (t.cpu() for t in cache.read(torch.arange(4, device=DEV)))
    assert rk[1, 0, 3] == 6 * 448 and rv[2, 1, 17] == -6 * 448      # saturated
    assert rk[0, 1, 16:32].isnan().all()
    clean = sa.FP4KVCache.empty(1, 2, 64, 16)
    k2, v2 = (torch.where(t.isfinite(), t, torch.zeros_like(t)) for t in (k, v))
    clean.append(k2.to(DEV), v2.to(DEV), torch.arange(4, device=DEV))
    ck, cv = (t.cpu() for t in clean.read(torch.arange(4, device=DEV)))
    for a, b, x in ((rk, ck, k), (rv, cv, v)):
        fine = x.view(4, 2, 4, 16).isfinite().all(-1, keepdim=True).expand(4, 2, 4, 16).reshape(4, 2, 64)
        assert torch.equal(a[fine], b[fine])


@pytest.mark.parametrize("T,Hq,H,D,rot,adjacent", [(1, 4, 1, 128, 128, False), (45, 32, 8, 128, 64, False), (100, 3, 3, 64, 64, True), (21, 10, 5, 96, 96, False)])
def test_norm_rope_append_is_both_steps(T, Hq, H, D, rot, adjacent):
    g = gen(T)
    x = normal(g, T, Hq + 2 * H, D).to(DEV)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    cos, sin = (t.to(DEV) for t in angles(64, rot, g))
    pos = torch.randint(64, (T,), generator=g).to(DEV)
    qw, kw, off = (normal(g, *s).to(DEV) for s in ((D,), (D,), (H, D)))
    slots = torch.randperm(256, generator=g)[:T].to(DEV)
    one, two = (sa.FP4KVCache(torch.zeros(4, H, sa.FP4KVCache.page_bytes(D, 64), dtype=torch.uint8, device=DEV), D, 64, off) for _ in range(2))
    got = sa.qk_norm_rope_append(q, k, v, one, slots, cos, sin, pos, qw, kw, adjacent_pairs=adjacent)
    a, b = sa.qk_norm_rope(q, k, cos, sin, pos, qw, kw, adjacent_pairs=adjacent)
    two.append(b, v, slots)
    assert torch.equal(got, a) and torch.equal(one.data, two.data)


# ------------------------------------------------------------------------------------------------ attention
def make_cache(g, kv_lens, H, D, page, offset=False, outlier=1.0):
    """A cache whose unwritten places hold arbitrary bytes and NaN scales, its table, and the data on the CPU."""
    pages = [-(-n // page) for n in kv_lens]
    total = sum(pages) + 2
    data = torch.randint(256, (total, H, sa.FP4KVCache.page_bytes(D, page)), generator=g, dtype=torch.uint8).to(DEV)
    data[torch.rand(data.shape, generator=g) < 0.1] = 0x7f
    off = normal(g, H, D).to(DEV) if offset else None
    cache = sa.FP4KVCache(data, D, page, off)
    ids = torch.randperm(total, generator=g)[:sum(pages)].tolist()
    cols = max(1, max(pages) + 1)
    table = torch.full((len(kv_lens), cols), -1, dtype=torch.int32)
    for b, n in enumerate(kv_lens):
        for j in range(pages[b]):
            table[b, j] = ids.pop()
        if n:
            slots = table[b, torch.arange(n) // page].long() * page + torch.arange(n) % page
            k = normal(g, n, H, D) * outlier
            cache.append((k + (off.cpu() if offset else 0)).to(BF).to(DEV), normal(g, n, H, D).to(DEV), slots.to(DEV))
    return cache, table


def check(q, cache, table, kv_lens, q_lens, **kw):
    """Calls the operator and compares out and LSE; returns them."""
    i32 = dict(dtype=torch.int32, device=DEV)
    cu = np.concatenate(([0], np.cumsum(q_lens)))
    plain = kw.pop("no_cu", False)
    args = dict(max_seqlen_q=max(q_lens)) if not plain else {}
    out, lse = sa.sageattn_kvcache(q, cache, table.to(DEV), torch.tensor(kv_lens, **i32), None if plain else torch.tensor(cu, **i32), return_lse=True, check_status=True,
                                   is_causal=kw.get("causal", True), sm_scale=kw.get("scale"), **args)
    alone = sa.sageattn_kvcache(q, cache, table.to(DEV), torch.tensor(kv_lens, **i32), None if plain else torch.tensor(cu, **i32),
                                is_causal=kw.get("causal", True), sm_scale=kw.get("scale"), **args)
    assert torch.equal(out[:cu[-1]], alone[:cu[-1]])           # the same bits without the LSE, and from call to call
    want, wl, tol, ltol = R.attend(q.cpu(), cache.data.cpu().numpy(), cache.head_dim, cache.page_size, table.tolist(), kv_lens, q_lens,
                                   k_offset=None if cache.k_offset is None else cache.k_offset.cpu(), **kw)
    got, gl = out.double().cpu().numpy()[:cu[-1]], lse.double().cpu().numpy()[:cu[-1]]
    want, wl, tol, ltol = want[:cu[-1]], wl[:cu[-1]], tol[:cu[-1]], ltol[:cu[-1]]
    empty = np.isneginf(wl)
    assert np.array_equal(np.isneginf(gl), empty) and not got[empty].any()
    worst = (np.abs(got - want)[~empty] / tol[~empty]).max() if (~empty).any() else 0
    assert worst <= 1, worst
    off = np.abs(gl[~empty] - wl[~empty]) / ltol[~empty]
    assert (off <= 1).all(), off.max()
    return out, lse


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("kv_lens,Hq,H,page", [
    ([1], 1, 1, 16), ([15, 16, 17, 31, 32, 33], 4, 1, 16), ([63, 64, 65, 127, 128, 129], 8, 2, 64), ([300, 1, 0, 777], 8, 1, 32), ([1500], 14, 2, 128),
    ([2049, 100], 16, 1, 64), ([513], 24, 1, 16), ([1000, 1000], 6, 6, 64)])
def test_one_token(kv_lens, Hq, H, page, D):
    g = gen(sum(kv_lens) + D)
    cache, table = make_cache(g, kv_lens, H, D, page, offset=len(kv_lens) % 2 == 0)
    q = normal(g, len(kv_lens), Hq, D).to(DEV)
    check(q, cache, table, kv_lens, [1] * len(kv_lens), no_cu=True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kv_lens,q_lens,Hq,H,D,page", [
    ([5, 40, 200], [5, 1, 3], 4, 2, 128, 16), ([100, 33, 64], [7, 0, 64], 2, 1, 64, 32), ([3, 0, 50], [9, 4, 20], 4, 1, 128, 64),
    ([260], [130], 4, 2, 128, 64), ([300, 17], [200, 17], 3, 1, 64, 16), ([700], [33], 7, 1, 128, 128), ([150, 90], [20, 90], 2, 2, 96, 32), ([64], [12], 1, 1, 8, 16),
    ([400, 260], [257, 129], 8, 2, 128, 64)])
def test_several_tokens(kv_lens, q_lens, Hq, H, D, page, causal):
    g = gen(sum(kv_lens) + sum(q_lens))
    cache, table = make_cache(g, kv_lens, H, D, page, offset=True)
    # heads further apart than they are long, and a padded batch
    q = normal(g, sum(q_lens) + 3, Hq + 2, D).to(DEV)[:, 1:1 + Hq]
    check(q, cache, table, kv_lens, q_lens, causal=causal)


@pytest.mark.parametrize("kv_lens,q_lens,Hq,H,D", [
    ([129, 0, 1000, 256], [1] * 4, 8, 2, 128), ([640], [1], 3, 1, 64), ([1153, 300], [6, 2], 4, 1, 128), ([2000, 90, 1], [5, 3, 4], 5, 1, 64),
    ([700, 1200], [8, 5], 4, 2, 64), ([1100], [4], 4, 1, 128), ([500, 700], [3, 1], 6, 2, 96), ([900], [2], 2, 1, 8), ([600, 5], [1, 1], 4, 4, 40)])
def test_keys_of_an_item_over_a_few_ctas(kv_lens, q_lens, Hq, H, D):
    """Two to eleven blocks of keys over two, four or eight CTAs, some of which then have none."""
    g = gen(sum(kv_lens) + Hq)
    cache, table = make_cache(g, kv_lens, H, D, 64, offset=True)
    check(normal(g, sum(q_lens), Hq, D).to(DEV), cache, table, kv_lens, q_lens)


@pytest.mark.parametrize("tokens,D", [(1, 128), (1, 64), (5, 128), (6, 64)])
def test_more_items_than_fit_at_once(tokens, D):
    g = gen(21 + tokens)
    kv_lens = torch.randint(400, (60,), generator=g).tolist()
    kv_lens[7] = 520
    cache, table = make_cache(g, kv_lens, 4, D, 16)
    q_lens = torch.randint(tokens + 1, (60,), generator=g).tolist() if tokens > 1 else [1] * 60
    q_lens[5] = tokens
    check(normal(g, sum(q_lens), 16, D).to(DEV), cache, table, kv_lens, q_lens)


@pytest.mark.parametrize("heads,tokens,keys,D", [(150, 33, 2100, 128), (151, 49, 2300, 64)])
def test_keys_of_the_last_round_are_split(heads, tokens, keys, D):
    """Two and three items more than the chip has SMs."""
    g = gen(heads)
    cache, table = make_cache(g, [keys], heads, D, 64, offset=True)
    check(normal(g, tokens, heads, D).to(DEV), cache, table, [keys], [tokens])


@pytest.mark.parametrize("tokens,D", [(2, 128), (5, 128), (6, 64), (8, 64)])
def test_long_rows_of_several_tokens(tokens, D):
    g = gen(31 + tokens)
    cache, table = make_cache(g, [9001, 130], 1, D, 128, offset=True)
    check(normal(g, 2 * tokens, 4, D).to(DEV), cache, table, [9001, 130], [tokens, tokens])


def test_many_ranges_of_keys():
    g = gen(9)
    kv_lens = [40001, 5, 20000]
    cache, table = make_cache(g, kv_lens, 1, 128, 64)
    check(normal(g, 3, 4, 128).to(DEV), cache, table, kv_lens, [1, 1, 1], no_cu=True)


@pytest.mark.parametrize("D,tokens", [(128, 1), (64, 6), (128, 150)])
def test_scales_of_scores_and_queries(D, tokens):
    """Large, small and very different queries of the rows of one tile: peaked and flat weights, and the power of two per row."""
    g = gen(11)
    cache, table = make_cache(g, [333], 1, D, 32, outlier=2.0)
    q = normal(g, tokens, 4, D) * torch.tensor([2.0 ** 4, 2.0 ** -30, 1.0, 0.0]).view(1, 4, 1).to(BF)
    check(q.to(DEV), cache, table, [333], [tokens])
    check(q.to(DEV), cache, table, [333], [tokens], scale=0.5)
    check((q * 2.0 ** -100).to(DEV), cache, table, [333], [tokens], scale=2.0 ** 90)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("tokens", [1, 5, 140])
def test_pages_that_are_not_in_the_cache(page, tokens):
    g = gen(13)
    cache, table = make_cache(g, [500, 200], 2, 128, page)
    table[0, 2], table[0, 4], table[1, 0] = -1, 10 ** 9, cache.num_pages
    table[1, 1:] = -1
    if page == 64:
        table[1, 1:] = -5
    check(normal(g, 2 * tokens, 4, 128).to(DEV), cache, table, [500, 200], [tokens, tokens])


@pytest.mark.parametrize("tokens,where", [(6, 60), (6, 63), (140, 150), (140, 230)])
def test_nan_among_unseen_keys_stays_out_of_rows(tokens, where):
    """A NaN value or key in the cache reaches the rows that see it and no others."""
    g = gen(17)
    n = tokens + 60 if tokens < 100 else tokens + 100
    for broken in "kv":
        cache, table = make_cache(g, [n], 1, 128, 32)
        q = normal(g, tokens, 4, 128).to(DEV)
        want = sa.sageattn_kvcache(q, cache, table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor([0, tokens], dtype=torch.int32, device=DEV), tokens)
        slot = table[0, where // 32].long() * 32 + where % 32
        k, v = cache.read(slot[None].to(DEV))
        (k if broken == "k" else v)[..., 16:32] = float("nan")
        cache.append(k, v, slot[None].to(DEV))
        got = sa.sageattn_kvcache(q, cache, table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor([0, tokens], dtype=torch.int32, device=DEV), tokens)
        first = where - (n - tokens)                           # the first row that sees it
        assert torch.equal(got[:max(first, 0)], want[:max(first, 0)])
        assert got[max(first, 0):, :, 16:32].isnan().all()


def test_rows_of_no_sequence_are_left_alone():
    g = gen(19)
    for q_lens in ([2, 3], [140, 3]):
        kv = [max(n, 100) for n in q_lens]
        cache, table = make_cache(g, kv, 2, 64, 16)
        T = sum(q_lens)
        q, out = normal(g, T + 4, 4, 64).to(DEV), torch.full((T + 4, 4, 64), 7.0, dtype=BF, device=DEV)
        cu = torch.tensor([0, q_lens[0], T], dtype=torch.int32, device=DEV)
        res = sa.sageattn_kvcache(q, cache, table.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV), cu, max_seqlen_q=max(q_lens), out=out)
        assert res is out and (out[T:] == 7).all() and (out[:T] != 7).any()


def test_a_cache_beyond_32_bits():
    """Pages whose bytes lie beyond 2^32, and a page number times its bytes beyond 2^31."""
    page, H, D = 128, 8, 128
    per = H * sa.FP4KVCache.page_bytes(D, page)
    pages = (2 ** 32 + 2 ** 28) // per + 2
    data = torch.empty(pages, H, per // H, dtype=torch.uint8, device=DEV)
    cache = sa.FP4KVCache(data, D, page)
    g = gen(23)
    ids = [pages - 1, 1, pages - 2, 2]
    small = sa.FP4KVCache.empty(4, H, D, page)
    k, v = normal(g, 500, H, D).to(DEV), normal(g, 500, H, D).to(DEV)
    place = torch.arange(500)
    far = (torch.tensor(ids)[place // page] * page + place % page).to(DEV)
    cache.append(k, v, far)
    small.append(k, v, place.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(cache.read(far), small.read(place.to(DEV))))
    lens = torch.tensor([500], dtype=torch.int32, device=DEV)
    for tokens in (1, 200):
        q, cu = normal(g, tokens, 16, D).to(DEV), torch.tensor([0, tokens], dtype=torch.int32, device=DEV)
        a = sa.sageattn_kvcache(q, cache, torch.tensor([ids], dtype=torch.int32, device=DEV), lens, cu, tokens)
        b = sa.sageattn_kvcache(q, small, torch.arange(4, dtype=torch.int32, device=DEV)[None], lens, cu, tokens)
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ a run of them, as a server makes it
def serve(steps, cache, g, Hq, H, D, B, cols, free):
    """Steps of B requests through the whole chain; -> per step (q, out), and the raw k, v of each request."""
    i32 = dict(dtype=torch.int32, device=DEV)
    lens, table = torch.zeros(B, **i32), torch.full((B, cols), -1, **i32)
    cos, sin = (t.to(DEV) for t in angles(512, D, g))
    kw, qw = normal(g, D).to(DEV), normal(g, D).to(DEV)
    ks, vs, res = [[] for _ in range(B)], [[] for _ in range(B)], []
    for new in steps:
        T = sum(new)
        t = sa.build_block_tables(lens, torch.tensor(new, **i32), table, free, cache.page_size, T + 2)
        x = normal(g, T + 2, Hq + 2 * H, D).to(DEV)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
        rq = sa.qk_norm_rope_append(q, k, v, cache, t.slots, cos, sin, t.positions, qw, kw)
        o = sa.sageattn_kvcache(rq, cache, table, t.kv_lens, t.cu_seqlens_q, max_seqlen_q=max(new))
        _, rk = sa.qk_norm_rope(q, k, cos, sin, t.positions, qw, kw)
        at = 0
        for b, n in enumerate(new):
            ks[b].append(rk[at:at + n])
            vs[b].append(v[at:at + n])
            at += n
        res.append((rq[:T], o[:T]))
        free = free[int(t.pages_taken):].contiguous()
        lens = t.kv_lens
    return res, [torch.cat(x) for x in ks], [torch.cat(x) for x in vs]


def test_serving_steps():
    """Prompts, then decoding and drafts: each step's attention equals that over a fresh cache with the same tokens, and is near attention
    over the unquantised ones."""
    Hq, H, D, B = 8, 2, 64, 3
    g = gen(29)
    cache = sa.FP4KVCache.empty(40, H, D, 16)
    steps = [[50, 7, 0], [1, 1, 130], [1, 1, 1], [4, 0, 2], [1, 16, 1]]
    res, ks, vs = serve(steps, cache, g, Hq, H, D, B, 12, torch.randperm(40, generator=g).to(torch.int32).to(DEV))
    lens = [0] * B
    for new, (q, o) in zip(steps, res):
        lens = [a + n for a, n in zip(lens, new)]
        fresh = sa.FP4KVCache.empty(40, H, D, 32)
        table, at = torch.full((B, 12), -1, dtype=torch.int32), 0
        for b in range(B):
            for j in range(-(-lens[b] // 32)):
                table[b, j] = at
                at += 1
            if lens[b]:
                place = torch.arange(lens[b])
                fresh.append(ks[b][:lens[b]], vs[b][:lens[b]], (table[b, place // 32].long() * 32 + place % 32).to(DEV))
        cu = torch.tensor(np.concatenate(([0], np.cumsum(new))), dtype=torch.int32, device=DEV)
        want = sa.sageattn_kvcache(q, fresh, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), cu, max_seqlen_q=max(new))
        # the same numbers, in chunks that may begin elsewhere: both within the bounds of _kv_reference, 2^-8 of the output above all
        assert torch.allclose(o.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
        at = 0
        for b, n in enumerate(new):
            if n:
                kf, vf = (x[b][:lens[b]].float().repeat_interleave(Hq // H, 1).transpose(0, 1) for x in (ks, vs))
                s = torch.matmul(q[at:at + n].float().transpose(0, 1), kf.transpose(1, 2)) * D ** -0.5
                s = s.masked_fill(torch.arange(lens[b], device=DEV) > torch.arange(lens[b] - n, lens[b], device=DEV)[:, None], float("-inf"))
                ref = torch.matmul(s.softmax(-1), vf).transpose(0, 1)
                assert torch.nn.functional.cosine_similarity(o[at:at + n].float().flatten(), ref.flatten(), 0) > 0.97
            at += n


def test_a_captured_step_replayed_on_another_stream():
    """A decoding step captured once: replays follow the contents of its buffers and give the bits of an eager call."""
    Hq, H, D, B, page = 8, 2, 128, 2, 16
    g = gen(31)
    i32 = dict(dtype=torch.int32, device=DEV)
    cache, table0 = make_cache(g, [70, 40], H, D, page)
    table = torch.full((B, 12), -1, **i32)
    table[:, :table0.shape[1]] = table0.to(DEV)
    more = torch.zeros(8, H, cache.data.shape[2], dtype=torch.uint8, device=DEV)
    cache = sa.FP4KVCache(torch.cat((cache.data, more)), D, page)
    free = torch.arange(cache.num_pages - 8, cache.num_pages, **i32)
    lens, new = torch.tensor([70, 40], **i32), torch.ones(B, **i32)
    x = normal(g, B, Hq + 2 * H, D).to(DEV)
    cos, sin = (t.to(DEV) for t in angles(512, D, g))

    def step():
        t = sa.build_block_tables(lens, new, table, free, page, B)
        q = sa.qk_norm_rope_append(x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:], cache, t.slots, cos, sin, t.positions)
        return sa.sageattn_kvcache(q, cache, table, t.kv_lens, t.cu_seqlens_q, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for _ in range(3):
        x.copy_(normal(g, B, Hq + 2 * H, D))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        got, gl = out.clone(), lse.clone()
        want, wl = step()
        assert torch.equal(got, want) and torch.equal(gl, wl)
        lens += 1


def test_two_calls_at_once():
    """The same call on two streams at a time: each has its own workspace."""
    g = gen(37)
    cache, table = make_cache(g, [9000, 8000], 2, 128, 64)
    q = normal(g, 2, 8, 128).to(DEV)
    table, lens = table.to(DEV), torch.tensor([9000, 8000], dtype=torch.int32, device=DEV)
    want = sa.sageattn_kvcache(q, cache, table, lens)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(sa.sageattn_kvcache(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_a_kept_attention_plan_does_not_let_another_tensor_through():
    g = gen(41)
    cache, table = make_cache(g, [40, 30], 1, 64, 16)
    i32 = dict(dtype=torch.int32, device=DEV)
    q, table, lens, cu = normal(g, 2, 2, 64).to(DEV), table.to(DEV), torch.tensor([40, 30], **i32), torch.tensor([0, 1, 2], **i32)
    want = sa.sageattn_kvcache(q, cache, table, lens, cu)
    assert torch.equal(sa.sageattn_kvcache(q, cache, table, lens), want)
    for kw in (dict(kv_lens=lens.long()), dict(kv_lens=lens.cpu()), dict(kv_lens=torch.zeros(4, **i32)[::2]), dict(cu_seqlens_q=cu.long()),
               dict(cu_seqlens_q=cu[:2]), dict(block_table=table.float()), dict(block_table=table.cpu())):
        with pytest.raises(ValueError):
            sa.sageattn_kvcache(**{**dict(q=q, cache=cache, block_table=table, kv_lens=lens, cu_seqlens_q=cu), **kw})


@pytest.mark.parametrize("tokens", [3, 70])
def test_nan_and_infinite_queries_stay_in_their_rows(tokens):
    g = gen(43)
    cache, table = make_cache(g, [300], 1, 128, 32)
    q = normal(g, tokens, 4, 128)
    bad = q.clone()
    bad[1, 2, 5], bad[2, 0, 100], bad[tokens - 1, 3] = float("nan"), float("inf"), float("-inf")
    i32 = dict(dtype=torch.int32, device=DEV)
    args = (cache, table.to(DEV), torch.tensor([300], **i32), torch.tensor([0, tokens], **i32), tokens)
    (a, al), (b, bl) = (sa.sageattn_kvcache(x.to(DEV), *args, return_lse=True) for x in (q, bad))
    hit = torch.zeros(tokens, 4, dtype=torch.bool)
    hit[1, 2] = hit[2, 0] = hit[tokens - 1, 3] = True
    assert a.isfinite().all() and b.cpu()[hit].isnan().all() and bl.cpu()[hit].isnan().all()
    want, _, tol, _ = R.attend(q, cache.data.cpu().numpy(), 128, 32, table.tolist(), [300], [tokens])
    off = np.abs(b.double().cpu().numpy() - want)[~hit.numpy()]
    assert (off <= tol[~hit.numpy()]).all()


def test_block_tables_without_free_pages_or_tokens():
    t, r = run_tables([5, 16], [3, 2], [[4, -1], [7, -1]], [], 16, 5)
    assert t.tolist() == [[4, -1], [7, -1]] and r.slots.tolist() == [69, 70, 71, -1, -1] and r.pages_taken.tolist() == [1]
    t, r = run_tables([5, 16], [0, 0], [[4, -1], [7, -1]], [], 16, 0)
    assert r.slots.numel() == r.positions.numel() == 0 and r.kv_lens.tolist() == [5, 16] and r.cu_seqlens_q.tolist() == [0, 0, 0]


def test_lengths_whose_sums_pass_32_bits():
    """Lengths that no cache can hold: the sums stop below 2^31, and every write stays in the table."""
    big = 2 ** 31 - 1
    i32 = dict(dtype=torch.int32, device=DEV)
    for before, new in (([0, 0, 0, 0], [big, big, big, 9]), ([big, 0, 7, 3], [big, 5, 1, 1]), ([0] * 40 + [3] * 3, [0] * 40 + [2 ** 30] * 3)):
        B = len(before)
        table = torch.full((B + 2, 8), 5, **i32)
        r = sa.build_block_tables(torch.tensor(before, **i32), torch.tensor(new, **i32), table[1:-1], torch.arange(4, **i32), 128, 100)
        fresh = [min(n, big - b) for b, n in zip(before, new)]
        assert r.kv_lens.tolist() == [b + n for b, n in zip(before, fresh)]
        assert r.cu_seqlens_q.tolist() == [min(sum(fresh[:i]), big) for i in range(B + 1)]
        assert r.pages_taken.item() == min(sum(-(-(b + n) // 128) + b // -128 for b, n in zip(before, fresh)), big)
        assert (table[0] == 5).all() and (table[-1] == 5).all()
        places = [b + t for b, n in zip(before, fresh) for t in range(min(n, 100))][:100]
        assert r.positions.tolist() == places + [0] * (100 - len(places))


def test_strides_of_single_rows_and_heads_say_nothing():
    g = gen(41)
    cache, table = make_cache(g, [50], 1, 64, 16)
    flat = normal(g, 1000).to(DEV)
    q = flat.as_strided((1, 3, 64), (77, 64, 1))
    want, lse = check(q, cache, table, [50], [1], no_cu=True)
    one = flat.as_strided((3, 1, 64), (64, 5, 1))
    k, v, slots = one, one, torch.arange(3, device=DEV)
    cache.append(k, v, slots)
    a, b = sa.qk_norm_rope(one, one.as_strided((3, 1, 64), (64, 3, 1)))
    assert torch.equal(a, one) and torch.equal(b, one)
    c = sa.qk_norm_rope(flat.as_strided((1, 3, 1, 64), (33, 64, 7, 1)), flat.as_strided((1, 3, 1, 64), (1, 64, 9, 1)))
    assert torch.equal(c[0][0], one) and torch.equal(c[1][0], one)


def test_one_plan_for_lengths_of_a_block_and_for_any_free_list():
    """Bounds that grow from step to step are held to, and so is each free list, though nothing is looked up anew."""
    g = gen(51)
    cache, table = make_cache(g, [300, 200], 2, 64, 16)
    q = normal(g, 2, 4, 64).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    lens, tab = torch.tensor([300, 200], **i32), table.to(DEV)
    for bound in (257, 258, 299, 300, 384, 200, 10 ** 6):
        n = [min(300, bound), min(200, bound)]
        a = sa.sageattn_kvcache(q, cache, tab, lens, max_seqlen_k=bound)
        b = sa.sageattn_kvcache(q, cache, tab, torch.tensor(n, **i32))
        want, _, tol, _ = R.attend(q.cpu(), cache.data.cpu().numpy(), 64, 16, table.tolist(), n, [1, 1])
        for x in (a, b):
            assert (np.abs(x.double().cpu().numpy() - want) <= tol).all()
    for free, tokens in (([7, 8, 9], 4), ([8], 4), ([], 5), ([5, 6, 7, 8], 3)):
        t = torch.full((1, 4), -7, **i32)
        r = sa.build_block_tables(torch.tensor([0], **i32), torch.tensor([3], **i32), t, torch.tensor(free, **i32), 16, tokens)
        page = free[0] if free else -1
        assert t.tolist() == [[page, -7, -7, -7]] and r.positions.tolist() == [0, 1, 2] + [0] * (tokens - 3)
        assert r.slots.tolist() == [page * 16 + i if free else -1 for i in range(3)] + [-1] * (tokens - 3)
