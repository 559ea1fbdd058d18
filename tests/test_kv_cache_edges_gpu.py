"""The 4-bit cache at its edges: lengths beyond what tables, bounds and outputs hold, the most requests, numbers that are none."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import sageattention_b200 as sa
from tests import _kv_reference as R
from tests.test_kv_cache_gpu import BF, DEV, check, gen, make_cache, normal

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("tokens,before", [(6, 200), (6, 9001), (150, 70), (150, 1300)])
@pytest.mark.parametrize("what", ["columns", "max_seqlen_k", "max_seqlen_q", "rows of q"])
def test_what_does_not_fit_is_left_out_and_moves_no_row(what, tokens, before, D):
    """Keys beyond the table's columns or max_seqlen_k, and rows beyond max_seqlen_q or q, are not there; a row that is sees its own
    place's keys as ever.  The reference takes each row as a sequence of its own."""
    g = gen(tokens + before + D)
    kv_lens, q_lens = [before + tokens, tokens, before // 2 + tokens], [tokens, tokens, tokens - 1]      # (the second: a prompt)
    cache, table = make_cache(g, kv_lens, 2, D, 16, offset=True)
    T, rows, max_q, keys = sum(q_lens), sum(q_lens), tokens, 16 * table.shape[1]
    if what == "columns":
        table = table[:, :(tokens // 2 if before < 100 else before + tokens // 2) // 16].contiguous()
        keys = 16 * table.shape[1]
    elif what == "max_seqlen_k":
        keys = tokens // 2 + 1 if before < 100 else before + tokens // 2 - 3
    elif what == "max_seqlen_q":
        max_q = tokens - 2
    else:
        rows = T - 3
    q = normal(g, rows, 4, D)
    out = torch.full((rows, 4, D), 7.0, dtype=BF, device=DEV)
    starts = np.concatenate(([0], np.cumsum(q_lens)))
    got, lse = sa.sageattn_kvcache(q.to(DEV), cache, table.to(DEV), torch.tensor(kv_lens, **I32), torch.tensor(starts, **I32), max_q, keys,
                                   return_lse=True, out=out, check_status=True)
    owner = [b for b, n in enumerate(q_lens) for _ in range(n)][:rows]
    place = [t for n in q_lens for t in range(n)][:rows]
    there = np.array([t < max_q for t in place])
    sees = [max(0, min(keys, kv_lens[b] - q_lens[b] + t + 1)) for b, t in zip(owner, place)]
    want, wl, tol, ltol = R.attend(q, cache.data.cpu().numpy(), D, 16, [table[b].tolist() for b in owner], sees, [1] * rows, k_offset=cache.k_offset.cpu())
    o, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    assert (o[~there] == 7).all()
    o, l, want, wl, tol, ltol = (x[there] for x in (o, l, want, wl, tol, ltol))
    assert (np.abs(o - want) <= tol).all()
    assert np.array_equal(np.isneginf(l), np.isneginf(wl)) and (np.abs(l - wl)[np.isfinite(wl)] <= ltol[np.isfinite(wl)]).all()


SHARED = """
import torch, sageattention_b200 as sa
from concurrent.futures import ThreadPoolExecutor
i32 = dict(dtype=torch.int32, device="cuda")

def one(B):
    new = torch.arange(B, **i32) % 3
    r = sa.build_block_tables(torch.zeros(B, **i32), new, torch.full((B, 1), -1, **i32), torch.arange(B, **i32), 16, 4)
    want = torch.cat((new.new_zeros(1), new.cumsum(0)))
    assert torch.equal(r.cu_seqlens_q.long(), want), B

for B in (6135, 6136, 6143, 6144, 6136, 16384, 6136):          # no larger one before the first four
    one(B)
with ThreadPoolExecutor(2) as pool:
    list(pool.map(one, [16384, 6200] * 200))
torch.cuda.synchronize()
print("fine")
"""


def test_block_tables_of_as_many_requests_as_shared_memory_holds():
    """In a process of its own: what the kernel may use is set once."""
    r = subprocess.run([sys.executable, "-c", SHARED], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("D", [128, 64, 72, 8])
def test_a_lone_nan_marks_its_block(D):
    """One NaN among finite channels (and beside the padding of a head dim that is no multiple of 16): the block reads back as NaN, and
    all others as they would without it."""
    g = gen(61 + D)
    T, H = 40, 2
    k, v = normal(g, T, H, D), normal(g, T, H, D)
    hit = torch.zeros(2, T, H, D, dtype=torch.bool)
    for i in range(T // 2):                                    # every channel in turn, and two in one block
        hit[i % 2, 2 * i, i % H, (7 * i) % D] = True
    hit[0, 1, 0, D - 1] = hit[0, 1, 0, D - 3] = True
    bad = [torch.where(h, torch.full_like(x, float("nan")), x) for h, x in zip(hit, (k, v))]
    slots = torch.randperm(64, generator=g)[:T].to(DEV)
    got, clean = [], []
    for res, (a, b) in ((got, bad), (clean, (k, v))):
        cache = sa.FP4KVCache.empty(4, H, D, 16)
        cache.append(a.to(DEV), b.to(DEV), slots)
        res += [t.cpu() for t in cache.read(slots)]
        fused = sa.FP4KVCache.empty(4, H, D, 16)               # the kernel with queries writes the same
        sa.qk_norm_rope_append(a[:, :1].to(DEV), a.to(DEV), b.to(DEV), fused, slots)
        assert all(torch.equal(x.nan_to_num(7e4), y.nan_to_num(7e4)) for x, y in zip((t.cpu() for t in fused.read(slots)), res[-2:]))
    for x, y, h in zip(got, clean, hit):
        pad = -D % 16
        block = torch.nn.functional.pad(h, (0, pad)).unflatten(-1, (-1, 16)).any(-1, keepdim=True).expand(T, H, (D + pad) // 16, 16).flatten(-2)[..., :D]
        assert x[block].isnan().all() and torch.equal(x[~block], y[~block])


@pytest.mark.parametrize("rot", [8, 24, 64])
def test_keys_of_positions_outside_the_table_are_nan(rot):
    """Also where the rotated channels end in the middle of a block."""
    g = gen(rot)
    q, k, v = normal(g, 4, 2, 64).to(DEV), normal(g, 4, 1, 64).to(DEV), normal(g, 4, 1, 64).to(DEV)
    cos, sin = torch.ones(3, rot // 2, device=DEV), torch.zeros(3, rot // 2, device=DEV)
    cache, slots = sa.FP4KVCache.empty(1, 1, 64, 16), torch.arange(4, device=DEV)
    sa.qk_norm_rope_append(q, k, v, cache, slots, cos, sin, torch.tensor([0, 3, 2, -1], device=DEV))
    rk, rv = cache.read(slots)
    end = -(-rot // 16) * 16
    assert rk[[1, 3], :, :end].isnan().all() and rk[[1, 3], :, end:].isfinite().all() and rk[[0, 2]].isfinite().all() and rv.isfinite().all()
    lens = torch.tensor([1, 2], **I32)
    o = sa.sageattn_kvcache(q[:2], cache, torch.zeros(2, 1, **I32), lens)
    assert o[0].isfinite().all() and o[1].isnan().all()


@pytest.mark.parametrize("D,heads,adjacent", [(128, 40, True), (64, 40, False), (128, 9, False)])
def test_norm_rope_in_place_over_many_rows(D, heads, adjacent):
    """A warp goes over a token's heads a few at a time, in a fused projection's own memory."""
    g = gen(D + heads)
    x = normal(g, 5000, 2 * heads + 1, D).to(DEV)
    cos, sin = (torch.randn(5000, D // 2, generator=g).to(DEV) for _ in range(2))
    w = normal(g, D).to(DEV)
    q, k, rest = x[:, :heads], x[:, heads:2 * heads], x[:, 2 * heads:].clone()
    want = sa.qk_norm_rope(q, k, cos, sin, None, w, w, adjacent_pairs=adjacent)
    got = sa.qk_norm_rope(q, k, cos, sin, None, w, w, adjacent_pairs=adjacent, out=(q, k))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is q and torch.equal(x[:, 2 * heads:], rest)


@pytest.mark.parametrize("D,tokens", [(64, 1), (128, 5), (64, 7), (128, 140)])
def test_outputs_of_the_callers_own(D, tokens):
    """Rows and heads further apart than they are long, in another order too: the bits of a call without ``out``, and nothing between them."""
    g = gen(71 + tokens)
    kv_lens, q_lens = [tokens + 300, tokens, 2500], [tokens, max(1, tokens - 1), tokens]
    cache, table = make_cache(g, kv_lens, 2, D, 32)
    T = sum(q_lens)
    q, cu = normal(g, T + 2, 4, D).to(DEV), torch.tensor(np.concatenate(([0], np.cumsum(q_lens))), **I32)
    args = (cache, table.to(DEV), torch.tensor(kv_lens, **I32), cu, tokens)
    want, lse = sa.sageattn_kvcache(q, *args, return_lse=True)
    for order in (False, True):
        wide = torch.full((T + 2, 9, D + 24) if not order else (9, T + 2, D + 24), 7.0, dtype=BF, device=DEV)
        inner = wide[:, 1:9:2, 8:D + 8] if not order else wide[1:9:2, :, 8:D + 8].transpose(0, 1)
        got, l2 = sa.sageattn_kvcache(q, *args, return_lse=True, out=inner)
        assert got is inner and torch.equal(inner[:T], want[:T]) and torch.equal(l2[:T], lse[:T])
        inner[:T] = 7
        assert (wide == 7).all()


@pytest.mark.parametrize("D,tokens", [(128, 1), (64, 6), (128, 60)])
def test_scores_as_large_as_they_may_be(D, tokens):
    """Scores near 9e7: the rounding of a maximum's product with the scale, 8 and more there, still leaves weights within fp16."""
    g = gen(73)
    cache, table = make_cache(g, [700], 1, D, 32, outlier=8.0)
    q = normal(g, tokens, 2, D) * 2.0 ** 17
    kk, _ = R.values(cache.data.cpu().numpy(), D, 32)
    keys = kk[table[0, torch.arange(700) // 32].numpy(), 0, np.arange(700) % 32]
    for size in (1e5, 1e7, 8.5e7):
        scale = size / np.abs(q.double().numpy() @ keys.T).max()
        out, lse = check(q.to(DEV), cache, table, [700], [tokens], scale=scale)
        assert out.isfinite().all() and lse.isfinite().all()
