"""The 4-bit cache without a GPU: what is refused (every refusal comes before the check of the device), storage sizes, the C entry
points' checks of arguments, and the restated storage itself."""
import ctypes as C
import subprocess

import numpy as np
import pytest
import torch

import sageattention_b200 as sa
from sageattention_b200 import _lib
from tests import _kv_reference as R

BF = torch.bfloat16


def cache(pages=4, heads=2, D=64, page=16, **kw):
    return sa.FP4KVCache.empty(pages, heads, D, page, device="cpu", **kw)


def ints(*v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype)


@pytest.mark.parametrize("D,page,nbytes", [(64, 16, 1152), (128, 16, 2304), (128, 64, 9216), (96, 32, 4608), (8, 128, 9216)])
def test_page_bytes(D, page, nbytes):
    assert sa.FP4KVCache.page_bytes(D, page) == nbytes
    assert cache(D=D, page=page).data.shape == (4, 2, nbytes)


@pytest.mark.parametrize("DS", [64, 128])
def test_a_record_has_a_place_for_everything_once(DS):
    every = np.concatenate([o.ravel() for o in R.offsets(DS)])
    assert sorted(every.tolist()) == list(range(18 * DS))


def test_restated_quantiser_against_the_oracle():
    from oracle import nvfp4
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(3)).to(BF).double().numpy()
    code, scale = R.quantise(x)
    packed, sf = nvfp4.quantize_nvfp4(x.astype(np.float32))
    assert np.array_equal(sf, scale)
    # the operator's quantiser multiplies by a rounded reciprocal, which moves some quotients that lie on a border between codes
    other = np.stack((packed & 15, packed >> 4), -1).reshape(code.shape)
    y = np.abs(x.reshape(64, 8, 16) / R.E4M3[scale][..., None]).reshape(code.shape)
    on_border = np.isin(y, (R.E2M1[1:] + R.E2M1[:-1]) / 2)
    assert on_border.any() and (other == code)[~on_border].all()
    err = np.abs(np.where(code < 8, R.E2M1[code % 8], -R.E2M1[code % 8]).reshape(64, 8, 16) * R.E4M3[scale][..., None] - x.reshape(64, 8, 16))
    # half a step of the code grid where steps are widest (2), or what saturation at 6 leaves of a scale rounded down by 2^-4
    assert (err <= R.E4M3[scale][..., None] * 1.0001).all()


@pytest.mark.parametrize("make,match", [
    (lambda: cache(page=48), "page_size"),
    (lambda: cache(D=136), "head_dim"),
    (lambda: cache(D=60), "head_dim"),
    (lambda: sa.FP4KVCache(torch.zeros(4, 2, 1152), 64, 16), "uint8"),
    (lambda: sa.FP4KVCache(torch.zeros(4, 2, 1150, dtype=torch.uint8), 64, 16), "bytes"),
    (lambda: sa.FP4KVCache(torch.zeros(2, 4, 1152, dtype=torch.uint8).transpose(0, 1), 64, 16), "contiguous"),
    (lambda: sa.FP4KVCache(torch.zeros(0, 2, 1152, dtype=torch.uint8), 64, 16), "pages"),
    (lambda: sa.FP4KVCache(torch.zeros(4 * 2 * 1152 + 1, dtype=torch.uint8)[1:].view(4, 2, 1152), 64, 16), "16-byte"),
    (lambda: cache(k_offset=torch.zeros(2, 32, dtype=BF)), "k_offset"),
])
def test_cache_refusals(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def tokens(T=3, H=2, D=64, dtype=BF):
    return torch.zeros(T, H, D, dtype=dtype)


@pytest.mark.parametrize("k,v,slots,exc,match", [
    (tokens(), tokens(), ints(0, 1, 2), ValueError, "slots must be torch.int64"),
    (tokens(), tokens(), ints(0, 1, dtype=torch.int64), ValueError, "slots must have shape"),
    (tokens(H=3), tokens(H=3), ints(0, 1, 2, dtype=torch.int64), ValueError, "k and v must be"),
    (tokens(), tokens(T=4), ints(0, 1, 2, dtype=torch.int64), ValueError, "k and v must be"),
    (tokens(dtype=torch.float16), tokens(), ints(0, 1, 2, dtype=torch.int64), AssertionError, "bfloat16"),
    (torch.zeros(3, 64, 2, dtype=BF).transpose(1, 2), tokens(), ints(0, 1, 2, dtype=torch.int64), ValueError, "contiguous"),
    (torch.zeros(3, 2, 68, dtype=BF)[..., :64], tokens(), ints(0, 1, 2, dtype=torch.int64), ValueError, "16-byte"),
    (tokens(), tokens(), ints(0, 1, 2, dtype=torch.int64), ValueError, "CUDA tensors only"),
])
def test_append_refusals(k, v, slots, exc, match):
    with pytest.raises(exc, match=match):
        cache().append(k, v, slots)


def test_read_refusals():
    with pytest.raises(ValueError, match="int64"):
        cache().read(ints(0))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        cache().read(ints(0, dtype=torch.int64))


def rope_args(**kw):
    a = dict(q=tokens(H=4), k=tokens(), cos=torch.ones(8, 32), sin=torch.zeros(8, 32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,exc,match", [
    (dict(q=tokens(T=4, H=4)), ValueError, "shapes"),
    (dict(q=tokens(H=4, D=32)), ValueError, "shapes"),
    (dict(q=tokens(H=4, dtype=torch.float32)), AssertionError, "bfloat16"),
    (dict(q=tokens(H=4, D=68), k=tokens(D=68)), ValueError, "head_dim"),
    (dict(q=tokens(H=4, D=136), k=tokens(D=136)), ValueError, "head_dim"),
    (dict(q=tokens()[0], k=tokens()[0]), ValueError, "4-D"),
    (dict(q=tokens()[None], k=tokens()[None], tensor_layout="DHN"), ValueError, "layout"),
    (dict(sin=None), ValueError, "together"),
    (dict(cos=torch.ones(8, 34), sin=torch.ones(8, 34)), ValueError, "rotated"),
    (dict(cos=torch.ones(8, 6), sin=torch.ones(8, 6)), ValueError, "rotated"),
    (dict(cos=torch.ones(8, 32, dtype=BF)), ValueError, "cos must be torch.float32"),
    (dict(sin=torch.ones(7, 32)), ValueError, "sin must have shape"),
    (dict(positions=ints(0, 1, 2, dtype=torch.int16)), ValueError, "positions"),
    (dict(positions=ints(0, 1)), ValueError, "positions must have shape"),
    (dict(q_weight=torch.ones(32, dtype=BF)), ValueError, "q_weight"),
    (dict(k_weight=torch.ones(64)), ValueError, "k_weight"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(), ValueError, "CUDA tensors only"),
])
def test_norm_rope_refusals(kw, exc, match):
    with pytest.raises(exc, match=match):
        sa.qk_norm_rope(**rope_args(**kw))


def test_norm_rope_append_refusals():
    slots = ints(0, 1, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="q must be"):
        sa.qk_norm_rope_append(tokens()[None], tokens()[None], tokens(), cache(), slots)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        sa.qk_norm_rope_append(tokens(H=4), tokens(), tokens(), cache(), slots)


def table_args(**kw):
    a = dict(lens_before=ints(3, 4), lens_new=ints(1, 1), block_table=torch.zeros(2, 4, dtype=torch.int32), free_pages=ints(5, 6), page_size=16, num_tokens=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(lens_before=ints(3, 4, dtype=torch.int64)), "lens_before must be torch.int32"),
    (dict(lens_new=ints(1)), "lens_new must have shape"),
    (dict(page_size=20), "page_size"),
    (dict(num_tokens=-1), "num_tokens"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 4)), "block_table"),
    (dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()), "rows of block_table"),
    (dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), "overlap"),
    (dict(free_pages=torch.zeros(2, 2, dtype=torch.int32)), "free_pages"),
    (dict(lens_before=torch.zeros(16385, dtype=torch.int32), lens_new=torch.zeros(16385, dtype=torch.int32)), "16384"),
    (dict(), "CUDA tensors only"),
])
def test_block_table_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        sa.build_block_tables(**table_args(**kw))


def attention_args(**kw):
    a = dict(q=tokens(T=2, H=4), cache=cache(), block_table=torch.zeros(2, 1, dtype=torch.int32), kv_lens=ints(3, 4))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,exc,match", [
    (dict(q=tokens(T=2, H=3)), ValueError, "num_qo_heads"),
    (dict(q=tokens(T=2, H=4, D=128)), ValueError, "q must be"),
    (dict(q=tokens(T=1, H=4)), ValueError, "a row for each sequence"),
    (dict(q=tokens(T=2, H=4, dtype=torch.float16)), AssertionError, "bfloat16"),
    (dict(kv_lens=ints(3, 4, dtype=torch.int64)), ValueError, "kv_lens"),
    (dict(cu_seqlens_q=ints(0, 1)), ValueError, "cu_seqlens_q must have shape"),
    (dict(cu_seqlens_q=ints(0, 1, 2), max_seqlen_q=0), ValueError, "max_seqlen_q"),
    (dict(max_seqlen_k=0), ValueError, "max_seqlen_k"),
    (dict(block_table=torch.zeros(1, 1, dtype=torch.int32)), ValueError, "block_table"),
    (dict(sm_scale=-0.1), ValueError, "sm_scale"),
    (dict(out=tokens(T=2, H=2)), ValueError, "outputs must have"),
    (dict(), ValueError, "CUDA tensors only"),
])
def test_attention_refusals(kw, exc, match):
    with pytest.raises(exc, match=match):
        sa.sageattn_kvcache(**attention_args(**kw))


def test_struct_layouts(tmp_path):
    pairs = {"sage3_kv_cache": _lib.KvCache, "sage3_kv_tables_args": _lib.KvTablesArgs, "sage3_kv_tokens_args": _lib.KvTokensArgs,
             "sage3_kv_attention_args": _lib.KvAttentionArgs}
    from tests.test_cabi_cpu import HEADER
    lines = "".join(
        f'  printf("%zu{" %zu" * len(c._fields_)}\\n", sizeof({n}), ' + ", ".join(f"offsetof({n}, {f[0]})" for f in c._fields_) + ");\n" for n, c in pairs.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "sage3_b200.h"\nint main(void) {\n' + lines + "  return 0;\n}\n")
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, cls in zip(got, pairs.values()):
        assert [int(x) for x in line.split()] == [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_], cls


def test_c_entry_points_check_arguments():
    """Nothing reaches the device: every one of these is refused by its sizes or pointers."""
    lib = _lib.load()
    A, U = _lib.ERR_ARGUMENT, _lib.ERR_UNSUPPORTED
    assert lib.sage3_kv_block_tables(None, None) == A
    assert lib.sage3_kv_tokens(None, None) == A
    assert lib.sage3_kv_attention(None, None) == A
    assert lib.sage3_kv_read(None, None, 1, None, None, None) == A
    one = 1 << 12                                              # an address that is never dereferenced

    def kv(**kw):
        c = _lib.KvCache(one, 4, 2, 16, 64, 64, None)
        for n, x in kw.items():
            setattr(c, n, x)
        return c

    for bad, want in ((dict(data=None), A), (dict(data=one + 8), A), (dict(num_pages=0), A), (dict(page_size=24), U), (dict(head_dim=60), U),
                      (dict(head_dim=72), U), (dict(head_dim_stored=96), U), (dict(k_offset=one + 2), A)):
        c = kv(**bad)
        assert lib.sage3_kv_read(C.byref(c), one, 1, one, one, None) == want, bad
    c = kv()
    assert lib.sage3_kv_read(C.byref(c), one, -1, one, one, None) == A
    assert lib.sage3_kv_read(C.byref(c), one, 0, None, None, None) == _lib.OK
    assert lib.sage3_kv_read(C.byref(c), one, 1, one + 8, one, None) == A

    def tok(**kw):
        a = _lib.KvTokensArgs()
        a.B, a.N, a.Hq, a.Hkv, a.D = 1, 1, 0, 2, 64
        a.k = a.v = _lib.Tensor(one, 0, 64, 128)
        a.cache, a.slots = C.pointer(c), one
        for n, x in kw.items():
            setattr(a, n, x)
        return lib.sage3_kv_tokens(C.byref(a), None)

    for bad, want in ((dict(D=60), U), (dict(D=136), U), (dict(Hkv=0), A), (dict(Hkv=3), A), (dict(Hq=1), A), (dict(slots=None), A), (dict(cache=None), A),
                      (dict(v=_lib.Tensor(None, 0, 0, 0)), A), (dict(k=_lib.Tensor(one, 0, 60, 128)), A), (dict(rot_dim=4), U), (dict(rot_dim=72), U),
                      (dict(rot_dim=64), A), (dict(k_weight=one, eps=-1.0), A), (dict(k_weight=one + 2), A)):
        assert tok(**bad) == want, bad
    assert tok(N=0) == _lib.OK

    def att(**kw):
        a = _lib.KvAttentionArgs(C.pointer(c), 1, 4, 1, 16, 1, one, 256, 64, one, 256, 64, None, None, one, one, 1, 1, 1, 0.0, one, 1 << 30)
        for n, x in kw.items():
            setattr(a, n, x)
        return lib.sage3_kv_attention(C.byref(a), None)

    for bad, want in ((dict(Hq=3), U), (dict(B=0), A), (dict(max_seqlen_k=0), A), (dict(columns=0), A), (dict(q=None), A), (dict(q=one + 2), A), (dict(kv_lens=None), A),
                      (dict(q_stride_n=250), A), (dict(workspace=one + 16), A), (dict(total_q=0), _lib.OK), (dict(B=2), A), (dict(cu_seqlens_q=one, max_seqlen_q=1 << 30), U)):
        assert att(**bad) == want, bad
    t = _lib.KvTablesArgs(one, one, one, one, 4, 2, 4, 1, 16, 2, one, one, one, one, one)
    for n, x, want in (("B", 0, A), ("B", 20000, U), ("columns", 5, A), ("page_size", 17, U), ("num_free", -1, A), ("free_pages", None, A), ("slots", None, A)):
        keep = getattr(t, n)
        setattr(t, n, x)
        assert lib.sage3_kv_block_tables(C.byref(t), None) == want, n
        setattr(t, n, keep)


def test_a_kept_plan_does_not_let_another_tensor_through(monkeypatch):
    """Types, shapes and layouts are looked at in every call, also where an earlier one with the same sizes was right."""
    from sageattention_b200 import kv_cache
    calls = []
    monkeypatch.setattr(kv_cache, "_check_device", lambda t: None)
    monkeypatch.setattr(kv_cache, "_run", lambda fn, struct, device, where: calls.append(where))
    monkeypatch.setattr(kv_cache, "_plans", {})
    monkeypatch.setattr(kv_cache, "_keep_plan", lambda key, plan: kv_cache._plans.setdefault(key, plan))
    c = cache()
    slots = ints(0, 1, 2, dtype=torch.int64)
    good = rope_args(positions=ints(0, 1, 2), q_weight=torch.ones(64, dtype=BF), k_weight=torch.ones(64, dtype=BF))
    bad = [dict(cos=torch.ones(8, 32, dtype=torch.float64)), dict(sin=torch.zeros(8, 64)[:, ::2]), dict(sin=None), dict(positions=ints(0, 1)),
           dict(positions=torch.zeros(6, dtype=torch.int32)[::2]), dict(q_weight=torch.ones(64)), dict(k_weight=torch.ones(128, dtype=BF)[::2]),
           dict(k_weight=torch.ones(32, dtype=BF))]
    sa.qk_norm_rope(**good)
    sa.qk_norm_rope_append(v=tokens(), cache=c, slots=slots, **good)
    c.append(tokens(), tokens(), slots)
    sa.build_block_tables(**table_args())
    assert len(calls) == 4
    for kw in bad:
        with pytest.raises(ValueError):
            sa.qk_norm_rope(**{**good, **kw})
        with pytest.raises(ValueError):
            sa.qk_norm_rope_append(v=tokens(), cache=c, slots=slots, **{**good, **kw})
    for s in (slots.int(), ints(0, 1, dtype=torch.int64), torch.zeros(6, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="slots"):
            sa.qk_norm_rope_append(v=tokens(), cache=c, slots=s, **good)
        with pytest.raises(ValueError, match="slots"):
            c.append(tokens(), tokens(), s)
    for kw in (dict(lens_new=ints(1, 1, dtype=torch.int64)), dict(lens_new=ints(1)), dict(free_pages=torch.zeros(4, dtype=torch.int32)[::2]),
               dict(block_table=torch.zeros(2, 4))):
        with pytest.raises(ValueError):
            sa.build_block_tables(**table_args(**kw))
    assert len(calls) == 4


def test_a_cache_keeps_its_tensors():
    c = cache()
    with pytest.raises(AttributeError):
        c.data = torch.zeros_like(c.data)
    with pytest.raises(AttributeError):
        c.k_offset = None


@pytest.mark.parametrize("kw,match", [
    (dict(max_seqlen_q=torch.tensor(2)), "not a tensor"), (dict(max_seqlen_k=torch.tensor(20)), "not a tensor"), (dict(sm_scale=torch.tensor(0.5)), "not a tensor"),
    (dict(sm_scale=1e-50), "sm_scale"), (dict(sm_scale=1e60), "sm_scale"), (dict(sm_scale=float("nan")), "sm_scale")])
def test_attention_numbers(kw, match):
    with pytest.raises(ValueError, match=match):
        sa.sageattn_kvcache(**attention_args(**kw))


def test_queries_beyond_the_grid():
    with pytest.raises(ValueError, match="too many"):
        sa.sageattn_kvcache(**attention_args(cu_seqlens_q=ints(0, 1, 2), max_seqlen_q=2 ** 30))


def test_a_table_of_more_keys_than_32_bits_count():
    wide = torch.zeros(attention_args()["block_table"].shape[0], 2 ** 26 + 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="too many"):
        sa.sageattn_kvcache(**attention_args(block_table=wide))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        sa.sageattn_kvcache(**attention_args(block_table=wide, max_seqlen_k=100))


def test_numbers_of_tables_and_rotation():
    with pytest.raises(ValueError, match="not a tensor"):
        sa.build_block_tables(**table_args(num_tokens=torch.tensor(3)))
    with pytest.raises(ValueError, match="not a tensor"):
        sa.qk_norm_rope(**rope_args(eps=torch.tensor(1e-6)))


def test_reading_more_tokens_than_the_kernel_counts():
    """Token numbers of the last, partly filled CTA must not pass 2^31."""
    c = _lib.KvCache(1 << 12, 4, 2, 16, 64, 64, None)
    for T in (2 ** 31 - 64, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
        assert _lib.load().sage3_kv_read(C.byref(c), 1 << 12, T, 1 << 12, 1 << 12, None) == _lib.ERR_UNSUPPORTED, T
    meta = sa.FP4KVCache.empty(4, 2, 64, 16, device="meta")
    with pytest.raises(ValueError, match="too many"):
        meta.read(torch.empty(2 ** 31 - 64, dtype=torch.int64, device="meta"))


def test_outputs_whose_elements_lie_on_one_another():
    wide = torch.zeros(3, 1, 64, dtype=BF).expand(3, 4, 64)
    steps = torch.zeros(512, dtype=BF).as_strided((3, 4, 64), (64, 8, 1))
    for bad in (wide, steps, torch.zeros(1, 4, 64, dtype=BF).expand(3, 4, 64)):
        with pytest.raises(ValueError, match="on one another"):
            sa.qk_norm_rope(**rope_args(out=(bad, tokens())))
        with pytest.raises(ValueError, match="on one another"):
            sa.qk_norm_rope_append(tokens(H=4), tokens(), tokens(), cache(), ints(0, 1, 2, dtype=torch.int64), out=bad)
        with pytest.raises(ValueError, match="on one another"):
            sa.sageattn_kvcache(**attention_args(q=tokens(T=3, H=4), out=bad))
    # slices, other orders of dimensions and dimensions of one are fine: the device is looked at next
    for good in (torch.zeros(3, 9, 80, dtype=BF)[:, 2:6, :64], torch.zeros(4, 3, 64, dtype=BF).transpose(0, 1)):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            sa.qk_norm_rope(**rope_args(out=(good, tokens())))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        sa.qk_norm_rope(**rope_args(q=tokens(T=1, H=1), k=tokens(T=1), out=(torch.zeros(64, dtype=BF).as_strided((1, 1, 64), (0, 0, 1)), tokens(T=1))))
