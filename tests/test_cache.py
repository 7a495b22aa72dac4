"""The 4-bit cache without a GPU: refusals on the host, the operators' shapes
on meta tensors, and the format's definition itself."""
import ctypes

import pytest
import torch

import splash_attention as sa
from splash_attention import _lib, cache as cm

import _cache as ref


def host_cache(pages=4, heads=2, d=64, page=16):
    """A cache object over CPU tensors, for checks that never launch."""
    c = cm.QuantizedKVCache.__new__(cm.QuantizedKVCache)
    G = -(-d // 32)
    mk = lambda tail, dt: torch.zeros((pages, heads, page) + tail, dtype=dt)  # noqa: E731
    c._hold(cm.QuantizedKVCache._describe(pages, heads, d, page), mk((16 * G,), torch.uint8),
            mk((G, 2), torch.bfloat16), mk((16 * G,), torch.uint8), mk((G, 2), torch.bfloat16))
    return c


def test_exports():
    assert sa.QuantizedKVCache is cm.QuantizedKVCache and sa.cache_attention is cm.cache_attention
    for n in ("cache_write", "cache_read", "cache_attention"):
        assert hasattr(torch.ops.adasplash, n)


@pytest.mark.parametrize("args,err,msg", [
    ((0, 2, 64, 64), ValueError, "num_pages"),
    ((4, 0, 64, 64), ValueError, "kv_heads"),
    ((4, 2, 129, 64), RuntimeError, "Head dimension too large"),
    ((4, 2, 0, 64), ValueError, "head dimension"),
    ((4, 2, 64, 48), ValueError, "page_size"),
    ((4, 2, 64, 64, "cpu"), RuntimeError, "CUDA"),
])
def test_construction_refusals(args, err, msg):
    with pytest.raises(err, match=msg):
        sa.QuantizedKVCache(*args)


def test_from_tensors_refusals():
    good = host_cache().tensors()
    with pytest.raises(RuntimeError, match="CUDA"):
        sa.QuantizedKVCache.from_tensors(*good, 64)
    with pytest.raises(TypeError):
        sa.QuantizedKVCache.from_tensors(None, *good[1:], 64)


@pytest.mark.parametrize("k,v,err,msg", [
    ((1, 2, 3, 64), (1, 2, 4, 64), ValueError, "must equal K shape"),
    ((1, 3, 3, 64), None, ValueError, "does not match the cache"),
    ((1, 2, 3, 32), None, ValueError, "does not match the cache"),
    ((2, 3, 64), None, ValueError, "4-D"),
    ((1, 2, 0, 64), None, ValueError, "no tokens"),
    ((1, 2, 3, 64), None, RuntimeError, "CUDA"),
])
def test_write_refusals(k, v, err, msg):
    K, V = torch.zeros(k), torch.zeros(v or k)
    with pytest.raises(err, match=msg):
        host_cache().write(K, V, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_write_dtype_refusals():
    K = torch.zeros(1, 2, 3, 64)
    with pytest.raises(TypeError, match="unsupported dtype"):
        host_cache().write(K.double(), K.double(), None, None)
    with pytest.raises(TypeError, match="same dtype"):
        host_cache().write(K, K.half(), None, None)


@pytest.mark.parametrize("shape,kw,err,msg", [
    ((1, 3, 1, 64), {}, ValueError, "not a multiple"),
    ((1, 4, 1, 32), {}, ValueError, "head dim"),
    ((1, 4, 65, 64), {}, ValueError, "at most 64"),
    ((0, 4, 1, 64), {}, ValueError, "empty"),
    ((1, 4, 64), {}, ValueError, "4-D"),
    ((1, 4, 1, 64), {"max_length": 0}, ValueError, "max_length"),
    ((1, 4, 1, 64), {}, RuntimeError, "CUDA"),
])
def test_attention_refusals(shape, kw, err, msg):
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(err, match=msg):
        sa.cache_attention(torch.zeros(shape), host_cache(), i[None], i, **kw)


def test_attention_refuses_other_types():
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="unsupported dtype"):
        sa.cache_attention(torch.zeros(1, 2, 1, 64, dtype=torch.float64), host_cache(), i[None], i)
    with pytest.raises(TypeError, match="QuantizedKVCache"):
        sa.cache_attention(torch.zeros(1, 2, 1, 64), None, i[None], i)


@pytest.mark.parametrize("t,err,msg", [
    (torch.zeros(3, dtype=torch.int32), ValueError, "shape"),
    (torch.zeros(2), TypeError, "integer"),
    (torch.zeros(2, dtype=torch.bool), TypeError, "integer"),
    ([0, 1], TypeError, "tensor"),
])
def test_integer_arguments(t, err, msg):
    with pytest.raises(err, match=msg):
        cm._i32(t, (2,), torch.device("cpu"), "lengths")


def test_wide_integers_do_not_wrap():
    got = cm._i32(torch.tensor([2 ** 32 + 5, -2 ** 40, 7]), (3,), torch.device("cpu"), "x")
    assert got.tolist() == [2 ** 31 - 1, -2 ** 31, 7]


def test_module_decodes_with_the_exact_threshold_only():
    i = torch.zeros(1, dtype=torch.int32)
    m = sa.AdaptiveSplashAttention(head_dim=64)
    with pytest.raises(ValueError, match="exact"):
        m.decode(torch.zeros(1, 2, 1, 64), host_cache(), i[None], i)
    m = sa.AdaptiveSplashAttention(head_dim=64, tau_mode="exact")
    with pytest.raises(RuntimeError, match="CUDA"):
        m.decode(torch.zeros(1, 2, 1, 64), host_cache(), i[None], i)


def _c(**kw):
    a = 1 << 20  # stand-in addresses: never dereferenced
    base = dict(pages=4, kv_heads=2, page_size=16, head_dim=64, k_codes=a, v_codes=a, k_params=a,
                v_params=a)
    base.update(kw)
    return _lib.Cache(**base)


@pytest.mark.parametrize("bad,msg", [
    (dict(pages=0), "pages"), (dict(pages=1 << 27), "too large"), (dict(kv_heads=0), "kv_heads"), (dict(page_size=24), "page_size"),
    (dict(page_size=512), "page_size"), (dict(head_dim=129), "too large"), (dict(head_dim=0), "head_dim"),
    (dict(k_codes=None), "NULL"), (dict(v_params=(1 << 20) + 8), "aligned"),
])
def test_c_entry_refuses_bad_caches(bad, msg):
    lib, a = _lib.load(), 1 << 20
    t = _lib.CacheTokens(batch=1, n=1, dtype=1, max_pages=1, page_table=a, start=a)
    assert lib.asa_cache_write(ctypes.byref(_c(**bad)), ctypes.byref(t), None, a, a, None) == 1
    assert msg in lib.asa_last_error().decode()


@pytest.mark.parametrize("bad,msg", [
    (dict(batch=0), "batch"), (dict(n=0), "n (0)"), (dict(max_pages=0), "max_pages"),
    (dict(dtype=3), "dtype"), (dict(page_table=None), "page_table"), (dict(n=1 << 27), "too many"), (dict(n=1 << 20, batch=1 << 8), "too many"),
    (dict(k_strides=(0, -4, 64)), "k_strides[1]"),
])
def test_c_entry_refuses_bad_tokens(bad, msg):
    lib, a = _lib.load(), 1 << 20
    base = dict(batch=1, n=1, dtype=1, max_pages=1, page_table=a, start=a)
    base.update(bad)
    t = _lib.CacheTokens(**base)
    assert lib.asa_cache_write(ctypes.byref(_c()), ctypes.byref(t), None, a, a, None) == 1
    assert msg in lib.asa_last_error().decode()


@pytest.mark.parametrize("bad,msg", [
    (dict(batch=0), "batch"), (dict(heads=3), "multiple"), (dict(nq=0), "nq"), (dict(nq=65), "nq"),
    (dict(dtype=-1), "dtype"), (dict(alpha=float("nan")), "alpha"), (dict(sm_scale=float("inf")), "sm_scale"),
    (dict(max_length=-1), "max_length"), (dict(max_pages=1 << 25), "2^28"),
    (dict(q_strides=(64, -1, 64)), "q_strides[1]"), (dict(batch=1 << 20), "too many"),
])
def test_c_entry_refuses_bad_queries(bad, msg):
    lib, a = _lib.load(), 1 << 20
    base = dict(batch=1, heads=4, nq=1, dtype=1, max_pages=4, max_length=0, alpha=1.5, sm_scale=0.1,
                page_table=a, lengths=a)
    base.update(bad)
    q = _lib.CacheQuery(**base)
    z = ctypes.c_size_t()
    assert lib.asa_cache_attention_workspace(ctypes.byref(_c()), ctypes.byref(q), ctypes.byref(z)) == 1
    assert msg in lib.asa_last_error().decode()
    assert lib.asa_cache_attention(ctypes.byref(_c()), ctypes.byref(q), a, a, a, None) == 1


def test_c_entry_refuses_null_operands():
    lib, a = _lib.load(), 1 << 20
    q = _lib.CacheQuery(batch=1, heads=4, nq=1, dtype=1, max_pages=4, alpha=1.5, sm_scale=0.1,
                        page_table=a, lengths=a)
    assert lib.asa_cache_attention(ctypes.byref(_c()), ctypes.byref(q), None, a, a, None) == 1
    q.lengths = None
    assert lib.asa_cache_attention(ctypes.byref(_c()), ctypes.byref(q), a, a, a, None) == 1
    t = _lib.CacheTokens(batch=1, n=1, dtype=1, max_pages=1, page_table=a)
    assert lib.asa_cache_read(ctypes.byref(_c()), ctypes.byref(t), None, a, a, None) == 1
    assert lib.asa_cache_write(None, ctypes.byref(t), None, a, a, None) == 1


def test_sizes_are_the_tensors():
    for d in (1, 32, 33, 80, 128):
        codes, params = ctypes.c_size_t(), ctypes.c_size_t()
        c = _c(head_dim=d, k_codes=None)
        assert _lib.load().asa_cache_query_sizes(ctypes.byref(c), ctypes.byref(codes), ctypes.byref(params)) == 0
        G = -(-d // 32)
        assert (codes.value, params.value) == (4 * 2 * 16 * 16 * G, 4 * 2 * 16 * 4 * G)


def test_struct_fields_match_the_header():
    from test_abi import _header_fields

    for name, cls in (("asa_cache", _lib.Cache), ("asa_cache_tokens", _lib.CacheTokens),
                      ("asa_cache_query", _lib.CacheQuery)):
        assert [f[0] for f in cls._fields_] == _header_fields(name)


def test_fake_shapes():
    m = dict(device="meta")
    pool = (torch.empty(5, 2, 16, 48, dtype=torch.uint8, **m), torch.empty(5, 2, 16, 3, 2, dtype=torch.bfloat16, **m)) * 2
    i = torch.empty(3, 4, dtype=torch.int32, **m)
    n = torch.empty(3, dtype=torch.int32, **m)
    Q = torch.empty(3, 6, 2, 80, dtype=torch.float16, **m)
    out = torch.ops.adasplash.cache_attention(*pool, 80, Q, i, n, None, 1.5, 0.1, None)
    assert (out.shape, out.dtype) == (Q.shape, Q.dtype)
    K, V = torch.ops.adasplash.cache_read(*pool, 80, i, n, 7, torch.float32, None)
    assert K.shape == V.shape == (3, 2, 7, 80) and K.dtype == torch.float32
    assert torch.ops.adasplash.cache_write(*pool, 80, K, V, i, n, None) is None


def test_every_value_is_within_half_a_step():
    """The definition's promise, on the 64-bit definition that the GPU tests
    compare codes with."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 80, generator=g) * torch.logspace(-6, 6, 200)[:, None]
    x[::3] += 5.0
    codes, s, m = ref.quantise(x)
    step = s.repeat_interleave(32, -1)[:, :80]
    assert bool(((ref.values(codes, s, m) - x.double()).abs() <= 0.5 * step).all())
    assert codes.min() == 0 and codes.max() == 15
