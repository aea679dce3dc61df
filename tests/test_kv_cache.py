"""Key-value cache checks that need no GPU: the ABI's structures, its refusals
on the host before anything is launched, and the page allocator."""
import ctypes

import pytest
import torch

import monarch_attention_b200 as mab
from monarch_attention_b200 import _lib
from oracle import kv_cache_oracle as oracle

def fill(p, **over):
    c = p.cache
    c.dtype = _lib.DTYPE_BF16
    for f in ("k_pages", "v_pages", "page_table", "status"):
        setattr(c, f, 4096)  # never read: every call here is refused
    c.k_stride[:] = c.v_stride[:] = [2048, 1024, 64]
    c.E, c.Hk, c.D, c.num_pages, c.page_size, c.max_pages = 2, 2, 64, 8, 16, 4
    p.dtype = _lib.DTYPE_BF16
    for name, v in over.items():
        obj = c if name.startswith("c_") else p
        setattr(obj, name[2:] if name.startswith("c_") else name, v)
    return p


CACHE_FAULTS = [
    (dict(c_struct_size=1), _lib.MA_ERR_BAD_PARAMS), (dict(struct_size=1), _lib.MA_ERR_BAD_PARAMS),
    (dict(c_dtype=9), 3), (dict(c_dtype=_lib.DTYPE_E4M3), 1), (dict(c_D=257), 2), (dict(c_D=0), 2),
    (dict(c_E=0), 2), (dict(c_Hk=0), 2), (dict(c_num_pages=0), 2), (dict(c_page_size=0), 2),
    (dict(c_max_pages=2 ** 28), 2), (dict(c_k_pages=None), 1), (dict(c_page_table=None), 1),
    (dict(c_status=None), 1), (dict(dtype=_lib.DTYPE_E4M3), 3), (dict(dtype=_lib.DTYPE_I8), 3),
]


@pytest.mark.parametrize("over,code", CACHE_FAULTS, ids=[str(list(f[0])[0]) + str(i) for i, f in enumerate(CACHE_FAULTS)])
@pytest.mark.parametrize("name", ["write", "read", "decode"])
def test_host_refuses_bad_cache(name, over, code):
    lib = mab.load_library()
    cls, fn = {"write": (_lib.MaCacheWriteParams, lib.ma_cache_write),
               "read": (_lib.MaCacheReadParams, lib.ma_cache_read),
               "decode": (_lib.MaDecodeParams, lib.ma_decode)}[name]
    assert fn(ctypes.byref(fill(cls(), **over)), None) == code
    assert lib.ma_last_error_detail()


@pytest.mark.parametrize("over,code", [
    (dict(T=0), 2), (dict(k=None), 1), (dict(start=None), 1), (dict(T=2 ** 30), 2),
])
def test_host_refuses_bad_write(over, code):
    lib = mab.load_library()
    good = dict(T=3, k=4096, v=4096, start=4096)
    assert lib.ma_cache_write(ctypes.byref(fill(_lib.MaCacheWriteParams(), **{**good, **over})), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(N=0), 2), (dict(v=None), 1), (dict(lengths=None), 1), (dict(N=2 ** 30), 2),
])
def test_host_refuses_bad_read(over, code):
    lib = mab.load_library()
    good = dict(N=3, k=4096, v=4096, lengths=4096)
    assert lib.ma_cache_read(ctypes.byref(fill(_lib.MaCacheReadParams(), **{**good, **over})), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(H=0), 2), (dict(H=3), 2), (dict(q=None), 1), (dict(out=None), 1), (dict(lengths=None), 1),
    (dict(dtype=_lib.DTYPE_F16), 3), (dict(mask=4096), 5), (dict(mask=4096, mask_dtype=7), 5),
    (dict(mask_dtype=1), 5), (dict(mask=4096, mask_dtype=1, mask_len=-1), 5),
    (dict(sm_scale=0.0), 9), (dict(sm_scale=float("nan")), 9), (dict(sm_scale=float("inf")), 9),
    (dict(workspace=None), 6), (dict(workspace_bytes=16), 6), (dict(workspace=4097), 6),
])
def test_host_refuses_bad_decode(over, code):
    lib = mab.load_library()
    good = dict(H=4, q=4096, out=4096, lengths=4096, sm_scale=0.1, workspace=4096,
                workspace_bytes=lib.ma_decode_workspace_bytes())
    assert lib.ma_decode(ctypes.byref(fill(_lib.MaDecodeParams(), **{**good, **over})), None) == code


def test_null_params():
    lib = mab.load_library()
    for fn in (lib.ma_cache_write, lib.ma_cache_read, lib.ma_decode):
        assert fn(None, None) == 1


def test_negative_strides_are_refused():
    lib = mab.load_library()
    p = fill(_lib.MaCacheReadParams(), N=3, k=4096, v=4096, lengths=4096)
    p.k_stride[2] = -64
    assert lib.ma_cache_read(ctypes.byref(p), None) == 4
    p = fill(_lib.MaCacheReadParams(), N=3, k=4096, v=4096, lengths=4096)
    p.cache.v_stride[0] = -1
    assert lib.ma_cache_read(ctypes.byref(p), None) == 4


def test_cpu_tensors_are_refused():
    cache = mab.PagedKVCache(4, 2, 64, max_seqs=2, max_len=32, page_size=16, device="cpu")
    x = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.append(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.attend(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.read()


def test_pages_are_handed_out_and_taken_back():
    cache = mab.PagedKVCache(6, 2, 20, max_seqs=2, max_len=64, page_size=16, dtype=torch.int8, device="cpu")
    assert cache.k_pages.shape == (6, 2, 16, 20) and cache.k_pages.stride()[2] == 32
    assert cache.scales[0].shape == (6, 2, 16)
    cache.reserve([17, 0])
    cache.reserve([17, 16])
    cache.reserve([1, 1])  # fewer: nothing changes
    t = cache.page_table
    used = t[t >= 0].tolist()
    assert cache.free_pages == 3 and len(set(used)) == 3 and (t[0, 2:] == -1).all()
    with pytest.raises(RuntimeError, match="full"):
        cache.reserve([64, 64])
    assert cache.free_pages == 3
    cache.free(0)
    assert cache.free_pages == 5 and (cache.page_table[0] == -1).all()
    cache.reserve([64, 16])
    ids = cache.page_table[cache.page_table >= 0].tolist()
    assert len(ids) == len(set(ids)) == 5
    with pytest.raises(ValueError):
        cache.reserve([1])
    with pytest.raises(ValueError):
        mab.PagedKVCache(4, 2, 257, max_seqs=1, max_len=8)
    with pytest.raises(TypeError):
        mab.PagedKVCache(4, 2, 64, max_seqs=1, max_len=8, dtype=torch.float64)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_oracle_codes_are_nearest(dtype):
    """The oracle's codes are within half a step of the value."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(50, 64, generator=g)
    c, s = oracle.quantise(x, dtype)
    err = (c.double() * s.double()[:, None] - x.double()).abs()
    # e4m3: half a unit of 3 bits behind the first, or half the smallest step
    step = 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * s.double()[:, None] \
        if dtype != torch.int8 else 0.5 * s.double()[:, None].expand_as(err)
    assert (err <= step * (1 + 2.0 ** -20)).all()
    z, zs = oracle.quantise(torch.zeros(2, 8), dtype)
    assert (z.float() == 0).all() and (zs > 0).all()


def test_binding_refuses_without_a_gpu():
    """The torch binding's checks raise Python exceptions with the shapes in them."""
    k = torch.zeros(2, 2, 4, 8)
    table, ln = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match=r"\(2, 2, 4, 8\) and \(1, 2, 4, 8\)"):
        mab.decode_attention(k, k, k[:1], table, ln)
    with pytest.raises(TypeError, match="Double"):
        mab.kv_cache_read(k, k.double(), table, ln, 4)
    with pytest.raises(TypeError, match="v_pages must be a tensor"):
        mab.kv_cache_write(k, k, k, None, table, ln)
    with pytest.raises(RuntimeError, match="CUDA"):
        mab.kv_cache_write(k, k, k, k, table, ln)
