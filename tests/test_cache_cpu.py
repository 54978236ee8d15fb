"""Paged-cache operators without a GPU: shapes of the shape-only kernels, refusals, the C entry points' checks of arguments."""
import ctypes as C

import pytest
import torch

import mha_manual  # noqa: F401
from nvfuserexamples_b200 import capi

ops = torch.ops.mha_manual


def meta(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def caches(bits=16, D=128, pages=10, H=2, page=32, dtype=torch.float16):
    if bits == 16:
        return dict(k_cache=meta(pages, H, page, D, dtype=dtype), v_cache=meta(pages, H, page, D, dtype=dtype)), {}
    return (dict(k_cache=meta(pages, H, page, D // 2, dtype=torch.uint8), v_cache=meta(pages, H, page, D // 2, dtype=torch.uint8)),
            dict(k_params=meta(pages, H, page, D // 32, 2), v_params=meta(pages, H, page, D // 32, 2)))


INT = dict(dtype=torch.int32)


@pytest.mark.parametrize("bits", [16, 4])
def test_shapes(bits):
    c, p = caches(bits)
    table, lens, cu = meta(3, 4, **INT), meta(3, **INT), meta(4, **INT)
    q, k = meta(7, 6, 128), meta(7, 2, 128)
    out = ops.kv_append(k, k, **c, block_table=table, seqlens=lens, cu_seqlens=cu, q=q, inv_freq=meta(64, dtype=torch.float32), **p)
    assert out.shape == q.shape and out.dtype == q.dtype
    assert ops.kv_append(k, k, **c, block_table=table, seqlens=lens, cu_seqlens=cu, **p) is None
    o, lse = ops.fmha_paged_fwd(q, **c, block_table=table, seqlens=lens, cu_seqlens=cu, max_seqlen_q=3, **p)
    assert o.shape == q.shape and lse.shape == (6, 7) and lse.dtype == torch.float32
    o, _ = ops.fmha_paged_fwd(q[:6], **c, block_table=table, seqlens=lens, **p)
    assert o.shape == (6, 6, 128)
    a, b = ops.kv_read(**c, block_table=table, cu_seqlens=cu, total_rows=50, **p, bf16=True)
    assert a.shape == b.shape == (50, 2, 128) and a.dtype == (torch.float16 if bits == 16 else torch.bfloat16)


def attend(**over):
    c, p = caches(over.pop("bits", 16), **over.pop("cache", {}))
    args = dict(q=meta(6, 6, 128), **c, **p, block_table=meta(3, 4, **INT), seqlens=meta(3, **INT))
    args.update(over)
    return ops.fmha_paged_fwd(**args)


def append(**over):
    c, p = caches(over.pop("bits", 16), **over.pop("cache", {}))
    args = dict(k=meta(6, 2, 128), v=meta(6, 2, 128), **c, **p, block_table=meta(3, 4, **INT), seqlens=meta(3, **INT))
    args.update(over)
    return ops.kv_append(**args)


@pytest.mark.parametrize("over", [
    dict(q=meta(6, 5, 128)), dict(q=meta(6, 6, 64)), dict(q=meta(6, 6, 128, dtype=torch.bfloat16)), dict(q=meta(7, 6, 128)), dict(seqlens=meta(4, **INT)),
    dict(block_table=meta(3, 4, dtype=torch.int64)), dict(block_table=meta(12, **INT)), dict(cu_seqlens=meta(4, **INT)), dict(cu_seqlens=meta(3, **INT), max_seqlen_q=2),
    dict(cache=dict(page=24)), dict(cache=dict(D=96), q=meta(6, 6, 96)), dict(v_cache=meta(10, 2, 16, 128)), dict(k_params=meta(10, 2, 32, 4, 2)),
    dict(bits=4, k_params=None), dict(bits=4, v_params=meta(10, 2, 32, 2, 2)), dict(bits=4, v_params=meta(10, 2, 32, 4, 2, dtype=torch.float32)),
    dict(cache=dict(pages=0)), dict(cache=dict(H=0)), dict(q=meta(6, 6, 128, dtype=torch.float32))])
def test_refusals_of_attention(over):
    with pytest.raises(RuntimeError):
        attend(**over)


@pytest.mark.parametrize("over", [
    dict(k=meta(6, 3, 128), v=meta(6, 3, 128)), dict(v=meta(5, 2, 128)), dict(k=meta(7, 2, 128), v=meta(7, 2, 128)), dict(q=meta(5, 4, 128)),
    dict(q=meta(6, 4, 128, dtype=torch.bfloat16)), dict(k=meta(6, 2, 128, dtype=torch.bfloat16), v=meta(6, 2, 128, dtype=torch.bfloat16)),
    dict(inv_freq=meta(65, dtype=torch.float32)), dict(inv_freq=meta(72, dtype=torch.float32)), dict(inv_freq=meta(12, dtype=torch.float32)),
    dict(inv_freq=meta(64, dtype=torch.float64)), dict(bits=4, inv_freq=meta(8, dtype=torch.float32)), dict(seqlens=meta(2, **INT)), dict(cu_seqlens=meta(6, **INT))])
def test_refusals_of_append(over):
    with pytest.raises(RuntimeError):
        append(**over)


def test_refusals_of_read():
    c, _ = caches()
    for over in (dict(cu_seqlens=meta(3, **INT)), dict(total_rows=-1)):
        args = dict(**c, block_table=meta(3, 4, **INT), cu_seqlens=meta(4, **INT), total_rows=9)
        args.update(over)
        with pytest.raises(RuntimeError):
            ops.kv_read(**args)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.fmha_paged_fwd(torch.zeros(1, 2, 64, dtype=torch.float16), x, x, torch.zeros(1, 1, **INT), torch.ones(1, **INT))


# ------------------------------------------------------------------------------------------------ the C entry points
def cache_struct(bits=16, **over):
    c = capi.KvCache()
    c.bits, c.pages, c.page_rows, c.H_kv, c.D = bits, 10, 32, 2, 128
    c.k = c.v = capi.Tensor4(0x1000, 2 * 32 * 128, 32 * 128, 128)
    c.k_params = c.v_params = capi.Tensor4(0x2000, 2 * 32 * 8, 32 * 8, 8)
    c.table, c.table_width, c.table_stride = 0x3000, 4, 4
    for k, v in over.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [(dict(bits=8), capi.FMHA_ERR_UNSUPPORTED), (dict(D=96), capi.FMHA_ERR_UNSUPPORTED), (dict(page_rows=24), capi.FMHA_ERR_BAD_ARG),
              (dict(page_rows=1 << 17), capi.FMHA_ERR_TOO_LARGE), (dict(H_kv=0), capi.FMHA_ERR_BAD_ARG), (dict(H_kv=70000), capi.FMHA_ERR_TOO_LARGE),
              (dict(table=None), capi.FMHA_ERR_BAD_ARG), (dict(table_width=1 << 27), capi.FMHA_ERR_TOO_LARGE), (dict(pages=-1), capi.FMHA_ERR_BAD_ARG),
              (dict(k=capi.Tensor4(0x1008, 8192, 4096, 128)), capi.FMHA_ERR_BAD_ARG), (dict(v=capi.Tensor4(0x1000, 8192, 4095, 128)), capi.FMHA_ERR_BAD_ARG),
              (dict(bits=4, k_params=capi.Tensor4(None, 512, 256, 8)), capi.FMHA_ERR_BAD_ARG), (dict(bits=4, v_params=capi.Tensor4(0x2000, 510, 256, 8)), capi.FMHA_ERR_BAD_ARG)]


def paged_params(cache=None, **over):
    p = capi.PagedParams()
    p.struct_bytes, p.dtype, p.B, p.H, p.total_rows, p.max_rows, p.scale = C.sizeof(p), capi.DTYPE_F16, 3, 6, 6, 2, 0.1
    p.q = p.o = capi.Tensor4(0x4000, 0, 128, 768)
    p.cache = cache or cache_struct()
    p.seqlens = 0x5000
    for k, v in over.items():
        setattr(p, k, v)
    return p


def append_params(cache=None, **over):
    p = capi.KvAppendParams()
    p.struct_bytes, p.dtype, p.B, p.H, p.total_rows = C.sizeof(p), capi.DTYPE_F16, 3, 6, 6
    p.q = p.q_out = capi.Tensor4(0x4000, 0, 128, 768)
    p.k = p.v = capi.Tensor4(0x4000, 0, 128, 256)
    p.cache = cache or cache_struct()
    p.seqlens, p.inv_freq, p.n_freq = 0x5000, 0x6000, 64
    for k, v in over.items():
        setattr(p, k, v)
    return p


def read_params(cache=None, **over):
    p = capi.KvReadParams()
    p.struct_bytes, p.dtype, p.B, p.total_rows = C.sizeof(p), capi.DTYPE_F16, 3, 6
    p.k = p.v = capi.Tensor4(0x4000, 0, 128, 256)
    p.cache = cache or cache_struct()
    p.cu_rows = 0x5000
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_caches_are_checked(over, code):
    lib = capi.load()
    c = cache_struct(**over)
    assert lib.fmha_sm100_paged_fwd(C.byref(paged_params(c)), None) == code
    assert lib.fmha_sm100_kv_append(C.byref(append_params(c)), None) == code
    assert lib.fmha_sm100_kv_read(C.byref(read_params(c)), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(struct_bytes=4), capi.FMHA_ERR_BAD_ARG), (dict(dtype=3), capi.FMHA_ERR_UNSUPPORTED), (dict(H=5), capi.FMHA_ERR_BAD_ARG), (dict(H=0), capi.FMHA_ERR_BAD_ARG),
    (dict(total_rows=7), capi.FMHA_ERR_BAD_ARG), (dict(scale=0.0), capi.FMHA_ERR_BAD_ARG), (dict(max_rows=0), capi.FMHA_ERR_BAD_ARG),
    (dict(max_rows=1 << 20), capi.FMHA_ERR_TOO_LARGE), (dict(seqlens=None), capi.FMHA_ERR_BAD_ARG), (dict(q=capi.Tensor4(0x4004, 0, 128, 768)), capi.FMHA_ERR_BAD_ARG),
    (dict(o=capi.Tensor4(0x4000, 0, 128, 764)), capi.FMHA_ERR_BAD_ARG), (dict(B=70000), capi.FMHA_ERR_TOO_LARGE), (dict(total_rows=0), capi.FMHA_OK)])
def test_argument_checks_of_attention(over, code):
    assert capi.load().fmha_sm100_paged_fwd(C.byref(paged_params(**over)), None) == code


def test_without_offsets_all_rows_take_part():
    assert capi.load().fmha_sm100_paged_fwd(C.byref(paged_params(max_rows=1)), None) == capi.FMHA_ERR_BAD_ARG   # two rows each
    assert capi.load().fmha_sm100_paged_fwd(C.byref(paged_params(max_rows=1, cu_rows=0x5000)), None) != capi.FMHA_ERR_BAD_ARG


@pytest.mark.parametrize("over,code", [
    (dict(struct_bytes=4), capi.FMHA_ERR_BAD_ARG), (dict(n_freq=65), capi.FMHA_ERR_UNSUPPORTED), (dict(n_freq=12), capi.FMHA_ERR_UNSUPPORTED),
    (dict(inv_freq=None), capi.FMHA_ERR_BAD_ARG), (dict(flags=2), capi.FMHA_ERR_BAD_ARG), (dict(total_rows=7), capi.FMHA_ERR_BAD_ARG),
    (dict(k=capi.Tensor4(0x4000, 0, 128, 252)), capi.FMHA_ERR_BAD_ARG), (dict(q_out=capi.Tensor4(None, 0, 128, 768)), capi.FMHA_ERR_BAD_ARG), (dict(total_rows=0), capi.FMHA_OK)])
def test_argument_checks_of_append(over, code):
    assert capi.load().fmha_sm100_kv_append(C.byref(append_params(**over)), None) == code


def test_four_bits_rotate_whole_groups():
    lib = capi.load()
    assert lib.fmha_sm100_kv_append(C.byref(append_params(cache_struct(4), n_freq=8)), None) == capi.FMHA_ERR_UNSUPPORTED


@pytest.mark.parametrize("over,code", [(dict(struct_bytes=4), capi.FMHA_ERR_BAD_ARG), (dict(cu_rows=None), capi.FMHA_ERR_BAD_ARG), (dict(B=0), capi.FMHA_ERR_BAD_ARG),
                                       (dict(k=capi.Tensor4(None, 0, 128, 256)), capi.FMHA_ERR_BAD_ARG), (dict(total_rows=0), capi.FMHA_OK)])
def test_argument_checks_of_read(over, code):
    assert capi.load().fmha_sm100_kv_read(C.byref(read_params(**over)), None) == code
