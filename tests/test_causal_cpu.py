"""Causal attention operators without a GPU: shapes of the shape-only kernels, refusals, the C entry points' checks of arguments."""
import ctypes as C

import pytest
import torch

import mha_manual  # noqa: F401
from nvfuserexamples_b200 import capi

ops = torch.ops.mha_manual


def meta(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_shapes():
    q, kv, cu = meta(40, 8, 128), meta(40, 2, 128), meta(4, dtype=torch.int32)
    o, lse = ops.fmha_causal_varlen_fwd(q, kv, kv, cu, 20)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (8, 40) and lse.dtype == torch.float32
    assert [x.shape for x in ops.fmha_causal_varlen_bwd(o, q, kv, kv, o, lse, cu, 20)] == [q.shape, kv.shape, kv.shape]
    assert ops.fmha_causal_varlen(q, kv, kv, cu, 20).shape == q.shape


@pytest.mark.parametrize("change", [dict(q=(40, 8, 96)), dict(k=(40, 3, 128)), dict(v=(39, 2, 128)), dict(k=(40, 2, 64)), dict(cu=(1,)), dict(max_seqlen=0),
                                    dict(dtype=torch.float32)])
def test_refusals(change):
    q, k, v = (meta(*change.get(n, s), dtype=change.get("dtype", torch.float16)) for n, s in (("q", (40, 8, 128)), ("k", (40, 2, 128)), ("v", (40, 2, 128))))
    with pytest.raises(RuntimeError):
        ops.fmha_causal_varlen_fwd(q, k, v, meta(*change.get("cu", (4,)), dtype=torch.int32), change.get("max_seqlen", 20))


def test_cpu_tensors_are_refused():
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.fmha_causal_varlen_fwd(q, q, q, torch.tensor([0, 4], dtype=torch.int32), 4)


def fwd_params(**over):
    p = capi.CausalFwdParams()
    p.struct_bytes, p.dtype, p.B, p.H, p.H_kv, p.max_seqlen, p.D, p.scale = C.sizeof(p), capi.DTYPE_F16, 2, 4, 2, 100, 64, 0.125
    p.q = p.k = p.v = p.o = capi.Tensor4(0x1000, 0, 64, 256)
    p.cu_seqlens, p.total_rows = 0x2000, 150
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(struct_bytes=8), capi.FMHA_ERR_BAD_ARG), (dict(D=96), capi.FMHA_ERR_UNSUPPORTED), (dict(dtype=5), capi.FMHA_ERR_UNSUPPORTED),
    (dict(H_kv=3), capi.FMHA_ERR_BAD_ARG), (dict(H_kv=0), capi.FMHA_ERR_BAD_ARG), (dict(B=70000), capi.FMHA_ERR_TOO_LARGE),
    (dict(B=65535, H=65535, H_kv=1, max_seqlen=1 << 20), capi.FMHA_ERR_TOO_LARGE), (dict(scale=-1.0), capi.FMHA_ERR_BAD_ARG),
    (dict(cu_seqlens=None), capi.FMHA_ERR_BAD_ARG), (dict(max_seqlen=0), capi.FMHA_ERR_BAD_ARG), (dict(total_rows=-1), capi.FMHA_ERR_BAD_ARG),
    (dict(q=capi.Tensor4(0x1008, 0, 64, 256)), capi.FMHA_ERR_BAD_ARG), (dict(k=capi.Tensor4(0x1000, 0, 60, 256)), capi.FMHA_ERR_BAD_ARG),
    (dict(total_rows=0), capi.FMHA_OK), (dict(B=0), capi.FMHA_OK)])
def test_argument_checks_of_the_c_entry(over, code):
    assert capi.load().fmha_sm100_causal_fwd(C.byref(fwd_params(**over)), None) == code


def test_workspace_and_checks_of_the_backward():
    lib = capi.load()
    p = capi.CausalBwdParams()
    p.struct_bytes, p.dtype, p.B, p.H, p.H_kv, p.max_seqlen, p.D, p.scale, p.total_rows = C.sizeof(p), capi.DTYPE_BF16, 2, 4, 2, 100, 64, 0.125, 150
    n = C.c_size_t()
    assert lib.fmha_sm100_causal_bwd_workspace_bytes(C.byref(p), C.byref(n)) == capi.FMHA_OK
    assert n.value >= 2 * 4 * 128 * 64 * 4 + 2 * 4 * 100 * 4
    assert lib.fmha_sm100_causal_bwd(C.byref(p), None) == capi.FMHA_ERR_BAD_ARG   # no tensors
    p.q = p.k = p.v = p.o = p.d_o = p.dq = p.dk = p.dv = capi.Tensor4(0x1000, 0, 64, 256)
    p.cu_seqlens, p.lse, p.workspace, p.workspace_bytes = 0x2000, 0x3000, 0x4000, n.value - 1
    assert lib.fmha_sm100_causal_bwd(C.byref(p), None) == capi.FMHA_ERR_BAD_ARG   # a workspace that is too small
    p.struct_bytes -= 4
    assert lib.fmha_sm100_causal_bwd(C.byref(p), None) == capi.FMHA_ERR_BAD_ARG
    assert lib.fmha_sm100_causal_bwd(None, None) == capi.FMHA_ERR_BAD_ARG


def workspace_bytes(lens, H, H_kv, D):
    p = capi.CausalBwdParams()
    p.struct_bytes, p.dtype, p.B, p.H, p.H_kv, p.max_seqlen, p.D, p.scale, p.total_rows = (
        C.sizeof(p), capi.DTYPE_BF16, len(lens), H, H_kv, max(lens), D, 0.125, sum(lens))
    n = C.c_size_t()
    assert capi.load().fmha_sm100_causal_bwd_workspace_bytes(C.byref(p), C.byref(n)) == capi.FMHA_OK
    return n.value


@pytest.mark.parametrize("lens", [[16384] + [247] * 199, [8192] + [92] * 511, [1] * 4000, [5000]], ids=["200", "512", "short", "one"])
@pytest.mark.parametrize("D,H", [(64, 16), (128, 16), (64, 32)])
def test_workspace_goes_by_rows(lens, D, H):
    """Whatever the longest sequence: dQ's sums (head dimension 64) and delta, a row of either per row and one tile more per sequence."""
    rows = sum(lens) + 128 * len(lens)
    assert workspace_bytes(lens, H, H, D) <= rows * H * 4 * (1 + (D if D == 64 else 0)) + 4096
