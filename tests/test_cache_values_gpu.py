"""Attention over a 4-bit cache whose values are small, large, or of keys with small probabilities, against plain attention in 64 bits.

Bound of o, element by element (p: probabilities; a value is b + s (1 + c/16)): P is rounded to fp16 for its product with b + s, and P times s once
more for that with c/16: 2^-11 of p |v| and of p s c/16, and the result's own rounding.  The kernel takes P 2^15-fold, or where scales are 2 and more down to
2^11-fold, and keeps the products at up to 2^9 to 2^16 times the largest scale; fp16's smallest step, 2^-24, thus rounds P by at most 2^-36 and a product
by at most 2^-33 of the largest scale (both per key, in units where a
row's largest P is 1, and a row's sum of P is at least that).  A score's rounding counts 2^-13 of p as in tests/reference64.py, for terms that add up to 8 in
absolute value; where they add up to more, as much more."""
import pytest
import torch

import mha_manual  # noqa: F401
from tests import cache_reference as ref
from tests.reference64 import SLACK, check, half_ulp

pytestmark = pytest.mark.gpu
ops = torch.ops.mha_manual


def randn(*shape, dtype, device, seed):
    return torch.randn(*shape, device=device, dtype=dtype, generator=torch.Generator(device=device).manual_seed(seed))


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def attention(c, q, lens, scale=None):
    """((o, bound), (lse, bound)) of one new row of every sequence."""
    rows, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    o, ob = (torch.zeros(rows, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, lb = (torch.empty(H, rows, dtype=torch.float64, device=q.device) for _ in range(2))
    for b, n in enumerate(lens):
        k = c.rows("k", b, n)[0]
        v, v_abs, by_code = c.rows("v", b, n)
        v_scale = c.params["v_params"][c.where(b, torch.arange(n, device=q.device))][..., 0].double()
        x = q[b].double().reshape(c.H, -1, D)
        s = torch.einsum("hgd,jhd->hgj", x, k) * scale
        terms = (torch.einsum("hgd,jhd->hgj", x.abs(), k.abs()).amax(-1, keepdim=True) * scale / 8).clamp(min=1.0)
        top = torch.logsumexp(s, -1, keepdim=True)
        p = (s - top).exp()
        out = torch.einsum("hgj,jhd->hgd", p, v)
        u = 2.0 ** -11
        e = (torch.einsum("hgj,jhd->hgd", (u + SLACK * terms) * p, v_abs) + u * torch.einsum("hgj,jhd->hgd", p, by_code) +
             n * (2.0 ** -36 * v_abs.max() + 2.0 ** -33 * v_scale.max()) + half_ulp(q.dtype) * out.abs())
        o[b], ob[b] = out.reshape(H, D), 1.01 * e.reshape(H, D)
        lse[:, b], lb[:, b] = top.reshape(H), 2.0 ** -12 * terms.reshape(H)
    return (o, ob), (lse, lb)


def filled(lens, H_kv, D, dtype, device, size, lift, sink):
    """Keys and values of lens[b] rows; the values are `size` large.  lift: the first key's scores are that much higher, for queries whose
    first value is 4; its values are `sink` large."""
    c = ref.Cache(len(lens), -(-max(lens) // 32), H_kv, D, 32, dtype, 4, device)
    for b, n in enumerate(lens):
        k, v = (randn(n, H_kv, D, dtype=dtype, device=device, seed=100 * b + i) for i in range(2))
        v *= size
        if lift:
            k[..., 0] = 0
            k[0, :, 0] = lift * D ** 0.5 / 4
            v[0] = v[0] * (sink / size)
        c.put(b, torch.arange(n, device=device), k, v)
    return c


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("H,H_kv", [(4, 2), (16, 1)])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e-5, 5000.0])
@pytest.mark.parametrize("lift,sink", [(0, 0), (14, 0), (17, 0), (17, 1), (20, 0)])
def test_values_of_all_sizes(cuda_device, D, dtype, H, H_kv, size, lift, sink):
    """Whole units and pieces of one; sink: of the first key's values, as a part of the others' size."""
    lens = [40, 4000, 513]
    c = filled(lens, H_kv, D, dtype, cuda_device, size, lift, sink * size)
    q = randn(len(lens), H, D, dtype=dtype, device=cuda_device, seed=7)
    if lift:
        q[..., 0] = 4
    o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints(lens, cuda_device), **c.params)
    ops.check_status()
    want_o, want_lse = attention(c, q, lens)
    check(o, (want_o[0], want_o[1] + (2.0 ** -25 if dtype == torch.float16 else 0)), "o")   # (the result's own smallest step)
    check(lse, want_lse, "lse")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("up", [True, False])
def test_sizes_that_change_along_a_sequence(cuda_device, D, up):
    """Values from 1e-6 to 1e4, growing or shrinking from key to key: the products' scale follows the largest."""
    lens, dtype = [900, 2500], torch.bfloat16
    c = ref.Cache(2, 79, 2, D, 32, dtype, 4, cuda_device)
    for b, n in enumerate(lens):
        k, v = (randn(n, 2, D, dtype=dtype, device=cuda_device, seed=10 * b + i) for i in range(2))
        size = torch.logspace(-6, 4, n, device=cuda_device, dtype=torch.float64)
        v = (v.double() * (size if up else size.flip(0))[:, None, None]).to(dtype)
        c.put(b, torch.arange(n, device=cuda_device), k, v)
    q = randn(2, 12, D, dtype=dtype, device=cuda_device, seed=7)
    o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints(lens, cuda_device), **c.params)
    ops.check_status()
    want_o, want_lse = attention(c, q, lens)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,sizes", [(torch.float16, [1, 1000, 1023, 1024, 5000, 15000]), (torch.bfloat16, [0.1, 1, 1000, 1024, 60000, 1e6, 3e8])])
def test_queries_of_all_sizes(cuda_device, D, dtype, sizes):
    """Large queries are scaled to the range of fp16, each row by a power of two of its own: heads of one tile from small to large, with
    the scale that makes the scores of each of them moderate in turn (and those of larger ones huge)."""
    lens, H = [700, 90], len(sizes)
    c = filled(lens, 1, D, dtype, cuda_device, 1.0, 0, 0)
    q = (randn(2, H, D, dtype=torch.float32, device=cuda_device, seed=3) * torch.tensor(sizes, device=cuda_device)[:, None]).to(dtype)
    for size in sizes:
        scale = 1.0 / size * D ** -0.5
        o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints(lens, cuda_device), scale=scale, **c.params)
        want_o, want_lse = attention(c, q, lens, scale)
        fine = torch.tensor([x <= 1e6 * size for x in sizes], device=cuda_device)   # scores below 2^24
        assert torch.isfinite(o[:, fine]).all() and torch.isfinite(lse[fine]).all()
        live = torch.tensor([x <= 100 * size for x in sizes], device=cuda_device)   # scores whose softmax 32 bits can tell
        check(o[:, live], (want_o[0][:, live], want_o[1][:, live]), f"o at {size}")
        check(lse[live], (want_lse[0][live], want_lse[1][live]), f"lse at {size}")
    ops.check_status()


def test_a_line_of_more_than_32_bits(cuda_device):
    """A sequence at the documented limit of rows, with so many key heads that their steps together pass 2^31.  Its pages do not exist (rows of
    zeros), so there is nothing to bring in: every key counts the same."""
    H, page, D = 66, 1 << 16, 64
    width = ((1 << 31) - page) // page
    k_cache = torch.zeros(1, H, page, D, dtype=torch.float16, device=cuda_device)
    table = torch.full((1, width), -1, dtype=torch.int32, device=cuda_device)
    q = randn(1, H, D, dtype=torch.float16, device=cuda_device, seed=1)
    n = width * page
    o, lse = ops.fmha_paged_fwd(q, k_cache, k_cache, table, ints([n], cuda_device))
    ops.check_status()
    assert (o == 0).all()
    assert (lse - torch.tensor(float(n)).log().item()).abs().max() < 2.0 ** -12 * 2
