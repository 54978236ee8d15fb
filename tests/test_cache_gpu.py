"""Paged caches in 16 and 4 bits: kv_append, kv_read and fmha_paged_fwd against plain torch (tests/cache_reference.py)."""
import pytest
import torch

import mha_manual  # noqa: F401
from tests import cache_reference as ref
from tests.reference64 import check

pytestmark = pytest.mark.gpu
ops = torch.ops.mha_manual
FREQ = {64: 32, 128: 64}


def randn(*shape, dtype, device, seed=1):
    return torch.randn(*shape, device=device, dtype=dtype, generator=torch.Generator(device=device).manual_seed(seed))


def ints(x, device, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=device)


def offsets(new, device, before=0):
    at = [before]
    for n in new:
        at.append(at[-1] + n)
    return ints(at, device)


def inv_freq(n, device):
    return (10000.0 ** (-torch.arange(n, device=device, dtype=torch.float64) / max(n, 1))).float()


def filled(lens, H_kv, D, page, dtype, bits, device, layout="pages", width=None, seed=5):
    """A cache that holds lens[b] random rows of every sequence."""
    width = width or max(1, -(-max(lens) // page))
    c = ref.Cache(len(lens), width, H_kv, D, page, dtype, bits, device, layout=layout, seed=seed)
    for b, n in enumerate(lens):
        if n > 0:
            k, v = (randn(n, H_kv, D, dtype=dtype, device=device, seed=100 * b + i) for i in range(2))
            c.put(b, torch.arange(n, device=device), k, v)
    return c


# ------------------------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page,layout", [(16, "pages"), (48, "rows"), (128, "joint")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(cuda_device, D, dtype, bits, page, layout, interleaved):
    """New rows at ragged positions: rotated k (and q), v as it is; all other rows keep their bits."""
    H, H_kv = 6, 2
    lens, new = [1, 16, 300, 47, 200, 5], [1, 16, 150, 0, 3, 2]
    n_freq = FREQ[D]
    c = filled([a - b for a, b in zip(lens, new)], H_kv, D, page, dtype, bits, cuda_device, layout, width=-(-300 // page))
    total = sum(new)
    q, k, v = randn(total, H, D, dtype=dtype, device=cuda_device, seed=2), *(randn(total, H_kv, D, dtype=dtype, device=cuda_device, seed=s) for s in (3, 4))
    before = [x.clone() for x in (c.k, c.v, *c.params.values())]
    freq, cu = inv_freq(n_freq, cuda_device), offsets(new, cuda_device)
    q_out = ops.kv_append(k, v, c.k, c.v, c.table, ints(lens, cuda_device), cu, q=q, inv_freq=freq, interleaved=interleaved, **c.params)
    pos = torch.cat([torch.arange(a - b, a, device=cuda_device) for a, b in zip(lens, new)])
    check(q_out, ref.rotate(q, pos, freq, interleaved), "q")
    k_rot = ref.rotate(k, pos, freq, interleaved)
    touched = torch.zeros(c.n, page, dtype=torch.bool, device=cuda_device)
    r = 0
    if bits == 4:   # what a 16-bit cache would hold is what is coded
        wide = ref.Cache(len(lens), c.table.shape[1], H_kv, D, page, dtype, 16, cuda_device)
        wide.table = c.table
        ops.kv_append(k, v, wide.k, wide.v, c.table, ints(lens, cuda_device), cu, inv_freq=freq, interleaved=interleaved)
    for b, n in enumerate(new):
        at = c.where(b, torch.arange(lens[b] - n, lens[b], device=cuda_device))
        touched[at[0], at[2]] = True
        rows = slice(r, r + n)
        r += n
        if bits == 16:
            check(c.k[at], (k_rot[0][rows], k_rot[1][rows]), "k")
            assert torch.equal(c.v[at], v[rows])
        else:
            for name in "kv":
                codes, params = ref.encode(getattr(wide, name)[at])
                assert torch.equal(getattr(c, name)[at], codes) and torch.equal(c.params[name + "_params"][at], params)
    for x, y in zip((c.k, c.v, *c.params.values()), before):
        old = ~touched[:, None, :].expand(c.n, H_kv, page)
        assert torch.equal(x[old].view(torch.uint8), y[old].view(torch.uint8))


@pytest.mark.parametrize("D,n_freq,bits", [(64, 0, 16), (64, 8, 16), (128, 16, 16), (128, 40, 16), (128, 32, 4), (64, 0, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_partial_rotation_and_one_row_each(cuda_device, D, n_freq, bits, interleaved):
    """Only the first 2 n_freq values are rotated; without offsets every sequence has the same number of rows."""
    lens = [3, 40, 17]
    c = filled([0, 0, 0], 3, D, 32, torch.float16, bits, cuda_device, width=2)
    k, v = (randn(6, 3, D, dtype=torch.float16, device=cuda_device, seed=s) for s in (1, 2))
    freq = inv_freq(n_freq, cuda_device)
    out = ops.kv_append(k, v, c.k, c.v, c.table, ints(lens, cuda_device), q=k, inv_freq=freq if n_freq else None, interleaved=interleaved, **c.params)
    pos = ints([1, 2, 38, 39, 15, 16], cuda_device)
    want = ref.rotate(k, pos, freq, interleaved)
    check(out, want, "q")
    for i in range(6):
        at = c.where(i // 2, pos[i])
        if bits == 16:
            assert torch.equal(c.k[at], out[i]) and torch.equal(c.v[at], v[i])
        else:
            assert torch.equal(c.k[at], ref.encode(out[i])[0]) and torch.equal(c.params["v_params"][at], ref.encode(v[i])[1])


def test_far_positions(cuda_device):
    """Angles of positions up to 2^30, as exact as near ones."""
    lens = [1 << 20, (1 << 27) + 12345, (1 << 30) - 7]
    freq = inv_freq(64, cuda_device)
    k = randn(3, 2, 128, dtype=torch.float16, device=cuda_device)
    c = ref.Cache(3, 1, 2, 128, 16, torch.float16, 16, cuda_device)
    before = c.k.clone()
    out = ops.kv_append(k, k, c.k, c.v, c.table, ints(lens, cuda_device), q=k, inv_freq=freq)
    pos = ints([n - 1 for n in lens], cuda_device)
    check(out, ref.rotate(k, pos, freq, False), "q")
    assert torch.equal(c.k.view(torch.int16), before.view(torch.int16))   # past the page table: not appended


@pytest.mark.parametrize("bits", [16, 4])
def test_rows_without_a_place_are_left_out(cuda_device, bits):
    """Rows outside the sequences, at negative positions, past the table, on pages that do not exist: nothing is written; q of the first two is zero."""
    D, page = 64, 16
    c = ref.Cache(3, 2, 2, D, page, torch.float16, bits, cuda_device)
    c.table[1] = ints([-1, c.n], cuda_device)
    c.table[2] = ints([1 << 30, -(1 << 31)], cuda_device)
    first = c.table[0, 0].item()
    q, k, v = (randn(60, h, D, dtype=torch.float16, device=cuda_device, seed=h) for h in (4, 2, 2))
    before = [x.clone() for x in (c.k, c.v, *c.params.values())]
    # sequence 0 has five rows and three of them positions; 1 and 2 have rows on bad pages and past the table
    cu = ints([3, 8, 28, 52], cuda_device)
    lens = ints([3, 20, 40], cuda_device)
    out = ops.kv_append(k, v, c.k, c.v, c.table, lens, cu, q=q, inv_freq=inv_freq(32, cuda_device), **c.params)
    assert (out[:5] == 0).all() and (out[52:] == 0).all() and (out[5:52] != 0).any(-1).all()
    for x, y in zip((c.k, c.v, *c.params.values()), before):
        same = (x.view(torch.uint8) == y.view(torch.uint8)).flatten(3).all(-1)
        same[first, :, :3] = True
        assert same.all()
    if bits == 16:
        assert torch.equal(c.v[first, :, :3], v[5:8].transpose(0, 1))


def test_values_that_four_bits_hold(cuda_device):
    """Equal values, one outlier, subnormal spreads, the largest of the type, infinities and NaNs."""
    D = 128
    rows = torch.zeros(8, 1, D, dtype=torch.bfloat16, device=cuda_device)
    rows[1] = 3.25
    rows[2, 0, 5] = 1000.0
    rows[3, 0, ::2] = 1e-7
    rows[4, 0, :40], rows[4, 0, 40:] = 3e38, -3e38
    rows[5, 0, 40] = float("inf")
    rows[6, 0, 100] = float("nan")
    rows[7] = randn(D, dtype=torch.bfloat16, device=cuda_device)
    c = ref.Cache(1, 1, 1, D, 16, torch.bfloat16, 4, cuda_device)
    ops.kv_append(rows, rows, c.k, c.v, c.table, ints([8], cuda_device), offsets([8], cuda_device), **c.params)
    k, v = ops.kv_read(c.k, c.v, c.table, offsets([8], cuda_device), 8, bf16=True, **c.params)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    assert torch.equal(k[:2], rows[:2])
    f = rows.float().clamp(-20000, 20000).unflatten(-1, (-1, 32))
    spread = f.amax(-1, keepdim=True) - f.amin(-1, keepdim=True)
    # half a code, the roundings of scale and base (2^-11 of at most twice the spread plus the value), and that of the result
    bound = spread / 30 + 2.0 ** -10 * (2 * spread + f.abs()) + 2.0 ** -8 * f.abs() + 2.0 ** -24
    fine = torch.isfinite(rows.float().unflatten(-1, (-1, 32))).all(-1, keepdim=True).expand_as(f)
    far = (k.float().unflatten(-1, (-1, 32)) - f).abs()
    assert (far <= bound)[fine].all()
    assert torch.isnan(k[5, 0, 32:64]).all() and torch.isnan(k[6, 0, 96:]).all() and torch.isfinite(k[5, 0, :32]).all() and torch.isfinite(k[6, 0, :96]).all()


@pytest.mark.parametrize("D,dtype,bits", [(64, torch.float16, 16), (128, torch.bfloat16, 16), (64, torch.bfloat16, 4), (128, torch.float16, 4)])
@pytest.mark.parametrize("page,layout", [(16, "joint"), (64, "rows"), (80, "pages")])
def test_read(cuda_device, D, dtype, bits, page, layout):
    lens = [1, 0, 33, 200, 65]
    c = filled(lens, 3, D, page, dtype, bits, cuda_device, layout, width=-(-200 // page))
    c.table[4, -1] = -1 if page > 65 else c.table[4, -1]
    cu = offsets(lens, cuda_device, before=2)
    total = 2 + sum(lens) + 5
    k, v = ops.kv_read(c.k, c.v, c.table, cu, total, bf16=dtype == torch.bfloat16, **c.params)
    assert k.dtype == v.dtype == dtype
    for name, x in (("k", k), ("v", v)):
        assert (x[:2] == 0).all() and (x[-5:] == 0).all()
        for b, n in enumerate(lens):
            if n:
                want = c.rows(name, b, n)[0]
                got = x[2 + sum(lens[:b]):][:n]
                if bits == 16:
                    assert torch.equal(got, want.to(dtype))
                else:
                    check(got, (want, torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -20), name)   # one rounding (of values up to eight in 32 bits first)


def test_read_past_the_table_and_of_missing_pages(cuda_device):
    c = filled([40], 2, 64, 16, torch.float16, 16, cuda_device)
    c.table[0, 1] = c.n + 5
    k, _ = ops.kv_read(c.k, c.v, c.table, ints([0, 70], cuda_device), 70)
    assert (k[16:32] == 0).all() and (k[48:] == 0).all()
    assert torch.equal(k[:16], c.rows("k", 0, 16)[0].half())


# ------------------------------------------------------------------------------------------------ attention
def attend(c, q, lens, new, device, cu=True, before=0, **kw):
    return ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints(lens, device), offsets(new, device, before) if cu else None, max(new), **kw, **c.params)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 48])
@pytest.mark.parametrize("H,H_kv", [(4, 4), (8, 2), (15, 1), (40, 2)])
def test_single_rows(cuda_device, D, dtype, bits, page, H, H_kv):
    lens = [1, 15, 16, 17, 63, 64, 65, 200, 0, 129]
    c = filled(lens, H_kv, D, page, dtype, bits, cuda_device)
    q = randn(len(lens), H, D, dtype=dtype, device=cuda_device)
    o, lse = attend(c, q, lens, [1] * len(lens), cuda_device, cu=False)
    ops.check_status()
    want_o, want_lse = ref.attention(c, q, lens, [1] * len(lens))
    check(o, want_o, "o")
    check(lse, want_lse, "lse")
    assert (o[8] == 0).all() and torch.isneginf(lse[:, 8]).all()      # a sequence without keys


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H,H_kv", [(2, 2), (12, 2), (16, 1)])
def test_several_new_rows(cuda_device, D, dtype, bits, H, H_kv):
    """Ragged numbers of new rows, each seeing one key more; more new rows than keys leaves the first ones without any."""
    lens, new = [70, 5, 300, 40, 2], [4, 5, 40, 0, 6]
    c = filled(lens, H_kv, D, 32, dtype, bits, cuda_device, layout="joint")
    q = randn(sum(new), H, D, dtype=dtype, device=cuda_device)
    o, lse = attend(c, q, lens, new, cuda_device)
    want_o, want_lse = ref.attention(c, q, lens, new)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")
    assert (o[49:53] == 0).all() and torch.isneginf(lse[:, 49:53]).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [16, 4])
def test_long_sequences_are_dealt_out(cuda_device, D, bits):
    """Lengths from one key to thousands in a batch: from one share to dozens."""
    lens, new = [9000, 1, 255, 4097, 520], [2, 1, 2, 2, 2]
    c = filled(lens, 2, D, 64, torch.bfloat16, bits, cuda_device, layout="rows")
    q = randn(sum(new), 6, D, dtype=torch.bfloat16, device=cuda_device)
    o, lse = attend(c, q, lens, new, cuda_device, scale=0.3)
    ops.check_status()
    want_o, want_lse = ref.attention(c, q, lens, new, scale=0.3)
    check(o, (want_o[0], want_o[1] * 4), "o")   # scores four times (at D = 64 2.4 times) as large as those of the bound's 32-bit term
    check(lse, (want_lse[0], want_lse[1] * 4), "lse")
    again = attend(c, q, lens, new, cuda_device, scale=0.3)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", [[512], [513], [641], [1000, 0, 64], [1, 1, 700, 1]])
def test_few_keys_in_small_pieces(cuda_device, D, dtype, bits, lens):
    """Around the length up to which units stay whole, and pieces of hardly more than their start."""
    new = [min(n, 1) for n in lens]
    c = filled(lens, 3, D, 16, dtype, bits, cuda_device)
    q = randn(sum(new), 6, D, dtype=dtype, device=cuda_device)
    o, lse = attend(c, q, lens, new, cuda_device)
    ops.check_status()
    want_o, want_lse = ref.attention(c, q, lens, new)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,H_kv", [(8, 4), (6, 6)])
def test_batches_in_four_bits(cuda_device, D, H, H_kv):
    """Fewer units than, about as many as and more than fill the chip."""
    for B in (20, 30, 70):
        lens = [5 + (37 * b * b) % 900 for b in range(B)]
        c = filled(lens, H_kv, D, 32, torch.float16, 4, cuda_device)
        q = randn(B, H, D, dtype=torch.float16, device=cuda_device)
        o, lse = attend(c, q, lens, [1] * B, cuda_device, cu=False)
        ops.check_status()
        want_o, want_lse = ref.attention(c, q, lens, [1] * B)
        check(o, want_o, "o")
        check(lse, want_lse, "lse")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("B", [3, 90])
def test_a_loose_maximum_of_new_rows(cuda_device, bits, B):
    """max_seqlen_q far above what any sequence has: tiles without rows."""
    lens, new = [(61 * b * b + 9) % 700 for b in range(B)], [b % 4 for b in range(B)]
    c = filled(lens, 2, 64, 32, torch.float16, bits, cuda_device)
    q = randn(sum(new), 8, 64, dtype=torch.float16, device=cuda_device)
    o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints(lens, cuda_device), offsets(new, cuda_device), 1000, **c.params)
    ops.check_status()
    want_o, want_lse = ref.attention(c, q, lens, new)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("scale", [1e-42, 1e-38, 1e-4])
def test_small_scales(cuda_device, bits, scale):
    """Down to subnormal numbers: means of the values."""
    lens = [40, 600]
    c = filled(lens, 2, 64, 16, torch.float16, bits, cuda_device)
    q = randn(2, 4, 64, dtype=torch.float16, device=cuda_device)
    o, lse = attend(c, q, lens, [1, 1], cuda_device, scale=scale)
    want_o, want_lse = ref.attention(c, q, lens, [1, 1], scale=scale)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")


@pytest.mark.parametrize("bits", [16, 4])
def test_rows_outside_sequences_and_past_max_rows(cuda_device, bits):
    lens, new = [50, 90], [3, 20]
    c = filled(lens, 2, 64, 16, torch.float16, bits, cuda_device)
    q = randn(40, 4, 64, dtype=torch.float16, device=cuda_device)
    o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints(lens, cuda_device), offsets(new, cuda_device, before=6), 7, **c.params)
    want_o, want_lse = ref.attention(c, q[6:29], lens, new)
    live = torch.zeros(40, dtype=torch.bool, device=cuda_device)
    live[6:9] = live[9:16] = True
    assert (o[~live] == 0).all() and torch.isneginf(lse[:, ~live]).all()
    check(o[6:16], (want_o[0][:10], want_o[1][:10]), "o")
    check(lse[:, 6:16], (want_lse[0][:, :10], want_lse[1][:, :10]), "lse")


@pytest.mark.parametrize("bits", [16, 4])
def test_pages_that_do_not_exist_read_as_zeros(cuda_device, bits):
    """Page numbers outside the cache are not followed: their rows take part as zeros.  A length past the table ends there."""
    lens = [100, 64]
    c = filled(lens, 2, 128, 32, torch.float16, bits, cuda_device)
    q = randn(2, 4, 128, dtype=torch.float16, device=cuda_device)
    clean_table = c.table.clone()
    for bad in (-1, c.n, (1 << 31) - 1, -(1 << 31)):
        c.table = clean_table.clone()
        c.table[0, 1] = bad
        o, lse = attend(c, q, [100, 1000], [1, 1], cuda_device, cu=False)
        # the same with a page of zeros in that place (sequence 1 has 4 pages of 32 rows; the last two are not filled)
        z = ref.Cache(2, 4, 2, 128, 32, torch.float16, bits, cuda_device)
        for name in "kv":
            getattr(z, name).copy_(getattr(c, name))
            for p in z.params:
                z.params[p].copy_(c.params[p])
        spare = next(i for i in range(c.n) if i not in clean_table.flatten().tolist())
        z.table = clean_table.clone()
        z.table[0, 1] = spare
        for x in (z.k, z.v, *z.params.values()):
            x[spare] = 0
        z_o, z_lse = attend(z, q, [100, 64], [1, 1], cuda_device, cu=False)
        assert torch.equal(o[0], z_o[0]) and torch.equal(lse[:, 0], z_lse[:, 0])
    ops.check_status()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_nan_in_a_row_that_is_seen_shows(cuda_device, bits):
    lens = [40, 40]
    c = filled(lens, 1, 64, 16, torch.float16, bits, cuda_device)
    if bits == 16:
        c.k[c.where(0, torch.tensor(7))] = float("nan")
    else:
        c.params["k_params"][c.where(0, torch.tensor(7))] = float("nan")
    q = randn(2, 2, 64, dtype=torch.float16, device=cuda_device)
    o, lse = attend(c, q, lens, [1, 1], cuda_device, cu=False)
    assert torch.isnan(o[0]).all() and torch.isfinite(o[1]).all() and torch.isfinite(lse[:, 1]).all()


def test_large_queries_stay_finite_in_fp16_products(cuda_device):
    """bf16 queries beyond the range of fp16, against a 4-bit cache."""
    c = filled([30], 1, 64, 16, torch.bfloat16, 4, cuda_device)
    q = randn(1, 2, 64, dtype=torch.bfloat16, device=cuda_device) * 1e6
    o, lse = attend(c, q, [30], [1], cuda_device, cu=False)
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_step_follows_its_tensors(cuda_device, bits):
    """Append and attend in a graph: replays go by the lengths, offsets and table of the moment; two graphs do not share anything."""
    H, H_kv, D, page, B = 8, 2, 128, 16, 3
    c = filled([500, 40, 7], H_kv, D, page, torch.float16, bits, cuda_device, width=40)
    lens = ints([500, 40, 7], cuda_device)
    q, k, v = (randn(B, h, D, dtype=torch.float16, device=cuda_device, seed=h) for h in (H, H_kv, H_kv + 1))
    v = v[:, :H_kv]
    freq = inv_freq(64, cuda_device)

    def step():
        lens.add_(1)
        turned = ops.kv_append(k, v, c.k, c.v, c.table, lens, q=q, inv_freq=freq, **c.params)
        return turned, *ops.fmha_paged_fwd(turned, c.k, c.v, c.table, lens, **c.params)

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(6):
        g, (turned, o, lse) = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        now = lens.tolist()
        assert now == [502 + i, 42 + i, 9 + i]
        want_o, want_lse = ref.attention(c, turned, now, [1, 1, 1])
        check(o, want_o, "o")
        check(lse, want_lse, "lse")


def test_other_streams_and_two_calls_at_once(cuda_device):
    lens = [3000, 900]
    c = filled(lens, 2, 64, 64, torch.bfloat16, 16, cuda_device)
    q = [randn(2, 8, 64, dtype=torch.bfloat16, device=cuda_device, seed=s) for s in range(4)]
    want = [attend(c, x, lens, [1, 1], cuda_device, cu=False) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(5):
        got = []
        for s, x in zip(streams, q):
            with torch.cuda.stream(s):
                got.append(attend(c, x, lens, [1, 1], cuda_device, cu=False))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_cache_past_32_bit_offsets(cuda_device):
    """A cache of more than 2^32 values, with the sequence's pages at its end."""
    H_kv, D, page = 8, 128, 64
    n = (1 << 32) // (H_kv * page * D) + 40
    if torch.cuda.mem_get_info()[0] < 20 * n * H_kv * page * D // 4:
        pytest.skip("not enough memory")
    k_cache = torch.zeros(n, H_kv, page, D, dtype=torch.bfloat16, device=cuda_device)
    v_cache = k_cache.clone()
    table = torch.arange(n - 1, n - 11, -1, device=cuda_device, dtype=torch.int32).reshape(1, -1)
    k, v, q = (randn(600, h, D, dtype=torch.bfloat16, device=cuda_device, seed=h) for h in (H_kv, H_kv, 16))
    cu, lens = offsets([600], cuda_device), ints([600], cuda_device)
    ops.kv_append(k, v, k_cache, v_cache, table, lens, cu)
    for x, y in zip(ops.kv_read(k_cache, v_cache, table, cu, 600), (k, v)):
        assert torch.equal(x, y)
    o, _ = ops.fmha_paged_fwd(q[:4], k_cache, v_cache, table, lens, ints([0, 4], cuda_device), 4)
    s = torch.einsum("ihd,jhd->hij", q[:4].double(), k.double().repeat_interleave(2, 1)) * D ** -0.5
    s = s.masked_fill(torch.arange(600, device=cuda_device) > torch.arange(596, 600, device=cuda_device)[:, None], float("-inf"))
    want = torch.einsum("hij,jhd->ihd", s.softmax(-1), v.double().repeat_interleave(2, 1))
    assert (o.double() - want).abs().max() < 2.0 ** -8   # |o| < 0.5: two roundings of 2^-9


@pytest.mark.parametrize("bits", [16, 4])
def test_prompt_then_decoding(cuda_device, bits):
    """Prompts by causal attention into the cache, then rows one by one and in twos: as causal attention over the whole sequences (in 4 bits as
    far as what the cache holds allows)."""
    H, H_kv, D, page, dtype = 8, 2, 64, 32, torch.float16
    full, prompt = [190, 77, 33], [180, 64, 1]
    freq = inv_freq(32, cuda_device)
    q, k, v = ([randn(n, h, D, dtype=dtype, device=cuda_device, seed=10 * n + h) for n in full] for h in (H, H_kv, H_kv))
    c = ref.Cache(3, 6, H_kv, D, page, dtype, bits, cuda_device)
    rows = lambda x, lo, hi: torch.cat([a[s:e] for a, s, e in zip(x, lo, hi)])  # noqa: E731
    cu, at = offsets(prompt, cuda_device), [0, 0, 0]
    turned = ops.kv_append(rows(k, at, prompt), rows(v, at, prompt), c.k, c.v, c.table, ints(prompt, cuda_device), cu, q=rows(q, at, prompt), inv_freq=freq, **c.params)
    kk, vv = ops.kv_read(c.k, c.v, c.table, cu, sum(prompt), **c.params)
    ops.fmha_causal_varlen_fwd(turned, kk, vv, cu, 180)
    outs, at = [[], [], []], list(prompt)
    while at != full:
        new = [min(2 if i else 1, n - a) for i, (n, a) in enumerate(zip(full, at))]
        hi = [a + n for a, n in zip(at, new)]
        cu = offsets(new, cuda_device)
        turned = ops.kv_append(rows(k, at, hi), rows(v, at, hi), c.k, c.v, c.table, ints(hi, cuda_device), cu, q=rows(q, at, hi), inv_freq=freq, **c.params)
        o, _ = ops.fmha_paged_fwd(turned, c.k, c.v, c.table, ints(hi, cuda_device), cu, max(new), **c.params)
        r = 0
        for b, n in enumerate(new):
            outs[b].append(o[r:r + n])
            r += n
        at = hi
    # the whole sequences at once
    cu, total = offsets(full, cuda_device), sum(full)
    pos = torch.cat([torch.arange(n, device=cuda_device) for n in full])
    turned = ref.rotate(torch.cat(q), pos, freq, False)[0].to(dtype)
    kk, vv = ops.kv_read(c.k, c.v, c.table, cu, total, **c.params)
    if bits == 16:
        check(kk, ref.rotate(torch.cat(k), pos, freq, False), "k")
        assert torch.equal(vv, torch.cat(v))
    whole, _ = ops.fmha_causal_varlen_fwd(turned, kk, vv, cu, 190)
    r = 0
    for b, n in enumerate(full):
        got = torch.cat(outs[b])
        want = whole[r + prompt[b]:r + n]
        r += n
        # two roundings of P and two of O on either side, of values of a few units; in 4 bits also those of the cache's values to fp16
        assert (got.double() - want.double()).abs().max() <= (4 if bits == 16 else 16) * 2.0 ** -11 * 3


@pytest.mark.parametrize("bits", [16, 4])
def test_other_layouts_of_the_arguments(cuda_device, bits):
    """Lines of a wider page table, int64 lengths and offsets, q and k as slices of one projection or with heads outermost, one head, one page."""
    lens, new, D = [45, 20, 64], [2, 1, 2], 64
    c = filled(lens, 2, D, 32, torch.float16, bits, cuda_device)
    wide = torch.full((3, 7), -5, dtype=torch.int32, device=cuda_device)
    wide[:, 2:4] = c.table
    x = randn(5, 10, D, dtype=torch.float16, device=cuda_device)
    q, k, v = x[:, :6], x[:, 6:8], x[:, 8:]
    args = (wide[:, 2:4], ints(lens, cuda_device, torch.int64), offsets(new, cuda_device).long())
    turned = ops.kv_append(k, v, c.k, c.v, *args, q=q, inv_freq=inv_freq(32, cuda_device), **c.params)
    heads_first = turned.transpose(0, 1).contiguous().transpose(0, 1)
    o, lse = ops.fmha_paged_fwd(heads_first, c.k, c.v, *args, 2, **c.params)
    want_o, want_lse = ref.attention(c, turned, lens, new)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")
    kk, vv = ops.kv_read(c.k, c.v, wide[:, 2:4], offsets(lens, cuda_device).long(), sum(lens), **c.params)
    plain = ops.kv_read(c.k, c.v, c.table, offsets(lens, cuda_device), sum(lens), **c.params)
    assert torch.equal(kk, plain[0]) and torch.equal(vv, plain[1])
    one = filled([30], 1, D, 32, torch.float16, bits, cuda_device)
    one.k, one.v, page = one.k[one.table[0, 0]:][:1], one.v[one.table[0, 0]:][:1], one.table[0, 0].item()
    one.params = {n: p[page:page + 1] for n, p in one.params.items()}
    one.table = torch.zeros_like(one.table)
    q1 = randn(1, 1, D, dtype=torch.float16, device=cuda_device)
    o, lse = attend(one, q1, [30], [1], cuda_device, cu=False)
    want_o, want_lse = ref.attention(one, q1, [30], [1])
    check(o, want_o, "o")
    check(lse, want_lse, "lse")


@pytest.mark.parametrize("bits", [16, 4])
def test_no_pages_and_no_rows(cuda_device, bits):
    c = filled([30, 10], 2, 64, 16, torch.float16, bits, cuda_device)
    q = randn(2, 4, 64, dtype=torch.float16, device=cuda_device)
    o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table[:, :0], ints([30, 10], cuda_device), **c.params)   # a table without entries: no keys
    assert (o == 0).all() and torch.isneginf(lse).all()
    o, lse = ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints([-3, 0], cuda_device), **c.params)
    assert (o == 0).all() and torch.isneginf(lse).all()
    o, lse = ops.fmha_paged_fwd(q[:0], c.k, c.v, c.table, ints([30, 10], cuda_device), **c.params)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    k = randn(0, 2, 64, dtype=torch.float16, device=cuda_device)
    out = ops.kv_append(k, k, c.k, c.v, c.table, ints([30, 10], cuda_device), q=q[:0], inv_freq=inv_freq(32, cuda_device), **c.params)
    assert out.shape == (0, 4, 64)
    assert ops.kv_read(c.k, c.v, c.table, ints([0, 0, 0], cuda_device), 0, **c.params)[0].shape == (0, 2, 64)


def test_many_sequences(cuda_device):
    """More sequences than lanes, several row tiles each, lengths of all kinds: the line of units is cut anywhere."""
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 700, (150,), generator=g).tolist()
    new = torch.randint(0, 6, (150,), generator=g).tolist()
    c = filled(lens, 2, 64, 16, torch.float16, 4, cuda_device)
    q, k = (randn(sum(new), h, 64, dtype=torch.float16, device=cuda_device, seed=h) for h in (10, 2))
    o, lse = attend(c, q, lens, new, cuda_device)
    ops.check_status()
    want_o, want_lse = ref.attention(c, q, lens, new)
    check(o, want_o, "o")
    check(lse, want_lse, "lse")
    live = [n >= m for n, m in zip(lens, new)]
    rows = torch.tensor([x for x, m in zip(live, new) for _ in range(m)], device=cuda_device)
    ops.kv_append(k, k, c.k, c.v, c.table, ints(lens, cuda_device), offsets(new, cuda_device), **c.params)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).to(cuda_device)
    seq = torch.tensor([b for b, m in enumerate(new) for _ in range(m)], device=cuda_device)
    at = (c.table[seq[rows], pos[rows] // 16].long(), slice(None), pos[rows] % 16)
    assert torch.equal(c.v[at], ref.encode(k[rows])[0])
    # offsets that decrease, lengths past everything: nothing outside the tensors is touched, and the call returns
    ops.fmha_paged_fwd(q, c.k, c.v, c.table, ints([2 ** 31 - 1] * 150, cuda_device), ints(list(range(150, -1, -1)), cuda_device), 5, **c.params)
    ops.kv_append(k, k, c.k.clone(), c.v.clone(), c.table, ints([2 ** 31 - 1] * 150, cuda_device), ints(list(range(150, -1, -1)), cuda_device),
                  **{n: p.clone() for n, p in c.params.items()})
    ops.kv_read(c.k, c.v, c.table, ints(list(range(150, -1, -1)), cuda_device), 200, **c.params)
    ops.check_status()


def test_operators_refuse_other_devices_and_types(cuda_device):
    c = filled([30], 2, 64, 16, torch.float16, 16, cuda_device)
    q = randn(1, 4, 64, dtype=torch.float16, device=cuda_device)
    lens = ints([30], cuda_device)
    for bad in (dict(block_table=c.table.cpu()), dict(seqlens=lens.cpu()), dict(v_cache=c.v.cpu()), dict(k_cache=c.k[..., :32], v_cache=c.v[..., :32]),
                dict(q=q[:, :, :32]), dict(q=randn(3, 2, 64, dtype=torch.float16, device=cuda_device).as_strided((1, 4, 64), (260, 65, 1))),
                dict(k_cache=c.k.transpose(2, 3)), dict(scale=-1.0)):
        args = dict(q=q, k_cache=c.k, v_cache=c.v, block_table=c.table, seqlens=lens)
        args.update(bad)
        with pytest.raises(RuntimeError):
            ops.fmha_paged_fwd(**args)
