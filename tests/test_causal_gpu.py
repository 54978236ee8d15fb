"""Causal attention of packed sequences with grouped heads (fmha_causal_varlen_fwd / _bwd / fmha_causal_varlen) against plain attention
in 64 bits, element by element (bounds: tests/reference64.py)."""
import pytest
import torch

import mha_manual  # noqa: F401
from tests import reference64 as ref64

pytestmark = pytest.mark.gpu
ops = torch.ops.mha_manual


def batch(lens, H, H_kv, D, dtype, device, seed=3, behind=0, before=0):
    g = torch.Generator(device=device).manual_seed(seed)
    rows = before + sum(lens) + behind
    q, d_o = (torch.randn(rows, H, D, device=device, dtype=dtype, generator=g) for _ in range(2))
    k, v = (torch.randn(rows, H_kv, D, device=device, dtype=dtype, generator=g) for _ in range(2))
    at = [before]
    for n in lens:
        at.append(at[-1] + n)
    return q, k, v, d_o, torch.tensor(at, dtype=torch.int32, device=device)


LENS = [[1], [2, 1, 3], [63, 64, 65], [127, 128, 129, 1], [255, 256, 257], [700, 5, 0, 131], [1100]]


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("H,H_kv", [(4, 4), (6, 2), (5, 1)])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_forward_and_gradients(cuda_device, D, dtype, H, H_kv, lens):
    q, k, v, d_o, cu = batch(lens, H, H_kv, D, dtype, cuda_device)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, max(lens))
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, max(lens))
    ops.check_status()
    ref = ref64.causal(q, k, v, lens, d_o)
    for name, x in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items():
        ref64.check(x, ref[name], name)


@pytest.mark.parametrize("D", [64, 128])
def test_many_heads_and_long_sequences(cuda_device, D):
    """Grids of several rounds: every CTA goes from item to item (at head dimension 128 in the kernel of two tiles)."""
    lens = [1500, 300, 2049, 1024, 777]
    q, k, v, d_o, cu = batch(lens, 32, 8, D, torch.bfloat16, cuda_device)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, max(lens))
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, max(lens))
    ops.check_status()
    ref = ref64.causal(q, k, v, lens, d_o)
    for name, x in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items():
        ref64.check(x, ref[name], name)
    again = ops.fmha_causal_varlen_fwd(q, k, v, cu, max(lens))
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    dq2, dk2, dv2 = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, max(lens))
    assert torch.equal(dk, dk2) and torch.equal(dv, dv2)      # summed over the group in a fixed order
    if D == 128:
        assert torch.equal(dq, dq2)


@pytest.mark.parametrize("D,H,H_kv", [(64, 8, 1), (128, 8, 1), (128, 12, 2)])
def test_few_key_heads_and_one_long_sequence(cuda_device, D, H, H_kv):
    """Query heads of a key head dealt out over items; their sums' places, and the scratch, go by rows and not by sequences times the longest."""
    lens = [3, 700, 1, 129, 0, 128, 40] + [5] * 40
    q, k, v, d_o, cu = batch(lens, H, H_kv, D, torch.bfloat16, cuda_device, before=7, behind=3)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 700)
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 700)
    used = torch.cuda.max_memory_allocated() - held
    ops.check_status()
    ref = ref64.causal(q, k, v, lens, d_o, offsets=cu[:-1].tolist())
    for name, x in dict(dq=dq, dk=dk, dv=dv).items():
        ref64.check(x[7:-3], (ref[name][0][7:-3], ref[name][1][7:-3]), name)
    tiles, rows = q.shape[0] // 128 + len(lens), 768 * len(lens)   # (rows: as many as the longest of every sequence, of dQ's sums at 64 and delta)
    assert used <= 4 * tiles * H_kv * 128 * D * 8 + rows * H * 4 * (1 + (D if D == 64 else 0)) + 3 * q.nbytes + (4 << 20)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[200, 77], [900, 40, 1300, 650] * 3], ids=["small", "large"])
def test_rows_outside_the_sequences_do_not_matter(cuda_device, D, lens):
    """Before the first and behind the last sequence lie NaNs and infinities; results are finite, and such rows come back as zeros."""
    H, H_kv = (4, 2) if len(lens) == 2 else (16, 4)
    q, k, v, d_o, cu = batch(lens, H, H_kv, D, torch.float16, cuda_device, before=37, behind=90)
    end = 37 + sum(lens)
    for x in (q, k, v, d_o):
        x[:37], x[end:] = float("nan"), float("inf")
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, max(lens))
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, max(lens))
    for x in (o, dq, dk, dv):
        assert (x[:37] == 0).all() and (x[end:] == 0).all()
    inner = slice(37, end)
    ref = ref64.causal(q[inner], k[inner], v[inner], lens, d_o[inner])
    for name, x in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        ref64.check(x[inner], ref[name], name)
    ref64.check(lse[:, inner], ref["lse"], "lse")


@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_stays_in_its_sequence(cuda_device, D):
    lens = [100, 150, 60]
    q, k, v, d_o, cu = batch(lens, 4, 2, D, torch.bfloat16, cuda_device)
    clean = ops.fmha_causal_varlen_fwd(q, k, v, cu, 150)
    for x in (q, k, v, d_o):
        x[100:250] = float("nan")
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 150)
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 150)
    for rows in (slice(0, 100), slice(250, 310)):
        assert torch.equal(o[rows], clean[0][rows])
        for x in (dq, dk, dv):
            assert torch.isfinite(x[rows]).all()


@pytest.mark.parametrize("D", [64, 128])
def test_layouts_streams_and_offsets_of_other_types(cuda_device, D):
    """Slices of one projection [rows, H + 2 H_kv, D], a gradient with stride 0, int64 offsets, another stream."""
    lens, H, H_kv = [140, 33, 290], 6, 3
    g = torch.Generator(device=cuda_device).manual_seed(4)
    x = torch.randn(sum(lens), H + 2 * H_kv, D, device=cuda_device, dtype=torch.float16, generator=g)
    q, k, v = x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:]
    cu = torch.tensor([0, 140, 173, 463], dtype=torch.int64, device=cuda_device)
    d_o = torch.randn(1, 1, D, device=cuda_device, dtype=torch.float16, generator=g).expand(sum(lens), H, D)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 290)
        dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 290)
    torch.cuda.current_stream().wait_stream(stream)
    ref = ref64.causal(q, k, v, lens, d_o)
    for name, y in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items():
        ref64.check(y, ref[name], name)


def test_scale_and_large_scores(cuda_device):
    """A scale of its own; scores of several hundred, whose softmax is nearly one key."""
    lens = [130, 520]
    q, k, v, d_o, cu = batch(lens, 4, 4, 128, torch.bfloat16, cuda_device)
    for scale in (0.02, 1.0):
        o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 520, scale)
        dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 520, scale)
        ref = ref64.causal(q, k, v, lens, d_o, scale=scale)
        for name, x in dict(o=o, dq=dq, dk=dk, dv=dv).items():
            # scale 1: scores of +-40 made of terms that add up to 90, and their rounding counts 11 times as much
            value, bound = ref[name]
            ref64.check(x, (value, bound * (1 if scale < 0.1 else 12)), f"{name} at {scale}")


@pytest.mark.parametrize("D", [64, 128])
def test_a_sequence_past_max_seqlen_is_cut(cuda_device, D):
    lens = [300, 120]
    q, k, v, d_o, cu = batch(lens, 4, 2, D, torch.float16, cuda_device)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 200)
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 200)
    ref = ref64.causal(q, k, v, [200, 120], d_o, offsets=[0, 300])
    for name, x in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        ref64.check(x, ref[name], name)
        assert (x[200:300] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_offsets_past_the_tensor(cuda_device, D):
    """Offsets that the host cannot see end at the tensor's last row; a sequence that begins before it has none."""
    q, k, v, d_o, _ = batch([400], 4, 2, D, torch.float16, cuda_device)
    cu = torch.tensor([0, 250, 900], dtype=torch.int32, device=cuda_device)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 700)
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 700)
    ref = ref64.causal(q, k, v, [250, 150], d_o)
    for name, x in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items():
        ref64.check(x, ref[name], name)
    bad = torch.tensor([-5, 100, 400], dtype=torch.int32, device=cuda_device)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, bad, 400)
    dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, bad, 400)
    ref = ref64.causal(q, k, v, [300], d_o, offsets=[100])
    for name, x in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        ref64.check(x[100:], (ref[name][0][100:], ref[name][1][100:]), name)
    ops.check_status()


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_autograd_and_differences(cuda_device, D, dtype):
    """The autograd operator gives the backward operator's gradients, and they match differences of a loss in 64 bits."""
    lens = [70, 200]
    q, k, v, d_o, cu = batch(lens, 4, 2, D, dtype, cuda_device)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = ops.fmha_causal_varlen(*leaves, cu, 200)
    grads = torch.autograd.grad(o, leaves, d_o)
    o2, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 200)
    assert torch.equal(o, o2)
    by_op = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o2, lse, cu, 200)
    for x, y in zip(grads[1:], by_op[1:]):
        assert torch.equal(x, y)

    def loss(x):   # in 64 bits
        total, r0 = 0.0, 0
        for n in lens:
            at = slice(r0, r0 + n)
            r0 += n
            s = torch.einsum("ihd,jhd->hij", x[0][at], x[1][at].repeat_interleave(2, 1)) * D ** -0.5
            s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=s.device).tril(), float("-inf"))
            total = total + (torch.einsum("hij,jhd->ihd", s.softmax(-1), x[2][at].repeat_interleave(2, 1)) * d_o[at].double()).sum()
        return total

    wide = [x.double() for x in (q, k, v)]
    g = torch.Generator(device=cuda_device).manual_seed(9)
    for i in range(3):
        step = torch.randn(wide[i].shape, device=cuda_device, dtype=torch.float64, generator=g)
        lo, hi = ([w + s * 1e-5 * step if j == i else w for j, w in enumerate(wide)] for s in (-1, 1))
        by_difference = (loss(hi) - loss(lo)) / 2e-5
        ref = ref64.causal(q, k, v, lens, d_o)[("dq", "dk", "dv")[i]]
        assert (by_difference - (ref[0] * step).sum()).abs() <= 1e-6 * (ref[0] * step).abs().sum()
        assert (by_difference - (grads[i].double() * step).sum()).abs() <= (ref[1] * step.abs()).sum() + 1e-6 * (ref[0] * step).abs().sum()


@pytest.mark.parametrize("D", [64, 128])
def test_graph_capture_of_a_step(cuda_device, D):
    lens = [150, 260]
    q, k, v, d_o, cu = batch(lens, 8, 2, D, torch.bfloat16, cuda_device)

    def step():
        o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 260)
        return (o, *ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 260))

    want = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for x in got:
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(zip(got, want)):
        if D == 128 or i != 1:
            assert torch.equal(x, y)


def test_no_rows_and_no_grad(cuda_device):
    q, k, v, d_o, cu = batch([5], 4, 2, 64, torch.float16, cuda_device)
    empty = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    o, lse = ops.fmha_causal_varlen_fwd(q[:0], k[:0], v[:0], empty, 1)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    assert [x.shape[0] for x in ops.fmha_causal_varlen_bwd(d_o[:0], q[:0], k[:0], v[:0], o, lse, empty, 1)] == [0, 0, 0]
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, empty, 5)   # one sequence without rows: all rows are outside
    assert (o == 0).all()
    with torch.inference_mode():
        assert not ops.fmha_causal_varlen(q, k, v, cu, 5).requires_grad


@pytest.mark.parametrize("D", [64, 128])
def test_one_long_document_among_many_short_ones(cuda_device, D):
    """The backward pass's scratch goes by rows; gradients at sequences that begin anywhere within a tile's rows."""
    lens, H, H_kv = [40] * 30 + [3001] + [1, 128, 127, 129, 256, 0, 60] * 8, 12, 6
    q, k, v, d_o, cu = batch(lens, H, H_kv, D, torch.float16, cuda_device, before=50, behind=9)
    o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, max(lens))
    for _ in range(2):   # (the scratch of the first call is the second one's, with what it left there)
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        dq, dk, dv = ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, max(lens))
        used = torch.cuda.max_memory_allocated() - held
        ops.check_status()
        ref = ref64.causal(q, k, v, lens, d_o, offsets=cu[:-1].tolist())
        for name, x in dict(dq=dq, dk=dk, dv=dv).items():
            ref64.check(x[50:-9], (ref[name][0][50:-9], ref[name][1][50:-9]), name)
            assert (x[:50] == 0).all() and (x[-9:] == 0).all()
        rows = q.shape[0] + 128 * len(lens)
        parts = 4 * rows * H_kv * D * 8   # at most, if a key head's query heads are dealt out
        assert used <= rows * H * 4 * (1 + (D if D == 64 else 0)) + parts + 3 * q.nbytes + (4 << 20)


@pytest.mark.parametrize("D", [64, 128])
def test_replays_start_from_clear_sums(cuda_device, D):
    """A captured forward and backward pass, replayed with other inputs: each replay's gradients, dq among them, are those of its inputs."""
    lens = [150, 260, 900]
    q, k, v, d_o, cu = batch(lens, 8, 4, D, torch.bfloat16, cuda_device)

    def step():
        o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, 900)
        return (o, *ops.fmha_causal_varlen_bwd(d_o, q, k, v, o, lse, cu, 900))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (11, 12, 13):
        for x, y in zip((q, k, v, d_o), batch(lens, 8, 4, D, torch.bfloat16, cuda_device, seed=seed)):
            x.copy_(y)
        for x in got:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        ref = ref64.causal(q, k, v, lens, d_o)
        for name, x in zip(("o", "dq", "dk", "dv"), got):
            ref64.check(x, ref[name], name)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,max_len,before,behind", [([200, 77], 200, 37, 90), ([900, 40, 1300, 650] * 3, 1300, 5, 2000), ([300, 120], 200, 0, 0), ([0], 5, 0, 300),
                                                        ([30, 0, 20], 30, 400, 500), ([2000, 700], 600, 3, 1)], ids=str)
def test_logsumexp_of_rows_outside_the_sequences(cuda_device, D, lens, max_len, before, behind):
    """-infinity, as their zeros are an empty sum: before the first and behind the last sequence, and past max_seqlen of one."""
    H, H_kv = (4, 2) if len(lens) < 5 else (16, 4)
    q, k, v, _, cu = batch(lens, H, H_kv, D, torch.bfloat16, cuda_device, before=before, behind=behind)
    for fill in (float("nan"), 3.0):
        torch.full((H, q.shape[0]), fill, device=cuda_device)   # (freed at once: what lies where the next tensors of this size are put)
        o, lse = ops.fmha_causal_varlen_fwd(q, k, v, cu, max_len)
        ops.check_status()
        live, at = torch.zeros(q.shape[0], dtype=torch.bool, device=cuda_device), before
        for n in lens:
            live[at:at + min(n, max_len)] = True
            at += n
        assert torch.isneginf(lse[:, ~live]).all() and torch.isfinite(lse[:, live]).all()
        assert (o[~live] == 0).all() and torch.isfinite(o).all()
