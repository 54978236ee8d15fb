"""The operators of autoregressive models in torch.compile and fake-tensor tracing (no GPU: meta tensors), and what kv_append tells autograd."""
import pytest
import torch

import mha_manual  # noqa: F401

ops = torch.ops.mha_manual
INT = dict(dtype=torch.int32)


def meta(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def caches(bits):
    if bits == 16:
        return meta(10, 2, 32, 128), meta(10, 2, 32, 128), {}
    return (meta(10, 2, 32, 64, dtype=torch.uint8), meta(10, 2, 32, 64, dtype=torch.uint8),
            dict(k_params=meta(10, 2, 32, 4, 2), v_params=meta(10, 2, 32, 4, 2)))


def compiled(f):
    torch._dynamo.reset()
    return torch.compile(f, fullgraph=True, backend="aot_eager")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("with_q", [True, False])
def test_a_step_with_append_compiles(bits, with_q):
    k_cache, v_cache, params = caches(bits)
    q, k, freq = meta(3, 6, 128), meta(3, 2, 128), meta(64, dtype=torch.float32)

    def step(q, k, k_cache, v_cache, table, lens, params):
        turned = ops.kv_append(k, k, k_cache, v_cache, table, lens, q=q if with_q else None, inv_freq=freq, **params)
        o, lse = ops.fmha_paged_fwd(turned if with_q else q, k_cache, v_cache, table, lens, **params)
        return o + 1, lse

    with torch.no_grad():
        o, lse = compiled(step)(q, k, k_cache, v_cache, meta(3, 4, **INT), meta(3, **INT), params)
    assert o.shape == q.shape and lse.shape == (6, 3)


@pytest.mark.parametrize("bits", [16, 4])
def test_reading_and_attention_compile(bits):
    k_cache, v_cache, params = caches(bits)

    def step(table, cu):
        k, v = ops.kv_read(k_cache, v_cache, table, cu, 50, **params)
        return k + v

    assert compiled(step)(meta(3, 4, **INT), meta(4, **INT)).shape == (50, 2, 128)


def test_causal_attention_compiles_with_its_gradients():
    q, k, cu = meta(40, 8, 128).requires_grad_(), meta(40, 2, 128).requires_grad_(), meta(4, **INT)
    f = compiled(lambda q, k, cu: ops.fmha_causal_varlen(q * 2, k, k, cu, 20).sum())
    f(q, k, cu).backward()
    assert q.grad.shape == q.shape and k.grad.shape == k.shape
    o, lse = compiled(lambda q, k, cu: ops.fmha_causal_varlen_fwd(q, k, k, cu, 20))(q.detach(), k.detach(), cu)
    assert o.shape == q.shape and lse.shape == (8, 40)


def test_changing_batches_compile_once_more():
    """Numbers of rows, sequences and pages that change from call to call are symbols after the second: no compilation for each."""
    from torch._dynamo.testing import CompileCounterWithBackend

    def step(q, k, k_cache, v_cache, table, lens):
        turned = ops.kv_append(k, k, k_cache, v_cache, table, lens, q=q)
        return ops.fmha_paged_fwd(turned, k_cache, v_cache, table, lens)[0]

    def train(q, k, cu):
        return ops.fmha_causal_varlen(q, k, k, cu, 20)

    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    f = torch.compile(step, fullgraph=True, backend=counter)
    with torch.no_grad():
        for B, pages, width in ((3, 10, 4), (5, 20, 6), (7, 35, 9), (11, 50, 10), (6, 31, 7)):
            cache = meta(pages, 2, 32, 128)
            assert f(meta(B, 6, 128), meta(B, 2, 128), cache, cache.clone(), meta(B, width, **INT), meta(B, **INT)).shape == (B, 6, 128)
    assert counter.frame_count == 2
    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    f = torch.compile(train, fullgraph=True, backend=counter)
    for B, rows in ((2, 40), (3, 50), (7, 90), (9, 33)):
        q, k = meta(rows, 8, 64).requires_grad_(), meta(rows, 2, 64).requires_grad_()
        f(q, k, meta(B + 1, **INT)).sum().backward()
        assert q.grad.shape == q.shape and k.grad.shape == k.shape
    assert counter.frame_count == 2


@pytest.mark.parametrize("bits", [16, 4])
def test_append_counts_as_a_write(bits):
    """The version counters of what is written move, so that autograd notices; of what is not, they do not."""
    k_cache, v_cache, params = caches(bits)
    k, q, table, lens = meta(3, 2, 128), meta(3, 6, 128), meta(3, 4, **INT), meta(3, **INT)
    written, read = (k_cache, v_cache, *params.values()), (k, q, table, lens)
    for kw in (dict(), dict(q=q)):
        before = [x._version for x in written], [x._version for x in read]
        assert (ops.kv_append(k, k, k_cache, v_cache, table, lens, **kw, **params) is None) == (not kw)
        assert all(x._version > n for x, n in zip(written, before[0]))
        assert [x._version for x in read] == before[1]
    with torch.inference_mode():
        ops.kv_append(k, k, k_cache, v_cache, table, lens, **params)
        c = caches(bits)
    with torch.no_grad():   # made in inference mode: no counter to move
        ops.kv_append(k, k, c[0], c[1], table, lens, q=q, **c[2])


def test_append_refuses_caches_that_want_gradients():
    k, table, lens = meta(3, 2, 128), meta(3, 4, **INT), meta(3, **INT)
    for bits, i in ((16, "k_cache"), (16, "v_cache"), (4, "k_params"), (4, "v_params")):
        k_cache, v_cache, c = caches(bits)
        c.update(k_cache=k_cache, v_cache=v_cache)
        c[i].requires_grad_()
        for kw in (dict(), dict(q=k)):
            with pytest.raises(RuntimeError, match="requires gradients"):
                ops.kv_append(k, k, block_table=table, seqlens=lens, **c, **kw)
            with torch.no_grad():
                ops.kv_append(k, k, block_table=table, seqlens=lens, **c, **kw)


def test_append_of_rows_that_want_gradients():
    """They are written as values; the rotated q has no gradient to give, and says so where one is asked for."""
    k_cache, v_cache, _ = caches(16)
    k, q = meta(3, 2, 128).requires_grad_(), meta(3, 6, 128).requires_grad_()
    ops.kv_append(k, k, k_cache, v_cache, meta(3, 4, **INT), meta(3, **INT), q=q)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("with_q", [True, False])
def test_a_compiled_step_writes_the_caches(cuda_device, bits, with_q):
    """Appending and attending, compiled and not, from the same caches: the same results and the same caches afterwards."""
    from tests import cache_reference as ref
    g = torch.Generator(device=cuda_device).manual_seed(2)
    lens = torch.tensor([40, 7, 64], dtype=torch.int32, device=cuda_device)
    q, k, v = (torch.randn(3, h, 128, device=cuda_device, dtype=torch.float16, generator=g) for h in (6, 2, 2))
    freq = torch.rand(64, device=cuda_device, generator=g)

    def step(k_cache, v_cache, table, params):
        turned = ops.kv_append(k, v, k_cache, v_cache, table, lens, q=q if with_q else None, inv_freq=freq, **params)
        return ops.fmha_paged_fwd(turned if with_q else q, k_cache, v_cache, table, lens, **params)

    results = []
    for f in (step, compiled(step)):
        c = ref.Cache(3, 2, 2, 128, 32, torch.float16, bits, cuda_device)
        for b, n in enumerate(lens.tolist()):
            rows = torch.randn(n, 2, 128, device=cuda_device, dtype=torch.float16, generator=torch.Generator(device=cuda_device).manual_seed(b))
            c.put(b, torch.arange(n, device=cuda_device), rows, rows)
        with torch.no_grad():
            out = f(c.k, c.v, c.table, c.params)
        results.append([x.view(torch.uint8) for x in (*out, c.k, c.v, *c.params.values())])
    for x, y in zip(*results):
        assert torch.equal(x, y)
