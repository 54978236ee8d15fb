"""The operators of autoregressive models: what a user has them do, as cases that can be timed and compared.

A case is a dict of plain values.  `path` says which entry points a pass goes through:

  prompt   torch.ops.mha_manual.fmha_causal_varlen_fwd: causal attention with grouped heads over packed prompts
  train    torch.ops.mha_manual.fmha_causal_varlen under autograd, and its gradients
  append   torch.ops.mha_manual.kv_append: new rows rotated by their positions and written into a paged cache; with a
           4-bit cache also kv_read, which gives the values that the cache holds
  read     torch.ops.mha_manual.kv_read: the rows of sequences out of a paged cache, in order, as 16-bit values
  paged    torch.ops.mha_manual.fmha_paged_fwd: a few new rows per sequence against all its rows in a paged cache

Lengths are spread evenly over [min_len, max_len], in an order drawn from the seed, so that the amount of work of a case
does not depend on the seed.  A cache is [pages, H_kv, page rows, D]; its pages are handed out in an order drawn from the seed.
A 4-bit cache holds two codes a byte and, for every 32 values of a row, a scale s and a base b in fp16: a code c stands for
b + s (1 + c / 16).
"""
import math
import random

import torch

own = False   # whether `run` makes the calls of this package; else it computes the same in elementary operations

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32          # values of a row that share a scale and a base
LIMIT4 = 20000.0    # values beyond it are held as it in 4 bits: scale and base then fit fp16


def _case(path, B, H, H_kv, D, dtype, min_len, max_len, page=0, bits=16, new=0, interleaved=False):
    return {"path": path, "B": B, "H": H, "H_kv": H_kv, "D": D, "dtype": dtype, "min_len": min_len, "max_len": max_len,
            "page": page, "bits": bits, "new": new, "interleaved": interleaved}


def listed():
    cases = [
        # a batch of long prompts, grouped heads: the largest
        ("prompt_long", _case("prompt", 4, 32, 8, 128, "bf16", 1500, 4096)),
        # many short and ragged prompts, head dimension 64
        ("prompt_ragged", _case("prompt", 11, 16, 4, 64, "fp16", 33, 900)),
        # a training step on packed documents, grouped heads
        ("train_grouped", _case("train", 6, 16, 4, 128, "bf16", 300, 2048)),
        # a training step with a key head per query head, head dimension 64, odd lengths
        ("train_plain_heads", _case("train", 13, 12, 12, 64, "fp16", 61, 1021)),
        # one decoding step's new rows: launches and latency
        ("append_step", _case("append", 64, 32, 8, 128, "bf16", 512, 4096, page=64, new=1)),
        # whole prompts into a cache of small pages
        ("append_prompt", _case("append", 8, 32, 8, 128, "bf16", 300, 2048, page=16, interleaved=True)),
        # whole prompts into a 4-bit cache, and the values it then holds
        ("append_4bit", _case("append", 5, 16, 4, 64, "fp16", 129, 2000, page=32, bits=4)),
        # sequences read back out of a 16-bit cache
        ("read_16bit", _case("read", 6, 32, 8, 128, "bf16", 200, 3000, page=64)),
        # sequences read back out of a 4-bit cache
        ("read_4bit", _case("read", 9, 16, 4, 64, "fp16", 100, 1700, page=16, bits=4)),
        # a few drafted rows per sequence against a 16-bit cache
        ("paged_drafts", _case("paged", 16, 32, 8, 128, "bf16", 200, 4000, page=16, new=4)),
        # a decoding step of a batch against a 4-bit cache
        ("paged_4bit_batch", _case("paged", 32, 32, 8, 128, "bf16", 1000, 8192, page=64, bits=4, new=1)),
        # two requests with very long contexts, 4 bits
        ("paged_4bit_long", _case("paged", 2, 32, 8, 128, "fp16", 90001, 131072, page=64, bits=4, new=1)),
    ]
    return [dict(c, name=name) for name, c in cases]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: a path drawn evenly, its sizes spread over the logarithm of that path's range."""
    path = rng.choice(("prompt", "prompt", "train", "append", "read", "paged", "paged", "paged"))
    heads = [(h, k) for h in (8, 12, 16, 32) for k in (1, 2, 4, 8, 12, 16) if h % k == 0 and h // k <= 16]
    bits = rng.choice((16, 4)) if path in ("append", "read", "paged") else 16
    page = rng.choice((16, 32, 64, 128, 48)) if path in ("append", "read", "paged") else 0
    most = {c["path"]: work(c) for c in listed() if c["name"] in ("prompt_long", "train_grouped", "append_prompt", "read_16bit", "paged_4bit_long")}
    while True:
        H, H_kv = rng.choice(heads)
        D, dtype = rng.choice((64, 128)), rng.choice(("fp16", "bf16"))
        new = 0
        if path == "prompt":
            B, hi = _log_int(rng, 1, 32), _log_int(rng, 1, 8000)
        elif path == "train":
            B, hi = _log_int(rng, 1, 24), _log_int(rng, 2, 4000)
        elif path == "append":
            B, hi = _log_int(rng, 1, 128), _log_int(rng, 1, 4000)
            new = rng.choice((0, 1, _log_int(rng, 1, 8)))
        elif path == "read":
            B, hi = _log_int(rng, 1, 32), _log_int(rng, 1, 6000)
        else:
            B, hi = _log_int(rng, 1, 96), _log_int(rng, 8, 100000)
            new = rng.choice((1, 1, _log_int(rng, 1, 8)))
        lo = max(1, new, int(hi * rng.uniform(0.2, 1.0)))
        c = _case(path, B, H, H_kv, D, dtype, lo, max(lo, hi), page, bits, new, rng.random() < 0.3)
        w, m = work(c), most[path]
        scores = B * H * max(lo, hi) ** 2 if path in ("prompt", "train") else 0   # of the padded plain form
        # the rows of the caches, unpacked, and those scores stay as large as the largest listed case's
        rows = B * H_kv * D * max(lo, hi) * (H // H_kv if path == "paged" else 1)
        if w["flops"] <= m["flops"] and w["bytes"] <= m["bytes"] and scores <= (4 if path == "prompt" else 1.2) * 5e8 and rows <= 1.1e9:
            return c


def _lengths(case):
    """Rows of the sequences (of a paged cache: with the new ones), before they are put in an order."""
    B, lo, hi = case["B"], case["min_len"], case["max_len"]
    return [hi] if B == 1 else [lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _inv_freq(D):
    return (10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)).float()


def prepare(case, seed):
    B, H, H_kv, D, page = (case[n] for n in ("B", "H", "H_kv", "D", "page"))
    path, dtype = case["path"], DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)

    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    s = {"case": dict(case), "max_len": max(lens)}
    dev = dict(dtype=torch.int32, device="cuda")
    new = lens if case["new"] == 0 else [case["new"]] * B   # rows of q (paged), of q, k and v (append)
    cu = [0]
    for n in lens if path in ("prompt", "train", "read") else new:
        cu.append(cu[-1] + n)
    s["cu"], s["total"], s["max_new"] = torch.tensor(cu, **dev), cu[-1], max(new)
    all_rows = [0]
    for n in lens:
        all_rows.append(all_rows[-1] + n)
    s["cu_all"], s["total_all"] = torch.tensor(all_rows, **dev), all_rows[-1]
    if path in ("prompt", "train"):
        s["q"], s["k"], s["v"] = normal(cu[-1], H, D), normal(cu[-1], H_kv, D), normal(cu[-1], H_kv, D)
        if path == "train":
            s["d_o"] = normal(cu[-1], H, D)
            for n in "qkv":
                s[n].requires_grad_()
        return s
    s["lens"] = torch.tensor(lens, **dev)
    width = -(-max(lens) // page)
    n_pages = B * width + 3
    s["table"] = torch.randperm(n_pages, device="cuda", generator=g)[:B * width].reshape(B, width).int()
    s["k_params"] = s["v_params"] = None
    if path == "append":
        s["q"], s["k"], s["v"] = normal(cu[-1], H, D), normal(cu[-1], H_kv, D), normal(cu[-1], H_kv, D)
        s["inv_freq"] = _inv_freq(D)
    elif path == "paged":
        s["q"] = normal(cu[-1], H, D)
    shape = (n_pages, H_kv, page)
    for n in "kv":
        if case["bits"] == 16:
            s[n + "_cache"] = normal(*shape, D)
        else:   # rows of N(0,1) values span some four units in 32 of them
            s[n + "_cache"] = torch.randint(0, 256, (*shape, D // 2), device="cuda", dtype=torch.uint8, generator=g)
            scale = torch.rand(*shape, D // GROUP, device="cuda", generator=g) * 2.5 + 3.5
            s[n + "_params"] = torch.stack((scale, -1.5 * scale + 0.3 * torch.randn(scale.shape, device="cuda", generator=g)), -1).half()
    return s


def run(s):
    c = s["case"]
    path = c["path"]
    if own:
        import mha_manual  # noqa: F401  registers torch.ops.mha_manual.*
        ops = torch.ops.mha_manual
        if path == "prompt":
            return ops.fmha_causal_varlen_fwd(s["q"], s["k"], s["v"], s["cu"], s["max_len"])
        if path == "train":
            o = ops.fmha_causal_varlen(s["q"], s["k"], s["v"], s["cu"], s["max_len"])
            return (o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["d_o"]))
        if path == "paged":
            cu = None if c["new"] == 1 else s["cu"]
            return ops.fmha_paged_fwd(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], cu, s["max_new"],
                                      k_params=s["k_params"], v_params=s["v_params"])
        if path == "append":
            cu = None if c["new"] == 1 else s["cu"]
            q = ops.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], cu, q=s["q"],
                              inv_freq=s["inv_freq"], interleaved=c["interleaved"], k_params=s["k_params"], v_params=s["v_params"])
            if c["bits"] == 16:
                return q, s["k_cache"], s["v_cache"]
        rows = ops.kv_read(s["k_cache"], s["v_cache"], s["table"], s["cu_all"], s["total_all"], k_params=s["k_params"],
                           v_params=s["v_params"], bf16=c["dtype"] == "bf16")
        return (q, *rows) if path == "append" else rows
    if path == "prompt":
        o, lse = _attention(s["q"].float(), s["k"].float(), s["v"].float(), s["cu"], s["max_len"])
        return o.to(s["q"].dtype), lse
    if path == "train":
        q, k, v = (s[n].detach().float().requires_grad_() for n in "qkv")
        o, _ = _attention(q, k, v, s["cu"], s["max_len"])
        grads = torch.autograd.grad(o, (q, k, v), s["d_o"].float())
        return tuple(x.to(s["q"].dtype) for x in (o.detach(), *grads))
    if path == "paged":
        return _paged(s)
    if path == "append":
        seq, row = _places(s["cu"], s["total"])
        pos = s["lens"][seq] - (s["cu"][1:] - s["cu"][:-1])[seq] + row
        q, k = (_rotated(s[n], pos, s["inv_freq"], c["interleaved"]) for n in "qk")
        where = (s["table"][seq, pos // c["page"]].long(), slice(None), (pos % c["page"]).long())
        if c["bits"] == 16:
            s["k_cache"][where], s["v_cache"][where] = k, s["v"]
            return q, s["k_cache"], s["v_cache"]
        s["k_cache"][where], s["k_params"][where] = _to4(k)
        s["v_cache"][where], s["v_params"][where] = _to4(s["v"])
    seq, row = _places(s["cu_all"], s["total_all"])
    where = (s["table"][seq, row // c["page"]].long(), slice(None), (row % c["page"]).long())
    rows = tuple(_values(s[n + "_cache"][where], None if c["bits"] == 16 else s[n + "_params"][where], DTYPES[c["dtype"]]) for n in "kv")
    return (q, *rows) if path == "append" else rows


def _places(cu, total):
    """Sequence and row within it of every packed row."""
    at = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    return seq, at - cu[seq]


def _attention(q, k, v, cu, max_len):
    """Causal attention over packed sequences, in 32 bits on padded copies."""
    (total, H, D), H_kv, B = q.shape, k.shape[1], cu.numel() - 1
    seq, row = _places(cu, total)

    def padded(x):   # [B, heads, max_len, D]
        return x.new_zeros(B, max_len, x.shape[1], D).index_put((seq, row), x).transpose(1, 2)

    qp = padded(q).unflatten(1, (H_kv, H // H_kv)) * D ** -0.5
    scores = qp @ padded(k).transpose(-1, -2).unsqueeze(2)
    later = torch.ones(max_len, max_len, dtype=torch.bool, device=q.device).triu(1)
    scores = scores.masked_fill(later, -math.inf)
    lse = torch.logsumexp(scores, -1)
    o = ((scores - lse[..., None]).exp() @ padded(v).unsqueeze(2)).flatten(1, 2)
    return o.transpose(1, 2)[seq, row], lse.flatten(1, 2).transpose(1, 2)[seq, row].T.contiguous()


def _rotated(x, pos, inv_freq, interleaved):
    """x [rows, heads, D] rotated by angles pos * inv_freq, in pairs (i, i + D/2) or (2i, 2i + 1)."""
    angle = (pos.double()[:, None] * inv_freq.double())[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    f = x.float()
    a, b = (f[..., ::2], f[..., 1::2]) if interleaved else f.chunk(2, -1)
    y = (a * cos - b * sin, b * cos + a * sin)
    return (torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)).to(x.dtype)


def _to4(x):
    """Codes [..., D/2] and (scale, base) [..., D/32, 2] of 16-bit values."""
    f = x.float().clamp(-LIMIT4, LIMIT4).unflatten(-1, (-1, GROUP))
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    scale = ((hi - lo) * (16.0 / 15.0)).half().float()
    base = (lo - scale).half().float()
    c = torch.where(scale > 0, (((f - base) / scale - 1.0) * 16.0).round().clamp(0, 15), 0.0)
    c = c.flatten(-2).to(torch.uint8)
    return c[..., ::2] | c[..., 1::2] << 4, torch.cat((scale, base), -1).half()


def _values(codes, params, dtype):
    """What cache rows hold, in `dtype` (None: 32 bits)."""
    if params is None:
        return codes.float() if dtype is None else codes
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    scale, base = params.float().unsqueeze(-1).unbind(-2)
    x = (base + scale * (1.0 + c / 16.0)).flatten(-2)
    return x if dtype is None else x.to(dtype)


def _paged(s):
    """Attention of new rows over a paged cache, in 32 bits on the pages put side by side."""
    c = s["case"]
    B, H, H_kv, D, T = (c[n] for n in ("B", "H", "H_kv", "D", "new"))
    table = s["table"].long()

    def rows(n):   # [B, H_kv, width * page, D]
        x = _values(s[n + "_cache"][table], None if c["bits"] == 16 else s[n + "_params"][table], None)
        return x.transpose(1, 2).flatten(2, 3)

    q = s["q"].float().reshape(B, T, H_kv, H // H_kv, D).permute(0, 2, 3, 1, 4) * D ** -0.5   # [B, H_kv, group, T, D]
    scores = q.flatten(2, 3) @ rows("k").transpose(-1, -2)
    last = s["lens"][:, None] - T + torch.arange(T, device="cuda")                             # the last row each one sees
    hidden = torch.arange(scores.shape[-1], device="cuda") > last[..., None]                   # [B, T, rows]
    scores = scores.unflatten(2, (-1, T)).masked_fill(hidden[:, None, None], -math.inf)
    lse = torch.logsumexp(scores, -1)
    o = (scores - lse[..., None]).exp().flatten(2, 3) @ rows("v")
    o = o.unflatten(2, (-1, T)).permute(0, 3, 1, 2, 4).reshape(B * T, H, D)
    return o.to(s["q"].dtype), lse.permute(1, 2, 0, 3).reshape(H, B * T)


def work(case):
    """Each input read once, each output written once; only scores that count are formed (4 D flops each forward, 10 D backward)."""
    B, H, H_kv, D, path = (case[n] for n in ("B", "H", "H_kv", "D", "path"))
    lens = _lengths(case)
    total = sum(lens)
    cached = 2 * D if case["bits"] == 16 else D // 2 + D // GROUP * 4      # bytes of a row of one head in the cache
    if path in ("prompt", "train"):
        scores = H * sum(n * (n + 1) // 2 for n in lens)
        if path == "prompt":
            return {"bytes": 2 * D * total * (2 * H + 2 * H_kv) + 4 * H * total, "flops": 4 * D * scores}
        return {"bytes": 2 * D * total * (4 * H + 4 * H_kv), "flops": 14 * D * scores}
    if path == "read":
        return {"bytes": 2 * total * H_kv * (cached + 2 * D), "flops": 0}
    new = total if case["new"] == 0 else B * case["new"]
    if path == "append":
        read_back = 2 * total * H_kv * (cached + 2 * D) if case["bits"] == 4 else 0
        return {"bytes": 2 * 2 * D * new * H + 2 * new * H_kv * (2 * D + cached) + read_back, "flops": 3 * D * new * (H + H_kv)}
    T = case["new"]
    seen = sum(n - T + t + 1 for n in lens for t in range(T))
    return {"bytes": 2 * total * H_kv * cached + 2 * 2 * D * new * H + 4 * H * new, "flops": 4 * D * H * seen}


def exact(case, seed):
    """What `run` returns, in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    c = case
    B, H, H_kv, D, page, path = (c[n] for n in ("B", "H", "H_kv", "D", "page", "path"))
    G, cu = H // H_kv, s["cu"].tolist()
    with torch.no_grad():
        if path in ("prompt", "train"):
            o = torch.zeros(cu[-1], H, D, dtype=torch.float64, device="cuda")
            lse = torch.zeros(H, cu[-1], dtype=torch.float64, device="cuda")
            grads = [torch.zeros_like(s[n], dtype=torch.float64) for n in "qkv"]
            for b in range(B):
                at = slice(cu[b], cu[b + 1])
                n = cu[b + 1] - cu[b]
                seen = torch.ones(n, n, dtype=torch.float64, device="cuda").tril()
                for h in range(H):
                    q, k, v = s["q"][at, h].double(), s["k"][at, h // G].double(), s["v"][at, h // G].double()
                    x = torch.einsum("id,jd->ij", q, k) / math.sqrt(D)
                    top = torch.where(seen > 0, x, -math.inf).max(1, keepdim=True).values
                    e = torch.exp(torch.minimum(x - top, torch.zeros_like(x))) * seen
                    total = e.sum(1, keepdim=True)
                    p = e / total
                    o[at, h], lse[h, at] = p @ v, (top + total.log())[:, 0]
                    if path == "train":
                        do = s["d_o"][at, h].double()
                        dp = do @ v.T
                        dx = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
                        grads[0][at, h] = dx @ k
                        grads[1][at, h // G] += dx.T @ q
                        grads[2][at, h // G] += p.T @ do
            return (o, lse) if path == "prompt" else (o, *grads)
        lens, table = s["lens"].tolist(), s["table"].tolist()

        def held(n, b, rows):   # [rows, H_kv, D] of sequence b
            pages = torch.tensor(table[b][:-(-rows // page)], device="cuda")
            x = s[n + "_cache"][pages]
            if c["bits"] == 16:
                x = x.double()
            else:
                par = s[n + "_params"][pages].double().repeat_interleave(GROUP, dim=3)
                code = torch.empty(*x.shape[:3], D, dtype=torch.float64, device="cuda")
                code[..., 0::2], code[..., 1::2] = (x % 16).double(), (x // 16).double()
                x = par[..., 1] + par[..., 0] * (16.0 + code) / 16.0
            return x.permute(0, 2, 1, 3).reshape(-1, H_kv, D)[:rows]

        if path == "read":
            return tuple(torch.cat([held(n, b, cu[b + 1] - cu[b]) for b in range(B)]) for n in "kv")
        if path == "append":
            pos = torch.cat([torch.arange(lens[b] - (cu[b + 1] - cu[b]), lens[b], device="cuda", dtype=torch.float64) for b in range(B)])
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(pos, s["inv_freq"].double()))[:, None]

            def rotated(x):
                x = x.double()
                z = torch.complex(x[..., ::2], x[..., 1::2]) if c["interleaved"] else torch.complex(x[..., :D // 2], x[..., D // 2:])
                z = z * turn
                return torch.view_as_real(z).flatten(-2) if c["interleaved"] else torch.cat((z.real, z.imag), -1)

            q, k, v = rotated(s["q"]), rotated(s["k"]), s["v"].double()
            if c["bits"] == 4:   # four bits stand for the nearest of sixteen values, not for the row itself
                return q, None, None
            caches = [s[n + "_cache"].double() for n in "kv"]
            for b in range(B):
                for r in range(cu[b], cu[b + 1]):
                    p = lens[b] - (cu[b + 1] - cu[b]) + r - cu[b]
                    caches[0][table[b][p // page], :, p % page], caches[1][table[b][p // page], :, p % page] = k[r], v[r]
            return (q, *caches)
        T = c["new"]
        o = torch.zeros(B * T, H, D, dtype=torch.float64, device="cuda")
        lse = torch.zeros(H, B * T, dtype=torch.float64, device="cuda")
        for b in range(B):
            k, v = held("k", b, lens[b]), held("v", b, lens[b])
            for t in range(T):
                n = lens[b] - T + t + 1
                x = torch.einsum("hgd,jhd->hgj", s["q"][b * T + t].double().reshape(H_kv, G, D), k[:n]) / math.sqrt(D)
                top = x.amax(-1, keepdim=True)
                e = torch.exp(x - top)
                o[b * T + t] = (torch.einsum("hgj,jhd->hgd", e, v[:n]) / e.sum(-1, keepdim=True)).reshape(H, D)
                lse[:, b * T + t] = (top + e.sum(-1, keepdim=True).log()).reshape(H)
        return o, lse
