"""A paged cache in plain torch: where rows lie, what 4 bits stand for, attention over it in 64 bits with the bounds of its roundings."""
import torch

from tests.reference64 import SLACK, half_ulp, tiny

GROUP = 32


class Cache:
    """k and v of B sequences in pages handed out at random.  layout: "pages" [pages, H, rows, D], "rows" [pages, rows, H, D] seen as the former,
    "joint" k and v of a page side by side.  What no row has been put into holds NaNs (4 bits: any codes, NaN scales)."""

    def __init__(self, B, width, H_kv, D, page, dtype, bits, device, seed=5, layout="pages", spare=3):
        g = torch.Generator(device=device).manual_seed(seed)
        n = B * width + spare
        self.B, self.H, self.D, self.page, self.bits, self.dtype, self.n = B, H_kv, D, page, bits, dtype, n
        self.table = torch.randperm(n, device=device, generator=g)[:B * width].reshape(B, width).int()
        cols = D if bits == 16 else D // 2

        def make():
            shape = {"pages": (n, H_kv, page, cols), "rows": (n, page, H_kv, cols), "joint": (n, 2, H_kv, page, cols)}[layout]
            if bits == 16:
                return torch.full(shape, float("nan"), dtype=dtype, device=device)
            return torch.randint(0, 256, shape, dtype=torch.uint8, device=device, generator=g)

        if layout == "joint":
            both = make()
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = (make() if layout == "pages" else make().transpose(1, 2) for _ in range(2))
        self.params = {}
        if bits == 4:
            self.params = {n + "_params": torch.full((self.n, H_kv, page, D // GROUP, 2), float("nan"), dtype=torch.float16, device=device) for n in "kv"}

    def where(self, b, pos):
        return self.table[b, pos // self.page].long(), slice(None), pos % self.page

    def put(self, b, pos, k, v):
        """Rows [n, H, D] of sequence b at positions `pos` [n]."""
        at = self.where(b, pos)
        for name, x in (("k", k), ("v", v)):
            if self.bits == 16:
                getattr(self, name)[at] = x
            else:
                getattr(self, name)[at], self.params[name + "_params"][at] = encode(x)

    def rows(self, name, b, n):
        """The first n rows of sequence b [n, H, D] in 64 bits: their values, what these are sums of in absolute values, and the part of that in which
        P has been multiplied by a scale and rounded again (4 bits)."""
        at = self.where(b, torch.arange(n, device=self.k.device))
        x = getattr(self, name)[at]
        if self.bits == 16:
            return x.double(), x.double().abs(), torch.zeros_like(x, dtype=torch.float64)
        c, s, base = decode_parts(x, self.params[name + "_params"][at])
        by_code = (s * c / 16).flatten(-2)
        return (base + s * (1 + c / 16)).flatten(-2), (base.abs() + s + s * c / 16).flatten(-2), by_code


def encode(x):
    """Codes and (scale, base) by the definition, in 32 bits operation by operation."""
    f = x.float().unflatten(-1, (-1, GROUP))
    bad = ~torch.isfinite(f).all(-1, keepdim=True)
    f = f.clamp(-20000.0, 20000.0)
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    s = ((hi - lo) * (16.0 / 15.0)).half().float()
    base = (lo - s).half().float()
    c = torch.where((s > 0) & ~bad, (((f - base) / s - 1.0) * 16.0).round().clamp(0, 15), 0.0).flatten(-2).to(torch.uint8)
    params = torch.cat((s, base), -1).masked_fill(bad, float("nan"))
    return c[..., ::2] | c[..., 1::2] << 4, params.half()


def decode_parts(codes, params):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
    s, base = params.double().unsqueeze(-1).unbind(-2)
    return c, s, base


def attention(cache, q, lens, new, scale=None):
    """(o, bound), (lse, bound) for packed rows q [sum(new), H, D]: the i-th new row of n sees lens[b] - n + i + 1 keys."""
    rows, H, D = q.shape
    G = H // cache.H
    scale = D ** -0.5 if scale is None else scale
    u = half_ulp(q.dtype)
    up = half_ulp(torch.float16 if cache.bits == 4 else q.dtype)   # P's type
    tp = tiny(torch.float16 if cache.bits == 4 else q.dtype)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    o, ob = zeros(rows, H, D), zeros(rows, H, D)
    lse, lb = torch.full((H, rows), float("-inf"), dtype=torch.float64, device=q.device), zeros(H, rows)
    r = 0
    for b, n in enumerate(new):
        total = max(lens[b], 0)
        if total:
            k = cache.rows("k", b, total)[0]
            v, v_abs, v_twice = cache.rows("v", b, total)
        for i in range(n):
            seen = lens[b] - n + i + 1
            if seen > 0:
                qq = q[r].double().reshape(cache.H, G, D)
                s = torch.einsum("hgd,jhd->hgj", qq, k[:seen]) * scale
                top = torch.logsumexp(s, -1, keepdim=True)
                p = (s - top).exp()
                out = torch.einsum("hgj,jhd->hgd", p, v[:seen])
                e = (torch.einsum("hgj,jhd->hgd", (up + SLACK) * p + tp, v_abs[:seen]) + up * torch.einsum("hgj,jhd->hgd", p, v_twice[:seen]) +
                     seen * tp * (cache.bits == 4) + u * out.abs())
                o[r], ob[r] = out.reshape(H, D), 1.01 * e.reshape(H, D)
                lse[:, r], lb[:, r] = top.reshape(H), 2.0 ** -12
            r += 1
    return (o, ob), (lse, lb)


def rotate(x, pos, inv_freq, interleaved):
    """(value, bound) of x [n, H, D] rotated by positions pos [n]."""
    y = x.double().clone()
    n = inv_freq.numel()
    angle = (pos.double()[:, None] * inv_freq.double())[:, None]
    c, s = angle.cos(), angle.sin()
    a = x[..., :2 * n:2].double() if interleaved else x[..., :n].double()
    b = x[..., 1:2 * n:2].double() if interleaved else x[..., n:2 * n].double()
    size = torch.zeros_like(y)
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one] = size[..., two] = a.abs() + b.abs()
    # cosine, sine, two products and a sum are rounded to 24 bits, the result to 16
    return y, torch.where(size > 0, half_ulp(x.dtype) * y.abs() + 2.0 ** -21 * size, 0.0)
