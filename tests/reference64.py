"""Plain attention in 64 bits, sequence by sequence and head by head, and how far a kernel may be from it.

Bounds, element by element, from the roundings a kernel makes (u = half a unit in the last place of its 16-bit type):
  o   P is rounded to 16 bits before P V, O once at the end:          u P|V| + u |o|
  dv  likewise:                                                       u P^T|dO| + u |dv|
  dq  dS is rounded to 16 bits, delta is formed from O as stored:     scale (u |dS| + u P rowsum|dO O|) |K| + u |dq|,  dk likewise
plus `SLACK` times the same sums of absolute values for what is done in 32 bits: a score is a sum of up to 128 products, whose rounding
(128 additions, 2^-24 each, of terms that add up to about 8 in absolute value) is the largest of it, 2^-14 of P; the exponential, the argument's
rounding and the sums over keys add less than that again.  In fp16 values below 2^-14 have an absolute rounding of up to 2^-25, which counts for
P and dS with every key (rescaled P is at least as large as P)."""
import torch

SLACK = 2.0 ** -13


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def causal(q, k, v, lens, d_o=None, scale=None, offsets=None):
    """Per output: (value, bound).  q [rows, H, D]; k, v [rows, H_kv, D]; rows outside the sequences stay zero, with bound zero."""
    dt, dev = q.dtype, q.device
    u, t = half_ulp(dt), tiny(dt)
    rows, H, D = q.shape
    G = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=dev)  # noqa: E731
    out = {"o": [zeros(q), zeros(q)], "lse": [torch.full((H, rows), float("nan"), dtype=torch.float64, device=dev)]}
    if d_o is not None:
        out.update(dq=[zeros(q), zeros(q)], dk=[zeros(k), zeros(k)], dv=[zeros(v), zeros(v)])
    r0 = 0
    for b, n in enumerate(lens):
        if offsets is not None:
            r0 = offsets[b]
        at = slice(r0, r0 + n)
        r0 += n
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device=dev).tril()
        for h in range(H):
            Q, K, V = q[at, h].double(), k[at, h // G].double(), v[at, h // G].double()
            s = (Q @ K.T * scale).masked_fill(~seen, float("-inf"))
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = (s - lse).exp()
            o = p @ V
            out["o"][0][at, h] = o
            out["o"][1][at, h] = (u + SLACK) * (p @ V.abs()) + u * o.abs() + t * (seen.double() @ V.abs())
            out["lse"][0][h, at] = lse[:, 0]
            if d_o is None:
                continue
            dO = d_o[at, h].double()
            dp = dO @ V.T
            dp_abs = dO.abs() @ V.abs().T
            delta, delta_abs = (dO * o).sum(1, keepdim=True), (dO * o).abs().sum(1, keepdim=True)
            ds = p * (dp - delta)
            e = u * ds.abs() + p * u * delta_abs + SLACK * p * (dp_abs + delta_abs) + t * seen.double()
            dq, dk, dv = ds @ K * scale, ds.T @ Q * scale, p.T @ dO
            out["dq"][0][at, h] = dq
            out["dq"][1][at, h] = scale * (e @ K.abs()) + u * dq.abs() + t
            out["dk"][0][at, h // G] += dk
            out["dk"][1][at, h // G] += scale * (e.T @ Q.abs())
            out["dv"][0][at, h // G] += dv
            out["dv"][1][at, h // G] += (u + SLACK) * (p.T @ dO.abs()) + t * (seen.double().T @ dO.abs())
    if d_o is not None:
        for n in ("dk", "dv"):
            out[n][1] += u * out[n][0].abs() + t
    out["lse"].append(torch.full_like(out["lse"][0], 2.0 ** -12))   # a score's rounding, absolute, and that of log2 of the sum
    return out


def check(got, ref, what):
    value, bound = ref
    live = torch.isfinite(value)
    got = got.double()
    assert torch.isfinite(got[live]).all(), f"{what}: non-finite values"
    far = (got - value).abs()[live] - bound[live]
    if far.numel():
        worst = int(far.argmax())
        assert far.max() <= 0, (f"{what}: {int((far > 0).sum())} of {far.numel()} out of bounds, worst by {far.max().item():.3e} "
                                f"(bound {bound[live][worst].item():.3e}, value {value[live][worst].item():.3e})")
