"""Plain 64-bit forms of the language-model operators, and how far a kernel that
keeps its sums in f32 may be from them.

A bf16 rounding is off by at most 2^-8 of the value.  The attention kernels round
twice: the weights p (bf16 or better, while their sum stays f32) and the result.
So, with A = sum p |v| / sum p,
    |got - want| <= 2^-8 A + 2^-8 (|want| + 2^-8 A) + (2 ds + m 2^-23) A,
where ds is the error of a score's exponent: the f32 dot product's D 2^-23 times
the sum of |q_d k_d| scale, two roundings of the exponent's argument and the
exponential's 2^-22, and m 2^-23 A bounds the f32 sums over m keys.
"""
import math


def visible(n, m, causal, window, device):
    import torch
    pos = torch.arange(n, device=device)[:, None] + (m - n)
    j = torch.arange(m, device=device)[None]
    ok = torch.ones((n, m), dtype=torch.bool, device=device)
    if causal:
        ok &= j <= pos
    if window:
        ok &= j > pos - window
    return ok


def attend(q, k, v, kv_heads, causal, window, scale):
    """One sequence: q [n][H][D], k and v [m][KV][D], f64.  Returns the result and
    the bound on a kernel's distance from it, both [n][H][D]."""
    import torch
    n, H, D = q.shape
    m, G = k.shape[0], H // kv_heads
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    if m == 0:
        return out, tol
    ok = visible(n, m, causal, window, q.device)
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        for a in range(0, n, 1024):
            qa, oka = q[a:a + 1024, h], ok[a:a + 1024]
            s = torch.where(oka, (qa @ kh.T) * scale, -math.inf)
            size = torch.where(oka, (qa.abs() @ kh.abs().T) * scale, 0.0)
            top = s.amax(1, keepdim=True)
            ds = D * 2.0 ** -23 * size.amax(1, keepdim=True) + 2.0 ** -22 * \
                (2 * s.where(oka, torch.zeros_like(s)).abs().amax(1, keepdim=True) + 1)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            p = torch.exp(s - top)
            total = p.sum(1, keepdim=True)
            seen = oka.any(1, keepdim=True)
            p = torch.where(seen, p / total, torch.zeros_like(p))
            # a key that a row does not see has no part in it, whatever it holds
            o = torch.zeros((qa.shape[0], D), dtype=q.dtype, device=q.device)
            A = torch.zeros_like(o)
            bad = ~torch.isfinite(vh).all(1)
            good = torch.where(bad[:, None], torch.zeros_like(vh), vh)
            o += p @ good
            A += p @ good.abs()
            for j in bad.nonzero()[:, 0].tolist():
                o += torch.where(oka[:, j:j + 1], p[:, j:j + 1] * vh[j], 0.0)
            out[a:a + 1024, h] = o
            r = 2.0 ** -8
            tol[a:a + 1024, h] = r * A + r * (o.abs() + r * A) + (2 * ds + m * 2.0 ** -23) * A
    return out, tol


def attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, causal, window, scale):
    """Lists of offsets; returns (want, tol) [rows][heads * D], NaN outside the
    sequences."""
    import torch
    want = torch.full((q.shape[0], heads * D), math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    for s in range(len(cu_q) - 1):
        a, b, c, d = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        if b > a:
            w, t = attend(q[a:b].double().view(b - a, heads, D),
                          k[c:d].double().view(d - c, kv_heads, D),
                          v[c:d].double().view(d - c, kv_heads, D), kv_heads, causal, window,
                          scale)
            want[a:b], tol[a:b] = w.reshape(b - a, -1), t.reshape(b - a, -1)
    return want, tol


def offsets(lens, first=0):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu
