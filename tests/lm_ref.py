"""Plain 64-bit forms of the language-model operators, and how far a kernel that
keeps its sums in f32 may be from them.

A bf16 rounding is off by at most 2^-8 of the value.  The attention kernels round
twice: the weights p (bf16 or better, while their sum stays f32) and the result.
So, with A = sum p |v| / sum p,
    |got - want| <= 2^-8 A + 2^-8 (|want| + 2^-8 A) + (2 ds + m 2^-23) A,
where ds is the error of a score's exponent: the f32 dot product's D 2^-23 times
the sum of |q_d k_d| scale, two roundings of the exponent's argument and the
exponential's 2^-22, and m 2^-23 A bounds the f32 sums over m keys.

The attention over the cache rounds p to f16 (2^-11) and, for keys whose weight is
under 2^-13 of the row's largest, to a multiple of 2^-24 of half a V scale's unit:
a code of 127 at most, off by 2^-25 * 127 * 2 < 2^-17 scales each, over the sum of
weights that counts the largest as 1.
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


def attend(q, k, v, kv_heads, causal, window, scale, p_round=2.0 ** -8, v_scale=0.0):
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
            tol[a:a + 1024, h] = p_round * A + r * (o.abs() + p_round * A) + \
                (2 * ds + m * 2.0 ** -23) * A
            if v_scale:
                rel = p / p.amax(1, keepdim=True).clamp(min=1e-300)
                tiny = ((rel < 2.0 ** -13) & oka).sum(1, keepdim=True)
                tol[a:a + 1024, h] += tiny * 2.0 ** -17 * v_scale / \
                    rel.sum(1, keepdim=True).clamp(min=1.0)
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


# ---- the 8-bit cache -------------------------------------------------------------

PAGE = 64


def page_scale(most):
    """The smallest bf16 s with 127 s >= most (f64, >= 0, of bf16 range), by bits."""
    import numpy as np
    if most == 0.0:
        return 0.0
    lo, hi = 0, 0x7f7f
    value = lambda b: float(np.array([b << 16], dtype=np.uint32).view(np.float32)[0])  # noqa: E731
    while lo < hi:
        mid = (lo + hi) // 2
        if 127.0 * value(mid) >= most:
            hi = mid
        else:
            lo = mid + 1
    return value(lo)


def kv8_append(codes, scales, x, cu, starts, table):
    """Appends in place: codes f64 [pages][KV][64][D], scales f64 [pages][KV], x f64
    [rows][KV][D], lists of offsets, starts and page ids."""
    import numpy as np
    KV = x.shape[1]
    for s in range(len(cu) - 1):
        n, done = cu[s + 1] - cu[s], 0
        while done < n:
            block, slot = divmod(starts[s] + done, PAGE)
            take = min(PAGE - slot, n - done)
            page = table[s][block]
            for h in range(KV):
                part = x[cu[s] + done:cu[s] + done + take, h]
                bad = not np.isfinite(part).all()
                size = math.nan if bad else page_scale(float(np.abs(part).max()))
                if slot:
                    was = scales[page, h]
                    size = math.nan if bad or math.isnan(was) else max(was, size)
                    if size > was:
                        codes[page, h, :slot] = np.rint(codes[page, h, :slot] * was / size)
                scales[page, h] = size
                if math.isnan(size):
                    codes[page, h, slot:slot + take] = 0
                else:
                    codes[page, h, slot:slot + take] = np.rint(part / size) if size else 0
            done += take


def kv8_attention(values_k, values_v, q, cu, lengths, table, heads, window, scale, v_scale):
    """values f64 [pages][KV][64][D]; lists; (want, tol) [rows][heads * D]."""
    import torch
    KV, D = values_k.shape[1], values_k.shape[3]
    want = torch.full((q.shape[0], heads * D), math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    for s, n in enumerate(lengths):
        a, b = cu[s], cu[s + 1]
        if b == a:
            continue
        t = torch.tensor(table[s][:(n + PAGE - 1) // PAGE], dtype=torch.long, device=q.device)
        k, v = (x[t].transpose(1, 2).reshape(-1, KV, D)[:n] for x in (values_k, values_v))
        w, e = attend(q[a:b].double().view(b - a, heads, D), k, v, KV, True, window, scale,
                      2.0 ** -11, v_scale)
        want[a:b], tol[a:b] = w.reshape(b - a, -1), e.reshape(b - a, -1)
    return want, tol
