"""Timing cases of the language-model operators: attention over packed prompts,
and the 8-bit key/value cache (append, read back, attention of new tokens).

`listed()` names the cases, `draw(rng)` makes one more of the same ranges,
`prepare(case, seed)` makes a case's inputs on the GPU, `run(state)` is one pass,
`work(case)` counts what a pass cannot do without and `exact(case, seed)` gives
the results in 64 bits.  With `own` false `run` computes the plain forms below;
with `own` true it calls this package's operators.

The definitions.  Query head h reads key/value head h // (heads / kv_heads).
Row i of a sequence with n queries and m keys stands at position m - n + i; with
`causal` it sees the keys j <= its position, with a `window` of w > 0 only those
above position - w.  o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j), over
the keys it sees; zero where it sees none.

The cache holds pages of 64 tokens, int8 codes [pages][kv_heads][64][head_dim]
with one bf16 scale for each page and head; token t of sequence s is slot t % 64
of page table[s][t // 64].  Appending tokens to a page takes the smallest bf16
scale with 127 scale >= |x| for all the new values, or the page's own where that
is larger and the page already holds tokens of the sequence; codes are
rint(x / scale), and codes that the page held are brought to a grown scale as
rint(code * old / new).
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 64


def _prompt(name, seqs, lo, hi, heads, kv_heads, head_dim, causal=True, window=0, prefix=0,
            lens_seed=1):
    c = {"kind": "prompt", "seqs": seqs, "lo": lo, "hi": hi, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "causal": causal, "window": window,
         "prefix": prefix, "lens_seed": lens_seed}
    return dict(c, name=name) if name else c


def _append(name, seqs, lo, hi, start, kv_heads, head_dim, lens_seed=1):
    c = {"kind": "append", "seqs": seqs, "lo": lo, "hi": hi, "start": start,
         "kv_heads": kv_heads, "head_dim": head_dim, "lens_seed": lens_seed}
    return dict(c, name=name) if name else c


def _decode(name, seqs, lo, hi, new, heads, kv_heads, head_dim, window=0, lens_seed=1):
    c = {"kind": "decode", "seqs": seqs, "lo": lo, "hi": hi, "new": new, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "lens_seed": lens_seed}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one caption of 256 tokens, the text length of a generation
        _prompt("prompt caption 256", 1, 256, 256, 32, 8, 128),
        # a batch of captions of mixed lengths in one call, 64-wide heads, queries,
        # keys and values as columns of one projection's output
        _prompt("prompt captions x16 hd64", 16, 9, 1024, 32, 4, 64, lens_seed=3),
        # one long instruction with its examples
        _prompt("prompt 8192", 1, 8192, 8192, 32, 8, 128),
        # a local layer of a caption encoder: 256-wide heads, a sliding window
        _prompt("prompt local hd256", 4, 500, 4001, 16, 8, 256, window=1024, lens_seed=4),
        # a later chunk of two prompts over what came before, five queries a key head
        _prompt("prompt chunk on prefix", 2, 333, 777, 20, 4, 128, prefix=6990, lens_seed=5),
        # every running sequence stores its newest token
        _append("append one x64", 64, 1, 1, 4096, 8, 128, lens_seed=6),
        # the prompts of a batch move into the cache, 256-wide heads
        _append("append prompts hd256", 6, 700, 2000, 0, 8, 256, lens_seed=7),
        # one user, short context: the latency of a token
        _decode("decode x1 1000", 1, 1000, 1000, 1, 32, 8, 128),
        # a served batch of mixed context lengths
        _decode("decode x64 to 8192", 64, 100, 8192, 1, 32, 8, 128, lens_seed=8),
        # one user, a very long context
        _decode("decode x1 131072", 1, 131072, 131072, 1, 32, 8, 128),
        # four proposed tokens a sequence checked at once, a local layer
        _decode("decode 4 new x16 hd256", 16, 200, 16384, 4, 16, 8, 256, window=4096, lens_seed=9),
        # a key head for every query head
        _decode("decode x32 hd64 ungrouped", 32, 5, 4096, 1, 16, 16, 64, lens_seed=10),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prompt", "append", "decode", "prompt", "decode"))
    head_dim = rng.choice((64, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8))
    lens_seed = rng.randrange(1 << 20)
    if kind == "append":
        hi = _log(rng, 1, 2000)
        return _append(None, _log(rng, 1, max(1, min(64, 12000 // hi))), _log(rng, 1, hi), hi,
                       rng.choice((0, _log(rng, 1, 4096))), kv_heads, head_dim, lens_seed)
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8) if kv_heads < 8 else (1, 2, 4))
    if kind == "prompt":
        hi = _log(rng, 1, 4096)
        seqs = _log(rng, 1, max(1, min(32, 6000 // hi)))
        return _prompt(None, seqs, _log(rng, 1, hi), hi, heads, kv_heads, head_dim,
                       causal=rng.random() < 0.8,
                       window=rng.choice((0, 0, _log(rng, 1, 2048))),
                       prefix=rng.choice((0, 0, _log(rng, 1, 3000))), lens_seed=lens_seed)
    new = rng.choice((1, 1, 1, 2, 3, 8))
    hi = _log(rng, new, 100000)
    seqs = _log(rng, 1, max(1, min(96, 200000 // hi)))
    return _decode(None, seqs, _log(rng, new, hi), hi, new, heads, kv_heads, head_dim,
                   window=rng.choice((0, 0, 0, _log(rng, 1, 8192))), lens_seed=lens_seed)


def _lens(case):
    """The sequences' lengths; for a prompt and an append those of the new rows."""
    r = random.Random(case["lens_seed"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _starts(case):
    """What each sequence of an append, or of a prompt's chunk, had before."""
    r = random.Random(case["lens_seed"] + 1)
    most = case["start"] if case["kind"] == "append" else case["prefix"]
    return [r.randint((most + 1) // 2, most) for _ in range(case["seqs"])]


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(g, blocks, kv_heads, head_dim):
    """Pages as they are after use: codes of normal values over scales that differ
    from page to page and head to head, and a table that leads to them in no order."""
    pages = int(sum(blocks))
    shape = (pages, kv_heads, BLOCK, head_dim)
    code = lambda: torch.randn(shape, generator=g, device="cuda").mul_(30).round_() \
        .clamp_(-127, 127).to(torch.int8)                               # noqa: E731
    scale = lambda: torch.randn((pages, kv_heads), generator=g, device="cuda").mul_(0.25) \
        .exp_().mul_(1 / 30).to(torch.bfloat16)                         # noqa: E731
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    cols = int(max(blocks))
    lens = torch.tensor(blocks, device="cuda")
    first = torch.cumsum(lens, 0) - lens
    at = first[:, None] + torch.arange(cols, device="cuda")[None, :]
    inside = torch.arange(cols, device="cuda")[None, :] < lens[:, None]
    table = torch.where(inside, order[at.clamp(max=pages - 1)], torch.zeros_like(order[:1]))
    return {"k": code(), "v": code(), "ks": scale(), "vs": scale(), "table": table.contiguous()}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lens, D, KV = _lens(case), case["head_dim"], case["kv_heads"]
    rnd = lambda rows, cols: torch.randn((rows, cols), generator=g, device="cuda") \
        .to(torch.bfloat16)                                             # noqa: E731
    s = {"case": case, "kv_heads": KV, "head_dim": D}
    if case["kind"] == "prompt":
        H, rows, before = case["heads"], sum(lens), _starts(case)
        keys = [n + b for n, b in zip(lens, before)]
        if sum(before):
            q, kv = rnd(rows, H * D), rnd(sum(keys), 2 * KV * D)
            k, v = kv[:, :KV * D], kv[:, KV * D:]
        else:  # columns of one fused projection
            qkv = rnd(rows, (H + 2 * KV) * D)
            q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + KV) * D], qkv[:, (H + KV) * D:]
        s.update(q=q, k=k, v=v, cu_q=_cu(lens), cu_k=_cu(keys), heads=H, max_q=max(lens),
                 max_k=max(keys), causal=case["causal"], window=case["window"],
                 scale=1.0 / math.sqrt(D))
    elif case["kind"] == "append":
        before = _starts(case)
        s.update(_cache(g, [(b + n + BLOCK - 1) // BLOCK for b, n in zip(before, lens)], KV, D))
        back = [b // BLOCK * BLOCK for b in before]
        s.update(x_k=rnd(sum(lens), KV * D), x_v=rnd(sum(lens), KV * D), cu=_cu(lens),
                 starts=_ints(before), back=_ints(back),
                 back_cu=_cu([b + n - r for b, n, r in zip(before, lens, back)]),
                 back_rows=sum(b + n - r for b, n, r in zip(before, lens, back)))
    else:
        H, new = case["heads"], case["new"]
        s.update(_cache(g, [(n + BLOCK - 1) // BLOCK for n in lens], KV, D))
        s.update(q=rnd(case["seqs"] * new, H * D), cu_q=_cu([new] * case["seqs"]), heads=H,
                 lengths=_ints(lens), max_q=new, max_len=max(lens), window=case["window"],
                 scale=1.0 / math.sqrt(D))
    return s


# ---- the package's operators ---------------------------------------------------

_ctx = None


def _package():
    global _ctx
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "vpipe-ltx-2.5_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ltx25_b200 as L
    if _ctx is None:
        _ctx = L.Context(torch.cuda.current_device())
    return L, _ctx


def _run_own(s):
    L, ctx = _package()
    kind = s["case"]["kind"]
    if kind == "prompt":
        return L.attention_packed(ctx, s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["heads"],
                                  s["kv_heads"], s["head_dim"], causal=s["causal"],
                                  window=s["window"], scale=s["scale"])
    cache = L.KV8Cache(s["k"], s["v"], s["ks"], s["vs"])
    if kind == "append":
        L.kv8_append(ctx, cache, s["x_k"], s["x_v"], s["cu"], s["starts"], s["table"])
        return L.kv8_read(ctx, cache, s["back_cu"], s["back"], s["table"], s["back_rows"])
    return L.kv8_attention(ctx, cache, s["q"], s["cu_q"], s["lengths"], s["table"], s["heads"],
                           s["max_len"], window=s["window"], scale=s["scale"])


# ---- plain forms ---------------------------------------------------------------

def _sequence_rows(cu, rows):
    """For each packed row its sequence and its place there."""
    r = torch.arange(rows, device=cu.device)
    seq = torch.searchsorted(cu, r, right=True) - 1
    return seq, r - cu[seq]


def _padded(x, cu, most, heads):
    """[rows][heads * D] -> f32 [seqs][heads][most][D]; rows past an end repeat the last."""
    n = x.shape[0]
    at = (cu[:-1, None] + torch.arange(most, device=x.device)).clamp(max=n - 1)
    return x[at].float().view(at.shape[0], most, heads, -1).transpose(1, 2)


def _attend(q, k, v, n, m, causal, window, scale):
    """q [S][H][mq][D], k and v [S][KV][mk][D], n and m the sequences' lengths."""
    S, H, mq, D = q.shape
    KV, mk = k.shape[1], k.shape[2]
    s = torch.matmul(q.reshape(S, KV, H // KV * mq, D), k.transpose(2, 3)).mul_(scale)
    s = s.view(S, KV, H // KV, mq, mk)
    j = torch.arange(mk, device=q.device)
    pos = (m - n)[:, None] + torch.arange(mq, device=q.device)
    seen = (j[None, None] < m[:, None, None]).expand(S, mq, mk)
    if causal:
        seen = seen & (j[None, None] <= pos[:, :, None])
    if window:
        seen = seen & (j[None, None] > pos[:, :, None] - window)
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, KV, H // KV * mq, mk), v).view(S, KV, H // KV, mq, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.view(S, H, mq, D)


def _packed(o, cu, rows):
    """f32 [seqs][heads][most][D] -> bf16 [rows][heads * D]."""
    seq, at = _sequence_rows(cu, rows)
    return o.transpose(1, 2)[seq, at].reshape(rows, -1).to(torch.bfloat16)


def _values(code, scale, table):
    """The cached values a table leads to: f32 [seqs][kv_heads][columns * 64][D]."""
    t = table.long()
    x = code[t].float().mul_(scale[t].float()[..., None, None])
    S, B, KV, _, D = x.shape
    return x.transpose(1, 2).reshape(S, KV, B * BLOCK, D)


def _page_scale(most):
    """The smallest bf16 s with 127 s >= most."""
    s = (most / 127).view(torch.int32).bitwise_and(-65536)
    up = 127 * s.view(torch.float32) < most
    return (s + up.int() * 65536).view(torch.float32)


def _store(code, scale, x, cu, starts, table):
    pages, KV, _, D = code.shape
    rows = x.shape[0]
    seq, i = _sequence_rows(cu, rows)
    pos = starts[seq] + i
    page = table[seq, pos // BLOCK].long()
    x = x.float().view(rows, KV, D)
    most = torch.zeros((pages, KV), device=x.device)
    most.scatter_reduce_(0, page[:, None].expand(rows, KV), x.abs().amax(-1), "amax")
    new = _page_scale(most)
    # the page each sequence continues, and what it held there
    held = torch.where(cu[1:] > cu[:-1], starts % BLOCK, torch.zeros_like(starts))
    first = table.gather(1, (starts // BLOCK).clamp(max=table.shape[1] - 1)[:, None].long())
    first = first[:, 0].long()
    before = scale[first].float()
    after = torch.where(held[:, None] > 0, torch.maximum(before, new[first]), new[first])
    grown = torch.round(code[first].float() * before[..., None, None] /
                        after[..., None, None].clamp(min=1e-30))
    keep = (torch.arange(BLOCK, device=x.device)[None] >= held[:, None])[:, None, :, None]
    code[first] = torch.where(keep, code[first], grown.to(torch.int8))
    new[first] = after
    touched = torch.zeros(pages, dtype=torch.bool, device=x.device)
    touched[page] = True
    scale.copy_(torch.where(touched[:, None], new, scale.float()).to(scale.dtype))
    c = torch.round(x / scale[page].float()[..., None].clamp(min=1e-30)).to(torch.int8)
    code[page[:, None], torch.arange(KV, device=x.device)[None], (pos % BLOCK)[:, None]] = c


def _read(code, scale, cu, starts, table, rows):
    seq, i = _sequence_rows(cu, rows)
    pos = starts[seq] + i
    page = table[seq, pos // BLOCK].long()
    at = torch.arange(code.shape[1], device=code.device)[None]
    x = code[page[:, None], at, (pos % BLOCK)[:, None]].float() * scale[page].float()[..., None]
    return x.view(rows, -1).to(torch.bfloat16)


def run(state):
    if own:
        return _run_own(state)
    s = state
    kind, KV = s["case"]["kind"], s["kv_heads"]
    if kind == "append":
        _store(s["k"], s["ks"], s["x_k"], s["cu"], s["starts"], s["table"])
        _store(s["v"], s["vs"], s["x_v"], s["cu"], s["starts"], s["table"])
        return tuple(_read(c, x, s["back_cu"], s["back"], s["table"], s["back_rows"])
                     for c, x in ((s["k"], s["ks"]), (s["v"], s["vs"])))
    q = _padded(s["q"], s["cu_q"], s["max_q"], s["heads"])
    n = s["cu_q"][1:] - s["cu_q"][:-1]
    if kind == "prompt":
        o = _attend(q, _padded(s["k"], s["cu_k"], s["max_k"], KV),
                    _padded(s["v"], s["cu_k"], s["max_k"], KV), n,
                    s["cu_k"][1:] - s["cu_k"][:-1], s["causal"], s["window"], s["scale"])
    else:
        o = _attend(q, _values(s["k"], s["ks"], s["table"]), _values(s["v"], s["vs"], s["table"]),
                    n, s["lengths"], True, s["window"], s["scale"])
    return _packed(o, s["cu_q"], s["q"].shape[0])


# ---- what a pass cannot do without ----------------------------------------------

def _seen(n, m, causal, window):
    """Pairs of a query and a key it sees, and the keys that any query sees."""
    pairs, low = 0, m
    for i in range(n):
        pos = m - n + i
        end = min(m, pos + 1) if causal else m
        begin = max(0, pos - window + 1) if window else 0
        pairs += max(0, end - begin)
        low = min(low, begin)
    return pairs, m - low


def work(case):
    lens, D, KV = _lens(case), case["head_dim"], case["kv_heads"]
    if case["kind"] == "append":
        before = _starts(case)
        rows = sum(lens)
        back = sum(b % BLOCK + n for b, n in zip(before, lens))
        # bf16 rows in and codes out, then codes in and bf16 rows out, keys and values
        return {"bytes": 2 * KV * D * (3 * rows + 3 * back), "flops": 2 * KV * D * (3 * rows + back)}
    H = case["heads"]
    if case["kind"] == "prompt":
        keys = [n + b for n, b in zip(lens, _starts(case))]
        seen = [_seen(n, m, case["causal"], case["window"]) for n, m in zip(lens, keys)]
        size, rows = 2 * 2 * KV * D, sum(lens)
    else:
        seen = [_seen(case["new"], n, True, case["window"]) for n in lens]
        size, rows = 2 * KV * D, case["new"] * len(lens)
    return {"bytes": size * sum(k for _, k in seen) + 2 * 2 * rows * H * D,
            "flops": 4 * H * D * sum(p for p, _ in seen)}


# ---- 64 bits ---------------------------------------------------------------------

def _exact_rows(q, k, v, causal, window, scale):
    """One sequence and one key head: q [n][G][D], k and v [m][D], all f64."""
    n, m = q.shape[0], k.shape[0]
    out = torch.zeros_like(q)
    step = max(1, (1 << 27) // max(1, q.shape[1] * m))
    for at in range(0, n, step):
        pos = torch.arange(at, min(n, at + step), device=q.device)[:, None] + (m - n)
        j = torch.arange(m, device=q.device)[None]
        ok = torch.ones((pos.shape[0], m), dtype=torch.bool, device=q.device)
        if causal:
            ok &= j <= pos
        if window:
            ok &= j > pos - window
        s = torch.einsum("ngd,md->ngm", q[at:at + step], k) * scale
        s = torch.where(ok[:, None], s, torch.full((), -math.inf, dtype=s.dtype, device=s.device))
        w = torch.softmax(s, -1).nan_to_num(0.0)
        out[at:at + step] = torch.einsum("ngm,md->ngd", w, v)
    return out


def _exact_scale(most):
    """The smallest number of 8 significant bits that is at least most / 127."""
    m, e = torch.frexp(most / 127)
    return torch.ldexp(torch.ceil(m * 256) / 256, e)


def exact(case, seed):
    s = prepare(case, seed)
    lens, D, KV = _lens(case), case["head_dim"], case["kv_heads"]
    if case["kind"] == "append":
        return tuple(_exact_append(case, s, c, x, n) for c, x, n in
                     (("k", "x_k", "ks"), ("v", "x_v", "vs")))
    H, G = case["heads"], case["heads"] // KV
    out = torch.empty((s["q"].shape[0], H, D), dtype=torch.float64, device="cuda")
    row = key = 0
    for i, n in enumerate(lens):
        new = n if case["kind"] == "prompt" else case["new"]
        q = s["q"][row:row + new].double().view(new, KV, G, D)
        if case["kind"] == "prompt":
            m = int(s["cu_k"][i + 1] - s["cu_k"][i])
            k = s["k"][key:key + m].double().view(m, KV, D)
            v = s["v"][key:key + m].double().view(m, KV, D)
            key, causal = key + m, case["causal"]
        else:
            t = s["table"][i, :(n + BLOCK - 1) // BLOCK].long()
            k, v = ((s[c][t].double() * s[x][t].double()[..., None, None]).transpose(1, 2)
                    .reshape(-1, KV, D)[:n] for c, x in (("k", "ks"), ("v", "vs")))
            causal = True
        for h in range(KV):
            out[row:row + new, h * G:(h + 1) * G] = _exact_rows(
                q[:, h], k[:, h], v[:, h], causal, case["window"], s["scale"])
        row += new
    return out.reshape(out.shape[0], H * D)


def _exact_append(case, s, code, x, scale):
    KV, D, out, row = case["kv_heads"], case["head_dim"], [], 0
    for i, (n, start) in enumerate(zip(_lens(case), _starts(case))):
        new = s[x][row:row + n].double().view(n, KV, D)
        row, done = row + n, 0
        while done < n:
            block, slot = divmod(start + done, BLOCK)
            take = min(BLOCK - slot, n - done)
            part = new[done:done + take].transpose(0, 1)
            page = int(s["table"][i, block])
            size = _exact_scale(part.abs().amax((1, 2)))[:, None, None]
            if slot:
                was = s[scale][page].double()[:, None, None]
                size = torch.maximum(size, was)
                held = torch.round(s[code][page, :, :slot].double() * was / size)
                out.append((held * size).transpose(0, 1))
            out.append((torch.round(part / size) * size).transpose(0, 1))
            done += take
    return torch.cat(out).reshape(-1, KV * D)
