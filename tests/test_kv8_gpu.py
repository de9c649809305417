"""The 8-bit key/value cache against its definition: codes and scales to the last
bit, values read back, attention of new tokens within lm_ref's bound, places outside
the cache, captured graphs, streams, refusals, and a run of all of it together."""
import math

import numpy as np
import pytest

import lm_ref

pytestmark = pytest.mark.gpu


def ints(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tables(blocks, seed=0, spare=3, cols=None):
    """Page ids for sequences of so many blocks, in no order, `spare` pages unused."""
    rng = np.random.default_rng(seed)
    pages = sum(blocks) + spare
    order = rng.permutation(pages).tolist()
    cols = max(blocks + [1]) if cols is None else cols
    out, at = [], 0
    for n in blocks:
        out.append(order[at:at + n] + [0] * (cols - n))
        at += n
    return out, pages


def cache_of(pages, kv_heads, D, seed=0, spread=0.5):
    """A used cache: codes of normal values, scales that differ."""
    import torch
    import ltx25_b200 as L
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def codes():
        return (torch.randn((pages, kv_heads, 64, D), generator=g, device="cuda") * 35).round() \
            .clamp(-127, 127).to(torch.int8)

    def scales():
        return (torch.randn((pages, kv_heads), generator=g, device="cuda") * spread).exp() \
            .mul(1 / 35).to(torch.bfloat16)

    return L.KV8Cache(codes(), codes(), scales(), scales())


def values(codes, scales):
    return codes.double() * scales.double()[:, :, None, None]


def host(t):
    return t.double().cpu().numpy().copy()


def check_append(ctx, cache, x_k, x_v, cu, starts, table):
    import torch
    import ltx25_b200 as L
    KV, D = cache.kv_heads, cache.head_dim
    want = []
    for codes, scales, x in ((cache.k, cache.k_scale, x_k), (cache.v, cache.v_scale, x_v)):
        c, s = host(codes), host(scales)
        lm_ref.kv8_append(c, s, host(x).reshape(-1, KV, D), cu, starts, table)
        want.append((c, s))
    L.kv8_append(ctx, cache, x_k, x_v, ints(cu), ints(starts), ints(table))
    torch.cuda.synchronize()
    ctx.check()
    for codes, scales, (c, s) in ((cache.k, cache.k_scale, want[0]),
                                  (cache.v, cache.v_scale, want[1])):
        np.testing.assert_array_equal(host(scales), s)
        np.testing.assert_array_equal(host(codes), c)


def rows_of(rows, cols, seed, scale=1.0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn((rows, cols), generator=g, device="cuda") * scale).to(torch.bfloat16)


@pytest.mark.parametrize("lens,starts,kv_heads,D", [
    ([1], [0], 1, 64), ([1], [63], 2, 128), ([1], [64], 2, 256), ([64], [0], 1, 128),
    ([65], [63], 2, 64), ([2], [63], 3, 128), ([0, 5, 0, 129, 1], [7, 60, 0, 1, 200], 2, 128),
    ([66, 1, 300], [63, 0, 31], 2, 256), ([1] * 40, list(range(30, 70)), 8, 128),
    ([500], [1000], 1, 64)])
def test_append_gives_the_definition_s_bits(ctx, lens, starts, kv_heads, D):
    blocks = [(s + n + 63) // 64 for s, n in zip(starts, lens)]
    table, pages = tables(blocks, seed=D)
    cu = lm_ref.offsets(lens)
    for scale in (1.0, 0.02):               # the page's own scale grows, or stays
        cache = cache_of(pages, kv_heads, D, seed=sum(lens) + D)
        check_append(ctx, cache, rows_of(cu[-1], kv_heads * D, 1, scale),
                     rows_of(cu[-1], kv_heads * D, 2, 3.0 * scale), cu, starts, table)


def test_append_decides_ties_and_edges(ctx):
    """Values of every magnitude: ties, subnormals, the largest numbers, zeros."""
    import torch
    D, pages = 256, 40
    rng = np.random.default_rng(7)
    bits = rng.integers(0, 1 << 16, size=(pages * 64, D)).astype(np.uint32)
    expo = np.repeat(np.linspace(0, 254, pages).astype(np.uint32), 64)[:, None]
    span = rng.integers(0, 9, size=bits.shape)
    bits = (bits & 0x807f) | (np.maximum(expo.astype(np.int64) - span, 0).astype(np.uint32) << 7)
    bits[64:128] = 0                                     # a page of zeros
    bits[128:192, :] = 0x8000                            # and of minus zeros
    # ties: s = 1 (the largest is 127), values n + 1/2 and n
    ties = (np.arange(64 * D) % 255 - 127) / 2.0
    ties[0] = 127.0
    bits[192:256] = (ties.reshape(64, D).astype(np.float32).view(np.uint32)) >> 16
    x = torch.from_numpy(bits.astype(np.uint16).view(np.int16)).view(torch.bfloat16).cuda()
    y = torch.from_numpy(bits[::-1].astype(np.uint16).view(np.int16)).view(torch.bfloat16).cuda()
    table, n = tables([pages])
    cache = cache_of(n, 1, D)
    check_append(ctx, cache, x, y, [0, pages * 64], [0], table)
    # the same, a page at a time from its middle: scales that grow by any factor
    for at in (0, 1, 30, 63):
        cache = cache_of(n, 1, D, seed=at, spread=20.0)
        m = pages
        xs = x[:m * 2].reshape(m * 2, D)[torch.randperm(m * 2, device="cuda")]
        ys = y[:m * 2].reshape(m * 2, D)[torch.randperm(m * 2, device="cuda")]
        tab = [[p] for p in table[0][:m]]
        check_append(ctx, cache, xs[:m], ys[:m], list(range(m + 1)), [at] * m, tab)


def test_append_marks_what_is_not_finite(ctx):
    D, KV = 128, 2
    table, pages = tables([3, 2])
    cache = cache_of(pages, KV, D)
    x = rows_of(150, KV * D, 3)
    y = rows_of(150, KV * D, 4)
    x[5, 7] = math.nan
    y[100, D + 1] = math.inf
    y[149, 3] = -math.inf
    check_append(ctx, cache, x, y, [0, 100, 150], [40, 64], table)
    # more tokens into a page that is marked leave it so
    check_append(ctx, cache, rows_of(2, KV * D, 5), rows_of(2, KV * D, 6), [0, 1, 2], [45, 114],
                 table)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_read_gives_the_values_back(ctx, D):
    import torch
    import ltx25_b200 as L
    KV, lens, starts = 3, [1, 0, 200, 64], [63, 5, 17, 64]
    table, pages = tables([(s + n + 63) // 64 for s, n in zip(starts, lens)])
    cache = cache_of(pages, KV, D)
    cu = lm_ref.offsets(lens, 2)
    wide = torch.full((cu[-1] + 5, 2 * KV * D), 7.0, device="cuda", dtype=torch.bfloat16)
    k, v = wide[:, :KV * D], wide[:, KV * D:]
    L.kv8_read(ctx, cache, ints(cu), ints(starts), ints(table), k.shape[0], k=k, v=v)
    torch.cuda.synchronize()
    ctx.check()
    for got, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want = torch.full_like(got, 7.0)
        x = values(codes, scales).to(torch.bfloat16)     # one rounding of an exact product
        for s, n in enumerate(lens):
            for i in range(n):
                t = starts[s] + i
                want[cu[s] + i] = x[table[s][t // 64], :, t % 64].reshape(-1)
        assert torch.equal(got, want)


CASES = [
    # new tokens, lengths, heads, kv_heads, D, window
    ([1], [1], 1, 1, 64, 0),
    ([1], [1], 4, 1, 128, 0),
    ([1], [64], 8, 2, 256, 0),
    ([1, 1, 1, 1], [63, 64, 65, 1000], 8, 2, 128, 0),
    ([1, 1, 1, 1], [63, 64, 65, 1000], 4, 4, 64, 0),
    ([1, 1, 1, 1], [15, 16, 17, 1000], 4, 2, 256, 0),
    ([1, 0, 1, 1], [0, 10, 5, 0], 4, 2, 128, 0),               # empty sequences
    ([3, 1, 5], [1, 0, 3], 4, 2, 64, 0),                       # tokens before the first
    ([4, 1, 7], [100, 3000, 7], 8, 2, 128, 0),                 # several new tokens
    ([4, 1, 7], [100, 3000, 7], 10, 2, 256, 0),
    ([4, 40, 7], [100, 3000, 7], 6, 2, 64, 0),
    ([33], [33], 20, 1, 128, 0),                               # more rows than a tile
    ([2], [700], 128, 1, 64, 0),
    ([1] * 5, [5, 200, 4000, 1, 777], 8, 8, 128, 1),           # windows
    ([1] * 5, [5, 200, 4000, 1, 777], 16, 2, 256, 130),
    ([3] * 5, [5, 200, 4000, 3, 777], 8, 2, 64, 100),
    ([1, 2], [300, 500], 4, 2, 128, 2147483647),
    ([1], [20000], 8, 1, 128, 0),
    ([1] * 64, [17 * i + 1 for i in range(64)], 16, 4, 128, 0),
    ([1] * 700, [(37 * i) % 211 for i in range(700)], 4, 2, 64, 0),
]


def attention_case(ctx, new, lengths, heads, kv_heads, D, window, qscale=1.0, spread=0.5):
    import torch
    table, pages = tables([(n + 63) // 64 for n in lengths], seed=len(new))
    cache = cache_of(pages, kv_heads, D, seed=sum(lengths), spread=spread)
    cu = lm_ref.offsets(new)
    q = rows_of(cu[-1], heads * D, 9, qscale)
    return cache, q, cu, table


def expect(cache, q, cu, lengths, table, heads, window):
    return lm_ref.kv8_attention(values(cache.k, cache.k_scale), values(cache.v, cache.v_scale), q,
                                cu, lengths, table, heads, window, cache.head_dim ** -0.5,
                                float(cache.v_scale.double().nan_to_num(0.0, 0.0, 0.0).max()))


def close(got, want, tol):
    import torch
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 1e-30, (float(over.max()), (over > 0).nonzero()[:5].tolist())


@pytest.mark.parametrize("new,lengths,heads,kv_heads,D,window", CASES)
def test_attention_matches_64_bits(ctx, new, lengths, heads, kv_heads, D, window):
    import torch
    import ltx25_b200 as L
    cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, window)
    got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, max(lengths),
                          window=window)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = expect(cache, q, cu, lengths, table, heads, window)
    close(got, want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("qscale,spread", [(8.0, 0.5), (1.0, 4.0), (1e-30, 0.5), (300.0, 3.0)])
def test_attention_over_far_apart_scales(ctx, D, qscale, spread):
    """Maxima that grow along the sequence, value scales that jump from page to page,
    queries far from 1."""
    import torch
    import ltx25_b200 as L
    new, lengths, heads, kv_heads = [1, 2, 1], [900, 1500, 64], 8, 2
    cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, 0, qscale, spread)
    got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, 1500)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = expect(cache, q, cu, lengths, table, heads, 0)
    close(got, want, tol)


@pytest.mark.parametrize("D,heads,kv_heads", [(64, 3, 3), (64, 16, 1), (128, 8, 2), (128, 40, 4),
                                              (256, 4, 2), (256, 9, 1)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_of_short_sequences(ctx, D, heads, kv_heads, window):
    """Lengths from nothing to a few stages a warp, one new token each or several or
    none, more new tokens than the sequence holds; the same with room for long ones."""
    import torch
    import ltx25_b200 as L
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 191, 400, 900, 2]
    for new in ([1] * 12, [1, 1, 2, 0, 5, 3, 0, 1, 4, 1, 2, 9]):
        cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, window)
        want, tol = expect(cache, q, cu, lengths, table, heads, window)
        for max_len in (900, 100000):
            got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads,
                                  max_len, window=window)
            torch.cuda.synchronize()
            ctx.check()
            close(got, want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("max_len", [0, 1, 300])
def test_longer_than_expected(ctx, D, max_len):
    """max_len sizes the launch; what a sequence holds beyond it counts all the same."""
    import torch
    import ltx25_b200 as L
    new, lengths, heads, kv_heads = [1, 2, 1], [5000, 700, 3], 4, 2
    cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, 0)
    got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, max_len)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = expect(cache, q, cu, lengths, table, heads, 0)
    close(got, want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("a,b", [(116, 100), (-90, -100), (100, 0)])
def test_attention_under_powers_of_two(ctx, D, a, b):
    """q by 2^a against K's scales by 2^-a, V's scales by 2^b: the products are the
    same and o is 2^b times as large.  Both are within f32's error of the same number,
    so they round to neighbours at most: a step of 2^-7."""
    import torch
    import ltx25_b200 as L
    new, lengths, heads, kv_heads = [1, 3], [900, 70], 4, 2
    cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, 0)
    far = L.KV8Cache(cache.k, cache.v, (cache.k_scale.double() * 2.0 ** -a).to(torch.bfloat16),
                     (cache.v_scale.double() * 2.0 ** b).to(torch.bfloat16))
    args = (ints(cu), ints(lengths), ints(table), heads, 900)
    near = L.kv8_attention(ctx, cache, q, *args).double()
    got = L.kv8_attention(ctx, far, (q.double() * 2.0 ** a).to(torch.bfloat16), *args).double()
    torch.cuda.synchronize()
    ctx.check()
    assert torch.isfinite(got).all()
    assert bool(((got * 2.0 ** -b - near).abs() <= near.abs() * 2.0 ** -7).all())


def steep_scales(exps, pages, kv_heads, table, lengths, seed):
    """V scales of powers of two, those of a sequence's pages taking `exps` in turn (or
    any of -133..60): bf16 [pages][kv_heads]."""
    import torch
    rng = np.random.default_rng(seed)
    e = np.zeros((pages, kv_heads), dtype=np.int64)
    for row, n in zip(table, lengths):
        for b in range((n + 63) // 64):
            for h in range(kv_heads):
                e[row[b], h] = rng.integers(-133, 61) if exps is None else exps[(b + h) % len(exps)]
    return torch.from_numpy(np.ldexp(1.0, e)).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("exps", [(0, -120), (-5, -5, -110), (0, -133), (-133,), (-121, -128, -133),
                                  (100, -20, -120, 40), (0, -60, 0, -70), None])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,max_len", [
    ([1, 2], [700, 1300], 8, 2, 1300), ([1, 3], [1900, 1300], 2, 2, 100000),
    ([1] * 16, [2500] * 16, 8, 8, 2500), ([3] * 6, [150] * 6, 12, 2, 20000)])
def test_attention_over_value_scales_at_the_ends_of_the_range(ctx, D, exps, new, lengths, heads,
                                                              kv_heads, max_len):
    """Pages whose V scales are up to 2^193 apart, subnormal ones among them.  Beside
    lm_ref's bound, in units of a sequence's largest V scale T:
      the lowest unit of O is max(2^-64 T / 32, 2^-126) or less; values of scales under
      2^-8 of it count as zero, codes of 127 at most: 2^-70 T;
      weights over the lowest unit round to 2^-25 of it a code: m 2^-18 of it for m
      keys, over a sum of at least 1;
      that lowest unit over the sum of weights (up to 2^6 m) may be subnormal: 2^-150 in
      2^-126 / (2^6 m), m 2^-18 of the result;
      and a bf16 result under 2^-126 rounds to 2^-134."""
    import torch
    import ltx25_b200 as L
    cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, 0)
    scales = steep_scales(exps, cache.pages, kv_heads, table, lengths, 3)
    cache = L.KV8Cache(cache.k, cache.v, cache.k_scale, scales)
    got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, max_len)
    torch.cuda.synchronize()
    ctx.check()
    assert torch.isfinite(got).all()
    k, v = values(cache.k, cache.k_scale), values(cache.v, scales)
    for s, n in enumerate(lengths):
        top = float(scales[table[s][:(n + 63) // 64]].double().max())
        rows = slice(cu[s], cu[s + 1])
        want, tol = lm_ref.kv8_attention(k, v, q[rows], [0, cu[s + 1] - cu[s]], [n], table[s:s + 1],
                                         heads, 0, D ** -0.5, top)
        tol = tol + 2.0 ** -70 * top + n * 2.0 ** -18 * max(2.0 ** -69 * top, 2.0 ** -126) + \
            n * 2.0 ** -18 * want.abs() + 2.0 ** -134
        over = (got[rows].double() - want).abs() - tol
        assert float(over.max()) <= 0, (s, float(over.max()), float(tol.max()))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lengths,max_len", [([300, 40], 300), ([9000, 700], 9000)])
def test_attention_of_the_largest_finite_numbers(ctx, D, lengths, max_len):
    """Up to 1e36: max|v| times the keys, D max|q| max|k|."""
    import torch
    import ltx25_b200 as L
    cache, q, cu, table = attention_case(ctx, [2, 1], lengths, 4, 2, D, 0, 3.0)
    kmax, vmax = (127 * float(s.double().max()) for s in (cache.k_scale, cache.v_scale))
    e = math.floor(math.log2(1e36 / (D * float(q.abs().max()) * kmax)) / 2)
    q, scale = q * 2.0 ** e, D ** -0.5 * 2.0 ** (-2 * e)
    cache = L.KV8Cache(cache.k, cache.v, cache.k_scale * 2.0 ** e, cache.v_scale *
                       2.0 ** math.floor(math.log2(1e36 / (lengths[0] * vmax))))
    got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), 4, max_len,
                          scale=scale)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.kv8_attention(values(cache.k, cache.k_scale),
                                     values(cache.v, cache.v_scale), q, cu, lengths, table, 4, 0,
                                     scale, float(cache.v_scale.double().max()))
    close(got, want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_does_not_look_past_a_row_s_tokens(ctx, D):
    """Scales of NaN on pages past the end, before the window, and on the page of a
    later new token; codes behind the last token of a page."""
    import torch
    import ltx25_b200 as L
    new, lengths, heads, kv_heads, window = [3, 1], [130, 300], 4, 2, 100
    table, pages = tables([4, 6])
    cache = cache_of(pages, kv_heads, D)
    # sequence 0: tokens 127, 128, 129 are new; page 2 (128..) is marked
    cache.k_scale[table[0][2]] = math.nan
    cache.v_scale[table[0][2]] = math.nan
    cache.v_scale[table[0][3]] = math.nan
    # sequence 1: position 299, window from 200: pages 0..2 are out of sight
    for b in (0, 1, 2, 5):
        cache.k_scale[table[1][b]] = math.nan
        cache.v_scale[table[1][b]] = math.inf
    cu = lm_ref.offsets(new)
    q = rows_of(4, heads * D, 9)
    got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, 300,
                          window=window)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = expect(cache, q, cu, lengths, table, heads, window)
    for row in (0, 3):
        close(got[row:row + 1], want[row:row + 1], tol[row:row + 1])
    assert got[1:3].isnan().all()


def test_rows_behind_the_last_sequence_and_given_workspaces(ctx):
    import torch
    import ltx25_b200 as L
    new, lengths, heads, kv_heads, D = [1, 3], [400, 90], 8, 2, 128
    cache, _, _, table = attention_case(ctx, new, lengths, heads, kv_heads, D, 0)
    q = rows_of(9, heads * D, 9)
    cu = [2, 3, 6]
    out = torch.full((9, heads * D), 7.0, device="cuda", dtype=torch.bfloat16)
    ws = torch.full((L.kv8_attention_workspace(ctx, D),), 0xff, device="cuda", dtype=torch.uint8)
    L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, 400, out=out,
                    workspace=ws)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = expect(cache, q, cu, lengths, table, heads, 0)
    close(out[2:6], want[2:6], tol[2:6])
    assert torch.all(out[:2] == 7.0) and torch.all(out[6:] == 7.0)


@pytest.mark.parametrize("given", [True, False])
def test_two_streams_and_two_graphs(ctx, given):
    """Calls that run at once, each with a workspace of its own (given, or left to the
    call), and graphs replayed after lengths changed on the device."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads, D, S = 8, 2, 128, 6
    table, pages = tables([40] * S)
    cache = cache_of(pages, kv_heads, D)
    cu = lm_ref.offsets([1] * S)
    t, c = ints(table), ints(cu)
    streams = [torch.cuda.Stream() for _ in range(2)]
    state = []
    for i, st in enumerate(streams):
        q, ln = rows_of(S, heads * D, i), ints([1] * S)
        ws = torch.empty(L.kv8_attention_workspace(ctx, D), device="cuda",
                         dtype=torch.uint8) if given else None
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        run = lambda q=q, ln=ln, ws=ws, out=out: L.kv8_attention(          # noqa: E731
            ctx, cache, q, c, ln, t, heads, 2560, out=out, workspace=ws)
        with torch.cuda.stream(st):
            run()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            run()
        state.append((st, g, q, ln, out, ws))     # what the graph holds addresses of
    rng = np.random.default_rng(0)
    for _ in range(3):
        lens = [rng.integers(0, 2561, S).tolist() for _ in state]
        for (st, g, q, ln, out, _), n in zip(state, lens):
            ln.copy_(ints(n))
        torch.cuda.synchronize()
        for st, g, *_ in state:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        ctx.check()
        for (st, g, q, ln, out, _), n in zip(state, lens):
            want, tol = expect(cache, q, cu, n, table, heads, 0)
            close(out, want, tol)


def test_the_same_call_gives_the_same_bits(ctx):
    import torch
    import ltx25_b200 as L
    new, lengths, heads, kv_heads, D = [1] * 7, [5, 4000, 900, 1, 64, 2222, 70], 8, 2, 128
    cache, q, cu, table = attention_case(ctx, new, lengths, heads, kv_heads, D, 0)
    a, b = (L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, 4000)
            for _ in range(2))
    assert torch.equal(a, b)
    # max_len only sizes the launch
    c = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(table), heads, 1)
    want, tol = expect(cache, q, cu, lengths, table, heads, 0)
    close(c, want, tol)


def test_places_outside_the_cache_are_not_followed(ctx):
    """The host sees neither lengths nor pages: the kernels leave out what they
    cannot reach and the context's check says so."""
    import torch
    import ltx25_b200 as L
    KV, D, heads = 2, 128, 4
    table, pages = tables([4, 4, 4])

    def marked():
        torch.cuda.synchronize()
        with pytest.raises(L.LtxError) as e:
            ctx.check()
        assert e.value.code == -6
        ctx.check()

    for page in (pages, -1, 2 ** 31 - 1, -2 ** 31):
        cache = cache_of(pages, KV, D)
        bad = [list(r) for r in table]
        bad[1][2] = page
        # append: the page's rows are left out, all others are stored
        x, y = rows_of(3 * 200, KV * D, 1), rows_of(3 * 200, KV * D, 2)
        k0, s0 = cache.k.clone(), cache.k_scale.clone()
        L.kv8_append(ctx, cache, x, y, ints([0, 200, 400, 600]), ints([0, 0, 0]), ints(bad))
        marked()
        c, s = host(k0), host(s0)
        keep_c, keep_s = c[table[1][2]].copy(), s[table[1][2]].copy()
        lm_ref.kv8_append(c, s, host(x).reshape(-1, KV, D), [0, 200, 400, 600], [0, 0, 0], table)
        c[table[1][2]], s[table[1][2]] = keep_c, keep_s
        np.testing.assert_array_equal(host(cache.k), c)
        np.testing.assert_array_equal(host(cache.k_scale), s)
        # read: its rows are left as they are
        k = torch.full((600, KV * D), 7.0, device="cuda", dtype=torch.bfloat16)
        v = k.clone()
        L.kv8_read(ctx, cache, ints([0, 200, 400, 600]), ints([0, 0, 0]), ints(bad), 600, k=k, v=v)
        marked()
        assert torch.all(k[328:392] == 7.0) and not torch.any(k[:328] == 7.0).item()
        # attention: its tokens are left out, the other sequences are whole
        q = rows_of(3, heads * D, 5)
        got = L.kv8_attention(ctx, cache, q, ints([0, 1, 2, 3]), ints([200] * 3), ints(bad), heads,
                              200)
        marked()
        want, tol = expect(cache, q, [0, 1, 2, 3], [200] * 3, table, heads, 0)
        close(got[[0, 2]], want[[0, 2]], tol[[0, 2]])
        assert torch.isfinite(got).all()
    cache = cache_of(pages, KV, D)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    x = rows_of(10, KV * D, 1)
    for start in (-1, 247, 257, 2 ** 31 - 1, -2 ** 31):       # 4 pages: 256 tokens
        L.kv8_append(ctx, cache, x, x, ints([0, 10]), ints([start]), ints(table[:1]))
        marked()
    for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)):
        assert torch.equal(a, b)
    for length in (-1, 257, 2 ** 31 - 1, -2 ** 31):
        got = L.kv8_attention(ctx, cache, x[:1, :].repeat(1, heads // KV), ints([0, 1]),
                              ints([length]), ints(table[:1]), heads, 256)
        marked()
        assert torch.isfinite(got).all()
    # offsets that descend or leave the tensor
    for cu in ([0, 30], [5, 2], [-7, 400], [2 ** 31 - 1, -2 ** 31]):
        L.kv8_append(ctx, cache, x, x, ints(cu), ints([0]), ints(table[:1]))
        L.kv8_attention(ctx, cache, rows_of(10, heads * D, 2), ints(cu), ints([100]),
                        ints(table[:1]), heads, 256)
        torch.cuda.synchronize()
    ctx.check()


@pytest.mark.parametrize("D,heads,kv_heads", [(64, 16, 2), (64, 3, 3), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("lengths,seqs", [([40, 64, 1], 3), ([300, 700, 64], 3), ([30000, 130, 64], 3),
                                          ([100, 5, 64], 400)])
@pytest.mark.parametrize("new,window", [(1, 0), (1, 20), (3, 33)])
def test_rows_without_a_page_are_zero(ctx, D, heads, kv_heads, lengths, seqs, new, window):
    """Every second sequence has no page at all, or none inside its window; the others are
    whole."""
    import torch
    import ltx25_b200 as L
    lengths = [max(new, lengths[i % len(lengths)]) for i in range(seqs)]
    cache, q, cu, table = attention_case(ctx, [new] * seqs, lengths, heads, kv_heads, D, window)
    bad = [list(r) for r in table]
    for s in range(0, seqs, 2):
        first = max(0, lengths[s] - new - window + 1) // 64 if window else 0
        for b in range(first, len(bad[s])):
            bad[s][b] = cache.pages if b % 3 else -1
    want, tol = expect(cache, q, cu, lengths, table, heads, window)
    for max_len in (1, max(lengths), 10 * max(lengths)):
        got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), ints(bad), heads, max_len,
                              window=window)
        torch.cuda.synchronize()
        with pytest.raises(L.LtxError) as e:
            ctx.check()
        assert e.value.code == -6
        got = got.view(seqs, new, -1)
        assert torch.all(got[::2] == 0)
        close(got[1::2], want.view(seqs, new, -1)[1::2], tol.view(seqs, new, -1)[1::2])


def test_a_scale_that_leaves_32_bits_is_refused(ctx):
    import torch
    import ltx25_b200 as L
    table, pages = tables([2])
    cache = cache_of(pages, 2, 64)
    args = (ints([0, 1]), ints([5]), ints(table), 4, 64)
    with pytest.raises(L.LtxError) as e:
        L.kv8_attention(ctx, cache, rows_of(1, 256, 2), *args, scale=3e38)
    assert e.value.code == -2
    torch.cuda.synchronize()
    ctx.check()


def test_refusals(ctx):
    import torch
    import ltx25_b200 as L
    KV, D, heads = 2, 64, 4
    table, pages = tables([2, 2])
    cache = cache_of(pages, KV, D)
    x, q = rows_of(8, KV * D, 1), rows_of(8, heads * D, 2)
    cu, n, t = ints([0, 4, 8]), ints([60, 64]), ints(table)

    def code(fn):
        with pytest.raises(L.LtxError) as e:
            fn()
        return e.value.code

    assert code(lambda: L.KV8Cache(cache.k[:, :, :32], cache.v, cache.k_scale, cache.v_scale)) == -2
    assert code(lambda: L.KV8Cache(cache.k, cache.v, cache.k_scale.float(), cache.v_scale)) == -2
    assert code(lambda: L.KV8Cache(cache.k, cache.v.cpu(), cache.k_scale, cache.v_scale)) == -2
    assert code(lambda: L.kv8_append(ctx, cache, x.float(), x, cu, n, t)) == -3
    assert code(lambda: L.kv8_append(ctx, cache, x[:, :64], x, cu, n, t)) == -2
    assert code(lambda: L.kv8_append(ctx, cache, x[:4], x, cu, n, t)) == -2
    assert code(lambda: L.kv8_append(ctx, cache, x, x, cu, n[:1], t)) == -2
    assert code(lambda: L.kv8_append(ctx, cache, x, x, cu, n, t.long())) == -2
    assert code(lambda: L.kv8_append(ctx, cache, x, x, cu, n, t[:1])) == -2
    assert code(lambda: L.kv8_append(ctx, cache, x, x, cu, n, t[:, :0])) == -2
    assert code(lambda: L.kv8_read(ctx, cache, cu, n, t, 8, k=x, v=x[:4])) == -2
    call = lambda **kw: L.kv8_attention(ctx, **{**dict(                     # noqa: E731
        cache=cache, q=q, cu_q=cu, lengths=n, table=t, heads=heads, max_len=64), **kw})
    assert code(lambda: call(heads=3)) == -2
    assert code(lambda: call(window=-1)) == -2
    assert code(lambda: call(scale=-1.0)) == -2
    assert code(lambda: call(max_len=-1)) == -2
    assert code(lambda: call(q=q.cpu())) == -2
    assert code(lambda: call(workspace=torch.empty(64, device="cuda"))) == -2
    ws = torch.empty(L.kv8_attention_workspace(ctx, D) + 16, dtype=torch.uint8, device="cuda")
    assert code(lambda: call(workspace=ws[1:])) == -8
    assert code(lambda: L.kv8_attention_workspace(ctx, 96)) == -2
    w96 = L.KV8Cache.empty(ctx, 2, 2, 96)
    x96 = torch.zeros((8, 192), device="cuda", dtype=torch.bfloat16)
    assert code(lambda: L.kv8_append(ctx, w96, x96, x96, cu, n, t)) == -2
    assert call(q=q[:0], cu_q=ints([0, 0, 0])).shape == (0, heads * D)
    torch.cuda.synchronize()
    ctx.check()


@pytest.mark.parametrize("D,heads,kv_heads,window", [(64, 6, 2, 0), (128, 8, 2, 0),
                                                     (256, 4, 2, 150)])
def test_a_prompt_then_token_after_token(ctx, D, heads, kv_heads, window):
    """As a caption model runs: the packed prompts' attention, their keys and values
    into the cache, a second chunk over what is read back, then single tokens whose
    attention reads the cache they were just appended to."""
    import torch
    import ltx25_b200 as L
    prompts, steps = [5, 190, 64], 70
    S, cols = len(prompts), kv_heads * D
    table, pages = tables([(n + 40 + steps + 63) // 64 for n in prompts])
    cache = L.KV8Cache.empty(ctx, pages, kv_heads, D)
    for t in (cache.k, cache.v):
        t.fill_(77)                                       # what an earlier use left
    cache.k_scale.fill_(math.nan)
    cache.v_scale.fill_(math.nan)
    t = ints(table)
    ref = [[np.zeros((pages, kv_heads, 64, D)), np.full((pages, kv_heads), 1.0)] for _ in range(2)]

    def append(k, v, cu, starts):
        L.kv8_append(ctx, cache, k, v, ints(cu), ints(starts), t)
        for (c, s), x in zip(ref, (k, v)):
            lm_ref.kv8_append(c, s, host(x).reshape(-1, kv_heads, D), cu, starts, table)

    def attend_cache(q, cu, lengths):
        got = L.kv8_attention(ctx, cache, q, ints(cu), ints(lengths), t, heads, max(lengths),
                              window=window)
        k, v = (torch.from_numpy(c * s[:, :, None, None]).cuda() for c, s in ref)
        want, tol = lm_ref.kv8_attention(k, v, q, cu, lengths, table, heads, window, D ** -0.5,
                                         float(ref[1][1].max()))
        close(got, want, tol)

    # the prompts
    cu = lm_ref.offsets(prompts)
    q, k, v = rows_of(cu[-1], heads * D, 1), rows_of(cu[-1], cols, 2), rows_of(cu[-1], cols, 3)
    got = L.attention_packed(ctx, q, k, v, ints(cu), ints(cu), heads, kv_heads, D, window=window)
    want, tol = lm_ref.attention_packed(q, k, v, cu, cu, heads, kv_heads, D, True, window,
                                        D ** -0.5)
    close(got, want, tol)
    append(k, v, cu, [0] * S)
    # a chunk of 40 tokens over all that came before, in bf16 from the cache
    cu = lm_ref.offsets([40] * S)
    q, k, v = rows_of(cu[-1], heads * D, 4), rows_of(cu[-1], cols, 5), rows_of(cu[-1], cols, 6)
    append(k, v, cu, prompts)
    lengths = [n + 40 for n in prompts]
    cu_k = lm_ref.offsets(lengths)
    rk, rv = L.kv8_read(ctx, cache, ints(cu_k), ints([0] * S), t, cu_k[-1])
    got = L.attention_packed(ctx, q, rk, rv, ints(cu), ints(cu_k), heads, kv_heads, D,
                             window=window)
    want, tol = lm_ref.attention_packed(q, rk, rv, cu, cu_k, heads, kv_heads, D, True, window,
                                        D ** -0.5)
    close(got, want, tol)
    attend_cache(q, cu, lengths)
    # single tokens
    cu = lm_ref.offsets([1] * S)
    for step in range(steps):
        q, k, v = (rows_of(S, c, 10 * step + i, 1.0 + step / 20)
                   for i, c in ((7, heads * D), (8, cols), (9, cols)))
        append(k, v, cu, lengths)
        lengths = [n + 1 for n in lengths]
        if step % 7 == 0 or step > steps - 4:
            attend_cache(q, cu, lengths)
    ctx.check()
    for (c, s), codes, scales in zip(ref, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        for i, n in enumerate(lengths):
            for b in range((n + 63) // 64):
                m = min(64, n - 64 * b)
                page = table[i][b]
                np.testing.assert_array_equal(host(codes)[page, :, :m], c[page, :, :m])
                np.testing.assert_array_equal(host(scales)[page], s[page])
