"""Attention over packed prompts against its formula in 64 bits: ragged and empty
sequences, rows that see nothing, grouped heads, windows, cached prefixes, head
widths 64 / 128 / 256, NaN and infinities wherever a row does not look, strides,
streams, captured graphs and refusals.  The bound is lm_ref's."""
import math

import pytest

import lm_ref

pytestmark = pytest.mark.gpu


def make(lens_q, lens_k, heads, kv_heads, D, seed=0, qscale=1.0, pad=0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    cu_q, cu_k = lm_ref.offsets(lens_q), lm_ref.offsets(lens_k)
    q = (torch.randn((cu_q[-1] + pad, heads * D), generator=g, device="cuda") * qscale)
    kv = torch.randn((cu_k[-1] + pad, 2 * kv_heads * D), generator=g, device="cuda")
    kv = kv.to(torch.bfloat16)
    return q.to(torch.bfloat16), kv[:, :kv_heads * D], kv[:, kv_heads * D:], cu_q, cu_k


def dev(cu):
    import torch
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def check(got, want, tol, cu_q):
    import torch
    a, b = cu_q[0], cu_q[-1]
    got, want, tol = got[a:b].double(), want[a:b], tol[a:b]
    assert torch.isfinite(got).all()
    over = (got - want).abs() - tol
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1e-30, (worst, (over > 0).nonzero()[:5].tolist())


CASES = [
    # lens_q, lens_k, heads, kv_heads, D, causal, window, qscale
    ([1], [1], 1, 1, 64, True, 0, 1.0),
    ([1], [1], 4, 4, 128, True, 0, 1.0),
    ([1], [1], 2, 1, 256, True, 0, 1.0),
    ([256], [256], 32, 8, 128, True, 0, 1.0),
    ([1, 2, 127, 128, 129, 1, 64, 255], None, 8, 2, 128, True, 0, 1.0),
    ([1, 2, 127, 128, 129, 1, 64, 255], None, 4, 4, 64, True, 0, 1.0),
    ([1, 2, 127, 128, 129, 1, 64, 257], None, 4, 1, 256, True, 0, 1.0),
    ([0, 5, 0, 300, 0], None, 4, 2, 128, True, 0, 1.0),
    ([0, 5, 0, 300, 0], [7, 5, 0, 400, 3], 4, 2, 64, False, 0, 1.0),
    ([10, 200, 3], [3, 0, 1], 4, 2, 128, True, 0, 1.0),        # rows that see nothing
    ([10, 200, 3], [3, 0, 1], 4, 2, 256, True, 0, 1.0),
    ([10, 200, 3], [3, 0, 1], 4, 2, 64, True, 2, 1.0),
    ([10, 5], [0, 0], 2, 2, 128, True, 0, 1.0),                # no keys at all
    ([1, 60, 129], [1000, 333, 1029], 6, 2, 128, True, 0, 1.0),  # after a prefix
    ([1, 60, 129], [1000, 333, 1029], 5, 1, 256, True, 0, 1.0),
    ([1, 60, 129], [1000, 333, 1029], 14, 2, 64, True, 100, 1.0),
    ([700], None, 7, 1, 128, True, 0, 1.0),
    ([300, 90], None, 64, 1, 64, True, 0, 1.0),
    ([40, 3], None, 128, 1, 64, True, 0, 1.0),
    ([40, 3], None, 127, 1, 128, True, 0, 1.0),
    ([500], None, 4, 2, 128, False, 0, 1.0),
    ([500, 77], [130, 900], 4, 2, 256, False, 0, 1.0),
    ([1000], None, 2, 2, 128, True, 1, 1.0),                   # itself alone
    ([1000], None, 2, 2, 128, True, 128, 1.0),
    ([1000, 444], None, 4, 2, 256, True, 300, 1.0),
    ([1000, 444], None, 4, 2, 64, False, 300, 1.0),
    ([1000], None, 2, 2, 64, True, 2147483647, 1.0),
    ([1500], None, 2, 2, 128, True, 0, 6.0),                   # maxima that grow
    ([1500], None, 2, 1, 64, False, 0, 6.0),
    ([900], None, 2, 1, 256, True, 0, 6.0),
    ([4099], None, 4, 1, 128, True, 0, 1.0),
    ([2500], None, 2, 2, 256, True, 1024, 1.0),
]


@pytest.mark.parametrize("lens_q,lens_k,heads,kv_heads,D,causal,window,qscale", CASES)
def test_packed_attention_matches_64_bits(ctx, lens_q, lens_k, heads, kv_heads, D, causal, window,
                                          qscale):
    import torch
    import ltx25_b200 as L
    lens_k = lens_q if lens_k is None else lens_k
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, sum(lens_q) + D, qscale)
    got = L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), heads, kv_heads, D,
                             causal=causal, window=window)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, causal, window,
                                        D ** -0.5)
    check(got, want, tol, cu_q)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_outside_the_sequences_are_left_alone(ctx, D, causal):
    """Rows before the first and behind the last sequence hold NaN and infinities
    and are neither read into a result nor written."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads, first = 4, 2, 3
    lens = [5, 130, 61]
    q, k, v, _, _ = make(lens, lens, heads, kv_heads, D, 5, pad=80)
    cu = lm_ref.offsets(lens, first)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=torch.bfloat16)
    for x in (q, k, v):
        x[:first] = bad[0]
        x[cu[-1]:] = bad[torch.arange(x.shape[0] - cu[-1], device="cuda") % 3][:, None]
    out = torch.full((q.shape[0], heads * D), 7.0, device="cuda", dtype=torch.bfloat16)
    L.attention_packed(ctx, q, k, v, dev(cu), dev(cu), heads, kv_heads, D, causal=causal, out=out)
    torch.cuda.synchronize()
    ctx.check()
    assert torch.all(out[:first] == 7.0) and torch.all(out[cu[-1]:] == 7.0)
    want, tol = lm_ref.attention_packed(q, k, v, cu, cu, heads, kv_heads, D, causal, 0, D ** -0.5)
    check(out, want, tol, cu)


def best_ms(fn, n=5):
    """The quickest of n calls on the device, after a first one."""
    import torch
    best = math.inf
    for i in range(n + 1):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        fn()
        b.record()
        torch.cuda.synchronize()
        if i > 0:
            best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("D,heads", [(64, 8), (128, 4), (256, 2)])
@pytest.mark.parametrize("lens_q,lens_k", [([64], [4000]), ([64] + [1] * 32, [4000] + [5] * 32)])
def test_rows_before_the_first_sequence_cost_no_work(ctx, D, heads, lens_q, lens_k):
    """200000 rows before the sequences take no longer than as many behind them: 0.14 ms
    against 1.1 to 1.3 where the first item is done again for every 128 to 512."""
    import torch
    import ltx25_b200 as L
    first = 200000
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, heads, D, 7, pad=first)
    q[first:] = q[:cu_q[-1]].clone()
    late = [first + c for c in cu_q]
    outs = [torch.full_like(q, 7.0) for _ in range(2)]
    ms = [best_ms(lambda: L.attention_packed(ctx, q, k, v, c, dev(cu_k), heads, heads, D,
                                             causal=False, out=o))
          for c, o in ((dev(cu_q), outs[0]), (dev(late), outs[1]))]
    ctx.check()
    n = cu_q[-1]
    assert torch.equal(outs[0][:n], outs[1][first:])
    assert torch.all(outs[0][n:] == 7.0) and torch.all(outs[1][:first] == 7.0)
    assert ms[1] < 2 * ms[0] + 0.1, ms


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, D, value):
    """NaN and infinities in the keys and values of a neighbour sequence, and of
    later tokens of the row's own."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads = 4, 2
    lens = [70, 90, 200]
    q, k, v, cu, _ = make(lens, lens, heads, kv_heads, D, 11)
    k[cu[1]:cu[2]] = value                   # the whole second sequence
    v[cu[1]:cu[2]] = value
    spot = cu[2] + 150                       # one token of the third: a few dims
    v[spot, 3:9] = value
    got = L.attention_packed(ctx, q, k, v, dev(cu), dev(cu), heads, kv_heads, D)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu, cu, heads, kv_heads, D, True, 0, D ** -0.5)
    for a, b in ((cu[0], cu[1]), (cu[2], spot)):
        over = (got[a:b].double() - want[a:b]).abs() - tol[a:b]
        assert torch.isfinite(got[a:b]).all()
        assert float(over.max()) <= 0
    # rows that do see it: the formula's own NaN or infinity, and only there
    seen, ref = got[spot:cu[3]].double(), want[spot:cu[3]]
    assert torch.equal(torch.isfinite(seen), torch.isfinite(ref))
    ok = torch.isfinite(ref)
    assert float(((seen - ref).abs() - tol[spot:cu[3]])[ok].max()) <= 0
    assert torch.equal(seen[~ok].isnan(), ref[~ok].isnan())


@pytest.mark.parametrize("D,heads,kv_heads", [(64, 8, 2), (64, 3, 3), (128, 8, 2), (128, 40, 40),
                                              (256, 4, 2)])
@pytest.mark.parametrize("lens_q,lens_k", [
    ([1, 15, 17, 70, 127, 129, 250, 300], None), ([400, 130], [1001, 16]), ([64], [8203]),
    ([900, 5], [3019, 4990]), ([3] * 40, [241 + 3 * i for i in range(40)])])
@pytest.mark.parametrize("causal,window", [(False, 0), (False, 90), (True, 0)])
def test_the_next_sequence_leaves_no_trace(ctx, D, heads, kv_heads, lens_q, lens_k, causal, window):
    """NaN and infinities in the keys and values right behind a sequence's last, on every
    second sequence and behind the last of all: the others get the bits that they get
    beside ordinary numbers."""
    import torch
    import ltx25_b200 as L
    lens_k = lens_q if lens_k is None else lens_k
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, 41, pad=130)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=torch.bfloat16)
    got = []
    for marked in (None, 0, 1):
        a, b = k.clone(), v.clone()
        for s in range(len(lens_k) + 1):
            if marked is not None and (s & 1) == marked:
                rows = slice(cu_k[s], cu_k[s + 1] if s < len(lens_k) else None)
                n = a[rows].shape[0]
                a[rows] = b[rows] = bad[torch.arange(n, device="cuda") % 3][:, None]
        got.append(L.attention_packed(ctx, q, a, b, dev(cu_q), dev(cu_k), heads, kv_heads, D,
                                      causal=causal, window=window))
    torch.cuda.synchronize()
    ctx.check()
    for marked in (0, 1):
        for s in range(1 - marked, len(lens_k), 2):
            rows = slice(cu_q[s], cu_q[s + 1])
            assert torch.equal(got[1 + marked][rows], got[0][rows]), (marked, s)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_next_sequence_costs_no_time(ctx, D):
    """3000 rows over 5003 keys of their own, all seen, in front of a sequence of NaN."""
    import torch
    import ltx25_b200 as L
    q, k, v, cu_q, cu_k = make([3000, 100], [5003, 100], 4, 4, D, 43)
    ms = []
    for value in (0.5, math.nan):
        k[5003:] = v[5003:] = value
        ms.append(best_ms(lambda: L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), 4, 4, D,
                                                     causal=False)))
    ctx.check()
    assert ms[1] < 1.5 * ms[0] + 0.1, ms


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens_q,lens_k", [([500], [500]), ([30], [9000])])
def test_the_largest_finite_numbers(ctx, D, lens_q, lens_k):
    """Up to 1e36: max|v| times the keys, D max|q| max|k|."""
    import torch
    import ltx25_b200 as L
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, 4, 2, D, 51, 3.0)
    e = math.floor(math.log2(1e36 / (D * float(q.abs().max()) * float(k.abs().max()))) / 2)
    q, k = q * 2.0 ** e, k * 2.0 ** e
    v = v * 2.0 ** math.floor(math.log2(1e36 / (lens_k[0] * float(v.abs().max()))))
    scale = D ** -0.5 * 2.0 ** (-2 * e)
    got = L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), 4, 2, D, scale=scale)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, 4, 2, D, True, 0, scale)
    check(got, want, tol, cu_q)


def test_rows_computed_again_over_long_keys(ctx):
    """A NaN in the last of 300000 values: the 127 rows in front of it see all others and
    are computed again, 32 of them by a warp, in 2.3 s.  What waits for them goes on
    waiting (2 s is its limit for a kernel that stands still) and does the rest."""
    import torch
    import ltx25_b200 as L
    D, n, m, short = 256, 128, 300000, 400
    lens_q, lens_k = [1] * short + [n], [3] * short + [m]
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, 1, 1, D, 47)
    v[-1, 5] = math.nan
    out = torch.full_like(q, 7.0)
    L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), 1, 1, D, out=out)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, 1, 1, D, True, 0, D ** -0.5)
    check(out[:-1], want[:-1], tol[:-1], [0, short + n - 1])
    assert torch.equal(out[-1].isnan(), want[-1].isnan()) and int(out[-1].isnan().sum()) == 1
    ok = ~want[-1].isnan()
    assert float(((out[-1].double() - want[-1]).abs() - tol[-1])[ok].max()) <= 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("where", ["k", "v", "both signs in v"])
def test_what_every_row_sees_reaches_it_alone(ctx, D, where):
    """A NaN, or infinities of both signs, near the start of a long prefix: NaN where
    the formula has it, in every row; the other columns and the other key head are
    what they were."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads, lens_q, lens_k = 4, 2, [200, 40], [9000, 300]
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, 13)
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, True, 0, D ** -0.5)
    bad = torch.zeros_like(want, dtype=torch.bool)
    if where == "k":
        k[70, 5] = math.nan
        bad[:200, :2 * D] = True             # the two query heads of key head 0
    else:
        v[70, 5] = math.nan if where == "v" else math.inf
        if where != "v":
            v[4000, 5] = -math.inf
        bad[:200, [5, D + 5]] = True
    got = L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), heads, kv_heads, D)
    torch.cuda.synchronize()
    ctx.check()
    assert torch.equal(got.isnan(), bad)
    assert float(((got.double() - want).abs() - tol)[~bad].max()) <= 0


def test_calls_beyond_the_kernels_counters_are_refused(ctx):
    """Before anything is read."""
    import torch
    import ltx25_b200 as L
    q, k, v, cu, _ = make([20], [20], 4, 2, 64)
    c = dev(cu)
    with pytest.raises(L.LtxError) as e:
        L.attention_packed(ctx, q, k, v, c, c, 4, 2, 64, scale=3e38)
    assert e.value.code == -2
    out = torch.zeros_like(q)
    rc = ctx.lib.ltx_attention_packed(
        ctx.h, q.data_ptr(), 256, k.data_ptr(), 256, v.data_ptr(), 256, out.data_ptr(), 256,
        c.data_ptr(), c.data_ptr(), 2 ** 29 + 1, 20, 20, 4, 2, 64, 1, 0, 0.125, 0)
    assert rc == -2
    torch.cuda.synchronize()
    ctx.check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ld", [0, 4, -8, 2 ** 31 - 1])
def test_no_keys_at_all(ctx, D, ld):
    """Rows without keys are zero, whatever stands for k and v."""
    import torch
    q, _, _, cu, _ = make([20, 1], [0, 0], 4, 2, D)
    c, none, out = dev(cu), dev([0, 0, 0]), torch.full_like(q, 7.0)
    rc = ctx.lib.ltx_attention_packed(
        ctx.h, q.data_ptr(), 4 * D, None, ld, None, ld, out.data_ptr(), 4 * D, c.data_ptr(),
        none.data_ptr(), 2, 21, 0, 4, 2, D, 1, 0, 0.125, 0)
    assert rc == 0
    torch.cuda.synchronize()
    ctx.check()
    assert torch.all(out == 0)


@pytest.mark.parametrize("D,heads,kv_heads", [(64, 8, 8), (128, 32, 4), (256, 12, 6)])
@pytest.mark.parametrize("causal,window,prefix", [(True, 0, 0), (True, 200, 0), (True, 0, 90),
                                                  (False, 0, 0), (False, 70, 33)])
@pytest.mark.parametrize("seqs", [2, 17, 32, 33])
def test_more_items_than_sms(ctx, D, heads, kv_heads, causal, window, prefix, seqs):
    """Items that wait for a place, of sequences of 0 to 1100 tokens: each is done, and
    done once, in whatever order; some sequences have no keys, some more rows than keys."""
    import random
    import torch
    import ltx25_b200 as L
    rng = random.Random(seqs * D + window)
    lens_q = [rng.choice([0, 1, rng.randint(2, 300), rng.randint(300, 1100)]) for _ in range(seqs)]
    lens_q[0] = 1100
    lens_k = [max(0, n + rng.choice([prefix, 0, -n, -5])) for n in lens_q]
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, 21)
    got = L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), heads, kv_heads, D, causal=causal,
                             window=window)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, causal, window,
                                        D ** -0.5)
    check(got, want, tol, cu_q)


LONG = [
    # lens_q, lens_k
    ([1], [4500]),
    ([64], [8200]),
    ([3, 40, 0, 130], [9000, 5000, 70, 12000]),
    ([70, 10, 200], [10, 20000, 0]),          # rows that see nothing beside a long sequence
    ([128, 1], [2049, 16384]),
]


@pytest.mark.parametrize("lens_q,lens_k", LONG)
@pytest.mark.parametrize("D,heads,kv_heads", [(64, 8, 1), (64, 3, 3), (128, 8, 2), (128, 5, 1),
                                              (256, 4, 2), (256, 1, 1)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 3001), (False, 0), (False, 7000)])
def test_few_rows_over_long_keys(ctx, lens_q, lens_k, D, heads, kv_heads, causal, window):
    """Keys that several SMs share, with NaN and infinities behind the last key."""
    import torch
    import ltx25_b200 as L
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, 31, 3.0, pad=140)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=torch.bfloat16)
    for x in (k, v):
        x[cu_k[-1]:] = bad[torch.arange(140, device="cuda") % 3][:, None]
    out = torch.full((q.shape[0], heads * D), 7.0, device="cuda", dtype=torch.bfloat16)
    L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), heads, kv_heads, D, causal=causal,
                       window=window, out=out)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, causal, window,
                                        D ** -0.5)
    check(out, want, tol, cu_q)
    assert torch.all(out[cu_q[-1]:] == 7.0)


def test_long_keys_shared_in_several_rounds(ctx):
    """More items than SMs, each shared all the same, in the order of their keys."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads, D, lens_q, lens_k = 16, 8, 256, [600, 500], [13000, 12000]
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, 33)
    got = L.attention_packed(ctx, q, k, v, dev(cu_q), dev(cu_k), heads, kv_heads, D)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, True, 0, D ** -0.5)
    check(got, want, tol, cu_q)


@pytest.mark.parametrize("lens_q,lens_k,heads,kv_heads,D", [
    ([777, 333], [7700, 7300], 20, 4, 128),
    ([1000], [9000], 20, 4, 128),
    ([5] * 8, [3000] * 8, 20, 20, 64),
    ([5, 1, 3, 0, 9, 5, 5, 5], [3000, 3001, 6000, 100, 2, 7000, 3000, 0], 20, 20, 64),
    ([5] * 8, [3000] * 8, 20, 20, 256),
    ([3, 2] * 17, [2500, 1900] * 17, 5, 5, 256),
])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 2100)])
def test_a_last_round_of_few_items(ctx, lens_q, lens_k, heads, kv_heads, D, causal, window):
    """Items that fill the SMs once and a little: the last ones are shared."""
    import torch
    import ltx25_b200 as L
    q, k, v, cu_q, cu_k = make(lens_q, lens_k, heads, kv_heads, D, 35, pad=30)
    out = torch.full((q.shape[0], heads * D), 7.0, device="cuda", dtype=torch.bfloat16)
    args = (ctx, q, k, v, dev(cu_q), dev(cu_k), heads, kv_heads, D)
    L.attention_packed(*args, causal=causal, window=window, out=out)
    torch.cuda.synchronize()
    ctx.check()
    want, tol = lm_ref.attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, D, causal, window,
                                        D ** -0.5)
    check(out, want, tol, cu_q)
    assert torch.all(out[cu_q[-1]:] == 7.0)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_rows_over_long_keys_captured(ctx, D):
    """The same bits again, and a graph replayed with other lengths, some of them short;
    NaN in values that only some rows see."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads = 4, 2
    q, k, v, _, _ = make([80], [16000], heads, kv_heads, D, 5)
    v[15990, 3] = math.nan
    cq, ck = dev([0, 50, 80]), dev([0, 9000, 16000])
    args = (ctx, q, k, v, cq, ck, heads, kv_heads, D)
    a, b = L.attention_packed(*args), L.attention_packed(*args)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.attention_packed(*args, out=out)
    for lq, lk in (([0, 50, 80], [0, 9000, 16000]), ([0, 1, 80], [0, 15900, 16000]),
                   ([5, 80, 80], [0, 100, 100]), ([0, 80, 80], [0, 0, 16000])):
        cq.copy_(dev(lq))
        ck.copy_(dev(lk))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        ctx.check()
        want, tol = lm_ref.attention_packed(q, k, v, lq, lk, heads, kv_heads, D, True, 0, D ** -0.5)
        rows = slice(lq[0], lq[-1])
        assert torch.equal(out[rows].isnan(), want[rows].isnan())
        ok = ~want[rows].isnan()
        assert float(((out[rows].double() - want[rows]).abs() - tol[rows])[ok].max()) <= 1e-30
        assert torch.all(out[:lq[0]] == 7.0) and torch.all(out[lq[-1]:] == 7.0)


FIRST = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import ltx25_b200 as L
ctx = L.Context(0)
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
for D in (64, 128, 256):
    q = torch.randn((40, 4 * D), device="cuda").to(torch.bfloat16)
    k = torch.randn((9000, 2 * D), device="cuda").to(torch.bfloat16)
    cu_q, cu_k, out = ints([0, 40]), ints([0, 9000]), torch.zeros_like(q)
    cache = L.KV8Cache.empty(ctx, 4, 2, D)
    cu, n, nine, t = ints([0, 9]), ints([0]), ints([9]), ints([[2, 0]])
    back = torch.zeros((9, 4 * D), device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(L.kv8_attention_workspace(ctx, D), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.attention_packed(ctx, q, k, k, cu_q, cu_k, 4, 2, D, out=out)
        L.kv8_append(ctx, cache, k[:9], k[:9], cu, n, t)
        L.kv8_attention(ctx, cache, q[:9], cu, nine, t, 4, 128, out=back, workspace=ws)
    g.replay()
    torch.cuda.synchronize()
    ctx.check()
    assert torch.equal(out, L.attention_packed(ctx, q, k, k, cu_q, cu_k, 4, 2, D))
    assert torch.equal(back, L.kv8_attention(ctx, cache, q[:9], cu, nine, t, 4, 128))
    for x in (out, back):
        assert bool(x.isfinite().all()) and bool((x != 0).any())
print("fine")
"""


def test_a_process_s_first_calls_may_be_captured(ctx):
    """Whatever a kernel is asked once happens during a capture then."""
    import os
    import subprocess
    import sys
    import ltx25_b200
    lib = os.path.dirname(os.path.dirname(os.path.abspath(ltx25_b200.__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST, lib], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_rows_of_one_projection_and_other_streams(ctx):
    """q, k and v as column slices of one buffer, on a stream of the caller's."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads, D = 8, 2, 64
    lens = [33, 200]
    cu = lm_ref.offsets(lens)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        qkv = torch.randn((cu[-1], (heads + 2 * kv_heads) * D), device="cuda").to(torch.bfloat16)
        c = dev(cu)
    q = qkv[:, :heads * D]
    k, v = qkv[:, heads * D:(heads + kv_heads) * D], qkv[:, (heads + kv_heads) * D:]
    got = L.attention_packed(ctx, q, k, v, c, c, heads, kv_heads, D, stream=st)
    st.synchronize()
    want, tol = lm_ref.attention_packed(q, k, v, cu, cu, heads, kv_heads, D, True, 0, D ** -0.5)
    check(got, want, tol, cu)


def test_captured_and_replayed_with_new_lengths(ctx):
    """One graph, replayed after the offsets changed on the device."""
    import torch
    import ltx25_b200 as L
    heads, kv_heads, D = 4, 1, 128
    q, k, v, _, _ = make([300], [300], heads, kv_heads, D, 3)
    c = dev([0, 100, 300])
    out = torch.zeros_like(q)
    L.attention_packed(ctx, q, k, v, c, c, heads, kv_heads, D, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.attention_packed(ctx, q, k, v, c, c, heads, kv_heads, D, out=out)
    for cu in ([0, 100, 300], [0, 1, 299], [17, 17, 230]):
        c.copy_(dev(cu))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        ctx.check()
        want, tol = lm_ref.attention_packed(q, k, v, cu, cu, heads, kv_heads, D, True, 0, D ** -0.5)
        check(out, want, tol, cu)
        assert torch.all(out[:cu[0]] == 7.0) and torch.all(out[cu[-1]:] == 7.0)


def test_the_same_call_gives_the_same_bits(ctx):
    import torch
    import ltx25_b200 as L
    lens = [411, 5, 900]
    q, k, v, cu, _ = make(lens, lens, 8, 2, 128, 9)
    a = L.attention_packed(ctx, q, k, v, dev(cu), dev(cu), 8, 2, 128)
    b = L.attention_packed(ctx, q, k, v, dev(cu), dev(cu), 8, 2, 128)
    assert torch.equal(a, b)


def test_refusals(ctx):
    import torch
    import ltx25_b200 as L
    q, k, v, cu, _ = make([20], [20], 4, 2, 64)
    c = dev(cu)

    def code(fn):
        with pytest.raises(L.LtxError) as e:
            fn()
        return e.value.code

    call = lambda **kw: L.attention_packed(ctx, **{**dict(                  # noqa: E731
        q=q, k=k, v=v, cu_q=c, cu_k=c, heads=4, kv_heads=2, head_dim=64), **kw})
    assert code(lambda: call(window=-1)) == -2
    assert code(lambda: call(scale=0.0)) == -2
    assert code(lambda: call(scale=math.nan)) == -2
    assert code(lambda: call(scale=math.inf)) == -2
    assert code(lambda: call(heads=4, kv_heads=3)) == -2
    assert code(lambda: call(q=q.float())) == -3
    assert code(lambda: call(q=q[:1].expand(20, -1))) == -2               # broadcast rows
    assert code(lambda: call(cu_q=c.long())) == -2
    assert code(lambda: call(cu_k=dev([0, 10, 20]))) == -2
    assert code(lambda: call(q=q.cpu())) == -2
    assert code(lambda: call(out=q[:10])) == -2
    wide = torch.zeros((20, 4 * 64 + 4), device="cuda", dtype=torch.bfloat16)
    assert code(lambda: call(q=wide[:, 1:257])) == -8
    assert code(lambda: call(q=wide[:, :256])) == -8
    w96 = torch.zeros((20, 96), device="cuda", dtype=torch.bfloat16)
    assert code(lambda: call(q=w96, k=w96, v=w96, heads=1, kv_heads=1, head_dim=96)) == -2
    none = L.attention_packed(ctx, q[:0], k, v, c, c, 4, 2, 64)            # nothing to do
    assert none.shape == (0, 256)
    torch.cuda.synchronize()
    ctx.check()
