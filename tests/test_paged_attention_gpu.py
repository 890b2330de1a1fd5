"""The paged key-value cache: append, attention of ragged batches of new tokens and of single
tokens, against the definition in 64 bits.

Tolerance of an output o = sum_j p_j v_j / l, from counting roundings (u = half a step of the
cache's type, w = 2^-24): scores are f32 sums of D exact products, off by at most
g = D w alpha sum_i |q_i k_ji| and three roundings of |s|; 2^x by the special function unit adds
2^-22 relative; p is rounded to the cache's type (u, or 2^-25 absolute where f16 is subnormal; p
is at most 2^8 times too large or small for its reference, which a floating type does not mind);
the sums over n keys are f32 (n w each, and the rescalings of a running maximum one w per 64 keys,
within that).  So |got - o| <= u |o| + A (u + 2 e + 2 n w) + F with e = g + 3 |s| w + 2^-21,
A = sum_j p_j |v_j| / l and F the flushed part.  An int8 code is within half a step of o / s_out
plus that bound over s_out; for a call with an int8 output p is two numbers of the cache's type, its
rounding and the rounding of what is left, and o is not rounded to that type: there the bound is
A (u^2 + 2 e + 2 n w) + F."""
import math

import pytest

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def make(seqs, heads, group, d, page, kind, seed=0, layout="token", scale=2.0, hide=None):
    """A cache that holds `seqs` = [(tokens, new tokens), ...], its pages in random order, unused slots
    and pages NaN, unused table entries out of range; queries for the new tokens."""
    import torch
    from lightship_b200.kv_cache import PagedKVCache
    dev = torch.device("cuda:0")
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, kind)
    used = [-(-max(n, 0) // page) for n, _ in seqs]
    most = max(used + [1]) + 1
    count = sum(used) + 2
    shape = {"token": (count, page, heads, d), "head": (count, heads, page, d)}[layout]
    k, v = (torch.full(shape, float("nan"), dtype=dt, device=dev) for _ in "kv")
    if layout == "head":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(count, generator=g)
    table = torch.full((len(seqs), most), -7, dtype=torch.int32)
    keys, values, at = [], [], 0
    for b, (n, _) in enumerate(seqs):
        ids = order[at:at + used[b]]
        at += used[b]
        table[b, :used[b]] = ids.int()
        kk = torch.randn(max(n, 0), heads, d, generator=g).to(dt)
        vv = torch.randn(max(n, 0), heads, d, generator=g).to(dt)
        keys.append(kk.to(dev))
        values.append(vv.to(dev))
        for i in range(used[b]):
            part = slice(i * page, min(n, (i + 1) * page))
            k[int(ids[i]), :part.stop - part.start] = kk[part].to(dev)
            v[int(ids[i]), :part.stop - part.start] = vv[part].to(dev)
    offsets = [0]
    for _, m in seqs:
        offsets.append(offsets[-1] + m)
    q = (scale * torch.randn(offsets[-1], heads * group, d, generator=g)).to(dt).to(dev)
    lens = torch.tensor([n for n, _ in seqs], dtype=torch.int32, device=dev)
    cache = PagedKVCache(k, v, table.to(dev), lens)
    return cache, q, torch.tensor(offsets, dtype=torch.int32, device=dev), keys, values


def define(q, pos, k, v, alpha, window, sinks, kind, fine=False):
    """(o, tolerance, whether it sees a key) for rows q [m, H, D] at positions pos over k, v [n, heads, D]."""
    import torch
    u = U[kind] ** 2 if fine else U[kind]
    m, hq, d = q.shape
    n, heads = k.shape[:2]
    o = torch.zeros(m, hq, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    j = torch.arange(n, device=q.device)
    see = j[None] <= pos[:, None]
    if window:
        see &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
    for h in range(hq):
        kk, vv = k[:, h // (hq // heads)].double(), v[:, h // (hq // heads)].double()
        s = alpha * (q[:, h].double() @ kk.T)
        g = alpha * (q[:, h].double().abs() @ kk.abs().T)
        s = torch.where(see, s, -math.inf)
        top = s.amax(1, keepdim=True).clamp(min=-1e300) if n else torch.zeros(m, 1, dtype=torch.float64, device=q.device)
        p = torch.exp(s - top)
        l = p.sum(1, keepdim=True).clamp(min=1e-300)
        o[:, h] = p @ vv / l
        e = torch.where(see, d * W * g + 3 * s.abs() * W + 2.0 ** -21, 0.0)
        f = torch.where(see, p.clamp(max=2.0 ** -25), 0.0) @ vv.abs() / l if kind == "float16" else 0.0
        tol[:, h] = (p * (u + 2 * e + 2 * n * W)) @ vv.abs() / l + f + 1e-30
        if not fine:
            tol[:, h] += U[kind] * o[:, h].abs()
        if kind == "float16":
            tol[:, h] += 2.0 ** -25
    return o, tol, see.any(1)


def check(got, q, offsets, keys, values, seqs, kind, window=0, sinks=0, alpha=None, s_out=None,
          fine=False):
    import torch
    d = q.shape[2]
    alpha = d ** -0.5 if alpha is None else alpha
    worst = 0.0
    for b, (n, m) in enumerate(seqs):
        if not m:
            continue
        rows = slice(int(offsets[b]), int(offsets[b + 1]))
        pos = torch.arange(n - m, n, device=q.device)
        o, tol, any_key = define(q[rows], pos, keys[b], values[b], alpha, window, sinks, kind, fine)
        assert bool((got[rows][~any_key] == 0).all())
        if s_out is not None:
            t = o / s_out
            off = (got[rows].double() - t.clamp(-128, 127)).abs() - 0.5 - tol / s_out
        else:
            off = (got[rows].double() - o).abs() - tol
        assert not bool(got[rows].isnan().any()), f"sequence {b}: NaN"
        worst = max(worst, float(off.max()))
    assert worst <= 0.0, worst


RAGGED = [(1, 1), (5, 5), (0, 0), (64, 64), (65, 1), (200, 200), (300, 17), (129, 128), (40, 0)]
SETS = [
    # seqs, heads, group, d, page
    (RAGGED, 2, 4, 128, 16),
    (RAGGED, 12, 1, 64, 8),
    (RAGGED, 1, 3, 64, 64),
    ([(700, 300), (513, 513)], 2, 5, 128, 32),
    ([(1000, 1000)], 1, 16, 64, 128),
    ([(257, 257), (90, 90)], 1, 40, 128, 256),
    ([(130, 130), (1, 1)], 1, 71, 64, 16),
    ([(4, 9), (0, 3), (20, 20)], 3, 2, 64, 16),       # more new tokens than places: rows before place 0
    ([(2500, 700)], 2, 12, 128, 64),
]
MASKS = [(0, 0), (1, 0), (100, 0), (64, 4), (33, 200), (5000, 3)]


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("index", range(len(SETS)))
def test_prefill(cuda, index, window, sinks, kind):
    import torch
    from lightship_b200 import ops
    seqs, heads, group, d, page = SETS[index]
    cache, q, offsets, keys, values = make(seqs, heads, group, d, page, kind, seed=index,
                                           layout="head" if index % 2 else "token")
    out = torch.full_like(q, 9.0)
    assert cache.prefill(q, offsets, window=window, sinks=sinks, out=out) is out
    check(out, q, offsets, keys, values, seqs, kind, window, sinks)
    ops.check_device()


@pytest.mark.parametrize("seqs,heads,group,d,page,window,sinks,kind", [
    ([(5000, 5000)], 8, 4, 128, 64, 0, 0, "float16"),
    ([(5000, 5000), (3000, 100), (1, 1), (2222, 2222)], 8, 2, 128, 16, 700, 9, "bfloat16"),
    ([(6000, 4000)], 6, 3, 64, 32, 300, 4, "float16"),
    ([(100 + 13 * i, 100) for i in range(60)], 4, 4, 64, 8, 0, 0, "bfloat16"),
])
def test_prefill_more_units_than_sms(cuda, seqs, heads, group, d, page, window, sinks, kind):
    """Many units of work for each SM, one after another."""
    from lightship_b200 import ops
    cache, q, offsets, keys, values = make(seqs, heads, group, d, page, kind, seed=11)
    for _ in range(3):
        out = cache.prefill(q, offsets, window=window, sinks=sinks)
    check(out, q, offsets, keys, values, seqs, kind, window, sinks)
    ops.check_device()


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1100, 0), (1030, 7), (1500, 2000), (5, 1200)])
@pytest.mark.parametrize("seqs,heads,group,d,page", [
    ([(9000, 16)], 8, 4, 128, 64),                                          # 8 units
    ([(4100, 70), (3, 3), (0, 0), (1500, 1), (2, 5), (129, 129)], 2, 4, 64, 16),
    ([(2500, 33), (700, 40), (1024, 1)], 1, 3, 128, 256),
    ([(1025, 200)], 12, 1, 64, 8),
    ([(3000, 64), (2900, 3), (90, 90)], 5, 8, 128, 32),
    ([(1300 + 3 * i, 5) for i in range(20)], 1, 2, 64, 16),
    ([(5000, 3)], 1, 71, 128, 128),
])
def test_prefill_few_rows_on_long_caches(cuda, seqs, heads, group, d, page, window, sinks, kind):
    """A unit's key tiles shared by a cluster: some parts empty, some masked whole, rows without a key."""
    import torch
    from lightship_b200 import ops
    cache, q, offsets, keys, values = make(seqs, heads, group, d, page, kind, seed=heads)
    more = dict(window=window, sinks=sinks)
    outs = [torch.full_like(q, 9.0) for _ in range(2)]
    for out in outs:
        cache.prefill(q, offsets, out=out, **more)
    check(outs[0], q, offsets, keys, values, seqs, kind, **more)
    assert torch.equal(outs[0], outs[1])
    q8 = torch.empty(q.shape, dtype=torch.int8, device=cuda)
    cache.prefill(q, offsets, out_i8=q8, s_out=0.02, **more)
    check(q8, q, offsets, keys, values, seqs, kind, s_out=0.02, fine=True, **more)
    ops.check_device()


def test_prefill_few_rows_back_to_back_and_captured(cuda):
    """Launches of clusters one behind the other, eager and replayed; rows around the batch stay."""
    import torch
    seqs = [(3000, 20), (2048, 30)]
    cache, q, offsets, keys, values = make(seqs, 4, 4, 128, 16, "float16", seed=4)
    wide = torch.cat([q[:3], q, q[:5]])
    out = torch.full_like(wide, 7.0)
    cache.prefill(wide, offsets + 3, out=out)
    for _ in range(20):
        cache.prefill(wide, offsets + 3, out=out)
    first = out.clone()
    check(first[3:-5], q, offsets, keys, values, seqs, "float16")
    assert bool((first[:3] == 7).all()) and bool((first[-5:] == 7).all())
    shifted = offsets + 3
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            cache.prefill(wide, shifted, out=out)
    out.fill_(7.0)
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("seqs,heads,group,d,page", [
    ([(1, 1), (64, 1), (65, 1), (0, 1), (1000, 1), (127, 1), (2, 1)], 2, 4, 128, 16),
    ([(200, 1)], 12, 1, 64, 16),
    ([(5000, 1), (3, 1)], 1, 8, 128, 64),
    ([(4097, 1)], 2, 3, 64, 8),
    ([(300 + 7 * i, 1) for i in range(40)], 2, 16, 64, 32),
    ([(777, 1), (778, 1)], 3, 17, 128, 256),
    ([(1500, 1), (10, 1)], 1, 71, 64, 128),
    ([(20000, 1)], 1, 6, 128, 32),
    ([(max(0, 9 - i), 1) for i in range(700)], 1, 2, 64, 8),
])
def test_decode(cuda, seqs, heads, group, d, page, window, sinks, kind):
    import torch
    from lightship_b200 import ops
    cache, q, offsets, keys, values = make(seqs, heads, group, d, page, kind, seed=len(seqs) + page,
                                           layout="head" if page > 16 else "token")
    out = torch.full_like(q, 9.0)
    assert cache.decode(q, window=window, sinks=sinks, out=out) is out
    check(out, q, offsets, keys, values, seqs, kind, window, sinks)
    again = cache.decode(q, window=window, sinks=sinks, workspace=cache.decode_workspace(q.shape[1]))
    assert torch.equal(out, again)
    ops.check_device()


@pytest.mark.parametrize("rounding", [0, 1])
@pytest.mark.parametrize("kind,d,group", [("float16", 64, 1), ("bfloat16", 128, 6)])
def test_int8_outputs(cuda, kind, d, group, rounding):
    """out_i8 alone, and beside out: within the bound, and the codes of saturated values."""
    import torch
    seqs = [(90, 90), (400, 33)]
    cache, q, offsets, keys, values = make(seqs, 2, group, d, 16, kind, seed=5)
    q8 = torch.empty(q.shape, dtype=torch.int8, device=cuda)
    assert cache.prefill(q, offsets, out_i8=q8, s_out=0.02, rounding=rounding) is q8
    check(q8, q, offsets, keys, values, seqs, kind, s_out=0.02)
    assert bool((q8 == -128).any())  # values past the range are there
    both = torch.empty_like(q8)
    out = torch.empty_like(q)
    cache.prefill(q, offsets, out=out, out_i8=both, s_out=0.02, rounding=rounding)
    assert torch.equal(both, q8)
    check(out, q, offsets, keys, values, seqs, kind)
    q1 = q[torch.tensor([89, 122], device=cuda)]
    d8 = torch.empty(q1.shape, dtype=torch.int8, device=cuda)
    one = torch.empty_like(q1)
    cache.decode(q1, out=one, out_i8=d8, s_out=0.02, rounding=rounding)
    last = [(90, 1), (400, 1)]
    check(d8, q1, torch.tensor([0, 1, 2]), keys, values, last, kind, s_out=0.02)
    check(one, q1, torch.tensor([0, 1, 2]), keys, values, last, kind)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,heads,group,window,sinks", [(64, 2, 4, 0, 0), (64, 1, 20, 300, 5), (128, 2, 4, 0, 0),
                                                        (128, 1, 3, 130, 0)])
def test_int8_codes_are_those_of_unrounded_probabilities(cuda, kind, d, heads, group, window, sinks):
    """Rounding p to the cache's type would move a code's value by up to a sixth of a step here."""
    import torch
    seqs = [(700, 300), (90, 90), (1, 1), (2600, 130), (5, 5)]
    cache, q, offsets, keys, values = make(seqs, heads, group, d, 16, kind, seed=12)
    more = dict(window=window, sinks=sinks)
    q8 = torch.empty(q.shape, dtype=torch.int8, device=cuda)
    cache.prefill(q, offsets, out_i8=q8, s_out=0.02, **more)
    check(q8, q, offsets, keys, values, seqs, kind, s_out=0.02, fine=True, **more)
    q1 = q[offsets[1:].long() - 1]
    d8 = torch.empty(q1.shape, dtype=torch.int8, device=cuda)
    cache.decode(q1, out_i8=d8, s_out=0.02, **more)
    check(d8, q1, torch.arange(len(seqs) + 1), keys, values, [(n, 1) for n, _ in seqs], kind, s_out=0.02, fine=True,
          **more)


@pytest.mark.parametrize("scale,alpha", [(30.0, None), (1e-3, None), (2.0, 1e-6), (100.0, 1.0)])
def test_sharp_and_flat_scores(cuda, scale, alpha):
    """Scores of several hundred (one key takes everything) and of nearly zero."""
    seqs = [(500, 500), (130, 1)]
    cache, q, offsets, keys, values = make(seqs, 1, 4, 64, 16, "float16", seed=3, scale=scale)
    check(cache.prefill(q, offsets, alpha=alpha), q, offsets, keys, values, seqs, "float16", alpha=alpha)
    import torch
    q1 = q[torch.tensor([499, 500], device=cuda)]
    check(cache.decode(q1, alpha=alpha), q1, torch.tensor([0, 1, 2]), keys, values, [(500, 1), (130, 1)], "float16",
          alpha=alpha)


def test_rising_scores_move_the_reference(cuda):
    """Every key scores higher than the one before it, by steps that sum to hundreds: the running maximum
    moves all the way."""
    import torch
    n, d = 600, 64
    for sign in (1.0, -1.0):
        cache, q, offsets, keys, values = make([(n, n)], 1, 2, d, 16, "float16", seed=1)
        ramp = (sign * torch.arange(n, device=cuda).half() / 64)[:, None, None].expand(n, 1, d)
        keys[0] = ramp.contiguous()
        cache.append(keys[0], values[0], offsets)
        q.fill_(1.0)
        check(cache.prefill(q, offsets, alpha=1.0), q, offsets, keys, values, [(n, n)], "float16", alpha=1.0)
        check(cache.decode(q[-1:], alpha=1.0), q[-1:], torch.tensor([0, 1]), keys, values, [(n, 1)], "float16", alpha=1.0)


def test_rows_around_the_batch_are_left(cuda):
    """Rows before the first offset and behind the last sequence keep what they held; strided queries."""
    import torch
    seqs = [(50, 50), (70, 3)]
    cache, q, offsets, keys, values = make(seqs, 2, 2, 64, 16, "float16", seed=9)
    wide = torch.randn(60, 12, 64, device=cuda).half()
    rows = offsets + 4
    wide[4:57, 3:7] = q
    out = torch.full((60, 4, 64), 5.0, dtype=torch.float16, device=cuda)
    cache.prefill(wide[:, 3:7], rows, out=out)
    check(out[4:57], q, offsets, keys, values, seqs, "float16")
    assert bool((out[:4] == 5).all()) and bool((out[57:] == 5).all())
    two = torch.randn(2, 9, 64, device=cuda).half()
    two[:, 2:6] = q[torch.tensor([49, 52], device=cuda)]
    check(cache.decode(two[:, 2:6]), two[:, 2:6], torch.tensor([0, 1, 2]), keys, values, [(50, 1), (70, 1)], "float16")


@pytest.mark.parametrize("d", [64, 128])
def test_places_that_no_row_sees_have_no_effect(cuda, d):
    """With a window, freed pages (table entry out of range) and NaN in every place outside it."""
    import torch
    from lightship_b200 import ops
    page, n, window, sinks = 16, 1000, 150, 5
    seqs = [(n, 20)]
    cache, q, offsets, keys, values = make(seqs, 1, 4, d, page, "float16", seed=4)
    table = cache.page_table
    low = n - 20 - window + 1  # first place in some row's window
    for j in range(sinks, low):
        cache.k[int(table[0, j // page]), j % page] = float("nan")
        cache.v[int(table[0, j // page]), j % page] = float("nan")
    freed = [i for i in range(n // page) if i * page >= sinks and (i + 1) * page <= low]
    assert len(freed) > 40
    table[0, freed] = -3
    check(cache.prefill(q, offsets, window=window, sinks=sinks), q, offsets, keys, values, seqs, "float16", window, sinks)
    for j in range(low, n - window):  # and for the last row alone
        cache.k[int(table[0, j // page]), j % page] = float("nan")
        cache.v[int(table[0, j // page]), j % page] = float("inf")
    one = cache.decode(q[-1:], window=window, sinks=sinks)
    check(one, q[-1:], torch.tensor([0, 1]), keys, values, [(n, 1)], "float16", window, sinks)
    ops.check_device()


def test_not_finite_values_that_are_seen(cuda):
    """NaN in K or V at a visible place gives NaN; an infinite key score wins or drops out."""
    import torch
    for where in ("k", "v"):
        cache, q, offsets, keys, values = make([(100, 100)], 1, 1, 64, 16, "float16", seed=2)
        getattr(cache, where)[int(cache.page_table[0, 0]), 3, 0, :] = float("nan")
        out = cache.prefill(q, offsets)
        assert bool(out[3:].isnan().all())
        assert bool(cache.decode(q[-1:]).isnan().all())
        if where == "k":  # a row that does not see the key
            assert not bool(out[:3].isnan().any())


def test_append_matches_definition(cuda):
    """New tokens of a ragged batch, out of a fused projection, in both layouts; all other places stay."""
    import torch
    from lightship_b200 import ops
    for layout, page, heads, d in (("token", 16, 2, 64), ("head", 8, 3, 128), ("token", 256, 1, 128), ("head", 64, 8, 64)):
        seqs = [(37, 5), (1, 1), (0, 0), (300, 300), (64, 64), (100, 0), (17, 1)]
        cache, q, offsets, keys, values = make(seqs, heads, 1, d, page, "float16", seed=page, layout=layout)
        before = cache.k.clone(), cache.v.clone()
        tokens = int(offsets[-1])
        fused = torch.randn(tokens + 4, 3 * heads, d, device=cuda).half()
        rows = offsets + 2
        cache.append(fused[:, heads:2 * heads], fused[:, 2 * heads:], rows)
        want = before[0].clone(), before[1].clone()
        for b, (n, m) in enumerate(seqs):
            for i in range(m):
                p = n - m + i
                at = int(cache.page_table[b, p // page])
                want[0][at, p % page] = fused[int(rows[b]) + i, heads:2 * heads]
                want[1][at, p % page] = fused[int(rows[b]) + i, 2 * heads:]
        for got, w in zip((cache.k, cache.v), want):
            assert torch.equal(got.view(torch.int16) if got.is_contiguous() else got.contiguous().view(torch.int16),
                               w.contiguous().view(torch.int16))
        ops.check_device()


def test_device_data_out_of_range(cuda):
    """Bad lengths, pages and offsets: the error word, no access out of range, the other sequences right."""
    import torch
    from lightship_b200 import _lib, ops
    from lightship_b200._lib import LightShipError
    seqs = [(40, 40), (50, 50), (30, 30)]
    cases = 6
    for case in range(cases):
        cache, q, offsets, keys, values = make(seqs, 1, 2, 64, 16, "float16", seed=case)
        tokens = q.shape[0]
        if case == 0:
            cache.kv_lens[1] = -5
        elif case == 1:
            cache.kv_lens[1] = 1 << 30
            cache.page_table[1].clamp_(min=0)
        elif case == 2:
            cache.page_table[1, 0] = cache.k.shape[0]
        elif case == 3:
            cache.page_table[1, 1] = -1
        elif case == 4:
            offsets[1], offsets[2] = 90, 40
        else:
            offsets[3] = 5000
        k0 = cache.k.clone()
        good = {4: [], 5: [0, 1]}.get(case, [0, 2])
        ops.check_device()
        out = cache.prefill(q, offsets)
        with pytest.raises(LightShipError) as e:
            ops.check_device()
        assert e.value.code == _lib.ERROR_EXECUTION_FAILED
        for b in good:
            at = slice(int(offsets[b]), int(offsets[b + 1]))
            check(out[at], q[at], torch.tensor([0, seqs[b][1]]), [keys[b]], [values[b]], [seqs[b]], "float16")
        if case < 4:
            one = cache.decode(q[torch.tensor([39, 89, 119], device=cuda)])
            with pytest.raises(LightShipError):
                ops.check_device()
            for b in good:
                check(one[b:b + 1], q[[39, 89, 119][b]][None], torch.tensor([0, 1]), [keys[b]], [values[b]],
                      [(seqs[b][0], 1)], "float16")
        new = torch.zeros(tokens, 1, 64, dtype=torch.float16, device=cuda)
        cache.append(new, new, offsets)
        if case != 1:  # a length past the table leaves room for the new tokens
            with pytest.raises(LightShipError):
                ops.check_device()
        else:
            try:
                ops.check_device()
            except LightShipError:
                pass
        assert cache.k.shape == k0.shape


def test_far_pages(cuda):
    """A cache whose offsets pass 32 bits: pages at both of its ends."""
    import torch
    from lightship_b200.kv_cache import PagedKVCache
    count, page, heads, d = 36000, 64, 8, 128  # 2.36e9 elements each
    k = torch.empty(count, page, heads, d, dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    n = 200
    table = torch.tensor([[count - 1, 0, count - 2, 33000]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    cache = PagedKVCache(k, v, table, lens)
    g = torch.Generator().manual_seed(1)
    kk, vv, q = (torch.randn(n, h, d, generator=g).bfloat16().to(cuda) for h in (heads, heads, heads * 2))
    off = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    cache.append(kk, vv, off)
    check(cache.prefill(q, off), q, off, [kk], [vv], [(n, n)], "bfloat16")
    check(cache.decode(q[-1:]), q[-1:], torch.tensor([0, 1]), [kk], [vv], [(n, 1)], "bfloat16")


def test_streams_and_graphs(cuda):
    """Prompt and token steps on another stream, and captured; two graphs that decode at the same time
    with a workspace each."""
    import torch
    from lightship_b200 import ops
    seqs = [(900, 1), (64, 1)]
    cache, q, offsets, keys, values = make(seqs, 2, 4, 128, 16, "bfloat16", seed=8)
    want = cache.decode(q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cache.decode(q)
        pre = cache.prefill(q, offsets)
    s.synchronize()
    assert torch.equal(got, want)
    check(pre, q, offsets, keys, values, seqs, "bfloat16")
    graphs, outs, qs = [], [], []
    for i in range(2):
        qs.append(q.clone())
        outs.append(torch.empty_like(q))
        ws = cache.decode_workspace(q.shape[1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.decode(qs[i], out=outs[i], workspace=ws)
        graphs.append((g, ws))
    qs[1].copy_(q.flip(0))
    cache.kv_lens.copy_(torch.tensor([900, 64], dtype=torch.int32))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    check(outs[1], qs[1], offsets, keys, values, seqs, "bfloat16")
    cache.kv_lens[0] = 700  # lengths are read when the graph runs
    graphs[0][0].replay()
    check(outs[0], q, offsets, [keys[0][:700], keys[1]], [values[0][:700], values[1]], [(700, 1), (64, 1)], "bfloat16")
    ops.check_device()


def test_prompt_chunks_and_tokens_agree(cuda):
    """A run as a server makes it: RMS norm to int8, the INT8 projections of Q, K and V with an f16 output,
    append, attention with an int8 output into the INT8 output projection; a prompt in one piece, in
    chunks, and its last tokens one at a time give the same hidden states."""
    import torch
    from lightship_b200 import ops
    from lightship_b200.backend import CudaBackend, DataType, OperatorDef, OperatorType, Quantization, Tensor
    from lightship_b200.kv_cache import PagedKVCache
    import numpy as np
    rng = np.random.default_rng(3)
    hidden, heads, kv, d, page, n = 512, 8, 2, 64, 16, 75
    be = CudaBackend()
    wq = rng.normal(0, 0.06, ((heads + 2 * kv) * d, hidden)).astype(np.float32)
    wo = rng.normal(0, 0.05, (hidden, heads * d)).astype(np.float32)
    gamma = torch.from_numpy(rng.uniform(0.8, 1.2, hidden).astype(np.float32)).to(cuda)
    x = torch.from_numpy(rng.normal(0, 1, (n, hidden)).astype(np.float32)).to(cuda)
    s_x, s_o = 4.0 / 127, 2.0 / 127

    def project(w, codes, s_in, out, residual=None):
        tin = Tensor("x", list(codes.shape), DataType.QInt8, codes, quantization=Quantization([s_in]))
        dt = DataType.F16 if out.dtype == torch.float16 else DataType.F32
        tout = Tensor("y", list(out.shape), dt, out)
        op = be.compile_operator(OperatorDef("fc", OperatorType.FullyConnected), None,
                                 [tin, Tensor("w", list(w.shape), DataType.F32, w)], [tout])
        ins = [tin] if residual is None else [tin, Tensor("r", list(residual.shape), DataType.F32, residual)]
        be.execute(op, ins, [tout], stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out

    def run(chunks):
        count = -(-n // page)
        k = torch.full((count, page, kv, d), float("nan"), dtype=torch.float16, device=cuda)
        v = torch.full_like(k, float("nan"))
        table = torch.arange(count, dtype=torch.int32, device=cuda).flip(0)[None].contiguous()
        lens = torch.zeros(1, dtype=torch.int32, device=cuda)
        cache = PagedKVCache(k, v, table, lens)
        outs, at = [], 0
        for m in chunks:
            part = x[at:at + m]
            codes = torch.empty(m, hidden, dtype=torch.int8, device=cuda)
            ops.rmsnorm(part, gamma, out_i8=codes, s_out=s_x)
            qkv = project(wq, codes, s_x, torch.empty(m, (heads + 2 * kv) * d, dtype=torch.float16, device=cuda))
            qkv = qkv.view(m, heads + 2 * kv, d)
            lens += m
            offsets = torch.tensor([0, m], dtype=torch.int32, device=cuda)
            cache.append(qkv[:, heads:heads + kv], qkv[:, heads + kv:], offsets)
            o = torch.empty(m, heads, d, dtype=torch.int8, device=cuda)
            if m == 1:
                cache.decode(qkv[:, :heads], window=40, sinks=3, out_i8=o, s_out=s_o)
            else:
                cache.prefill(qkv[:, :heads], offsets, window=40, sinks=3, out_i8=o, s_out=s_o)
            outs.append(project(wo, o.view(m, heads * d), s_o, torch.empty(m, hidden, device=cuda), part))
            at += m
        ops.check_device()
        return torch.cat(outs)

    whole = run([n])
    assert not bool(whole.isnan().any())
    # one code of one input moves an output by s_o * |w|: allow a few codes to fall the other way
    step = 4 * s_o * float(np.abs(wo).max())
    for chunks in ([20, 2, 33, 20], [70] + [1] * 5, [1] * 10 + [65]):
        assert float((run(chunks) - whole).abs().max()) <= step


def test_captured_token_steps(cuda):
    """One captured step - the lengths move on, the new keys and values are appended, the new token attends -
    replayed over many tokens, across page and tile borders, on top of other launches that overlap."""
    import torch
    from lightship_b200 import ops
    from lightship_b200.kv_cache import PagedKVCache
    heads, group, d, page, batch, steps = 2, 4, 128, 16, 3, 150
    g = torch.Generator().manual_seed(6)
    start = [0, 50, 700]
    most = -(-(max(start) + steps) // page)
    k = torch.full((batch * most + 1, page, heads, d), float("nan"), dtype=torch.float16, device=cuda)
    v = torch.full_like(k, float("nan"))
    table = torch.randperm(batch * most, generator=g)[:batch * most].view(batch, most).int().to(cuda)
    lens = torch.zeros(batch, dtype=torch.int32, device=cuda)
    cache = PagedKVCache(k, v, table, lens)
    keys = [torch.randn(n + steps, heads, d, generator=g).half().to(cuda) for n in start]
    values = [torch.randn(n + steps, heads, d, generator=g).half().to(cuda) for n in start]
    lens.copy_(torch.tensor(start, dtype=torch.int32))
    off = torch.tensor([0] + start, dtype=torch.int32).cumsum(0).int().to(cuda)
    cache.append(torch.cat([x[:n] for x, n in zip(keys, start)]), torch.cat([x[:n] for x, n in zip(values, start)]), off)
    one = torch.arange(batch + 1, dtype=torch.int32, device=cuda)
    kn = torch.empty(batch, heads, d, dtype=torch.float16, device=cuda)
    vn, q, x = torch.empty_like(kn), torch.empty(batch, heads * group, d, dtype=torch.float16, device=cuda), None
    out = torch.empty_like(q)
    x = torch.empty(batch, heads * group * d, dtype=torch.float16, device=cuda)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        lens.add_(1)
        cache.append(kn, vn, one)
        ops.rmsnorm(q.view(batch, -1), out=x)
        cache.decode(q, out=out)
    for t in range(steps):
        kn.copy_(torch.stack([y[n + t] for y, n in zip(keys, start)]))
        vn.copy_(torch.stack([y[n + t] for y, n in zip(values, start)]))
        q.copy_(2 * torch.randn(q.shape, generator=g).half())
        graph.replay()
        if t % 7 == 0 or t == steps - 1:
            now = [(n + t + 1, 1) for n in start]
            check(out, q, one, [y[:n] for y, (n, _) in zip(keys, now)], [y[:n] for y, (n, _) in zip(values, now)], now,
                  "float16")
    assert lens.tolist() == [n + steps for n in start]
    ops.check_device()


def test_two_streams_at_once(cuda):
    """Prompt and token calls of two caches on two streams, many at a time, give what they give alone."""
    import torch
    from lightship_b200 import ops
    a = make([(3000, 500), (100, 100)], 4, 2, 128, 16, "float16", seed=1)
    b = make([(5000, 1), (800, 1), (1, 1)], 4, 4, 64, 32, "bfloat16", seed=2)
    want = a[0].prefill(a[1], a[2]), b[0].decode(b[1])
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            got[0].append(a[0].prefill(a[1], a[2]))
        with torch.cuda.stream(streams[1]):
            got[1].append(b[0].decode(b[1]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)
    ops.check_device()


def test_first_call_inside_a_capture(cuda):
    """A process whose first use of the operators is a graph capture."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path.insert(0, %r)
from lightship_b200 import ops
from lightship_b200.kv_cache import PagedKVCache
k = torch.randn(80, 16, 2, 64, device="cuda").half()
v = torch.randn_like(k)
lens = torch.tensor([1200], dtype=torch.int32, device="cuda")
cache = PagedKVCache(k, v, torch.arange(80, dtype=torch.int32, device="cuda")[None], lens)
q = torch.randn(1, 4, 64, device="cuda").half()
off = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
new = torch.randn(1, 2, 64, device="cuda").half()
outs = [torch.zeros_like(q) for _ in range(2)]
x = torch.randn(3, 64, device="cuda")
y = torch.empty_like(x)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.rmsnorm(x, out=y)
    cache.append(new, new, off)
    cache.prefill(q, off, out=outs[0])
    cache.decode(q, out=outs[1])
g.replay()
torch.cuda.synchronize()
assert float((outs[0] - outs[1]).abs().max()) < 4e-3 and float(outs[0].abs().max()) > 0
assert torch.allclose(y, x / (x.square().mean(1, keepdim=True) + 1e-5).sqrt(), atol=1e-5)
ops.check_device()
""" % os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
