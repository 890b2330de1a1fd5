"""Paged attention at its limits."""
import math

import pytest

from tests.test_paged_attention_gpu import U, W, check, make

pytestmark = pytest.mark.gpu


# ---- probabilities far below the largest one

def _tail(n, heads, group, d, kind, x, new):
    """One key that scores 0 and n - 1 keys that score -x; the values are 0 there and 1 here."""
    import torch
    from lightship_b200.kv_cache import PagedKVCache
    page = 256
    pages = -(-n // page)
    dt = getattr(torch, kind)
    dev = torch.device("cuda:0")
    k = torch.zeros(pages, page, heads, d, dtype=dt, device=dev)
    v = torch.ones_like(k)
    k[..., 0] = -x
    k[0, 0], v[0, 0] = 0.0, 0.0
    cache = PagedKVCache(k, v, torch.arange(pages, dtype=torch.int32, device=dev)[None],
                         torch.tensor([n], dtype=torch.int32, device=dev))
    q = torch.zeros(new, heads * group, d, dtype=dt, device=dev)
    q[..., 0] = 1.0
    return cache, q, torch.tensor([0, new], dtype=torch.int32, device=dev)


# scores in f16: 2^-25.09, 2^-24.91 and 2^-28 of the largest probability
@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("x", [17.390625, 17.265625, 19.40625])
@pytest.mark.parametrize("n,heads,group,d,new", [
    (131072, 1, 4, 64, 0), (131072, 2, 1, 128, 0), (131072, 1, 40, 128, 0),         # single tokens
    (131072, 1, 4, 64, 3), (131072, 1, 1, 128, 40), (20000, 8, 4, 128, 700), (20000, 8, 4, 64, 700)])
def test_faint_keys_behind_a_strong_one(cuda, n, heads, group, d, new, x, kind):
    """What the faint keys give is N p / (1 + N p).  The bound is the one of test_paged_attention_gpu with
    what f16 still loses of p: single tokens hold 2^15 p, so half a step of its subnormals is 2^-40 of p;
    prompts hold 2^7 p (p reaches 2^8 there), 2^-32.  bf16 loses nothing: its exponents are f32's."""
    import torch
    x = float(torch.tensor(x, dtype=getattr(torch, kind)))
    cache, q, off = _tail(n, heads, group, d, kind, x, max(new, 1))
    first = n - max(new, 1)
    keys = torch.arange(first, n, dtype=torch.float64, device=cuda)  # faint keys that each row sees
    p = math.exp(-x)
    l = 1.0 + keys * p
    o = keys * p / l
    lost = 0.0 if kind == "bfloat16" else (2.0 ** -32 if new else 2.0 ** -40)
    e = 3 * x * W + 2.0 ** -21

    def bound(u):
        return o * (u + 2 * e + 2 * n * W) + keys * lost / l
    call = (lambda **kw: cache.prefill(q, off, alpha=1.0, **kw)) if new else (lambda **kw: cache.decode(q, alpha=1.0, **kw))
    got = call().double()
    tol = bound(U[kind]) + U[kind] * o + (2.0 ** -25 if kind == "float16" else 0.0)
    assert float(((got - o[:, None, None]).abs() - tol[:, None, None]).max()) <= 0.0
    s = float(o[-1]) / 100
    q8 = torch.empty(q.shape, dtype=torch.int8, device=cuda)
    call(out_i8=q8, s_out=s)
    off8 = (q8.double() - (o / s)[:, None, None]).abs() - 0.5 - (bound(U[kind] ** 2) / s)[:, None, None]
    assert float(off8.max()) <= 0.0


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_just_below_a_move_of_the_reference(cuda, d, kind):
    """Each tile of 128 keys scores 5.4 (2^7.8) above the one before it, and each second one lower again."""
    import torch
    n = 1100
    for up in ([0.0, 5.4], [0.0, 5.4, 10.8, 16.2, 5.4]):
        cache, q, offsets, keys, values = make([(n, n)], 2, 2, d, 16, kind, seed=2)
        steps = torch.tensor(up, device=cuda)[torch.arange(n, device=cuda) // 128 % len(up)]
        keys[0][..., 0] = steps[:, None].to(keys[0].dtype)
        keys[0][..., 1:] = 0.0
        q.fill_(0.0)
        q[..., 0] = 1.0
        cache.append(keys[0], values[0], offsets)
        check(cache.prefill(q, offsets, alpha=1.0), q, offsets, keys, values, [(n, n)], kind, alpha=1.0)
        check(cache.decode(q[-1:], alpha=1.0), q[-1:], torch.tensor([0, 1]), keys, values, [(n, 1)], kind, alpha=1.0)


# ---- bad device data, shown on the whole buffers

@pytest.mark.parametrize("case", ["negative length", "length past the table", "page past the cache", "negative page",
                                  "offsets that decrease", "offset past the tokens", "more tokens than places"])
def test_append_of_bad_device_data_writes_nothing_else(cuda, case):
    """Guard pages on both sides of the cache: the well-formed sequences' places take their tokens, the bad
    one's good places theirs, everything else stays to the bit, and the error word is raised."""
    import torch
    from lightship_b200 import _lib, ops
    from lightship_b200._lib import LightShipError
    from lightship_b200.kv_cache import PagedKVCache
    page, heads, d, pages, guard, most = 16, 2, 64, 12, 5, 4
    g = torch.Generator().manual_seed(3)
    whole = [torch.randn(pages + 2 * guard, page, heads, d, generator=g).half().to(cuda) for _ in range(2)]
    k, v = (w[guard:guard + pages] for w in whole)
    table = torch.tensor([[3, 8, 1, -1], [10, 0, 5, 11], [7, 2, 4, -1]], dtype=torch.int32)
    lens, offs = [40, 50, 30], [0, 40, 90, 120]
    if case == "negative length":
        lens[1] = -5
    elif case == "length past the table":
        lens[1] = 1 << 30
    elif case == "page past the cache":
        table[1, 0] = pages
    elif case == "negative page":
        table[1, 1] = -1
    elif case == "offsets that decrease":
        offs[1], offs[2] = 90, 40
    elif case == "offset past the tokens":
        offs[3] = 5000
    else:
        lens[1] = 20
    tokens = 120
    new = [torch.randn(tokens, heads, d, generator=g).half().to(cuda) for _ in range(2)]
    want = [w.clone() for w in whole]
    for b in range(3):
        begin, end = offs[b], offs[b + 1]
        if not 0 <= begin <= end <= tokens:
            continue
        n = min(max(lens[b], 0), most * page)
        for t in range(begin, end):
            p = n - (end - begin) + t - begin
            if p < 0 or not 0 <= int(table[b, p // page]) < pages:
                continue
            at = guard + int(table[b, p // page])
            for w, x in zip(want, new):
                w[at, p % page] = x[t]
    cache = PagedKVCache(k, v, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda))
    ops.check_device()
    cache.append(new[0], new[1], torch.tensor(offs, dtype=torch.int32, device=cuda))
    with pytest.raises(LightShipError) as e:
        ops.check_device()
    assert e.value.code == _lib.ERROR_EXECUTION_FAILED
    for got, w in zip(whole, want):
        assert torch.equal(got.view(torch.int16), w.view(torch.int16))


@pytest.mark.parametrize("d", [64, 128])
def test_infinite_scores(cuda, d):
    """A key that scores -inf drops out; one that scores +inf makes NaN of the rows that see it and of no
    other."""
    import torch
    n, at = 300, 37
    for sign in (-1.0, 1.0):
        cache, q, offsets, keys, values = make([(n, n)], 1, 2, d, 16, "float16", seed=6)
        q.abs_().clamp_(min=0.01)
        cache.k[int(cache.page_table[0, at // 16]), at % 16, 0, 5] = sign * math.inf
        out, one = cache.prefill(q, offsets), cache.decode(q[-1:])
        if sign > 0:
            assert bool(out[at:].isnan().all()) and bool(one.isnan().all())
            check(out[:at], q[:at], torch.tensor([0, at]), [keys[0][:at]], [values[0][:at]], [(at, at)], "float16")
            continue
        left = [i for i in range(n) if i != at]
        rows = torch.cat([out[:at], out[at + 1:]])  # the row of the place itself sees the keys before it
        qs = torch.cat([q[:at], q[at + 1:]])
        off = torch.tensor([0, n - 1])
        check(rows, qs, off, [keys[0][left]], [values[0][left]], [(n - 1, n - 1)], "float16")
        check(out[at:at + 1], q[at:at + 1], torch.tensor([0, 1]), [keys[0][:at]], [values[0][:at]], [(at, 1)], "float16")
        check(one, q[-1:], torch.tensor([0, 1]), [keys[0][left]], [values[0][left]], [(n - 1, 1)], "float16")


# ---- what a call takes does not hang on the table's width or on empty slots

def _time(call):
    """us a call: the best of several replays of twenty captured ones."""
    import torch
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            call()
    best = math.inf
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(15):
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        best = min(best, begin.elapsed_time(end) * 1e3 / 20)
    return best


@pytest.mark.parametrize("live", [[0, 1, 2, 3], [0, 700, 2000, 4095], [4092, 4093, 4094, 4095], [31, 32, 64, 1000]])
@pytest.mark.parametrize("longest", [200, 3000])
def test_decode_of_a_batch_padded_with_empty_slots(cuda, longest, live):
    """Four sequences among 4096 slots: the values, zeros for the others, and a time that does not follow
    where the empty slots are."""
    import torch
    slots = 4096
    lens = {b: n for b, n in zip(live, [longest, 100, 1, longest - 50])}
    seqs = [(lens.get(b, 0), 1) for b in range(slots)]
    cache, q, offsets, keys, values = make(seqs, 2, 4, 128, 16, "float16", seed=live[1])
    out = torch.full_like(q, 9.0)
    ws = cache.decode_workspace(8)
    cache.decode(q, out=out, workspace=ws)
    rows = torch.tensor(live, device=cuda)
    check(out[rows], q[rows], torch.arange(5), [keys[b] for b in live], [values[b] for b in live],
          [seqs[b] for b in live], "float16")
    out[rows] = 0.0
    assert bool((out == 0).all())
    packed = cache.kv_lens.clone()
    took = _time(lambda: cache.decode(q, out=out, workspace=ws))
    cache.kv_lens.zero_()
    cache.kv_lens[-4:] = packed[rows]
    cache.page_table[-4:] = cache.page_table[rows].clone()
    assert took <= 2 * _time(lambda: cache.decode(q, out=out, workspace=ws))


def _widened(cache, places):
    """The same cache under a table of `places` per sequence."""
    import torch
    from lightship_b200.kv_cache import PagedKVCache
    page = cache.k.shape[1]
    table = torch.full((cache.batch, places // page), -1, dtype=torch.int32, device=cache.device)
    table[:, :cache.page_table.shape[1]] = cache.page_table[:, :places // page]
    return PagedKVCache(cache.k, cache.v, table, cache.kv_lens)


def test_short_prompts_under_a_wide_table(cuda):
    """A table with room for 8192 places a sequence: the rows are those of a fitted table, to the bit, and the
    call does not pay for a cluster's exchange (7.4, 8.5 and 10.5 us fitted; 9.1, 10.8 and 13.5 wide; with the
    exchange 11.3, 13.7 and 15.3)."""
    import torch
    took = [0.0, 0.0]
    for kind, n, heads, group, d, page in (("float16", 100, 12, 1, 64, 16), ("float16", 100, 8, 4, 128, 64),
                                           ("bfloat16", 256, 8, 4, 128, 64)):
        cache, q, offsets, keys, values = make([(n, n)], heads, group, d, page, kind, seed=n)
        wide = _widened(cache, 8192)
        outs = [torch.full_like(q, 9.0) for _ in range(2)]
        codes = [torch.full(q.shape, 99, dtype=torch.int8, device=cuda) for _ in range(2)]
        for i, c in enumerate((cache, wide)):
            c.prefill(q, offsets, out=outs[i], out_i8=codes[i], s_out=0.02)
            took[i] += _time(lambda: c.prefill(q, offsets, out=outs[i]))
        check(outs[1], q, offsets, keys, values, [(n, n)], kind)
        assert torch.equal(codes[0], codes[1])
        wide.prefill(q, offsets, out=outs[1])
        assert torch.equal(outs[0], outs[1])
    assert took[1] <= 1.4 * took[0], took


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 3), (3000, 0)])
def test_short_and_long_units_of_one_call(cuda, window, sinks, kind):
    """Clusters that share their unit beside such that leave it to one CTA: 7, 8, 9 and 15 key tiles, one, none."""
    from lightship_b200 import ops
    seqs = [(896, 30), (897, 30), (1024, 9), (1025, 1), (1152, 7), (1920, 33), (5, 5), (1, 1), (0, 0), (0, 3), (6000, 12)]
    for heads, group, d in ((1, 2, 64), (1, 4, 128)):
        cache, q, offsets, keys, values = make(seqs, heads, group, d, 16, kind, seed=d)
        wide = _widened(cache, 65536)
        for c in (cache, wide):
            check(c.prefill(q, offsets, window=window, sinks=sinks), q, offsets, keys, values, seqs, kind, window, sinks)
    ops.check_device()


@pytest.mark.parametrize("live", [[0, 1, 2, 3], [0, 300, 800, 1023], [1020, 1021, 1022, 1023], list(range(5, 1024, 33)),
                                  list(range(31, 1024, 31))])
def test_prefill_of_a_batch_padded_with_empty_slots(cuda, live):
    """Up to 32 prompts among 1024 slots take what they take alone and one look at the batch (32 rounds of
    loads that come from L2, under 0.8 us each); 33 are right too."""
    import torch
    slots = 1024
    lens = {b: (1500, 700, 100, 1100)[i % 4] // (1 if len(live) == 4 else 4) for i, b in enumerate(live)}
    seqs = [(lens.get(b, 0), lens.get(b, 0) // (1 + b % 2)) for b in range(slots)]
    cache, q, offsets, keys, values = make(seqs, 4, 4, 128, 16, "float16", seed=len(live))
    out = torch.full_like(q, 9.0)
    cache.prefill(q, offsets, out=out)
    check(out, q, offsets, keys, values, seqs, "float16")
    if len(live) > 32:
        return
    from lightship_b200.kv_cache import PagedKVCache
    rows = torch.tensor(live, device=cuda)
    alone = PagedKVCache(cache.k, cache.v, cache.page_table[rows].contiguous(), cache.kv_lens[rows].contiguous())
    off = torch.cat([offsets[rows], offsets[-1:]])
    again = torch.empty_like(out)
    took = _time(lambda: cache.prefill(q, offsets, out=out)), _time(lambda: alone.prefill(q, off, out=again))
    assert torch.equal(out, again)
    assert took[0] <= took[1] + 25.0, took
