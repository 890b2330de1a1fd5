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
