"""GPU: the 4-bit cache and its attention where values are very small, very large or outweighed, and prompts against a bound that holds
the roundings the prompt kernel states.

Prompts on dense rows: keys and values are given to the oracle as the kernel has them, rounded through float32 to the type (float16: at most
65504), so that what is left is
 * a score: products accumulated in float32 over at most 128 columns, 2^-17 of the sum of |q| |k| (and of one), twice with the ratio to the sum;
 * the weights' rounding to the type, h = finfo(type).eps / 2 of the weighted sum of |v|; float16 weights below 2^-14 are off by 2^-25, where
   the largest of a row is 2^7 at least: 2^-32 of the sum of |v| over the positions;
 * sums of n positions in float32, 16 at a time: n / 16 additions of 2^-22 at most of the weighted sum of |v|;
 * the output's rounding, h of it, and of the smallest normal number below that.
Attention over the codes, 16-bit types: weights and their products with s are float16, 2^-11 with the ratio to the sum, of the weighted sums of
|v| and of s code, instead of h; the rest as above (scores: the same bound covers eight groups)."""
import numpy as np
import pytest

from oracle import cache4_np as O

pytestmark = pytest.mark.gpu
HALVES = ["bfloat16", "float16"]


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def held(x):
    """Rows [batch, seq, heads, dim] as the cache holds them: [batch, heads, seq, dim]."""
    return O.held(host(x)).transpose(0, 2, 1, 3)


def dense(torch, x, dtype):
    y = torch.from_numpy(np.clip(x, -65504, 65504) if dtype == "float16" else x).to(torch.float32)
    return y.to(getattr(torch, dtype)).double().numpy()


def rows(torch, rng, shape, dtype, size=1.0):
    x = (rng.standard_normal(shape) + rng.standard_normal(shape[-2:])) * size
    return torch.from_numpy(x.astype(np.float32)).cuda().to(getattr(torch, dtype))


def needs(torch, cache, dtype, heads, seq, high, window=0):
    from rotor_b200 import abi, ops
    return abi.lib.rotor_b200_cache4_attend_workspace_bytes(cache._ref, ops.type_code(getattr(torch, dtype)), heads, seq, high, window)


def bound_of(torch, dtype, want, size, reach, weight, many, sum_v, spare):
    half, tiny = torch.finfo(getattr(torch, dtype)).eps / 2, torch.finfo(getattr(torch, dtype)).smallest_normal
    return (size * (weight + np.expm1(2.0 ** -16 * (reach[..., None] + 1)) + many / 16 * 2.0 ** -22) + spare * sum_v + half * np.abs(want) + half * tiny
            + 1e-30)


def prompt(torch, seed, dtype, batch, seq, heads, kv, dim, past, window=0, sinks=False, scale=None):
    """(output, its oracle, the bound); the call is one that goes over dense rows."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(seed)
    total = max(past) + seq
    cache = Cache4(batch, kv, total, dim)
    assert needs(torch, cache, dtype, heads, seq, max(past), window) >= 4 * batch * kv * total * dim
    k, v = rows(torch, rng, (batch, total, kv, dim), "bfloat16"), rows(torch, rng, (batch, total, kv, dim), "bfloat16")
    cache.append(k, v, 0)
    q = torch.from_numpy(rng.standard_normal((batch, seq, heads, dim)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    s = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if sinks else None
    lengths = torch.tensor(past, dtype=torch.int32, device="cuda")
    got = cache.attend(q, lengths, scale=scale, window=window, sinks=s, longest=max(past))
    kd, vd = dense(torch, held(k), dtype), dense(torch, held(v), dtype)
    use = dim ** -0.5 if scale is None else scale
    args = past, use, window, None if s is None else host(s)
    want, size, reach = O.attend(host(q), kd, vd, *args)
    bound = bound_of(torch, dtype, want, size, reach, torch.finfo(getattr(torch, dtype)).eps / 2, total, np.abs(vd).sum(2).max(), 2.0 ** -32)
    return got, want, bound, (host(q), kd, vd, args)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("seq,heads,kv,dim,past,kw", [
    (300, 20, 5, 128, 0, {}), (300, 6, 6, 96, 77, {}), (300, 8, 2, 32, 3, {}), (260, 8, 2, 128, 300, {"scale": 1.5}), (300, 8, 2, 128, 0, {"scale": 6.0}),
    (300, 12, 4, 64, 150, {"scale": -9.0, "sinks": True}), (400, 6, 2, 96, 0, {"scale": 3.0}), (300, 8, 1, 128, 300, {"window": 99, "scale": 0.7})])
def test_prompts_within_the_roundings_that_are_stated(torch, seq, heads, kv, dim, past, kw, dtype):
    """... and a bound that says something: outputs of zeros, of the next query row, of the next head and without a row's last position
    are outside of it."""
    batch = 8
    got, want, bound, (q, kd, vd, args) = prompt(torch, seq + heads + dim, dtype, batch, seq, heads, kv, dim, [past] * batch, **kw)
    err = np.abs(host(got) - want)
    assert np.all(err <= bound), float((err / bound).max())
    outside = lambda other: (np.abs(other - want) > bound).mean()
    assert outside(np.zeros_like(want)) > 0.9 and outside(-want) > 0.9
    assert outside(np.roll(want, 1, 1)) > 0.5 and outside(np.roll(want, 1, 2)) > 0.5
    if past:      # every row sees a position less: with sharp scores that is the one that counts in one row of so many
        short = O.attend(q[:1], kd[:1], vd[:1], [past - 1], *args[1:])[0]
        assert (np.abs(short - want[:1]) > bound[:1]).mean() > 0.5 / (past + seq)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("seq,heads,kv,dim,past,kw", [
    (24, 8, 8, 128, 333, {}), (9, 16, 4, 64, 100, {"scale": 1.0}), (40, 4, 2, 128, 50, {"scale": 3.0}), (20, 12, 3, 96, 80, {"sinks": True, "window": 31}),
    (30, 4, 2, 256, 60, {"scale": 1.0})])
def test_portions_over_the_codes(torch, seq, heads, kv, dim, past, kw, dtype):
    """More than sixteen query rows a KV head, on the kernel that rounds no keys."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(seq + dim)
    batch, total, kw = 1, past + seq, dict(kw)
    cache = Cache4(batch, kv, total, dim)
    assert needs(torch, cache, dtype, heads, seq, past, kw.get("window", 0)) < 4 * batch * kv * total * dim
    k, v = rows(torch, rng, (batch, total, kv, dim), "float32"), rows(torch, rng, (batch, total, kv, dim), "float32")
    cache.append(k, v, 0)
    q = torch.from_numpy(rng.standard_normal((batch, seq, heads, dim)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    s = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if kw.pop("sinks", False) else None
    got = cache.attend(q, past, sinks=s, **kw)
    want, size, reach = O.attend(host(q), held(k), held(v), [past], kw.get("scale", dim ** -0.5), kw.get("window", 0), None if s is None else host(s),
                                 O.coded(host(v)).transpose(0, 2, 1, 3))
    bound = bound_of(torch, dtype, want, size, reach, 2.0 ** -11, total, 0.0, 0.0)
    err = np.abs(host(got) - want)
    assert np.all(err <= bound), float((err / bound).max())
    assert (np.abs(want) > bound).mean() > 0.9


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("seq,batch", [(1, 1), (256, 8)])
def test_one_position_outweighs_thousands(torch, seq, batch, dtype):
    """One key is 2^25.5 times the others' weight and has values of zero: the outputs are what all the others give together.

    Weights are off by 2^-32 of the largest (float16: half of 2^-24, the largest being 2^7 or more) or in float32 calls 2^-35 (half of 2^-24 in a
    term held 2^10 times as large, the largest being 1 or more): times the sum of |v|, which is the others' number at most."""
    from rotor_b200.cache4 import Cache4
    past, kv, heads, dim = 6000, 1, 8, 64
    total = past + seq
    cache = Cache4(batch, kv, total, dim)
    if seq > 1 and dtype != "float32":
        assert needs(torch, cache, dtype, heads, seq, past) >= 4 * batch * kv * total * dim
    k, v = torch.zeros((1, total, 1, dim), device="cuda"), torch.ones((1, total, 1, dim), device="cuda")
    v[..., 1::2] = -0.5
    k[0, 3, 0, 0], v[0, 3] = 15.0, 0.0
    cache.append(k.expand(batch, -1, -1, -1), v.expand(batch, -1, -1, -1), 0)
    q = torch.zeros((1, seq, heads, dim), device="cuda", dtype=getattr(torch, dtype))
    q[..., 0] = 25.5 * np.log(2) / 15
    got = host(cache.attend(q.repeat(batch, 1, 1, 1), past, scale=1.0))      # (rows that lie apart, as the prompt kernel asks)
    x = float(host(q[0, 0, 0, 0])) * 15
    n = past + np.arange(seq)[:, None, None]                  # others that a row sees
    share = n * np.exp(-x) / (1 + n * np.exp(-x))
    want = share * O.held(host(v[0, 0, 0]))
    half = torch.finfo(getattr(torch, dtype)).eps / 2
    bound = np.abs(want) * (half + max(half, 2.0 ** -11) + np.expm1(2.0 ** -16 * (x + 1)) + total / 16 * 2.0 ** -22) + 2.0 ** -32 * n + half * 2.0 ** -14
    if dtype == "float32":
        bound = np.abs(want) * (half + 2.0 ** -21 + np.expm1(2.0 ** -16 * (x + 1)) + total / 16 * 2.0 ** -22) + 2.0 ** -35 * n
    err = np.abs(got - want)
    assert np.all(err <= bound), float((err / bound).max())


@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("seq", [1, 20])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e-5, "mixed", "mixed rows", 3000.0])
def test_float32_weights_at_values_of_any_size(torch, size, seq, dim):
    """The queries are short, so that what the scores' sums leave does not hide what the weights' two terms leave: a score is off by
    2^-19 of the sum of |q| |k| (four additions of a group, its scaling, up to six groups, 2^-23 each; queries as two terms, 2^-22) and by the
    exponential (its argument, up to 16, 2^-21; its result, 2^-22): 2^-20, twice with the ratio to the sum.  Weights as two terms, alone and times s,
    are off by 2^-22 each, 2^-20 with the ratio; sums over the positions add 2^-23 a tile.  2^-17 of the weighted sums of |v| and of s code
    holds all of them.  ("mixed": groups of 1, 1e-2, 1e-4 and 1 in turn, "mixed rows": the positions.)"""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(21)
    batch, heads, kv, past = 2, 8, 2, 150
    total = past + seq
    cache = Cache4(batch, kv, total, dim)
    sizes = np.array([1.0, 1e-2, 1e-4, 1.0])
    factor = np.repeat(sizes[np.arange(dim // 32) % 4], 32) if size == "mixed" else sizes[np.arange(total) % 4][:, None, None] if size == "mixed rows" else size
    k = rows(torch, rng, (batch, total, kv, dim), "float32")
    v = torch.from_numpy((rng.standard_normal((batch, total, kv, dim)) * factor).astype(np.float32)).cuda()
    cache.append(k, v, 0)
    q = torch.from_numpy((rng.standard_normal((batch, seq, heads, dim)) * 0.02).astype(np.float32)).cuda()
    got = host(cache.attend(q, past, scale=dim ** -0.5))
    want, weighted, reach = O.attend(host(q), held(k), held(v), [past] * batch, dim ** -0.5, 0, None, O.coded(host(v)).transpose(0, 2, 1, 3))
    assert reach.max() < 1.0
    err, bound = np.abs(got - want), 2.0 ** -17 * weighted + 2.0 ** -24 * np.abs(want)
    assert np.all(err <= bound), float((err / bound).max())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-6, "mixed", "growing", 3000.0])
def test_16_bit_calls_at_values_of_any_size(torch, size, dtype):
    """Groups of one size, groups of several, and positions whose values grow by a power of two every few rows: 2^-11 of the weighted sums
    as everywhere, and the type's own steps."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(22)
    batch, heads, kv, past, dim = 2, 8, 2, 300, 128
    for seq in (1, 4):
        total = past + seq
        cache = Cache4(batch, kv, total, dim)
        factor = (np.repeat([1.0, 1e-2, 30.0, 1.0], 32) if size == "mixed" else 2.0 ** (np.arange(total) // 16 - 9.0)[:, None, None] if size == "growing"
                  else size)
        k = rows(torch, rng, (batch, total, kv, dim), "float32")
        v = torch.from_numpy((rng.standard_normal((batch, total, kv, dim)) * factor).astype(np.float32)).cuda()
        cache.append(k, v, 0)
        q = torch.from_numpy(rng.standard_normal((batch, seq, heads, dim)).astype(np.float32)).cuda().to(getattr(torch, dtype))
        got = cache.attend(q, past)
        want, weighted, reach = O.attend(host(q), held(k), held(v), [past] * batch, dim ** -0.5, 0, None, O.coded(host(v)).transpose(0, 2, 1, 3))
        bound = bound_of(torch, dtype, want, weighted, reach, 2.0 ** -11, total, 0.0, 0.0)
        err = np.abs(host(got) - want)
        assert np.all(err <= bound), (seq, float((err / bound).max()))


def test_magnitudes_above_the_largest_float16(torch):
    """They are stored as 65504 is: where a group's smallest value rounds up, that is not the highest code."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(23)
    x = np.empty((16, 64), np.float32)
    x[:8] = 65490.0
    x[8:] = rng.uniform(60000, 65504, (8, 64))
    x[8:12, :32] = rng.uniform(65400, 65504, (4, 32))
    big = [70000.0, np.inf, 1e30, 65505.0]
    for r in range(16):
        x[r, 5 + r], x[r, 40] = big[r % 4], big[(r + 1) % 4]
    x[3, 9], x[5, 41] = np.nan, -np.inf
    for sign in (1, -1):
        for dtype in ("float32", "bfloat16", "float16"):
            t = torch.from_numpy((sign * x).reshape(1, 16, 1, 64)).cuda().to(getattr(torch, dtype))
            cache = Cache4(1, 1, 16, 64)
            cache.append(t, t.flip(1), 0)
            k, v = cache.read(0, 16)
            want = held(t).astype(np.float32).astype(np.float64)
            assert np.array_equal(host(k), want) and np.array_equal(host(v), want[:, :, ::-1])


@pytest.mark.parametrize("seq", [1, 300])
def test_finite_float16_rows_stay_finite(torch, seq):
    """From a step of 4096 on m + 15 s can lie above the largest float16: it is read as that, and weighted sums end there too."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(24)
    batch, kv, dim, total = 8, 2, 64, 400
    x = rng.uniform(-65504, 65504, (batch, total, kv, dim))
    x[..., 0] = x[..., 32] = 65504
    x[..., 1], x[..., 33] = rng.uniform(-65504, -1000, (2, batch, total, kv))
    t = torch.from_numpy(x).cuda().half()
    assert t.isfinite().all()
    cache = Cache4(batch, kv, total, dim)
    cache.append(t, t, 0)
    want = held(t)
    assert want.max() > 65520
    k, v = cache.read(0, total, torch.float16)
    assert np.array_equal(host(k), dense(torch, want, "float16")) and torch.equal(k, v)
    assert host(cache.read(0, total)[0]).max() > 65520      # (float32 holds what the codes stand for)
    q = torch.zeros((batch, seq, 4, dim), device="cuda", dtype=torch.float16)
    out = cache.attend(q, total - seq, window=1)            # every row's own position
    assert out.isfinite().all()
    own = np.repeat(want[:, :, total - seq:].transpose(0, 2, 1, 3), 2, 2)
    # 2^-11 for the weight, of |v| and of s code, and the output's half step
    assert np.all(np.abs(host(out) - np.clip(own, -65504, 65504)) <= 2.0 ** -11 * (np.abs(own) + 2 * 65504 + 32) + 2.0 ** -11 * np.abs(own))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("seq", [1, 7, 300])
def test_scores_of_any_size(torch, seq, dtype):
    """Scores of 1e31 to 1e34, all below zero: the largest takes everything, as among small ones."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(25)
    batch, kv, dim, total = 4, 2, 64, 350
    k = torch.full((batch, total, kv, dim), 2.0, device="cuda")
    best = torch.from_numpy(rng.integers(0, total - seq + 1, (batch, kv))).cuda()
    for b in range(batch):
        for h in range(kv):
            k[b, best[b, h], h] = 1.0
    v = rows(torch, rng, (batch, total, kv, dim), "float32")
    cache = Cache4(batch, kv, total, dim)
    cache.append(k, v, 0)
    want = torch.stack([torch.stack([cache.read(0, total)[1][b, h, best[b, h]] for h in range(kv)]) for b in range(batch)])
    for size in (1.0, 1e29, 1e31, 1e33):
        got = cache.attend(torch.full((batch, seq, kv, dim), -size, device="cuda", dtype=getattr(torch, dtype)), total - seq, scale=10.0)
        # one weight: 2^-11 with s, the value's and the output's rounding
        bound = want.abs().double() * 2.0 ** -7 + (2.0 ** -10 if dtype != "float32" else 2.0 ** -20) * 8
        assert ((got.double() - want[:, None].double()).abs() <= bound[:, None]).all(), size
