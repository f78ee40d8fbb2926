"""GPU: the 4-bit cache and the attention over it against oracle/cache4_np.py.

What is read back is compared bit by bit: the definition decides every code, and a value is one rounding of m + s code to float32
and one more to the type asked for.  Attention is off by
 * the rounding of its outputs, half a step of the type: finfo(type).eps / 2 of the value, and of smallest_normal below that (float16: 2^-25;
   a row that a sink outweighs by e^28 has outputs of 4e-13, which are zeros in float16);
 * the rounding of the weights: float16 (2^-11 at most, with the ratio to the sum of weights that are not rounded) of the weighted sums
   of |v| and of s code for 16-bit types, two terms (2^-21) for float32.  (s code, because a value is m + s code and the rounded weight
   p s multiplies the code alone: where m and s code cancel, p s code (1 + e) + p m = p v + e p s code.);
 * 16-bit calls of more than 16 query rows a KV head: keys, values and weights may be rounded to the type, h = finfo(type).eps / 2 each, which
   is h of the weighted sum of |v| for the weights and for the values, and h of |q| |k| for a score, twice with the ratio to the sum;
 * scores: products accumulated in float32 over at most 256 columns and 8 groups, each addition off by 2^-23 of the sum of |q| |k|:
   fewer than 64 of them, so 2^-17 of it, which is the relative error of a weight, twice with the ratio to the sum.
Scores that are off by d each change a weight's ratio to the sum by factors between e^(-2 d) and e^(2 d), so by at most e^(2 d) - 1 of it:
2 d where that is small, but not for scores of hundreds in 16-bit types (2 d = 2^-10 of 750 is 0.73, and e^0.73 - 1 = 1.08)."""
import numpy as np
import pytest

from oracle import cache4_np as O

pytestmark = pytest.mark.gpu
TYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def make(torch, rng, shape, dtype, size=1.0, offset=1.0):
    x = rng.standard_normal(shape) * size + offset * rng.standard_normal(shape[-2:])
    return torch.from_numpy(x.astype(np.float32)).cuda().to(getattr(torch, dtype))


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def rounded(torch, x, dtype):
    """Exact values through float32 to the type, as the cache gives them."""
    return torch.from_numpy(x.astype(np.float32)).to(getattr(torch, dtype)).float().numpy().astype(np.float64)


def held(x):
    """Rows [batch, seq, heads, dim] as the cache holds them: [batch, heads, seq, dim]."""
    return O.held(host(x)).transpose(0, 2, 1, 3)


def check_attention(torch, got, want, size, reach, dtype, kv):
    half = torch.finfo(getattr(torch, dtype)).eps / 2
    weight = 2.0 ** -21 if dtype == "float32" else 2.0 ** -11
    score = 2.0 ** -16
    if dtype != "float32" and want.shape[1] * want.shape[2] // kv > 16 and want.shape[3] <= 128:
        weight, score = 2 * half, 2 * half + score
    bound = half * np.abs(want) + size * (weight + np.expm1(score * (reach[..., None] + 1))) + half * torch.finfo(getattr(torch, dtype)).smallest_normal + 1e-30
    err = np.abs(host(got) - want)
    assert np.all(err <= bound), float((err / bound).max())


def attend_case(torch, seed, batch, seq, heads, kv, dim, past, window=0, sinks=False, dtype="float32", room=None, scale=None, size=1.0,
                q_size=1.0, lengths=None):
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(seed)
    past = [past] * batch if isinstance(past, int) else past
    total = max(past) + seq
    cache = Cache4(batch, kv, room or total, dim)
    k, v = make(torch, rng, (batch, total, kv, dim), "bfloat16", size, size), make(torch, rng, (batch, total, kv, dim), "bfloat16", size, size)
    cache.append(k, v, 0)
    q = make(torch, rng, (batch, seq, heads, dim), dtype, q_size, 0.0)
    s = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if sinks else None
    if len(set(past)) > 1 or lengths:
        got = cache.attend(q, torch.tensor(past, dtype=torch.int32, device="cuda"), scale=scale, window=window, sinks=s, longest=lengths)
    else:
        got = cache.attend(q, past[0], scale=scale, window=window, sinks=s)
    assert got.shape == q.shape and got.dtype == q.dtype
    want = O.attend(host(q), held(k), held(v), past, dim ** -0.5 if scale is None else scale, window, None if s is None else host(s),
                    O.coded(host(v)).transpose(0, 2, 1, 3))
    check_attention(torch, got, *want, dtype, kv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_what_is_written_is_read(torch, dim, dtype):
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(dim)
    batch, kv, seq, past = 2, 3, 37, 5
    cache = Cache4(batch, kv, 50, dim)
    assert cache.max_seq == 64
    k, v = make(torch, rng, (batch, seq, kv, dim), dtype), make(torch, rng, (batch, seq, kv, dim), dtype)
    cache.append(k, v, past)
    for out in TYPES:
        for x, y in zip((k, v), cache.read(past, past + seq, getattr(torch, out))):
            assert y.dtype is getattr(torch, out)
            assert np.array_equal(host(y), rounded(torch, held(x), out))
    a, b = cache.read(0, cache.max_seq)
    for y in (a, b):      # nothing else was touched
        assert not y[:, :, :past].any() and not y[:, :, past + seq:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_strides(torch, dtype):
    """Columns of stacked rows, transposed heads, a broadcast sequence, rows that begin off a 16-byte boundary."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(1)
    stacked = make(torch, rng, (2, 9, 7, 64), dtype)
    heads_first = make(torch, rng, (2, 3, 9, 64), dtype).transpose(1, 2)
    one = make(torch, rng, (1, 9, 3, 64), dtype).expand(2, 9, 3, 64)
    wide = make(torch, rng, (2, 9, 3, 67), dtype)[..., 1:65]
    for k, v in ((stacked[:, :, 1:4], stacked[:, :, 4:]), (heads_first, one), (wide, heads_first)):
        cache = Cache4(2, 3, 16, 64)
        cache.append(k, v, 2)
        for x, y in zip((k, v), cache.read(2, 11)):
            assert np.array_equal(host(y), rounded(torch, held(x), "float32"))


def test_values_at_the_edges(torch):
    """Constant, zero, tiny and huge groups, infinities, NaN, groups of nothing but NaN, quotients on a border between two codes."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(2)
    x = rng.standard_normal((16, 128)).astype(np.float32)
    x[0] = 0.0
    x[1] = 0.1
    x[2] *= 1e-6
    x[3] *= 1e-9
    x[4] *= 1e30
    x[5, 3], x[5, 40] = np.inf, -np.inf
    x[6, 5], x[6, 70:100] = np.nan, np.nan
    x[7] = np.nan
    x[8] = np.tile(np.arange(32) / 2.0, 4) % 15.5          # halves: m 0, s 1
    x[9] = np.tile(np.arange(32) * 15 / 31.0, 4)
    x[10] = 1000 + x[10] * 1e-3                            # an offset much larger than the step
    x[11] = np.tile(np.r_[np.zeros(31), 15 * 2.0 ** -10], 4)
    x[12, :32] = -0.0
    x[13] = np.float32(65504) * np.sign(x[13])
    for dtype in TYPES:
        t = torch.from_numpy(x.reshape(1, 16, 1, 128)).cuda().to(getattr(torch, dtype))
        cache = Cache4(1, 1, 16, 128)
        cache.append(t, t.flip(1), 0)
        k, v = cache.read(0, 16)
        want = held(t)
        assert np.isfinite(want).all()
        assert np.array_equal(host(k), rounded(torch, want, "float32"))
        assert np.array_equal(host(v), rounded(torch, want[:, :, ::-1], "float32"))


def test_many_random_rows_bit_by_bit(torch):
    """Three million values of a few sizes: the rare quotients that float32 arithmetic does not settle are among them."""
    from rotor_b200.cache4 import Cache4
    g = torch.Generator(device="cuda").manual_seed(3)
    for dtype, size in (("bfloat16", 1.0), ("float32", 3.7), ("float16", 0.02)):
        x = (torch.randn((1, 4096, 2, 128), generator=g, device="cuda") * size + size).to(getattr(torch, dtype))
        cache = Cache4(1, 2, 4096, 128)
        cache.append(x, x, 0)
        k, v = cache.read(0, 4096)
        assert torch.equal(k, v)
        assert np.array_equal(host(k), rounded(torch, held(x), "float32"))


def test_lengths_on_the_device(torch):
    """A start per sequence; rows past the end of the cache are left out, and a length outside the cache is taken as its nearest bound."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(4)
    cache = Cache4(5, 2, 32, 64)
    k, v = make(torch, rng, (5, 9, 2, 64), "float32"), make(torch, rng, (5, 9, 2, 64), "float32")
    past = [0, 11, 27, 40, -3]
    cache.append(k, v, torch.tensor(past, dtype=torch.int32, device="cuda"))
    for x, y in zip((k, v), cache.read(0, 32)):
        want = np.zeros((5, 2, 32, 64))
        for b, p in enumerate(past):
            p = min(max(p, 0), 32)
            n = min(9, 32 - p)
            want[b, :, p:p + n] = held(x)[b, :, :n]
        assert np.array_equal(host(y), rounded(torch, want, "float32"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (20, 5), (8, 1), (9, 1), (33, 1), (6, 6)])
def test_one_token(torch, heads, kv, dtype):
    for past in (0, 1, 15, 16, 300):
        attend_case(torch, past + heads, 2, 1, heads, kv, 128, past, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_every_head_size(torch, dim, dtype):
    attend_case(torch, dim, 2, 1, 4, 2, dim, 77, dtype=dtype)
    attend_case(torch, dim, 1, 7, 12, 2, dim, 130, dtype=dtype, sinks=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seq,heads,kv,past", [(2, 4, 1, 0), (5, 5, 5, 19), (16, 2, 1, 3), (33, 6, 2, 90), (130, 3, 1, 0), (64, 20, 5, 200)])
def test_portions_and_prompts(torch, seq, heads, kv, past, dtype):
    attend_case(torch, seq, 2, seq, heads, kv, 64, past, dtype=dtype)
    attend_case(torch, seq + 1, 1, seq, heads, kv, 128, past, dtype=dtype, window=21)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("seq,heads,kv,dim,past,kw", [
    (300, 20, 5, 128, 0, {}), (257, 12, 4, 64, 200, {}), (300, 6, 6, 96, [0, 77], {}), (300, 8, 2, 32, 3, {}), (200, 64, 8, 128, 100, {}),
    (300, 8, 1, 128, [300, 5], {"window": 99}), (290, 9, 3, 64, [400, 0], {"window": 130, "sinks": True}), (300, 8, 2, 128, 0, {"sinks": True}),
    (520, 7, 1, 128, 0, {"scale": -0.07}), (256, 16, 4, 128, 0, {"scale": 0.0}), (260, 8, 2, 128, 900, {"scale": 1.5}),
    (300, 8, 2, 128, 0, {"scale": 6.0}), (300, 12, 4, 64, 150, {"scale": -9.0, "sinks": True}), (600, 6, 2, 96, 0, {"scale": 3.0})])
def test_prompts_on_the_prompt_kernel(torch, seq, heads, kv, dim, past, kw, dtype):
    """Sizes that are worth dense rows: the workspace holds them."""
    from rotor_b200 import abi, ops
    from rotor_b200.cache4 import Cache4
    batch = 8
    past = past if isinstance(past, int) else past * 4
    high = past if isinstance(past, int) else max(past)
    need = abi.lib.rotor_b200_cache4_attend_workspace_bytes(Cache4(batch, kv, high + seq, dim)._ref, ops.type_code(getattr(torch, dtype)), heads, seq, high,
                                                            kw.get("window", 0))
    assert need >= 4 * batch * kv * (high + seq) * dim
    attend_case(torch, seq + heads, batch, seq, heads, kv, dim, past, dtype=dtype, lengths=None if isinstance(past, int) else high, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 5000])
def test_windows_and_sinks(torch, window, dtype):
    attend_case(torch, window, 2, 3, 6, 2, 64, [40, 333], window=window, sinks=True, dtype=dtype)
    attend_case(torch, window, 2, 1, 8, 2, 128, [0, 200], window=window, dtype=dtype, lengths=200)


@pytest.mark.parametrize("lengths", [None, 699, 700, 10 ** 6])
def test_unequal_lengths_and_bounds(torch, lengths):
    attend_case(torch, 7, 6, 1, 8, 2, 64, [0, 1, 63, 64, 500, 699], dtype="bfloat16", lengths=lengths)
    attend_case(torch, 8, 3, 4, 8, 2, 64, [0, 17, 612], dtype="float32", lengths=lengths)


@pytest.mark.parametrize("seq", [1, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_above_the_bound_are_taken_as_it(torch, seq, dtype):
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(18)
    cache = Cache4(2, 1, 200, 64)
    k = make(torch, rng, (2, 200, 1, 64), dtype)
    cache.append(k, k, 0)
    q = make(torch, rng, (2, seq, 2, 64), dtype)
    past = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")
    assert torch.equal(cache.attend(q, past(120, 60), longest=100), cache.attend(q, past(100, 60), longest=100))


@pytest.mark.parametrize("dtype", TYPES)
def test_long_cache(torch, dtype):
    attend_case(torch, 9, 1, 1, 8, 1, 64, 20001, dtype=dtype)
    attend_case(torch, 10, 1, 2, 2, 2, 128, 5000, dtype=dtype, room=9000)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-5, 1e-3, 300.0])
def test_values_of_any_size(torch, size, dtype):
    """Keys and values of that size; queries that bring the scores back to the usual range."""
    attend_case(torch, 11, 2, 1, 8, 2, 128, 150, size=size, q_size=1 / size, dtype=dtype if size > 1e-4 or dtype != "float16" else "float32")


def test_sharp_and_flat_scores(torch):
    for scale in (0.0, 5.0, -1.0):
        attend_case(torch, 12, 2, 3, 8, 2, 64, 100, scale=scale)


def test_queries_that_are_no_numbers_stay_among_themselves(torch):
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(13)
    for seq in (1, 40):
        cache = Cache4(1, 1, 64, 64)
        k = make(torch, rng, (1, 50, 1, 64), "float32")
        cache.append(k, k, 0)
        q = make(torch, rng, (1, seq, 8, 64), "float32")
        clean = cache.attend(q, 50 - seq)
        q[0, 0, 3, 5], q[0, 0, 4, 0], q[0, 0, 6] = float("nan"), float("inf"), 0.0
        got = cache.attend(q, 50 - seq)
        assert got[0, 0, 3].isnan().all() and got[0, 0, 4].isnan().all()
        others = [0, 1, 2, 5, 7]
        assert torch.equal(got[0, 0, others], clean[0, 0, others]) and torch.equal(got[0, 1:], clean[0, 1:])
        want = O.held(host(k))[0, :51 - seq, 0].mean(0)
        assert np.abs(host(got[0, 0, 6]) - want).max() < 1e-5 * np.abs(O.held(host(k))).max()


def test_rows_behind_a_sequence_do_not_matter(torch):
    """Rows that an earlier, longer sequence left behind the present one's end, the largest numbers among them."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(14)
    for dtype in ("float32", "bfloat16"):
        for seq in (1, 5, 64):
            a, b = Cache4(2, 2, 256, 64), Cache4(2, 2, 256, 64)
            junk = torch.full((2, 256, 2, 64), 60000.0, device="cuda")
            junk[..., ::2] = -60000.0
            b.append(junk, junk, 0)
            k, v = make(torch, rng, (2, 70 + seq, 2, 64), dtype), make(torch, rng, (2, 70 + seq, 2, 64), dtype)
            q = make(torch, rng, (2, seq, 4, 64), dtype)
            past = torch.tensor([70, 3], dtype=torch.int32, device="cuda")
            for c in (a, b):
                c.append(k, v, 0)
                c.append(k[:, :seq], v[:, :seq], past)
            assert torch.equal(a.attend(q, past), b.attend(q, past))


def test_query_rows_of_any_strides(torch):
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(15)
    for dtype in TYPES:
        for seq in (3, 40):
            cache = Cache4(2, 2, 64, 64)
            k = make(torch, rng, (2, 64, 2, 64), dtype)
            cache.append(k, k, 0)
            row = make(torch, rng, (2, seq, 9, 64), dtype)
            odd = make(torch, rng, (2, seq, 6, 65), dtype)[..., 1:]
            turned = make(torch, rng, (2, 6, seq, 64), dtype).transpose(1, 2)
            for q in (row[:, :, 3:], odd, turned, row[:1, :, :6].expand(2, seq, 6, 64)):
                want = O.attend(host(q), held(k), held(k), [5, 5], 0.125, 0, None, O.coded(host(k)).transpose(0, 2, 1, 3))
                check_attention(torch, cache.attend(q, 5), *want, dtype, 2)


def test_empty_calls(torch):
    from rotor_b200.cache4 import Cache4
    cache = Cache4(2, 2, 16, 64)
    none = torch.empty((2, 0, 2, 64), device="cuda")
    cache.append(none, none, 16)
    assert cache.attend(torch.empty((2, 0, 4, 64), device="cuda"), 3).shape == (2, 0, 4, 64)
    k, v = cache.read(4, 4)
    assert k.shape == v.shape == (2, 2, 0, 64)


def test_a_query_beyond_the_cache_with_a_window_gives_zeros(torch):
    """A length at the cache's end: the query's own row was not stored, and its window holds no other."""
    from rotor_b200.cache4 import Cache4
    cache = Cache4(1, 1, 16, 64)
    ones = torch.ones((1, 16, 1, 64), device="cuda")
    cache.append(ones, ones, 0)
    past = torch.tensor([16], dtype=torch.int32, device="cuda")
    assert not cache.attend(torch.ones((1, 1, 2, 64), device="cuda"), past, window=1).any()
    assert (cache.attend(torch.ones((1, 1, 2, 64), device="cuda"), past, window=2) == 1).all()


@pytest.mark.parametrize("seq,dtype", [(1, "float32"), (1, "bfloat16"), (24, "float32"), (24, "bfloat16"), (24, "float16")])
def test_captured_steps_follow_the_lengths(torch, seq, dtype):
    """Append and attend captured once on a side stream and replayed with other inputs and lengths."""
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(16)
    batch, kv, dim = 2, 2, 64
    cache, plain = Cache4(batch, kv, 128, dim), Cache4(batch, kv, 128, dim)
    k, v, q = (torch.zeros((batch, seq, n, dim), device="cuda", dtype=getattr(torch, dtype)) for n in (kv, kv, 8))
    past = torch.zeros(batch, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.append(k, v, past)
        cache.attend(q, past)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            cache.append(k, v, past)
            out = cache.attend(q, past)
    torch.cuda.current_stream().wait_stream(stream)
    lengths = np.array([0, 40])
    for _ in range(3):
        for t in (k, v, q):
            t.copy_(make(torch, rng, tuple(t.shape), dtype))
        past.copy_(torch.from_numpy(lengths.astype(np.int32)))
        graph.replay()
        plain.append(k, v, past)
        assert torch.equal(out, plain.attend(q, past))
        lengths += seq


def test_repeated_calls_give_the_same_bits(torch):
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(17)
    cache = Cache4(3, 2, 1000, 128)
    k = make(torch, rng, (3, 1000, 2, 128), "bfloat16")
    cache.append(k, k.flip(1), 0)
    for seq in (1, 50):
        q = make(torch, rng, (3, seq, 8, 128), "bfloat16")
        first = cache.attend(q, 900)
        for _ in range(3):
            assert torch.equal(cache.attend(q, 900), first)


def test_prompts_a_few_sequences_at_a_time(torch):
    """Dense rows of more than a GiB are made for some of the sequences at a time: each gets the bits that it gets alone."""
    from rotor_b200 import abi, ops
    from rotor_b200.cache4 import Cache4
    batch, kv, room, dim, heads, seq = 5, 8, 65536 + 256, 128, 32, 256
    torch.manual_seed(5)
    cache = Cache4(batch, kv, room, dim)
    for at in range(0, room, 4096):
        k, v = (torch.randn((batch, min(4096, room - at), kv, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        cache.append(k, v, at)
    q = torch.randn((batch, seq, heads, dim), device="cuda", dtype=torch.bfloat16)
    past = torch.tensor([65536, 100, 40000, 0, 65000], dtype=torch.int32, device="cuda")
    each = 4 * kv * (65536 + seq) * dim
    bytes_of = lambda c: abi.lib.rotor_b200_cache4_attend_workspace_bytes(c._ref, ops.type_code(q.dtype), heads, seq, 65536, 0)
    assert 3 * each < bytes_of(cache) < 4 * each
    got = cache.attend(q, past, longest=65536)
    for b in range(batch):
        alone = Cache4(1, kv, room, dim)
        for mine, all_ in zip(alone._tensors(), cache._tensors()):
            mine.copy_(all_[b:b + 1])
        assert each <= bytes_of(alone) < 2 * each
        assert torch.equal(alone.attend(q[b:b + 1], past[b:b + 1], longest=65536), got[b:b + 1]), b


def test_offsets_beyond_32_bits(torch):
    """The last sequence's codes lie 5.3 GB behind the first one's, and the same rows give the same bits there."""
    from rotor_b200.cache4 import Cache4
    torch.manual_seed(6)
    batch, room = 80, 131072
    cache = Cache4(batch, 8, room, 128)
    assert (batch - 1) * cache.k_codes.stride(0) > 2 ** 32
    k, v = (torch.randn((1, 600, 8, 128), device="cuda", dtype=torch.bfloat16).expand(batch, -1, -1, -1) for _ in range(2))
    cache.append(k, v, room - 600)
    for rows, held in zip(cache.read(room - 600, room, dtype=torch.float32), (k, v)):
        assert torch.equal(rows[0], rows[-1]) and (rows[0] - held[0].transpose(0, 1)).abs().max() < 1.0
    for seq in (1, 9, 200):
        q = torch.randn((1, seq, 64, 128), device="cuda", dtype=torch.bfloat16).expand(batch, -1, -1, -1)
        for x in (q, q.contiguous()):
            out = cache.attend(x, room - seq, window=700)
            assert torch.equal(out[0], out[-1]) and out[0].abs().max() > 0
    mark = cache.v_codes[-1, :, -16:].clone()
    cache.v_codes[-8, :, -16:] = 0
    cache.reorder(torch.arange(8, device="cuda").flip(0).repeat(batch // 8, 1))
    assert torch.equal(cache.v_codes[-8, :, -16:], mark) and not cache.v_codes[-1, :, -16:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_reading_to_any_address(torch, dtype):
    """Buffers that begin at multiples of 16 bytes, and not of 32, get the same bits."""
    from rotor_b200 import abi, ops
    from rotor_b200.cache4 import Cache4
    cache = Cache4(2, 3, 50, 96)
    cache.append(*make(torch, np.random.default_rng(9), (2, 2, 40, 3, 96), dtype), 5)
    want = cache.read(3, 41, dtype=getattr(torch, dtype))
    off = 16 // want[0].element_size()
    got = [torch.full((want[0].numel() + 2 * off,), 7.0, dtype=want[0].dtype, device="cuda") for _ in range(2)]
    assert all(g.data_ptr() % 32 == 0 for g in got)
    status = abi.lib.rotor_b200_cache4_read(cache._ref, 3, 41, got[0][off:].data_ptr(), got[1].data_ptr(), ops.type_code(want[0].dtype), abi.stream())
    assert status == 0
    for g, w, at in zip(got, want, (off, 0)):
        assert torch.equal(g[at:at + w.numel()], w.reshape(-1)) and (g[:at] == 7).all() and (g[at + w.numel():] == 7).all()


def test_prompts_to_any_address(torch):
    """Outputs that begin at a multiple of 16 bytes, and not of 32, get the same bits, and nothing beside them is written."""
    import ctypes as C
    from rotor_b200 import abi, ops
    from rotor_b200.cache4 import Cache4
    torch.manual_seed(8)
    cache = Cache4(8, 2, 300, 64)
    cache.append(*torch.randn((2, 8, 300, 2, 64), device="cuda"), 0)
    q = torch.randn((8, 300, 16, 64), device="cuda", dtype=torch.bfloat16)
    want, code, n = cache.attend(q, 0), ops.type_code(q.dtype), q.numel()
    need = abi.lib.rotor_b200_cache4_attend_workspace_bytes(cache._ref, code, 16, 300, 0, 0)
    assert need >= 4 * 8 * 2 * 300 * 64
    work, out = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.full((n + 16,), 7.0, dtype=q.dtype, device="cuda")
    status = abi.lib.rotor_b200_cache4_attend(cache._ref, q.data_ptr(), code, (C.c_int64 * 3)(*q.stride()[:3]), 16, 300, 0, None, 0, 64 ** -0.5, 0,
                                              None, out[8:].data_ptr(), work.data_ptr(), need, abi.stream())
    assert status == 0 and out.data_ptr() % 32 == 0
    assert torch.equal(out[8:n + 8].view_as(want), want) and (out[:8] == 7).all() and (out[n + 8:] == 7).all()


def test_another_device_is_refused(torch):
    from rotor_b200.cache4 import Cache4
    cache = Cache4(1, 1, 16, 32)
    x = torch.zeros((1, 1, 1, 32), device="cuda")
    cache._device += 1
    for call in (lambda: cache.append(x, x, 0), lambda: cache.read(0, 1), lambda: cache.attend(x, 0)):
        with pytest.raises(ValueError, match="current CUDA device"):
            call()


FRESH = """
import torch
from rotor_b200 import ops
from rotor_b200.cache4 import Cache4
torch.manual_seed(3)
def calls():
    cache = Cache4(8, 2, 400, 128)
    k, v = (torch.randn((8, 300, 2, 128), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn((8, 300, 8, 128), device="cuda", dtype=torch.bfloat16)
    wide = torch.randn((16, 8, 40000), device="cuda")
    one = torch.randn((1, 2, 500), device="cuda")
    scores = torch.zeros((16, 8), device="cuda")
    def run():
        cache.append(k, v, 0)
        return (*cache.read(0, 300), cache.attend(q, 0), cache.attend(q[:, :1].contiguous(), 299), *ops.beam_select(wide, scores, 9),
                *ops.beam_select(one, scores[:1, :2], 3))
    return run
run = calls()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
print("same")
"""


def test_the_first_call_of_a_process_may_be_captured(torch):
    import os
    import subprocess
    import sys
    import rotor_b200
    here = os.path.dirname(os.path.dirname(rotor_b200.__file__))
    r = subprocess.run([sys.executable, "-c", FRESH], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=here + os.pathsep + os.environ.get("PYTHONPATH", "")))
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


def test_refusals(torch):
    from rotor_b200.cache4 import Cache4
    cache = Cache4(2, 2, 32, 64)
    x = torch.zeros((2, 4, 2, 64), device="cuda")
    q = torch.zeros((2, 4, 4, 64), device="cuda")
    past = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: Cache4(2, 2, 32, 80), lambda: Cache4(0, 2, 32, 64), lambda: cache.append(x, x, 29), lambda: cache.append(x, x, -1),
                lambda: cache.append(x, x.half(), 0), lambda: cache.append(x, x[:, :3], 0), lambda: cache.append(x[..., :32], x[..., :32], 0),
                lambda: cache.append(x.double(), x.double(), 0), lambda: cache.append(x.cpu(), x.cpu(), 0),
                lambda: cache.append(x.transpose(2, 3).contiguous().transpose(2, 3), x, 0), lambda: cache.append(x, x, past.long()),
                lambda: cache.append(x, x, past[:1]), lambda: cache.append(x, x, past.cpu()), lambda: cache.read(3, 2), lambda: cache.read(0, 33),
                lambda: cache.read(0, 3, torch.int8), lambda: cache.attend(q[:, :, :3], 0), lambda: cache.attend(q, 29),
                lambda: cache.attend(q, 0, window=-1), lambda: cache.attend(q, 0, sinks=torch.zeros(3, device="cuda")),
                lambda: cache.attend(q, 0, sinks=torch.zeros(4, device="cuda", dtype=torch.float64)), lambda: cache.attend(q[:1], 0),
                lambda: cache.attend(q[0], 0)):
        with pytest.raises(ValueError):
            bad()
