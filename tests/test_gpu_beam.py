"""GPU: beam search's selection and the reordering of states against oracle/beam_np.py.

Beams and tokens are compared exactly: the inputs keep candidates that are not equal further apart than the selection's error (float32
exponentials and sums of a row: 2^-20 of the sum at most, so 1e-6 of a score).  Scores are off by that and by their rounding to float32."""
import numpy as np
import pytest

from oracle import beam_np as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def check(torch, logits, scores, count, ended=None, pad=0):
    from rotor_b200 import ops
    e = None if ended is None else torch.from_numpy(ended).cuda()
    got = ops.beam_select(logits, torch.from_numpy(scores.astype(np.float32)).cuda(), count, ended=e, pad=pad)
    want = O.select(logits.float().cpu().numpy(), scores.astype(np.float32), count, ended, pad)
    assert [g.dtype for g in got] == [torch.float32, torch.int64, torch.int64]
    s, b, t = (g.cpu().numpy() for g in got)
    # the inputs are what they should be: neighbours of the chosen are equal or further apart than the error
    v = O.select(logits.float().cpu().numpy(), scores.astype(np.float32), min(count + 1, logits.shape[1] * logits.shape[2]), ended, pad)[0]
    with np.errstate(invalid="ignore"):
        gaps = -np.diff(v, axis=1)
    assert not np.any((gaps > 1e-12) & (gaps < 2e-6)), "choose another seed"
    assert np.array_equal(b, want[1]) and np.array_equal(t, want[2])
    fine = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(s), fine)
    assert np.all(np.abs(s[fine] - want[0][fine]) <= 1e-6 + np.abs(want[0][fine]) * 2.0 ** -24)


def inputs(torch, seed, groups, width, vocab, dtype="float32", size=3.0):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((rng.standard_normal((groups, width, vocab)) * size).astype(np.float32)).cuda().to(getattr(torch, dtype))
    return x, -10 - 4 * rng.random((groups, width))


@pytest.mark.parametrize("groups,width,vocab,count", [(1, 1, 1, 1), (1, 4, 10, 8), (2, 3, 257, 6), (1, 4, 8192, 8), (1, 4, 8193, 8),
                                                      (3, 8, 30001, 16), (2, 32, 1000, 64), (1, 1, 128256, 64), (5, 2, 50000, 1)])
def test_selection(torch, groups, width, vocab, count):
    x, s = inputs(torch, vocab + count, groups, width, vocab)
    check(torch, x, s, count)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_types_with_many_equal_logits(torch, dtype):
    """Sixteen bits: equal logits within a row, the lower token first."""
    x, s = inputs(torch, 5, 2, 4, 20000, dtype, 1.0)
    check(torch, x, s, 16)


def test_all_equal(torch):
    """Every candidate of a beam is worth the same, in one slice and over several."""
    for vocab in (40, 1500, 8000, 20000):
        x = torch.zeros((2, 3, vocab), device="cuda")
        check(torch, x, np.array([[-3.0, -2.0, -2.0], [-1.0, -1.0, -1.0]]), 40)


def test_two_values(torch):
    """Thousands at the top value, spread over the row."""
    rng = np.random.default_rng(6)
    x = torch.from_numpy((rng.random((1, 2, 30000)) < 0.3).astype(np.float32)).cuda()
    check(torch, x, np.array([[-1.0, -1.5]]), 64)


def test_nothing_but_one_beam_at_the_start(torch):
    """The first step of a search: the other beams have no score yet."""
    x, _ = inputs(torch, 7, 2, 4, 999)
    check(torch, x, np.array([[0, -np.inf, -np.inf, -np.inf]] * 2), 8)


def test_ended_beams(torch):
    x, s = inputs(torch, 8, 3, 4, 5000)
    ended = np.array([[False] * 4, [True, False, True, False], [True] * 4])
    s[1, 0], s[2] = -0.5, [-4, -2, -3, -2]
    check(torch, x, s, 8, ended, pad=17)


@pytest.mark.parametrize("kept", [0, 1, 5, 7])
def test_masked_vocabulary(torch, kept):
    """-inf, the lowest float and NaN in masked places; too few candidates for the places."""
    x, s = inputs(torch, 9, 2, 2, 3000)
    for fill in (float("-inf"), float("nan")):
        y = x.clone()
        y[:, :, kept:] = fill
        check(torch, y, s, 16)
    y = x.clone()
    y[:, :, kept:] = torch.finfo(torch.float32).min
    check(torch, y, s, 4)


def test_rows_and_beams_that_offer_nothing(torch):
    x, s = inputs(torch, 10, 1, 6, 2000)
    x[0, 1, 7] = float("inf")
    x[0, 2] = float("-inf")
    s[0, 3], s[0, 4] = np.nan, np.inf
    check(torch, x, s, 12)
    check(torch, x[:, 1:5], s[:, 1:5], 5)
    check(torch, x, s, 9, np.array([[False, False, False, True, True, True]]), pad=3)


def test_signed_zeros_and_large_offsets(torch):
    x, s = inputs(torch, 11, 1, 2, 100)
    x[0, 0, ::2], x[0, 0, 1::2] = 0.0, -0.0
    check(torch, x, s, 30)
    y, s = inputs(torch, 12, 1, 2, 100, size=1.0)
    check(torch, y * 1e4, s * 1e3, 5)


def test_strided_logits(torch):
    """Rows cut out of wider ones, on and off 16-byte boundaries, and groups that share rows."""
    rng = np.random.default_rng(13)
    wide = torch.from_numpy((rng.standard_normal((2, 5, 1003)) * 3).astype(np.float32)).cuda()
    s = -10 - 4 * rng.random((2, 3))
    for x in (wide[:, 1:4, :1000], wide[:, ::2, 3:], wide[:1, :3].expand(2, 3, 1003), wide[:, :3, 4:]):
        check(torch, x, s, 6)


def test_selection_repeats_its_bits_and_replays(torch):
    from rotor_b200 import ops
    x, s = inputs(torch, 14, 4, 4, 30000, "bfloat16", 0.5)
    s = torch.from_numpy(s.astype(np.float32)).cuda()
    first = [t.clone() for t in ops.beam_select(x, s, 8)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.beam_select(x, s, 8)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = ops.beam_select(x, s, 8)
    torch.cuda.current_stream().wait_stream(stream)
    y = x.flip(0).clone()
    x.copy_(y)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, ops.beam_select(y, s, 8)))


@pytest.mark.parametrize("width", [1, 2, 4, 5, 8, 9, 16, 17, 32])
def test_states_follow_their_beams(torch, width):
    from rotor_b200 import ops
    rng = np.random.default_rng(width)
    groups = 3
    beams = rng.integers(0, width, (groups, width))
    beams[1] = np.roll(np.arange(width), 1)               # a cycle through all rows
    states = [torch.from_numpy(rng.integers(0, 256, (groups * width, *shape)).astype(np.uint8)).cuda()
              for shape in ((3, 40, 16), (7,), (1,), (2, 9, 6), (4, 12))]
    states.append(torch.from_numpy(rng.standard_normal((groups * width, 2, 50, 8))).cuda())
    states.append(torch.zeros((groups * width, 0), device="cuda"))
    want = [O.reorder(t.cpu().numpy(), beams) for t in states]
    ops.reorder_states(states, torch.from_numpy(beams).cuda())
    for t, w in zip(states, want):
        assert np.array_equal(t.cpu().numpy(), w)


@pytest.mark.parametrize("length", [0, 1, 17, 40])
def test_only_the_filled_positions_move(torch, length):
    from rotor_b200 import ops
    rng = np.random.default_rng(length)
    beams = rng.integers(0, 4, (2, 4))
    for shape, axis in (((8, 3, 40, 16), 2), ((8, 40, 5), 1), ((8, 2, 3, 40), 3)):
        for dtype in (torch.float32, torch.uint8, torch.bfloat16):
            t = torch.from_numpy(rng.integers(0, 200, shape).astype(np.float32)).cuda().to(dtype)
            whole = torch.from_numpy(rng.standard_normal((8, 3))).cuda()
            before, other = t.float().cpu().numpy(), O.reorder(whole.cpu().numpy(), beams)
            at = (slice(None),) * axis + (slice(0, length),)
            want = before.copy()
            want[at] = O.reorder(before, beams)[at]
            ops.reorder_states([(t, axis), whole], torch.from_numpy(beams).cuda(), length=length)
            assert np.array_equal(t.float().cpu().numpy(), want)
            assert np.array_equal(whole.cpu().numpy(), other)


def test_beams_that_are_none_leave_their_rows(torch):
    from rotor_b200 import ops
    beams = torch.tensor([[1, -1, 7, 2 ** 40]], device="cuda")
    t = torch.arange(4, device="cuda")[:, None].repeat(1, 33)
    ops.reorder_states([t], beams)
    assert t[:, 0].tolist() == [1, 1, 2, 3] and t[:, 32].tolist() == [1, 1, 2, 3]


def test_many_states_and_rows_apart(torch):
    """More states than one launch describes, rows of a wider buffer."""
    from rotor_b200 import ops
    rng = np.random.default_rng(20)
    beams = rng.integers(0, 3, (2, 3))
    buffer = torch.from_numpy(rng.standard_normal((6, 150, 11)).astype(np.float32)).cuda()
    before = buffer.cpu().numpy()
    ops.reorder_states([buffer[:, i] for i in range(0, 150, 2)], torch.from_numpy(beams).cuda())
    want = before.copy()
    want[:, ::2] = O.reorder(before, beams)[:, ::2]
    assert np.array_equal(buffer.cpu().numpy(), want)


def test_refusals(torch):
    from rotor_b200 import ops
    x, s = torch.zeros((2, 3, 10), device="cuda"), torch.zeros((2, 3), device="cuda")
    e = torch.zeros((2, 3), dtype=torch.bool, device="cuda")
    b, t = torch.zeros((2, 3), dtype=torch.int64, device="cuda"), torch.zeros((6, 4, 5), device="cuda")
    for bad in (lambda: ops.beam_select(x, s, 0), lambda: ops.beam_select(x, s, 31), lambda: ops.beam_select(x[0], s, 1),
                lambda: ops.beam_select(x, s[:1], 1), lambda: ops.beam_select(x, s.double(), 1), lambda: ops.beam_select(x.double(), s, 1),
                lambda: ops.beam_select(x.cpu(), s, 1), lambda: ops.beam_select(x, s, 1, ended=e, pad=10),
                lambda: ops.beam_select(x, s, 1, ended=e.int()), lambda: ops.beam_select(x.transpose(1, 2).contiguous().transpose(1, 2), s, 1),
                lambda: ops.beam_select(torch.zeros((1, 33, 4), device="cuda"), torch.zeros((1, 33), device="cuda"), 1),
                lambda: ops.beam_select(torch.zeros((1, 2, 100), device="cuda"), torch.zeros((1, 2), device="cuda"), 65),
                lambda: ops.reorder_states([t[:5]], b), lambda: ops.reorder_states([t], b.int()), lambda: ops.reorder_states([t], b.cpu()),
                lambda: ops.reorder_states([t.transpose(1, 2)], b), lambda: ops.reorder_states([t[:1].expand(6, 4, 5)], b),
                lambda: ops.reorder_states([(t, 1)], b, length=5), lambda: ops.reorder_states([(t, 3)], b, length=1),
                lambda: ops.reorder_states([(t, 0)], b, length=1), lambda: ops.reorder_states([t, t], b), lambda: ops.reorder_states([t.cpu()], b)):
        with pytest.raises(ValueError):
            bad()
    assert all(o.shape == (0, 4) for o in ops.beam_select(x[:0], s[:0], 4))
    ops.reorder_states([], b)
    ops.reorder_states([t[:0]], b[:0])
