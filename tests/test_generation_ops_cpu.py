"""CPU: what the 4-bit cache's and beam search's C entry points refuse before any CUDA call, and their oracles."""
import ctypes as C

import numpy as np
import pytest

from oracle import beam_np, cache4_np
from rotor_b200 import abi
from rotor_b200.abi import lib

ARG, SHAPE, WORKSPACE = 1, 3, 4
A = 1 << 20      # an address that is never read


def cache(**kw):
    c = abi.Cache4(2, 2, 32, 64, A, A, A, A, A, A)
    for k, v in kw.items():
        setattr(c, k, v)
    return C.byref(c)


def strides(*s):
    return (C.c_int64 * 3)(*(s or (256, 128, 64)))


@pytest.mark.parametrize("kw,status", [({"batch": 0}, ARG), ({"kv_heads": -1}, ARG), ({"dim": 80}, SHAPE), ({"dim": 160}, SHAPE), ({"dim": 512}, SHAPE),
                                       ({"max_seq": 0}, ARG), ({"max_seq": 40}, SHAPE), ({"max_seq": (1 << 26) + 16}, SHAPE), ({"batch": 65536}, SHAPE),
                                       ({"k_codes": None}, ARG), ({"v_step": None}, ARG), ({"k_least": A + 2}, ARG)])
def test_descriptions_of_a_cache(kw, status):
    assert lib.rotor_b200_cache4_append(cache(**kw), A, A, 0, strides(), strides(), 1, 0, None, None) == status
    assert lib.rotor_b200_cache4_read(cache(**kw), 0, 1, A, A, 0, None) == status
    assert lib.rotor_b200_cache4_attend(cache(**kw), A, 0, strides(), 4, 1, 0, None, 0, 1.0, 0, None, A, A, 1 << 30, None) == status
    assert lib.rotor_b200_cache4_attend_workspace_bytes(cache(**kw), 0, 4, 1, 0, 0) == 0


def test_calls_on_a_cache():
    c = cache()
    for args in ((None, A, 0, strides(), strides(), 1, 0), (A, None, 0, strides(), strides(), 1, 0), (A, A, 3, strides(), strides(), 1, 0),
                 (A, A, 0, None, strides(), 1, 0), (A, A, 0, strides(), strides(), 0, 0), (A, A, 0, strides(), strides(), 33, 0),
                 (A, A, 0, strides(), strides(), 2, 31), (A, A, 0, strides(), strides(), 1, -1), (A, A, 0, strides(-1, 1, 1), strides(), 1, 0),
                 (A + 2, A, 0, strides(), strides(), 1, 0), (A, A, 0, strides(), strides(), 1, 2 ** 31 - 1)):
        assert lib.rotor_b200_cache4_append(c, *args, None, None) == ARG
    for args in ((-1, 4, A, A, 0), (4, 4, A, A, 0), (0, 33, A, A, 0), (0, 4, None, A, 0), (0, 4, A + 8, A, 0), (0, 4, A, A, -1)):
        assert lib.rotor_b200_cache4_read(c, *args, None) == ARG

    def attend(q=A, dtype=0, s=strides(), heads=4, seq=1, past=0, longest=0, window=0, out=A, ws=A, size=1 << 30):
        return lib.rotor_b200_cache4_attend(c, q, dtype, s, heads, seq, past, None, longest, 1.0, window, None, out, ws, size, None)
    for kw in ({"q": None}, {"dtype": 7}, {"s": None}, {"s": strides(1, -1, 1)}, {"heads": 3}, {"heads": 0}, {"seq": 0}, {"seq": 33}, {"past": 32},
               {"past": -1}, {"longest": -1}, {"window": -1}, {"out": None}, {"out": A + 4}, {"ws": A + 8}, {"q": A + 1}):
        assert attend(**kw) == ARG, kw
    assert lib.rotor_b200_cache4_attend_workspace_bytes(c, 0, 4, 1, 5, 0) > 0
    c = cache(max_seq=8192)
    need = lib.rotor_b200_cache4_attend_workspace_bytes(c, 0, 4, 1, 8000, 0)
    assert need > 0 and attend(past=8000, size=need - 1) == WORKSPACE and attend(past=8000, ws=None, size=0) == WORKSPACE
    assert attend(heads=65536) == SHAPE and lib.rotor_b200_cache4_attend_workspace_bytes(c, 0, 65536, 1, 5, 0) == 0


def test_selections():
    def select(logits=A, dtype=0, gs=30, bs=10, scores=A, ended=None, groups=2, width=3, vocab=10, count=4, pad=0, out=A, ws=None):
        return lib.rotor_b200_beam_select(logits, dtype, gs, bs, scores, ended, groups, width, vocab, count, pad, out, A, A, ws, 0, None)
    for kw in ({"logits": None}, {"dtype": 3}, {"gs": -1}, {"scores": None}, {"out": None}, {"ws": A + 8}, {"ended": A, "pad": 10},
               {"ended": A, "pad": -1}, {"logits": A + 2}):
        assert select(**kw) == ARG, kw
    for kw in ({"groups": 0}, {"width": 33}, {"count": 0}, {"count": 65}, {"count": 31}, {"width": 3, "vocab": 2 ** 30}, {"groups": 30000}):
        assert select(**kw) == SHAPE, kw


def test_reorderings():
    def move(beams=A, groups=2, width=3, n=1, **kw):
        s = dict(data=A, row_stride=64, segment_stride=16, segment_bytes=16, segments=4)
        s.update(kw)
        return lib.rotor_b200_reorder_states((abi.State * 2)(abi.State(**s), abi.State(**s)), n, beams, groups, width, None)
    for kw in ({"beams": None}, {"groups": 0}, {"width": 0}, {"n": 0}, {"data": None}, {"segments": 0}, {"segment_stride": 8}, {"row_stride": 63}, {"n": 2}):
        assert move(**kw) == ARG, kw
    assert move(width=33) == SHAPE and move(groups=65536) == SHAPE


def test_the_oracles_levels_are_the_nearest():
    """Every value is held by the nearest of its group's sixteen levels, and a search by hand agrees with the selection."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)) * 3 + 1
    q, s, m = cache4_np.quantise(x)
    levels = m.astype(float)[..., None] + s.astype(float)[..., None] * np.arange(16)
    nearest = np.abs(x.reshape(50, 2, 32)[..., None] - levels[:, :, None]).min(-1)
    assert np.allclose(np.abs(x - cache4_np.values(q, s, m)).reshape(50, 2, 32), nearest, rtol=0, atol=1e-12)
    logits, scores = rng.standard_normal((1, 2, 5)), np.array([[-1.0, -1.2]])
    flat = [(scores[0, w] + logits[0, w, v] - np.log(np.exp(logits[0, w]).sum()), w, v) for w in range(2) for v in range(5)]
    best = sorted(flat, key=lambda c: -c[0])[:4]
    got = beam_np.select(logits, scores, 4)
    assert [(b, t) for b, t in zip(got[1][0], got[2][0])] == [(w, v) for _, w, v in best]
    assert np.allclose(got[0][0], [c[0] for c in best])
    assert np.array_equal(beam_np.reorder(np.arange(6), np.array([[2, 2, 0], [1, 5, -1]])), [2, 2, 0, 4, 4, 5])


def test_beams_are_searched_behind_one_prompt():
    from rotor_b200.__main__ import main
    for args in (["--prompt", "1", "--prompt", "2"], ["--prompt", "1", "--sampling", "top-k"]):
        with pytest.raises(SystemExit):
            main(["generate", "--model", "nowhere", "--beams", "2"] + args)
