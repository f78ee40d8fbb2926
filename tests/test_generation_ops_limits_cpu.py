"""CPU: limits of the generation operators' C entry points that are checked before anything is launched."""
import pytest

from rotor_b200 import abi
from rotor_b200.abi import lib

ARG, SHAPE = 1, 3
A = 1 << 20      # an address that is never read


LONG = [(dict(segment_bytes=2 ** 31 + 1, segments=1, row_stride=2 ** 34 + 1), [SHAPE]),
        (dict(segment_bytes=2 ** 31 - 1, segments=3, segment_stride=2 ** 31 + 1, row_stride=2 ** 34 + 1), [SHAPE]),
        # (bytes of a row that 64 bits do not hold)
        (dict(segment_bytes=2 ** 46, segments=2 ** 30, segment_stride=2 ** 46, row_stride=2 ** 63), [ARG, SHAPE])]


@pytest.mark.parametrize("at", [0, 63, 64, 72])
@pytest.mark.parametrize("long,refusals", LONG)
def test_states_with_too_many_pieces_are_refused_before_any_is_moved(at, long, refusals):
    """More than a launch's 64 states, one of them too long: the call is refused as a whole.  (Without a GPU a launch would give another
    status, and with one nothing is launched.)"""
    states = (abi.State * 73)()
    for i in range(73):
        s = dict(data=A + 4096 * i, row_stride=64, segment_stride=16, segment_bytes=16, segments=4)
        states[i] = abi.State(**{**s, **long, "data": s["data"] + 1} if i == at else s)
    assert lib.rotor_b200_reorder_states(states, 73, A, 2, 3, None) in refusals
