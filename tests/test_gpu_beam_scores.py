"""GPU: how far the scores of beam search's selection are from 64 bits.

A row's log-sum-exp is a float32 sum of exponentials.  Of a term e^-t its argument is off by t (2^-24 for the difference, 2^-24 for the product with
log2(e), 2^-26 for that constant), and t is on average no more than the logarithm of the number of logits: 12.5 of 2^18; the exponential is off by 2^-22;
a thread adds at most 64 rounds of 2^18 logits, 3 additions before each, and some 10 join the threads and the parts: 2^-24 each.  Together
less than 2^-17 (7.6e-6).  Scores that are close to what the log-sum-exp takes off bring the result near zero, where float32 shows it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("groups,width,vocab", [(1, 1, 300), (1, 4, 102400), (16, 8, 128256), (1, 1, 262144), (40, 1, 50000)])
@pytest.mark.parametrize("kind", ["normal", "flat", "peaked", "equal"])
def test_scores_against_64_bits(torch, groups, width, vocab, kind):
    from rotor_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn((groups, width, vocab), generator=g, device="cuda") * {"normal": 2.5, "flat": 0.01, "peaked": 8.0, "equal": 0.0}[kind]
    x += torch.arange(width, device="cuda")[:, None] * 37.0 - 1000.0
    lse = torch.logsumexp(x.double(), -1)
    scores = (lse - x.double().amax(-1)).float()
    got, beams, tokens = ops.beam_select(x, scores, min(width, 4))
    at = (torch.arange(groups, device="cuda")[:, None], beams, tokens)
    want = scores.double()[at[0], beams] + x.double()[at] - lse[at[0], beams]
    assert want.abs().max() < 1.0
    err = (got.double() - want).abs().max().item()
    print(kind, groups, width, vocab, "%.3g" % err)
    assert err <= 2.0 ** -17 + want.abs().max().item() * 2.0 ** -24


def test_one_beams_candidates_are_in_the_order_of_their_logits(torch):
    """... however close they are: neighbouring floats, and equal ones by their tokens."""
    from rotor_b200 import ops
    rng = np.random.default_rng(1)
    base = np.float32(9.0)                 # above all others
    x = rng.standard_normal((2, 3, 5000)).astype(np.float32)
    order = rng.permutation(5000)[:20]
    near = base
    for k, token in enumerate(order):      # pairs of equal ones, each pair one step above the next
        x[:, 1, token] = near
        if k % 2:
            near = np.nextafter(near, np.float32(0))
    scores = torch.tensor([[-50.0, -1.0, -50.0]] * 2, device="cuda")
    s, b, t = ops.beam_select(torch.from_numpy(x).cuda(), scores, 20)
    want = [int(v) for k in range(0, 20, 2) for v in sorted(order[k:k + 2])]
    assert (b == 1).all() and t[0].tolist() == want and t[1].tolist() == want
    assert (s.diff(dim=1) <= 0).all()
