"""GPU: beam search through the models and over the 4-bit cache, against searches that recompute every beam from its first token.

The searches have to agree in every token: the seeds are ones whose candidates lie further apart at each cut than the two ways' logits
differ (checked with the reference's own values)."""
import numpy as np
import pytest

import golden_inputs as G
import likerax_models as LM
import miborax_models as MM
from oracle import beam_np, cache4_np

pytestmark = pytest.mark.gpu


def plain_search(logits_of, prompts, width, steps, eos=None):
    """logits_of(token lists) -> float64 [lists, vocab].  Returns per prompt [(tokens, score)] in the order of the beams, and the smallest
    distance between a candidate that went on and the best that did not."""
    n = len(prompts)
    beams = [[list(p)] for p in prompts]
    scores, ended, gap = [[0.0] for _ in range(n)], [[False] for _ in range(n)], np.inf
    for _ in range(steps):
        for b in range(n):
            x = logits_of(beams[b])[None]
            args = np.array([scores[b]]), np.array([ended[b]]), eos or 0
            s, w, t = beam_np.select(x, args[0], width, args[1], args[2])
            more = beam_np.select(x, args[0], min(width + 1, x.shape[1] * x.shape[2]), args[1], args[2])[0]
            gap = min(gap, *[d for d in -np.diff(more[0]) if np.isfinite(d)])
            over = [ended[b][i] for i in w[0]]
            beams[b] = [beams[b][i] + [int(v)] for i, v in zip(w[0], t[0])]
            scores[b], ended[b] = list(s[0]), [o or v == eos for o, v in zip(over, t[0])]
    out = []
    for b in range(n):
        found = []
        for tokens, score in zip(beams[b], scores[b]):
            new = tokens[len(prompts[b]):]
            found.append((new[:new.index(eos)] if eos in new else new, score))
        out.append(found)
    return out, gap


def model_of(kind):
    if kind == "bitnet":
        from rotor_b200 import semantics
        from rotor_b200.synth import model_from_oracle_params
        om, prompt = G.tiny_model("hd64")
        return model_from_oracle_params(om, semantics=semantics.REFERENCE.with_(causal=True), max_seq=64), prompt
    m, M = (LM.make(LM.config([LM.layer(chunk=20), LM.layer(ff=None, chunk=33)], loop=(0, 1, 2)), seed=1), LM) if kind == "likerax" else (
        MM.make(MM.config([MM.window(20), MM.full(), MM.window(11, kv_from=0, mlp=None)]), seed=1), MM)
    return M.load(m, max_seq=64, dtype="float32"), np.random.default_rng(3).integers(0, m["cfg"]["vocab"], 7)


def logits_by_model(model):
    return lambda lists: np.stack([model.forward(np.array(x))[0][-1] for x in lists]).astype(np.float64)


@pytest.mark.parametrize("kind", ["bitnet", "likerax", "miborax"])
@pytest.mark.parametrize("width,steps", [(1, 5), (3, 7), (8, 12)])
def test_models_search(kind, width, steps):
    model, prompt = model_of(kind)
    (want,), gap = plain_search(logits_by_model(model), [prompt], width, steps)
    got = model.generate_beams(prompt, width, steps)
    assert gap > 1e-4, "choose another seed"
    assert [ids for ids, _ in got] == [ids for ids, _ in want]
    assert np.allclose([s for _, s in got], [s for _, s in want], atol=1e-4 * steps)
    if width == 1:
        assert got[0][0] == model.generate_greedy(prompt, steps)


@pytest.mark.parametrize("kind", ["bitnet", "likerax"])
def test_ended_beams_keep_their_place(kind):
    """The token most beams take second ends them; results are put in order by their score per token."""
    model, prompt = model_of(kind)
    first = model.generate_beams(prompt, 4, 6)
    eos = first[0][0][1]
    (want,), gap = plain_search(logits_by_model(model), [prompt], 4, 11, eos)
    assert gap > 1e-4, "choose another seed"
    for penalty in (0.0, 1.0):
        got = model.generate_beams(prompt, 4, 11, eos=eos, length_penalty=penalty)
        order = sorted(want, key=lambda r: -r[1] / (len(r[0]) + (len(r[0]) < 11)) ** penalty)
        assert [ids for ids, _ in got] == [ids for ids, _ in order]
        assert any(len(ids) < 11 for ids, _ in got)


def test_two_prompts_and_reuse():
    """Two prompts at once give what each gives alone, and a search leaves nothing behind."""
    model, prompt = model_of("bitnet")
    other = prompt[::-1].copy()
    both = model.generate_beams(np.stack([prompt, other]), 3, 6)
    assert [ids for ids, _ in both[0]] == [ids for ids, _ in model.generate_beams(prompt, 3, 6)]
    assert [ids for ids, _ in both[1]] == [ids for ids, _ in model.generate_beams(other, 3, 6)]
    assert model.generate_beams(prompt, 2, 0) == [([], 0.0)] * 2


def test_refusals():
    model, prompt = model_of("likerax")
    for bad in (lambda: model.generate_beams(prompt, 0, 3), lambda: model.generate_beams(prompt, 33, 3), lambda: model.generate_beams(prompt[:0], 2, 3),
                lambda: model.generate_beams(np.stack([prompt] * 9), 4, 3), lambda: model.generate_beams(prompt, 2, 3, eos=10 ** 6)):
        with pytest.raises(ValueError):
            bad()


def test_command_line(tmp_path, capsys):
    from rotor_b200.__main__ import main
    m = LM.make(LM.config([LM.layer(chunk=20)]), seed=1)
    model, folder = LM.load(m, max_seq=32), LM.write(m, tmp_path)
    assert main(["generate", "--model", folder, "--prompt", "1 2 3", "--beams", "3", "--max-new-tokens", "5"]) == 0
    lines = capsys.readouterr().out.strip().splitlines()
    want = model.generate_beams([1, 2, 3], 3, 5)
    assert [[int(t) for t in l.split()[1:]] for l in lines] == [ids for ids, _ in want]


def test_a_search_over_the_four_bit_cache():
    """A model of one attention layer whose cache is held in four bits: append, attend, select and reorder as a program calls them, against
    a search in 64 bits that quantises and attends anew for every beam."""
    import torch
    from rotor_b200 import ops
    from rotor_b200.cache4 import Cache4
    rng = np.random.default_rng(5)
    groups, width, steps, heads, kv, dim, vocab, n_prompt = 2, 4, 9, 8, 2, 64, 300, 21
    f = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()
    embed, head = f(vocab, heads * dim) * 2, f(heads * dim, vocab) / 12
    prompts = rng.integers(0, vocab, (groups, n_prompt))

    def rows(ids):                                       # queries, keys and values of tokens [..., seq]
        x = embed[ids]
        return [t.unflatten(-1, (-1, dim)) for t in (x, x[..., :kv * dim].flip(-1), x[..., -kv * dim:])]

    def logits_of(lists):
        out = []
        for ids in lists:
            q, k, v = (t[None].double().cpu().numpy() for t in rows(torch.tensor(ids, device="cuda")))
            k, v = (cache4_np.held(t).transpose(0, 2, 1, 3) for t in (k, v))
            y, _, _ = cache4_np.attend(q[:, -1:], k, v, [len(ids) - 1], dim ** -0.5)
            out.append((y.reshape(-1) + q[0, -1].reshape(-1)) @ head.double().cpu().numpy())
        return np.stack(out)

    want, gap = plain_search(logits_of, [list(p) for p in prompts], width, steps)
    assert gap > 1e-4, "choose another seed"

    cache = Cache4(groups * width, kv, n_prompt + steps, dim)
    ids = torch.from_numpy(prompts).cuda().repeat_interleave(width, 0)
    scores = torch.full((groups, width), float("-inf"), device="cuda")
    scores[:, 0] = 0.0
    history = torch.zeros((groups * width, steps), dtype=torch.int64, device="cuda")
    past = 0
    for step in range(steps):
        q, k, v = rows(ids)
        cache.append(k, v, past)
        y = cache.attend(q, past)[:, -1] + q[:, -1]
        past += ids.shape[1]
        logits = (y.reshape(groups, width, -1).double() @ head.double()).float()
        scores, beams, tokens = ops.beam_select(logits, scores, width)
        ops.reorder_states(cache.states() + [history], beams, length=(past + 15) // 16 * 16)
        history[:, step] = tokens.view(-1)
        ids = tokens.view(-1, 1)
    got = history.view(groups, width, steps).tolist()
    assert got == [[t for t, _ in g] for g in want]
    assert np.allclose(scores.cpu().numpy(), [[s for _, s in g] for g in want], atol=1e-4)
