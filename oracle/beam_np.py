"""Plain statement of beam search's selection and of the reordering of states (NumPy, float64)."""
import numpy as np


def select(logits, scores, count, ended=None, pad=0):
    """(scores, beams, tokens), each [groups, count]: the best candidates of [groups, width, vocab], the lowest place first among equals."""
    logits, scores = np.asarray(logits, dtype=np.float64), np.asarray(scores, dtype=np.float64)
    groups, width, vocab = logits.shape
    out = np.empty((groups, count)), np.empty((groups, count), np.int64), np.empty((groups, count), np.int64)
    for g in range(groups):
        value = np.full((width, vocab), -np.inf)
        for w in range(width):
            x = np.where(np.isnan(logits[g, w]), -np.inf, logits[g, w])
            if not np.isfinite(scores[g, w]):
                continue
            if ended is not None and ended[g, w]:
                value[w, pad] = scores[g, w]
            elif np.isfinite(x.max()):
                value[w] = scores[g, w] + (x - (x.max() + np.log(np.exp(x - x.max()).sum())))
        order = np.argsort(-value.reshape(-1), kind="stable")[:count]
        out[0][g], out[1][g], out[2][g] = value.reshape(-1)[order], order // vocab, order % vocab
    return out


def reorder(state, beams):
    """Row b * width + w of the result is row b * width + beams[b, w]; a beam that is none of the group leaves its row."""
    state, (groups, width) = np.asarray(state), beams.shape
    source = np.where((beams >= 0) & (beams < width), beams, np.arange(width))
    return state[(source + width * np.arange(groups)[:, None]).reshape(-1)]
