"""Float64 restatement of beam search's selection (include/kvhip.h).  Test infrastructure only."""
import numpy as np


def beam_select(logits, scores, count, done=None, pad_token=0):
    """logits [B,K,V], scores [B,K] or None -> (rows, tokens, scores), each [B,count]."""
    B, K, V = logits.shape
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, float(np.finfo(np.float32).max)))
    rows, tokens = np.full((B, count), -1), np.full((B, count), -1)
    best = np.full((B, count), -np.inf)
    for b in range(B):
        found = []
        for k in range(K):
            own = 0.0 if scores is None else float(scores[b, k])
            own = -np.inf if np.isnan(own) else own
            if done is not None and done[b, k]:
                found.append((own, k, 0.0, pad_token))
                continue
            top = x[b, k].max()
            log = np.log(np.exp(x[b, k] - top).sum()) if top > -np.inf else 0.0
            for t in np.lexsort((np.arange(V), -x[b, k]))[:count]:
                s = -np.inf if own == -np.inf or x[b, k, t] == -np.inf else own + ((x[b, k, t] - top) - log)
                found.append((s, k, x[b, k, t], int(t)))
        found.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
        for i, (s, k, _, t) in enumerate(found[:count]):
            rows[b, i], tokens[b, i], best[b, i] = b * K + k, t, s
    return rows, tokens, best
