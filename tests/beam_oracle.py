"""Beam search in plain NumPy and Python, in 64 bits: what tests/test_gpu_beam_*.py hold the library to."""
import numpy as np


def select(x, scores, n):
    """x [B * K, V] float (masked tokens -inf), scores [B, K]: lists per sequence of (score, beam, token, logit), the n best in order,
    and the log-normalisers [B, K]."""
    B, K = scores.shape
    x = np.asarray(x, np.float64).reshape(B, K, -1)
    out, norms = [], np.full((B, K), -np.inf)
    for b in range(B):
        found = []
        for k in range(K):
            c, row = float(scores[b, k]), x[b, k]
            if not np.isfinite(c):
                continue
            m = np.max(row)
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                s = np.exp(row - m).sum()
            if not (np.isfinite(s) and np.isfinite(m)):
                norms[b, k] = np.nan
                continue
            norms[b, k] = m + np.log(s)
            ids = np.flatnonzero(row > -np.inf)
            ids = ids[np.lexsort((ids, -row[ids]))][:n]
            found += [(c + ((row[v] - m) - np.log(s)), k, int(v), row[v]) for v in ids]
        found.sort(key=lambda f: (-f[0], f[1], -f[3], f[2]))
        out.append(found[:n])
    return out, norms


class Search:
    """stg_beam_start / stg_beam_advance for one sequence."""

    def __init__(self, beams, max_steps, eos=(), pad=0, norms=None, early=False):
        self.K, self.T, self.eos, self.pad, self.early = beams, max_steps, set(eos), pad, early
        self.norms = [float(t + 1) for t in range(max_steps)] if norms is None else norms
        self.beams = [(pad, k, 0.0 if k == 0 else -np.inf) for k in range(beams)]
        self.pool, self.trail, self.steps, self.done = [], [], 0, False

    def _offer(self, score, step, parent, token):
        with np.errstate(over="ignore"):
            q = np.float32(np.float64(score) / self.norms[step])
        if q > -np.inf:
            self.pool.append((q, step, parent, token))
            self.pool.sort(key=lambda e: -e[0])  # stable: an equal one stands behind the older
            del self.pool[self.K:]

    def dead(self):
        self.beams = [(self.pad, k, -np.inf) for k in range(self.K)]

    def advance(self, candidates, finish=False):
        """candidates: (token, parent, float32 score), best first."""
        if self.done or self.steps >= self.T:
            self.dead()
            return
        t, live = self.steps, []
        for i, (tok, par, sc) in enumerate(candidates):
            if not (tok >= 0 and 0 <= par < self.K and sc > -np.inf):
                continue
            if tok in self.eos:
                if i < self.K:
                    self._offer(sc, t, par, tok)
            elif len(live) < self.K:
                live.append((tok, par, sc))
        self.beams = live + [(self.pad, k, -np.inf) for k in range(len(live), self.K)]
        self.trail.append([(tok, par) for tok, par, _ in self.beams])
        self.steps += 1
        last = finish or self.steps == self.T
        if last:
            for tok, par, sc in live:
                self._offer(sc, t, par, tok)
        full = len(self.pool) == self.K
        if last or not live or (full and (self.early or self.pool[-1][0] >= np.float32(np.float64(live[0][2]) / self.norms[t]))):
            self.done = True
            self.dead()


def backtrace(tokens, parents, step, parent, token, pad):
    """tokens, parents [T, K] of one sequence: (padded row of T tokens, length)."""
    T, K = tokens.shape
    row = [pad] * T
    if not 0 <= step < T:
        return row, 0
    row[step] = token
    k = parent
    for t in range(step - 1, -1, -1):
        if not 0 <= k < K:
            break
        row[t] = int(tokens[t, k])
        k = int(parents[t, k])
    return row, step + 1
