"""Plain 64-bit implementations of the decode operators (8-bit K/V cache, attention, beam search) for
their tests, written position by position from the definitions in include/stt_b200.h."""
import math

import numpy as np

BLOCK, EMIN = 16, -100


def exponent(amax: float) -> int:
    """Smallest e >= EMIN with amax <= 127 * 2^e."""
    if amax == 0:
        return EMIN
    e = math.frexp(amax / 127.0)[1] - 2
    while amax > math.ldexp(127.0, e):
        e += 1
    return max(EMIN, e)


class RefCache:
    """One half (K or V) of a cache: codes [seqs, heads, cap, dim] and exponents [seqs, heads, cap / 16]."""

    def __init__(self, codes, exps):
        self.codes, self.exps = codes.astype(np.int64), exps.astype(np.int64)
        self.cap = codes.shape[2]

    def append(self, seq, pos, x):
        """x [count, heads, dim] in f64 at positions pos .. pos + count - 1."""
        count = x.shape[0]
        b = pos // BLOCK * BLOCK if count else pos
        while b < pos + count:
            lo, hi = max(b, pos), min(b + BLOCK, pos + count)
            at, blk, old = b % self.cap, b % self.cap // BLOCK, lo - b
            for h in range(x.shape[1]):
                new = x[lo - pos:hi - pos, h]
                fin = np.where(np.isfinite(new), new, 0.0)
                e = exponent(float(np.abs(fin).max()))
                if old:
                    was = int(self.exps[seq, h, blk])
                    e = max(e, was)
                    self.codes[seq, h, at:at + old] = np.rint(np.ldexp(self.codes[seq, h, at:at + old].astype(float), was - e))
                q = np.rint(np.ldexp(np.where(np.isnan(new), 0.0, new), -e))
                self.codes[seq, h, at + old:at + old + hi - lo] = np.clip(q, -127, 127)
                self.exps[seq, h, blk] = e
            b += BLOCK

    def values(self, seq, positions):
        """[positions, heads, dim]."""
        slot = np.asarray(positions, dtype=np.int64) % self.cap
        c = self.codes[seq][:, slot].astype(np.float64)
        return np.ldexp(c, self.exps[seq][:, slot // BLOCK][..., None]).transpose(1, 0, 2)


def attention(k: RefCache, v: RefCache, seq, pos, q, scale, window=0, start=0):
    """q [count, heads, dim] at positions pos ..; returns (out, sum over |q||k| scale's maximum)."""
    count, heads, dim = q.shape
    group = heads // k.codes.shape[1]
    out = np.zeros((count, heads, dim))
    ring = -(-(pos + count) // BLOCK) * BLOCK - k.cap
    biggest = 0.0
    for t in range(count):
        P = pos + t
        lo = max(0, start, ring, P + 1 - window if window else 0)
        if lo > P:
            continue
        kk, vv = k.values(seq, range(lo, P + 1)), v.values(seq, range(lo, P + 1))
        for j in range(heads):
            s = kk[:, j // group] @ q[t, j] * scale
            biggest = max(biggest, float((np.abs(kk[:, j // group]) @ np.abs(q[t, j])).max()) * abs(scale))
            w = np.exp(s - s.max())
            out[t, j] = w @ vv[:, j // group] / w.sum()
    return out, biggest


def select(logits, scores, done=None, eos=-1):
    """logits [batch, beams, vocab], scores [batch, beams]: (scores, parents, tokens, done), best first,
    equal candidates by the lowest beam * vocab + token."""
    batch, beams, vocab = logits.shape
    x = logits.astype(np.float64)
    total = np.full((batch, beams, vocab), -np.inf)
    for g in range(batch):
        for b in range(beams):
            s = float(scores[g, b])
            if done is not None and done[g, b]:
                if eos >= 0:
                    total[g, b, eos] = s
                continue
            top = x[g, b].max()
            if not s < math.inf or not top < math.inf or top == -math.inf or s == -math.inf:
                continue
            total[g, b] = ((x[g, b] - top) - math.log(np.exp(x[g, b] - top).sum())) + s
    flat = total.reshape(batch, -1)
    at = np.argsort(-flat, axis=1, kind="stable")[:, :beams]
    parents, tokens = at // vocab, at % vocab
    ended = tokens == eos
    if done is not None:
        ended |= np.take_along_axis(np.asarray(done, bool), parents, 1)
    return np.take_along_axis(flat, at, 1), parents, tokens, ended
