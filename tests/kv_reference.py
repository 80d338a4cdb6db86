"""A plain restatement of the paged int8 cache: appending in the f32 steps that its definition names (numpy has no fused
multiply-add, so they are the same bits), attention in 64 bits."""
import numpy as np

BLOCK, SCALE_MIN, LARGEST = 16, np.float32(2.0 ** -40), np.float32(131008.0)


def rotate(x, cos, sin, rot, interleaved):
    """x f32 [n, heads, d], cos / sin f32 [n, rot/2]."""
    y, half = x.copy(), rot // 2
    e = np.arange(half)
    one, two = (2 * e, 2 * e + 1) if interleaved else (e, e + half)
    c, s = cos[:, None], sin[:, None]
    with np.errstate(invalid="ignore"):
        y[:, :, one] = x[:, :, one] * c - x[:, :, two] * s
        y[:, :, two] = x[:, :, two] * c + x[:, :, one] * s
    return y


def quantise(y, inv):
    with np.errstate(invalid="ignore"):
        q = np.rint(y * inv)
    return np.clip(np.nan_to_num(q, nan=0.0, posinf=127, neginf=-127), -127, 127).astype(np.int8)


class Cache:
    """k, v int8 [pages, kv_heads, page, d]; ks, vs float32 [pages, kv_heads, page / 16]."""

    def __init__(self, rng, pages, kv_heads, d, page):
        self.kv_heads, self.d, self.page = kv_heads, d, page
        self.k, self.v = [rng.integers(-127, 128, (pages, kv_heads, page, d)).astype(np.int8) for _ in range(2)]
        self.ks, self.vs = [(rng.random((pages, kv_heads, page // BLOCK)) * 0.02 + 0.01).astype(np.float32) for _ in range(2)]

    def copy(self):
        c = object.__new__(Cache)
        c.__dict__.update({k: v.copy() if isinstance(v, np.ndarray) else v for k, v in self.__dict__.items()})
        return c

    def _store(self, cache, scale, y, pages, first):
        """y f32 [n, kv_heads, d] become the tokens from position `first` on of the sequence with these pages."""
        n = y.shape[0]
        for block in range(first // BLOCK, -(-(first + n) // BLOCK)):
            lo, hi = max(first, block * BLOCK), min(first + n, (block + 1) * BLOCK)
            page, at = pages[lo // self.page], lo % self.page
            inside = at // BLOCK
            new, begin = y[lo - first:hi - first], lo - block * BLOCK
            with np.errstate(invalid="ignore"):
                top = np.minimum(np.nanmax(np.nan_to_num(np.abs(new), nan=0.0, posinf=np.inf), axis=(0, 2)), LARGEST)
            old = scale[page, :, inside].copy() if begin else np.zeros(self.kv_heads, np.float32)
            s = np.maximum(np.maximum(top / np.float32(127.0), old), SCALE_MIN)
            if begin:
                slots = slice(inside * BLOCK, inside * BLOCK + begin)
                ratio = np.where(s > old, old / s, np.float32(1.0)).astype(np.float32)
                cache[page, :, slots] = quantise(cache[page, :, slots].astype(np.float32), ratio[:, None, None])
            slots = slice(inside * BLOCK + begin, inside * BLOCK + begin + hi - lo)
            cache[page, :, slots] = quantise(new, (np.float32(1.0) / s)[None, :, None]).transpose(1, 0, 2)
            scale[page, :, inside] = s

    def append(self, q, k, v, cos, sin, table, q_start, kv_len, rot, interleaved):
        """q f16 [tokens, heads, d], k, v f16 [tokens, kv_heads, d]; the rotated q in f32 (rows of no sequence: zeros)."""
        out = np.zeros(q.shape, np.float32)
        for b, kv in enumerate(kv_len):
            r0, r1 = q_start[b], q_start[b + 1]
            if r1 == r0:
                continue
            first = kv - (r1 - r0)
            yq, yk = q[r0:r1].astype(np.float32), k[r0:r1].astype(np.float32)
            if rot:
                yq, yk = [rotate(x, cos[first:kv], sin[first:kv], rot, interleaved) for x in (yq, yk)]
            out[r0:r1] = yq
            self._store(self.k, self.ks, yk, table[b], first)
            self._store(self.v, self.vs, v[r0:r1].astype(np.float32), table[b], first)
        return out

    def values(self, table, kv):
        """Keys and values of a sequence's tokens, f64 [kv, kv_heads, d]."""
        pages = np.asarray(table[:-(-kv // self.page)], np.int64)
        got = []
        for cache, scale in ((self.k, self.ks), (self.v, self.vs)):
            s = np.maximum(scale[pages], SCALE_MIN).astype(np.float64).repeat(BLOCK, axis=2)[..., None]
            with np.errstate(invalid="ignore"):  # what lies behind the last token may be anything
                got.append((cache[pages] * s).transpose(0, 2, 1, 3).reshape(-1, self.kv_heads, self.d)[:kv])
        return got

    def attend(self, q, table, q_start, kv_len, causal=True):
        """(out f64 [tokens, heads, d], bound on the error of the f16 kernels' outputs); see `attention_bound`."""
        heads = q.shape[1]
        out, bound = [np.zeros(q.shape) for _ in range(2)]
        for b, kv in enumerate(kv_len):
            r0, r1 = q_start[b], q_start[b + 1]
            if r1 == r0 or kv == 0:
                continue
            k, v = self.values(table[b], kv)
            vs = np.maximum(self.vs[np.asarray(table[b][:-(-kv // self.page)], np.int64)], SCALE_MIN)
            seen = np.arange(kv)[None] < (kv - (r1 - r0) + np.arange(r1 - r0) + 1 if causal else np.full(r1 - r0, kv))[:, None]
            for h in range(heads):
                g = h // (heads // self.kv_heads)
                out[r0:r1, h], bound[r0:r1, h] = attention(q[r0:r1, h].astype(np.float64), k[:, g], v[:, g], seen,
                                                           float(vs[:, g].max()))
        return out, bound


def attention(q, k, v, seen, vs_max):
    """One head: (out, bound).  What the kernels may be off by:
      out       rounded to f16:                          2^-11 |o| (2^-25 below f16's normal range)
      P         rounded to f16 before P V:               2^-11 sum p |v|, and 2^-25 * 127 vs per key for what is below the
                normal range (the largest P is at least 1 when no score is masked, and P = p vs / max (p vs))
      scores    f32 products of up to d terms:           (d + 4) 2^-24 sum |q k| / sqrt(d) on each exponent, counted twice:
                in P and in the sum
      the sum and the output's accumulation in f32:      (keys + 16) 2^-24 sum p |v|
    """
    n, d = q.shape
    x = np.where(seen, q @ k.T / np.sqrt(d), -np.inf)
    top = x.max(1, keepdims=True)
    p = np.exp(x - np.where(np.isinf(top), 0.0, top))
    total = p.sum(1, keepdims=True)
    p /= np.where(total == 0, 1.0, total)
    o = p @ v
    spread = p @ np.abs(v)
    score = ((d + 4) * 2.0 ** -24 * np.where(seen, np.abs(q) @ np.abs(k).T, 0).max(1) / np.sqrt(d))[:, None]
    keys = seen.sum(1)[:, None]
    return o, 2.0 ** -11 * np.abs(o) + 2.0 ** -24 + spread * (2.0 ** -11 + 2 * score + (keys + 16) * 2.0 ** -24) + \
        keys * 2.0 ** -25 * 127 * vs_max
