"""Plain restatements of the serving operators in 64 bits (numpy), and the
buffers their tests put on the device.  Shared by test_gpu_serve.py and
test_gpu_paged_decoder.py."""
import numpy as np

TINY, BIG = np.float32(2.0 ** -126), np.float32(8454659 * 2.0 ** 98)
TYPES = {"f32": 0, "bf16": 1, "i8": 2}


def to_bf16(x):
    """fp32 -> bf16 bits, to nearest even; NaN stays NaN."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_bf16(b):
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def quantise(x):
    """(int8 rows, scales) of fp32 rows (last axis)."""
    with np.errstate(all="ignore"):
        top = np.abs(x).max(-1).astype(np.float32)
        s = np.clip(top / np.float32(127), TINY, BIG).astype(np.float32)
        q = np.clip(np.rint((x / s[..., None]).astype(np.float32)), -127, 127)
    bad = ~np.isfinite(x).all(-1)
    s = np.where(bad, np.float32(np.nan), s)
    return np.where(bad[..., None], 0, q).astype(np.int8), s


class Pool:
    """One layer's cache on the host: its stored form and the numbers it stands for."""

    def __init__(self, type, num_pages, page, Hkv, hd, k=None, v=None):
        self.type, self.num, self.page, self.Hkv, self.hd = type, num_pages, page, Hkv, hd
        shape = (num_pages, Hkv, page, hd)
        k = np.zeros(shape, np.float32) if k is None else k
        v = np.zeros(shape, np.float32) if v is None else v
        self.k, self.ks = self.store(k)
        self.v, self.vs = self.store(v)

    def store(self, x):
        if self.type == "f32":
            return np.ascontiguousarray(x, np.float32).copy(), None
        if self.type == "bf16":
            return to_bf16(x), None
        return quantise(x)

    def numbers(self, which):
        x, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        if self.type == "f32":
            return x.astype(np.float64)
        if self.type == "bf16":
            return from_bf16(x).astype(np.float64)
        return x.astype(np.float64) * s.astype(np.float64)[..., None]

    def upload(self, dev, trlm):
        self.ptr = [dev.upload(a) if a is not None else None for a in (self.k, self.v, self.ks, self.vs)]
        return trlm.KvCache(k=self.ptr[0], v=self.ptr[1], k_scale=self.ptr[2], v_scale=self.ptr[3],
                            type=TYPES[self.type], num_pages=self.num, page_size=self.page, kv_heads=self.Hkv,
                            head_dim=self.hd)

    def download(self, dev):
        """(k, v, k_scale, v_scale) as the device holds them."""
        return [dev.download(p, a.shape, a.dtype) if p else None
                for p, a in zip(self.ptr, (self.k, self.v, self.ks, self.vs))]


class Seqs:
    """Sequences of given new and held lengths, with pages dealt at random."""

    def __init__(self, rng, q_len, kv_len, page, spare_pages=2, spare_rows=0, tables=None):
        self.n, self.q_len, self.kv_len = len(q_len), list(q_len), list(kv_len)
        self.q_start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.used = int(self.q_start[-1])
        self.rows = max(1, self.used + spare_rows)
        self.page = page
        self.per = max(1, -(-max(kv_len) // page)) + 1
        self.num = self.n * self.per + spare_pages
        self.pages = rng.permutation(self.num)[:self.n * self.per].reshape(self.n, self.per).astype(np.int32) \
            if tables is None else tables
        self.max_q, self.max_kv = max(1, max(q_len)), max(1, max(kv_len))

    def upload(self, dev, trlm):
        self.ptr = [dev.upload(a) for a in (self.q_start, np.array(self.kv_len, np.int32), self.pages)]
        return trlm.KvSeqs(n=self.n, rows=self.rows, q_start=self.ptr[0], kv_len=self.ptr[1], pages=self.ptr[2],
                           max_pages=self.pages.shape[1], max_q=self.max_q, max_kv=self.max_kv)

    def spans(self):
        """(sequence, first row, rows, position of the first row, tokens held)."""
        return [(i, int(self.q_start[i]), self.q_len[i], self.kv_len[i] - self.q_len[i], self.kv_len[i])
                for i in range(self.n)]

    def cells(self, pool, i, first, last):
        """(page or -1, row in the page) of sequence i's positions first .. last - 1."""
        p = np.arange(first, last)
        ok = (p >= 0) & (p // self.page < self.pages.shape[1])
        pg = np.where(ok, self.pages[i][np.clip(p // self.page, 0, self.pages.shape[1] - 1)], -1)
        return np.where((pg >= 0) & (pg < pool.num), pg, -1), p % self.page


def rotate(x, cos, sin, rot, half):
    """x [.., hd] fp32, tables [.., rot / 2]: exact products, rounded once."""
    a = x.astype(np.float64)
    y = a.copy()
    lo, hi = (a[..., :rot // 2], a[..., rot // 2:rot]) if half else (a[..., 0:rot:2], a[..., 1:rot:2])
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    y0, y1 = lo * c - hi * s, lo * s + hi * c
    if half:
        y[..., :rot // 2], y[..., rot // 2:rot] = y0, y1
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = y0, y1
    return y.astype(np.float32)


def attention(pool, seqs, q, H, scale):
    """(out, bound) in 64 bits: out [rows, H, hd] (zeros where nothing is seen) and for each row and head how far fp32
    arithmetic may be off.  With u = 2^-24, a score in units of log2 is off by at most (hd + 8) u A_t, A_t = scale
    log2(e) sum |q_d k_d| (hd products and sums, the query's scaling, the operands' 22 to 24 bits), and by 2^-29 of the
    row's largest number times the other operand's magnitudes (what the operands' splits leave): a weight relatively by
    d_t = ln 2 times that, 2^-22 for the power and its split, and n u for the sum over n weights.  What all weights
    share cancels.  Numerator and denominator: (sum w_t |v_t| d_t + sum w_t d_t sum w_t |v_t| / sum w_t) / sum w_t, |v_t|
    the row's largest; twice, for the splits and their join, and
    2^-120 where values come near the end of fp32's range."""
    hd, G = pool.hd, H // pool.Hkv
    out = np.zeros((seqs.rows, H, hd))
    bound = np.zeros((seqs.rows, H))
    K, V = pool.numbers("k"), pool.numbers("v")
    u = 2.0 ** -24
    for i, r0, m, first, held in seqs.spans():
        pg, at = seqs.cells(pool, i, 0, held)
        for j in range(m):
            see = np.flatnonzero(pg[:max(0, first + j + 1)] >= 0)
            if not see.size:
                continue
            for h in range(H):
                k, v = K[pg[see], h // G, at[see]], V[pg[see], h // G, at[see]]
                x = q[r0 + j, h * hd:(h + 1) * hd].astype(np.float64)
                z = k @ x * scale
                w = np.exp(z - z.max())
                out[r0 + j, h] = w @ v / w.sum()
                ak, ax, top = np.abs(k), np.abs(x), np.abs(v).max(1)
                A = ak @ ax * (hd + 8) * u + (ak.max(1) * ax.sum() + ak.sum(1) * ax.max()) * 2.0 ** -29
                d = 0.6932 * np.abs(scale) * 1.4427 * A + 2.0 ** -22 + see.size * u
                bound[r0 + j, h] = 2 * (w @ (top * d) + (w @ d) * (w @ top) / w.sum()) / w.sum() + 2.0 ** -120
    return out, bound


def rules(x, history=None, hist_len=None, gen_start=None, rep=None, freq=None, pres=None, bias_ids=None, bias=None,
          n_bias=None, mask=None):
    """(out, bound) of logits x [rows, V] in 64 bits.  Bound: half a unit of the last place for the quotient or
    product, and one for each later sum and product, of the largest magnitude that goes through (5 of 2^-24)."""
    rows, V = x.shape
    y = x.astype(np.float64)
    big = np.abs(y)
    for r in range(rows):
        if history is not None:
            L = min(max(int(hist_len[r]), 0), history.shape[1])
            g = 0 if gen_start is None else int(gen_start[r])
            for t in set(int(t) for t in history[r, :L] if t < V):
                p = 1.0 if rep is None else float(rep[r])
                y[r, t] = y[r, t] / p if y[r, t] > 0 else y[r, t] * p
                big[r, t] = max(big[r, t], abs(y[r, t]))
            for t in set(int(t) for j, t in enumerate(history[r, :L]) if j >= g and t < V):
                c = int(np.sum(history[r, max(g, 0):L] == t))
                d = (0.0 if freq is None else float(freq[r]) * c) + (0.0 if pres is None else float(pres[r]))
                y[r, t] -= d
                big[r, t] = max(big[r, t], abs(d), abs(y[r, t]))
        if bias_ids is not None:
            n = min(max(int(n_bias[r]), 0), bias_ids.shape[1])
            for t, b in {int(t): float(b) for t, b in zip(bias_ids[r, :n], bias[r, :n])}.items():
                if t < V:
                    y[r, t] += b
                    big[r, t] = max(big[r, t], abs(b), abs(y[r, t]))
        if mask is not None:
            open_ = (mask[r][np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1
            y[r, open_ == 0] = -np.inf
    return y, 5 * 2.0 ** -24 * big
