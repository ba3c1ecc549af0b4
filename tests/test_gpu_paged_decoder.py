"""The paged decoder (gpu_paged_*), which runs the serving operators together.

  - prompts, chunks of prompts and single tokens of sequences of their own
    lengths, in one call: the last tokens' logits equal the oracle's full
    forward of each sequence (fp32 cache), within 1e-4 of max|logits|, as the
    decoder's do (head_dim 16, 32, 64);
  - with every cache type, a plain restatement of the model in 64 bits that
    attends over the keys and values read back from the decoder gives its
    logits within 1e-4, and its own keys and values are those read back within
    half a step of the type;
  - rules, greedy picks and sampling on the logits;
  - refusals change nothing; pages come back and are used again.
"""
import numpy as np
import pytest

import serve_ref as ref

pytestmark = pytest.mark.gpu


class Box:
    def __init__(self, trlm, orc, V, D, H, L, F, params=None):
        self.shape = (V, D, H, L, F)
        self.model = orc.Model(V, D, H, L, F)
        self.params = self.model.init(1337, 1) if params is None else params
        self.hm = trlm.HostModel(V, D, H, L, F, self.params)
        self.tr = trlm.Trainer(self.hm, 1, 8)
        self.trlm, self.decs = trlm, []

    def decoder(self, *a, **k):
        d = self.trlm.PagedDecoder(self.tr, *a, **k)
        self.decs.append(d)
        return d

    def __enter__(self):
        return self

    def __exit__(self, *_):
        for d in self.decs:
            d.destroy()
        self.tr.destroy()
        self.hm.close()

    def last_row(self, tokens):
        t = np.ascontiguousarray(tokens, np.uint32)
        return self.model.forward_logits(self.params, t, 1, t.size).reshape(t.size, -1)[-1]


def near(got, want, tol=1e-4):
    err = np.abs(got.astype(np.float64) - want).max() / np.abs(want).max()
    assert err <= tol, err


@pytest.mark.parametrize("V,D,H,L,F,page", [(61, 32, 2, 2, 48, 16), (97, 64, 2, 2, 96, 16), (83, 128, 2, 2, 160, 32),
                                            (59, 96, 6, 2, 50, 64)])
def test_sequences_of_their_own_lengths(trlm, orc, V, D, H, L, F, page):
    rng = np.random.default_rng(1)
    with Box(trlm, orc, V, D, H, L, F) as b:
        dec = b.decoder(5, 200, 40, page)
        text = {s: rng.integers(0, V, 200).astype(np.uint32) for s in range(5)}
        held = dict.fromkeys(text, 0)
        # prompts; a chunk beside single tokens; a new sequence beside both; long chunks (the many-rows kernel)
        for call in ([(3, 7), (0, 1), (1, 40)], [(0, 1), (3, 1), (1, 1)], [(1, 90), (3, 1), (4, 17), (0, 1)],
                     [(2, 130)], [(2, 1), (4, 66), (0, 15), (1, 2), (3, 1)]):
            dec.extend([s for s, _ in call], [text[s][held[s]:held[s] + m] for s, m in call])
            for s, m in call:
                held[s] += m
            got = dec.logits()
            for r, (s, _) in enumerate(call):
                assert dec.length(s) == held[s]
                near(got[r], b.last_row(text[s][:held[s]]))
            assert np.array_equal(dec.greedy(), np.argmax(got, axis=1))
            assert dec.free_pages() == 40 - sum(-(-held[s] // page) for s in held)


def forward64(b, tokens, caches, H, noise=None):
    """The model in 64 bits, attention over the given caches [(k, v)] per layer; (last logits, [(k, v)] of its own).
    With a generator as noise, every query is off by up to 2^-20 of the largest one."""
    V, D, _, L, F = b.shape
    p, off, t = [], 0, np.asarray(tokens, np.int64)
    for s in b.hm.shapes:
        p.append(b.params[off:off + int(np.prod(s))].reshape(s).astype(np.float64))
        off += int(np.prod(s))
    hd, n = D // H, t.size
    # the angles are the framework's own numbers, formed in fp32 (at position 100 a 64-bit angle is 1e-5 away)
    freq = (10000.0 ** np.float64(np.float32(-2.0 * np.arange(hd // 2) / hd))).astype(np.float32)
    ang = (np.arange(n, dtype=np.float32)[:, None] * freq[None, :]).astype(np.float64)
    c, s_ = np.cos(ang)[:, None, :], np.sin(ang)[:, None, :]

    def turn(x):
        y = x.reshape(n, H, hd)
        e, o = y[..., 0::2], y[..., 1::2]
        return np.stack([e * c - o * s_, e * s_ + o * c], -1).reshape(n, D)

    def norm(x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w

    x, own = p[0][t], []
    for l in range(L):
        an, wqkv, bqkv, wo, bo, fn, wgu, bgu, wd, bd = p[1 + 10 * l:11 + 10 * l]
        qkv = norm(x, an) @ wqkv + bqkv
        q, k, v = turn(qkv[:, :D]), turn(qkv[:, D:2 * D]), qkv[:, 2 * D:]
        own.append((k, v))
        if noise is not None:
            q = q + 2.0 ** -20 * np.abs(q).max() * noise.uniform(-1, 1, q.shape)
        K, W = [a.astype(np.float64) for a in caches[l]]
        att = np.zeros((n, D))
        for h in range(H):
            i = slice(h * hd, (h + 1) * hd)
            z = q[:, i] @ K[:, i].T / np.sqrt(hd)
            z[np.triu_indices(n, 1)] = -np.inf
            w = np.exp(z - z.max(-1, keepdims=True))
            att[:, i] = w @ W[:, i] / w.sum(-1, keepdims=True)
        x = x + att @ wo + bo
        gu = norm(x, fn) @ wgu + bgu
        g, u = gu[:, :F], gu[:, F:]
        x = x + (g / (1 + np.exp(-g)) * u) @ wd + bd
    return norm(x[-1:], p[-1])[0] @ p[0].T, own


@pytest.mark.parametrize("name,kv", [("f32", 0), ("bf16", 1), ("i8", 2)])
def test_every_cache_type(trlm, orc, name, kv):
    V, D, H, L, F = 89, 128, 2, 3, 96
    rng = np.random.default_rng(2)
    with Box(trlm, orc, V, D, H, L, F) as b0:
        params = (6 * b0.params).astype(np.float32)       # sharper scores than a fresh model's
    with Box(trlm, orc, V, D, H, L, F, params) as b:
        dec = b.decoder(3, 150, 30, 16, kv)
        text = rng.integers(0, V, (3, 150)).astype(np.uint32)
        held = [0, 0, 0]
        for call in ([(0, 20), (2, 90)], [(2, 1), (0, 1), (1, 33)], [(0, 1), (1, 1), (2, 1)], [(1, 70), (0, 1)]):
            dec.extend([s for s, _ in call], [text[s][held[s]:held[s] + m] for s, m in call])
            for s, m in call:
                held[s] += m
        got = dec.logits()
        for r, s in enumerate((1, 0)):
            caches = [dec.read(s, l) for l in range(L)]
            want, own = forward64(b, text[s][:held[s]], caches, H)
            near(got[r], want)
            # Half a step of the type, 2^-16 of the largest number for the fp32 products before it, and from the second
            # layer on what the queries' rounding does to the attention below. With numbers of 30 and heads of 64 a
            # score q.k/8 reaches hundreds: a query off by 2^-22 of its size, as fp32 sums of 128 products are, moves a
            # score of 300 by 1e-4 or more, and where two keys share a row their weights by a quarter of that, times
            # the difference of their values (50): 1e-3, many times 2^-16 of 30, at such a row and no other. So the
            # 64-bit model is asked: four times what its own numbers move by with its queries off by 2^-20.
            moved = forward64(b, text[s][:held[s]], caches, H, np.random.default_rng(7))[1]
            for l in range(L):
                for mine, cached, other in zip(own[l], caches[l], moved[l]):
                    x = mine.reshape(held[s], H, D // H)
                    slack = 2.0 ** -16 * np.abs(x).max() + 4 * np.abs(other - mine).max(1)[:, None, None]
                    assert np.median(slack) < 1e-3              # few rows are like that
                    if name == "i8":
                        step = (0.5 / 127) * np.abs(x).max(-1, keepdims=True)
                    else:
                        step = (2.0 ** -8 if name == "bf16" else 2.0 ** -24) * np.abs(x)
                    assert np.all(np.abs(cached.reshape(x.shape) - x) <= 1.001 * step + slack)


def test_rules_picks_and_sampling(trlm, orc):
    V, D, H, L, F = 113, 64, 2, 2, 96
    rng = np.random.default_rng(3)
    with Box(trlm, orc, V, D, H, L, F) as b:
        dec = b.decoder(4, 64, 20, 16, trlm.KV_BF16)
        prompt = [rng.integers(0, V, m).astype(np.uint32) for m in (9, 1, 30)]
        more = [rng.integers(0, V, m).astype(np.uint32) for m in (1, 2, 1)]
        order = [2, 0, 3]
        dec.extend(order, prompt)
        dec.extend(order[::-1], more)
        before = dec.logits()
        full = [np.concatenate([prompt[2 - r], more[r]]) for r in range(3)]
        hist = np.zeros((3, 40), np.uint32)
        for r in range(3):
            hist[r, :full[r].size] = full[r]
        a = dict(rep=np.array([1.3, 1.0, 2.0], np.float32), freq=np.array([0.2, 0.0, 0.1], np.float32),
                 pres=np.array([0.0, 0.5, 0.1], np.float32), bias_ids=rng.integers(0, V, (3, 4)).astype(np.uint32),
                 bias=rng.standard_normal((3, 4)).astype(np.float32), n_bias=np.array([4, 0, 2], np.uint32),
                 mask=rng.integers(0, 2 ** 32, (3, 4), dtype=np.uint64).astype(np.uint32))
        a["mask"][1] = 0                                     # a grammar that leaves nothing
        dec.rules(a["rep"], a["freq"], a["pres"], a["bias_ids"], a["bias"], a["n_bias"], a["mask"])
        got = dec.logits()
        want, bound = ref.rules(before, hist, [f.size for f in full], [prompt[2 - r].size for r in range(3)], **a)
        fine = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), fine) and np.all(np.abs(got[fine] - want[fine]) <= bound[fine])
        assert np.array_equal(dec.greedy(), [np.argmax(got[0]), 0, np.argmax(got[2])])
        rngs = (trlm.PCGState * 3)(*[trlm.libs()[0].pcg_seed(4242, 7 + r) for r in range(3)])
        mirror = [orc.pcg_stream(4242, 7 + r) for r in range(3)]
        pick = dec.sample(rngs, 0.85)
        for r in (0, 2):
            assert pick[r] == orc.sample_next(got[r], 0.85, mirror[r])
            assert a["mask"][r][pick[r] // 32] >> (pick[r] % 32) & 1
        assert pick[1] == V - 1


def test_refusals_change_nothing_and_pages_come_back(trlm, orc):
    V, D, H, L, F = 61, 32, 2, 1, 48
    rng = np.random.default_rng(4)
    with Box(trlm, orc, V, D, H, L, F) as b:
        dec = b.decoder(3, 100, 8, 16)
        text = rng.integers(0, V, (3, 100)).astype(np.uint32)
        with pytest.raises(trlm.Refused):
            dec.rules()                                      # no logits yet
        dec.extend([0, 1], [text[0][:50], text[1][:60]])     # 4 + 4 pages: all of them
        assert dec.free_pages() == 0
        before = dec.logits()
        for seqs, toks in (([2], [text[2][:1]]), ([0, 2], [text[0][50:51], text[2][:5]]), ([1], [text[1][60:65]]),
                           ([0, 0], [text[0][50:51], text[0][51:52]]), ([3], [text[0][:1]]), ([0], [text[0][:0]]),
                           ([0], [np.array([V], np.uint32)]), ([0], [np.zeros(51, np.uint32)]), ([], [])):
            with pytest.raises(trlm.Refused):
                dec.extend(seqs, toks)
            assert [dec.length(s) for s in range(4)] == [50, 60, 0, 0] and dec.free_pages() == 0
        assert np.array_equal(dec.logits(), before)
        ids, one = np.zeros((2, 3), np.uint32), np.ones(2, np.float32)
        with pytest.raises(trlm.Refused):
            dec.rules(bias_ids=ids, bias=np.ones((2, 3), np.float32), n_bias=np.array([1, 4], np.uint32))
        with pytest.raises(trlm.Refused):
            dec.rules(bias_ids=ids)
        for bad in (dict(repetition=one[:1]), dict(mask=np.zeros((2, 1), np.uint32)), dict(bias_ids=ids, bias=one)):
            with pytest.raises(ValueError):
                dec.rules(**bad)
        with pytest.raises(ValueError):
            dec.extend([0, 1], [text[0][:1]])
        with pytest.raises(ValueError):
            dec.sample((trlm.PCGState * 1)(), 1.0)
        dec.rules()                                          # none: the logits as they are
        assert np.array_equal(dec.logits(), before)
        with pytest.raises(trlm.Refused):
            dec.read(0, 1)
        dec.extend([0], [text[0][50:55]])                    # room in its last page
        near(dec.logits()[0], b.last_row(text[0][:55]))
        dec.release(1)
        assert dec.length(1) == 0 and dec.free_pages() == 4
        dec.extend([2, 0], [text[2][:30], text[0][55:56]])   # another sequence in the pages that came back
        got = dec.logits()
        near(got[0], b.last_row(text[2][:30]))
        near(got[1], b.last_row(text[0][:56]))
        dec.release(0)
        dec.extend([0], [text[1][:80]])                      # a slot again
        near(dec.logits()[0], b.last_row(text[1][:80]))
        k, v = dec.read(1, 0)
        assert k.shape == (0, D) and v.shape == (0, D)


def test_model_sized_batch(trlm, orc):
    """The model's own width and vocabulary, 64 sequences of ragged lengths, prompts and then steps: equal to the
    decoder (pinned to the oracle) run one sequence at a time, within 1e-4."""
    V, D, H, L, F = 31769, 384, 6, 2, 1024
    rng = np.random.default_rng(5)
    with Box(trlm, orc, V, D, H, L, F) as b:
        dec = b.decoder(64, 128, 64 * 2, 64)
        lens = rng.integers(1, 120, 64)
        text = [rng.integers(0, V, m + 2).astype(np.uint32) for m in lens]
        dec.extend(np.arange(64), [t[:-2] for t in text])
        dec.extend(np.arange(64), [t[-2:-1] for t in text])
        dec.extend(np.arange(64), [t[-1:] for t in text])
        got = dec.logits()
        one = trlm.Decoder(b.tr, 1, 128)
        for s in rng.permutation(64)[:6]:
            one.prefill(text[s][None])
            near(got[s], one.logits()[0])
        one.destroy()
