"""The serving operators (trlm_serve.h) against their definitions in 64 bits.

  - trlm_kv_append equals the definition bit for bit (rotation rounded once,
    bf16 to nearest even, 8-bit integers and scales) for every head width,
    cache type and rotary layout, with shared heads, padded row strides,
    empty sequences, rows behind the last one, tokens without a page, rows
    that are not finite and rows at both ends of the range;
  - trlm_kv_read returns those numbers;
  - trlm_attn_paged is within the bound of fp32 arithmetic (serve_ref.py) from
    one token to long chunks, contexts of every length around a tile, a page
    and a split, shared heads, rows that see nothing, missing pages, and
    whatever lies in places that a row does not see;
  - trlm_logits_rules within its bound at aligned and unaligned rows;
  - calls captured into a HIP graph follow their buffers at every replay.
"""
import ctypes as C
import math

import numpy as np
import pytest

import serve_ref as ref

pytestmark = pytest.mark.gpu

ALL_HD = [16, 32, 64, 128]
ALL_TYPES = ["f32", "bf16", "i8"]


@pytest.fixture(scope="module")
def box(trlm):
    dev = trlm.Device()
    serve = trlm.Serve(dev)
    yield dev, serve
    serve.close()
    dev.close()


def bits(a):
    a = np.ascontiguousarray(a)
    return a.view({1: np.uint8, 2: np.uint16, 4: np.uint32}[a.dtype.itemsize])


def same(got, want):
    """Equal bit for bit, NaNs of any pattern equal."""
    if got.dtype.kind == "f":
        return np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(
            bits(got)[~np.isnan(got)], bits(want)[~np.isnan(want)])
    return np.array_equal(got, want)


# ---------------------------------------------------------------- append, read

def tables(max_pos, rot):
    a = np.arange(max_pos)[:, None] * 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))[None, :]
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def append_case(trlm, box, rng, type, hd, H, Hkv, q_len, kv_len, page, rot, half, spare_rows=0, pad=0, max_pos=None,
                special=None, tables_of=None, in_place=False):
    """One append and one read, compared with the definition."""
    dev, serve = box
    dev.current()
    seqs = ref.Seqs(rng, q_len, kv_len, page, spare_rows=spare_rows)
    if tables_of is not None:
        seqs.pages = tables_of(seqs.pages)
    shape = (seqs.num, Hkv, page, hd)
    old = rng.standard_normal((2,) + shape).astype(np.float32)
    pool = ref.Pool(type, seqs.num, page, Hkv, hd, old[0], old[1])
    ld = (H + 2 * Hkv) * hd + pad
    qkv = rng.standard_normal((seqs.rows, ld)).astype(np.float32)
    if special is not None:
        special(qkv, H, Hkv, hd)
    max_pos = max_pos or seqs.max_kv
    cos, sin = tables(max_pos, rot)
    cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
    d_qkv = dev.upload(qkv)
    ldqo = ld if in_place else H * hd + 4
    q_before = qkv if in_place else rng.standard_normal((seqs.rows, ldqo)).astype(np.float32)
    d_out = d_qkv if in_place else dev.upload(q_before)
    d_cos, d_sin = (dev.upload(cos), dev.upload(sin)) if rot else (None, None)
    rows = trlm.KvRows(q=d_qkv if H else None, k=d_qkv + 4 * H * hd, v=d_qkv + 4 * (H + Hkv) * hd, ldq=ld, ldk=ld,
                       ldv=ld, q_out=d_out if H else None, ldqo=ldqo, heads=H, cos_t=d_cos, sin_t=d_sin,
                       max_pos=max_pos if rot else 0, rot_dim=rot, rot_half=int(half))
    serve.append(cache, s, rows)
    got_q = dev.download(d_out, q_before.shape)
    got = pool.download(dev)

    # the definition
    want_q = q_before.copy()
    src = qkv.copy()
    reads = [np.full((seqs.rows, Hkv * hd), 7.0, np.float32) for _ in "kv"]
    for i, r0, m, first, held in seqs.spans():
        pg, at = seqs.cells(pool, i, first, held)
        for j in range(m):
            r, pos = r0 + j, first + j
            for o in reads:
                o[r] = 0
            if pos < 0 or (rot and pos >= max_pos) or pg[j] < 0:
                # not written: reads what was there, where there is a place
                if pos >= 0 and pg[j] >= 0:
                    for o, w in zip(reads, "kv"):
                        o[r] = pool.numbers(w)[pg[j], :, at[j]].astype(np.float32).ravel()
                continue
            x = src[r, :(H + 2 * Hkv) * hd].reshape(-1, hd)
            with np.errstate(all="ignore"):
                t = ref.rotate(x[:H + Hkv], cos[pos], sin[pos], rot, half) if rot else x[:H + Hkv]
                if H:
                    want_q[r, :H * hd] = t[:H].ravel()
                for name, y in (("k", t[H:]), ("v", x[H + Hkv:])):
                    stored, scale = pool.store(y)
                    getattr(pool, name)[pg[j], :, at[j]] = stored
                    if scale is not None:
                        getattr(pool, name + "s")[pg[j], :, at[j]] = scale
    for i, r0, m, first, held in seqs.spans():
        pg, at = seqs.cells(pool, i, first, held)
        for j in range(m):
            if first + j >= 0 and pg[j] >= 0:
                for o, w in zip(reads, "kv"):
                    with np.errstate(all="ignore"):
                        o[r0 + j] = pool.numbers(w)[pg[j], :, at[j]].astype(np.float32).ravel()
    assert same(got_q, want_q)
    for g, w in zip(got, (pool.k, pool.v, pool.ks, pool.vs)):
        assert g is None or same(g, w)

    ldr = Hkv * hd + 4
    before = np.full((seqs.rows, ldr), 7.0, np.float32)
    d_k, d_v = dev.upload(before), dev.upload(before)
    serve.read(cache, s, d_k, d_v, ldr)
    for p, w in zip((d_k, d_v), reads):
        g = dev.download(p, before.shape)
        assert same(g[:, :Hkv * hd], w)
        assert np.all(g[:, Hkv * hd:] == 7.0)
    for p in [d_qkv, d_k, d_v] + ([] if in_place else [d_out]) + ([d_cos, d_sin] if rot else []):
        dev.free(p)
    for p in pool.ptr + seqs.ptr:
        if p:
            dev.free(p)


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd", ALL_HD)
@pytest.mark.parametrize("half", [False, True])
def test_append_and_read(trlm, box, type, hd, half):
    rng = np.random.default_rng(hd * 10 + half)
    append_case(trlm, box, rng, type, hd, 6, 2, [5, 0, 1, 33], [5, 9, 40, 64], 16, hd, half, spare_rows=3, pad=8)
    append_case(trlm, box, rng, type, hd, 3, 3, [1] * 7, [1, 16, 17, 31, 32, 33, 100], 32, hd // 2, half)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_append_many_rows(trlm, box, type):
    """Enough rows for four of them per lane group, ragged against it."""
    rng = np.random.default_rng(3)
    append_case(trlm, box, rng, type, 64, 12, 4, [700, 1, 399, 0, 1023], [900, 1, 399, 12, 1030], 64, 64, True)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_append_keys_and_values_alone_without_rotation(trlm, box, type):
    rng = np.random.default_rng(4)
    append_case(trlm, box, rng, type, 64, 0, 2, [3, 4], [3, 20], 16, 0, False)


@pytest.mark.parametrize("half", [False, True])
def test_append_turns_queries_in_place(trlm, box, half):
    rng = np.random.default_rng(5)
    append_case(trlm, box, rng, "f32", 64, 4, 2, [7, 2], [7, 20], 16, 32, half, in_place=True, spare_rows=2)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_append_passes_over_tokens_without_place(trlm, box, type):
    """Pages of -1 and past the pool, positions past the tables, more new tokens than held (positions below zero)."""
    rng = np.random.default_rng(6)

    def holes(t):
        t = t.copy()
        t[0, 1], t[1, 0], t[2, 0] = -1, 2 ** 31 - 1, 10 ** 6
        return t

    append_case(trlm, box, rng, type, 32, 2, 1, [40, 5, 3, 9], [40, 5, 3, 4], 16, 32, False, tables_of=holes)
    append_case(trlm, box, rng, type, 32, 2, 1, [40, 5], [40, 5], 16, 32, True, max_pos=33)


def test_append_rows_at_the_ends_of_the_range(trlm, box):
    """8 bits: rows of zeros, of denormals, of the largest numbers, and rows that are not finite (read back as NaN)."""
    rng = np.random.default_rng(7)

    def special(x, H, Hkv, hd):
        k = x[:, H * hd:(H + Hkv) * hd]
        v = x[:, (H + Hkv) * hd:(H + 2 * Hkv) * hd]
        v[0] = 0
        v[1] = 1e-42
        v[2] = np.float32(3.4028235e38)
        v[3, ::2] = -np.float32(3.4028235e38)
        v[4, 3] = np.inf
        v[5, 7] = np.nan
        v[6] *= np.float32(1e-30)
        k[7] *= np.float32(1e30)
        v[8] = np.float32(127) * np.float32(2.0 ** -130)

    append_case(trlm, box, rng, "i8", 64, 2, 2, [12], [12], 16, 0, False, special=special)
    append_case(trlm, box, rng, "bf16", 64, 2, 2, [12], [12], 16, 0, False, special=special)
    append_case(trlm, box, rng, "f32", 64, 2, 2, [12], [12], 16, 0, False, special=special)


# ---------------------------------------------------------------- attention

def attn_case(trlm, box, rng, type, hd, H, Hkv, q_len, kv_len, page, spare_rows=0, pad=0, garbage=None, tables_of=None,
              max_q=None, max_kv=None, scale=None, std=1.0, numbers=None):
    """trlm_attn_paged against serve_ref.attention; returns (out, want, seqs)."""
    dev, serve = box
    dev.current()
    seqs = ref.Seqs(rng, q_len, kv_len, page, spare_rows=spare_rows)
    if tables_of is not None:
        seqs.pages = tables_of(seqs.pages)
    if max_q:
        seqs.max_q = max_q
    if max_kv:
        seqs.max_kv = max_kv
    shape = (seqs.num, Hkv, page, hd)
    kv = [std * rng.standard_normal(shape).astype(np.float32), rng.standard_normal(shape).astype(np.float32)]
    if numbers is not None:
        numbers(rng, *kv)
    pool = ref.Pool(type, seqs.num, page, Hkv, hd, *kv)
    ldq, ldo = H * hd + pad, H * hd + 2 * pad
    q = std * rng.standard_normal((seqs.rows, ldq)).astype(np.float32)
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    want, bound = ref.attention(pool, seqs, q, H, scale)
    if garbage is not None:
        garbage(pool, seqs)
    cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
    before = rng.standard_normal((seqs.rows, ldo)).astype(np.float32)
    d_q, d_out = dev.upload(q), dev.upload(before)
    ws_bytes = serve.attn_workspace(cache, s, H)
    ws = dev.upload(np.full(max(ws_bytes // 4, 1), np.nan, np.float32)) if ws_bytes else None
    serve.attn(cache, s, d_q, ldq, H, scale, d_out, ldo, ws, ws_bytes)
    got = dev.download(d_out, before.shape)
    for p in pool.ptr + seqs.ptr + [d_q, d_out, ws]:
        if p:
            dev.free(p)
    used = seqs.used
    assert np.array_equal(got[used:], before[used:]), "rows behind the last sequence"
    assert np.array_equal(got[:, H * hd:], before[:, H * hd:]), "columns behind the heads"
    out = got[:used, :H * hd].reshape(used, H, hd)
    err = np.abs(out - want[:used])
    worst = (err.max(-1) / np.maximum(bound[:used], 2.0 ** -60)).max() if used else 0.0
    assert np.all(err <= bound[:used][..., None]), (worst, err.max())
    return out, want, seqs


def lengths_around(*marks):
    return sorted({max(0, m + d) for m in marks for d in (-1, 0, 1)})


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd", ALL_HD)
@pytest.mark.parametrize("H,Hkv", [(2, 2), (8, 1), (6, 2)])
def test_attn_single_tokens(trlm, box, type, hd, H, Hkv):
    """Contexts of every length around a 16-key group, a block, the waves' share, a page and a split."""
    kv = [k for k in lengths_around(1, 16, 32, 64, 128, 256) if k] + [0, 517]
    rng = np.random.default_rng(hd + H)
    attn_case(trlm, box, rng, type, hd, H, Hkv, [1] * len(kv), kv, 16 if hd < 64 else 64, spare_rows=2, pad=4)


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd", ALL_HD)
@pytest.mark.parametrize("H,Hkv", [(2, 2), (4, 1), (6, 2)])
def test_attn_chunks(trlm, box, type, hd, H, Hkv):
    """A few to many new tokens over cached ones and alone, empty sequences, new tokens without room (q > kv)."""
    rng = np.random.default_rng(7 * hd + H)
    attn_case(trlm, box, rng, type, hd, H, Hkv, [5, 0, 17, 64, 1, 33, 6], [9, 30, 17, 200, 70, 65, 4], 32, spare_rows=1)


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_attn_long_chunks(trlm, box, type, hd):
    rng = np.random.default_rng(11 * hd)
    attn_case(trlm, box, rng, type, hd, 4, 2, [300, 129, 255], [300, 700, 257], 64)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_attn_many_query_heads_to_one(trlm, box, type):
    rng = np.random.default_rng(13)
    attn_case(trlm, box, rng, type, 64, 40, 1, [1, 2, 7], [100, 90, 300], 16)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_attn_one_long_context(trlm, box, type):
    """One sequence over 5,000 tokens in shuffled pages: many splits, joined; with bounds well above the lengths."""
    rng = np.random.default_rng(17)
    attn_case(trlm, box, rng, type, 64, 2, 1, [1], [5001], 16)
    attn_case(trlm, box, rng, type, 64, 2, 1, [1, 3, 1], [130, 2000, 1], 64, max_q=64)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_attn_ignores_what_no_row_sees(trlm, box, type):
    """NaN and infinity in page tails, in pages of nobody, and in tokens after a row's own."""
    rng = np.random.default_rng(19)

    def garbage(pool, seqs):
        used = np.zeros((pool.num, pool.page), bool)
        for i, _, _, _, held in seqs.spans():
            pg, at = seqs.cells(pool, i, 0, held)
            used[pg, at] = True
        for n, (x, s) in enumerate(((pool.k, pool.ks), (pool.v, pool.vs))):
            if pool.type == "i8":
                s.transpose(0, 2, 1)[~used] = np.nan if n else np.inf
            else:
                dead = {"f32": np.float32(np.nan), "bf16": np.uint16(0x7f80)}[pool.type]
                x.transpose(0, 2, 1, 3)[~used] = dead

    attn_case(trlm, box, rng, type, 64, 4, 2, [1, 1, 9, 70], [1, 33, 41, 77], 32, garbage=garbage)
    attn_case(trlm, box, rng, type, 128, 4, 4, [1, 300], [1, 333], 32, garbage=garbage)


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd,q_len,kv_len,at", [(64, 10, 40, 35), (64, 10, 40, 39), (64, 200, 260, 100), (128, 40, 40, 0),
                                                (128, 150, 700, 690), (16, 3, 33, 32)])
def test_attn_what_is_not_finite_stays_with_rows_that_see_it(trlm, box, type, what, hd, q_len, kv_len, at):
    """A value and a key that are not finite at token `at`: NaN for the rows at and after it, nothing for the others."""
    dev, serve = box
    dev.current()
    rng = np.random.default_rng(23)
    for which in "kv":
        seqs = ref.Seqs(rng, [q_len], [kv_len], 16)
        shape = (seqs.num, 1, 16, hd)
        pool = ref.Pool(type, seqs.num, 16, 1, hd, rng.standard_normal(shape).astype(np.float32),
                        rng.standard_normal(shape).astype(np.float32))
        q = rng.standard_normal((seqs.rows, hd)).astype(np.float32)
        want, bound = ref.attention(pool, seqs, q, 1, 0.25)
        pg, pos = seqs.cells(pool, 0, at, at + 1)
        if type == "i8":
            (pool.ks if which == "k" else pool.vs)[pg[0], 0, pos[0]] = np.nan
        else:
            w = np.float32(what)
            (pool.k if which == "k" else pool.v)[pg[0], 0, pos[0], 3] = w if type == "f32" else ref.to_bf16(
                np.array([w]))[0]
        cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
        d_q, d_out = dev.upload(q), dev.empty(q.nbytes)
        ws_bytes = serve.attn_workspace(cache, s, 1)
        ws = dev.empty(ws_bytes) if ws_bytes else None
        serve.attn(cache, s, d_q, hd, 1, 0.25, d_out, hd, ws, ws_bytes)
        out = dev.download(d_out, q.shape)
        sees = kv_len - q_len + np.arange(q_len) >= at
        assert np.all(np.abs(out[~sees] - want[~sees, 0]) <= bound[~sees])
        if which == "k" and type != "i8" and np.isinf(what):
            # an infinite key's score is infinite with the sign of q_3 what: below zero its weight is 2^-inf = 0, so
            # by the definition the row is the attention over the other keys; NaN is allowed too (an infinite fp32
            # number has no split)
            others = ref.Pool("f32", pool.num, 16, 1, hd, pool.numbers("k"), pool.numbers("v"))
            others.k[pg[0], 0, pos[0]] = 0
            others.k[pg[0], 0, pos[0], 3] = np.sign(what) * 1e30
            without, _ = ref.attention(others, seqs, q, 1, 0.25)
            for r in np.flatnonzero(sees):
                # (a row that sees this key alone is then one without a token to see: zeros)
                rest = np.zeros(hd) if kv_len - q_len + r == 0 else without[r, 0]
                low = q[r, 3] * what < 0 and np.all(np.abs(out[r] - rest) <= bound[r])
                assert np.all(np.isnan(out[r])) or low, r
        elif which == "k" or type == "i8":
            assert np.all(np.isnan(out[sees]))
        else:
            assert np.all(~np.isfinite(out[sees][:, 3]))
            rest = np.delete(np.arange(hd), 3)
            assert np.all(np.abs(out[sees][:, rest] - want[sees, 0][:, rest]) <= bound[sees])


@pytest.mark.parametrize("type", ALL_TYPES)
def test_attn_missing_pages_hold_nothing(trlm, box, type):
    rng = np.random.default_rng(29)

    def holes(t):
        t = t.copy()
        t[0, 1], t[1, 0], t[2] = -1, 2 ** 30, -5
        return t

    out, _, seqs = attn_case(trlm, box, rng, type, 64, 4, 2, [1, 20, 3], [70, 50, 33], 16, tables_of=holes)
    assert np.all(out[21:] == 0)      # every page missing: rows without a token to see


@pytest.mark.parametrize("std", [1e-3, 30.0])
def test_attn_flat_and_sharp(trlm, box, std):
    """Nearly equal weights and nearly one-hot ones."""
    rng = np.random.default_rng(31)
    attn_case(trlm, box, rng, "f32", 64, 2, 2, [1, 70], [300, 300], 32, std=std)


def rows_of_all_sizes(rng, k, v):
    """Key and value rows of magnitudes 2^-30 .. 2^30 in no order (keys: to 2^6), some of zeros alone."""
    shape = k.shape[:3] + (1,)
    k *= (2.0 ** rng.integers(-30, 7, shape)).astype(np.float32)
    v *= (2.0 ** rng.integers(-30, 31, shape)).astype(np.float32)
    k[rng.random(k.shape[:3]) < 0.1] = 0
    v[rng.random(k.shape[:3]) < 0.1] = 0


def pages_of_all_sizes(rng, k, v):
    """Magnitudes that change from page to page, to the ends of fp32's range for values."""
    k *= (2.0 ** rng.integers(-20, 5, (k.shape[0], 1, 1, 1))).astype(np.float32)
    v *= (2.0 ** rng.integers(-120, 121, (k.shape[0], 1, 1, 1))).astype(np.float32)


def weightless_giants(rng, k, v):
    """Every eighth key against the queries' mean with a value 2^60 times the others': its weight is 0."""
    k[:, :, ::8] = 0
    k[:, :, ::8, 0] = -3000
    v[:, :, ::8] *= np.float32(2.0 ** 60)


@pytest.mark.parametrize("numbers", [rows_of_all_sizes, pages_of_all_sizes, weightless_giants])
@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_attn_numbers_of_every_magnitude(trlm, box, numbers, type, hd):
    """Neighbours of very different size do not cost one another's precision; single tokens and chunks."""
    rng = np.random.default_rng(47)
    attn_case(trlm, box, rng, type, hd, 2, 1, [1, 70, 2, 150], [77, 130, 200, 150], 16, numbers=numbers)


@pytest.mark.parametrize("std", [2.0 ** -40, 2.0 ** 20])
def test_attn_queries_of_every_magnitude(trlm, box, std):
    """A chunk whose queries are scaled row by row; the scale argument undoes the mean of it."""
    rng = np.random.default_rng(53)
    attn_case(trlm, box, rng, "f32", 64, 2, 2, [1, 100], [100, 300], 32, std=std, scale=0.125 / std / std)


def test_attn_repeats_bit_for_bit(trlm, box):
    outs = []
    for _ in range(2):
        rng = np.random.default_rng(37)
        outs.append(attn_case(trlm, box, rng, "f32", 64, 4, 2, [1, 140, 1], [3000, 900, 5], 32)[0])
    assert np.array_equal(bits(outs[0]), bits(outs[1]))


# ---------------------------------------------------------------- rules

def rules_case(trlm, box, rng, rows, V, hist, bias, mask, pad, in_place=False, parts="rfpg", logits=None):
    dev, serve = box
    dev.current()
    ld = V + pad
    x = (3 * rng.standard_normal((rows, ld))).astype(np.float32) if logits is None else logits
    a = dict(rows=rows, vocab=V, ld=ld, ld_out=ld if in_place else ld + pad)
    r, bufs = {}, {}
    if hist:
        r["history"] = np.minimum(rng.zipf(1.3, (rows, hist)), V + 5).astype(np.uint32)     # some past the vocabulary
        r["history"][:, -1] = 2 ** 32 - 1
        r["hist_len"] = rng.integers(-1, hist + 2, rows).astype(np.int32)
        r["gen_start"] = rng.integers(0, hist + 1, rows).astype(np.int32) if "g" in parts else None
        r["rep"] = (1 + rng.random(rows)).astype(np.float32) if "r" in parts else None
        r["freq"] = rng.random(rows).astype(np.float32) if "f" in parts else None
        r["pres"] = rng.random(rows).astype(np.float32) if "p" in parts else None
    if bias:
        r["bias_ids"] = rng.integers(0, V + 2, (rows, bias)).astype(np.uint32)
        r["bias_ids"][:, bias // 2] = r["bias_ids"][:, 0]                     # the same id twice
        r["bias"] = (5 * rng.standard_normal((rows, bias))).astype(np.float32)
        r["n_bias"] = rng.integers(-1, bias + 2, rows).astype(np.int32)
    if mask:
        r["mask"] = rng.integers(0, 2 ** 32, (rows, (V + 31) // 32 + 1), dtype=np.uint64).astype(np.uint32)
        r["mask"][0] = 0                                                      # leaves nothing
    with np.errstate(all="ignore"):
        want, bound = ref.rules(x[:, :V], **{k: v for k, v in r.items() if v is not None})
    p = {k: dev.upload(v) for k, v in r.items() if v is not None}
    d_x = dev.upload(x)
    before = np.full((rows, a["ld_out"]), 7.0, np.float32)
    d_o = d_x if in_place else dev.upload(before)
    serve.logits_rules(trlm.LogitsRules(
        logits=d_x, out=d_o, **a, history=p.get("history"), hist_len=p.get("hist_len"), gen_start=p.get("gen_start"),
        ld_hist=hist, repetition=p.get("rep"), frequency=p.get("freq"), presence=p.get("pres"),
        bias_ids=p.get("bias_ids"), bias=p.get("bias"), n_bias=p.get("n_bias"), ld_bias=bias, mask=p.get("mask"),
        ld_mask=(V + 31) // 32 + 1 if mask else 0))
    got = dev.download(d_o, (rows, a["ld_out"]))
    for q in list(p.values()) + [d_x] + ([] if in_place else [d_o]):
        dev.free(q)
    assert np.array_equal(got[:, V:], x[:, V:] if in_place else before[:, V:])
    got = got[:, :V]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert np.all(np.abs(got[fine] - want[fine]) <= bound[fine])
    return got


@pytest.mark.parametrize("V,pad", [(1, 0), (3, 1), (31, 0), (33, 3), (1000, 0), (1024, 0), (1025, 3), (4099, 1),
                                   (31769, 3), (31769, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules_sizes(trlm, box, V, pad, in_place):
    rng = np.random.default_rng(V + pad)
    rules_case(trlm, box, rng, 3, V, 40, 6, True, pad, in_place)


@pytest.mark.parametrize("rows,V", [(70, 31769), (1030, 16001)])
def test_rules_many_rows(trlm, box, rows, V):
    """Enough rows for the wide slices, aligned and not."""
    rng = np.random.default_rng(rows)
    rules_case(trlm, box, rng, rows, V, 300, 9, True, (-V) % 4)
    rules_case(trlm, box, rng, rows, V, 300, 9, True, (-V) % 4 + 1)


@pytest.mark.parametrize("hist,bias,mask,parts", [(0, 0, True, ""), (0, 5, False, ""), (50, 0, False, "rfpg"),
                                                  (50, 0, False, "r"), (50, 0, False, "f"), (50, 0, False, "pg"),
                                                  (0, 0, False, ""), (2000, 700, True, "rfp")])
def test_rules_parts(trlm, box, hist, bias, mask, parts):
    rng = np.random.default_rng(hist + bias)
    rules_case(trlm, box, rng, 5, 777, hist, bias, mask, 3, parts=parts)


def test_rules_keep_what_is_not_finite(trlm, box):
    rng = np.random.default_rng(41)
    x = rng.standard_normal((4, 204)).astype(np.float32)
    x[:, 1], x[:, 2], x[:, 3], x[:, 4], x[:, 5] = np.nan, np.inf, -np.inf, 0.0, -0.0
    rules_case(trlm, box, rng, 4, 201, 60, 4, False, 3, logits=x)


# ---------------------------------------------------------------- graphs

def _runtime():
    with open("/proc/self/maps") as fh:
        paths = {line.split()[-1] for line in fh if "libamdhip64.so" in line}
    assert len(paths) == 1, paths
    return C.CDLL(paths.pop())


def test_captured_calls_follow_their_buffers(trlm, box):
    """Append, attention and rules in one graph, replayed with other lengths, tokens and pages, eager calls between."""
    dev, serve = box
    dev.current()
    hip = _runtime()
    rng = np.random.default_rng(43)
    H, Hkv, hd, page, V, n = 4, 2, 64, 16, 300, 3
    seqs = ref.Seqs(rng, [1] * n, [600] * n, page)
    shape = (seqs.num, Hkv, page, hd)
    pool = ref.Pool("i8", seqs.num, page, Hkv, hd, rng.standard_normal(shape).astype(np.float32),
                    rng.standard_normal(shape).astype(np.float32))
    cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
    ld = (H + 2 * Hkv) * hd
    cos, sin = tables(700, hd)
    qkv0 = np.zeros((n, ld), np.float32)
    d = {k: dev.upload(v) for k, v in dict(
        qkv=qkv0, cos=cos, sin=sin, out=np.zeros((n, H * hd), np.float32), logits=np.zeros((n, V), np.float32),
        edited=np.zeros((n, V), np.float32), hist=np.zeros((n, 20), np.uint32), len=np.zeros(n, np.int32),
        rep=np.full(n, 1.5, np.float32)).items()}
    d["q"] = dev.empty(4 * n * H * hd)
    rows = trlm.KvRows(q=d["qkv"], k=d["qkv"] + 4 * H * hd, v=d["qkv"] + 4 * (H + Hkv) * hd, ldq=ld, ldk=ld, ldv=ld,
                       q_out=d["q"], ldqo=H * hd, heads=H, cos_t=d["cos"], sin_t=d["sin"], max_pos=700, rot_dim=hd,
                       rot_half=1)
    ws_bytes = serve.attn_workspace(cache, s, H)
    ws = dev.empty(ws_bytes)
    assert ws_bytes
    edit = trlm.LogitsRules(logits=d["logits"], out=d["edited"], rows=n, vocab=V, ld=V, ld_out=V, history=d["hist"],
                            hist_len=d["len"], ld_hist=20, repetition=d["rep"])

    def step():
        serve.append(cache, s, rows)
        serve.attn(cache, s, d["q"], H * hd, H, 0.125, d["out"], H * hd, ws, ws_bytes)
        serve.logits_rules(edit)

    step()
    dev.sync()
    stream, graph, exe = C.c_void_p(dev.ctx.stream), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0

    def put(p, a):
        a = np.ascontiguousarray(a)
        dev.hip.hip_h2d(p, a.ctypes.data, a.nbytes)

    try:
        for lens in ([1, 17, 599], [300, 0, 64], [2, 130, 600], [600, 600, 600]):
            qkv = rng.standard_normal((n, ld)).astype(np.float32)
            logits = rng.standard_normal((n, V)).astype(np.float32)
            hist, hl = rng.integers(0, V, (n, 20)).astype(np.uint32), rng.integers(0, 21, n).astype(np.int32)
            seqs.pages = rng.permutation(seqs.num)[:seqs.pages.size].reshape(seqs.pages.shape).astype(np.int32)
            seqs.kv_len = lens
            for p, a in ((d["qkv"], qkv), (d["logits"], logits), (d["hist"], hist), (d["len"], hl),
                         (seqs.ptr[1], np.array(lens, np.int32)), (seqs.ptr[2], seqs.pages)):
                put(p, a)
            before = pool.download(dev)
            outs = []
            for eager in (False, True, False):
                for p, a in zip(pool.ptr, before):
                    put(p, a)
                if eager:
                    step()
                else:
                    assert hip.hipGraphLaunch(exe, stream) == 0
                dev.sync()
                outs.append([dev.download(d["out"], (n, H * hd)), dev.download(d["edited"], (n, V))]
                            + pool.download(dev))
            for got in outs:
                for a, b in zip(got, outs[1]):
                    assert same(a, b)
            pool.k, pool.v, pool.ks, pool.vs = outs[1][2:]
            q = dev.download(d["q"], (n, H * hd))
            want, bound = ref.attention(pool, seqs, q, H, 0.125)
            seen = np.array(lens) > 0
            assert np.all(np.abs(outs[0][0].reshape(n, H, hd) - want)[seen] <= bound[seen][..., None])
            assert np.all(outs[0][0][~seen] == 0)
            y, b = ref.rules(logits, hist, hl, rep=np.full(n, 1.5))
            assert np.all(np.abs(outs[0][1] - y) <= b)
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


# ---------------------------------------------------------------- calls at the edges of what is allowed

@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("q_len,kv_len,spare,max_q", [([10], [40], 90, 100), ([1], [700], 299, 300), ([0], [9], 64, 64),
                                                      ([10, 3], [500, 3], 187, 100), ([1, 100], [1, 100], 99, 100),
                                                      ([3, 70], [900, 900], 0, 400)])
def test_attn_bounds_wider_than_the_call(trlm, box, type, q_len, kv_len, spare, max_q):
    """max_q and rows are bounds: a call that could hold long chunks and holds short ones."""
    attn_case(trlm, box, np.random.default_rng(47), type, 64, 4, 2, q_len, kv_len, 32, spare_rows=spare, max_q=max_q)


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("q_len,kv_len", [([300], [100]), ([400, 1, 200], [30, 9, 0])])
def test_attn_more_new_tokens_than_kept(trlm, box, type, q_len, kv_len):
    """The first of them see nothing, and the plan does not count on them."""
    attn_case(trlm, box, np.random.default_rng(49), type, 64, 4, 2, q_len, kv_len, 32)


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("page", [16, 65536])
def test_page_sizes_at_the_ends(trlm, box, type, page):
    rng = np.random.default_rng(53)
    attn_case(trlm, box, rng, type, 16, 2, 1, [1, 90, 7], [17, 90, 1500], page)
    append_case(trlm, box, rng, type, 16, 2, 1, [1, 90, 7], [17, 90, 1500], page, 16, False)


@pytest.mark.parametrize("type", ALL_TYPES)
def test_starts_out_of_range_are_kept_to_the_rows(trlm, box, type):
    """Row ranges that break the rules (negative, descending, past the end): nothing outside the buffers is touched."""
    dev, serve = box
    dev.current()
    rng = np.random.default_rng(59)
    H, Hkv, hd, page, rows, guard = 4, 2, 64, 16, 90, 40
    ld = (H + 2 * Hkv) * hd
    for starts in ([-5, 3, 2, 1000, 80], [50, 20, 90, 2 ** 31 - 1, -2 ** 31], [-2 ** 31, -1, 0, 40, 2 ** 31 - 1]):
        for max_q in (4, 90):
            seqs = ref.Seqs(rng, [20] * 4, [33] * 4, page)
            shape = (seqs.num, Hkv, page, hd)
            pool = ref.Pool(type, seqs.num, page, Hkv, hd, rng.standard_normal(shape).astype(np.float32),
                            rng.standard_normal(shape).astype(np.float32))
            seqs.q_start, seqs.rows, seqs.max_q, seqs.max_kv = np.array(starts, np.int32), rows, max_q, 3000
            seqs.kv_len = [33, 2 ** 31 - 1, -2 ** 31, 5]
            cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
            cos, sin = tables(64, hd)
            whole = rng.standard_normal((rows + 2 * guard, ld)).astype(np.float32)
            d_x, d_cos, d_sin = dev.upload(whole), dev.upload(cos), dev.upload(sin)
            x = d_x + 4 * guard * ld
            d_o, d_k, d_v = [dev.upload(whole) for _ in range(3)]
            rows_ = trlm.KvRows(q=x, k=x + 4 * H * hd, v=x + 4 * (H + Hkv) * hd, ldq=ld, ldk=ld, ldv=ld, q_out=x, ldqo=ld,
                                heads=H, cos_t=d_cos, sin_t=d_sin, max_pos=64, rot_dim=hd, rot_half=0)
            ws_bytes = serve.attn_workspace(cache, s, H)
            edge = np.full(1024, 3.0, np.float32)
            d_ws = dev.upload(np.concatenate([edge, np.zeros(ws_bytes // 4, np.float32), edge]))
            serve.append(cache, s, rows_)
            serve.attn(cache, s, x, ld, H, 0.125, d_o + 4 * guard * ld, ld, d_ws + 4096, ws_bytes)
            serve.read(cache, s, d_k + 4 * guard * ld, d_v + 4 * guard * ld, ld)
            for p in (d_x, d_o, d_k, d_v):
                got = dev.download(p, whole.shape)
                assert np.array_equal(got[:guard], whole[:guard]) and np.array_equal(got[-guard:], whole[-guard:])
            got = dev.download(d_ws, (2048 + ws_bytes // 4,))
            assert np.array_equal(got[:1024], edge) and np.array_equal(got[-1024:], edge)
            for p in pool.ptr + seqs.ptr + [d_x, d_o, d_k, d_v, d_cos, d_sin, d_ws]:
                if p:
                    dev.free(p)


@pytest.mark.parametrize("type,numbers", [("f32", 2 ** 32), ("bf16", 2 ** 32), ("i8", 5 * 2 ** 30)])
def test_offsets_past_32_bits(trlm, box, type, numbers):
    """A pool of more than 2^32 numbers, the pages in use at both of its ends; rows 2^30 floats apart."""
    dev, serve = box
    dev.current()
    rng = np.random.default_rng(61)
    H, Hkv, hd, page = 2, 2, 64, 64
    num = numbers // (Hkv * page * hd) + 3
    small = ref.Seqs(rng, [100, 1], [100, 1], page)
    small.pages = np.array([[0, 1], [2, 3]], np.int32)
    pool = ref.Pool(type, 4, page, Hkv, hd)
    size = {"f32": 4, "bf16": 2, "i8": 1}[type]
    d = {n: dev.hip.hip_alloc(num * Hkv * page * hd * size) for n in "kv"}
    sc = {n: dev.hip.hip_alloc(num * Hkv * page * 4) for n in "kv"} if type == "i8" else dict(k=None, v=None)
    cache = trlm.KvCache(k=d["k"], v=d["v"], k_scale=sc["k"], v_scale=sc["v"], type=ref.TYPES[type], num_pages=num,
                         page_size=page, kv_heads=Hkv, head_dim=hd)
    far = small.pages.copy()
    small.pages = np.array([[num - 1, 0], [num - 3, num - 2]], np.int32)
    s = small.upload(dev, trlm)
    small.pages = far
    ld = 3 * H * hd
    x = rng.standard_normal((101, ld)).astype(np.float32)
    d_x = dev.upload(x)
    serve.append(cache, s, trlm.KvRows(q=None, k=d_x + 4 * H * hd, v=d_x + 8 * H * hd, ldq=0, ldk=ld, ldv=ld, q_out=None,
                                       ldqo=0, heads=0, cos_t=None, sin_t=None, max_pos=0, rot_dim=0, rot_half=0))
    for r in range(101):
        pg, at = small.pages[0 if r < 100 else 1][r % 100 // page], r % 100 % page
        for j, n in enumerate("kv"):
            stored, scale = pool.store(x[r, (1 + j) * H * hd:(2 + j) * H * hd].reshape(Hkv, hd))
            getattr(pool, n)[pg, :, at] = stored
            if scale is not None:
                getattr(pool, n + "s")[pg, :, at] = scale
    outs = [dev.empty(4 * 101 * Hkv * hd) for _ in "kv"]
    serve.read(cache, s, outs[0], outs[1], Hkv * hd)
    for n, o in zip("kv", outs):
        got = dev.download(o, (101, Hkv, hd))
        for r in range(101):
            pg, at = small.pages[0 if r < 100 else 1][r % 100 // page], r % 100 % page
            assert np.array_equal(got[r], pool.numbers(n)[pg, :, at].astype(np.float32))
    want, bound = ref.attention(pool, small, x, H, 0.125)
    ws_bytes = serve.attn_workspace(cache, s, H)
    ws, d_o = dev.empty(ws_bytes), dev.empty(4 * 101 * H * hd)
    serve.attn(cache, s, d_x, ld, H, 0.125, d_o, H * hd, ws, ws_bytes)
    assert np.all(np.abs(dev.download(d_o, (101, H, hd)) - want) <= bound[..., None])
    if type == "bf16":
        # the second sequence's token and two more rows, 2^30 floats apart (row 2 is 2^31 floats and 2^33 bytes in)
        wide = ref.Seqs(rng, [2, 1], [100, 1], page)
        wide.pages = np.array([[num - 1, 0], [num - 3, num - 2]], np.int32)
        s2 = wide.upload(dev, trlm)
        gap = 2 ** 30
        d_q, d_w = [dev.hip.hip_alloc(4 * (2 * gap + H * hd)) for _ in "qo"]
        y = x[98:]
        for r in range(3):
            row = np.ascontiguousarray(y[r, :H * hd])
            dev.hip.hip_h2d(d_q + 4 * r * gap, row.ctypes.data, row.nbytes)
        ws2 = dev.empty(serve.attn_workspace(cache, s2, H))
        serve.attn(cache, s2, d_q, gap, H, 0.125, d_w, gap, ws2, serve.attn_workspace(cache, s2, H))
        for r in range(3):
            got = dev.download(d_w + 4 * r * gap, (H, hd))
            assert np.all(np.abs(got - want[98 + r]) <= bound[98 + r][:, None])
        rule = trlm.LogitsRules(logits=d_q, out=d_w, rows=3, vocab=H * hd, ld=gap, ld_out=gap)
        serve.logits_rules(rule)
        for r in range(3):
            assert np.array_equal(dev.download(d_w + 4 * r * gap, (H * hd,)), y[r, :H * hd])
        for p in [d_q, d_w, ws2] + wide.ptr:
            dev.free(p)
    for p in list(d.values()) + [p for p in sc.values() if p] + outs + [d_x, ws, d_o] + small.ptr:
        dev.free(p)


def test_two_contexts_at_once(trlm, box):
    """Two contexts, each with its own stream, handle and workspace, their calls queued in turn before either is waited
    for: the same as alone."""
    dev, serve = box
    dev2 = trlm.Device()
    serve2 = trlm.Serve(dev2)
    rng = np.random.default_rng(67)
    H, Hkv, hd, page = 4, 2, 64, 32
    jobs = []
    for d, e in ((dev, serve), (dev2, serve2)):
        d.current()
        seqs = ref.Seqs(rng, [1, 200, 3], [900, 400, 3], page)
        shape = (seqs.num, Hkv, page, hd)
        pool = ref.Pool("bf16", seqs.num, page, Hkv, hd, rng.standard_normal(shape).astype(np.float32),
                        rng.standard_normal(shape).astype(np.float32))
        q = rng.standard_normal((seqs.rows, H * hd)).astype(np.float32)
        cache, s = pool.upload(d, trlm), seqs.upload(d, trlm)
        n = e.attn_workspace(cache, s, H)
        jobs.append((d, e, cache, s, d.upload(q), d.empty(q.nbytes), d.empty(n), n, ref.attention(pool, seqs, q, H, 0.125),
                     q.shape))
    for _ in range(20):
        for d, e, cache, s, q, o, ws, n, _, _ in jobs:
            d.current()
            e.attn(cache, s, q, H * hd, H, 0.125, o, H * hd, ws, n)
    for d, e, cache, s, q, o, ws, n, (want, bound), shape in jobs:
        d.current()
        got = d.download(o, shape).reshape(-1, H, hd)
        assert np.all(np.abs(got - want) <= bound[..., None])
    dev2.current()
    serve2.close()
    dev2.close()
    dev.current()


@pytest.mark.parametrize("type", ALL_TYPES)
@pytest.mark.parametrize("hd", ALL_HD)
def test_attn_mixed_batches(trlm, box, type, hd):
    """Long chunks beside single tokens: row tiles found among the sequences' counts; more of them than the rows with one
    sequence at its longest suggest (taken in turns); more sequences than a workgroup has threads; long ones anywhere."""
    rng = np.random.default_rng(71 + hd)
    attn_case(trlm, box, rng, type, hd, 2, 1, [1, 300, 1, 0, 2, 1], [50, 400, 1, 7, 600, 33], 32, spare_rows=3)
    attn_case(trlm, box, rng, type, hd, 2, 2, [70] * 6, [90, 70, 200, 70, 71, 300], 16, max_q=420)
    if hd == 64:
        attn_case(trlm, box, rng, type, hd, 2, 2, [66] * 20 + [1] * 20, [66] * 20 + [200] * 20, 16, max_q=1340)
        n = 1100
        q, kv = np.ones(n, int), rng.integers(1, 40, n)
        for at, m in ((0, 140), (513, 70), (1025, 65), (1099, 300)):
            q[at], kv[at] = m, m + 9
        attn_case(trlm, box, rng, type, hd, 1, 1, q.tolist(), kv.tolist(), 16, spare_rows=1)


def test_attn_mixed_batch_captured(trlm, box):
    """One graph of a mixed batch, replayed with the long sequences elsewhere."""
    dev, serve = box
    dev.current()
    hip = _runtime()
    rng = np.random.default_rng(73)
    H, Hkv, hd, page, n = 2, 1, 64, 16, 12
    seqs = ref.Seqs(rng, [1] * 10 + [300, 90], [320] * n, page)
    shape = (seqs.num, Hkv, page, hd)
    pool = ref.Pool("bf16", seqs.num, page, Hkv, hd, rng.standard_normal(shape).astype(np.float32),
                    rng.standard_normal(shape).astype(np.float32))
    q = rng.standard_normal((seqs.rows, H * hd)).astype(np.float32)
    cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
    d_q, d_o = dev.upload(q), dev.upload(q)
    ws_bytes = serve.attn_workspace(cache, s, H)
    ws = dev.empty(ws_bytes)

    def step():
        serve.attn(cache, s, d_q, H * hd, H, 0.125, d_o, H * hd, ws, ws_bytes)

    step()
    dev.sync()
    stream, graph, exe = C.c_void_p(dev.ctx.stream), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    try:
        for lens in ([1] * 10 + [300, 90], [65] * 6 + [1] * 6, [0, 200, 1, 70, 0, 0, 120, 9, 0, 0, 0, 0], [1] * n):
            seqs.q_len, seqs.kv_len = lens, [m + int(rng.integers(0, 20)) for m in lens]
            seqs.q_start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            for p, a in ((seqs.ptr[0], seqs.q_start), (seqs.ptr[1], np.array(seqs.kv_len, np.int32))):
                dev.hip.hip_h2d(p, a.ctypes.data, a.nbytes)
            want, bound = ref.attention(pool, seqs, q, H, 0.125)
            outs = []
            for eager in (False, True, False):
                dev.hip.hip_h2d(d_o, q.ctypes.data, q.nbytes)
                if eager:
                    step()
                else:
                    assert hip.hipGraphLaunch(exe, stream) == 0
                dev.sync()
                outs.append(dev.download(d_o, q.shape))
            assert same(outs[0], outs[1]) and same(outs[2], outs[1])
            used = int(seqs.q_start[-1])
            assert np.array_equal(outs[0][used:], q[used:])
            err = np.abs(outs[0][:used].reshape(used, H, hd) - want[:used])
            assert np.all(err <= bound[:used][..., None])
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


def test_first_call_of_a_handle_captured(trlm, box):
    """A handle finds its kernels at their first use, which may be inside a capture."""
    dev, _ = box
    dev.current()
    serve = trlm.Serve(dev)
    hip = _runtime()
    rng = np.random.default_rng(79)
    H, Hkv, hd, page = 2, 1, 32, 16
    seqs = ref.Seqs(rng, [1, 80], [700, 90], page)
    shape = (seqs.num, Hkv, page, hd)
    pool = ref.Pool("i8", seqs.num, page, Hkv, hd, rng.standard_normal(shape).astype(np.float32),
                    rng.standard_normal(shape).astype(np.float32))
    q = rng.standard_normal((seqs.rows, H * hd)).astype(np.float32)
    cache, s = pool.upload(dev, trlm), seqs.upload(dev, trlm)
    d_q, d_o = dev.upload(q), dev.empty(q.nbytes)
    ws_bytes = serve.attn_workspace(cache, s, H)
    ws = dev.empty(ws_bytes)
    dev.sync()
    stream, graph, exe = C.c_void_p(dev.ctx.stream), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    serve.attn(cache, s, d_q, H * hd, H, 0.2, d_o, H * hd, ws, ws_bytes)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    want, bound = ref.attention(pool, seqs, q, H, 0.2)
    try:
        for _ in range(3):
            assert hip.hipGraphLaunch(exe, stream) == 0
            dev.sync()
            got = dev.download(d_o, q.shape).reshape(-1, H, hd)
            assert np.all(np.abs(got - want) <= bound[..., None])
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
        serve.close()
