"""Serving operators: a paged K/V cache, the attention that reads it, and the rules on the logits that follow.

Four operators, all on device buffers through the C ABI as turkce-llm_amd/trlm.py binds it:

  append  trlm_kv_append: rotary positions of the new tokens' queries and keys (interleaved or half layout, the
          whole head or its first part), the keys and values written into the cache's pages as fp32, bf16 or 8 bits
          with a scale for each token and head.
  read    trlm_kv_read: the cache's rows of given tokens back as fp32 rows.  An 8-bit append is followed by the
          read of the same tokens, so that the stored values come back as the numbers they stand for.
  attn    trlm_attn_paged: causal attention of each sequence's new tokens (one, a few, or a long chunk) over all its
          cached tokens, read from the pages; the heads may share keys and values in groups.
  rules   trlm_logits_rules: repetition, frequency and presence penalties from each row's tokens, a bias list and a
          grammar's bit mask, from one buffer of logits to another.

Sizes come from the repository's model (V 31769, 6 heads of 64, B8 T1024, 64 sequences of decode) and from generic
heads that share keys and values (32 on 8 of 128, 16 on 2 of 64); draw() spreads over what lies between.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": 0, "bf16": 1, "i8": 2}        # the binding's KV_F32, KV_BF16, KV_I8
BYTES = {"f32": 4, "bf16": 2, "i8": 1}
TINY, BIG = 2.0 ** -126, float(0x810203) * 2.0 ** 98   # the scales' bounds: no division by zero, 127 * BIG is finite


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of 64 sequences of the model: the smallest call, where latency counts
        _cache("append", "append 64 tokens f32", n=64, q=1, kv=1024, H=6, Hkv=6, hd=64, page=64, type="f32"),
        # a training batch's worth of prompt tokens into an 8-bit cache, half-layout rotation, and read back
        _cache("append", "append 8x1024 i8 + read", n=8, q=1024, kv=1024, H=32, Hkv=8, hd=128, page=64, type="i8",
               half=True),
        # sequences leave a bf16 cache whole (to a host, another GPU): ragged lengths
        _cache("read", "read 16 sequences bf16", n=16, q=4096, kv=4096, H=8, Hkv=8, hd=128, page=32, type="bf16",
               ragged=True),
        # one user of the model: a single token over a short context
        _cache("attn", "attn 1 token kv 1000 f32", n=1, q=1, kv=1000, H=6, Hkv=6, hd=64, page=64, type="f32"),
        # a decode step of 64 sequences of the model, ragged contexts
        _cache("attn", "attn 64 tokens kv 1024 f32", n=64, q=1, kv=1024, H=6, Hkv=6, hd=64, page=64, type="f32",
               ragged=True),
        # a decode step over long contexts held in 8 bits, four query heads to a cached one
        _cache("attn", "attn 32 tokens kv 8192 i8", n=32, q=1, kv=8192, H=32, Hkv=8, hd=128, page=128, type="i8",
               ragged=True),
        # drafted tokens checked in one call: a few queries each, odd and empty sequences among them
        _cache("attn", "attn 24x5 drafted bf16", n=24, q=5, kv=2000, H=16, Hkv=2, hd=64, page=16, type="bf16",
               ragged=True),
        # the prompts of a training-sized batch of the model from an empty cache
        _cache("attn", "attn 8x1024 prompts f32", n=8, q=1024, kv=1024, H=6, Hkv=6, hd=64, page=64, type="f32"),
        # one chunk of a long prompt over what is cached already
        _cache("attn", "attn chunk 2048 kv 16384 bf16", n=1, q=2048, kv=16384, H=32, Hkv=8, hd=128, page=64,
               type="bf16"),
        # one user of the model: penalties and a grammar over one row
        _rules("rules 1 row", rows=1, V=31769, hist=300, bias=8, mask=True),
        # 64 sequences of the model, rows padded to 16 bytes as the decoder keeps them
        _rules("rules 64 rows", rows=64, V=31769, hist=1024, bias=16, mask=True),
        # many sequences over a large vocabulary, penalties alone
        _rules("rules 256 rows V 131072", rows=256, V=131072, hist=2048, bias=0, mask=False),
    ]


def _cache(op, name, *, n, q, kv, H, Hkv, hd, page, type, ragged=False, half=False, rot=None):
    c = dict(op=op, n=n, q=q, kv=kv, H=H, Hkv=Hkv, hd=hd, page=page, type=type, ragged=ragged)
    if op == "append":
        c |= dict(half=half, rot=hd if rot is None else rot)
    return dict(c, name=name) if name else c


def _rules(name, *, rows, V, hist, bias, mask, pad=True):
    c = dict(op="rules", rows=rows, V=V, hist=hist, bias=bias, mask=mask, pad=pad)
    return dict(c, name=name) if name else c


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attn", "attn", "attn", "rules"])
    if op == "rules":
        while True:
            rows, V = _logint(rng, 1, 256), _logint(rng, 50, 131072)
            if rows * V <= 2 ** 24:
                break
        hist, bias = rng.choice([0, _logint(rng, 1, 4096)]), rng.choice([0, 3, 40])
        return _rules(None, rows=rows, V=V, hist=hist, bias=bias, mask=rng.random() < 0.5 or not hist + bias,
                      pad=rng.random() < 0.75)
    hd = rng.choice([16, 32, 64, 64, 128, 128])
    Hkv, G = rng.choice([1, 2, 3, 6, 8]), rng.choice([1, 1, 2, 4, 5, 8])
    H, page, type = Hkv * G, rng.choice([16, 32, 64, 128]), rng.choice(["f32", "bf16", "i8"])
    shape = dict(H=H, Hkv=Hkv, hd=hd, page=page, type=type)
    if op == "append":
        while True:
            n, q = _logint(rng, 1, 128), rng.choice([1, _logint(rng, 1, 2048)])
            if n * q * (H + 2 * Hkv) * hd <= 6e7:
                break
        half = rng.random() < 0.5
        return _cache(op, None, n=n, q=q, kv=q + _logint(rng, 1, 2048), ragged=rng.random() < 0.5, half=half,
                      rot=rng.choice([hd, hd // 2]), **shape)
    if op == "read":
        while True:
            n, kv = _logint(rng, 1, 64), _logint(rng, 1, 8192)
            if n * kv * Hkv * hd <= 6e7:
                break
        return _cache(op, None, n=n, q=rng.choice([kv, max(1, kv // 3)]), kv=kv, ragged=True, **shape)
    while True:
        mode = rng.choice(["token", "token", "few", "chunk"])
        q = {"token": 1, "few": rng.randint(2, 16), "chunk": _logint(rng, 17, 2048)}[mode]
        n, kv = _logint(rng, 1, 8 if mode == "chunk" else 96), q + _logint(rng, 1, 16384)
        if n * kv * Hkv * hd <= 1.3e8 and n * H * q * kv <= 4e8 and n * H * q * kv * hd <= 6e10:
            break
    return _cache(op, None, n=n, q=q, kv=kv, ragged=rng.random() < 0.6, **shape)


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)


def _normal(gen, *shape, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std


def _lengths(c):
    """Each sequence's new tokens and its tokens in all, a case's own.  Ragged: from a tenth of the longest on, one
    sequence of the longest, and of more than two the second without new tokens."""
    n, q, kv = c["n"], c["q"], c["kv"]
    g = torch.Generator().manual_seed(1000 * kv + 10 * n + q)
    if not c["ragged"]:
        return [q] * n, [kv] * n
    qs, kvs = [], []
    for i in range(n):
        f = 0.1 + 0.9 * float(torch.rand((), generator=g)) if i else 1.0
        k = max(1, int(kv * f))
        m = max(1, int(q * (0.1 + 0.9 * float(torch.rand((), generator=g))))) if i and 1 < q < kv else q
        m = k if q == kv else min(m, k)
        qs.append(0 if i == 1 and n > 2 else m)
        kvs.append(k)
    return qs, kvs


def _quantise(x):
    """8 bits for each row of the last axis: (values in [-127, 127] as fp32, scale)."""
    top = x.abs().amax(-1, keepdim=True)
    s = (top / torch.full_like(top, 127.0)).clamp(TINY, BIG)     # a quotient: by a number torch would multiply
    return torch.round(x / s).clamp(-127, 127), s


def prepare(case, seed):
    return _prepare_rules(case, seed) if case["op"] == "rules" else _prepare_cache(case, seed)


def _prepare_cache(c, seed):
    gen = _gen(seed)
    n, H, Hkv, hd, page, type = c["n"], c["H"], c["Hkv"], c["hd"], c["page"], c["type"]
    qs, kvs = _lengths(c)
    rows = sum(qs)
    per = -(-max(kvs) // page)
    num = n * per + 3                       # a few pages more than are in use
    order = torch.randperm(num, generator=gen, device="cuda")
    s = {"case": c, "rows": rows, "max_q": max(qs), "max_kv": max(kvs), "num_pages": num}
    s["pages"] = order[:n * per].reshape(n, per).to(torch.int32).contiguous()
    s["q_start"] = torch.tensor([0] + [sum(qs[:i + 1]) for i in range(n)], dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    # keys with a few large channels, as rotated keys have; values near the normal
    shape = (num, Hkv, page, hd)
    if c["op"] == "append":
        for x in "kv":
            s[x] = torch.zeros(shape, device="cuda", dtype=_torch_type(type))
            s[x + "_scale"] = torch.zeros(shape[:3], device="cuda") if type == "i8" else None
        # the projections' rows side by side, as the model's QKV product leaves them
        s["qkv"] = _normal(gen, rows, (H + 2 * Hkv) * hd) * (1.0 + 4.0 * (torch.rand(
            (H + 2 * Hkv) * hd, generator=gen, device="cuda") < 0.03))
        s["q_out"] = torch.zeros((rows, H * hd), device="cuda")
        s["max_pos"] = max(kvs)
        angle = torch.arange(max(kvs), dtype=torch.float64)[:, None] * 10000.0 ** (
            -2.0 * torch.arange(c["rot"] // 2, dtype=torch.float64) / c["rot"])[None, :]
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    else:
        big = 1.0 + 4.0 * (torch.rand(hd, generator=gen, device="cuda") < 0.03)
        for x, f in (("k", big), ("v", 1.0)):
            t = _normal(gen, *shape) * f
            if type == "i8":
                t, scale = _quantise(t)
                s[x + "_scale"] = scale[..., 0].contiguous()
            else:
                s[x + "_scale"] = None
            s[x] = t.to(_torch_type(type))
            del t
    if c["op"] == "attn":
        s["q"] = _normal(gen, rows, H * hd)
        s["out"] = torch.zeros((rows, H * hd), device="cuda")
    else:
        for x in ("k_read", "v_read"):
            s[x] = torch.zeros((rows, Hkv * hd), device="cuda")
    return s


def _torch_type(type):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}[type]


def _prepare_rules(c, seed):
    gen = _gen(seed)
    rows, V, hist = c["rows"], c["V"], c["hist"]
    ld = (V + 3) // 4 * 4 if c["pad"] else V
    s = {"case": c, "logits": _normal(gen, rows, ld, std=3.0), "out": torch.zeros((rows, ld), device="cuda")}
    if hist:
        # a few tokens come again and again, as in text; each row of a length of its own
        u = torch.rand((rows, hist), generator=gen, device="cuda", dtype=torch.float64)
        s["history"] = (V ** u).long().sub(1).clamp(0, V - 1).to(torch.int32)
        s["hist_len"] = torch.randint(0, hist + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        s["gen_start"] = (s["hist_len"] * torch.rand(rows, generator=gen, device="cuda")).to(torch.int32)
        s["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=gen, device="cuda")
        s["frequency"] = 0.3 * torch.rand(rows, generator=gen, device="cuda")
        s["presence"] = 0.5 * torch.rand(rows, generator=gen, device="cuda")
    if c["bias"]:
        s["bias_ids"] = torch.randint(0, V, (rows, c["bias"]), generator=gen, device="cuda", dtype=torch.int32)
        s["bias"] = _normal(gen, rows, c["bias"], std=4.0)
        s["n_bias"] = torch.randint(0, c["bias"] + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if c["mask"]:
        # a grammar allows whole runs of tokens: a tenth of the words are open
        words = (V + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen, device="cuda", dtype=torch.int64)
        keep = torch.rand((rows, words), generator=gen, device="cuda") < 0.1
        s["mask"] = torch.where(keep, bits, torch.zeros_like(bits)).to(torch.int32)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "read": _plain_read, "attn": _plain_attn, "rules": _plain_rules}[
        state["case"]["op"]](state["case"], state)


def _rows_of(s):
    """Of every row: its sequence and its token's position there."""
    rows = torch.arange(s["rows"], device="cuda")
    seq = torch.bucketize(rows, s["q_start"][1:].long(), right=True)
    start, end = s["q_start"].long()[seq], s["q_start"].long()[seq + 1]
    return seq, s["kv_len"].long()[seq] - end + rows, rows - start


def _slots(s, seq, pos):
    page = s["case"]["page"]
    return s["pages"].long()[seq, pos // page], pos % page


def _stored(s, x, page, slot):
    """Cached rows [.., Hkv, hd] as fp32."""
    t = s[x].permute(0, 2, 1, 3)[page, slot].float()
    return t * s[x + "_scale"].permute(0, 2, 1)[page, slot][..., None] if s["case"]["type"] == "i8" else t


def _rotate(c, x, cos, sin):
    """x [rows, heads, hd] turned by each row's angles, computed in 64 bits and rounded once."""
    r = c["rot"]
    a = x.double()
    a, b = (a[..., :r // 2], a[..., r // 2:r]) if c["half"] else (a[..., 0:r:2], a[..., 1:r:2])
    cs, sn = cos.double()[:, None, :], sin.double()[:, None, :]
    y0, y1 = (a * cs - b * sn).float(), (a * sn + b * cs).float()
    y = torch.cat([y0, y1], -1) if c["half"] else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _plain_append(c, s):
    H, Hkv, hd = c["H"], c["Hkv"], c["hd"]
    seq, pos, _ = _rows_of(s)
    page, slot = _slots(s, seq, pos)
    x = s["qkv"].reshape(s["rows"], H + 2 * Hkv, hd)
    cos, sin = s["cos"][pos], s["sin"][pos]
    s["q_out"].copy_(_rotate(c, x[:, :H], cos, sin).reshape(s["rows"], -1))
    for name, t in (("k", _rotate(c, x[:, H:H + Hkv], cos, sin)), ("v", x[:, H + Hkv:])):
        if c["type"] == "i8":
            t, scale = _quantise(t)
            s[name + "_scale"].permute(0, 2, 1)[page, slot] = scale[..., 0]
        s[name].permute(0, 2, 1, 3)[page, slot] = t.to(s[name].dtype)
    if c["type"] == "i8":
        return [s["q_out"]] + _plain_read(c, s)
    return [s["q_out"], s["k"], s["v"]]


def _plain_read(c, s):
    seq, pos, _ = _rows_of(s)
    page, slot = _slots(s, seq, pos)
    for x in "kv":
        s[x + "_read"].copy_(_stored(s, x, page, slot).reshape(s["rows"], -1))
    return [s["k_read"], s["v_read"]]


def _plain_attn(c, s):
    n, H, Hkv, hd, mq, mk = c["n"], c["H"], c["Hkv"], c["hd"], s["max_q"], s["max_kv"]
    G = H // Hkv
    seq, pos, at = _rows_of(s)
    q = torch.zeros((n, mq, H, hd), device="cuda")
    q[seq, at] = s["q"].reshape(s["rows"], H, hd)
    q = q.reshape(n, mq, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(n * Hkv, G * mq, hd)
    j = torch.arange(mk, device="cuda")
    held = (j < s["kv_len"][:, None])
    where = torch.where(held, j, torch.zeros_like(j))
    page, slot = _slots(s, torch.arange(n, device="cuda")[:, None], where)
    k, v = (_stored(s, x, page, slot).permute(0, 2, 1, 3).reshape(n * Hkv, mk, hd) for x in "kv")
    S = torch.matmul(q * (1.0 / math.sqrt(hd)), k.transpose(1, 2).contiguous())
    del k
    first = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1])).long()
    seen = (j <= first[:, None, None] + torch.arange(mq, device="cuda")[:, None]) & held[:, None, :]
    S = S.reshape(n, H, mq, mk).masked_fill_(~seen[:, None], -math.inf)
    m = S.amax(-1, keepdim=True)
    S = S.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = S.sum(-1, keepdim=True)
    o = torch.matmul(S.reshape(n * Hkv, G * mq, mk), v).reshape(n, H, mq, hd) / total
    s["out"].copy_(o.permute(0, 2, 1, 3)[seq, at].reshape(s["rows"], -1))
    return s["out"]


def _plain_rules(c, s):
    rows, V = c["rows"], c["V"]
    x = s["logits"][:, :V].clone()
    row = torch.arange(rows, device="cuda")[:, None]
    if c["hist"]:
        at = torch.arange(c["hist"], device="cuda")
        held = at < s["hist_len"][:, None]
        made = held & (at >= s["gen_start"][:, None])
        ids = s["history"].long()
        seen = torch.zeros((rows, V), device="cuda").scatter_add_(1, ids, held.float()) > 0
        count = torch.zeros((rows, V), device="cuda").scatter_add_(1, ids, made.float())
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = torch.where(count > 0, x - (s["frequency"][:, None] * count + s["presence"][:, None]), x)
    if c["bias"]:
        # an id that stands more than once takes its last entry
        at = torch.arange(c["bias"], device="cuda").expand(rows, -1)
        at = torch.where(at < s["n_bias"][:, None], at, torch.full_like(at, -1))
        last = torch.full((rows, V), -1, device="cuda", dtype=torch.int64)
        last.scatter_reduce_(1, s["bias_ids"].long(), at, "amax")
        x = torch.where(last >= 0, x + s["bias"].gather(1, last.clamp(min=0)), x)
    if c["mask"]:
        t = torch.arange(V, device="cuda")
        open_ = (s["mask"][:, t // 32] >> (t % 32).to(torch.int32)) & 1
        x = x.masked_fill(open_ == 0, -math.inf)
    s["out"][:, :V] = x
    return s["out"][:, :V]


# ---------------------------------------------------------------- the framework's calls

_kept = None


def _program():
    """What a serving program keeps: the context, the operators' handle and one workspace."""
    global _kept
    if _kept is None:
        if "trlm_amd" not in sys.modules:
            path = os.path.join(ROOT, "turkce-llm_amd", "trlm.py")
            spec = importlib.util.spec_from_file_location("trlm_amd", path)
            mod = importlib.util.module_from_spec(spec)
            sys.modules["trlm_amd"] = mod
            spec.loader.exec_module(mod)
        trlm = sys.modules["trlm_amd"]
        dev = trlm.Device()
        _kept = {"trlm": trlm, "dev": dev, "serve": trlm.Serve(dev), "ws": None}
    return _kept


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _plan(s, p):
    """The call's argument blocks, made once for a state."""
    trlm, c = p["trlm"], s["case"]
    if c["op"] == "rules":
        ld = s["logits"].shape[1]
        return trlm.LogitsRules(
            logits=_ptr(s["logits"]), out=_ptr(s["out"]), rows=c["rows"], vocab=c["V"], ld=ld, ld_out=ld,
            history=_ptr(s.get("history")), hist_len=_ptr(s.get("hist_len")), gen_start=_ptr(s.get("gen_start")),
            ld_hist=c["hist"], repetition=_ptr(s.get("repetition")), frequency=_ptr(s.get("frequency")),
            presence=_ptr(s.get("presence")), bias_ids=_ptr(s.get("bias_ids")), bias=_ptr(s.get("bias")),
            n_bias=_ptr(s.get("n_bias")), ld_bias=c["bias"], mask=_ptr(s.get("mask")), ld_mask=(c["V"] + 31) // 32)
    cache = trlm.KvCache(k=_ptr(s["k"]), v=_ptr(s["v"]), k_scale=_ptr(s["k_scale"]), v_scale=_ptr(s["v_scale"]),
                         type=TYPES[c["type"]], num_pages=s["num_pages"], page_size=c["page"], kv_heads=c["Hkv"],
                         head_dim=c["hd"])
    seqs = trlm.KvSeqs(n=c["n"], rows=s["rows"], q_start=_ptr(s["q_start"]), kv_len=_ptr(s["kv_len"]),
                       pages=_ptr(s["pages"]), max_pages=s["pages"].shape[1], max_q=s["max_q"], max_kv=s["max_kv"])
    rows = None
    if c["op"] == "append":
        ld, hd = s["qkv"].shape[1], c["hd"]
        at = s["qkv"].data_ptr()
        rows = trlm.KvRows(q=at, k=at + 4 * c["H"] * hd, v=at + 4 * (c["H"] + c["Hkv"]) * hd, ldq=ld, ldk=ld, ldv=ld,
                           q_out=_ptr(s["q_out"]), ldqo=c["H"] * hd, heads=c["H"], cos_t=_ptr(s["cos"]),
                           sin_t=_ptr(s["sin"]), max_pos=s["max_pos"], rot_dim=c["rot"], rot_half=int(c["half"]))
    return cache, seqs, rows


def _run_own(s):
    c, p = s["case"], _program()
    serve = p["serve"]
    if "plan" not in s:
        s["plan"] = _plan(s, p)
    p["dev"].current()
    if c["op"] == "rules":
        serve.logits_rules(s["plan"])
        return s["out"][:, :c["V"]]
    cache, seqs, rows = s["plan"]
    if c["op"] == "attn":
        if "ws_bytes" not in s:
            s["ws_bytes"] = serve.attn_workspace(cache, seqs, c["H"])
            if s["ws_bytes"] and (p["ws"] is None or p["ws"].numel() < s["ws_bytes"]):
                p["dev"].sync()
                p["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device="cuda")
        D = c["H"] * c["hd"]
        serve.attn(cache, seqs, s["q"].data_ptr(), D, c["H"], 1.0 / math.sqrt(c["hd"]), s["out"].data_ptr(), D,
                   _ptr(p["ws"]), s["ws_bytes"])
        return s["out"]
    if c["op"] == "append":
        serve.append(cache, seqs, rows)
        if c["type"] != "i8":
            return [s["q_out"], s["k"], s["v"]]
    ld = c["Hkv"] * c["hd"]
    serve.read(cache, seqs, s["k_read"].data_ptr(), s["v_read"].data_ptr(), ld)
    return ([s["q_out"]] if c["op"] == "append" else []) + [s["k_read"], s["v_read"]]


# ---------------------------------------------------------------- what a pass needs

def _seen(c):
    """(rows, cached tokens read, pairs of a query and a key) of a case."""
    qs, kvs = _lengths(c)
    pairs = sum(m * (k - m) + m * (m + 1) // 2 for m, k in zip(qs, kvs))
    return sum(qs), sum(k for m, k in zip(qs, kvs) if m), pairs


def work(case):
    c = case
    if c["op"] == "rules":
        words = (c["V"] + 31) // 32 if c["mask"] else 0
        return {"bytes": c["rows"] * (8 * c["V"] + 4 * words + 2 * c["hist"] + 4 * c["bias"]),
                "flops": 4 * c["rows"] * c["V"]}
    rows, held, pairs = _seen(c)
    kv_row = c["Hkv"] * (c["hd"] * BYTES[c["type"]] + (4 if c["type"] == "i8" else 0)) * 2
    q_row, f_row = 4 * c["H"] * c["hd"], 8 * c["Hkv"] * c["hd"]
    if c["op"] == "attn":
        return {"bytes": 2 * rows * q_row + held * kv_row, "flops": 4 * pairs * c["H"] * c["hd"]}
    if c["op"] == "read":
        return {"bytes": rows * (kv_row + f_row), "flops": rows * 2 * c["Hkv"] * c["hd"]}
    b = rows * (2 * q_row + f_row + kv_row + 4 * c["rot"])
    if c["type"] == "i8":
        b += rows * (kv_row + f_row)
    return {"bytes": b, "flops": rows * (c["H"] + c["Hkv"]) * c["rot"] * 3}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rules":
        return _exact_rules(c, s)
    n, page, H, Hkv, hd = c["n"], c["page"], c["H"], c["Hkv"], c["hd"]
    q_start, kv_len = s["q_start"].tolist(), s["kv_len"].tolist()
    spans = [(q_start[i], q_start[i + 1], kv_len[i]) for i in range(n)]

    def cells(i, first, last):
        p = torch.arange(first, last, device="cuda")
        return s["pages"][i].long()[p // page], p % page

    def held(x, i, first, last):
        """Sequence i's cached rows of positions first .. last - 1, [positions, Hkv, hd]."""
        pg, at = cells(i, first, last)
        t = s[x].double()[pg, :, at] if s[x].numel() < 2 ** 27 else torch.stack(
            [s[x][pg, h, at].double() for h in range(Hkv)], 1)
        if c["type"] == "i8":
            t = t * s[x + "_scale"].double()[pg, :, at][..., None]
        return t

    if c["op"] == "read":
        out = [torch.zeros((s["rows"], Hkv * hd), dtype=torch.float64, device="cuda") for _ in "kv"]
        for o, x in zip(out, "kv"):
            for i, (a, b, t) in enumerate(spans):
                o[a:b] = held(x, i, t - (b - a), t).flatten(1)
        return out
    if c["op"] == "append":
        return _exact_append(c, s, spans, cells)
    out = torch.zeros((s["rows"], H, hd), dtype=torch.float64, device="cuda")
    for i, (a, b, t) in enumerate(spans):
        if a == b:
            continue
        k, v = held("k", i, 0, t), held("v", i, 0, t)
        pos = torch.arange(t - (b - a), t, device="cuda")
        hidden = torch.arange(t, device="cuda")[None, :] > pos[:, None]
        for h in range(H):
            z = s["q"][a:b, h * hd:(h + 1) * hd].double() @ k[:, h // (H // Hkv)].T.contiguous() / math.sqrt(hd)
            w = torch.softmax(z.masked_fill_(hidden, -math.inf), -1)
            out[a:b, h] = w @ v[:, h // (H // Hkv)].contiguous()
    return out.reshape(s["rows"], -1)


def _exact_append(c, s, spans, cells):
    """The rotation by complex numbers in 64 bits; what a cache holds is a number of fp32 (the definition's), in 8 bits
    the nearest of 255 steps of a scale that is itself one of fp32, each quotient rounded to fp32."""
    H, Hkv, hd, r = c["H"], c["Hkv"], c["hd"], c["rot"]
    pos = torch.cat([torch.arange(t - (b - a), t, device="cuda") for a, b, t in spans])
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None, :]
    x = s["qkv"].double().reshape(s["rows"], H + 2 * Hkv, hd).clone()
    front = x[:, :H + Hkv, :r]
    two = front.reshape(*front.shape[:2], 2, r // 2).transpose(-1, -2) if c["half"] else front.reshape(
        *front.shape[:2], r // 2, 2)
    turned = torch.view_as_real(torch.view_as_complex(two.contiguous()) * turn)
    x[:, :H + Hkv, :r] = (turned.transpose(-1, -2) if c["half"] else turned).reshape(front.shape)
    q = x[:, :H].reshape(s["rows"], -1)
    kept = []
    for name, y in (("k", x[:, H:H + Hkv]), ("v", x[:, H + Hkv:])):
        if c["type"] == "i8":
            y = y.float().double()
            scale = (y.abs().amax(-1, keepdim=True) / 127.0).float().double().clamp(TINY, BIG)
            kept.append((torch.round((y / scale).float().double()) * scale).reshape(s["rows"], -1))
        else:
            pool = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
            for i, (a, b, t) in enumerate(spans):
                pg, at = cells(i, t - (b - a), t)
                pool[pg, :, at] = y[a:b]
            kept.append(pool)
    return [q] + kept


def _exact_rules(c, s):
    rows, V = c["rows"], c["V"]
    x = s["logits"][:, :V].double()
    host = {k: s[k].cpu() for k in ("history", "hist_len", "gen_start", "bias_ids", "n_bias") if k in s}
    for i in range(rows):
        if c["hist"]:
            L, g = int(host["hist_len"][i]), int(host["gen_start"][i])
            ids = torch.unique(host["history"][i, :L].long()).cuda()
            r = float(s["repetition"][i])
            z = x[i, ids]
            x[i, ids] = torch.where(z > 0, z / r, z * r)
            ids, times = torch.unique(host["history"][i, min(g, L):L].long(), return_counts=True)
            x[i, ids.cuda()] -= float(s["frequency"][i]) * times.double().cuda() + float(s["presence"][i])
        if c["bias"]:
            last = {int(t): j for j, t in enumerate(host["bias_ids"][i, :int(host["n_bias"][i])].tolist())}
            for t, j in last.items():
                x[i, t] += s["bias"][i, j].double()
    if c["mask"]:
        bits = s["mask"].cpu().numpy().view("u1")          # little-endian words: bit t of the row is token t
        import numpy as np
        open_ = torch.from_numpy(np.unpackbits(bits, axis=1, bitorder="little")[:, :V].astype(bool)).cuda()
        x = torch.where(open_, x, torch.full_like(x, -math.inf))
    return x
