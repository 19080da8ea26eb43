"""Attention of a text encoder's prompts and of the tokens that follow them over
an 8-bit key/value cache, as cases that can be timed and compared.

Three kinds of case:

  seqs    attention within packed sequences (documents): shared key heads, causal
          or not, a prefix that everyone sees, scores capped by a tanh, a bias
          that falls with the distance;
  fill    new tokens written to the cache (8 bits, one scale for each page of 64
          tokens, head and K or V), and the pages they touched read back;
  cached  new tokens' attention over the cache: one token, a few, or a chunk.

The cache is a byte pool: for each page and head the 64 x hd bytes of K, then of
V (values q + 128, in the order of _k_values and _v_values), and behind all pages
one fp32 scale (a power of two) for each page, head and K or V.
"""
import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64
DTYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}


def listed():
    return [
        # a one-line prompt through a text encoder layer, fp32 as the linears leave it: the smallest call
        {"name": "prompt_37", "kind": "seqs", "type": "F32", "heads": 64, "kv": 8, "hd": 128, "seqs": 1, "lo": 37, "hi": 37,
         "mix": 0, "causal": True, "cap": 0.0, "alibi": False, "prefix": 0.0, "tail": 0, "fused": False},
        # the longest prompt the text encoder is given, q, k and v in one buffer
        {"name": "prompt_600", "kind": "seqs", "type": "F32", "heads": 64, "kv": 8, "hd": 128, "seqs": 1, "lo": 600, "hi": 600,
         "mix": 0, "causal": True, "cap": 0.0, "alibi": False, "prefix": 0.0, "tail": 0, "fused": True},
        # a batch of documents of very different lengths packed behind each other, capped scores
        {"name": "packed_documents", "kind": "seqs", "type": "BF16", "heads": 40, "kv": 8, "hd": 128, "seqs": 24, "lo": 17,
         "hi": 1500, "mix": 3, "causal": True, "cap": 50.0, "alibi": False, "prefix": 0.0, "tail": 5, "fused": False},
        # instructions seen from everywhere before a text with distance bias, narrow heads of their own keys
        {"name": "prefix_distance", "kind": "seqs", "type": "F16", "heads": 16, "kv": 16, "hd": 64, "seqs": 3, "lo": 1021,
         "hi": 2047, "mix": 5, "causal": True, "cap": 0.0, "alibi": True, "prefix": 0.25, "tail": 0, "fused": True},
        # one long document: the largest product
        {"name": "long_document", "kind": "seqs", "type": "BF16", "heads": 64, "kv": 8, "hd": 128, "seqs": 1, "lo": 8192,
         "hi": 8192, "mix": 0, "causal": True, "cap": 0.0, "alibi": False, "prefix": 0.0, "tail": 0, "fused": False},
        # a batch of prompts written to an empty cache
        {"name": "fill_prompts", "kind": "fill", "type": "F32", "kv": 8, "hd": 128, "seqs": 16, "lo": 100, "hi": 600, "mix": 1,
         "held_lo": 0, "held_hi": 0},
        # one token of each of many sequences, behind what the cache holds
        {"name": "append_tokens", "kind": "fill", "type": "BF16", "kv": 8, "hd": 128, "seqs": 64, "lo": 1, "hi": 1, "mix": 2,
         "held_lo": 100, "held_hi": 4000},
        # the next token of one short conversation: latency
        {"name": "token_alone", "kind": "cached", "type": "F32", "heads": 64, "kv": 8, "hd": 128, "seqs": 1, "lo": 300, "hi": 300,
         "new_lo": 1, "new_hi": 1, "mix": 0, "cap": 0.0, "alibi": False},
        # the next token of a batch of conversations of different lengths
        {"name": "token_batch", "kind": "cached", "type": "BF16", "heads": 64, "kv": 8, "hd": 128, "seqs": 32, "lo": 200,
         "hi": 8192, "new_lo": 1, "new_hi": 1, "mix": 4, "cap": 0.0, "alibi": False},
        # the next token behind two whole books
        {"name": "token_far", "kind": "cached", "type": "F16", "heads": 40, "kv": 8, "hd": 128, "seqs": 2, "lo": 120011,
         "hi": 131071, "new_lo": 1, "new_hi": 1, "mix": 6, "cap": 0.0, "alibi": True},
        # a few proposed tokens checked at once, capped scores, narrow heads
        {"name": "few_tokens", "kind": "cached", "type": "F32", "heads": 16, "kv": 4, "hd": 64, "seqs": 24, "lo": 500, "hi": 5000,
         "new_lo": 2, "new_hi": 6, "mix": 7, "cap": 30.0, "alibi": False},
        # the next chunk of long prompts over what the cache holds of them
        {"name": "chunk", "kind": "cached", "type": "BF16", "heads": 64, "kv": 8, "hd": 128, "seqs": 2, "lo": 12000, "hi": 16500,
         "new_lo": 500, "new_hi": 512, "mix": 8, "cap": 0.0, "alibi": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["seqs"] * 5 + ["fill"] * 2 + ["cached"] * 5)
    qt = rng.choice(["F32", "F16", "BF16"])
    hd = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8]) if rng.random() < 0.8 else kv
    mix = rng.randint(0, 10 ** 6)
    if kind == "seqs":
        seqs = _log_int(rng, 1, 40)
        hi = _log_int(rng, 1, 8000 // seqs)
        return {"kind": kind, "type": qt, "heads": heads, "kv": kv, "hd": hd, "seqs": seqs, "lo": max(1, hi // rng.choice([1, 3, 20])),
                "hi": hi, "mix": mix, "causal": rng.random() < 0.8, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "alibi": rng.random() < 0.3,
                "prefix": rng.choice([0.0, 0.0, 0.2, 0.6]), "tail": rng.choice([0, 0, 3]), "fused": rng.random() < 0.5}
    if kind == "fill":
        seqs = _log_int(rng, 1, 100)
        hi = _log_int(rng, 1, 16000 // seqs)
        held = rng.choice([0, _log_int(rng, 1, 3000)])
        return {"kind": kind, "type": qt, "kv": kv, "hd": hd, "seqs": seqs, "lo": max(1, hi // 4), "hi": hi, "mix": mix,
                "held_lo": held // 3, "held_hi": held}
    form = rng.choice(["token", "token", "few", "chunk"])
    new = 1 if form == "token" else rng.randint(2, 9) if form == "few" else _log_int(rng, 10, 600)
    seqs = _log_int(rng, 1, 48 if form != "chunk" else 4)
    hi = max(new, _log_int(rng, 1, (400000 if form != "chunk" else 40000) // seqs))
    return {"kind": kind, "type": qt, "heads": heads, "kv": kv, "hd": hd, "seqs": seqs, "lo": max(new, hi // rng.choice([1, 4, 30])), "hi": hi,
            "new_lo": max(1, new // 2) if form != "token" else 1, "new_hi": new, "mix": mix,
            "cap": rng.choice([0.0, 0.0, 30.0]), "alibi": rng.random() < 0.3}


# ---------------------------------------------------------------------------
# Shapes of a case: what a scheduler knows on the host
# ---------------------------------------------------------------------------
def _spread(rng, n, lo, hi):
    return [_log_int(rng, lo, hi) if 0 < lo < hi else rng.randint(lo, hi) for _ in range(n)]


def _shape(case):
    """New tokens and tokens held (the new ones among them) of each sequence."""
    rng = random.Random(case["mix"])
    if case["kind"] == "cached":
        new = _spread(rng, case["seqs"], case["new_lo"], case["new_hi"])
        return new, [max(a, b) for a, b in zip(new, _spread(rng, case["seqs"], case["lo"], case["hi"]))]
    new = _spread(rng, case["seqs"], case["lo"], case["hi"])
    if case["kind"] == "seqs":
        return new, new
    return new, [a + b for a, b in zip(new, _spread(rng, case["seqs"], case["held_lo"], case["held_hi"]))]


def _offsets(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _prefixes(case, new):
    return [int(n * case["prefix"]) for n in new] if case["prefix"] else None


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rows(g, n, heads, hd, dtype, kind):
    """q, k or v rows [n][heads * hd] as a layer's projections give them: keys with a few strong channels and an offset in some,
    queries that make scores of a few units."""
    x = torch.randn(n, heads, hd, generator=g, device=DEV)
    if kind == "k":
        x[..., ::32] *= 3.0
        x[..., 5::32] += 1.5
    if kind == "q":
        x *= 1.5
    return x.reshape(n, heads * hd).to(dtype)


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device=DEV)


def _pow2(e):
    """2^e as fp32, exactly (e from -126 to 127)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The smallest e >= -100 with amax <= 127 * 2^e."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, torch.where(m <= 127.0 / 128.0, x - 7, x - 6).clamp(min=-100), torch.full_like(x, -100))


def _pool_parts(pool, pages, kv, hd):
    """The pool's bytes [pages][kv][2][64 hd] and scales [pages][kv][2], in place."""
    n = pages * kv * 2 * PAGE * hd
    return pool[:n].view(pages, kv, 2, PAGE * hd), pool[n:].view(torch.float32).view(pages, kv, 2)


def _k_values(raw, hd):
    """Bytes [..., 64 hd] of K -> [..., 64, hd]: token 16 t + i, channel 64 c + 16 g + b."""
    n = raw.dim() - 1
    x = raw.reshape(*raw.shape[:-1], 4, hd // 64, 4, 16, 16)  # t, c, g, i, b
    return x.permute(*range(n), n, n + 3, n + 1, n + 2, n + 4).reshape(*raw.shape[:-1], PAGE, hd)


def _k_bytes(x, hd):
    n = x.dim() - 2
    y = x.reshape(*x.shape[:-2], 4, 16, hd // 64, 4, 16)  # t, i, c, g, b
    return y.permute(*range(n), n, n + 2, n + 3, n + 1, n + 4).reshape(*x.shape[:-2], PAGE * hd)


def _v_values(raw, hd):
    """Bytes [..., 64 hd] of V -> [..., 64, hd]: token 16 t + 4 g + r, channel 16 c + i."""
    n = raw.dim() - 1
    x = raw.reshape(*raw.shape[:-1], hd // 16, 4, 16, 4, 4)  # c, g, i, t, r
    return x.permute(*range(n), n + 3, n + 1, n + 4, n, n + 2).reshape(*raw.shape[:-1], PAGE, hd)


def _v_bytes(x, hd):
    n = x.dim() - 2
    y = x.reshape(*x.shape[:-2], 4, 4, 4, hd // 16, 16)  # t, g, r, c, i
    return y.permute(*range(n), n + 3, n + 1, n + 4, n, n + 2).reshape(*x.shape[:-2], PAGE * hd)


def _filled_pool(g, pages, kv, hd):
    """A pool whose pages are full of quantised keys and values."""
    pool = torch.empty(pages * kv * 2 * (PAGE * hd + 4), dtype=torch.uint8, device=DEV)
    raw, scale = _pool_parts(pool, pages, kv, hd)
    step = max(1, (1 << 26) // (PAGE * kv * hd))  # bounded scratch
    for p in range(0, pages, step):
        n = min(step, pages - p)
        for which, to_bytes in ((0, _k_bytes), (1, _v_bytes)):
            x = _rows(g, n * PAGE, kv, hd, torch.float32, "kv"[which]).reshape(n, PAGE, kv, hd).transpose(1, 2)
            s = _pow2(_exponent(x.abs().amax((-2, -1))))
            scale[p:p + n, :, which] = s
            raw[p:p + n, :, which] = to_bytes(((x / s[..., None, None]).round() + 128).to(torch.uint8), hd)
    return pool


def _inputs(case, seed):
    g = _gen(seed)
    new, held = _shape(case)
    first, dt, kv, hd = _offsets(new), DTYPES[case["type"]], case["kv"], case["hd"]
    s = {"case": case, "new": new, "held": held, "n": first[-1], "first": _int32(first), "rows": first[-1]}
    if case["kind"] != "seqs":  # pages of the sequences, in no order, in a pool with a few more
        need = [-(-h // PAGE) for h in held]
        s["max_pages"], s["pages"] = max(need), sum(need) + 3
        order = torch.randperm(s["pages"], generator=g, device=DEV).to(torch.int32)
        s["table"] = torch.zeros(len(need), s["max_pages"], dtype=torch.int32, device=DEV)
        for i, (a, n) in enumerate(zip(_offsets(need), need)):
            s["table"][i, :n] = order[a:a + n]
        s["pool"] = _filled_pool(g, s["pages"], kv, hd)
        s["len"] = _int32(held)
    if case["kind"] == "fill":
        s["k"], s["v"] = (_rows(g, s["n"], kv, hd, dt, c) for c in "kv")
        back = [h - (h - n) // PAGE * PAGE for n, h in zip(new, held)]  # the touched pages' tokens
        s["back"], s["back_first"] = sum(back), _int32(_offsets(back))
        s["ko"], s["vo"] = (torch.empty(s["back"], kv * hd, dtype=dt, device=DEV) for _ in "kv")
        return s
    heads = case["heads"]
    if case["alibi"]:
        s["slopes"] = _slopes(heads)
    if case["kind"] == "seqs":
        s["rows"] = s["n"] + case["tail"]  # rows behind the last sequence stay as they are
        if case["fused"]:
            qkv = torch.cat([_rows(g, s["rows"], h, hd, dt, c) for h, c in ((heads, "q"), (kv, "k"), (kv, "v"))], 1)
            s["qkv"] = qkv
            s["q"], s["k"], s["v"] = qkv.split([heads * hd, kv * hd, kv * hd], 1)
        else:
            s["q"], s["k"], s["v"] = (_rows(g, s["rows"], h, hd, dt, c) for h, c in ((heads, "q"), (kv, "k"), (kv, "v")))
        pre = _prefixes(case, new)
        if pre:
            s["prefix"] = _int32(pre)
    else:
        s["q"] = _rows(g, s["n"], heads, hd, dt, "q")
    s["o"] = torch.full((s["rows"], heads * hd), 0.25, dtype=dt, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    new, held = s["new"], s["held"]
    # which sequence and which token of it each row is (the plain form's index lists)
    s["row_seq"] = torch.repeat_interleave(torch.arange(len(new), device=DEV), s["first"].diff().long())
    s["row_at"] = torch.arange(s["n"], device=DEV) - s["first"].long()[s["row_seq"]]
    if case["kind"] == "fill":
        touched = [(i, p) for i, (n, h) in enumerate(zip(new, held)) for p in range((h - n) // PAGE, -(-h // PAGE))]
        s["touched"] = torch.tensor(touched, dtype=torch.int64, device=DEV)
        seqs = torch.repeat_interleave(torch.arange(len(new), device=DEV), s["back_first"].diff().long())
        at = torch.arange(s["back"], device=DEV) - s["back_first"].long()[seqs]
        pages = _offsets([-(-h // PAGE) - (h - n) // PAGE for n, h in zip(new, held)])
        s["back_page"], s["back_slot"] = torch.tensor(pages, device=DEV)[seqs] + at // PAGE, at % PAGE  # page: of the touched ones
    if own:
        s["call"] = _handles(s)
    return s


# ---------------------------------------------------------------------------
# One pass: the framework's calls
# ---------------------------------------------------------------------------
def _handles(s):
    """What a program keeps between calls: the settings, the cache's description, the workspace."""
    from fasth3inc_amd import fh3 as F
    F.init(0)
    c = s["case"]
    h = {"F": F, "type": {"F32": F.FH3_QUANT_F32, "F16": F.FH3_QUANT_F16, "BF16": F.FH3_QUANT_BF16}[c["type"]]}
    if c["kind"] != "fill":
        h["cfg"] = F.attn_cfg(c["heads"], c["kv"], c["hd"], h["type"], causal=c.get("causal", True), softcap=c["cap"],
                              d_slopes=_at(s, "slopes"))
    if c["kind"] != "seqs":
        assert s["pool"].numel() == F.kv_pool_bytes(c["kv"], c["hd"], s["pages"])
        h["kv"] = F.kv_cache(c["kv"], c["hd"], s["pages"], s["max_pages"], _at(s, "pool"), _at(s, "table"), _at(s, "len"))
    if c["kind"] == "cached":
        h["bytes"] = F.kv_attention_workspace_bytes(h["cfg"], h["kv"], s["n"], len(s["new"]))
        h["ws"] = torch.empty(max(1, h["bytes"]), dtype=torch.uint8, device=DEV)
    return h


def _at(s, name):
    return s[name].data_ptr() if name in s else None


def _run_own(s):
    c, h = s["case"], s["call"]
    F, n_seq = h["F"], len(s["new"])
    if c["kind"] == "seqs":
        F.attention_seqs_dev(h["cfg"], _at(s, "q"), _at(s, "k"), _at(s, "v"), _at(s, "o"), s["rows"], n_seq, _at(s, "first"),
                             _at(s, "prefix"), ldq=s["q"].stride(0), ldk=s["k"].stride(0), ldv=s["v"].stride(0))
        return s["o"]
    if c["kind"] == "fill":
        F.kv_append_dev(h["kv"], h["type"], _at(s, "k"), _at(s, "v"), s["n"], n_seq, _at(s, "first"))
        F.kv_read_dev(h["kv"], h["type"], _at(s, "ko"), _at(s, "vo"), s["back"], n_seq, _at(s, "back_first"))
        return {"k": s["ko"], "v": s["vo"]}
    F.kv_attention_dev(h["cfg"], h["kv"], _at(s, "q"), _at(s, "o"), s["n"], n_seq, h["ws"].data_ptr(), h["bytes"], _at(s, "first"))
    return s["o"]


# ---------------------------------------------------------------------------
# One pass: the plain form
# ---------------------------------------------------------------------------
def _weigh(score, dist, seen, c, slopes):
    """Weights of scores [..., kv, group, i, j] (unscaled), seen and dist [..., 1, 1, i, j]: softmax over what is seen, zeros for none."""
    score = score * (1.0 / math.sqrt(c["hd"]))
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    if c["alibi"]:
        score = score - slopes.view(c["kv"], -1, 1, 1) * dist.abs()
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    return w / torch.where(total == 0, torch.ones_like(total), total)


def _plain_seqs(s):
    c, n = s["case"], s["n"]
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    q = s["q"][:n].float().reshape(n, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
    k = s["k"][:n].float().reshape(n, kv, hd).permute(1, 2, 0).contiguous()
    v = s["v"][:n].float().reshape(n, kv, hd).permute(1, 0, 2).contiguous()
    dist = s["row_at"][:, None] - s["row_at"][None, :]
    seen = s["row_seq"][:, None] == s["row_seq"][None, :]
    if c["causal"]:
        open_to = dist >= 0
        if "prefix" in s:
            open_to = open_to | (s["row_at"] < s["prefix"].long()[s["row_seq"]])[None, :]
        seen = seen & open_to
    w = _weigh(torch.matmul(q, k).reshape(kv, -1, n, n), dist.float(), seen, c, s.get("slopes"))
    o = torch.matmul(w.reshape(kv, -1, n), v).reshape(kv, -1, n, hd).permute(2, 0, 1, 3).reshape(n, heads * hd)
    return torch.cat([o.to(s["o"].dtype), s["o"][n:]])


def _plain_fill(s):
    c = s["case"]
    kv, hd = c["kv"], c["hd"]
    raw, scale = _pool_parts(s["pool"], s["pages"], kv, hd)
    seq, page = s["touched"][:, 0], s["touched"][:, 1]
    ids, length = s["table"].long()[seq, page], s["len"].long()[seq, None]
    begin = length - s["first"].diff().long()[seq, None]
    slot = page[:, None] * PAGE + torch.arange(PAGE, device=DEV)
    fresh, held = ((slot >= begin) & (slot < length))[:, None, :, None], (slot < begin)[:, None, :, None]
    row = (s["first"].long()[seq, None] + slot - begin).clamp(0, s["n"] - 1)
    out = []
    for which, (x, values, to_bytes) in enumerate(((s["k"], _k_values, _k_bytes), (s["v"], _v_values, _v_bytes))):
        x = x.float().reshape(-1, kv, hd)[row].transpose(1, 2)
        fine = torch.where(fresh & torch.isfinite(x), x.abs(), torch.zeros_like(x))
        need = _pow2(_exponent(fine.amax((-2, -1))))
        before = scale[ids, :, which]
        after = torch.where(held.any(2)[..., 0], torch.maximum(before, need), need)
        old = values(raw[ids, :, which], hd).float() - 128
        old = torch.where(held, (old * (before / after)[..., None, None]).round(), old)
        put = torch.nan_to_num(x / after[..., None, None], nan=0.0).round().clamp(-127, 127)
        now = torch.where(fresh, put, old)
        raw[ids, :, which] = to_bytes((now + 128).to(torch.uint8), hd)
        scale[ids, :, which] = after
        got = (now * after[..., None, None])[s["back_page"], :, s["back_slot"]]
        out.append(got.reshape(-1, kv * hd).to(DTYPES[c["type"]]))
    return {"k": out[0], "v": out[1]}


def _plain_cached(s):
    c, n_seq = s["case"], len(s["new"])
    heads, kv, hd, most = c["heads"], c["kv"], c["hd"], max(s["new"])
    raw, scale = _pool_parts(s["pool"], s["pages"], kv, hd)
    ids = s["table"].long()
    got = []
    for which, values in ((0, _k_values), (1, _v_values)):
        x = (values(raw[ids][:, :, :, which], hd).float() - 128) * scale[ids][:, :, :, which, None, None]
        got.append(x.transpose(1, 2).reshape(n_seq, kv, -1, hd))
    at = torch.arange(most, device=DEV)
    count = s["first"].diff().long()
    row = (s["first"].long()[:-1, None] + at).clamp(max=s["n"] - 1)
    q = s["q"].float().reshape(-1, kv, heads // kv, hd)[row].permute(0, 2, 3, 1, 4).reshape(n_seq, kv, -1, hd)
    keys = torch.arange(got[0].shape[2], device=DEV)
    dist = (s["len"].long() - count)[:, None, None] + at[None, :, None] - keys
    seen = ((dist >= 0) & (keys < s["len"][:, None, None]))[:, None, None]
    score = torch.matmul(q, got[0].transpose(-1, -2).contiguous()).reshape(n_seq, kv, -1, most, keys.numel())
    w = _weigh(score, dist.float()[:, None, None], seen, c, s.get("slopes"))
    o = torch.matmul(w.reshape(n_seq, kv, -1, keys.numel()), got[1]).reshape(n_seq, kv, -1, most, hd)
    return o.permute(0, 3, 1, 2, 4)[s["row_seq"], s["row_at"]].reshape(-1, heads * hd).to(s["o"].dtype)


def run(s):
    if own:
        return _run_own(s)
    return {"seqs": _plain_seqs, "fill": _plain_fill, "cached": _plain_cached}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(case, new, held):
    """Query-key pairs that are computed, of one head."""
    if case["kind"] == "cached":
        return sum(n * (h - n) + n * (n + 1) // 2 for n, h in zip(new, held))
    if not case["causal"]:
        return sum(n * n for n in new)
    pre = _prefixes(case, new) or [0] * len(new)
    return sum(n * (n + 1) // 2 + p * (p - 1) // 2 for n, p in zip(new, pre))


def work(case):
    new, held = _shape(case)
    size, n, kv, hd = DTYPES[case["type"]].itemsize, sum(new), case["kv"], case["hd"]
    if case["kind"] == "fill":
        back = sum(h - (h - a) // PAGE * PAGE for a, h in zip(new, held))
        return {"bytes": 2 * kv * hd * (n * (size + 1) + back * (size + 1)), "flops": 0}
    rows = 2 * size * n * case["heads"] * hd  # q and o
    rows += 2 * kv * hd * (size * n if case["kind"] == "seqs" else sum(held))
    return {"bytes": rows, "flops": 4 * case["heads"] * hd * _pairs(case, new, held)}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definition, sequence by sequence and head by head
# ---------------------------------------------------------------------------
def _exact_head(q, k, v, pos, c, slope, prefix, causal):
    """One head's outputs for queries at positions pos over keys 0 .. len(k) - 1."""
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=DEV)
    j = torch.arange(k.shape[0], device=DEV)
    step = max(1, (1 << 26) // max(1, k.shape[0]))
    for r in range(0, q.shape[0], step):
        i = pos[r:r + step, None]
        a = (q[r:r + step] @ k.t().contiguous()) / math.sqrt(c["hd"])
        if c["cap"]:
            a = torch.tanh(a / c["cap"]) * c["cap"]
        if slope is not None:
            a = a - float(slope) * (i - j).abs().double()
        if causal:
            a[(j > i) & (j >= prefix)] = -math.inf
        out[r:r + step] = torch.softmax(a, -1) @ v
    return out


def _exact_seqs(case, s):
    kv, hd, group = case["kv"], case["hd"], case["heads"] // case["kv"]
    out = s["o"].double()
    pre = _prefixes(case, s["new"]) or [0] * len(s["new"])
    for i, (a, n) in enumerate(zip(_offsets(s["new"]), s["new"])):
        for h in range(case["heads"]):
            m = h // group
            q, k, v = (s[x][a:a + n, y * hd:(y + 1) * hd].double() for x, y in (("q", h), ("k", m), ("v", m)))
            slope = s["slopes"][h] if case["alibi"] else None
            out[a:a + n, h * hd:(h + 1) * hd] = _exact_head(q, k, v, torch.arange(n, device=DEV), case, slope, pre[i], case["causal"])
    return out


def _byte_at(which, token, channel, hd):
    """Where in its 64 hd bytes a value stands."""
    if which == 0:
        return (((token // 16 * (hd // 64) + channel // 64) * 4 + channel % 64 // 16) * 16 + token % 16) * 16 + channel % 16
    return ((channel // 16 * 4 + token % 16 // 4) * 16 + channel % 16) * 16 + token // 16 * 4 + token % 4


def _exact_values(case, s, seq, which, begin, end):
    """Cached values of tokens begin .. end - 1 of a sequence, [tokens][kv][hd], as 64-bit numbers (integers and scales)."""
    kv, hd = case["kv"], case["hd"]
    t, d = torch.arange(begin, end, device=DEV), torch.arange(hd, device=DEV)
    base = s["table"][seq].long()[t // PAGE][:, None] * kv + torch.arange(kv, device=DEV)
    at = (base[..., None] * 2 + which) * (PAGE * hd) + _byte_at(which, (t % PAGE)[:, None, None], d, hd)
    scales = s["pool"][s["pages"] * kv * 2 * PAGE * hd:].view(torch.float32)
    return s["pool"][at].double() - 128, scales[base * 2 + which].double()


def _exact_cached(case, s):
    kv, hd, group = case["kv"], case["hd"], case["heads"] // case["kv"]
    out = torch.empty(s["n"], case["heads"] * hd, dtype=torch.float64, device=DEV)
    for i, (a, n, held) in enumerate(zip(_offsets(s["new"]), s["new"], s["held"])):
        (k, ks), (v, vs) = (_exact_values(case, s, i, w, 0, held) for w in (0, 1))
        k, v = k * ks[..., None], v * vs[..., None]
        pos = held - n + torch.arange(n, device=DEV)
        for h in range(case["heads"]):
            q = s["q"][a:a + n, h * hd:(h + 1) * hd].double()
            slope = s["slopes"][h] if case["alibi"] else None
            out[a:a + n, h * hd:(h + 1) * hd] = _exact_head(q, k[:, h // group], v[:, h // group], pos, case, slope, 0, True)
    return out


def _two_to(e):
    """2^e as a 64-bit number, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_fill(case, s):
    kv, hd = case["kv"], case["hd"]
    out = {"k": [], "v": []}
    for i, (a, n, held) in enumerate(zip(_offsets(s["new"]), s["new"], s["held"])):
        begin = held - n
        for which, name in ((0, "k"), (1, "v")):
            x = s[name][a:a + n].double().reshape(n, kv, hd)
            for p in range(begin // PAGE, -(-held // PAGE)):
                lo, hi = max(begin, p * PAGE), min(held, (p + 1) * PAGE)
                part = x[lo - begin:hi - begin]
                top = part.abs().amax((0, 2))
                e = torch.ceil(torch.log2(top / 127)).clamp(min=-100)
                e = torch.where(top > 127 * _two_to(e), e + 1, torch.where(top <= 127 * _two_to(e - 1), e - 1, e))
                unit = _two_to(e.clamp(min=-100))
                if lo > p * PAGE:
                    q, before = _exact_values(case, s, i, which, p * PAGE, lo)
                    unit = torch.maximum(unit, before[0])
                    out[name].append(torch.round(q * (before / unit)[..., None]) * unit[:, None])
                out[name].append(torch.round(part / unit[:, None]) * unit[:, None])
    return {name: torch.cat(parts).reshape(-1, kv * hd) for name, parts in out.items()}


def exact(case, seed):
    new, held = _shape(case)
    if case["kind"] == "fill":
        return _exact_fill(case, _inputs(case, seed)) if sum(new) < 40000 else None
    if case["heads"] * _pairs(case, new, held) > 5e9 or case["heads"] * len(new) > 4000:
        return None
    return (_exact_seqs if case["kind"] == "seqs" else _exact_cached)(case, _inputs(case, seed))
