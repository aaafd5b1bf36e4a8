"""Measured cases of the operators that verify a tree of drafted tokens.

A verification step of speculative decoding takes up to 64 drafted tokens per
sequence through these operators, in this order:

* rope      -- rotary positions on q heads and KV rows (interleaved or half
               layout, part of the head, YaRN-scaled frequencies) and the
               inverse rotation of the attention's output;
* kv_write  -- the tokens' latent KV rows rotated, quantised and written into
               a paged cache; kv_read -- rows of the cache read back;
* tree_attn -- every drafted token attends to its sequence's cached context
               and to its own ancestors in the tree;
* logits    -- repetition, frequency and presence penalties, token biases and
               a grammar mask on the head's logits, and the greedy token.

A cache row is d - tail e4m3 codes, `tail` f16 values and one power-of-two
scale (an E8M0 byte): element = code * scale. The scale is the smallest power
of two that brings the row's largest magnitude to 448 or below.

`run` computes the plain form in torch, or with `own` set calls the framework.
"""
import math
import os
import sys

import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"


def _framework():
    path = os.path.join(REPO, "deepseek-v4-in-c_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dsv4_b200
    return dsv4_b200


def listed():
    return [
        # the query of one decoded token: 64 heads of 512, the last 64 rotated
        dict(name="rope-1", op="rope", tokens=1, heads=64, width=512, rd=64, first=448, layout="interleaved",
             inverse=False, scaled=False, src="f32", dst="bf16"),
        # de-rotation of the attention outputs of a 32-token tree
        dict(name="rope-inv-32", op="rope", tokens=32, heads=64, width=512, rd=64, first=448, layout="interleaved",
             inverse=True, scaled=True, src="bf16", dst="f32"),
        # queries of a long prompt, half layout, a rotated part in front
        dict(name="rope-2048", op="rope", tokens=2048, heads=64, width=512, rd=128, first=0, layout="half",
             inverse=False, scaled=True, src="f32", dst="bf16"),
        # the drafted tokens' rows of 4 sequences rotated, quantised and cached in one call
        dict(name="write-64", op="kv_write", n=64, d=512, tail=64, page=64, src="f32", rope=True),
        # a long prompt's rows into the cache, with padding rows that are skipped
        dict(name="write-16000", op="kv_write", n=16000, d=576, tail=64, page=64, src="bf16", rope=False),
        # a cached context gathered back, as for a copy to another host
        dict(name="read-16384", op="kv_read", n=16384, d=512, tail=64, page=64, dst="bf16"),
        # one decoded token over a short context
        dict(name="attn-1x700", op="tree_attn", batch=1, tokens=1, heads=64, d=512, tail=64, page=64, ctx=700,
             ragged=False, dtype="bf16"),
        # a batch of ragged sequences, 7 drafted tokens each
        dict(name="attn-8x7x4100", op="tree_attn", batch=8, tokens=7, heads=64, d=512, tail=64, page=64, ctx=4100,
             ragged=True, dtype="bf16"),
        # decode of 8 sequences over 32768 positions of 512 + 64 elements
        dict(name="attn-8x1x32768", op="tree_attn", batch=8, tokens=1, heads=64, d=576, tail=64, page=64, ctx=32768,
             ragged=False, dtype="f16"),
        # a 16-token tree per sequence over long contexts
        dict(name="attn-4x16x32768", op="tree_attn", batch=4, tokens=16, heads=64, d=512, tail=64, page=64,
             ctx=32768, ragged=False, dtype="bf16"),
        # one token's logits under a grammar with a short history
        dict(name="logits-1", op="logits", rows=1, vocab=129280, hist=600, bias=16, mask=True, dtype="f32"),
        # the logits of 64 rows, long histories
        dict(name="logits-64", op="logits", rows=64, vocab=129280, hist=8192, bias=300, mask=True, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


SHAPES = [(512, 64), (576, 64), (320, 64), (256, 0), (448, 128), (64, 0), (128, 64)]


def draw(rng):
    op = rng.choice(["rope", "kv_write", "kv_read", "tree_attn", "tree_attn", "logits"])
    if op == "rope":
        width = rng.choice([64, 128, 192, 320, 512, 576, 2 * rng.randint(16, 288)])
        rd = min(width, rng.choice([32, 64, 128, 2 * rng.randint(1, 64)]))
        return dict(op=op, tokens=_log(rng, 1, 2000), heads=rng.choice([1, 16, 64, rng.randint(1, 64)]), width=width,
                    rd=rd, first=rng.choice([0, width - rd]), layout=rng.choice(["interleaved", "half"]),
                    inverse=rng.random() < 0.5, scaled=rng.random() < 0.5, src=rng.choice(sorted(TYPES)),
                    dst=rng.choice(sorted(TYPES)))
    if op in ("kv_write", "kv_read"):
        d, tail = rng.choice(SHAPES)
        c = dict(op=op, n=_log(rng, 1, 16000), d=d, tail=tail, page=rng.choice([16, 32, 64, 128]))
        if op == "kv_read":
            return dict(c, dst=rng.choice(sorted(TYPES)))
        return dict(c, src=rng.choice(sorted(TYPES)), rope=tail > 0 and rng.random() < 0.5)
    if op == "tree_attn":
        d, tail = rng.choice(SHAPES)
        c = dict(op=op, batch=_log(rng, 1, 16), tokens=_log(rng, 1, 64), heads=rng.choice([1, 8, 16, 64, 64, 128]),
                 d=d, tail=tail, page=rng.choice([16, 32, 64, 128]), ctx=_log(rng, 1, 32768), ragged=rng.random() < 0.6,
                 dtype=rng.choice(["bf16", "f16"]))
        most = work(listed()[9])["flops"]
        full = work(dict(c, ragged=False))["flops"]
        return dict(c, ctx=max(1, int(c["ctx"] * min(1.0, 0.9 * most / full))))
    return dict(op="logits", rows=_log(rng, 1, 60), vocab=rng.choice([129280, 4096, _log(rng, 500, 129280)]),
                hist=rng.choice([0, _log(rng, 1, 8192)]), bias=rng.choice([0, _log(rng, 1, 300)]),
                mask=rng.random() < 0.7, dtype=rng.choice(sorted(TYPES)))


# ------------------------------------------------------------------ inputs

BASE, FACTOR, ORIG, FAST, SLOW = 10000.0, 16.0, 65536, 32.0, 1.0      # the model's rotary settings
FAR = 1048576                                                         # and its longest position


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _ints(g, lo, hi, shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=dtype)


def _latent(g, n, d):
    """Latent KV rows: normalised to unit RMS, a shared direction in all of them."""
    x = _normal(g, n, d) + 0.5 * _normal(g, 1, d)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def _frequencies(rd, scaled):
    """Angle per position of each pair, in double: base^(-2i/rd), under YaRN
    divided by the factor where the wavelength exceeds the trained context and
    blended over the ramp between beta_fast and beta_slow turns of it."""
    i = torch.arange(rd // 2, dtype=torch.float64)
    f = 1.0 / BASE ** (2 * i / rd)
    if scaled:
        at = [rd * math.log(ORIG / (b * 2 * math.pi)) / (2 * math.log(BASE)) for b in (FAST, SLOW)]
        lo, hi = max(0, math.floor(at[0])), min(rd - 1, math.ceil(at[1]))
        ramp = ((i - lo) / (hi - lo if hi != lo else 0.001)).clamp(0, 1)
        f = f / FACTOR * ramp + f * (1 - ramp)
    return f.to(DEV)


def _empty_cache(n_slots, page, d, tail):
    pages = -(-n_slots // page)
    return (torch.zeros((pages, page, d + tail), dtype=torch.uint8, device=DEV),
            torch.zeros((pages, page), dtype=torch.uint8, device=DEV))


def _plan(case, s):
    """What a program of the framework keeps from call to call."""
    B = _framework()
    s["B"] = B
    if case["op"] == "rope" or case.get("rope"):
        rd = case["rd"] if case["op"] == "rope" else case["tail"]
        scaled = case.get("scaled", True)
        half = case.get("layout") == "half"
        s["cfg"] = B.rope_cfg(rd, BASE, layout=B.ROPE_HALF if half else B.ROPE_INTERLEAVED,
                              factor=FACTOR if scaled else 1.0, orig=ORIG if scaled else 0, beta_fast=FAST,
                              beta_slow=SLOW)
    if "codes" in s:
        s["cache"] = B.KvCache(s["codes"], s["scales"], case["d"], case["tail"])
    if case["op"] == "tree_attn":
        s["scratch"] = torch.empty(B.tree_attn_scratch(case["heads"], case["d"], case["tokens"], case["batch"],
                                                       case["ctx"]), dtype=torch.uint8, device=DEV)
    if case["op"] == "logits":
        s["adj"] = B.LogitAdjust(hist=s["hist"], hist_len=s["hist_len"], n_prompt=s["n_prompt"], rep=s["rep"],
                                 freq=s["freq"], pres=s["pres"], bias_ids=s["bias_ids"], bias=s["bias"],
                                 bias_len=s["bias_len"], mask=s["mask"])


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "rope":
        n, h, w = case["tokens"], case["heads"], case["width"]
        s["x"] = _normal(g, n, h, w).to(TYPES[case["src"]])
        s["pos"] = _ints(g, 0, FAR, (n,))
        s["out"] = torch.zeros((n, h, w), dtype=TYPES[case["dst"]], device=DEV)
    elif op in ("kv_write", "kv_read"):
        n, d, tail, page = case["n"], case["d"], case["tail"], case["page"]
        slots = -(-(n + n // 4 + 1) // page) * page
        s["codes"], s["scales"] = _empty_cache(slots, page, d, tail)
        rows = _latent(g, n, d)
        s["slots"] = torch.randperm(slots, generator=g, device=DEV)[:n]
        s["slots"][torch.rand(n, generator=g, device=DEV) < 0.02] = -1        # padding: no row of the cache
        if op == "kv_write":
            s["rows"] = rows.to(TYPES[case["src"]])
            s["pos"] = _ints(g, 0, FAR, (n,))
        else:
            at = torch.randperm(slots, generator=g, device=DEV)
            full = _latent(g, slots, d)
            _store(s["codes"], s["scales"], full, at, tail)
            s["out"] = torch.zeros((n, d), dtype=TYPES[case["dst"]], device=DEV)
    elif op == "tree_attn":
        b, t, h, d, tail, page = (case[k] for k in ("batch", "tokens", "heads", "d", "tail", "page"))
        most = case["ctx"]
        per = -(-(most + t) // page)
        pool = b * per + 3
        s["codes"], s["scales"] = _empty_cache(pool * page, page, d, tail)
        _store(s["codes"], s["scales"], _latent(g, pool * page, d), torch.arange(pool * page, device=DEV), tail)
        s["pages"] = torch.randperm(pool, generator=g, device=DEV)[:b * per].to(torch.int32).view(b, per)
        s["ctx"] = torch.full((b,), most, dtype=torch.int32, device=DEV)
        s["n_draft"] = torch.full((b,), t, dtype=torch.int32, device=DEV)
        if case["ragged"]:
            s["ctx"] = _ints(g, 0, most + 1, (b,))
            s["n_draft"] = _ints(g, 1, t + 1, (b,))
        s["mask"] = _trees(g, b, t)
        s["q"] = (2.0 * _normal(g, b, t, h, d)).to(TYPES[case["dtype"]])
        s["sink"] = _normal(g, h)
        s["out"] = torch.zeros((b, t, h, d), dtype=TYPES[case["dtype"]], device=DEV)
        s["scale"] = d ** -0.5
    else:
        r, v = case["rows"], case["vocab"]
        s["x"] = (3.0 * _normal(g, r, v)).to(TYPES[case["dtype"]])
        # token ids of text: a few frequent ones, a long tail
        u = torch.rand((r, max(1, case["hist"])), generator=g, device=DEV)
        s["hist"] = (u.pow(6) * v).to(torch.int32).clamp_(max=v - 1)
        s["hist_len"] = _ints(g, case["hist"] // 2, case["hist"] + 1, (r,))
        s["n_prompt"] = (s["hist_len"].float() * torch.rand(r, generator=g, device=DEV)).to(torch.int32)
        s["rep"] = 1.0 + 0.3 * torch.rand(r, generator=g, device=DEV)
        s["freq"] = 0.4 * torch.rand(r, generator=g, device=DEV)
        s["pres"] = 0.6 * torch.rand(r, generator=g, device=DEV)
        s["bias_ids"] = _ints(g, 0, v, (r, max(1, case["bias"])))
        s["bias"] = 2.0 * _normal(g, r, max(1, case["bias"]))
        s["bias_len"] = torch.full((r,), case["bias"], dtype=torch.int32, device=DEV)
        s["mask"] = None
        if case["mask"]:
            words = -(-v // 32)
            # a grammar allows a few per cent of the vocabulary
            bits = [_ints(g, -2 ** 31, 2 ** 31, (r, words), torch.int64) for _ in range(4)]
            s["mask"] = (bits[0] & bits[1] & bits[2] & bits[3]).to(torch.int32)
        s["out"] = torch.zeros((r, v), dtype=TYPES[case["dtype"]], device=DEV)
        s["token"] = torch.zeros(r, dtype=torch.int32, device=DEV)
    if own:
        _plan(case, s)
    return s


def _trees(g, b, t):
    """Ancestor masks of random trees: token i's parent is an earlier token, or
    the context alone; bit j of token i's mask says that i attends to j."""
    up = (torch.rand((b, t), generator=g, device=DEV) * (torch.arange(t, device=DEV) + 1)).long() - 1
    see = torch.eye(t, dtype=torch.bool, device=DEV).expand(b, t, t)
    step = torch.zeros((b, t, t + 1), device=DEV)
    step.scatter_(2, torch.where(up < 0, t, up)[..., None], 1.0)
    step = step[..., :t]
    reach = see.float()
    for _ in range(6):                                   # 2^6 generations: any tree of 64 tokens
        reach = ((reach + reach @ step) > 0).float()
        step = ((step @ step) > 0).float()
    bit = torch.ones(t, dtype=torch.int64, device=DEV) << torch.arange(t, device=DEV)
    return (reach.long() * bit).sum(-1)


# -------------------------------------------------------------- plain forms

def _angles(pos, rd, scaled):
    th = pos.double()[:, None] * _frequencies(rd, scaled)
    return th.cos().float(), th.sin().float()


def _rotated(x, c, s, first, rd, half, inverse):
    """x [n][h][w] in 32 bits with elements first .. first + rd rotated."""
    part = x[..., first:first + rd]
    a, b = (part[..., :rd // 2], part[..., rd // 2:]) if half else (part[..., 0::2], part[..., 1::2])
    c, s = c[:, None], (-s if inverse else s)[:, None]
    re, im = a * c - b * s, a * s + b * c
    turned = torch.cat((re, im), -1) if half else torch.stack((re, im), -1).flatten(-2)
    return torch.cat((x[..., :first], turned, x[..., first + rd:]), -1)


def _store(codes, scales, rows, slots, tail):
    """Quantise 32-bit rows into the cache rows `slots` (-1: none)."""
    d = rows.shape[1]
    top = rows.abs().amax(-1)
    m, e = torch.frexp(top.double() / 448.0)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(top > 0, e, -127).clamp(-127, 127)
    y = rows * torch.pow(2.0, -e.double()).float()[:, None]
    put = slots >= 0
    at = slots[put]
    flat = codes.view(-1, d + tail)
    packed = torch.cat((y[:, :d - tail].to(torch.float8_e4m3fn).view(torch.uint8),
                        y[:, d - tail:].to(torch.float16).contiguous().view(torch.uint8)), -1)
    flat[at] = packed[put]
    scales.view(-1)[at] = (e + 127).to(torch.uint8)[put]


def _values(codes, scales, d, tail, slots):
    """The 32-bit values of cache rows."""
    raw = codes.view(-1, d + tail)[slots]
    head = raw[..., :d - tail].contiguous().view(torch.float8_e4m3fn).float()
    end = raw[..., d - tail:].contiguous().view(torch.float16).float()
    scale = torch.pow(2.0, scales.view(-1)[slots].double() - 127).float()
    return torch.cat((head, end), -1) * scale[..., None]


def _cache_out(s):
    c = s["case"]
    n = c["d"] - c["tail"]
    return {"codes": s["codes"][..., :n].view(torch.float8_e4m3fn),
            "tail": s["codes"][..., n:].view(torch.float16), "scales": s["scales"].view(torch.float8_e8m0fnu)}


def _slots_of(pages, page, count):
    j = torch.arange(count, device=pages.device)
    return pages.long()[:, j // page] * page + j % page


def _seen(s):
    """[batch][tokens][position]: what each drafted token attends to."""
    t, count = s["case"]["tokens"], s["case"]["ctx"] + s["case"]["tokens"]
    j = torch.arange(count, device=DEV)[None, None]
    ctx, nd = s["ctx"].long()[:, None, None], s["n_draft"].long()[:, None, None]
    k = (j - ctx).clamp(0, 63)
    return (j < ctx) | ((j >= ctx) & (j - ctx < nd) & (((s["mask"][..., None] >> k) & 1) == 1)
                        & (torch.arange(t, device=DEV)[None, :, None] < nd))


def _plain_attn(s):
    c = s["case"]
    b, t, h, d, tail = (c[k] for k in ("batch", "tokens", "heads", "d", "tail"))
    v = _values(s["codes"], s["scales"], d, tail, _slots_of(s["pages"], c["page"], c["ctx"] + t))
    score = (s["q"].float().view(b, t * h, d) @ v.transpose(1, 2)).mul_(s["scale"]).view(b, t, h, -1)
    score.masked_fill_(~_seen(s)[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True) + (s["sink"][:, None] - top).exp()
    o = (p.view(b, t * h, -1) @ v).view(b, t, h, d) / total
    drafted = torch.arange(t, device=DEV)[None] < s["n_draft"][:, None]
    return torch.where(drafted[..., None, None], o.to(s["out"].dtype), s["out"])


def _plain_logits(s):
    x = s["x"].float()
    r, v = x.shape
    at = torch.arange(s["hist"].shape[1], device=DEV)[None]
    some = torch.zeros((r, v), dtype=torch.int32, device=DEV)
    count = torch.zeros((r, v), dtype=torch.int32, device=DEV)
    ids = s["hist"].long()
    some.scatter_add_(1, ids, (at < s["hist_len"][:, None]).int())
    count.scatter_add_(1, ids, ((at < s["hist_len"][:, None]) & (at >= s["n_prompt"][:, None])).int())
    rep = s["rep"][:, None]
    y = torch.where(some > 0, torch.where(x > 0, x / rep, x * rep), x)
    y = y - s["freq"][:, None] * count.float()
    y = torch.where(count > 0, y - s["pres"][:, None], y)
    on = torch.arange(s["bias"].shape[1], device=DEV)[None] < s["bias_len"][:, None]
    add = torch.zeros((r, v), dtype=torch.float64, device=DEV)
    add.scatter_add_(1, s["bias_ids"].long(), torch.where(on, s["bias"], 0.0).double())
    y = y + add.float()
    if s["mask"] is not None:
        k = torch.arange(v, device=DEV)
        y = torch.where(((s["mask"][:, k // 32] >> (k % 32)) & 1) == 1, y, -math.inf)
    y = y.to(s["out"].dtype)
    top = y.float().amax(-1, keepdim=True)
    first = torch.where(y.float() == top, torch.arange(v, device=DEV)[None], v).amin(-1)
    return {"logits": y, "token": torch.where(top[:, 0] > -math.inf, first, -1).to(torch.int32)}


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        B = s["B"]
        if op == "rope":
            B.rope_dev(s["out"], s["x"], s["pos"], s["cfg"], case["first"], inverse=case["inverse"])
            return s["out"]
        if op == "kv_write":
            if case["rope"]:
                B.kv_write_dev(s["cache"], s["rows"], s["slots"], rope=s["cfg"], pos=s["pos"])
            else:
                B.kv_write_dev(s["cache"], s["rows"], s["slots"])
            return _cache_out(s)
        if op == "kv_read":
            B.kv_read_dev(s["out"], s["cache"], s["slots"])
            return s["out"]
        if op == "tree_attn":
            B.tree_attn_dev(s["out"], s["q"], s["cache"], s["pages"], s["ctx"], s["n_draft"], s["mask"], s["sink"],
                            case["ctx"], s["scale"], s["scratch"])
            return s["out"]
        B.logits_dev(s["out"], s["x"], s["token"], s["adj"])
        return {"logits": s["out"], "token": s["token"]}
    if op == "rope":
        c, sn = _angles(s["pos"], case["rd"], case["scaled"])
        x = _rotated(s["x"].float(), c, sn, case["first"], case["rd"], case["layout"] == "half", case["inverse"])
        return x.to(s["out"].dtype)
    if op == "kv_write":
        rows = s["rows"].float()
        if case["rope"]:
            c, sn = _angles(s["pos"], case["tail"], True)
            rows = _rotated(rows[:, None], c, sn, case["d"] - case["tail"], case["tail"], False, False)[:, 0]
        _store(s["codes"], s["scales"], rows, s["slots"], case["tail"])
        return _cache_out(s)
    if op == "kv_read":
        v = _values(s["codes"], s["scales"], case["d"], case["tail"], s["slots"].clamp(min=0))
        return torch.where(s["slots"][:, None] >= 0, v, 0.0).to(s["out"].dtype)
    if op == "tree_attn":
        return _plain_attn(s)
    return _plain_logits(s)


# ------------------------------------------------------------- in 64 bits

def _turn64(x, pos, rd, first, half, inverse, scaled):
    """The rotation as complex numbers."""
    x = x.double().clone()
    th = pos.double()[:, None, None] * _frequencies(rd, scaled)
    z = torch.polar(torch.ones_like(th), -th if inverse else th)
    part = x[..., first:first + rd]
    w = torch.complex(part[..., :rd // 2], part[..., rd // 2:]) if half else \
        torch.view_as_complex(part.reshape(*part.shape[:-1], rd // 2, 2).contiguous())
    w = w * z
    x[..., first:first + rd] = torch.cat((w.real, w.imag), -1) if half else torch.view_as_real(w).flatten(-2)
    return x


def _pow2(e):
    """2^e exactly, from the bits of a double."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest64(v, bits, low):
    """v rounded to `bits` fraction bits, the exponent no lower than `low`: ties to even."""
    step = _pow2((torch.frexp(v.abs().clamp(min=2.0 ** low))[1] - 1).clamp(min=low) - bits)
    return torch.round(v / step) * step


def _rows64(s, slots):
    """Values of cache rows, decoded from the bits."""
    c = s["case"]
    n = c["d"] - c["tail"]
    raw = s["codes"].reshape(-1, c["d"] + c["tail"])[slots].long()
    k = raw[..., :n]
    e, m = (k >> 3) & 15, (k & 7).double()
    mag = torch.where(e > 0, (8 + m) * _pow2(e - 10), m * 2.0 ** -9)
    mag = torch.where((k & 127) == 127, math.nan, mag)
    u = raw[..., n::2] + 256 * raw[..., n + 1::2]
    f, w = (u >> 10) & 31, (u & 1023).double()
    end = torch.where(f > 0, (1024 + w) * _pow2(f - 25), w * 2.0 ** -24)
    v = torch.cat((torch.where(k > 127, -mag, mag), torch.where(u >= 1 << 15, -end, end)), -1)
    return v * _pow2(s["scales"].reshape(-1)[slots].long() - 127)[..., None]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rope":
        return _turn64(s["x"], s["pos"], case["rd"], case["first"], case["layout"] == "half", case["inverse"],
                       case["scaled"])
    if op == "kv_write":
        d, tail = case["d"], case["tail"]
        x = s["rows"].double()
        if case["rope"]:
            x = _turn64(x[:, None], s["pos"], tail, d - tail, False, False, True)[:, 0]
        e = torch.ceil(torch.log2(x.abs().amax(-1) / 448.0)).clamp(min=-127)
        y = x * _pow2(-e)[:, None]
        y = torch.cat((_nearest64(y[:, :d - tail], 3, -6), _nearest64(y[:, d - tail:], 10, -14)), -1)
        put = s["slots"] >= 0
        full = torch.zeros((s["scales"].numel(), d), dtype=torch.float64, device=DEV)
        full[s["slots"][put]] = y[put]
        scales = torch.full((s["scales"].numel(),), 2.0 ** -127, dtype=torch.float64, device=DEV)
        scales[s["slots"][put]] = _pow2(e[put])
        full = full.view(*s["scales"].shape, d)
        return {"codes": full[..., :d - tail].contiguous(), "tail": full[..., d - tail:].contiguous(),
                "scales": scales.view(s["scales"].shape)}
    if op == "kv_read":
        v = _rows64(s, s["slots"].clamp(min=0))
        v[s["slots"] < 0] = 0.0
        return v
    if op == "tree_attn":
        b, t, h, d = (case[k] for k in ("batch", "tokens", "heads", "d"))
        see = _seen(s)
        out = torch.zeros((b, t, h, d), dtype=torch.float64, device=DEV)
        for i in range(b):
            n = int(s["ctx"][i] + s["n_draft"][i])
            v = _rows64(s, _slots_of(s["pages"][i:i + 1], case["page"], n)[0])
            for k in range(int(s["n_draft"][i])):
                z = s["q"][i, k].double() @ v.T * s["scale"]
                z[:, ~see[i, k, :n]] = -math.inf
                w = torch.cat((z, s["sink"].double()[:, None]), -1)     # the sink takes its share and gives nothing
                out[i, k] = torch.softmax(w, -1)[:, :n] @ v
        return out
    x, r, v = s["x"].double(), case["rows"], case["vocab"]
    for i in range(r):
        n, p = int(s["hist_len"][i]), int(s["n_prompt"][i])
        seen = torch.bincount(s["hist"][i, :n].long(), minlength=v) > 0
        count = torch.bincount(s["hist"][i, p:n].long(), minlength=v).double()
        rep = s["rep"][i].double()
        x[i, seen] = torch.where(x[i, seen] > 0, x[i, seen] / rep, x[i, seen] * rep)
        x[i] -= s["freq"][i].double() * count + s["pres"][i].double() * (count > 0)
        k = int(s["bias_len"][i])
        x[i].index_add_(0, s["bias_ids"][i, :k].long(), s["bias"][i, :k].double())
        if s["mask"] is not None:
            word = s["mask"][i].long() & 0xFFFFFFFF
            on = (word[:, None] >> torch.arange(32, device=DEV)) & 1
            x[i, on.flatten()[:v] == 0] = -math.inf
    return {"logits": x, "token": None}


# --------------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": n * case["width"] * (SIZE[case["src"]] + SIZE[case["dst"]]) + 4 * case["tokens"],
                "flops": 3 * n * case["rd"]}
    if op in ("kv_write", "kv_read"):
        n, d = case["n"], case["d"]
        other = SIZE[case["src" if op == "kv_write" else "dst"]]
        return {"bytes": n * (d * other + d + case["tail"] + 1 + 8), "flops": 2 * n * d}
    if op == "tree_attn":
        b, t, h, d = (case[k] for k in ("batch", "tokens", "heads", "d"))
        share = 0.5 if case["ragged"] else 1.0           # ragged lengths are half the longest on average
        rows = b * (share * case["ctx"] + t)
        pairs = b * (share * t if t > 1 else t) * h * (share * case["ctx"] + t / 2)
        return {"bytes": rows * (d + case["tail"] + 1) + 2 * b * t * h * d * 2, "flops": 4 * pairs * d}
    r, v = case["rows"], case["vocab"]
    return {"bytes": r * (2 * v * SIZE[case["dtype"]] + 4 * 0.75 * case["hist"] + 8 * case["bias"]
                          + (v / 8 if case["mask"] else 0)), "flops": 4 * r * v}
