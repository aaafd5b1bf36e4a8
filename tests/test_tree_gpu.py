"""The tree-verification operators on the B200 against plain computations in
64 bits (torch float64 on the device, from the definition).

Tolerances come from the roundings that the definition and the kernels make:
u(t) = finfo(t).eps / 2 for one rounding to type t; a float product or sum
2^-24 of its value.
"""
import numpy as np
import pytest

import dsv4_b200 as B

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def dev():
    return B.init()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def unit(t):
    """Half a step of type t relative to the value, and below the normal range."""
    f = torch.finfo(t)
    return f.eps / 2, f.tiny * f.eps / 2


def close(got, want, tol):
    """|got - want| <= tol everywhere; NaN and infinities in the same places."""
    g, w = got.double(), want.double()
    fin = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    assert torch.equal(g[~fin & ~torch.isnan(w)], w[~fin & ~torch.isnan(w)])
    bad = (g - w).abs() > tol
    bad &= fin
    assert not bad.any(), (int(bad.sum()), float(((g - w).abs() / tol)[fin].max()))


# -------------------------------------------------------------------- rope

def turned(x, pos, cfg, first, inverse):
    """The rotation in double, and |a| + |b| of each element's pair."""
    x = x.double().clone()
    n = cfg.rd // 2
    th = pos.double()[:, None, None] * torch.tensor(list(cfg.freq[:n]), dtype=torch.float64, device="cuda")
    c, s = th.cos(), th.sin() * (-1 if inverse else 1)
    size = torch.zeros_like(x)
    ia = torch.arange(n, device="cuda") if cfg.layout == B.ROPE_HALF else 2 * torch.arange(n, device="cuda")
    ib = ia + n if cfg.layout == B.ROPE_HALF else ia + 1
    a, b = x[..., first + ia], x[..., first + ib]
    size[..., first + ia] = size[..., first + ib] = a.abs() + b.abs()
    x[..., first + ia], x[..., first + ib] = a * c - b * s, a * s + b * c
    return x, size


def rope_tol(want, size, dt):
    """cos and sin are rounded once (their angle is good to 1e-15), then each
    product and the sum: 3 roundings on |a| + |b|; then the output's."""
    rel, low = unit(dt)
    return 3.01 * U32 * size + (rel * (1 + 2 ** -20)) * want.abs() + low


ROPES = [  # tokens, heads, width, rd, first, layout, src, dst
    (1, 64, 512, 64, 448, 0, "f32", "bf16"), (5, 3, 512, 64, 448, 1, "bf16", "f32"), (7, 1, 64, 64, 0, 0, "f16", "f16"),
    (33, 16, 320, 64, 256, 0, "f32", "f32"), (2, 4, 576, 256, 320, 1, "bf16", "bf16"), (3, 2, 37, 34, 3, 0, "f32", "f16"),
    (3, 2, 37, 34, 1, 1, "bf16", "bf16"), (257, 2, 24, 8, 8, 0, "f16", "f32"), (4, 5, 40, 16, 16, 1, "f32", "bf16"),
    (1, 1, 2, 2, 0, 0, "f32", "f32"), (1300, 2, 64, 32, 0, 1, "bf16", "f16")]


@pytest.mark.parametrize("n,h,w,rd,first,layout,src,dst", ROPES)
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(n, h, w, rd, first, layout, src, dst, inverse):
    g = gen(n + w)
    cfg = B.rope_cfg(rd, 1e4, layout=layout, factor=16.0, orig=65536)
    x = normal(g, n, h, w).to(DT[src])
    pos = torch.randint(-5, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    pos[-1] = 2 ** 31 - 1                                   # the farthest position
    pos[0] = 0 if n > 1 else pos[0]
    want, size = turned(x, pos, cfg, first, inverse)
    out = torch.full((n, h, w), 7.0, dtype=DT[dst], device="cuda")
    B.rope_dev(out, x, pos, cfg, first, inverse=inverse)
    tol = rope_tol(want, size, DT[dst])
    close(out, want, tol)
    # strided: heads inside a wider row, tokens apart, odd offsets
    pad = torch.full((n, h + 1, w + 5), 3.0, dtype=DT[src], device="cuda")
    pad[:, :h, 1:1 + w] = x
    dest = torch.full((n, h + 2, w + 3), 9.0, dtype=DT[dst], device="cuda")
    B.rope_dev(dest[:, 1:1 + h, 2:2 + w], pad[:, :h, 1:1 + w], pos, cfg, first, inverse=inverse)
    close(dest[:, 1:1 + h, 2:2 + w], want, tol)
    dest[:, 1:1 + h, 2:2 + w] = 9.0
    assert torch.all(dest == 9.0)                          # nothing beside it was written
    # in place
    y = x.clone()
    B.rope_dev(y, y, pos, cfg, first, inverse=inverse)
    close(y, want, rope_tol(want, size, DT[src]))


def test_rope_broadcast_heads_and_gradient():
    """x shared by all heads (stride 0); the inverse is the gradient: the
    formula's transpose, and differences of sum(w * rope(x))."""
    g = gen(3)
    cfg = B.rope_cfg(16, 1e4, layout=B.ROPE_HALF)
    x = normal(g, 6, 1, 24).expand(6, 4, 24)
    pos = torch.arange(6, dtype=torch.int32, device="cuda") * 11
    out = torch.empty((6, 4, 24), device="cuda")
    B.rope_dev(out, x, pos, cfg, 4)
    want, size = turned(x, pos, cfg, 4, False)
    close(out, want, rope_tol(want, size, torch.float32))
    w = normal(g, 6, 4, 24)
    grad = torch.empty_like(w)
    B.rope_dev(grad, w, pos, cfg, 4, inverse=True)
    for e in (0, 4, 9, 12, 19, 23):                        # the map is linear: a step of 1 has no remainder
        step = torch.zeros((6, 4, 24), device="cuda")
        step[..., e] = 1.0
        up, dn = torch.empty_like(step), torch.empty_like(step)
        B.rope_dev(up, step, pos, cfg, 4)
        B.rope_dev(dn, -step, pos, cfg, 4)
        diff = ((up.double() - dn.double()) * w.double()).sum(-1) / 2
        # two weighted roundings of the differences, three of the gradient
        assert torch.all((diff - grad[..., e].double()).abs() <= 8 * U32 * w.double().abs().sum(-1))


# ------------------------------------------------------------- quantised cache

def nearest(v, bits, low):
    """v rounded to `bits` fraction bits with exponents from `low`, ties to even."""
    e = (torch.frexp(v.abs().clamp(min=2.0 ** low))[1] - 1).clamp(min=low)
    step = torch.ldexp(torch.ones_like(v), e - bits)
    return torch.round(v / step) * step


def two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def decode(cache, slots):
    """Values of cache rows from the bits, in double."""
    n = cache.d - cache.tail
    raw = cache.codes.view(-1, cache.d + cache.tail)[slots].long()
    k = raw[:, :n]
    e, m = (k >> 3) & 15, (k & 7).double()
    mag = torch.where(e > 0, (8 + m) * two(e - 10), m * 2.0 ** -9)
    mag = torch.where((k & 127) == 127, np.nan, mag)
    u = raw[:, n::2] + 256 * raw[:, n + 1::2]
    f, w = (u >> 10) & 31, (u & 1023).double()
    end = torch.where(f > 0, (1024 + w) * two(f - 25), w * 2.0 ** -24)
    v = torch.cat((torch.where(k > 127, -mag, mag), torch.where(u >= 1 << 15, -end, end)), -1)
    b = cache.scales.view(-1)[slots].long()
    return torch.where(b[:, None] == 255, np.nan, v * two(b - 127)[:, None])


def same(a, b):
    """Equal values, NaN in the same places."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def quantised(x, tail):
    """Row values after quantisation, and the scale bytes, by the definition: a
    row with an infinity or a NaN is NaN, byte 255."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[:, None], 0.0, x)
    top = x.abs().amax(-1)
    m, e = torch.frexp(top / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-127)
    e = torch.where(top > 0, e, -127)
    y = x * two(-e)[:, None]
    n = x.shape[1] - tail
    y = torch.cat((nearest(y[:, :n], 3, -6), nearest(y[:, n:], 10, -14)), -1)
    return (torch.where(bad[:, None], np.nan, y * two(e)[:, None]),
            torch.where(bad, 255, e + 127).to(torch.uint8))


KV = [(1, 64, 0, 64, "f32"), (5, 512, 64, 16, "bf16"), (33, 576, 64, 64, "f16"), (300, 320, 64, 1, "f32"),
      (17, 128, 128, 4, "bf16"), (1000, 448, 128, 128, "f32"), (9, 256, 0, 32, "f16")]


@pytest.mark.parametrize("n,d,tail,page,src", KV)
def test_kv_round_trip(n, d, tail, page, src):
    g = gen(d + n)
    x = normal(g, n, d) * torch.exp(3 * normal(g, n, 1))
    x[:, 3] *= 1e-4                                        # far below the largest: subnormal codes
    if n > 4:
        x[0] = 0.0
        x[1] = 448.0 * 2.0 ** -7                           # on the border of a scale
        x[2] = 448.0 * 2.0 ** -7 * (1 + 2.0 ** -7)         # just above it
        x[3] *= 2.0 ** -12
    if n > 8 and src != "f16":
        x[5] *= 1e-38 / x[5].abs().max()                   # the smallest scale
        x[6] *= 3e38 / x[6].abs().max()
    x = x.to(DT[src])
    pages = -(-(2 * n + 3) // page)
    c = B.KvCache.empty(pages, page, d, tail)
    c.codes.fill_(0x5A)
    c.scales.fill_(0x33)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
    B.kv_write_dev(c, x, slots)
    want, scale = quantised(x, tail)
    assert torch.equal(c.scales.view(-1)[slots], scale)
    assert same(decode(c, slots), want)                    # exactly the nearest codes
    other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    other[slots] = False
    assert torch.all(c.codes.view(-1, d + tail)[other] == 0x5A) and torch.all(c.scales.view(-1)[other] == 0x33)
    for dst in DT.values():
        out = torch.full((n, d), 5.0, dtype=dst, device="cuda")
        B.kv_read_dev(out, c, slots)
        assert same(out, want.float().to(dst))             # code * scale is exact in float
    # rows that are not 16-byte aligned, and a strided destination
    wide = torch.zeros((n, d + 3), dtype=DT[src], device="cuda")
    wide[:, 1:1 + d] = x
    c2 = B.KvCache.empty(pages, page, d, tail)
    B.kv_write_dev(c2, wide[:, 1:1 + d], slots)
    assert torch.equal(c2.codes.view(-1, d + tail)[slots], c.codes.view(-1, d + tail)[slots])
    dest = torch.full((n, d + 5), 5.0, device="cuda")
    B.kv_read_dev(dest[:, 3:3 + d], c, slots)
    assert same(dest[:, 3:3 + d].double(), want.float().double())
    assert torch.all(dest[:, :3] == 5.0) and torch.all(dest[:, 3 + d:] == 5.0)


def test_kv_moved_rows_keep_their_values():
    """Rows read into f32 and written elsewhere read back the same: a largest
    code that was rounded down to a power of two halves the scale, which
    doubles codes and tail exactly."""
    g = gen(50)
    n, d, tail = 2000, 512, 64
    c = B.KvCache.empty(2 * n // 16, 16, d, tail)
    x = normal(g, n, d) * torch.exp(4 * normal(g, n, 1))
    x[::5] = x[::5].clamp(-1, 1) * 224.01 * 2.0 ** -9       # the largest just above half the range
    x[3], x[4] = 0.0, float("nan")
    at = torch.randperm(2 * n, generator=g, device="cuda")
    first, then = torch.empty_like(x), torch.empty_like(x)
    B.kv_write_dev(c, x, at[:n])
    B.kv_read_dev(first, c, at[:n])
    B.kv_write_dev(c, first, at[n:])
    B.kv_read_dev(then, c, at[n:])
    assert torch.equal(then.nan_to_num(nan=7.0), first.nan_to_num(nan=7.0)) and then[4].isnan().all()


def test_kv_skipped_and_bad_values():
    c = B.KvCache.empty(3, 8, 128, 64)
    x = normal(gen(1), 6, 128)
    x[1, 5], x[2, 100], x[3, 0] = float("nan"), float("inf"), -float("inf")
    slots = torch.tensor([-1, 3, 4, 5, 24, 7], device="cuda")
    B.kv_write_dev(c, x, slots)
    out = torch.full((8, 128), 9.0, device="cuda")
    B.kv_read_dev(out, c, torch.tensor([-1, 3, 4, 5, 24, 7, 0, -(1 << 40)], device="cuda"))
    assert torch.isnan(out[1:4]).all() and not out[[0, 4, 6, 7]].any()
    assert torch.equal(out[5].double(), quantised(x[5:6], 64)[0][0])
    assert int((c.codes != 0).any(-1).sum()) == 1          # NaN rows hold zero codes
    assert torch.all(c.scales.view(-1)[3:6] == 255)
    B.kv_write_dev(c, x[:0], slots[:0])
    B.kv_read_dev(out[:0], c, slots[:0])


@pytest.mark.parametrize("layout", [B.ROPE_INTERLEAVED, B.ROPE_HALF])
@pytest.mark.parametrize("d,tail,rd,src", [(512, 64, 64, "f32"), (128, 64, 34, "bf16"), (576, 64, 256, "f16"), (64, 0, 64, "f32")])
def test_kv_write_rotates(layout, d, tail, rd, src):
    """Rotation and quantisation in one call: the stored values are within half
    a code step (and the rotation's float roundings) of the rotated rows."""
    n = 37
    g = gen(d + rd)
    cfg = B.rope_cfg(rd, 1e4, layout=layout, factor=16.0, orig=65536)
    x = normal(g, n, d).to(DT[src])
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    c = B.KvCache.empty(2, 32, d, tail)
    slots = torch.randperm(64, generator=g, device="cuda")[:n]
    B.kv_write_dev(c, x, slots, rope=cfg, pos=pos)
    want, size = turned(x[:, None], pos, cfg, d - rd, False)
    want, size = want[:, 0], size[:, 0]
    s = two(c.scales.view(-1)[slots].long() - 127)[:, None]
    top = want.abs().amax(-1, keepdim=True)
    assert torch.all(top <= 448 * s * (1 + 2 ** -20)) and torch.all(top > 224 * s * (1 - 2 ** -20))
    half = torch.cat((torch.maximum(want[:, :d - tail].abs() * 2.0 ** -4, s * 2.0 ** -10),
                      torch.maximum(want[:, d - tail:].abs() * 2.0 ** -11, s * 2.0 ** -25)), -1)
    close(decode(c, slots), want, half * (1 + 2 ** -18) + 4 * U32 * size)


# ---------------------------------------------------------------- attention

def tree_case(seed, b, t, h, d, tail, page, ctx, dtype, ragged=False, spread=2.0, extra=3):
    g = gen(seed)
    per = -(-(ctx + t) // page)
    pool = b * per + extra
    c = B.KvCache.empty(pool, page, d, tail)
    x = normal(g, pool * page, d) + 0.5 * normal(g, 1, d)
    x *= torch.exp(0.5 * normal(g, pool * page, 1))        # rows of different scales
    B.kv_write_dev(c, x, torch.arange(pool * page, device="cuda"))
    pages = torch.randperm(pool, generator=g, device="cuda")[:b * per].to(torch.int32).view(b, per)
    cl = torch.full((b,), ctx, dtype=torch.int32, device="cuda")
    nd = torch.full((b,), t, dtype=torch.int32, device="cuda")
    if ragged:
        cl = torch.randint(0, ctx + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        nd = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        cl[0], nd[-1] = 0, t
    rng = np.random.default_rng(seed)
    mask = torch.from_numpy(np.stack([B.tree_mask([int(rng.integers(-1, i)) for i in range(t)]) for _ in range(b)])).cuda()
    q = (spread * normal(g, b, t, h, d)).to(dtype)
    sink = normal(g, h)
    return dict(c=c, pages=pages, ctx=cl, nd=nd, mask=mask, q=q, sink=sink, scale=d ** -0.5, max_ctx=ctx)


def plain_tree(k):
    """o and its tolerance, in double, token by token."""
    q, c = k["q"], k["c"]
    b, t, h, d = q.shape
    want = torch.full(q.shape, 11.0, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    page, total = c.codes.shape[1], c.scales.numel()
    for i in range(b):
        n, m = int(k["ctx"][i]), int(k["nd"][i])
        j = torch.arange(n + m, device="cuda")
        pg = k["pages"][i].long()[j // page]
        good = (pg >= 0) & (pg < c.codes.shape[0])
        slot = torch.where(good, pg * page + j % page, 0)
        assert slot.numel() == 0 or int(slot.max()) < total
        v = decode(c, slot)
        for a in range(m):
            bits = int(k["mask"][i, a]) & (2 ** 64 - 1)
            see = good.clone()
            for z in range(m):
                see[n + z] &= bool((bits >> z) & 1)
            w = v[see]
            if w.shape[0] == 0:
                want[i, a] = 0.0
                continue
            z = q[i, a].double() @ w.T * k["scale"]
            top = z.amax(-1, keepdim=True)
            p = (z - top).exp()
            den = p.sum(-1, keepdim=True)
            if k["sink"] is not None:
                den = den + (k["sink"].double()[:, None] - top).exp()
            want[i, a] = p @ w / den
            # a score is a float sum of d products whose partial sums are held
            # in float: each of the d / 16 accumulations is off by at most
            # 2^-22 of the sum of magnitudes; q is held in f16 relative to the
            # largest of its tile (2^-24 of that); the exponential adds 2^-21
            qa = q[i, a].double().abs()
            mag = abs(k["scale"]) * (qa @ w.abs().T).amax(-1, keepdim=True)
            part = abs(k["scale"]) * float(q.double().abs().max()) * 2.0 ** -24 * w.abs().sum(-1).max()
            delta = mag * (d / 16 + 4) * 2.0 ** -22 + part + 2.0 ** -21
            # a weight is rounded to f16 (2^-11, and 2^-25 of the largest
            # weight), so is one output; sums of n weights in float
            size = p @ w.abs() / den
            low = 2.0 ** -22 * w.abs().sum(0, keepdim=True) / den
            rel, tiny = unit(q.dtype)
            tol[i, a] = size * (2.0 ** -11 + 2 * delta + 2.0 ** -16) + low + rel * 1.001 * want[i, a].abs() + tiny
    return want, tol


def run_tree(k, out=None, scratch=None, stream=None):
    q = k["q"]
    b, t, h, d = q.shape
    if scratch is None:
        scratch = torch.empty(B.tree_attn_scratch(h, d, t, b, k["max_ctx"]), dtype=torch.uint8, device="cuda")
        scratch.fill_(255)                                 # NaN wherever something is read before it is written
    if out is None:
        out = torch.full(q.shape, 11.0, dtype=q.dtype, device="cuda")
    B.tree_attn_dev(out, q, k["c"], k["pages"], k["ctx"], k["nd"], k["mask"], k["sink"], k["max_ctx"], k["scale"],
                    scratch, stream=stream)
    return out


TREES = [  # batch, tokens, heads, d, tail, page, ctx
    (1, 1, 64, 512, 64, 64, 0), (1, 1, 64, 512, 64, 64, 1), (1, 1, 1, 64, 0, 16, 127), (2, 3, 5, 128, 64, 1, 128),
    (1, 2, 64, 512, 64, 64, 129), (3, 7, 16, 320, 64, 32, 500), (2, 64, 4, 64, 0, 16, 63), (1, 5, 128, 256, 0, 128, 300),
    (1, 1, 64, 576, 64, 64, 1000), (2, 4, 48, 576, 64, 64, 255), (1, 17, 64, 448, 128, 64, 640), (5, 1, 8, 192, 192, 2, 70),
    (1, 3, 64, 512, 64, 4096, 5000), (2, 2, 64, 512, 512, 64, 200), (1, 33, 3, 384, 64, 8, 191)]


@pytest.mark.parametrize("b,t,h,d,tail,page,ctx", TREES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_tree_attn(b, t, h, d, tail, page, ctx, dtype, ragged):
    k = tree_case(b * 1000 + t * 100 + d, b, t, h, d, tail, page, ctx, DT[dtype], ragged)
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)
    k["sink"] = None
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)


@pytest.mark.parametrize("b,ctx", [(1, 20000), (3, 6000), (40, 900)])
def test_tree_attn_splits(b, ctx):
    """Contexts that are split over blocks and joined, and many sequences."""
    k = tree_case(b, b, 3, 64, 512, 64, 64, ctx, torch.bfloat16, ragged=b > 1)
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)


def test_tree_attn_sharp_and_flat():
    """One position far above the others at the start, the end and the middle,
    growing scores (the running maximum rises in every tile), equal scores."""
    k = tree_case(5, 1, 2, 64, 512, 64, 64, 1500, torch.bfloat16, spread=8.0)
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)
    c = k["c"]
    page = c.codes.shape[1]
    j = torch.arange(1502, device="cuda")
    slot = k["pages"][0].long()[j // page] * page + j % page
    base = normal(gen(9), 1, 512)
    rise = torch.linspace(0.01, 6.0, 1502, device="cuda")[:, None]
    for rows in (base * rise, base * rise.flip(0), base.expand(1502, 512) + 0.0):
        B.kv_write_dev(c, rows.contiguous(), slot)
        k["q"] = (3.0 * base * torch.ones((1, 2, 64, 1), device="cuda")).to(torch.bfloat16)
        want, tol = plain_tree(k)
        close(run_tree(k), want, tol)


def test_tree_attn_scale_range():
    """Rows whose scales are far apart: large rows with little weight beside
    small rows that carry it, rows of zeros, the smallest and largest scales."""
    k = tree_case(6, 1, 2, 64, 256, 0, 64, 700, torch.float16)
    c = k["c"]
    rows = normal(gen(4), c.scales.numel(), 256)
    rows[::7] *= 2.0 ** -9
    rows[1::7] *= 2.0 ** 5
    rows[2::7] = 0.0
    B.kv_write_dev(c, rows, torch.arange(c.scales.numel(), device="cuda"))
    k["q"] = (normal(gen(5), 1, 2, 64, 256) * 0.5).half()
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)
    for f in (2.0 ** -100, 2.0 ** 100):
        B.kv_write_dev(c, rows * f, torch.arange(c.scales.numel(), device="cuda"))
        k["scale"] = 256 ** -0.5 / f
        k["q"] = k["q"].bfloat16()
        want, tol = plain_tree(k)
        if f > 1:                                          # values beyond f16: bf16 outputs
            close(run_tree(k), want, tol)
        else:
            close(run_tree(k), want, tol + 2.0 ** -133)


def test_tree_attn_nothing_and_masked_nan():
    """An empty mask over an empty context gives zeros; NaN rows behind the
    context, in unseen drafts and on skipped pages stay out."""
    k = tree_case(7, 2, 4, 64, 512, 64, 16, 40, torch.bfloat16)
    c = k["c"]
    k["ctx"][1] = 0
    k["mask"][1, 2] = 0
    k["mask"][0, 1] = 0b1101 & ~0b0010
    page = 16

    def slot(b, j):
        return int(k["pages"][b, j // page]) * page + j % page

    bad = torch.full((1, 512), float("nan"), device="cuda")
    for b, j in ((0, 41), (1, 3)):                         # the unseen draft 1 of sequence 0; draft 3 of sequence 1
        B.kv_write_dev(c, bad, torch.tensor([slot(b, j)], device="cuda"))
    k["mask"][0, 1:] &= ~0b0010
    k["mask"][0, 0] = 1
    k["mask"][1] &= ~0b1000
    k["pages"][1, 1:] = -1
    want, tol = plain_tree(k)
    assert torch.isfinite(want).all() and not want[1, 2].any()
    # garbage in every byte that is no row of a sequence: codes and scales of all ones are NaN
    used = torch.zeros(c.scales.numel(), dtype=torch.bool, device="cuda")
    for b in range(2):
        for j in range(int(k["ctx"][b]) + 4):
            if 0 <= int(k["pages"][b, j // page]) < c.codes.shape[0]:
                used[slot(b, j)] = True
    c.codes.view(-1, 576)[~used] = 255
    c.scales.view(-1)[~used] = 255
    close(run_tree(k), want, tol)
    # a NaN row that is seen makes its tokens NaN, and only those
    k["mask"][0, 2] |= 0b0010
    out = run_tree(k)
    assert torch.isnan(out[0, 2]).all()
    keep = torch.ones((2, 4), dtype=torch.bool, device="cuda")
    keep[0, 2] = False
    close(out[keep], want[keep], tol[keep])


def test_tree_attn_bad_pages_and_lengths():
    """Pages outside the cache are skipped; lengths beyond the launch's are cut
    to it, negative ones count as none."""
    k = tree_case(8, 3, 2, 16, 128, 64, 16, 100, torch.float16)
    k["pages"][0, 2] = -1
    k["pages"][1, 0] = k["c"].codes.shape[0]
    k["pages"][2, 6] = 2 ** 31 - 1                          # the drafts' own page
    k["pages"][2, 3] = -2 ** 31
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)
    k["ctx"][0], k["ctx"][1], k["nd"][2] = 10 ** 9, -5, 99
    k2 = dict(k, ctx=torch.tensor([100, 0, 100], dtype=torch.int32, device="cuda"),
              nd=torch.tensor([2, 2, 2], dtype=torch.int32, device="cuda"))
    want, tol = plain_tree(k2)
    close(run_tree(k), want, tol)
    k["nd"][1] = -3
    k2["nd"][1] = 0
    want, tol = plain_tree(k2)
    out = run_tree(k)
    assert torch.all(out[1] == 11.0)
    close(out, want, tol)
    k["pages"].fill_(-1)
    out = run_tree(k)
    assert not out[0].any() and not out[2].any()


def test_tree_attn_far_offsets():
    """Rows more than 2^31 bytes into the cache."""
    page, d, tail = 4096, 512, 64
    pages = (1 << 31) // (page * (d + tail)) + 40
    c = B.KvCache.empty(pages, page, d, tail)
    last = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    j = torch.arange(2 * page, device="cuda")
    slots = last[0].long()[j // page] * page + j % page
    assert int(slots.min()) * (d + tail) > 1 << 31
    x = normal(gen(12), 2 * page, d)
    B.kv_write_dev(c, x, slots)
    got = torch.empty_like(x)
    B.kv_read_dev(got, c, slots)
    assert torch.equal(got.double(), quantised(x, tail)[0])
    k = dict(c=c, pages=last, ctx=torch.tensor([5000], dtype=torch.int32, device="cuda"),
             nd=torch.tensor([2], dtype=torch.int32, device="cuda"), mask=torch.tensor([[1, 3]], device="cuda"),
             q=normal(gen(13), 1, 2, 64, d).bfloat16(), sink=normal(gen(14), 64), scale=d ** -0.5, max_ctx=5000)
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)


def test_tree_attn_strides_streams_and_graphs():
    """q and o inside wider rows; a side stream; a captured call replayed with
    other contents, lengths and masks; equal results call after call."""
    k = tree_case(15, 2, 3, 64, 512, 64, 64, 900, torch.bfloat16)
    want, tol = plain_tree(k)
    ref = run_tree(k)
    close(ref, want, tol)
    wide = torch.zeros((2, 3, 70, 512), dtype=torch.bfloat16, device="cuda")
    wide[:, :, 3:67] = k["q"]
    dest = torch.full((2, 3, 66, 512), 11.0, dtype=torch.bfloat16, device="cuda")
    run_tree(dict(k, q=wide[:, :, 3:67]), out=dest[:, :, 1:65])
    assert torch.equal(dest[:, :, 1:65], ref)
    assert torch.all(dest[:, :, 0] == 11.0) and torch.all(dest[:, :, 65] == 11.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert torch.equal(_after(side, lambda: run_tree(k, stream=side)), ref)
    scratch = torch.empty(B.tree_attn_scratch(64, 512, 3, 2, 900), dtype=torch.uint8, device="cuda")
    out = torch.full(k["q"].shape, 11.0, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_tree(k, out=out, scratch=scratch)
    for ctx, nd in ((900, 3), (0, 1), (400, 2)):
        k["ctx"].fill_(ctx)
        k["nd"].fill_(nd)
        k["q"].copy_(normal(gen(ctx), *k["q"].shape))
        out.fill_(11.0)
        graph.replay()
        torch.cuda.synchronize()
        want, tol = plain_tree(k)
        close(out, want, tol)
        assert torch.equal(out, run_tree(k))


def test_tree_attn_shares_blocks_by_length():
    """Many sequences of very different lengths, some without tokens: the
    blocks that short ones leave go to the long ones."""
    k = tree_case(31, 70, 3, 16, 128, 64, 16, 2500, torch.bfloat16, ragged=True)
    k["ctx"][5::7] = 0
    k["ctx"][::11] = 2500
    k["nd"][3::9] = 0
    want, tol = plain_tree(k)
    got = run_tree(k)
    close(got, want, tol)
    assert torch.equal(run_tree(k), got)
    k["nd"].zero_()
    assert torch.all(run_tree(k) == 11.0)                  # nothing drafted: nothing written


@pytest.mark.parametrize("d,tail", [(64, 64), (128, 0), (256, 64), (384, 64), (448, 64), (512, 64), (576, 64)])
@pytest.mark.parametrize("heads", [8, 64])
def test_tree_attn_many_tiles(d, tail, heads):
    """Every row width through many key tiles of one block: all places for keys
    and values are used again and again."""
    k = tree_case(40 + d, 37, 4, heads, d, tail, 64, 1400, torch.bfloat16)
    if heads == 64:
        k["ctx"][1:] = torch.arange(36, dtype=torch.int32, device="cuda")
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)


def test_tree_attn_one_long_among_short():
    k = tree_case(32, 33, 2, 64, 512, 64, 64, 3000, torch.float16)
    k["ctx"].fill_(10)
    k["ctx"][32] = 3000
    want, tol = plain_tree(k)
    close(run_tree(k), want, tol)


def test_tree_attn_thousands_of_sequences():
    """More sequences than the blocks share among, with room for long contexts."""
    b, d, page = 4100, 64, 65536
    c = B.KvCache.empty(2, page, d, 0)
    x = normal(gen(33), 600, d)
    at = torch.cat((torch.arange(300), page + torch.arange(300))).cuda()
    B.kv_write_dev(c, x, at)
    pages = torch.zeros((b, 17), dtype=torch.int32, device="cuda")
    pages[:, 0] = torch.arange(b, device="cuda") % 2
    g = gen(34)
    ctx = torch.randint(0, 299, (b,), generator=g, device="cuda", dtype=torch.int32)
    q = normal(g, b, 1, 2, d).bfloat16()
    k = dict(c=c, pages=pages, ctx=ctx, nd=torch.ones(b, dtype=torch.int32, device="cuda"),
             mask=torch.ones((b, 1), dtype=torch.int64, device="cuda"), q=q, sink=None, scale=0.2, max_ctx=1 << 20)
    got = run_tree(k)
    some = torch.tensor([0, 1, 31, 32, 4095, 4096, 4099], device="cuda")
    part = dict(k, pages=pages[some], ctx=ctx[some], nd=k["nd"][some], mask=k["mask"][some], q=q[some])
    want, tol = plain_tree(part)
    close(got[some], want, tol)
    assert torch.all((got != 11.0).any(-1))                # every sequence has been written


def test_two_streams_at_once():
    """Calls on two streams at a time, each with scratch of its own."""
    k = [tree_case(35 + i, 2, 4, 64, 512, 64, 64, 1500, torch.bfloat16, ragged=bool(i)) for i in range(2)]
    ref = [run_tree(x) for x in k]
    x = 3 * normal(gen(37), 2, 20000)
    tok = torch.empty(2, dtype=torch.int32, device="cuda")
    B.logits_dev(None, x, tok)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    room = [torch.empty(B.tree_attn_scratch(64, 512, 4, 2, 1500), dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [[torch.full_like(r, 11.0) for _ in range(6)] for r in ref]
    toks = [[torch.empty_like(tok) for _ in range(6)] for _ in range(2)]
    torch.cuda.synchronize()
    for n in range(6):
        for i in range(2):
            run_tree(k[i], out=outs[i][n], scratch=room[i], stream=side[i])
            B.logits_dev(None, x, toks[i][n], stream=side[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i]) for o in outs[i]) and all(torch.equal(t, tok) for t in toks[i])
    assert B.lib().dsv4b_tree_attn_status() == 0           # no bounded wait has run out


def _after(stream, fn):
    out = fn()
    stream.synchronize()
    return out


# ------------------------------------------------------------------- logits

def plain_logits(x, hist, hl, npr, rep, freq, pres, ids, bias, bl, mask):
    """Adjusted logits in double and the sum of magnitudes along the way."""
    y = x.double().clone()
    r, v = y.shape
    size = y.abs()
    for i in range(r):
        if hist is not None:
            h = [int(t) for t in hist[i, :max(0, int(hl[i]))]]
            n = int(npr[i]) if npr is not None else 0
            seen = sorted({t for t in h if 0 <= t < v})
            if rep is not None and seen:
                z = y[i, seen]
                y[i, seen] = torch.where(z > 0, z / rep[i].double(), z * rep[i].double())
                size[i] = torch.maximum(size[i], y[i].abs())
            count = torch.zeros(v, dtype=torch.float64, device="cuda")
            for t in h[max(0, n):]:
                if 0 <= t < v:
                    count[t] += 1
            for amount, times in ((freq, count), (pres, (count > 0).double())):
                if amount is not None:
                    y[i] -= amount[i].double() * times
                    size[i] += (amount[i].double() * times).abs()
        if bias is not None:
            for k in range(max(0, int(bl[i]))):
                t = int(ids[i, k])
                if 0 <= t < v:
                    y[i, t] += bias[i, k].double()
                    size[i, t] += bias[i, k].double().abs()
        if mask is not None:
            on = torch.tensor([(int(mask[i, t // 32]) >> (t % 32)) & 1 for t in range(v)], device="cuda")
            y[i, on == 0] = -np.inf
    return y, size


def greedy(y):
    top = y.float().amax(-1)
    out = []
    for i in range(y.shape[0]):
        at = (y[i].float() == top[i]).nonzero().flatten()
        out.append(int(at[0]) if float(top[i]) > -np.inf else -1)
    return out


LOGITS = [(1, 1, 0, 0, False, "f32"), (3, 1000, 40, 5, True, "f32"), (2, 131, 9, 200, True, "bf16"),
          (4, 65543, 300, 30, True, "f16"), (2, 4096, 2500, 64, False, "bf16"), (70, 517, 8, 1, True, "f32"),
          (1, 70001, 100, 12, True, "f32")]


@pytest.mark.parametrize("r,v,hist,nb,masked,dt", LOGITS)
def test_logits(r, v, hist, nb, masked, dt):
    g = gen(r * 31 + v)
    x = (3 * normal(g, r, v)).to(DT[dt])
    kw = dict(hist=None, hist_len=None, n_prompt=None, rep=None, freq=None, pres=None, bias_ids=None, bias=None,
              bias_len=None, mask=None)
    if hist:
        kw["hist"] = torch.randint(-3, min(v, 60) + 3, (r, hist), generator=g, device="cuda", dtype=torch.int32)
        kw["hist_len"] = torch.randint(0, hist + 1, (r,), generator=g, device="cuda", dtype=torch.int32)
        kw["hist_len"][0] = hist + 5                       # cut to the row
        kw["n_prompt"] = torch.randint(-1, hist, (r,), generator=g, device="cuda", dtype=torch.int32)
        kw["rep"] = 0.5 + torch.rand(r, generator=g, device="cuda")
        kw["freq"], kw["pres"] = 0.3 * normal(g, r), normal(g, r)
    if nb:
        kw["bias_ids"] = torch.randint(-1, min(v, 90), (r, nb), generator=g, device="cuda", dtype=torch.int32)
        kw["bias"] = 2 * normal(g, r, nb)
        kw["bias_len"] = torch.full((r,), nb, dtype=torch.int32, device="cuda")
    if masked:
        words = (v + 31) // 32 + 1
        kw["mask"] = torch.randint(-2 ** 31, 2 ** 31, (r, words), generator=g, device="cuda").to(torch.int32)
        kw["mask"][-1] = 0                                 # a row that allows nothing
    hl = None if not hist else kw["hist_len"].clamp(max=hist)
    want, size = plain_logits(x, kw["hist"], hl, kw["n_prompt"], kw["rep"], kw["freq"], kw["pres"], kw["bias_ids"],
                              kw["bias"], kw["bias_len"], kw["mask"])
    rel, low = unit(DT[dt])
    # at most six float roundings on the way, then the output's
    tol = 6.01 * U32 * size + rel * (1 + 2 ** -20) * want.abs().nan_to_num(posinf=0) + low
    adj = B.LogitAdjust(**kw)
    out = torch.full((r, v), 5.0, dtype=DT[dt], device="cuda")
    tok = torch.full((r,), 77, dtype=torch.int32, device="cuda")
    B.logits_dev(out, x, tok, adj)
    close(out, want, tol)
    assert tok.tolist() == greedy(out)
    if masked:
        assert tok[-1] == -1
    only = torch.full((r,), 77, dtype=torch.int32, device="cuda")
    B.logits_dev(None, x, only, adj)                       # the token alone
    assert torch.equal(only, tok)
    pad = torch.full((r, v + 3), 5.0, dtype=DT[dt], device="cuda")
    pad[:, 1:1 + v] = x
    B.logits_dev(pad[:, 1:1 + v], pad[:, 1:1 + v], None, adj)     # in place, unaligned, no token
    assert torch.equal(pad[:, 1:1 + v], out)
    assert torch.all(pad[:, 0] == 5.0) and torch.all(pad[:, 1 + v:] == 5.0)


def test_logits_plain_and_special_values():
    """No adjustment copies and picks; ties go to the lowest index across
    blocks; infinities and NaN."""
    x = torch.zeros((4, 30000), device="cuda")
    x[0, [29999, 17, 12000]] = 4.0
    x[1] = -np.inf
    x[2, 5], x[2, 20000] = float("nan"), 1.0
    x[3, 9], x[3, 7] = np.inf, -np.inf
    out, tok = torch.empty_like(x), torch.empty(4, dtype=torch.int32, device="cuda")
    B.logits_dev(out, x, tok)
    assert torch.equal(out.nan_to_num(nan=123.0), x.nan_to_num(nan=123.0))
    assert tok.tolist() == [17, -1, 20000, 9]
    x.fill_(float("nan"))
    B.logits_dev(None, x, tok)
    assert tok.tolist() == [-1] * 4


@pytest.mark.parametrize("v,hist,span,nb,dt", [
    (129280, 60000, 129280, 3000, "f32"),       # more named tokens in a block's share than it settles at once
    (129280, 60000, 9000, 0, "bf16"),           # the same in the first shares alone
    (129280, 5000, 700, 0, "f32"),              # a long history of few tokens
    (40000, 0, 40000, 30000, "f16"),            # biases alone
    (600001, 40000, 600001, 500, "f32"),        # a vocabulary of two runs a block
    (600001, 70000, 150000, 9, "bf16")])
def test_logits_many_named(v, hist, span, nb, dt):
    """Histories and bias lists that fill, and overflow, what a block settles at once."""
    g = gen(v + hist)
    x = (3 * normal(g, 2, v)).to(DT[dt])
    kw = {}
    y, size = x.double(), x.double().abs()
    if hist:
        h = torch.randint(0, span, (2, hist), generator=g, device="cuda", dtype=torch.int32)
        n = torch.tensor([hist // 3, 0], dtype=torch.int32, device="cuda")
        rep, freq, pres = 0.5 + torch.rand(2, generator=g, device="cuda"), 0.1 * normal(g, 2), normal(g, 2)
        kw.update(hist=h, hist_len=torch.full((2,), hist, dtype=torch.int32, device="cuda"), n_prompt=n, rep=rep,
                  freq=freq, pres=pres)
        for i in range(2):
            seen = torch.bincount(h[i].long(), minlength=v) > 0
            count = torch.bincount(h[i, int(n[i]):].long(), minlength=v).double()
            r = rep[i].double()
            y[i] = torch.where(seen, torch.where(y[i] > 0, y[i] / r, y[i] * r), y[i])
            size[i] = torch.maximum(size[i], y[i].abs()) + (freq[i].double() * count).abs() + pres[i].double().abs()
            y[i] -= freq[i].double() * count + pres[i].double() * (count > 0)
    if nb:
        ids = torch.randint(0, v, (2, nb), generator=g, device="cuda", dtype=torch.int32)
        bias = normal(g, 2, nb)
        kw.update(bias_ids=ids, bias=bias, bias_len=torch.full((2,), nb, dtype=torch.int32, device="cuda"))
        for i in range(2):
            y[i].index_add_(0, ids[i].long(), bias[i].double())
            size[i].index_add_(0, ids[i].long(), bias[i].double().abs())
    rel, low = unit(DT[dt])
    # at most six float roundings on the way, then the output's
    tol = 6.01 * U32 * size + rel * (1 + 2 ** -20) * y.abs() + low
    out, tok = torch.empty_like(x), torch.empty(2, dtype=torch.int32, device="cuda")
    B.logits_dev(out, x, tok, B.LogitAdjust(**kw))
    close(out, y, tol)
    assert tok.tolist() == greedy(out)
    B.logits_dev(x, x, None, B.LogitAdjust(**kw))
    assert torch.equal(x, out)


def test_logits_duplicate_biases_are_ordered():
    """A token named many times gets the sum in list order, the same every time."""
    v, n = 5000, 900
    x = torch.zeros((1, v), device="cuda")
    ids = torch.full((1, n), 4321, dtype=torch.int32, device="cuda")
    ids[0, ::3] = 17
    b = normal(gen(2), 1, n) * torch.exp(6 * normal(gen(3), 1, n))
    adj = B.LogitAdjust(bias_ids=ids, bias=b, bias_len=torch.tensor([n], dtype=torch.int32, device="cuda"))
    out, tok = torch.empty_like(x), torch.empty(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        B.logits_dev(out, x, tok, adj)
        for t in (17, 4321):
            s = np.float64(0)
            for i in range(n):
                if int(ids[0, i]) == t:
                    s += np.float64(b[0, i].item())
            assert out[0, t].item() == np.float32(s)


# --------------------------------------------------------------- together

def test_verification_step():
    """The operators as one step uses them: rotate and cache the drafted rows,
    rotate the queries, attend over context and tree, rotate the outputs back,
    project to logits, adjust and choose -- eagerly and as one captured graph."""
    g = gen(21)
    b, t, h, d, rd, tail, page, ctx, v = 2, 4, 64, 512, 64, 64, 64, 300, 2000
    cfg = B.rope_cfg(rd, 1.6e5, factor=16.0, orig=65536)
    per = -(-(ctx + t) // page)
    c = B.KvCache.empty(b * per, page, d, tail)
    pages = torch.randperm(b * per, generator=g, device="cuda").to(torch.int32).view(b, per)
    j = torch.arange(ctx + t, device="cuda")
    slots = pages.long()[:, j // page] * page + j % page
    rows = normal(g, b, ctx + t, d)
    B.kv_write_dev(c, rows[:, :ctx].reshape(-1, d).contiguous(), slots[:, :ctx].reshape(-1), rope=cfg,
                   pos=j[:ctx].int().repeat(b))
    parents = [-1, 0, 0, 1]
    mask = torch.from_numpy(B.tree_mask(parents)).cuda().expand(b, t).contiguous()
    depth = torch.tensor([0, 1, 1, 2], dtype=torch.int32, device="cuda")
    pos = (ctx + depth).repeat(b)
    q32, head = normal(g, b * t, h, d), normal(g, h * d, v) * 0.01
    new = rows[:, ctx:].reshape(-1, d).contiguous()
    at = slots[:, ctx:].reshape(-1).contiguous()
    k = dict(c=c, pages=pages, ctx=torch.full((b,), ctx, dtype=torch.int32, device="cuda"), nd=None, mask=mask,
             q=torch.empty((b, t, h, d), dtype=torch.bfloat16, device="cuda"), sink=normal(g, h), scale=d ** -0.5,
             max_ctx=ctx)
    o = torch.empty_like(k["q"])
    back = torch.empty((b * t, h, d), device="cuda")
    lg, tok = torch.empty((b * t, v), device="cuda"), torch.empty(b * t, dtype=torch.int32, device="cuda")
    scratch = torch.empty(B.tree_attn_scratch(h, d, t, b, ctx), dtype=torch.uint8, device="cuda")
    hist = torch.randint(0, v, (b * t, 30), generator=g, device="cuda", dtype=torch.int32)
    adj = B.LogitAdjust(hist=hist, hist_len=torch.full((b * t,), 30, dtype=torch.int32, device="cuda"),
                        rep=torch.full((b * t,), 1.2, device="cuda"))

    def step():
        B.kv_write_dev(c, new, at, rope=cfg, pos=pos)
        B.rope_dev(k["q"].view(b * t, h, d), q32, pos, cfg, d - rd)
        run_tree(k, out=o, scratch=scratch)
        B.rope_dev(back, o.view(b * t, h, d), pos, cfg, d - rd, inverse=True)
        torch.matmul(back.view(b * t, -1), head, out=lg)
        B.logits_dev(lg, lg, tok, adj)

    step()
    want, size = turned(q32, pos, cfg, d - rd, False)
    close(k["q"].view(b * t, h, d), want, rope_tol(want, size, torch.bfloat16))
    plain = dict(k, nd=torch.full((b,), t, dtype=torch.int32, device="cuda"))
    ow, tol = plain_tree(plain)
    close(o, ow, tol)
    bw, size = turned(o.view(b * t, h, d), pos, cfg, d - rd, True)
    close(back, bw, rope_tol(bw, size, torch.float32))
    assert tok.tolist() == greedy(lg)
    first = (o.clone(), lg.clone(), tok.clone())
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                             # the projection's library set-up stays out of the capture
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        step()
    for x in (o, lg, tok):
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, first[0]) and torch.equal(lg, first[1]) and torch.equal(tok, first[2])


def test_python_refusals():
    c = B.KvCache.empty(2, 16, 128, 64)
    x = torch.zeros((3, 128), device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    cfg = B.rope_cfg(64, 1e4)
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: B.kv_write_dev(c, x[:, :64], slots), lambda: B.kv_write_dev(c, x.double(), slots),
                lambda: B.kv_write_dev(c, x, slots.int()), lambda: B.kv_write_dev(c, x, slots[:2]),
                lambda: B.kv_write_dev(c, x, slots.cpu()), lambda: B.kv_write_dev(c, x.cpu(), slots),
                lambda: B.kv_write_dev(c, x, slots, rope=cfg), lambda: B.kv_read_dev(x.t(), c, slots),
                lambda: B.rope_dev(x.view(3, 1, 128), x.view(3, 1, 128), pos.long(), cfg, 0),
                lambda: B.rope_dev(x.view(3, 2, 64), x.view(3, 1, 128), pos, cfg, 0),
                lambda: B.KvCache(c.codes, c.scales[:1], 128, 64), lambda: B.KvCache(c.codes, c.scales, 160, 32),
                lambda: B.KvCache(c.codes.cpu(), c.scales.cpu(), 128, 64), lambda: B.KvCache.empty(2, 12, 128, 64),
                lambda: B.logits_dev(x, x.half(), None), lambda: B.LogitAdjust(rep=torch.ones(3, device="cuda")),
                lambda: B.LogitAdjust(hist=slots[None].int()),
                lambda: B.logits_dev(x, x, None, B.LogitAdjust(mask=torch.zeros((2, 4), dtype=torch.int32, device="cuda")))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        B.rope_dev(x.view(3, 1, 128), x.view(3, 1, 128), pos, cfg, 65)       # past the head's end
    with pytest.raises(RuntimeError):
        B.logits_dev(None, x, torch.zeros(3, dtype=torch.int32, device="cuda"),
                     B.LogitAdjust(mask=torch.zeros((3, 3), dtype=torch.int32, device="cuda")))


def test_on_a_second_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x = torch.randn((3, 2, 64), device="cuda:1")
    out = torch.empty_like(x)
    cfg = B.rope_cfg(64, 1e4)
    B.rope_dev(out, x, torch.arange(3, dtype=torch.int32, device="cuda:1"), cfg, 0)
    torch.cuda.synchronize("cuda:1")
    assert torch.cuda.current_device() == 0
    assert torch.allclose(out[0], x[0])
