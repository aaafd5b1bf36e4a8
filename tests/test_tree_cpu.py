"""The tree-verification operators' host side: frequencies, ancestor masks,
scratch sizes, and the refusal of bad arguments before any device work. CPU
only: without a device an accepted call gets as far as its launch, which fails
with -2, and a refused one returns -1."""
import ctypes as C

import numpy as np
import pytest

import dsv4_b200 as B


def yarn(rd, base, factor, orig, fast, slow):
    """The reference's scaled frequencies (src/core/dsv4_rope.c:48-99)."""
    i = np.arange(rd // 2)
    f = base ** (-2.0 * i / rd)
    if orig:
        at = [rd * np.log(orig / (b * 2 * np.pi)) / (2 * np.log(base)) for b in (fast, slow)]
        lo, hi = max(0, np.floor(at[0])), min(rd - 1, np.ceil(at[1]))
        ramp = np.clip((i - lo) / ((hi - lo) or 0.001), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    return f


@pytest.mark.parametrize("rd,base,factor,orig", [(64, 1e4, 1.0, 0), (64, 1.6e5, 16.0, 65536), (2, 1e4, 4.0, 8),
                                                 (256, 5e5, 8.0, 8192), (34, 1e4, 16.0, 65536)])
def test_rope_frequencies(rd, base, factor, orig):
    c = B.rope_cfg(rd, base, factor=factor, orig=orig)
    want = yarn(rd, base, factor, orig, 32.0, 1.0)
    got = np.array(c.freq[:rd // 2])
    assert np.max(np.abs(got / want - 1)) < 1e-14     # a few roundings of pow and the blend in double
    assert not any(c.freq[rd // 2:]) and c.rd == rd and c.layout == B.ROPE_INTERLEAVED


@pytest.mark.parametrize("bad", [dict(rd=0), dict(rd=3), dict(rd=258), dict(rd=-2), dict(layout=2), dict(base=1.0),
                                 dict(base=float("nan")), dict(factor=0.0), dict(factor=float("inf")), dict(orig=-1),
                                 dict(orig=4, beta_fast=0.0), dict(orig=4, beta_slow=float("nan"))])
def test_rope_init_refuses(bad):
    with pytest.raises(RuntimeError):
        B.rope_cfg(**dict(dict(rd=64, base=1e4), **bad))


def test_tree_mask():
    assert list(B.tree_mask([-1, 0, 0, 2, -1])) == [1, 3, 5, 13, 16]
    chain = B.tree_mask(list(range(-1, 63)))
    assert chain[63] == -1 and chain[0] == 1             # 64 ancestors fill the word
    for bad in ([0], [-1, 1], [-2], [-1] * 65):
        with pytest.raises(ValueError):
            B.tree_mask(bad)


@pytest.mark.parametrize("bad", [(0, 512, 1, 1, 1), (1025, 512, 1, 1, 1), (64, 500, 1, 1, 1), (64, 640, 1, 1, 1),
                                 (64, 512, 0, 1, 1), (64, 512, 65, 1, 1), (64, 512, 1, 0, 1), (64, 512, 1, 65536, 1),
                                 (64, 512, 1, 1, -1)])
def test_scratch_refuses(bad):
    with pytest.raises(ValueError):
        B.tree_attn_scratch(*bad)


def test_scratch_is_bounded():
    """Scratch covers every split of every row tile and no more than a few
    hundred of them for any context."""
    assert B.tree_attn_scratch(64, 512, 1, 1, 0) >= 16
    a, b = B.tree_attn_scratch(64, 512, 1, 1, 1 << 20), B.tree_attn_scratch(64, 512, 1, 1, 1 << 30)
    assert 0 < a <= 1 << 28 and 0 < b <= 1 << 28


# ------------------------------------------------------------- refusals
# One accepted call per entry, then the same call with one argument changed.

P = 1 << 20                    # an aligned address that no call dereferences on the host
Q = 1 << 30


def no_device():
    if B.lib().dsv4_cuda_available():
        pytest.skip("launches with made-up addresses: only without a device")


def call(name, args, **change):
    a = dict(args)
    for k, v in change.items():
        assert k in a, k
        a[k] = v
    return getattr(B.lib(), name)(*a.values())


ROPE = dict(out=P, out_dt=B.F32, out_tok=512 * 8, out_head=512, x=Q, x_dt=B.BF16, x_tok=512 * 8, x_head=512, cfg=None,
            pos=P, n_tok=3, n_heads=8, width=512, first=448, inverse=0, stream=None)


def test_rope_refusals():
    no_device()
    c = B.rope_cfg(64, 1e4)
    args = dict(ROPE, cfg=C.byref(c))
    assert call("dsv4b_rope", args) == -2
    for ok in (dict(x_head=0), dict(x_tok=0), dict(first=0), dict(n_tok=1, out_tok=512 * 8),
               dict(x=P, x_dt=B.F32), dict(x=P + 3 * 512 * 8 * 4)):
        assert call("dsv4b_rope", args, **ok) == -2, ok
    for none in (dict(n_tok=0), dict(n_heads=0)):
        assert call("dsv4b_rope", args, **none) == 0
    for bad in (dict(out=None), dict(x=None), dict(pos=None), dict(cfg=None), dict(out_dt=B.E4M3), dict(x_dt=4),
                dict(x_dt=-1), dict(out=P + 2), dict(x=Q + 1), dict(pos=P + 2), dict(n_tok=-1), dict(n_heads=-1),
                dict(width=0), dict(first=-1), dict(first=449), dict(width=32), dict(out_head=511),
                dict(out_tok=511 * 8), dict(x_head=-1), dict(x_tok=-512),
                dict(x=P), dict(x=P + 512, x_dt=B.F32)):            # overlapping, not in place
        assert call("dsv4b_rope", args, **bad) == -1, bad
    for bad in ((63, 0), (258, 0), (64, 2), (0, 0)):
        c2 = B.RopeCfg()
        c2.rd, c2.layout = bad
        assert call("dsv4b_rope", args, cfg=C.byref(c2)) == -1


CACHE = dict(codes=P, scales=P, n_pages=10, page_rows=64, d=512, tail=64)
BAD_CACHES = (dict(codes=None), dict(scales=None), dict(codes=P + 8), dict(n_pages=0), dict(n_pages=1 << 31),
              dict(page_rows=0), dict(page_rows=48), dict(page_rows=1 << 17), dict(d=0), dict(d=500), dict(d=640),
              dict(tail=-64), dict(tail=32), dict(tail=576))


def cache(**change):
    return C.byref(B.KvqC(*dict(CACHE, **change).values()))


def test_kv_refusals():
    no_device()
    r = B.rope_cfg(64, 1e4)
    write = dict(c=cache(), rows=Q, dt=B.BF16, stride=512, slots=P, n=5, rope=C.byref(r), pos=P, stream=None)
    read = dict(c=cache(), out=Q, dt=B.F16, stride=512, slots=P, n=5, stream=None)
    assert call("dsv4b_kv_write", write) == -2 and call("dsv4b_kv_read", read) == -2
    assert call("dsv4b_kv_write", write, rope=None, pos=None) == -2
    assert call("dsv4b_kv_write", write, n=0) == 0 and call("dsv4b_kv_read", read, n=0) == 0
    for bad in BAD_CACHES:
        assert call("dsv4b_kv_write", write, c=cache(**bad)) == -1, bad
        assert call("dsv4b_kv_read", read, c=cache(**bad)) == -1, bad
    for bad in (dict(c=None), dict(dt=B.E4M3), dict(stride=511), dict(slots=None), dict(slots=P + 4), dict(n=-1)):
        assert call("dsv4b_kv_write", write, **bad) == -1, bad
        assert call("dsv4b_kv_read", read, **bad) == -1, bad
    for bad in (dict(rows=None), dict(rows=Q + 1), dict(pos=None), dict(pos=P + 1)):
        assert call("dsv4b_kv_write", write, **bad) == -1, bad
    for bad in (dict(out=None), dict(out=Q + 1)):
        assert call("dsv4b_kv_read", read, **bad) == -1, bad
    long = B.rope_cfg(256, 1e4)
    assert call("dsv4b_kv_write", write, c=cache(d=128), stride=128, rope=C.byref(long)) == -1


def test_tree_attn_refusals():
    no_device()
    n = B.tree_attn_scratch(64, 512, 8, 2, 1000)
    args = dict(o=P, q=Q, dt=B.BF16, o_tok=64 * 512, q_tok=64 * 512, c=cache(), pages=P, max_pages=16, ctx=P,
                n_draft=None, mask=P, sink=None, n_heads=64, n_tok=8, batch=2, max_ctx=1000, scale=0.1, scratch=P,
                bytes=n, stream=None)
    assert call("dsv4b_tree_attn", args) == -2
    for ok in (dict(n_draft=P), dict(sink=P), dict(q_tok=64 * 512 + 8), dict(max_ctx=0)):
        assert call("dsv4b_tree_attn", args, **ok) == -2, ok
    assert call("dsv4b_tree_attn", args, batch=0) == 0 and call("dsv4b_tree_attn", args, n_tok=0) == 0
    for bad in BAD_CACHES:
        assert call("dsv4b_tree_attn", args, c=cache(**bad)) == -1, bad
    for bad in (dict(o=None), dict(q=None), dict(c=None), dict(pages=None), dict(ctx=None), dict(mask=None),
                dict(scratch=None), dict(o=P + 8), dict(q=Q + 2), dict(pages=P + 1), dict(ctx=P + 2), dict(mask=P + 4),
                dict(sink=P + 1), dict(n_draft=P + 1), dict(scratch=P + 8), dict(dt=B.F32), dict(dt=B.E4M3),
                dict(o_tok=64 * 512 - 8), dict(q_tok=64 * 512 + 4), dict(n_heads=0), dict(n_heads=1025),
                dict(n_tok=65), dict(n_tok=-1), dict(batch=-1), dict(batch=65536), dict(max_ctx=-1),
                dict(max_ctx=16 * 64 - 7), dict(max_pages=0), dict(max_pages=15), dict(bytes=n - 1),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(q=P), dict(q=P + 16 * 64 * 512)):
        assert call("dsv4b_tree_attn", args, **bad) == -1, bad


def test_tree_attn_refuses_caches_past_its_offsets():
    """A row's place is kept in 32 bits of 64-byte steps."""
    no_device()
    args = dict(o=P, q=Q, dt=B.BF16, o_tok=64 * 512, q_tok=64 * 512, c=None, pages=P, max_pages=16, ctx=P, n_draft=None,
                mask=P, sink=None, n_heads=64, n_tok=8, batch=2, max_ctx=1000, scale=0.1, scratch=P,
                bytes=B.tree_attn_scratch(64, 512, 8, 2, 1000), stream=None)
    steps = (512 + 64) // 64
    most = (2 ** 32 - 2) // steps // 64                   # pages of 64 rows
    assert call("dsv4b_tree_attn", args, c=cache(n_pages=most)) == -2
    assert call("dsv4b_tree_attn", args, c=cache(n_pages=most + 1)) == -1
    assert call("dsv4b_tree_attn", args, c=cache(n_pages=2 ** 31 - 1)) == -1


def test_status_without_a_device():
    no_device()
    assert B.lib().dsv4b_tree_attn_status() == -1


def test_logits_refusals():
    no_device()
    full = dict(hist=P, hist_stride=9, hist_len=P, n_prompt=P, rep=P, freq=P, pres=P, bias_ids=P, bias=P,
                bias_stride=4, bias_len=P, mask=P, mask_stride=32)

    def adj(**change):
        return C.byref(B.LogitAdjustC(*dict(full, **change).values()))

    args = dict(out=P, x=Q, dt=B.F32, os=1000, xs=1000, token=P, adj=adj(), rows=3, vocab=1000, stream=None)
    assert call("dsv4b_logits", args) == -2
    for ok in (dict(adj=None), dict(out=None), dict(token=None), dict(out=Q), dict(adj=adj(n_prompt=None, rep=None)),
               dict(adj=adj(mask=None)), dict(adj=adj(bias=None, bias_ids=None))):
        assert call("dsv4b_logits", args, **ok) == -2, ok
    assert call("dsv4b_logits", args, rows=0) == 0
    for bad in (dict(x=None), dict(out=None, token=None), dict(dt=B.E4M3), dict(dt=7), dict(os=999), dict(xs=999),
                dict(rows=-1), dict(vocab=0), dict(out=Q + 4), dict(out=Q, os=1001), dict(x=Q + 2), dict(out=P + 1),
                dict(token=P + 2), dict(adj=adj(hist_len=None)), dict(adj=adj(hist=None)), dict(adj=adj(hist_stride=-1)),
                dict(adj=adj(bias_ids=None)), dict(adj=adj(bias_len=None)), dict(adj=adj(bias=None)),
                dict(adj=adj(bias_stride=-1)), dict(adj=adj(mask_stride=31)), dict(adj=adj(mask=P + 2))):
        assert call("dsv4b_logits", args, **bad) == -1, bad
    assert call("dsv4b_logits", args, adj=adj(hist_stride=1 << 30)) == -2
    for bad in (adj(hist_stride=(1 << 30) + 1), adj(bias_stride=(1 << 30) + 1)):
        assert call("dsv4b_logits", args, adj=bad) == -1
