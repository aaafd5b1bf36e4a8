"""The tree-verification operators' host side where a call is allowed but
unusual. CPU only: without a device an accepted call gets as far as its launch,
which fails with -2, and a refused one returns -1."""
import ctypes as C

import numpy as np
import pytest

import dsv4_b200 as B
import test_tree_cpu as T

P, Q = T.P, T.Q


def test_scratch_grows_with_every_size():
    """Scratch for the largest call is enough for every smaller one, to the call's own check."""
    rng = np.random.default_rng(0)
    top = 1024, 576, 64, 65535, 1 << 30
    for _ in range(3000):
        big = [int(np.exp(rng.uniform(0, np.log(m)))) for m in top]
        big[1] = 64 * (1 + big[1] * 9 // 577)
        big[4] -= 1
        small = [int(rng.integers(1, m + 1)) for m in big[:4]] + [0]
        small[1], small[4] = big[1], int(rng.integers(0, big[4] + 1))
        a, b = B.tree_attn_scratch(*small), B.tree_attn_scratch(*big)
        assert 16 <= a <= b <= 220 << 20, (small, big)


def test_a_smaller_call_takes_the_largest_call_s_scratch():
    T.no_device()
    room = B.tree_attn_scratch(64, 512, 16, 64, 32768)
    for batch in (64, 16, 8, 4, 2, 1):
        for tok in (16, 5, 1):
            args = dict(o=P, q=Q << 4, dt=B.BF16, o_tok=64 * 512, q_tok=64 * 512, c=T.cache(n_pages=40000), pages=P,
                        max_pages=513, ctx=P, n_draft=None, mask=P, sink=None, n_heads=64, n_tok=tok, batch=batch,
                        max_ctx=32768, scale=0.1, scratch=P, bytes=room, stream=None)
            assert T.call("dsv4b_tree_attn", args) == -2, (batch, tok)


def test_selftest_refusals():
    T.no_device()
    f = B.lib().dsv4b_tree_attn_selftest
    assert f(1000, None) == -2
    for bad in (0, -1, 1000001):
        assert f(bad, None) == -1


def test_rope_takes_heads_by_heads():
    """out may lie heads first, in place too; overlapping heads are refused."""
    T.no_device()
    c = B.rope_cfg(64, 1e4)
    args = dict(T.ROPE, cfg=C.byref(c), out_tok=512, out_head=3 * 512)
    assert T.call("dsv4b_rope", args) == -2
    assert T.call("dsv4b_rope", args, x_tok=512, x_head=3 * 512) == -2
    assert T.call("dsv4b_rope", args, x=P, x_dt=B.F32, x_tok=512, x_head=3 * 512) == -2
    for bad in (dict(out_head=3 * 512 - 1), dict(out_tok=511), dict(out_tok=0), dict(out_tok=-512),
                dict(x=P, x_dt=B.F32)):
        assert T.call("dsv4b_rope", args, **bad) == -1, bad


def test_column_ranges_of_one_array_do_not_overlap():
    """Input and output as parts of the same rows, tokens or heads."""
    T.no_device()
    c = B.rope_cfg(64, 1e4)
    w, h, n = 512, 8, 3
    rope = dict(T.ROPE, cfg=C.byref(c), x_dt=B.F32, x=P, out_tok=2 * h * w, x_tok=2 * h * w)
    assert T.call("dsv4b_rope", rope, out=P + 4 * h * w) == -2               # heads 8 .. 15 of each token
    assert T.call("dsv4b_rope", rope, out=P, x=P + 4 * h * w) == -2
    heads = dict(rope, out_head=2 * w, x_head=2 * w)
    assert T.call("dsv4b_rope", heads, out=P + 4 * w) == -2                  # the second half of each head
    by_head = dict(rope, out_tok=w, x_tok=w, out_head=2 * n * w, x_head=2 * n * w)
    assert T.call("dsv4b_rope", by_head, out=P + 4 * n * w) == -2
    for bad in (dict(rope, out=P + 4 * h * w - 4), dict(rope, out=P + 4 * h * w + 4), dict(heads, out=P + 4 * w - 4),
                dict(heads, out=P + 4 * w + 4), dict(by_head, out=P + 4 * n * w + 4),
                dict(rope, out=P + 4 * h * w, x_tok=2 * h * w + 1), dict(rope, out=P + 4 * h * w, x_dt=B.BF16),
                dict(rope, out=P + 4 * w, x_head=0, x_tok=w)):
        assert T.call("dsv4b_rope", bad) == -1
    assert T.call("dsv4b_rope", rope, out=P + 4 * h * w, x_head=0) == -2     # one head of x for all
    t = 64 * 512
    attn = dict(o=P + 2 * t, q=P, dt=B.BF16, o_tok=2 * t, q_tok=2 * t, c=T.cache(), pages=P, max_pages=16, ctx=P,
                n_draft=None, mask=P, sink=None, n_heads=64, n_tok=8, batch=2, max_ctx=1000, scale=0.1, scratch=P,
                bytes=B.tree_attn_scratch(64, 512, 8, 2, 1000), stream=None)
    assert T.call("dsv4b_tree_attn", attn) == -2 and T.call("dsv4b_tree_attn", attn, o=P, q=P + 2 * t) == -2
    assert T.call("dsv4b_tree_attn", attn, o=P + 2 * t - 16) == -1 and T.call("dsv4b_tree_attn", attn, q_tok=t) == -1
    lg = dict(out=P + 4000, x=P, dt=B.F32, os=2000, xs=2000, token=P, adj=None, rows=3, vocab=1000, stream=None)
    assert T.call("dsv4b_logits", lg) == -2
    assert T.call("dsv4b_logits", lg, out=P + 3996) == -1 and T.call("dsv4b_logits", lg, xs=1000) == -1


def test_sizes_past_32_bits_are_refused():
    """Not cut to their low 32 bits."""
    far = 1 << 32
    for bad in ((64 + far, 512, 1, 1, 1), (64, 512 + far, 1, 1, 1), (64, 512, 1 + far, 1, 1), (64, 512, 1, 1 + far, 1),
                (64, 512, 1, 1, 1 + far), (64, 512, 1, 1, -far)):
        with pytest.raises(ValueError):
            B.tree_attn_scratch(*bad)
    for bad in (dict(rd=64 + far), dict(layout=far), dict(orig=far + 8)):
        with pytest.raises(ValueError):
            B.rope_cfg(**dict(dict(rd=64, base=1e4), **bad))
