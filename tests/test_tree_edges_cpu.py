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
