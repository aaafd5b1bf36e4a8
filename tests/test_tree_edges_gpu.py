"""The tree-verification operators on the B200 where a call is allowed but
unusual: cache rows of very different magnitude, layouts, streams, scratch of
another size, errors of earlier calls. Against the same 64-bit definitions and
roundings as test_tree_gpu.py.
"""
import os
import subprocess
import sys

import pytest

import dsv4_b200 as B
import test_tree_gpu as T

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DT, close, gen, normal = T.DT, T.close, T.gen, T.normal


@pytest.fixture(scope="module", autouse=True)
def dev():
    return B.init()


# ---------------------------------------------- rows of different magnitude

def slots_of(k, b, n):
    page = k["c"].codes.shape[1]
    j = torch.arange(n, device="cuda")
    return k["pages"][b].long()[j // page] * page + j % page


def weighted(k):
    """o and its tolerance in double, where every error counts with the weight
    of its key, so that rows without weight lend no slack:

    * a score is a float sum whose partial sums are off by at most 2^-22 of the
      key's sum of magnitudes, d / 16 + 4 of them (f16 products are exact; q is
      held in f16 to 2^-38 of its largest element at least);
    * exponents are below 2^9 and rounded in float (2^-16), ex2 adds 2^-22: a
      weight and the sum of weights each move by less than 2^-15;
    * a weight is rounded to f16: 2^-11 of it, or half the smallest step, 2^-25,
      where the row's largest is held at 2^7 / sqrt(2) or more: 2^-31.5 of the
      largest p times scale, for each code;
    * the output is rounded once, past the type's largest value to infinity."""
    q, c = k["q"], k["c"]
    b, t, h, d = q.shape
    want = torch.full(q.shape, 11.0, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    rel, tiny = T.unit(q.dtype)
    for i in range(b):
        n, m = int(k["ctx"][i]), int(k["nd"][i])
        slot = slots_of(k, i, n + m)
        v = T.decode(c, slot)
        s = T.two(c.scales.view(-1)[slot].long() - 127)
        for a in range(m):
            bits = int(k["mask"][i, a])
            see = torch.ones(n + m, dtype=torch.bool, device="cuda")
            for z in range(m):
                see[n + z] = bool((bits >> z) & 1)
            w, sc = v[see], s[see]
            x = q[i, a].double()
            z = x @ w.T * k["scale"]
            top = z.amax(-1, keepdim=True)
            p = (z - top).exp()
            den = p.sum(-1, keepdim=True) + (k["sink"].double()[:, None] - top).exp()
            want[i, a] = p @ w / den
            delta = abs(k["scale"]) * ((d / 16 + 4) * 2.0 ** -22 * (x.abs() @ w.abs().T)
                                       + 2.0 ** -38 * x.abs().amax(-1, keepdim=True) * w.abs().sum(-1))
            pd = torch.where(p > 0, p * delta, 0.0)
            size = p @ w.abs() / den
            low = 2.0 ** -31.5 * (p * sc).amax(-1, keepdim=True) * (w.abs() / sc[:, None]).sum(0) / den
            tol[i, a] = ((pd @ w.abs()) / den + size * (2.0 ** -11 + 2.0 ** -15 + pd.sum(-1, keepdim=True) / den) + low
                         + rel * 1.001 * want[i, a].abs() + tiny)
    f = torch.finfo(q.dtype)
    return torch.where(want.abs() >= f.max * (1 + f.eps / 4), want * float("inf"), want), tol


@pytest.mark.parametrize("g", [0, 4, 8, 14, 18, 22, 26, 40, 100])
@pytest.mark.parametrize("where", ["opposite", "hidden", "both"])
@pytest.mark.parametrize("b,t,h,ctx,dtype", [(1, 3, 64, 700, "bf16"), (2, 2, 4, 1500, "f16"), (150, 2, 8, 300, "bf16")])
def test_small_rows_beside_large_ones(g, where, b, t, h, ctx, dtype):
    """Rows 2^g larger than the rest that weigh nothing (opposite to q) or are
    hidden from every token but their own: the small rows carry the output."""
    d = 512
    k = T.tree_case(60 + g, b, t, h, d, 64, 64, ctx, DT[dtype])
    u = normal(gen(61), d).sign()
    k["q"] = (normal(gen(62), b, t, h, d) + u).to(DT[dtype])
    rows = normal(gen(63), k["c"].scales.numel(), d)
    for i in range(b):
        at = slots_of(k, i, ctx + t)
        if where != "hidden":
            rows[at[[3, ctx // 2, ctx - 1]]] = -u * 2.0 ** g
        if where != "opposite":
            rows[at[ctx + t - 1]] = u * 2.0 ** g             # the last token's own row
    k["mask"] &= ~(1 << (t - 1))
    if where == "hidden" and g < 30:
        k["mask"][0, t - 1] |= 1 << (t - 1)                  # one token sees it: that row alone carries its output
    B.kv_write_dev(k["c"], rows, torch.arange(rows.shape[0], device="cuda"))
    want, tol = weighted(k)
    close(T.run_tree(k), want, tol)


def test_rows_of_every_magnitude():
    """Scales over 200 powers of two in one context, each scale's rows among
    the heaviest for some head; zero rows between them."""
    d, n = 256, 900
    k = T.tree_case(70, 2, 2, 16, d, 64, 64, n, torch.bfloat16)
    g = gen(71)
    rows = normal(g, k["c"].scales.numel(), d) * torch.exp2(torch.randint(-100, 4, (k["c"].scales.numel(), 1), generator=g,
                                                                         device="cuda").float())
    rows[::5] = 0.0
    B.kv_write_dev(k["c"], rows, torch.arange(rows.shape[0], device="cuda"))
    want, tol = weighted(k)
    close(T.run_tree(k), want, tol)


@pytest.mark.parametrize("f", [2.0 ** -120, 2.0 ** -126, 2.0 ** 110])
def test_rows_at_the_ends_of_the_scales(f):
    """Rows whose scale byte is 0 or near it (float's subnormal numbers among
    them), and rows near float's largest; zero rows between them."""
    k = T.tree_case(80, 2, 3, 16, 128, 64, 64, 700, torch.bfloat16)
    rows = normal(gen(81), k["c"].scales.numel(), 128)
    rows[::9] = 0.0
    rows[1::9] *= 2.0 ** -6
    B.kv_write_dev(k["c"], rows * f, torch.arange(rows.shape[0], device="cuda"))
    k["scale"] = min(128 ** -0.5 / f, 2.0 ** 100)
    want, tol = weighted(k)
    close(T.run_tree(k), want, tol)


# ------------------------------------------------------------------- layouts

@pytest.mark.parametrize("n,h,w,rd,first,layout,src,dst", [(5, 8, 512, 64, 448, 0, "f32", "bf16"), (33, 3, 64, 32, 16, 1, "bf16", "f32"),
                                                           (7, 4, 37, 34, 3, 0, "f16", "f16"), (200, 2, 24, 8, 8, 1, "f32", "f32")])
def test_rope_heads_first(n, h, w, rd, first, layout, src, dst):
    """[heads, tokens, width] seen as [tokens, heads, width], in x, out or both, and in place."""
    g = gen(n)
    cfg = B.rope_cfg(rd, 1e4, layout=layout)
    x = normal(g, n, h, w).to(DT[src])
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    want, size = T.turned(x, pos, cfg, first, False)
    xt = x.transpose(0, 1).contiguous()
    for a in (x, xt.transpose(0, 1)):
        out = torch.full((h, n + 2, w), 7.0, dtype=DT[dst], device="cuda")
        B.rope_dev(out[:, 1:1 + n].transpose(0, 1), a, pos, cfg, first)
        close(out[:, 1:1 + n].transpose(0, 1), want, T.rope_tol(want, size, DT[dst]))
        assert torch.all(out[:, 0] == 7.0) and torch.all(out[:, 1 + n:] == 7.0)
    B.rope_dev(xt.transpose(0, 1), xt.transpose(0, 1), pos, cfg, first)
    close(xt.transpose(0, 1), want, T.rope_tol(want, size, DT[src]))


def test_parts_of_one_array():
    """Input and output beside each other in the same tokens, heads or rows."""
    g = gen(55)
    cfg = B.rope_cfg(32, 1e4)
    buf = normal(g, 6, 4, 128)
    x, pos = buf[..., :64].clone(), torch.arange(6, dtype=torch.int32, device="cuda") * 9
    want, size = T.turned(x, pos, cfg, 16, False)
    B.rope_dev(buf[..., 64:], buf[..., :64], pos, cfg, 16)
    close(buf[..., 64:], want, T.rope_tol(want, size, torch.float32))
    assert torch.equal(buf[..., :64], x)
    k = T.tree_case(56, 2, 3, 8, 128, 64, 64, 300, torch.bfloat16)
    ref = T.run_tree(k)
    both = torch.cat((k["q"], torch.full_like(k["q"], 11.0)), 2)
    T.run_tree(dict(k, q=both[:, :, :8]), out=both[:, :, 8:])
    assert torch.equal(both[:, :, 8:], ref) and torch.equal(both[:, :, :8], k["q"])
    rows = torch.cat((3 * normal(g, 5, 1000), torch.zeros((5, 1000), device="cuda")), 1)
    B.logits_dev(rows[:, 1000:], rows[:, :1000], None)
    assert torch.equal(rows[:, 1000:], rows[:, :1000])


# ------------------------------------------------------------------- scratch

def test_one_scratch_for_smaller_calls():
    """Scratch of the largest call, its bytes NaN, serves smaller batches, trees
    and contexts, which are cut otherwise."""
    h, d = 64, 128
    room = torch.empty(B.tree_attn_scratch(h, d, 16, 40, 6000), dtype=torch.uint8, device="cuda")
    for b, t, ctx in ((40, 16, 900), (16, 16, 2000), (3, 2, 6000), (1, 1, 6000), (40, 1, 300), (1, 16, 0)):
        k = T.tree_case(90 + b, b, t, h, d, 64, 64, ctx, torch.bfloat16, ragged=b > 1)
        room.fill_(255)
        want, tol = T.plain_tree(k)
        close(T.run_tree(k, scratch=room), want, tol)


# -------------------------------------------------------------------- status

def test_status_waits_for_every_stream():
    """A call that is still queued on a side stream has ended before its status
    is given."""
    k = T.tree_case(95, 1, 1, 8, 128, 64, 64, 300, torch.bfloat16)
    ref = T.run_tree(k)
    out = torch.full_like(ref, 11.0)
    room = torch.empty(B.tree_attn_scratch(8, 128, 1, 1, 300), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                     # about 50 ms
        T.run_tree(k, out=out, scratch=room)
    assert B.lib().dsv4b_tree_attn_status() == 0
    assert side.query()
    assert torch.equal(out, ref)


def test_status_reports_a_wait_once():
    """A wait that ran out is in the next status, and not in the one after."""
    assert B.tree_attn_status()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert B.lib().dsv4b_tree_attn_selftest(1000, side.cuda_stream) == 0
    assert not B.tree_attn_status()
    assert B.tree_attn_status() and B.lib().dsv4b_tree_attn_status() == 0
    k = T.tree_case(96, 1, 1, 8, 128, 64, 64, 300, torch.bfloat16)
    want, tol = T.plain_tree(k)
    close(T.run_tree(k), want, tol)
    assert B.tree_attn_status(torch.cuda.current_device())


# -------------------------------------------------------------------- errors

def test_an_earlier_error_is_not_this_call_s():
    """An allocation of this library that failed (824 GB, refused at once) leaves
    its error code behind; launches that follow succeed, and say so. In a
    process of its own, as the code stays there."""
    code = """
import ctypes as C, numpy as np, torch, dsv4_b200 as B, test_tree_gpu as T
B.init()
buf = np.zeros(4, np.float32)
fail = C.CDLL(B.LIB_PATH).dsv4b_peer_selftest
fail.argtypes = [C.c_int, C.c_int, C.c_uint, C.c_int, C.c_void_p, C.c_void_p]
assert fail(64, (1 << 30) - 4, 1, 1, buf.ctypes.data, buf.ctypes.data) == -1
x = T.normal(T.gen(57), 2, 3, 64)
out, pos = torch.empty_like(x), torch.arange(2, dtype=torch.int32, device="cuda")
B.rope_dev(out, x, pos, B.rope_cfg(64, 1e4), 0)
c, at = B.KvCache.empty(1, 16, 64, 0), torch.arange(2, device="cuda")
B.kv_write_dev(c, x[:, 0].contiguous(), at)
B.kv_read_dev(out[:, 0], c, at)
B.logits_dev(None, x[:, 0], torch.empty(2, dtype=torch.int32, device="cuda"))
k = T.tree_case(58, 1, 2, 8, 128, 64, 64, 2000, torch.bfloat16)
want, tol = T.plain_tree(k)
T.close(T.run_tree(k), want, tol)
print("every launch succeeded")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join((here, os.path.dirname(B.LIB_PATH))))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "every launch succeeded" in r.stdout, r.stderr


# ------------------------------------------------------------------- streams

def test_memory_of_a_call_on_another_stream_is_kept():
    """Tensors dropped while a side stream has yet to run the call that reads or
    writes them: their memory is not given out before."""
    side = torch.cuda.Stream()
    g = gen(59)
    cfg = B.rope_cfg(64, 1e4)
    cache = B.KvCache.empty(4, 64, 512, 64)
    k = T.tree_case(60, 1, 2, 8, 128, 64, 64, 2000, torch.bfloat16)
    hist = torch.randint(0, 3000, (5, 700), generator=g, device="cuda", dtype=torch.int32)
    ref = T.run_tree(k)

    def calls(stream):
        """A call of each kind on tensors of its own; the outputs, and where the rest lay."""
        x, pos = normal(gen(1), 300, 2, 512), torch.arange(300, dtype=torch.int32, device="cuda")
        rows, slots = normal(gen(2), 200, 512), torch.arange(200, device="cuda")
        lg, rep = 3 * normal(gen(3), 5, 3000), torch.full((5,), 1.3, device="cuda")
        adj = B.LogitAdjust(hist=hist.clone(), hist_len=torch.full((5,), 700, dtype=torch.int32, device="cuda"), rep=rep)
        q, mask = k["q"].clone(), k["mask"].clone()
        scratch = torch.empty(B.tree_attn_scratch(8, 128, 2, 1, 2000), dtype=torch.uint8, device="cuda")
        outs = [torch.zeros_like(x), torch.zeros((200, 512), device="cuda"), torch.zeros_like(lg),
                torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros_like(q)]
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                torch.cuda._sleep(200_000_000)             # about 100 ms
        B.rope_dev(outs[0], x, pos, cfg, 0, stream=stream)
        B.kv_write_dev(cache, rows, slots, rope=cfg, pos=pos[:200], stream=stream)
        B.kv_read_dev(outs[1], cache, slots, stream=stream)
        B.logits_dev(outs[2], lg, outs[3], adj, stream=stream)
        T.run_tree(dict(k, q=q, mask=mask), out=outs[4], scratch=scratch, stream=stream)
        return outs, [t.data_ptr() for t in (x, pos, rows, slots, lg, rep, adj.keep[0], adj.keep[1], q, mask, scratch)], \
            [(t.shape, t.dtype) for t in (x, pos, rows, slots, lg, rep, adj.keep[0], adj.keep[1], q, mask, scratch)]

    want = calls(None)[0]
    torch.cuda.synchronize()
    got, at, kinds = calls(side)
    later = [torch.zeros(s, dtype=d, device="cuda") for s, d in kinds for _ in range(3)]
    assert not side.query()                                # the calls are still to come
    assert not {t.data_ptr() for t in later} & set(at)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(got[4], ref)


def test_sizes_past_32_bits_are_refused():
    far = 1 << 32
    x = torch.zeros((3, 1, 128), device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    k = T.tree_case(97, 1, 1, 8, 128, 64, 64, 60, torch.bfloat16)
    scratch = torch.empty(B.tree_attn_scratch(8, 128, 1, 1, 60), dtype=torch.uint8, device="cuda")
    for bad in (lambda: B.rope_dev(x, x, pos, B.rope_cfg(64, 1e4), far), lambda: T.run_tree(dict(k, max_ctx=60 + far), scratch=scratch)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------- values and sizes

def test_query_rows_that_are_not_finite_spoil_no_others():
    for dtype in (torch.bfloat16, torch.float16):
        k = T.tree_case(100, 2, 3, 16, 256, 64, 64, 900, dtype)
        want, tol = T.plain_tree(k)
        ref = T.run_tree(k)
        bad = torch.zeros(k["q"].shape[:3], dtype=torch.bool, device="cuda")
        k["q"][0, 1, 3, 7], k["q"][1, 2, 15, 255], k["q"][1, 0, 0] = float("nan"), float("inf"), -float("inf")
        bad[0, 1, 3] = bad[1, 2, 15] = bad[1, 0, 0] = True
        out = T.run_tree(k)
        assert torch.isnan(out[bad]).all()
        close(out[~bad], want[~bad], tol[~bad])
        assert torch.equal(out[~bad], ref[~bad])


@pytest.mark.parametrize("scale", [0.0, -0.05, 2.0 ** -140])
def test_scales_of_any_sign(scale):
    k = dict(T.tree_case(101, 2, 3, 16, 256, 64, 64, 900, torch.bfloat16), scale=scale)
    want, tol = T.plain_tree(k)
    close(T.run_tree(k), want, tol)


def test_sinks_at_their_ends():
    """An infinite sink takes everything, one of -infinity nothing, NaN its own head."""
    k = T.tree_case(102, 2, 2, 8, 128, 64, 64, 1500, torch.bfloat16)
    free, tol = T.plain_tree(dict(k, sink=None))
    want, tol2 = T.plain_tree(k)
    k["sink"][1], k["sink"][2], k["sink"][3] = float("inf"), -float("inf"), float("nan")
    out = T.run_tree(k)
    assert not out[:, :, 1].any() and torch.isnan(out[:, :, 3]).all()
    close(out[:, :, 2], free[:, :, 2], tol[:, :, 2])
    for h in (0, 4, 5, 6, 7):
        close(out[:, :, h], want[:, :, h], tol2[:, :, h])


def test_most_heads_and_tokens():
    k = T.tree_case(103, 1, 64, 1024, 64, 0, 64, 200, torch.bfloat16)
    out = T.run_tree(k)
    for t in (0, 1, 31, 63):
        part = dict(k, q=k["q"][:, t:t + 1], mask=k["mask"][:, t:t + 1])
        # one token's row of the definition: its mask over all 64 drafted rows
        n = 200 + 64
        v = T.decode(k["c"], slots_of(k, 0, n))
        see = torch.ones(n, dtype=torch.bool, device="cuda")
        bits = int(part["mask"][0, 0])
        for z in range(64):
            see[200 + z] = bool((bits >> z) & 1)
        z = part["q"][0, 0].double() @ v[see].T * k["scale"]
        w = torch.cat((z, k["sink"].double()[:, None]), -1).softmax(-1)[:, :-1]
        mag = (k["scale"] * part["q"][0, 0].double().abs() @ v[see].abs().T).amax(-1, keepdim=True)
        delta = mag * 8 * 2.0 ** -22 + 2.0 ** -15               # d / 16 + 4 partial sums of a score, as above
        want = w @ v[see]
        size = w @ v[see].abs()
        close(out[0, t], want, size * (2.0 ** -11 + 2 * delta) + 2.0 ** -20 * v.abs().amax() + 2.0 ** -8 * 1.001 * want.abs())


def test_a_given_stream_inside_a_capture():
    """stream= naming the stream that is being captured."""
    k = T.tree_case(104, 1, 2, 8, 128, 64, 64, 900, torch.bfloat16)
    ref = T.run_tree(k)
    out = torch.full_like(ref, 11.0)
    scratch = torch.empty(B.tree_attn_scratch(8, 128, 2, 1, 900), dtype=torch.uint8, device="cuda")
    x = 3 * normal(gen(105), 2, 5000)
    tok, first = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    B.logits_dev(None, x, first)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        T.run_tree(k, out=out, scratch=scratch, stream=side)
        B.logits_dev(None, x, tok, stream=side)
    for _ in range(2):
        out.fill_(11.0)
        tok.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(tok, first)


def test_more_rows_of_logits_than_a_launch_takes():
    r, v = 32770, 40
    g = gen(106)
    x = 3 * normal(g, r, v)
    kw = dict(hist=torch.randint(0, v, (r, 5), generator=g, device="cuda", dtype=torch.int32),
              hist_len=torch.randint(0, 6, (r,), generator=g, device="cuda", dtype=torch.int32),
              n_prompt=torch.randint(0, 3, (r,), generator=g, device="cuda", dtype=torch.int32),
              rep=0.5 + torch.rand(r, generator=g, device="cuda"), freq=0.3 * normal(g, r), pres=normal(g, r),
              bias_ids=torch.randint(0, v, (r, 3), generator=g, device="cuda", dtype=torch.int32), bias=normal(g, r, 3),
              bias_len=torch.full((r,), 3, dtype=torch.int32, device="cuda"),
              mask=torch.randint(-2 ** 31, 2 ** 31, (r, 2), generator=g, device="cuda").to(torch.int32))
    out, tok = torch.empty_like(x), torch.empty(r, dtype=torch.int32, device="cuda")
    B.logits_dev(out, x, tok, B.LogitAdjust(**kw))
    rows = torch.tensor([0, 1, 32766, 32767, 32768, 32769], device="cuda")
    part = {n: t[rows] for n, t in kw.items()}
    want, size = T.plain_logits(x[rows], part["hist"], part["hist_len"], part["n_prompt"], part["rep"], part["freq"],
                                part["pres"], part["bias_ids"], part["bias"], part["bias_len"], part["mask"])
    # at most six float roundings on the way, then the output's
    close(out[rows], want, 6.01 * T.U32 * size + T.U32 * (1 + 2 ** -20) * want.abs().nan_to_num(posinf=0) + 2.0 ** -149)
    top = out.amax(-1)
    first = torch.where(out == top[:, None], torch.arange(v, device="cuda"), v).amin(-1)
    assert torch.equal(tok.long(), torch.where(top > -float("inf"), first, -1))


@pytest.mark.parametrize("g", [-60, 0, 20, 60, 90])
def test_hidden_nan_rows_at_any_magnitude(g):
    """A NaN row that one token sees and the others do not, among rows near 2^g."""
    k = T.tree_case(107, 1, 4, 16, 128, 64, 64, 500, torch.bfloat16)
    rows = normal(gen(108), k["c"].scales.numel(), 128) * 2.0 ** g
    at = slots_of(k, 0, 504)
    rows[at[502]] = float("nan")
    k["mask"][0] = torch.tensor([1, 3, 4, 11], device="cuda")
    B.kv_write_dev(k["c"], rows, torch.arange(rows.shape[0], device="cuda"))
    k["scale"] *= 2.0 ** -g
    out = T.run_tree(k)
    assert torch.isnan(out[0, 2]).all()
    B.kv_write_dev(k["c"], torch.zeros((1, 128), device="cuda"), at[502:503])
    want, tol = weighted(k)
    keep = torch.tensor([0, 1, 3], device="cuda")
    close(out[:, keep], want[:, keep], tol[:, keep])
