// capi_tree.cu - C ABI of the tree-verification operators: argument checks,
// then the kernels. Every check runs on the host before any device work, so a
// refused call (-1) has touched nothing.
#include <math.h>

#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tree.h"

using namespace dsv4b;

namespace {

bool row_dt(int dt) { return dt == DSV4B_F32 || dt == DSV4B_BF16 || dt == DSV4B_F16; }

bool cache_ok(const dsv4b_kvq *c)
{
    if (!c || !c->codes || !c->scales || ((uintptr_t)c->codes & 15)) return false;
    if (c->d < 64 || c->d > DSV4B_KVQ_MAX_D || (c->d & 63) || c->tail < 0 || c->tail > c->d || (c->tail & 63)) return false;
    if (c->page_rows < 1 || c->page_rows > 65536 || (c->page_rows & (c->page_rows - 1))) return false;
    return c->n_pages > 0 && c->n_pages <= 0x7fffffffL;
}

bool rope_arg(const dsv4b_rope_cfg *r, RopeArg &a)
{
    if (!r || r->rd < 2 || r->rd > DSV4B_ROPE_MAX || (r->rd & 1)) return false;
    if (r->layout != DSV4B_ROPE_INTERLEAVED && r->layout != DSV4B_ROPE_HALF) return false;
    for (int i = 0; i < kRopePairs; i++) a.freq[i] = i < r->rd / 2 ? r->freq[i] : 0.0;
    a.rd = r->rd;
    a.half = r->layout == DSV4B_ROPE_HALF;
    return true;
}

// A strided array [n0][n1][n2] in bytes; strides in elements, all >= 0.
struct Span {
    uintptr_t at;
    long n[2], step[2], row;
    Span(const void *p, int size, long n0, long s0, long n1, long s1, long n2)
        : at((uintptr_t)p), n{n0, n1}, step{s0 * size, s1 * size}, row(n2 * size)
    {
    }
    // Bytes past `at` that its elements reach, by their place modulo `period`
    // (0: their place itself).
    uintptr_t reach(long period) const
    {
        uintptr_t r = (uintptr_t)row;
        for (int i = 0; i < 2; i++)
            if (period == 0 || step[i] % period) r += (uintptr_t)(n[i] - 1) * step[i];
        return r;
    }
    // Whether an element may lie in both: not when the whole ranges are apart,
    // or the places within a common period (column ranges of one wider array).
    bool meets(const Span &o) const
    {
        if (at + reach(0) <= o.at || o.at + o.reach(0) <= at) return false;
        for (long p : step) {
            if (p <= 0) continue;
            const uintptr_t d = (o.at % p + p - at % p) % p;
            if (d >= reach(p) && d + o.reach(p) <= (uintptr_t)p) return false;
        }
        return true;
    }
};

bool aligned(const void *p, size_t n) { return ((uintptr_t)p % n) == 0; }

}  // namespace

extern "C" int dsv4b_rope_init(dsv4b_rope_cfg *r, int rd, int layout, double base, double factor, int orig,
                               double beta_fast, double beta_slow)
{
    if (!r || rd < 2 || rd > DSV4B_ROPE_MAX || (rd & 1)) return -1;
    if (layout != DSV4B_ROPE_INTERLEAVED && layout != DSV4B_ROPE_HALF) return -1;
    if (!(base > 1.0) || !isfinite(base) || !(factor > 0.0) || !isfinite(factor) || orig < 0) return -1;
    if (orig > 0 && (!(beta_fast > 0.0) || !(beta_slow > 0.0) || !isfinite(beta_fast) || !isfinite(beta_slow))) return -1;
    double lo = 0.0, hi = 0.0;
    if (orig > 0) {         // src/core/dsv4_rope.c:48-99
        const double twopi = 2.0 * 3.14159265358979323846;
        lo = floor((double)rd * log((double)orig / (beta_fast * twopi)) / (2.0 * log(base)));
        hi = ceil((double)rd * log((double)orig / (beta_slow * twopi)) / (2.0 * log(base)));
        if (lo < 0.0) lo = 0.0;
        if (hi > rd - 1) hi = rd - 1;
        if (lo == hi) hi += 0.001;
    }
    for (int i = 0; i < DSV4B_ROPE_MAX / 2; i++) {
        double f = 0.0;
        if (i < rd / 2) {
            f = 1.0 / pow(base, (double)(2 * i) / (double)rd);
            if (orig > 0) {
                double ramp = ((double)i - lo) / (hi - lo);
                ramp = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
                f = f / factor * ramp + f * (1.0 - ramp);
            }
        }
        r->freq[i] = f;
    }
    r->rd = rd;
    r->layout = layout;
    return 0;
}

extern "C" int dsv4b_rope(void *out, int out_dt, long out_tok, long out_head, const void *x, int x_dt, long x_tok,
                          long x_head, const dsv4b_rope_cfg *r, const int *pos, int n_tok, int n_heads, int width,
                          int first, int inverse, void *stream)
{
    RopeArg a;
    if (!row_dt(out_dt) || !row_dt(x_dt) || !rope_arg(r, a) || n_tok < 0 || n_heads < 0 || width < 1) return -1;
    if (first < 0 || first > width - a.rd) return -1;
    if (n_tok == 0 || n_heads == 0) return 0;
    const int os = row_dt_size(out_dt), xs = row_dt_size(x_dt);
    if (!out || !x || !pos || !aligned(out, os) || !aligned(x, xs) || !aligned(pos, 4)) return -1;
    if (x_head < 0 || x_tok < 0) return -1;
    // no two heads of out overlap: a token's heads lie together, or a head's tokens
    if (!(out_head >= width && out_tok >= (long)(n_heads - 1) * out_head + width) &&
        !(out_tok >= width && out_head >= (long)(n_tok - 1) * out_tok + width))
        return -1;
    const bool inplace = out == x && out_dt == x_dt && out_tok == x_tok && out_head == x_head;
    if (!inplace && Span(out, os, n_tok, out_tok, n_heads, out_head, width)
                        .meets(Span(x, xs, n_tok, x_tok, n_heads, x_head, width)))
        return -1;
    const RopeCall c = {out, x, out_dt, x_dt, out_tok, out_head, x_tok, x_head, pos, n_tok, n_heads, width, first,
                        inverse ? 1 : 0, inplace ? 1 : 0};
    return rope(c, a, stream_of(stream));
}

extern "C" int dsv4b_kv_write(const dsv4b_kvq *c, const void *rows, int dt, long row_stride, const long long *slots,
                              int n, const dsv4b_rope_cfg *r, const int *pos, void *stream)
{
    RopeArg a;
    if (!cache_ok(c) || !row_dt(dt) || n < 0) return -1;
    if (r && (!rope_arg(r, a) || a.rd > c->d)) return -1;
    if (n == 0) return 0;
    if (!rows || !slots || row_stride < c->d || !aligned(rows, row_dt_size(dt)) || !aligned(slots, 8)) return -1;
    if (r && (!pos || !aligned(pos, 4))) return -1;
    return kv_write(*c, rows, dt, row_stride, slots, n, r ? &a : nullptr, pos, stream_of(stream));
}

extern "C" int dsv4b_kv_read(const dsv4b_kvq *c, void *out, int dt, long row_stride, const long long *slots, int n,
                             void *stream)
{
    if (!cache_ok(c) || !row_dt(dt) || n < 0) return -1;
    if (n == 0) return 0;
    if (!out || !slots || row_stride < c->d || !aligned(out, row_dt_size(dt)) || !aligned(slots, 8)) return -1;
    return kv_read(*c, out, dt, row_stride, slots, n, stream_of(stream));
}

static bool tree_sizes(int n_heads, int d, int n_tok, int batch, int max_ctx)
{
    return n_heads >= 1 && n_heads <= 1024 && d >= 64 && d <= DSV4B_KVQ_MAX_D && !(d & 63) && n_tok >= 1 &&
           n_tok <= DSV4B_TREE_MAX && batch >= 1 && batch <= 65535 && max_ctx >= 0 && max_ctx <= (1 << 30);
}

extern "C" size_t dsv4b_tree_attn_scratch(int n_heads, int d, int n_tok, int batch, int max_ctx)
{
    return tree_sizes(n_heads, d, n_tok, batch, max_ctx) ? tree_attn_bytes(n_heads, d, n_tok, batch, max_ctx) : 0;
}

extern "C" int dsv4b_tree_attn(void *o, const void *q, int dt, long o_tok, long q_tok, const dsv4b_kvq *c,
                               const int *pages, int max_pages, const int *ctx, const int *n_draft,
                               const unsigned long long *mask, const float *sink, int n_heads, int n_tok, int batch,
                               int max_ctx, float scale, void *scratch, size_t scratch_bytes, void *stream)
{
    if ((dt != DSV4B_BF16 && dt != DSV4B_F16) || !cache_ok(c) || batch < 0 || n_tok < 0) return -1;
    if (batch == 0 || n_tok == 0) return 0;
    if (!tree_sizes(n_heads, c->d, n_tok, batch, max_ctx) || !isfinite(scale)) return -1;
    if (!o || !q || !pages || !ctx || !mask || !scratch) return -1;
    if (!aligned(o, 16) || !aligned(q, 16) || !aligned(pages, 4) || !aligned(ctx, 4) || !aligned(mask, 8) ||
        !aligned(scratch, 16) || !aligned(sink, 4) || !aligned(n_draft, 4))
        return -1;
    // the kernel holds a row's place as 32 bits of 64-byte steps
    if ((long long)c->n_pages * c->page_rows > 0xFFFFFFFEll / ((c->d + c->tail) >> 6)) return -1;
    const long w = (long)n_heads * c->d;
    if (o_tok < w || q_tok < w || (o_tok & 7) || (q_tok & 7)) return -1;
    if (max_pages < 1 || (long long)max_pages * c->page_rows < (long long)max_ctx + n_tok) return -1;
    const long nt = (long)batch * n_tok;
    if (Span(o, 2, nt, o_tok, 1, 0, w).meets(Span(q, 2, nt, q_tok, 1, 0, w))) return -1;
    if (scratch_bytes < tree_attn_bytes(n_heads, c->d, n_tok, batch, max_ctx)) return -1;
    const TreeAttn a = {o, q, dt, o_tok, q_tok, *c, pages, max_pages, ctx, n_draft, mask, sink,
                        n_heads, n_tok, batch, max_ctx, scale};
    return tree_attn(a, scratch, stream_of(stream));
}

extern "C" int dsv4b_tree_attn_status(void) { return tree_attn_status(); }

extern "C" int dsv4b_tree_attn_selftest(int limit_us, void *stream)
{
    if (limit_us < 1 || limit_us > 1000000) return -1;
    return tree_attn_selftest(limit_us, stream_of(stream));
}

extern "C" int dsv4b_logits(void *out, const void *x, int dt, long out_stride, long x_stride, int *token,
                            const dsv4b_logit_adjust *adj, int rows, int vocab, void *stream)
{
    if (!row_dt(dt) || rows < 0 || vocab < 1 || vocab > (1 << 30)) return -1;
    const dsv4b_logit_adjust none = {};
    const dsv4b_logit_adjust a = adj ? *adj : none;
    if (a.hist && (!a.hist_len || a.hist_stride < 0 || a.hist_stride > (1 << 30))) return -1;
    if (!a.hist && (a.rep || a.freq || a.pres || a.n_prompt)) return -1;
    if (a.bias && (!a.bias_ids || !a.bias_len || a.bias_stride < 0 || a.bias_stride > (1 << 30))) return -1;
    if (!a.bias && a.bias_ids) return -1;
    if (a.mask && a.mask_stride < (vocab + 31) / 32) return -1;
    if (rows == 0) return 0;
    if (!x || (!out && !token) || x_stride < vocab || (out && out_stride < vocab)) return -1;
    const int sz = row_dt_size(dt);
    if (!aligned(x, sz) || !aligned(out, sz) || !aligned(token, 4) || !aligned(a.hist, 4) || !aligned(a.bias_ids, 4) ||
        !aligned(a.bias, 4) || !aligned(a.mask, 4))
        return -1;
    // in place, or apart
    if (out && !(out == x && out_stride == x_stride) &&
        Span(out, sz, rows, out_stride, 1, 0, vocab).meets(Span(x, sz, rows, x_stride, 1, 0, vocab)))
        return -1;
    return logits(out, x, dt, out ? out_stride : 0, x_stride, token, a, rows, vocab, stream_of(stream));
}
