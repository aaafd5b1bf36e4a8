// tree_attn.cu - attention of a tree of drafted tokens over the quantised
// paged cache. For drafted token t of sequence b and head h
//
//   o = sum_j p_j v_j / (sum_j p_j + exp(sink_h - M)),  p_j = exp(s_j - M),
//   s_j = scale * (q . v_j),   v_j = the cache row of position j (keys and
//   values are the same rows, one KV head for all heads),
//
// over the context positions j < ctx[b] and over the drafted positions
// ctx[b] + k whose bit k is set in mask[b][t]. The sink counts in the
// denominator only (src/core/dsv4_attn.c:84-92); with nothing to attend to
// the output is zero. Tokens t >= n_draft[b] are not written.
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tree.h"

namespace dsv4b {

constexpr int TA_W = 8;                             // heads (warps) per block
constexpr int TA_E = DSV4B_KVQ_MAX_D / 64;          // element pairs per lane

// grid (n_tok, ceil(heads / TA_W), batch); a warp owns one head's running
// maximum, sum and output; lane l holds elements 64 k + 2 l, 2 l + 1.
template <int DT>
__global__ void __launch_bounds__(TA_W * 32)
k_tree_attn_simple(const __grid_constant__ TreeAttn a)
{
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, b = blockIdx.z, lane = threadIdx.x & 31, h = blockIdx.y * TA_W + (threadIdx.x >> 5);
    const int nd = a.n_draft ? min(max(__ldcg(a.n_draft + b), 0), a.n_tok) : a.n_tok;
    if (h >= a.n_heads || t >= nd) return;
    const int ctx = min(max(__ldcg(a.ctx + b), 0), a.max_ctx), d = a.c.d, dq = d - a.c.tail;
    const unsigned long long mask = __ldcg(a.mask + (size_t)b * a.n_tok + t);
    const size_t qi = ((size_t)b * a.n_tok + t) * a.q_tok + (size_t)h * d;
    float2 q[TA_E], o[TA_E];
#pragma unroll
    for (int k = 0; k < TA_E; k++) {
        const int e = 64 * k + 2 * lane;
        q[k] = o[k] = make_float2(0.f, 0.f);
        if (e < d) q[k] = make_float2(ld_row1<DT>(a.q, qi + e), ld_row1<DT>(a.q, qi + e + 1));
    }
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < ctx + nd; j++) {
        if (j >= ctx && !((mask >> (j - ctx)) & 1)) continue;
        const int pg = __ldcg(a.pages + (size_t)b * a.max_pages + j / a.c.page_rows);
        if (pg < 0 || pg >= a.c.n_pages) continue;
        const size_t slot = (size_t)pg * a.c.page_rows + j % a.c.page_rows;
        const unsigned char *row = (const unsigned char *)a.c.codes + slot * (d + a.c.tail);
        const float s = e8m0(__ldcg((const unsigned char *)a.c.scales + slot));
        float2 v[TA_E];
        float acc = 0.f;
#pragma unroll
        for (int k = 0; k < TA_E; k++) {
            const int e = 64 * k + 2 * lane;
            v[k] = make_float2(0.f, 0.f);
            if (e < dq) v[k] = e4m3x2(__ldcg((const unsigned short *)(row + e)));
            else if (e < d) {
                const unsigned u = __ldcg((const unsigned *)(row + dq + 2 * (e - dq)));
                v[k] = __half22float2(*(const __half2 *)&u);
            }
            acc += q[k].x * v[k].x + q[k].y * v[k].y;
        }
        const float z = warp_sum_f(acc) * s * a.scale, mn = fmaxf(m, z), f = m == -INFINITY ? 0.f : expf(m - mn);
        const float p = expf(z - mn);
        l = l * f + p;
        m = mn;
#pragma unroll
        for (int k = 0; k < TA_E; k++) {
            o[k].x = o[k].x * f + p * s * v[k].x;
            o[k].y = o[k].y * f + p * s * v[k].y;
        }
    }
    if (a.sink && l > 0.f) l += expf(a.sink[h] - m);
    const float inv = m == -INFINITY ? 0.f : 1.0f / l;
    const size_t oi = ((size_t)b * a.n_tok + t) * a.o_tok + (size_t)h * d;
#pragma unroll
    for (int k = 0; k < TA_E; k++) {
        const int e = 64 * k + 2 * lane;
        if (e < d) {
            st_row1<DT>(a.o, oi + e, o[k].x * inv);
            st_row1<DT>(a.o, oi + e + 1, o[k].y * inv);
        }
    }
}

size_t tree_attn_bytes(int n_heads, int d, int n_tok, int batch, int max_ctx)
{
    return 16;
}

int tree_attn(const TreeAttn &a, void *scratch, cudaStream_t st)
{
    const dim3 grid(a.n_tok, (a.n_heads + TA_W - 1) / TA_W, a.batch);
    if (a.dt == DSV4B_BF16) launch(k_tree_attn_simple<DSV4B_BF16>, grid, dim3(TA_W * 32), 0, st, a);
    else launch(k_tree_attn_simple<DSV4B_F16>, grid, dim3(TA_W * 32), 0, st, a);
    return cudaPeekAtLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace dsv4b
