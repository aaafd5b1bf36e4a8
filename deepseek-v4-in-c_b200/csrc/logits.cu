// logits.cu - adjusting a row of logits before a token is chosen, and the
// greedy choice. For token v of a row, in this order, each step rounded to
// float and off where its array is absent:
//
//   seen in the history:  x > 0 ? x / rep : x * rep
//   c = its count among the generated part of the history:
//                         x -= freq * c;  if c > 0:  x -= pres
//   biases:               x += the row's biases for v (summed in double)
//   grammar:              x = -inf where v's bit is clear
//
// and token = the lowest index of the largest x (of the stored, rounded
// value), -1 when no x is above -inf; a NaN is never chosen.
//
// Bound by HBM at many rows (2 * vocab * size a row) and by latency at one. A
// cluster of 8 blocks owns a row: each block takes runs of the vocabulary,
// counts the history that falls into its run in shared memory (integer
// atomics, so the order of arrival cannot show), and makes one pass over the
// logits; the blocks' best (value, index) pairs meet in the first block's
// shared memory, so the greedy token needs neither scratch nor a second
// launch.
#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tree.h"

namespace cg = cooperative_groups;

namespace dsv4b {

constexpr int LG_C = 8;                 // blocks of a row (a portable cluster)
constexpr int LG_T = 512;
constexpr int LG_RUN = 8192;            // tokens handled at once: 32 KB of counters, 32 KB of bias links

// A history word in shared memory: the count of generated occurrences, and
// the top bit when the token occurs in the prompt.
constexpr unsigned LG_SEEN = 0x80000000u;
// A bias link: the first list entry of the token, and a bit when there are
// more.
constexpr unsigned LG_NONE = 0xFFFFFFFFu, LG_MORE = 0x80000000u;

struct LogitsCall {
    void *out;
    const void *x;
    long out_stride, x_stride;
    int *token;
    dsv4b_logit_adjust a;
    int vocab, run;
};

// (value, index): larger value, ties to the lower index; index -1 = none.
__device__ __forceinline__ void better(float &v, int &i, float ov, int oi)
{
    if (oi >= 0 && (i < 0 || ov > v || (ov == v && oi < i))) {
        v = ov;
        i = oi;
    }
}

template <int DT, bool VEC>
__global__ void __cluster_dims__(LG_C, 1, 1) __launch_bounds__(LG_T)
k_logits(LogitsCall c)
{
    pdl_trigger();
    pdl_wait();
    extern __shared__ unsigned cnt[];           // [run]
    unsigned *link = cnt + c.run;               // [run] when there are biases
    __shared__ float sv[LG_T / 32], best_v[LG_C];
    __shared__ int si[LG_T / 32], best_i[LG_C];
    const int row = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x;
    const dsv4b_logit_adjust &a = c.a;
    const char *x = reinterpret_cast<const char *>(c.x) + (size_t)row * c.x_stride * row_dt_size(DT);
    char *out = c.out ? reinterpret_cast<char *>(c.out) + (size_t)row * c.out_stride * row_dt_size(DT) : nullptr;
    const int *hist = a.hist ? a.hist + (size_t)row * a.hist_stride : nullptr;
    const int hl = hist ? min(__ldcg(a.hist_len + row), (int)min(a.hist_stride, 0x7fffffffL)) : 0;
    const int np = hist && a.n_prompt ? __ldcg(a.n_prompt + row) : 0;
    const int *bid = a.bias ? a.bias_ids + (size_t)row * a.bias_stride : nullptr;
    const float *bias = a.bias ? a.bias + (size_t)row * a.bias_stride : nullptr;
    const int bl = bias ? min(__ldcg(a.bias_len + row), (int)min(a.bias_stride, 0x7fffffffL)) : 0;
    const unsigned *mask = a.mask ? a.mask + (size_t)row * a.mask_stride : nullptr;
    const float rep = a.rep ? __ldcg(a.rep + row) : 1.0f, freq = a.freq ? __ldcg(a.freq + row) : 0.0f;
    const float pres = a.pres ? __ldcg(a.pres + row) : 0.0f;
    float bv = -INFINITY;
    int bi = -1;
    // every block of the cluster has started before one writes to the first
    if (c.token) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    for (int r0 = rank * c.run; r0 < c.vocab; r0 += LG_C * c.run) {
        const int m = min(c.run, c.vocab - r0);
        if (hist || bias) {
            __syncthreads();                    // the counters of the run before are read
            for (int i = tid; i < m; i += LG_T) {
                if (hist) cnt[i] = 0;
                if (bias) link[i] = LG_NONE;
            }
            __syncthreads();
            for (int i = tid; i < hl; i += LG_T) {
                const unsigned k = (unsigned)(__ldcg(hist + i) - r0);
                if (k < (unsigned)m) {
                    if (i >= np) atomicAdd(cnt + k, 1u);
                    else atomicOr(cnt + k, LG_SEEN);
                }
            }
            for (int i = tid; i < bl; i += LG_T) {
                const unsigned k = (unsigned)(__ldcg(bid + i) - r0);
                if (k < (unsigned)m) atomicMin(link + k, (unsigned)i);
            }
            __syncthreads();
            if (bl > 1) {
                for (int i = tid; i < bl; i += LG_T) {
                    const unsigned k = (unsigned)(__ldcg(bid + i) - r0);
                    if (k < (unsigned)m && (link[k] & ~LG_MORE) != (unsigned)i) atomicOr(link + k, LG_MORE);
                }
                __syncthreads();
            }
        }
        auto adjust = [&](int k, float v, unsigned bits) {
            if (hist) {
                const unsigned w = cnt[k];
                if (w) {
                    const unsigned n = w & ~LG_SEEN;
                    v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    if (n) {
                        v = __fsub_rn(v, __fmul_rn(freq, (float)n));
                        v = __fsub_rn(v, pres);
                    }
                }
            }
            if (bias) {
                const unsigned l = link[k];
                if (l != LG_NONE) {
                    const int i = (int)(l & ~LG_MORE);
                    double s = (double)__ldcg(bias + i);
                    if (l & LG_MORE)            // the token's other entries, in list order
                        for (int j = i + 1; j < bl; j++)
                            if (__ldcg(bid + j) == r0 + k) s += (double)__ldcg(bias + j);
                    v = __fadd_rn(v, (float)s);
                }
            }
            return (bits & 1u) ? v : -INFINITY;
        };
        if constexpr (VEC) {
            const int groups = (m + 7) >> 3;
            for (int g = tid; g < groups; g += LG_T) {
                const int k0 = g << 3;
                float v[8];
                const int left = min(8, m - k0);
                if (left == 8) {
                    widen8<DT>(ld_raw8<DT, true>(x, (size_t)r0 + k0), v);
                } else {
                    for (int j = 0; j < 8; j++) v[j] = j < left ? ld_row1<DT>(x, (size_t)r0 + k0 + j) : -INFINITY;
                }
                const unsigned w = mask ? __ldcg(mask + ((r0 + k0) >> 5)) >> ((r0 + k0) & 31) : 0xFFu;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (j >= left) break;
                    v[j] = adjust(k0 + j, v[j], w >> j);
                    if constexpr (DT == DSV4B_BF16) v[j] = __bfloat162float(__float2bfloat16_rn(v[j]));
                    if constexpr (DT == DSV4B_F16) v[j] = __half2float(__float2half_rn(v[j]));
                    if (v[j] > bv) bv = v[j], bi = r0 + k0 + j;
                }
                if (out) {
                    if (left == 8) st_row8<DT, true>(out, (size_t)r0 + k0, v);
                    else
                        for (int j = 0; j < left; j++) st_row1<DT>(out, (size_t)r0 + k0 + j, v[j]);
                }
            }
        } else {
            for (int k = tid; k < m; k += LG_T) {
                const int t = r0 + k;
                const unsigned w = mask ? __ldcg(mask + (t >> 5)) >> (t & 31) : 1u;
                float v = adjust(k, ld_row1<DT>(x, (size_t)t), w);
                if constexpr (DT == DSV4B_BF16) v = __bfloat162float(__float2bfloat16_rn(v));
                if constexpr (DT == DSV4B_F16) v = __half2float(__float2half_rn(v));
                if (v > bv) bv = v, bi = t;
                if (out) st_row1<DT>(out, (size_t)t, v);
            }
        }
    }
    if (!c.token) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
    if ((tid & 31) == 0) sv[tid >> 5] = bv, si[tid >> 5] = bi;
    __syncthreads();
    cg::cluster_group cl = cg::this_cluster();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid == 0) {
        for (int w = 1; w < LG_T / 32; w++) better(bv, bi, sv[w], si[w]);
        *cl.map_shared_rank(&best_v[rank], 0) = bv;
        *cl.map_shared_rank(&best_i[rank], 0) = bi;
    }
    cl.sync();
    if (rank == 0 && tid == 0) {
        for (int w = 1; w < LG_C; w++) better(bv, bi, best_v[w], best_i[w]);
        c.token[row] = bi;
    }
}

int logits(void *out, const void *x, int dt, long out_stride, long x_stride, int *token,
           const dsv4b_logit_adjust &a, int rows, int vocab, cudaStream_t st)
{
    if (rows <= 0 || vocab <= 0) return 0;
    LogitsCall c = {out, x, out_stride, x_stride, token, a, vocab, 0};
    const int share = ((vocab + LG_C - 1) / LG_C + 31) & ~31;     // whole mask words a run
    c.run = share < LG_RUN ? share : LG_RUN;
    const int sz = row_dt_size(dt);
    const bool vec = !(((uintptr_t)x | (uintptr_t)out) & 15) && !((x_stride * sz) & 15) && !((out_stride * sz) & 15);
    const size_t smem = (size_t)c.run * 4 * (a.bias ? 2 : 1);
    DSV4B_ROW_DT(dt, DT, {
        if (smem_optin(k_logits<DT, true>, LG_RUN * 8) || smem_optin(k_logits<DT, false>, LG_RUN * 8)) return -2;
        for (int r0 = 0; r0 < rows; r0 += 32768) {
            const int nr = rows - r0 < 32768 ? rows - r0 : 32768;
            LogitsCall p = c;
            p.x = reinterpret_cast<const char *>(x) + (size_t)r0 * x_stride * sz;
            if (out) p.out = reinterpret_cast<char *>(out) + (size_t)r0 * out_stride * sz;
            if (token) p.token = token + r0;
            if (a.hist) p.a.hist += (size_t)r0 * a.hist_stride, p.a.hist_len += r0;
            if (a.n_prompt) p.a.n_prompt += r0;
            if (a.rep) p.a.rep += r0;
            if (a.freq) p.a.freq += r0;
            if (a.pres) p.a.pres += r0;
            if (a.bias) p.a.bias += (size_t)r0 * a.bias_stride, p.a.bias_ids += (size_t)r0 * a.bias_stride, p.a.bias_len += r0;
            if (a.mask) p.a.mask += (size_t)r0 * a.mask_stride;
            if (vec) launch(k_logits<DT, true>, dim3(LG_C, nr), dim3(LG_T), smem, st, p);
            else launch(k_logits<DT, false>, dim3(LG_C, nr), dim3(LG_T), smem, st, p);
        }
    });
    return cudaPeekAtLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace dsv4b
