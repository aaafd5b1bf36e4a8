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
// cluster of 4 or 8 blocks owns a row; chunks of 64 tokens are dealt to the
// blocks in turn, as the frequent tokens of a text lie together at the low end
// of a vocabulary. Few of a block's tokens are in the history or the bias
// list, so these are settled apart, and the pass over the logits only looks
// up what they became:
//
//   mark     a bitmap of the block's named tokens, and a list of the history
//            that falls to the block
//   place    a slot for each marked token, by prefix sums of the bitmap
//   count    its occurrences and its first bias, by integer atomics, so the
//            order of arrival cannot show
//   settle   its adjusted value, one thread a slot, kept in the slot
//   stream   all its tokens, eight logits a thread at a time: a marked one is
//            taken from its slot; mask, rounding, best value
//
// The blocks' best (value, index) pairs meet in the first block's shared
// memory, so the greedy token needs neither scratch nor a second launch.
//
// Measured at 129280 floats a row: 8.8 us for one row with 600 tokens of
// history (5.7 without), 29 us for 64 rows with up to 8192 (16.1 without
// history and biases, where the traffic alone takes 10.5); the rest is the
// latency of the five steps, which two blocks a multiprocessor overlap only in
// part. A block keeps 4096 entries of the history that fall to it and 2048 named
// tokens; past either it reads the lists again, past the second once for every
// 2048 of its tokens: 167 us for 64 rows with up to 20000 tokens of text, 351
// with up to 60000 (418 with 60000 drawn evenly, 48000 of them distinct); one row
// 20, 87 and 159 us.
#include <cooperative_groups.h>

#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tree.h"

namespace cg = cooperative_groups;

namespace dsv4b {

// Threads of a block, two blocks a multiprocessor. At 64 rows 512 threads take
// 29 us, 256 take 38 (fewer loads in flight) and 1024, one block, 40.
constexpr int LG_T = 512;
constexpr int LG_CHUNK = 64;            // tokens dealt to a block at a time
constexpr int LG_RUN = 65536;           // tokens of a block at a time: 16 bits number them
constexpr int LG_SLOTS = 2048;          // named tokens settled at once; a run with more is cut into parts this long
constexpr int LG_LIST = 4096;           // history entries kept; a longer list is read again

// A slot's count: the generated occurrences, and the top bit when the token
// occurs in the prompt. The same bit of a list entry marks the prompt's.
constexpr unsigned LG_SEEN = 0x80000000u;
constexpr unsigned LG_NONE = 0xFFFFFFFFu;       // a slot without a bias

// Rows that get 8 blocks each; more get 4, which read the history half as
// often. Measured at 129280 floats, 2000 tokens of history, 50 biases, a mask
// (us by 8 / by 4 blocks a row): 1 row 9.5 / 12.1, 16 rows 13.0 / 12.9,
// 32 rows 15.7 / 17.6, 48 rows 27.7 / 21.8, 64 rows 29.6 / 23.0: the step
// comes where the blocks no longer all fit on the device at once.
constexpr int LG_FEW = 36;

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

// Dynamic shared memory of a run of `run` tokens (a multiple of 64).
__host__ __device__ inline size_t lg_smem(int run, bool named, bool bias)
{
    if (!named) return 0;
    return LG_LIST * 4 + LG_SLOTS * (4 + 2) + (bias ? LG_SLOTS * 4 + LG_SLOTS / 8 : 0) + (size_t)run / 32 * (4 + 2);
}

// LG_C blocks a row.
template <int DT, bool VEC, int LG_C>
__global__ void __cluster_dims__(LG_C, 1, 1) __launch_bounds__(LG_T, 2)
k_logits(LogitsCall c)
{
    pdl_trigger();
    pdl_wait();
    extern __shared__ unsigned sm[];
    __shared__ float sv[LG_T / 32], best_v[LG_C];
    __shared__ int si[LG_T / 32], best_i[LG_C];
    __shared__ unsigned n_list, n_slots;
    const int row = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const dsv4b_logit_adjust &a = c.a;
    const char *x = reinterpret_cast<const char *>(c.x) + (size_t)row * c.x_stride * row_dt_size(DT);
    char *out = c.out ? reinterpret_cast<char *>(c.out) + (size_t)row * c.out_stride * row_dt_size(DT) : nullptr;
    const int *hist = a.hist ? a.hist + (size_t)row * a.hist_stride : nullptr;
    const int *bid = a.bias ? a.bias_ids + (size_t)row * a.bias_stride : nullptr;
    const float *bias = a.bias ? a.bias + (size_t)row * a.bias_stride : nullptr;
    const unsigned *mask = a.mask ? a.mask + (size_t)row * a.mask_stride : nullptr;
    const bool named = hist || bias;
    unsigned *list = sm, *cnt = list + LG_LIST, *link = cnt + LG_SLOTS, *many = link + (bias ? LG_SLOTS : 0);
    unsigned *bits = many + (bias ? LG_SLOTS / 32 : 0);
    unsigned short *tok = reinterpret_cast<unsigned short *>(bits + c.run / 32), *base = tok + LG_SLOTS;

    // Number k of the block's run in the run of the cluster that starts at r0.
    auto token_of = [&](int r0, int k) { return r0 + ((k / LG_CHUNK) * LG_C + rank) * LG_CHUNK + k % LG_CHUNK; };
    // eight logits and their mask bits, asked for ahead of their use
    Raw8<DT> nx;
    unsigned nm = 0xFFFFFFFFu;              // the mask's whole word: shifting it here would wait for it
    auto ask = [&](int r0, int k, int end) {
        const int t0 = token_of(r0, k);
        if (k >= end || t0 >= c.vocab) return;
        if (t0 + 8 <= c.vocab) nx = ld_raw8<DT, VEC>(x, (size_t)t0);
        if (mask) nm = __ldcg(mask + (t0 >> 5));
    };
    ask(0, tid * 8, c.run);

    // so is the start of the history, and its length: used only later on
    int ahead[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
        ahead[j] = hist && j * LG_T + tid < a.hist_stride ? __ldcg(hist + j * LG_T + tid) : -1;
    const int hist_len = hist ? __ldcg(a.hist_len + row) : 0, np = hist && a.n_prompt ? __ldcg(a.n_prompt + row) : 0;
    const int bias_len = bias ? __ldcg(a.bias_len + row) : 0;
    const float rep = a.rep ? __ldcg(a.rep + row) : 1.0f, freq = a.freq ? __ldcg(a.freq + row) : 0.0f;
    const float pres = a.pres ? __ldcg(a.pres + row) : 0.0f;
    float bv = -INFINITY;
    int bi = -1;
    // every block of the cluster has started before one writes to the first
    // (relaxed: nothing is handed over, and a release would wait for the loads)
    if (c.token) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    for (long at = 0; at < c.vocab; at += (long)LG_C * c.run) {
        const int r0 = (int)at, here = min(LG_C * c.run, c.vocab - r0);       // the cluster's tokens
        const int chunks = (here + LG_CHUNK - 1) / LG_CHUNK, m = (chunks - rank + LG_C - 1) / LG_C * LG_CHUNK;
        const int hl = min(hist_len, (int)a.hist_stride), bl = min(bias_len, (int)a.bias_stride);
        // the block's number of token r0 + u, ~0 for one that is not its own
        auto number_of = [&](unsigned u) {
            const unsigned q = u / LG_CHUNK;
            return u < (unsigned)here && q % LG_C == (unsigned)rank ? q / LG_C * LG_CHUNK + u % LG_CHUNK : 0xFFFFFFFFu;
        };
        // fn(i, k) for entries from .. n of a list of tokens, four at a time: k
        // the block's number of entry i's token, then of i + LG_T's, and so on;
        // whole warps, the four loads in flight together
        auto each = [&](const int *ids, int from, int n, auto fn) {
            for (int i = from + tid; (i & ~31) < n; i += 4 * LG_T) {
                unsigned k[4];
#pragma unroll
                for (int j = 0; j < 4; j++) k[j] = i + j * LG_T < n ? (unsigned)__ldcg(ids + i + j * LG_T) - (unsigned)r0 : 0xFFFFFFFFu;
#pragma unroll
                for (int j = 0; j < 4; j++) k[j] = number_of(k[j]);
                fn(i, k);
            }
        };
        auto place = [&](int w0, int w1) {      // slots of the marked tokens of bitmap words w0 .. w1
            for (int w = w0 + (tid & ~31); w < w1; w += LG_T) {
                const int n = w + lane < w1 ? __popc(bits[w + lane]) : 0;
                int to = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, to, o);
                    if (lane >= o) to += up;
                }
                unsigned first = 0;
                if (lane == 31) first = atomicAdd(&n_slots, (unsigned)to);
                first = __shfl_sync(0xffffffffu, first, 31);
                if (w + lane < w1) base[w + lane] = (unsigned short)(first + to - n);
            }
            for (int i = tid; i < LG_SLOTS; i += LG_T) {
                cnt[i] = 0;
                if (bias) link[i] = LG_NONE;
            }
            if (bias)
                for (int i = tid; i < LG_SLOTS / 32; i += LG_T) many[i] = 0;
        };
        auto slot_of = [&](unsigned k) { return base[k >> 5] + __popc(bits[k >> 5] & ((1u << (k & 31)) - 1u)); };
        if (named) {
            __syncthreads();                    // the run before is done
            for (int i = tid; i < (m + 31) >> 5; i += LG_T) bits[i] = 0;
            if (tid == 0) n_list = n_slots = 0;
            __syncthreads();
            // (one entry for equal tokens of a warp, found by matching, takes
            // longer than the repeated atomics: 1.5 us at 64 rows)
            auto mark = [&](int i, const unsigned (&k)[4]) {
                unsigned who[4];
                int all = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    who[j] = __ballot_sync(0xffffffffu, k[j] != 0xFFFFFFFFu);
                    all += __popc(who[j]);
                }
                if (!all) return;
                int p = 0;
                if (lane == 0) p = (int)atomicAdd(&n_list, (unsigned)all);
                p = __shfl_sync(0xffffffffu, p, 0);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int at = p + __popc(who[j] & ((1u << lane) - 1u));
                    p += __popc(who[j]);
                    if (k[j] == 0xFFFFFFFFu) continue;
                    atomicOr(bits + (k[j] >> 5), 1u << (k[j] & 31));
                    if (at < LG_LIST) list[at] = k[j] | (i + j * LG_T < np ? LG_SEEN : 0u);
                }
            };
            if (r0 == 0 && (tid & ~31) < hl) {
                unsigned k[4];
#pragma unroll
                for (int j = 0; j < 4; j++) k[j] = j * LG_T + tid < hl ? number_of((unsigned)ahead[j]) : 0xFFFFFFFFu;
                mark(tid, k);
            }
            each(hist, r0 == 0 ? 4 * LG_T : 0, hl, mark);
            each(bid, 0, bl, [&](int, const unsigned (&k)[4]) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (k[j] != 0xFFFFFFFFu) atomicOr(bits + (k[j] >> 5), 1u << (k[j] & 31));
            });
            __syncthreads();
            place(0, (m + 31) >> 5);
            __syncthreads();
        }
        const bool whole = !named || n_slots <= LG_SLOTS;
        const int part = whole ? m : LG_SLOTS;
        for (int s0 = 0; s0 < m; s0 += part) {
            const int len = min(part, m - s0);
            if (!whole) {
                __syncthreads();                // the part before is done
                if (tid == 0) n_slots = 0;
                __syncthreads();
                place(s0 >> 5, (s0 + len + 31) >> 5);
                __syncthreads();
            }
            if (named) {
                auto count = [&](unsigned k, bool prompt) {
                    if (k - s0 >= (unsigned)len) return;
                    const int s = slot_of(k);
                    tok[s] = (unsigned short)k;
                    if (prompt) atomicOr(cnt + s, LG_SEEN);
                    else atomicAdd(cnt + s, 1u);
                };
                const int nl = (int)n_list;
                if (nl <= LG_LIST)
                    for (int i = tid; i < nl; i += LG_T) count(list[i] & ~LG_SEEN, list[i] & LG_SEEN);
                else                            // the list is cut short: the history again
                    each(hist, 0, hl, [&](int i, const unsigned (&k)[4]) {
#pragma unroll
                        for (int j = 0; j < 4; j++) count(k[j], i + j * LG_T < np);
                    });
                each(bid, 0, bl, [&](int i, const unsigned (&k)[4]) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (k[j] - s0 >= (unsigned)len) continue;
                        const int s = slot_of(k[j]);
                        tok[s] = (unsigned short)k[j];
                        if (atomicMin(link + s, (unsigned)(i + j * LG_T)) != LG_NONE)
                            atomicOr(many + (s >> 5), 1u << (s & 31));
                    }
                });
                __syncthreads();
                const int ns = (int)n_slots;
                for (int j0 = tid & ~31; j0 < ns; j0 += LG_T) {
                    const int j = j0 + lane;
                    const bool on = j < ns;
                    const int t = on ? token_of(r0, tok[j]) : 0;
                    const unsigned w = on ? cnt[j] : 0;
                    float v = on ? ld_row1<DT>(x, (size_t)t) : 0.0f;
                    if (w) {
                        const unsigned n = w & ~LG_SEEN;
                        v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                        if (n) {
                            v = __fsub_rn(v, __fmul_rn(freq, (float)n));
                            v = __fsub_rn(v, pres);
                        }
                    }
                    if (bias) {
                        const unsigned l = on ? link[j] : LG_NONE;
                        double s = l != LG_NONE ? (double)__ldcg(bias + l) : 0.0;
                        // a token that is named again: the warp looks for its
                        // other entries and adds them in list order
                        for (unsigned rest = many[j0 >> 5]; rest; rest &= rest - 1) {
                            const int who = __ffs(rest) - 1;
                            const int want = __shfl_sync(0xffffffffu, t, who);
                            for (int i0 = __shfl_sync(0xffffffffu, (int)l, who) + 1; i0 < bl; i0 += 128) {
                                int id[4];
#pragma unroll
                                for (int u = 0; u < 4; u++) {
                                    const int i = i0 + u * 32 + lane;
                                    id[u] = i < bl ? __ldcg(bid + i) : -1;
                                }
#pragma unroll
                                for (int u = 0; u < 4; u++)
                                    for (unsigned hit = __ballot_sync(0xffffffffu, id[u] == want); hit; hit &= hit - 1)
                                        if (lane == who) s += (double)__ldcg(bias + i0 + u * 32 + __ffs(hit) - 1);
                            }
                        }
                        if (l != LG_NONE) v = __fadd_rn(v, (float)s);
                    }
                    if (on) cnt[j] = __float_as_uint(v);
                }
                __syncthreads();
            }
            const int end = s0 + len;
            if (r0 || s0) ask(r0, s0 + tid * 8, end);
            for (int k = s0 + tid * 8; k < end; k += LG_T * 8) {
                const int t0 = token_of(r0, k), left = min(8, c.vocab - t0);
                if (left <= 0) break;
                float v[8];
                if (left == 8) {
                    widen8<DT>(nx, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] = j < left ? ld_row1<DT>(x, (size_t)t0 + j) : -INFINITY;
                }
                const unsigned on = nm >> (t0 & 31);
                ask(r0, k + LG_T * 8, end);
                if (named) {
                    const unsigned its = bits[k >> 5] >> (k & 31) & 0xFFu;
                    if (its) {
                        const unsigned *s = cnt + slot_of(k);
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (its >> j & 1u) v[j] = __uint_as_float(s[__popc(its & ((1u << j) - 1u))]);
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (!(on >> j & 1u)) v[j] = -INFINITY;
                    if constexpr (DT == DSV4B_BF16) v[j] = __bfloat162float(__float2bfloat16_rn(v[j]));
                    if constexpr (DT == DSV4B_F16) v[j] = __half2float(__float2half_rn(v[j]));
                    top = fmaxf(top, v[j]);                     // passes over NaN
                }
                if (top > bv) {
                    bv = top;
#pragma unroll
                    for (int j = 7; j >= 0; j--)
                        if (v[j] == top) bi = t0 + j;
                }
                if (out) {
                    if (left == 8) st_row8<DT, VEC>(out, (size_t)t0, v);
                    else
                        for (int j = 0; j < left; j++) st_row1<DT>(out, (size_t)t0 + j, v[j]);
                }
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
        // the pair is handed over; a releasing barrier would wait for every
        // thread's stores of logits
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
    const int nb = rows <= LG_FEW ? 8 : 4;
    const int share = ((vocab + nb - 1) / nb + LG_CHUNK - 1) / LG_CHUNK * LG_CHUNK;
    c.run = share < LG_RUN ? share : LG_RUN;
    const int sz = row_dt_size(dt);
    const bool vec = !(((uintptr_t)x | (uintptr_t)out) & 15) && !((x_stride * sz) & 15) && !((out_stride * sz) & 15);
    const size_t smem = lg_smem(c.run, a.hist || a.bias, a.bias), most = lg_smem(LG_RUN, true, true);
    cudaError_t e = cudaSuccess;
    DSV4B_ROW_DT(dt, DT, {
        const auto k = nb == 8 ? (vec ? k_logits<DT, true, 8> : k_logits<DT, false, 8>)
                               : (vec ? k_logits<DT, true, 4> : k_logits<DT, false, 4>);
        if (smem_optin(k, most)) return -2;
        for (int r0 = 0; r0 < rows && e == cudaSuccess; r0 += 32768) {
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
            e = launch(k, dim3(nb, nr), dim3(LG_T), smem, st, p);
        }
    });
    return e == cudaSuccess ? 0 : -2;
}

}  // namespace dsv4b
