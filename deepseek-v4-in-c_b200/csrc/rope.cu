// rope.cu - rotary positions of query heads, KV rows and attention outputs.
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),   t = pos * freq[i]
//
// for the rd/2 pairs of a head's rotated part; pair i is (2i, 2i+1) in the
// interleaved layout and (i, i + rd/2) in the half layout. The inverse turns
// by -t: it is the transpose, so also the gradient of the rotation.
//
// The angle is formed and reduced in double -- at position 2^20 a float angle
// is off by 0.06 radians -- and only its cosine and sine are rounded to
// float. The reference precomputes tables in double on the host
// (src/core/dsv4_rope.c:48-99); here a block computes its token's rd/2 pairs
// itself, which bounds neither the position nor the context.
//
// Bound by HBM: x read once and out written once (in place: the rotated part
// only). A block owns one token and a run of its heads, so a pair's cosine
// and sine are computed once per block and read from shared memory; the first
// groups are asked for before. Measured with 64 heads of 512 elements: 2048
// tokens f32 -> bf16, 128 elements in halves, in 73.5 us, 5.5 TB/s (3 groups
// in flight a thread 79; 8 of them 110, as fewer threads fit); 32 tokens
// bf16 -> f32, 64 elements in pairs turned back, in 4.0 us; one in 2.6 us. Element
// by element, where no 16-byte groups fit (heads of 510 elements, 126 of them in
// pairs): 188 us for the 2048 tokens, 8.6 for 32, 3.2 for one.
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tree.h"

namespace dsv4b {

constexpr int RP_T = 256;       // threads per block
constexpr int RP_U = 4;         // groups in flight per thread

// Group kinds of one head: 8 elements copied, 8 elements of interleaved
// pairs, or 8 + 8 elements of half-layout pairs. Every element is read by the
// thread that writes it (its pair partner included), so out may be x.
template <int XDT, int ODT>
__global__ void __launch_bounds__(RP_T)
k_rope(RopeCall c, const __grid_constant__ RopeArg r, int heads_per_block)
{
    pdl_trigger();
    pdl_wait();
    __shared__ float2 cs[kRopePairs];
    const int t = blockIdx.x, h0 = blockIdx.y * heads_per_block;
    const int nh = min(heads_per_block, c.n_heads - h0), np = r.rd >> 1;
    const size_t xb = (size_t)t * c.x_tok + (size_t)h0 * c.x_head, ob = (size_t)t * c.out_tok + (size_t)h0 * c.out_head;
    const int rot = r.half ? r.rd >> 4 : r.rd >> 3;            // rotated groups of a head
    const int still = c.inplace ? 0 : (c.width - r.rd) >> 3;   // copied groups
    const int per = rot + still, n = per * nh;
    const int pos = __ldcg(c.pos + t);
    for (int first = 0; first < n; first += RP_T * RP_U) {
        const int u0 = first + threadIdx.x;
        Raw8<XDT> a[RP_U], b[RP_U];
        int at[RP_U], kind[RP_U];           // element of the head; rotated group or -1
        size_t hx[RP_U];
#pragma unroll
        for (int k = 0; k < RP_U; k++) {
            const int u = u0 + k * RP_T;
            if (u >= n) continue;
            const int h = u / per, g = u - h * per;
            hx[k] = (size_t)h;
            kind[k] = g < rot ? g : -1;
            const int e = (g - rot) << 3;
            at[k] = g < rot ? c.first + (g << 3) : (e < c.first ? e : e + r.rd);
            const size_t i = xb + hx[k] * c.x_head + at[k];
            a[k] = ld_raw8<XDT, true>(c.x, i);
            if (kind[k] >= 0 && r.half) b[k] = ld_raw8<XDT, true>(c.x, i + np);
        }
        if (first == 0) {                   // the angles, while the first groups travel
            for (int i = threadIdx.x; i < np; i += RP_T) {
                float2 a = rope_angle(pos, r.freq[i]);
                if (c.inverse) a.y = -a.y;
                cs[i] = a;
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < RP_U; k++) {
            if (u0 + k * RP_T >= n) continue;
            const size_t i = ob + hx[k] * c.out_head + at[k];
            float v[8], w[8];
            widen8<XDT>(a[k], v);
            if (kind[k] >= 0) {
                if (r.half) {
                    widen8<XDT>(b[k], w);
#pragma unroll
                    for (int j = 0; j < 8; j++) turn(v[j], w[j], cs[8 * kind[k] + j]);
                    st_row8<ODT, true>(c.out, i + np, w);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) turn(v[2 * j], v[2 * j + 1], cs[4 * kind[k] + j]);
                }
            }
            st_row8<ODT, true>(c.out, i, v);
        }
    }
}

// Any width, offset, stride or alignment: one pair or one copied element per
// thread.
template <int XDT, int ODT>
__global__ void __launch_bounds__(RP_T)
k_rope_any(RopeCall c, const __grid_constant__ RopeArg r, int heads_per_block)
{
    pdl_trigger();
    pdl_wait();
    __shared__ float2 cs[kRopePairs];
    const int t = blockIdx.x, h0 = blockIdx.y * heads_per_block;
    const int nh = min(heads_per_block, c.n_heads - h0), np = r.rd >> 1;
    const int pos = __ldcg(c.pos + t);
    for (int i = threadIdx.x; i < np; i += RP_T) {
        float2 a = rope_angle(pos, r.freq[i]);
        if (c.inverse) a.y = -a.y;
        cs[i] = a;
    }
    __syncthreads();
    const int per = np + (c.inplace ? 0 : c.width - r.rd);
    for (int u = threadIdx.x; u < per * nh; u += RP_T) {
        const int h = u / per, g = u - h * per;
        const size_t xi = (size_t)t * c.x_tok + (size_t)(h0 + h) * c.x_head;
        const size_t oi = (size_t)t * c.out_tok + (size_t)(h0 + h) * c.out_head;
        if (g < np) {
            const int ea = c.first + (r.half ? g : 2 * g), eb = r.half ? ea + np : ea + 1;
            float a = ld_row1<XDT>(c.x, xi + ea), b = ld_row1<XDT>(c.x, xi + eb);
            turn(a, b, cs[g]);
            st_row1<ODT>(c.out, oi + ea, a);
            st_row1<ODT>(c.out, oi + eb, b);
        } else {
            int e = g - np;
            if (e >= c.first) e += r.rd;
            st_row1<ODT>(c.out, oi + e, ld_row1<XDT>(c.x, xi + e));
        }
    }
}

int rope(const RopeCall &c, const RopeArg &r, cudaStream_t st)
{
    if (c.n_tok <= 0 || c.n_heads <= 0) return 0;
    // 16-byte groups: every group of 8 elements starts on a group boundary
    const bool vec = !(c.width & 7) && !(c.first & 7) && !(r.rd & (r.half ? 15 : 7)) &&
                     !((c.x_tok | c.x_head | c.out_tok | c.out_head) & 7) &&
                     !(((uintptr_t)c.x | (uintptr_t)c.out) & 15);
    // a block takes as many of a token's heads as leave a block for each SM:
    // 32 tokens of 64 heads take 4.0 us so, 4.7 with two blocks an SM, 6.5 with
    // four, as each block looks up the frequencies and turns its pairs anew
    int hpb = c.n_heads;
    while (hpb > 1 && (long)c.n_tok * ((c.n_heads + hpb - 1) / hpb) < 148) hpb = (hpb + 1) / 2;
    const dim3 grid(c.n_tok, (c.n_heads + hpb - 1) / hpb);
    if (grid.y > 65535) return -1;
    cudaError_t e = cudaSuccess;
    DSV4B_ROW_DT(c.x_dt, XDT, DSV4B_ROW_DT(c.out_dt, ODT, {
        if (vec) e = launch(k_rope<XDT, ODT>, grid, dim3(RP_T), 0, st, c, r, hpb);
        else e = launch(k_rope_any<XDT, ODT>, grid, dim3(RP_T), 0, st, c, r, hpb);
    }));
    return e == cudaSuccess ? 0 : -2;
}

}  // namespace dsv4b
