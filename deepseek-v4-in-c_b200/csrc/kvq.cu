// kvq.cu - the quantised cache: latent KV rows written and read back.
//
// A row of d elements is held as d - tail e4m3 codes, `tail` f16 values and
// one E8M0 byte: element = code * s, s = 2^(byte - 127). s is the smallest
// power of two with max|x| <= 448 s, so no code saturates, x / s is exact and
// the only rounding is the code's: 2^-4 relative for e4m3 (while |x| is above
// 2^-14.8 of the row's largest), 2^-11 for the tail. One scale per row: e4m3
// keeps its mantissa over 14 binades below the largest element, so blocks of
// a row would gain nothing for normalised latent rows, and with one scale the
// attention multiplies scores and weights by s instead of every element. An
// all-zero row has byte 0; a row with an infinity or a NaN is stored as byte
// 255 over zero codes and reads back as NaN (no code is ever NaN, so a masked
// row cannot leak into a sum).
//
// Bound by HBM (d * size + d + tail + 1 bytes a row). One warp per row, 8
// elements per lane and group of 256: the row stays in registers between the
// maximum and the codes, so it is read once. Measured at tail 64: 16000 bf16 rows
// of d 576 written in 7.7 to 8.1 us, 16384 of d 512 read in 5.9 us, both with
// about 2 us of launch and ramp on traffic that takes 4.4 and 4.0 us. At d 512,
// 16000 rows take 6.8 us, and rotated 9.9 (13.3 from float): a rotated row costs
// 427 warp instructions, one of d 576 that is not 295, and 62 to 66 % of the issue
// slots are used. 64 rows rotated and written in 3.0 us. Blocks of 4 or 8 warps take
// the same, of 2 or 16 longer (9.6, 9.1 us).
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tree.h"

namespace dsv4b {

constexpr int KQ_W = 8;                                // warps (rows) per block
constexpr int KQ_G = (DSV4B_KVQ_MAX_D + 255) / 256;    // 256-element groups of a row

// E8M0 byte of a row whose largest magnitude has the float bits m: with
// |x| = f 2^E, f in [1, 2), and 448 = 1.75 * 2^8, the exponent is E - 8, one
// more when f > 1.75. Zero and subnormal maxima get byte 0 (2^-127).
__device__ __forceinline__ int row_scale_byte(unsigned m)
{
    if (m >= 0x7F800000u) return 255;
    const int b = (int)(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return b < 0 ? 0 : b;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(KQ_W * 32)
k_kv_write(dsv4b_kvq c, const void *rows, long row_stride, const long long *slots, int n, int has_rope,
           const __grid_constant__ RopeArg r, const int *pos)
{
    pdl_trigger();
    pdl_wait();
    __shared__ float2 cs_s[KQ_W][kRopePairs];
    __shared__ double freq[kRopePairs];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * KQ_W + warp;
    const long long slot = i < n ? __ldcg(slots + i) : -1;
    const bool live = slot >= 0 && slot < (long long)c.n_pages * c.page_rows;
    const size_t base = (size_t)i * row_stride;
    Raw8<DT> raw[KQ_G];
#pragma unroll
    for (int g = 0; g < KQ_G; g++)
        if (i < n && g * 256 + lane * 8 < c.d) raw[g] = ld_raw8<DT, VEC>(rows, base + g * 256 + lane * 8);
    float2 *cs = cs_s[warp];
    const int first = c.d - r.rd, np = r.rd >> 1;
    if (has_rope) {
        const int p = i < n ? __ldcg(pos + i) : 0;
        // a warp's lanes take turns at an array of the arguments: once a block
        if (threadIdx.x < np) freq[threadIdx.x] = r.freq[threadIdx.x];
        __syncthreads();
        if (live)
            for (int k = lane; k < np; k += 32) cs[k] = rope_angle(p, freq[k]);
        __syncwarp();
    }
    if (!live) return;
    float v[KQ_G][8];
    unsigned m = 0;
#pragma unroll
    for (int g = 0; g < KQ_G; g++) {
        const int e = g * 256 + lane * 8;
        if (e >= c.d) continue;
        widen8<DT>(raw[g], v[g]);
        if (has_rope && e + 8 > first) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int k = e + j - first;
                if (r.half) {
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int kk = k + q;
                        if (kk < 0) continue;
                        float a = kk < np ? v[g][j + q] : ld_row1<DT>(rows, base + first + kk - np);
                        float b = kk < np ? ld_row1<DT>(rows, base + first + kk + np) : v[g][j + q];
                        turn(a, b, cs[kk < np ? kk : kk - np]);
                        v[g][j + q] = kk < np ? a : b;
                    }
                } else if (k >= 0) {
                    turn(v[g][j], v[g][j + 1], cs[k >> 1]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[g][j]) & 0x7FFFFFFFu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    const int b = row_scale_byte(m);
    // 1 / s = 2^(127 - b), exact; 0 for the byte that marks a NaN row
    const float inv = b == 255 ? 0.0f : __uint_as_float((unsigned)(254 - b) << 23);
    const int dq = c.d - c.tail;
    unsigned char *row = reinterpret_cast<unsigned char *>(c.codes) + (size_t)slot * (c.d + c.tail);
#pragma unroll
    for (int g = 0; g < KQ_G; g++) {
        const int e = g * 256 + lane * 8;
        if (e >= c.d) continue;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = b == 255 ? 0.0f : __fmul_rn(v[g][j], inv);
        if (e < dq) {
            unsigned w[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j], y[4 * j + 1]), __NV_SATFINITE, __NV_E4M3);
                const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j + 2], y[4 * j + 3]), __NV_SATFINITE, __NV_E4M3);
                w[j] = lo | (hi << 16);
            }
            *reinterpret_cast<uint2 *>(row + e) = make_uint2(w[0], w[1]);
        } else {
            st_row8<DSV4B_F16, true>(row + dq, (size_t)(e - dq), y);
        }
    }
    if (lane == 0) reinterpret_cast<unsigned char *>(c.scales)[slot] = (unsigned char)b;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(KQ_W * 32)
k_kv_read(dsv4b_kvq c, void *out, long row_stride, const long long *slots, int n)
{
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, i = blockIdx.x * KQ_W + (threadIdx.x >> 5);
    if (i >= n) return;
    const long long slot = __ldcg(slots + i);
    const bool live = slot >= 0 && slot < (long long)c.n_pages * c.page_rows;
    const int dq = c.d - c.tail;
    const unsigned char *row = reinterpret_cast<const unsigned char *>(c.codes) + (size_t)(live ? slot : 0) * (c.d + c.tail);
    const float s = live ? e8m0(__ldcg(reinterpret_cast<const unsigned char *>(c.scales) + slot)) : 0.0f;
    uint4 raw[KQ_G];
#pragma unroll
    for (int g = 0; g < KQ_G; g++) {
        const int e = g * 256 + lane * 8;
        raw[g] = make_uint4(0, 0, 0, 0);
        if (!live || e >= c.d) continue;
        if (e < dq) {
            const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(row + e));
            raw[g].x = w.x;
            raw[g].y = w.y;
        } else {
            raw[g] = __ldcg(reinterpret_cast<const uint4 *>(row + dq + 2 * (e - dq)));
        }
    }
#pragma unroll
    for (int g = 0; g < KQ_G; g++) {
        const int e = g * 256 + lane * 8;
        if (e >= c.d) continue;
        float v[8];
        if (e < dq) {
            const unsigned w[2] = {raw[g].x, raw[g].y};
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float2 a = e4m3x2((uint16_t)(w[j] & 0xFFFFu)), b = e4m3x2((uint16_t)(w[j] >> 16));
                v[4 * j] = a.x, v[4 * j + 1] = a.y, v[4 * j + 2] = b.x, v[4 * j + 3] = b.y;
            }
        } else {
            Raw8<DSV4B_F16> h;
            h.w[0] = raw[g];
            widen8<DSV4B_F16>(h, v);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = __fmul_rn(v[j], s);
        st_row8<DT, VEC>(out, (size_t)i * row_stride + e, v);
    }
}

static bool rows_vec(const void *p, int dt, long row_stride)
{
    return !((uintptr_t)p & 15) && !((row_stride * row_dt_size(dt)) & 15);
}

int kv_write(const dsv4b_kvq &c, const void *rows, int dt, long row_stride, const long long *slots, int n,
             const RopeArg *r, const int *pos, cudaStream_t st)
{
    if (n <= 0) return 0;
    RopeArg none = {};
    const dim3 grid((n + KQ_W - 1) / KQ_W);
    cudaError_t e = cudaSuccess;
    DSV4B_ROW_DT(dt, DT, {
        if (rows_vec(rows, dt, row_stride))
            e = launch(k_kv_write<DT, true>, grid, dim3(KQ_W * 32), 0, st, c, rows, row_stride, slots, n, r ? 1 : 0,
                       r ? *r : none, pos);
        else
            e = launch(k_kv_write<DT, false>, grid, dim3(KQ_W * 32), 0, st, c, rows, row_stride, slots, n, r ? 1 : 0,
                       r ? *r : none, pos);
    });
    return e == cudaSuccess ? 0 : -2;
}

int kv_read(const dsv4b_kvq &c, void *out, int dt, long row_stride, const long long *slots, int n,
            cudaStream_t st)
{
    if (n <= 0) return 0;
    const dim3 grid((n + KQ_W - 1) / KQ_W);
    cudaError_t e = cudaSuccess;
    DSV4B_ROW_DT(dt, DT, {
        if (rows_vec(out, dt, row_stride))
            e = launch(k_kv_read<DT, true>, grid, dim3(KQ_W * 32), 0, st, c, out, row_stride, slots, n);
        else
            e = launch(k_kv_read<DT, false>, grid, dim3(KQ_W * 32), 0, st, c, out, row_stride, slots, n);
    });
    return e == cudaSuccess ? 0 : -2;
}

}  // namespace dsv4b
