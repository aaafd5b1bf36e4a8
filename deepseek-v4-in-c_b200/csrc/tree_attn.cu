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
//
// Every head of every drafted token reads the same rows, so T tokens of H
// heads do 4 T H d flops per row of d + tail bytes: at H = 64 the tensor
// cores bound the kernel from the first token on. It runs on tcgen05 with
// the keys on the M side:
//
//   S^T [128 keys][rows] = V Q^T      A = V  (K-major),  B = Q  (K-major)
//   O^T [128 dims][rows] += V^T P^T   A = V^T (M-major), B = P^T (N-major)
//
// rows = up to 64 (token, head) pairs. All of O stays in TMEM: d/128 blocks
// of `rows` columns (the other way round, with queries on the M side, O
// [128][512] alone would fill TMEM).
//
// What bounds the products is shared memory: an MMA with both operands there reads
// 128 x 16 + rows x 16 f16, at 128 bytes a cycle 48 cycles for 64 rows where
// the tensor core needs 32 (measured: 48.5; with A in TMEM 32.5). So the first
// product takes V from TMEM, and the second -- whose A is V transposed, which
// only a shared-memory descriptor can express -- from shared memory. The
// TMEM copy also lets the first product run ahead of the second by more than
// a tile while shared memory holds one tile (128 rows of 512 f16 are 128 KB),
// which hides the softmax.
//
// A block takes one tile of rows and a run of 128-key tiles, cut into chunk
// pairs of 128 elements:
//   8 widening warps four threads to a key: read the codes (64-byte runs, one
//                    or two pairs in flight), widen e4m3 to f16 -- exact, the
//                    row scale stays outside -- into a TMEM ring of 2 to 4
//                    pairs;
//   8 copying warps  from there to shared memory once the second product has
//                    freed the pair's place (128-byte swizzle; V^T is the
//                    same bytes, M-major);
//   2 MMA warps      one issues S pair by pair, one O;
//   2 look-up warps  the next tile's row scales, and a request to L2 for the
//                    rows of the tile after it;
//   8 softmax warps  thread = one key and half of the rows.
//
// Measured (d 512, 64 heads, bf16): 16 tokens on 4 contexts of 32768 positions
// 420 us, 655 TFLOP/s; 7 tokens on 8 contexts of up to 4100 40 us; one token on
// 700 positions 14 us. With d 576, one token on 8 contexts of 32768 99 us. What
// bounds it is no unit but the hand-over between the roles: a tile of 64 rows
// takes 6300 cycles, of which the MMAs need 2600, and leaving out all MMAs,
// all exponentials or all loads shortens the call by 3, 0 and 5 %. Shared
// memory and TMEM are full, so no role can run further ahead. Beside its
// tiles a block costs 9 to 15 us: the first rows' way from DRAM, q, the first
// references, the output.
//
// Numbers. Cache row j has the scale byte e_j; x_j is its score as a power of
// two. Each of the tile's rows has two references of its own over the keys it
// sees: M for x, and R for x + e, which is what a key gives to O. p_j =
// 2^(x_j - M) and its sum are float. The weight that multiplies codes is
// 2^(x_j + e_j - R + 8), rounded once to f16: half a step is 2^-11 of it, or
// 2^-31 of the row's largest below f16's normal range. So a large cache row
// that is hidden or weighs nothing takes no bits from small ones that weigh
// much (with one reference of scales for all rows, 2^20 between them cost 8 %
// of the output and 2^26 all of it). References are raised only when a score
// passes M by 2^8 or a weight 2^15.5, which fits f16: O^T is almost never
// rescaled, and no tile needs the exact maximum, only two comparisons per score
// and one vote per tile. q is widened or scaled per row by a power of two into
// f16 (exact unless an element is below 2^-29 of its row's largest). S and O
// are float.
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"
#include "tcgen05.cuh"
#include "tree.h"

namespace dsv4b {
namespace {

constexpr int TA_KEYS = 128;                        // keys of a tile (M of S^T)
constexpr int TA_SOFT = 8, TA_LOAD = 8, TA_COPY = 8;    // softmax, widening and copying warps
constexpr int TA_RING = 4;                          // most pairs of the TMEM ring
constexpr int TA_WCOPY = TA_SOFT + TA_LOAD, TA_WMMA = TA_WCOPY + TA_COPY;   // MMA and look-up warps: the last four
constexpr int TA_T = 32 * (TA_WMMA + 4);
// Registers: 896 threads are launched with 72 each. A softmax thread holds two
// floats for each of its NR / 2 rows, a widening one the codes of the pairs in
// flight (two, one at 64 rows); no role may spill (shared memory leaves next to
// no L1, so a spilled register comes back from L2: 64 rows with 40 registers a
// copying thread, 8 fewer, take 582 us where these take 416).
template <int NR>
struct Regs {
    static constexpr int soft = NR == 64 ? 128 : NR == 48 ? 112 : 88, load = NR == 64 ? 56 : 72;
    static constexpr int copy = NR >= 48 ? 48 : 56, mma = 40;
    static_assert(2 * (soft + load + copy) + mma <= 7 * 72, "more registers than the block is launched with");
};
constexpr int TA_ROWS = 64;                         // most rows of a tile (N)
constexpr int TA_SLOT = TA_KEYS * 128;              // bytes of one 64-element chunk
constexpr int TA_PLACES = 7;                        // most chunk pairs in shared memory
constexpr int TA_SMEM = 232448;                     // a block's limit
constexpr int TA_SPLITS = 128;
constexpr float TA_RAISE = 8.0f;                    // log2 of p that raises the references
constexpr float TA_LIFT = 8.0f, TA_FULL = 15.5f;    // log2 of the weight at R, and of one that raises them
constexpr float TA_UNSEEN = -120.0f;                // 8 - (R - M) of a row that has seen nothing: any number

struct Parts {              // one entry per (block, row of its tile)
    float *o;               // [d] the block's own average
    float2 *ml;             // reference (log2) and sum of its weights
    int2 *seq;              // per sequence: its first block, blocks a row tile
};

struct Args {
    TreeAttn a;
    Parts part;
    int nch, places, ring, page_shift, nr;          // chunks of a row; pairs in shared memory and in TMEM; rows of a tile
    int nsplit, per;                                // splits and their key tiles when all contexts are the longest
};

struct Shared {             // behind the operand tiles
    uint64_t v_full[TA_PLACES], v_empty[TA_PLACES], k_full[TA_RING], k_done[TA_RING];
    uint64_t q_full, key_full, s_full, s_free, p_full, pv_done;
    uint64_t rowmask[TA_ROWS], out_at[TA_ROWS];     // a row's tree mask, and its first output element
    float cq[TA_ROWS], nm[TA_ROWS];     // score factor of a row, and its negated reference M
    float rr[TA_ROWS], dr[TA_ROWS];     // R - M, and 8 - (R - M) as a whole number
    float bs[TA_ROWS], dmax[2];         // 2^(dr + 127), and the largest dr of each half of the rows
    float fo[TA_ROWS], fl[TA_ROWS], wmax[4][TA_ROWS], rmax[4][TA_ROWS], lsum[4][TA_ROWS];
    int kx[TA_KEYS];        // each key's scale byte, -1: not there
    int seq, tile, tb, nt;  // the block's share: sequence (-1: none), row tile, first key tile, key tiles
    int ctx, nd;            // the sequence's context and drafted tokens
    uint32_t tmem;
    int dead;
};

__device__ __align__(64) unsigned char g_zero_row[2 * DSV4B_KVQ_MAX_D];  // a position that is not there
__device__ int g_gave_up;   // a bounded wait ran out (dsv4b_tree_attn_status)

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// 2^e for an integer e, 0 below the normal range and infinity above it.
__device__ __forceinline__ float pow2i(int e)
{
    return __uint_as_float(e < -126 ? 0u : e > 127 ? 0x7F800000u : (uint32_t)(e + 127) << 23);
}

// Among the 4 softmax warps of a half of the rows (named barriers 1 and 2):
// a vote, and a barrier.
__device__ __forceinline__ bool soft_any(bool p, int wg)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                 "barrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)p), "r"(wg + 1) : "memory");
    return r != 0;
}
__device__ __forceinline__ void soft_sync(int wg) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(wg + 1) : "memory"); }

// A widening thread's codes of a chunk pair (16 of each chunk for two keys),
// and the two rows.
struct Unit {
    uint32_t w[16], r0, r1;         // rows as 64-byte steps from the cache's start; TA_NOROW
};
constexpr uint32_t TA_NOROW = 0xFFFFFFFFu;
__device__ __forceinline__ void ld16(uint32_t *w, const unsigned char *p)
{
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}

__device__ __forceinline__ uint32_t e4m3x2_f16(uint32_t v)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)v));
    return r;
}

__device__ __forceinline__ void st_smem8(uint32_t a, uint32_t x, uint32_t y)
{
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void st_smem16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ void warp_wait(const uint64_t *bar, uint32_t parity, volatile int *dead)
{
    tc::warp_wait(tc::smem_u32(bar), parity, dead);
}
__device__ __forceinline__ void warp_arrive(const uint64_t *bar, int lane)
{
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(tc::smem_u32(bar));
}

// q rows to f16 for warp w of the 16 that share the work: one warp a row,
// scaled so that the largest magnitude lies in [2^14, 2^15) (f16 rows are
// taken as they are).
template <int NR>
__device__ __forceinline__ void widen_q(const TreeAttn &a, Shared &sh, uint32_t q_s, int r0, int nr, int b, int w, int lane)
{
    const int H = a.n_heads, d = a.c.d;
    constexpr int NV = 3;                       // 256-element parts of a row
    auto row = [&](int r) {
        const int t = (r0 + r) / H;
        return reinterpret_cast<const unsigned short *>(a.q) + ((size_t)b * a.n_tok + t) * a.q_tok +
               (size_t)(r0 + r - t * H) * d;
    };
    auto read = [&](int r, uint4 (&v)[NV]) {
        const unsigned short *q = row(r);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = i * 256 + lane * 8;
            v[i] = make_uint4(0, 0, 0, 0);
            if (r < nr && e < d) v[i] = __ldcg(reinterpret_cast<const uint4 *>(q + e));
        }
    };
    auto put = [&](int r, uint4 (&v)[NV]) {
        int kq = 0;
        if (a.dt == DSV4B_BF16) {
            uint32_t top2 = 0;          // magnitudes order as 16-bit integers
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (i * 256 >= d) break;
                top2 = __vmaxs2(top2, __vmaxs2(__vmaxs2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu), __vmaxs2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu)));
            }
            uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xFFFFu, top2 >> 16));
            if (top >= 0x7F80u) {       // infinities and NaN set no scale
                top = 0;
#pragma unroll 1
                for (int i = 0; i < d / 32; i++) {
                    const uint32_t m = r < nr ? __ldcg(row(r) + i * 32 + lane) & 0x7FFFu : 0u;
                    if (m < 0x7F80u) top = max(top, m);
                }
                top = __reduce_max_sync(0xffffffffu, top);
            }
            if (top) kq = max((int)(top >> 7) - 127 - 14, -112);
            const float f = pow2i(-kq);
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (i * 256 >= d) break;
                uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 x = mul2(bf16x2(u[k]), make_float2(f, f));
                    u[k] = pack2<DSV4B_F16>(x.x, x.y);
                }
                v[i] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
        const uint32_t dst = q_s + r * 128;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int e = i * 256 + lane * 8;
            if (e >= d) continue;
            // elements 16 q + 4 i go to place 16 i + 4 q of the chunk
            const uint32_t chunk = dst + (e >> 6) * (NR * 128), q4 = (e >> 4) & 3, i4 = (e >> 2) & 3, sw = (r & 7) << 4;
            st_smem8(chunk + ((32 * i4 + 8 * q4) ^ sw), v[i].x, v[i].y);
            st_smem8(chunk + ((32 * (i4 + 1) + 8 * q4) ^ sw), v[i].z, v[i].w);
        }
        if (lane == 0) sh.cq[r] = a.scale * 1.4426950408889634f * pow2i(kq);
    };
    // two rows' loads at a time
    constexpr int W = TA_SOFT + TA_COPY;
    uint4 v[NV], u[NV];
#pragma unroll 1
    for (int r = w; r < NR; r += 2 * W) {
        read(r, v);
        if (r + W < NR) read(r + W, u);
        put(r, v);
        if (r + W < NR) put(r + W, u);
    }
}


// The largest of a warp's values; a NaN counts only among NaN.
__device__ __forceinline__ float warp_top(float x)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

// Combine N values per lane over the 32 lanes of a warp: lane i gets the
// result of value i (N <= 32), by halving exchanges.
template <int N, typename F>
__device__ __forceinline__ float across(const float (&x)[N], float none, int lane, F op)
{
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = i < N ? x[i < N ? i : 0] : none;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; i++) {
            const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
            v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
        }
    }
    return v[0];
}

// The block's share of the work, by one warp. The host cuts every context as
// if it were the longest (it does not know the lengths); here the blocks that
// shorter contexts and smaller trees leave over go to the others: key tiles a
// block = the fewest for which all sequences' blocks fit in the grid. (Eight
// contexts of up to 4100 positions, 7 drafted tokens: 72 us cut by the longest,
// 42 so; equal contexts pay 0.4 us a block for it.) Not where the host's plan
// leaves contexts whole: 8 sequences of 16 tokens, 64 heads, under a longest
// context of 32768 fill 128 blocks uncut, and take 787 us also when seven of the
// contexts have 1000 positions, as the blocks of the eighth walk it alone.
// Sequences are numbered through, a sequence's row tiles in turn, the splits
// of a row tile side by side.
constexpr int TA_STASH = 4096;              // sequences whose lengths fit in `len`; more keep the host's cut
template <int NR>
__device__ __forceinline__ void share(const Args &g, Shared &sh, int2 *len, int lane)
{
    const TreeAttn &a = g.a;
    const bool even = g.nsplit > 1 && a.batch <= TA_STASH;
    auto length = [&](int b) {              // context and drafted tokens of sequence b
        return make_int2(min(max(__ldcg(a.ctx + b), 0), a.max_ctx),
                         a.n_draft ? min(max(__ldcg(a.n_draft + b), 0), a.n_tok) : a.n_tok);
    };
    auto tiles = [&](int2 l) {              // its key tiles and row tiles
        return l.y ? make_int2((l.x + l.y + TA_KEYS - 1) / TA_KEYS, (l.y * a.n_heads + NR - 1) / NR) : make_int2(0, 0);
    };
    int per = g.per;
    if (even) {
        int top = 1;
        for (int b = lane; b < a.batch; b += 32) {
            len[b] = length(b);
            top = max(top, tiles(len[b]).x);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        // eight parts a step: its seven counts do not wait for one another
        for (int lo = (top + TA_SPLITS - 1) / TA_SPLITS; lo < per;) {
            const int step = (per - lo + 7) >> 3;
            unsigned blocks[7] = {};
            for (int b = lane; b < a.batch; b += 32) {
                const int2 l = tiles(len[b]);
#pragma unroll
                for (int i = 0; i < 7; i++) {
                    const int mid = lo + i * step;
                    blocks[i] = min(blocks[i] + l.y * ((l.x + mid - 1) / mid), 1u << 26);
                }
            }
            int more = 0;                   // candidates lo, lo + step, ... that need too many blocks
#pragma unroll
            for (int i = 0; i < 7; i++) more += __reduce_add_sync(0xffffffffu, blocks[i]) > gridDim.x;
            if (more < 7) per = min(per, lo + more * step);
            if (more > 0) lo = min(per, lo + (more - 1) * step + 1);
        }
    }
    unsigned first = 0;                     // block of sequence b0's first
    int seq = -1, tile = 0, tb = 0, nt = 0;
    for (int b0 = 0; b0 < a.batch && seq < 0; b0 += 32) {
        const int b = b0 + lane;
        const int2 at_b = b >= a.batch ? make_int2(0, 0) : even ? len[b] : length(b), l = tiles(at_b);
        const int ns = (l.x + per - 1) / per;
        const unsigned mine = l.y * ns;
        unsigned end = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned up = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += up;
        }
        end += first;
        const unsigned here = __ballot_sync(0xffffffffu, blockIdx.x < end);
        first = __shfl_sync(0xffffffffu, end, 31);
        if (!here) continue;
        seq = b0 + __ffs(here) - 1;
        if (lane == __ffs(here) - 1) {
            const int at = blockIdx.x - (end - mine), split = at % ns, even_per = (l.x + ns - 1) / ns;
            tile = at / ns;
            tb = split * even_per;
            nt = min(l.x - tb, even_per);
            if (at == 0 && g.nsplit > 1) g.part.seq[b] = make_int2((int)(end - mine), ns);
            sh.tile = tile, sh.tb = tb, sh.nt = nt;
            sh.ctx = at_b.x, sh.nd = at_b.y;
        }
    }
    if (lane == 0) sh.seq = seq;
}

template <int NR>
__global__ void __launch_bounds__(TA_T, 1)
k_tree_attn(const __grid_constant__ Args g)
{
    pdl_wait();
    constexpr int NC = NR / 2;                  // rows of a softmax thread
    const TreeAttn &a = g.a;
    extern __shared__ unsigned char ta_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int H = a.n_heads, d = a.c.d, nch = g.nch, VP = g.places;
    const uint32_t base = (tc::smem_u32(ta_raw) + 1023u) & ~1023u;
    const uint32_t q_s = base, p_s = q_s + nch * NR * 128, kv_s = p_s + TA_KEYS * 128;
    Shared &sh = *reinterpret_cast<Shared *>(ta_raw + (kv_s - tc::smem_u32(ta_raw)) + VP * 2 * TA_SLOT);
    volatile int *dead = &sh.dead;
    const int npair = (nch + 1) >> 1;

    if (warp == TA_WMMA) tc::tmem_alloc(tc::smem_u32(&sh.tmem), 512);
    if (warp == 1) share<NR>(g, sh, reinterpret_cast<int2 *>(ta_raw + (base - tc::smem_u32(ta_raw))), lane);
    if (tid == 0) {
        for (int s = 0; s < VP; s++) {
            tc::mbar_init(tc::smem_u32(&sh.v_full[s]), TA_COPY);
            tc::mbar_init(tc::smem_u32(&sh.v_empty[s]), 1);
        }
        for (int r = 0; r < g.ring; r++) {
            tc::mbar_init(tc::smem_u32(&sh.k_full[r]), TA_LOAD);
            tc::mbar_init(tc::smem_u32(&sh.k_done[r]), 1 + TA_COPY);
        }
        tc::mbar_init(tc::smem_u32(&sh.q_full), TA_SOFT + TA_COPY);
        tc::mbar_init(tc::smem_u32(&sh.key_full), 2);
        tc::mbar_init(tc::smem_u32(&sh.s_full), 1);
        tc::mbar_init(tc::smem_u32(&sh.s_free), TA_SOFT);
        tc::mbar_init(tc::smem_u32(&sh.p_full), TA_SOFT);
        tc::mbar_init(tc::smem_u32(&sh.pv_done), 1);
        tc::mbar_init_fence();
        sh.dead = 0;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = sh.tmem;
    // the same in every lane, which the compiler cannot see of a load
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int b = uniform(sh.seq);
    if (b < 0) {
        __syncthreads();
        if (warp == TA_WMMA) tc::tmem_free(tmem, 512);
        return;
    }
    const int r0 = uniform(sh.tile) * NR, tb = uniform(sh.tb), nt = uniform(sh.nt);
    const int nd = uniform(sh.nd), ctx = uniform(sh.ctx), nr = min(NR, nd * H - r0), n = ctx + nd;
    const size_t prow = (size_t)blockIdx.x * NR;
    const int nblk = npair;                             // 128-element blocks of O^T
    const uint32_t o_col = 0, s_col = nblk * NR, k_col = s_col + NR;    // TMEM columns
    const int KR = g.ring;

    if (warp >= TA_SOFT && warp < TA_WCOPY) {
        // --------------------------------------------------------- widening
        if (Regs<NR>::load < 72) tc::reg_dec<Regs<NR>::load>();
        // Four lanes share a key: lane 4r + q holds elements 16q .. 16q + 15 of
        // a chunk for keys r and r + 8 of the warp's 16, so that a load reads
        // whole 64-byte runs of 8 rows (with a key per lane it took 4 times
        // the shared-memory cycles). The 16x256b store puts them 4 elements at
        // a time at places 16 i + 4 q of the chunk, i < 4: TMEM holds each
        // chunk in that order, which q follows and the copy undoes.
        const int lane0 = (warp & 3) * 32 + ((warp - TA_SOFT) >> 2) * 16, q4 = lane & 3;
        const int ndq = (d - a.c.tail) >> 6, shift = g.page_shift, rm = a.c.page_rows - 1;
        const int *pages = a.pages + (size_t)b * a.max_pages;
        const uint32_t row_steps = (d + a.c.tail) >> 6;
        int pos = tb * TA_KEYS + lane0 + (lane >> 2);   // of the next rows to look up
        auto page_at = [&](int q) { return q < n ? __ldcg(pages + (q >> shift)) : -1; };
        auto row_at = [&](int pg, int q) {
            return (unsigned)pg < (unsigned)a.c.n_pages ? (uint32_t)((((size_t)pg << shift) + (q & rm)) * row_steps) : TA_NOROW;
        };
        auto at_row = [&](uint32_t r) {
            return (r == TA_NOROW ? g_zero_row : reinterpret_cast<const unsigned char *>(a.c.codes) + ((size_t)r << 6)) + 16 * q4;
        };
        int pg0 = page_at(pos), pg1 = page_at(pos + 8);
        uint32_t row0, row1;
        auto next_rows = [&]() {
            row0 = row_at(pg0, pos);
            row1 = row_at(pg1, pos + 8);
            pos += TA_KEYS;
            pg0 = page_at(pos);
            pg1 = page_at(pos + 8);
        };
        next_rows();
        // the first rows into L2 at once, a cache line a lane: fetching pair by
        // pair would wait for DRAM each time
        for (int o = 128 * q4; o < d + a.c.tail; o += 512) {
            if (row0 != TA_NOROW) asm volatile("prefetch.global.L2 [%0];" ::"l"(at_row(row0) - 16 * q4 + o));
            if (row1 != TA_NOROW) asm volatile("prefetch.global.L2 [%0];" ::"l"(at_row(row1) - 16 * q4 + o));
        }
        int fp = 0, left = nt;                          // pair to fetch; tiles left
        auto fetch = [&](Unit &u) {
            if (left == 0) return;
            u.r0 = row0;
            u.r1 = row1;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const unsigned char *at = at_row(r ? row1 : row0) + 128 * fp;
#pragma unroll
                for (int s = 0; s < 2; s++)
                    if (2 * fp + s < ndq) ld16(u.w + 8 * s + 4 * r, at + 64 * s);
            }
            if (++fp == npair) {
                fp = 0;
                left--;
                next_rows();
            }
        };
        const uint32_t k_mine = tmem + ((uint32_t)lane0 << 16) + k_col;
        const int pairs = nt * npair;
        int slot = 0, par = 1, p = 0;                   // ring place, parity of its last use, pair of the tile
        int i = 0;
        auto put = [&](Unit &u) {
            const uint32_t dst = k_mine + 64 * slot;
            if (i >= KR) warp_wait(&sh.k_done[slot], par, dead);
            tc::fence_after();
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int c = 2 * p + s;
                uint32_t h[16];
                if (c < ndq) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            h[4 * k + 2 * r] = e4m3x2_f16(u.w[8 * s + 4 * r + k] & 0xFFFFu);
                            h[4 * k + 2 * r + 1] = e4m3x2_f16(u.w[8 * s + 4 * r + k] >> 16);
                        }
                    }
                    tc::tmem_st_16x256(dst + 32 * s, h);
                } else if (c < nch) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const unsigned char *at = at_row(r ? u.r1 : u.r0) + ndq * 64 + (c - ndq) * 128 + 16 * q4;
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            uint32_t t[4];
                            ld16(t, at + 16 * k);
                            h[8 * k + 2 * r] = t[0], h[8 * k + 2 * r + 1] = t[1];
                            h[8 * k + 4 + 2 * r] = t[2], h[8 * k + 4 + 2 * r + 1] = t[3];
                        }
                    }
                    tc::tmem_st_16x256(dst + 32 * s, h);
                }
            }
            fetch(u);
            tc::tmem_wait_st();
            tc::fence_before();
            warp_arrive(&sh.k_full[slot], lane);
            i++;
            if (++p == npair) p = 0;
            if (++slot == KR) slot = 0, par ^= 1;
        };
        // two pairs in flight, in registers of their own: a copy between them
        // would wait for the load
        Unit u0;
        fetch(u0);
        if constexpr (NR < 64) {
            Unit u1;
            fetch(u1);
            while (i < pairs) {
                put(u0);
                if (i < pairs) put(u1);
            }
        } else {
            while (i < pairs) put(u0);
        }
    } else if (warp >= TA_WCOPY && warp < TA_WMMA) {
        // ---------------------------------------------------------- copying
        tc::reg_dec<Regs<NR>::copy>();
        widen_q<NR>(a, sh, q_s, r0, nr, b, TA_SOFT + warp - TA_WCOPY, lane);
        tc::fence_async_smem();
        warp_arrive(&sh.q_full, lane);
        const int quad = warp & 3, half = (warp - TA_WCOPY) >> 2, key = quad * 32 + lane;
        const uint32_t k_mine = tmem + ((uint32_t)quad << 21) + k_col + 32 * half, sw = key & 7;
        const int pairs = nt * npair;
        int p = 0, slot = 0, kpar = 0, place = 0, vpar = 1;
        for (int i = 0; i < pairs; i++) {
            const int c = 2 * p + half;
            uint32_t h[32];
            warp_wait(&sh.k_full[slot], kpar, dead);
            tc::fence_after();
            if (c < nch) {
                tc::tmem_ld32(k_mine + 64 * slot, h);
                tc::tmem_wait_ld(h);
                tc::fence_before();
            }
            warp_arrive(&sh.k_done[slot], lane);
            if (i >= VP) warp_wait(&sh.v_empty[place], vpar, dead);
            if (c < nch) {
                const uint32_t dst = kv_s + (2 * place + half) * TA_SLOT + key * 128;
#pragma unroll
                for (int k = 0; k < 8; k++) {           // elements 8k .. 8k + 7 are at places 32 (k % 2) + 4 (k / 2)
                    const int r = 16 * (k & 1) + 2 * (k >> 1);
                    st_smem16(dst + ((k ^ sw) << 4), h[r], h[r + 1], h[r + 8], h[r + 9]);
                }
                tc::fence_async_smem();
            }
            warp_arrive(&sh.v_full[place], lane);
            if (++slot == KR) slot = 0, kpar ^= 1;
            if (++place == VP) place = 0, vpar ^= 1;
            if (++p == npair) p = 0;
        }
    } else if (warp >= TA_WMMA) {
        // ------------------------------------------------------- MMA issue
        tc::reg_dec<Regs<NR>::mma>();
        // Two warps, one for each product, each in the order of the pairs: the
        // tensor core takes what is ready of either.
        const int pairs = nt * npair;
        if (warp == TA_WMMA) {
            constexpr uint32_t id_s = tc::idesc_f16(128, NR, false, false);
            const uint64_t q_d = tc::sdesc(q_s, 16, 1024);
            int p = 0, j = 0, slot = 0, kpar = 0;
            warp_wait(&sh.q_full, 0, dead);
            for (int v = 0; v < pairs; v++) {
                if (p == 0 && j > 0) warp_wait(&sh.s_free, (j - 1) & 1, dead);
                warp_wait(&sh.k_full[slot], kpar, dead);
                tc::fence_after();
                if (tc::elect_one()) {
                    const uint32_t ka = tmem + k_col + 64 * slot;
                    const uint64_t qb = q_d + (uint64_t)(2 * p * NR * 8);
#pragma unroll
                    for (int k = 0; k < 4; k++) tc::mma_f16_ta(tmem + s_col, ka + 8 * k, qb + 2 * k, id_s, p > 0 || k > 0);
                    if (2 * p + 1 < nch) {
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc::mma_f16_ta(tmem + s_col, ka + 32 + 8 * k, qb + NR * 8 + 2 * k, id_s, true);
                    }
                    tc::mma_commit(tc::smem_u32(&sh.k_done[slot]));
                    if (p == npair - 1) tc::mma_commit(tc::smem_u32(&sh.s_full));
                }
                __syncwarp();
                if (++slot == KR) slot = 0, kpar ^= 1;
                if (++p == npair) p = 0, j++;
            }
        } else if (warp == TA_WMMA + 1) {
            constexpr uint32_t id_o = tc::idesc_f16(128, NR, true, true);
            const uint64_t p_d = tc::sdesc(p_s, 16, 1024);
            // a last single chunk: its second half repeats the first, into
            // TMEM lanes that nothing reads
            const uint64_t v_d2 = tc::sdesc(kv_s, TA_SLOT, 1024), v_d1 = tc::sdesc(kv_s, 0, 1024);
            int p = 0, j = 0, place = 0, vpar = 0;
            for (int v = 0; v < pairs; v++) {
                if (p == 0) warp_wait(&sh.p_full, j & 1, dead);
                warp_wait(&sh.v_full[place], vpar, dead);
                tc::fence_after();
                if (tc::elect_one()) {
                    const uint64_t va = (2 * p + 1 < nch ? v_d2 : v_d1) + (uint64_t)(2 * place * (TA_SLOT >> 4));
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        tc::mma_f16(tmem + o_col + p * NR, va + 128 * k, p_d + 128 * k, id_o, j > 0 || k > 0);
                    tc::mma_commit(tc::smem_u32(&sh.v_empty[place]));
                    if (p == npair - 1) tc::mma_commit(tc::smem_u32(&sh.pv_done));
                }
                __syncwarp();
                if (++place == VP) place = 0, vpar ^= 1;
                if (++p == npair) p = 0, j++;
            }
        }
        if (warp > TA_WMMA + 1) {
            // Two warps look up, for the softmax, the scale bytes of each tile's
            // rows, and ask the L2 for the rows two tiles ahead. A tile's
            // loads are all sent before any is used.
            const int key = (warp - TA_WMMA - 2) * 64 + lane, shift = g.page_shift, rm = a.c.page_rows - 1;
            const int *pages = a.pages + (size_t)b * a.max_pages;
            int pos = tb * TA_KEYS + key;               // of tile j, key 0 of the thread's two
            auto page_at = [&](int q) { return q < n ? __ldcg(pages + (q >> shift)) : -1; };
            auto scale_at = [&](int pg, int q) {
                return (unsigned)pg < (unsigned)a.c.n_pages
                           ? (int)__ldcg(reinterpret_cast<const unsigned char *>(a.c.scales) + ((size_t)pg << shift) + (q & rm))
                           : -1;
            };
            auto ask = [&](int pg, int q) {
                if ((unsigned)pg < (unsigned)a.c.n_pages)
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                        reinterpret_cast<const unsigned char *>(a.c.codes) + (((size_t)pg << shift) + (q & rm)) * (d + a.c.tail)),
                        "r"(d + a.c.tail));
            };
            int pa = page_at(pos), pb = page_at(pos + 32);
            int pa1 = page_at(pos + TA_KEYS), pb1 = page_at(pos + TA_KEYS + 32);
            int ka = scale_at(pa, pos), kb = scale_at(pb, pos + 32);
            pa = page_at(pos + 2 * TA_KEYS);
            pb = page_at(pos + 2 * TA_KEYS + 32);
            for (int j = 0; j < nt; j++) {              // pa1, pb1: tile j + 1; pa, pb: tile j + 2
                const int ka1 = scale_at(pa1, pos + TA_KEYS), kb1 = scale_at(pb1, pos + TA_KEYS + 32);
                if (j + 2 < nt) {
                    ask(pa, pos + 2 * TA_KEYS);
                    ask(pb, pos + 2 * TA_KEYS + 32);
                }
                pa1 = pa, pb1 = pb;
                pa = page_at(pos + 3 * TA_KEYS), pb = page_at(pos + 3 * TA_KEYS + 32);
                if (j > 0) warp_wait(&sh.s_free, (j - 1) & 1, dead);
                sh.kx[key] = ka;
                sh.kx[key + 32] = kb;
                warp_arrive(&sh.key_full, lane);
                ka = ka1, kb = kb1;
                pos += TA_KEYS;
            }
        }
        if (warp <= TA_WMMA + 1) {
            if (*dead) {        // let what was issued finish before TMEM is freed
                const uint64_t t0 = tc::now_ns();
                while (tc::now_ns() - t0 < 1000000ull) {}
            }
        }
    } else {
        // --------------------------------------------------------- softmax
        tc::reg_inc<Regs<NR>::soft>();
        const int wg = warp >> 2, key = (warp & 3) * 32 + lane, c0 = wg * NC;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        widen_q<NR>(a, sh, q_s, r0, nr, b, warp, lane);
        if (tid < NR) {
            const int r = tid, t = (r0 + r) / H;
            sh.nm[r] = INFINITY;
            sh.rr[r] = -INFINITY;
            sh.dr[r] = TA_UNSEEN;
            sh.bs[r] = pow2i((int)TA_UNSEEN + 127);
            if (r % NC == 0) sh.dmax[r / NC] = TA_UNSEEN;
            sh.out_at[r] = ((uint64_t)b * a.n_tok + t) * a.o_tok + (uint64_t)(r0 + r - t * H) * d;
            sh.rowmask[r] = r < nr ? __ldcg(a.mask + (size_t)b * a.n_tok + t) : 0ull;
        }
        tc::fence_async_smem();
        warp_arrive(&sh.q_full, lane);
        warp_wait(&sh.q_full, 0, dead);
        float l[NC];
#pragma unroll
        for (int i = 0; i < NC; i++) l[i] = 0.0f;
        const int old = ctx - tb * TA_KEYS;             // context positions from the first tile on
        for (int j = 0; j < nt; j++) {
            warp_wait(&sh.key_full, j & 1, dead);
            const int kx = sh.kx[key];
            const bool valid = kx >= 0;
            const int draft = j * TA_KEYS + key - old;
            const bool drafts = (j + 1) * TA_KEYS > old;          // the tile holds drafted rows
            const float ks = e8m0((uint8_t)kx);         // NaN for a NaN row: so are its scores and weights
            const float kf = (float)kx;
            float dmax = sh.dmax[wg];
            warp_wait(&sh.s_full, j & 1, dead);
            tc::fence_after();
            float x[NC];
            // scores times the row's factor and key's scale; hidden ones -inf
            auto scores = [&](bool lift) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < NC; i += 8) tc::tmem_ld8(tmem + lanes + s_col + c0 + i, x + i);
                tc::tmem_wait_ld(x);
#pragma unroll
                for (int i = 0; i < NC; i += 4) {
                    const float4 cq = *reinterpret_cast<const float4 *>(&sh.cq[c0 + i]);
                    const float4 nm = lift ? *reinterpret_cast<const float4 *>(&sh.nm[c0 + i]) : make_float4(0.f, 0.f, 0.f, 0.f);
                    // factors first: a large row's scale times S alone can pass
                    // float's range where the score does not
                    const float2 u = fma2(make_float2(x[i], x[i + 1]), mul2(make_float2(ks, ks), make_float2(cq.x, cq.y)), make_float2(nm.x, nm.y));
                    const float2 v = fma2(make_float2(x[i + 2], x[i + 3]), mul2(make_float2(ks, ks), make_float2(cq.z, cq.w)), make_float2(nm.z, nm.w));
                    x[i] = u.x, x[i + 1] = u.y, x[i + 2] = v.x, x[i + 3] = v.y;
                }
                if (drafts && draft >= 0) {             // past 63: no key, set below
#pragma unroll
                    for (int i = 0; i < NC; i++)
                        if (!((sh.rowmask[c0 + i] >> (draft & 63)) & 1)) x[i] = -INFINITY;
                }
                if (!valid) {
#pragma unroll
                    for (int i = 0; i < NC; i++) x[i] = -INFINITY;
                }
            };
            // exponents of the weights of x[i .. i + 3], from those of p
            auto weights = [&](int i, float2 &u, float2 &v) {
                const float4 dr = *reinterpret_cast<const float4 *>(&sh.dr[c0 + i]);
                u = add2(make_float2(x[i], x[i + 1]), add2(make_float2(kf, kf), make_float2(dr.x, dr.y)));
                v = add2(make_float2(x[i + 2], x[i + 3]), add2(make_float2(kf, kf), make_float2(dr.z, dr.w)));
            };
            // S is in registers: its columns are free. Before any wait for the
            // second product, which the MMA warp issues behind the next S.
            auto free_s = [&]() {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(tc::smem_u32(&sh.s_free));
            };
            scores(true);
            float over = -INFINITY;
#pragma unroll
            for (int i = 0; i < NC; i++) over = fmaxf(over, x[i]);
            float full = over + (kf + dmax);            // no weight is above it
            if (full > TA_FULL && over <= TA_RAISE) {
                full = -INFINITY;
#pragma unroll
                for (int i = 0; i < NC; i += 4) {
                    float2 u, v;
                    weights(i, u, v);
                    full = fmaxf(fmaxf(full, fmaxf(u.x, u.y)), fmaxf(v.x, v.y));
                }
            }
            if (soft_any(over > TA_RAISE || full > TA_FULL, wg)) {
                // raise the references: the rows' maxima over the tile (fmaxf
                // takes no NaN). R is kept relative to M: scores can be so
                // large that a scale byte added to one is lost.
                scores(false);
                free_s();
                float mine = -INFINITY, mine_r = -INFINITY;
#pragma unroll
                for (int i = 0; i < NC; i++) {
                    const float m = warp_top(x[i]);
                    if (lane == i) mine = m;
                }
                // scales within a factor of two: the largest of them serves as
                // the maxima of x + e - m, one too high at most (one maximum a
                // row instead of two: 22.6 us at 3 x 5 tokens of d = 256 on up to
                // 8000 became 24.1 without this, 23.3 with it)
                const bool some = valid && kx < 255;
                const int most = __reduce_max_sync(0xffffffffu, some ? kx : -1);
                if (most - __reduce_min_sync(0xffffffffu, some ? kx : 255) <= 1) {
                    if (mine != -INFINITY) mine_r = (float)most;
                } else {
#pragma unroll
                    for (int i = 0; i < NC; i++) {
                        const float m = __shfl_sync(0xffffffffu, mine, i);
                        const float q = warp_top(m == -INFINITY ? m : (x[i] - m) + kf);
                        if (lane == i) mine_r = q;
                    }
                }
                if (lane < NC) {
                    sh.wmax[warp & 3][c0 + lane] = fmaxf(mine, -INFINITY);
                    sh.rmax[warp & 3][c0 + lane] = fmaxf(mine_r, -INFINITY);
                }
                soft_sync(wg);
                if ((warp & 3) == 0) {
                    const int r = c0 + min(lane, NC - 1);
                    const float mo = -sh.nm[r], d0 = sh.dr[r];
                    const float mn = fmaxf(fmaxf(mo, fmaxf(sh.wmax[0][r], sh.wmax[1][r])), fmaxf(sh.wmax[2][r], sh.wmax[3][r]));
                    float rn = -INFINITY;
                    if (mn != -INFINITY) {
                        rn = (mo - mn) + sh.rr[r];
#pragma unroll
                        for (int w = 0; w < 4; w++) rn = fmaxf(rn, (sh.wmax[w][r] - mn) + sh.rmax[w][r]);
                    }
                    const float dn = mn == -INFINITY ? TA_UNSEEN : TA_LIFT - rintf(rn);
                    const float top = warp_top(dn);
                    __syncwarp();
                    if (lane < NC) {
                        sh.fl[r] = mo == -INFINITY ? 0.0f : ex2(mo - mn);
                        sh.fo[r] = mo == -INFINITY ? 0.0f : ex2((mo - mn) + (dn - d0));
                        sh.nm[r] = -mn;
                        sh.rr[r] = rn;
                        sh.dr[r] = dn;
                        sh.bs[r] = pow2i(min((int)dn, 0) + 127);    // finite: a warp without keys multiplies 0 by it
                        if (lane == 0) sh.dmax[wg] = top;
                    }
                }
                soft_sync(wg);
                dmax = sh.dmax[wg];
#pragma unroll
                for (int i = 0; i < NC; i++) l[i] *= sh.fl[c0 + i];
                if (j > 0) {
                    warp_wait(&sh.pv_done, (j - 1) & 1, dead);
                    tc::fence_after();
                    for (int p = 0; p < nblk; p++)
#pragma unroll
                        for (int i = 0; i < NC; i += 8) {
                            float y[8];
                            tc::tmem_ld8(tmem + lanes + o_col + p * NR + c0 + i, y);
                            tc::tmem_wait_ld(y);
#pragma unroll
                            for (int k = 0; k < 8; k++) y[k] *= sh.fo[c0 + i + k];
                            tc::tmem_st8(tmem + lanes + o_col + p * NR + c0 + i, y);
                        }
                    tc::tmem_wait_st();
                }
#pragma unroll
                for (int i = 0; i < NC; i++) x[i] = x[i] == -INFINITY ? x[i] : x[i] + sh.nm[c0 + i];
            } else {
                free_s();
            }
            // weights: sums of p in float, the f16 operand of the second product.
            // p 2^(e + dr) as p (2^(e - 127) 2^(dr + 127)) while no factor leaves
            // float's range for any row, which takes scales 2^93 apart; else by
            // an exponential of its own (for every weight, that takes 7 % longer:
            // 449 us against 419 at 4 x 16 tokens on 32768).
            uint32_t pw[NC / 2];
            if (!__any_sync(0xffffffffu, valid && !(dmax <= 0.0f && kf + dmax <= 100.0f))) {
                const float as = valid && kx < 255 ? ks : 0.0f;     // a NaN row's p is NaN, or 0 where it is hidden
#pragma unroll
                for (int i = 0; i < NC; i += 4) {
                    const float4 bs = *reinterpret_cast<const float4 *>(&sh.bs[c0 + i]);
                    const float2 p = make_float2(ex2(x[i]), ex2(x[i + 1])), q = make_float2(ex2(x[i + 2]), ex2(x[i + 3]));
                    const float2 u = mul2(p, mul2(make_float2(as, as), make_float2(bs.x, bs.y)));
                    const float2 v = mul2(q, mul2(make_float2(as, as), make_float2(bs.z, bs.w)));
                    pw[i / 2] = pack2<DSV4B_F16>(u.x, u.y);
                    pw[i / 2 + 1] = pack2<DSV4B_F16>(v.x, v.y);
                    const float2 s = add2(make_float2(l[i], l[i + 1]), p), t = add2(make_float2(l[i + 2], l[i + 3]), q);
                    l[i] = s.x, l[i + 1] = s.y, l[i + 2] = t.x, l[i + 3] = t.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NC; i += 4) {
                    float2 u, v;
                    weights(i, u, v);
                    pw[i / 2] = pack2<DSV4B_F16>(ex2(u.x), ex2(u.y));
                    pw[i / 2 + 1] = pack2<DSV4B_F16>(ex2(v.x), ex2(v.y));
                    const float2 s = add2(make_float2(l[i], l[i + 1]), make_float2(ex2(x[i]), ex2(x[i + 1])));
                    const float2 t = add2(make_float2(l[i + 2], l[i + 3]), make_float2(ex2(x[i + 2]), ex2(x[i + 3])));
                    l[i] = s.x, l[i + 1] = s.y, l[i + 2] = t.x, l[i + 3] = t.y;
                }
            }
            if (j > 0) warp_wait(&sh.pv_done, (j - 1) & 1, dead);
            const uint32_t dst = p_s + key * 128;
#pragma unroll
            for (int i = 0; i < NC; i += 8)
                st_smem16(dst + ((((c0 + i) >> 3) ^ (key & 7)) << 4), pw[i / 2], pw[i / 2 + 1], pw[i / 2 + 2], pw[i / 2 + 3]);
            tc::fence_async_smem();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_u32(&sh.p_full));
        }
        // row sums: the warp's 32 keys (lane = row), then the four warps
        const float mine = across<NC>(l, 0.0f, lane, [](float p, float q) { return p + q; });
        if (lane < NC) sh.lsum[warp & 3][c0 + lane] = mine;
        soft_sync(wg);
        warp_wait(&sh.pv_done, (nt - 1) & 1, dead);
        tc::fence_after();
        if (key < NC && c0 + key < nr) {
            const int r = c0 + key;
            const float m = -sh.nm[r], sum = (sh.lsum[0][r] + sh.lsum[1][r]) + (sh.lsum[2][r] + sh.lsum[3][r]);
            float den = sum;
            if (g.nsplit > 1) {
                g.part.ml[prow + r] = make_float2(m, sum);
            } else if (a.sink && m != -INFINITY) {
                den += ex2(__ldcg(a.sink + (r0 + r) % H) * 1.4426950408889634f - m);
            }
            // O = 2^dr sum p 2^e code; 0 where nothing was seen. dr lies in
            // -247 .. 8: it is set where the largest p is 1
            const int t = -(int)sh.dr[r] - 127, h = max(t, -126);
            sh.fo[r] = m == -INFINITY && sum == 0.0f ? 0.0f : pow2i(t - h) / den;
            sh.fl[r] = pow2i(h);
        }
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    // The join may start to launch: earlier it would take room from blocks to
    // come (0.6 us at 700 positions).
    pdl_trigger();
    // O out of TMEM by six groups of four warps, 16 rows at a time: lane = an
    // element of the output
    if (warp < TA_WMMA) {
        const int key = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        constexpr int NQ = NR / 16;
#pragma unroll 1
        for (int w = warp >> 2; w < npair * NQ; w += TA_WMMA / 4) {
            const int p = w / NQ, c0 = (w - p * NQ) * 16, e = p * 128 + key;
            if (c0 >= nr) continue;
            float x[16];
            tc::tmem_ld8(tmem + lanes + o_col + p * NR + c0, x);
            tc::tmem_ld8(tmem + lanes + o_col + p * NR + c0 + 8, x + 8);
            tc::tmem_wait_ld(x);
            if (e >= d) continue;
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = x[i] * sh.fo[c0 + i] * sh.fl[c0 + i];
            if (g.nsplit > 1) {
                float *o = g.part.o + (prow + c0) * d + e;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    if (c0 + i < nr) *o = x[i];
                    o += d;
                }
            } else if (a.dt == DSV4B_BF16) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (c0 + i < nr) st_row1<DSV4B_BF16>(a.o, sh.out_at[c0 + i] + e, x[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (c0 + i < nr) st_row1<DSV4B_F16>(a.o, sh.out_at[c0 + i] + e, x[i]);
            }
        }
        tc::fence_before();
    }
    __syncthreads();
    if (warp == TA_WMMA) {
        tc::fence_after();
        tc::tmem_free(tmem, 512);
    }
    if (tid == 0 && sh.dead) g_gave_up = 1;
}

// One row per block: the splits' averages weighted by their sums, joined in
// split order; the sink joins the denominator.
__global__ void __launch_bounds__(128)
k_tree_join(const __grid_constant__ Args g)
{
    pdl_trigger();
    pdl_wait();
    const TreeAttn &a = g.a;
    __shared__ float wt[TA_SPLITS];
    const int H = a.n_heads, r = blockIdx.x, b = blockIdx.y, t = r / H, d = a.c.d, tid = threadIdx.x, lane = tid & 31;
    const int nd = a.n_draft ? min(max(__ldcg(a.n_draft + b), 0), a.n_tok) : a.n_tok;
    const int2 seq = __ldcg(g.part.seq + b);    // of a sequence without tokens: not written, not used
    if (t >= nd) return;
    const int nsplit = seq.y;
    const size_t rows = g.nr, p0 = ((size_t)seq.x + (size_t)(r / g.nr) * nsplit) * rows + r % g.nr;
    if (tid < 32) {
        float2 ml[TA_SPLITS / 32];
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < TA_SPLITS / 32; i++) {
            const int s = lane + 32 * i;
            ml[i] = s < nsplit ? __ldcg(g.part.ml + p0 + s * rows) : make_float2(-INFINITY, 0.0f);
            M = fmaxf(M, ml[i].x);
        }
        M = warp_max_f(M);
        float den = 0.0f;
#pragma unroll
        for (int i = 0; i < TA_SPLITS / 32; i++) {
            // a split with a sum but no reference holds a NaN row
            ml[i].y = ml[i].x == -INFINITY && ml[i].y == 0.0f ? 0.0f : ml[i].y * ex2(ml[i].x - M);
            den += ml[i].y;
        }
        den = warp_sum_f(den);
        if (a.sink && M != -INFINITY) den += ex2(__ldcg(a.sink + (r - t * H)) * 1.4426950408889634f - M);
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
        for (int i = 0; i < TA_SPLITS / 32; i++)
            if (lane + 32 * i < nsplit) wt[lane + 32 * i] = ml[i].y * inv;
    }
    __syncthreads();
    const size_t o = ((size_t)b * a.n_tok + t) * a.o_tok + (size_t)(r - t * H) * d;
    for (int e = 4 * tid; e < d; e += 512) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < nsplit; s++) {
            const float w = wt[s];
            if (w == 0.0f) continue;                    // nothing in it, or nothing of it left
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(g.part.o + (p0 + s * rows) * d + e));
            acc.x += w * v.x, acc.y += w * v.y, acc.z += w * v.z, acc.w += w * v.w;
        }
        uint2 u;
        if (a.dt == DSV4B_BF16) u = make_uint2(pack2<DSV4B_BF16>(acc.x, acc.y), pack2<DSV4B_BF16>(acc.z, acc.w));
        else u = make_uint2(pack2<DSV4B_F16>(acc.x, acc.y), pack2<DSV4B_F16>(acc.z, acc.w));
        *reinterpret_cast<uint2 *>(reinterpret_cast<unsigned short *>(a.o) + o + e) = u;
    }
}

// A wait that nothing ends: it runs out, as a call's would, and is reported.
__global__ void __launch_bounds__(32) k_tree_wait_test(uint64_t limit_ns)
{
    __shared__ uint64_t bar;
    __shared__ int dead;
    if (threadIdx.x == 0) {
        tc::mbar_init(tc::smem_u32(&bar), 1);
        tc::mbar_init_fence();
        dead = 0;
    }
    __syncwarp();
    tc::warp_wait(tc::smem_u32(&bar), 0, &dead, limit_ns);
    __syncwarp();
    if (threadIdx.x == 0 && *(volatile int *)&dead) g_gave_up = 1;
}

// How a call is cut: rows of a tile, splits of the context, key tiles of a
// split; blocks in all (where contexts are split, whole waves of 148: shorter
// contexts leave some to the others).
struct Plan {
    int nr, tiles, nsplit, per;
    long blocks;
};

// Rows of partial outputs that a call may use: none while one key tile holds
// every position, else what any cut takes (whole waves of 148 blocks), up to ten
// waves of 64-row blocks. It grows with every size, so scratch for the largest call
// serves all smaller ones, although these are cut into more splits. The times
// below would choose more than ten waves for batches of about a hundred long
// contexts, for 3 % less time on average and 16 % at most.
constexpr long TA_PARTS = 10l * 148 * TA_ROWS;
long part_rows(int n_heads, int n_tok, int batch, int max_ctx)
{
    const long kt = (max_ctx + n_tok + TA_KEYS - 1) / TA_KEYS, s = kt < TA_SPLITS ? kt : TA_SPLITS;
    if (kt < 2) return 0;
    const long most = ((long)n_heads * n_tok + TA_ROWS - 1) * batch * s + 148l * TA_ROWS;
    return most < TA_PARTS ? most : TA_PARTS;
}

// The pair (rows of a tile, splits) of least time on 148 SMs, one block each,
// by what a block costs: microseconds per tile and beside its tiles, measured
// over 700 to 32768 positions at d = 512 and, past it, 576 (a narrower row's
// tiles take less, but the pairs compare much the same). A tile's time hardly depends on its rows (the
// 128 keys are widened all the same), so many rows win once the blocks fill
// the machine, and few rows before that. Past d = 512 a tile of 64 rows leaves
// TMEM two pairs of keys and shared memory four of five: 5.2 us a tile, still
// less than two tiles of 32 (one token on 8 contexts of 32768 at d = 576: 99
// us, with 32 rows 124, with 48 137).
Plan plan(int n_heads, int d, int n_tok, int batch, int max_ctx)
{
    static const double tile[2][4] = {{2.9, 3.1, 3.2, 3.4}, {3.3, 3.6, 4.1, 5.2}}, block_us[4] = {9.0, 11.0, 12.5, 15.0};
    const double *tile_us = tile[d > 512];
    Plan best = {};
    double cost = 0.0;
    const long R = (long)n_heads * n_tok, room = part_rows(n_heads, n_tok, batch, max_ctx);
    const int kt = (max_ctx + n_tok + TA_KEYS - 1) / TA_KEYS;
    for (int i = 3; i >= 0; i--) {
        const int nr = 16 * (i + 1);
        const long tiles = (R + nr - 1) / nr, units = tiles * batch;
        for (int s = 1; s <= TA_SPLITS && s <= kt && units * s <= 0x7fffff00l; s++) {
            const int per = (kt + s - 1) / s;
            if ((kt + per - 1) / per != s) continue;
            const long blocks = s == 1 ? units : (units * s + 147) / 148 * 148;
            if (s > 1 && blocks * nr > room) break;
            double c = (double)((units * s + 147) / 148) * (per * tile_us[i] + block_us[i]);
            // the join: a launch, and the partial outputs once through L2
            if (s > 1) c += 3.0 + (double)s * batch * R * d * 8 / 6.5e6;
            if (best.nr == 0 || c < cost) {
                cost = c;
                best = {nr, (int)tiles, s, per, blocks};
            }
        }
    }
    return best;
}

template <int NR>
int run(const Args &g, const Plan &p, size_t smem, cudaStream_t st)
{
    if (smem_optin(k_tree_attn<NR>, TA_SMEM)) return -2;
    PdlChain chain;
    cudaError_t e = launch(k_tree_attn<NR>, dim3((unsigned)p.blocks), dim3(TA_T), smem, st, g);
    if (p.nsplit > 1 && e == cudaSuccess) e = launch(k_tree_join, dim3(g.a.n_tok * g.a.n_heads, g.a.batch), dim3(128), 0, st, g);
    return e == cudaSuccess ? 0 : -2;
}

}  // namespace

size_t tree_attn_bytes(int n_heads, int d, int n_tok, int batch, int max_ctx)
{
    return (size_t)part_rows(n_heads, n_tok, batch, max_ctx) * ((size_t)d * 4 + sizeof(float2)) + (size_t)batch * sizeof(int2) + 16;
}

int tree_attn(const TreeAttn &a, void *scratch, cudaStream_t st)
{
    const Plan p = plan(a.n_heads, a.c.d, a.n_tok, a.batch, a.max_ctx);
    Args g = {};
    g.a = a;
    g.nch = a.c.d / 64;
    g.nsplit = p.nsplit;
    g.per = p.per;
    while ((1 << g.page_shift) < a.c.page_rows) g.page_shift++;
    g.part.o = reinterpret_cast<float *>(scratch);
    const size_t prows = (size_t)p.blocks * p.nr;
    g.part.ml = reinterpret_cast<float2 *>(g.part.o + prows * a.c.d);
    g.part.seq = reinterpret_cast<int2 *>(g.part.ml + prows);
    g.nr = p.nr;
    const int fixed = 1024 + g.nch * p.nr * 128 + TA_KEYS * 128 + (int)sizeof(Shared);
    // at least 4: 64 rows of 576 elements leave 135 KB
    g.places = (TA_SMEM - fixed) / (2 * TA_SLOT);
    if (g.places > TA_PLACES) g.places = TA_PLACES;
    // at least 2 pairs (64 rows, d > 512: 5 blocks of 64 columns beside S)
    g.ring = (512 - ((g.nch + 1) / 2 + 1) * p.nr) / 64;
    if (g.ring > TA_RING) g.ring = TA_RING;
    size_t smem = (size_t)fixed + (size_t)g.places * 2 * TA_SLOT;
    // one block per SM: each takes all of TMEM
    if (smem < 120 * 1024) smem = 120 * 1024;
    switch (p.nr) {
    case 16: return run<16>(g, p, smem, st);
    case 32: return run<32>(g, p, smem, st);
    case 48: return run<48>(g, p, smem, st);
    default: return run<64>(g, p, smem, st);
    }
}

int tree_attn_status()
{
    int v = 0;
    // the copy alone would wait for no stream that was made non-blocking
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    if (cudaMemcpyFromSymbol(&v, g_gave_up, sizeof v) != cudaSuccess) return -1;
    if (v == 0) return 0;
    v = 0;
    return cudaMemcpyToSymbol(g_gave_up, &v, sizeof v) == cudaSuccess ? 1 : -1;
}

int tree_attn_selftest(int limit_us, cudaStream_t st)
{
    return launch(k_tree_wait_test, dim3(1), dim3(32), 0, st, (uint64_t)limit_us * 1000) == cudaSuccess ? 0 : -2;
}

}  // namespace dsv4b
