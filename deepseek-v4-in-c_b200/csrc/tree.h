// tree.h - the operators of a tree-verification step: rotary positions, the
// quantised paged cache, attention of drafted tokens over it, and logits
// adjustment. Arguments are checked by the C ABI (capi_tree.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include "../../include/dsv4_b200.h"

namespace dsv4b {

constexpr int kRopePairs = DSV4B_ROPE_MAX / 2;

// A rotation as a kernel parameter: pair i turns by pos * freq[i].
struct RopeArg {
    double freq[kRopePairs];
    int rd, half;
};

// x [n_tok][n_heads][width] -> out, elements first .. first + rd of every
// head rotated; strides in elements. inplace: out is x, only the rotated
// elements are written.
struct RopeCall {
    void *out;
    const void *x;
    int out_dt, x_dt;
    long out_tok, out_head, x_tok, x_head;
    const int *pos;
    int n_tok, n_heads, width, first, inverse, inplace;
};
int rope(const RopeCall &c, const RopeArg &r, cudaStream_t st);

// rows [n][d] (stride in elements) into / out of the cache rows slots[n];
// r (may be null) rotates the last r->rd elements before quantisation.
int kv_write(const dsv4b_kvq &c, const void *rows, int dt, long row_stride, const long long *slots, int n,
             const RopeArg *r, const int *pos, cudaStream_t st);
int kv_read(const dsv4b_kvq &c, void *out, int dt, long row_stride, const long long *slots, int n,
            cudaStream_t st);

struct TreeAttn {
    void *o;
    const void *q;
    int dt;                         // DSV4B_BF16 or DSV4B_F16
    long o_tok, q_tok;              // elements from one token's heads to the next's
    dsv4b_kvq c;
    const int *pages;               // [batch][max_pages]
    int max_pages;
    const int *ctx, *n_draft;       // [batch]; n_draft may be null (n_tok each)
    const unsigned long long *mask; // [batch][n_tok]
    const float *sink;              // [n_heads] or null
    int n_heads, n_tok, batch, max_ctx;
    float scale;
};
size_t tree_attn_bytes(int n_heads, int d, int n_tok, int batch, int max_ctx);
int tree_attn(const TreeAttn &a, void *scratch, cudaStream_t st);

int tree_attn_status();
int tree_attn_selftest(int limit_us, cudaStream_t st);

int logits(void *out, const void *x, int dt, long out_stride, long x_stride, int *token,
           const dsv4b_logit_adjust &a, int rows, int vocab, cudaStream_t st);

}  // namespace dsv4b
