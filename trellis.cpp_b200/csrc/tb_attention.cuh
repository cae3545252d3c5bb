// Arguments shared by the attention kernels (tb_attention.cu, tb_attention_tc.cu).
#pragma once

#include "tb_common.cuh"

struct AttnArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;                      // [nq][heads] or null
    const int32_t* q_off;
    const int32_t* k_off;
    int64_t nq, nk;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;   // in elements
    int nset, heads, kv_heads, group, dim, causal;
    int unit;                        // query tokens of a block
    float scale_log2;                // scale * log2(e): scores in powers of two
    int nsplit;                      // ranges the keys are cut into
    float* part;                     // [nsplit][nq][heads][dim] partial rows (normalised), null with one range
    float* part_lse;                 // [nsplit][nq][heads] their log sums, base 2; -inf: no key, row not written
    int* err;
};

// The plan of a kernel that may cut the keys: how many ranges.
int tb_attn_tc_nsplit(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int heads, int kv_heads, int dim);
// 16-bit operands on tensor cores; nq, nk, nset > 0. args.nsplit as planned, part and part_lse set.
tb_status tb_attn_tc_launch(tb_ctx* ctx, const AttnArgs& args, tb_dtype dtype, tb_dtype out_dtype);
