// Arguments shared by the attention kernels (tb_attention.cu, tb_attention_tc.cu).
#pragma once

#include <cuda.h>

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

// The kernels' plans: how many ranges the keys are cut into.
int tb_attn_tc_nsplit(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int heads, int kv_heads, int dim);
int tb_attn_few_nsplit(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int kv_heads, int group);
// The kernel of few rows a set takes the call (16-bit operands).
bool tb_attn_few(int64_t nq, int nset, int group);
// 16-bit operands on tensor cores; nq, nk, nset > 0. args.nsplit as planned, part and part_lse set.
tb_status tb_attn_tc_launch(tb_ctx* ctx, const AttnArgs& args, tb_dtype dtype, tb_dtype out_dtype);
tb_status tb_attn_few_launch(tb_ctx* ctx, const AttnArgs& args, tb_dtype dtype, tb_dtype out_dtype);
// Tensor map over [rows][heads][dim] (strides in elements), boxes of 64 columns x box_heads x box_rows.
tb_status tb_attn_encode(tb_ctx* ctx, CUtensorMap* map, tb_dtype dtype, const void* base, int dim, int64_t heads, int64_t head,
                         int64_t rows, int64_t row, uint32_t box_heads, uint32_t box_rows);
