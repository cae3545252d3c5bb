// Attention within packed sets: entry point, argument checks and the CUDA-core kernel of the
// 32-bit mode. For query row i of set s, head h, with k and v of head h / (heads / kv_heads):
//   p_j = exp(scale q_i.k_j - m_i),  m_i = max_j scale q_i.k_j,
//   out_i = sum_j p_j v_j / sum_j p_j,   lse_i = m_i + log sum_j p_j
// over the set's keys j (causal: j <= i + keys - queries, so the last query sees every key).
// One pass over the keys keeps the running maximum, sum and output; when the maximum rises, the
// sum and output so far are scaled by exp(old - new).
//
// k_attn_cc: one block takes 64 rows (a row is a query token and one of the heads that share a key
// head, so a group's heads read the keys once) and walks the keys 64 at a time: scores by 4 x 4
// register tiles from shared memory, softmax over 16 lanes a row, output by 4 x (dim / 16) tiles.
// Bound by the FFMA rate and the shared-memory reads that feed it.
#include "tb_packed.cuh"

#include <algorithm>
#include <cmath>

#include "tb_attention.cuh"

namespace {

using namespace tbpk;

constexpr int kCcThreads = 256, kCcRows = 64, kCcKeys = 64;

template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T, class O, int D>
__global__ void __launch_bounds__(kCcThreads) k_attn_cc(const __grid_constant__ AttnArgs a) {
    constexpr int LD = D + 4;                       // row stride of q and k tiles: no bank is hit twice
    extern __shared__ float sm[];
    float* sq = sm;                                 // [64][LD]
    float* sk = sq + kCcRows * LD;                  // [64][LD]
    float* sv = sk + kCcKeys * LD;                  // [64][D]
    float* sp = sv + kCcKeys * D;                   // [64][68]
    __shared__ Item it;
    __shared__ uint32_t scan[32];
    const int kvh = blockIdx.x % a.kv_heads;
    find_item(a.q_off, a.nset, a.nq, a.unit, blockIdx.x / a.kv_heads, a.err, &it, scan);
    if (it.set < 0) return;
    // causal: the last rows of a set see the most keys; they go first
    const int piece = a.causal ? (int)(it.items - 1 - it.item) : (int)it.item;
    int64_t k0, k1;
    set_range(a.k_off, it.set, a.nk, k0, k1, a.err);
    const int nq = (int)(it.hi - it.lo), nk = (int)(k1 - k0), g = a.group;
    const int t0 = piece * a.unit, rows = min(a.unit, nq - t0) * g;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

    for (int i = threadIdx.x; i < kCcRows * (D / 8); i += kCcThreads) {
        const int r = i / (D / 8), d = i % (D / 8) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        if (r < rows && d < a.dim)
            load8<T>(reinterpret_cast<const T*>(a.q) + (it.lo + t0 + r / g) * a.q_row + (int64_t)(kvh * g + r % g) * a.q_head + d, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) sq[r * LD + d + j] = v[j] * a.scale_log2;
    }
    int lim[4];                                     // keys that the thread's rows see
    float m[4], l[4], o[4][D / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        lim[i] = r >= rows ? 0 : (a.causal ? max(0, min(nk, t0 + r / g + nk - nq + 1)) : nk);
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[i][j] = 0.f;
    }
    const int last_t = t0 + (rows - 1) / g;
    const int end = a.causal ? max(0, min(nk, last_t + nk - nq + 1)) : nk;
    for (int kb = 0; kb < end; kb += kCcKeys) {
        __syncthreads();
        for (int i = threadIdx.x; i < kCcKeys * (D / 8); i += kCcThreads) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;
            float kv[8], vv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) kv[j] = vv[j] = 0.f;
            if (kb + r < nk && d < a.dim) {         // keys past the set stay zero
                load8<T>(reinterpret_cast<const T*>(a.k) + (k0 + kb + r) * a.k_row + (int64_t)kvh * a.k_head + d, kv);
                load8<T>(reinterpret_cast<const T*>(a.v) + (k0 + kb + r) * a.v_row + (int64_t)kvh * a.v_head + d, vv);
            }
            store8<float>(sk + r * LD + d, kv);
            store8<float>(sv + r * D + d, vv);
        }
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            float4 qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(sq + (ty * 4 + i) * LD + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
                    s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
                    s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
                    s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (kb + tx + 16 * j >= lim[i]) s[i][j] = -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int d = 8; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mx = fmaxf(mx, m[i]);
            const float ref = mx == -INFINITY ? 0.f : mx;       // no key so far: every p is 0
            const float al = exp2f(m[i] - ref);
            m[i] = mx;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(s[i][j] - ref);
                sum += p;
                sp[(ty * 4 + i) * 68 + tx + 16 * j] = p;
            }
            l[i] = fmaf(l[i], al, sum);                          // the lane's own keys; joined at the end
#pragma unroll
            for (int j = 0; j < D / 16; ++j) o[i][j] *= al;
        }
        __syncwarp();                               // a row's 16 lanes are one half of a warp
#pragma unroll 2
        for (int kk = 0; kk < kCcKeys; kk += 4) {
            float4 p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(sp + (ty * 4 + i) * 68 + kk);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(sv + (kk + q) * D + c * 64 + tx * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float pq = q == 0 ? p[i].x : q == 1 ? p[i].y : q == 2 ? p[i].z : p[i].w;
                        o[i][4 * c] = fmaf(pq, v.x, o[i][4 * c]);
                        o[i][4 * c + 1] = fmaf(pq, v.y, o[i][4 * c + 1]);
                        o[i][4 * c + 2] = fmaf(pq, v.z, o[i][4 * c + 2]);
                        o[i][4 * c + 3] = fmaf(pq, v.w, o[i][4 * c + 3]);
                    }
                }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        float sum = l[i];
#pragma unroll
        for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (r >= rows) continue;
        const int64_t t = it.lo + t0 + r / g;
        const int h = kvh * g + r % g;
        const bool none = lim[i] == 0;              // a row without a key: out 0, lse -inf
        const float inv = none ? 0.f : 1.f / sum;
        O* out = reinterpret_cast<O*>(a.out) + t * a.out_row + (int64_t)h * a.out_head;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = c * 64 + tx * 4 + j;
                if (d < a.dim) out[d] = from_f32<O>(none ? 0.f : o[i][4 * c + j] * inv);
            }
        if (a.lse && tx == 0)
            a.lse[t * a.heads + h] = none ? -INFINITY : (m[i] + log2f(sum)) * 0.69314718055994530942f;
    }
}

template <class T, class O, int D>
tb_status launch_cc(tb_ctx* ctx, AttnArgs a) {
    constexpr size_t sm = sizeof(float) * (2 * 64 * (D + 4) + 64 * D + 64 * 68);
    a.unit = std::max(1, kCcRows / a.group);
    const int64_t items = ((a.nq + a.unit - 1) / a.unit + a.nset) * a.kv_heads;
    if (items > INT32_MAX) return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: too many rows times heads");
    TB_CUDA_TRY(ctx, cudaFuncSetAttribute(k_attn_cc<T, O, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
    k_attn_cc<T, O, D><<<(unsigned)items, kCcThreads, sm, ctx->stream>>>(a);
    TB_LAUNCH_CHECK(ctx, "k_attn_cc");
    return TB_OK;
}

template <class T, class O>
tb_status launch_cc_dim(tb_ctx* ctx, const AttnArgs& a) {
    return a.dim <= 64 ? launch_cc<T, O, 64>(ctx, a) : launch_cc<T, O, 128>(ctx, a);
}

bool bad_stride(int64_t count, int64_t stride, int64_t unit) { return count > 1 && (stride <= 0 || stride % unit != 0); }

// The checks that need no device; fills the kernels' arguments.
tb_status attn_args(tb_ctx* ctx, const tb_attention_params* p, AttnArgs& a) {
    if (!p) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: null parameters");
    if (p->dtype != TB_F32 && p->dtype != TB_F16 && p->dtype != TB_BF16)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: bad dtype");
    if (p->out_dtype != TB_F32 && p->out_dtype != p->dtype)
        return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_attention: out_dtype must be TB_F32 or the operand dtype");
    if (p->nq < 0 || p->nk < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: rows < 0, or heads not a multiple of kv_heads");
    if (p->head_dim < 8 || p->head_dim % 8 != 0 || p->head_dim > 128)
        return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_attention: head_dim must be a multiple of 8 up to 128");
    if (p->heads / p->kv_heads > 64)
        return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_attention: at most 64 heads may share a key head");
    if (p->nset < 0 || (!p->q_offsets != !p->k_offsets) || (!p->q_offsets && p->nset != 1))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: give both offset tables, or neither with nset 1");
    if (!(p->scale > 0.f) || !std::isfinite(p->scale))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: scale must be positive and finite");
    // a tile past the last row still has a 32-bit row number
    if (p->nq > (int64_t)INT32_MAX - 1024 || p->nk > (int64_t)INT32_MAX - 1024 || p->nset > 65536 || p->heads > 65536)
        return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: rows must be <= 2^31-1025, sets and heads at most 65536");
    const int64_t unit = 16 / (int64_t)tb_dtype_size(p->dtype), ounit = 16 / (int64_t)tb_dtype_size(p->out_dtype);
    if (bad_stride(p->nq, p->q_row, unit) || bad_stride(p->heads, p->q_head, unit) || bad_stride(p->nk, p->k_row, unit) ||
        bad_stride(p->kv_heads, p->k_head, unit) || bad_stride(p->nk, p->v_row, unit) ||
        bad_stride(p->kv_heads, p->v_head, unit) || bad_stride(p->nq, p->out_row, ounit) ||
        bad_stride(p->heads, p->out_head, ounit))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: strides must be positive multiples of 16 bytes");
    if (!tb_rows_disjoint(p->nq, p->out_row, p->heads, p->out_head, p->head_dim))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: rows or heads of out overlap");
    if (p->nq > 0 && (!p->q || !p->out)) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: null pointer");
    if (p->nk > 0 && (!p->k || !p->v)) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: null pointer");
    if (!tb_aligned16(p->q) || !tb_aligned16(p->k) || !tb_aligned16(p->v) || !tb_aligned16(p->out))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: q / k / v / out must be 16-byte aligned");
    if (p->nq > 0 && (p->out == p->q || p->out == p->k || p->out == p->v))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: out must not alias q, k or v");
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.out = p->out;
    a.lse = p->lse;
    a.q_off = p->q_offsets;
    a.k_off = p->k_offsets;
    a.nq = p->nq;
    a.nk = p->nk;
    a.q_row = p->nq > 1 ? p->q_row : 0;
    a.k_row = p->nk > 1 ? p->k_row : 0;
    a.v_row = p->nk > 1 ? p->v_row : 0;
    a.out_row = p->nq > 1 ? p->out_row : 0;
    a.q_head = p->heads > 1 ? p->q_head : 0;
    a.k_head = p->kv_heads > 1 ? p->k_head : 0;
    a.v_head = p->kv_heads > 1 ? p->v_head : 0;
    a.out_head = p->heads > 1 ? p->out_head : 0;
    a.nset = p->nset;
    a.heads = p->heads;
    a.kv_heads = p->kv_heads;
    a.group = p->heads / p->kv_heads;
    a.dim = p->head_dim;
    a.causal = p->causal ? 1 : 0;
    a.scale_log2 = p->scale * 1.44269504088896340736f;
    a.err = ctx->d_err;
    return TB_OK;
}

}  // namespace

extern "C" size_t tb_attention_workspace_bytes(const tb_ctx* ctx, const tb_attention_params* p) {
    if (!ctx || !p || (p->dtype != TB_F16 && p->dtype != TB_BF16) || p->heads < 1 || p->kv_heads < 1 ||
        p->heads % p->kv_heads != 0 || p->heads / p->kv_heads > 64 || p->head_dim < 1)
        return 0;
    return tb_attn_tc_workspace(ctx, p->nq, p->nk, p->nset, p->heads, p->kv_heads, p->head_dim);
}

extern "C" tb_status tb_attention(tb_ctx* ctx, const tb_attention_params* p) {
    if (!ctx) return TB_ERR_INVALID_ARG;
    AttnArgs a{};
    const tb_status s = attn_args(ctx, p, a);
    if (s != TB_OK) return s;
    if (a.nq == 0 || a.nset == 0) return TB_OK;
    const size_t need = tb_attention_workspace_bytes(ctx, p);
    if (need && (!p->workspace || p->workspace_bytes < need || !tb_aligned16(p->workspace)))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: workspace too small or not 16-byte aligned");
    tb_device_guard guard;
    TB_CUDA_TRY(ctx, guard.enter(ctx->device));
    if (p->dtype == TB_F32) return launch_cc_dim<float, float>(ctx, a);
    if (a.nk > 0) return tb_attn_tc_launch(ctx, a, p->dtype, p->out_dtype, p->workspace);
    // no key rows to describe to the tensor cores' loads: every row is 0
    if (p->dtype == TB_F16)
        return p->out_dtype == TB_F32 ? launch_cc_dim<__half, float>(ctx, a) : launch_cc_dim<__half, __half>(ctx, a);
    return p->out_dtype == TB_F32 ? launch_cc_dim<__nv_bfloat16, float>(ctx, a)
                                  : launch_cc_dim<__nv_bfloat16, __nv_bfloat16>(ctx, a);
}
