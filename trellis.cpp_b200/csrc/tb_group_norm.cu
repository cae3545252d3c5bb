// GroupNorm with an activation over packed sets, channels last: for set s and group g (the
// c / groups consecutive channels of the group over the set's rows)
//   mean, var = the mean and variance of those values,
//   out = act((x - mean) / sqrt(var + eps) * w[channel] + b[channel]).
//
// Three passes: k_gn_stats cuts the sets into pieces of rows, one block a piece, and writes each
// group's mean and sum of squared deviations; k_gn_merge joins a set's pieces; k_gn_apply
// normalises. Statistics: a thread takes 8 channels, reads rows in batches of four and joins each
// batch's mean and squared deviations with its running ones (no difference of large sums, so a
// mean far from zero costs no digits); entries are joined as
//   mean = sum n_i mean_i / N,  M2 = sum M2_i + sum n_i (mean_i - mean)^2,
// in 64 bits, always in the same order, so results repeat to the bit. Bound by memory.
#include "tb_packed.cuh"

#include <algorithm>

namespace {

using namespace tbpk;

constexpr int kGnThreads = 256;
constexpr int kGnMaxC = 2048;

struct GnArgs {
    const void* x;
    void* out;
    const int32_t* off;
    const float* w;
    const float* b;
    int64_t n;
    int nset, c, groups, unit;
    float eps;
    int act;
    float2* part;     // [pieces][groups] mean, M2
    float2* stat;     // [nset][groups] mean, 1 / sqrt(var + eps)
    int* err;
};

template <class T>
__global__ void __launch_bounds__(kGnThreads) k_gn_stats(const __grid_constant__ GnArgs a) {
    __shared__ Item it;
    __shared__ uint32_t scan[32];
    extern __shared__ float2 ent[];                 // [row lanes][c] mean, M2 of a thread's channels
    __shared__ int cnt[kGnThreads];                 // rows of a row lane
    find_item(a.off, a.nset, a.n, a.unit, blockIdx.x, a.err, &it, scan);
    if (it.set < 0) return;
    const int tc = a.c / 8, lanes = kGnThreads / tc;
    const int ry = threadIdx.x / tc, c0 = (threadIdx.x % tc) * 8;
    const int64_t r0 = it.lo + (int64_t)it.item * a.unit, r1 = min(it.hi, r0 + a.unit);
    if (ry < lanes) {
        float mean[8], m2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) mean[j] = m2[j] = 0.f;
        int n = 0;
        const T* x = reinterpret_cast<const T*>(a.x) + c0;
        int64_t r = r0 + ry;
        for (; r + 3 * lanes < r1; r += 4 * lanes) {
            float v[4][8];
#pragma unroll
            for (int q = 0; q < 4; ++q) load8<T>(x + (r + (int64_t)q * lanes) * a.c, v[q]);
            const float f = 4.f / (float)(n + 4), g = f * (float)n;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float m = 0.25f * ((v[0][j] + v[1][j]) + (v[2][j] + v[3][j]));
                float s = 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float d = v[q][j] - m;
                    s = fmaf(d, d, s);
                }
                const float d = m - mean[j];
                mean[j] = fmaf(d, f, mean[j]);
                m2[j] += fmaf(d * d, g, s);
            }
            n += 4;
        }
        for (; r < r1; r += lanes) {
            float v[8];
            load8<T>(x + r * a.c, v);
            ++n;
            const float f = 1.f / (float)n;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = v[j] - mean[j];
                mean[j] = fmaf(d, f, mean[j]);
                m2[j] = fmaf(d, v[j] - mean[j], m2[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ent[ry * a.c + c0 + j] = make_float2(mean[j], m2[j]);
        if (c0 == 0) cnt[ry] = n;
    }
    __syncthreads();
    // a warp joins the entries of one group after another
    const int cg = a.c / a.groups, lane = threadIdx.x & 31;
    const double total = (double)(r1 - r0) * cg;
    for (int g = threadIdx.x >> 5; g < a.groups; g += kGnThreads / 32) {
        double s = 0;
        for (int e = lane; e < lanes * cg; e += 32) s += (double)cnt[e / cg] * ent[(e / cg) * a.c + g * cg + e % cg].x;
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const double m = s / total;
        double q = 0;
        for (int e = lane; e < lanes * cg; e += 32) {
            const float2 v = ent[(e / cg) * a.c + g * cg + e % cg];
            const double d = v.x - m;
            q += v.y + cnt[e / cg] * (d * d);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) q += __shfl_xor_sync(0xffffffffu, q, d);
        if (lane == 0) a.part[(int64_t)blockIdx.x * a.groups + g] = make_float2((float)m, (float)q);
    }
}

// One warp joins the pieces of one group of one set.
__global__ void __launch_bounds__(kGnThreads) k_gn_merge(const __grid_constant__ GnArgs a) {
    __shared__ uint32_t first_s;
    const int set = blockIdx.x, lane = threadIdx.x & 31;
    // the set's first piece: the pieces of the sets before it
    uint32_t before = 0;
    for (int s = threadIdx.x; s < set; s += kGnThreads) {
        int64_t lo, hi;
        set_range(a.off, s, a.n, lo, hi, a.err);
        before += (uint32_t)((hi - lo + a.unit - 1) / a.unit);
    }
    if (threadIdx.x == 0) first_s = 0;
    __syncthreads();
    if (before) atomicAdd(&first_s, before);
    __syncthreads();
    int64_t lo, hi;
    set_range(a.off, set, a.n, lo, hi, a.err);
    if (hi == lo) return;
    const int pieces = (int)((hi - lo + a.unit - 1) / a.unit), cg = a.c / a.groups;
    const int last = (int)(hi - lo - (int64_t)(pieces - 1) * a.unit);
    for (int g = blockIdx.y * (kGnThreads / 32) + (threadIdx.x >> 5); g < a.groups; g += gridDim.y * (kGnThreads / 32)) {
        const float2* p = a.part + (int64_t)first_s * a.groups + g;
        double s = 0;
        for (int i = lane; i < pieces; i += 32) s += (double)(i == pieces - 1 ? last : a.unit) * p[(int64_t)i * a.groups].x;
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const double m = s / (double)(hi - lo);
        double q = 0;
        for (int i = lane; i < pieces; i += 32) {
            const float2 v = p[(int64_t)i * a.groups];
            const double d = v.x - m;
            q += v.y + (double)(i == pieces - 1 ? last : a.unit) * cg * (d * d);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) q += __shfl_xor_sync(0xffffffffu, q, d);
        if (lane == 0)
            a.stat[(int64_t)set * a.groups + g] =
                make_float2((float)m, (float)(1.0 / sqrt(q / ((double)(hi - lo) * cg) + (double)a.eps)));
    }
}

template <class T, class O>
__global__ void __launch_bounds__(kGnThreads) k_gn_apply(const __grid_constant__ GnArgs a) {
    __shared__ Item it;
    __shared__ uint32_t scan[32];
    find_item(a.off, a.nset, a.n, a.unit, blockIdx.x, a.err, &it, scan);
    if (it.set < 0) return;
    const int tc = a.c / 8, lanes = kGnThreads / tc;
    const int ry = threadIdx.x / tc, c0 = (threadIdx.x % tc) * 8;
    if (ry >= lanes) return;
    const int64_t r0 = it.lo + (int64_t)it.item * a.unit, r1 = min(it.hi, r0 + a.unit);
    const int cg = a.c / a.groups;
    float mean[8], f[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 s = a.stat[(int64_t)it.set * a.groups + (c0 + j) / cg];
        mean[j] = s.x;
        f[j] = a.w ? s.y * a.w[c0 + j] : s.y;
        b[j] = a.b ? a.b[c0 + j] : 0.f;
    }
    const T* x = reinterpret_cast<const T*>(a.x) + c0;
    O* o = reinterpret_cast<O*>(a.out) + c0;
    for (int64_t r = r0 + ry; r < r1; r += lanes) {
        float v[8];
        load8<T>(x + r * a.c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = fmaf(v[j] - mean[j], f[j], b[j]);
            if (a.act) v[j] = tb_silu(v[j]);
        }
        store8<O>(o + r * a.c, v);
    }
}

// Rows of a piece: about eight pieces an SM over the whole array, 16 rows at least.
int gn_unit(int num_sms, int64_t n) {
    const int64_t pieces = 8ll * num_sms;
    return (int)std::max<int64_t>(16, (n + pieces - 1) / pieces);
}
int64_t gn_pieces(int num_sms, int64_t n, int nset) {
    const int unit = gn_unit(num_sms, n);
    return (n + unit - 1) / unit + nset;
}

template <class T>
void launch_gn(const GnArgs& a, bool f32_out, int64_t pieces, cudaStream_t st) {
    const size_t sm = (size_t)(kGnThreads / (a.c / 8)) * a.c * sizeof(float2);
    k_gn_stats<T><<<(unsigned)pieces, kGnThreads, sm, st>>>(a);
    k_gn_merge<<<dim3((unsigned)a.nset, (unsigned)((a.groups + 7) / 8)), kGnThreads, 0, st>>>(a);
    if (f32_out) k_gn_apply<T, float><<<(unsigned)pieces, kGnThreads, 0, st>>>(a);
    else k_gn_apply<T, T><<<(unsigned)pieces, kGnThreads, 0, st>>>(a);
}

}  // namespace

extern "C" size_t tb_group_norm_workspace_bytes(const tb_ctx* ctx, int64_t n, int groups, int nset) {
    if (!ctx || n <= 0 || groups < 1 || nset < 1) return 0;
    return (size_t)(gn_pieces(ctx->num_sms, n, nset) + nset) * groups * sizeof(float2);
}

extern "C" tb_status tb_group_norm(tb_ctx* ctx, const void* x, tb_dtype x_dtype, const int32_t* offsets, int nset,
                                   int64_t n, int c, int groups, const float* w, const float* b, float eps,
                                   tb_epilogue act, tb_dtype out_dtype, void* out, void* workspace,
                                   size_t workspace_bytes) {
    if (!ctx) return TB_ERR_INVALID_ARG;
    if (x_dtype != TB_F32 && x_dtype != TB_F16 && x_dtype != TB_BF16)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: bad dtype");
    if (out_dtype != TB_F32 && out_dtype != x_dtype)
        return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_group_norm: out_dtype must be TB_F32 or x's dtype");
    if (n < 0 || c <= 0 || c % 8 != 0 || c > kGnMaxC)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: needs n >= 0 and c a multiple of 8 up to 2048");
    if (groups < 1 || c % groups != 0) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: groups must divide c");
    if (nset < 0 || (!offsets && nset != 1))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: nset < 0, or no offsets and nset != 1");
    if (act != TB_EPI_NONE && act != TB_EPI_SILU) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: bad activation");
    if (!(eps >= 0.f)) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: eps must not be negative");
    if (n == 0 || nset == 0) return TB_OK;
    if (n >= (int64_t)INT32_MAX || nset > 65536)
        return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_group_norm: n must be < 2^31-1 and nset at most 65536");
    if (!x || !out) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: null pointer");
    if (!tb_aligned16(x) || !tb_aligned16(out))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: x / out must be 16-byte aligned");
    if (out == x && out_dtype != x_dtype)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: in place needs out_dtype equal to x's dtype");
    if (!workspace || workspace_bytes < tb_group_norm_workspace_bytes(ctx, n, groups, nset) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: workspace too small or not 16-byte aligned");
    const int64_t pieces = gn_pieces(ctx->num_sms, n, nset);
    GnArgs a{};
    a.x = x;
    a.out = out;
    a.off = offsets;
    a.w = w;
    a.b = b;
    a.n = n;
    a.nset = nset;
    a.c = c;
    a.groups = groups;
    a.unit = gn_unit(ctx->num_sms, n);
    a.eps = eps;
    a.act = act == TB_EPI_SILU;
    a.part = reinterpret_cast<float2*>(workspace);
    a.stat = a.part + pieces * groups;
    a.err = ctx->d_err;
    tb_device_guard guard;
    TB_CUDA_TRY(ctx, guard.enter(ctx->device));
    if (x_dtype == TB_F32) launch_gn<float>(a, true, pieces, ctx->stream);
    else if (x_dtype == TB_F16) launch_gn<__half>(a, out_dtype == TB_F32, pieces, ctx->stream);
    else launch_gn<__nv_bfloat16>(a, out_dtype == TB_F32, pieces, ctx->stream);
    TB_LAUNCH_CHECK(ctx, "tb_group_norm");
    return TB_OK;
}
