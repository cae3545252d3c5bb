// Attention within packed sets: entry point, argument checks and the CUDA-core kernel of the
// 32-bit mode. For query row i of set s, head h, with k and v of head h / (heads / kv_heads):
//   p_j = exp(scale q_i.k_j - m_i),  m_i = max_j scale q_i.k_j,
//   out_i = sum_j p_j v_j / sum_j p_j,   lse_i = m_i + log sum_j p_j
// over the set's keys j (causal: j <= i + keys - queries, so the last query sees every key).
// One pass over the keys keeps the running maximum, sum and output; when the maximum rises, the
// sum and output so far are scaled by exp(old - new).
//
// k_attn_cc: one block takes 64 rows (a row is a query token and one of the heads that share a key
// head, so a group's heads read the keys once) and walks the keys 64 at a time. Scores and output are
// the same product of two tiles in shared memory, 8 x 4 values a thread: the values are laid in the
// tile, so 16 bytes are two pairs of neighbours of the summed axis for packed FMAs, and the two halves
// of a pair's sum meet at the end. Bound by what feeds the FMAs: a warp's step is 12 16-byte loads, 4
// cycles of the SM's shared-memory path each, and 64 packed FMAs, 2 cycles of its scheduler each, so
// the path is busy 192 cycles for 128 of the four schedulers' FMAs: 47 us of the 94 (22 TFLOP/s) that 800
// and 600 rows, 8 heads of 64 take (4 x 4 values a thread, 256 threads, unpacked: 107 us). The rest: blocks
// of keys are loaded between two barriers and used at once, 368 CTAs fill one wave of two an SM and part of
// another, and the parts' join takes 10 us.
#include "tb_packed.cuh"

#include <algorithm>
#include <cmath>

#include "tb_attention.cuh"

namespace {

using namespace tbpk;

constexpr int kCcThreads = 128, kCcRows = 64, kCcKeys = 64, kCcLd = 68;

template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// x[i][j] = sum over n < N of a[i * 8 rows][n] b[j * 16 rows][n]. Row strides of 4 modulo 32 words: the
// 16 rows of b and the two of a that a warp reads at once lie in different banks.
template <int N, int LDA, int LDB>
__device__ __forceinline__ void tile_product(const float* a, const float* b, float (&x)[8][4]) {
    f2 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0;
#pragma unroll 2
    for (int n = 0; n < N; n += 4) {
        ulonglong2 bv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[j] = *reinterpret_cast<const ulonglong2*>(b + 16 * j * LDB + n);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const ulonglong2 av = *reinterpret_cast<const ulonglong2*>(a + 8 * i * LDA + n);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fma2(av.y, bv[j].y, fma2(av.x, bv[j].x, acc[i][j]));
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpack(acc[i][j]);
            x[i][j] = f.x + f.y;
        }
}

// Operands are 32-bit; without keys nothing is read, and O alone counts.
template <class O, int D>
__global__ void __launch_bounds__(kCcThreads, 2) k_attn_cc(const __grid_constant__ AttnArgs a) {
    constexpr int LD = D + 4, V4 = D / 64;
    extern __shared__ float sm[];
    float* sq = sm;                                 // [64][LD]
    float* sk = sq + kCcRows * LD;                  // [64][LD], then the weights [64][68]
    float* sv = sk + kCcKeys * LD;                  // [D][68]: values of a column side by side
    float* sp = sk;
    uint32_t idx = blockIdx.x;
    const int split = idx % a.nsplit;
    idx /= a.nsplit;
    const int kvh = idx % a.kv_heads;
    check_table(a.q_off, a.nset, a.nq, a.err);
    check_table(a.k_off, a.nset, a.nk, a.err);
    const Item it = find_item(a.q_off, a.nset, a.nq, a.unit, idx / a.kv_heads, a.err);
    if (it.set < 0) return;
    // causal: the last rows of a set see the most keys; they go first
    const int piece = a.causal ? (int)(it.items - 1 - it.item) : (int)it.item;
    int64_t k0, k1;
    set_range(a.k_off, it.set, a.nk, k0, k1, a.err);
    const int nq = (int)(it.hi - it.lo), nk = (int)(k1 - k0), g = a.group;
    const int t0 = piece * a.unit, rows = min(a.unit, nq - t0) * g;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;     // rows ty + 8 i

    int lim[8];                                     // keys that the thread's rows see
    float m[8], l[8], o[8][4 * V4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = ty + 8 * i;
        lim[i] = r >= rows ? 0 : (a.causal ? max(0, min(nk, t0 + r / g + nk - nq + 1)) : nk);
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 4 * V4; ++j) o[i][j] = 0.f;
    }
    const int last_t = t0 + (rows - 1) / g;
    const int end = a.causal ? max(0, min(nk, last_t + nk - nq + 1)) : nk;
    const int all = (end + kCcKeys - 1) / kCcKeys;
    const int first = (int)((int64_t)all * split / a.nsplit) * kCcKeys;
    const int stop = min(end, (int)((int64_t)all * (split + 1) / a.nsplit) * kCcKeys);
    if (first < stop)
        for (int i = threadIdx.x; i < kCcRows * (D / 8); i += kCcThreads) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
            if (r < rows && d < a.dim)
                load8<float>(reinterpret_cast<const float*>(a.q) + (it.lo + t0 + r / g) * a.q_row + (int64_t)(kvh * g + r % g) * a.q_head + d, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= a.scale_log2;
            store8<float>(sq + r * LD + d, v);
        }
    for (int kb = first; kb < stop; kb += kCcKeys) {
        __syncthreads();
        for (int i = threadIdx.x; i < kCcKeys * (D / 8); i += kCcThreads) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;     // a row's columns on neighbouring lanes
            const int vr = i % kCcKeys, vd = i / kCcKeys * 8;   // rows on neighbouring lanes: turned without conflicts
            float kv[8], vv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) kv[j] = vv[j] = 0.f;    // keys past the set stay zero
            if (kb + r < nk && d < a.dim)
                load8<float>(reinterpret_cast<const float*>(a.k) + (k0 + kb + r) * a.k_row + (int64_t)kvh * a.k_head + d, kv);
            if (kb + vr < nk && vd < a.dim)
                load8<float>(reinterpret_cast<const float*>(a.v) + (k0 + kb + vr) * a.v_row + (int64_t)kvh * a.v_head + vd, vv);
            store8<float>(sk + r * LD + d, kv);
#pragma unroll
            for (int j = 0; j < 8; ++j) sv[(vd + j) * kCcLd + vr] = vv[j];
        }
        __syncthreads();
        float s[8][4];
        tile_product<D, LD, LD>(sq + ty * LD, sk + tx * LD, s);
        __syncthreads();                            // every warp is through with the keys
#pragma unroll
        for (int i = 0; i < 8; ++i) {
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
                sp[(ty + 8 * i) * kCcLd + tx + 16 * j] = p;
            }
            l[i] = fmaf(l[i], al, sum);                          // the lane's own keys; joined at the end
#pragma unroll
            for (int j = 0; j < 4 * V4; ++j) o[i][j] *= al;
        }
        __syncwarp();                               // a row's 16 lanes are one half of a warp
#pragma unroll
        for (int c = 0; c < V4; ++c) {
            tile_product<kCcKeys, kCcLd, kCcLd>(sp + ty * kCcLd, sv + (c * 64 + tx) * kCcLd, s);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][4 * c + j] += s[i][j];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = ty + 8 * i;
        float sum = l[i];
#pragma unroll
        for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (r >= rows) continue;
        const int64_t t = it.lo + t0 + r / g;
        const int h = kvh * g + r % g;
        const bool none = sum == 0.f;       // a row without a key, or without a score above -inf: out 0, lse -inf
        const float lg = none ? -INFINITY : m[i] + log2f(sum);
        const float inv = none ? 0.f : 1.f / sum;
        if (a.part) {
            const int64_t at = ((int64_t)split * a.nq + t) * a.heads + h;
            if (tx == 0) a.part_lse[at] = lg;
            if (none) continue;
#pragma unroll
            for (int j = 0; j < 4 * V4; ++j)
                if (tx + 16 * j < a.dim) a.part[at * a.dim + tx + 16 * j] = o[i][j] * inv;
            continue;
        }
        O* out = reinterpret_cast<O*>(a.out) + t * a.out_row + (int64_t)h * a.out_head;
#pragma unroll
        for (int j = 0; j < 4 * V4; ++j)
            if (tx + 16 * j < a.dim) out[tx + 16 * j] = from_f32<O>(none ? 0.f : o[i][j] * inv);
        if (a.lse && tx == 0) a.lse[t * a.heads + h] = lg * 0.69314718055994530942f;
    }
}

// Blocks of the CUDA-core kernel before the keys are cut.
int64_t cc_items(int64_t nq, int nset, int kv_heads, int group) {
    const int unit = kCcRows / group;
    return ((nq + unit - 1) / unit + nset) * kv_heads;
}
// Fewer CTAs than three an SM are cut, down to a block of keys each for sets of the average length or to two
// if all keys are one set's, which the host does not know: a block takes a lone CTA 4 to 11 us, a range
// without keys next to nothing. (800 and 600 rows, 8 heads of 64, 192 CTAs: 104 us whole, 93 cut in two
// and joined; 870 rows beside four small sets, one head of 128: 150 and 34; 57 and 91 rows, 8 heads of
// 128: 29 and 22; three sets of 64, one block each: 13 us, 16 if cut all the same.)
int cc_nsplit(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int kv_heads, int group) {
    const int64_t items = cc_items(nq, nset, kv_heads, group);
    const int64_t blocks = std::max((nk / nset + kCcKeys - 1) / kCcKeys, nk / kCcKeys / 2);
    return (int)std::max<int64_t>(1, std::min<int64_t>({3ll * ctx->num_sms / items, blocks, 32}));
}

template <class O, int D>
tb_status launch_cc(tb_ctx* ctx, AttnArgs a) {
    constexpr size_t sm = sizeof(float) * (2 * 64 * (D + 4) + D * kCcLd);
    a.unit = kCcRows / a.group;
    const int64_t items = cc_items(a.nq, a.nset, a.kv_heads, a.group) * a.nsplit;
    if (items > INT32_MAX) return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: too many rows times heads");
    TB_CUDA_TRY(ctx, cudaFuncSetAttribute(k_attn_cc<O, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
    k_attn_cc<O, D><<<(unsigned)items, kCcThreads, sm, ctx->stream>>>(a);
    TB_LAUNCH_CHECK(ctx, "k_attn_cc");
    return TB_OK;
}

// Joins the partial rows: with lg_s the base-2 log sum of part s and M their maximum,
//   out = sum_s 2^(lg_s - M) out_s / sum_s 2^(lg_s - M),  lse = (M + log2(that sum)) / log2(e).
// A warp a row and head: a lane takes one part's weight (at most 32), then four values of the row.
template <class O>
__global__ void __launch_bounds__(128) k_attn_join(const __grid_constant__ AttnArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t row = at / a.heads, h = at % a.heads, step = a.nq * a.heads;
    int64_t lo = 0, hi = a.nq;
    if (a.q_off) {
        lo = min(max((int64_t)a.q_off[0], (int64_t)0), a.nq);
        hi = min((int64_t)a.q_off[a.nset], a.nq);
    }
    if (row < lo || row >= hi) return;
    const float lg = lane < a.nsplit ? a.part_lse[lane * step + at] : -INFINITY;
    float mx = lg;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    // a log sum that is no number does not show in the maximum: it goes by its weight
    const float w = lg == -INFINITY ? 0.f : exp2f(lg - mx);
    const int c0 = lane * 4;
    float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const float* part = a.part + at * a.dim + (c0 < a.dim ? c0 : 0);
#pragma unroll 8
    for (int s = 0; s < a.nsplit; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(part + s * step * a.dim);
        const float ws = __shfl_sync(0xffffffffu, w, s);
        const bool written = __shfl_sync(0xffffffffu, lg, s) != -INFINITY;     // else whatever was there
        sum += ws;
        o[0] = written ? fmaf(ws, v.x, o[0]) : o[0];
        o[1] = written ? fmaf(ws, v.y, o[1]) : o[1];
        o[2] = written ? fmaf(ws, v.z, o[2]) : o[2];
        o[3] = written ? fmaf(ws, v.w, o[3]) : o[3];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (lane == 0 && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994530942f;
    if (c0 >= a.dim) return;
    O* out = reinterpret_cast<O*>(a.out) + row * a.out_row + h * a.out_head + c0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    if (sizeof(O) == 4) {
        *reinterpret_cast<float4*>(out) = make_float4(o[0], o[1], o[2], o[3]);
    } else {
        using H = typename std::conditional<sizeof(O) == 4, __half, O>::type;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack2(o[0], o[1], H()), pack2(o[2], o[3], H()));
    }
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
    // scores are taken in powers of two
    if (!(p->scale > 0.f) || !std::isfinite(p->scale * 1.44269504088896340736f))
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
    const tb_rows o = tb_head_rows(p->out, p->nq, p->out_row, p->heads, p->out_head, p->head_dim, p->out_dtype);
    if (p->nq > 0 && (p->out == p->q || p->out == p->k || p->out == p->v ||
                      tb_rows_overlap(o, tb_head_rows(p->q, p->nq, p->q_row, p->heads, p->q_head, p->head_dim, p->dtype)) ||
                      tb_rows_overlap(o, tb_head_rows(p->k, p->nk, p->k_row, p->kv_heads, p->k_head, p->head_dim, p->dtype)) ||
                      tb_rows_overlap(o, tb_head_rows(p->v, p->nk, p->v_row, p->kv_heads, p->v_head, p->head_dim, p->dtype))))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: out must not overlap q, k or v");
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

// Ranges that the kernel for these arguments cuts the keys into; 1 without keys.
static int attn_nsplit(const tb_ctx* ctx, tb_dtype dtype, int64_t nq, int64_t nk, int nset, int heads, int kv_heads, int dim) {
    if (nq <= 0 || nk <= 0 || nset <= 0) return 1;
    if (dtype == TB_F32) return cc_nsplit(ctx, nq, nk, nset, kv_heads, heads / kv_heads);
    if (tb_attn_few(nq, nset, heads / kv_heads)) return tb_attn_few_nsplit(ctx, nq, nk, nset, kv_heads, heads / kv_heads);
    return tb_attn_tc_nsplit(ctx, nq, nk, nset, heads, kv_heads, dim);
}

extern "C" size_t tb_attention_workspace_bytes(const tb_ctx* ctx, const tb_attention_params* p) {
    if (!ctx || !p || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0 || p->heads / p->kv_heads > 64 ||
        p->head_dim < 1)
        return 0;
    const int n = attn_nsplit(ctx, p->dtype, p->nq, p->nk, p->nset, p->heads, p->kv_heads, p->head_dim);
    return n > 1 ? (size_t)n * p->nq * p->heads * (p->head_dim + 1) * sizeof(float) : 0;
}

extern "C" tb_status tb_attention(tb_ctx* ctx, const tb_attention_params* p) {
    if (!ctx) return TB_ERR_INVALID_ARG;
    AttnArgs a{};
    tb_status s = attn_args(ctx, p, a);
    if (s != TB_OK) return s;
    if (a.nq == 0 || a.nset == 0) return TB_OK;
    a.nsplit = attn_nsplit(ctx, p->dtype, a.nq, a.nk, a.nset, a.heads, a.kv_heads, a.dim);
    if (a.nsplit > 1) {
        const size_t rows = (size_t)a.nsplit * a.nq * a.heads;
        if (!p->workspace || p->workspace_bytes < rows * (a.dim + 1) * sizeof(float) || !tb_aligned16(p->workspace))
            return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_attention: workspace too small or not 16-byte aligned");
        if ((a.nq * a.heads + 3) / 4 > INT32_MAX) return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: too many rows times heads");
        a.part = reinterpret_cast<float*>(p->workspace);
        a.part_lse = a.part + rows * a.dim;
    }
    tb_device_guard guard;
    TB_CUDA_TRY(ctx, guard.enter(ctx->device));
    // without key rows there is nothing to describe to the TMA loads: every row is 0
    if (p->dtype != TB_F32 && a.nk > 0)
        s = tb_attn_few(a.nq, a.nset, a.group) ? tb_attn_few_launch(ctx, a, p->dtype, p->out_dtype)
                                               : tb_attn_tc_launch(ctx, a, p->dtype, p->out_dtype);
    else if (p->out_dtype == TB_F16) s = launch_cc<__half, 128>(ctx, a);
    else if (p->out_dtype == TB_BF16) s = launch_cc<__nv_bfloat16, 128>(ctx, a);
    else s = a.dim <= 64 ? launch_cc<float, 64>(ctx, a) : launch_cc<float, 128>(ctx, a);
    if (s != TB_OK || !a.part) return s;
    const unsigned blocks = (unsigned)((a.nq * a.heads + 3) / 4);
    if (p->out_dtype == TB_F32) k_attn_join<float><<<blocks, 128, 0, ctx->stream>>>(a);
    else if (p->out_dtype == TB_F16) k_attn_join<__half><<<blocks, 128, 0, ctx->stream>>>(a);
    else k_attn_join<__nv_bfloat16><<<blocks, 128, 0, ctx->stream>>>(a);
    TB_LAUNCH_CHECK(ctx, "k_attn_join");
    return TB_OK;
}
