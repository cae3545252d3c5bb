// Rotary positions with several axes: the pair p of every head of row i turns by the angle
//   pos[i][axis(p)] * f_p,   (a, b) -> (a cos - b sin, a sin + b cos),
// where the first sections[0] pairs of a head take axis 0 (a voxel's x), the next sections[1] axis
// 1, and so on; pairs past the last section keep their bits (no product with a sine of 0, which would
// carry a value that is no number to its partner). f_p = theta^(-j / sections[axis])
// with j the pair's place in its section, or theta^(-p / (head_dim/2)) with frequencies shared by
// the axes. inverse turns by the negative angle, which is the transpose: the gradient's way back.
//
// Angles: far positions times a 32-bit frequency lose the phase (position 1e5 at f = 1: 4e-3), so
// the angle is counted in revolutions in 64 bits, its whole part dropped, and the rest given to
// sincospif in 32 bits. A thread owns a few pairs of one row and computes their sines once for
// all heads it turns. Bound by memory: each value is read and written once.
#include "tb_packed.cuh"

#include <algorithm>
#include <cmath>

namespace {

using namespace tbpk;

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 128;

struct RopeArgs {
    const void* x;
    void* out;
    const int32_t* pos;       // column of axis 0 of row 0
    int64_t n, x_row, x_head, out_row, out_head;
    int pos_stride, heads, half, chunks, heads_per;
    int turned;               // pairs that turn; those behind are kept
    float sign;               // -1 turns backwards
    double freq[kRopeMaxPairs];      // revolutions per position
    uint8_t axis[kRopeMaxPairs];
};

// P pairs of one head as they lie in memory: elements 2p, 2p+1 (PAIRS), otherwise p and p + half. Words
// of 16 bytes, of 8 where a half of a head is no multiple of them; streamed past the caches' end.
template <class T, int P, bool PAIRS> struct Pairs {
    static constexpr int kBytes = PAIRS ? 2 * P * (int)sizeof(T) : P * (int)sizeof(T);   // of each run
    static constexpr int kRuns = PAIRS ? 1 : 2;
    using W = typename std::conditional<kBytes % 16 == 0, uint4, uint2>::type;
    static constexpr int kWords = kBytes / (int)sizeof(W);
    W w[kRuns * kWords];
    __device__ __forceinline__ void load(const T* h, int p0, int half) {
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                w[r * kWords + i] = __ldcs(reinterpret_cast<const W*>(h + (PAIRS ? 2 * p0 : r * half + p0)) + i);
    }
    __device__ __forceinline__ void store(T* h, int p0, int half) const {
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                __stcs(reinterpret_cast<W*>(h + (PAIRS ? 2 * p0 : r * half + p0)) + i, w[r * kWords + i]);
    }
    // turns the pairs by c, s; KEPT: the first `left` of them
    template <bool KEPT> __device__ __forceinline__ void turn(const float* c, const float* s, int left) {
        uint32_t* u = reinterpret_cast<uint32_t*>(w);
        constexpr int per = 4 / (int)sizeof(T);                   // elements of a 32-bit word
#pragma unroll
        for (int i = 0; i < P; i += (PAIRS ? 1 : per)) {
            if (PAIRS) {
                float a, b;
                get(u, 2 * i, &a, &b);
                if (!KEPT || i < left) put(u, 2 * i, a * c[i] - b * s[i], a * s[i] + b * c[i]);
            } else {
                float x[2], y[2];
#pragma unroll
                for (int e = 0; e < per; ++e) {
                    const float a = value(u, i + e), b = value(u, P + i + e);
                    x[e] = a * c[i + e] - b * s[i + e];
                    y[e] = a * s[i + e] + b * c[i + e];
                }
                if (per == 2) {
                    const uint32_t ka = u[i / 2], kb = u[(P + i) / 2];
                    const uint32_t m = !KEPT || i + 1 < left ? 0xffffffffu : i < left ? 0xffffu : 0u;   // the halves that turn
                    put(u, i, x[0], x[1]);
                    put(u, P + i, y[0], y[1]);
                    u[i / 2] = (u[i / 2] & m) | (ka & ~m);
                    u[(P + i) / 2] = (u[(P + i) / 2] & m) | (kb & ~m);
                } else if (!KEPT || i < left) {
                    u[i] = __float_as_uint(x[0]);
                    u[P + i] = __float_as_uint(y[0]);
                }
            }
        }
    }

private:
    using H = typename std::conditional<sizeof(T) == 4, __half, T>::type;
    static __device__ __forceinline__ float value(const uint32_t* u, int i) {
        if (sizeof(T) == 4) return __uint_as_float(u[i]);
        float v[2];
        unpack2(u[i / 2], v, H());
        return v[i % 2];
    }
    // elements i (even) and i + 1
    static __device__ __forceinline__ void get(const uint32_t* u, int i, float* a, float* b) {
        a[0] = value(u, i);
        b[0] = value(u, i + 1);
    }
    static __device__ __forceinline__ void put(uint32_t* u, int i, float x, float y) {
        if (sizeof(T) == 4) {
            u[i] = __float_as_uint(x);
            u[i + 1] = __float_as_uint(y);
        } else {
            u[i / 2] = pack2(x, y, H());
        }
    }
};

// KEPT: some pairs keep their bits. A kernel of its own, since the choice costs 2% where all turn (131072 x
// 16 heads of 128, halves, f16: 180 us against 176).
template <class T, int P, bool PAIRS, bool KEPT>
__global__ void __launch_bounds__(kRopeThreads) k_rope(const __grid_constant__ RopeArgs r) {
    constexpr int kBatch = 4;                       // heads whose loads go before the first store
    const int64_t t = (int64_t)blockIdx.x * kRopeThreads + threadIdx.x;
    const int64_t row = t / r.chunks;
    if (row >= r.n) return;
    const int p0 = (int)(t - row * r.chunks) * P;
    const int h0 = blockIdx.y * r.heads_per, h1 = min(r.heads, h0 + r.heads_per);
    const T* x = reinterpret_cast<const T*>(r.x) + row * r.x_row + h0 * r.x_head;
    T* o = reinterpret_cast<T*>(r.out) + row * r.out_row + h0 * r.out_head;
    Pairs<T, P, PAIRS> v[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
        if (h0 + q < h1) v[q].load(x + q * r.x_head, p0, r.half);
    float c[P], s[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const double turns = (double)r.pos[row * r.pos_stride + r.axis[p0 + i]] * r.freq[p0 + i];
        sincospif(2.f * (float)(turns - rint(turns)), s + i, c + i);
        s[i] *= r.sign;
    }
    for (int h = h0; h < h1; h += kBatch) {
#pragma unroll
        for (int q = 0; q < kBatch; ++q)
            if (h + q < h1) {
                v[q].template turn<KEPT>(c, s, r.turned - p0);
                v[q].store(o + q * r.out_head, p0, r.half);
            }
        x += kBatch * r.x_head;
        o += kBatch * r.out_head;
#pragma unroll
        for (int q = 0; q < kBatch; ++q)
            if (h + kBatch + q < h1) v[q].load(x + q * r.x_head, p0, r.half);
    }
}

template <class T, bool KEPT>
void launch_rope(const RopeArgs& r, bool pairs, int per, dim3 grid, cudaStream_t stream) {
    if (pairs) k_rope<T, 4, true, KEPT><<<grid, kRopeThreads, 0, stream>>>(r);
    else if (per == 8) k_rope<T, 8, false, KEPT><<<grid, kRopeThreads, 0, stream>>>(r);
    else k_rope<T, 4, false, KEPT><<<grid, kRopeThreads, 0, stream>>>(r);
}
template <class T>
void launch_rope(const RopeArgs& r, bool pairs, int per, dim3 grid, cudaStream_t stream) {
    if (r.turned < r.half) launch_rope<T, true>(r, pairs, per, grid, stream);
    else launch_rope<T, false>(r, pairs, per, grid, stream);
}

}  // namespace

extern "C" tb_status tb_rope(tb_ctx* ctx, const tb_rope_params* p) {
    if (!ctx) return TB_ERR_INVALID_ARG;
    if (!p) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: null parameters");
    if (p->dtype != TB_F32 && p->dtype != TB_F16 && p->dtype != TB_BF16)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: bad dtype");
    if (p->n < 0 || p->heads < 1) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: n < 0 or heads < 1");
    if (p->head_dim < 8 || p->head_dim % 8 != 0 || p->head_dim > 2 * kRopeMaxPairs)
        return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_rope: head_dim must be a multiple of 8 up to 256");
    if (p->layout != TB_ROPE_PAIRS && p->layout != TB_ROPE_HALVES)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: bad layout");
    if (p->freqs != TB_ROPE_FREQS_AXIS && p->freqs != TB_ROPE_FREQS_JOINT)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: bad frequency rule");
    if (p->axes < 1 || p->axes > 4 || p->coord_stride < p->axes)
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: needs 1 to 4 axes and coord_stride >= axes");
    if (!(p->theta > 0) || !std::isfinite(p->theta)) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: theta must be positive");
    const int half = p->head_dim / 2;
    int64_t total = 0;
    for (int a = 0; a < p->axes; ++a) {
        if (p->sections[a] < 1) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: a section needs at least one pair");
        total += p->sections[a];
    }
    if (total > half) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: the sections have more pairs than a head");
    if (p->n == 0) return TB_OK;
    if (p->n >= (int64_t)INT32_MAX) return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_rope: n must be < 2^31-1");
    if (!p->x || !p->out || !p->coords) return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: null pointer");
    const int64_t unit = 16 / (int64_t)tb_dtype_size(p->dtype);
    const bool rows = p->n > 1, hds = p->heads > 1;          // a single row's or head's stride is not used
    if (!tb_aligned16(p->x) || !tb_aligned16(p->out) || (rows && (p->x_row % unit || p->out_row % unit)) ||
        (hds && (p->x_head % unit || p->out_head % unit)))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: pointers and strides must be multiples of 16 bytes");
    if (!tb_rows_disjoint(p->n, p->out_row, p->heads, p->out_head, p->head_dim))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: rows or heads of out overlap");
    if (p->out == p->x && ((rows && p->out_row != p->x_row) || (hds && p->out_head != p->x_head)))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: in place needs equal strides");
    if (p->out != p->x && tb_rows_overlap(tb_head_rows(p->out, p->n, p->out_row, p->heads, p->out_head, p->head_dim, p->dtype),
                                          tb_head_rows(p->x, p->n, p->x_row, p->heads, p->x_head, p->head_dim, p->dtype)))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_rope: out must be x or not overlap it");

    RopeArgs r;
    r.x = p->x;
    r.out = p->out;
    r.pos = p->coords + (p->coord_stride - p->axes);
    r.n = p->n;
    r.x_row = p->x_row;
    r.x_head = p->x_head;
    r.out_row = p->out_row;
    r.out_head = p->out_head;
    r.pos_stride = p->coord_stride;
    r.heads = p->heads;
    r.half = half;
    r.sign = p->inverse ? -1.f : 1.f;
    const double lg = std::log2(p->theta), turn = 0.15915494309189533577;   // 1 / (2 pi)
    int q = 0;
    for (int a = 0; a < p->axes; ++a)
        for (int j = 0; j < p->sections[a]; ++j, ++q) {
            const double power = p->freqs == TB_ROPE_FREQS_JOINT ? (double)q / half : (double)j / p->sections[a];
            r.freq[q] = turn * std::exp2(-power * lg);
            r.axis[q] = (uint8_t)a;
        }
    r.turned = q;
    for (; q < half; ++q) {
        r.freq[q] = 0.0;
        r.axis[q] = 0;
    }
    const bool pairs = p->layout == TB_ROPE_PAIRS;
    const int per = !pairs && p->dtype != TB_F32 && half % 8 == 0 ? 8 : 4;
    r.chunks = half / per;
    const int64_t blocks = (p->n * r.chunks + kRopeThreads - 1) / kRopeThreads;
    // A thread turns as many heads as leave four blocks an SM: its sines serve them all, but 600 rows of
    // 64 on one block each 24 heads leave most SMs idle (9.9 us against 4.8 with the heads spread).
    const int64_t split = std::max<int64_t>(1, std::min<int64_t>(p->heads, 4ll * ctx->num_sms / blocks));
    r.heads_per = (int)((p->heads + split - 1) / split);
    tb_device_guard guard;
    TB_CUDA_TRY(ctx, guard.enter(ctx->device));
    const dim3 grid((unsigned)blocks, (unsigned)((p->heads + r.heads_per - 1) / r.heads_per));
    if (p->dtype == TB_F32) launch_rope<float>(r, pairs, per, grid, ctx->stream);
    else if (p->dtype == TB_F16) launch_rope<__half>(r, pairs, per, grid, ctx->stream);
    else launch_rope<__nv_bfloat16>(r, pairs, per, grid, ctx->stream);
    TB_LAUNCH_CHECK(ctx, "k_rope");
    return TB_OK;
}
