// Attention within packed sets of few query rows (bf16 / f16 operands): a new token or a few against
// the keys so far. The mathematics and the entry point are in tb_attention.cu.
//
// Bound by reading the keys and values once, so the kernel is laid out for loads under way: a CTA takes
// 16 rows (a row is a token and one of the heads that share a key head) and a range of the keys, its W
// warps every W-th 16 keys of them. A warp has a ring of its own (24 KB) that one lane fills by TMA, runs
// its own softmax and meets the others at the end only. Its products are warp-level m16n8k16 MMAs: the
// rows fill one fragment, where the 128-row tiles of tb_attention_tc.cu would run the softmax of 128
// rows for them. 64 tokens of 32/8 heads of 128 against 2048 keys each: 82 us, 6.5 TB/s; 16 against 1
// to 8192 keys (63k): 54 us, 5.0 TB/s, the longest set's CTAs last. (The next step's scores before this
// one's softmax: 61 us, the ring then holds one step less under way.)
#include "tb_packed.cuh"
#include "tb_tc_ptx.cuh"

#include <algorithm>

#include "tb_attention.cuh"

namespace {

using namespace tbtc;
using namespace tbpk;

constexpr int kFewRows = 16;
constexpr int kStep = 16;              // keys of a warp's step
// Steps of one accumulation of a warp's MMAs (32768 keys): they cut what they add below the sum's last
// place instead of rounding it, and long sums come out short (a warp's 65536, 262144 and 1M keys of equal
// weight in f16: -0.02, -0.14 and -0.65%). Further ones are added up in 32 bits.
constexpr int kChain = 2048;

template <int D> struct FewGeom {
    static constexpr int kBoxes = D / 64;
    static constexpr int kBox = kStep * 128;                      // 16 rows of 64 columns
    static constexpr int kBytes = 2 * kBoxes * kBox;              // a step's K and V
    static constexpr int kStages = 24576 / kBytes;
    static constexpr int kRing = kStages * kBytes;                // of a warp
};

__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_frag(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_frag_turned(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16-byte word w of row `row` in boxes of 64 columns, 128-byte swizzle
template <int D> __device__ __forceinline__ uint32_t word_at(uint32_t base, int row, int w) {
    return base + (w >> 3) * FewGeom<D>::kBox + row * 128 + (((w ^ row) & 7) << 4);
}

template <class T, class O, int D, int W>
__global__ void __launch_bounds__(32 * W, 8 / W)
k_attn_few(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnArgs a) {
    using G = FewGeom<D>;
    constexpr int kBlock = kStep * W;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[W * G::kStages];
    __shared__ float s_max[W][kFewRows], s_sum[W][kFewRows];
    __shared__ int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, col = lane & 3;
    uint32_t idx = blockIdx.x;
    const int split = idx % a.nsplit;
    idx /= a.nsplit;
    const int kvh = idx % a.kv_heads;
    if (threadIdx.x == 0) s_abort = 0;
    if (threadIdx.x < W * G::kStages) {
        mbar_init(smem_u32(bars + threadIdx.x), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    check_table(a.q_off, a.nset, a.nq, a.err);
    check_table(a.k_off, a.nset, a.nk, a.err);
    const Item it = find_item(a.q_off, a.nset, a.nq, a.unit, idx / a.kv_heads, a.err);
    if (it.set < 0) return;
    __syncthreads();                                    // the barriers
    int64_t k0, k1;
    set_range(a.k_off, it.set, a.nk, k0, k1, a.err);
    const int nq = (int)(it.hi - it.lo), nk = (int)(k1 - k0), g = a.group;
    const int t0 = (int)it.item * a.unit, rows = min(a.unit, nq - t0) * g;
    const int end = a.causal ? max(0, min(nk, t0 + (rows - 1) / g + 1 + nk - nq)) : nk;
    const int all = (end + kBlock - 1) / kBlock;
    const int first = (int)((int64_t)all * split / a.nsplit) * kBlock;
    const int stop = min(end, (int)((int64_t)all * (split + 1) / a.nsplit) * kBlock);
    const int kb0 = first + warp * kStep, steps = max(0, (stop - kb0 + kBlock - 1) / kBlock);

    uint8_t* ring = smem_align1024(smem_raw) + warp * G::kRing;
    const uint32_t ring0 = smem_u32(ring), bar0 = smem_u32(bars + warp * G::kStages);
    auto load = [&](int i, int st) {                    // by one lane
        const uint32_t to = ring0 + st * G::kBytes, bar = bar0 + 8 * st;
        mbar_arrive_expect_tx(bar, G::kBytes);
        const int key = (int)k0 + kb0 + i * kBlock;
#pragma unroll
        for (int b = 0; b < G::kBoxes; ++b) tma_load_3d(to + b * G::kBox, &kmap, b * 64, kvh, key, bar);
#pragma unroll
        for (int b = 0; b < G::kBoxes; ++b) tma_load_3d(to + (G::kBoxes + b) * G::kBox, &vmap, b * 64, kvh, key, bar);
    };
    if (lane == 0)
        for (int i = 0; i < G::kStages && i < steps; ++i) load(i, i);
    __syncwarp();

    // the thread's rows are quad and quad + 8
    uint32_t qf[D / 16][4];
    int lim[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int r = quad + 8 * e;
        lim[e] = r >= rows ? 0 : (a.causal ? max(0, min(nk, t0 + r / g + nk - nq + 1)) : nk);
        const T* q = reinterpret_cast<const T*>(a.q) + (it.lo + t0 + r / g) * a.q_row + (int64_t)(kvh * g + r % g) * a.q_head;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const int d = k * 16 + col * 2;
            qf[k][e] = r < rows && d < a.dim ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
            qf[k][2 + e] = r < rows && d + 8 < a.dim ? *reinterpret_cast<const uint32_t*>(q + d + 8) : 0u;
        }
    }
    // p in f16 starts at 2^7 instead of 1: small p keep their digits
    constexpr float lift = std::is_same<T, __half>::value ? 7.f : 0.f;
    const float c = a.scale_log2;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    // What came before this accumulation, against the maxima in keep[D / 2 + e]. Indexed from a number
    // that the compiler does not know, so that it lies in local memory and takes no registers.
    float keep[D / 2 + 2];
    int zero = 0;
    asm volatile("" : "+r"(zero));
    auto add_kept = [&]() {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float had = keep[zero + D / 2 + e], f = had == -INFINITY ? 0.f : ex2(had - m[e]);
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int x = 2 * e; x < 2 * e + 2; ++x) o[n][x] = fmaf(keep[zero + 4 * n + x], f, o[n][x]);
        }
    };

    int st = 0, round = 0;
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
        if (__builtin_expect(i > 0 && i % kChain == 0, 0)) {
            if (i > kChain) add_kept();
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    keep[zero + 4 * n + x] = o[n][x];
                    o[n][x] = 0.f;
                }
            keep[zero + D / 2] = m[0];
            keep[zero + D / 2 + 1] = m[1];
        }
        ok = __all_sync(0xffffffffu, mbar_wait(bar0 + 8 * st, round, &s_abort, a.err));
        if (!ok) break;
        const uint32_t ks = ring0 + st * G::kBytes, vs = ks + G::kBoxes * G::kBox;
        const int kb = kb0 + i * kBlock;
        if (kb + kStep > nk) {
            // rows of V behind the set's last key belong to others and may hold no numbers, which a p of
            // 0 would not cancel; a warp's last step
            for (int w = lane; w < (kb + kStep - nk) * (D / 8); w += 32)
                *reinterpret_cast<uint4*>(ring + st * G::kBytes + G::kBoxes * G::kBox + (w % (D / 8) >> 3) * G::kBox +
                                          (nk - kb + w / (D / 8)) * 128 + (w & 7) * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                uint32_t kf[4];
                load_frag(word_at<D>(ks, n * 8 + (lane & 7), k * 4 + (lane >> 3)), kf);
                mma(s[n], qf[2 * k], kf[0], kf[1], T());
                mma(s[n], qf[2 * k + 1], kf[2], kf[3], T());
            }
        }
        float p[2][4], top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            top[e] = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float& v = s[n][2 * e + x];
                    v = kb + n * 8 + col * 2 + x < lim[e] ? v * c : -INFINITY;
                    top[e] = fmaxf(top[e], v);
                }
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float next = fmaxf(m[e], top[e]), al = next == -INFINITY ? 1.f : ex2(m[e] - next);
                m[e] = next;
                l[e] *= al;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                    o[n][2 * e] *= al;
                    o[n][2 * e + 1] *= al;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float ref = m[e] == -INFINITY ? 0.f : m[e] - lift;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    p[n][2 * e + x] = ex2(s[n][2 * e + x] - ref);
                    l[e] += p[n][2 * e + x];
                }
        }
        // rounded to the operands' type, which the MMA takes (what that costs: exp_block in tb_attention_tc.cu)
        const uint32_t pf[4] = {pack2(p[0][0], p[0][1], T()), pack2(p[0][2], p[0][3], T()), pack2(p[1][0], p[1][1], T()),
                                pack2(p[1][2], p[1][3], T())};
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            uint32_t vf[4];
            load_frag_turned(word_at<D>(vs, (lane >> 3 & 1) * 8 + (lane & 7), 2 * n + (lane >> 4)), vf);
            mma(o[2 * n], pf, vf[0], vf[1], T());
            mma(o[2 * n + 1], pf, vf[2], vf[3], T());
        }
        __syncwarp();                                   // the step has been read
        if (lane == 0 && i + G::kStages < steps) load(i + G::kStages, st);
        __syncwarp();
        if (++st == G::kStages) {
            st = 0;
            round ^= 1;
        }
    }
    if (steps > kChain) add_kept();
    if (!ok) {                                          // loads may still be in flight
        const long long w0 = clock64();
        while (clock64() - w0 < 20000000) { }
    }
    // The warps meet: each leaves its rows in its own ring.
    float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        const int r = quad + 8 * e;
        if (col == 0) {
            s_max[warp][r] = m[e];
            s_sum[warp][r] = l[e];
        }
        if (r < rows)
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float2*>(mine + r * D + n * 8 + col * 2) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
    }
    __syncthreads();
    if (s_abort) return;
    const uint8_t* rings = smem_align1024(smem_raw);
    for (int w = threadIdx.x; w < rows * (D / 8); w += 32 * W) {
        const int r = w / (D / 8), d = w % (D / 8) * 8;
        float mx = s_max[0][r];
#pragma unroll
        for (int e = 1; e < W; ++e) mx = fmaxf(mx, s_max[e][r]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float f = ex2(s_max[e][r] - ref);
            const float* from = reinterpret_cast<const float*>(rings + e * G::kRing) + r * D + d;
            sum = fmaf(f, s_sum[e][r], sum);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = fmaf(f, from[j], v[j]);
        }
        const bool none = sum == 0.f;                   // a row without a key here, or without a score above -inf
        const float inv = none ? 0.f : 1.f / sum, lg = none ? -INFINITY : mx - lift + log2f(sum);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = none ? 0.f : v[j] * inv;
        const int64_t t = it.lo + t0 + r / g;
        const int h = kvh * g + r % g;
        if (a.part) {
            const int64_t at = ((int64_t)split * a.nq + t) * a.heads + h;
            if (d == 0) a.part_lse[at] = lg;
            if (!none && d < a.dim) store8<float>(a.part + at * a.dim + d, v);
        } else {
            if (d == 0 && a.lse) a.lse[t * a.heads + h] = lg * 0.69314718055994530942f;
            if (d < a.dim) store8<O>(reinterpret_cast<O*>(a.out) + t * a.out_row + (int64_t)h * a.out_head + d, v);
        }
    }
}

int64_t few_items(int64_t nq, int nset, int kv_heads, int group) {
    const int unit = kFewRows / group;
    return ((nq + unit - 1) / unit + nset) * kv_heads;
}

// CTAs of a call that cuts no keys, without the empty ones.
int64_t few_ctas(int64_t nq, int nset, int kv_heads, int group) {
    const int unit = kFewRows / group;
    return std::max<int64_t>((nq + unit - 1) / unit, std::min<int64_t>(nset, nq)) * kv_heads;
}

template <class T, class O, int D, int W>
tb_status launch(tb_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnArgs& a, unsigned grid) {
    constexpr size_t sm = (size_t)W * FewGeom<D>::kRing + 1024;
    TB_CUDA_TRY(ctx, cudaFuncSetAttribute(k_attn_few<T, O, D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
    k_attn_few<T, O, D, W><<<grid, 32 * W, sm, ctx->stream>>>(km, vm, a);
    TB_LAUNCH_CHECK(ctx, "k_attn_few");
    return TB_OK;
}
template <class T, class O>
tb_status launch_dim(tb_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnArgs& a, unsigned grid) {
    // one CTA an SM of eight warps, two of four where there are more (8 x 4 tokens, 16 heads of 128, 4096
    // keys, 128 CTAs: 47 us with eight warps, 50 with four and the keys cut in two)
    if (few_ctas(a.nq, a.nset, a.kv_heads, a.group) <= ctx->num_sms)
        return a.dim <= 64 ? launch<T, O, 64, 8>(ctx, km, vm, a, grid) : launch<T, O, 128, 8>(ctx, km, vm, a, grid);
    return a.dim <= 64 ? launch<T, O, 64, 4>(ctx, km, vm, a, grid) : launch<T, O, 128, 4>(ctx, km, vm, a, grid);
}

}  // namespace

// Sets of 16 rows at most, on average. (16 tokens of 32/8 heads of 64 against 1 to 8192 keys: 40 us here, 61
// in 128-row tiles; 16 x 12 heads of 64 against 300 keys: 8 and 15; 8 x 16 rows of 128 against 4096
// keys: 48 and 55.)
bool tb_attn_few(int64_t nq, int nset, int group) { return group <= kFewRows && (nq + nset - 1) / nset * group <= kFewRows; }

// Keys are cut only where one CTA an SM leaves SMs idle, into 512 keys at least: a CTA costs some 8 us
// besides its keys and eight warps keep enough loads under way for the SM. (One token, 32/8 heads of
// 128, 8192 keys: 84 us whole, 15 cut in 16; 4 such tokens: 30 us, with twice the ranges 33; 16 x
// 1..8192: 54 whole, 56 in two.)
int tb_attn_few_nsplit(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int kv_heads, int group) {
    const int64_t ctas = few_ctas(nq, nset, kv_heads, group);
    return (int)std::max<int64_t>(1, std::min<int64_t>({ctx->num_sms / ctas, nk / nset / 512, 32}));
}

tb_status tb_attn_few_launch(tb_ctx* ctx, const AttnArgs& args, tb_dtype dtype, tb_dtype out_dtype) {
    AttnArgs a = args;
    a.unit = kFewRows / a.group;
    const int64_t items = few_items(a.nq, a.nset, a.kv_heads, a.group) * a.nsplit;
    if (items > INT32_MAX) return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: too many rows times heads");
    CUtensorMap km, vm;
    tb_status s = tb_attn_encode(ctx, &km, dtype, a.k, a.dim, a.kv_heads, a.k_head, a.nk, a.k_row, 1, kStep);
    if (s == TB_OK) s = tb_attn_encode(ctx, &vm, dtype, a.v, a.dim, a.kv_heads, a.v_head, a.nk, a.v_row, 1, kStep);
    if (s != TB_OK) return s;
    const unsigned grid = (unsigned)items;
    if (dtype == TB_F16)
        return out_dtype == TB_F32 ? launch_dim<__half, float>(ctx, km, vm, a, grid) : launch_dim<__half, __half>(ctx, km, vm, a, grid);
    return out_dtype == TB_F32 ? launch_dim<__nv_bfloat16, float>(ctx, km, vm, a, grid)
                               : launch_dim<__nv_bfloat16, __nv_bfloat16>(ctx, km, vm, a, grid);
}
