// GroupNorm with an activation over packed sets, channels last: for set s and group g (the
// c / groups consecutive channels of the group over the set's rows)
//   mean, var = the mean and variance of those values,
//   out = act((x - mean) / sqrt(var + eps) * w[channel] + b[channel]).
//
// Up to kGnSmall rows (so no set is longer) one kernel: a block takes one set and a slab of
// channels that holds whole groups, and reads its rows twice, the second time from the caches. Longer
// arrays take three passes: k_gn_stats cuts the sets into pieces of rows, one block a piece, and
// writes each group's mean and sum of squared deviations; k_gn_merge joins a set's pieces;
// k_gn_apply normalises, last pieces first, which L2 still holds.
//
// Statistics: a thread takes 8 channels, reads rows in batches and joins each batch's mean and
// squared deviations with its running ones (no difference of large sums, so a mean far from zero
// costs no digits); entries are joined as
//   mean = sum n_i mean_i / N,  M2 = sum M2_i + sum n_i (mean_i - mean)^2
// always in the same order, so results repeat to the bit. Bound by memory: 262144 x 512 of bf16 in
// 8 sets take 148 us; under the profiler 53 of 152 are the statistics (5.1 TB/s) and 7 their join.
#include "tb_packed.cuh"

#include <algorithm>

namespace {

using namespace tbpk;

constexpr int kGnThreads = 256;
constexpr int kGnMaxC = 2048;
// The bytes at the array's end that k_gn_stats leaves in L2 for k_gn_apply, which begins with them; the
// others go first. (262144 x 512 of bf16: 150 us with 60 MB, 152 with 90 MB, 156 without hints.)
constexpr int64_t kGnKeep = 60 << 20;

struct GnArgs {
    const void* x;
    void* out;
    const int32_t* off;
    const float* w;
    const float* b;
    int64_t n;
    int nset, c, groups, slab;
    int unit, unit_out;   // rows of a piece of k_gn_stats, of k_gn_apply
    float eps;
    int act;
    float2* part;     // [pieces][groups] mean, M2
    float2* stat;     // [nset][groups] mean, 1 / sqrt(var + eps)
    int* err;
};

// A thread's running statistics of 8 channels, two in a register pair.
struct Running {
    f2 mean[4], m2[4];
    int n;
    __device__ void clear() {
#pragma unroll
        for (int j = 0; j < 4; ++j) mean[j] = m2[j] = pack(0.f, 0.f);
        n = 0;
    }
    // joins k rows (a power of two's share is exact) of mean m and squared deviations d2
    __device__ void join(const f2* m, const f2* d2, int k) {
        const float f = (float)k / (float)(n + k), g = f * (float)n;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f2 d = sub2(m[j], mean[j]);
            mean[j] = fma2(d, pack(f, f), mean[j]);
            m2[j] = add2(m2[j], fma2(mul2(d, d), pack(g, g), d2[j]));
        }
        n += k;
    }
};

// 16 bytes with a policy for their stay in L2.
__device__ __forceinline__ uint4 load16(const void* p, uint64_t policy) {
    uint4 v;
    asm volatile("ld.global.L2::cache_hint.v4.b32 {%0,%1,%2,%3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t l2_policy(bool keep) {
    uint64_t normal, first;
    asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(normal));
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
    return keep ? normal : first;
}

// 8 values of 16-bit or 32-bit type as they come from memory: 16-byte words, unpacked when used, so
// that a batch of rows in flight takes few registers.
template <class T> struct Raw8 {
    static constexpr int kRows = 8;      // rows of a batch, in flight together
    uint4 w;
    __device__ void load(const T* p, uint64_t policy) { w = load16(p, policy); }
    __device__ void load_last(const T* p) { w = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ void get(f2* v) const {
        float x[8];
        unpack8<T>(w, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = pack(x[2 * j], x[2 * j + 1]);
    }
};
template <> struct Raw8<float> {
    static constexpr int kRows = 4;
    float4 a, b;
    __device__ void load(const float* p, uint64_t policy) {
        const uint4 u = load16(p, policy), v = load16(p + 4, policy);
        a = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        b = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ void load_last(const float* p) {
        a = __ldcs(reinterpret_cast<const float4*>(p));
        b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ void get(f2* v) const {
        v[0] = pack(a.x, a.y);
        v[1] = pack(a.z, a.w);
        v[2] = pack(b.x, b.y);
        v[3] = pack(b.z, b.w);
    }
};

// Rows r, r + step, ... below r1 of the thread's 8 channels (x: of row 0).
template <class T>
__device__ __forceinline__ void gn_read(Running& s, const T* x, int64_t c, int64_t r, int64_t r1, int64_t step,
                                        uint64_t policy) {
    constexpr int R = Raw8<T>::kRows;
    const f2 zero = pack(0.f, 0.f);
    for (; r < r1; r += R * step) {
        const int k = r + (R - 1) * step < r1 ? R : (int)((r1 - r + step - 1) / step);
        Raw8<T> raw[R];
        f2 m[4] = {zero, zero, zero, zero}, d2[4] = {zero, zero, zero, zero}, v[4];
        if (k == R) {
#pragma unroll
            for (int q = 0; q < R; ++q) raw[q].load(x + (r + q * step) * c, policy);
#pragma unroll
            for (int q = 0; q < R; ++q) {
                raw[q].get(v);
#pragma unroll
                for (int j = 0; j < 4; ++j) m[j] = add2(m[j], v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) m[j] = mul2(m[j], pack(1.f / R, 1.f / R));
#pragma unroll
            for (int q = 0; q < R; ++q) {
                raw[q].get(v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f2 d = sub2(v[j], m[j]);
                    d2[j] = fma2(d, d, d2[j]);
                }
            }
        } else {                         // the last rows, fewer than a batch, in flight together as well
#pragma unroll
            for (int q = 0; q < R; ++q)
                if (q < k) raw[q].load(x + (r + q * step) * c, policy);
            // the share of a third or so is not exact: it multiplies differences from the first row
            f2 first[4];
            raw[0].get(first);
#pragma unroll
            for (int q = 1; q < R; ++q)
                if (q < k) {
                    raw[q].get(v);
#pragma unroll
                    for (int j = 0; j < 4; ++j) m[j] = add2(m[j], sub2(v[j], first[j]));
                }
            const float share = 1.f / (float)k;
#pragma unroll
            for (int j = 0; j < 4; ++j) m[j] = fma2(m[j], pack(share, share), first[j]);
#pragma unroll
            for (int q = 0; q < R; ++q)
                if (q < k) {
                    raw[q].get(v);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f2 d = sub2(v[j], m[j]);
                        d2[j] = fma2(d, d, d2[j]);
                    }
                }
        }
        s.join(m, d2, k);
    }
}

// A mean of entries (mean_i, M2_i, n_i) in two rounds: m from the plain sum, a few steps off, then
// d = sum n_i (mean_i - m), which is near 0 and so keeps its digits, and q = sum M2_i + n_i (mean_i - m)^2;
// the mean is m + d / N, rounded once, and M2 = q - d^2 / N.
__device__ __forceinline__ void gn_add(float off, float m2, float n, float& d, float& q) {
    d = fmaf(n, off, d);
    q += fmaf(n, off * off, m2);
}
__device__ __forceinline__ void gn_settle(float& m, float& m2, float d, float q, float share) {
    const float e = d * share;
    m2 = fmaf(-d, e, q);
    m += e;
}

// Joins the block's threads: `lanes` row lanes of tc threads, 8 channels a thread. Where groups are
// whole threads (cg % 8 == 0) a thread joins its channels first. A group's entries lie together and a
// team of up to 32 threads adds them up; put(g, mean, M2) by its first thread.
template <class F>
__device__ __forceinline__ void gn_join(const Running& s, int ry, int tx, int lanes, int groups, int cg, float rows,
                                        float4* ent, F put) {
    const bool whole = cg % 8 == 0;
    const int ge = whole ? cg / 8 : cg, each = lanes * ge;        // entries of a row lane's group, of a group
    if (ry < lanes) {
        float mean[8], m2[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 a = unpack(s.mean[j]), b = unpack(s.m2[j]);
            mean[2 * j] = a.x;
            mean[2 * j + 1] = a.y;
            m2[2 * j] = b.x;
            m2[2 * j + 1] = b.y;
        }
        if (whole) {
            float d = 0.f, q = 0.f;
#pragma unroll
            for (int j = 1; j < 8; ++j) d += mean[j] - mean[0];
            const float m = fmaf(d, 0.125f, mean[0]);
#pragma unroll
            for (int j = 0; j < 8; ++j) q += m2[j] + (float)s.n * ((mean[j] - m) * (mean[j] - m));
            ent[tx / ge * each + ry * ge + tx % ge] = make_float4(m, q, 8.f * (float)s.n, 0.f);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int ch = tx * 8 + j;
                ent[ch / ge * each + ry * ge + ch % ge] = make_float4(mean[j], m2[j], (float)s.n, 0.f);
            }
        }
    }
    __syncthreads();
    int team = 32;
    while (team > 1 && groups * team > kGnThreads) team /= 2;
    const int sub = threadIdx.x & (team - 1);
    const float share = 1.f / (rows * (float)cg);
    for (int g0 = (threadIdx.x & ~31) / team; g0 < groups; g0 += kGnThreads / team) {
        const int g = g0 + (threadIdx.x & 31) / team;             // whole warps take part in the exchange
        const float4* e = ent + (g < groups ? g : 0) * each;
        auto all = [&](float v) {
            for (int k = team / 2; k; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
            return v;
        };
        float m = 0.f, d = 0.f, q = 0.f;
        for (int i = sub; i < each; i += team) m = fmaf(e[i].z, e[i].x, m);
        m = all(m) * share;
        for (int i = sub; i < each; i += team) gn_add(e[i].x - m, e[i].y, e[i].z, d, q);
        gn_settle(m, q, all(d), all(q), share);
        if (sub == 0 && g < groups) put(g, m, q);
    }
}

// Normalises rows r, r + step, ... below r1 of the thread's 8 channels.
template <class T, class O>
__device__ __forceinline__ void gn_write(const GnArgs& a, const f2* mean, const f2* f, const f2* b, int ch, int64_t r,
                                         int64_t r1, int64_t step) {
    constexpr int R = 4;                 // rows in flight: their loads go before the first store
    const T* x = reinterpret_cast<const T*>(a.x) + ch;
    O* o = reinterpret_cast<O*>(a.out) + ch;
    auto one = [&](const Raw8<T>& raw, int64_t row) {
        f2 v[4];
        float y[8];
        raw.get(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = fma2(sub2(v[j], mean[j]), f[j], b[j]);
            if (a.act) v[j] = silu2(v[j]);
            const float2 z = unpack(v[j]);
            y[2 * j] = z.x;
            y[2 * j + 1] = z.y;
        }
        store8<O>(o + row * a.c, y);
    };
    for (; r + (R - 1) * step < r1; r += R * step) {
        Raw8<T> raw[R];
#pragma unroll
        for (int q = 0; q < R; ++q) raw[q].load_last(x + (r + q * step) * a.c);
#pragma unroll
        for (int q = 0; q < R; ++q) one(raw[q], r + q * step);
    }
    Raw8<T> raw[R];
#pragma unroll
    for (int q = 0; q < R; ++q)
        if (r + q * step < r1) raw[q].load_last(x + (r + q * step) * a.c);
#pragma unroll
    for (int q = 0; q < R; ++q)
        if (r + q * step < r1) one(raw[q], r + q * step);
}

template <class T>
__global__ void __launch_bounds__(kGnThreads, 2) k_gn_stats(const __grid_constant__ GnArgs a) {
    extern __shared__ float4 ent[];
    check_table(a.off, a.nset, a.n, a.err);
    const Item it = find_item(a.off, a.nset, a.n, a.unit, blockIdx.x, a.err);
    if (it.set < 0) return;
    const int tc = a.c / 8, lanes = kGnThreads / tc;
    const int ry = threadIdx.x / tc, tx = threadIdx.x % tc;
    const int64_t r0 = it.lo + (int64_t)it.item * a.unit, r1 = min(it.hi, r0 + a.unit);
    Running s;
    s.clear();
    const uint64_t policy = l2_policy((a.n - r0) * a.c * (int64_t)sizeof(T) < kGnKeep);
    if (ry < lanes) gn_read<T>(s, reinterpret_cast<const T*>(a.x) + tx * 8, a.c, r0 + ry, r1, lanes, policy);
    float2* part = a.part + (int64_t)blockIdx.x * a.groups;
    gn_join(s, ry, tx, lanes, a.groups, a.c / a.groups, (float)(r1 - r0), ent,
            [&](int g, float m, float q) { part[g] = make_float2(m, q); });
}

// One block joins the pieces of a set's groups, one group after another.
__global__ void __launch_bounds__(128) k_gn_merge(const __grid_constant__ GnArgs a) {
    __shared__ float acc[2][4];
    const int set = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t lo, hi;
    set_range(a.off, set, a.n, lo, hi, a.err);
    if (hi == lo) return;
    const int pieces = (int)((hi - lo + a.unit - 1) / a.unit);
    const float cg = (float)(a.c / a.groups), each = (float)a.unit * cg;
    const float last = (float)(hi - lo - (int64_t)(pieces - 1) * a.unit) * cg, share = 1.f / ((float)(hi - lo) * cg);
    auto join = [&](float& x, float& y) {           // the block's sums, in a fixed order
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, d);
            y += __shfl_xor_sync(0xffffffffu, y, d);
        }
        if (lane == 0) {
            acc[0][warp] = x;
            acc[1][warp] = y;
        }
        __syncthreads();
        x = (acc[0][0] + acc[0][1]) + (acc[0][2] + acc[0][3]);
        y = (acc[1][0] + acc[1][1]) + (acc[1][2] + acc[1][3]);
        __syncthreads();
    };
    for (int g = blockIdx.y; g < a.groups; g += gridDim.y) {
        const float2* p = a.part + (int64_t)first_item(a.off, set, a.n, a.unit) * a.groups + g;
        float m = 0.f, d = 0.f, q = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x; i < pieces; i += 128) m = fmaf(i == pieces - 1 ? last : each, p[(int64_t)i * a.groups].x, m);
        join(m, d);
        m *= share;
        d = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x; i < pieces; i += 128) {
            const float2 v = p[(int64_t)i * a.groups];
            gn_add(v.x - m, v.y, i == pieces - 1 ? last : each, d, q);
        }
        join(d, q);
        gn_settle(m, q, d, q, share);
        if (threadIdx.x == 0) a.stat[(int64_t)set * a.groups + g] = make_float2(m, 1.f / sqrtf(fmaf(q, share, a.eps)));
    }
}

// Mean, factor and shift of the thread's 8 channels from its groups' statistics.
__device__ __forceinline__ void gn_factors(const GnArgs& a, const float2* stat, int ch, int first_group, f2* mean, f2* f, f2* b) {
    const int cg = a.c / a.groups;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float2 s = stat[(ch + j) / cg - first_group], t = stat[(ch + j + 1) / cg - first_group];
        mean[j / 2] = pack(s.x, t.x);
        f[j / 2] = a.w ? mul2(pack(s.y, t.y), pack(a.w[ch + j], a.w[ch + j + 1])) : pack(s.y, t.y);
        b[j / 2] = a.b ? pack(a.b[ch + j], a.b[ch + j + 1]) : pack(0.f, 0.f);
    }
}

template <class T, class O>
__global__ void __launch_bounds__(kGnThreads, sizeof(T) == 4 ? 3 : 4) k_gn_apply(const __grid_constant__ GnArgs a) {
    const Item it = find_item(a.off, a.nset, a.n, a.unit_out, gridDim.x - 1 - blockIdx.x, a.err);
    if (it.set < 0) return;
    const int tc = a.c / 8, lanes = kGnThreads / tc;
    const int ry = threadIdx.x / tc, ch = (threadIdx.x % tc) * 8;
    if (ry >= lanes) return;
    const int64_t r0 = it.lo + (int64_t)it.item * a.unit_out, r1 = min(it.hi, r0 + a.unit_out);
    f2 mean[4], f[4], b[4];
    gn_factors(a, a.stat + (int64_t)it.set * a.groups, ch, 0, mean, f, b);
    gn_write<T, O>(a, mean, f, b, ch, r0 + ry, r1, lanes);
}

// Small arrays: block (set, slab of a.slab channels, whole groups).
template <class T, class O>
__global__ void __launch_bounds__(kGnThreads) k_gn_small(const __grid_constant__ GnArgs a) {
    extern __shared__ float4 ent[];
    __shared__ float2 stat[16];                     // a slab has at most 16 groups
    int64_t lo, hi;
    set_range(a.off, blockIdx.x, a.n, lo, hi, a.err);
    if (hi == lo) return;
    const int tc = a.slab / 8, lanes = kGnThreads / tc, cg = a.c / a.groups;
    const int ry = threadIdx.x / tc, tx = threadIdx.x % tc, ch0 = blockIdx.y * a.slab, ch = ch0 + tx * 8;
    Running s;
    s.clear();
    if (ry < lanes) gn_read<T>(s, reinterpret_cast<const T*>(a.x) + ch, a.c, lo + ry, hi, lanes, l2_policy(true));
    const float count = (float)(hi - lo) * cg;
    gn_join(s, ry, tx, lanes, a.slab / cg, cg, (float)(hi - lo), ent,
            [&](int g, float m, float q) { stat[g] = make_float2(m, 1.f / sqrtf(q / count + a.eps)); });
    __syncthreads();
    if (ry >= lanes) return;
    f2 mean[4], f[4], b[4];
    gn_factors(a, stat, ch, ch0 / cg, mean, f, b);
    gn_write<T, O>(a, mean, f, b, ch, lo + ry, hi, lanes);
}

// Channels of a block of the small kernel: the fewest that are whole groups and whole threads and, where
// the array has them, 32 bytes of a row. At most 16 groups.
int gn_slab(int c, int cg, int size) {
    int slab = cg;
    while (slab % 8) slab += cg;                    // divides c, which is a multiple of 8 and of cg
    while (slab * size < 32 && c % (2 * slab) == 0) slab *= 2;
    return slab;
}

// One launch where three would take longer than a second reading by few blocks (800 x 128: 7 us in one,
// 12 in three; 8192 x 512: 24 and 17). Measured with 32 groups. The rule looks at rows alone, and a set of
// few wide groups has few blocks: 4096 x 2048 of bf16 takes 39 us with 32 groups, 268 with 4 and 1060 with
// one, where three launches take 18 (4097 rows).
constexpr int kGnSmall = 4096;
// Pieces an SM: one wave of k_gn_stats's blocks, whose join costs as much as some rows (16384 x 512:
// 22 us with two, 32 with eight); one of k_gn_apply's, or two smaller ones where the array is larger
// than L2 and the pass long enough to have a tail (65536 x 512: 47 us with four, 49 with eight;
// 262144 x 512: 151 and 148).
constexpr int kGnPieces = 2;
int gn_pieces_out(int64_t n, int c, tb_dtype t) { return n * c * (int64_t)tb_dtype_size(t) > 2 * kGnKeep ? 8 : 4; }

// Rows of a piece, so that the sets' ends included there are `per` pieces an SM, and 16 rows at least.
int gn_unit(int num_sms, int64_t n, int nset, int per) {
    const int64_t pieces = (int64_t)per * num_sms - std::min(nset, per * num_sms / 2);
    return (int)std::max<int64_t>(16, (n + pieces - 1) / pieces);
}
int64_t gn_pieces(int64_t n, int nset, int unit) { return (n + unit - 1) / unit + nset; }

template <class T>
void launch_gn(const GnArgs& a, bool f32_out, cudaStream_t st) {
    if (a.slab) {
        const int cg = a.c / a.groups;
        const size_t sm = (size_t)(kGnThreads / (a.slab / 8)) * a.slab / (cg % 8 == 0 ? 8 : 1) * sizeof(float4);
        const dim3 grid((unsigned)a.nset, (unsigned)(a.c / a.slab));
        if (f32_out) k_gn_small<T, float><<<grid, kGnThreads, sm, st>>>(a);
        else k_gn_small<T, T><<<grid, kGnThreads, sm, st>>>(a);
        return;
    }
    const size_t sm = (size_t)(kGnThreads / (a.c / 8)) * a.c / (a.c / a.groups % 8 == 0 ? 8 : 1) * sizeof(float4);
    k_gn_stats<T><<<(unsigned)gn_pieces(a.n, a.nset, a.unit), kGnThreads, sm, st>>>(a);
    const unsigned gy = (unsigned)std::min(a.groups, std::max(1, 4096 / a.nset));
    k_gn_merge<<<dim3((unsigned)a.nset, gy), 128, 0, st>>>(a);
    const unsigned blocks = (unsigned)gn_pieces(a.n, a.nset, a.unit_out);
    if (f32_out) k_gn_apply<T, float><<<blocks, kGnThreads, 0, st>>>(a);
    else k_gn_apply<T, T><<<blocks, kGnThreads, 0, st>>>(a);
}

}  // namespace

extern "C" size_t tb_group_norm_workspace_bytes(const tb_ctx* ctx, int64_t n, int c, int groups, int nset) {
    if (!ctx || n <= 0 || c < 1 || groups < 1 || c % groups != 0 || nset < 1 || n <= kGnSmall) return 0;
    return (size_t)(gn_pieces(n, nset, gn_unit(ctx->num_sms, n, nset, kGnPieces)) + nset) * groups * sizeof(float2);
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
    if (out != x && tb_rows_overlap({out, 1, 0, n * c * (int64_t)tb_dtype_size(out_dtype)},
                                    {x, 1, 0, n * c * (int64_t)tb_dtype_size(x_dtype)}))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: out must be x or not overlap it");
    const size_t need = tb_group_norm_workspace_bytes(ctx, n, c, groups, nset);
    if (need && (!workspace || workspace_bytes < need || !tb_aligned16(workspace)))
        return tb_fail(ctx, TB_ERR_INVALID_ARG, "tb_group_norm: workspace too small or not 16-byte aligned");
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
    a.unit = gn_unit(ctx->num_sms, n, nset, kGnPieces);
    a.unit_out = gn_unit(ctx->num_sms, n, nset, gn_pieces_out(n, c, x_dtype));
    a.slab = n <= kGnSmall ? gn_slab(c, c / groups, (int)tb_dtype_size(x_dtype)) : 0;
    a.eps = eps;
    a.act = act == TB_EPI_SILU;
    a.part = reinterpret_cast<float2*>(workspace);
    a.stat = a.part + gn_pieces(n, nset, a.unit) * groups;
    a.err = ctx->d_err;
    tb_device_guard guard;
    TB_CUDA_TRY(ctx, guard.enter(ctx->device));
    if (x_dtype == TB_F32) launch_gn<float>(a, true, ctx->stream);
    else if (x_dtype == TB_F16) launch_gn<__half>(a, out_dtype == TB_F32, ctx->stream);
    else launch_gn<__nv_bfloat16>(a, out_dtype == TB_F32, ctx->stream);
    TB_LAUNCH_CHECK(ctx, "tb_group_norm");
    return TB_OK;
}
