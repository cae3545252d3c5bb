// Packed sets: rows of one array that hold one set (object, sequence) after another, set s in
// rows offsets[s] .. offsets[s+1]-1 of an int32 device array [nset + 1]. Shared by the operators
// over packed sets (tb_attention*.cu, tb_group_norm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tb_common.cuh"
#include "tb_set_walk.cuh"

namespace tbpk {

// Reports every bad offset of a table once, the blocks of the launch together.
__device__ __forceinline__ void check_table(const int32_t* off, int nset, int64_t n, int* err) {
    int64_t lo, hi;
    if (off)
        for (int64_t s = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; s < nset; s += (int64_t)gridDim.x * blockDim.x)
            set_range(off, (int)s, n, lo, hi, err);
}

// The sets cut into pieces of `unit` rows, in order. Set s has the numbers from first_item(s) =
// offsets[s] / unit + s on, at least as many as it has pieces (a few stay without one), so a set's
// numbers need one entry of the table and the set of a number is found by search. Numbers are below
// n / unit + nset, 32 bits.
__device__ __forceinline__ uint32_t first_item(const int32_t* off, int s, int64_t n, int unit) {
    const int64_t o = off ? off[s] : 0;
    return (uint32_t)(o < 0 ? 0 : o > n ? n : o) / (uint32_t)unit + (uint32_t)s;
}
struct Item {
    int set;        // -1: the number is without a piece
    uint32_t item;  // which piece of the set
    uint32_t items; // pieces of the set
    int64_t lo, hi; // the set's rows
};
// Piece number `idx`, by whole warps: a step looks at 32 places, three steps find one of 32768 sets.
__device__ __forceinline__ Item find_item(const int32_t* off, int nset, int64_t n, int unit, uint32_t idx, int* err) {
    const int lane = threadIdx.x & 31;
    int s = 0;
    for (int span = nset; span > 1;) {
        const int step = (span + 31) / 32, at = lane * step;
        const uint32_t below = __ballot_sync(0xffffffffu, at < span && first_item(off, s + min(at, span - 1), n, unit) <= idx);
        const int k = below ? 31 - __clz(below) : 0;
        s += k * step;
        span = min(step, span - k * step);
    }
    Item it;
    set_range(off, s, n, it.lo, it.hi, err);
    const uint32_t first = first_item(off, s, n, unit);
    it.items = (uint32_t)((it.hi - it.lo + unit - 1) / unit);
    it.item = idx - first;
    it.set = idx >= first && it.item < it.items ? s : -1;
    return it;
}

// ---- two 32-bit values in one instruction ----------------------------------------------------------
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack(float a, float b) {
    f2 y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float2 unpack(f2 x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ f2 sub2(f2 a, f2 b) {
    f2 y;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
// 2^x, about 2 steps off; 0 far below, inf far above
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// v / (1 + e^-v) of two values, by one reciprocal of the two sums' product (the exponential unit sets the
// pace). The sums stop at 2^63, whose product still has a reciprocal: below -43.7 the result is v 2^-63
// where it should fall on towards 0, at most 1e-17 |v| off.
__device__ __forceinline__ f2 silu2(f2 v) {
    const float2 e = unpack(mul2(v, pack(-1.44269504088896340736f, -1.44269504088896340736f)));
    const float2 d = unpack(add2(pack(ex2(fminf(e.x, 63.f)), ex2(fminf(e.y, 63.f))), pack(1.f, 1.f)));
    const float r = rcp(d.x * d.y);
    return mul2(v, mul2(pack(d.y, d.x), pack(r, r)));
}

// ---- 8 consecutive elements of a 16-byte aligned row as float ------------------------------------
template <class T> __device__ __forceinline__ void load8(const T* p, float* v);
template <> __device__ __forceinline__ void load8<float>(const float* p, float* v) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void unpack2(uint32_t w, float* v, __nv_bfloat16) {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float* v, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    v[0] = f.x;
    v[1] = f.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T> __device__ __forceinline__ void unpack8(uint4 w, float* v) {
    unpack2(w.x, v, T());
    unpack2(w.y, v + 2, T());
    unpack2(w.z, v + 4, T());
    unpack2(w.w, v + 6, T());
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* v) {
    unpack8<__nv_bfloat16>(*reinterpret_cast<const uint4*>(p), v);
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float* v) {
    unpack8<__half>(*reinterpret_cast<const uint4*>(p), v);
}
template <class T> __device__ __forceinline__ void store8(T* p, const float* v) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                                              pack2(v[6], v[7], T()));
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float* v) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

}  // namespace tbpk

// The calling thread's current device is put back when the call returns.
struct tb_device_guard {
    int prev = -1;
    cudaError_t enter(int device) {
        cudaError_t e = cudaGetDevice(&prev);
        if (e == cudaSuccess && prev != device) return cudaSetDevice(device);
        prev = -1;
        return e;
    }
    ~tb_device_guard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};
