// Packed sets and the walk over them that one warp makes. No more than warp intrinsics, so that a
// host program can run it on lanes of its own; tb_packed.cuh includes it.
#pragma once

#include <stdint.h>

namespace tbpk {

// Rows [lo, hi) of a set. The table lives in device memory, so it is checked here: an offset that
// is negative, smaller than the one before it or past the array's n rows is clamped (no kernel
// reads or writes outside the array) and reported through the context's error word.
__device__ __forceinline__ void set_range(const int32_t* off, int s, int64_t n, int64_t& lo, int64_t& hi, int* err) {
    if (!off) {
        lo = 0;
        hi = n;
        return;
    }
    const int64_t a = off[s], b = off[s + 1];
    if (a < 0 || b < a || b > n) atomicCAS(err, 0, TB_DEVERR_BAD_OFFSETS);
    lo = a < 0 ? 0 : (a > n ? n : a);
    hi = b < lo ? lo : (b > n ? n : b);
}

// The query rows of all sets cut into pieces of `unit` rows, numbered in order without gaps; finds the
// set of a number. Lane l holds set set0 + l of the 32 in hand. Numbers that grow move on from there;
// one that lies before them starts over, since the tiles that a running CTA takes over come in no
// promised order.
struct SetWalk {
    int set0 = -32;
    uint32_t base = 0, total = 0;       // pieces of the sets before those in hand, of those
    uint32_t inc = 0, cnt = 0;          // pieces up to and with the lane's set, of it
    int qlo = 0, qn = 0, klo = 0, kn = 0;   // the lane's set: first rows and counts, below 2^31

    struct Piece {
        int q0, nq, k0, nk;             // the set's query rows and keys
        uint32_t at, of;                // which of the set's pieces, and how many there are
    };
    // False for a number behind the last piece. By a whole warp.
    __device__ __forceinline__ bool find(const int32_t* q_off, const int32_t* k_off, int nset, int64_t nq, int64_t nk, int unit,
                                         uint32_t number, int lane, int* err, Piece& p) {
        if (number < base) {
            set0 = -32;
            base = total = 0;
        }
        while (number >= base + total && set0 + 32 < nset) {
            base += total;
            set0 += 32;
            cnt = 0;
            if (set0 + lane < nset) {
                int64_t lo, hi;
                set_range(q_off, set0 + lane, nq, lo, hi, err);
                qlo = (int)lo;
                qn = (int)(hi - lo);
                set_range(k_off, set0 + lane, nk, lo, hi, err);
                klo = (int)lo;
                kn = (int)(hi - lo);
                cnt = ((uint32_t)qn + (uint32_t)unit - 1) / (uint32_t)unit;
            }
            inc = cnt;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, inc, d);
                if (lane >= d) inc += v;
            }
            total = __shfl_sync(0xffffffffu, inc, 31);
        }
        if (number >= base + total) return false;
        const int src = __ffs(__ballot_sync(0xffffffffu, base + inc > number)) - 1;
        p.of = __shfl_sync(0xffffffffu, cnt, src);
        p.at = number - base - (__shfl_sync(0xffffffffu, inc, src) - p.of);
        p.q0 = __shfl_sync(0xffffffffu, qlo, src);
        p.nq = __shfl_sync(0xffffffffu, qn, src);
        p.k0 = __shfl_sync(0xffffffffu, klo, src);
        p.nk = __shfl_sync(0xffffffffu, kn, src);
        return true;
    }
};

}  // namespace tbpk
