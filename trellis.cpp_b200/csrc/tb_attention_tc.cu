// Attention within packed sets on tcgen05 (bf16 / f16 operands); the mathematics and the entry point
// are in tb_attention.cu.
//
// One CTA takes 256 query rows of one key head as two tiles of 128 (a row is a token and one of the
// heads that share the key head, so the keys of a group are read once) and walks the keys in
// blocks of 128: S = Q K^T into 128 TMEM columns a tile, softmax by one warpgroup a tile (a thread
// owns a row: no exchange between threads), P over S's columns as the A operand of O += P V, which
// stays in TMEM. While one tile's warpgroup computes its softmax the tensor pipe works on the other
// tile. One warp streams Q, K and V by TMA, one a tile issues the MMAs.
//
// The running maximum moves only when a block's exceeds it by more than 2^8 (in units of p): until
// then p grows to at most 2^8, which the 32-bit sums hold as well, and O need not be scaled; the
// result is the same since the sum carries the same factor. A block's S is committed after the
// tile's last P V, so O is at rest while the softmax warps scale it.
//
// With few query rows a set (ALT) one tile holds them and the two halves of the CTA take every
// other block of keys; with few CTAs the keys are also cut into `nsplit` ranges. Both leave partial
// rows (32 bits, normalised, with their log sums) that k_attn_join adds up in a fixed order.
#include "tb_packed.cuh"
#include "tb_tc_ptx.cuh"

#include <algorithm>

#include "tb_attention.cuh"

namespace {

using namespace tbtc;
using namespace tbpk;

constexpr int kThreads = 384;          // warps 0-3 and 4-7 softmax, 8 and 9 MMA, 10 TMA, 11 idle
// Registers: 65536 / 384 threads allows 168 at launch; the third warpgroup gives up what the two
// softmax warpgroups need to hold a row of S. 2 * 208 + 88 = 3 * 168.
constexpr int kRegsSoftmax = 208, kRegsOther = 88;
constexpr int kKeys = 128;             // keys of a block
constexpr float kRaise = 8.f;          // the maximum follows when a block's is 2^8 above it
#ifndef TB_FIRST
#define TB_FIRST 96
#endif
constexpr int kFirst = TB_FIRST;             // keys of a block whose p the products may read early
#ifndef TB_POLY
#define TB_POLY 3
#endif
constexpr int kPoly = TB_POLY;         // of every 8 pairs of exponentials, those by polynomial

struct TcArgs {
    AttnArgs a;
    float* part;                       // [nsp][nq][heads][dim] partial rows, null without splits
    float* part_lse;                   // [nsp][nq][heads], base 2
    int nsplit, tile_tokens;           // key ranges; tokens of a 128-row tile
    uint32_t idesc_s, idesc_o, q_bytes;
};

template <int D, bool ALT> struct Geom {
    static constexpr int kBoxes = D / 64;
    static constexpr int kTileBytes = kBoxes * 16384;         // 128 rows x D, boxes of 64 columns
    static constexpr int kQTiles = ALT ? 1 : 2;
    static constexpr int kStages = D == 64 ? 10 : (ALT ? 6 : 5);
    static constexpr int kBars = 2 * kStages + 1 + 2 + 2 + 2 + 2 + 2 + 1;
    static constexpr size_t kSmem = (size_t)(kQTiles + kStages) * kTileBytes + 8 * kBars + 16 + 1024;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// Shared-memory descriptors of tiles in the 128-byte swizzle: low word (address >> 4) | leading
// offset << 16, high word 8-row groups 1024 bytes apart. Q and K have their K dimension (the head's
// columns) contiguous; V is the B operand with N (the head's columns) contiguous, its boxes of 64
// columns 16384 bytes apart.
__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                   "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                   "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]),
                   "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]),
                   "=f"(v[30]), "=f"(v[31])
                 : "r"(taddr));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 2^x of two values on the FMA pipes, beside the exponential unit: x = i + f with i the nearest whole
// number, 2^f by the cubic of least relative error on [-1/2, 1/2] (exchange method, 7.5e-5: an
// eighth of a half step of f16), times 2^i put together from its bits. x is taken at -126 at
// least; a value that is no number stays one (the product keeps it).
__device__ __forceinline__ float2 ex2_poly(f2 x) {
    float2 v = unpack(x);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(-126.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(-126.f));
    x = pack(v.x, v.y);
    const f2 r = add2(x, pack(12582912.f, 12582912.f));                     // 1.5 * 2^23: whole numbers
    const f2 f = fma2(add2(r, pack(-12582912.f, -12582912.f)), pack(-1.f, -1.f), x);
    f2 y = fma2(pack(0.0551716685f, 0.0551716685f), f, pack(0.242611125f, 0.242611125f));
    y = fma2(y, f, pack(0.693260968f, 0.693260968f));
    y = fma2(y, f, pack(0.999928057f, 0.999928057f));
    const float2 i = unpack(r);
    const float e0 = __uint_as_float((__float_as_uint(i.x) << 23) + 0x3f800000u);
    const float e1 = __uint_as_float((__float_as_uint(i.y) << 23) + 0x3f800000u);
    return unpack(mul2(y, pack(e0, e1)));
}

// p = 2^(s c + ref) of a row's 128 scores, left in s and, rounded to T, in the TMEM columns from `ts`.
// NPOLY of every 8 pairs go by polynomial, which shares the work between the exponential unit (4
// lanes a cycle and scheduler: 1024 cycles a block and warp, as long as the tile's products) and the
// FMA pipes. A hidden score (-inf) has to give exactly 0: masked blocks use NPOLY 0.
template <class T, int NPOLY>
__device__ __forceinline__ void exp_block(float* s, float c, float ref, uint32_t ts, uint32_t half_bar, int lane) {
    const f2 c2 = pack(c, c), ref2 = pack(ref, ref);
#pragma unroll
    for (int quarter = 0; quarter < 4; ++quarter) {
        float* v = s + quarter * 32;
#pragma unroll
        for (int q = 0; q < 32; q += 2) {
            const float2 x = unpack(fma2(pack(v[q], v[q + 1]), c2, ref2));
            v[q] = x.x;
            v[q + 1] = x.y;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if ((q & 7) * NPOLY / 8 == ((q & 7) + 1) * NPOLY / 8) {
                v[2 * q] = ex2(v[2 * q]);
                v[2 * q + 1] = ex2(v[2 * q + 1]);
            }
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if ((q & 7) * NPOLY / 8 != ((q & 7) + 1) * NPOLY / 8) {
                const float2 y = ex2_poly(pack(v[2 * q], v[2 * q + 1]));
                v[2 * q] = y.x;
                v[2 * q + 1] = y.y;
            }
        uint32_t w[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) w[q] = pack2(v[2 * q], v[2 * q + 1], T());
        tmem_st_x16(ts + quarter * 16, w);
        if (quarter == kFirst / 32 - 1) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(half_bar);
        }
    }
}

// What one CTA works on, in shared memory.
struct Job {
    int64_t q0, k0;        // first query row and key row of the set
    int nq, nk;            // rows of the set
    int t0;                // first token of the CTA, in the set
    int blk0;              // first key block
    int n[2];              // key blocks of each tile (ALT: of the CTA, n[0])
};

template <class T, class O, int D, bool ALT>
__global__ void __launch_bounds__(kThreads, 1)
k_attn_tc(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
          const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcArgs p) {
    using G = Geom<D, ALT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Item it_s;
    __shared__ uint32_t scan[32];
    uint8_t* smem = smem_align1024(smem_raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (G::kQTiles + G::kStages) * G::kTileBytes);
    uint32_t* s_misc = reinterpret_cast<uint32_t*>(bars + G::kBars);       // [0] tmem, [1] abort
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_misc + 1);
    const uint32_t b0 = smem_u32(bars);
    auto full = [&](int s) { return b0 + 8u * s; };
    auto empty = [&](int s) { return b0 + 8u * (G::kStages + s); };
    const uint32_t bq = b0 + 8u * (2 * G::kStages);
    auto sfull = [&](int i) { return bq + 8u * (1 + i); };
    auto pfull = [&](int i) { return bq + 8u * (3 + i); };
    auto ofull = [&](int i) { return bq + 8u * (5 + i); };
    auto phalf = [&](int i) { return bq + 8u * (7 + i); };
    auto turn = [&](int i) { return bq + 8u * (9 + i); };
    const uint32_t drain = bq + 8u * 11;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AttnArgs& a = p.a;

    uint32_t idx = blockIdx.x;
    const int split = idx % p.nsplit;
    idx /= p.nsplit;
    const int kvh = idx % a.kv_heads;
    find_item(a.q_off, a.nset, a.nq, a.unit, idx / a.kv_heads, a.err, &it_s, scan);
    if (it_s.set < 0) return;
    Job j;
    {
        int64_t k1;
        set_range(a.k_off, it_s.set, a.nk, j.k0, k1, a.err);
        j.q0 = it_s.lo;
        j.nq = (int)(it_s.hi - it_s.lo);
        j.nk = (int)(k1 - j.k0);
        // causal: the last rows of a set see the most keys; they go first
        j.t0 = (a.causal ? (int)(it_s.items - 1 - it_s.item) : (int)it_s.item) * a.unit;
        int nb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int first = j.t0 + (ALT ? 0 : i * p.tile_tokens), last = min(first + p.tile_tokens, j.nq) - 1;
            const int end = a.causal ? max(0, min(j.nk, last + 1 + j.nk - j.nq)) : j.nk;
            nb[i] = first < j.nq ? (end + kKeys - 1) / kKeys : 0;
        }
        const int all = max(nb[0], nb[1]);
        j.blk0 = (int)((int64_t)all * split / p.nsplit);
        const int blk1 = (int)((int64_t)all * (split + 1) / p.nsplit);
        j.n[0] = max(0, min(blk1, nb[0]) - j.blk0);
        j.n[1] = max(0, min(blk1, nb[1]) - j.blk0);
    }
    const int nmax = max(j.n[0], j.n[1]);

    if (threadIdx.x == 0) {
        for (int s = 0; s < G::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), ALT ? 1 : 2);        // every tile that reads it
        }
        mbar_init(bq, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(sfull(i), 1);
            mbar_init(pfull(i), 4);
            mbar_init(phalf(i), 4);
            mbar_init(turn(i), 1);
            mbar_init(ofull(i), 1);
        }
        mbar_init(drain, 2);
        s_misc[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(s_misc)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_misc[0];
    const uint32_t sq = smem_u32(smem), skv = sq + G::kQTiles * G::kTileBytes;
    int issued = 0;

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsOther));
    if (warp == 10) {
        // ------------------------------------------------------------------ TMA producer
        if (nmax > 0 && elect_one()) {
            const bool two = !ALT && j.n[1] > 0;
            mbar_arrive_expect_tx(bq, p.q_bytes * (two ? 2u : 1u));
            for (int t = 0; t < (two ? 2 : 1); ++t)
                for (int b = 0; b < G::kBoxes; ++b)
                    tma_load_3d(sq + t * G::kTileBytes + b * 16384, &qmap, b * 64, kvh * a.group,
                                (int)j.q0 + j.t0 + t * p.tile_tokens, bq);
            // blocks in the order in which the MMA warp needs them: K0 V0 K1 V1 ...;
            // ALT: K0 K1 V0 K2 V1 ... (two blocks are in work)
            for (int it = 0; it < 2 * nmax; ++it) {
                bool is_v = it & 1;
                int blk = it >> 1;
                if (ALT) {
                    is_v = it == 2 * nmax - 1 || (it > 0 && !(it & 1));
                    blk = it == 0 ? 0 : it == 2 * nmax - 1 ? nmax - 1 : is_v ? (it - 2) / 2 : (it + 1) / 2;
                }
                const int s = it % G::kStages;
                if (it >= G::kStages && !mbar_wait(empty(s), (uint32_t)((it / G::kStages - 1) & 1), s_abort, a.err)) break;
                mbar_arrive_expect_tx(full(s), G::kTileBytes);
                for (int b = 0; b < G::kBoxes; ++b)
                    tma_load_3d(skv + s * G::kTileBytes + b * 16384, is_v ? &vmap : &kmap, b * 64, kvh,
                                (int)j.k0 + (j.blk0 + blk) * kKeys, full(s));
                issued = it + 1;
            }
        }
        issued = __shfl_sync(0xffffffffu, __reduce_max_sync(0xffffffffu, issued), 0);
        __syncwarp();
    } else if (warp < 10) {
        // ------------------------------------------------------------------ MMA issuers, one a tile
        // A wait costs some 150 cycles of dependent instructions even when its phase is over, and one
        // warp for both tiles left the tensor pipe idle for 1600 of 3600 cycles a block; so each tile
        // has its own, the ring's place is counted along and descriptors differ by constants.
        const int i = warp - 8;
        bool ok = nmax > 0;
        uint32_t stage = 0, round = 0;               // ring place of the next item
        auto wait = [&](uint32_t bar, uint32_t par) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, par, s_abort, a.err));
            return ok;
        };
        auto take = [&]() {                          // the next ring item once it has landed
            const uint32_t st = stage;
            wait(full(st), round);
            if (++stage == G::kStages) {
                stage = 0;
                round ^= 1;
            }
            return st;
        };
        auto release = [&](uint32_t st) {
            if (elect_one()) tc_commit(empty(st));
            __syncwarp();
        };
        const uint32_t qlo = (sq >> 4) | (1u << 16), klo = (skv >> 4) | (1u << 16), vlo = (skv >> 4) | (1024u << 16);
        constexpr uint32_t kHi = 64u | (1u << 14) | (2u << 29);
        // S of tile i = Q K^T with K in ring place st
        auto mma_s = [&](uint32_t st) {
            const uint32_t ql = qlo + (ALT ? 0u : (uint32_t)(i * (G::kTileBytes >> 4))), kl = klo + st * (G::kTileBytes >> 4);
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t o = (uint32_t)((k >> 2) * 1024 + (k & 3) * 2);
                    if (k * 16 < a.dim)
                        tc_mma(tmem + (uint32_t)(i * 128), desc64(ql + o, kHi), desc64(kl + o, kHi), p.idesc_s, k ? 1u : 0u);
                }
                tc_commit(sfull(i));
            }
            __syncwarp();
        };
        // The tiles take turns, a block's P V and the next S together: issued at once they would finish
        // together, and both softmaxes would then wait for the tensor pipe and it for them.
        auto my_turn = [&](int k) {
            if (!ALT && (i || k)) wait(turn(i), (uint32_t)((k - 1 + i) & 1));
            return ok;
        };
        auto pass = [&]() {
            if (!ALT && lane == 0) mbar_arrive(turn(1 - i));
        };
        // O of tile i += P V over the block's first `keys` keys, the early ones as soon as their p is there
        auto mma_o = [&](uint32_t st, int blk, bool first, int keys, uint32_t par) {
            const uint32_t vl = vlo + st * (G::kTileBytes >> 4);
            const uint32_t td = tmem + 256u + (uint32_t)(i * D), ta = tmem + (uint32_t)(i * 128);
            if (!my_turn(blk + 1) || !wait(phalf(i), par)) return false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kFirst / 16; ++k)
                    if (k * 16 < keys) tc_mma_ts(td, ta + k * 8, desc64(vl + k * 128, kHi), p.idesc_o, first && k == 0 ? 0u : 1u);
            }
            __syncwarp();
            if (!wait(pfull(i), par)) return false;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = kFirst / 16; k < kKeys / 16; ++k)
                    if (k * 16 < keys) tc_mma_ts(td, ta + k * 8, desc64(vl + k * 128, kHi), p.idesc_o, 1u);
            }
            __syncwarp();
            return true;
        };
        auto last = [&]() {
            if (elect_one()) tc_commit(ofull(i));
            __syncwarp();
        };
        // The rows of V behind the set's last key belong to others and may hold no numbers, which a
        // p of 0 would not cancel: those of the last 16 that the products read become 0.
        auto clean = [&](uint32_t st, int keys) {
            if (keys >= kKeys || (keys & 15) == 0) return;
            uint8_t* v = smem + (G::kQTiles + st) * G::kTileBytes;
            for (int c = lane; c < (16 - (keys & 15)) * 8 * G::kBoxes; c += 32) {
                const int row = keys + c / (8 * G::kBoxes), x = c % (8 * G::kBoxes);
                *reinterpret_cast<uint4*>(v + (x >> 3) * 16384 + row * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        int keys = j.nk - j.blk0 * kKeys;            // left from the block on
        wait(bq, 0);
        if (!ALT) {
            const int n = j.n[i];                    // the other tile may have more blocks: their places pass
            const uint32_t k0 = take();
            if (my_turn(0)) {
                if (n > 0) mma_s(k0);
                pass();
                release(k0);
            }
            for (int b = 0; b < nmax && ok; ++b, keys -= kKeys) {
                const uint32_t v = take(), k = b + 1 < nmax ? take() : 0;
                if (!ok) break;
                if (b < n) {
                    clean(v, keys);
                    if (!mma_o(v, b, b == 0, keys, (uint32_t)(b & 1))) break;
                    if (b + 1 < n) mma_s(k);
                    else last();
                } else if (!my_turn(b + 1)) {
                    break;
                }
                pass();
                release(v);
                if (b + 1 < nmax) release(k);
            }
        } else {
            // ring: K0 K1 V0 K2 V1 ...; this tile's blocks are i, i + 2, ...
            const int n = nmax;
            auto skip = [&]() {
                if (++stage == G::kStages) {
                    stage = 0;
                    round ^= 1;
                }
            };
            if (i == 0) {
                const uint32_t k = take();
                if (ok) {
                    mma_s(k);
                    release(k);
                }
                if (n > 1) skip();
            } else if (n > 1) {
                skip();
                const uint32_t k = take();
                if (ok) {
                    mma_s(k);
                    release(k);
                }
            }
            for (int b = 0; b < n && ok; ++b, keys -= kKeys) {
                if ((b & 1) != i) {                  // the other tile's V and K
                    skip();
                    if (b + 2 < n) skip();
                    continue;
                }
                const uint32_t v = take(), k = b + 2 < n ? take() : 0;
                if (!ok) break;
                clean(v, keys);
                if (!mma_o(v, b, b < 2, keys, (uint32_t)((b >> 1) & 1))) break;
                if (b + 2 < n) mma_s(k);
                else last();
                release(v);
                if (b + 2 < n) release(k);
            }
        }
        // every MMA has completed before the TMEM is freed (also after an abort)
        if (elect_one()) tc_commit(drain);
        __syncwarp();
        const long long t0 = clock64();
        while (!mbar_try_wait(drain, 0) && clock64() - t0 < kWaitCycles) { }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kRegsSoftmax));
        // ------------------------------------------------------------------ softmax and output
        const int i = warp >> 2, r = (warp & 3) * 32 + lane;
        const int t = j.t0 + (ALT ? 0 : i * p.tile_tokens) + r / a.group;
        const int h = kvh * a.group + r % a.group;
        const bool valid = r < p.tile_tokens * a.group && t < j.nq;
        const int lim = !valid ? j.nk : a.causal ? max(0, min(j.nk, t + 1 + j.nk - j.nq)) : j.nk;   // keys the row sees
        const int wlim = __reduce_min_sync(0xffffffffu, lim);
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ts = lane_base + (uint32_t)(i * 128), to = lane_base + 256u + (uint32_t)(i * D);
        const float c = a.scale_log2;
        // p in f16 starts at 2^7 instead of 1 (2^15 after the largest rise): small p keep their digits
        constexpr float lift = std::is_same<T, __half>::value ? 7.f : 0.f;
        const int n = ALT ? (j.n[0] + 1 - i) / 2 : j.n[i];
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int b = 0; b < n; ++b) {
            const int key0 = (j.blk0 + (ALT ? 2 * b + i : b)) * kKeys;
            if (!__all_sync(0xffffffffu, mbar_wait(sfull(i), (uint32_t)(b & 1), s_abort, a.err))) { ok = false; break; }
            tc_fence_after();
            float s[128];
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld_x32(ts + q * 32, s + q * 32);
            tmem_wait_ld();
            const bool masked = wlim < key0 + kKeys;
            if (masked) {
                const int left = lim - key0;
#pragma unroll
                for (int q = 0; q < 128; ++q) s[q] = q < left ? s[q] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int q = 4; q < 124; q += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[q + e], s[q + 4 + e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[124 + e]);
            const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
            if (b == 0) {
                m = mn;
            } else if (__any_sync(0xffffffffu, (mn - m) * c > kRaise)) {
                const float al = mn == m ? 1.f : ex2((m - mn) * c);
                m = mn;
                l *= al;
#pragma unroll 1
                for (int q = 0; q < D; q += 32) {
                    float o[32];
                    tmem_ld_x32(to + q, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] *= al;
                    tmem_st_x32(to + q, reinterpret_cast<const uint32_t*>(o));
                }
            }
            const float ref = lift - (m == -INFINITY ? 0.f : m * c);
            // p in quarters of 32 keys; the products start on the first kFirst keys
            if (masked) exp_block<T, 0>(s, c, ref, ts, phalf(i), lane);
            else exp_block<T, kPoly>(s, c, ref, ts, phalf(i), lane);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull(i));
            f2 sum[2] = {pack(s[0], s[1]), pack(s[2], s[3])};
#pragma unroll
            for (int q = 4; q < 128; q += 4) {
                sum[0] = add2(sum[0], pack(s[q], s[q + 1]));
                sum[1] = add2(sum[1], pack(s[q + 2], s[q + 3]));
            }
            const float2 both = unpack(add2(sum[0], sum[1]));
            l += both.x + both.y;
        }
        if (n > 0 && ok) {
            ok = __all_sync(0xffffffffu, mbar_wait(ofull(i), 0, s_abort, a.err));
            tc_fence_after();
        }
        if (ok) {
            const bool none = n == 0 || lim <= (j.blk0 + (ALT ? i : 0)) * kKeys;    // the row sees no key here
            const float inv = none ? 0.f : 1.f / l;
            const float lg = none ? -INFINITY : m * c - lift + log2f(l);
            const int64_t row = j.q0 + t;
            if (p.part) {
                const int64_t at = ((int64_t)(ALT ? 2 * split + i : split) * a.nq + row) * a.heads + h;
                if (valid) p.part_lse[at] = lg;
                float* out = p.part + at * a.dim;
                if (n > 0) {
#pragma unroll 1
                    for (int q = 0; q < D; q += 32) {
                        float o[32];
                        __syncwarp();
                        tmem_ld_x32(to + q, o);
                        tmem_wait_ld();
                        if (!valid || none) continue;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (q + e < a.dim)
                                *reinterpret_cast<float4*>(out + q + e) =
                                    make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
                    }
                }
            } else {
                if (valid && a.lse) a.lse[row * a.heads + h] = lg * 0.69314718055994530942f;
                O* out = reinterpret_cast<O*>(a.out) + row * a.out_row + (int64_t)h * a.out_head;
#pragma unroll 1
                for (int q = 0; q < D; q += 32) {
                    float o[32];
                    __syncwarp();
                    if (n > 0) {
                        tmem_ld_x32(to + q, o);
                        tmem_wait_ld();
                    }
                    if (!valid) continue;
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = none ? 0.f : o[e] * inv;
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        if (q + e < a.dim) store8<O>(out + q + e, o + e);
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 10 && lane == 0 && *s_abort) {
        // after an abort, TMA loads still in flight land before the CTA exits
        const long long t0 = clock64();
        for (int it = max(0, issued - G::kStages); it < issued; ++it)
            while (!mbar_try_wait(full(it % G::kStages), (uint32_t)((it / G::kStages) & 1)) && clock64() - t0 < kWaitCycles) { }
        while (nmax > 0 && !mbar_try_wait(bq, 0) && clock64() - t0 < kWaitCycles) { }
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the partial rows: with lg_s the base-2 log sum of part s and M their maximum,
//   out = sum_s 2^(lg_s - M) out_s / sum_s 2^(lg_s - M),  lse = (M + log2(that sum)) / log2(e).
// A warp a row and head, parts in order.
template <class O>
__global__ void __launch_bounds__(256) k_attn_join(const __grid_constant__ TcArgs p, int nsp) {
    const AttnArgs& a = p.a;
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, hi = a.nq;
    if (a.q_off) {
        lo = min(max((int64_t)a.q_off[0], (int64_t)0), a.nq);
        hi = min((int64_t)a.q_off[a.nset], a.nq);
    }
    const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t row = at / a.heads, h = at % a.heads;
    if (row < lo || row >= hi) return;
    const int64_t step = a.nq * a.heads;
    float mx = -INFINITY;
    for (int s = lane; s < nsp; s += 32) mx = fmaxf(mx, p.part_lse[s * step + at]);
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const int c0 = lane * 4;
    // a log sum that is no number does not show in the maximum: it goes by its weight
    for (int s = 0; s < nsp; ++s) {
        const float lg = p.part_lse[s * step + at];
        if (lg == -INFINITY) continue;              // no key here, nothing was written
        const float w = exp2f(lg - mx);
        sum += w;
        if (c0 < a.dim) {
            const float4 v = *reinterpret_cast<const float4*>(p.part + (s * step + at) * a.dim + c0);
            o[0] = fmaf(w, v.x, o[0]);
            o[1] = fmaf(w, v.y, o[1]);
            o[2] = fmaf(w, v.z, o[2]);
            o[3] = fmaf(w, v.w, o[3]);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (lane == 0 && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994530942f;
    if (c0 >= a.dim) return;
    O* out = reinterpret_cast<O*>(a.out) + row * a.out_row + h * a.out_head + c0;
    if (sizeof(O) == 4) {
        *reinterpret_cast<float4*>(out) = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    } else {
        using H = typename std::conditional<sizeof(O) == 4, __half, O>::type;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack2(o[0] * inv, o[1] * inv, H()), pack2(o[2] * inv, o[3] * inv, H()));
    }
}

struct Plan {
    bool alt;
    int tile_tokens, unit, nsplit, nsp;
    int64_t items;
};

// ALT when an average set's rows fit one tile. Keys are cut where the CTAs would not fill the SMs.
Plan attn_plan(int num_sms, int64_t nq, int64_t nk, int nset, int kv_heads, int group) {
    Plan l;
    l.tile_tokens = 128 / group;
    l.alt = (nq + nset - 1) / nset <= l.tile_tokens;
    l.unit = l.alt ? l.tile_tokens : 2 * l.tile_tokens;
    const int64_t pieces = (nq + l.unit - 1) / l.unit;
    const int64_t ctas = std::max<int64_t>(pieces, std::min<int64_t>(nset, nq)) * kv_heads;
    const int64_t blocks = (nk / nset + kKeys - 1) / kKeys;          // of an average set
    l.nsplit = 1;
    if (ctas < 2 * num_sms)
        l.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({4ll * num_sms / ctas, blocks / 8, 32}));
    l.nsp = l.alt ? 2 * l.nsplit : (l.nsplit > 1 ? l.nsplit : 0);
    l.items = (pieces + nset) * kv_heads * l.nsplit;
    return l;
}

tb_status encode(tb_ctx* ctx, CUtensorMap* map, tb_dtype dtype, const void* base, int dim, int64_t heads, int64_t head,
                 int64_t rows, int64_t row, uint32_t box_heads, uint32_t box_rows) {
    if (!ctx->encode_tiled) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        TB_CUDA_TRY(ctx, cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        if (!fn || q != cudaDriverEntryPointSuccess)
            return tb_fail(ctx, TB_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
        ctx->encode_tiled = fn;
    }
    const cuuint64_t gdim[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t stride[2] = {(cuuint64_t)(heads > 1 ? head : dim) * 2, (cuuint64_t)(rows > 1 ? row : dim) * 2};
    const cuuint32_t box[3] = {64, box_heads, box_rows}, es[3] = {1, 1, 1};
    const CUresult cr = reinterpret_cast<EncodeTiledFn>(ctx->encode_tiled)(
        map, dtype == TB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
        gdim, stride, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? TB_OK : tb_fail(ctx, TB_ERR_CUDA, "cuTensorMapEncodeTiled failed for tb_attention");
}

template <class T, class O, int D, bool ALT>
tb_status launch(tb_ctx* ctx, const TcArgs& p, const Plan& l, const CUtensorMap& qm, const CUtensorMap& km,
                 const CUtensorMap& vm) {
    constexpr size_t sm = Geom<D, ALT>::kSmem;
    if (sm > (size_t)ctx->max_smem_optin) return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_attention: shared memory too small");
    TB_CUDA_TRY(ctx, cudaFuncSetAttribute(k_attn_tc<T, O, D, ALT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
    k_attn_tc<T, O, D, ALT><<<(unsigned)l.items, kThreads, sm, ctx->stream>>>(qm, km, vm, p);
    TB_LAUNCH_CHECK(ctx, "k_attn_tc");
    if (p.part) {
        k_attn_join<O><<<(unsigned)((p.a.nq * p.a.heads + 7) / 8), 256, 0, ctx->stream>>>(p, l.nsp);
        TB_LAUNCH_CHECK(ctx, "k_attn_join");
    }
    return TB_OK;
}

template <class T, class O>
tb_status launch_any(tb_ctx* ctx, const TcArgs& p, const Plan& l, const CUtensorMap& qm, const CUtensorMap& km,
                     const CUtensorMap& vm) {
    if (p.a.dim <= 64) return l.alt ? launch<T, O, 64, true>(ctx, p, l, qm, km, vm) : launch<T, O, 64, false>(ctx, p, l, qm, km, vm);
    return l.alt ? launch<T, O, 128, true>(ctx, p, l, qm, km, vm) : launch<T, O, 128, false>(ctx, p, l, qm, km, vm);
}

}  // namespace

size_t tb_attn_tc_workspace(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int heads, int kv_heads, int dim) {
    if (nq <= 0 || nk <= 0 || nset <= 0) return 0;
    const Plan l = attn_plan(ctx->num_sms, nq, nk, nset, kv_heads, heads / kv_heads);
    return (size_t)l.nsp * nq * heads * (dim + 1) * sizeof(float);
}

tb_status tb_attn_tc_launch(tb_ctx* ctx, const AttnArgs& args, tb_dtype dtype, tb_dtype out_dtype, void* workspace) {
    TcArgs p{};
    p.a = args;
    const AttnArgs& a = p.a;
    const Plan l = attn_plan(ctx->num_sms, a.nq, a.nk, a.nset, a.kv_heads, a.group);
    if (l.items > INT32_MAX || (l.nsp && (a.nq * a.heads + 7) / 8 > INT32_MAX))
        return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: too many rows times heads");
    p.a.unit = l.unit;
    p.tile_tokens = l.tile_tokens;
    p.nsplit = l.nsplit;
    if (l.nsp) {
        p.part = reinterpret_cast<float*>(workspace);
        p.part_lse = p.part + (size_t)l.nsp * a.nq * a.heads * a.dim;
    }
    const uint32_t fmt = dtype == TB_BF16 ? 1u : 0u;
    const uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
    p.idesc_s = base | (16u << 17);
    p.idesc_o = base | (1u << 16) | ((uint32_t)((a.dim + 15) / 16 * 2) << 17);        // B (V) with N contiguous
    p.q_bytes = (uint32_t)((a.dim <= 64 ? 1 : 2) * 128 * a.group * l.tile_tokens);
    CUtensorMap qm, km, vm;
    tb_status s = encode(ctx, &qm, dtype, a.q, a.dim, a.heads, a.q_head, a.nq, a.q_row, (uint32_t)a.group, (uint32_t)l.tile_tokens);
    if (s == TB_OK) s = encode(ctx, &km, dtype, a.k, a.dim, a.kv_heads, a.k_head, a.nk, a.k_row, 1, kKeys);
    if (s == TB_OK) s = encode(ctx, &vm, dtype, a.v, a.dim, a.kv_heads, a.v_head, a.nk, a.v_row, 1, kKeys);
    if (s != TB_OK) return s;
    if (dtype == TB_F16)
        return out_dtype == TB_F32 ? launch_any<__half, float>(ctx, p, l, qm, km, vm) : launch_any<__half, __half>(ctx, p, l, qm, km, vm);
    return out_dtype == TB_F32 ? launch_any<__nv_bfloat16, float>(ctx, p, l, qm, km, vm)
                               : launch_any<__nv_bfloat16, __nv_bfloat16>(ctx, p, l, qm, km, vm);
}
