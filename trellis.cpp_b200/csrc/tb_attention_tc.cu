// Attention within packed sets on tcgen05 (bf16 / f16 operands); the mathematics and the entry point
// are in tb_attention.cu.
//
// A CTA takes 128 query rows of one key head (a row is a token and one of the heads that share the key
// head, so a group reads its keys once) and walks the keys in blocks of 128: S = Q K^T into one of
// three 128-column TMEM buffers, softmax by a thread a row (no exchange), P over its S as the A operand
// of O += P V, which stays in TMEM. Two softmax warpgroups take every other block; with three buffers
// one block's S is ready and another's P V in work while they compute, so neither they nor the tensor
// pipe wait for the other's latencies. (Two tiles of rows a CTA with one buffer each, the other way
// to overlap them, left a chain S - softmax - P V of 3450 cycles for work of 2050 a pair of blocks.)
//
// Heads of more than 64 columns (PAIR): two CTAs of a cluster share each product as M = 256: each holds
// its own rows' Q, S, P and O, one half of each block's keys for S and one half of the head's columns
// of V for P V. Per CTA that halves the keys' way from L2 and the shared-memory reads, which a lone
// CTA's products would saturate.
//
// The rows' reference starts as the first block's maximum and moves only when a later block's exceeds it
// by more than 2^8: until then p grows to at most 2^8, which the 32-bit sums hold as well. It is that
// maximum itself, whose p is 1 and loses nothing where p is rounded to the operand type: a row that sees
// one key gives its value (with the next whole power of two, p came out up to half a step off).
// The warpgroups hand it on from block to block through shared memory; the one that raises it waits
// until the block before has been added and scales O.
//
// The launch has a CTA (pair) for each tile, but those that run take over tiles that have not started
// (clusterlaunchcontrol), so the next tile's loads and first products run while the last one's softmax
// and output finish (a CTA a tile paid some 4 us for them) and no SM idles while others have work
// left. One warp finds the tiles in the tables of sets.
//
// With few CTAs the keys are cut into `nsplit` ranges, which leave partial rows (32 bits, normalised,
// with their log sums) that are added up in a fixed order (k_attn_join in tb_attention.cu).
#include "tb_packed.cuh"
#include "tb_tc_ptx.cuh"

#include <algorithm>

#include "tb_attention.cuh"

namespace {

using namespace tbtc;
using namespace tbpk;

constexpr int kThreads = 384;
constexpr int kMma = 8, kTma = 9, kList = 10;      // warps 0-3 and 4-7 softmax, products (odd CTA of a pair: passes on), TMA, list
// Registers: 65536 / 384 threads allows 168 at launch; the third warpgroup gives up what the two
// softmax warpgroups need to hold a row of S. 2 * 216 + 72 = 3 * 168.
constexpr int kRegsSoftmax = 216, kRegsOther = 72;
constexpr int kKeys = 128;             // keys of a block
constexpr int kJobs = 2;               // tiles read ahead of the one in work, and it
constexpr int kBufs = 3;               // S buffers
constexpr float kRaise = 8.f;          // the reference follows when a block's maximum is 2^8 above it
// Blocks of one accumulation in TMEM (32768 keys). The tensor core cuts what it adds to O below O's last
// place instead of rounding it, so long sums come out short, by a share that grows with their length: at
// 2^18, 2^20 and 2^22 keys of equal weight -0.14, -0.65 and -2.7% in f16 (-0.02, -0.45 and -2.5% in
// bf16). A longer range is taken in segments, whose O the softmax threads add up in 32 bits.
constexpr int kChain = 256;
struct TcArgs {
    AttnArgs a;
    int tile_tokens;                   // tokens of a 128-row tile
    int wide;                          // output rows (or partial rows) start at multiples of 32 bytes
    uint32_t idesc_s, idesc_o, q_bytes;   // q_bytes: what one tile's boxes deliver
};

template <int D, bool PAIR> struct Geom {
    static constexpr int kBoxes = D / 64;
    static constexpr int kQBytes = kBoxes * 16384;                // 128 rows x D, boxes of 64 columns
    static constexpr int kBytes = kBoxes * 16384 / (PAIR ? 2 : 1);   // a CTA's share of a block's K, of its V
    static constexpr int kStages = 196608 / (2 * kBytes);         // of a K and a V each
    static constexpr int kBars = (2 * kStages + 2 + 3 * kBufs + 2 + 8 + 4 + 2 * kJobs + 1 + 9 + 1) / 2 * 2;
    static constexpr size_t kUsed = (size_t)kQBytes + 2 * kStages * kBytes + 2048 + 8 * kBars + kJobs * 48 + 48;
    static constexpr size_t kSlack = 448;                         // for a base that is no multiple of 1024
    static constexpr size_t kSmem = kUsed + kSlack;
};

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

// The maximum that keeps a value that is no number: it then makes its whole row none.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float max2(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// p = 2^(s c + ref) of a row's 128 scores, rounded to T into the TMEM columns from `ts`; returns the sum of
// the unrounded ones. T, since the tensor core takes P in V's type: a second product with what the rounding
// leaves would double P V, and the rounded result is as far off by itself (bf16 1.7e-3 against 64 bits, with
// this 2.1 to 2.3e-3); 32-bit operands have a kernel without it. The exponentials take 1024 cycles of their
// unit a block, as long as the products of a wide block, but neither sets the pace (59 and 58% busy at 128
// columns, 52 and 25% at 64): a turn of a softmax warpgroup does, some 3400 cycles with two under way.
// (A share of the exponentials by a cubic on the FMA pipes, 1 or 2 of 8: 1507 -> 1559 and 1659 us at 16384 x
// 12 x 128; not measured at 64 columns.)
template <class T> __device__ __forceinline__ float exp_block(const float* s, float c, float ref, uint32_t ts) {
    const f2 c2 = pack(c, c), ref2 = pack(ref, ref);
    f2 sum[2];
#pragma unroll
    for (int quarter = 0; quarter < 4; ++quarter) {
        const float* v = s + quarter * 32;
        uint32_t w[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            float2 y = unpack(fma2(pack(v[2 * q], v[2 * q + 1]), c2, ref2));
            y.x = ex2(y.x);
            y.y = ex2(y.y);
            w[q] = pack2(y.x, y.y, T());
            sum[q & 1] = quarter || q >= 2 ? add2(sum[q & 1], pack(y.x, y.y)) : pack(y.x, y.y);
        }
        tmem_st_x16(ts + quarter * 16, w);
    }
    const float2 all = unpack(add2(sum[0], sum[1]));
    return all.x + all.y;
}

// Hand-offs inside a CTA, or across the pair: those order tcgen05 operations only (see tb_tc_ptx.cuh).
template <bool PAIR> __device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t par, volatile int* ab, int* err) {
    return PAIR ? mbar_wait_cluster_relaxed(bar, par, ab, err) : mbar_wait(bar, par, ab, err);
}
template <bool PAIR> __device__ __forceinline__ void commit(uint32_t bar) {
    if (PAIR) tc_commit_pair(bar, 0x3);
    else tc_commit(bar);
}

// A place in a ring of N and the parity of its round.
template <int N> struct Ring {
    uint32_t at = 0, round = 0;
    __device__ __forceinline__ void step() {
        if (++at == N) {
            at = 0;
            round ^= 1;
        }
    }
};

// A job of the list: a tile (query rows of a set, a key head, a range of its key blocks) or a segment of
// one. 12 words.
struct Job {
    int q0, nq, k0, nk;    // the set's rows
    int first;             // the tile's first token, in the set
    int blk0, n;           // key blocks
    int kvh, split, end;   // end: the list is done
    int seg;               // of a tile in segments: bit 0 some came before, bit 1 some follow
    int pad;
};

// 32 values of a row at p, as far as `left` says (a multiple of 8). Lanes are rows, so each store is a
// sector or two of its own: 32 bytes at once where the rows allow it.
template <class O> __device__ __forceinline__ void store_row(O* p, const float* v, int left, bool wide) {
    constexpr int n = 32 / (int)sizeof(O);               // values of 32 bytes
    if (wide && left >= 32) {
#pragma unroll
        for (int e = 0; e < 32; e += n) {
            uint32_t w[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if (sizeof(O) == 4) {
                    w[q] = __float_as_uint(v[e + q]);
                } else {
                    using H = typename std::conditional<sizeof(O) == 4, __half, O>::type;
                    w[q] = pack2(v[(e + 2 * q) % 32], v[(e + 2 * q + 1) % 32], H());
                }
            }
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                         :: "l"(p + e), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        }
    } else {
#pragma unroll
        for (int e = 0; e < 32; e += 8)
            if (e < left) store8<O>(p + e, v + e);
    }
}

template <class T, class O, int D, bool PAIR>
__device__ __forceinline__ void attn_tc(const CUtensorMap& qmap, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                        const TcArgs& p) {
    using G = Geom<D, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_align1024(smem_raw);
    uint8_t* ring = smem + G::kQBytes;
    float* s_ref = reinterpret_cast<float*>(ring + 2 * G::kStages * G::kBytes);   // [2][128] the rows' reference, by tile
    float* s_sum = s_ref + 256;                                                   // [2][128] the warpgroups' sums
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_sum + 256);
    Job* s_job = reinterpret_cast<Job*>(bars + G::kBars);
    uint32_t* s_take = reinterpret_cast<uint32_t*>(s_job + kJobs);                // [4] the tile taken over, as answered
    uint32_t* s_next = s_take + 4;                                                // [4] its number, for the odd CTA
    uint32_t* s_misc = s_next + 4;                                                // [0] tmem, [1] abort
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_misc + 1);
    const uint32_t b0 = smem_u32(bars);
    auto full = [&](uint32_t s) { return b0 + 8u * s; };
    auto empty = [&](uint32_t s) { return b0 + 8u * (G::kStages + s); };
    const uint32_t bq = b0 + 8u * (2 * G::kStages), qempty = bq + 8u;
    auto sfull = [&](uint32_t s) { return bq + 8u * (2 + s); };
    auto pfull = [&](uint32_t s) { return bq + 8u * (2 + kBufs + s); };
    auto pvdone = [&](uint32_t s) { return bq + 8u * (2 + 2 * kBufs + s); };
    const uint32_t ofull = bq + 8u * (2 + 3 * kBufs), oempty = ofull + 8u;
    auto handed = [&](int wg, int q) { return ofull + 8u * (2 + 4 * wg + q); };   // the reference, to a warp
    auto sums = [&](int q) { return ofull + 8u * (10 + q); };
    auto jfull = [&](uint32_t s) { return ofull + 8u * (14 + s); };
    auto jempty = [&](uint32_t s) { return ofull + 8u * (14 + kJobs + s); };
    const uint32_t drain = ofull + 8u * (14 + 2 * kJobs), taken = drain + 8u;
    auto told = [&](uint32_t s) { return taken + 8u * (1 + s); };
    auto heard = [&](uint32_t s) { return taken + 8u * (5 + s); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AttnArgs& a = p.a;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    if ((size_t)(smem - smem_raw) > G::kSlack) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, TB_DEVERR_SMEM_BASE);
        return;                            // both CTAs of a pair
    }

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < G::kStages; ++s) {
            mbar_init(full(s), PAIR && leader ? 2 : 1);         // its own TMA and the odd CTA's, passed on
            mbar_init(empty(s), 1);
        }
        mbar_init(bq, 1);
        mbar_init(qempty, 1);
        for (uint32_t s = 0; s < kBufs; ++s) {
            mbar_init(sfull(s), 1);
            mbar_init(pfull(s), PAIR ? 8 : 4);                  // the warps of both CTAs, at the even one
            mbar_init(pvdone(s), 1);
        }
        mbar_init(ofull, 1);
        mbar_init(oempty, PAIR ? 16 : 8);
        for (int q = 0; q < 4; ++q) {
            mbar_init(handed(0, q), 1);
            mbar_init(handed(1, q), 1);
            mbar_init(sums(q), 2);
        }
        for (uint32_t s = 0; s < kJobs; ++s) {
            mbar_init(jfull(s), 1);
            mbar_init(jempty(s), 10);                           // softmax warps, products, TMA
        }
        mbar_init(drain, 1);
        mbar_init(taken, 1);
        for (uint32_t s = 0; s < 4; ++s) {
            mbar_init(told(s), 1);
            mbar_init(heard(s), 1);
        }
        s_misc[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMma) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                         :: "r"(smem_u32(s_misc)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                         :: "r"(smem_u32(s_misc)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
    }
    __syncthreads();
    if (PAIR) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = s_misc[0], tmem_o = tmem + kBufs * 128u;
    const uint32_t sq = smem_u32(smem), skv = sq + G::kQBytes;

    Ring<kJobs> jr;
    // The next tile of the list, in place until it is released; null at the list's end.
    auto next_job = [&]() -> const Job* {
        if (!__all_sync(0xffffffffu, mbar_wait(jfull(jr.at), jr.round, s_abort, a.err))) return nullptr;
        const Job* j = s_job + jr.at;
        return j->end ? nullptr : j;
    };
    auto release_job = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(jempty(jr.at));
        jr.step();
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsOther));
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t par) {
            if (ok) ok = __all_sync(0xffffffffu, wait_bar<PAIR>(bar, par, s_abort, a.err));
            return ok;
        };
        auto wait_own = [&](uint32_t bar, uint32_t par) {        // a barrier that this CTA alone takes part in
            ok = __all_sync(0xffffffffu, mbar_wait(bar, par, s_abort, a.err));
            return ok;
        };
        // The rows of V behind the set's last key belong to others and may hold no numbers, which a p
        // of 0 would not cancel: those of the last 16 that the products read become 0.
        auto clean = [&](uint32_t st, int keys) {
            constexpr int per = G::kBytes / kKeys / 16;         // 16-byte words of a key's row
            uint8_t* v = ring + st * (2 * G::kBytes) + G::kBytes;
            for (int w = lane; w < (16 - (keys & 15)) * per; w += 32) {
                const int row = keys + w / per, x = w % per;
                *reinterpret_cast<uint4*>(v + (x >> 3) * 16384 + row * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        // A tile's items of the ring: item j holds the K of its block j and the V of block j - lag, what the
        // products of one round read. One barrier to wait for, one to free.
        Job j;
        if (warp == kList) {
            // -------------------------------------------------------------- the list
            // Tiles in the order set, piece of the set (causal: the last ones, which see the most keys, come
            // first), key head, range of keys; taken over in whatever order they are given.
            SetWalk walk;
            uint32_t number = PAIR ? cluster_id_x() : blockIdx.x, jobs = 0;
            for (uint32_t k = 0;; ++k) {
                const bool over = number == 0xffffffffu;         // none left to take over
                uint32_t idx = over ? 0 : number;
                const int split = idx % a.nsplit;
                idx /= a.nsplit;
                const int kvh = idx % a.kv_heads;
                SetWalk::Piece at{};                             // the launch has some more tiles than there are
                if (over || walk.find(a.q_off, a.k_off, a.nset, a.nq, a.nk, a.unit, idx / a.kv_heads, lane, a.err, at)) {
                    Job o;
                    o.q0 = at.q0;
                    o.nq = at.nq;
                    o.k0 = at.k0;
                    o.nk = at.nk;
                    o.first = (int)(a.causal ? at.of - 1 - at.at : at.at) * a.unit;
                    const int end = a.causal ? max(0, min(o.nk, min(o.first + a.unit, o.nq) + o.nk - o.nq)) : o.nk;
                    const int all = (end + kKeys - 1) / kKeys;
                    o.blk0 = (int)((int64_t)all * split / a.nsplit);
                    const int stop = over ? o.blk0 : (int)((int64_t)all * (split + 1) / a.nsplit);
                    o.kvh = kvh;
                    o.split = split;
                    o.end = over ? 1 : 0;
                    o.seg = 0;
                    // The wait for a place takes a job's time at most: a segment's, not a tile's of any length.
                    do {
                        o.n = min(stop - o.blk0, kChain);
                        o.seg = (o.seg & 1) | (o.blk0 + o.n < stop ? 2 : 0);
                        if (jobs >= kJobs && !wait_own(jempty(jr.at), jr.round ^ 1)) break;
                        if (lane == 0) {
                            int4* dst = reinterpret_cast<int4*>(s_job + jr.at);
                            dst[0] = make_int4(o.q0, o.nq, o.k0, o.nk);
                            dst[1] = make_int4(o.first, o.blk0, o.n, o.kvh);
                            dst[2] = make_int4(o.split, o.end, o.seg, 0);
                            mbar_arrive(jfull(jr.at));
                        }
                        __syncwarp();
                        jr.step();
                        ++jobs;
                        o.blk0 += o.n;
                        o.seg |= 1;
                    } while (o.blk0 < stop);
                }
                if (over || !ok) break;
                if (leader) {
                    if (elect_one()) {
                        mbar_arrive_expect_tx(taken, 16);
                        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                                     :: "r"(smem_u32(s_take)), "r"(taken) : "memory");
                    }
                    __syncwarp();
                    if (!__all_sync(0xffffffffu, mbar_wait(taken, k & 1, s_abort, a.err))) break;
                    uint32_t x, got;
                    asm volatile("{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t"
                                 "ld.shared.b128 h, [%2];\n\t"
                                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
                                 "selp.u32 %1, 1, 0, p;\n\tmov.u32 %0, 0;\n\t"
                                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
                                 : "=r"(x), "=r"(got) : "r"(smem_u32(s_take)) : "memory");
                    number = got ? (PAIR ? x / 2 : x) : 0xffffffffu;
                    fence_proxy_async_smem();                    // read before the next answer is written
                    __syncwarp();
                    // one of four places for the odd CTA, once it has read what was there
                    if (PAIR && k >= 4 && !__all_sync(0xffffffffu, mbar_wait_cluster(heard(k & 3), ((k >> 2) - 1) & 1, s_abort, a.err)))
                        break;
                    if (PAIR && lane == 0) {
                        asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, 1;\n\t"
                                     "st.shared::cluster.u32 [ra], %1;\n\t}"
                                     :: "r"(smem_u32(s_next + (k & 3))), "r"(number) : "memory");
                        mbar_arrive_cluster(told(k & 3), 1);
                    }
                } else {
                    if (!__all_sync(0xffffffffu, mbar_wait_cluster(told(k & 3), k >> 2 & 1, s_abort, a.err))) break;
                    number = *reinterpret_cast<volatile uint32_t*>(s_next + (k & 3));
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(heard(k & 3), 0);
                }
            }
        } else if (warp == kTma) {
            // -------------------------------------------------------------- TMA producer
            Ring<G::kStages> r;
            uint32_t used = 0, tiles = 0;
            while (const Job* from = next_job()) {
                j = *from;
                release_job();
                if (j.n == 0) continue;
                const int lag = min(j.n, kBufs), items = j.n + lag;
                if (tiles && !wait(qempty, (tiles - 1) & 1)) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(bq, p.q_bytes);
                    for (int b = 0; b < G::kBoxes; ++b)
                        tma_load_3d(sq + b * 16384, &qmap, b * 64, j.kvh * a.group, j.q0 + j.first + (int)rank * p.tile_tokens, bq);
                }
                __syncwarp();
                for (int i = 0; i < items; ++i, r.step(), ++used) {
                    if (used >= G::kStages && !wait(empty(r.at), r.round ^ 1)) break;
                    if (elect_one()) {
                        const uint32_t k_at = skv + r.at * (2 * G::kBytes), v_at = k_at + G::kBytes;
                        mbar_arrive_expect_tx(full(r.at), i < j.n && i >= lag ? 2 * G::kBytes : G::kBytes);
                        const int key = j.k0 + (j.blk0 + i) * kKeys;
                        if (i < j.n)
                            for (int x = 0; x < G::kBoxes; ++x)
                                tma_load_3d(k_at + x * (PAIR ? 8192 : 16384), &kmap, x * 64, j.kvh,
                                            key + (PAIR ? (int)rank * 64 : 0), full(r.at));
                        if (i >= lag)
                            for (int x = 0; x < (PAIR ? 1 : G::kBoxes); ++x)
                                tma_load_3d(v_at + x * 16384, &vmap, (PAIR ? (int)rank : x) * 64, j.kvh, key - lag * kKeys, full(r.at));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                ++tiles;
            }
        } else if (warp == kMma && leader) {
            // -------------------------------------------------------------- the products
            // One warp issues both: a block's P V and, into the buffer that it frees, the S three blocks on.
            // MMAs of one thread run in order, so nothing is waited for between the two. Its instructions
            // are the pace where the softmax keeps up: a wait costs some 150 cycles even when its phase is
            // over, an MMA issued by a thread on its own 100 instead of 40. Descriptors differ by
            // constants: low word (address >> 4) | leading offset << 16, high word 8-row groups 1024 bytes
            // apart in the 128-byte swizzle. Q and K have their K dimension (the head's columns)
            // contiguous; V is the B operand with N (the head's columns) contiguous, boxes of 64 columns
            // 16384 bytes apart.
            constexpr uint32_t kHi = 64u | (1u << 14) | (2u << 29);
            const uint32_t qlo = (sq >> 4) | (1u << 16), klo = (skv >> 4) | (1u << 16);
            const uint32_t vlo = ((skv + G::kBytes) >> 4) | (1024u << 16);
            const int dim = a.dim;
            Ring<G::kStages> r;
            Ring<kBufs> u, us;                       // P V's and S's buffers
            uint32_t tiles = 0;
            auto mma_s = [&](bool last) {            // by the elected thread
                const uint32_t kl = klo + r.at * (2 * G::kBytes >> 4), td = tmem + us.at * 128;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint64_t qd = (uint64_t)kHi << 32 | (qlo + (k >> 2) * 1024 + (k & 3) * 2);
                    const uint64_t kd = (uint64_t)kHi << 32 | (kl + (k >> 2) * (PAIR ? 512 : 1024) + (k & 3) * 2);
                    if (k * 16 < dim) {
                        if (PAIR) tc_mma_ss_pair(td, qd, kd, p.idesc_s, k ? 1u : 0u);
                        else tc_mma(td, qd, kd, p.idesc_s, k ? 1u : 0u);
                    }
                }
                commit<PAIR>(sfull(us.at));
                if (last) commit<PAIR>(qempty);
            };
            while (const Job* from = ok ? next_job() : nullptr) {
                const int n = from->n;
                int keys = from->nk - from->blk0 * kKeys;
                release_job();
                if (n == 0) continue;
                const int lag = min(n, kBufs);
                ok = __all_sync(0xffffffffu, mbar_wait(bq, tiles & 1, s_abort, a.err));
                for (int b = 0; b < lag && ok; ++b, r.step(), us.step()) {
                    if (!wait(full(r.at), r.round)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_s(b == n - 1);
                        commit<PAIR>(empty(r.at));
                    }
                    __syncwarp();
                }
                for (int b = 0; b < n && ok; ++b, r.step(), u.step(), keys -= kKeys) {
                    if (!wait(full(r.at), r.round)) break;
                    if (keys < kKeys && (keys & 15)) clean(r.at, keys);
                    // the last tile's O has been read
                    if (b == 0 && tiles && !wait(oempty, (tiles - 1) & 1)) break;
                    if (!wait(pfull(u.at), u.round)) break;
                    tc_fence_after();
                    const bool more = b + lag < n;
                    if (elect_one()) {
                        const uint32_t vl = vlo + r.at * (2 * G::kBytes >> 4), pa = tmem + u.at * 128;
#pragma unroll
                        for (int k = 0; k < kKeys / 16; ++k) {
                            const uint64_t vd = (uint64_t)kHi << 32 | (vl + k * 128);
                            if (k * 16 < keys) {
                                if (PAIR) tc_mma_ts_pair(tmem_o, pa + k * 8, vd, p.idesc_o, b || k ? 1u : 0u);
                                else tc_mma_ts(tmem_o, pa + k * 8, vd, p.idesc_o, b || k ? 1u : 0u);
                            }
                        }
                        commit<PAIR>(pvdone(u.at));
                        if (more) mma_s(b + lag == n - 1);
                        commit<PAIR>(empty(r.at));
                        if (b == n - 1) commit<PAIR>(ofull);
                    }
                    __syncwarp();
                    if (more) us.step();
                }
                ++tiles;
            }
            // every MMA has completed before the TMEM is freed (also after an abort)
            if (elect_one()) PAIR ? tc_commit_pair(drain, 0x1) : tc_commit(drain);
            __syncwarp();
        } else if (PAIR && !leader && warp == kMma) {
            // -------------------------------------------------------------- odd CTA: what has landed, passed on
            Ring<G::kStages> r;
            uint32_t tiles = 0;
            while (const Job* from = ok ? next_job() : nullptr) {
                j = *from;
                release_job();
                if (j.n == 0) continue;
                const int lag = min(j.n, kBufs), items = j.n + lag, tail = j.nk - (j.blk0 + j.n - 1) * kKeys;
                ok = __all_sync(0xffffffffu, mbar_wait(bq, tiles & 1, s_abort, a.err));
                for (int i = 0; i < items && ok; ++i, r.step()) {
                    ok = __all_sync(0xffffffffu, mbar_wait(full(r.at), r.round, s_abort, a.err));
                    if (!ok) break;
                    const bool dirty = i == items - 1 && tail < kKeys && (tail & 15);
                    if (dirty) clean(r.at, tail);
                    if (lane == 0) {
                        if (dirty) mbar_arrive_cluster(full(r.at), 0);          // its zeros before the products
                        else mbar_arrive_cluster_relaxed(full(r.at), 0);
                    }
                }
                ++tiles;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kRegsSoftmax));
        // ------------------------------------------------------------------ softmax and output
        // The warpgroups take turns over the blocks of all tiles.
        const int wg = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quad * 32) << 16, to = tmem_o + lane_base;
        const int rt = r / a.group;           // the row's token in a tile
        const float c = a.scale_log2;
        // p in f16 starts at 2^7 instead of 1 (2^15 after the largest rise): small p keep their digits
        constexpr float lift = std::is_same<T, __half>::value ? 7.f : 0.f;
        Ring<kBufs> u;
        // A tile in segments: the thread's columns of O and the row's sum so far, against the reference in
        // keep[W]. Indexed from a number that the compiler does not know, so that it lies in local memory and
        // takes no registers from the softmax.
        constexpr int W = D / 2;                     // each warpgroup writes half of the head's columns
        float keep[W + 2];
        int zero = 0;
        asm volatile("" : "+r"(zero));
        uint32_t tiles = 0, blocks = 0, turns = 0;   // jobs with keys, blocks of all jobs, hand-offs received
        bool ok = true;
        while (const Job* job = ok ? next_job() : nullptr) {
            const int n = job->n, seg = job->seg;
            // the keys from the tile's first block on that the row sees; rows past the set see all
            auto rows = [&](int& t, int& h) {
                t = job->first + (int)rank * p.tile_tokens + rt;
                h = job->kvh * a.group + r - rt * a.group;
                return rt < p.tile_tokens && t < job->nq;
            };
            int lim, wlim;
            {
                int t, h;
                const int nk = job->nk;
                lim = !rows(t, h) ? nk : a.causal ? max(0, min(nk, t + 1 + nk - job->nq)) : nk;
                lim -= job->blk0 * kKeys;
                wlim = __reduce_min_sync(0xffffffffu, lim);
            }
            float* refs = s_ref + (tiles & 1) * 128;
            float ref = -INFINITY, l = 0.f;          // of the warpgroup's own blocks; -inf: no key so far
            float shift = lift;                      // what scores are shifted by: lift - ref
            for (int b = 0; b < n; ++b, ++blocks, u.step()) {
                if ((int)(blocks & 1) != wg) continue;
                const uint32_t ts = tmem + u.at * 128u + lane_base;
                if (!__all_sync(0xffffffffu, wait_bar<PAIR>(sfull(u.at), u.round, s_abort, a.err))) { ok = false; break; }
                tc_fence_after();
                float s[kKeys];
#pragma unroll
                for (int q = 0; q < kKeys; q += 32) tmem_ld_x32(ts + q, s + q);
                // meanwhile: the reference after the block before, from the other warpgroup
                float now = -INFINITY;
                if (blocks > 0) {
                    if (!__all_sync(0xffffffffu, mbar_wait(handed(wg, quad), turns & 1, s_abort, a.err))) { ok = false; break; }
                    ++turns;
                    if (b > 0) now = refs[r];
                }
                tmem_wait_ld();
                const bool masked = wlim < (b + 1) * kKeys;
                if (masked) {
                    const int left = lim - b * kKeys, least = wlim - b * kKeys;
#pragma unroll
                    for (int e = 0; e < kKeys; e += 32) {
                        if (least >= e + 32) continue;   // all of it
#pragma unroll
                        for (int q = e; q < e + 32; ++q) s[q] = q < left ? s[q] : -INFINITY;
                    }
                }
                float mx[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = max3(s[e], s[e + 4], s[e + 8]);
#pragma unroll
                for (int q = 12; q < kKeys - 4; q += 8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[q + e], s[q + 4 + e]);
                }
                const float top = max3(max3(mx[0], mx[1], s[kKeys - 4]), max3(mx[2], mx[3], s[kKeys - 3]),
                                       max2(s[kKeys - 2], s[kKeys - 1])) * c;
                const bool raise = !(top - now <= kRaise) && !(top == -INFINITY && now == -INFINITY);
                if (b == 0 || __any_sync(0xffffffffu, raise || now != ref)) {
                    const float next = raise ? top : now;
                    refs[r] = next;
                    if (b > 0 && __any_sync(0xffffffffu, raise)) {
                        // O is at rest once the block before has been added
                        const uint32_t before = u.at ? u.at - 1 : kBufs - 1, par = u.at ? u.round : u.round ^ 1;
                        if (!__all_sync(0xffffffffu, wait_bar<PAIR>(pvdone(before), par, s_abort, a.err))) { ok = false; break; }
                        tc_fence_after();
                        const float al = raise ? ex2(now - next) : 1.f;
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
                    __syncwarp();                    // the references before the hand-off
                    l = next == ref ? l : l * ex2(ref - next);
                    ref = next;
                    shift = lift - (ref == -INFINITY ? 0.f : ref);
                }
                if (lane == 0) mbar_arrive(handed(1 - wg, quad));
                __syncwarp();                        // the hand-off first: the exponentials are not moved ahead of it
                l += exp_block<T>(s, c, shift, ts);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster_relaxed(pfull(u.at), 0);
                    else mbar_arrive(pfull(u.at));
                }
            }
            float total = 0.f;
            if (n > 0 && ok) {
                ok = __all_sync(0xffffffffu, wait_bar<PAIR>(ofull, tiles & 1, s_abort, a.err));
                tc_fence_after();
                // both warpgroups' sums against the last reference
                const float last = refs[r];
                s_sum[wg * 128 + r] = ref == last ? l : ref == -INFINITY ? 0.f : l * ex2(ref - last);
                ref = last;
                __syncwarp();
                if (lane == 0) mbar_arrive(sums(quad));
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(sums(quad), tiles & 1, s_abort, a.err));
                total = s_sum[r] + s_sum[128 + r];
            }
            if (!ok) break;
            auto o_read = [&]() {                    // O may be written again
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster_relaxed(oempty, 0);
                    else mbar_arrive(oempty);
                }
            };
            if (__builtin_expect(seg, 0)) {
                // O and what the thread has of the segments before: to be kept, after the last one back into TMEM
                const float had = seg & 1 ? keep[zero + W] : -INFINITY, top = fmaxf(had, ref);
                const float mine = ref == -INFINITY ? 0.f : ex2(ref - top), before = had == -INFINITY ? 0.f : ex2(had - top);
                total = fmaf(total, mine, seg & 1 ? keep[zero + W + 1] * before : 0.f);
                ref = top;
                keep[zero + W] = ref;
                keep[zero + W + 1] = total;
#pragma unroll 1
                for (int w = 0; w < W; w += 32) {
                    float o[32];
                    __syncwarp();
                    tmem_ld_x32(to + wg * W + w, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        o[e] = fmaf(o[e], mine, seg & 1 ? keep[zero + w + e] * before : 0.f);
                        keep[zero + w + e] = o[e];
                    }
                    if (!(seg & 2)) tmem_st_x32(to + wg * W + w, reinterpret_cast<const uint32_t*>(o));
                }
                tmem_wait_st();
                if (seg & 2) {
                    o_read();
                    ++tiles;
                    release_job();
                    continue;
                }
            }
            int t, h;
            const bool valid = rows(t, h), none = total == 0.f;            // the row sees no key here, or none above -inf
            const float inv = none ? 0.f : 1.f / total;
            const int64_t row = (int64_t)job->q0 + t;
            const int64_t at = ((int64_t)job->split * a.nq + row) * a.heads + h;
            if (valid && wg == 0 && (a.part || a.lse)) {
                const float lg = none ? -INFINITY : ref - lift + log2f(total);
                if (a.part) a.part_lse[at] = lg;
                else a.lse[row * a.heads + h] = lg * 0.69314718055994530942f;
            }
            float* part = a.part + at * a.dim;
            O* out = reinterpret_cast<O*>(a.out) + row * a.out_row + (int64_t)h * a.out_head;
#pragma unroll 1
            for (int w = 0; w < W; w += 32) {
                const int q = wg * W + w;
                float o[32];
                __syncwarp();
                if (n > 0) {
                    tmem_ld_x32(to + q, o);
                    tmem_wait_ld();
                    if (w + 32 >= W) o_read();
                }
                if (!valid || (a.part && none)) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = none ? 0.f : o[e] * inv;
                if (a.part) store_row<float>(part + q, o, a.dim - q, p.wide);
                else store_row<O>(out + q, o, a.dim - q, p.wide);
            }
            if (n > 0) ++tiles;
            release_job();
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMma && leader) {
        const long long w0 = clock64();
        while (!mbar_try_wait(drain, 0) && clock64() - w0 < kWaitCycles) { }
    }
    if (*s_abort && threadIdx.x == 0) {
        // after an abort: wait out the loads that may still be in flight
        const long long w0 = clock64();
        while (clock64() - w0 < 20000000) { }
    }
    __syncthreads();
    if (PAIR) cluster_sync_all();
    if (warp == kMma) {
        tc_fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

template <class T, class O, int D>
__global__ void __launch_bounds__(kThreads, 1)
k_attn_tc(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
          const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcArgs p) {
    attn_tc<T, O, D, false>(qmap, kmap, vmap, p);
}
template <class T, class O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_attn_pair(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
            const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcArgs p) {
    attn_tc<T, O, 128, true>(qmap, kmap, vmap, p);
}

struct Plan {
    bool pair;
    int tile_tokens, unit, nsplit;
    int64_t items;                     // tiles, at most
};

// Pairs for wide heads where an average set's rows fill more than one CTA (16384 rows, 12 heads of 128:
// 1.53 ms, a CTA a tile 1.59; eight causal sets of 1 to 4096 rows, 16/4 heads: 183 us and 202; where rows
// fill one CTA at most a pair's other half is idle: 62 us and 118 for 16 single rows). Keys are cut
// where the CTAs would not fill the SMs, into ranges of four blocks at least in a set of the average
// length, of eight if all keys are one set's (100 rows, 12 heads, 20000 keys: 32 us, whole 129; 300 rows, 8
// heads, 2048 keys: 14 and 16; 100 rows against 8000 keys beside three sets of 3, 4 heads: 20 and 37; two
// sets of 40 rows, 16 heads, 8192 keys: 38, 34 with ranges twice as long, whole 60).
Plan attn_plan(int num_sms, int64_t nq, int64_t nk, int nset, int kv_heads, int group, int dim) {
    Plan l;
    l.tile_tokens = 128 / group;
    l.pair = dim > 64 && (nq + nset - 1) / nset > l.tile_tokens;
    l.unit = l.pair ? 2 * l.tile_tokens : l.tile_tokens;
    const int64_t pieces = (nq + l.unit - 1) / l.unit;
    const int64_t ctas = std::max<int64_t>(pieces, std::min<int64_t>(nset, nq)) * kv_heads * (l.pair ? 2 : 1);
    const int64_t blocks = std::max((nk / nset + kKeys - 1) / kKeys / 4, nk / kKeys / 8);
    l.nsplit = 1;
    if (ctas < num_sms) l.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({4ll * num_sms / ctas, blocks, 32}));
    l.items = (pieces + nset) * kv_heads * l.nsplit;
    return l;
}

template <class T, class O>
tb_status launch(tb_ctx* ctx, const TcArgs& p, const Plan& l, const CUtensorMap& qm, const CUtensorMap& km,
                 const CUtensorMap& vm) {
    const bool wide = p.a.dim > 64;
    const size_t sm = l.pair ? Geom<128, true>::kSmem : wide ? Geom<128, false>::kSmem : Geom<64, false>::kSmem;
    const void* kernel = l.pair ? (const void*)k_attn_pair<T, O>
                                : wide ? (const void*)k_attn_tc<T, O, 128> : (const void*)k_attn_tc<T, O, 64>;
    if (sm > (size_t)ctx->max_smem_optin) return tb_fail(ctx, TB_ERR_UNSUPPORTED, "tb_attention: shared memory too small");
    TB_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
    const unsigned grid = (unsigned)(l.pair ? 2 * l.items : l.items);
    if (l.pair) k_attn_pair<T, O><<<grid, kThreads, sm, ctx->stream>>>(qm, km, vm, p);
    else if (wide) k_attn_tc<T, O, 128><<<grid, kThreads, sm, ctx->stream>>>(qm, km, vm, p);
    else k_attn_tc<T, O, 64><<<grid, kThreads, sm, ctx->stream>>>(qm, km, vm, p);
    TB_LAUNCH_CHECK(ctx, "k_attn_tc");
    return TB_OK;
}

}  // namespace

tb_status tb_attn_encode(tb_ctx* ctx, CUtensorMap* map, tb_dtype dtype, const void* base, int dim, int64_t heads, int64_t head,
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

int tb_attn_tc_nsplit(const tb_ctx* ctx, int64_t nq, int64_t nk, int nset, int heads, int kv_heads, int dim) {
    return attn_plan(ctx->num_sms, nq, nk, nset, kv_heads, heads / kv_heads, dim).nsplit;
}

tb_status tb_attn_tc_launch(tb_ctx* ctx, const AttnArgs& args, tb_dtype dtype, tb_dtype out_dtype) {
    TcArgs p{};
    p.a = args;
    const AttnArgs& a = p.a;
    const Plan l = attn_plan(ctx->num_sms, a.nq, a.nk, a.nset, a.kv_heads, a.group, a.dim);
    if (2 * l.items > INT32_MAX) return tb_fail(ctx, TB_ERR_TOO_LARGE, "tb_attention: too many rows times heads");
    p.a.unit = l.unit;
    p.tile_tokens = l.tile_tokens;
    {
        const int64_t size = (int64_t)tb_dtype_size(out_dtype);
        const bool rows = (reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_row * size) | (uintptr_t)(a.out_head * size)) % 32 == 0;
        p.wide = a.part ? reinterpret_cast<uintptr_t>(a.part) % 32 == 0 : rows;
    }
    const uint32_t fmt = dtype == TB_BF16 ? 1u : 0u;
    const uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((l.pair ? 16u : 8u) << 24);
    p.idesc_s = base | (16u << 17);
    // B (V) with N contiguous; a pair's halves are 64 columns each, behind the head's last one zeros
    p.idesc_o = base | (1u << 16) | ((l.pair ? 16u : (uint32_t)((a.dim + 15) / 16 * 2)) << 17);
    p.q_bytes = (uint32_t)((a.dim <= 64 ? 1 : 2) * 128 * a.group * l.tile_tokens);
    CUtensorMap qm, km, vm;
    tb_status s = tb_attn_encode(ctx, &qm, dtype, a.q, a.dim, a.heads, a.q_head, a.nq, a.q_row, (uint32_t)a.group, (uint32_t)l.tile_tokens);
    if (s == TB_OK) s = tb_attn_encode(ctx, &km, dtype, a.k, a.dim, a.kv_heads, a.k_head, a.nk, a.k_row, 1, l.pair ? 64 : kKeys);
    if (s == TB_OK) s = tb_attn_encode(ctx, &vm, dtype, a.v, a.dim, a.kv_heads, a.v_head, a.nk, a.v_row, 1, kKeys);
    if (s != TB_OK) return s;
    if (dtype == TB_F16)
        return out_dtype == TB_F32 ? launch<__half, float>(ctx, p, l, qm, km, vm) : launch<__half, __half>(ctx, p, l, qm, km, vm);
    return out_dtype == TB_F32 ? launch<__nv_bfloat16, float>(ctx, p, l, qm, km, vm)
                               : launch<__nv_bfloat16, __nv_bfloat16>(ctx, p, l, qm, km, vm);
}
