// g4_tree_attention.cu -- attention of a tree of drafted tokens over each sequence's cached
// keys and the node's own ancestors.
//
// Row (s, i) of q sits at position base + depth(i) and sees the cached keys j < base (of the
// last `window` positions when sliding) and the drafted rows of its ancestors and itself.
//
// Every row of a sequence reads the same K/V, so the sequence's nodes x heads query rows are
// the M side of two tensor-core products per tile of 128 keys, S = Q K^T and O += P V, with
// 128 rows per CTA (16 nodes of 8 heads).  Per tile and 128 rows that is 4 * 128 * 128 * hd
// FLOP against 512 * hd B of K/V: 128 FLOP/B per CTA, so one CTA's worth of nodes is bound by
// reading the cache (at 148 SMs even one node's 8 rows keep the tensor pipe ahead of HBM), and
// four CTAs of one sequence (64 nodes) by the products.  Weights go to the second product as a
// bf16 head and a bf16 tail, which makes it twice as long: half as much tensor work again as the
// 2048 clocks per tile at hd 256.
#include <algorithm>
#include <type_traits>

#include "g4_attention.cuh"
#include "g4_common.cuh"
#include "g4_tcgen05.cuh"
#include "g4_tree.cuh"

namespace {

using namespace g4dev;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 128;        // keys per tile = MMA N of the scores
constexpr int kRowsPerCta = 128;  // MMA M
constexpr int kRest = 3 * 1024;   // shared memory besides Q and the ring
// Four threads per query row, each with a quarter of a tile's keys (scores are read once and stay in
// registers) and of O's columns: four warps per scheduler hide each other's latencies.  32 sequences
// of 512 rows over 4160 keys at hd 256 (before weights had tails, which take these 59.6 us to 71.1):
// 59.6 us, with two threads per row (scores read twice) 60.6; one per row, a warp per scheduler, took
// 4500 clocks per tile instead of 2800.
constexpr int kParts = 4;
constexpr int kSoftmaxWarps = 4 * kParts;
constexpr int kKeysPerThread = kTile / kParts;
constexpr int kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr int kThreads = kSoftmaxThreads + 64;  // + TMA warp + MMA warp

// Shared memory: Q [HD/64 boxes][128 rows][128 B], then a ring of equal slots that K and V
// granules pass through in the order the MMA warp uses them: K(0), K(1), V(0), K(2), V(1), ...
// A K granule holds whole 64-column boxes of all 128 keys (K-major operand: 8-row groups 1024 B
// apart); a V granule holds every column of kVKeys keys (MN-major operand: 64-column chunks
// kVKeys * 128 B apart, 8-key groups 1024 B apart).  hd 512: a CTA computes all scores but only
// 256 columns of O, because O (f32) and the two score buffers share 512 TMEM columns.
//
// kPair: two CTAs of a cluster take 256 rows together (tcgen05 cta_group::2).  Each holds its own
// rows of Q, S, P and O, but half of K's keys and half of V's columns, which the tensor cores of
// both read: half the L2 and shared-memory traffic per row.  The even CTA issues every product;
// commits arrive in both, and the odd one's MMA warp tells it when a granule has landed there.
// Taken at hd 256 and 512 where a sequence has more than 128 rows: one sequence over a long cache at
// hd 512, whose CTAs read K for 256 columns of V only, 90.4 us in single CTAs, 75.2 in pairs; 32 x 64
// nodes over 4160 keys 184 and 156, at hd 256 79.5 and 71.1 (100 x 20 nodes over 500 keys, where start
// and drain count: 31.0 and 35.0).  At hd 128 the pair's longer chain of arrivals costs more than its
// traffic saves: 51.2 and 53.5 us, in the short contexts 22.5 and 26.0.
template <int HD, bool kPair>
struct TreeCfg {
    static constexpr int HDV = HD < 256 ? HD : 256;           // O columns per CTA
    static constexpr int OCOLS = HDV < 128 ? 32 : HDV / kParts;  // O columns per thread (hd 64: of the first parts)
    static constexpr int NV = HD / HDV;                        // CTAs (pairs) per 128 (256) rows
    static constexpr int QBYTES = HD * 256;
    static constexpr int KKEYS = kPair ? kTile / 2 : kTile;    // of a tile's keys in this CTA's K
    static constexpr int VCOLS = kPair ? HDV / 2 : HDV;        // columns of this CTA's V
    static constexpr int SLOT = HD == 64 ? 16384 : 32768;
    static constexpr int KGRAN = HD * KKEYS * 2 / SLOT;        // granules per K tile
    static constexpr int KBOX = KKEYS * 128;                   // bytes of a K box
    static constexpr int KBOXES = SLOT / KBOX;                 // boxes per K granule
    static constexpr int VGRAN = VCOLS * 256 / SLOT;
    static constexpr int VKEYS = kTile / VGRAN;                // keys per V granule
    static constexpr int VBOX = VKEYS * 128;                   // bytes of a V box
    static constexpr int SLOTS = SLOT == 16384 ? 8 : (229376 - QBYTES) / SLOT;
    static constexpr int SMEM = QBYTES + SLOTS * SLOT + kRest;  // the rest: TreeShared
    static_assert(SMEM <= 232448, "shared memory");
    static_assert(!kPair || HD >= 256, "pairs are for the wide heads");
};

struct TreeAttnParams {
    const uint16_t* q;
    const uint16_t* v;  // the cache's values (its tensor map's)
    uint16_t* out;
    float* part_o;   // [nsplit][nseq * nodes * heads][HD] (nsplit > 1)
    float2* part_ml; // [nsplit][HD / HDV][nseq * nodes * heads]: running maximum (base 2), sum
    uint32_t* err;
    g4_tree tree;
    const int32_t* seq_pos;
    int seq_base, pos0, seq_stride, heads, sliding, window, ring, limit, nsplit, nseq, history_ready;
    int krows, vrows;  // rows of the tensor maps' boxes (the whole granule, or a part in ring caches)
};

// Tiles that not every row sees whole: the drafted rows lie in one or two, and the rows' windows start
// less than 64 keys apart, the first of them at the first key of the first tile.
constexpr int kMasked = 3;
struct TreeShared {
    uint64_t full[8], empty[8];
    uint64_t peer_full[8];  // pairs: the granule has landed in the odd CTA
    uint64_t q_full, s_full[2], p_ready[2], o_done[2], v_full, scanned, drained;
    uint32_t tmem;
    uint32_t poison[kMasked][4];  // keys of each masked tile whose V row is not finite
    int masked_key[kMasked];      // and its first key
    uint32_t poisoned;            // whether there are any
    int parents[G4_TREE_MAX_NODES];
    int mx[3][kRowsPerCta];  // a row's maximum, ordered as integers (three tiles in turn)
};

static_assert(sizeof(TreeShared) <= kRest, "shared memory");

__device__ __forceinline__ float ex2(float x) {  // 2^x to 2^-22, 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Shared-memory operand descriptors in 128-byte swizzle, 8-row groups 1024 B apart (g4_tcgen05.cuh:
// sw128_desc), as two words: the high one is a constant, the low one moves by address / 16, so a
// step costs the issuing thread one add (rebuilding the 64-bit descriptor per MMA: +25 clocks each).
// `chunk`: for an MN-major operand, the distance of its 64-element chunks in bytes.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t chunk = 16) { return saddr >> 4 | (chunk >> 4) << 16; }
template <bool kPair>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi));
}
template <bool kPair>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
            "mov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
            "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
            "mov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
            "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi));
}
// Arrives on `bar` (in both CTAs of a pair) when the products issued so far have completed.
template <bool kPair>
__device__ __forceinline__ void commit_to(uint64_t* bar) {
    if constexpr (kPair)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        tc_commit(bar);
}
template <bool kPair>
__device__ __forceinline__ void tree_tmem_alloc(uint32_t* dst) {
    if constexpr (kPair) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        tmem_alloc(dst, 512);
    }
}
template <bool kPair>
__device__ __forceinline__ void tree_tmem_dealloc(uint32_t tmem) {
    if constexpr (kPair)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else
        tmem_dealloc(tmem, 512);
}
// Every thread of the pair (of the CTA).
template <bool kPair>
__device__ __forceinline__ void pair_sync() {
    if constexpr (kPair)
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    else
        __syncthreads();
}
// The address of a shared-memory object in CTA `rank` of the pair.
__device__ __forceinline__ uint32_t in_cta(const void* p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// Arrives on a barrier of either CTA.  kRemote: stores to the other CTA's shared memory come before
// it; that release at cluster scope costs 1300 to 4000 clocks.  Without any, what comes before is
// local and complete: a copy that the thread has seen land, tensor-memory stores (tcgen05.wait::st
// and tcgen05.fence) or stores to its own shared memory behind a proxy fence, which the products
// read there.
template <bool kRemote>
__device__ __forceinline__ void arrive_in(uint64_t* bar, int rank) {
    if constexpr (kRemote)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar, rank)) : "memory");
    else
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar, rank)) : "memory");
}
__device__ __forceinline__ void or_in(uint32_t* word, int rank, uint32_t bits) {
    asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(in_cta(word, rank)), "r"(bits) : "memory");
}
// A warp's wait.  kRemote: the other CTA arrives on the barrier.
template <bool kRemote>
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t site) {
    if constexpr (!kRemote) return mbar_wait_warp(bar, parity, err, site);
    bool ok = true;
    unsigned long long t0 = 0;
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity), "r"(kPollSuspendNs)
            : "memory");
        if (done) break;
        if (t0 == 0) t0 = globaltimer_ns();
        else if (globaltimer_ns() - t0 > kWaitLimitNs) {
            raise_error(err, G4_DEVERR_TIMEOUT, site);
            ok = false;
            break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
constexpr uint32_t kTransposeB = 1u << 16;
// Weights lie over the scores they come from, each thread's 32 over its own: 16 columns of heads (bf16
// pairs), then 16 of tails.  TMEM column of the heads of the 16-key step i.
__device__ __forceinline__ int p_col(int i) { return (i >> 1) * kKeysPerThread + (i & 1) * 8; }
constexpr int kTail = kKeysPerThread / 2;
// Floats (but NaN) in the order of integers, and back.
__device__ __forceinline__ int ordered(int bits) { return bits < 0 ? bits ^ 0x7fffffff : bits; }
constexpr int kLowest = (int)0x807fffff;  // ordered(-inf)

// Bits [lo, hi) of the word that covers columns 32 w .. 32 w + 31.
__device__ __forceinline__ uint32_t range_word(int lo, int hi, int w) {
    const int a = max(lo - 32 * w, 0), b = min(hi - 32 * w, 32);
    if (a >= b) return 0u;
    return (b == 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u);
}

// What one sequence's CTAs share.
struct TreeSeq {
    int base, lo, ntiles;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnParams& p, int s) {
    TreeSeq t;
    t.base = p.seq_pos[p.seq_base + s] + p.pos0;
    t.lo = p.sliding ? max(0, t.base - p.window + 1) : 0;  // the root's window reaches furthest back
    t.ntiles = (t.base + p.tree.nodes - t.lo + kTile - 1) / kTile;
    return t;
}
// Sequences whose rows do not fit are left out.
__device__ __forceinline__ bool tree_seq_fits(const TreeAttnParams& p, const TreeSeq& t, int count) {
    return t.base >= 0 && (long long)t.base + count <= p.limit;
}

template <int HD, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
tree_attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const TreeAttnParams p) {
    using C = TreeCfg<HD, kPair>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {  // the swizzle needs it, and nothing is left to move the base (never seen)
        raise_error(p.err, G4_DEVERR_TIMEOUT, 716);
        return;
    }
    uint8_t* qsm = smem;
    uint8_t* ring = smem + C::QBYTES;
    TreeShared& sh = *reinterpret_cast<TreeShared*>(ring + C::SLOTS * C::SLOT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kPair ? blockIdx.x & 1 : 0, unit = kPair ? blockIdx.x >> 1 : blockIdx.x;
    const int vhalf = unit % C::NV, mtile = kPair ? unit / C::NV * 2 + rank : unit / C::NV;
    const int s = blockIdx.y, split = blockIdx.z;
    const int n = p.tree.nodes;

    pdl_trigger();
    // With history_ready the positions and the cached rows below base are final already.
    if (!p.history_ready) pdl_wait();
    // What the prologue reads goes out at once, before the first use of any of it.
    constexpr int CH = HD / 8;  // 16-byte chunks per row
    constexpr int PER = kRowsPerCta * CH / kSoftmaxThreads;
    const int f0 = mtile * kRowsPerCta;
    const size_t grow = (size_t)s * n * p.heads;  // the sequence's first row of q and out
    const uint4* qg = reinterpret_cast<const uint4*>(p.q + (grow + f0) * HD);
    int parent = -1;
    auto prologue_loads = [&]() {
        // Q into the swizzled operand layout.  Rows behind the sequence's count are products of no
        // consequence; rows behind its nodes are zero.
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int u = i * kSoftmaxThreads + threadIdx.x, qr = u / CH, c = u % CH;
            const bool in = f0 + qr < n * p.heads;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             smem_u32(qsm + (c >> 3) * 16384 + qr * 128 + (((c & 7) ^ (qr & 7)) << 4))),
                         "l"(in ? qg + u : reinterpret_cast<const uint4*>(p.q)), "r"(in ? 16 : 0)
                         : "memory");
        }
        if (threadIdx.x < n) parent = p.tree.parents[(size_t)s * p.tree.parent_stride + threadIdx.x];
    };
    const TreeSeq ts = tree_seq(p, s);
    if (warp < kSoftmaxWarps && !p.history_ready) prologue_loads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
            mbar_init(&sh.peer_full[i], 1);
        }
        constexpr int kArrivals = kSoftmaxWarps * (kPair ? 2 : 1);  // a warp each
        mbar_init(&sh.q_full, kArrivals);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_ready[i], kArrivals);
            mbar_init(&sh.o_done[i], 1);
        }
        mbar_init(&sh.v_full, 1);
        mbar_init(&sh.scanned, kArrivals);
        mbar_init(&sh.drained, 1);
        fence_mbar_init();
    }
    if (warp == kSoftmaxWarps + 1) tree_tmem_alloc<kPair>(&sh.tmem);
    // This split's tiles; tile t covers keys lo + (t0 + t) * 128 ...
    const int t0 = (int)((unsigned)split * (unsigned)ts.ntiles / (unsigned)p.nsplit);
    int nt = (int)((unsigned)(split + 1) * (unsigned)ts.ntiles / (unsigned)p.nsplit) - t0;
    const int key0 = ts.lo + t0 * kTile;
    if (ts.base < 0 || ts.base > p.limit) nt = 0;
    if (!p.history_ready) {  // no used row among this CTA's (this pair's)
        const int c = tree_count(p.tree, s, nullptr);
        if ((mtile - rank) * kRowsPerCta >= c * p.heads || !tree_seq_fits(p, ts, c)) nt = 0;
    }
    tc_fence_before();
    pair_sync<kPair>();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t o_tmem = tmem + 256;

    // Every row sees every key of a tile in [all_lo, base); the softmax threads look through the V
    // rows of the others ("masked" tiles) before the product reads them.
    const int all_lo = p.sliding ? ts.base + n - p.window : 0;
    auto masked_tile = [&](int t) { return key0 + t * kTile < all_lo || key0 + (t + 1) * kTile > ts.base; };

    // Granules in ring order: K(0) first, then K(t + 1) before V(t).
    constexpr int G = C::KGRAN + C::VGRAN;
    auto k_granule = [&](int t) { return t == 0 ? 0 : C::KGRAN + (t - 1) * G; };
    auto v_granule = [&](int t) { return C::KGRAN + t * G + (t + 1 < nt ? C::KGRAN : 0); };

    if (warp == kSoftmaxWarps) {
        // ------------------------------------------------ TMA producer --
        if (lane == 0 && nt > 0) {
            prefetch_tensor_map(&kmap);
            prefetch_tensor_map(&vmap);
            bool ok = true, waited = !p.history_ready;
            int g = 0;
            const int seq = p.seq_base + s;
            // `boxes` 64-column boxes of `keys` keys, from column box `box`: one copy where the map's box
            // covers them, else (a ring cache's rows are contiguous for `mirror` keys only) one per box and part.
            auto load = [&](const CUtensorMap* map, int slot, int box, int boxes, int key, int keys, int part) {
                uint8_t* to = ring + slot * C::SLOT;
                const int row0 = seq * p.seq_stride;
                if (part == keys) {
                    tma_load_3d(to, map, &sh.full[slot], 0, row0 + (p.ring ? key % p.ring : key), box);
                } else {
                    for (int r = 0; r < keys; r += part)
                        for (int b = 0; b < boxes; ++b)
                            tma_load_3d(to + b * keys * 128 + r * 128, map, &sh.full[slot], 0, row0 + (key + r) % p.ring,
                                        box + b);
                }
            };
            auto claim = [&]() {
                const int slot = g % C::SLOTS;
                if (g >= C::SLOTS) ok = ok && mbar_wait(&sh.empty[slot], ((g / C::SLOTS) - 1) & 1, p.err, 701);
                if (ok) mbar_arrive_expect_tx(&sh.full[slot], C::SLOT);
                return slot;
            };
            for (int t = -1; t < nt && ok; ++t) {
                if (t + 1 < nt) {
                    const int k0 = key0 + (t + 1) * kTile;
                    if (!waited && k0 + kTile > ts.base) {  // the tile reaches the drafted rows
                        pdl_wait();
                        waited = true;
                    }
                    for (int a = 0; a < C::KGRAN && ok; ++a, ++g) {
                        const int slot = claim();
                        if (!ok) break;
                        load(&kmap, slot, a * C::KBOXES, C::KBOXES, k0 + rank * C::KKEYS, C::KKEYS, p.krows);
                    }
                }
                if (t >= 0) {
                    const int k0 = key0 + t * kTile;
                    for (int a = 0; a < C::VGRAN && ok; ++a, ++g) {
                        const int slot = claim();
                        if (!ok) break;
                        load(&vmap, slot, vhalf * 4 + rank * (C::VCOLS / 64), C::VCOLS / 64, k0 + a * C::VKEYS, C::VKEYS, p.vrows);
                    }
                }
            }
            // Do not leave while copies may still be landing.
            for (int i = g > C::SLOTS ? g - C::SLOTS : 0; i < g; ++i)
                mbar_wait(&sh.full[i % C::SLOTS], (i / C::SLOTS) & 1, p.err, 702);
        }
    } else if (warp == kSoftmaxWarps + 1) {
        // --------------------------------------------------- MMA issuer --
        // The warp stays together (its waits and addresses are uniform); one lane issues.
        int slot = 0;
        uint32_t phase = 0;  // of the slot that comes next in ring order
        auto next = [&]() {
            if (++slot == C::SLOTS) slot = 0, phase ^= 1;
        };
        if (kPair && rank == 1) {
            // Only tells the even CTA (and, of a masked tile's V, the softmax threads) what has landed here.
            bool ok = true;
            int handed = 0;
            for (int t = -1; t < nt && ok && nt > 0; ++t) {
                for (int a = 0; a < (t + 1 < nt ? C::KGRAN : 0) + (t >= 0 ? C::VGRAN : 0) && ok; ++a) {
                    ok = wait_on<false>(&sh.full[slot], phase, p.err, 714);
                    if (ok && lane == 0) arrive_in<false>(&sh.peer_full[slot], 0);
                    __syncwarp();
                    next();
                }
                if (ok && t >= 0 && masked_tile(t)) {
                    // One hand-over at a time: this warp follows the copies, which may be tiles ahead.
                    if (handed > 0) ok = wait_on<true>(&sh.scanned, (handed - 1) & 1, p.err, 717);
                    if (ok && lane == 0) mbar_arrive(&sh.v_full);
                    ++handed;
                }
                __syncwarp();
            }
        } else if (nt > 0) {
            constexpr int kM = kPair ? 256 : 128;
            constexpr uint32_t qk_idesc = mma_idesc_bf16(kM, kTile);
            constexpr uint32_t pv_idesc = mma_idesc_bf16(kM, C::HDV) | kTransposeB;
            const uint32_t qa = desc_lo(smem_u32(qsm)), ka = desc_lo(smem_u32(ring));
            const uint32_t va = desc_lo(smem_u32(ring), C::VBOX);
            bool ok = wait_on<kPair>(&sh.q_full, 0, p.err, 703);
            auto landed = [&](int sl, uint32_t ph) {
                ok = ok && wait_on<false>(&sh.full[sl], ph, p.err, 704);
                if (kPair) ok = ok && wait_on<true>(&sh.peer_full[sl], ph, p.err, 705);
                return ok;
            };
            auto scores = [&](int t) {
#pragma unroll
                for (int a = 0; a < C::KGRAN; ++a) {
                    if (!landed(slot, phase)) return;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t b = ka + slot * (C::SLOT >> 4), d = tmem + (t & 1) * 128;
#pragma unroll
                        for (int i = 0; i < C::KBOXES * 4; ++i)
                            mma_ss<kPair>(d, qa + (((a * C::KBOXES + i / 4) * 16384 + (i % 4) * 32) >> 4),
                                          b + (((i / 4) * C::KBOX + (i % 4) * 32) >> 4), qk_idesc, (a | i) ? 1u : 0u);
                        commit_to<kPair>(&sh.empty[slot]);
                        if (a == C::KGRAN - 1) commit_to<kPair>(&sh.s_full[t & 1]);
                    }
                    __syncwarp();
                    next();
                }
            };
            if (ok) scores(0);
            for (int t = 0; t < nt && ok; ++t) {
                if (t + 1 < nt) scores(t + 1);
                if (ok && masked_tile(t)) {  // hand V to the softmax threads (only this warp can follow the ring)
                    int sl = slot;
                    uint32_t ph = phase;
                    for (int a = 0; a < C::VGRAN && ok; ++a) {
                        ok = wait_on<false>(&sh.full[sl], ph, p.err, 708);
                        if (++sl == C::SLOTS) sl = 0, ph ^= 1;
                    }
                    if (ok && lane == 0) mbar_arrive(&sh.v_full);
                    __syncwarp();
                }
                ok = ok && wait_on<kPair>(&sh.p_ready[t & 1], (t >> 1) & 1, p.err, 706);
#pragma unroll
                for (int a = 0; a < C::VGRAN; ++a) {
                    if (!landed(slot, phase)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t b = va + slot * (C::SLOT >> 4), w = tmem + (t & 1) * 128;
#pragma unroll
                        for (int i = 0; i < C::VKEYS / 16; ++i) {
                            const uint32_t head = w + p_col(a * (C::VKEYS / 16) + i), bv = b + i * (2048 >> 4);
                            mma_ts<kPair>(o_tmem, head, bv, pv_idesc, (a | i) || t > 0 ? 1u : 0u);
                            mma_ts<kPair>(o_tmem, head + kTail, bv, pv_idesc, 1u);
                        }
                        commit_to<kPair>(&sh.empty[slot]);
                        if (a == C::VGRAN - 1) commit_to<kPair>(&sh.o_done[t & 1]);
                    }
                    __syncwarp();
                    next();
                }
            }
            // Do not free the tensor memory while products may still be running (after a failed wait).
            if (elect_one()) commit_to<kPair>(&sh.drained);
            __syncwarp();
            wait_on<false>(&sh.drained, 0, p.err, 711);
        }
    } else {
        // ------------------ softmax: kParts threads (warps w, w + 4, ...) per query row --
        const int part = warp >> 2, r = (warp & 3) * 32 + lane;
        const int f = f0 + r;
        if (p.history_ready) {
            pdl_wait();
            prologue_loads();
        }
        int count = tree_count(p.tree, s, p.err);
        if (!tree_seq_fits(p, ts, count)) {
            if (threadIdx.x == 0 && blockIdx.x == 0 && split == 0) raise_error(p.err, G4_DEVERR_BAD_INDEX);
            count = 0;
        }
        if (threadIdx.x < n) {
            const bool good = parent >= -1 && parent < (int)threadIdx.x;
            if (!good && (int)threadIdx.x < count) raise_error(p.err, G4_DEVERR_BAD_INDEX);
            sh.parents[threadIdx.x] = good ? parent : -1;
        }
        if (threadIdx.x < kMasked * 4) sh.poison[threadIdx.x >> 2][threadIdx.x & 3] = 0u;
        if (threadIdx.x == 0) sh.poisoned = 0u;
        const int rows = count * p.heads;              // of this sequence
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        auto tell = [&](uint64_t* bar) {  // the issuing CTA, once per warp
            __syncwarp();
            if (lane == 0) {
                if (kPair && rank == 1) arrive_in<false>(bar, 0);
                else mbar_arrive(bar);
            }
        };
        tell(&sh.q_full);
        if (part < 2) sh.mx[part][r] = kLowest;
        auto softmax_sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory"); };
        auto row_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(2 + (warp & 3)), "n"(32 * kParts) : "memory"); };
        softmax_sync();  // parents
        const bool live = f < rows;
        const bool warp_live = f - lane < rows;
        // The row's visible drafted rows (bit = node) and first visible cached key.
        unsigned long long seen = 0ull;
        int first = 0x7fffffff;
        if (live) {
            int up = 0;
            for (int a = f / p.heads; a >= 0; a = sh.parents[a], ++up)
                if (!p.sliding || up < p.window) seen |= 1ull << a;
            first = p.sliding ? ts.base + up - p.window : 0;  // up = depth + 1
        }
        // Which of the keys k0 + 32 w .. + 31 the row sees.
        auto visible = [&](int k0, int w) {
            const int d = ts.base - k0, sft = 32 * w - d;  // node 0 is column d: the word's drafted bits start at node sft
            const unsigned long long bits = sft >= 64 || sft <= -32 ? 0ull : sft >= 0 ? seen >> sft : seen << -sft;
            return live ? range_word(first - k0, d, w) | (uint32_t)bits : 0u;
        };
        const uint32_t s_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + part * kKeysPerThread;
        const uint32_t o_part = o_tmem + ((uint32_t)((warp & 3) * 32) << 16) + part * C::OCOLS;
        const bool has_o = part * C::OCOLS < C::HDV;
        float m = -INFINITY, mu = 0.f, l = 0.f;
        // A warp whose wait gave up keeps to the barriers of the others and does nothing else.
        bool ok = true;
        int nmasked = 0;
        for (int t = 0; t < nt; ++t) {
            const int k0 = key0 + t * kTile;
            const bool masked = masked_tile(t);
            ok = ok && wait_on<false>(&sh.s_full[t & 1], (t >> 1) & 1, p.err, 707);
            tc_fence_after();
            uint32_t x[32];
            int* const mx = sh.mx[t % 3];
            if (warp_live && ok) {
                tmem_ld_32x32b_x32(s_tmem + (t & 1) * 128, x);
                tmem_ld_wait(x);
                if (masked) {
                    const uint32_t v = visible(k0, part);
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = v >> i & 1u ? x[i] : 0xff800000u;
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(x[i]));
                atomicMax(&mx[r], ordered(__float_as_int(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])))));
            }
            row_sync();
            if (warp_live && ok) {
                const float tm = __int_as_float(ordered(mx[r]));
                if (part == 0) sh.mx[(t + 2) % 3][r] = kLowest;  // last read before this tile's barrier
                // The weights are taken against a maximum that may be stale by up to 2^8 (P and the
                // sums have the range for it), so O is rescaled only when it is exceeded.
                const bool grow_m = tm > m && !((tm - m) * kLog2e <= 8.f);
                float factor = 1.f;
                if (grow_m) {
                    factor = m == -INFINITY ? 0.f : ex2((m - tm) * kLog2e);
                    m = tm;
                    mu = m * kLog2e;
                    l *= factor;
                }
                if (t > 0 && has_o && __any_sync(0xffffffffu, grow_m)) {
                    ok = wait_on<false>(&sh.o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, p.err, 709);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < C::OCOLS; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_part + c, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_st_32x32b_x32(o_part + c, o);
                    }
                }
                // P as a bf16 head and a bf16 tail (the product's operand type): 2^-16 of a weight is lost,
                // as in g4_attention_rows, so that verifying a token and decoding it differ by no more than
                // the order of their sums.  In heads alone a weight loses 2^-8, which is as much again as the
                // rounding of the result (2.2e-3 of its norm instead of 1.65e-3).
                uint32_t w[32];
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float a = ex2(fmaf(__uint_as_float(x[2 * i]), kLog2e, -mu));
                    const float b = ex2(fmaf(__uint_as_float(x[2 * i + 1]), kLog2e, -mu));
                    l0 += a;
                    l1 += b;
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(b), "f"(a));
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
                        : "=r"(w[kTail + i])
                        : "f"(b - __uint_as_float(w[i] & 0xffff0000u)), "f"(a - __uint_as_float(w[i] << 16)));
                }
                tmem_st_32x32b_x32(s_tmem + (t & 1) * 128, w);
                l += l0 + l1;
                tmem_st_wait();
            }
            if (masked) {
                // What a row does not see must not reach its product: 0 * NaN.  Thread = key and a part of the
                // columns: rows behind base + count become 0; values that are not finite become 0 and
                // are remembered, for the rows that see them.
                const int key = threadIdx.x & 127, vrow = key % C::VKEYS, g = v_granule(t) + key / C::VKEYS;
                uint32_t* poison = sh.poison[nmasked];
                if (threadIdx.x == 0) sh.masked_key[nmasked] = k0;
                ok = ok && wait_on<false>(&sh.v_full, nmasked & 1, p.err, 712);
                ok = ok && wait_on<false>(&sh.full[g % C::SLOTS], (g / C::SLOTS) & 1, p.err, 713);  // of this phase now
                ++nmasked;
                if (ok) {
                    uint8_t* vr = ring + (g % C::SLOTS) * C::SLOT + vrow * 128;
                    const bool outside = k0 + key >= ts.base + count;
                    bool bad = false;
                    auto at = [&](int i) {
                        const int c = part * (C::VCOLS / (8 * kParts)) + i;
                        return reinterpret_cast<uint4*>(vr + (c >> 3) * C::VBOX + (((c & 7) ^ (vrow & 7)) << 4));
                    };
                    // an exponent of all ones carries into the bit above it
                    auto odd = [](uint32_t e) { return ((e & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
                    uint32_t any = 0u;
#pragma unroll 8
                    for (int i = 0; i < C::VCOLS / (8 * kParts); ++i) {
                        const uint4 w = *at(i);
                        any |= odd(w.x) | odd(w.y) | odd(w.z) | odd(w.w);
                    }
                    if (outside || any) {
#pragma unroll 1
                        for (int i = 0; i < C::VCOLS / (8 * kParts); ++i) {
                            const uint4 w = *at(i);
                            auto clean = [&](uint32_t e) {
                                const uint32_t o = odd(e);
                                return outside ? 0u : e & ((o & 0x8000u ? 0u : 0xffffu) | (o & 0x80000000u ? 0u : 0xffff0000u));
                            };
                            *at(i) = make_uint4(clean(w.x), clean(w.y), clean(w.z), clean(w.w));
                        }
                        bad = !outside;
                    }
                    if (bad) {
                        atomicOr(&poison[key >> 5], 1u << lane);
                        sh.poisoned = 1u;
                        if (kPair) {  // its rows see the same keys
                            or_in(&poison[key >> 5], rank ^ 1, 1u << lane);
                            or_in(&sh.poisoned, rank ^ 1, 1u);
                        }
                    }
                    fence_proxy_async_smem();
                }
                if (kPair) {
                    __syncwarp();
                    if (lane == 0) {
                        arrive_in<true>(&sh.scanned, 0);
                        arrive_in<true>(&sh.scanned, 1);
                    }
                    ok = wait_on<true>(&sh.scanned, (nmasked - 1) & 1, p.err, 715) && ok;
                } else {
                    softmax_sync();
                }
            }
            tc_fence_before();
            tell(&sh.p_ready[t & 1]);
        }
        // ---- O of the row ----
        if (nt > 0) {
            // The last product is done, so Q and the ring have been read for the last time.  (A warp whose
            // wait gave up writes nothing: copies may be landing yet.)
            ok = ok && wait_on<false>(&sh.o_done[(nt - 1) & 1], ((nt - 1) >> 1) & 1, p.err, 710);
            float* const sums = reinterpret_cast<float*>(ring + C::SLOTS * C::SLOT) - kParts * kRowsPerCta;  // behind the staged rows
            static_assert(kRowsPerCta * C::HDV * 4 + kParts * kRowsPerCta * 4 <= C::QBYTES + C::SLOTS * C::SLOT, "staging");
            if (ok) sums[part * kRowsPerCta + r] = l;
            row_sync();
            if (ok) {
                l = 0.f;
                for (int i = 0; i < kParts; ++i) l += sums[i * kRowsPerCta + r];
            }
        }
        tc_fence_after();
        if (nt > 0 && warp_live && ok && has_o && sh.poisoned) {
            // What was taken out of V comes back into its column of the rows that see it, as if the product
            // had met it.
            const size_t row0 = (size_t)(p.seq_base + s) * p.seq_stride;
            const uint16_t* v = p.v + row0 * HD + vhalf * C::HDV + part * C::OCOLS;
#pragma unroll 1
            for (int c = 0; c < C::OCOLS; c += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_part + c, o);
                tmem_ld_wait(o);
#pragma unroll 1
                for (int w = 0; w < nmasked * 4; ++w) {
                    const int k0 = sh.masked_key[w >> 2];
                    for (uint32_t bits = sh.poison[w >> 2][w & 3] & visible(k0, w & 3); bits; bits &= bits - 1) {
                        const int key = k0 + 32 * (w & 3) + __ffs(bits) - 1;
                        const uint16_t* e = v + (size_t)(p.ring ? key % p.ring : key) * HD + c;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if ((e[i] & 0x7f80u) == 0x7f80u)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float((uint32_t)e[i] << 16));
                    }
                }
                __syncwarp();
                tmem_st_32x32b_x32(o_part + c, o);
            }
            tmem_st_wait();
        }
        // Rows leave through shared memory: written
        // by row, 16-byte chunks permuted within 128 B against bank conflicts, read back along the
        // rows, so that global stores are whole lines.  (Stores from the row's own thread touch 32
        // lines each: 5 to 10 thousand clocks per CTA.)
        if (nt > 0 && warp_live) {
            const size_t nrows = (size_t)p.nseq * n * p.heads;
            const float inv = 1.f / l;
            auto stage = [&](auto whole_c) {
                constexpr bool whole = decltype(whole_c)::value;
                constexpr int rowb = C::HDV * (whole ? 2 : 4), chunks = rowb / 16;  // of a staged row
                uint8_t* const mine = smem + r * rowb;
                if (ok && has_o) {
#pragma unroll 1
                    for (int c = 0; c < C::OCOLS; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_part + c, o);
                        tmem_ld_wait(o);
                        const int col = part * C::OCOLS + c;
#pragma unroll
                        for (int i = 0; i < (whole ? 4 : 8); ++i) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if (whole)
                                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
                                        : "=r"(w[k])
                                        : "f"(__uint_as_float(o[(8 * i + 2 * k + 1) & 31]) * inv),
                                          "f"(__uint_as_float(o[(8 * i + 2 * k) & 31]) * inv));
                                else
                                    w[k] = o[4 * i + k];
                            }
                            const int ch = (whole ? col / 8 : col / 4) + i;
                            *reinterpret_cast<uint4*>(mine + (((ch & ~7) | ((ch ^ r) & 7)) << 4)) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    if (!whole && live && part == 0)
                        p.part_ml[(split * C::NV + vhalf) * nrows + grow + f] = make_float2(mu, l);
                }
                row_sync();
                if (ok) {
                    const int row0 = (warp & 3) * 32;  // the row group
                    uint8_t* const to = (whole ? reinterpret_cast<uint8_t*>(p.out) : reinterpret_cast<uint8_t*>(p.part_o)) +
                                        ((whole ? 0 : split * nrows) + grow + f0) * (HD * (whole ? 2 : 4)) + vhalf * rowb;
#pragma unroll 8
                    for (int u = part * 32 + lane; u < 32 * chunks; u += 32 * kParts) {
                        const int rr = row0 + u / chunks, ch = u % chunks;
                        if (f0 + rr < rows)
                            *reinterpret_cast<uint4*>(to + (size_t)rr * (HD * (whole ? 2 : 4)) + ch * 16) =
                                *reinterpret_cast<const uint4*>(smem + rr * rowb + (((ch & ~7) | ((ch ^ rr) & 7)) << 4));
                    }
                }
            };
            if (p.nsplit == 1) stage(std::true_type{});
            else stage(std::false_type{});
        } else if (nt == 0 && p.nsplit > 1 && live && part == 0) {
            const size_t nrows = (size_t)p.nseq * n * p.heads;
            p.part_ml[(split * C::NV + vhalf) * nrows + grow + f] = make_float2(0.f, 0.f);
        }
    }
    tc_fence_before();
    __syncwarp();
    pair_sync<kPair>();  // (of a pair: neither leaves while the other may read its shared memory)
    if (warp == kSoftmaxWarps + 1) {
        __syncwarp();
        tc_fence_after();
        tree_tmem_dealloc<kPair>(tmem);
    }
}

// Joins the splits of a row: out = sum_i 2^(mu_i - mu) O_i / sum_i 2^(mu_i - mu) l_i.  One CTA per
// row and HDV columns, a thread per two columns.  The splits' (mu, l) and the first 16 splits'
// columns are read at once: one round trip (columns after the factors: 1.4 us more of the 15.5 us of
// one sequence's 8 nodes over 4096 keys).  A split that saw none of the row's keys has l = 0 and is
// left out (its O was not written).
constexpr int kMaxSplits = 160;
template <int HD>
__global__ void __launch_bounds__(TreeCfg<HD, false>::HDV / 2) tree_combine_kernel(const TreeAttnParams p) {
    using C = TreeCfg<HD, false>;
    constexpr int T = C::HDV / 2;
    __shared__ float2 ml[kMaxSplits];
    pdl_trigger();
    const size_t row = blockIdx.x;
    const int vhalf = blockIdx.y;
    const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
    const int s = (int)(row / (p.tree.nodes * p.heads)), node = (int)(row / p.heads) - s * p.tree.nodes;
    pdl_wait();
    // The first splits' columns are on their way before it is known which of them count.
    constexpr int B = 16;
    const float2* o = reinterpret_cast<const float2*>(p.part_o + row * HD + vhalf * C::HDV) + threadIdx.x;
    auto column = [&](int i) { return i < p.nsplit ? __ldg(o + i * nrows * (HD / 2)) : make_float2(0.f, 0.f); };
    float2 v[B];
#pragma unroll
    for (int b = 0; b < B; ++b) v[b] = column(b);
    for (int i = threadIdx.x; i < p.nsplit; i += T) ml[i] = p.part_ml[(i * C::NV + vhalf) * nrows + row];
    const int count = tree_count(p.tree, s, nullptr);
    const bool used = node < count && tree_seq_fits(p, tree_seq(p, s), count);
    __syncthreads();
    if (!used) return;
    float mu = -INFINITY;
    for (int i = 0; i < p.nsplit; ++i) mu = ml[i].y != 0.f ? fmaxf(mu, ml[i].x) : mu;
    float l = 0.f, a0 = 0.f, a1 = 0.f;
    for (int i0 = 0; i0 < p.nsplit; i0 += B) {
        if (i0 > 0) {
#pragma unroll
            for (int b = 0; b < B; ++b) v[b] = column(i0 + b);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (i0 + b >= p.nsplit || ml[i0 + b].y == 0.f) continue;  // (its columns were not written)
            const float f = ex2(ml[i0 + b].x - mu);
            l += f * ml[i0 + b].y;
            a0 += f * v[b].x;
            a1 += f * v[b].y;
        }
    }
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(a1 / l), "f"(a0 / l));
    reinterpret_cast<uint32_t*>(p.out + row * HD + vhalf * C::HDV)[threadIdx.x] = w;
}

template <int HD, bool kPair>
g4_status launch_tree_attention_t(g4_ctx* ctx, const g4_kv* kv, TreeAttnParams p) {
    using C = TreeCfg<HD, kPair>;
    const int mtiles = (p.tree.nodes * p.heads + kRowsPerCta - 1) / kRowsPerCta;
    const int longest = (p.sliding && p.window < p.seq_stride ? p.window : p.seq_stride) + p.tree.nodes;
    const int ntiles = (longest + kTile - 1) / kTile;
    const int across = (kPair ? (mtiles + 1) / 2 * 2 : mtiles) * C::NV;  // CTAs of a sequence and split
    const long long ctas = (long long)across * p.nseq;
    // Split the keys while that adds CTAs to SMs without one: down to one tile per split up to 16
    // splits (which the join reads in one round trip), then to two.  One sequence of 8 nodes over 4096
    // keys: 14.3 us at one tile, 14.2 so, 15.0 at two, 15.2 at three; 8 sequences with a window of 512
    // (five tiles): 14.8, 16.9 and 18.9 at one, two and three.  A split costs a start, a drain, the join
    // and the partial rows' way to L2 and back, so it has to save four tiles: 64 sequences of 16 nodes
    // with a window of 512 take 34.8 us in two splits (two tiles saved), 21.1 whole, 32 of them 23.5 in
    // three (three saved) and 20.1, 16 of them 17.1 in five (four saved) and 20.1.
    int nsplit = (int)std::max<long long>(
        1, std::min<long long>({ctx->num_sms / ctas, std::max(ntiles / 2, std::min(ntiles, 16)), kMaxSplits}));
    if (ntiles - (ntiles + nsplit - 1) / nsplit < 4) nsplit = 1;
    p.nsplit = nsplit;
    const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
    if (nsplit > 1) {
        const size_t ob = nsplit * nrows * HD * sizeof(float);
        g4_status st = g4::ensure_workspace(ctx, ob + (size_t)nsplit * C::NV * nrows * sizeof(float2));
        if (st) return st;
        p.part_o = static_cast<float*>(ctx->ws);
        p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ctx->ws) + ob);
    }
    static std::atomic<uint64_t> attr_set{0};
    if (!(attr_set.load() & (1ull << ctx->device))) {
        G4_CHECK_CUDA(cudaFuncSetAttribute(tree_attention_kernel<HD, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           C::SMEM));
        attr_set.fetch_or(1ull << ctx->device);
    }
    const g4_tree_maps& maps = kv->tree[kPair];
    p.krows = maps.krows;
    p.vrows = maps.vrows;
    g4_status st = g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<HD, kPair>, dim3(across, p.nseq, nsplit),
                              dim3(kThreads), C::SMEM, kPair ? 2 : 1, maps.k, maps.v, p);
    if (st || nsplit == 1) return st;
    // The join is set up while the attention runs, and waits for it (griddepcontrol).
    const bool pdl = ctx->pdl;
    ctx->pdl = true;
    st = g4::launch(ctx, "tree_combine_kernel", tree_combine_kernel<HD>, dim3((unsigned)nrows, C::NV), dim3(C::HDV / 2), 0, 1,
                    p);
    ctx->pdl = pdl;
    return st;
}
template <int HD>
g4_status launch_tree_attention(g4_ctx* ctx, const g4_kv* kv, const TreeAttnParams& p) {
    if constexpr (HD >= 256) {
        if (p.tree.nodes * p.heads > kRowsPerCta) return launch_tree_attention_t<HD, true>(ctx, kv, p);
    }
    return launch_tree_attention_t<HD, false>(ctx, kv, p);
}

template <int HD, bool kPair>
g4_status tree_maps(g4_kv* kv) {
    using C = TreeCfg<HD, kPair>;
    g4_tree_maps& m = kv->tree[kPair];
    const int contiguous = kv->ring ? kv->mirror : kTile;
    m.krows = std::min(C::KKEYS, contiguous);
    m.vrows = std::min(C::VKEYS, contiguous);
    const uint64_t dims[3] = {64, (uint64_t)kv->rows_total, HD / 64}, pitch[2] = {HD * 2, 128};
    const uint32_t kbox[3] = {64, (uint32_t)m.krows, m.krows == C::KKEYS ? (uint32_t)C::KBOXES : 1u};
    const uint32_t vbox[3] = {64, (uint32_t)m.vrows, m.vrows == C::VKEYS ? C::VCOLS / 64u : 1u};
    g4_status st = g4::encode_tensor_map_3d(&m.k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv->k, dims, pitch, kbox,
                                            CU_TENSOR_MAP_SWIZZLE_128B);
    if (st) return st;
    return g4::encode_tensor_map_3d(&m.v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv->v, dims, pitch, vbox,
                                    CU_TENSOR_MAP_SWIZZLE_128B);
}
template <int HD>
g4_status tree_maps_all(g4_kv* kv) {
    g4_status st = tree_maps<HD, false>(kv);
    if constexpr (HD >= 256) {
        if (!st) st = tree_maps<HD, true>(kv);
    }
    return st;
}

}  // namespace

namespace g4 {

g4_status make_tree_maps(g4_kv* kv) {
    switch (kv->hd) {
        case 64: return tree_maps_all<64>(kv);
        case 128: return tree_maps_all<128>(kv);
        case 256: return tree_maps_all<256>(kv);
        default: return tree_maps_all<512>(kv);
    }
}

}  // namespace g4

extern "C" g4_status g4_attention_tree(g4_ctx* ctx, const void* q_bf16, const g4_kv* kv, int rows, int heads, int hd,
                                       const g4_rows* map, const g4_tree* tree, int seq_stride, int sliding, int window,
                                       void* out_bf16) {
    g4_status st = g4::check_tree_rows("g4_attention_tree", map, tree, rows);
    if (st) return st;
    if (heads < 1 || heads > 8)
        return g4::set_error(G4_ERR_UNSUPPORTED, "g4_attention_tree: %d heads per KV head (1..8 supported)", heads);
    if (sliding && window < 1) return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: window %d", window);
    if ((reinterpret_cast<uintptr_t>(q_bf16) | reinterpret_cast<uintptr_t>(out_bf16)) % 16 != 0)
        return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: q and out must be 16-byte aligned");
    if (!kv || !q_bf16 || !out_bf16) return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: null argument");
    st = g4::use_device(ctx);
    if (st) return st;
    if (hd != kv->hd) return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: hd %d != cache hd %d", hd, kv->hd);
    if (kv->device != ctx->device)
        return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: the cache is on device %d, the context on %d",
                             kv->device, ctx->device);
    if (kv->ring && seq_stride != kv->seq_rows)
        return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: seq_stride %d of a ring cache must be its %d rows per "
                             "sequence", seq_stride, kv->seq_rows);
    if (rows == 0) return G4_OK;
    const int nseq = rows / tree->nodes;
    if (nseq > 65535) return g4::set_error(G4_ERR_UNSUPPORTED, "g4_attention_tree: %d sequences (65535 supported)", nseq);
    if (seq_stride < 1 || ((long long)map->seq_base + nseq) * seq_stride > kv->rows_total)
        return g4::set_error(G4_ERR_RANGE, "g4_attention_tree: sequences beyond the cache (%d rows)", kv->rows_total);
    st = g4::check_ring("g4_attention_tree", kv, sliding, window, tree->nodes);
    if (st) return st;
    const TreeAttnParams p{static_cast<const uint16_t*>(q_bf16), kv->v, static_cast<uint16_t*>(out_bf16), nullptr, nullptr,
                           ctx->d_err, *tree, map->seq_pos, map->seq_base, map->pos0, seq_stride, heads,
                           sliding ? 1 : 0, window, kv->ring, kv->ring ? kv->capacity : seq_stride, 1, nseq,
                           (map->flags & G4_ROWS_HISTORY_READY) ? 1 : 0};
    switch (hd) {
        case 64: return launch_tree_attention<64>(ctx, kv, p);
        case 128: return launch_tree_attention<128>(ctx, kv, p);
        case 256: return launch_tree_attention<256>(ctx, kv, p);
        case 512: return launch_tree_attention<512>(ctx, kv, p);
        default: return g4::set_error(G4_ERR_UNSUPPORTED, "g4_attention_tree: head dim %d (64/128/256/512 supported)", hd);
    }
}
