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
// four CTAs of one sequence (64 nodes) by the products.
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
// Two threads per query row, each with half of a tile's keys and half of O's columns: two warps
// per scheduler hide each other's latencies (one warp per scheduler: 4500 clocks per tile).
constexpr int kSoftmaxWarps = 8;
constexpr int kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr int kThreads = kSoftmaxThreads + 64;  // + TMA warp + MMA warp

// Shared memory: Q [HD/64 boxes][128 rows][128 B], then a ring of equal slots that K and V
// granules pass through in the order the MMA warp uses them: K(0), K(1), V(0), K(2), V(1), ...
// A K granule holds whole 64-column boxes of all 128 keys (K-major operand: 8-row groups 1024 B
// apart); a V granule holds every column of kVKeys keys (MN-major operand: 64-column chunks
// kVKeys * 128 B apart, 8-key groups 1024 B apart).  hd 512: a CTA computes all scores but only
// 256 columns of O, because O (f32) and the two score buffers share 512 TMEM columns.
template <int HD>
struct TreeCfg {
    static constexpr int HDV = HD < 256 ? HD : 256;           // O columns per CTA
    static constexpr int NV = HD / HDV;                        // CTAs per 128 rows
    static constexpr int QBYTES = HD * 256;
    static constexpr int SLOT = HD == 64 ? 16384 : 32768;
    static constexpr int KGRAN = HD * 256 / SLOT;              // granules per K tile
    static constexpr int KBOXES = SLOT / 16384;                // boxes per K granule
    static constexpr int VGRAN = HDV * 256 / SLOT;
    static constexpr int VKEYS = kTile / VGRAN;                // keys per V granule
    static constexpr int VBOX = VKEYS * 128;                   // bytes of a V box
    static constexpr int SLOTS = HD == 64 ? 8 : (229376 - QBYTES) / SLOT;
    static constexpr int SMEM = QBYTES + SLOTS * SLOT + 3072;  // the rest: alignment (1008), TreeShared
    static_assert(SMEM <= 232448, "shared memory");
};

struct TreeAttnParams {
    const uint16_t* q;
    uint16_t* out;
    float* part_o;   // [nsplit][nseq * nodes * heads][HD] (nsplit > 1)
    float2* part_ml; // [nsplit][HD / HDV][nseq * nodes * heads]: running maximum (base 2), sum
    uint32_t* err;
    g4_tree tree;
    const int32_t* seq_pos;
    int seq_base, pos0, seq_stride, heads, sliding, window, ring, limit, nsplit, nseq, history_ready;
    int krows, vrows;  // rows of the tensor maps' boxes (the whole granule, or a part in ring caches)
};

struct TreeShared {
    uint64_t full[8], empty[8];
    uint64_t q_full, s_full[2], p_ready[2], o_done[2], v_full, drained;
    uint32_t tmem;
    uint32_t poison[3][4];  // keys of a masked tile whose V row is not finite (three tiles in turn)
    int parents[G4_TREE_MAX_NODES];
    float mx[2][2][kRowsPerCta];  // a row's maximum of each half (two tiles in turn); at the end its sums
};

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
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi));
}
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
constexpr uint32_t kTransposeB = 1u << 16;
// Weights (bf16 pairs) lie over the scores they come from, each half of a tile over its own half:
// TMEM column of the 16-key step i.
__device__ __forceinline__ int p_col(int i) { return (i >> 2) * 64 + (i & 3) * 8; }

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

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
tree_attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const TreeAttnParams p) {
    using C = TreeCfg<HD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* qsm = smem;
    uint8_t* ring = smem + C::QBYTES;
    TreeShared& sh = *reinterpret_cast<TreeShared*>(ring + C::SLOTS * C::SLOT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int mtile = blockIdx.x / C::NV, vhalf = blockIdx.x % C::NV;
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
                         "l"(qg + (in ? u : 0)), "r"(in ? 16 : 0)
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
        }
        mbar_init(&sh.q_full, kSoftmaxThreads);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_ready[i], kSoftmaxThreads);
            mbar_init(&sh.o_done[i], 1);
        }
        mbar_init(&sh.v_full, 1);
        mbar_init(&sh.drained, 1);
        fence_mbar_init();
    }
    if (warp == kSoftmaxWarps + 1) tmem_alloc(&sh.tmem, 512);
    // This split's tiles; tile t covers keys lo + (t0 + t) * 128 ...
    const int t0 = (int)((unsigned)split * (unsigned)ts.ntiles / (unsigned)p.nsplit);
    int nt = (int)((unsigned)(split + 1) * (unsigned)ts.ntiles / (unsigned)p.nsplit) - t0;
    const int key0 = ts.lo + t0 * kTile;
    if (ts.base < 0 || ts.base > p.limit) nt = 0;
    if (!p.history_ready) {  // no used row among this CTA's
        const int c = tree_count(p.tree, s, nullptr);
        if (mtile * kRowsPerCta >= c * p.heads || !tree_seq_fits(p, ts, c)) nt = 0;
    }
    tc_fence_before();
    __syncthreads();
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
                        load(&kmap, slot, a * C::KBOXES, C::KBOXES, k0, kTile, p.krows);
                    }
                }
                if (t >= 0) {
                    const int k0 = key0 + t * kTile;
                    for (int a = 0; a < C::VGRAN && ok; ++a, ++g) {
                        const int slot = claim();
                        if (!ok) break;
                        load(&vmap, slot, vhalf * 4, C::HDV / 64, k0 + a * C::VKEYS, C::VKEYS, p.vrows);
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
        if (nt > 0) {
            constexpr uint32_t qk_idesc = mma_idesc_bf16(128, kTile);
            constexpr uint32_t pv_idesc = mma_idesc_bf16(128, C::HDV) | kTransposeB;
            const uint32_t qa = desc_lo(smem_u32(qsm)), ka = desc_lo(smem_u32(ring));
            const uint32_t va = desc_lo(smem_u32(ring), C::VBOX);
            bool ok = mbar_wait_warp(&sh.q_full, 0, p.err, 703);
            int slot = 0;
            uint32_t phase = 0;  // of the slot that comes next in ring order
            auto next = [&]() {
                if (++slot == C::SLOTS) slot = 0, phase ^= 1;
            };
            auto scores = [&](int t) {
#pragma unroll
                for (int a = 0; a < C::KGRAN; ++a) {
                    ok = ok && mbar_wait_warp(&sh.full[slot], phase, p.err, 704);
                    if (!ok) return;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t b = ka + slot * (C::SLOT >> 4), d = tmem + (t & 1) * 128;
#pragma unroll
                        for (int i = 0; i < C::KBOXES * 4; ++i)
                            mma_ss(d, qa + (((a * C::KBOXES + i / 4) * 16384 + (i % 4) * 32) >> 4),
                                   b + (((i / 4) * 16384 + (i % 4) * 32) >> 4), qk_idesc, (a | i) ? 1u : 0u);
                        tc_commit(&sh.empty[slot]);
                        if (a == C::KGRAN - 1) tc_commit(&sh.s_full[t & 1]);
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
                        ok = mbar_wait_warp(&sh.full[sl], ph, p.err, 708);
                        if (++sl == C::SLOTS) sl = 0, ph ^= 1;
                    }
                    if (ok && lane == 0) mbar_arrive(&sh.v_full);
                    __syncwarp();
                }
                ok = ok && mbar_wait_warp(&sh.p_ready[t & 1], (t >> 1) & 1, p.err, 705);
#pragma unroll
                for (int a = 0; a < C::VGRAN; ++a) {
                    ok = ok && mbar_wait_warp(&sh.full[slot], phase, p.err, 706);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t b = va + slot * (C::SLOT >> 4), w = tmem + (t & 1) * 128;
#pragma unroll
                        for (int i = 0; i < C::VKEYS / 16; ++i)
                            mma_ts(o_tmem, w + p_col(a * (C::VKEYS / 16) + i), b + i * (2048 >> 4), pv_idesc,
                                   (a | i) || t > 0 ? 1u : 0u);
                        tc_commit(&sh.empty[slot]);
                        if (a == C::VGRAN - 1) tc_commit(&sh.o_done[t & 1]);
                    }
                    __syncwarp();
                    next();
                }
            }
            // Do not free the tensor memory while products may still be running (after a failed wait).
            if (elect_one()) tc_commit(&sh.drained);
            __syncwarp();
            mbar_wait_warp(&sh.drained, 0, p.err, 711);
        }
    } else {
        // ------------------ softmax: two threads (warps w, w + 4) per query row --
        const int half = warp >> 2, r = (warp & 3) * 32 + lane;
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
        if (threadIdx.x < 4) sh.poison[0][threadIdx.x] = 0u;
        const int rows = count * p.heads;              // of this sequence
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(&sh.q_full);
        asm volatile("bar.sync 1, 256;" ::: "memory");  // parents
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
        const uint32_t s_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * 64;
        const uint32_t o_half = o_tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * (C::HDV / 2);
        float m = -INFINITY, mu = 0.f, l = 0.f;
        // A warp whose wait gave up keeps to the barriers of the others and does nothing else.
        bool ok = true;
        int nmasked = 0;
        for (int t = 0; t < nt; ++t) {
            const int k0 = key0 + t * kTile;
            const bool masked = masked_tile(t);
            ok = ok && mbar_wait_warp(&sh.s_full[t & 1], (t >> 1) & 1, p.err, 707);
            tc_fence_after();
            uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
            if (masked) {
                vis[0] = visible(k0, 2 * half);
                vis[1] = visible(k0, 2 * half + 1);
            }
            float tm = -INFINITY;
            if (warp_live && ok) {
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t x[32];
                    tmem_ld_32x32b_x32(s_tmem + (t & 1) * 128 + c * 32, x);
                    tmem_ld_wait(x);
                    if (masked) {
                        const uint32_t v = c ? vis[1] : vis[0];
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = v >> i & 1u ? x[i] : 0xff800000u;
                    }
                    float m4[4] = {tm, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(x[i]));
                    tm = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                }
                sh.mx[t & 1][half][r] = tm;
            }
            asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
            if (warp_live && ok) {
                tm = fmaxf(tm, sh.mx[t & 1][half ^ 1][r]);
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
                if (t > 0 && __any_sync(0xffffffffu, grow_m)) {
                    ok = mbar_wait_warp(&sh.o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, p.err, 709);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < C::HDV / 2; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_half + c, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_st_32x32b_x32(o_half + c, o);
                    }
                }
                // P in bf16 (the product's operand type; at most 1 part in 256 per weight) over the
                // scores just read; l sums the rounded weights, so they are weights of sum 1.
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t x[32], w[16];
                    tmem_ld_32x32b_x32(s_tmem + (t & 1) * 128 + c * 32, x);
                    tmem_ld_wait(x);
                    if (masked) {
                        const uint32_t v = c ? vis[1] : vis[0];
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = v >> i & 1u ? x[i] : 0xff800000u;
                    }
                    float l0 = 0.f, l1 = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float a = ex2(fmaf(__uint_as_float(x[2 * i]), kLog2e, -mu));
                        const float b = ex2(fmaf(__uint_as_float(x[2 * i + 1]), kLog2e, -mu));
                        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(b), "f"(a));
                        l0 += __uint_as_float(w[i] << 16);
                        l1 += __uint_as_float(w[i] & 0xffff0000u);
                    }
                    tmem_st_32x32b_x16(s_tmem + (t & 1) * 128 + c * 16, w);
                    l += l0 + l1;
                }
                tmem_st_wait();
            }
            if (masked) {
                // What no row sees must not reach the product: 0 * NaN.  Thread = key and half of the
                // columns: rows behind base + count become 0; values that are not finite become 0 and
                // are remembered.
                const int key = threadIdx.x & 127, vrow = key % C::VKEYS, g = v_granule(t) + key / C::VKEYS;
                uint32_t* poison = sh.poison[nmasked % 3];
                if (threadIdx.x < 4) sh.poison[(nmasked + 1) % 3][threadIdx.x] = 0u;  // last read two masked tiles ago
                ok = ok && mbar_wait_warp(&sh.v_full, nmasked & 1, p.err, 712);
                ok = ok && mbar_wait_warp(&sh.full[g % C::SLOTS], (g / C::SLOTS) & 1, p.err, 713);  // of this phase now
                ++nmasked;
                if (ok) {
                    uint8_t* vr = ring + (g % C::SLOTS) * C::SLOT + vrow * 128;
                    const bool outside = k0 + key >= ts.base + count;
                    bool bad = false;
                    auto at = [&](int i) {
                        const int c = half * (C::HDV / 16) + i;
                        return reinterpret_cast<uint4*>(vr + (c >> 3) * C::VBOX + (((c & 7) ^ (vrow & 7)) << 4));
                    };
                    // an exponent of all ones carries into the bit above it
                    auto odd = [](uint32_t e) { return ((e & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
                    uint32_t any = 0u;
#pragma unroll 8
                    for (int i = 0; i < C::HDV / 16; ++i) {
                        const uint4 w = *at(i);
                        any |= odd(w.x) | odd(w.y) | odd(w.z) | odd(w.w);
                    }
                    if (outside || any) {
#pragma unroll 1
                        for (int i = 0; i < C::HDV / 16; ++i) {
                            const uint4 w = *at(i);
                            auto clean = [&](uint32_t e) {
                                const uint32_t o = odd(e);
                                return outside ? 0u : e & ((o & 0x8000u ? 0u : 0xffffu) | (o & 0x80000000u ? 0u : 0xffff0000u));
                            };
                            *at(i) = make_uint4(clean(w.x), clean(w.y), clean(w.z), clean(w.w));
                        }
                        bad = !outside;
                    }
                    if (bad) atomicOr(&poison[key >> 5], 1u << lane);
                    fence_proxy_async_smem();
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 1
                for (int w = 0; w < 4; ++w)
                    if (poison[w] & visible(k0, w)) l = __int_as_float(0x7fffffff);  // sees a V row that is not finite
            }
            tc_fence_before();
            mbar_arrive(&sh.p_ready[t & 1]);
        }
        // ---- O of the row ----
        if (nt > 0) {
            // mx[nt & 1] was last read before the barrier of tile nt - 1
            sh.mx[nt & 1][half][r] = l;
            asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
            l += sh.mx[nt & 1][half ^ 1][r];
            ok = ok && mbar_wait_warp(&sh.o_done[(nt - 1) & 1], ((nt - 1) >> 1) & 1, p.err, 710);
        }
        tc_fence_after();
        // Rows leave through shared memory (Q and the ring have been read for the last time): written
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
                if (ok) {
#pragma unroll 1
                    for (int c = 0; c < C::HDV / 2; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_half + c, o);
                        tmem_ld_wait(o);
                        const int col = half * (C::HDV / 2) + c;
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
                    if (!whole && live && half == 0)
                        p.part_ml[(split * C::NV + vhalf) * nrows + grow + f] = make_float2(mu, l);
                }
                asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
                if (ok) {
                    const int row0 = (warp & 3) * 32;  // the pair's 32 rows
                    uint8_t* const to = (whole ? reinterpret_cast<uint8_t*>(p.out) : reinterpret_cast<uint8_t*>(p.part_o)) +
                                        ((whole ? 0 : split * nrows) + grow + f0) * (HD * (whole ? 2 : 4)) + vhalf * rowb;
#pragma unroll 8
                    for (int u = half * 32 + lane; u < 32 * chunks; u += 64) {
                        const int rr = row0 + u / chunks, ch = u % chunks;
                        if (f0 + rr < rows)
                            *reinterpret_cast<uint4*>(to + (size_t)rr * (HD * (whole ? 2 : 4)) + ch * 16) =
                                *reinterpret_cast<const uint4*>(smem + rr * rowb + (((ch & ~7) | ((ch ^ rr) & 7)) << 4));
                    }
                }
            };
            if (p.nsplit == 1) stage(std::true_type{});
            else stage(std::false_type{});
        } else if (nt == 0 && p.nsplit > 1 && live && half == 0) {
            const size_t nrows = (size_t)p.nseq * n * p.heads;
            p.part_ml[(split * C::NV + vhalf) * nrows + grow + f] = make_float2(0.f, 0.f);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the splits of a row: out = sum_i 2^(mu_i - mu) O_i / sum_i 2^(mu_i - mu) l_i.  One CTA per
// row and HDV columns, a thread per two columns.  The splits' (mu, l) are read at once, then every
// split's columns independently: two round trips.  A split that saw none of the row's keys has
// l = 0 and is left out (its O was not written).
constexpr int kMaxSplits = 160;
template <int HD>
__global__ void __launch_bounds__(TreeCfg<HD>::HDV / 2) tree_combine_kernel(const TreeAttnParams p) {
    using C = TreeCfg<HD>;
    constexpr int T = C::HDV / 2;
    __shared__ float2 ml[kMaxSplits];
    pdl_trigger();
    const size_t row = blockIdx.x;
    const int vhalf = blockIdx.y;
    const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
    const int s = (int)(row / (p.tree.nodes * p.heads)), node = (int)(row / p.heads) - s * p.tree.nodes;
    pdl_wait();
    for (int i = threadIdx.x; i < p.nsplit; i += T) ml[i] = p.part_ml[(i * C::NV + vhalf) * nrows + row];
    const int count = tree_count(p.tree, s, nullptr);
    const bool used = node < count && tree_seq_fits(p, tree_seq(p, s), count);
    __syncthreads();
    if (!used) return;
    float mu = -INFINITY;
    for (int i = 0; i < p.nsplit; ++i) mu = ml[i].y != 0.f ? fmaxf(mu, ml[i].x) : mu;
    const float2* o = reinterpret_cast<const float2*>(p.part_o + row * HD + vhalf * C::HDV) + threadIdx.x;
    float l = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll 8
    for (int i = 0; i < p.nsplit; ++i) {
        const bool use = ml[i].y != 0.f;
        const float f = use ? ex2(ml[i].x - mu) : 0.f;
        const float2 v = use ? __ldg(o + i * nrows * (HD / 2)) : make_float2(0.f, 0.f);
        l += f * ml[i].y;
        a0 += f * v.x;
        a1 += f * v.y;
    }
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(a1 / l), "f"(a0 / l));
    reinterpret_cast<uint32_t*>(p.out + row * HD + vhalf * C::HDV)[threadIdx.x] = w;
}

template <int HD>
g4_status launch_tree_attention(g4_ctx* ctx, const g4_kv* kv, TreeAttnParams p) {
    using C = TreeCfg<HD>;
    const int mtiles = (p.tree.nodes * p.heads + kRowsPerCta - 1) / kRowsPerCta;
    const int longest = (p.sliding && p.window < p.seq_stride ? p.window : p.seq_stride) + p.tree.nodes;
    const int ntiles = (longest + kTile - 1) / kTile;
    const long long ctas = (long long)mtiles * C::NV * p.nseq;
    // Split the keys while that adds CTAs to SMs without one, at three tiles or more per split: a
    // split costs its CTA's start and drain (about three tiles' time) and the join.  One sequence
    // of 8 nodes over 4096 keys: 15.0 us at two tiles, 15.3 at three, 19.1 at six; 64 sequences
    // with a window of 512 (five tiles): 28.6 us in two splits, 19.9 whole.
    int nsplit = (int)std::max<long long>(1, std::min<long long>({ctx->num_sms / ctas, ntiles / 3, kMaxSplits}));
    p.nsplit = nsplit;
    if (nsplit > 1) {
        const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
        const size_t ob = nsplit * nrows * HD * sizeof(float);
        g4_status st = g4::ensure_workspace(ctx, ob + (size_t)nsplit * C::NV * nrows * sizeof(float2));
        if (st) return st;
        p.part_o = static_cast<float*>(ctx->ws);
        p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(ctx->ws) + ob);
    }
    static std::atomic<uint64_t> attr_set{0};
    if (!(attr_set.load() & (1ull << ctx->device))) {
        G4_CHECK_CUDA(cudaFuncSetAttribute(tree_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set.fetch_or(1ull << ctx->device);
    }
    p.krows = kv->tree_krows;
    p.vrows = kv->tree_vrows;
    g4_status st = g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<HD>, dim3(mtiles * C::NV, p.nseq, nsplit),
                              dim3(kThreads), C::SMEM, 1, kv->tree_kmap, kv->tree_vmap, p);
    if (st || nsplit == 1) return st;
    const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
    // The join is set up while the attention runs, and waits for it (griddepcontrol).
    const bool pdl = ctx->pdl;
    ctx->pdl = true;
    st = g4::launch(ctx, "tree_combine_kernel", tree_combine_kernel<HD>,
                      dim3((unsigned)nrows, C::NV), dim3(C::HDV / 2), 0, 1, p);
    ctx->pdl = pdl;
    return st;
}

template <int HD>
g4_status tree_maps(g4_kv* kv) {
    using C = TreeCfg<HD>;
    const int contiguous = kv->ring ? kv->mirror : kTile;
    kv->tree_krows = std::min(kTile, contiguous);
    kv->tree_vrows = std::min(C::VKEYS, contiguous);
    const uint64_t dims[3] = {64, (uint64_t)kv->rows_total, HD / 64}, pitch[2] = {HD * 2, 128};
    const uint32_t kbox[3] = {64, (uint32_t)kv->tree_krows, kv->tree_krows == kTile ? (uint32_t)C::KBOXES : 1u};
    const uint32_t vbox[3] = {64, (uint32_t)kv->tree_vrows, kv->tree_vrows == C::VKEYS ? C::HDV / 64u : 1u};
    g4_status st = g4::encode_tensor_map_3d(&kv->tree_kmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv->k, dims, pitch, kbox,
                                            CU_TENSOR_MAP_SWIZZLE_128B);
    if (st) return st;
    return g4::encode_tensor_map_3d(&kv->tree_vmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv->v, dims, pitch, vbox,
                                    CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

namespace g4 {

g4_status make_tree_maps(g4_kv* kv) {
    switch (kv->hd) {
        case 64: return tree_maps<64>(kv);
        case 128: return tree_maps<128>(kv);
        case 256: return tree_maps<256>(kv);
        default: return tree_maps<512>(kv);
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
    const TreeAttnParams p{static_cast<const uint16_t*>(q_bf16), static_cast<uint16_t*>(out_bf16), nullptr, nullptr,
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
