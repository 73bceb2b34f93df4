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

#include "g4_attention.cuh"
#include "g4_common.cuh"
#include "g4_tcgen05.cuh"
#include "g4_tree.cuh"

namespace {

using namespace g4dev;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 128;        // keys per tile = MMA N of the scores
constexpr int kRowsPerCta = 128;  // MMA M
constexpr int kSoftmaxThreads = 128;
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
    static constexpr int BOXROWS = HD == 64 ? 128 : 16384 / HD;  // rows of a TMA box
    static constexpr int SLOTS = HD == 64 ? 8 : (229376 - QBYTES) / SLOT;
    static constexpr int SMEM = QBYTES + SLOTS * SLOT + 2048;  // + alignment, barriers, parents
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
};

struct TreeShared {
    uint64_t full[8], empty[8];
    uint64_t q_full, s_full[2], p_ready[2], o_done[2], v_full, drained;
    uint32_t tmem;
    uint32_t poison[3][4];  // keys of a masked tile whose V row is not finite (three tiles in turn)
    int parents[G4_TREE_MAX_NODES];
};

__device__ __forceinline__ float ex2(float x) {  // 2^x to 2^-22, 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// MN-major operand in 128-byte swizzle: 64-element chunks `chunk` bytes apart, 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t chunk) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
constexpr uint32_t kTransposeB = 1u << 16;

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
    const TreeSeq ts = tree_seq(p, s);
    // This split's tiles; tile t covers keys lo + (t0 + t) * 128 ...
    const int t0 = (int)((long long)split * ts.ntiles / p.nsplit);
    int nt = (int)((long long)(split + 1) * ts.ntiles / p.nsplit) - t0;
    const int key0 = ts.lo + t0 * kTile;
    if (ts.base < 0 || ts.base > p.limit) nt = 0;
    if (!p.history_ready) {  // no used row among this CTA's
        const int c = tree_count(p.tree, s, nullptr);
        if (mtile * kRowsPerCta >= c * p.heads || !tree_seq_fits(p, ts, c)) nt = 0;
    }

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
    if (warp == 5) tmem_alloc(&sh.tmem, 512);
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

    if (warp == 4) {
        // ------------------------------------------------ TMA producer --
        if (lane == 0 && nt > 0) {
            prefetch_tensor_map(&kmap);
            prefetch_tensor_map(&vmap);
            bool ok = true, waited = !p.history_ready;
            int g = 0;
            const int seq = p.seq_base + s;
            auto load = [&](const CUtensorMap* map, int slot, uint32_t off, int x, int key) {
                const int row = seq * p.seq_stride + (p.ring ? key % p.ring : key);
                tma_load_2d(ring + slot * C::SLOT + off, map, &sh.full[slot], x, row);
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
#pragma unroll
                        for (int b = 0; b < C::KBOXES; ++b)
#pragma unroll
                            for (int r = 0; r < kTile; r += C::BOXROWS)
                                load(&kmap, slot, b * 16384 + r * 128, (a * C::KBOXES + b) * 64, k0 + r);
                    }
                }
                if (t >= 0) {
                    const int k0 = key0 + t * kTile;
                    for (int a = 0; a < C::VGRAN && ok; ++a, ++g) {
                        const int slot = claim();
                        if (!ok) break;
#pragma unroll
                        for (int b = 0; b < C::HDV / 64; ++b)
#pragma unroll
                            for (int r = 0; r < C::VKEYS; r += C::BOXROWS)
                                load(&vmap, slot, b * C::VBOX + r * 128, vhalf * 256 + b * 64, k0 + a * C::VKEYS + r);
                    }
                }
            }
            // Do not leave while copies may still be landing.
            for (int i = g > C::SLOTS ? g - C::SLOTS : 0; i < g; ++i)
                mbar_wait(&sh.full[i % C::SLOTS], (i / C::SLOTS) & 1, p.err, 702);
        }
    } else if (warp == 5) {
        // --------------------------------------------------- MMA issuer --
        if (lane == 0 && nt > 0) {
            constexpr uint32_t qk_idesc = mma_idesc_bf16(128, kTile);
            constexpr uint32_t pv_idesc = mma_idesc_bf16(128, C::HDV) | kTransposeB;
            const uint32_t qa = smem_u32(qsm), ra = smem_u32(ring);
            bool ok = mbar_wait(&sh.q_full, 0, p.err, 703);
            auto scores = [&](int t) {
                for (int a = 0; a < C::KGRAN && ok; ++a) {
                    const int g = k_granule(t) + a, slot = g % C::SLOTS;
                    ok = mbar_wait(&sh.full[slot], (g / C::SLOTS) & 1, p.err, 704);
                    if (!ok) return;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < C::KBOXES * 4; ++i)
                        tc_mma_ss(tmem + (t & 1) * 128, sw128_desc(qa + (a * C::KBOXES + i / 4) * 16384 + (i % 4) * 32),
                                  sw128_desc(ra + slot * C::SLOT + (i / 4) * 16384 + (i % 4) * 32), qk_idesc,
                                  (a | i) ? 1u : 0u);
                    tc_commit(&sh.empty[slot]);
                }
                tc_commit(&sh.s_full[t & 1]);
            };
            if (ok) scores(0);
            for (int t = 0; t < nt && ok; ++t) {
                if (t + 1 < nt) scores(t + 1);
                if (ok && masked_tile(t)) {  // hand V to the softmax threads (only this thread can follow the ring)
                    for (int a = 0; a < C::VGRAN && ok; ++a) {
                        const int g = v_granule(t) + a;
                        ok = mbar_wait(&sh.full[g % C::SLOTS], (g / C::SLOTS) & 1, p.err, 708);
                    }
                    if (ok) mbar_arrive(&sh.v_full);
                }
                ok = ok && mbar_wait(&sh.p_ready[t & 1], (t >> 1) & 1, p.err, 705);
                for (int a = 0; a < C::VGRAN && ok; ++a) {
                    const int g = v_granule(t) + a, slot = g % C::SLOTS;
                    ok = mbar_wait(&sh.full[slot], (g / C::SLOTS) & 1, p.err, 706);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < C::VKEYS / 16; ++i)
                        tc_mma_ts(o_tmem, tmem + (t & 1) * 128 + (a * (C::VKEYS / 16) + i) * 8,
                                  mn_desc(ra + slot * C::SLOT + i * 2048, C::VBOX), pv_idesc, (t | a | i) ? 1u : 0u);
                    tc_commit(&sh.empty[slot]);
                }
                if (ok) tc_commit(&sh.o_done[t & 1]);
            }
            // Do not free the tensor memory while products may still be running (after a failed wait).
            tc_commit(&sh.drained);
            mbar_wait(&sh.drained, 0, p.err, 711);
        }
    } else {
        // ------------------------------ softmax: thread = one query row --
        if (p.history_ready) pdl_wait();
        int count = tree_count(p.tree, s, p.err);
        if (!tree_seq_fits(p, ts, count)) {
            if (threadIdx.x == 0 && blockIdx.x == 0 && split == 0) raise_error(p.err, G4_DEVERR_BAD_INDEX);
            count = 0;
        }
        if (threadIdx.x < n) sh.parents[threadIdx.x] = threadIdx.x < count ? tree_parent(p.tree, s, threadIdx.x, p.err) : -1;
        if (threadIdx.x < 4) sh.poison[0][threadIdx.x] = 0u;
        const int rows = count * p.heads;              // of this sequence
        const int f0 = mtile * kRowsPerCta, f = f0 + threadIdx.x;
        const size_t grow = (size_t)s * n * p.heads;   // the sequence's first row of q and out
        if (nt > 0) {
            // Q into the swizzled operand layout; rows that are not used are zero.
            constexpr int CH = HD / 8, PER = CH;       // 16-byte chunks per row = per thread
            const uint4* qg = reinterpret_cast<const uint4*>(p.q + (grow + f0) * HD);
            for (int i0 = 0; i0 < PER; i0 += 8) {
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int u = (i0 + i) * kSoftmaxThreads + threadIdx.x;
                    v[i] = f0 + u / CH < rows ? qg[u] : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int u = (i0 + i) * kSoftmaxThreads + threadIdx.x, r = u / CH, c = u % CH;
                    *reinterpret_cast<uint4*>(qsm + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[i];
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&sh.q_full);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");  // parents
        const bool live = f < rows;
        const bool warp_live = f - lane < rows;
        // The row's visible drafted rows (bit = node) and first visible cached key.
        unsigned long long seen = 0ull;
        int first = 0x7fffffff;
        if (live) {
            const int node = f / p.heads;
            int up = 0;
            for (int a = node; a >= 0; a = sh.parents[a], ++up)
                if (!p.sliding || up < p.window) seen |= 1ull << a;
            first = p.sliding ? ts.base + up - p.window : 0;  // up = depth + 1
        }
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        float m = -INFINITY, mu = 0.f, l = 0.f;
        // A warp whose wait gave up keeps to the barriers of the others and does nothing else.
        bool ok = true;
        int nmasked = 0;
        for (int t = 0; t < nt; ++t) {
            const int k0 = key0 + t * kTile;
            const bool masked = masked_tile(t);
            ok = ok && mbar_wait_warp(&sh.s_full[t & 1], (t >> 1) & 1, p.err, 707);
            tc_fence_after();
            uint32_t vis[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
            if (masked) {
                // What no row sees must not reach the product: 0 * NaN.  Thread = key: rows outside
                // [lo, base + count) become 0; values that are not finite become 0 and are remembered.
                const int key = k0 + threadIdx.x, vrow = threadIdx.x % C::VKEYS;
                const int g = v_granule(t) + threadIdx.x / C::VKEYS;
                uint32_t* poison = sh.poison[nmasked % 3];
                if (threadIdx.x < 4) sh.poison[(nmasked + 1) % 3][threadIdx.x] = 0u;  // last read two masked tiles ago
                ok = ok && mbar_wait_warp(&sh.v_full, nmasked & 1, p.err, 712);
                ok = ok && mbar_wait_warp(&sh.full[g % C::SLOTS], (g / C::SLOTS) & 1, p.err, 713);  // of this phase now
                ++nmasked;
                if (ok) {
                    uint8_t* vr = ring + (g % C::SLOTS) * C::SLOT + vrow * 128;
                    const bool outside = key >= ts.base + count;
                    bool bad = false;
#pragma unroll 4
                    for (int c = 0; c < C::HDV / 8; ++c) {
                        uint4* at = reinterpret_cast<uint4*>(vr + (c >> 3) * C::VBOX + (((c & 7) ^ (vrow & 7)) << 4));
                        uint4 w = *at;
                        uint32_t* e = reinterpret_cast<uint32_t*>(&w);
                        bool fix = outside;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool b0 = (e[i] & 0x7f80u) == 0x7f80u, b1 = (e[i] & 0x7f800000u) == 0x7f800000u;
                            if (outside) e[i] = 0u;
                            else e[i] &= (b0 ? 0xffff0000u : 0xffffffffu) & (b1 ? 0x0000ffffu : 0xffffffffu);
                            bad = bad || b0 || b1;
                            fix = fix || b0 || b1;
                        }
                        if (fix) *at = w;
                    }
                    if (bad && !outside) atomicOr(&poison[threadIdx.x >> 5], 1u << lane);
                    fence_proxy_async_smem();
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int d = ts.base - k0;  // column of node 0
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int sft = 32 * w - d;  // drafted bits start at node sft
                    const unsigned long long bits = sft >= 64 || sft <= -32 ? 0ull : sft >= 0 ? seen >> sft : seen << -sft;
                    vis[w] = live ? range_word(first - k0, d, w) | (uint32_t)bits : 0u;
                    if (vis[w] & poison[w]) l = __int_as_float(0x7fffffff);  // sees a V row that is not finite
                }
            }
            if (warp_live && ok) {
                float x[kTile];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    tmem_ld_32x32b_x32(tmem + lane_off + (t & 1) * 128 + c * 32, *reinterpret_cast<uint32_t(*)[32]>(x + c * 32));
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(x + c * 32));
                if (masked) {
#pragma unroll
                    for (int c = 0; c < kTile; ++c) x[c] = (vis[c >> 5] >> (c & 31)) & 1u ? x[c] : -INFINITY;
                }
                float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int c = 4; c < kTile; ++c) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
                const float tm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
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
                    for (int c = 0; c < C::HDV; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_tmem + lane_off + c, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_st_32x32b_x32(o_tmem + lane_off + c, o);
                    }
                }
                // P in bf16 (the product's operand type; at most 1 part in 256 per weight) over the
                // scores just read; l sums the rounded weights, so they are weights of sum 1.
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float a = ex2(fmaf(x[h * 64 + 2 * i], kLog2e, -mu));
                        const float b = ex2(fmaf(x[h * 64 + 2 * i + 1], kLog2e, -mu));
                        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(b), "f"(a));
                        l0 += __uint_as_float(w[i] << 16);
                        l1 += __uint_as_float(w[i] & 0xffff0000u);
                    }
                    tmem_st_32x32b_x32(tmem + lane_off + (t & 1) * 128 + h * 32, w);
                }
                l += l0 + l1;
                tmem_st_wait();
            }
            tc_fence_before();
            mbar_arrive(&sh.p_ready[t & 1]);
        }
        // ---- O of the row ----
        if (nt > 0 && ok) ok = mbar_wait_warp(&sh.o_done[(nt - 1) & 1], ((nt - 1) >> 1) & 1, p.err, 710);
        tc_fence_after();
        if (warp_live && ok) {
            const float inv = 1.f / l;
            const size_t row = grow + f;
            const size_t nrows = (size_t)p.nseq * n * p.heads;
            if (p.nsplit > 1 && live) p.part_ml[(split * C::NV + vhalf) * nrows + row] = make_float2(mu, nt > 0 ? l : 0.f);
            if (nt > 0) {
#pragma unroll 1
                for (int c = 0; c < C::HDV; c += 32) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_tmem + lane_off + c, o);
                    tmem_ld_wait(o);
                    if (!live) continue;
                    if (p.nsplit == 1) {
                        uint4* to = reinterpret_cast<uint4*>(p.out + row * HD + vhalf * 256 + c);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
                                    : "=r"(w[k])
                                    : "f"(__uint_as_float(o[8 * i + 2 * k + 1]) * inv), "f"(__uint_as_float(o[8 * i + 2 * k]) * inv));
                            to[i] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
                        uint4* to = reinterpret_cast<uint4*>(p.part_o + (split * nrows + row) * HD + vhalf * 256 + c);
#pragma unroll
                        for (int i = 0; i < 8; ++i) to[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the splits of a row: out = sum_i 2^(mu_i - mu) O_i / sum_i 2^(mu_i - mu) l_i, one warp per
// row and HDV columns.  A split that saw none of the row's keys has l = 0 and is left out (its O
// is not read).
constexpr int kCombineWarps = 4;
template <int HD>
__global__ void __launch_bounds__(kCombineWarps * 32) tree_combine_kernel(const TreeAttnParams p) {
    using C = TreeCfg<HD>;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, vhalf = blockIdx.y;
    const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
    const size_t row = (size_t)blockIdx.x * kCombineWarps + (threadIdx.x >> 5);
    if (row >= nrows) return;
    const int s = (int)(row / (p.tree.nodes * p.heads)), node = (int)(row / p.heads) - s * p.tree.nodes;
    const int count = tree_count(p.tree, s, nullptr);
    if (node >= count || !tree_seq_fits(p, tree_seq(p, s), count)) return;
    const float2* ml = p.part_ml + vhalf * nrows + row;
    float mu = -INFINITY;
    for (int i = lane; i < p.nsplit; i += 32) {
        const float2 v = ml[i * (C::NV * nrows)];
        if (v.y != 0.f) mu = fmaxf(mu, v.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mu = fmaxf(mu, __shfl_xor_sync(0xffffffffu, mu, o));
    constexpr int E = C::HDV / 64;
    float acc[2 * E], l = 0.f;
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < p.nsplit; ++i) {
        const float2 v = ml[i * (C::NV * nrows)];
        const bool use = v.y != 0.f;
        const float f = use ? ex2(v.x - mu) : 0.f;
        l += f * v.y;
        const float2* o = reinterpret_cast<const float2*>(p.part_o + (i * nrows + row) * HD + vhalf * C::HDV);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 w = use ? o[e * 32 + lane] : make_float2(0.f, 0.f);
            acc[2 * e] += f * w.x;
            acc[2 * e + 1] += f * w.y;
        }
    }
    const float inv = 1.f / l;
    uint32_t* out = reinterpret_cast<uint32_t*>(p.out + row * HD + vhalf * C::HDV);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        uint32_t w;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(acc[2 * e + 1] * inv), "f"(acc[2 * e] * inv));
        out[e * 32 + lane] = w;
    }
}

template <int HD>
g4_status launch_tree_attention(g4_ctx* ctx, const g4_kv* kv, TreeAttnParams p) {
    using C = TreeCfg<HD>;
    const int mtiles = (p.tree.nodes * p.heads + kRowsPerCta - 1) / kRowsPerCta;
    const int longest = (p.sliding && p.window < p.seq_stride ? p.window : p.seq_stride) + p.tree.nodes;
    const int ntiles = (longest + kTile - 1) / kTile;
    const long long ctas = (long long)mtiles * C::NV * p.nseq;
    // Split the keys while that adds CTAs to SMs without one, at two tiles or more per split.
    int nsplit = (int)std::max<long long>(1, std::min<long long>(ctx->num_sms / ctas, ntiles / 2));
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
    const CUtensorMap& km = HD == 64 ? kv->kmap_narrow : kv->kmap;
    const CUtensorMap& vm = HD == 64 ? kv->vmap_narrow : kv->vmap;
    g4_status st = g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<HD>, dim3(mtiles * C::NV, p.nseq, nsplit),
                              dim3(kThreads), C::SMEM, 1, km, vm, p);
    if (st || nsplit == 1) return st;
    const size_t nrows = (size_t)p.nseq * p.tree.nodes * p.heads;
    return g4::launch(ctx, "tree_combine_kernel", tree_combine_kernel<HD>,
                      dim3((unsigned)((nrows + kCombineWarps - 1) / kCombineWarps), C::NV), dim3(kCombineWarps * 32), 0, 1, p);
}

}  // namespace

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
    if (kv->ctx->device != ctx->device)
        return g4::set_error(G4_ERR_INVALID, "g4_attention_tree: the cache is on device %d, the context on %d",
                             kv->ctx->device, ctx->device);
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
