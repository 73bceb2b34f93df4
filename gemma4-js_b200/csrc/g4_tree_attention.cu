// g4_tree_attention.cu -- attention of a tree of drafted tokens over each sequence's cached
// keys and the node's own ancestors.
//
// Row (s, i) of q sits at position base + depth(i) and sees the cached keys j < base (of the
// last `window` positions when sliding) and the drafted rows of its ancestors and itself.
#include "g4_attention.cuh"
#include "g4_common.cuh"
#include "g4_tree.cuh"

namespace {

using namespace g4dev;

// Round to nearest even with NaN kept: the integer rule of f32_to_bf16_bits carries the NaN that
// arithmetic gives (all mantissa bits set) into -0.
__device__ __forceinline__ uint16_t out_bits(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

struct TreeAttnParams {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    uint32_t* err;
    g4_tree tree;
    const int32_t* seq_pos;
    int seq_base, pos0, seq_stride, heads, sliding, window, ring, limit;
};

// One warp per (row, head); lane l holds columns l, l + 32, ...
template <int HD>
__global__ void __launch_bounds__(256) tree_attention_kernel(TreeAttnParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int E = HD / 32;
    const int h = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = p.tree.nodes, node = blockIdx.x, s = blockIdx.y;
    const int count = tree_count(p.tree, s, p.err);
    if (node >= count) return;
    const WarpTree wt = load_warp_tree(p.tree, s, count, p.err);
    const int seq = p.seq_base + s, base = p.seq_pos[seq] + p.pos0;
    if (base < 0 || (long long)base + count > p.limit) {
        if (threadIdx.x == 0) raise_error(p.err, G4_DEVERR_BAD_INDEX);
        return;
    }
    const int depth = warp_tree_depth(wt, node);
    const size_t row = ((size_t)s * n + node) * p.heads + h;
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = bf16_bits_to_f32(p.q[row * HD + e * 32 + lane]);
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    auto visit = [&](int pos) {
        const size_t at = ((size_t)seq * p.seq_stride + (p.ring ? pos % p.ring : pos)) * HD + lane;
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) d += q[e] * bf16_bits_to_f32(p.k[at + e * 32]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
        const float mn = fmaxf(m, d), a = expf(m - mn), w = expf(d - mn);
        l = l * a + w;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * bf16_bits_to_f32(p.v[at + e * 32]);
    };
    for (int j = p.sliding ? max(0, base + depth - p.window + 1) : 0; j < base; ++j) visit(j);
    int up = 0;
    for (int a = node; a >= 0 && (!p.sliding || up < p.window); a = wt.parent(a), ++up) visit(base + a);
#pragma unroll
    for (int e = 0; e < E; ++e) p.out[row * HD + e * 32 + lane] = out_bits(o[e] / l);
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
    const TreeAttnParams p{static_cast<const uint16_t*>(q_bf16), kv->k, kv->v, static_cast<uint16_t*>(out_bf16),
                           ctx->d_err, *tree, map->seq_pos, map->seq_base, map->pos0, seq_stride, heads,
                           sliding ? 1 : 0, window, kv->ring, kv->ring ? kv->capacity : seq_stride};
    const dim3 grid(tree->nodes, nseq), block(heads * 32);
    switch (hd) {
        case 64: return g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<64>, grid, block, 0, 1, p);
        case 128: return g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<128>, grid, block, 0, 1, p);
        case 256: return g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<256>, grid, block, 0, 1, p);
        case 512: return g4::launch(ctx, "tree_attention_kernel", tree_attention_kernel<512>, grid, block, 0, 1, p);
        default: return g4::set_error(G4_ERR_UNSUPPORTED, "g4_attention_tree: head dim %d (64/128/256/512 supported)", hd);
    }
}
