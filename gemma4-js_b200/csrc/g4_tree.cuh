// g4_tree.cuh -- trees of drafted tokens (the public struct is g4_tree in include/g4w4.h):
// checks shared by the entry points and the per-warp walk up a node's ancestors.
#pragma once
#include "g4_common.cuh"

namespace g4dev {

// Nodes of sequence s that are used: counts[s] clamped to [0, nodes].
__device__ __forceinline__ int tree_count(const g4_tree& t, int s, uint32_t* err) {
    if (!t.counts) return t.nodes;
    const int c = t.counts[s];
    if (c >= 0 && c <= t.nodes) return c;
    raise_error(err, G4_DEVERR_BAD_INDEX);
    return c < 0 ? 0 : t.nodes;
}

// parents[i] of sequence s; one outside [-1, i) counts as -1 and raises the error word.
__device__ __forceinline__ int tree_parent(const g4_tree& t, int s, int i, uint32_t* err) {
    const int p = t.parents[(size_t)s * t.parent_stride + i];
    if (p >= -1 && p < i) return p;
    raise_error(err, G4_DEVERR_BAD_INDEX);
    return -1;
}

// A warp's copy of one sequence's parents: lane l holds nodes l and l + 32 (one round trip for
// the whole tree; the walk itself is shuffles).
struct WarpTree {
    int lo, hi;
    __device__ __forceinline__ int parent(int i) const {  // i uniform across the warp
        return __shfl_sync(0xffffffffu, i < 32 ? lo : hi, i & 31);
    }
};
__device__ __forceinline__ WarpTree load_warp_tree(const g4_tree& t, int s, int count, uint32_t* err) {
    const int lane = threadIdx.x & 31;
    WarpTree w{-1, -1};
    if (lane < count) w.lo = tree_parent(t, s, lane, err);
    if (lane + 32 < count) w.hi = tree_parent(t, s, lane + 32, err);
    return w;
}
// The number of ancestors of node i (uniform across the warp).
__device__ __forceinline__ int warp_tree_depth(const WarpTree& w, int i) {
    int d = 0;
    for (int a = w.parent(i); a >= 0; a = w.parent(a)) ++d;  // parents are below their node: ends
    return d;
}

}  // namespace g4dev

namespace g4 {

inline g4_status check_tree(const char* name, const g4_tree* tree) {
    if (!tree || !tree->parents) return set_error(G4_ERR_INVALID, "%s: null tree", name);
    if (tree->nodes < 1 || tree->nodes > G4_TREE_MAX_NODES)
        return set_error(G4_ERR_UNSUPPORTED, "%s: %d nodes (1..%d supported)", name, tree->nodes, G4_TREE_MAX_NODES);
    if (tree->parent_stride != 0 && tree->parent_stride < tree->nodes)
        return set_error(G4_ERR_INVALID, "%s: parent_stride %d of %d nodes", name, tree->parent_stride, tree->nodes);
    return G4_OK;
}

// The rows map of a drafted tree: device positions, rows_per_seq = nodes, whole sequences.
inline g4_status check_tree_rows(const char* name, const g4_rows* map, const g4_tree* tree, int rows) {
    g4_status st = check_tree(name, tree);
    if (st) return st;
    if (!map || !map->seq_pos) return set_error(G4_ERR_INVALID, "%s: null rows map or positions", name);
    if (map->rows_per_seq != tree->nodes)
        return set_error(G4_ERR_INVALID, "%s: %d rows per sequence, trees of %d nodes", name, map->rows_per_seq,
                         tree->nodes);
    if (rows < 0 || rows % tree->nodes != 0)
        return set_error(G4_ERR_INVALID, "%s: %d rows (a multiple of %d nodes)", name, rows, tree->nodes);
    if (map->seq_base < 0) return set_error(G4_ERR_INVALID, "%s: seq_base %d", name, map->seq_base);
    return G4_OK;
}

}  // namespace g4
