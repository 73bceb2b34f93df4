// g4_kv_rows.cu -- whole K/V rows of the caches: accepting the path of a drafted tree, moving
// its rows together, and forking a sequence's rows into other sequences.
//
// A cache row is hd bf16 values (128 B .. 1 KiB), so everything here is 16-byte copies; one
// launch serves every layer's cache (their pointers travel as a kernel argument).
#include "g4_attention.cuh"
#include "g4_common.cuh"
#include "g4_tree.cuh"

namespace {

using namespace g4dev;

constexpr int kMaxCaches = 48;  // caches per launch (32 B each, of the 4 KiB of arguments)
constexpr int kMaxPairs = 128;  // fork pairs per launch

struct CacheRef {
    uint16_t *k, *v;
    int hd, stride;    // stride: rows per sequence
    int ring, mirror;  // ring caches: position p in slot p % ring, slots below mirror again at ring + slot
};
struct CacheTable {
    CacheRef c[kMaxCaches];
    int limit;     // positions run below this in every cache of the call (also those of other launches):
    int smallest;  // and its smallest ring: a sequence is moved in all caches or in none
};
__device__ __forceinline__ uint4* row_ptr(const CacheRef& c, int is_v, int seq, int slot) {
    return reinterpret_cast<uint4*>((is_v ? c.v : c.k) + ((size_t)seq * c.stride + slot) * c.hd);
}

// One warp per sequence: lane l holds nodes l and l + 32; a step of the walk is two ballots.
__global__ void __launch_bounds__(128) tree_accept_kernel(g4_tree tree, int nseq, const int32_t* __restrict__ tokens,
                                                          const int32_t* __restrict__ picks, int32_t* __restrict__ path,
                                                          int32_t* __restrict__ accepted, int32_t* __restrict__ next,
                                                          uint32_t* err) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, s = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (s >= nseq) return;
    const int n = tree.nodes;
    const int count = tree_count(tree, s, err);
    const WarpTree w = load_warp_tree(tree, s, count, err);
    const size_t row = (size_t)s * n;
    const bool in0 = lane < count, in1 = lane + 32 < count;
    const int tok0 = in0 ? tokens[row + lane] : 0, tok1 = in1 ? tokens[row + lane + 32] : 0;
    const int pick0 = in0 ? picks[row + lane] : 0, pick1 = in1 ? picks[row + lane + 32] : 0;
    int len = 0, cur = 0;
    int out0 = -1, out1 = -1;  // lane l keeps path entries l and l + 32
    int pick = 0;
    if (count > 0) {
        for (;;) {
            if (lane == (len & 31)) (len < 32 ? out0 : out1) = cur;
            ++len;
            pick = __shfl_sync(0xffffffffu, cur < 32 ? pick0 : pick1, cur & 31);
            const unsigned m0 = __ballot_sync(0xffffffffu, in0 && w.lo == cur && tok0 == pick);
            const unsigned m1 = __ballot_sync(0xffffffffu, in1 && w.hi == cur && tok1 == pick);
            if (!(m0 | m1)) break;
            cur = m0 ? __ffs(m0) - 1 : __ffs(m1) + 31;  // a child is above its parent: the walk ends
        }
    }
    if (lane < n) path[row + lane] = out0;
    if (lane + 32 < n) path[row + lane + 32] = out1;
    if (lane == 0) {
        accepted[s] = len;
        if (len > 0) next[s] = pick;
    }
}

// One warp per (sequence, cache, K or V).  Row j of the path moves down from base + path[j] to
// base + j (path[j] >= j, rising), so no row is read after a lower-numbered step wrote it:
// steps run in batches of 256 / (row in 16-byte units), every load of a batch before its first
// store.  A few rows of 0.5 KiB: bound by the latency of one batch (two dependent round trips:
// path and positions, then the rows).
__global__ void __launch_bounds__(128) kv_compact_kernel(const __grid_constant__ CacheTable table, int ncache,
                                                         const int32_t* __restrict__ seq_pos, int seq_base, int nseq,
                                                         int nodes, const int32_t* __restrict__ path,
                                                         const int32_t* __restrict__ accepted, uint32_t* err) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (unit >= (long long)nseq * ncache * 2) return;
    const int which = (int)(unit % (ncache * 2)), s = (int)(unit / (ncache * 2));
    const CacheRef c = table.c[which >> 1];
    const int seq = seq_base + s, base = seq_pos[seq];
    const int len = accepted[s];
    int p0 = lane < nodes ? path[(size_t)s * nodes + lane] : 0;
    int p1 = lane + 32 < nodes ? path[(size_t)s * nodes + lane + 32] : 0;
    // A rising path inside the tree, drafted rows inside the cache.
    const int up1 = __shfl_up_sync(0xffffffffu, p1, 1), up0 = __shfl_up_sync(0xffffffffu, p0, 1);
    const int last0 = __shfl_sync(0xffffffffu, p0, 31);
    bool ok = len >= 0 && len <= nodes && base >= 0;
    if (lane < len) ok = ok && p0 < nodes && p0 > (lane ? up0 : -1);
    if (lane + 32 < len) ok = ok && p1 < nodes && p1 > (lane ? up1 : last0);
    if (len > 0) {
        const int last = __shfl_sync(0xffffffffu, len <= 32 ? p0 : p1, (len - 1) & 31);
        const long long end = (long long)base + last;
        ok = ok && end < table.limit && nodes <= table.smallest;
    }
    if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) raise_error(err, G4_DEVERR_BAD_INDEX);
        return;
    }
    const int chunks = c.hd >> 3;      // 16-byte units of a row (8 .. 64)
    const int batch = 256 / chunks;    // rows per batch: 8 units per lane
    for (int j0 = 0; j0 < len; j0 += batch) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int j = j0 + (u * 32 + lane) / chunks, col = (u * 32 + lane) % chunks;
            const int a = __shfl_sync(0xffffffffu, p0, j & 31), b = __shfl_sync(0xffffffffu, p1, j & 31);
            const int from = j < 32 ? a : b;
            if (j < len && from != j) {
                const int pos = base + from;
                v[u] = row_ptr(c, which & 1, seq, c.ring ? pos % c.ring : pos)[col];
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int j = j0 + (u * 32 + lane) / chunks, col = (u * 32 + lane) % chunks;
            const int a = __shfl_sync(0xffffffffu, p0, j & 31), b = __shfl_sync(0xffffffffu, p1, j & 31);
            const int from = j < 32 ? a : b;
            if (j < len && from != j) {
                const int pos = base + j, slot = c.ring ? pos % c.ring : pos;
                row_ptr(c, which & 1, seq, slot)[col] = v[u];
                if (c.ring && slot < c.mirror) row_ptr(c, which & 1, seq, c.ring + slot)[col] = v[u];
            }
        }
        __syncwarp();
    }
}

struct ForkTable {
    int ngroups;
    int src[kMaxPairs];        // per group: the source sequence
    int first[kMaxPairs + 1];  // per group: its destinations are dst[first .. next group's first)
    int dst[kMaxPairs];
};

// CTA (chunk, cache and K/V, group): 16 KiB of the source's rows, read once into registers and
// stored to every destination of the group.  Bound by the stores' bandwidth; the grid covers a
// full cache because the length is known on the device only, and CTAs behind it leave at once.
constexpr int kForkUnits = 4;  // 16-byte units per thread
constexpr int kForkThreads = 256;
__global__ void __launch_bounds__(kForkThreads) kv_fork_kernel(const __grid_constant__ CacheTable table,
                                                               const __grid_constant__ ForkTable pairs,
                                                               int32_t* __restrict__ seq_pos, int set_pos,
                                                               uint32_t* err) {
    pdl_trigger();
    pdl_wait();
    const int which = blockIdx.y, grp = blockIdx.z;
    const CacheRef c = table.c[which >> 1];
    const int src = pairs.src[grp], d0 = pairs.first[grp], d1 = pairs.first[grp + 1];
    const int len = seq_pos[src];
    if (len < 0 || len > table.limit) {
        if (threadIdx.x == 0) raise_error(err, G4_DEVERR_BAD_INDEX);
        return;
    }
    if (set_pos && blockIdx.x == 0 && blockIdx.y == 0)
        for (int d = d0 + threadIdx.x; d < d1; d += blockDim.x) seq_pos[pairs.dst[d]] = len;
    const int chunks = c.hd >> 3;
    const long long units = (long long)c.stride * chunks;
    const int held = c.ring ? min(len, c.ring) : len;          // slots in use
    const int again = c.ring ? min(held, c.mirror) : 0;        // of them repeated after the ring
    const long long u0 = (long long)blockIdx.x * (kForkThreads * kForkUnits) + threadIdx.x;
    uint4 v[kForkUnits];
    bool in[kForkUnits];
    const uint4* from = row_ptr(c, which & 1, src, 0);
#pragma unroll
    for (int i = 0; i < kForkUnits; ++i) {
        const long long u = u0 + i * kForkThreads;
        const int row = (int)(u / chunks);
        in[i] = u < units && (row < held || (c.ring && row >= c.ring && row - c.ring < again));
        if (in[i]) v[i] = from[u];
    }
    for (int d = d0; d < d1; ++d) {
        uint4* to = row_ptr(c, which & 1, pairs.dst[d], 0);
#pragma unroll
        for (int i = 0; i < kForkUnits; ++i)
            if (in[i]) to[u0 + i * kForkThreads] = v[i];
    }
}

}  // namespace

namespace {

// The checks both row movers share: caches of this device, each once, holding sequences up to
// `last_seq`.
g4_status check_caches(const char* name, const g4_ctx* ctx, g4_kv* const* kvs, int nkv, int seq_stride, long long last_seq) {
    if (!kvs || nkv < 0) return g4::set_error(G4_ERR_INVALID, "%s: null caches", name);
    for (int i = 0; i < nkv; ++i) {
        const g4_kv* kv = kvs[i];
        if (!kv) return g4::set_error(G4_ERR_INVALID, "%s: null cache %d", name, i);
        if (kv->device != ctx->device)
            return g4::set_error(G4_ERR_INVALID, "%s: cache %d is on device %d, the context on %d", name, i,
                                 kv->device, ctx->device);
        for (int j = 0; j < i; ++j)
            if (kvs[j] == kv) return g4::set_error(G4_ERR_INVALID, "%s: caches %d and %d are the same", name, j, i);
        const int stride = kv->ring ? kv->seq_rows : seq_stride;
        if (stride < 1) return g4::set_error(G4_ERR_INVALID, "%s: seq_stride %d", name, seq_stride);
        if ((last_seq + 1) * stride > kv->rows_total)
            return g4::set_error(G4_ERR_RANGE, "%s: sequence %lld beyond cache %d (%d rows)", name, last_seq, i,
                                 kv->rows_total);
    }
    return G4_OK;
}

// Up to kMaxCaches caches from kvs[first].
int fill_table(CacheTable* t, g4_kv* const* kvs, int first, int nkv, int seq_stride) {
    t->limit = t->smallest = 0x7fffffff;
    for (int i = 0; i < nkv; ++i) {
        const int limit = kvs[i]->ring ? kvs[i]->capacity : seq_stride;
        t->limit = limit < t->limit ? limit : t->limit;
        if (kvs[i]->ring && kvs[i]->ring < t->smallest) t->smallest = kvs[i]->ring;
    }
    int n = 0;
    for (; n < kMaxCaches && first + n < nkv; ++n) {
        const g4_kv* kv = kvs[first + n];
        t->c[n] = kv->ring ? CacheRef{kv->k, kv->v, kv->hd, kv->seq_rows, kv->ring, kv->mirror}
                           : CacheRef{kv->k, kv->v, kv->hd, seq_stride, 0, 0};
    }
    return n;
}

}  // namespace

extern "C" {

g4_status g4_tree_accept(g4_ctx* ctx, const g4_tree* tree, int nseq, const int32_t* tokens, const int32_t* picks,
                         int32_t* path_out, int32_t* accepted_out, int32_t* next_out) {
    g4_status st = g4::check_tree("g4_tree_accept", tree);
    if (st) return st;
    if (nseq < 0 || !tokens || !picks || !path_out || !accepted_out || !next_out)
        return g4::set_error(G4_ERR_INVALID, "g4_tree_accept: bad arguments");
    st = g4::use_device(ctx);
    if (st || nseq == 0) return st;
    return g4::launch(ctx, "tree_accept_kernel", tree_accept_kernel, dim3((nseq + 3) / 4), dim3(128), 0, 1, *tree, nseq,
                      tokens, picks, path_out, accepted_out, next_out, ctx->d_err);
}

g4_status g4_kv_compact(g4_ctx* ctx, g4_kv* const* kvs, int nkv, int seq_stride, const int32_t* seq_pos, int seq_base,
                        int nseq, int nodes, const int32_t* path, const int32_t* accepted) {
    if (!seq_pos || !path || !accepted || nseq < 0 || seq_base < 0)
        return g4::set_error(G4_ERR_INVALID, "g4_kv_compact: bad arguments");
    if (nodes < 1 || nodes > G4_TREE_MAX_NODES)
        return g4::set_error(G4_ERR_UNSUPPORTED, "g4_kv_compact: %d nodes (1..%d supported)", nodes, G4_TREE_MAX_NODES);
    g4_status st = g4::use_device(ctx);
    if (st) return st;
    st = check_caches("g4_kv_compact", ctx, kvs, nkv, seq_stride, (long long)seq_base + nseq - 1);
    if (st || nseq == 0) return st;
    for (int first = 0; first < nkv; first += kMaxCaches) {
        CacheTable t;
        const int n = fill_table(&t, kvs, first, nkv, seq_stride);
        const long long warps = (long long)nseq * n * 2;
        st = g4::launch(ctx, "kv_compact_kernel", kv_compact_kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, 1, t,
                        n, seq_pos, seq_base, nseq, nodes, path, accepted, ctx->d_err);
        if (st) return st;
    }
    return G4_OK;
}

g4_status g4_kv_fork(g4_ctx* ctx, g4_kv* const* kvs, int nkv, int seq_stride, int32_t* seq_pos, const int32_t* src,
                     const int32_t* dst, int n) {
    if (!seq_pos || n < 0 || (n > 0 && (!src || !dst))) return g4::set_error(G4_ERR_INVALID, "g4_kv_fork: bad arguments");
    int last = -1;
    for (int i = 0; i < n; ++i) {
        if (src[i] < 0 || dst[i] < 0)
            return g4::set_error(G4_ERR_RANGE, "g4_kv_fork: sequence %d -> %d", src[i], dst[i]);
        for (int j = 0; j < n; ++j) {
            if (src[j] == dst[i])
                return g4::set_error(G4_ERR_INVALID, "g4_kv_fork: sequence %d is a source and a destination", dst[i]);
            if (j < i && dst[j] == dst[i])
                return g4::set_error(G4_ERR_INVALID, "g4_kv_fork: sequence %d is a destination twice", dst[i]);
        }
        last = src[i] > last ? src[i] : last;
        last = dst[i] > last ? dst[i] : last;
    }
    g4_status st = g4::use_device(ctx);
    if (st) return st;
    st = check_caches("g4_kv_fork", ctx, kvs, nkv, seq_stride, last);
    if (st || n == 0) return st;
    if (nkv == 0) return g4::set_error(G4_ERR_INVALID, "g4_kv_fork: no caches");
    for (int p0 = 0; p0 < n; p0 += kMaxPairs) {
        const int m = n - p0 < kMaxPairs ? n - p0 : kMaxPairs;
        ForkTable f{};
        int at = 0;
        for (int i = 0; i < m; ++i) {  // pairs of one source together
            bool seen = false;
            for (int g = 0; g < f.ngroups; ++g) seen = seen || f.src[g] == src[p0 + i];
            if (seen) continue;
            f.src[f.ngroups] = src[p0 + i];
            f.first[f.ngroups++] = at;
            for (int j = i; j < m; ++j)
                if (src[p0 + j] == src[p0 + i]) f.dst[at++] = dst[p0 + j];
        }
        f.first[f.ngroups] = at;
        for (int first = 0; first < nkv; first += kMaxCaches) {
            CacheTable t;
            const int nc = fill_table(&t, kvs, first, nkv, seq_stride);
            long long most = 1;  // CTAs for the largest cache of this launch
            for (int i = 0; i < nc; ++i) {
                const long long u = (long long)t.c[i].stride * (t.c[i].hd / 8);
                const long long b = (u + kForkThreads * kForkUnits - 1) / (kForkThreads * kForkUnits);
                most = b > most ? b : most;
            }
            st = g4::launch(ctx, "kv_fork_kernel", kv_fork_kernel, dim3((unsigned)most, nc * 2, f.ngroups),
                            dim3(kForkThreads), 0, 1, t, f, seq_pos, first + kMaxCaches >= nkv ? 1 : 0, ctx->d_err);
            if (st) return st;
        }
    }
    return G4_OK;
}

}  // extern "C"
