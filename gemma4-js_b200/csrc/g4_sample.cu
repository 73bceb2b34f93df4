// g4_sample.cu -- one token per row of f32 logits: temperature, top-k, top-p, min-p and a given
// uniform number per row.
//
// With w_i = exp((l_i - m) / T), m the highest logit, the filters keep a prefix of the ranking
// by (l descending, index ascending), and the pick is an inverse cumulative sum in index order.
// Sums of up to 786432 weights decide which token a border falls on, so weights and sums are
// 64-bit (32-bit weights would move a border past a token in one row of some hundred).
//
// Three launches:
//   summary  reads the logits once (bound by HBM) and leaves, per group of 4 .. 512 consecutive
//            logits (at most 2048 groups a row), the highest key and, for rows whose settings
//            need the mass of the whole row, the group's weight relative to its highest logit.
//   finish   one CTA per row works from the groups: the k-th highest group maximum bounds the
//            k-th highest logit from below, so only the about k groups above it are read again
//            (64 of 2048 groups: 32 KB of a 1 MB row) and ranked.  Rows it cannot settle that
//            way (a nucleus of more than some thousand tokens, top-k above 1024, masses of ties)
//            go to a queue.
//   general  a cluster of CTAs holds a queued row in shared memory and narrows the threshold of
//            each filter by sums over the row; right for every row, some 20 times the cost.
#include <algorithm>

#include <cooperative_groups.h>

#include "g4_common.cuh"

namespace {

using namespace g4dev;
namespace cg = cooperative_groups;

constexpr int kMaxVocab = 786432;
constexpr int kMaxGroups = 2048;
constexpr int kMaxTopK = 1024;   // of the finish kernel
constexpr int kCand = 2048;      // candidates the finish kernel ranks

struct SampleParams {
    const float* logits;
    long long ld;
    int rows, vocab;
    float cap;
    g4_sampling how;
    int32_t* ids;
    float* probs;
    uint32_t* gkey;   // [rows][groups] highest key of each group
    double* gmass;    // [rows][groups] sum of exp((l - group's highest) / T)
    int* queue;       // [0] rows left to the general kernel, then the rows
    int gshift, groups;
};

// Monotone key of a logit: larger logit, larger key; 0 for what is never picked (NaN, -inf).
__device__ __forceinline__ uint32_t logit_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);  // -0 ties with +0
    const uint32_t k = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return l > -INFINITY ? k : 0u;
}
constexpr uint32_t kLowestKey = 0x00800000u;  // of -FLT_MAX
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// A row's settings with what is off made explicit.
enum Mode { kTopK, kAll, kMinP, kTopP, kGeneral };
struct RowSettings {
    double c;         // log2(e) / temperature
    double p, mp;     // p >= 1: off; mp = 0: off
    int k;            // 0: off
    Mode mode;
};
__device__ __forceinline__ RowSettings row_settings(const SampleParams& P, int r) {
    RowSettings s;
    const float t = P.how.temperature ? P.how.temperature[r] : 1.f;
    const float tp = P.how.top_p ? P.how.top_p[r] : 1.f;
    const float mp = P.how.min_p ? P.how.min_p[r] : 0.f;
    s.k = P.how.top_k ? P.how.top_k[r] : 0;
    if (s.k < 1 || s.k >= P.vocab) s.k = 0;
    s.p = tp < 1.f ? (double)tp : 2.0;
    s.mp = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
    s.c = 1.4426950408889634 / (double)t;
    if (!(t > 0.f)) {  // the greedy pick
        s.k = 1, s.c = 1.0, s.p = 2.0, s.mp = 0.0;
    } else if (s.p <= 0.0) {
        s.k = 1, s.p = 2.0;
    }
    s.mode = s.k > kMaxTopK ? kGeneral : s.k ? kTopK : s.p < 1.0 ? kTopP : s.mp > 0.0 ? kMinP : kAll;
    return s;
}

// 2^y for y <= 0, relative error below 3e-15 (0 below 2^-1021): y = k / 32 + f, |f| <= 1/64, a
// table of 2^(j/32) and the Taylor polynomial of 2^f to the fifth power (the table-driven method
// of P. T. P. Tang, 1989).  12 double-precision operations; `table` is shared memory.
__device__ __forceinline__ double exp2_64(double y, const double* table) {
    const double magic = 211106232532992.0;  // 1.5 * 2^47: one unit in the last place is 1/32
    const double t = y + magic;
    const int k = __double2loint(t);
    const double f = y - (t - magic);
    double q = 0.0013333558146428443;
    q = fma(q, f, 0.009618129107628477);
    q = fma(q, f, 0.05550410866482158);
    q = fma(q, f, 0.24022650695910072);
    q = fma(q, f, 0.6931471805599453);
    q = fma(q, f, 1.0);
    q *= table[k & 31];
    return y < -1021.0 ? 0.0 : __hiloint2double(__double2hiint(q) + ((k >> 5) << 20), __double2loint(q));
}
__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 32.0));
}
// exp((v - m) / T); +inf logits (m = +inf) share the whole weight.
__device__ __forceinline__ double weight(float v, float m, double c, const double* table) {
    if (v == m) return 1.0;
    if (m == INFINITY) return 0.0;
    return exp2_64(((double)v - (double)m) * c, table);
}

__device__ __forceinline__ float capped(float v, float cap) { return cap > 0.f ? tanhf(v / cap) * cap : v; }

// ---------------------------------------------------------------- summary --
// A warp takes 512 consecutive logits at a time as four chunks of 128.  kVec: rows are 16-byte
// aligned and a lane holds 4 consecutive logits of each chunk; else a lane holds logits lane,
// lane + 32, ... of it.  Groups of up to 128 lie inside a chunk, larger ones join chunks.
constexpr int kSumWarps = 8;
template <bool kVec>
__global__ void __launch_bounds__(kSumWarps * 32) sample_summary_kernel(const SampleParams P, int segments) {
    __shared__ double table[32];
    pdl_trigger();
    pdl_wait();
    fill_table(table);
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) P.queue[0] = 0;
    const int lane = threadIdx.x & 31;
    const int r = (int)(blockIdx.x / (unsigned)segments);
    const int base = ((int)(blockIdx.x - (unsigned)r * segments) * kSumWarps + (threadIdx.x >> 5)) * 512;
    if (base >= P.vocab) return;
    const float* row = P.logits + (size_t)r * P.ld;
    float v[4][4];
    auto index = [&](int i, int e) { return base + i * 128 + (kVec ? lane * 4 + e : e * 32 + lane); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (kVec && index(i, 3) < P.vocab) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(row + index(i, 0)));
            v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = index(i, e) < P.vocab ? row[index(i, e)] : -INFINITY;
        }
    }
    const RowSettings st = row_settings(P, r);
    const bool mass = st.mode == kAll || st.mode == kTopP;
    if (P.cap > 0.f) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = capped(v[i][e], P.cap);
    }
    const int gs = 1 << P.gshift;
    // Units that one warp reduction covers: a chunk (kVec) or 32 logits of it.
    constexpr int U = kVec ? 1 : 4;
    const int lanes = min(32, kVec ? gs >> 2 : gs);  // lanes of a unit that share a group
    uint32_t key[4][U];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t k = kVec ? max(max(logit_key(v[i][0]), logit_key(v[i][1])), max(logit_key(v[i][2]), logit_key(v[i][3])))
                              : logit_key(v[i][u]);
            for (int o = 1; o < lanes; o <<= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
            key[i][u] = k;
        }
    }
    // Groups of several units.
    const int span = gs / (kVec ? 128 : 32);  // units per group, if more than one
    if (!kVec && span >= 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            key[i][0] = key[i][U > 1 ? 1 : 0] = max(key[i][0], key[i][U > 1 ? 1 : 0]);
            key[i][U > 2 ? 2 : 0] = key[i][U > 3 ? 3 : 0] = max(key[i][U > 2 ? 2 : 0], key[i][U > 3 ? 3 : 0]);
            if (span >= 4) {
                const uint32_t k = max(key[i][0], key[i][U > 2 ? 2 : 0]);
#pragma unroll
                for (int u = 0; u < U; ++u) key[i][u] = k;
            }
        }
    }
    if (gs >= 256) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            key[0][u] = key[1][u] = max(key[0][u], key[1][u]);
            key[2][u] = key[3][u] = max(key[2][u], key[3][u]);
            if (gs >= 512) key[0][u] = key[1][u] = key[2][u] = key[3][u] = max(key[0][u], key[2][u]);
        }
    }
    double sum[4][U];
    if (mass) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int u = 0; u < U; ++u) sum[i][u] = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int u = kVec ? 0 : e;
                const uint32_t k = key[i][u];
                const float g = key_logit(k);
                if (k != 0u && logit_key(v[i][e]) != 0u) sum[i][u] += weight(v[i][e], g, st.c, table);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                for (int o = 1; o < lanes; o <<= 1) sum[i][u] += __shfl_xor_sync(0xffffffffu, sum[i][u], o);
        }
    }
    uint32_t* gk = P.gkey + (size_t)r * P.groups;
    double* gm = P.gmass + (size_t)r * P.groups;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = base + i * 128 + (kVec ? lane * 4 : u * 32 + lane);
            if (at & (gs - 1)) continue;  // the first lane of the group's first unit writes
            const int g = at >> P.gshift;
            if (g >= P.groups) continue;
            gk[g] = key[i][u];
            if (!mass) continue;
            double s = sum[i][u];
            if (!kVec && span >= 2) {
                if (U > 1 && u + 1 < U) s += sum[i][(u + 1) % U];
                if (span >= 4 && u == 0) s += sum[i][2 % U] + sum[i][3 % U];
            }
            if (gs >= 256 && i + 1 < 4) {
                double t = 0.0;
#pragma unroll
                for (int w = 0; w < U; ++w) t += sum[(i + 1) & 3][w];
                s += t;
                if (gs >= 512 && i == 0) {
#pragma unroll
                    for (int w = 0; w < U; ++w) s += sum[2][w] + sum[3][w];
                }
            }
            gm[g] = s;
        }
    }
}

// ------------------------------------------------- block-wide building blocks --
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

struct BlockScratch {
    double d[2][kWarps];
    uint32_t u[2][kWarps];
};
// Sum over the block of an int / double, given to every thread; `flip` alternates two buffers so
// that one barrier per call is enough.
__device__ __forceinline__ int block_sum_int(int v, BlockScratch& s, int& flip) {
    v = __reduce_add_sync(0xffffffffu, v);
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) s.u[flip][threadIdx.x >> 5] = (uint32_t)v;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) t += (int)s.u[flip][i];
    return t;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, BlockScratch& s, int& flip) {
    v = __reduce_max_sync(0xffffffffu, v);
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) s.u[flip][threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) t = max(t, s.u[flip][i]);
    return t;
}
__device__ __forceinline__ double block_sum(double v, BlockScratch& s, int& flip) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) s.d[flip][threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) t += s.d[flip][i];
    return t;
}
// Sum over the threads before this one; *total gets the whole.
__device__ __forceinline__ double block_prefix(double v, BlockScratch& s, int& flip, double* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    double x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    flip ^= 1;
    if (lane == 31) s.d[flip][w] = x;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i == w) before = all;
        all += s.d[flip][i];
    }
    *total = all;
    double left = __shfl_up_sync(0xffffffffu, x, 1);
    if (lane == 0) left = 0.0;
    return before + left;
}

// Bitonic sort of n = a power of two 64-bit values in shared memory, largest first.
__device__ __forceinline__ void block_sort_desc(unsigned long long* a, int n) {
    for (int size = 2; size <= n; size <<= 1) {
        for (int step = size >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < n / 2; t += kThreads) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const unsigned long long x = a[i], y = a[j];
                const bool desc = (i & size) == 0;
                if ((x < y) == desc) a[i] = y, a[j] = x;
            }
        }
    }
    __syncthreads();
}
__device__ __forceinline__ int pow2_at_least(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

__device__ __forceinline__ double row_uniform(const SampleParams& P, int r) {
    const float u = P.how.uniform[r];
    return u >= 0.f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0;
}

// ----------------------------------------------------------------- finish --
struct FinishShared {
    double table[32];
    unsigned long long cand[kCand];  // key << 32 | ~index; then index << 32 | position
    double w[kCand];
    uint16_t glist[kMaxGroups];
    BlockScratch scratch;
    double zk;
    int n, ng, kept;
};

__global__ void __launch_bounds__(kThreads) sample_finish_kernel(const SampleParams P, int vec) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    FinishShared& S = *reinterpret_cast<FinishShared*>(smem_raw);
    pdl_trigger();
    fill_table(S.table);
    if (threadIdx.x == 0) S.n = S.ng = S.kept = 0;
    pdl_wait();
    int flip = 0;
    const int r = blockIdx.x, G = P.groups, gs = 1 << P.gshift;
    const float* row = P.logits + (size_t)r * P.ld;
    const RowSettings st = row_settings(P, r);
    const uint32_t* gk = P.gkey + (size_t)r * G;
    uint32_t key[kMaxGroups / kThreads];
    constexpr int KG = kMaxGroups / kThreads;
    uint32_t top = 0, low = 0;
#pragma unroll
    for (int i = 0; i < KG; ++i) {
        const int g = i * kThreads + threadIdx.x;
        key[i] = g < G ? gk[g] : 0u;
    }
#pragma unroll
    for (int i = 0; i < KG; ++i) {
        top = max(top, key[i]);
        if (key[i]) low = max(low, ~key[i]);
    }
    top = block_max(top, S.scratch, flip);
    if (top == 0u) {
        if (threadIdx.x == 0) {
            P.ids[r] = -1;
            if (P.probs) P.probs[r] = 0.f;
        }
        return;
    }
    const float m = key_logit(top);
    const double u = row_uniform(P, r);
    auto leave = [&]() {  // to the general kernel
        if (threadIdx.x == 0) P.queue[1 + atomicAdd(P.queue, 1)] = r;
    };
    if (st.mode == kGeneral) {
        leave();
        return;
    }
    if (st.mode == kAll) {
        // Groups in index order, four consecutive ones per thread.
        const double* gm = P.gmass + (size_t)r * G;
        double x[KG], own = 0.0, total;
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            const int g = threadIdx.x * KG + i;
            x[i] = g < G && gk[g] ? gm[g] * weight(key_logit(gk[g]), m, st.c, S.table) : 0.0;
            own += x[i];
        }
        const double before = block_prefix(own, S.scratch, flip, &total);
        const double target = u * total;
        // The thread whose groups hold the target; its first group past it (the last positive one
        // where rounding leaves none).
        if (own > 0.0 && before <= target) {
            // the highest such thread wins
            atomicMax(&S.ng, (int)threadIdx.x + 1);
        }
        __syncthreads();
        if (S.ng == (int)threadIdx.x + 1) {
            double c = before;
            int g = 0;
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                if (x[i] > 0.0 && c <= target) {
                    g = threadIdx.x * KG + i;
                    S.w[0] = c;
                }
                c += x[i];
            }
            S.n = g;
        }
        __syncthreads();
        if (threadIdx.x < 32) {  // the pick inside the group
            const int lane = threadIdx.x;
            double c = S.w[0];
            int pick = -1;
            double wp = 0.0;
            for (int o = 0; o < gs; o += 32) {
                const int i = (S.n << P.gshift) + o + lane;
                double w = 0.0;
                if (o + lane < gs && i < P.vocab) {
                    const float v = capped(row[i], P.cap);
                    if (logit_key(v)) w = weight(v, m, st.c, S.table);
                }
                double s = w;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, s, d);
                    if (lane >= d) s += y;
                }
                const unsigned past = __ballot_sync(0xffffffffu, w > 0.0 && c + s > target);
                const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
                const int from = past ? __ffs(past) - 1 : some ? 31 - __clz(some) : 0;
                if (some) {
                    pick = (S.n << P.gshift) + o + from;
                    wp = __shfl_sync(0xffffffffu, w, from);
                }
                if (past) break;
                c += __shfl_sync(0xffffffffu, s, 31);
            }
            if (lane == 0) {
                P.ids[r] = pick;
                if (P.probs) P.probs[r] = (float)(wp / total);
            }
        }
        return;
    }

    // Candidates: every logit with key >= bound, from the groups whose maximum reaches it.
    uint32_t bound;
    double total = 0.0;
    if (st.mode == kMinP) {
        // the lowest key that weighs mp or more: w falls with the key
        uint32_t lo = kLowestKey, hi = top;  // hi keeps
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (weight(key_logit(mid), m, st.c, S.table) >= st.mp) hi = mid;
            else lo = mid + 1;
        }
        bound = hi;
    } else {
        low = ~block_max(low, S.scratch, flip);  // the lowest group maximum
        uint32_t lo = low, hi = top + 1;          // [lo, hi): what counts >= lo is enough, >= hi is not
        if (st.mode == kTopK) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < KG; ++i) c += key[i] != 0u;
            if (block_sum_int(c, S.scratch, flip) < st.k) {
                lo = 1;
            } else {
                while (hi - lo > 1) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    c = 0;
#pragma unroll
                    for (int i = 0; i < KG; ++i) c += key[i] >= mid;
                    c = block_sum_int(c, S.scratch, flip);
                    if (c >= st.k) {
                        lo = mid;
                        if (c <= st.k + st.k / 8 + 4) break;  // few enough
                    } else {
                        hi = mid;
                    }
                }
            }
        } else {
            // Nucleus: the weights of the highest group maxima are a lower bound of what the logits
            // above them weigh.
            const double* gm = P.gmass + (size_t)r * G;
            double own = 0.0;
            float w[KG];
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const int g = i * kThreads + threadIdx.x;
                const double x = key[i] ? weight(key_logit(key[i]), m, st.c, S.table) : 0.0;
                w[i] = (float)x;
                own += key[i] ? x * gm[g] : 0.0;
            }
            total = block_sum(own, S.scratch, flip);
            const float need = (float)(st.p * total * 1.0001);
            auto above = [&](uint32_t at) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < KG; ++i) s += key[i] >= at ? w[i] : 0.f;
                return block_sum((double)s, S.scratch, flip);
            };
            if (above(low) < need) {
                leave();
                return;
            }
            while (hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                const double a = above(mid);
                if (a >= need) {
                    lo = mid;
                    if (a <= need * 1.01) break;
                } else {
                    hi = mid;
                }
            }
        }
        bound = lo;
    }
#pragma unroll
    for (int i = 0; i < KG; ++i)
        if (key[i] >= bound) S.glist[atomicAdd(&S.ng, 1)] = (uint16_t)(i * kThreads + threadIdx.x);
    __syncthreads();
    const int ng = S.ng;
    if (ng > kCand / 2 && P.vocab > 4 * kCand) {  // too many to rank here (a short row is tried whole)
        leave();
        return;
    }
    const int qs = gs >> 2, quads = ng * qs;  // four consecutive logits at a time
#pragma unroll 4
    for (int q = threadIdx.x; q < quads; q += kThreads) {
        const int i0 = ((int)S.glist[q / qs] << P.gshift) + (q % qs) * 4;
        float v[4];
        if (vec && i0 + 3 < P.vocab) {
            const float4 f = *reinterpret_cast<const float4*>(row + i0);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i0 + e < P.vocab ? row[i0 + e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t k = logit_key(capped(v[e], P.cap));
            if (k >= bound) {
                const int at = atomicAdd(&S.n, 1);
                if (at < kCand) S.cand[at] = (unsigned long long)k << 32 | (0xffffffffu - (unsigned)(i0 + e));
            }
        }
    }
    __syncthreads();
    const int n = S.n;
    if (n > kCand) {
        leave();
        return;
    }
    int n2 = pow2_at_least(n);
    for (int i = n + threadIdx.x; i < n2; i += kThreads) S.cand[i] = 0ull;
    block_sort_desc(S.cand, n2);
    // Ranks 4t .. 4t + 3: weights, their running sum and where it ends the prefix.
    constexpr int E = kCand / kThreads;
    const int limit = st.mode == kTopK ? min(st.k, n) : n;
    double w[E], own = 0.0, all;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = threadIdx.x * E + e;
        w[e] = i < limit ? weight(key_logit((uint32_t)(S.cand[i] >> 32)), m, st.c, S.table) : 0.0;
        if (i < n2) S.w[i] = w[e];
        own += w[e];
    }
    double run = block_prefix(own, S.scratch, flip, &all);
    if (st.mode != kTopP) total = all;
    const double need = st.p * total;
    if (st.mode == kTopP && all < need) {
        leave();
        return;
    }
    // kept: the longest prefix that the filters leave.
    if (threadIdx.x == 0) S.kept = limit;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = threadIdx.x * E + e;
        run += w[e];
        if (i < limit && ((st.p < 1.0 && run >= need) || (i + 1 < limit && st.mp > 0.0 && S.w[i + 1] < st.mp)))
            atomicMin(&S.kept, i + 1);
    }
    __syncthreads();
    const int kept = S.kept;
    // The kept ones in index order.
    n2 = pow2_at_least(kept);
    for (int i = threadIdx.x; i < n2; i += kThreads) {
        // ~index << 32 | position: largest first is lowest index first
        S.cand[i] = i < kept ? (S.cand[i] & 0xffffffffull) << 32 | (unsigned)i : 0ull;
    }
    block_sort_desc(S.cand, n2);
    own = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = threadIdx.x * E + e;
        w[e] = i < kept ? S.w[(uint32_t)S.cand[i]] : 0.0;
        own += w[e];
    }
    run = block_prefix(own, S.scratch, flip, &all);
    const double target = u * all;
    // The first rank whose running sum exceeds the target; the highest positive one at or below it
    // is the same rank: sums before it do not exceed the target.
    if (threadIdx.x == 0) S.n = 0;
    __syncthreads();
    int mine = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (w[e] > 0.0 && run <= target) mine = threadIdx.x * E + e;
        run += w[e];
    }
    if (mine >= 0) atomicMax(&S.n, mine);
    __syncthreads();
    if (mine >= 0 && mine == S.n) {
        const unsigned long long c = S.cand[mine];
        P.ids[r] = (int)(0xffffffffu - (unsigned)(c >> 32));
        if (P.probs) P.probs[r] = (float)(S.w[(uint32_t)c] / all);
    }
}

// ---------------------------------------------------------------- general --
// A cluster of up to 16 CTAs takes queued rows, each CTA with its part of the row in shared
// memory (warps own consecutive segments of 128 * J logits).
constexpr int kMaxCluster = 16;
constexpr int kPick = 1024;  // logits ranked at the end of a search
constexpr int kWays = 8;

struct GeneralShared {
    double table[32];
    double xd[2][kMaxCluster][kWays];  // per rank: sums of a step
    int xn[2][kMaxCluster][kWays];     // per rank: counts of a step
    uint32_t xlow[kMaxCluster];        // per rank: ~ the lowest key
    unsigned long long cand[kPick];
    BlockScratch scratch;
    double wsum[kWarps];
    int wcnt[kWarps];
    double red[kWarps][kWays];
    int redn[kWarps][kWays];
    uint32_t found_key;
    int found_idx, ncand, work;
};
// The kept prefix: keys above `key`, and equal ones up to index `idx`.
struct Limit {
    uint32_t key;
    int idx;
};

struct General {
    const SampleParams& P;
    GeneralShared& S;
    const float* chunk;
    cg::cluster_group cluster;
    int rank, ranks, J, r, flip, xflip;
    float m;
    uint32_t top, low;  // highest and lowest key of the row
    double c;

    __device__ int first_index() const { return rank * kThreads * 4 * J; }
    __device__ bool inside(uint32_t k, int i, const Limit& lim) const {
        return k != 0u && (k > lim.key || (k == lim.key && i <= lim.idx));
    }
    // f(index, logit) over this thread's logits, in the warp's segment.
    template <class F>
    __device__ void each(F f) const {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        for (int j = 0; j < J; ++j) {
            const int o = (w * J + j) * 128 + lane * 4;
            const float4 v = *reinterpret_cast<const float4*>(chunk + o);
            const int i = first_index() + o;
            f(i, v.x);
            f(i + 1, v.y);
            f(i + 2, v.z);
            f(i + 3, v.w);
        }
    }
    // Sums over the cluster of kWays doubles and counts per thread (added in rank order).
    __device__ void cluster_sums(double (&d)[kWays], int (&n)[kWays]) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
        for (int i = 0; i < kWays; ++i) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d[i] += __shfl_xor_sync(0xffffffffu, d[i], o);
            n[i] = __reduce_add_sync(0xffffffffu, n[i]);
            if (lane == 0) S.red[w][i] = d[i], S.redn[w][i] = n[i];
        }
        __syncthreads();
        xflip ^= 1;
        if (threadIdx.x < ranks * kWays) {
            const int to = threadIdx.x / kWays, i = threadIdx.x % kWays;
            double s = 0.0;
            int t = 0;
            for (int k = 0; k < kWarps; ++k) s += S.red[k][i], t += S.redn[k][i];
            *cluster.map_shared_rank(&S.xd[xflip][rank][i], to) = s;
            *cluster.map_shared_rank(&S.xn[xflip][rank][i], to) = t;
        }
        cluster.sync();
#pragma unroll
        for (int i = 0; i < kWays; ++i) {
            d[i] = 0.0, n[i] = 0;
            for (int k = 0; k < ranks; ++k) d[i] += S.xd[xflip][k][i], n[i] += S.xn[xflip][k][i];
        }
    }
    __device__ double mass(const Limit& lim, bool count) {
        double d[kWays] = {};
        int n[kWays] = {};
        each([&](int i, float v) {
            const uint32_t k = logit_key(v);
            if (inside(k, i, lim)) d[0] += count ? 1.0 : weight(v, m, c, S.table);
        });
        cluster_sums(d, n);
        return d[0];
    }

    // The shortest prefix inside `lim` whose weight (number, if count) is at least t.  [lo, hi) are
    // the keys where it ends, `above` what the keys from hi on weigh; each step cuts them in eight,
    // in turn evenly in value (which suits what logits look like) and in key (which ends after at
    // most eleven steps).
    __device__ Limit search(const Limit& lim, double t, bool count) {
        uint32_t lo = low, hi = top + 1;
        double above = 0.0;
        int inside_n = 0x7fffffff;
        for (int step = 0; inside_n > kPick && hi - lo > 1; ++step) {
            uint32_t cut[kWays];
            const float a = key_logit(lo), b = key_logit(hi - 1);
            const bool even = (step & 1) == 0 && a > -3.0e38f && b < 3.0e38f && a < b;
#pragma unroll
            for (int i = 0; i < kWays; ++i) {
                uint32_t k = lo + (uint32_t)((unsigned long long)(hi - lo) * i / kWays);
                if (even && i > 0) k = logit_key((float)((double)a + ((double)b - (double)a) * (i / (double)kWays)));
                cut[i] = i == 0 ? lo : min(max(k, cut[i - 1]), hi);
            }
            double d[kWays] = {};
            int n[kWays] = {};
            each([&](int i, float v) {
                const uint32_t k = logit_key(v);
                if (k >= lo && k < hi && inside(k, i, lim)) {
                    const double w = count ? 1.0 : weight(v, m, c, S.table);
#pragma unroll
                    for (int q = 0; q < kWays; ++q)
                        if (k >= cut[q]) d[q] += w, n[q] += 1;
                }
            });
            cluster_sums(d, n);
            int at = 0;
#pragma unroll
            for (int q = 1; q < kWays; ++q)
                if (cut[q] < hi && above + d[q] >= t) at = q;
            uint32_t nlo = lo, nhi = hi;
            double nabove = above;
            int na = 0;
#pragma unroll
            for (int q = 0; q < kWays; ++q) {
                if (q == at) nlo = cut[q], na = n[q];
                if (q == at + 1 && cut[q] < hi) nhi = cut[q], nabove = above + d[q], na -= n[q];
            }
            lo = nlo, hi = nhi, above = nabove, inside_n = na;
        }
        if (inside_n > kPick) return nth_equal(lim, lo, above, t, count, inside_n);
        // Rank what is left in CTA 0.
        if (threadIdx.x == 0) S.ncand = 0;
        cluster.sync();
        int* cnt = cluster.map_shared_rank(&S.ncand, 0);
        unsigned long long* list = cluster.map_shared_rank(&S.cand[0], 0);
        each([&](int i, float v) {
            const uint32_t k = logit_key(v);
            if (k >= lo && k < hi && inside(k, i, lim))
                list[atomicAdd(cnt, 1)] = (unsigned long long)k << 32 | (0xffffffffu - (unsigned)i);
        });
        cluster.sync();
        if (rank == 0) {
            const int n = S.ncand, n2 = pow2_at_least(n);
            for (int i = n + threadIdx.x; i < n2; i += kThreads) S.cand[i] = 0ull;
            block_sort_desc(S.cand, n2);
            constexpr int E = kPick / kThreads;
            double w[E], own = 0.0, all;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = threadIdx.x * E + e;
                w[e] = i < n ? (count ? 1.0 : weight(key_logit((uint32_t)(S.cand[i] >> 32)), m, c, S.table)) : 0.0;
                own += w[e];
            }
            double run = above + block_prefix(own, S.scratch, flip, &all);
            if (threadIdx.x == 0) S.work = n - 1;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                run += w[e];
                if (threadIdx.x * E + e < n && run >= t) atomicMin(&S.work, threadIdx.x * E + e);
            }
            __syncthreads();
            if (threadIdx.x < ranks) {
                const unsigned long long f = S.cand[S.work];
                *cluster.map_shared_rank(&S.found_key, threadIdx.x) = (uint32_t)(f >> 32);
                *cluster.map_shared_rank(&S.found_idx, threadIdx.x) = (int)(0xffffffffu - (unsigned)f);
            }
        }
        cluster.sync();
        return Limit{S.found_key, S.found_idx};
    }

    // The search ended at one key shared by `n` logits of one weight: the first of them, in index
    // order, that reach t.
    __device__ Limit nth_equal(const Limit& lim, uint32_t key, double above, double t, bool count, int n) {
        const double w = count ? 1.0 : weight(key_logit(key), m, c, S.table);
        const double q = ceil((t - above) / w);
        const int need = q >= (double)n ? n : q > 1.0 ? (int)q : 1;
        double d[kWays] = {};
        int own[kWays] = {};
        each([&](int i, float v) { own[0] += logit_key(v) == key && inside(key, i, lim); });
        const int mine = own[0];
        cluster_sums(d, own);
        int before = 0;
        for (int k = 0; k < rank; ++k) before += S.xn[xflip][k][0];
        const int here = S.xn[xflip][rank][0];
        if (before < need && need <= before + here) {  // the whole CTA
            const int lane = threadIdx.x & 31, w0 = threadIdx.x >> 5;
            const int in_warp = __reduce_add_sync(0xffffffffu, mine);
            if (lane == 0) S.wcnt[w0] = in_warp;
            __syncthreads();
            int wb = before;
            for (int k = 0; k < w0; ++k) wb += S.wcnt[k];
            if (wb < need && need <= wb + in_warp) {
                for (int j = 0; j < J; ++j) {
                    const int o = (w0 * J + j) * 128 + lane * 4, i0 = first_index() + o;
                    int eq[4], cnt = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) cnt += eq[e] = logit_key(chunk[o + e]) == key && inside(key, i0 + e, lim);
                    int x = cnt;
#pragma unroll
                    for (int s = 1; s < 32; s <<= 1) {
                        const int y = __shfl_up_sync(0xffffffffu, x, s);
                        if (lane >= s) x += y;
                    }
                    int at = wb + x - cnt;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        at += eq[e];
                        if (eq[e] && at == need)
                            for (int k = 0; k < ranks; ++k) *cluster.map_shared_rank(&S.found_idx, k) = i0 + e;
                    }
                    wb += __shfl_sync(0xffffffffu, x, 31);
                }
            }
        }
        cluster.sync();
        return Limit{key, S.found_idx};
    }

    // The pick in index order among what `lim` and mp keep.
    __device__ void pick(const Limit& lim, double mp, double u) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        auto kept = [&](int i, float v) {
            if (!inside(logit_key(v), i, lim)) return 0.0;
            const double x = weight(v, m, c, S.table);
            return x < mp ? 0.0 : x;
        };
        double d[kWays] = {};
        int n[kWays] = {};
        each([&](int i, float v) { d[0] += kept(i, v); });
        double ws = d[0];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
        if (lane == 0) S.wsum[w] = ws;
        cluster_sums(d, n);
        // The last CTA, warp and lane with something at or below the target hold the pick.
        const double total = d[0], target = u * total;
        double before = 0.0, start = 0.0;
        int owner = 0;
        for (int k = 0; k < ranks; ++k) {
            if (S.xd[xflip][k][0] > 0.0 && before <= target) owner = k, start = before;
            before += S.xd[xflip][k][0];
        }
        if (owner != rank) return;
        int ow = 0;
        before = start;
        for (int k = 0; k < kWarps; ++k) {
            if (S.wsum[k] > 0.0 && before <= target) ow = k, start = before;
            before += S.wsum[k];
        }
        if (ow != w) return;
        int best = -1;
        double bw = 0.0, run = start;
        for (int j = 0; j < J; ++j) {
            const int o = (w * J + j) * 128 + lane * 4, i0 = first_index() + o;
            double x[4], s = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) s += x[e] = kept(i0 + e, chunk[o + e]);
            double y = s;
#pragma unroll
            for (int q = 1; q < 32; q <<= 1) {
                const double z = __shfl_up_sync(0xffffffffu, y, q);
                if (lane >= q) y += z;
            }
            double at = run + (y - s);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (x[e] > 0.0 && at <= target) best = i0 + e, bw = x[e];
                at += x[e];
            }
            run += __shfl_sync(0xffffffffu, y, 31);
        }
        const int last = __reduce_max_sync(0xffffffffu, best);
        if (best == last && best >= 0) {
            P.ids[r] = best;
            if (P.probs) P.probs[r] = (float)(bw / total);
        }
    }
};

__global__ void __launch_bounds__(kThreads) sample_general_kernel(const SampleParams P, int J) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    GeneralShared& S = *reinterpret_cast<GeneralShared*>(smem_raw);
    float* chunk = reinterpret_cast<float*>(smem_raw + ((sizeof(GeneralShared) + 15) & ~size_t(15)));
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    pdl_trigger();
    fill_table(S.table);
    pdl_wait();
    cluster.sync();  // every CTA of the cluster runs before any writes to another's shared memory
    General g{P, S, chunk, cluster, rank, ranks, J, 0, 0, 0, 0.f, 0u, 0u, 0.0};
    const int queued = P.queue[0];
    for (int q = blockIdx.x / ranks; q < queued; q += gridDim.x / ranks) {
        const int r = P.queue[1 + q];
        const float* row = P.logits + (size_t)r * P.ld;
        g.r = r;
        __syncthreads();
        const int i0 = g.first_index(), per = kThreads * 4 * J;
        uint32_t top = 0, low = 0;
#pragma unroll 8
        for (int o = threadIdx.x; o < per; o += kThreads) {
            const float v = i0 + o < P.vocab ? capped(row[i0 + o], P.cap) : -INFINITY;
            chunk[o] = v;
            const uint32_t k = logit_key(v);
            if (k) low = max(low, ~k);
        }
        for (int i = threadIdx.x; i < P.groups; i += kThreads) top = max(top, P.gkey[(size_t)r * P.groups + i]);
        g.top = block_max(top, S.scratch, g.flip);  // (its barrier also closes the loads of the chunk)
        g.m = key_logit(g.top);
        low = block_max(low, S.scratch, g.flip);
        if (threadIdx.x < ranks) *cluster.map_shared_rank(&S.xlow[rank], threadIdx.x) = low;
        cluster.sync();
        low = 0;
        for (int k = 0; k < ranks; ++k) low = max(low, S.xlow[k]);
        g.low = ~low;
        const RowSettings st = row_settings(P, r);
        g.c = st.c;
        Limit lim{0u, 0};
        if (st.k && g.mass(lim, true) > (double)st.k) lim = g.search(lim, (double)st.k, true);
        if (st.p < 1.0) lim = g.search(lim, st.p * g.mass(lim, false), false);
        g.pick(lim, st.mp, row_uniform(P, r));
        cluster.sync();  // the exchange buffers are free again
    }
}

}  // namespace

extern "C" g4_status g4_sample(g4_ctx* ctx, const float* logits, long long ld, int rows, int vocab, float cap,
                               const g4_sampling* how, int32_t* ids_out, float* probs_out) {
    if (rows < 0 || vocab < 1 || ld < vocab || !how)
        return g4::set_error(G4_ERR_INVALID, "g4_sample: rows %d, vocab %d, row pitch %lld", rows, vocab, ld);
    if (vocab > kMaxVocab) return g4::set_error(G4_ERR_UNSUPPORTED, "g4_sample: vocab %d (%d supported)", vocab, kMaxVocab);
    if (rows > 0 && (!logits || !how->uniform || !ids_out))
        return g4::set_error(G4_ERR_INVALID, "g4_sample: null argument");
    g4_status st = g4::use_device(ctx);
    if (st || rows == 0) return st;
    SampleParams P{logits, ld, rows, vocab, cap, *how, ids_out, probs_out, nullptr, nullptr, nullptr, 2, 0};
    while (((vocab + (1 << P.gshift) - 1) >> P.gshift) > kMaxGroups) ++P.gshift;
    P.groups = (vocab + (1 << P.gshift) - 1) >> P.gshift;
    const long long segments = (vocab + kSumWarps * 512 - 1) / (kSumWarps * 512);
    if (segments * rows > 0x7fffffffLL)
        return g4::set_error(G4_ERR_UNSUPPORTED, "g4_sample: %d rows of %d logits", rows, vocab);
    const size_t ng = (size_t)rows * P.groups;
    st = g4::ensure_workspace(ctx, ng * sizeof(double) + ng * sizeof(uint32_t) + ((size_t)rows + 1) * sizeof(int));
    if (st) return st;
    P.gmass = static_cast<double*>(ctx->ws);
    P.gkey = reinterpret_cast<uint32_t*>(P.gmass + ng);
    P.queue = reinterpret_cast<int*>(P.gkey + ng);
    const int vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (ld % 4 == 0 || rows == 1);

    // The general kernel's cluster: parts of at most 16384 logits if 16 CTAs are enough for that.
    int ranks = 1;
    while (ranks < kMaxCluster && (vocab + ranks - 1) / ranks > 2 * kThreads * 4) ranks <<= 1;
    const int J = (vocab + ranks * kThreads * 4 - 1) / (ranks * kThreads * 4);
    const size_t gsmem = ((sizeof(GeneralShared) + 15) & ~size_t(15)) + (size_t)J * kThreads * 4 * sizeof(float);
    static std::atomic<uint64_t> attr_set{0};
    if (!(attr_set.load() & (1ull << ctx->device))) {
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_finish_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)sizeof(FinishShared)));
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_general_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_general_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr_set.fetch_or(1ull << ctx->device);
    }
    st = g4::launch(ctx, "sample_summary_kernel", vec ? sample_summary_kernel<true> : sample_summary_kernel<false>,
                    dim3((unsigned)(segments * rows)), dim3(kSumWarps * 32), 0, 1, P, (int)segments);
    if (st) return st;
    // The two that follow are set up while their predecessor runs, and wait for it (griddepcontrol).
    const bool pdl = ctx->pdl;
    ctx->pdl = true;
    st = g4::launch(ctx, "sample_finish_kernel", sample_finish_kernel, dim3(rows), dim3(kThreads), sizeof(FinishShared), 1, P,
                    vec);
    // Only top-k, top-p and min-p can leave a row to the general kernel.
    if (!st && (how->top_k || how->top_p || how->min_p)) {
        const int clusters = std::max(1, std::min(rows, 128 / ranks));
        st = g4::launch(ctx, "sample_general_kernel", sample_general_kernel, dim3(clusters * ranks), dim3(kThreads), gsmem,
                        ranks, P, J);
    }
    ctx->pdl = pdl;
    return st;
}
