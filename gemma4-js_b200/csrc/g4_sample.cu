// g4_sample.cu -- one token per row of f32 logits: temperature, top-k, top-p, min-p and a given
// uniform number per row.
//
// With w_i = exp((l_i - m) / T), m the highest logit, the filters keep a prefix of the ranking
// by (l descending, index ascending), and the pick is an inverse cumulative sum in index order.
// Sums of up to 786432 weights decide which token a border falls on, so weights and sums are
// 64-bit (32-bit weights would move a border past a token in one row of some hundred).
//
// Three launches, and a fourth before the last where a top_p is given without a top_k:
//   summary  reads the logits once (bound by HBM) and leaves, per group of 4 .. 512 consecutive
//            logits (at most 2048 groups a row), the highest key and, for rows whose settings
//            need the mass of the whole row, the group's weight relative to its highest logit.
//   finish   one CTA per row works from the groups: the k-th highest group maximum bounds the
//            k-th highest logit from below, so only the about k groups above it are read again
//            (64 of 2048 groups: 32 KB of a 1 MB row) and ranked.  Rows it cannot settle that
//            way (a nucleus of more than some thousand tokens, top-k above 1024, masses of ties)
//            go to a queue, rows of one rank never.
//   nucleus  a cluster of CTAs reads a queued row with a top-p alone twice: once to find what the
//            prefix can end on, once for its sum and end.
//   general  a cluster of CTAs holds a queued row in shared memory and narrows the threshold of
//            each filter by sums over the row; right for every row.
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
    double* rowmass;  // [rows] weight of the whole row, for rows left to the general kernel with a top_p and no top_k
    uint32_t* rowkey; // [rows] highest key, for rows left to the nucleus kernel
    int* queue;       // [0] rows left to the general kernel, then the rows
    int* nucleus;     // the same for the nucleus kernel; null: not launched
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
// The key before k, without the one of -0, which no logit has and which compares like +0's.
__device__ __forceinline__ uint32_t key_before(uint32_t k) { return k == 0x80000000u ? 0x7ffffffeu : k - 1u; }

// A row's settings with what is off made explicit.
enum Mode { kTopK, kAll, kMinP, kTopP, kGeneral };
struct RowSettings {
    float t;          // temperature
    double p, mp;     // p >= 1: off; mp = 0: off
    int k;            // 0: off
    Mode mode;
    __device__ __forceinline__ double scale() const { return 1.4426950408889634 / (double)t; }  // log2(e) / T
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
    s.t = t;
    if (!(t > 0.f)) {  // the greedy pick
        s.k = 1, s.t = 1.f, s.p = 2.0, s.mp = 0.0;
    } else if (s.p <= 0.0) {
        s.k = 1, s.p = 2.0;
    }
    // (a long top-k with a min-p and no top-p is the min-p's prefix, cut at k ranks)
    s.mode = s.k > kMaxTopK ? (s.p >= 1.0 && s.mp > 0.0 ? kMinP : kGeneral) : s.k ? kTopK : s.p < 1.0 ? kTopP : s.mp > 0.0 ? kMinP : kAll;
    return s;
}

// 2^(d c) for d c <= 0 to 2e-14 (0 below 2^-1021): d c = n + f with |f| <= 1/2, and the polynomial
// of degree 9 that interpolates 2^f in the Chebyshev nodes of [-1/2, 1/2].  13 operations of the
// double-precision pipe, 64 a clock and SM.  A table of 2^(j/32) in shared memory saves five of
// them and costs more in bank conflicts: 52 us against 21 for the summary of 64 rows of 262144.
__constant__ double kExp2[10] = {1.0000000000000135,    0.69314718055995,      0.240226506956403,     0.05550410866444768,
                                 0.009618129193942167,  0.0013333558230170627, 0.00015403433746224196, 1.5252657257186041e-05,
                                 1.3259646250270451e-06, 1.020869083593037e-07};
__device__ __forceinline__ double exp2_64(double d, double c) {
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: one unit in the last place is 1
    const double t = fma(d, c, magic);
    const double f = fma(d, c, magic - t);
    const int n = __double2loint(t);
    double q = kExp2[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) q = fma(q, f, kExp2[i]);
    // The bits of t are those of magic plus n as a 64-bit number (a NaN's are not near).
    const bool in = __double2hiint(t) - 0x43380000 == n >> 31 && n >= -1021;
    return in ? __hiloint2double(__double2hiint(q) + (n << 20), __double2loint(q)) : 0.0;
}
// exp((v - m) / T), 0 for logits that are never picked; +inf logits (m = +inf) share the whole
// weight.  Free of branches: the chains of several logits run beside one another (behind branches
// they ran one after the other, 350 clocks each: 48 us against 19 for 64 rows of 262144).
__device__ __forceinline__ double weight(float v, float m, double c) {
    const double w = exp2_64((double)v - (double)m, c);
    return v == m ? 1.0 : w;
}

// g4_softcap's arithmetic, but a mask (-inf) stays one; out of line, because 16 to 32 copies of it
// in code that seldom runs it cost more in instruction fetches than the calls.
__device__ __noinline__ float softcap(float v, float cap) { return v > -INFINITY ? tanhf(v / cap) * cap : v; }
__device__ __noinline__ float4 softcap4(float4 v, float cap) {
    return make_float4(softcap(v.x, cap), softcap(v.y, cap), softcap(v.z, cap), softcap(v.w, cap));
}
__device__ __forceinline__ float capped(float v, float cap) { return cap > 0.f ? softcap(v, cap) : v; }

// ---------------------------------------------------------------- summary --
// A warp takes 512 consecutive logits at a time as four chunks of 128.  kVec: rows are 16-byte
// aligned and a lane holds 4 consecutive logits of each chunk; else a lane holds logits lane,
// lane + 32, ... of it.  Groups of up to 128 lie inside a chunk, larger ones join chunks.
constexpr int kSumWarps = 8;
template <bool kVec>
__global__ void __launch_bounds__(kSumWarps * 32) sample_summary_kernel(const SampleParams P, int segments) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        P.queue[0] = 0;
        if (P.nucleus) P.nucleus[0] = 0;
    }
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
            const float4 f = __ldg(reinterpret_cast<const float4*>(row + index(i, 0)));
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
            for (int e = 0; e < 4; ++e) v[i][e] = softcap(v[i][e], P.cap);
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
            // fmaxf passes over NaN
            uint32_t k = logit_key(kVec ? fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3])) : v[i][u]);
            if (lanes == 32) {
                k = __reduce_max_sync(0xffffffffu, k);
            } else {
                for (int o = 1; o < lanes; o <<= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
            }
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
        const double c = st.scale();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int u = 0; u < U; ++u) sum[i][u] = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int u = kVec ? 0 : e;
                sum[i][u] += weight(v[i][e], key_logit(key[i][u]), c);  // a group without any: against NaN, 0
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

// The same for rows in 16-byte pieces and groups of 128 logits or more (vocabularies above 131072):
// a warp walks `blocks` blocks of 512 with the next one's loads in flight, and the four chunks'
// sums are reduced together (12 shuffles of a double where one after the other they take 40).
__global__ void __launch_bounds__(kSumWarps * 32) sample_summary_wide_kernel(const SampleParams P, int segments, int blocks) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        P.queue[0] = 0;
        if (P.nucleus) P.nucleus[0] = 0;
    }
    const int lane = threadIdx.x & 31;
    const int r = (int)(blockIdx.x / (unsigned)segments);
    const int warp = (int)(blockIdx.x - (unsigned)r * segments) * kSumWarps + (threadIdx.x >> 5);
    const float* row = P.logits + (size_t)r * P.ld;
    float4 next[4];
    auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = base + i * 128 + lane * 4;
            next[i] = at < P.vocab ? __ldg(reinterpret_cast<const float4*>(row + at))
                                   : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
    };
    int base = warp * blocks * 512;
    if (base >= P.vocab) return;
    load(base);
    const RowSettings st = row_settings(P, r);
    const bool mass = st.mode == kAll || st.mode == kTopP;
    const double c = mass ? st.scale() : 0.0;
    for (int k = 0; k < blocks && base < P.vocab; ++k, base += 512) {
        float v[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i][0] = next[i].x, v[i][1] = next[i].y, v[i][2] = next[i].z, v[i][3] = next[i].w;
        if (k + 1 < blocks) load(base + 512);
        if (P.cap > 0.f) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] = softcap(v[i][e], P.cap);
        }
        uint32_t key[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)  // fmaxf passes over NaN
            key[i] = __reduce_max_sync(0xffffffffu, logit_key(fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]))));
        if (P.gshift >= 8) key[0] = key[1] = max(key[0], key[1]), key[2] = key[3] = max(key[2], key[3]);
        if (P.gshift >= 9) key[0] = key[1] = key[2] = key[3] = max(key[0], key[2]);
        // Lane 8 i speaks for chunk i.
        const int i = lane >> 3, g = (base + i * 128) >> P.gshift;
        const bool writes = (lane & 7) == 0 && ((base + i * 128) & ((1 << P.gshift) - 1)) == 0 && g < P.groups;
        if (writes) P.gkey[(size_t)r * P.groups + g] = i < 2 ? (i == 0 ? key[0] : key[1]) : (i == 2 ? key[2] : key[3]);
        if (!mass) continue;
        double s[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float m = key_logit(key[q]);  // a group without any: NaN, and all weights 0
            s[q] = (weight(v[q][0], m, c) + weight(v[q][1], m, c)) + (weight(v[q][2], m, c) + weight(v[q][3], m, c));
        }
        const bool hi = lane & 16, odd = lane & 8;
        double a = hi ? s[2] : s[0], b = hi ? s[3] : s[1];
        a += __shfl_xor_sync(0xffffffffu, hi ? s[0] : s[2], 16);
        b += __shfl_xor_sync(0xffffffffu, hi ? s[1] : s[3], 16);
        double t = odd ? b : a;
        t += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (P.gshift >= 8) t += __shfl_xor_sync(0xffffffffu, t, 8);
        if (P.gshift >= 9) t += __shfl_xor_sync(0xffffffffu, t, 16);
        if (writes) P.gmass[(size_t)r * P.groups + g] = t;
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
    double t = s.d[flip][threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
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
    double y = lane < kWarps ? s.d[flip][lane] : 0.0;  // sums of the warps up to and with `lane`
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
        const double z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    *total = __shfl_sync(0xffffffffu, y, kWarps - 1);
    double before = __shfl_sync(0xffffffffu, y, w > 0 ? w - 1 : 0);
    if (w == 0) before = 0.0;
    double left = __shfl_up_sync(0xffffffffu, x, 1);
    if (lane == 0) left = 0.0;
    return before + left;
}

// Bitonic sort of n2 = a power of two up to kThreads 64-bit values in shared memory, largest first.
// Values stay in registers: partners less than 32 away come by shuffle, the others through `a` and
// `b` in turn, one barrier a step.
__device__ __forceinline__ void block_sort_desc(unsigned long long* a, unsigned long long* b, int n2) {
    const int t = threadIdx.x;
    __syncthreads();
    unsigned long long v = t < n2 ? a[t] : 0ull;
    bool second = true;  // the buffer that may be written: a's values have been read after the next barrier
    for (int size = 2; size <= n2; size <<= 1) {
        for (int step = size >> 1; step > 0; step >>= 1) {
            unsigned long long* const buf = second ? b : a;
            if (step >= 32) {
                buf[t] = v;
                __syncthreads();
                second = !second;
            }
            const unsigned long long o = step >= 32 ? buf[t ^ step] : __shfl_xor_sync(0xffffffffu, v, step);
            const bool larger = ((t & size) == 0) == ((t & step) == 0);  // this one keeps the larger
            v = (o > v) == larger ? o : v;
        }
    }
    __syncthreads();
    if (t < n2) a[t] = v;
    __syncthreads();
}
__device__ __forceinline__ int pow2_at_least(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

__device__ __forceinline__ double row_uniform(const SampleParams& P, int r) {
    const float u = P.how.uniform[r];
    return u >= 0.f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0;
}

// ----------------------------------------------------------------- finish --
constexpr int kFew = 256;
struct FinishShared {
    unsigned long long cand[kCand];  // key << 32 | ~index; then ~index << 32 | position
    unsigned long long cand2[kCand];
    double w[kCand];
    uint16_t glist[kMaxGroups];
    BlockScratch scratch;
    double zk;
    int n, ng, kept, found, pick;
    uint32_t hist[256], found_above, found_in;
    int rank[kFew];
    int begin[kThreads + 1], cursor[kThreads];
};

// Sorts S.cand[0 .. n), n <= kCand distinct values, largest first.  bin(value) in [0, kThreads) falls
// as the value rises: values go to their bin's place, and inside it (a handful, if bin spreads them)
// each counts the larger ones.  Two bitonic sorts of 2048 values in its place took 50 us of a row.
template <class Bin>
__device__ __forceinline__ void bin_sort_desc(FinishShared& S, int n, Bin bin) {
    const int t = threadIdx.x, lane = t & 31;
    S.cursor[t] = 0;
    __syncthreads();
    for (int i = t; i < n; i += kThreads) atomicAdd(&S.cursor[bin(S.cand[i])], 1);
    __syncthreads();
    const int own = S.cursor[t];
    int x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) S.begin[t >> 5] = x;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) before += w < t >> 5 ? S.begin[w] : 0;
    __syncthreads();
    S.begin[t] = S.cursor[t] = before + x - own;
    if (t == 0) S.begin[kThreads] = n;
    __syncthreads();
    for (int i = t; i < n; i += kThreads) {
        const unsigned long long v = S.cand[i];
        S.cand2[atomicAdd(&S.cursor[bin(v)], 1)] = v;
    }
    __syncthreads();
    for (int i = t; i < n; i += kThreads) {
        const unsigned long long v = S.cand2[i];
        const int b = bin(v), from = S.begin[b], to = S.begin[b + 1];
        int larger = 0;
        for (int j = from; j < to; ++j) larger += S.cand2[j] > v;
        S.cand[from + larger] = v;
    }
    __syncthreads();
}

// The end of a row with at most kFew candidates: ranks by counting (several threads per candidate)
// instead of sorts, whose 28 barriers for 128 candidates cost 6400 clocks.
template <class Leave>
__device__ __forceinline__ void finish_few(const SampleParams& P, FinishShared& S, const RowSettings& st, int r, int n,
                                           float m, double c, double u, double total, int& flip, Leave leave) {
    const int n2 = max(32, pow2_at_least(n)), parts = kThreads / n2, part = threadIdx.x / n2, i = threadIdx.x & (n2 - 1);
    const int t = threadIdx.x;
    if (i < n) {
        const unsigned long long me = S.cand[i];
        int above = 0;
#pragma unroll 4
        for (int j = part; j < n; j += parts) above += S.cand[j] > me;
        if (above) atomicAdd(&S.rank[i], above);
    }
    __syncthreads();
    unsigned long long* sorted = S.cand + kFew;
    if (t < n) sorted[S.rank[t]] = S.cand[t];
    __syncthreads();
    const int limit = st.k ? min(st.k, n) : n;
    const double w = t < limit ? weight(key_logit((uint32_t)(sorted[t] >> 32)), m, c) : 0.0;
    if (t < n) S.w[t] = w;
    if (t == 0) S.kept = limit;
    double all;
    const double run = block_prefix(w, S.scratch, flip, &all) + w;
    if (st.mode != kTopP) total = all;
    const double need = st.p * total;
    if (st.mode == kTopP && st.mp == 0.0 && all < need) {
        leave(total);
        return;
    }
    // kept: the shortest prefix of the filters.
    const unsigned ends = __ballot_sync(
        0xffffffffu, t < limit && ((st.p < 1.0 && run >= need) || (t + 1 < limit && st.mp > 0.0 && S.w[t + 1] < st.mp)));
    if (ends && (t & 31) == 0) atomicMin(&S.kept, t + __ffs(ends));
    __syncthreads();
    const int kept = S.kept;
    if (t == kept - 1) S.zk = run;
    // What lies before each kept one in index order.
    double* before = S.w + kFew;  // [parts][n2]
    if (i < kept) {
        const uint32_t me = (uint32_t)sorted[i];  // ~index
        double s0 = 0.0;
#pragma unroll 4
        for (int j = part; j < kept; j += parts) s0 += (uint32_t)sorted[j] > me ? S.w[j] : 0.0;
        before[part * n2 + i] = s0;
    }
    __syncthreads();
    const double target = u * S.zk;
    int mine = -1, at = -1;
    if (t < kept && w > 0.0) {
        double s0 = 0.0;
        for (int q = 0; q < parts; ++q) s0 += before[q * n2 + t];
        mine = (int)(0xffffffffu - (uint32_t)sorted[t]);
        // the highest index with no more than the target before it
        if (s0 <= target) at = mine;
    }
    at = __reduce_max_sync(0xffffffffu, at);
    if (at >= 0 && (t & 31) == 0) atomicMax(&S.pick, at);
    __syncthreads();
    if (mine >= 0 && mine == S.pick) {
        P.ids[r] = mine;
        if (P.probs) P.probs[r] = (float)(w / S.zk);
    }
}

__global__ void __launch_bounds__(kThreads, 2) sample_finish_kernel(const SampleParams P, int vec) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    FinishShared& S = *reinterpret_cast<FinishShared*>(smem_raw);
    pdl_trigger();
    if (threadIdx.x == 0) S.n = S.ng = S.kept = 0, S.pick = -1;
    if (threadIdx.x < kFew) S.rank[threadIdx.x] = 0;
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
    auto leave = [&](double mass) {  // to one of the kernels that follow
        if (threadIdx.x != 0) return;
        int* const queue = P.nucleus && st.mode == kTopP && st.mp == 0.0 ? P.nucleus : P.queue;
        P.rowmass[r] = mass, P.rowkey[r] = top;
        queue[1 + atomicAdd(queue, 1)] = r;
    };
    if (st.mode == kGeneral) {
        leave(0.0);
        return;
    }
    if (st.k == 1) {
        // One rank: the lowest index of the highest logit, from the first group that has it.  However many
        // share it, so no such row is left to the kernels that follow: a call with temperatures alone has none.
        uint32_t first = 0;  // ~ the group
#pragma unroll
        for (int i = 0; i < KG; ++i)
            if (key[i] == top) first = max(first, ~(uint32_t)(i * kThreads + threadIdx.x));
        const int g = (int)~block_max(first, S.scratch, flip);
        if (threadIdx.x < 32) {
            for (int o = 0; o < gs; o += 32) {
                const int i = (g << P.gshift) + o + (int)threadIdx.x;
                const bool has = o + (int)threadIdx.x < gs && i < P.vocab && logit_key(capped(row[i], P.cap)) == top;
                const unsigned who = __ballot_sync(0xffffffffu, has);
                if (!who) continue;
                if ((int)threadIdx.x == __ffs(who) - 1) {
                    P.ids[r] = i;
                    if (P.probs) P.probs[r] = 1.f;
                }
                break;
            }
        }
        return;
    }
    if (st.mode == kAll) {
        // Groups in index order, four consecutive ones per thread.
        const double c = st.scale();
        const double* gm = P.gmass + (size_t)r * G;
        double x[KG], own = 0.0, total;
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            const int g = threadIdx.x * KG + i;
            x[i] = g < G && gk[g] ? gm[g] * weight(key_logit(gk[g]), m, c) : 0.0;
            own += x[i];
        }
        const double before = block_prefix(own, S.scratch, flip, &total);
        const double target = u * total;
        // The thread whose groups hold the target; its first group past it (the last positive one
        // where rounding leaves none).
        const unsigned holds = __ballot_sync(0xffffffffu, own > 0.0 && before <= target);  // the highest such thread wins
        if (holds && (threadIdx.x & 31) == 0) atomicMax(&S.ng, (int)threadIdx.x + 32 - __clz(holds));
        __syncthreads();
        if (S.ng == (int)threadIdx.x + 1) {
            double run = before;
            int g = 0;
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                if (x[i] > 0.0 && run <= target) {
                    g = threadIdx.x * KG + i;
                    S.w[0] = run;
                }
                run += x[i];
            }
            S.n = g;
        }
        __syncthreads();
        if (threadIdx.x < 32) {  // the pick inside the group
            const int lane = threadIdx.x;
            double run = S.w[0];
            int pick = -1;
            double wp = 0.0;
            for (int o = 0; o < gs; o += 32) {
                const int i = (S.n << P.gshift) + o + lane;
                double w = 0.0;
                if (o + lane < gs && i < P.vocab) {
                    const float v = capped(row[i], P.cap);
                    if (logit_key(v)) w = weight(v, m, c);
                }
                double s = w;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, s, d);
                    if (lane >= d) s += y;
                }
                const unsigned past = __ballot_sync(0xffffffffu, w > 0.0 && run + s > target);
                const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
                const int from = past ? __ffs(past) - 1 : some ? 31 - __clz(some) : 0;
                if (some) {
                    pick = (S.n << P.gshift) + o + from;
                    wp = __shfl_sync(0xffffffffu, w, from);
                }
                if (past) break;
                run += __shfl_sync(0xffffffffu, s, 31);
            }
            if (lane == 0) {
                P.ids[r] = pick;
                if (P.probs) P.probs[r] = (float)(wp / total);
            }
        }
        return;
    }

    // Candidates: every logit with key >= bound, from the groups whose maximum reaches it.
    const double c = st.scale();
    uint32_t bound;
    double total = 0.0;
    const bool whole = P.vocab <= kCand;  // every logit may be a candidate
    // A top-p with a min-p: either the prefix ends among the logits that weigh mp or more, or all of
    // those are kept; no others are looked at.
    const bool floored = st.mode == kTopP && st.mp > 0.0;
    if (floored) {
        const double* gm = P.gmass + (size_t)r * G;
        double own = 0.0;
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            const int g = i * kThreads + threadIdx.x;
            own += g < G ? weight(key_logit(key[i]), m, c) * gm[g] : 0.0;
        }
        total = block_sum(own, S.scratch, flip);
    }
    if (st.mode == kMinP || floored) {
        // The lowest key that weighs mp or more (w falls with the key): every thread tries one of 512
        // keys of what is left.
        uint32_t lo = kLowestKey, hi = top;  // hi keeps
        const double at = (double)m + (double)st.t * log(st.mp);  // where it is, but for roundings
        if (m < 3.0e38f && at > -3.0e38) {
            const uint32_t k = logit_key((float)at);
            const uint32_t a = max(k, kLowestKey + 200u) - 200u, b = min(k + 200u, top);
            if (a < b && weight(key_logit(b), m, c) >= st.mp && weight(key_logit(a), m, c) < st.mp) lo = a, hi = b;
        }
        while (lo < hi) {
            const uint32_t span = hi - lo;
            auto cut = [&](int t) { return lo + (uint32_t)((unsigned long long)span * (unsigned)t / kThreads); };
            const int below = __syncthreads_count(weight(key_logit(cut(threadIdx.x)), m, c) < st.mp);
            const uint32_t nhi = below < kThreads ? cut(below) : hi;
            lo = below > 0 ? cut(below - 1) + 1 : lo;
            hi = nhi;
        }
        bound = hi;
    } else {
        // The highest bound that the group maxima reach often enough (top-k: k of them; top-p: maxima
        // that weigh what is needed, in units of 2^-20), by a histogram of what is left in 256 parts.
        low = ~block_max(low, S.scratch, flip);
        uint32_t val[KG], need;
        if (st.mode == kTopK) {
#pragma unroll
            for (int i = 0; i < KG; ++i) val[i] = 1;
            need = (uint32_t)st.k;
        } else {
            const double* gm = P.gmass + (size_t)r * G;
            double own = 0.0;
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const int g = i * kThreads + threadIdx.x;
                const double x = weight(key_logit(key[i]), m, c);
                val[i] = (uint32_t)(x * 1048576.0);
                own += g < G ? x * gm[g] : 0.0;
            }
            total = block_sum(own, S.scratch, flip);
            const double fixed = st.p * total * 1048576.0 + kMaxGroups;
            if (fixed > 2147483648.0 && !whole) {  // more than all maxima can weigh
                leave(total);
                return;
            }
            need = (uint32_t)fmin(fixed, 4294967295.0);
        }
        uint32_t lo = low, hi = top + 1, above = 0;
        bool enough = false;
        if (st.mode == kTopK && st.k <= kThreads / 4) {
            // Few: the maxima of each thread's four groups will do, one barrier per halving.
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < KG; ++i) mine = max(mine, key[i]);
            if (__syncthreads_count(mine >= low) >= st.k) {
                enough = true;
                while (hi - lo > 1) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    const int count = __syncthreads_count(mine >= mid);
                    if (count >= st.k) lo = mid;
                    else hi = mid;
                    if (count >= st.k && count <= st.k + st.k / 8 + 4) break;
                }
            }
        }
        for (bool done = enough; !done;) {
            const uint32_t span = hi - lo;
            const int shift = max(0, 24 - __clz(span - 1 | 1u));
            if (threadIdx.x < 256) S.hist[threadIdx.x] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < KG; ++i)
                if (key[i] >= lo && key[i] < hi && key[i]) atomicAdd(&S.hist[(key[i] - lo) >> shift], val[i]);
            __syncthreads();
            if (threadIdx.x < 32) {  // lane l: parts 8 l .. 8 l + 7; sums from the top
                uint32_t h[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += h[i] = S.hist[threadIdx.x * 8 + i];
                uint32_t from = sum;  // of this lane's parts and all above
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t x = __shfl_down_sync(0xffffffffu, from, o);
                    if (threadIdx.x + o < 32) from += x;
                }
                const unsigned ok = __ballot_sync(0xffffffffu, above + from >= need);
                if (ok == 0u) {
                    if (threadIdx.x == 0) S.found = -1;
                } else if ((int)threadIdx.x == 31 - __clz(ok)) {
                    uint32_t run = above + from - sum;
                    int at = 7;
#pragma unroll
                    for (int i = 7; i >= 0; --i) {
                        at = i;
                        if (run + h[i] >= need) break;
                        run += h[i];
                    }
                    S.found = threadIdx.x * 8 + at;
                    S.found_above = run;
                    S.found_in = h[at];
                }
            }
            __syncthreads();
            const int at = S.found;
            if (at < 0) break;  // all of the maxima are not enough
            enough = true;
            const uint32_t part = lo + ((uint32_t)at << shift);
            if (hi - part > 1u << shift) hi = part + (1u << shift);
            lo = part;
            above = S.found_above;
            if (shift == 0 || above + S.found_in <= need + need / 8 + (st.mode == kTopK ? 4 : 0)) done = true;
        }
        if (!enough && st.mode == kTopP && !whole) {
            leave(total);
            return;
        }
        bound = enough ? lo : 1u;
    }
#pragma unroll
    for (int i = 0; i < KG; ++i)
        if (key[i] >= bound) S.glist[atomicAdd(&S.ng, 1)] = (uint16_t)(i * kThreads + threadIdx.x);
    __syncthreads();
    const int ng = S.ng;
    // Too many to read here (a short row is tried whole): by one CTA 1024 groups take 60 us, by the
    // general kernel's cluster the whole row some 20.
    if (ng > (st.mode == kTopK ? kCand / 2 : kCand / 8) && P.vocab > 4 * kCand) {
        leave(total);
        return;
    }
    const int qshift = P.gshift - 2, quads = ng << qshift;  // four consecutive logits at a time
    const float least = key_logit(max(bound, kLowestKey));  // (NaN compares false)
    auto place = [&](int q) { return ((int)S.glist[q >> qshift] << P.gshift) + (q & ((1 << qshift) - 1)) * 4; };
    auto fetch = [&](int at) {
        float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (vec) {
            if (at < P.vocab) f = __ldg(reinterpret_cast<const float4*>(row + at));
        } else {
            if (at < P.vocab) f.x = __ldg(row + at);
            if (at + 1 < P.vocab) f.y = __ldg(row + at + 1);
            if (at + 2 < P.vocab) f.z = __ldg(row + at + 2);
            if (at + 3 < P.vocab) f.w = __ldg(row + at + 3);
        }
        return f;
    };
    // Eight in flight: the some hundred groups of a usual row are one round trip.  A bit per logit
    // first; the few that count are read once more: 4.3 of a row's 18 thousand clocks (every four
    // logits handed to a function that lists them, three in flight: 7.5 thousand).  64 registers, at
    // the price of a few spills: with 82, one CTA per SM, 256 rows took 65 us instead of 59.
    constexpr int B = 8;
#pragma unroll 1
    for (int q = threadIdx.x; q < quads; q += B * kThreads) {
        float4 f[B];
#pragma unroll
        for (int b = 0; b < B; ++b) f[b] = fetch(q + b * kThreads < quads ? place(q + b * kThreads) : P.vocab);
        if (P.cap > 0.f) {
#pragma unroll
            for (int b = 0; b < B; ++b) f[b] = softcap4(f[b], P.cap);
        }
        uint32_t bits = 0;
#pragma unroll
        for (int b = 0; b < B; ++b)
            bits |= (f[b].x >= least ? 1u : 0u) << 4 * b | (f[b].y >= least ? 2u : 0u) << 4 * b |
                    (f[b].z >= least ? 4u : 0u) << 4 * b | (f[b].w >= least ? 8u : 0u) << 4 * b;
        if (!bits) continue;
        int to = atomicAdd(&S.n, __popc(bits));
#pragma unroll 1
        for (; bits && to < kCand; bits &= bits - 1, ++to) {
            const int k = __ffs(bits) - 1, i = place(q + (k >> 2) * kThreads) + (k & 3);
            S.cand[to] = (unsigned long long)logit_key(capped(__ldg(row + i), P.cap)) << 32 | (0xffffffffu - (unsigned)i);
        }
    }
    __syncthreads();
    const int n = S.n;
    if (n > kCand) {
        leave(total);
        return;
    }
    if (n <= kFew) {
        finish_few(P, S, st, r, n, m, c, u, total, flip, leave);
        return;
    }
    uint32_t least_key = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) least_key = max(least_key, ~(uint32_t)(S.cand[i] >> 32));
    const float lowest = key_logit(~block_max(least_key, S.scratch, flip)), parts = (float)kThreads / (m - lowest);
    bin_sort_desc(S, n, [&](unsigned long long v) {
        if (!(parts < 3.0e38f)) return 0;  // equal logits, or infinite ones
        return kThreads - 1 - min(kThreads - 1, (int)((key_logit((uint32_t)(v >> 32)) - lowest) * parts));
    });
    // Ranks 4t .. 4t + 3: weights, their running sum and where it ends the prefix.
    constexpr int E = kCand / kThreads;
    const int limit = st.k ? min(st.k, n) : n;
    double w[E], own = 0.0, all;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = threadIdx.x * E + e;
        w[e] = i < limit ? weight(key_logit((uint32_t)(S.cand[i] >> 32)), m, c) : 0.0;
        if (i < n) S.w[i] = w[e];
        own += w[e];
    }
    double run = block_prefix(own, S.scratch, flip, &all);
    if (st.mode != kTopP) total = all;
    const double need = st.p * total;
    if (st.mode == kTopP && st.mp == 0.0 && all < need) {
        leave(total);
        return;
    }
    // kept: the longest prefix that the filters leave.
    if (threadIdx.x == 0) S.kept = limit;
    __syncthreads();
    int upto = limit;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = threadIdx.x * E + e;
        run += w[e];
        if (i < limit && ((st.p < 1.0 && run >= need) || (i + 1 < limit && st.mp > 0.0 && S.w[i + 1] < st.mp)))
            upto = min(upto, i + 1);
    }
    upto = __reduce_min_sync(0xffffffffu, upto);
    if ((threadIdx.x & 31) == 0 && upto < limit) atomicMin(&S.kept, upto);
    __syncthreads();
    const int kept = S.kept;
    // The kept ones in index order.
    for (int i = threadIdx.x; i < kept; i += kThreads)
        S.cand[i] = (S.cand[i] & 0xffffffffull) << 32 | (unsigned)i;  // ~index << 32 | position: lowest index first
    __syncthreads();
    bin_sort_desc(S, kept, [&](unsigned long long v) {
        return (int)((unsigned long long)(0xffffffffu - (uint32_t)(v >> 32)) * kThreads / (unsigned)P.vocab);
    });
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
    const int last = __reduce_max_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0 && last >= 0) atomicMax(&S.n, last);
    __syncthreads();
    if (mine >= 0 && mine == S.n) {
        const unsigned long long c = S.cand[mine];
        P.ids[r] = (int)(0xffffffffu - (unsigned)(c >> 32));
        if (P.probs) P.probs[r] = (float)(S.w[(uint32_t)c] / all);
    }
}

// ---------------------------------------------------------------- nucleus --
// A cluster of up to 8 CTAs takes a queued row with a top-p alone and reads it twice, from L2 where
// the batch fits there.  No logit that weighs less than (1 - p) total / vocab is kept (all of those
// together weigh less than what top-p may drop), so the logits from there to the highest are
// counted in 8192 parts of even width.  A part's number times the weight of its middle is right to
// a factor of half a part's width, so the parts where the prefix can end are known for certain:
// some 0.1 % of the mass around it.  The second pass sums what lies above them exactly and lists
// what lies in them; CTA 0 finds the end of the prefix in the list.  The sums of the segments (512
// logits), with what is kept of the list, then give the pick's segment.  Weights of the list are
// summed as integers, so that the order of the list, which the atomics decide, does not matter.
// Rows whose list is too long (a top_p close to 1 over a flat row, or equal logits) go on to the
// general kernel.
//
// Its share of a call with 64 rows of 262144 logits and a top_p around 0.9 (some twenty rows come
// here): 53 us, of the general kernel in its place 118; 200 such rows: the call takes 260 us instead
// of 528, one row 30 instead of 35.  What bounds it is the chain of steps of a row, about 66
// thousand clocks of two passes (four segments of a warp one after the other in each) and seven
// barriers of the cluster.  1024 threads with one segment in registers: with 512 threads and the
// next segment's loads in flight, at two CTAs per SM (64 registers, spills), the call took 128 us,
// at one 106; this way 101.
constexpr int kMaxCluster = 16;
constexpr int kMaxRanks = 8;   // of the nucleus kernel: a thread has one of the parts or more
constexpr int kWide = 1024;    // its threads
constexpr int kWideWarps = kWide / 32;
constexpr int kParts = 8192;
constexpr int kList = 8192;
constexpr int kSegment = 512;      // at most kWide segments per CTA
constexpr int kFixed = 50;         // bits of a listed weight: kList of them reach 2^63, and lose 2^-37 of the highest in all
constexpr int kCount = 256;      // listed logits ranked by counting

struct NucleusShared {
    union {
        uint32_t own[kParts + 32];         // this CTA's numbers, and a lane's of what lies below
        unsigned long long listed[kList];  // all lists: key << 32 | ~index
    };
    union {
        uint32_t num[kParts];  // the row's numbers in this CTA's parts
        uint2 list[kList];     // key, index
    };
    union {
        float staged[kWideWarps][kSegment];  // a warp's segment
        unsigned long long listed_weight[kList];
        double weight[kSegment + kSegment / 16];  // of the pick's segment
    };
    double seg[kWide];  // per segment: weight above the listed parts
    unsigned long long seg_listed[kWide];
    unsigned long long few_weight[kWide];
    uint16_t few[kCount];
    double scratch[2 * kWideWarps];
    double xpart[kMaxCluster];                // per rank: estimated weight of its parts
    double xmass[kMaxCluster];                // per rank: weight above
    unsigned long long xlisted[kMaxCluster];  // per rank: kept of the list
    int xn[kMaxCluster];                      // per rank: length of the list
    int xfirst[kMaxCluster], xlast[kMaxCluster];
    double start;
    unsigned long long past;
    int n, first, last, at, nfew, fine;
    uint32_t end_key;  // the prefix ends with this key,
    int end_index;     // of equal ones at this index; -1: not found
};

// Out of line: for code that runs once or twice per row.
__device__ __noinline__ double exp2_call(double d, double c) { return exp2_64(d, c); }
template <class T>
struct Scan {
    T before, all;
};
// Sum over the threads before this one, and over all.
template <class T>
__device__ __noinline__ Scan<T> block_scan(T v, void* scratch) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    T* const sums = static_cast<T*>(scratch);
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[w] = x;
    __syncthreads();
    T y = sums[lane];  // a warp each
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    static_assert(kWideWarps == 32, "a lane per warp");
    const T warps = __shfl_sync(0xffffffffu, y, w > 0 ? w - 1 : 0), left = __shfl_up_sync(0xffffffffu, x, 1);
    return {(w > 0 ? warps : T(0)) + (lane > 0 ? left : T(0)), __shfl_sync(0xffffffffu, y, 31)};
}

__global__ void __launch_bounds__(kWide, 1) sample_nucleus_kernel(const SampleParams P, int vec) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    NucleusShared& S = *reinterpret_cast<NucleusShared*>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x / ranks >= P.nucleus[0]) return;  // nothing for this cluster
    cluster.sync();  // every CTA of the cluster runs before any reaches into another's shared memory
    const int segments = ((P.vocab + kSegment - 1) / kSegment + ranks - 1) / ranks;  // of a CTA
    const int first = rank * segments * kSegment;
    const int queued = P.nucleus[0];
#pragma unroll 1
    for (int q = blockIdx.x / ranks; q < queued; q += gridDim.x / ranks, cluster.sync()) {
        const int r = P.nucleus[1 + q];
        const float* row = P.logits + (size_t)r * P.ld;
        const float temperature = P.how.temperature ? P.how.temperature[r] : 1.f;
        const double p = (double)P.how.top_p[r], total = P.rowmass[r], t = p * total;
        const double c = 1.4426950408889634 / (double)temperature;
        const double u = row_uniform(P, r);
        const float m = key_logit(P.rowkey[r]);
        auto leave = [&]() {
            if (rank == 0 && threadIdx.x == 0) P.queue[1 + atomicAdd(P.queue, 1)] = r;
        };
        // The lowest logit of interest, rounded down (by far more than the roundings of this line).
        const float bound = log2f((float)((1.0 - p) * total) / (float)P.vocab) - 0.01f;
        float a = fmaf(bound * 0.6931472f, temperature, m);
        a -= fabsf(a) * 1e-6f + fabsf(m) * 1e-6f;
        const float scale = (float)kParts / (m - a);
        const double part = 1.0 / (double)scale, width = c * part;  // of a part: in logits, in powers of two
        if (!(a > -3.0e38f && m < 3.0e38f && scale > 0.f && scale < 3.0e38f && width < 1.0 / 64.0)) {
            leave();
            continue;
        }
        auto part_of = [&](float v) { return min(kParts - 1, (int)((v - a) * scale)); };
        // Highest key of quarter `lane` of a segment (lanes 0 .. 3), from the groups.
        auto quarter_key = [&](int s) {
            uint32_t k = 0;
            const int at = first + s * kSegment + lane * 128;
            if (lane < 4 && s < segments && at < P.vocab) {
                const int g = at >> P.gshift, end = min(P.groups, g + max(1, 128 >> P.gshift));
#pragma unroll 1
                for (int i = g; i < end; ++i) k = max(k, P.gkey[(size_t)r * P.groups + i]);
            }
            return k;
        };
        // f(s, quarters read, lane's 16 logits) for each of the warp's segments with a logit from `least` on.  Quarters
        // without (by their highest key) are not read.
        auto each_segment = [&](float least, auto f) {
            uint32_t key = quarter_key(warp);
#pragma unroll 1
            for (int s = warp; s < segments; s += kWideWarps) {
                const unsigned wanted = __ballot_sync(0xffffffffu, key_logit(key) >= least);  // (key 0 is a NaN's)
                key = quarter_key(s + kWideWarps);
                if (!wanted) continue;
                float v[16];
                const int base = first + s * kSegment;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[4 * i] = v[4 * i + 1] = v[4 * i + 2] = v[4 * i + 3] = -INFINITY;
                    if (!(wanted >> i & 1u)) continue;
                    if (vec) {
                        const int at = base + i * 128 + lane * 4;
                        if (at < P.vocab) {
                            const float4 q4 = __ldg(reinterpret_cast<const float4*>(row + at));
                            v[4 * i] = q4.x, v[4 * i + 1] = q4.y, v[4 * i + 2] = q4.z, v[4 * i + 3] = q4.w;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (base + i * 128 + e * 32 + lane < P.vocab) v[4 * i + e] = __ldg(row + base + i * 128 + e * 32 + lane);
                    }
                }
                if (P.cap > 0.f) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] = softcap(v[k], P.cap);
                }
                f(s, wanted, v);
            }
        };
        {
            uint4* const z = reinterpret_cast<uint4*>(S.own);
#pragma unroll 1
            for (int i = threadIdx.x; i < kParts / 4; i += kWide) z[i] = make_uint4(0, 0, 0, 0);
        }
        S.seg[threadIdx.x] = 0.0;
        S.seg_listed[threadIdx.x] = 0;
        if (threadIdx.x == 0) S.n = S.first = S.last = S.nfew = 0, S.at = S.end_index = S.fine = -1, S.past = 0;
        __syncthreads();
        each_segment(a, [&](int, unsigned wanted, const float (&v)[16]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(wanted >> i & 1u)) continue;
#pragma unroll
                for (int k = 4 * i; k < 4 * i + 4; ++k)
                    atomicAdd(&S.own[v[k] >= a ? part_of(v[k]) : kParts + lane], 1u);  // free of branches
            }
        });
        cluster.barrier_arrive();
        // This CTA's share of the parts, from the top, E per thread.
        const int E = kParts / kWide / ranks, top = kParts - 1 - (rank * kWide + (int)threadIdx.x) * E;
        const double step = exp2_64(-width, 1.0);
        const double wtop = exp2_64((double)a + ((double)top + 0.5) * part - (double)m, c);
        const double off = exp2_64(-0.51 * width, 1.0);  // a part's true weight: the estimate times off .. 1 / off
        double x = 0.0, w = wtop;
        cluster.barrier_wait();
#pragma unroll 2
        for (int e = 0; e < E; ++e, w *= step) {
            uint32_t n = 0;
#pragma unroll 4
            for (int k = 0; k < ranks; ++k) n += *cluster.map_shared_rank(&S.own[top - e], k);
            S.num[threadIdx.x * E + e] = n;
            x += (double)n * w;
        }
        const Scan<double> parts = block_scan(x, S.scratch);
        if ((int)threadIdx.x < ranks) *cluster.map_shared_rank(&S.xpart[rank], threadIdx.x) = parts.all;
        cluster.sync();
        double run = parts.before;
#pragma unroll 1
        for (int k = 0; k < rank; ++k) run += S.xpart[k];
        int hi = -1, lo = -1;
        w = wtop;
#pragma unroll 1
        for (int e = 0; e < E; ++e, w *= step) {
            run += (double)S.num[threadIdx.x * E + e] * w;
            if (hi < 0 && run >= t * off) hi = top - e;
            if (lo < 0 && run * off >= t) lo = top - e;
        }
        hi = __reduce_max_sync(0xffffffffu, hi), lo = __reduce_max_sync(0xffffffffu, lo);
        if (lane == 0 && hi >= 0) atomicMax(&S.last, hi);
        if (lane == 0 && lo >= 0) atomicMax(&S.first, lo);
        __syncthreads();
        if ((int)threadIdx.x < ranks) {
            *cluster.map_shared_rank(&S.xfirst[rank], threadIdx.x) = S.first;
            *cluster.map_shared_rank(&S.xlast[rank], threadIdx.x) = S.last;
        }
        cluster.sync();
        int b0 = 0, b1 = 0;  // the prefix ends in these parts
#pragma unroll 1
        for (int k = 0; k < ranks; ++k) b0 = max(b0, S.xfirst[k]), b1 = max(b1, S.xlast[k]);
        // The values of the list, a float more on each side: only what is listed has to be in there.
        const uint32_t klo = logit_key((float)((double)a + (double)b0 * part)), khi = logit_key((float)((double)a + (double)(b1 + 1) * part));
        const float least = b0 > 0 ? key_logit(klo - 1) : a, past_list = b1 < kParts - 1 ? key_logit(khi + 1) : INFINITY;
        each_segment(least, [&](int s, unsigned wanted, const float (&v)[16]) {
            // What lies above is written side by side, so that full warps weigh it.
            int count = 0;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(wanted >> i & 1u)) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = v[4 * i + e];
                    if (!__any_sync(0xffffffffu, x >= least)) continue;
                    const unsigned above = __ballot_sync(0xffffffffu, x >= past_list);
                    if (x >= past_list) {
                        S.staged[warp][count + __popc(above & ((1u << lane) - 1u))] = x;
                    } else if (x >= least) {
                        const int at = atomicAdd(&S.n, 1);
                        if (at < kList)
                            S.list[at] = make_uint2(logit_key(x), (uint32_t)(first + s * kSegment + i * 128 + (vec ? lane * 4 + e : e * 32 + lane)));
                    }
                    count += __popc(above);
                }
            }
            if (count == 0) return;
            __syncwarp();
            double sum = 0.0;
#pragma unroll 2
            for (int j = lane; j < count; j += 32) sum += weight(S.staged[warp][j], m, c);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) S.seg[s] = sum;
        });
        __syncthreads();
        const Scan<double> segs = block_scan(S.seg[threadIdx.x], S.scratch);
        if ((int)threadIdx.x < ranks) {
            *cluster.map_shared_rank(&S.xmass[rank], threadIdx.x) = segs.all;
            *cluster.map_shared_rank(&S.xn[rank], threadIdx.x) = S.n;
        }
        cluster.sync();
        double above = 0.0;
        int n = 0;
#pragma unroll 1
        for (int k = 0; k < ranks; ++k) above += S.xmass[k], n += S.xn[k];
        if (n > kList) {
            leave();
            continue;
        }
        // Listed weights in units of 2^-kFixed of a power of two that none exceeds.
        const double high = fmin((double)a + ((double)b1 + 1.01) * part, (double)m);
        const int e2 = kFixed - (int)ceil((high - (double)m) * c);
        const double unit = __hiloint2double((1023 - e2) << 20, 0), per = __hiloint2double((1023 + e2) << 20, 0);
        auto fixed = [&](uint32_t key) {
            const float v = key_logit(key);
            return (unsigned long long)((v == m ? 1.0 : exp2_call((double)v - (double)m, c)) * per);
        };
        if (rank == 0) {
#pragma unroll 1
            for (int j = threadIdx.x; j < n; j += kWide) {
                int i = j, k = 0;
                while (i >= S.xn[k]) i -= S.xn[k++];
                const uint2 f = *cluster.map_shared_rank(&S.list[i], k);
                S.listed[j] = (unsigned long long)f.x << 32 | (0xffffffffu - f.y);
                S.listed_weight[j] = fixed(f.x);
                if (j < kCount) S.few[j] = (uint16_t)j;
            }
            __syncthreads();
            const double need = (t - above) * per;
            unsigned long long past = 0;  // what the listed above those to rank weigh
            int left = n;
            if (n > kCount) {
                // 1024 parts of even width again: what is listed in the one where the prefix ends is ranked.
                const float from = (float)((double)a + (double)b0 * part), fine = (float)kWide * scale / (float)(b1 + 1 - b0);
                auto fine_of = [&](unsigned long long f) {
                    return max(0, min(kWide - 1, (int)((key_logit((uint32_t)(f >> 32)) - from) * fine)));
                };
                S.few_weight[threadIdx.x] = 0;
                __syncthreads();
#pragma unroll 2
                for (int j = threadIdx.x; j < n; j += kWide) atomicAdd(&S.few_weight[fine_of(S.listed[j])], S.listed_weight[j]);
                __syncthreads();
                const unsigned long long mine = S.few_weight[kWide - 1 - threadIdx.x];
                const Scan<unsigned long long> sc = block_scan(mine, S.scratch);
                if (!((double)sc.before >= need) && (double)(sc.before + mine) >= need) S.fine = kWide - 1 - (int)threadIdx.x, S.past = sc.before;
                __syncthreads();
                const int fine_at = S.fine;
                past = S.past;
#pragma unroll 1
                for (int j = threadIdx.x; j < n; j += kWide) {
                    if (fine_of(S.listed[j]) != fine_at) continue;
                    const int at = atomicAdd(&S.nfew, 1);
                    if (at < kCount) S.few[at] = (uint16_t)j;
                }
                __syncthreads();
                left = S.nfew;
            }
            if (left <= kCount && (int)threadIdx.x < left) {
                const int mine = S.few[threadIdx.x];
                const unsigned long long me = S.listed[mine];
                unsigned long long upto = past;
#pragma unroll 4
                for (int j = 0; j < left; ++j) {
                    const int i = S.few[j];
                    upto += S.listed[i] >= me ? S.listed_weight[i] : 0ull;
                }
                if ((double)upto >= need && !((double)(upto - S.listed_weight[mine]) >= need)) {  // one of them at most
#pragma unroll 1
                    for (int k = 0; k < ranks; ++k) {
                        *cluster.map_shared_rank(&S.end_key, k) = (uint32_t)(me >> 32);
                        *cluster.map_shared_rank(&S.end_index, k) = (int)(0xffffffffu - (uint32_t)me);
                    }
                }
            }
        }
        cluster.sync();
        const uint32_t end_key = S.end_key;
        const int end_index = S.end_index;
        if (end_index < 0) {
            leave();
            continue;
        }
        unsigned long long listed = 0;
#pragma unroll 1
        for (int j = threadIdx.x; j < S.n; j += kWide) {
            const uint2 f = S.list[j];
            if (f.x > end_key || (f.x == end_key && (int)f.y <= end_index)) {
                const unsigned long long y = fixed(f.x);
                listed += y;
                atomicAdd(&S.seg_listed[((int)f.y - first) / kSegment], y);
            }
        }
        listed = block_scan(listed, S.scratch).all;
        if ((int)threadIdx.x < ranks) *cluster.map_shared_rank(&S.xlisted[rank], threadIdx.x) = listed;
        cluster.sync();
        // The last CTA, segment and lane with something at or below the target hold the pick.
        double in_rank = 0.0, upto_rank = 0.0;
        if (lane < ranks) in_rank = S.xmass[lane] + (double)S.xlisted[lane] * unit;
        upto_rank = in_rank;
#pragma unroll
        for (int o = 1; o < kMaxCluster; o <<= 1) {
            const double z = __shfl_up_sync(0xffffffffu, upto_rank, o);
            if (lane >= o) upto_rank += z;
        }
        const double kept = __shfl_sync(0xffffffffu, upto_rank, kMaxCluster - 1), target = u * kept;
        double before = __shfl_up_sync(0xffffffffu, upto_rank, 1);
        if (lane == 0) before = 0.0;
        const unsigned holds = __ballot_sync(0xffffffffu, lane < ranks && in_rank > 0.0 && before <= target);
        const int owner = 31 - __clz(holds | 1u);
        const double start = __shfl_sync(0xffffffffu, before, owner);
        if (owner != rank) continue;
        const double y = S.seg[threadIdx.x] + (double)S.seg_listed[threadIdx.x] * unit;
        before = start + block_scan(y, S.scratch).before;
        const int held = __reduce_max_sync(0xffffffffu, y > 0.0 && before <= target ? (int)threadIdx.x : -1);
        if (lane == 0 && held >= 0) atomicMax(&S.at, held);
        __syncthreads();
        if (S.at == (int)threadIdx.x) S.start = before;
        __syncthreads();
        if (warp == 0 && S.at >= 0) {
            const int base = first + S.at * kSegment;
            const float lim = key_logit(end_key);
            auto slot = [](int i) { return i + (i >> 4); };  // (a lane's 16 are read without bank conflicts)
            float v[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = base + k * 32 + lane < P.vocab ? __ldg(row + base + k * 32 + lane) : -INFINITY;
            if (P.cap > 0.f) {
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = softcap(v[k], P.cap);
            }
            float* const to = S.staged[kWideWarps - 1];  // (behind the weights)
#pragma unroll
            for (int k = 0; k < 16; ++k) to[k * 32 + lane] = v[k];
#pragma unroll 4
            for (int k = 0; k < 16; ++k) {
                const int i = base + k * 32 + lane;
                const float l = to[k * 32 + lane];
                const double wk = weight(l, m, c);
                S.weight[slot(k * 32 + lane)] = l > lim || (l == lim && i <= end_index) ? wk : 0.0;
            }
            __syncwarp();
            double own = 0.0;
#pragma unroll 4
            for (int k = 0; k < 16; ++k) own += S.weight[slot(lane * 16 + k)];
            double upto = own;
#pragma unroll 1
            for (int o = 1; o < 32; o <<= 1) {
                const double z = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += z;
            }
            double left = __shfl_up_sync(0xffffffffu, upto, 1);  // (upto - own would be 0 beside a much larger own)
            if (lane == 0) left = 0.0;
            double at = S.start + left, bw = 0.0;
            int best = -1;
#pragma unroll 4
            for (int k = 0; k < 16; ++k) {
                const double wk = S.weight[slot(lane * 16 + k)];
                if (wk > 0.0 && at <= target) best = base + lane * 16 + k, bw = wk;
                at += wk;
            }
            const int pick = __reduce_max_sync(0xffffffffu, best);
            if (best == pick && best >= 0) {
                P.ids[r] = best;
                if (P.probs) P.probs[r] = (float)(bw / kept);
            }
        }
    }
}

// ---------------------------------------------------------------- general --
// A cluster of up to 16 CTAs takes queued rows, each CTA with its part of the row in shared
// memory (warps own consecutive segments of 128 * J logits).
constexpr int kPick = kThreads;  // logits ranked at the end of a search
constexpr int kWays = 4;
constexpr int kBins = 256;

struct GeneralShared {
    double xd[2][kMaxCluster][kWays];  // per rank: sums of a step
    int xn[2][kMaxCluster][kWays];     // per rank: counts of a step
    uint32_t xlow[kMaxCluster];        // per rank: ~ the lowest key
    unsigned long long cand[kPick], cand2[kPick];
    BlockScratch scratch;
    double wsum[kWarps];
    int wcnt[kWarps];
    double red[kWarps][kWays];
    int redn[kWarps][kWays];
    uint32_t hist[kMaxCluster][kBins];  // per rank: number (at most 49152) and mean place of a part's logits
    uint32_t own_hist[kBins + 32], own_place[kBins + 32];  // the last 32: a lane's of what lies outside
    double above, past_at, n_at, n_b0, n_b1;
    float found_v;
    int found_idx, ncand, at, b0, b1, verdict;
};
// A kept prefix: logits above v, and equal ones up to index idx.  (Comparisons of floats leave NaN
// out and take -0 for +0, as the keys do.)
struct Limit {
    float v;
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
    __device__ static bool inside(float v, int i, const Limit& lim) { return v > lim.v || (v == lim.v && i <= lim.idx); }
    // f(index, four logits from it on) over this thread's logits, in the warp's segment.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        for (int j = 0; j < J; ++j) {
            const int o = (w * J + j) * 128 + lane * 4;
            const float4 q = *reinterpret_cast<const float4*>(chunk + o);
            const float v[4] = {q.x, q.y, q.z, q.w};
            f(first_index() + o, v);
        }
    }
    // The sum of weight over this thread's logits that keep(index, logit) takes.  A bit per logit
    // first, then only those: of a nucleus of some thousand tokens each thread has a few of 32.
    template <class K>
    __device__ __forceinline__ double weigh(K keep) const {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        double sum = 0.0;
        for (int j0 = 0; j0 < J; j0 += 8) {
            uint32_t bits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j0 + j >= J) break;
                const int o = (w * J + j0 + j) * 128 + lane * 4;
                const float4 q = *reinterpret_cast<const float4*>(chunk + o);
                const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) bits |= (keep(first_index() + o + e, v[e]) ? 1u : 0u) << (j * 4 + e);
            }
            while (__any_sync(0xffffffffu, bits != 0u)) {
                if (bits) {
                    const int k = __ffs(bits) - 1;
                    bits &= bits - 1;
                    sum += weight(chunk[(w * J + j0 + (k >> 2)) * 128 + lane * 4 + (k & 3)], m, c);
                }
            }
        }
        return sum;
    }
    // Sums over the cluster of N doubles and counts per thread (added in rank order).
    template <int N>
    __device__ __forceinline__ void cluster_sums(double (&d)[N], int (&n)[N]) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d[i] += __shfl_xor_sync(0xffffffffu, d[i], o);
            n[i] = __reduce_add_sync(0xffffffffu, n[i]);
            if (lane == 0) S.red[w][i] = d[i], S.redn[w][i] = n[i];
        }
        __syncthreads();
        xflip ^= 1;
        if (w < N) {  // warp i: value i of the CTA, sent to every rank
            double s = lane < kWarps ? S.red[lane][w] : 0.0;
            const int t = __reduce_add_sync(0xffffffffu, lane < kWarps ? S.redn[lane][w] : 0);
#pragma unroll
            for (int o = 1; o < kWarps; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            s = __shfl_sync(0xffffffffu, s, 0);
            if (lane < ranks) {
                *cluster.map_shared_rank(&S.xd[xflip][rank][w], lane) = s;
                *cluster.map_shared_rank(&S.xn[xflip][rank][w], lane) = t;
            }
        }
        cluster.sync();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            d[i] = 0.0, n[i] = 0;
            for (int k = 0; k < ranks; ++k) d[i] += S.xd[xflip][k][i], n[i] += S.xn[xflip][k][i];
        }
    }
    // What the logits above `past` inside `lim` weigh, and how many are inside `lim` at all.
    __device__ double mass(const Limit& lim, float past) {
        double d[1] = {weigh([&](int i, float v) { return v > past && inside(v, i, lim); })};
        int n[1] = {0};
        cluster_sums(d, n);
        return d[0];
    }
    __device__ int number(const Limit& lim) {
        double d[1] = {0.0};
        int n[1] = {0};
        each([&](int i, const float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) n[0] += inside(v[e], i + e, lim);
        });
        cluster_sums(d, n);
        return n[0];
    }

    // The shortest prefix inside `lim` whose weight (or number, if count) is at least t, from
    // histograms: 256 parts of the keys [lo, hi), even in value, then the parts around the one where
    // the number (exactly) or the weight (number times the weight in the mean place, some 1e-3 off at
    // first) passes t, with the exact weight of all above them, until at most kPick logits are left;
    // those are ranked.  *ok is false where that does not end on the prefix (ties, or a border nearer
    // than the estimate): search() does then.  Every CTA of the cluster computes the same steps from
    // the same sums, in one order.
    __device__ Limit estimate(const Limit& lim, double t, bool count, bool* ok) {
        uint32_t lo = low, hi = top + 1;
        double above = 0.0;
        *ok = false;
        cluster.sync();  // (a histogram of an earlier call may still be read)
        for (int step = 0; step < 5; ++step) {
            const float a = key_logit(lo), b = key_logit(key_before(hi));
            if (!(a > -3.0e38f && b < 3.0e38f && a < b)) return lim;
            const float scale = (float)kBins / (b - a);
            if (!(scale < 3.0e38f && scale > 0.f)) return lim;
            auto bin = [&](float v) { return min(kBins - 1, (int)((v - a) * scale)); };
            if (threadIdx.x < kBins) S.own_hist[threadIdx.x] = S.own_place[threadIdx.x] = 0;
            if (threadIdx.x == 0) S.at = -1, S.b0 = kBins, S.b1 = -1;
            __syncthreads();
            each([&](int i, const float (&v)[4]) {
                int at[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // free of branches
                    at[e] = v[e] >= a && v[e] <= b && inside(v[e], i + e, lim) ? bin(v[e]) : kBins + (int)(threadIdx.x & 31);
                    atomicAdd(&S.own_hist[at[e]], 1u);
                }
                if (!count) {  // its place in the part, in 1/32768
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        atomicAdd(&S.own_place[at[e]], (uint32_t)(((v[e] - a) * scale - (float)at[e]) * 32768.f));
                }
            });
            if (step > 0) cluster.sync();  // the last step's histograms have been read
            __syncthreads();
            if (threadIdx.x < kBins) {
                const uint32_t n = S.own_hist[threadIdx.x];
                S.own_hist[threadIdx.x] = n << 16 | (n ? min(S.own_place[threadIdx.x] / n, 65535u) : 0u);
            }
            __syncthreads();
            for (int x = threadIdx.x; x < kBins * ranks; x += kThreads)
                *cluster.map_shared_rank(&S.hist[rank][x % kBins], x / kBins) = S.own_hist[x % kBins];
            cluster.sync();
            // Parts from the top: thread i has part 255 - i.
            const int q = kBins - 1 - (int)threadIdx.x;
            uint32_t n = 0;
            double x = 0.0;
            if (q >= 0) {
                float place = 0.f;
                for (int k = 0; k < ranks; ++k) {
                    const uint32_t h = S.hist[k][q];
                    n += h >> 16;
                    place += (float)(h >> 16) * (float)(h & 65535u);
                }
                x = (double)n;
                if (!count && n) x *= weight(fminf(a + ((float)q + place / (float)n * (1.f / 32768.f)) / scale, m), m, c);
            }
            double all;
            const double before = above + block_prefix(x, S.scratch, flip, &all);
            const double past = block_prefix((double)n, S.scratch, flip, &all);  // logits in the parts above
            if (count && step == 0 && all <= t) {  // no more than are asked for
                *ok = true;
                return lim;
            }
            if (q >= 0 && before < t && before + x >= t) atomicMax(&S.at, q);
            __syncthreads();
            const int at = max(S.at, 0);
            if (q == at) S.past_at = past, S.n_at = (double)n;
            __syncthreads();
            // The window: that part, and for an estimate some hundred logits (a part at least) on each side.
            if (q >= 0) {
                const double side = count ? -1.0 : step == 0 ? kPick / 4 : kPick / 10;
                if (q == at || (q > at && S.past_at - past <= side)) atomicMax(&S.b1, q);
                if (q == at || (q < at && past + n - S.past_at - S.n_at <= side)) atomicMin(&S.b0, q);
            }
            __syncthreads();
            const int b0 = count ? at : max(0, min(S.b0, at - 1)), b1 = count ? at : min(kBins - 1, max(S.b1, at + 1));
            if (q == b1) S.above = before, S.n_b1 = past;
            if (q == b0) S.n_b0 = past + n;
            __syncthreads();
            above = S.above;
            const double in = S.n_b0 - S.n_b1;
            // The keys of the window: the lowest in part b0, the lowest past part b1 (parts rise with the
            // keys; the searches start next to where the part's border is in value).
            auto edge = [&](int part) {
                uint32_t l = lo, h = hi;  // the first key in [l, h] whose part is `part` or more (hi: none)
                const uint32_t guess = logit_key(fminf(fmaxf(a + part / scale, a), b));
                const uint32_t g0 = max(guess, lo + 64u) - 64u, g1 = min(guess + 64u, hi - 1);
                if (bin(key_logit(g0)) < part && bin(key_logit(g1)) >= part) l = g0, h = g1;
                while (l < h) {
                    const uint32_t mid = l + ((h - l) >> 1);
                    if (bin(key_logit(mid)) >= part) h = mid;
                    else l = mid + 1;
                }
                return l;
            };
            const uint32_t nlo = b0 > 0 ? edge(b0) : lo, nhi = b1 < kBins - 1 ? edge(b1 + 1) : hi;
            if (in > (double)kPick && nlo == lo && nhi == hi) return lim;
            lo = nlo, hi = nhi;
            if (!count) above = mass(lim, key_logit(key_before(hi)));
            if (!(above < t)) return lim;
            if (in <= (double)kPick) return rank_window(lim, lo, hi, above, t, count, ok);
        }
        return lim;
    }

    // The same by exact sums: [lo, hi) are the keys where the prefix ends, `above` what the keys from
    // hi on weigh; each step cuts them in four, in turn evenly in value and in key (which ends after
    // at most sixteen steps).
    __device__ Limit search(const Limit& lim, double t, bool count) {
        uint32_t lo = low, hi = top + 1;
        double above = 0.0;
        int inside_n = 0x7fffffff;
        for (int step = 0; inside_n > kPick && hi - lo > 1; ++step) {
            uint32_t cut[kWays];
            float cutv[kWays];
            const float a = key_logit(lo), b = key_logit(key_before(hi));
            const bool even = (step & 1) == 0 && a > -3.0e38f && b < 3.0e38f && a < b;
#pragma unroll
            for (int i = 0; i < kWays; ++i) {
                uint32_t k = lo + (uint32_t)((unsigned long long)(hi - lo) * i / kWays);
                if (even && i > 0) k = logit_key((float)((double)a + ((double)b - (double)a) * (i / (double)kWays)));
                cut[i] = i == 0 ? lo : min(max(k, cut[i - 1]), hi);
                cutv[i] = cut[i] < hi ? key_logit(cut[i]) : INFINITY;  // (an empty part: at most +inf logits, unused)
            }
            double d[kWays] = {};
            int n[kWays] = {};
            each([&](int i, const float (&v)[4]) {
                bool in[4], any = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    in[e] = v[e] >= a && v[e] <= b && inside(v[e], i + e, lim);
                    any = any || in[e];
                }
                if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double w = count ? 1.0 : weight(v[e], m, c);
#pragma unroll
                    for (int q = 0; q < kWays; ++q) {
                        const bool here = in[e] && v[e] >= cutv[q];
                        d[q] += here ? w : 0.0;
                        n[q] += here;
                    }
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
        if (inside_n > kPick) return nth_equal(lim, key_logit(lo), above, t, count, inside_n);
        bool ok;
        return rank_window(lim, lo, hi, above, t, count, &ok);
    }

    // Ranks the logits with keys in [lo, hi) (at most kPick) in CTA 0: the end of the shortest prefix
    // that reaches t, where all keys from hi on weigh `above`.  *ok: there is one.
    __device__ Limit rank_window(const Limit& lim, uint32_t lo, uint32_t hi, double above, double t, bool count, bool* ok) {
        if (threadIdx.x == 0) S.ncand = 0;
        cluster.sync();
        int* cnt = cluster.map_shared_rank(&S.ncand, 0);
        unsigned long long* list = cluster.map_shared_rank(&S.cand[0], 0);
        const float a = key_logit(lo), b = key_logit(key_before(hi));
        each([&](int i, const float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v[e] >= a && v[e] <= b && inside(v[e], i + e, lim)) {
                    const int at = atomicAdd(cnt, 1);
                    if (at < kPick) list[at] = (unsigned long long)logit_key(v[e]) << 32 | (0xffffffffu - (unsigned)(i + e));
                }
            }
        });
        cluster.sync();
        if (rank == 0) {
            const int n = min(S.ncand, kPick), t0 = threadIdx.x;
            if (t0 < n) S.own_hist[t0 & (kBins - 1)] = 0;
            __syncthreads();
            if (n <= kBins) {  // ranks by counting, two threads per logit
                const int i = t0 & (kBins - 1);
                int over = 0;
                if (i < n) {
                    const unsigned long long me = S.cand[i];
#pragma unroll 4
                    for (int j = t0 >> 8; j < n; j += 2) over += S.cand[j] > me;
                    atomicAdd(&S.own_hist[i], (uint32_t)over);
                }
                __syncthreads();
                if (t0 < n) S.cand2[S.own_hist[t0]] = S.cand[t0];
                __syncthreads();
                if (t0 < n) S.cand[t0] = S.cand2[t0];
                __syncthreads();
            } else {
                const int n2 = pow2_at_least(n);
                for (int i = n + t0; i < n2; i += kThreads) S.cand[i] = 0ull;
                block_sort_desc(S.cand, S.cand2, n2);
            }
            const double w = t0 >= n ? 0.0 : count ? 1.0 : weight(key_logit((uint32_t)(S.cand[t0] >> 32)), m, c);
            if (t0 == 0) S.at = n;
            double all;
            const double run = above + block_prefix(w, S.scratch, flip, &all) + w;
            if (t0 < n && run >= t) atomicMin(&S.at, t0);
            __syncthreads();
            if (t0 < ranks) {
                const int at = S.at;
                const unsigned long long f = S.cand[at < n ? at : max(n - 1, 0)];  // the last one, if a rounding left none
                *cluster.map_shared_rank(&S.found_v, t0) = key_logit((uint32_t)(f >> 32));
                *cluster.map_shared_rank(&S.found_idx, t0) = (int)(0xffffffffu - (unsigned)f);
                *cluster.map_shared_rank(&S.verdict, t0) = at < n;
            }
        }
        cluster.sync();
        *ok = S.verdict != 0;
        return Limit{S.found_v, S.found_idx};
    }

    // The search ended at one value shared by `n` logits: the first of them, in index order, that
    // reach t.
    __device__ Limit nth_equal(const Limit& lim, float value, double above, double t, bool count, int n) {
        const double w = count ? 1.0 : weight(value, m, c);
        const double q = ceil((t - above) / w);
        const int need = q >= (double)n ? n : q > 1.0 ? (int)q : 1;
        double d[1] = {0.0};
        int own[1] = {0};
        auto equal = [&](int i, float v) { return v == value && inside(v, i, lim); };
        each([&](int i, const float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) own[0] += equal(i + e, v[e]);
        });
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
                    for (int e = 0; e < 4; ++e) cnt += eq[e] = equal(i0 + e, chunk[o + e]);
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
        return Limit{value, S.found_idx};
    }

    // The pick in index order among what `lim` and mp keep.
    __device__ void pick(const Limit& lim, double mp, double u) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        auto kept = [&](float v) {
            const double x = weight(v, m, c);
            return x < mp ? 0.0 : x;
        };
        // min_p as a value: w rises with the logit
        float least = lim.v;
        if (mp > 0.0) {
            uint32_t lo = kLowestKey, hi = top;
            while (lo < hi) {
                const uint32_t span = hi - lo;
                auto cut = [&](int t) { return lo + (uint32_t)((unsigned long long)span * (unsigned)t / kThreads); };
                const int below = __syncthreads_count(weight(key_logit(cut(threadIdx.x)), m, c) < mp);
                const uint32_t nhi = below < kThreads ? cut(below) : hi;
                lo = below > 0 ? cut(below - 1) + 1 : lo;
                hi = nhi;
            }
            least = key_logit(hi);
        }
        double d[1] = {weigh([&](int i, float v) { return v >= least && inside(v, i, lim); })};
        int n[1] = {0};
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
            for (int e = 0; e < 4; ++e) s += x[e] = chunk[o + e] >= least && inside(chunk[o + e], i0 + e, lim) ? kept(chunk[o + e]) : 0.0;
            double y = s;
#pragma unroll
            for (int q = 1; q < 32; q <<= 1) {
                const double z = __shfl_up_sync(0xffffffffu, y, q);
                if (lane >= q) y += z;
            }
            double left = __shfl_up_sync(0xffffffffu, y, 1);  // (y - s would be 0 beside a much larger s)
            if (lane == 0) left = 0.0;
            double at = run + left;
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

__global__ void __launch_bounds__(kThreads, 2) sample_general_kernel(const SampleParams P, int J, int vec) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    GeneralShared& S = *reinterpret_cast<GeneralShared*>(smem_raw);
    float* chunk = reinterpret_cast<float*>(smem_raw + ((sizeof(GeneralShared) + 15) & ~size_t(15)));
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x / ranks >= P.queue[0]) return;  // nothing for this cluster
    cluster.sync();  // every CTA of the cluster runs before any writes to another's shared memory
    General g{P, S, chunk, cluster, rank, ranks, J, 0, 0, 0, 0.f, 0u, 0u, 0.0};
    const int queued = P.queue[0];
    for (int q = blockIdx.x / ranks; q < queued; q += gridDim.x / ranks) {
        const int r = P.queue[1 + q];
        const float* row = P.logits + (size_t)r * P.ld;
        g.r = r;
        __syncthreads();
        const int i0 = g.first_index();
        uint32_t top = 0, low = 0;
        constexpr int B = 8;  // loads of a thread in flight
        for (int j0 = 0; j0 < J; j0 += B) {
            float4 v[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int i = i0 + ((j0 + b) * kThreads + threadIdx.x) * 4;
                v[b] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (vec) {
                    if (j0 + b < J && i < P.vocab) v[b] = __ldg(reinterpret_cast<const float4*>(row + i));
                } else if (j0 + b < J) {
                    if (i < P.vocab) v[b].x = __ldg(row + i);
                    if (i + 1 < P.vocab) v[b].y = __ldg(row + i + 1);
                    if (i + 2 < P.vocab) v[b].z = __ldg(row + i + 2);
                    if (i + 3 < P.vocab) v[b].w = __ldg(row + i + 3);
                }
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                if (j0 + b >= J) break;
                if (P.cap > 0.f)
                    v[b] = make_float4(softcap(v[b].x, P.cap), softcap(v[b].y, P.cap), softcap(v[b].z, P.cap),
                                       softcap(v[b].w, P.cap));
                *reinterpret_cast<float4*>(chunk + ((j0 + b) * kThreads + threadIdx.x) * 4) = v[b];
                const float e[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t k = logit_key(e[q]);
                    low = k ? max(low, ~k) : low;
                }
            }
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
        g.c = st.scale();
        Limit lim{-INFINITY, -1};
        auto prefix = [&](double t, bool count) {
            bool ok;
            const Limit e = g.estimate(lim, t, count, &ok);
            if (ok) return e;
            return count && g.number(lim) <= t ? lim : g.search(lim, t, count);
        };
        if (st.k) lim = prefix((double)st.k, true);
        if (st.p < 1.0) {
            double total = 0.0;
            if (st.k) {
                total = g.mass(lim, -INFINITY);
            } else {
                total = P.rowmass[r];
            }
            lim = prefix(st.p * total, false);
        }
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
    SampleParams P{logits, ld, rows, vocab, cap, *how, ids_out, probs_out, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 2, 0};
    while (((vocab + (1 << P.gshift) - 1) >> P.gshift) > kMaxGroups) ++P.gshift;
    P.groups = (vocab + (1 << P.gshift) - 1) >> P.gshift;
    const long long segments = (vocab + kSumWarps * 512 - 1) / (kSumWarps * 512);
    if (segments * rows > 0x7fffffffLL)
        return g4::set_error(G4_ERR_UNSUPPORTED, "g4_sample: %d rows of %d logits", rows, vocab);
    const size_t ng = (size_t)rows * P.groups;
    st = g4::ensure_workspace(ctx, (ng + rows) * sizeof(double) + (ng + rows) * sizeof(uint32_t) + 2 * ((size_t)rows + 1) * sizeof(int));
    if (st) return st;
    P.gmass = static_cast<double*>(ctx->ws);
    P.rowmass = P.gmass + ng;
    P.gkey = reinterpret_cast<uint32_t*>(P.rowmass + rows);
    P.rowkey = P.gkey + ng;
    P.queue = reinterpret_cast<int*>(P.rowkey + rows);
    // With a top_k few rows are left over, and the launch would cost more than it saves.
    if (how->top_p && !how->top_k) P.nucleus = P.queue + rows + 1;
    const int vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (ld % 4 == 0 || rows == 1);
    const int vec4 = vec && vocab % 4 == 0;  // every row in whole 16-byte pieces

    // The general kernel's cluster: parts of at most 16384 logits if 16 CTAs are enough for that, and
    // down to 4096 while two CTAs per SM hold a cluster for every row.
    int ranks = 1;
    while (ranks < kMaxCluster && ((vocab + ranks - 1) / ranks > 8 * kThreads * 4 ||
                                   ((vocab + ranks - 1) / ranks > 2 * kThreads * 4 && 2LL * ranks * rows <= 2 * ctx->num_sms)))
        ranks <<= 1;
    const int J = (vocab + ranks * kThreads * 4 - 1) / (ranks * kThreads * 4);
    const size_t gsmem = ((sizeof(GeneralShared) + 15) & ~size_t(15)) + (size_t)J * kThreads * 4 * sizeof(float);
    static_assert(24 * kThreads * 16 + sizeof(GeneralShared) + 16 <= 227 * 1024, "the longest row's parts fit");
    static std::atomic<uint64_t> attr_set{0};
    if (!(attr_set.load() & (1ull << ctx->device))) {
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_finish_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)sizeof(FinishShared)));
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_general_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_general_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_nucleus_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)sizeof(NucleusShared)));
        G4_CHECK_CUDA(cudaFuncSetAttribute(sample_nucleus_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr_set.fetch_or(1ull << ctx->device);
    }
    if (vec4 && P.gshift >= 7) {
        // Blocks per warp: up to four, while some eight waves of warps are left.
        const long long all = (long long)rows * ((vocab + 511) / 512);
        const int blocks = (int)std::max<long long>(1, std::min<long long>(4, all / (ctx->num_sms * 48 * 2)));
        const int seg = (vocab + kSumWarps * 512 * blocks - 1) / (kSumWarps * 512 * blocks);
        st = g4::launch(ctx, "sample_summary_wide_kernel", sample_summary_wide_kernel, dim3((unsigned)((long long)seg * rows)),
                        dim3(kSumWarps * 32), 0, 1, P, seg, blocks);
    } else {
        st = g4::launch(ctx, "sample_summary_kernel", vec ? sample_summary_kernel<true> : sample_summary_kernel<false>,
                        dim3((unsigned)(segments * rows)), dim3(kSumWarps * 32), 0, 1, P, (int)segments);
    }
    if (st) return st;
    // The two that follow are set up while their predecessor runs, and wait for it (griddepcontrol).
    const bool pdl = ctx->pdl;
    ctx->pdl = true;
    st = g4::launch(ctx, "sample_finish_kernel", sample_finish_kernel, dim3(rows), dim3(kThreads), sizeof(FinishShared), 1, P,
                    vec4);
    if (!st && P.nucleus) {
        // One wave of clusters, if half of the rows come there, while a CTA has 8192 logits or more (64 rows
        // of 262144 in clusters of 8, of which a third came: 128 us, in clusters of 4: 104).
        int per = 1;
        while (per < kMaxRanks && (vocab > per * kWide * kSegment ||
                                     (2LL * per * rows <= 2 * ctx->num_sms && vocab >= 2 * per * 8192)))
            per <<= 1;
        st = g4::launch(ctx, "sample_nucleus_kernel", sample_nucleus_kernel,
                        dim3(std::max(1, std::min(rows, ctx->num_sms / per)) * per), dim3(kWide), sizeof(NucleusShared),
                        per, P, vec4);
    }
    // Only top-k, top-p and min-p can leave a row to the general kernel.
    if (!st && (how->top_k || how->top_p || how->min_p)) {
        const int clusters = std::max(1, std::min(rows, 2 * ctx->num_sms / ranks));
        st = g4::launch(ctx, "sample_general_kernel", sample_general_kernel, dim3(clusters * ranks), dim3(kThreads), gsmem,
                        ranks, P, J, vec4);
    }
    ctx->pdl = pdl;
    return st;
}
