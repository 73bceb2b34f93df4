// g4_sample.cu -- one token per row of f32 logits: temperature, top-k, top-p, min-p and a given
// uniform number per row.
//
// With w_i = exp((l_i - m) / T), m the highest logit, the filters keep a prefix of the ranking
// by (l descending, index ascending), so each is a threshold (key, index): an element is kept
// when its key is above, or equal with an index not above.  A threshold is the answer to "the
// shortest prefix whose weight reaches t" with weights w (top-p) or 1 (top-k).  Sums decide
// which token a border falls on, so they are 64-bit.
#include "g4_common.cuh"

namespace {

using namespace g4dev;

constexpr int kThreads = 1024;

struct SampleParams {
    const float* logits;
    long long ld;
    int vocab;
    float cap;
    g4_sampling how;
    int32_t* ids;
    float* probs;
};

// Monotone key of a logit: larger logit, larger key; 0 for what is never picked (NaN, -inf).
__device__ __forceinline__ uint32_t logit_key(float l) {
    if (!(l > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(l + 0.f);  // -0 ties with +0
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

struct Limit {
    uint32_t key;
    int idx;
};

struct RowView {
    const float* l;
    int vocab;
    float cap, m;
    double inv_t;
    __device__ float at(int i) const { return cap > 0.f ? tanhf(l[i] / cap) * cap : l[i]; }
    __device__ double weight(float v) const { return v == m ? 1.0 : exp(((double)v - (double)m) * inv_t); }
};

__device__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) s += red[i];
    return s;
}

__device__ __forceinline__ bool inside(uint32_t k, int i, const Limit& lim) {
    return k > lim.key || (k == lim.key && k != 0u && i <= lim.idx);
}

// Sum over the elements inside `lim` with key >= from, of their weights (or their number).
template <bool kCount>
__device__ double mass(const RowView& R, const Limit& lim, uint32_t from, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < R.vocab; i += kThreads) {
        const float v = R.at(i);
        const uint32_t k = logit_key(v);
        if (k >= from && inside(k, i, lim)) s += kCount ? 1.0 : R.weight(v);
    }
    return block_sum(s, red);
}

// The shortest prefix inside `lim` whose weight (or number) is at least t > 0.
template <bool kCount>
__device__ Limit search(const RowView& R, const Limit& lim, double t, double* red) {
    uint32_t key = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = key | (1u << bit);
        if (mass<kCount>(R, lim, c, red) >= t) key = c;
    }
    if (key == 0) return lim;  // all of it weighs less (a rounding of t)
    const double above = key == 0xffffffffu ? 0.0 : mass<kCount>(R, lim, key + 1, red);
    const double at = mass<kCount>(R, lim, key, red) - above;
    // of the elements with this key, all of one weight, the first `need`
    const double number = mass<true>(R, lim, key, red) - (key == 0xffffffffu ? 0.0 : mass<true>(R, lim, key + 1, red));
    const double need = fmax(1.0, ceil((t - above) / (at / number)));
    int lo = 0, hi = R.vocab - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        double c = 0.0;
        for (int i = threadIdx.x; i <= mid; i += kThreads) {
            const uint32_t k = logit_key(R.at(i));
            c += k == key && inside(k, i, lim) ? 1.0 : 0.0;
        }
        if (block_sum(c, red) >= need) hi = mid;
        else lo = mid + 1;
    }
    return Limit{key, lo};
}

__global__ void __launch_bounds__(kThreads) sample_kernel(SampleParams p) {
    __shared__ double red[kThreads / 32];
    __shared__ unsigned long long best;
    __shared__ double part[kThreads];
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x;
    RowView R{p.logits + (size_t)r * p.ld, p.vocab, p.cap, 0.f, 1.0};
    if (threadIdx.x == 0) best = 0ull;
    __syncthreads();
    unsigned long long mine = 0ull;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
        const unsigned long long k = ((unsigned long long)logit_key(R.at(i)) << 32) | (0xffffffffu - (unsigned)i);
        mine = k > mine ? k : mine;
    }
    atomicMax(&best, mine);
    __syncthreads();
    const uint32_t top = (uint32_t)(best >> 32);
    const int first = (int)(0xffffffffu - (unsigned)best);
    const float T = p.how.temperature ? p.how.temperature[r] : 1.f;
    if (top == 0u || !(T > 0.f)) {
        if (threadIdx.x == 0) {
            p.ids[r] = top == 0u ? -1 : first;
            if (p.probs) p.probs[r] = top == 0u ? 0.f : 1.f;
        }
        return;
    }
    R.m = R.at(first);
    R.inv_t = 1.0 / (double)T;
    Limit lim{1u, p.vocab};
    const int k = p.how.top_k ? p.how.top_k[r] : 0;
    if (k >= 1 && k < p.vocab && mass<true>(R, lim, 1u, red) > (double)k) lim = search<true>(R, lim, (double)k, red);
    const float tp = p.how.top_p ? p.how.top_p[r] : 1.f;
    if (tp <= 0.f) lim = Limit{top, first};
    else if (tp < 1.f) lim = search<false>(R, lim, (double)tp * mass<false>(R, lim, 1u, red), red);
    const float mpf = p.how.min_p ? p.how.min_p[r] : 0.f;
    const double mp = mpf > 0.f ? fmin((double)mpf, 1.0) : 0.0;
    auto kept = [&](float v, int i) {
        if (!inside(logit_key(v), i, lim)) return 0.0;
        const double w = R.weight(v);
        return mp > 0.0 && w < mp ? 0.0 : w;
    };
    // index order: each thread sums a run of consecutive indices
    const int run = (p.vocab + kThreads - 1) / kThreads;
    const int i0 = threadIdx.x * run, i1 = min(p.vocab, i0 + run);
    double s = 0.0;
    for (int i = i0; i < i1; ++i) s += kept(R.at(i), i);
    part[threadIdx.x] = s;
    __syncthreads();
    double before = 0.0, total = 0.0;
    for (int t = 0; t < kThreads; ++t) {
        if (t == threadIdx.x) before = total;
        total += part[t];
    }
    float u = p.how.uniform[r];
    u = u >= 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
    const double target = (double)u * total;
    if (before <= target && before + s > target) {
        double c = before;
        int pick = -1;
        double w = 0.0;
        for (int i = i0; i < i1; ++i) {
            const double x = kept(R.at(i), i);
            if (x > 0.0) pick = i, w = x;  // the last positive one when rounding keeps c at the target
            c += x;
            if (c > target) break;
        }
        p.ids[r] = pick;
        if (p.probs) p.probs[r] = (float)(w / total);
    }
}

}  // namespace

extern "C" g4_status g4_sample(g4_ctx* ctx, const float* logits, long long ld, int rows, int vocab, float cap,
                               const g4_sampling* how, int32_t* ids_out, float* probs_out) {
    if (rows < 0 || vocab < 1 || ld < vocab || !how)
        return g4::set_error(G4_ERR_INVALID, "g4_sample: rows %d, vocab %d, row pitch %lld", rows, vocab, ld);
    if (vocab > 786432) return g4::set_error(G4_ERR_UNSUPPORTED, "g4_sample: vocab %d (786432 supported)", vocab);
    if (rows > 0 && (!logits || !how->uniform || !ids_out))
        return g4::set_error(G4_ERR_INVALID, "g4_sample: null argument");
    const g4_status st = g4::use_device(ctx);
    if (st || rows == 0) return st;
    const SampleParams p{logits, ld, vocab, cap, *how, ids_out, probs_out};
    return g4::launch(ctx, "sample_kernel", sample_kernel, dim3(rows), dim3(kThreads), 0, 1, p);
}
