// Token log probabilities with entropy and the best alternatives, and their gradient (include/ntc_ops.h).
#include "ops_common.hpp"

namespace ntc_ops {

// One row's softmax, kept while it is read once: the largest x so far, and over e = exp2((x - m) k) the sums of e and of
// e (x - m) k, with k = log2(e) / T. log2 sum exp2(x k) = m k + log2 s, and the entropy is ln 2 (log2 s - t / s).
// m starts at the type's lowest value and not at -inf, so that x - m is never inf - inf; a row of only -inf ends with s = 0.
struct Soft { float m, s, t; };
__device__ __forceinline__ void soft_add(Soft& a, float x, float k) {
    const float d = (x - a.m) * k;
    const float e = fast_exp2(d);
    a.s += e;
    a.t = __builtin_fmaf(e, fmaxf(d, -1e30f), a.t);   // (an e of 0 has d = -inf)
}
__device__ __forceinline__ void soft_raise(Soft& a, float m, float k) {   // m >= a.m
    const float d = fmaxf((a.m - m) * k, -1e30f), f = fast_exp2(d);
    a.t = f * __builtin_fmaf(a.s, d, a.t);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ void soft_join(Soft& a, Soft b, float k) {
    const float m = fmaxf(a.m, b.m);
    soft_raise(a, m, k);
    soft_raise(b, m, k);
    a.s += b.s;
    a.t += b.t;
}

// log p of one value, in nats: not through (x - m) k, which overflows for a mask of the lowest value
__device__ __forceinline__ float log_prob(float x, float m, float inv_t, float log_s) { return (x - m) * inv_t - kLn2 * log_s; }

__device__ __forceinline__ long long token_of(const ntc_logprobs_desc& d, long long outer, long long inner) {
    const long long at = outer * d.token_outer_stride + inner * d.token_inner_stride;
    return d.token_bytes == 8 ? ((const long long*)d.tokens)[at] : ((const int*)d.tokens)[at];
}

// (v, i) comes before (w, j): larger value, then lower index
__device__ __forceinline__ bool before(float v, long long i, float w, long long j) { return v > w || (v == w && i < j); }
__device__ __forceinline__ float order_of(float x) { return x != x ? -NTC_INF : x; }

template <class T> __global__ void __launch_bounds__(256) k_logprobs_row(ntc_logprobs_desc d) {
    const long long row = blockIdx.x, outer = row / d.inner_rows, inner = row % d.inner_rows;
    const T* x = (const T*)d.logits + outer * d.outer_stride + inner * d.inner_stride;
    const float inv_t = 1.0f / d.temperature, k = kLog2e / d.temperature;
    __shared__ Soft part[256];
    __shared__ float bv[256];
    __shared__ long long bi[256];
    Soft a = { kLowest, 0.0f, 0.0f };
    for (long long i = threadIdx.x; i < d.V; i += 256) {
        const float v = (float)x[i];
        if (v > a.m) soft_raise(a, v, k);
        soft_add(a, v, k);
    }
    part[threadIdx.x] = a;
    __syncthreads();
    for (int w = 128; w; w >>= 1) {
        if (threadIdx.x < w) { Soft b = part[threadIdx.x]; soft_join(b, part[threadIdx.x + w], k); part[threadIdx.x] = b; }
        __syncthreads();
    }
    a = part[0];
    const bool none = a.s == 0.0f;
    const float log_s = fast_log2(a.s);
    if (threadIdx.x == 0) {
        const long long t = token_of(d, outer, inner);
        float lp = 0.0f;
        if (t != d.ignore_index) lp = t < 0 || t >= d.V ? __builtin_nanf("") : none ? -NTC_INF : log_prob((float)x[t], a.m, inv_t, log_s);
        d.logprob[row] = lp;
        d.entropy[row] = none ? 0.0f : kLn2 * (log_s - a.t / a.s);
        d.stats[2 * row] = none ? -NTC_INF : a.m;
        d.stats[2 * row + 1] = log_s;
    }
    float pv = NTC_INF;
    long long pi = -1;
    for (int r = 0; r < d.top; r++) {
        float v = -NTC_INF;
        long long at = d.V;
        for (long long i = threadIdx.x; i < d.V; i += 256) {
            const float w = order_of((float)x[i]);
            if (before(pv, pi, w, i) && before(w, i, v, at)) { v = w; at = i; }
        }
        bv[threadIdx.x] = v;
        bi[threadIdx.x] = at;
        __syncthreads();
        for (int w = 128; w; w >>= 1) {
            if (threadIdx.x < w && before(bv[threadIdx.x + w], bi[threadIdx.x + w], bv[threadIdx.x], bi[threadIdx.x])) {
                bv[threadIdx.x] = bv[threadIdx.x + w];
                bi[threadIdx.x] = bi[threadIdx.x + w];
            }
            __syncthreads();
        }
        pv = bv[0];
        pi = bi[0];
        __syncthreads();
        if (threadIdx.x == 0) {
            d.top_ids[row * d.top + r] = pi;
            d.top_logprobs[row * d.top + r] = none ? -NTC_INF : log_prob(pv, a.m, inv_t, log_s);
        }
    }
}

template <class T> __global__ void __launch_bounds__(256) k_logprobs_grad(ntc_logprobs_desc d) {
    const long long row = blockIdx.x, outer = row / d.inner_rows, inner = row % d.inner_rows;
    const T* x = (const T*)d.logits + outer * d.outer_stride + inner * d.inner_stride;
    T* dx = (T*)d.dlogits + row * d.V;
    const float k = kLog2e / d.temperature, inv_t = 1.0f / d.temperature;
    const float m = d.stats[2 * row], log_s = d.stats[2 * row + 1], H = d.entropy[row];
    const long long t = token_of(d, outer, inner);
    const bool none = m == -NTC_INF, out = t != d.ignore_index && (t < 0 || t >= d.V);
    const float glp = d.g_logprob && t != d.ignore_index ? d.g_logprob[row] : 0.0f;
    const float gh = d.g_entropy ? d.g_entropy[row] : 0.0f;
    float all = glp;
    if (d.g_top) for (int r = 0; r < d.top; r++) all += d.g_top[row * d.top + r];
    if (out) all = __builtin_nanf("");
    for (long long i = threadIdx.x; i < d.V; i += 256) {
        const float lp = ((float)x[i] - m) * k - log_s, p = fast_exp2(lp);
        float g = i == t ? glp : 0.0f;
        if (d.g_top) for (int r = 0; r < d.top; r++) g += d.top_ids[row * d.top + r] == i ? d.g_top[row * d.top + r] : 0.0f;
        g -= p * (all + gh * __builtin_fmaf(kLn2, fmaxf(lp, -160.0f), H));
        dx[i] = (T)(none ? 0.0f : g * inv_t);
    }
}

static int check(const ntc_logprobs_desc* d, bool backward, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->rows < 0 || d->V < 1 || d->inner_rows < 1) return refuse(why, cap, "rows >= 0, inner_rows >= 1 and V >= 1 are needed");
    if (d->V > 0x7fffffff || d->rows > 0x7fffffff) return refuse(why, cap, "at most 2^31 - 1 rows and values of a row");
    if (d->dtype < 0 || d->dtype > 2) return refuse(why, cap, "logits are 32-bit floats, bfloat16 or float16");
    if (d->token_bytes != 4 && d->token_bytes != 8) return refuse(why, cap, "tokens are 32- or 64-bit integers");
    if (d->top < 0 || d->top > NTC_MAX_TOP || d->top > d->V) return refuse(why, cap, "top is 0 to 32 and at most V");
    if (!(d->temperature > 0.0f) || d->temperature > 3e38f) return refuse(why, cap, "temperature is positive and finite");
    if (d->rows == 0) return 0;
    if (!d->logits || !d->tokens || !d->stats || !d->entropy) return refuse(why, cap, "a null pointer");
    if (!backward && (!d->logprob || (d->top && (!d->top_ids || !d->top_logprobs)))) return refuse(why, cap, "a null pointer");
    if (backward && (!d->dlogits || (d->g_top && !d->top_ids))) return refuse(why, cap, "a null pointer");
    return 0;
}

}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" size_t ntc_op_token_logprobs_workspace(int64_t, int64_t, int32_t) { return 0; }

extern "C" int ntc_op_token_logprobs(const ntc_logprobs_desc* d, void* stream, char* why, size_t cap) {
    if (const int r = check(d, false, why, cap)) return r;
    if (!d->rows) return 0;
    const auto go = [&](auto kernel) { kernel<<<(unsigned)d->rows, 256, 0, (hipStream_t)stream>>>(*d); };
    d->dtype == NTC_F32 ? go(k_logprobs_row<f32>) : d->dtype == NTC_BF16 ? go(k_logprobs_row<bf16>) : go(k_logprobs_row<f16>);
    return launched(why, cap);
}

extern "C" int ntc_op_token_logprobs_backward(const ntc_logprobs_desc* d, void* stream, char* why, size_t cap) {
    if (const int r = check(d, true, why, cap)) return r;
    if (!d->rows) return 0;
    const auto go = [&](auto kernel) { kernel<<<(unsigned)d->rows, 256, 0, (hipStream_t)stream>>>(*d); };
    d->dtype == NTC_F32 ? go(k_logprobs_grad<f32>) : d->dtype == NTC_BF16 ? go(k_logprobs_grad<bf16>) : go(k_logprobs_grad<f16>);
    return launched(why, cap);
}
