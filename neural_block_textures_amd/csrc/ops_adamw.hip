// AdamW over many tensors, with its state in 32 bits or in 8 (include/ntc_ops.h).
#include <math.h>

#include "device_common.hpp"
#include "ops_common.hpp"

namespace ntc_ops {

constexpr int kAdamTPB = 256, kLane = 4, kWaveBlocks = 4;    // a wave's 4 blocks of 256 values, 4 a lane
constexpr int kBatch = 160;                                   // tensors of one launch: their gradients travel as arguments
constexpr uint32_t kNsAdam = 5;                               // stream of the counter noise (1 to 4: the ES trainer's)
static_assert(kAdamTPB / 64 * kWaveBlocks * NTC_STATE_BLOCK == NTC_ADAMW_CHUNK, "a block of threads is a chunk");

struct AdamGrads {
    const void* g[kBatch];
    float rate[kBatch], root[kBatch];        // lr / (1 - b1^c), 1 / sqrt(1 - b2^c)
    uint8_t type[kBatch];
};
struct AdamArgs {
    const ntc_adamw_tensor* tensors;
    const int32_t* chunk_tensor;
    long long chunk0;
    int tensor0;
    void *m, *v;
    uint8_t *me, *ve;
    float* master;
    float b1, nb1, b2, nb2, eps, keep;
    uint64_t head;
};

// Four values from position i of a buffer of type `type` (uniform over the block) as floats: whole runs where all four are
// there and aligned, else one by one; 0 past the end.
__device__ __forceinline__ void load4(float (&o)[4], const void* p, int type, long long i, long long n, bool aligned) {
    if (type == NTC_F32) {
        const float* q = (const float*)p + i;
        if (aligned && i + 4 <= n) { const auto r = *(const Run<float, 4>*)q; for (int j = 0; j < 4; j++) o[j] = r.v[j]; }
        else for (int j = 0; j < 4; j++) o[j] = i + j < n ? q[j] : 0.0f;
    } else if (type == NTC_BF16) {
        const bf16* q = (const bf16*)p + i;
        if (aligned && i + 4 <= n) { const auto r = *(const Run<bf16, 4>*)q; for (int j = 0; j < 4; j++) o[j] = (float)r.v[j]; }
        else for (int j = 0; j < 4; j++) o[j] = i + j < n ? (float)q[j] : 0.0f;
    } else {
        const f16* q = (const f16*)p + i;
        if (aligned && i + 4 <= n) { const auto r = *(const Run<f16, 4>*)q; for (int j = 0; j < 4; j++) o[j] = (float)r.v[j]; }
        else for (int j = 0; j < 4; j++) o[j] = i + j < n ? (float)q[j] : 0.0f;
    }
}
__device__ __forceinline__ void store4(const float (&o)[4], void* p, int type, long long i, long long n, bool aligned) {
    if (type == NTC_F32) {
        float* q = (float*)p + i;
        if (aligned && i + 4 <= n) { Run<float, 4> r; for (int j = 0; j < 4; j++) r.v[j] = o[j]; *(Run<float, 4>*)q = r; }
        else for (int j = 0; j < 4; j++) if (i + j < n) q[j] = o[j];
    } else if (type == NTC_BF16) {
        bf16* q = (bf16*)p + i;
        if (aligned && i + 4 <= n) { Run<bf16, 4> r; for (int j = 0; j < 4; j++) r.v[j] = (bf16)o[j]; *(Run<bf16, 4>*)q = r; }
        else for (int j = 0; j < 4; j++) if (i + j < n) q[j] = (bf16)o[j];
    } else {
        f16* q = (f16*)p + i;
        if (aligned && i + 4 <= n) { Run<f16, 4> r; for (int j = 0; j < 4; j++) r.v[j] = (f16)o[j]; *(Run<f16, 4>*)q = r; }
        else for (int j = 0; j < 4; j++) if (i + j < n) q[j] = (f16)o[j];
    }
}
__device__ __forceinline__ bool aligned4(const void* p, int type) { return ((uintptr_t)p & (type == NTC_F32 ? 15 : 7)) == 0; }

// 2^(b - 127), b from 0 to 254
__device__ __forceinline__ float power_of(int b) { return __uint_as_float(b > 0 ? (uint32_t)b << 23 : 1u << 22); }

// ---------------------------------------------------------------- 8-bit states
// The value of a code without its sign (kTop: the exponent that stands for [1, 2)); exact, and `scale` is a power of two.
template <int kTop> __device__ __forceinline__ float decode8(uint32_t c, float scale) {
    const float normal = __uint_as_float((c + 8u * (127 - kTop)) << 20);
    const float small = (float)c * __uint_as_float((uint32_t)(127 - 2 - kTop) << 23);
    return (c >= 8 ? normal : small) * scale;
}
// a >= 0, at most 1.875, to its code: the 16 bits r are added below the last kept bit
template <int kTop> __device__ __forceinline__ uint32_t encode8(float a, uint32_t r) {
    const uint32_t normal = ((__float_as_uint(a) + (r << 4)) >> 20) - 8u * (127 - kTop);
    const float small = a * __uint_as_float((uint32_t)(127 + kTop + 2) << 23) + (float)r * 0x1p-16f;
    return a >= __uint_as_float((uint32_t)(127 + 1 - kTop) << 23) ? normal : (uint32_t)small;
}
// The largest of 64 lanes' a >= 0 (NaN counts as the largest: bit patterns are compared), and the block's exponent byte from it.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t b) {
    for (int w = 1; w < 64; w <<= 1) { const uint32_t o = __shfl_xor(b, w); b = o > b ? o : b; }
    return b;
}
__device__ __forceinline__ int exponent_byte(uint32_t most) {
    const int e = (int)(most >> 23) + ((most & 0x7fffffu) > 0x700000u ? 1 : 0);
    return (most >> 23) >= 254u ? 255 : e;
}

// four values a lane of one block, to codes
struct Codes { uint32_t m, v; int me, ve; };
__device__ __forceinline__ Codes encode_block(const float (&m)[4], const float (&v)[4], const uint32_t (&rm)[4], const uint32_t (&rv)[4]) {
    uint32_t bm = 0, bv = 0;
    for (int j = 0; j < 4; j++) {
        const uint32_t a = __float_as_uint(m[j]) & 0x7fffffffu, b = __float_as_uint(v[j]) & 0x7fffffffu;
        bm = a > bm ? a : bm;
        bv = b > bv ? b : bv;
    }
    Codes c = { 0, 0, exponent_byte(wave_max_bits(bm)), exponent_byte(wave_max_bits(bv)) };
    const float sm = power_of(254 - (c.me == 255 ? 254 : c.me)), sv = power_of(254 - (c.ve == 255 ? 254 : c.ve));
    for (int j = 0; j < 4; j++) {
        const uint32_t sign = m[j] < 0.0f ? 128u : 0u;
        uint32_t a = encode8<15>(fabsf(m[j]) * sm, rm[j]) | sign, b = encode8<31>(v[j] * sv, rv[j]);
        b = b == 0 && v[j] * sv > 0.0f ? 1u : b;
        c.m |= (c.me == 255 ? 0u : a) << (8 * j);
        c.v |= (c.ve == 255 ? 0u : b) << (8 * j);
    }
    return c;
}
__device__ __forceinline__ void decode_block(uint32_t cm, uint32_t cv, int me, int ve, float (&m)[4], float (&v)[4]) {
    const float sm = me == 255 ? __builtin_nanf("") : power_of(me), sv = ve == 255 ? __builtin_nanf("") : power_of(ve);
    for (int j = 0; j < 4; j++) {
        const uint32_t a = (cm >> (8 * j)) & 255u, b = (cv >> (8 * j)) & 255u;
        const float x = decode8<15>(a & 127u, sm);
        m[j] = a & 128u ? -x : x;
        v[j] = decode8<31>(b, sv);
    }
}

template <int kBits, bool kMaster> __global__ void __launch_bounds__(kAdamTPB) k_adamw(AdamArgs A, AdamGrads G) {
    const long long chunk = A.chunk0 + blockIdx.x;
    const int ti = A.chunk_tensor[chunk], gi = ti - A.tensor0;
    const void* g_ptr = G.g[gi];
    if (!g_ptr) return;
    const ntc_adamw_tensor T = A.tensors[ti];
    const float rate = G.rate[gi], root = G.root[gi];
    const int gt = G.type[gi];
    const bool g_al = aligned4(g_ptr, gt), p_al = aligned4(T.param, T.param_type);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long base = (chunk - T.first_chunk) * NTC_ADAMW_CHUNK + wave * (kWaveBlocks * NTC_STATE_BLOCK) + lane * kLane;
#pragma unroll
    for (int u = 0; u < kWaveBlocks; u++) {
        const long long i = base + u * NTC_STATE_BLOCK, at = T.state_offset + i;
        if (i - lane * kLane >= T.numel) break;      // the whole block lies past the end
        float g[4], p[4], m[4], v[4];
        load4(g, g_ptr, gt, i, T.numel, g_al);
        if (kMaster) { const auto r = *(const Run<float, 4>*)(A.master + at); for (int j = 0; j < 4; j++) p[j] = r.v[j]; }
        else load4(p, T.param, T.param_type, i, T.numel, p_al);
        if (kBits == 8) {
            decode_block(*(const uint32_t*)((const uint8_t*)A.m + at), *(const uint32_t*)((const uint8_t*)A.v + at), A.me[at >> 8], A.ve[at >> 8], m, v);
        } else {
            const auto r = *(const Run<float, 4>*)((const float*)A.m + at), q = *(const Run<float, 4>*)((const float*)A.v + at);
            for (int j = 0; j < 4; j++) { m[j] = r.v[j]; v[j] = q.v[j]; }
        }
        for (int j = 0; j < 4; j++) {
            m[j] = m[j] * A.b1 + g[j] * A.nb1;
            v[j] = v[j] * A.b2 + (g[j] * g[j]) * A.nb2;
            p[j] = p[j] * A.keep - rate * (m[j] / (sqrtf(v[j]) * root + A.eps));
        }
        if (kBits == 8) {
            uint32_t rm[4], rv[4];
            for (int j = 0; j < 4; j += 2) {
                const uint64_t h = ntc_hip::noise_bits(A.head, (uint64_t)(at + j) >> 1);
                rm[j] = (uint32_t)h & 0xffffu;
                rv[j] = (uint32_t)(h >> 16) & 0xffffu;
                rm[j + 1] = (uint32_t)(h >> 32) & 0xffffu;
                rv[j + 1] = (uint32_t)(h >> 48);
            }
            const Codes c = encode_block(m, v, rm, rv);
            *(uint32_t*)((uint8_t*)A.m + at) = c.m;
            *(uint32_t*)((uint8_t*)A.v + at) = c.v;
            if (lane == 0) { A.me[at >> 8] = (uint8_t)c.me; A.ve[at >> 8] = (uint8_t)c.ve; }
        } else {
            Run<float, 4> r, q;
            for (int j = 0; j < 4; j++) { r.v[j] = m[j]; q.v[j] = v[j]; }
            *(Run<float, 4>*)((float*)A.m + at) = r;
            *(Run<float, 4>*)((float*)A.v + at) = q;
        }
        if (kMaster) { Run<float, 4> r; for (int j = 0; j < 4; j++) r.v[j] = p[j]; *(Run<float, 4>*)(A.master + at) = r; }
        store4(p, T.param, T.param_type, i, T.numel, p_al);
    }
}

__global__ void __launch_bounds__(256) k_adamw_moments(const uint8_t* cm, const uint8_t* cv, const uint8_t* me, const uint8_t* ve, long long n, float* om,
                                                       float* ov) {
    const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    float m[4], v[4];
    decode_block(*(const uint32_t*)(cm + at), *(const uint32_t*)(cv + at), me[at >> 8], ve[at >> 8], m, v);
    Run<float, 4> r, q;
    for (int j = 0; j < 4; j++) { r.v[j] = m[j]; q.v[j] = v[j]; }
    *(Run<float, 4>*)(om + at) = r;
    *(Run<float, 4>*)(ov + at) = q;
}
__global__ void __launch_bounds__(256) k_adamw_encode(const float* im, const float* iv, long long n, uint8_t* cm, uint8_t* cv, uint8_t* me, uint8_t* ve) {
    const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;    // whole waves: n is a multiple of 256
    if (at >= n) return;
    const auto r = *(const Run<float, 4>*)(im + at), q = *(const Run<float, 4>*)(iv + at);
    float m[4], v[4];
    for (int j = 0; j < 4; j++) { m[j] = r.v[j]; v[j] = q.v[j]; }
    const uint32_t half[4] = { 32768, 32768, 32768, 32768 };
    const Codes c = encode_block(m, v, half, half);
    *(uint32_t*)(cm + at) = c.m;
    *(uint32_t*)(cv + at) = c.v;
    if ((threadIdx.x & 63) == 0) { me[at >> 8] = (uint8_t)c.me; ve[at >> 8] = (uint8_t)c.ve; }
}

}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" int ntc_op_adamw(const ntc_adamw_desc* d, void* stream, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->n < 0 || d->n > (1 << 30)) return refuse(why, cap, "a tensor count from 0 to 2^30");
    if (d->state_bits != 8 && d->state_bits != 32) return refuse(why, cap, "states are held in 8 or 32 bits");
    if (!(d->beta1 >= 0.0 && d->beta1 < 1.0) || !(d->beta2 >= 0.0 && d->beta2 < 1.0)) return refuse(why, cap, "betas are in [0, 1)");
    if (!(d->lr >= 0.0) || !(d->eps >= 0.0) || !(d->weight_decay >= 0.0)) return refuse(why, cap, "lr, eps and weight_decay are not negative");
    if (d->n == 0) return 0;
    if (!d->tensors || !d->chunk_tensor || !d->first_chunk || !d->grads || !d->grad_types || !d->steps || !d->exp_avg || !d->exp_avg_sq)
        return refuse(why, cap, "a null pointer");
    if (d->state_bits == 8 && (!d->exp_avg_exp || !d->exp_avg_sq_exp)) return refuse(why, cap, "8-bit states have exponents");
    for (int64_t i = 0; i < d->n; i++) {
        if (d->grads[i] && d->steps[i] < 1) return refuse(why, cap, "steps count from 1");
        if (d->grad_types[i] < 0 || d->grad_types[i] > 2) return refuse(why, cap, "gradients are 32-bit floats, bfloat16 or float16");
        if (d->first_chunk[i + 1] < d->first_chunk[i] || d->first_chunk[i + 1] > 0x7fffffff) return refuse(why, cap, "chunks in order, fewer than 2^31");
    }
    AdamArgs A;
    A.tensors = d->tensors;
    A.chunk_tensor = d->chunk_tensor;
    A.m = d->exp_avg;
    A.v = d->exp_avg_sq;
    A.me = d->exp_avg_exp;
    A.ve = d->exp_avg_sq_exp;
    A.master = d->master;
    A.b1 = (float)d->beta1;
    A.nb1 = (float)(1.0 - d->beta1);
    A.b2 = (float)d->beta2;
    A.nb2 = (float)(1.0 - d->beta2);
    A.eps = (float)d->eps;
    A.keep = (float)(1.0 - d->lr * d->weight_decay);
    A.head = ntc_hip::noise_head(d->seed, kNsAdam, d->calls, 0);
    int32_t last = -1;
    float rate = 0, root = 0;
    for (int64_t t0 = 0; t0 < d->n; t0 += kBatch) {
        const int64_t t1 = t0 + kBatch < d->n ? t0 + kBatch : d->n;
        AdamGrads G;
        bool any = false;
        for (int64_t t = t0; t < t1; t++) {
            if (d->grads[t] && d->steps[t] != last) {     // (nearly always all tensors are at the same step)
                last = d->steps[t];
                rate = (float)(d->lr / (1.0 - pow(d->beta1, last)));
                root = (float)(1.0 / sqrt(1.0 - pow(d->beta2, last)));
            }
            G.g[t - t0] = d->grads[t];
            G.rate[t - t0] = rate;
            G.root[t - t0] = root;
            G.type[t - t0] = (uint8_t)d->grad_types[t];
            any |= d->grads[t] != nullptr;
        }
        const int64_t blocks = d->first_chunk[t1] - d->first_chunk[t0];
        if (!any || !blocks) continue;
        A.chunk0 = d->first_chunk[t0];
        A.tensor0 = (int)t0;
        const auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, kAdamTPB, 0, (hipStream_t)stream>>>(A, G); };
        if (d->state_bits == 8) d->master ? go(k_adamw<8, true>) : go(k_adamw<8, false>);
        else d->master ? go(k_adamw<32, true>) : go(k_adamw<32, false>);
        if (const int r = launched(why, cap)) return r;
    }
    return 0;
}

static int check_state(const void* a, const void* b, const void* c, const void* e, const void* m, const void* v, int64_t n, char* why, size_t cap) {
    if (n < 0 || n % NTC_STATE_BLOCK || n > (int64_t)1 << 40) return refuse(why, cap, "a state is a multiple of 256 values");
    if (n && (!a || !b || !c || !e || !m || !v)) return refuse(why, cap, "a null pointer");
    return 0;
}

extern "C" int ntc_op_adamw_moments(const void* cm, const void* cv, const uint8_t* me, const uint8_t* ve, int64_t n, float* m, float* v, void* stream, char* why,
                                    size_t cap) {
    if (const int r = check_state(cm, cv, me, ve, m, v, n, why, cap)) return r;
    if (!n) return 0;
    k_adamw_moments<<<(unsigned)((n + 1023) / 1024), 256, 0, (hipStream_t)stream>>>((const uint8_t*)cm, (const uint8_t*)cv, me, ve, n, m, v);
    return launched(why, cap);
}

extern "C" int ntc_op_adamw_encode(const float* m, const float* v, int64_t n, void* cm, void* cv, uint8_t* me, uint8_t* ve, void* stream, char* why, size_t cap) {
    if (const int r = check_state(cm, cv, me, ve, m, v, n, why, cap)) return r;
    if (!n) return 0;
    k_adamw_encode<<<(unsigned)((n + 1023) / 1024), 256, 0, (hipStream_t)stream>>>(m, v, n, (uint8_t*)cm, (uint8_t*)cv, me, ve);
    return launched(why, cap);
}
