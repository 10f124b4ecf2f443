// AdamW over many tensors, with its state in 32 bits or in 8 (include/ntc_ops.h).
#include <math.h>

#include "device_common.hpp"
#include "ops_common.hpp"

namespace ntc_ops {

constexpr int kAdamTPB = 256, kLane = 4, kWaveBlocks = 4;    // a wave's 4 blocks of 256 values, 4 a lane
constexpr int kBatch = 400, kRates = 16;                      // tensors of one launch, and different steps among them: gradients travel as arguments (of at most 4 KiB)
constexpr uint32_t kNsAdam = 5;                               // stream of the counter noise (1 to 4: the ES trainer's)
static_assert(kAdamTPB / 64 * kWaveBlocks * NTC_STATE_BLOCK == NTC_ADAMW_CHUNK, "a block of threads is a chunk");

struct AdamGrads {
    const void* g[kBatch];
    float rate[kRates], root[kRates];        // lr / (1 - b1^c), 1 / sqrt(1 - b2^c)
    uint8_t kind[kBatch];                    // the gradient's type, and 4 times its place among the rates
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
static_assert(sizeof(AdamGrads) + sizeof(AdamArgs) <= 4096, "arguments of a launch");

// Four values from position i of a buffer of type `type` (uniform over the block) as floats: whole runs where all four are
// there, else one by one; 0 past the end.
template <class T> __device__ __forceinline__ void load4_of(float (&o)[4], const T* q, long long left) {
    if (left >= 4) { const auto r = *(const LooseRun<T, 4>*)q; for (int j = 0; j < 4; j++) o[j] = (float)r.v[j]; }
    else for (int j = 0; j < 4; j++) o[j] = j < left ? (float)q[j] : 0.0f;
}
template <class T> __device__ __forceinline__ void store4_of(const float (&o)[4], T* q, long long left) {
    if (left >= 4) { LooseRun<T, 4> r; for (int j = 0; j < 4; j++) r.v[j] = (T)o[j]; *(LooseRun<T, 4>*)q = r; }
    else for (int j = 0; j < 4; j++) if (j < left) q[j] = (T)o[j];
}
__device__ __forceinline__ void load4(float (&o)[4], const void* p, int type, long long i, long long n) {
    if (type == NTC_F32) load4_of(o, (const float*)p + i, n - i);
    else if (type == NTC_BF16) load4_of(o, (const bf16*)p + i, n - i);
    else load4_of(o, (const f16*)p + i, n - i);
}
__device__ __forceinline__ void store4(const float (&o)[4], void* p, int type, long long i, long long n) {
    if (type == NTC_F32) store4_of(o, (float*)p + i, n - i);
    else if (type == NTC_BF16) store4_of(o, (bf16*)p + i, n - i);
    else store4_of(o, (f16*)p + i, n - i);
}

// 2^(b - 127), b from 0 to 254
__device__ __forceinline__ float power_of(int b) { return __uint_as_float(b > 0 ? (uint32_t)b << 23 : 1u << 22); }

// ---------------------------------------------------------------- 8-bit states
// A code's bits are the top bits of a 32-bit float whose exponents are 2^(127 - kTop) too small (kTop: the exponent that stands for
// [1, 2)), the smallest codes being that float's own subnormals: two exact products by powers of two are the whole conversion.
template <int kTop> __device__ __forceinline__ float decode8(uint32_t c20, float scale) {   // c20: the code without sign, at bit 20
    return __uint_as_float(c20) * __uint_as_float((uint32_t)(254 - kTop) << 23) * scale;
}
// 0 <= a * scale <= 1.875 to its code: 16 random bits r are added below the last kept bit. (Below the smallest power the product is
// rounded 20 bits below the last kept one.)
template <int kTop> __device__ __forceinline__ uint32_t encode8(float a, float scale, uint32_t r) {
    return (__float_as_uint(a * scale * __uint_as_float((uint32_t)kTop << 23)) + (r << 4)) >> 20;
}
// the block's exponent byte from the bits of its largest magnitude (NaN counts as the largest)
__device__ __forceinline__ int exponent_byte(uint32_t most) {
    const int e = (int)(most >> 23) + ((most & 0x7fffffu) > 0x700000u ? 1 : 0);
    return (most >> 23) >= 254u ? 255 : e;
}

// four values a lane of one block, to codes
struct Codes { uint32_t m, v; int me, ve; };
__device__ __forceinline__ Codes encode_block(const float (&m)[4], const float (&v)[4], const uint32_t (&rm)[4], const uint32_t (&rv)[4]) {
    const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    uint32_t bm = 0, bv = 0;
    for (int j = 0; j < 4; j++) {
        bm = larger(bm, __float_as_uint(m[j]) & 0x7fffffffu);
        bv = larger(bv, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    bm = __builtin_amdgcn_readfirstlane(reduce64(bm, larger));
    bv = __builtin_amdgcn_readfirstlane(reduce64(bv, larger));
    Codes c = { 0, 0, exponent_byte(bm), exponent_byte(bv) };
    const float sm = power_of(254 - c.me), sv = power_of(254 - c.ve);
    for (int j = 0; j < 4; j++) {
        const uint32_t a = encode8<15>(fabsf(m[j]), sm, rm[j]) | (__float_as_uint(m[j]) >> 24 & 128u);
        uint32_t b = encode8<31>(v[j], sv, rv[j]);
        const uint32_t least = __float_as_uint(v[j]) < 1u ? 0u : 1u;     // v > 0 is not rounded to 0
        b = b > least ? b : least;
        c.m |= a << (8 * j);
        c.v |= b << (8 * j);
    }
    if (c.me == 255) c.m = 0;
    if (c.ve == 255) c.v = 0;
    return c;
}
__device__ __forceinline__ void decode_block(uint32_t cm, uint32_t cv, int me, int ve, float (&m)[4], float (&v)[4]) {
    const float sm = me == 255 ? __builtin_nanf("") : power_of(me), sv = ve == 255 ? __builtin_nanf("") : power_of(ve);
    for (int j = 0; j < 4; j++) {
        const uint32_t a = cm >> (8 * j), b = cv >> (8 * j);
        m[j] = __uint_as_float(__float_as_uint(decode8<15>((a & 127u) << 20, sm)) | (a & 128u) << 24);
        v[j] = decode8<31>((b & 255u) << 20, sv);
    }
}

// ---------------------------------------------------------------- the step
// Four values of one tensor. The division and the root are the hardware's, an ulp each: a 2^-22 of the update, where p keeps 2^-24 of itself. They take a
// subnormal number as 0, which eps hides unless it is small. `kSmall`, it is: small v are taken 2^64 times and the sum 2^24 times as large (2^28 bf16 values
// with an 8-bit state 531 us against 507; with 32-bit state the same).
template <bool kSmall> __device__ __forceinline__ void update(const AdamArgs& A, float rate, float root, const float (&g)[4], float (&p)[4], float (&m)[4], float (&v)[4]) {
    for (int j = 0; j < 4; j++) {
        m[j] = m[j] * A.b1 + g[j] * A.nb1;
        v[j] = v[j] * A.b2 + (g[j] * g[j]) * A.nb2;
        if (kSmall) {
            const bool low = v[j] < 0x1p-96f;
            const float below = __builtin_amdgcn_sqrtf(low ? v[j] * 0x1p64f : v[j]) * (low ? root * 0x1p-32f : root) + A.eps;
            p[j] = p[j] * A.keep - rate * (m[j] * __builtin_amdgcn_rcpf(below * 0x1p24f) * 0x1p24f);
        } else {
            p[j] = p[j] * A.keep - rate * (m[j] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[j]) * root + A.eps));
        }
    }
}
__device__ __forceinline__ void random16(uint64_t at, uint32_t (&rm)[4], uint32_t (&rv)[4]) {   // at: head + (position / 2) phi
    for (int j = 0; j < 4; j += 2) {
        const uint64_t h = ntc_hip::mix64(at + (j ? ntc_hip::kPhi64 : 0));
        rm[j] = (uint32_t)h & 0xffffu;
        rv[j] = (uint32_t)h >> 16;
        rm[j + 1] = (uint32_t)(h >> 32) & 0xffffu;
        rv[j + 1] = (uint32_t)(h >> 48);
    }
}

// A wave's blocks that lie whole in its tensor (all four, or `count`): everything is read first, so that the memory has four blocks' requests at
// once; kG32, kP32: the gradient and the tensor are 32-bit. They may lie at any element's address.
template <class R, int kSize> struct __attribute__((packed, aligned(kSize))) Loose { R v; };
struct __attribute__((packed)) LooseWord { uint32_t v; };
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool k32> struct Raw { using type = std::conditional_t<k32, u32x4, u32x2>; };
template <bool k32> __device__ __forceinline__ void widen(float (&o)[4], const typename Raw<k32>::type& r, int type) {
    if constexpr (k32) { const auto f = __builtin_bit_cast(Run<float, 4>, r); for (int j = 0; j < 4; j++) o[j] = f.v[j]; }
    else if (type == NTC_BF16) { const auto f = __builtin_bit_cast(Run<bf16, 4>, r); for (int j = 0; j < 4; j++) o[j] = (float)f.v[j]; }
    else { const auto f = __builtin_bit_cast(Run<f16, 4>, r); for (int j = 0; j < 4; j++) o[j] = (float)f.v[j]; }
}
template <bool k32> __device__ __forceinline__ typename Raw<k32>::type narrow(const float (&p)[4], int type) {
    if constexpr (k32) { Run<float, 4> f; for (int j = 0; j < 4; j++) f.v[j] = p[j]; return __builtin_bit_cast(u32x4, f); }
    else if (type == NTC_BF16) { Run<bf16, 4> f; for (int j = 0; j < 4; j++) f.v[j] = (bf16)p[j]; return __builtin_bit_cast(u32x2, f); }
    else { Run<f16, 4> f; for (int j = 0; j < 4; j++) f.v[j] = (f16)p[j]; return __builtin_bit_cast(u32x2, f); }
}
template <int kBits, bool kMaster, bool kSmall, bool kG32, bool kP32, bool kAll> __device__ __forceinline__ void whole_blocks(const AdamArgs& A, const ntc_adamw_tensor& T, const void* g_ptr, int gt, float rate,
                                                                                                                 float root, long long i0, int count) {
    using GR = typename Raw<kG32>::type;
    using PR = typename Raw<kP32>::type;
    using GL = Loose<GR, kG32 ? 4 : 2>;
    using PL = Loose<PR, kP32 ? 4 : 2>;
    using SR = std::conditional_t<kBits == 8, uint32_t, float4>;
    const GL* gp = (const GL*)((const uint8_t*)g_ptr + i0 * (kG32 ? 4 : 2));
    PL* pp = (PL*)((uint8_t*)T.param + i0 * (kP32 ? 4 : 2));
    const long long at = T.state_offset + i0;
    SR* mp = (SR*)((uint8_t*)A.m + at * (kBits / 8));
    SR* vp = (SR*)((uint8_t*)A.v + at * (kBits / 8));
    float4* wp = (float4*)(A.master + at);
    GR g[kWaveBlocks];
    PR p[kWaveBlocks];
    SR m[kWaveBlocks], v[kWaveBlocks];
    float4 w[kWaveBlocks];
    uint32_t me = 0, ve = 0;
#pragma unroll
    for (int u = 0; u < kWaveBlocks; u++) {
        if (!kAll && u >= count) break;
        g[u] = gp[64 * u].v;
        if (kMaster) w[u] = wp[64 * u];
        else p[u] = pp[64 * u].v;
        m[u] = mp[64 * u];
        v[u] = vp[64 * u];
    }
    if constexpr (kBits == 8 && kAll) {                      // a wave's four blocks' exponents are a word, at any byte
        me = __builtin_amdgcn_readfirstlane(((const LooseWord*)(A.me + (at >> 8)))->v);
        ve = __builtin_amdgcn_readfirstlane(((const LooseWord*)(A.ve + (at >> 8)))->v);
    } else if constexpr (kBits == 8) {
        const int lane = threadIdx.x & 63;                   // lane u the exponents of block u
        const uint32_t em = lane < count ? A.me[(at >> 8) + lane] : 0, ev = lane < count ? A.ve[(at >> 8) + lane] : 0;
        for (int u = 0; u < kWaveBlocks; u++) { me |= __builtin_amdgcn_readlane(em, u) << (8 * u); ve |= __builtin_amdgcn_readlane(ev, u) << (8 * u); }
    }
    uint32_t new_me = 0, new_ve = 0;
    uint64_t noise = A.head + (uint64_t)(at >> 1) * ntc_hip::kPhi64;
#pragma unroll
    for (int u = 0; u < kWaveBlocks; u++) {
        if (!kAll && u >= count) break;
        float gf[4], pf[4], mf[4], vf[4];
        widen<kG32>(gf, g[u], gt);
        if (kMaster) { pf[0] = w[u].x; pf[1] = w[u].y; pf[2] = w[u].z; pf[3] = w[u].w; }
        else widen<kP32>(pf, p[u], T.param_type);
        if constexpr (kBits == 8) decode_block(m[u], v[u], (me >> (8 * u)) & 255, (ve >> (8 * u)) & 255, mf, vf);
        else { mf[0] = m[u].x; mf[1] = m[u].y; mf[2] = m[u].z; mf[3] = m[u].w; vf[0] = v[u].x; vf[1] = v[u].y; vf[2] = v[u].z; vf[3] = v[u].w; }
        update<kSmall>(A, rate, root, gf, pf, mf, vf);
        if constexpr (kBits == 8) {
            uint32_t rm[4], rv[4];
            random16(noise + (uint64_t)(128 * u) * ntc_hip::kPhi64, rm, rv);
            const Codes c = encode_block(mf, vf, rm, rv);
            mp[64 * u] = c.m;
            vp[64 * u] = c.v;
            new_me |= (uint32_t)c.me << (8 * u);
            new_ve |= (uint32_t)c.ve << (8 * u);
        } else {
            mp[64 * u] = float4{ mf[0], mf[1], mf[2], mf[3] };
            vp[64 * u] = float4{ vf[0], vf[1], vf[2], vf[3] };
        }
        if (kMaster) wp[64 * u] = float4{ pf[0], pf[1], pf[2], pf[3] };
        pp[64 * u].v = narrow<kP32>(pf, T.param_type);
    }
    if (kBits == 8 && !kAll) {
        const int lane = threadIdx.x & 63;
        if (lane < count) {
            A.me[(at >> 8) + lane] = (uint8_t)(new_me >> (8 * lane));
            A.ve[(at >> 8) + lane] = (uint8_t)(new_ve >> (8 * lane));
        }
    } else if (kBits == 8 && (threadIdx.x & 63) == 0) {
        ((LooseWord*)(A.me + (at >> 8)))->v = new_me;
        ((LooseWord*)(A.ve + (at >> 8)))->v = new_ve;
    }
}

// One pass over everything: memory bounds it (2^28 bf16 values with a 32-bit copy and state, 7.5 GB: 1406 us, 5.3 TB/s, where a copy reaches 5.0; 8-bit
// state and no copy, 2.7 GB: 507 us where many follow each other, 5.3 TB/s, 555 over the first twenty). A block takes 4096 values of one tensor, a wave 1024 of them, 256 (a block of an 8-bit state) at a
// time: blocks never span tensors, whose pointers are one lookup each, and small tensors (240 of 1 to 400000 values, 24 us; six of a small decoder, 4)
// cost a launch between them, not one each.
template <int kBits, bool kMaster, bool kSmall> __global__ void __launch_bounds__(kAdamTPB) k_adamw(AdamArgs A, AdamGrads G) {
    const long long chunk = A.chunk0 + blockIdx.x;
    const int ti = A.chunk_tensor[chunk], gi = ti - A.tensor0;
    const void* g_ptr = G.g[gi];
    if (!g_ptr) return;
    const ntc_adamw_tensor T = A.tensors[ti];
    const int kind = G.kind[gi], gt = kind & 3;
    const float rate = G.rate[kind >> 2], root = G.root[kind >> 2];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long long wave_base = (chunk - T.first_chunk) * NTC_ADAMW_CHUNK + wave * (kWaveBlocks * NTC_STATE_BLOCK), base = wave_base + lane * kLane;
    const long long blocks = (T.numel - wave_base) >> 8;     // whole ones from here on
    const bool g32 = gt == NTC_F32, p32 = T.param_type == NTC_F32;
    const auto whole = [&](auto all, int count) {
        if (g32) p32 ? whole_blocks<kBits, kMaster, kSmall, true, true, all.value>(A, T, g_ptr, gt, rate, root, base, count) : whole_blocks<kBits, kMaster, kSmall, true, false, all.value>(A, T, g_ptr, gt, rate, root, base, count);
        else p32 ? whole_blocks<kBits, kMaster, kSmall, false, true, all.value>(A, T, g_ptr, gt, rate, root, base, count) : whole_blocks<kBits, kMaster, kSmall, false, false, all.value>(A, T, g_ptr, gt, rate, root, base, count);
    };
    if (blocks >= kWaveBlocks) { whole(std::true_type(), kWaveBlocks); return; }
    if (blocks > 0) whole(std::false_type(), (int)blocks);
    // the tensor's last, ragged block
    const long long i = base + (blocks > 0 ? blocks : 0) * NTC_STATE_BLOCK, at = T.state_offset + i;
    if (i - lane * kLane < T.numel) {
        float g[4], p[4], m[4], v[4];
        load4(g, g_ptr, gt, i, T.numel);
        if (kMaster) { const auto r = *(const Run<float, 4>*)(A.master + at); for (int j = 0; j < 4; j++) p[j] = r.v[j]; }
        else load4(p, T.param, T.param_type, i, T.numel);
        if (kBits == 8) {
            decode_block(*(const uint32_t*)((const uint8_t*)A.m + at), *(const uint32_t*)((const uint8_t*)A.v + at), A.me[at >> 8], A.ve[at >> 8], m, v);
        } else {
            const auto r = *(const Run<float, 4>*)((const float*)A.m + at), q = *(const Run<float, 4>*)((const float*)A.v + at);
            for (int j = 0; j < 4; j++) { m[j] = r.v[j]; v[j] = q.v[j]; }
        }
        update<kSmall>(A, rate, root, g, p, m, v);
        if (kBits == 8) {
            uint32_t rm[4], rv[4];
            random16(A.head + (uint64_t)(at >> 1) * ntc_hip::kPhi64, rm, rv);
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
        store4(p, T.param, T.param_type, i, T.numel);
    }
}

__global__ void __launch_bounds__(256) k_adamw_moments(const uint8_t* cm, const uint8_t* cv, const uint8_t* me, const uint8_t* ve, long long n, float* om,
                                                       float* ov) {
    const long long at = (block_number() * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    float m[4], v[4];
    decode_block(*(const uint32_t*)(cm + at), *(const uint32_t*)(cv + at), me[at >> 8], ve[at >> 8], m, v);
    Run<float, 4> r, q;
    for (int j = 0; j < 4; j++) { r.v[j] = m[j]; q.v[j] = v[j]; }
    *(Run<float, 4>*)(om + at) = r;
    *(Run<float, 4>*)(ov + at) = q;
}
__global__ void __launch_bounds__(256) k_adamw_encode(const float* im, const float* iv, long long n, uint8_t* cm, uint8_t* cv, uint8_t* me, uint8_t* ve) {
    const long long at = (block_number() * 256 + threadIdx.x) * 4;    // whole waves: n is a multiple of 256
    if (at >= n) return;
    const auto r = *(const Run<float, 4>*)(im + at), q = *(const Run<float, 4>*)(iv + at);
    float m[4], v[4];
    for (int j = 0; j < 4; j++) { m[j] = r.v[j]; v[j] = q.v[j] <= 0.0f ? 0.0f : q.v[j]; }   // (v has no sign: a set bit would reach into the next code)
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
    if (!d->first_chunk || !d->grads || !d->grad_types || !d->steps) return refuse(why, cap, "a null pointer");
    const bool values = d->first_chunk[d->n] > d->first_chunk[0];          // (tensors of no values have no state either)
    if (values && (!d->tensors || !d->chunk_tensor || !d->exp_avg || !d->exp_avg_sq)) return refuse(why, cap, "a null pointer");
    if (values && d->state_bits == 8 && (!d->exp_avg_exp || !d->exp_avg_sq_exp)) return refuse(why, cap, "8-bit states have exponents");
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
    for (int64_t t0 = 0, t1; t0 < d->n; t0 = t1) {
        AdamGrads G;
        int32_t steps[kRates];
        int rates = 0;
        bool any = false, small = false;
        for (t1 = t0; t1 < d->n && t1 - t0 < kBatch; t1++) {
            int r = 0;
            if (d->grads[t1]) {                           // (nearly always all tensors are at the same step)
                while (r < rates && steps[r] != d->steps[t1]) r++;
                if (r == kRates) break;
                if (r == rates) {
                    steps[r] = d->steps[t1];
                    G.rate[r] = (float)(d->lr / (1.0 - pow(d->beta1, steps[r])));
                    G.root[r] = (float)(1.0 / sqrt(1.0 - pow(d->beta2, steps[r])));
                    // a lost root of up to 2^-63 and its correction, against half a unit of eps
                    small = small || !(A.eps >= 0x1p-39f * G.root[r]);
                    rates++;
                }
                any = true;
            }
            G.g[t1 - t0] = d->grads[t1];
            G.kind[t1 - t0] = (uint8_t)(d->grad_types[t1] | r << 2);
        }
        const int64_t blocks = d->first_chunk[t1] - d->first_chunk[t0];
        if (!any || !blocks) continue;
        A.chunk0 = d->first_chunk[t0];
        A.tensor0 = (int)t0;
        const auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, kAdamTPB, 0, (hipStream_t)stream>>>(A, G); };
        const auto with = [&](auto is_small) {
            constexpr bool s = is_small.value;
            if (d->state_bits == 8) d->master ? go(k_adamw<8, true, s>) : go(k_adamw<8, false, s>);
            else d->master ? go(k_adamw<32, true, s>) : go(k_adamw<32, false, s>);
        };
        small ? with(std::true_type()) : with(std::false_type());
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
    k_adamw_moments<<<grid_of((n + 1023) / 1024), 256, 0, (hipStream_t)stream>>>((const uint8_t*)cm, (const uint8_t*)cv, me, ve, n, m, v);
    return launched(why, cap);
}

extern "C" int ntc_op_adamw_encode(const float* m, const float* v, int64_t n, void* cm, void* cv, uint8_t* me, uint8_t* ve, void* stream, char* why, size_t cap) {
    if (const int r = check_state(cm, cv, me, ve, m, v, n, why, cap)) return r;
    if (!n) return 0;
    k_adamw_encode<<<grid_of((n + 1023) / 1024), 256, 0, (hipStream_t)stream>>>(m, v, n, (uint8_t*)cm, (uint8_t*)cv, me, ve);
    return launched(why, cap);
}
