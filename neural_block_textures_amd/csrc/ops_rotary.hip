// Rotary positions of several axes (include/ntc_ops.h: ntc_op_rotary).
//
// A pair (a, b) of a head's elements that belongs to axis m and has frequency f is turned by the angle pos[m] f:
//   a' = a cos - b sin,  b' = a sin + b cos;  backwards by the angle's negative.
// An angle is a 64-bit fraction of a turn: f / 2 pi, rounded to units of 2^-64, times the position, modulo 2^64, which no position is too far
// for: the angle is off by no more than the frequency is, 2^-57 of it. Its quarters of a turn are its top bits, and sine and cosine come from their
// power series on the rest, to 2^-23.
//
// A thread takes a token's run of pairs, makes their sines and cosines once, and turns that run in several heads of queries and
// keys. Bound by memory: every value is read and written once.
#include <math.h>

#include "ops_common.hpp"

namespace ntc_ops {
namespace {

constexpr int kMostPairs = 128, kMostAxes = 8;

struct RotaryArgs {
    const void* positions;
    long long position_stride, tokens;
    const void* x[2];
    void* y[2];
    long long token_stride[2], head_stride[2];
    int heads[2];
    int head_dim, pairs, backward;
    int units, turned_units;          // runs of a head, and those of them that are turned
    int heads_each, head_groups;
    unsigned long long turn[kMostPairs];  // f / 2 pi, in units of 2^-64
    uint8_t axis[kMostPairs];
};

// cos and sin of a 64-bit fraction of a turn
__device__ __forceinline__ void cos_sin(unsigned long long t, float& c, float& s) {
    const unsigned quarter = (unsigned)((t + (1ull << 61)) >> 62);
    const long long rest = (long long)(t - ((unsigned long long)quarter << 62));     // [-1/8, 1/8) of a turn
    const float x = (float)(int)(rest >> 30) * (6.283185307179586f * 0x1p-34f), z = x * x;
    const float sine = __builtin_fmaf(x * z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float cosine = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const float a = quarter & 1 ? sine : cosine, b = quarter & 1 ? cosine : sine;
    c = (quarter + 1) & 2 ? -a : a;
    s = quarter & 2 ? -b : b;
}

// kRun elements in one access; kBeside: a pair's elements lie beside each other, else half of what is turned apart.
template <class T, int kRun, bool kBeside, class P> __global__ void __launch_bounds__(256) k_rotary(RotaryArgs d) {
    constexpr int kPairs = kBeside ? kRun / 2 : kRun;
    const long long id = block_number() * 256 + threadIdx.x;
    const int unit = (int)(id % d.units);
    const long long rest = id / d.units;
    const int group = (int)(rest % d.head_groups);
    const long long token = rest / d.head_groups;
    if (token >= d.tokens) return;
    const int all = d.heads[0] + d.heads[1], h0 = group * d.heads_each, h1 = h0 + d.heads_each < all ? h0 + d.heads_each : all;
    const bool turned = unit < d.turned_units;
    float c[kPairs], s[kPairs];
    if (turned) {
        const P* pos = (const P*)d.positions + token * d.position_stride;
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const int p = unit * kPairs + i;
            cos_sin((unsigned long long)(long long)pos[d.axis[p]] * d.turn[p], c[i], s[i]);
            if (d.backward) s[i] = -s[i];
        }
    }
    const int first = turned ? unit * (kBeside ? kRun : kPairs) : 2 * d.pairs + (unit - d.turned_units) * kRun;
    for (int h = h0; h < h1; h++) {
        const int t = h >= d.heads[0], own = t ? h - d.heads[0] : h;
        const T* x = (const T*)d.x[t] + token * d.token_stride[t] + own * d.head_stride[t] + first;
        T* y = (T*)d.y[t] + (token * d.heads[t] + own) * d.head_dim + first;
        using R = LooseRun<T, kRun>;
        if (!turned) { *(R*)y = *(const R*)x; continue; }
        if constexpr (kBeside) {
            const R in = *(const R*)x;
            R out;
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                const float a = (float)in.v[2 * i], b = (float)in.v[2 * i + 1];
                out.v[2 * i] = (T)__builtin_fmaf(a, c[i], -(b * s[i]));
                out.v[2 * i + 1] = (T)__builtin_fmaf(a, s[i], b * c[i]);
            }
            *(R*)y = out;
        } else {
            const R lo = *(const R*)x, hi = *(const R*)(x + d.pairs);
            R a2, b2;
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                const float a = (float)lo.v[i], b = (float)hi.v[i];
                a2.v[i] = (T)__builtin_fmaf(a, c[i], -(b * s[i]));
                b2.v[i] = (T)__builtin_fmaf(a, s[i], b * c[i]);
            }
            *(R*)y = a2;
            *(R*)(y + d.pairs) = b2;
        }
    }
}

const char* wrong(const ntc_rotary_desc* d) {
    if (!d) return "no description";
    if (d->tokens < 0 || d->heads[0] < 0 || d->heads[1] < 0 || (int64_t)d->heads[0] + d->heads[1] > 1 << 20) return "tokens and heads from 0 on, at most 2^20 heads, are needed";
    if (d->head_dim < 2 || d->head_dim > 1 << 16 || d->head_dim % 2) return "a head has 2 to 65536 elements, an even number";
    if (d->axes < 1 || d->axes > kMostAxes) return "positions have 1 to 8 axes";
    int64_t pairs = 0;
    for (int a = 0; a < d->axes; a++) {
        if (d->sections[a] < 0) return "an axis has 0 pairs or more";
        pairs += d->sections[a];
    }
    if (pairs < 1 || pairs > kMostPairs || 2 * pairs > d->head_dim) return "the axes have 1 to 128 pairs together, and no more than a head's elements make";
    if (!(d->base >= 1) || d->base > 1e300) return "base must be a number from 1 on";
    if (d->dtype < 0 || d->dtype > NTC_F16) return "values are float32, bfloat16 or float16";
    if (d->position_bytes != 4 && d->position_bytes != 8) return "positions are 4 or 8 bytes wide";
    if (d->tokens && !d->positions) return "null pointer";
    for (int t = 0; t < 2; t++) if (d->tokens && d->heads[t] && (!d->x[t] || !d->y[t])) return "null pointer";
    return nullptr;
}

}  // namespace
}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" int ntc_op_rotary(const ntc_rotary_desc* d, void* stream, char* why, size_t cap) {
    if (const char* w = wrong(d)) return refuse(why, cap, w);
    const int heads = d->heads[0] + d->heads[1];
    if (!d->tokens || !heads) return 0;
    RotaryArgs a = {};
    a.positions = d->positions;
    a.position_stride = d->position_stride;
    a.tokens = d->tokens;
    for (int t = 0; t < 2; t++) {
        a.x[t] = d->x[t]; a.y[t] = d->y[t];
        a.token_stride[t] = d->token_stride[t]; a.head_stride[t] = d->head_stride[t];
        a.heads[t] = d->heads[t];
    }
    a.head_dim = d->head_dim;
    a.backward = d->backward != 0;
    for (int m = 0; m < d->axes; m++) a.pairs += d->sections[m];
    // (each frequency from the one before it, in 64 bits: off by 2^-57 at most after 128 of them, where a power for each would be 13 us of host work for 64)
    long double f = 1, ratio = d->one_ladder ? powl(d->base, -1.0L / a.pairs) : 1;
    for (int m = 0, p = 0; m < d->axes; m++) {
        if (!d->one_ladder && d->sections[m]) { f = 1; ratio = powl(d->base, -1.0L / d->sections[m]); }
        for (int j = 0; j < d->sections[m]; j++, p++, f *= ratio) {
            a.turn[p] = (unsigned long long)(f * (0x1p64L / 6.283185307179586476925286766559005768L) + 0.5L);
            a.axis[p] = (uint8_t)m;
        }
    }
    // The widest access, up to 16 bytes, that divides what is turned and what is not. (Rows may start at any element.)
    int run = 16 / (int)type_size(d->dtype);
    while ((d->interleaved ? 2 * a.pairs : a.pairs) % run || (d->head_dim - 2 * a.pairs) % run) run /= 2;
    const bool beside = d->interleaved != 0;                   // (runs have 2 elements at least then: heads are even)
    a.turned_units = d->interleaved ? 2 * a.pairs / run : a.pairs / run;
    a.units = a.turned_units + (d->head_dim - 2 * a.pairs) / run;
    // Heads that share a thread's sines: as many as leave 2^19 threads (a card full of them); then a quarter of the work is theirs and not the sines'.
    const int64_t each = a.tokens * a.units;
    int64_t groups = ((1 << 19) + each - 1) / each;
    if (groups > heads) groups = heads;
    a.heads_each = (int)((heads + groups - 1) / groups);
    a.head_groups = (heads + a.heads_each - 1) / a.heads_each;
    const dim3 grid = grid_of((each * a.head_groups + 255) / 256);
    const hipStream_t s = (hipStream_t)stream;
    const auto with = [&](auto type, auto run_, auto beside_, auto position) { k_rotary<decltype(type), run_.value, beside_.value, decltype(position)><<<grid, 256, 0, s>>>(a); };
    const auto with_position = [&](auto type, auto run_, auto beside_) { d->position_bytes == 8 ? with(type, run_, beside_, (int64_t)0) : with(type, run_, beside_, (int32_t)0); };
    const auto with_run = [&](auto type) {
        using T = decltype(type);
#define NTC_RUN(R) if (run == R) return beside && R > 1 ? with_position(type, std::integral_constant<int, R>{}, std::bool_constant<(R > 1)>{}) : with_position(type, std::integral_constant<int, R>{}, std::false_type{})
        if constexpr (sizeof(T) == 2) NTC_RUN(8);
        NTC_RUN(4); NTC_RUN(2); NTC_RUN(1);
#undef NTC_RUN
    };
    if (d->dtype == NTC_F32) with_run(f32{});
    else if (d->dtype == NTC_BF16) with_run(bf16{});
    else with_run(f16{});
    return launched(why, cap);
}
