// Rotary positions of several axes (include/ntc_ops.h: ntc_op_rotary).
//
// A pair (a, b) of a head's elements that belongs to axis m and has frequency f is turned by the angle pos[m] f:
//   a' = a cos - b sin,  b' = a sin + b cos;  backwards by the angle's negative.
// An angle is a 64-bit fraction of a turn: f / 2 pi, rounded to units of 2^-64, times the position, modulo 2^64. It is off by no more than the position times 2^-57 f (f's own error)
// and 2^-65 of a turn (f's rounding, all that is left of slow frequencies): some 2^-24 at positions of 2^33, and in proportion. Its quarters of a turn are its top bits, and sine and cosine come from their
// power series on the rest, to 2^-23.
//
// A block takes a few tokens: their sines and cosines are made once, into shared memory, and serve all heads of queries and keys, whose elements
// are then read and written in the order in which they lie. Bound by memory: every value is read and written once. 50176 tokens of 32 heads of 128 bfloat16: 173 us (4.8 TB/s); 65536 of
// 16 heads of 32, whose values the last-level cache holds: 30 (4.5 TB/s); one token: 4, the launch.
#include <math.h>

#include "ops_common.hpp"

namespace ntc_ops {
namespace {

constexpr int kMostPairs = 128, kMostAxes = 8, kTable = 1024;

struct RotaryArgs {
    const void* positions;
    long long position_stride, tokens;
    const void* x[2];
    void* y[2];
    long long token_stride[2], head_stride[2];
    int heads[2];
    int head_dim, pairs, backward;
    int units, turned_units;              // runs of a head, and those of them that are turned
    int block_tokens, block_heads, head_blocks;
    unsigned unit_magic, head_magic, pair_magic;   // ceil(2^32 / n), 0 for 1: of units, of a block's heads, of pairs
    unsigned long long turn[kMostPairs];  // f / 2 pi, in units of 2^-64
    int axis[kMostPairs];
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

// kRun elements as one access to any element's address. (As integers: the compiler stores a structure of 16-bit floats in pieces of 2 to 8 bytes, and 65536 tokens of 16 heads then take 45 us.)
template <int kBytes> struct Piece;
template <> struct Piece<16> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Piece<8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Piece<4> { typedef uint32_t type __attribute__((aligned(2))); };
template <> struct Piece<2> { typedef uint16_t type; };
template <class T, int kRun> using PieceOf = typename Piece<kRun * (int)sizeof(T)>::type;

// x / n for x n < 2^32
__device__ __forceinline__ int quotient(int x, unsigned magic) { return magic ? (int)__umulhi((unsigned)x, magic) : x; }

// kRun elements in one access; kBeside: a pair's elements lie beside each other, else half of what is turned apart.
template <class T, int kRun, bool kBeside, class P> __global__ void __launch_bounds__(256) k_rotary(RotaryArgs d) {
    constexpr int kPairs = kBeside ? kRun / 2 : kRun;
    __shared__ alignas(16) float cosines[kTable], sines[kTable];     // [tokens][pairs]
    const long long block = block_number();
    const int group = (int)(block % d.head_blocks);
    const long long first = block / d.head_blocks * d.block_tokens;
    if (first >= d.tokens) return;
    const int tokens = d.tokens - first < d.block_tokens ? (int)(d.tokens - first) : d.block_tokens;
    const int all = d.heads[0] + d.heads[1], h0 = group * d.block_heads, heads = h0 + d.block_heads < all ? d.block_heads : all - h0, items = tokens * d.block_heads * d.units;
    using R = Run<T, kRun>;
    using W = PieceOf<T, kRun>;
    const auto load = [](const T* p) { return __builtin_bit_cast(R, *(const W*)p); };
    const auto store = [](T* p, const R& r) { *(W*)p = __builtin_bit_cast(W, r); };
    const int rest = d.head_dim - 2 * d.pairs;
    constexpr int kBatch = 4;                              // runs whose loads are on their way together
    R lo[kBatch], hi[kBatch];
    T* to[kBatch];
    int angle[kBatch];                                     // of the first pair in the table; -1: not turned, -2: no run
    const auto fetch = [&](int i0) {
#pragma unroll
        for (int n = 0; n < kBatch; n++) {
            const int i = i0 + 256 * n, row = quotient(i, d.unit_magic), unit = i - row * d.units, t = quotient(row, d.head_magic), own = row - t * d.block_heads;
            const int which = h0 + own >= d.heads[0], h = which ? h0 + own - d.heads[0] : h0 + own;
            const bool turned = unit < d.turned_units;
            // the last run of what is turned, and of the rest, ends where these do: it lies over the one before it where they are no multiple of it (what both write is the same)
            const int pair = unit * kPairs < d.pairs - kPairs ? unit * kPairs : d.pairs - kPairs, beyond = (unit - d.turned_units) * kRun, room = rest > kRun ? rest - kRun : 0;
            const int at = turned ? (kBeside ? 2 * pair : pair) : 2 * d.pairs + (beyond < room ? beyond : room);
            angle[n] = i >= items || own >= heads ? -2 : turned ? t * d.pairs + pair : -1;
            to[n] = (T*)d.y[which] + ((first + t) * d.heads[which] + h) * d.head_dim + at;
            if (angle[n] == -2) continue;
            const T* x = (const T*)d.x[which] + (first + t) * d.token_stride[which] + h * d.head_stride[which] + at;
            if (turned || rest >= kRun) lo[n] = load(x);
            else {
#pragma unroll
                for (int k = 0; k < kRun; k++) lo[n].v[k] = k < rest ? x[k] : (T)0.f;
            }
            if (!kBeside && turned) hi[n] = load(x + d.pairs);
        }
    };
    fetch(threadIdx.x);                                    // (on their way while the table is made)
    for (int i = threadIdx.x; i < tokens * d.pairs; i += 256) {
        const int t = quotient(i, d.pair_magic), p = i - t * d.pairs;
        const long long at = (long long)((const P*)d.positions)[(first + t) * d.position_stride + d.axis[p]];
        float c, s;
        cos_sin((unsigned long long)at * d.turn[p], c, s);
        cosines[i] = c;
        sines[i] = d.backward ? -s : s;
    }
    __syncthreads();
    for (int i0 = threadIdx.x;;) {
#pragma unroll
        for (int n = 0; n < kBatch; n++) {
            if (angle[n] == -2) continue;
            if (angle[n] == -1) {
                if (rest >= kRun) store(to[n], lo[n]);
                else {
#pragma unroll
                    for (int k = 0; k < kRun; k++) if (k < rest) to[n][k] = lo[n].v[k];
                }
                continue;
            }
            float c[kPairs], s[kPairs];
#pragma unroll
            for (int k = 0; k < kPairs; k++) { c[k] = cosines[angle[n] + k]; s[k] = sines[angle[n] + k]; }
            R out, out2;
#pragma unroll
            for (int k = 0; k < kPairs; k++) {
                const float a = (float)(kBeside ? lo[n].v[2 * k] : lo[n].v[k]), b = (float)(kBeside ? lo[n].v[2 * k + 1] : hi[n].v[k]);
                const T a2 = (T)__builtin_fmaf(a, c[k], -(b * s[k])), b2 = (T)__builtin_fmaf(a, s[k], b * c[k]);
                if constexpr (kBeside) { out.v[2 * k] = a2; out.v[2 * k + 1] = b2; }
                else { out.v[k] = a2; out2.v[k] = b2; }
            }
            store(to[n], out);
            if constexpr (!kBeside) store(to[n] + d.pairs, out2);
        }
        if ((i0 += 256 * kBatch) >= items) break;
        fetch(i0);
    }
}

const char* wrong(const ntc_rotary_desc* d) {
    if (!d) return "no description";
    if (d->tokens < 0 || d->heads[0] < 0 || d->heads[1] < 0 || (int64_t)d->heads[0] + d->heads[1] > 1 << 20) return "tokens and heads from 0 on, at most 2^20 heads, are needed";
    if (d->head_dim < 2 || d->head_dim > 1 << 14 || d->head_dim % 2) return "a head has 2 to 16384 elements, an even number";
    if (((int64_t)d->heads[0] + d->heads[1]) * d->head_dim > 1 << 28) return "a token has at most 2^28 elements";
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
            a.axis[p] = m;
        }
    }
    // The widest access, up to 16 bytes, that what is turned holds; what is not turned is copied by the same. (Rows may start at any element. 65536 tokens of 4 heads of 256 bfloat16: 50 us with 8 pairs or
    // more, 68, 98 and 166 with 4, 2 and 1.)
    int run = 16 / (int)type_size(d->dtype);
    const bool beside = d->interleaved != 0;                   // (pairs in one run)
    while (run > (beside ? 2 * a.pairs : a.pairs)) run /= 2;
    const int run_pairs = beside ? run / 2 : run;
    a.turned_units = (a.pairs + run_pairs - 1) / run_pairs;
    a.units = a.turned_units + (d->head_dim - 2 * a.pairs + run - 1) / run;
    // Tokens of a block: as many as give each thread four runs, where the table holds them; heads of one token in several blocks where tokens are few.
    const auto magic = [](int n) { return n > 1 ? (unsigned)((((uint64_t)1 << 32) + n - 1) / n) : 0u; };
    constexpr int kItems = 1024;
    const int row = heads * a.units;
    a.block_tokens = kItems / row < 1 ? 1 : kItems / row;
    if (a.block_tokens > kTable / a.pairs) a.block_tokens = kTable / a.pairs;
    while (a.block_tokens > 1 && d->tokens / a.block_tokens < 512) a.block_tokens /= 2;
    a.block_heads = heads;
    while (a.block_heads > 1 && a.block_tokens * a.block_heads * a.units > kItems) a.block_heads = (a.block_heads + 1) / 2;
    while (a.block_tokens == 1 && a.block_heads > 1 && a.block_heads * a.units > 256 && d->tokens * ((heads + a.block_heads - 1) / a.block_heads) < 512) a.block_heads = (a.block_heads + 1) / 2;
    a.head_blocks = (heads + a.block_heads - 1) / a.block_heads;
    a.unit_magic = magic(a.units);
    a.head_magic = magic(a.block_heads);
    a.pair_magic = magic(a.pairs);
    const dim3 grid = grid_of((d->tokens + a.block_tokens - 1) / a.block_tokens * a.head_blocks);
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
