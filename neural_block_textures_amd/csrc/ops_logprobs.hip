// Token log probabilities with entropy and the best alternatives, and their gradient (include/ntc_ops.h).
#include <string.h>

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

// log p of one value, in nats: not through (x - m) k, which overflows for a mask of the lowest value, and on halves, since the difference itself may
__device__ __forceinline__ float log_prob(float x, float m, float inv_t, float log_s) { return 2.0f * ((0.5f * x - 0.5f * m) * inv_t) - kLn2 * log_s; }

__device__ __forceinline__ long long token_of(const ntc_logprobs_desc& d, long long outer, long long inner) {
    const long long at = outer * d.token_outer_stride + inner * d.token_inner_stride;
    return d.token_bytes == 8 ? ((const long long*)d.tokens)[at] : ((const int*)d.tokens)[at];
}

template <class T> __device__ __forceinline__ const T* row_of(const ntc_logprobs_desc& d, long long row, long long& outer, long long& inner) {
    outer = 0;
    inner = row;
    if (d.inner_rows < d.rows) {                            // (fewer than 2^31 rows: a 64-bit division is a tenth of a short row's work)
        outer = (uint32_t)row / (uint32_t)d.inner_rows;
        inner = (uint32_t)row % (uint32_t)d.inner_rows;
    }
    return (const T*)d.logits + outer * d.outer_stride + inner * d.inner_stride;
}
// Row first + own: first is the same in all lanes.
template <class T> __device__ __forceinline__ const T* row_of(const ntc_logprobs_desc& d, long long first, int own) {
    if (d.inner_rows < d.rows) {
        long long outer, inner;
        return row_of<T>(d, first + own, outer, inner);
    }
    return (const T*)d.logits + first * d.inner_stride + own * d.inner_stride;
}
// What stands at a row's token: 0 where there is none.
template <class T> __device__ __forceinline__ float value_at(const ntc_logprobs_desc& d, const T* x, long long t) { return t != d.ignore_index && t >= 0 && t < d.V ? (float)x[t] : 0.0f; }
// The results of a row but its alternatives, from its softmax with the largest value m (kLowest or less: see none) and the token's value.
__device__ __forceinline__ void write_row(const ntc_logprobs_desc& d, long long row, float at_token, long long t, float m, float log_s, float ratio, bool none, float inv_t) {
    float lp = 0.0f;
    if (t != d.ignore_index) lp = t < 0 || t >= d.V ? __builtin_nanf("") : none ? -NTC_INF : log_prob(at_token, m, inv_t, log_s);
    d.logprob[row] = lp;
    d.entropy[row] = none ? 0.0f : kLn2 * (log_s - ratio);
    d.stats[2 * row] = none ? -NTC_INF : m;
    d.stats[2 * row + 1] = log_s;
}

// Sixteen bytes of a row at its ragged end: the `left` values (fewer than a run) from x[at] on, zeros after them, and their store.
typedef unsigned __int128 Bits;
template <class T> __device__ __forceinline__ Bits last_run(const T* x, int V, int at, int left) {
    constexpr int kVec = 16 / (int)sizeof(T);
    if (V >= kVec) return __builtin_bit_cast(Bits, *(const LooseRun<T, kVec>*)(x + V - kVec)) >> (8 * (int)sizeof(T) * (kVec - left));
    LooseRun<T, kVec> r = {};
    for (int j = 0; j < kVec; j++) if (j < left) r.v[j] = x[at + j];
    return __builtin_bit_cast(Bits, r);
}
template <class T> __device__ __forceinline__ void store_last(T* to, Bits w, int left) {
    uint8_t* p = (uint8_t*)to;
    const int bytes = left * (int)sizeof(T);
    if (bytes & 8) { *(LooseRun<uint16_t, 4>*)p = __builtin_bit_cast(LooseRun<uint16_t, 4>, (uint64_t)w); p += 8; w >>= 64; }
    if (bytes & 4) { *(LooseRun<uint16_t, 2>*)p = __builtin_bit_cast(LooseRun<uint16_t, 2>, (uint32_t)w); p += 4; w >>= 32; }
    if (bytes & 2) *(uint16_t*)p = (uint16_t)w;
}

// ---------------------------------------------------------------- short rows
// Integers that order as floats do (-0 as 0), and back.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t h = __float_as_uint(x + 0.0f);
    return h ^ ((uint32_t)((int)h >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// The same for 16-bit types, two to a word, as signed 16-bit integers: a magnitude or its negative.
template <class T> struct Half {
    typedef short s2 __attribute__((ext_vector_type(2)));
    static constexpr int kInf = type_code<T> == NTC_BF16 ? 0x7f80 : 0x7c00, kNone = -0x8000;   // larger magnitudes are NaN; no value's key
    static __device__ __forceinline__ s2 order(uint32_t w) {
        const s2 x = __builtin_bit_cast(s2, w), sign = x >> (short)15;
        return __builtin_bit_cast(s2, (w & 0x7fff7fffu) ^ __builtin_bit_cast(uint32_t, sign)) - sign;
    }
    static __device__ __forceinline__ float value(int k) {
        const uint16_t h = (uint16_t)(k < 0 ? -k | 0x8000 : k);
        return (float)__builtin_bit_cast(T, h);
    }
};

__device__ __forceinline__ uint32_t above(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t below(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ int above(int a, int b) { return a > b ? a : b; }
__device__ __forceinline__ int below(int a, int b) { return a < b ? a : b; }
// A lane's three best keys, in order. 16-bit types: the index is in the key.
constexpr int kNoKey = (int)0x80000000;
struct Three {
    int a = kNoKey, b = kNoKey, c = kNoKey;
    __device__ __forceinline__ static int middle(int x, int y, int z) { return above(below(x, y), below(above(x, y), z)); }   // one instruction
    __device__ __forceinline__ void add(int k) { c = middle(b, c, k); b = middle(a, b, k); a = above(a, k); }
    __device__ __forceinline__ void next() { a = b; b = c; c = kNoKey; }
};
// With the index beside the key; added in ascending order, so that the first of equals stays ahead.
struct ThreePlaced {                                          // (0: none)
    uint32_t a = 0, b = 0, c = 0, ia = ~0u, ib = ~0u, ic = ~0u;
    __device__ __forceinline__ void add(uint32_t k, uint32_t i) {
        const bool pa = k > a, pb = k > b, pc = k > c;
        c = pb ? b : pc ? k : c;
        ic = pb ? ib : pc ? i : ic;
        b = pa ? a : pb ? k : b;
        ib = pa ? ia : pb ? i : ib;
        a = pa ? k : a;
        ia = pa ? i : ia;
    }
    __device__ __forceinline__ void next() { a = b; b = c; c = 0; ia = ib; ib = ic; ic = ~0u; }
};

// A group of kGroup lanes holds a row in registers, 16 neighbouring values a lane: the largest, then the sums, then the alternatives one by
// one, from the lanes' three best, through LDS to whole runs of the results. A 16-bit value's key is ordered two at a time and leaves half a
// word to its index (from the top down, in a row of at most 1024): one word orders values and indices both. A 32-bit value's index is found in
// a second reduction. What is written of rows is left to one lane a row (and one an alternative), since a wave's instructions cost as much for 4 rows
// as for 64. Bound by vector instructions (359 a wave with 4 alternatives): 262144 rows of 256 bf16 values 42 us with 4 alternatives, 3.6 TB/s; 400000
// x 64 14.3 us without, at the rate of their bytes.
constexpr int kShort = 1024;                                 // the longest such row
// Sixteen values in descending order: exchanges of pairs, halves merged odd with even.
template <class K> __device__ __forceinline__ void sort16(K (&a)[16]) {
#pragma unroll
    for (int p = 1; p < 16; p *= 2)
#pragma unroll
        for (int k = p; k; k /= 2)
#pragma unroll
            for (int j = 0; j < 16 - k; j++)
                if (j >= k % p && ((j - k % p) / k) % 2 == 0 && j / (2 * p) == (j + k) / (2 * p)) {
                    const K x = a[j], y = a[j + k];
                    a[j] = x > y ? x : y;
                    a[j + k] = x > y ? y : x;
                }
}
//
// The sums are taken on products x k - m k, one operation fewer a value than on differences, where these stay exact: |m k| up to `most` = 2^24 (its
// rounding, which every exponent is off by, is then at most 1/2 and is taken out again; past 2^31 it would be beyond an exponential's range), k from 2^-60
// on (what is past a row's end stands as -lim, and exp2(-lim k) has to be 0; `most` is -1 for smaller ones), and no product that overflows to an infinity
// whose e of 0 would give 0 * inf: values below -lim (`low`: that as a 16-bit key) go with the infinities and NaN.
template <class T, int kGroup, bool kSorted> __global__ void __launch_bounds__(256) k_logprobs_short(ntc_logprobs_desc d, float lim, int low, float most, float k, float inv_t) {
    constexpr int kEach = 16, kVec = 16 / (int)sizeof(T), kRows = 256 / kGroup;
    constexpr bool kPlaced = sizeof(T) == 4;
    static_assert(kGroup * kEach <= kShort, "indices of 10 bits");
    using H = Half<T>;
    using s2 = typename H::s2;
    __shared__ uint32_t keys[kRows][NTC_MAX_TOP], places[kPlaced ? kRows : 1][NTC_MAX_TOP];
    __shared__ Soft stat[kRows];
    using Key = std::conditional_t<kPlaced, unsigned long long, int>;
    __shared__ Key lists[kSorted ? kEach + 1 : 1][256];
    const int in = threadIdx.x % kGroup, own = threadIdx.x / kGroup;
    const long long first = block_number() * kRows;
    if (first >= d.rows) return;
    const int last_row = d.rows - first < kRows ? (int)(d.rows - first) - 1 : kRows - 1;   // of this block; past it the same again, not written
    // A row's lanes have its sums, but what is written of rows is left to one lane each, once all have theirs: what it needs is asked for now.
    long long token = 0;
    float at_token = 0.0f;
    const T* token_row = nullptr;
    if ((int)threadIdx.x <= last_row) {
        long long outer, inner;
        token_row = row_of<T>(d, first + threadIdx.x, outer, inner);
        token = token_of(d, outer, inner);
    }
    const T* x = row_of<T>(d, first, own < last_row ? own : last_row);
    const int V = (int)d.V, at = in * kEach;
    float v[kEach];
    s2 pair[kEach / 2], least = { 0, 0 };                    // keys of 16-bit values, and the least of the whole vectors'
    bool odd = false;                                        // a 16-bit value below -lim, infinity or NaN
#pragma unroll
    for (int i = 0; i < kEach; i += kVec) {
        const int left = V - at - i;                         // of this vector's values
        if (left >= kVec) {
            const auto r = *(const LooseRun<T, kVec>*)(x + at + i);
#pragma unroll
            for (int j = 0; j < kVec; j++) v[i + j] = (float)r.v[j];
            if constexpr (!kPlaced) {
                const uint4 w = __builtin_bit_cast(uint4, r);
                const uint32_t words[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    pair[i / 2 + q] = H::order(words[q]);
                    least = __builtin_elementwise_min(least, pair[i / 2 + q]);
                }
            }
        } else {
            Bits w = 0, inside = 0;                          // this lane's values, and ones where there are any
            if (left > 0) {
                w = last_run(x, V, at + i, left);
                inside = ~(Bits)0 >> (8 * (int)sizeof(T) * (kVec - left));
            }
            const auto r = __builtin_bit_cast(LooseRun<T, kVec>, w);
#pragma unroll
            for (int j = 0; j < kVec; j++) v[i + j] = j < left ? (float)r.v[j] : kPlaced ? -NTC_INF : -lim;
            if constexpr (!kPlaced) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const s2 key = H::order((uint32_t)(w >> 32 * q));
                    const uint32_t in_row = (uint32_t)(inside >> 32 * q);
                    least = __builtin_elementwise_min(least, key);   // (past the end: 0)
                    pair[i / 2 + q] = __builtin_bit_cast(s2, (__builtin_bit_cast(uint32_t, key) & in_row) | (0x80008000u & ~in_row));
                }
            }
        }
    }
    const auto larger = [](float a, float b) { return fmaxf(a, b); };
    const auto sum = [](float a, float b) { return a + b; };
    float m;
    if constexpr (kPlaced) {
        m = v[0];
#pragma unroll
        for (int j = 1; j < kEach; j++) m = fmaxf(m, v[j]);
        m = reduce<kGroup>(m, larger);
    } else {
        const auto most = [&] {
            s2 p = pair[0];
#pragma unroll
            for (int q = 1; q < kEach / 2; q++) p = __builtin_elementwise_max(p, pair[q]);
            return above((int)p[0], (int)p[1]);
        };
        int top = most();
        odd = top >= H::kInf || below((int)least[0], (int)least[1]) <= -low;
        odd = __ballot(odd) != 0;
        if (odd) {                                           // a NaN counts as -inf in the order
            asm volatile("");                                // (a branch, not selections that every row would make)
#pragma unroll
            for (int q = 0; q < kEach / 2; q++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int c = pair[q][h];
                    pair[q][h] = (short)(c > H::kInf || (c < -H::kInf && c != H::kNone) ? -H::kInf : c);
                }
            top = most();
        }
        top = reduce<kGroup>(top, [](int a, int b) { return above(a, b); });
        m = H::value(top);
    }
    if (token_row) at_token = value_at(d, token_row, token);
    const float mm = m == -NTC_INF ? 0.0f : m;              // nothing left: every exponential is 0
    float s = 0.0f, t = 0.0f;
    const float mk = mm * k, off = __builtin_fmaf(mm, k, -mk);
    if (__ballot(!(fabsf(mk) <= most)) == 0) {              // the exponents are `off` too large
        if (!kPlaced && !odd) {
#pragma unroll
            for (int j = 0; j < kEach; j++) {
                const float q = __builtin_fmaf(v[j], k, -mk), e = fast_exp2(q);
                s += e;
                t = __builtin_fmaf(e, q, t);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kEach; j++) {
                const float q = __builtin_fmaf(v[j], k, -mk), e = fast_exp2(q);
                s += e;
                t = __builtin_fmaf(e, fmaxf(q, -1e30f), t);  // (an e of 0 may have q = -inf)
            }
        }
        const float f = fast_exp2(-off);
        t = f * __builtin_fmaf(-s, off, t);
        s *= f;
    } else {
#pragma unroll
        for (int j = 0; j < kEach; j++) {
            const float q = ((at + j < V ? v[j] : -NTC_INF) - mm) * k, e = fast_exp2(q);
            s += e;
            t = __builtin_fmaf(e, fmaxf(q, -1e30f), t);
        }
    }
    s = reduce<kGroup>(s, sum);
    t = reduce<kGroup>(t, sum);
    if (in == 0) stat[own] = { mm, s, t };
    if (d.top) {
        if constexpr (kPlaced) {
            if (__ballot(s != s)) {                              // a NaN somewhere (or +inf): in the order it counts as -inf
#pragma unroll
                for (int j = 0; j < kEach; j++) v[j] = v[j] != v[j] ? -NTC_INF : v[j];
            }
            uint32_t key[kEach];
#pragma unroll
            for (int j = 0; j < kEach; j++) key[j] = order_key(v[j]);
            if (V < kGroup * kEach) {
                asm volatile("");
#pragma unroll
                for (int j = 0; j < kEach; j++) key[j] = at + j < V ? key[j] : 0;   // below every key of a value
            }
            if constexpr (kSorted) {
                Key all[kEach];
#pragma unroll
                for (int j = 0; j < kEach; j++) all[j] = (Key)key[j] << 32 | (uint32_t)~(at + j);
                sort16(all);
#pragma unroll
                for (int j = 0; j < kEach; j++) lists[j][threadIdx.x] = all[j];
                lists[kEach][threadIdx.x] = 0;
                const Key* next = &lists[0][threadIdx.x];
                Key head = all[0];
                for (int r = 0; r < d.top; r++) {
                    const uint32_t mine = (uint32_t)(head >> 32), last = reduce<kGroup>(mine, [](uint32_t a, uint32_t b) { return above(a, b); });
                    const uint32_t place = reduce<kGroup>(mine == last ? (uint32_t)head : 0u, [](uint32_t a, uint32_t b) { return above(a, b); });
                    if (in == 0) { keys[own][r] = last; places[own][r] = ~place; }
                    if (mine == last && (uint32_t)head == place) next += 256;
                    head = *next;
                }
            } else {
            ThreePlaced best;
#pragma unroll
            for (int j = 0; j < kEach; j++) best.add(key[j], (uint32_t)(at + j));
            for (int r = 0; r < d.top; r++) {
                const uint32_t last = reduce<kGroup>(best.a, [](uint32_t a, uint32_t b) { return above(a, b); });
                const uint32_t place = reduce<kGroup>(best.a == last ? best.ia : ~0u, [](uint32_t a, uint32_t b) { return below(a, b); });
                const bool took = best.a == last && best.ia == place;
                if (in == 0) { keys[own][r] = last; places[own][r] = place; }
                if (took) best.next();
                if (__ballot(took && best.a == 0 && r + 1 < d.top)) {   // a lane has given its three: again from those that come after the last
                    asm volatile("");
                    best = {};
#pragma unroll
                    for (int j = 0; j < kEach; j++) {
                        const bool open = key[j] < last || (key[j] == last && (uint32_t)(at + j) > place);
                        best.add(open ? key[j] : 0, (uint32_t)(at + j));
                    }
                }
            }
            }
        } else {
            // Values in the upper half, the index from the top down in the lower one: its last four bits now, the lane's once the three are known.
            const auto key = [&](int j) { return (int)__builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, pair[j / 2]), (uint32_t)(15 - j), j & 1 ? 0x07060100u : 0x05040100u); };
            const int lane_bits = kShort - kEach - at;
            if constexpr (kSorted) {
                int all[kEach];
#pragma unroll
                for (int j = 0; j < kEach; j++) all[j] = key(j);
                sort16(all);
#pragma unroll
                for (int j = 0; j < kEach; j++) lists[j][threadIdx.x] = all[j];
                lists[kEach][threadIdx.x] = kNoKey;
                const int* next = &lists[0][threadIdx.x];
                int head = all[0] | lane_bits;
                for (int r = 0; r < d.top; r++) {
                    const int last = reduce<kGroup>(head, [](int a, int b) { return above(a, b); });
                    if (in == 0) keys[own][r] = (uint32_t)last;
                    if (head == last) next += 256;
                    head = *next | lane_bits;
                }
            } else {
            Three best;
#pragma unroll
            for (int j = 0; j < kEach; j++) best.add(key(j));
            best.a |= lane_bits; best.b |= lane_bits; best.c |= lane_bits;
            for (int r = 0; r < d.top; r++) {
                const int last = reduce<kGroup>(best.a, [](int a, int b) { return above(a, b); });
                const bool took = best.a == last;
                if (in == 0) keys[own][r] = (uint32_t)last;
                if (took) best.next();
                if (__ballot(took && best.a >> 16 == H::kNone && r + 1 < d.top)) {
                    int bits = lane_bits;
                    asm volatile("" : "+v"(bits));               // (else the comparisons' words would be made for every row)
                    best = {};
#pragma unroll
                    for (int j = 0; j < kEach; j++) best.add((key(j) | bits) < last ? key(j) : kNoKey);
                    best.a |= lane_bits; best.b |= lane_bits; best.c |= lane_bits;
                }
            }
            }
        }
    }
    __syncthreads();
    if ((int)threadIdx.x <= last_row) {
        const Soft a = stat[threadIdx.x];
        write_row(d, first + threadIdx.x, at_token, token, a.m, fast_log2(a.s), a.t * __builtin_amdgcn_rcpf(a.s), a.s == 0.0f, inv_t);
    }
    // alternatives by the other waves first
    for (int e = threadIdx.x ^ 192; e < (last_row + 1) * d.top; e += 256) {
        const int own = e / d.top, r = e % d.top;
        const uint32_t found = keys[own][r];
        uint32_t place;
        float w;
        if constexpr (kPlaced) { place = places[own][r]; w = key_value(found); }
        else { place = kShort - 1 - (found & (kShort - 1)); w = H::value((int)found >> 16); }
        const Soft a = stat[own];
        d.top_ids[first * d.top + e] = place;
        // (a NaN in the row has made the sum NaN, which swallows what stands for it here)
        d.top_logprobs[first * d.top + e] = a.s == 0.0f ? -NTC_INF : log_prob(w, a.m, inv_t, fast_log2(a.s));
    }
}

// ---------------------------------------------------------------- long rows
// The best values of what a wave has read: up to 64 candidates in LDS that its chunks add to; full, they are put in order (each counts
// those before it) and the first `top` stay. Empty places of a finished list are (-inf, kNoIndex).
constexpr int kNoIndex = 0x7fffffff, kCandidates = 64;
struct Best { float v; int i; };
__device__ __forceinline__ unsigned long long place_key(float w, int j) { return (unsigned long long)order_key(w) << 32 | (uint32_t)~j; }   // larger: comes first
struct Candidates {
    float* v;
    int* i;
    int n = 0, ordered = 0;                                  // the same in all lanes; the first `ordered` are in order
    __device__ __forceinline__ void put_in_order(int top) {
        const int lane = lane_id();
        if (n == ordered) return;
        wave_shared();
        const float w = lane < n ? v[lane] : -NTC_INF;
        const int j = lane < n ? i[lane] : kNoIndex;
        const uint32_t key = lane < n ? order_key(w) : 0;
        const unsigned long long mine = (unsigned long long)key << 32 | (uint32_t)~j;
        int before = 0;
        for (int l = 0; l < n; l += 4) {                     // (lanes past n come after all others)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const unsigned long long other = (unsigned long long)(uint32_t)__builtin_amdgcn_readlane(key, l + u) << 32 | (uint32_t)__builtin_amdgcn_readlane(~j, l + u);
                before += other > mine;
            }
        }
        wave_shared();
        if (lane < n && before < top) { v[before] = w; i[before] = j; }
        n = ordered = n < top ? n : top;
        wave_shared();
    }
    // lanes of `ask` add (w, j); returns those that found no place
    __device__ __forceinline__ unsigned long long add(unsigned long long ask, float w, int j) {
        const int at = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(ask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ask, 0u));
        const bool mine = ask >> lane_id() & 1;
        if (mine && at < kCandidates) { v[at] = w; i[at] = j; }
        const unsigned long long rest = __ballot(mine && at >= kCandidates);
        n += __builtin_popcountll(ask) - __builtin_popcountll(rest);
        return rest;
    }
};
// A bound that the K-th largest of 64 lanes' values reaches, within a 2^-10 of its size: its highest bits, one by one.
__device__ __forceinline__ float kth_largest(float x, int k) {
    const uint32_t key = order_key(x != x ? -NTC_INF : x);
    uint32_t t = 0;
#pragma unroll
    for (uint32_t bit = 1u << 31; bit >= 1u << 13; bit >>= 1)
        if (__builtin_popcountll(__ballot(key >= (t | bit))) >= k) t |= bit;
    return t <= 0x007fffffu ? -NTC_INF : key_value(t);
}

// The best of up to 64 lists in LDS (list p's values at v + p stride, indices at i + p stride, in order): all lists' first, then all second ones,
// as many ranks at a time as fit 64 lanes, until a rank has nothing that comes before the `top` values found so far. `list` is empty.
__device__ __forceinline__ Best merge(Candidates& list, const float* v, const int* i, int stride, int lists, int top) {
    const int lane = lane_id(), ranks = 64 / lists, p = lane % lists, r0 = lane / lists;
    unsigned long long bar = 0;                              // (every value's key is above 0)
    for (int r = r0; __ballot(r < top && r0 < ranks); r += ranks) {
        const bool in = r < top && r0 < ranks;
        const float w = in ? v[p * stride + r] : -NTC_INF;
        const int j = in ? i[p * stride + r] : kNoIndex;
        unsigned long long ask = __ballot(j != kNoIndex && place_key(w, j) > bar);
        if (!ask) break;
        while (ask) {
            ask = list.add(ask, w, j);
            if (list.n < kCandidates) break;
            list.put_in_order(top);
            bar = place_key(list.v[top - 1], list.i[top - 1]);
            ask &= __ballot(place_key(w, j) > bar);
        }
        if (list.n >= top + 16) {
            list.put_in_order(top);
            bar = place_key(list.v[top - 1], list.i[top - 1]);
        }
    }
    list.put_in_order(top);
    return lane < list.n ? Best{ list.v[lane], list.i[lane] } : Best{ -NTC_INF, kNoIndex };
}

// A lane's value of another lane (0 where there is none): rows of 16 shifted, or a row's last lane to those after.
template <int kCtrl, int kRows = 0xf> __device__ __forceinline__ uint32_t before(uint32_t x) { return __builtin_amdgcn_update_dpp(0, x, kCtrl, kRows, 0xf, false); }

// What a lane reads at a time: kRun values in vectors of 16 bytes.
template <class T> struct Long { static constexpr int kVec = 16 / (int)sizeof(T), kVecs = 2, kRun = kVec * kVecs, kChunk = 64 * kRun; };

// Adds all values of a chunk that reach `least`, in ascending order of index, if the list has room for them: each lane's places
// from a prefix sum over the lanes, of both vectors at once.
template <int kRun> __device__ __forceinline__ bool add_run(Candidates& list, const float (&v)[kRun], float least, int base) {
    constexpr int kVec = kRun / 2;
    uint32_t low = 0, high = 0;
#pragma unroll
    for (int j = 0; j < kVec; j++) { low += v[j] >= least; high += v[kVec + j] >= least; }
    const uint32_t own = low | high << 16;
    uint32_t x = own;
    x += before<0x111>(x);
    x += before<0x112>(x);
    x += before<0x114>(x);
    x += before<0x118>(x);                                   // within rows of 16 lanes
    x += before<0x142, 0xa>(x);                              // the last lane's of row 0 to row 1, of 2 to 3
    x += before<0x143, 0xc>(x);                              // lane 31's to rows 2 and 3
    const uint32_t total = __builtin_amdgcn_readlane(x, 63);
    const int n = list.n + (int)(total & 0xffffu) + (int)(total >> 16);
    if (n > kCandidates) return false;
    x -= own;
    int at = list.n + (int)(x & 0xffffu), at1 = list.n + (int)(total & 0xffffu) + (int)(x >> 16);
    base += lane_id() * kVec;
#pragma unroll
    for (int j = 0; j < kVec; j++) if (v[j] >= least) { list.v[at] = v[j]; list.i[at++] = base + j; }
#pragma unroll
    for (int j = 0; j < kVec; j++) if (v[kVec + j] >= least) { list.v[at1] = v[kVec + j]; list.i[at1++] = base + 64 * kVec + j; }
    list.n = n;
    return true;
}

// A wave's share of a row: chunks first, first + step, .. below `end` (chunks of kChunk values, the last one ragged).
// The sums are each lane's own, on a floor that only rises: exp2(x k - m k) is one fused operation and an exponential, with m held
// within lim so that neither product overflows. A row whose values all lie below -lim, or reach past lim, or hold NaN ends with s = 0, infinite or
// NaN and is read again by scan_again(). Values become candidates where their lane's largest of a chunk passes what `top` values are known to
// reach: its own, or those of another wave of the row (bar: as an integer that orders; only ever raised).
// A chunk's terms are added to each other first, and sixteen chunks' sums before they join the rest: added one by one, what is below half a unit of the
// sum would be lost, always downwards (131072 values, one of them 16.75 above the rest: log p off by 1.1e-4 so, by 1e-6 now; 0.3% of the time).
constexpr uint32_t kLowestKey = 0x00800000u;                 // kLowest as an integer that orders
template <class T> __device__ __forceinline__ void scan(const T* x, int V, int first, int step, int end, float k, float lim, int top, Soft& a, Candidates& list, uint32_t* bar) {
    using L = Long<T>;
    const int lane = lane_id();
    a = { -lim, 0.0f, 0.0f };
    float mk = -lim * k, far_s = 0.0f, far_t = 0.0f;         // sums of the chunks before the last few
    int near = 0;
    float least = kLowest;                                   // the least value that a candidate may have
    bool fresh = true;
    for (int c = first; c < end; c += step) {
        float v[L::kRun];
        const int base = c * L::kChunk;
        const int at0 = base + lane * L::kVec;
        const uint32_t others = top && bar ? *(volatile uint32_t*)bar : 0;
        if (base + L::kChunk <= V) {
#pragma unroll
            for (int i = 0; i < L::kVecs; i++) {
                const auto r = *(const LooseRun<T, L::kVec>*)(x + at0 + i * 64 * L::kVec);
#pragma unroll
                for (int j = 0; j < L::kVec; j++) v[i * L::kVec + j] = (float)r.v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < L::kVecs; i++) {
                const int at = at0 + i * 64 * L::kVec, left = V - at;
                Bits w = 0;
                if (left >= L::kVec) w = __builtin_bit_cast(Bits, *(const LooseRun<T, L::kVec>*)(x + at));
                else if (left > 0) w = last_run(x, V, at, left);
                const auto r = __builtin_bit_cast(LooseRun<T, L::kVec>, w);
#pragma unroll
                for (int j = 0; j < L::kVec; j++) v[i * L::kVec + j] = j < left ? (float)r.v[j] : -NTC_INF;
            }
        }
        float cm = v[0];
#pragma unroll
        for (int j = 1; j < L::kRun; j++) cm = fmaxf(cm, v[j]);
        if (cm > a.m) {
            a.m = fminf(cm, lim);
            const float was = mk, f = fast_exp2(was - a.m * k);   // between the rounded products, which the exponents are taken on
            mk = a.m * k;
            a.t = f * __builtin_fmaf(a.s, was - mk, a.t);
            a.s *= f;
            far_t = f * __builtin_fmaf(far_s, was - mk, far_t);
            far_s *= f;
        }
        float s = 0.0f, t = 0.0f;
#pragma unroll
        for (int j = 0; j < L::kRun; j++) {
            const float d = __builtin_fmaf(v[j], k, -mk), e = fast_exp2(d);
            s += e;
            t = __builtin_fmaf(e, fmaxf(d, -1e30f), t);
        }
        a.s += s;
        a.t += t;
        if (++near == 16) {
            far_s += a.s;
            far_t += a.t;
            a.s = a.t = 0.0f;
            near = 0;
        }
        if (!top) continue;
        least = fmaxf(least, key_value(others > kLowestKey ? others : kLowestKey));
        if (fresh) {
            least = fmaxf(least, kth_largest(cm, top));      // at least `top` values of the first chunk reach it
            if (bar && lane == 0) atomicMax(bar, order_key(least));
        }
        fresh = false;
        const unsigned long long lanes = __ballot(cm >= least);
        if (!lanes) continue;
        if (!(__builtin_popcountll(lanes) > 4 && add_run(list, v, least, base))) {
#pragma unroll
            for (int j = 0; j < L::kRun; j++) {
                unsigned long long ask = __ballot(v[j] >= least);
                while (ask) {
                    ask = list.add(ask, v[j], base + (j / L::kVec) * 64 * L::kVec + lane * L::kVec + j % L::kVec);
                    if (list.n == kCandidates) {
                        list.put_in_order(top);
                        least = fmaxf(least, list.v[top - 1]);
                        ask &= __ballot(v[j] >= least);
                    }
                }
            }
        }
        if (list.n >= top + 16) {                            // its last may only be passed, by later indices
            list.put_in_order(top);
            const uint32_t next = order_key(list.v[top - 1]) + 1;
            least = fmaxf(least, key_value(next));
            if (bar && lane == 0) atomicMax(bar, next - 1);
        }
    }
    if (top) {
        list.put_in_order(top);
        if (lane >= list.n && lane < top) { list.v[lane] = -NTC_INF; list.i[lane] = kNoIndex; }
    }
    a.s += far_s;
    a.t += far_t;
    if (a.s == 0.0f) return;                                 // (nothing above the floor: its m k has no meaning)
    // the sums were taken on the rounded m k: to those on m itself
    const float off = __builtin_fmaf(a.m, k, -mk);           // m k - fl(m k): every exponent was that much too large
    a.t -= a.s * off;
    const float f = fast_exp2(-off);
    a.t *= f;
    a.s *= f;
}

// The same sums for any values: on differences, which do not overflow where the values do not differ that much. One wave, whole row.
template <class T> __device__ __forceinline__ Soft scan_again(const T* x, int V, float k) {
    float m = kLowest;
    for (int i = lane_id(); i < V; i += 64) m = fmaxf(m, (float)x[i]);
    m = reduce64(m, [](float p, float q) { return fmaxf(p, q); });
    Soft a = { m, 0.0f, 0.0f }, near = a;
    int runs = 0;
    for (int base = 0; base < V; base += 64 * 16) {
        Soft run = { m, 0.0f, 0.0f };
        for (int i = base + lane_id(), u = 0; u < 16 && i < V; i += 64, u++) soft_add(run, (float)x[i], k);
        near.s += run.s;
        near.t += run.t;
        if (++runs % 16 == 0 || base + 64 * 16 >= V) {
            a.s += near.s;
            a.t += near.t;
            near.s = near.t = 0.0f;
        }
    }
    const auto sum = [](float p, float q) { return p + q; };
    a.s = reduce64(a.s, sum);
    a.t = reduce64(a.t, sum);
    return a;
}
// Whether a joined sum is that of an ordinary row: its largest value adds 1, and there are fewer than 2^31. (Less: all lie below the floor, and what is
// small beside them has been lost; more: they reach past lim, and the second sum may have overflowed first.)
__device__ __forceinline__ bool plain_sum(float s) { return s > 0.5f && s < 0x1p40f; }

__device__ __forceinline__ Soft join_lanes(Soft a, float k) {
    const auto sum = [](float p, float q) { return p + q; };
    const float m = reduce64(a.m, [](float p, float q) { return fmaxf(p, q); });
    soft_raise(a, m, k);
    a.s = reduce64(a.s, sum);
    a.t = reduce64(a.t, sum);
    return a;
}

// The rest of a row, by one wave that has its joined sums and best values: odd rows read again, places of the list that no number above -inf
// took filled with the first indices that hold -inf or NaN, and everything written.
template <class T> __device__ __forceinline__ void finish(const ntc_logprobs_desc& d, long long row, const T* x, long long t, Soft a, Best best) {
    const int lane = lane_id(), V = (int)d.V;
    const float inv_t = 1.0f / d.temperature, k = kLog2e / d.temperature;
    if (!plain_sum(a.s)) a = scan_again(x, V, k);
    const bool none = a.s == 0.0f;
    const float log_s = fast_log2(a.s);
    if (lane == 0) write_row(d, row, value_at(d, x, t), t, a.m, log_s, a.t / a.s, none, inv_t);
    if (!d.top) return;
    int have = __builtin_popcountll(__ballot(lane < d.top && best.i != kNoIndex));
    for (int i = 0; have < d.top && i < V; i += 64) {
        const bool low = i + lane < V && !((float)x[i + lane < V ? i + lane : 0] > -NTC_INF);
        unsigned long long ask = __ballot(low);
        while (ask && have < d.top) {
            const int l = __builtin_ctzll(ask);
            ask &= ask - 1;
            if (lane == have) { best.v = -NTC_INF; best.i = i + l; }
            have++;
        }
    }
    if (lane < d.top) {
        d.top_ids[row * d.top + lane] = best.i;
        d.top_logprobs[row * d.top + lane] = none ? -NTC_INF : log_prob(best.v, a.m, inv_t, log_s);
    }
}

// Memory bounds it where rows are many and alternatives few (bf16 4096 x 131072 with 16: 215 us, 5.0 TB/s; 8190 x 50001 without: 162 us, 5.1 TB/s), the
// two launches and the dependent steps of one wave's search where rows are few (1 x 131072: 4.9 us; with 8 alternatives 10.9, the 6 more being a bound
// from 19 ballots, one wave's ranking of candidates lane by lane, and two merges in series).
// kWaves waves (of a block of 4) read a row; with kParts a block reads the part blockIdx.y of a row and leaves its sums and list in the workspace.
template <class T, int kWaves, bool kParts> __global__ void __launch_bounds__(256) k_logprobs_long(ntc_logprobs_desc d, float lim, int part_chunks) {
    __shared__ Soft soft[4];
    constexpr int kLists = kWaves > 1 ? 5 : 4;               // (the last: of all waves)
    __shared__ float list_v[kLists][kCandidates];
    __shared__ int list_i[kLists][kCandidates];
    __shared__ uint32_t bar;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id();
    const long long row = (kParts ? blockIdx.x : block_number()) * (4 / kWaves) + wave / kWaves;
    if (row >= d.rows) return;                               // (kWaves 1: a wave on its own; else whole blocks)
    if (kWaves > 1) {
        if (threadIdx.x == 0) bar = 0;
        __syncthreads();
    }
    long long outer, inner;
    const T* x = row_of<T>(d, row, outer, inner);
    const float k = kLog2e / d.temperature;
    const int V = (int)d.V, chunks = (V + Long<T>::kChunk - 1) / Long<T>::kChunk;
    const int begin = kParts ? (int)blockIdx.y * part_chunks : 0, end = kParts && begin + part_chunks < chunks ? begin + part_chunks : chunks;
    Soft a;
    Candidates list = { list_v[wave], list_i[wave] };
    scan(x, V, begin + wave % kWaves, kWaves, end, k, lim, d.top, a, list, kWaves > 1 ? &bar : nullptr);
    a = join_lanes(a, k);
    Best best = { -NTC_INF, kNoIndex };
    if (kWaves > 1) {
        if (lane == 0) soft[wave] = a;
        __syncthreads();
        if (wave) return;
        for (int w = 1; w < kWaves; w++) soft_join(a, soft[w], k);
        if (d.top) {
            Candidates all = { list_v[kLists - 1], list_i[kLists - 1] };
            best = merge(all, list_v[0], list_i[0], kCandidates, kWaves, d.top);
        }
    } else if (lane < d.top) {
        best = { list.v[lane], list.i[lane] };
    }
    if (!kParts) { finish(d, row, x, token_of(d, outer, inner), a, best); return; }
    const int parts = gridDim.y;
    float* to = (float*)d.workspace + (row * parts + blockIdx.y) * (4 + 2 * d.top);
    if (lane == 0) { to[0] = a.m; to[1] = a.s; to[2] = a.t; }
    if (lane < d.top) { to[4 + lane] = best.v; ((int*)to)[4 + d.top + lane] = best.i; }
}

// Joins a row's parts: part p's sums and list in lane p.
constexpr int kMostParts = 64;
template <class T> __global__ void __launch_bounds__(256) k_logprobs_join(ntc_logprobs_desc d, int parts) {
    __shared__ float all[kMostParts * (4 + 2 * NTC_MAX_TOP)], list_v[kCandidates];
    __shared__ int list_i[kCandidates];
    const long long row = blockIdx.x;
    const int lane = lane_id(), size = 4 + 2 * d.top;
    const float* from = (const float*)d.workspace + row * parts * size;
    for (int i = threadIdx.x; i < parts * size; i += 256) all[i] = from[i];
    __syncthreads();
    if (threadIdx.x >= 64) return;
    long long outer, inner;
    const T* x = row_of<T>(d, row, outer, inner);
    const float k = kLog2e / d.temperature;
    Soft a = { kLowest, 0.0f, 0.0f };
    if (lane < parts) a = { all[lane * size], all[lane * size + 1], all[lane * size + 2] };
    a = join_lanes(a, k);
    Best best = { -NTC_INF, kNoIndex };
    Candidates list = { list_v, list_i };
    if (d.top) best = merge(list, all + 4, (const int*)all + 4 + d.top, size, parts, d.top);
    finish(d, row, x, token_of(d, outer, inner), a, best);
}

// ---------------------------------------------------------------- gradient
// dx_v = -p_v (a + g_H (log p_v + H)) / T, with a the sum of all g_logprob, and more at the token and the alternatives. One read and one write of the
// row, from its stats: memory bounds it (bf16 8190 x 50001: 345 us, 4.75 TB/s). A wave takes two vectors a lane of one row. The few places that get
// more are held one a lane and looked for a chunk at a time.
constexpr int kGradVecs = 2;
template <class T> __global__ void __launch_bounds__(256) k_logprobs_grad(ntc_logprobs_desc d, int row_chunks) {
    constexpr int kVec = 16 / (int)sizeof(T), kChunk = 64 * kVec;
    const int lane = lane_id();
    const long long unit = block_number() * 4 + (threadIdx.x >> 6), row = unit / row_chunks;
    if (row >= d.rows) return;
    const int V = (int)d.V, begin = (int)(unit % row_chunks) * (kGradVecs * kChunk);
    long long outer, inner;
    const T* x = row_of<T>(d, row, outer, inner);
    T* dx = (T*)d.dlogits + row * d.V;
    const float k = kLog2e / d.temperature, inv_t = 1.0f / d.temperature;
    const float m = d.stats[2 * row], log_s = d.stats[2 * row + 1], H = d.entropy[row];
    const long long t = token_of(d, outer, inner);
    const bool none = m == -NTC_INF, out = t != d.ignore_index && (t < 0 || t >= d.V);
    const float glp = d.g_logprob && t != d.ignore_index ? d.g_logprob[row] : 0.0f;
    const float gh = d.g_entropy ? d.g_entropy[row] : 0.0f;
    const bool tops = d.g_top != nullptr;
    // lane 0: the token; lanes 1 to top: the alternatives
    int place = -1;
    float extra = 0.0f;
    if (lane == 0 && !out && t != d.ignore_index) { place = (int)t; extra = glp; }
    if (tops && lane >= 1 && lane <= d.top) { place = (int)d.top_ids[row * d.top + lane - 1]; extra = d.g_top[row * d.top + lane - 1]; }
    float all = reduce64(extra, [](float p, float q) { return p + q; });
    if (out) all = __builtin_nanf("");
    // a token that is an alternative too gets both at once: they may nearly cancel
    const bool twice = lane && place >= 0 && place == t;
    const bool moved = __ballot(twice) != 0;
    if (twice) extra += glp;
    if (lane == 0 && moved) place = -1;
    extra *= inv_t;
    const float na = -all * inv_t * 0x1p-24f, nh = -gh * inv_t * 0x1p-24f;
#pragma unroll
    for (int c = 0; c < kGradVecs; c++) {
        const int base = begin + c * kChunk, at = base + lane * kVec;
        if (base >= V) break;
        T r[kVec];
        const bool full = at + kVec <= V;
        if (full) { const auto q = *(const LooseRun<T, kVec>*)(x + at); for (int j = 0; j < kVec; j++) r[j] = q.v[j]; }
        else { const auto q = __builtin_bit_cast(LooseRun<T, kVec>, at < V ? last_run(x, V, at, V - at) : (Bits)0); for (int j = 0; j < kVec; j++) r[j] = q.v[j]; }
        float g[kVec];
#pragma unroll
        for (int j = 0; j < kVec; j++) {
            // (the exponential's instruction gives 0 for what is below 2^-126: probabilities are taken times 2^24)
            const float lp = ((float)r[j] - m) * k - log_s, p = fast_exp2(lp + 24.0f);
            g[j] = p * __builtin_fmaf(nh, __builtin_fmaf(kLn2, fmaxf(lp, -160.0f), H), na);
        }
        unsigned long long here = __ballot(place >= base && place < base + kChunk);
        while (here) {
            const int l = __builtin_ctzll(here);
            here &= here - 1;
            const int off = __builtin_amdgcn_readlane(place, l) - at;
            const float e = read_lane(extra, l);
#pragma unroll
            for (int j = 0; j < kVec; j++) g[j] += off == j ? e : 0.0f;
        }
        LooseRun<T, kVec> o;
#pragma unroll
        for (int j = 0; j < kVec; j++) o.v[j] = (T)(none ? 0.0f : g[j]);
        if (full) *(LooseRun<T, kVec>*)(dx + at) = o;
        else if (at < V) store_last(dx + at, __builtin_bit_cast(Bits, o), V - at);
    }
}

// Short rows: a group of kGroup lanes holds a row, 16 values a lane, as forward. The places that get more are a lane's each, and are added
// where the group has laid its gradients in LDS (bf16 400000 x 256: 93 us, 4.4 TB/s; a wave to a row as below 254).
template <class T, int kGroup> __global__ void __launch_bounds__(256) k_logprobs_grad_short(ntc_logprobs_desc d, float k, float inv_t) {
    constexpr int kEach = 16, kVec = 16 / (int)sizeof(T), kRows = 256 / kGroup;
    __shared__ float4 laid[kEach / 4][256];
    const int in = threadIdx.x % kGroup, own = threadIdx.x / kGroup;
    const long long first = block_number() * kRows;
    if (first >= d.rows) return;
    const long long row = first + own < d.rows ? first + own : d.rows - 1;   // past the end the last row again, not written
    const int V = (int)d.V, at = in * kEach;
    long long outer, inner;
    const T* x = row_of<T>(d, row, outer, inner);
    LooseRun<T, kVec> r[kEach / kVec];
#pragma unroll
    for (int i = 0; i < kEach / kVec; i++) {
        const int left = V - at - i * kVec;
        r[i] = {};
        if (left >= kVec) r[i] = *(const LooseRun<T, kVec>*)(x + at + i * kVec);
        else if (left > 0) r[i] = __builtin_bit_cast(LooseRun<T, kVec>, last_run(x, V, at + i * kVec, left));
    }
    const float m = d.stats[2 * row], log_s = d.stats[2 * row + 1], H = d.entropy[row];
    const long long t = token_of(d, outer, inner);
    const bool none = m == -NTC_INF, ignored = t == d.ignore_index, out = !ignored && (t < 0 || t >= d.V);
    const float glp = d.g_logprob && !ignored ? d.g_logprob[row] : 0.0f;
    const float gh = d.g_entropy ? d.g_entropy[row] : 0.0f;
    const int tops = d.g_top ? d.top : 0;
    float all = 0.0f;
    for (int e = in; e < tops; e += kGroup) all += d.g_top[row * d.top + e];
    all = reduce<kGroup>(all, [](float p, float q) { return p + q; }) + glp;
    if (out) all = __builtin_nanf("");
    const float na = -all * inv_t * 0x1p-24f, nh = -gh * inv_t * 0x1p-24f;
    float g[kEach];
#pragma unroll
    for (int j = 0; j < kEach; j++) {
        const float lp = ((float)r[j / kVec].v[j % kVec] - m) * k - log_s, p = fast_exp2(lp + 24.0f);   // (times 2^24, as below)
        g[j] = p * __builtin_fmaf(nh, __builtin_fmaf(kLn2, fmaxf(lp, -160.0f), H), na);
    }
#pragma unroll
    for (int q = 0; q < kEach / 4; q++) laid[q][threadIdx.x] = float4{ g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3] };
    wave_shared();
    const auto add = [&](int place, float extra) {
        float* to = (float*)&laid[(place % kEach) / 4][own * kGroup + place / kEach] + place % 4;
        *to += extra * inv_t;
    };
    bool joined = out || ignored;                            // the token, where it is an alternative too, is added with it: the two may nearly cancel
    for (int e0 = 0; e0 < tops; e0 += kGroup) {
        const int e = e0 + in;
        const long long id = e < tops ? d.top_ids[row * d.top + e] : -1;
        const int place = id < V ? (int)id : -1;
        const bool both = place >= 0 && place == t && !ignored;
        if (place >= 0) add(place, d.g_top[row * d.top + e] + (both ? glp : 0.0f));
        const unsigned long long found = __ballot(both) >> (lane_id() & ~(kGroup - 1));
        joined |= (kGroup == 64 ? found : found & ((1ull << (kGroup % 64)) - 1)) != 0;
    }
    if (in == 0 && !joined) add((int)t, glp);
    wave_shared();
#pragma unroll
    for (int q = 0; q < kEach / 4; q++) { const float4 o = laid[q][threadIdx.x]; g[4 * q] = o.x; g[4 * q + 1] = o.y; g[4 * q + 2] = o.z; g[4 * q + 3] = o.w; }
    if (first + own >= d.rows) return;
    T* dx = (T*)d.dlogits + row * d.V + at;
#pragma unroll
    for (int i = 0; i < kEach / kVec; i++) {
        const int left = V - at - i * kVec;
        LooseRun<T, kVec> o;
#pragma unroll
        for (int j = 0; j < kVec; j++) o.v[j] = (T)(none ? 0.0f : g[i * kVec + j]);
        if (left >= kVec) *(LooseRun<T, kVec>*)(dx + i * kVec) = o;
        else if (left > 0) store_last(dx + i * kVec, __builtin_bit_cast(Bits, o), left);
    }
}

// How long rows are read: waves a row, and blocks a row where there are few rows. A wave to a row puts alternatives in order once, not four
// times, and joins nothing, but needs rows for every SIMD and leaves them unevenly done (bf16, one wave against four: 5000 x 10000 21.0 against 28.0 us,
// with 32 alternatives 51 against 75; 16384 x 20000 129 against 149; 2500 x 30000 with 4 44.6 against 41.1; 8190 x 50001 168 against 162, with 16
// 196 against 234; float32 with 4 4096 x 30000 89 against 96, 8192 x 50000 323 against 279; 1500 x 20000 18.8 against 14.8). Blocks to a row cost a
// second launch (1 x 131072 4.9 against 16 us, with 4 9.8 against 27; 100 x 24000 with 4 10.1 against 12.3; 1 x 9000 5.1 against 4.0; 500 x 24000 9.5
// against 7.8).
struct Reading { int waves, parts, part_chunks; };
template <class T> static Reading reading(int64_t rows, int64_t V, int top) {
    const int64_t chunks = (V + Long<T>::kChunk - 1) / Long<T>::kChunk;
    const bool one = rows >= 4096 ? chunks <= 32 || (top >= 4 && (sizeof(T) == 2 || chunks <= 64)) : rows >= 2048 && chunks <= 16;
    Reading r = { one ? 1 : 4, 1, (int)chunks };
    if (r.waves == 4 && rows < 384 && chunks > 16) {
        int64_t parts = 1024 / rows;
        if (parts > kMostParts) parts = kMostParts;
        if (parts > chunks / 4) parts = chunks / 4;
        r.part_chunks = (int)((chunks + parts - 1) / parts);
        r.parts = (int)((chunks + r.part_chunks - 1) / r.part_chunks);
    }
    return r;
}

template <class T> static void forward(const ntc_logprobs_desc& d, hipStream_t s) {
    const auto blocks = [&](int per) { return grid_of((d.rows + per - 1) / per); };
    const float k = kLog2e / d.temperature, lim = 1e30f / (k > 1.0f ? k : 1.0f);   // values up to lim times k stay far from overflow
    const float most = k >= 0x1p-60f ? 0x1p24f : -1.0f;
    uint32_t bits;
    memcpy(&bits, &lim, 4);
    const int low = type_code<T> == NTC_BF16 ? (int)(bits >> 16) : lim > 65504.0f ? 0x7c00 : 0;   // lim as such a type's bits (float16: its infinity's, or every row is looked at)
    // Up to 512 values, and 1024 of 16 bits, a row is held in registers, in the fewest lanes of 16 values (against reading it as a long one: bf16
    // 200000 x 256 23 against 96 us, 50000 x 1000 with 4 alternatives 38 against 46; float32 100000 x 512 31 against 40, but 50000 x 1000 54 against 37).
    // Short rows of many alternatives sort each lane's values first, where that beats finding its three best again and again (bf16, with 32: 400000 x 64
    // 55 us against 79, 50000 x 1024 77 against 83; with 8 29 against 31 and 46 against 40; float32 with 16: 400000 x 64 60 against 80,
    // 100000 x 512 89 against 78).
    const auto shorts = [&](auto group) {
        constexpr int g = group.value;
        const dim3 grid = blocks(256 / g);
        constexpr int from = sizeof(T) == 4 ? (g > 12 ? g : 12) : g > 16 ? g / 2 : 8;
        if constexpr (from <= NTC_MAX_TOP)
            if (d.top >= from) { k_logprobs_short<T, g, true><<<grid, 256, 0, s>>>(d, lim, low, most, k, 1.0f / d.temperature); return; }
        k_logprobs_short<T, g, false><<<grid, 256, 0, s>>>(d, lim, low, most, k, 1.0f / d.temperature);
    };
    if (d.V <= 64) return shorts(std::integral_constant<int, 4>());
    if (d.V <= 128) return shorts(std::integral_constant<int, 8>());
    if (d.V <= 256) return shorts(std::integral_constant<int, 16>());
    if (d.V <= 512) return shorts(std::integral_constant<int, 32>());
    if constexpr (sizeof(T) == 2)
        if (d.V <= kShort) return shorts(std::integral_constant<int, 64>());
    const Reading r = reading<T>(d.rows, d.V, d.top);
    if (r.waves == 1) k_logprobs_long<T, 1, false><<<blocks(4), 256, 0, s>>>(d, lim, 0);
    else if (r.parts == 1) k_logprobs_long<T, 4, false><<<blocks(1), 256, 0, s>>>(d, lim, 0);
    else {
        k_logprobs_long<T, 4, true><<<dim3((unsigned)d.rows, r.parts), 256, 0, s>>>(d, lim, r.part_chunks);
        k_logprobs_join<T><<<(unsigned)d.rows, 256, 0, s>>>(d, r.parts);
    }
}
template <class T> static size_t workspace(int64_t rows, int64_t V, int top) {
    const Reading r = reading<T>(rows, V, top);
    return r.parts == 1 ? 0 : (size_t)rows * r.parts * (4 + 2 * top) * 4;
}
template <class T> static void backward(const ntc_logprobs_desc& d, hipStream_t s) {
    constexpr int kVec = 16 / (int)sizeof(T);
    const auto shorts = [&](auto group) {
        constexpr int g = group.value;
        k_logprobs_grad_short<T, g><<<grid_of((d.rows + 256 / g - 1) / (256 / g)), 256, 0, s>>>(d, kLog2e / d.temperature, 1.0f / d.temperature);
    };
    if (d.V <= 64) return shorts(std::integral_constant<int, 4>());
    if (d.V <= 128) return shorts(std::integral_constant<int, 8>());
    if (d.V <= 256) return shorts(std::integral_constant<int, 16>());
    if (d.V <= 512) return shorts(std::integral_constant<int, 32>());
    if (d.V <= kShort) return shorts(std::integral_constant<int, 64>());
    const int64_t row_chunks = (d.V + 64 * kVec * kGradVecs - 1) / (64 * kVec * kGradVecs);
    k_logprobs_grad<T><<<grid_of((d.rows * row_chunks + 3) / 4), 256, 0, s>>>(d, (int)row_chunks);
}

static int check(const ntc_logprobs_desc* d, bool backward, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->rows < 0 || d->V < 1 || d->inner_rows < 1) return refuse(why, cap, "rows >= 0, inner_rows >= 1 and V >= 1 are needed");
    if (d->V > 0x7fff0000 || d->rows > 0x7fffffff) return refuse(why, cap, "fewer than 2^31 rows, and at most 2^31 - 2^16 values of a row");
    if (d->dtype < 0 || d->dtype > 2) return refuse(why, cap, "logits are 32-bit floats, bfloat16 or float16");
    if (d->token_bytes != 4 && d->token_bytes != 8) return refuse(why, cap, "tokens are 32- or 64-bit integers");
    if (d->top < 0 || d->top > NTC_MAX_TOP || d->top > d->V) return refuse(why, cap, "top is 0 to 32 and at most V");
    // (below, 1 / T is infinite; above, differences of logits that overflow would still have an exponential)
    if (!(d->temperature >= 0x1p-127f && d->temperature <= 0x1p120f)) return refuse(why, cap, "temperature is from 2^-127 to 2^120");
    if (d->rows == 0) return 0;
    if (!d->logits || !d->tokens || !d->stats || !d->entropy) return refuse(why, cap, "a null pointer");
    if (!backward && (!d->logprob || (d->top && (!d->top_ids || !d->top_logprobs)))) return refuse(why, cap, "a null pointer");
    if (backward && (!d->dlogits || (d->g_top && !d->top_ids))) return refuse(why, cap, "a null pointer");
    return 0;
}

}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" size_t ntc_op_token_logprobs_workspace(int64_t rows, int64_t V, int32_t dtype, int32_t top) {
    if (rows < 1 || V < 1 || top < 0 || top > NTC_MAX_TOP) return 0;
    return dtype == NTC_F32 ? workspace<f32>(rows, V, top) : workspace<bf16>(rows, V, top);
}

extern "C" int ntc_op_token_logprobs(const ntc_logprobs_desc* d, void* stream, char* why, size_t cap) {
    if (const int r = check(d, false, why, cap)) return r;
    if (!d->rows) return 0;
    if (!d->workspace && ntc_op_token_logprobs_workspace(d->rows, d->V, d->dtype, d->top)) return refuse(why, cap, "a null workspace");
    const hipStream_t s = (hipStream_t)stream;
    d->dtype == NTC_F32 ? forward<f32>(*d, s) : d->dtype == NTC_BF16 ? forward<bf16>(*d, s) : forward<f16>(*d, s);
    return launched(why, cap);
}

extern "C" int ntc_op_token_logprobs_backward(const ntc_logprobs_desc* d, void* stream, char* why, size_t cap) {
    if (const int r = check(d, true, why, cap)) return r;
    if (!d->rows) return 0;
    const hipStream_t s = (hipStream_t)stream;
    d->dtype == NTC_F32 ? backward<f32>(*d, s) : d->dtype == NTC_BF16 ? backward<bf16>(*d, s) : backward<f16>(*d, s);
    return launched(why, cap);
}
