// Layer norm and its gradients (include/ntc_ops.h: ntc_op_layer_norm).
//
// With mu and s the mean and 1 / sqrt(variance + eps) of a row, h = (x - mu) s and y = h w + b; backwards, with t = g w,
//   dx = s (t - mean t - h mean(t h)),   dw = sum over rows of g h,   db = sum over rows of g.
// A row is read once and kept in registers: 8 to 64 lanes of a wave, or two to sixteen waves to a row, 8 or 16 values a lane, the next row on its way meanwhile. The variance is
// taken on differences from the mean, in a second pass over the registers. Backwards a block walks through many rows and adds up its
// columns' dw and db on the way; a second, small launch adds the blocks' sums, in order, so that results repeat bit for bit.
//
// Bound by memory: forward reads and writes a row once, backward reads two rows and writes one. 16384 rows of 8192 bfloat16: 105 us forward (5.1 TB/s), 157 and 5 for the sums
// backward (5.1 TB/s); 65536 rows of 256: 15, and 20 and 4; a call of one row: 4.6, the launch.
#include "ops_common.hpp"

namespace ntc_ops {
namespace {

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y, *dx;
    float* stats;             // [rows][2]: mean, 1 / sqrt(variance + eps)
    float* parts;             // [blocks][2][C]: sums of a block's rows, of dw and of db
    long long rows, x_stride, dy_stride;
    int C, w_f32;             // w_f32: weight and bias are 32-bit
    float eps;
};

// 16 bytes of a row, as they lie
struct Words { uint32_t w[4]; };
template <class T> constexpr int kRunOf = 16 / (int)sizeof(T);
template <class T> __device__ __forceinline__ float value(const Words& x, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(x.w[i]);
    else if constexpr (std::is_same_v<T, bf16>) return __uint_as_float(i & 1 ? x.w[i / 2] & 0xffff0000u : x.w[i / 2] << 16);
    else return (float)__builtin_bit_cast(T, (uint16_t)(x.w[i / 2] >> 16 * (i & 1)));
}
// The values from p on, of which n are the row's. `past`: what follows the row may be read as well (another row does); values past n are any then, else 0.
template <class T> __device__ __forceinline__ Words load_run(const T* p, int n, bool past) {
    constexpr int kN = kRunOf<T>;
    if (n >= kN || (past && n > 0)) return __builtin_bit_cast(Words, *(const LooseRun<T, kN>*)p);
    Words r = {};
#pragma unroll
    for (int i = 0; i < kN; i++)
        if (i < n) {
            if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(p[i]);
            else r.w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << 16 * (i & 1);
        }
    return r;
}
// kN values of a weight's type W (32-bit ones in two runs where the row's are 16-bit)
template <class W, int kN> __device__ __forceinline__ void load_values(const W* p, int n, float* v) {
#pragma unroll
    for (int k = 0; k < kN; k += kRunOf<W>) {
        const Words r = load_run<W>(p + k, n - k, false);
#pragma unroll
        for (int i = 0; i < kRunOf<W>; i++) v[k + i] = value<W>(r, i);
    }
}
// (weights and biases: null stands for `none`)
template <class T, int kN> __device__ __forceinline__ void load_weights(const void* w, int f32_, int c, int C, float none, float* v) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < kN; i++) v[i] = none;
    } else if (f32_) load_values<float, kN>((const float*)w + c, C - c, v);
    else load_values<T, kN>((const T*)w + c, C - c, v);
}
template <class T, int kN> __device__ __forceinline__ void store_values(T* p, int n, const float* v) {
    if (n >= kN) {
        LooseRun<T, kN> r;
#pragma unroll
        for (int i = 0; i < kN; i++) r.v[i] = (T)v[i];
        *(LooseRun<T, kN>*)p = r;
    } else {
#pragma unroll
        for (int i = 0; i < kN; i++) if (i < n) p[i] = (T)v[i];
    }
}

// The sum over a row's lanes: kLanes of a wave, or kWaves waves through shared memory (`at`: kWaves floats that nobody reads any more).
template <int kLanes, int kWaves> __device__ __forceinline__ float row_sum(float x, float* at) {
    x = reduce<kLanes>(x, [](float a, float b) { return a + b; });
    if constexpr (kWaves > 1) {
        if (lane_id() == 0) at[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0;
#pragma unroll
        for (int i = 0; i < kWaves; i++) x += at[i];
    }
    return x;
}

// kLanes lanes of a wave (kWaves = 1) or kWaves whole waves to a row, kValues values a lane in runs of 16 bytes.
template <class T, int kLanes, int kWaves, int kValues> struct Shape {
    static constexpr int kRun = kRunOf<T>, kRuns = kValues / kRun, kThreads = kWaves > 1 ? 64 * kWaves : 256, kGroup = kLanes * kWaves, kGroups = kThreads / kGroup;
    static __device__ __forceinline__ int column(int run) { return (run * kGroup + (int)threadIdx.x % kGroup) * kRun; }
};

template <class T, int kLanes, int kWaves, int kValues> __global__ void __launch_bounds__(kWaves > 1 ? 64 * kWaves : 256) k_norm(NormArgs d) {
    using S = Shape<T, kLanes, kWaves, kValues>;
    constexpr int kRun = S::kRun, kRuns = S::kRuns;
    __shared__ float sums[2][kWaves];
    float w[kValues], b[kValues];
#pragma unroll
    for (int r = 0; r < kRuns; r++) {
        load_weights<T, kRun>(d.w, d.w_f32, S::column(r), d.C, 1.f, w + r * kRun);
        load_weights<T, kRun>(d.b, d.w_f32, S::column(r), d.C, 0.f, b + r * kRun);
    }
    const float inv = 1.f / (float)d.C;
    const long long step = (long long)gridDim.x * S::kGroups, own = (long long)blockIdx.x * S::kGroups + threadIdx.x / S::kGroup;
    const bool apart = d.x_stride >= d.C && d.C >= kRun;          // (a run that begins in a row ends in the next at the latest)
    Words next[kRuns];                                     // of the row after this one, on its way meanwhile
    const auto load = [&](long long row) {
        const T* x = (const T*)d.x + row * d.x_stride;
#pragma unroll
        for (int r = 0; r < kRuns; r++) next[r] = load_run<T>(x + S::column(r), row < d.rows ? d.C - S::column(r) : 0, apart && row + 1 < d.rows);
    };
    load(own);
    for (long long first = (long long)blockIdx.x * S::kGroups, row = own; first < d.rows; first += step, row += step) {
        const bool live = row < d.rows;
        float v[kValues], sum = 0, square = 0;
#pragma unroll
        for (int r = 0; r < kRuns; r++)
#pragma unroll
            for (int i = 0; i < kRun; i++) {
                v[r * kRun + i] = S::column(r) + i < d.C ? value<T>(next[r], i) : 0.f;
                sum += v[r * kRun + i];
            }
        if (first + step < d.rows) load(row + step);
        const float mean = row_sum<kLanes, kWaves>(sum, sums[0]) * inv;
#pragma unroll
        for (int r = 0; r < kRuns; r++)
#pragma unroll
            for (int i = 0; i < kRun; i++) {
                float& z = v[r * kRun + i];
                z = S::column(r) + i < d.C ? z - mean : 0.f;
                square = __builtin_fmaf(z, z, square);
            }
        const float s = 1.f / __builtin_sqrtf(row_sum<kLanes, kWaves>(square, sums[1]) * inv + d.eps);
        if (live) {
            T* y = (T*)d.y + row * d.C;
#pragma unroll
            for (int r = 0; r < kRuns; r++) {
                float o[kRun];
#pragma unroll
                for (int i = 0; i < kRun; i++) o[i] = __builtin_fmaf(v[r * kRun + i] * s, w[r * kRun + i], b[r * kRun + i]);
                store_values<T, kRun>(y + S::column(r), d.C - S::column(r), o);
            }
            if (d.stats && threadIdx.x % S::kGroup == 0) *(float2*)(d.stats + 2 * row) = make_float2(mean, s);
        }
    }
}

template <class T, int kLanes, int kWaves, int kValues> __global__ void __launch_bounds__(kWaves > 1 ? 64 * kWaves : 256) k_norm_back(NormArgs d) {
    using S = Shape<T, kLanes, kWaves, kValues>;
    constexpr int kRun = S::kRun, kRuns = S::kRuns;
    __shared__ float sums[4][kWaves];
    __shared__ float joined[S::kGroups > 1 ? S::kGroups * S::kGroup * kValues : 1];
    float w[kValues], dw[kValues] = {}, db[kValues] = {};
#pragma unroll
    for (int r = 0; r < kRuns; r++) load_weights<T, kRun>(d.w, d.w_f32, S::column(r), d.C, 1.f, w + r * kRun);
    const float inv = 1.f / (float)d.C;
    const long long step = (long long)gridDim.x * S::kGroups, own = (long long)blockIdx.x * S::kGroups + threadIdx.x / S::kGroup;
    const bool apart = d.x_stride >= d.C && d.dy_stride >= d.C && d.C >= kRun;
    Words next_x[kRuns], next_g[kRuns];
    float2 next_st;
    const auto load = [&](long long row) {
        const T *x = (const T*)d.x + row * d.x_stride, *dy = (const T*)d.dy + row * d.dy_stride;
#pragma unroll
        for (int r = 0; r < kRuns; r++) {
            const int n = row < d.rows ? d.C - S::column(r) : 0;
            const bool past = apart && row + 1 < d.rows;
            next_x[r] = load_run<T>(x + S::column(r), n, past);
            next_g[r] = load_run<T>(dy + S::column(r), n, past);
        }
        next_st = row < d.rows ? *(const float2*)(d.stats + 2 * row) : make_float2(0.f, 0.f);
    };
    load(own);
    int turn = 0;
    for (long long first = (long long)blockIdx.x * S::kGroups, row = own; first < d.rows; first += step, row += step, turn ^= 2) {
        const bool live = row < d.rows;
        const float2 st = next_st;
        float h[kValues], g[kValues], a = 0, c = 0;
#pragma unroll
        for (int r = 0; r < kRuns; r++)
#pragma unroll
            for (int i = 0; i < kRun; i++) {
                const int k = r * kRun + i;
                const bool in = live && S::column(r) + i < d.C;
                h[k] = in ? (value<T>(next_x[r], i) - st.x) * st.y : 0.f;
                g[k] = in ? value<T>(next_g[r], i) : 0.f;
            }
        if (first + step < d.rows) load(row + step);
#pragma unroll
        for (int k = 0; k < kValues; k++) {
            dw[k] = __builtin_fmaf(g[k], h[k], dw[k]);
            db[k] += g[k];
            g[k] *= w[k];
            a += g[k];
            c = __builtin_fmaf(g[k], h[k], c);
        }
        if (!d.dx) continue;
        a = row_sum<kLanes, kWaves>(a, sums[turn]) * inv;
        c = row_sum<kLanes, kWaves>(c, sums[turn + 1]) * inv;
        if (live) {
            T* dx = (T*)d.dx + row * d.C;
#pragma unroll
            for (int r = 0; r < kRuns; r++) {
                float o[kRun];
#pragma unroll
                for (int i = 0; i < kRun; i++) o[i] = st.y * (g[r * kRun + i] - a - h[r * kRun + i] * c);
                store_values<T, kRun>(dx + S::column(r), d.C - S::column(r), o);
            }
        }
    }
    if (!d.parts) return;
    // the block's groups' sums joined, first dw's and then db's
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* v = which ? db : dw;
        float* to = d.parts + ((long long)blockIdx.x * 2 + which) * d.C;
        if constexpr (S::kGroups > 1) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kRuns; r++)
#pragma unroll
                for (int i = 0; i < kRun; i++) joined[threadIdx.x / S::kGroup * (S::kGroup * kValues) + S::column(r) + i] = v[r * kRun + i];
            __syncthreads();
            for (int c = threadIdx.x; c < d.C; c += S::kThreads) {
                float sum = 0;
                for (int k = 0; k < S::kGroups; k++) sum += joined[k * (S::kGroup * kValues) + c];
                to[c] = sum;
            }
        } else {
#pragma unroll
            for (int r = 0; r < kRuns; r++)
#pragma unroll
                for (int i = 0; i < kRun; i++) {
                    const int c = S::column(r) + i;
                    if (c < d.C) to[c] = v[r * kRun + i];
                }
        }
    }
}

// Rows that no block holds: read three times (backward: twice, and once more for the columns' sums), the later times from the caches. 4096 rows of 12000 bfloat16 with all gradients: 190 us, where
// their bytes at a copy's rate are 99; of 20000, 342 of 165.
constexpr int kWide = 1024;
__device__ __forceinline__ float block_sum(float x, float* at) { return row_sum<64, kWide / 64>(x, at); }
template <class T, class F> __device__ __forceinline__ void for_runs(int C, F f) {       // f(first column of a run, its columns)
    for (int c = threadIdx.x * kRunOf<T>; c < C; c += kWide * kRunOf<T>) f(c, C - c);
}
template <class T> __global__ void __launch_bounds__(kWide) k_norm_wide(NormArgs d) {
    __shared__ float sums[2][kWide / 64];
    constexpr int kRun = kRunOf<T>;
    const float inv = 1.f / (float)d.C;
    for (long long row = blockIdx.x; row < d.rows; row += gridDim.x) {
        const T* x = (const T*)d.x + row * d.x_stride;
        float sum = 0, square = 0;
        for_runs<T>(d.C, [&](int c, int n) {
            const Words r = load_run<T>(x + c, n, false);
#pragma unroll
            for (int i = 0; i < kRun; i++) sum += value<T>(r, i);
        });
        const float mean = block_sum(sum, sums[0]) * inv;
        for_runs<T>(d.C, [&](int c, int n) {
            const Words r = load_run<T>(x + c, n, false);
#pragma unroll
            for (int i = 0; i < kRun; i++) { const float z = i < n ? value<T>(r, i) - mean : 0.f; square = __builtin_fmaf(z, z, square); }
        });
        const float s = 1.f / __builtin_sqrtf(block_sum(square, sums[1]) * inv + d.eps);
        for_runs<T>(d.C, [&](int c, int n) {
            const Words r = load_run<T>(x + c, n, false);
            float w[kRun], b[kRun], o[kRun];
            load_weights<T, kRun>(d.w, d.w_f32, c, d.C, 1.f, w);
            load_weights<T, kRun>(d.b, d.w_f32, c, d.C, 0.f, b);
#pragma unroll
            for (int i = 0; i < kRun; i++) o[i] = __builtin_fmaf((value<T>(r, i) - mean) * s, w[i], b[i]);
            store_values<T, kRun>((T*)d.y + row * d.C + c, n, o);
        });
        if (d.stats && threadIdx.x == 0) *(float2*)(d.stats + 2 * row) = make_float2(mean, s);
    }
}
template <class T> __global__ void __launch_bounds__(kWide) k_norm_wide_back(NormArgs d) {
    __shared__ float sums[4][kWide / 64];
    constexpr int kRun = kRunOf<T>;
    const float inv = 1.f / (float)d.C;
    int turn = 0;
    for (long long row = blockIdx.x; row < d.rows; row += gridDim.x, turn ^= 2) {
        const T *x = (const T*)d.x + row * d.x_stride, *dy = (const T*)d.dy + row * d.dy_stride;
        const float2 st = *(const float2*)(d.stats + 2 * row);
        const auto run = [&](int c, int n, float* t, float* h) {
            const Words rx = load_run<T>(x + c, n, false), rg = load_run<T>(dy + c, n, false);
            load_weights<T, kRun>(d.w, d.w_f32, c, d.C, 1.f, t);
#pragma unroll
            for (int i = 0; i < kRun; i++) {
                t[i] = i < n ? t[i] * value<T>(rg, i) : 0.f;
                h[i] = i < n ? (value<T>(rx, i) - st.x) * st.y : 0.f;
            }
        };
        float a = 0, b = 0;
        for_runs<T>(d.C, [&](int c, int n) {
            float t[kRun], h[kRun];
            run(c, n, t, h);
#pragma unroll
            for (int i = 0; i < kRun; i++) { a += t[i]; b = __builtin_fmaf(t[i], h[i], b); }
        });
        a = block_sum(a, sums[turn]) * inv;
        b = block_sum(b, sums[turn + 1]) * inv;
        for_runs<T>(d.C, [&](int c, int n) {
            float t[kRun], h[kRun];
            run(c, n, t, h);
#pragma unroll
            for (int i = 0; i < kRun; i++) t[i] = st.y * (t[i] - a - h[i] * b);
            store_values<T, kRun>((T*)d.dx + row * d.C + c, n, t);
        });
    }
}
// ... and their columns' sums: 256 columns and a run of rows to a block.
template <class T> __global__ void __launch_bounds__(256) k_norm_wide_columns(NormArgs d) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= d.C) return;
    float dw = 0, db = 0;
    for (long long row = blockIdx.y; row < d.rows; row += gridDim.y) {
        const float2 st = *(const float2*)(d.stats + 2 * row);
        const float g = (float)((const T*)d.dy)[row * d.dy_stride + c];
        dw = __builtin_fmaf(g, ((float)((const T*)d.x)[row * d.x_stride + c] - st.x) * st.y, dw);
        db += g;
    }
    d.parts[(blockIdx.y * 2ll) * d.C + c] = dw;
    d.parts[(blockIdx.y * 2ll + 1) * d.C + c] = db;
}

// dw and db from the blocks' sums: 32 columns to a block, 32 threads to a column.
template <class W> __global__ void __launch_bounds__(1024) k_norm_join(const float* parts, int blocks, int C, W* dw, W* db) {
    __shared__ float part[32][33];
    const unsigned c = (unsigned)block_number() * 32 + (threadIdx.x & 31), all = 2u * C, k = threadIdx.x >> 5;
    float sum = 0;
    if (c < all)
#pragma unroll 8
        for (int p = (int)k; p < blocks; p += 32) sum += parts[(long long)p * 2 * C + c];
    part[k][threadIdx.x & 31] = sum;
    __syncthreads();
    if (k || c >= all) return;
    sum = 0;
    for (int i = 0; i < 32; i++) sum += part[i][threadIdx.x];
    W* to = c < (unsigned)C ? dw : db;
    if (to) to[c < (unsigned)C ? c : c - C] = (W)sum;
}

// ---------------------------------------------------------------- launches
// A row's lanes and values: as few lanes as hold it in 8 values each, up to a wave, then more values, then more waves. (Lanes beyond a row's end
// are idle, and a value more a lane is cheaper than a step more in the sums.)
struct Plan { int lanes, waves, values; };
Plan plan_of(int64_t C) {
    if (C <= 64) return { 8, 1, 8 };
    if (C <= 128) return { 16, 1, 8 };
    if (C <= 256) return { 32, 1, 8 };
    if (C <= 512) return { 64, 1, 8 };
    if (C <= 1024) return { 64, 1, 16 };
    if (C <= 2048) return { 64, 2, 16 };
    if (C <= 4096) return { 64, 4, 16 };
    if (C <= 8192) return { 64, 8, 16 };
    if (C <= 16384) return { 64, 16, 16 };
    return { 0, 0, 0 };
}
// (Backwards a lane also keeps its columns' sums: sixteen waves' registers do not hold sixteen values.)
Plan back_plan_of(int64_t C) { return C <= 8192 ? plan_of(C) : Plan{ 0, 0, 0 }; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t groups_of(const Plan& p) { return p.waves > 1 ? 1 : 256 / p.lanes; }
template <class T, class F> void with_shape(const Plan& p, F f) {
    const auto go = [&](auto l, auto w, auto v) { f(Shape<T, l.value, w.value, v.value>{}, l, w, v); };
#define NTC_SHAPE(L, W, V) if (p.lanes == L && p.waves == W && p.values == V) return go(std::integral_constant<int, L>{}, std::integral_constant<int, W>{}, std::integral_constant<int, V>{})
    NTC_SHAPE(8, 1, 8); NTC_SHAPE(16, 1, 8); NTC_SHAPE(32, 1, 8); NTC_SHAPE(64, 1, 8); NTC_SHAPE(64, 1, 16);
    NTC_SHAPE(64, 2, 16); NTC_SHAPE(64, 4, 16); NTC_SHAPE(64, 8, 16); NTC_SHAPE(64, 16, 16);
#undef NTC_SHAPE
}
template <class F> void with_type(int t, F f) {
    if (t == NTC_F32) f(f32{});
    else if (t == NTC_BF16) f(bf16{});
    else f(f16{});
}
// Blocks that walk through the rows backwards, each with sums of its own.
int64_t back_blocks(int64_t rows, int64_t C) {
    const Plan p = back_plan_of(C);
    if (!p.lanes) return rows < 64 ? rows : 64;
    const int64_t n = ceil_div(rows, groups_of(p)), most = p.waves > 4 ? 256 : p.waves > 2 ? 512 : 1024;
    return n < most ? n : most;
}

const char* wrong(const ntc_layer_norm_desc* d, bool back) {
    if (!d) return "no description";
    if (d->rows < 0 || d->C < 1 || d->C >= (int64_t)1 << 30) return "rows >= 0 and 1 <= C < 2^30 are needed";
    if (d->dtype < 0 || d->dtype > NTC_F16) return "values are float32, bfloat16 or float16";
    if (d->weight_type != NTC_F32 && d->weight_type != d->dtype) return "weight and bias are of the values' type, or float32";
    if (!(d->eps >= 0) || d->eps > 3.4e38f) return "eps must be a number from 0 on";
    if (!d->rows) return nullptr;
    if (!d->x || (!back && !d->y) || (back && (!d->dy || !d->stats))) return "null pointer";
    if (back && (d->dweight || d->dbias) && !d->workspace) return "null workspace";
    if (((uintptr_t)d->stats | (uintptr_t)d->workspace) % 8) return "stats and workspace start at a multiple of 8 bytes";
    return nullptr;
}
NormArgs args_of(const ntc_layer_norm_desc* d) {
    NormArgs a = {};
    a.x = d->x; a.w = d->weight; a.b = d->bias; a.dy = d->dy; a.y = d->y; a.dx = d->dx;
    a.stats = d->stats;
    a.rows = d->rows; a.x_stride = d->x_stride; a.dy_stride = d->dy_stride;
    a.C = (int)d->C; a.w_f32 = d->weight_type == NTC_F32;
    a.eps = d->eps;
    return a;
}

}  // namespace
}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" {

int ntc_op_layer_norm(const ntc_layer_norm_desc* d, void* stream, char* why, size_t cap) {
    if (const char* w = wrong(d, false)) return refuse(why, cap, w);
    if (!d->rows) return 0;
    const NormArgs a = args_of(d);
    const Plan p = plan_of(d->C);
    const hipStream_t s = (hipStream_t)stream;
    with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t n = p.lanes ? ceil_div(a.rows, groups_of(p)) : a.rows;
        // 12 blocks (of 8 and 16 waves: 4) for each of 256 compute units at most, each with as many rows. Half and twice as many are within 5% (65536 rows of 256: 13 us with any; 16384 of 8192: 108,
        // 108, 110), but for 16 waves: 3000 rows of 16000 take 44, 50 and 55 us with 2, 4 and 8.
        const unsigned grid = (unsigned)ceil_div(n, ceil_div(n, 256 * (p.waves > 4 ? 4 : 12)));
        if (!p.lanes) k_norm_wide<T><<<grid, kWide, 0, s>>>(a);
        else with_shape<T>(p, [&](auto shape, auto l, auto w, auto v) { k_norm<T, l.value, w.value, v.value><<<grid, decltype(shape)::kThreads, 0, s>>>(a); });
    });
    return launched(why, cap);
}

size_t ntc_op_layer_norm_workspace(int64_t rows, int64_t C) { return rows < 1 || C < 1 ? 0 : (size_t)back_blocks(rows, C) * 2 * C * sizeof(float); }

int ntc_op_layer_norm_backward(const ntc_layer_norm_desc* d, void* stream, char* why, size_t cap) {
    if (const char* w = wrong(d, true)) return refuse(why, cap, w);
    const hipStream_t s = (hipStream_t)stream;
    NormArgs a = args_of(d);
    const bool sums = d->dweight || d->dbias;
    const int64_t blocks = back_blocks(d->rows, d->C);
    if (sums) a.parts = (float*)d->workspace;
    if (d->rows && (sums || d->dx)) {
        const Plan p = back_plan_of(d->C);
        with_type(d->dtype, [&](auto t) {
            using T = decltype(t);
            if (p.lanes) {
                with_shape<T>(p, [&](auto shape, auto l, auto w, auto v) {
                    if constexpr (w.value < 16) k_norm_back<T, l.value, w.value, v.value><<<(unsigned)blocks, decltype(shape)::kThreads, 0, s>>>(a);
                });
            } else {
                if (a.dx) k_norm_wide_back<T><<<(unsigned)(a.rows < 4096 ? a.rows : 4096), kWide, 0, s>>>(a);
                if (sums) k_norm_wide_columns<T><<<dim3((unsigned)((a.C + 255) / 256), (unsigned)blocks), 256, 0, s>>>(a);
            }
        });
        if (const int rc = launched(why, cap)) return rc;
    }
    if (!sums) return 0;
    with_type(d->weight_type, [&](auto t) {
        using W = decltype(t);
        k_norm_join<W><<<grid_of((2 * d->C + 31) / 32, 1024), 1024, 0, s>>>(a.parts, (int)(d->rows ? blocks : 0), a.C, (W*)d->dweight, (W*)d->dbias);
    });
    return launched(why, cap);
}

}  // extern "C"
