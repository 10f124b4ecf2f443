// Matrices in 8-bit floating point with a power-of-two scale for each block of 128, and their products (include/ntc_ops.h).
#include <type_traits>

#include "ops_common.hpp"

namespace ntc_ops {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float power_of(int b) { return __uint_as_float(b > 0 ? (uint32_t)b << 23 : 1u << 22); }   // 2^(b - 127), b from 0 to 254
// The exponent byte of a block whose largest finite magnitude has these bits: amax <= 448 * 2^(E - 127).
__device__ __forceinline__ int exp_byte(uint32_t most) {
    const int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 0 ? 0 : e;
}
// Four values to codes of a block whose scale is 2^(byte - 127); the instruction divides by the power itself.
template <class T> __device__ __forceinline__ uint32_t to_codes4(T a, T b, T c, T d, float scale) {
    typedef short s2 __attribute__((ext_vector_type(2)));
    s2 r = { 0, 0 };
    if constexpr (std::is_same_v<T, bf16>) {
        typedef __bf16 two __attribute__((ext_vector_type(2)));
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, two{ a, b }, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, two{ c, d }, scale, true);
    } else if constexpr (std::is_same_v<T, f16>) {
        typedef _Float16 two __attribute__((ext_vector_type(2)));
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, two{ a, b }, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, two{ c, d }, scale, true);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
    }
    return __builtin_bit_cast(uint32_t, r);
}

// Largest magnitudes of finite values, as integers that order like them: 16-bit types two to a word, so that one instruction
// takes two; of_max() gives the bits of the 32-bit float.
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <class T> struct Magnitude {                       // bf16 and f16
    static constexpr uint32_t kInf = type_code<T> == NTC_BF16 ? 0x7f80u : 0x7c00u;
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max_pair(a, b); }
    // of eight values; non-finite ones count as 0 (seldom there: looked for once all eight are joined)
    static __device__ __forceinline__ uint32_t of(const Run<T, 8>& x) {
        const uint4 w = __builtin_bit_cast(uint4, x);
        const uint32_t v[4] = { w.x & 0x7fff7fffu, w.y & 0x7fff7fffu, w.z & 0x7fff7fffu, w.w & 0x7fff7fffu };
        uint32_t m = max_pair(max_pair(v[0], v[1]), max_pair(v[2], v[3]));
        if (__builtin_expect(__ballot(max_word(m & 0xffffu, m >> 16) >= kInf) != 0, 0)) {   // (a branch of the whole wave: else it would be computed always)
            m = 0;
            for (int i = 0; i < 4; i++) m = max_pair(m, ((v[i] & 0xffffu) >= kInf ? 0u : v[i] & 0xffffu) | (v[i] >> 16 >= kInf ? 0u : v[i] & 0xffff0000u));
        }
        return m;
    }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t m) {
        const uint16_t h = (uint16_t)max_word(m & 0xffffu, m >> 16);
        return __float_as_uint((float)__builtin_bit_cast(T, h));
    }
    // of eight rows of eight values, two to a word; non-finite ones as 0
    static constexpr int kWords = 4;
    static __device__ __forceinline__ void all(const Run<T, 8> (&x)[8], uint32_t (&m)[8][kWords]) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint4 v = __builtin_bit_cast(uint4, x[i]);
            m[i][0] = v.x & 0x7fff7fffu; m[i][1] = v.y & 0x7fff7fffu; m[i][2] = v.z & 0x7fff7fffu; m[i][3] = v.w & 0x7fff7fffu;
#pragma unroll
            for (int q = 0; q < 4; q++) any = max_pair(any, m[i][q]);
        }
        if (__builtin_expect(__ballot(max_word(any & 0xffffu, any >> 16) >= kInf) != 0, 0)) {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) m[i][q] = ((m[i][q] & 0xffffu) >= kInf ? 0u : m[i][q] & 0xffffu) | (m[i][q] >> 16 >= kInf ? 0u : m[i][q] & 0xffff0000u);
        }
    }
    // the float bits of each row's largest over 16 lanes, two rows to a word on the way
    static __device__ __forceinline__ void rows(const uint32_t (&m)[8][kWords], uint32_t (&bits)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint32_t a = max_pair(max_pair(m[i][0], m[i][1]), max_pair(m[i][2], m[i][3])), b = max_pair(max_pair(m[i + 1][0], m[i + 1][1]), max_pair(m[i + 1][2], m[i + 1][3]));
            const uint32_t both = reduce16(max_pair(__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(b, a, 0x07060302u)), max_pair);
            bits[i] = float_bits(both & 0xffffu);
            bits[i + 1] = float_bits(both >> 16);
        }
    }
    static __device__ __forceinline__ uint32_t column_bits(const uint32_t (&m)[kWords], int j) { return float_bits(j & 1 ? m[j >> 1] >> 16 : m[j >> 1] & 0xffffu); }
};
template <> struct Magnitude<f32> {
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max_word(a, b); }
    static __device__ __forceinline__ uint32_t one(float x) {
        const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
        return a < 0x7f800000u ? a : 0u;
    }
    static __device__ __forceinline__ uint32_t of(const Run<float, 8>& x) {
        uint32_t m = 0;
        for (int j = 0; j < 8; j++) m = max_word(m, one(x.v[j]));
        return m;
    }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t m) { return m; }
    static constexpr int kWords = 8;
    static __device__ __forceinline__ void all(const Run<float, 8> (&x)[8], uint32_t (&m)[8][kWords]) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) m[i][j] = one(x[i].v[j]);
    }
    static __device__ __forceinline__ void rows(const uint32_t (&m)[8][kWords], uint32_t (&bits)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t a = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) a = max_word(a, m[i][j]);
            bits[i] = reduce16(a, max_word);
        }
    }
    static __device__ __forceinline__ uint32_t column_bits(const uint32_t (&m)[kWords], int j) { return m[j]; }
};

// ---------------------------------------------------------------- to 8 bits
// A block of 256 threads takes a 128 x 128 tile: thread t holds 8 columns (8 (t % 16) ..) of the 8 rows 8 (t / 16) .., so that a
// row's largest is a reduction over 16 lanes, and a column's codes of 8 rows are one 8-byte word of the transposed tile. x is
// read once for both orders. Bound by memory where it is large (bf16 8192 x 8192, 1 x 128 blocks: 34.6 us, 5.8 TB/s; both orders 51), by the tile's own
// latency where it is not (128 x 128, both orders: 4.6 us; 4096 x 4096 15.8 us, 4.2 TB/s: loads, largest values, codes and stores of all tiles
// go in step).
template <class T> struct QuantizeSpace {
    alignas(16) uint32_t most[4][16 * Magnitude<T>::kWords];
    alignas(16) uint8_t tile[128 * 128];                   // transposed; word w of 8 rows of column c at w ^ (c / 8)
};
template <class T, bool kBlock> __device__ __forceinline__ void quantize_tile(const ntc_fp8_quantize_desc& d, long long tile_r, long long tile_c, QuantizeSpace<T>& space) {
    using Mag = Magnitude<T>;
    auto& most = space.most;
    auto& tile = space.tile;
    const long long r0 = tile_r * 128, c0 = tile_c * 128;
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    const int rows = d.R - r0 < 128 ? (int)(d.R - r0) : 128, cols = d.K - c0 < 128 ? (int)(d.K - c0) : 128;   // of this tile
    const T* from = (const T*)d.x + (r0 + 8 * rg) * d.row_stride + c0 + 8 * cg;
    Run<T, 8> x[8];
    if (rows == 128 && cols == 128) {
#pragma unroll
        for (int i = 0; i < 8; i++) { const auto v = *(const LooseRun<T, 8>*)(from + i * d.row_stride); for (int j = 0; j < 8; j++) x[i].v[j] = v.v[j]; }
    } else {
        // At the edges what is past them counts as 0; rows past the end read the last one instead, so that no branch is between the loads.
        const T* const tile0 = (const T*)d.x + r0 * d.row_stride + c0;
        const int left = cols - 8 * cg;                     // of this lane's eight columns
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = Run<T, 8>{};
        if (left >= 8) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const auto v = *(const LooseRun<T, 8>*)(tile0 + (8 * rg + i < rows ? 8 * rg + i : rows - 1) * d.row_stride + 8 * cg);
                for (int j = 0; j < 8; j++) x[i].v[j] = v.v[j];
            }
        } else if (left > 0 && sizeof(T) == 2 && d.K >= 8) {  // from the last eight of the row
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const auto v = *(const LooseRun<T, 8>*)((const T*)d.x + (r0 + (8 * rg + i < rows ? 8 * rg + i : rows - 1)) * d.row_stride + d.K - 8);
                if constexpr (sizeof(T) == 2) x[i] = __builtin_bit_cast(Run<T, 8>, __builtin_bit_cast(unsigned __int128, v) >> (16 * (8 - left)));
            }
        } else if (left > 0) {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const T v = tile0[(8 * rg + i < rows ? 8 * rg + i : rows - 1) * d.row_stride + 8 * cg + (j < left ? j : 0)];
                    x[i].v[j] = j < left ? v : (T)0.0f;
                }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) if (8 * rg + i >= rows) x[i] = Run<T, 8>{};
    }
    const long long code_stride = ntc_fp8_code_stride(d.K), exp_stride = ntc_fp8_exp_stride(d.K), code_stride_t = ntc_fp8_code_stride(d.R), exp_stride_t = ntc_fp8_exp_stride(d.R);
    // a row of exponents is written by the tile that has its block; the last one also clears what follows
    const bool last_c = c0 + 128 >= d.K, last_r = r0 + 128 >= d.R;
    const auto put_exp = [](uint8_t* row, long long at, int byte, bool last, long long stride) {
        row[at] = (uint8_t)byte;
        if (last) for (long long k = at + 1; k < stride; k++) row[k] = 0;
    };
    const auto byte_of = [](uint64_t packed, int i) { return (int)((packed >> (8 * i)) & 255); };
    uint32_t mag[8][Mag::kWords];
    Mag::all(x, mag);
    int block_byte = 0;
    if (kBlock) {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int q = 0; q < Mag::kWords; q++) b = Mag::join(b, mag[i][q]);
        b = reduce64(b, Mag::join);
        if ((threadIdx.x & 63) == 0) most[wave][0] = b;
        __syncthreads();
        b = Mag::join(Mag::join(most[0][0], most[1][0]), Mag::join(most[2][0], most[3][0]));
        block_byte = exp_byte(Mag::float_bits(b));
        if (threadIdx.x == 0) {
            if (d.codes) put_exp(d.exps + tile_r * exp_stride, tile_c, block_byte, last_c, exp_stride);
            if (d.codes_t) put_exp(d.exps_t + tile_c * exp_stride_t, tile_r, block_byte, last_r, exp_stride_t);
        }
    }
    if (d.codes) {
        uint8_t* to = d.codes + (r0 + 8 * rg) * code_stride + c0 + 8 * cg;
        uint32_t bits[8];
        uint64_t bytes = 0;
        if (!kBlock) Mag::rows(mag, bits);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int byte = kBlock ? block_byte : exp_byte(bits[i]);
            bytes |= (uint64_t)byte << (8 * i);
            const float s = power_of(byte);
            uint2 o;
            o.x = to_codes4(x[i].v[0], x[i].v[1], x[i].v[2], x[i].v[3], s);
            o.y = to_codes4(x[i].v[4], x[i].v[5], x[i].v[6], x[i].v[7], s);
            if (8 * rg + i < rows) *(uint2*)(to + i * code_stride) = o;
        }
        // lane i of the row group's 16 has row i's exponent to write
        if (!kBlock && cg < 8 && 8 * rg + cg < rows) put_exp(d.exps + (r0 + 8 * rg + cg) * exp_stride, tile_c, byte_of(bytes, cg), last_c, exp_stride);
    }
    if (!d.codes_t) return;
    uint32_t col[Mag::kWords];
    if (!kBlock) {
#pragma unroll
        for (int q = 0; q < Mag::kWords; q++) {
            col[q] = mag[0][q];
#pragma unroll
            for (int i = 1; i < 8; i++) col[q] = Mag::join(col[q], mag[i][q]);
            col[q] = reduce_rows(col[q], Mag::join);
        }
        if ((threadIdx.x & 48) == 0)
#pragma unroll
            for (int q = 0; q < Mag::kWords; q++) most[wave][Mag::kWords * cg + q] = col[q];
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int q = 0; q < Mag::kWords; q++) col[q] = Mag::join(col[q], most[w][Mag::kWords * cg + q]);
    }
    uint64_t bytes = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int byte = kBlock ? block_byte : exp_byte(Mag::column_bits(col, j));
        bytes |= (uint64_t)byte << (8 * j);
        const float s = power_of(byte);
        uint2 o;
        o.x = to_codes4(x[0].v[j], x[1].v[j], x[2].v[j], x[3].v[j], s);
        o.y = to_codes4(x[4].v[j], x[5].v[j], x[6].v[j], x[7].v[j], s);
        *(uint2*)(tile + 128 * (8 * cg + j) + 8 * (rg ^ cg)) = o;
    }
    if (!kBlock && rg < 8 && 8 * cg + rg < cols) put_exp(d.exps_t + (c0 + 8 * cg + rg) * exp_stride_t, tile_r, byte_of(bytes, rg), last_r, exp_stride_t);
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const int c = 32 * p + (threadIdx.x >> 3), part = threadIdx.x & 7, g = c >> 3;
        const uint4 v = *(const uint4*)(tile + 128 * c + 8 * ((2 * part) ^ (g & 14)));
        if (c < cols) *(uint4*)(d.codes_t + (c0 + c) * code_stride_t + r0 + 16 * part) = g & 1 ? uint4{ v.z, v.w, v.x, v.y } : v;
    }
}

constexpr int kGridRows = 1 << 15;                           // of tiles, in a grid's second dimension; more go into its third
template <class T, bool kBlock> __global__ void __launch_bounds__(256) k_fp8_quantize(ntc_fp8_quantize_desc d) {
    __shared__ QuantizeSpace<T> space;
    const long long tile_r = blockIdx.y + (long long)blockIdx.z * kGridRows;
    if (tile_r * 128 >= d.R) return;
    quantize_tile<T, kBlock>(d, tile_r, blockIdx.x, space);
}
// Two matrices, the first in blocks of 1 x 128, the second of 128 x 128 (a layer's values and its weights): a launch less.
template <class T> __global__ void __launch_bounds__(256) k_fp8_quantize_pair(ntc_fp8_quantize_desc a, ntc_fp8_quantize_desc b, uint32_t tiles_a, uint32_t across_a, uint32_t across_b) {
    __shared__ QuantizeSpace<T> space;
    const uint32_t tile = blockIdx.x;
    if (tile < tiles_a) quantize_tile<T, false>(a, tile / across_a, tile % across_a, space);
    else quantize_tile<T, true>(b, (tile - tiles_a) / across_b, (tile - tiles_a) % across_b, space);
}

// ---------------------------------------------------------------- products
// v_mfma_scale_f32_32x32x64: lane l holds 32 bytes of row l % 32 at k = 32 (l / 32) of each operand, and that row's exponent byte;
// the result's element i of lane l is (first operand's row 8 (i / 4) + 4 (l / 32) + i % 4, second's row l % 32). The first operand is B
// here, so that four of a lane's results are neighbours in C's row.
//
// A block of four waves makes a TM x TN tile of C, a quarter each. The tiles of A and B come 64 columns at a time straight
// into LDS (a stage; kStages of them in turn), stages ahead of the registers that the products are fed from, which are themselves
// one stage ahead of the products: one barrier a stage, and no product waits for a load of its own stage. In LDS a row is 64 bytes, and the 16-byte
// piece c of row r lies at c ^ swizzle(r), which spreads any 8 or 16 rows' pieces over all banks.
//
// Bound by the matrix instructions and the power they draw (8192 x 8192 x 8192: 416 us alone, 2.64 PFLOP/s, 500 to 515 for the first five in a row, 402 where hundreds follow; the instructions alone, from registers, 3.8 PFLOP/s on random
// data and 4.9 on zeros; the library's product with one scale for a matrix 3.05). 256 x 256 tiles read each operand byte from LDS half as often as 128 x
// 128 ones, and the four waves' SIMDs hold nothing else.
constexpr int kStages = 4;
__device__ __forceinline__ int swizzle(int r) { return ((r >> 1) & 3) ^ ((r >> 3) & 1); }

__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }
// 16 (4) bytes a lane from base + off to LDS at `to` + 16 (4) lane: `to` is the same in all lanes. Nothing waits for it but a vmcnt
// of the caller's; the compiler's own waits only become stricter by loads that it does not count.
__device__ __forceinline__ void to_lds16(uint32_t to, uint32_t off, const uint8_t* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(uint32_t to, uint32_t off, const uint8_t* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" :: "s"(to), "v"(off), "s"(base) : "memory", "m0");
}

// until at most n of the wave's loads are on their way
template <int n> __device__ __forceinline__ void wait_loads() {
    static_assert(n < 64, "the counter has 6 bits");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | ((n >> 4) << 14));
}

struct MatmulArgs {
    const uint8_t *a, *ae, *b, *be;
    void* c;
    long long M, N, ldc;
    int stride, estride;      // bytes of a row of codes and of exponents
    int blocks;               // of 128 columns
    int a_shift, b_shift;     // log2 of the rows of a block
    int tiles_m, tiles_n;
    int split_blocks;         // blocks of one part of the sum, a multiple of 4
};

template <int TM, int TN, class C, bool kParts> __global__ void __launch_bounds__(256, TM > 128 ? 1 : TM > 64 ? 2 : 4) k_fp8_matmul(MatmulArgs d) {
    constexpr int RM = TM / 64, RN = TN / 64;              // 32-row tiles of a wave
    constexpr int kLoads = (TM + TN) / 64;                 // 1 KiB loads a wave and stage
    constexpr int kStage = (TM + TN) * 64;
    __shared__ alignas(16) uint8_t lds[kStages * kStage + 2 * 4 * (TM + TN)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Blocks are dealt to the 8 XCDs in turn, each with an L2 of its own: every XCD takes a run of parts and tiles, which it walks in
    // columns of up to 8 rows, so that neighbours share their operands there (256 x 256 x 65536 in 64 parts without it: 15.5 us, every operand read twice).
    const int tiles = d.tiles_m * d.tiles_n, each = gridDim.x / 8, rest = gridDim.x % 8, xcd = blockIdx.x % 8;
    int tile = xcd * each + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
    const int part = kParts ? tile / tiles : 0;
    tile -= part * tiles;
    const int group = tile / (8 * d.tiles_n), first = group * 8, high = d.tiles_m - first < 8 ? d.tiles_m - first : 8;
    const int tm = first + (tile - group * 8 * d.tiles_n) % high, tn = (tile - group * 8 * d.tiles_n) / high;
    const long long m0 = (long long)tm * TM, n0 = (long long)tn * TN;
    const int rows_m = d.M - m0 < TM ? (int)(d.M - m0) : TM, rows_n = d.N - n0 < TN ? (int)(d.N - n0) : TN;   // rows past the end read the last one
    const int block0 = part * d.split_blocks;
    const int blocks = kParts && d.blocks - block0 > d.split_blocks ? d.split_blocks : d.blocks - block0;

    // what this lane loads: pieces of rows of A (the first TM / 64 loads of a wave) and of B
    const uint8_t* base_a = d.a + m0 * d.stride + block0 * 128;
    const uint8_t* base_b = d.b + n0 * d.stride + block0 * 128;
    uint32_t off[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const bool is_a = i < TM / 64;
        const int r = 16 * (4 * (is_a ? i : i - TM / 64) + wave) + (lane >> 2), rows = is_a ? rows_m : rows_n;
        off[i] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)d.stride + 16 * ((lane & 3) ^ swizzle(r));
    }
    const uint8_t* ebase_a = d.ae + (m0 >> d.a_shift) * d.estride + block0;
    const uint8_t* ebase_b = d.be + (n0 >> d.b_shift) * d.estride + block0;
    constexpr int kExpLoads = (TM + TN + 255) / 256;
    uint32_t eoff[kExpLoads];
#pragma unroll
    for (int i = 0; i < kExpLoads; i++) {                  // exponents of 64 rows: the blocks' words of A, then of B
        const int at = 64 * (4 * i + wave), r = at < TM ? at + lane : at - TM + lane, rows = at < TM ? rows_m : rows_n;
        eoff[i] = (uint32_t)((r < rows ? r : rows - 1) >> (at < TM ? d.a_shift : d.b_shift)) * (uint32_t)d.estride;
    }
    const uint32_t lds0 = lds_address(lds);
    const int stages = 2 * blocks;
    const auto load = [&](int s, int i) {                  // load i of stage s; past the end the last stage again, so that every stage has as many
        const int k = 64 * (s < stages ? s : stages - 1);
        to_lds16(lds0 + (s % kStages) * kStage + 1024 * wave + 4096 * i, off[i], (i < TM / 64 ? base_a : base_b) + k);
    };
    const auto load_exps = [&](int g) {                    // a word of four blocks' exponents for each row, two groups in turn
        const int b = 4 * g < blocks ? 4 * g : 4 * ((blocks - 1) / 4);
#pragma unroll
        for (int i = 0; i < kExpLoads; i++) {
            const int at = 64 * (4 * i + wave);
            if ((TM + TN) % 256 == 0 || at < TM + TN) to_lds4(lds0 + kStages * kStage + (g & 1) * 4 * (TM + TN) + 4 * at, eoff[i], (at < TM ? ebase_a : ebase_b) + b);
        }
    };

    const int wm = (wave >> 1) * (TM / 2), wn = (wave & 1) * (TN / 2), r32 = lane & 31, half = lane >> 5;
    v8i fa[2][RM], fb[2][RN];
    int ea[RM], eb[RN], na[RM], nb[RN];                    // exponents of this group of four blocks and of the next
    // Half an operand: the 2 (RM + RN) pieces of a stage in the order in which its products need them (A's first tile, B's, A's others).
    const auto fetch = [&](int s, int set, int p) {
        const bool is_a = p < 2 || p >= 2 * RN + 2;
        const int i = p < 2 ? 0 : is_a ? (p - 2 * RN) >> 1 : (p - 2) >> 1, r = (is_a ? wm : TM + wn) + 32 * i + r32, h = p & 1;
        const int4 x = *(const int4*)(lds + (s % kStages) * kStage + 64 * r + 16 * ((2 * half + h) ^ swizzle(r)));
        v8i& to = is_a ? fa[set][i] : fb[set][i];
        to[4 * h] = x.x; to[4 * h + 1] = x.y; to[4 * h + 2] = x.z; to[4 * h + 3] = x.w;
    };
    const auto fetch_exps = [&](int g) {
        const int* at = (const int*)(lds + kStages * kStage) + (g & 1) * (TM + TN);
#pragma unroll
        for (int i = 0; i < RM; i++) na[i] = at[wm + 32 * i + r32];
#pragma unroll
        for (int i = 0; i < RN; i++) nb[i] = at[TM + wn + 32 * i + r32];
    };
    v16f acc[RM][RN] = {};
    // The next stage's loads have landed, in every wave (all but the newest kStages - 3 stages' have); and every wave has its operands of the stage before (their products
    // have been issued), so that the buffer they came from is free.
    const auto arrive = [&] {
        __builtin_amdgcn_sched_barrier(0);
        wait_loads<(kStages - 3) * kLoads>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    // A stage: its RM RN products and, spread evenly between them, the reads of the next stage and the loads of the one kStages - 1 later. A wave has
    // its SIMD to itself and issues in order: what is not spread holds the products up. kByte: the block's byte of the exponents' words.
    const auto stage = [&](int s, auto set_, auto byte_, auto&& first, auto&& last) {
        constexpr int n = RM * RN, reads = 2 * (RM + RN), set = set_.value, kByte = byte_.value;
        arrive();
#pragma unroll
        for (int q = 0; q < n; q++) {
            const int i = q / RN, j = q % RN;
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[set][j], fa[set][i], acc[i][j], 0, 0, kByte, eb[j], kByte, ea[i]);
            if (q == 0) first();
#pragma unroll
            for (int p = q * reads / n; p < (q + 1) * reads / n; p++) fetch(s + 1, set ^ 1, p);
#pragma unroll
            for (int p = q * kLoads / n; p < (q + 1) * kLoads / n; p++) load(s + kStages - 1, p);
            if (q == n - 1) last();
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const auto none = [] {};
    const auto next_exps = [&] {
#pragma unroll
        for (int i = 0; i < RM; i++) ea[i] = na[i];
#pragma unroll
        for (int i = 0; i < RN; i++) eb[i] = nb[i];
    };

    load_exps(0);
#pragma unroll
    for (int i = 0; i < (kStages - 1) * kLoads; i++) load(i / kLoads, i % kLoads);
    wait_loads<(kStages - 2) * kLoads>();                  // the exponents and stage 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < 2 * (RM + RN); p++) fetch(0, 0, p);
    fetch_exps(0);
    using std::integral_constant;
    const integral_constant<int, 0> c0;
    const integral_constant<int, 1> c1;
    const integral_constant<int, 2> c2;
    const integral_constant<int, 3> c3;
    int b = 0;
    for (; b + 4 <= blocks; b += 4) {                      // the loads of group b / 4 + 1 have 7 stages until they are read
        next_exps();
        stage(2 * b, c0, c0, [&] { load_exps((b >> 2) + 1); }, none);
        stage(2 * b + 1, c1, c0, none, none);
        stage(2 * b + 2, c0, c1, none, none);
        stage(2 * b + 3, c1, c1, none, none);
        stage(2 * b + 4, c0, c2, none, none);
        stage(2 * b + 5, c1, c2, none, none);
        stage(2 * b + 6, c0, c3, none, none);
        stage(2 * b + 7, c1, c3, none, [&] { fetch_exps((b >> 2) + 1); });
    }
    next_exps();
    for (; b < blocks; b++) {                              // one to three blocks more
        stage(2 * b, c0, c0, none, none);
        stage(2 * b + 1, c1, c0, none, none);
#pragma unroll
        for (int i = 0; i < RM; i++) ea[i] = (unsigned)ea[i] >> 8;
#pragma unroll
        for (int i = 0; i < RN; i++) eb[i] = (unsigned)eb[i] >> 8;
    }
    wait_loads<0>();                                       // loads past the end must not land after the block has gone

    C* const quarter = (C*)d.c + (long long)part * d.M * d.N + (m0 + wm) * d.ldc + n0 + wn;
    const int left_m = rows_m - wm, left_n = rows_n - wn;
    // kGuard 0: the tile is whole; 1: its rows may end; 2: its columns too
    const auto put = [&](C* to, const auto& run, int m, int n, auto guard) {
        constexpr int R = sizeof(run) / sizeof(C);
        if (guard.value && m >= left_m) return;
        if (guard.value < 2 || n + R <= left_n) *(LooseRun<C, R>*)to = *(const LooseRun<C, R>*)&run;
        else for (int k = 0; k < R; k++) if (n + k < left_n) to[k] = run.v[k];
    };
    const auto store = [&](auto guard) {
    if constexpr (sizeof(C) == 2) {
        // Four results a lane are 8 bytes of a row: 32 rows of the wave's quarter at a time go through LDS, so that rows are stored whole.
        constexpr int kRow = TN, kPieces = kRow / 16;       // bytes of a row of the quarter, and its 16-byte pieces
        __builtin_amdgcn_s_barrier();                       // every wave has its last operands
        asm volatile("" ::: "memory");
        uint8_t* own = lds + wave * 32 * kRow;
#pragma unroll
        for (int i = 0; i < RM; i++) {
#pragma unroll
            for (int j = 0; j < RN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    Run<C, 4> o;
                    for (int k = 0; k < 4; k++) o.v[k] = (C)acc[i][j][4 * q + k];
                    *(Run<C, 4>*)(own + r32 * kRow + 16 * ((4 * j + q) ^ (r32 & (kPieces - 1))) + 8 * half) = o;
                }
            wave_shared();
#pragma unroll
            for (int p = 0; p < 32 * kPieces / 64; p++) {
                const int r = p * (64 / kPieces) + lane / kPieces, piece = lane % kPieces;
                const Run<C, 8> x = *(const Run<C, 8>*)(own + r * kRow + 16 * (piece ^ (r & (kPieces - 1))));
                put(quarter + (32 * i + r) * d.ldc + 8 * piece, x, 32 * i + r, 8 * piece, guard);
            }
            wave_shared();
        }
    } else {
#pragma unroll
        for (int i = 0; i < RM; i++)
#pragma unroll
            for (int j = 0; j < RN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int m = 32 * i + r32, n = 32 * j + 8 * q + 4 * half;
                    Run<C, 4> o;
                    for (int k = 0; k < 4; k++) o.v[k] = (C)acc[i][j][4 * q + k];
                    put(quarter + m * d.ldc + n, o, m, n, guard);
                }
    }
    };
    // (one branch for the whole tile: a guard at every store of a full one is 5% of the largest product)
    if (rows_n < TN) store(std::integral_constant<int, 2>());
    else if (rows_m < TM) store(std::integral_constant<int, 1>());
    else store(std::integral_constant<int, 0>());
}

// Few rows of A: bound by the bytes of B (one row by 4096 x 4096 5.9 us, 2.9 TB/s and mostly the launch and the first loads; by 8192 x 4096 8.1 us,
// 4.2 TB/s). A block takes 16 rows of B, its waves a share of the columns each, straight from memory into the
// operands' registers (v_mfma_scale_f32_16x16x128: lane l holds 32 bytes of row l % 16 at k = 32 (l / 16); result i is (first operand's row
// 4 (l / 16) + i, second's row l % 16)), and the waves' sums are added in LDS, in order. A's rows are kM tiles of 16 (past the end the last row
// again); floats are taken to 8 bits here, each wave what it needs, which saves a launch: a row's block is 32 values in each of 4 lanes.
struct FewArgs {
    const void* a;
    const uint8_t *ae, *b, *be;
    void* c;
    long long N, a_stride, ldc;
    int M, K, blocks, stride, estride, a_shift, b_shift;
};
template <class A> __device__ __forceinline__ v8i to_codes(const Run<A, 8> (&x)[4], int& byte) {
    using Mag = Magnitude<A>;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) m = Mag::join(m, Mag::of(x[i]));
    byte = exp_byte(reduce_rows(Mag::float_bits(m), [](uint32_t p, uint32_t q) { return p > q ? p : q; }));
    const float s = power_of(byte);
    v8i r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        r[2 * i] = (int)to_codes4(x[i].v[0], x[i].v[1], x[i].v[2], x[i].v[3], s);
        r[2 * i + 1] = (int)to_codes4(x[i].v[4], x[i].v[5], x[i].v[6], x[i].v[7], s);
    }
    return r;
}
constexpr int kFewWaves = 8;
// kM x kN tiles of 16 x 16: a wave converts (or reads) a block of A's columns once for kN tiles of B.
template <class A, int kM, int kN, class C> __global__ void __launch_bounds__(64 * kFewWaves) k_fp8_few(FewArgs d) {
    constexpr bool kFp8 = std::is_same_v<A, uint8_t>;
    constexpr int kRegs = kM * (kFp8 ? 8 : 8 * (int)sizeof(A)) + kN * 8;                       // registers of a block of columns in flight
    constexpr int kAhead = kRegs > 64 ? 1 : kRegs > 32 ? 2 : 4;
    __shared__ float sums[kFewWaves][kM * kN][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const long long n0 = block_number() * (16 * kN);
    const uint8_t *b[kN], *be[kN];
#pragma unroll
    for (int i = 0; i < kN; i++) {
        const long long n = n0 + 16 * i + r < d.N ? n0 + 16 * i + r : d.N - 1;
        b[i] = d.b + n * d.stride + 32 * g;
        be[i] = d.be + (n >> d.b_shift) * d.estride;
    }
    const A* a[kM];
    const uint8_t* ae[kM];
#pragma unroll
    for (int i = 0; i < kM; i++) {
        const int m = 16 * i + r < d.M ? 16 * i + r : d.M - 1;
        a[i] = (const A*)d.a + (long long)m * (kFp8 ? d.stride : d.a_stride) + 32 * g;
        ae[i] = kFp8 ? d.ae + (long long)(m >> d.a_shift) * d.estride : nullptr;
    }
    const auto codes = [](const uint8_t* p) {
        const uint4 x = *(const uint4*)p, y = *(const uint4*)(p + 16);
        return v8i{ (int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w };
    };
    v4f acc[kM][kN] = {};
    for (int k0 = wave; k0 < d.blocks; k0 += kFewWaves * kAhead) {
        v8i w[kAhead][kN];
        int we[kAhead][kN];
        std::conditional_t<kFp8, v8i, Run<A, 8>[4]> x[kAhead][kM];
        int xe[kAhead][kM];
        // A's first, so that they are converted while B's are on the way
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int k = k0 + kFewWaves * u;
            if (k >= d.blocks) break;
#pragma unroll
            for (int i = 0; i < kM; i++) {
                if constexpr (kFp8) {
                    x[u][i] = codes(a[i] + 128ll * k);
                    xe[u][i] = ae[i][k];
                } else {
                    const int left = d.K - 128 * k - 32 * g;   // values of this lane's 32 that are there
                    const A* from = a[i] + 128ll * k;
                    if (128 * k + 128 <= d.K) {
#pragma unroll
                        for (int j = 0; j < 4; j++) { const auto v = *(const LooseRun<A, 8>*)(from + 8 * j); for (int e = 0; e < 8; e++) x[u][i][j].v[e] = v.v[e]; }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) for (int e = 0; e < 8; e++) x[u][i][j].v[e] = 8 * j + e < left ? from[8 * j + e] : (A)0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int k = k0 + kFewWaves * u;
            if (k >= d.blocks) break;
#pragma unroll
            for (int i = 0; i < kN; i++) {
                w[u][i] = codes(b[i] + 128ll * k);
                we[u][i] = be[i][k];
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (k0 + kFewWaves * u >= d.blocks) break;
#pragma unroll
            for (int i = 0; i < kM; i++) {
                v8i code;
                if constexpr (kFp8) code = x[u][i];
                else code = to_codes<A>(x[u][i], xe[u][i]);
#pragma unroll
                for (int j = 0; j < kN; j++) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[u][j], code, acc[i][j], 0, 0, 0, we[u][j], 0, xe[u][i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kM; i++)
#pragma unroll
        for (int j = 0; j < kN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) sums[wave][i * kN + j][r][4 * g + q] = acc[i][j][q];
    __syncthreads();
    for (int at = threadIdx.x; at < kM * kN * 256; at += 64 * kFewWaves) {
        const int n = at % (16 * kN), m = at / (16 * kN);
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWaves; w++) s += sums[w][(m >> 4) * kN + (n >> 4)][m & 15][n & 15];
        if (m < d.M && n0 + n < d.N) ((C*)d.c)[m * d.ldc + n0 + n] = (C)s;
    }
}
// Up to 16 rows, which may be floats (17 rows as floats 9.5 us by 4096 x 4096 and 23.0 by 12000 x 4096, taken to 8 bits before 11.3 and 21.7; 32 rows
// 13.5 and 28.3 against 13.5 and 25.8); up to 32 while B's pairs of tiles are at most one to a CU (32 rows by 8192 x 4096: 15.7 us so, 19.4 in tiles of
// 64 x 64; by 12000 x 4096 25.8 and 19.8; by 12000 x 12000 62 and 33). More rows go into tiles (64 by 4096 x 4096: 19.4 us so, 17.6 in tiles).
constexpr int kFloatRows = 16;
static bool few_rows(int64_t M, int64_t N) { return M <= 16 || (M <= 32 && N <= 32 * 256); }

// The parts of a split sum, added in a fixed order: a block takes 256 results, four a lane, each of its four waves every fourth part.
template <class C> __global__ void __launch_bounds__(256) k_fp8_join(const float* parts, int n_parts, long long size, long long N, long long ldc, C* c) {
    __shared__ float4 sums[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long at = ((long long)blockIdx.x * 64 + lane) * 4;
    float4 s = { 0, 0, 0, 0 };
    if (at + 4 <= size) {
#pragma unroll 8
        for (int p = wave; p < n_parts; p += 4) {
            const auto v = *(const LooseRun<float, 4>*)(parts + p * size + at);
            s.x += v.v[0]; s.y += v.v[1]; s.z += v.v[2]; s.w += v.v[3];
        }
    } else if (at < size) {
        for (int p = wave; p < n_parts; p += 4) {
            const float* v = parts + p * size + at;
            s.x += v[0];
            if (at + 1 < size) s.y += v[1];
            if (at + 2 < size) s.z += v[2];
        }
    }
    if (wave) sums[wave - 1][lane] = s;
    __syncthreads();
    if (wave) return;
    for (int w = 0; w < 3; w++) { const float4 o = sums[w][lane]; s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w; }
    Run<C, 4> o;
    o.v[0] = (C)s.x; o.v[1] = (C)s.y; o.v[2] = (C)s.z; o.v[3] = (C)s.w;
    if (ldc == N && at + 4 <= size) { *(LooseRun<C, 4>*)(c + at) = *(const LooseRun<C, 4>*)&o; return; }
    for (int k = 0; k < 4; k++) if (at + k < size) c[(at + k) / N * ldc + (at + k) % N] = o.v[k];
}

// How a product is divided. Tiles of 256 x 256 (one to a CU) where they fill the chip and the sum is long enough for what they cost to begin and end
// (8192 x 8192 x 512: 51 us against 59 in tiles of 128; 65536 x 256 x 256: 14.6 against 12.7); of 128 x 128 (two) where there are more than 128
// (1003 x 2077 x 1500: 8.1 against 9.7 in tiles of 64); else of 64 x 64 (1000 x 1000 x 1000: 4.8 against 7.0, 512 x 4096 x 4096: 16.8 against 18.4).
// Long sums of few such tiles go into parts of at least 16 blocks of columns, which a second launch adds, from 48 blocks on (256 x 256 x 65536: 15.9
// against 198; 1024 x 1024 x 8192: 23.0 against 27.9; 64 x 4096 x 8192: 12.5 against 27.2, x 6144 12.5 against 11.5; with 32 blocks 64 x 4096 x 4096 9.3
// against 8.7, 256 x 4096 x 4096 16.5 against 10.3, 64 x 1024 x 4096 8.0 against 8.6).
struct Plan { int tile, parts, split_blocks; };
static Plan plan_of(int64_t M, int64_t N, int64_t K) {
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const auto tiles_of = [&](int64_t t) { return up(M, t) * up(N, t); };
    const int64_t blocks = up(K, 128);
    Plan p = { tiles_of(256) >= 200 && blocks >= 4 ? 256 : tiles_of(128) > 128 ? 128 : 64, 1, (int)blocks };
    const int64_t tiles = tiles_of(p.tile);
    if (p.tile == 64 && tiles <= 256 && blocks >= 48) {
        int64_t parts = 512 / tiles;
        if (parts > blocks / 16) parts = blocks / 16;
        p.split_blocks = (int)(up(up(blocks, parts), 4) * 4);
        p.parts = (int)up(blocks, p.split_blocks);
    }
    return p;
}

}  // namespace ntc_ops

using namespace ntc_ops;

static int check_quantize(const ntc_fp8_quantize_desc* d, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->R < 0 || d->K < 0 || d->row_stride < 0) return refuse(why, cap, "sizes and strides are not negative");
    if (d->dtype < 0 || d->dtype > 2) return refuse(why, cap, "x is 32-bit floats, bfloat16 or float16");
    if (d->block_rows != 1 && d->block_rows != 128) return refuse(why, cap, "blocks are 1 x 128 or 128 x 128");
    if (!d->codes && !d->codes_t) return refuse(why, cap, "nothing to write");
    if (d->R > (int64_t)1 << 36 || (d->K + 127) / 128 >= 1 << 24) return refuse(why, cap, "at most 2^36 rows, and fewer than 2^31 columns");
    if (d->R && d->K && (!d->x || (d->codes && !d->exps) || (d->codes_t && !d->exps_t))) return refuse(why, cap, "a null pointer");
    return 0;
}

extern "C" int ntc_op_fp8_quantize(const ntc_fp8_quantize_desc* d, void* stream, char* why, size_t cap) {
    if (const int r = check_quantize(d, why, cap)) return r;
    if (!d->R || !d->K) return 0;
    const int64_t down = (d->R + 127) / 128;
    const dim3 grid((unsigned)((d->K + 127) / 128), (unsigned)(down < kGridRows ? down : kGridRows), (unsigned)((down + kGridRows - 1) / kGridRows));
    const auto go = [&](auto kernel) { kernel<<<grid, 256, 0, (hipStream_t)stream>>>(*d); };
    if (d->block_rows == 128) d->dtype == NTC_F32 ? go(k_fp8_quantize<f32, true>) : d->dtype == NTC_BF16 ? go(k_fp8_quantize<bf16, true>) : go(k_fp8_quantize<f16, true>);
    else d->dtype == NTC_F32 ? go(k_fp8_quantize<f32, false>) : d->dtype == NTC_BF16 ? go(k_fp8_quantize<bf16, false>) : go(k_fp8_quantize<f16, false>);
    return launched(why, cap);
}

extern "C" int ntc_op_fp8_quantize_pair(const ntc_fp8_quantize_desc* a, const ntc_fp8_quantize_desc* b, void* stream, char* why, size_t cap) {
    if (const int r = check_quantize(a, why, cap)) return r;
    if (const int r = check_quantize(b, why, cap)) return r;
    if (a->block_rows != 1 || b->block_rows != 128) return refuse(why, cap, "a pair's blocks are 1 x 128 and 128 x 128");
    const int64_t across_a = (a->K + 127) / 128, across_b = (b->K + 127) / 128, tiles_a = (a->R + 127) / 128 * across_a, tiles_b = (b->R + 127) / 128 * across_b;
    if (!tiles_a || !tiles_b || a->dtype != b->dtype || tiles_a + tiles_b >= 1 << 24) {
        if (const int r = ntc_op_fp8_quantize(a, stream, why, cap)) return r;
        return ntc_op_fp8_quantize(b, stream, why, cap);
    }
    const auto go = [&](auto kernel) { kernel<<<(unsigned)(tiles_a + tiles_b), 256, 0, (hipStream_t)stream>>>(*a, *b, (uint32_t)tiles_a, (uint32_t)across_a, (uint32_t)across_b); };
    a->dtype == NTC_F32 ? go(k_fp8_quantize_pair<f32>) : a->dtype == NTC_BF16 ? go(k_fp8_quantize_pair<bf16>) : go(k_fp8_quantize_pair<f16>);
    return launched(why, cap);
}

extern "C" size_t ntc_op_fp8_matmul_workspace(int64_t M, int64_t N, int64_t K, int32_t) {
    if (M < 1 || N < 1 || K < 1 || few_rows(M, N)) return 0;
    const Plan p = plan_of(M, N, K);
    return p.parts > 1 ? (size_t)p.parts * M * N * 4 : 0;
}
extern "C" int64_t ntc_op_fp8_matmul_float_rows(void) { return kFloatRows; }

template <class A, int kM, class C> static void launch_few(const FewArgs& F, hipStream_t s) {
    // two tiles of B a wave where that still leaves a block to each CU (one row by 8192 x 4096: 8.1 us against 10.1; 4096 x 4096: 7.7 against 5.9)
    if (F.N >= 32 * 256) k_fp8_few<A, kM, 2, C><<<grid_of((F.N + 31) / 32), 64 * kFewWaves, 0, s>>>(F);
    else k_fp8_few<A, kM, 1, C><<<grid_of((F.N + 15) / 16), 64 * kFewWaves, 0, s>>>(F);
}
template <class C> static void run_few(const ntc_fp8_matmul_desc* d, hipStream_t s) {
    const FewArgs F = { d->a, d->a_exps, d->b, d->b_exps, d->c, d->N, d->a_stride, d->ldc, (int)d->M, (int)d->K, (int)((d->K + 127) / 128), (int)ntc_fp8_code_stride(d->K),
                        (int)ntc_fp8_exp_stride(d->K), d->a_block_rows == 128 ? 7 : 0, d->b_block_rows == 128 ? 7 : 0 };
    if (d->a_type == NTC_F32) launch_few<f32, 1, C>(F, s);
    else if (d->a_type == NTC_BF16) launch_few<bf16, 1, C>(F, s);
    else if (d->a_type == NTC_F16) launch_few<f16, 1, C>(F, s);
    else if (d->M <= 16) launch_few<uint8_t, 1, C>(F, s);
    else launch_few<uint8_t, 2, C>(F, s);
}

template <int T, class C> static void launch_matmul(const MatmulArgs& A, int parts, hipStream_t s) {
    const unsigned tiles = (unsigned)(A.tiles_m * A.tiles_n);
    if constexpr (T == 64)
        if (parts > 1) { k_fp8_matmul<T, T, float, true><<<tiles * parts, 256, 0, s>>>(A); return; }
    k_fp8_matmul<T, T, C, false><<<tiles, 256, 0, s>>>(A);
}

template <class C> static void run_matmul(const ntc_fp8_matmul_desc* d, hipStream_t s) {
    const Plan p = plan_of(d->M, d->N, d->K);
    MatmulArgs A;
    A.a = (const uint8_t*)d->a;
    A.ae = d->a_exps;
    A.b = d->b;
    A.be = d->b_exps;
    A.M = d->M;
    A.N = d->N;
    A.stride = (int)ntc_fp8_code_stride(d->K);
    A.estride = (int)ntc_fp8_exp_stride(d->K);
    A.blocks = (int)((d->K + 127) / 128);
    A.a_shift = d->a_block_rows == 128 ? 7 : 0;
    A.b_shift = d->b_block_rows == 128 ? 7 : 0;
    A.tiles_m = (int)((d->M + p.tile - 1) / p.tile);
    A.tiles_n = (int)((d->N + p.tile - 1) / p.tile);
    A.split_blocks = p.split_blocks;
    A.c = p.parts > 1 ? d->workspace : d->c;
    A.ldc = p.parts > 1 ? d->N : d->ldc;
    if (p.tile == 256) launch_matmul<256, C>(A, 1, s);
    else if (p.tile == 128) launch_matmul<128, C>(A, 1, s);
    else launch_matmul<64, C>(A, p.parts, s);
    if (p.parts > 1) k_fp8_join<C><<<(unsigned)((d->M * d->N + 255) / 256), 256, 0, s>>>((const float*)d->workspace, p.parts, d->M * d->N, d->N, d->ldc, (C*)d->c);
}

extern "C" int ntc_op_fp8_matmul(const ntc_fp8_matmul_desc* d, void* stream, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->M < 0 || d->N < 0 || d->K < 0) return refuse(why, cap, "sizes are not negative");
    if (d->a_type < 0 || d->a_type > NTC_FP8) return refuse(why, cap, "A is 8-bit codes, or 32-bit floats, bfloat16 or float16");
    if (d->a_type != NTC_FP8 && d->M > kFloatRows) return refuse(why, cap, "A of more than 16 rows is given in 8 bits");
    if (d->a_type != NTC_FP8 && d->a_stride < 0) return refuse(why, cap, "strides are not negative");
    if (d->c_type < 0 || d->c_type > 2) return refuse(why, cap, "C is 32-bit floats, bfloat16 or float16");
    if ((d->a_block_rows != 1 && d->a_block_rows != 128) || (d->b_block_rows != 1 && d->b_block_rows != 128)) return refuse(why, cap, "blocks are 1 x 128 or 128 x 128");
    if (d->ldc < d->N) return refuse(why, cap, "C's rows overlap");
    if (d->K > 1 << 23 || d->M > (int64_t)1 << 36 || d->N > (int64_t)1 << 36 || (d->M + 127) / 128 * ((d->N + 127) / 128) >= 1 << 24)
        return refuse(why, cap, "K at most 2^23, and fewer than 2^24 tiles of 128 x 128");
    if (!d->M || !d->N) return 0;
    if (!d->K) return refuse(why, cap, "K is at least 1");
    const bool codes = d->a_type == NTC_FP8;
    if (!d->c || !d->a || (codes && !d->a_exps) || !d->b || !d->b_exps) return refuse(why, cap, "a null pointer");
    if ((((codes ? (uintptr_t)d->a : 0) | (uintptr_t)d->b) & 15) || (((codes ? (uintptr_t)d->a_exps : 0) | (uintptr_t)d->b_exps) & 3))
        return refuse(why, cap, "codes start at multiples of 16 bytes, exponents of 4");
    if (!d->workspace && ntc_op_fp8_matmul_workspace(d->M, d->N, d->K, d->a_type)) return refuse(why, cap, "a null workspace");
    const hipStream_t s = (hipStream_t)stream;
    if (few_rows(d->M, d->N)) {
        d->c_type == NTC_F32 ? run_few<f32>(d, s) : d->c_type == NTC_BF16 ? run_few<bf16>(d, s) : run_few<f16>(d, s);
        return launched(why, cap);
    }
    d->c_type == NTC_F32 ? run_matmul<f32>(d, s) : d->c_type == NTC_BF16 ? run_matmul<bf16>(d, s) : run_matmul<f16>(d, s);
    return launched(why, cap);
}
