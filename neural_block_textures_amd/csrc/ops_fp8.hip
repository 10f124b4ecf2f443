// Matrices in 8-bit floating point with a power-of-two scale for each block of 128, and their products (include/ntc_ops.h).
#include "ops_common.hpp"

namespace ntc_ops {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float power_of(int b) { return __uint_as_float(b > 0 ? (uint32_t)b << 23 : 1u << 22); }   // 2^(b - 127), b from 0 to 254
// The bits of |x|, 0 where x is not finite.
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
    return a < 0x7f800000u ? a : 0u;
}
// The exponent byte of a block whose largest finite magnitude has these bits: amax <= 448 * 2^(E - 127).
__device__ __forceinline__ int exp_byte(uint32_t most) {
    const int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 0 ? 0 : e;
}
__device__ __forceinline__ uint32_t to_fp8x4(float a, float b, float c, float d) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return r;
}

// ---------------------------------------------------------------- to 8 bits
// A block of 256 threads takes a 128 x 128 tile: thread t holds 8 columns (8 (t % 16) ..) of the 8 rows 8 (t / 16) .., so that a
// row's largest is a reduction over 16 lanes, and a column's codes of 8 rows are one 8-byte word of the transposed tile.
template <class T, bool kBlock> __global__ void __launch_bounds__(256) k_fp8_quantize(ntc_fp8_quantize_desc d) {
    __shared__ uint32_t most[4][128];
    __shared__ alignas(16) uint8_t tile[128][144];
    const long long r0 = (long long)blockIdx.y * 128, c0 = (long long)blockIdx.x * 128;
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    const long long c = c0 + 8 * cg, r = r0 + 8 * rg;
    float x[8][8];
    for (int i = 0; i < 8; i++)
        for (int j = 0; j < 8; j++) x[i][j] = r + i < d.R && c + j < d.K ? (float)((const T*)d.x)[(r + i) * d.row_stride + c + j] : 0.0f;
    const long long code_stride = ntc_fp8_code_stride(d.K), exp_stride = ntc_fp8_exp_stride(d.K), blocks = (d.K + 127) / 128;
    const long long code_stride_t = ntc_fp8_code_stride(d.R), exp_stride_t = ntc_fp8_exp_stride(d.R), blocks_t = (d.R + 127) / 128;
    int block_byte = 0;
    if (kBlock) {
        uint32_t b = 0;
        for (int i = 0; i < 8; i++) for (int j = 0; j < 8; j++) { const uint32_t a = finite_bits(x[i][j]); b = a > b ? a : b; }
        for (int w = 1; w < 64; w <<= 1) { const uint32_t o = __shfl_xor(b, w); b = o > b ? o : b; }
        if ((threadIdx.x & 63) == 0) most[wave][0] = b;
        __syncthreads();
        for (int w = 0; w < 4; w++) b = most[w][0] > b ? most[w][0] : b;
        block_byte = exp_byte(b);
        if (threadIdx.x == 0) {
            if (d.codes) {
                uint8_t* e = d.exps + blockIdx.y * exp_stride;
                e[blockIdx.x] = (uint8_t)block_byte;
                if (blockIdx.x == blocks - 1) for (long long k = blocks; k < exp_stride; k++) e[k] = 0;
            }
            if (d.codes_t) {
                uint8_t* e = d.exps_t + blockIdx.x * exp_stride_t;
                e[blockIdx.y] = (uint8_t)block_byte;
                if (blockIdx.y == blocks_t - 1) for (long long k = blocks_t; k < exp_stride_t; k++) e[k] = 0;
            }
        }
    }
    if (d.codes) {
        for (int i = 0; i < 8; i++) {
            int byte = block_byte;
            if (!kBlock) {
                uint32_t b = 0;
                for (int j = 0; j < 8; j++) { const uint32_t a = finite_bits(x[i][j]); b = a > b ? a : b; }
                for (int w = 1; w < 16; w <<= 1) { const uint32_t o = __shfl_xor(b, w); b = o > b ? o : b; }
                byte = exp_byte(b);
                if (cg == 0 && r + i < d.R) {
                    uint8_t* e = d.exps + (r + i) * exp_stride;
                    e[blockIdx.x] = (uint8_t)byte;
                    if (blockIdx.x == blocks - 1) for (long long k = blocks; k < exp_stride; k++) e[k] = 0;
                }
            }
            if (r + i >= d.R) continue;
            const float s = power_of(254 - byte);
            uint2 o;
            o.x = to_fp8x4(x[i][0] * s, x[i][1] * s, x[i][2] * s, x[i][3] * s);
            o.y = to_fp8x4(x[i][4] * s, x[i][5] * s, x[i][6] * s, x[i][7] * s);
            *(uint2*)(d.codes + (r + i) * code_stride + c) = o;
        }
    }
    if (!d.codes_t) return;
    if (!kBlock) {
        for (int j = 0; j < 8; j++) {
            uint32_t b = 0;
            for (int i = 0; i < 8; i++) { const uint32_t a = finite_bits(x[i][j]); b = a > b ? a : b; }
            for (int w = 16; w < 64; w <<= 1) { const uint32_t o = __shfl_xor(b, w); b = o > b ? o : b; }
            if ((threadIdx.x & 48) == 0) most[wave][8 * cg + j] = b;
        }
        __syncthreads();
    }
    for (int j = 0; j < 8; j++) {
        int byte = block_byte;
        if (!kBlock) {
            uint32_t b = 0;
            for (int w = 0; w < 4; w++) b = most[w][8 * cg + j] > b ? most[w][8 * cg + j] : b;
            byte = exp_byte(b);
            if (rg == 0 && c + j < d.K) {
                uint8_t* e = d.exps_t + (c + j) * exp_stride_t;
                e[blockIdx.y] = (uint8_t)byte;
                if (blockIdx.y == blocks_t - 1) for (long long k = blocks_t; k < exp_stride_t; k++) e[k] = 0;
            }
        }
        const float s = power_of(254 - byte);
        uint2 o;
        o.x = to_fp8x4(x[0][j] * s, x[1][j] * s, x[2][j] * s, x[3][j] * s);
        o.y = to_fp8x4(x[4][j] * s, x[5][j] * s, x[6][j] * s, x[7][j] * s);
        *(uint2*)&tile[8 * cg + j][8 * rg] = o;
    }
    __syncthreads();
    for (int p = 0; p < 4; p++) {
        const int col = 32 * p + (threadIdx.x >> 3), part = threadIdx.x & 7;
        if (c0 + col < d.K) *(uint4*)(d.codes_t + (c0 + col) * code_stride_t + r0 + 16 * part) = *(const uint4*)&tile[col][16 * part];
    }
}

// ---------------------------------------------------------------- products
// v_mfma_scale_f32_16x16x128: lane l holds 32 bytes of row l % 16 at k = 32 (l / 16) of each operand and that row's exponent; the
// result's element i of lane l is (first operand's row 4 (l / 16) + i, second's row l % 16). The first operand is B here, so
// that a lane's four results are neighbours in C's row.
template <class C> __global__ void __launch_bounds__(256) k_fp8_matmul(ntc_fp8_matmul_desc d) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const long long m0 = (long long)blockIdx.y * 64 + 32 * (wave >> 1), n0 = (long long)blockIdx.x * 64 + 32 * (wave & 1);
    const long long code_stride = ntc_fp8_code_stride(d.K), exp_stride = ntc_fp8_exp_stride(d.K);
    long long am[2], bn[2];
    for (int i = 0; i < 2; i++) {
        am[i] = m0 + 16 * i + r < d.M ? m0 + 16 * i + r : d.M - 1;
        bn[i] = n0 + 16 * i + r < d.N ? n0 + 16 * i + r : d.N - 1;
    }
    v4f acc[2][2] = {};
    for (long long k = 0; k < d.K; k += 128) {
        v8i a[2], b[2];
        int ea[2], eb[2];
        for (int i = 0; i < 2; i++) {
            a[i] = *(const v8i*)((const uint8_t*)d.a + am[i] * code_stride + k + 32 * g);
            b[i] = *(const v8i*)(d.b + bn[i] * code_stride + k + 32 * g);
            ea[i] = d.a_exps[am[i] / d.a_block_rows * exp_stride + k / 128];
            eb[i] = d.b_exps[bn[i] / d.b_block_rows * exp_stride + k / 128];
        }
        for (int i = 0; i < 2; i++)
            for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a[i], acc[i][j], 0, 0, 0, eb[j], 0, ea[i]);
    }
    for (int i = 0; i < 2; i++)
        for (int j = 0; j < 2; j++) {
            const long long m = m0 + 16 * i + r, n = n0 + 16 * j + 4 * g;
            if (m >= d.M) continue;
            for (int q = 0; q < 4; q++) if (n + q < d.N) ((C*)d.c)[m * d.ldc + n + q] = (C)acc[i][j][q];
        }
}

}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" int ntc_op_fp8_quantize(const ntc_fp8_quantize_desc* d, void* stream, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->R < 0 || d->K < 0 || d->row_stride < 0) return refuse(why, cap, "sizes and strides are not negative");
    if (d->dtype < 0 || d->dtype > 2) return refuse(why, cap, "x is 32-bit floats, bfloat16 or float16");
    if (d->block_rows != 1 && d->block_rows != 128) return refuse(why, cap, "blocks are 1 x 128 or 128 x 128");
    if (!d->codes && !d->codes_t) return refuse(why, cap, "nothing to write");
    const int64_t gy = (d->R + 127) / 128, gx = (d->K + 127) / 128;
    if (gy > 65535 || gx > 0x7fffffff) return refuse(why, cap, "at most 65535 * 128 rows");
    if (!gx || !gy) return 0;
    if (!d->x || (d->codes && !d->exps) || (d->codes_t && !d->exps_t)) return refuse(why, cap, "a null pointer");
    const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)gx, (unsigned)gy), 256, 0, (hipStream_t)stream>>>(*d); };
    if (d->block_rows == 128) d->dtype == NTC_F32 ? go(k_fp8_quantize<f32, true>) : d->dtype == NTC_BF16 ? go(k_fp8_quantize<bf16, true>) : go(k_fp8_quantize<f16, true>);
    else d->dtype == NTC_F32 ? go(k_fp8_quantize<f32, false>) : d->dtype == NTC_BF16 ? go(k_fp8_quantize<bf16, false>) : go(k_fp8_quantize<f16, false>);
    return launched(why, cap);
}

extern "C" size_t ntc_op_fp8_matmul_workspace(int64_t, int64_t, int64_t) { return 0; }
extern "C" int64_t ntc_op_fp8_matmul_float_rows(void) { return 0; }

extern "C" int ntc_op_fp8_matmul(const ntc_fp8_matmul_desc* d, void* stream, char* why, size_t cap) {
    if (!d) return refuse(why, cap, "no description");
    if (d->M < 0 || d->N < 0 || d->K < 0) return refuse(why, cap, "sizes are not negative");
    if (d->a_type != NTC_FP8) return refuse(why, cap, "A is a matrix in 8 bits");
    if (d->c_type < 0 || d->c_type > 2) return refuse(why, cap, "C is 32-bit floats, bfloat16 or float16");
    if ((d->a_block_rows != 1 && d->a_block_rows != 128) || (d->b_block_rows != 1 && d->b_block_rows != 128)) return refuse(why, cap, "blocks are 1 x 128 or 128 x 128");
    if (d->ldc < d->N) return refuse(why, cap, "C's rows overlap");
    const int64_t gy = (d->M + 63) / 64, gx = (d->N + 63) / 64;
    if (gy > 65535 || gx > 0x7fffffff) return refuse(why, cap, "at most 65535 * 64 rows");
    if (!gx || !gy) return 0;
    if (!d->c || (d->K && (!d->a || !d->a_exps || !d->b || !d->b_exps))) return refuse(why, cap, "a null pointer");
    const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)gx, (unsigned)gy), 256, 0, (hipStream_t)stream>>>(*d); };
    d->c_type == NTC_F32 ? go(k_fp8_matmul<f32>) : d->c_type == NTC_BF16 ? go(k_fp8_matmul<bf16>) : go(k_fp8_matmul<f16>);
    return launched(why, cap);
}
