// Attention over packed sequences, and its gradients (include/ntc_ops.h: ntc_op_attention).
//
// Forward, for a sequence's queries i and keys j: s = c q_i k_j (c = scale log2 e), p = 2^(s - m), o = sum p v / sum p, keys taken 64 at a time with a
// running m and sum (rows are rescaled where a maximum rises by more than 2^8). Backward: p = 2^(s - lse), dS = p (dO v - D).
// The query heads that share a key head are rows of one matrix: row r of a sequence is query r / G, head r % G of the G. So keys and values are read
// once for all of them, single tokens fill a tile, and the gradients of shared heads are sums over rows like any other.
//
// Matrix products are 32 x 32 x 16. A lane holds one column of a result and 16 of its rows, and 8 neighbouring values of one row of an operand.
// Scores are made transposed (keys x queries): a lane's column is a query, its maximum and sum are the lane's own (and its other half's), and the scores, rounded, are at once the
// second operand of the product that sums over keys; which keys stand at which place of that sum does not matter as long as the other
// operand has them in the same order: 8 places of half h are keys 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3 of sixteen. That operand
// (values or keys, transposed) comes from LDS by the transposing read, four keys of a column at a time. The keys' and values' gradients go the same way with
// queries and keys exchanged. No score leaves a register.
#include "ops_common.hpp"

namespace ntc_ops {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <class T> __device__ __forceinline__ v16f product(v4u a, v4u b, v16f c) {
    if constexpr (std::is_same_v<T, bf16>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T v2 __attribute__((ext_vector_type(2)));
    const v2 x = { (T)a, (T)b };
    return __builtin_bit_cast(uint32_t, x);
}
// c and both halves of x
template <class T> __device__ __forceinline__ float add2(uint32_t x, float c) {
    typedef T v2 __attribute__((ext_vector_type(2)));
    const v2 one = { (T)1.f, (T)1.f };
    if constexpr (std::is_same_v<T, bf16>) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, x), one, c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, x), one, c, false);
}
// of lanes l and l ^ 32
__device__ __forceinline__ float other_half(float x) {
    const uint32_t b = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(lane_id() < 32 ? (uint32_t)p[1] : (uint32_t)p[0]);
}

struct Operand3 { const char* p; long long row, head, batch; };    // strides in bytes
struct AttentionArgs {
    Operand3 q, k, v, d_o;
    void *out, *rest, *dq, *dk, *dv;
    float *lse, *log_sums, *deltas;    // backward [q_rows][q_heads]: log2 sum exp less kShift, dO o times the sequence's power of two over 2^kShift
    float *extents_v, *extents_do;     // float16, backward: the largest |v| and |dO| of each kExtentRows rows of a sequence
    int v_extents, v_extents_each, do_extents, do_extents_each;    // how many in all, and of each sequence where there are no ends
    const int *cu_q, *cu_k, *k_lens;
    long long q_rows, k_rows;
    int sequences, q_each, k_each;     // rows of a sequence where there are no ends
    int q_heads, k_heads, group, D, causal;
    unsigned group_magic;              // ceil(2^32 / group): x / group is the high word of the product with it where x group < 2^32; 0 for 1
    int parts;                         // of a sequence's keys (dk and dv: of its rows), joined by a second launch; their sums:
    float* part_sums;                  // forward [parts][q_rows][q_heads][D]; backward dk's [parts][k_rows][k_heads][D], then dv's; dq's [parts][q_rows][q_heads][D], then part_rests
    float* part_rests;                 // [parts][q_rows][q_heads]: what the rounded dS add up to
    float2* part_stats;                // forward [parts][q_rows][q_heads]: m c (float16: less 7) and the sum of probabilities (-1: of keys whose scores are all -inf)
    int line_heads;                    // log2 of how many heads share a line of the cache (128 bytes)
    int tiles, tiles_each;             // tiles of rows (or keys) in all, and of each sequence where there are no ends
    float scale, c;                    // c: scale log2 e
};

constexpr int kRows = 128, kKeys = 64, kExtentRows = 32;

// ---------------------------------------------------------------- which rows
struct Span { int b; long long row; int n; long long start; };     // sequence, its first row in all, its rows, the byte where they start
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long cut(long long x, long long lo, long long hi) { return x < lo ? lo : x > hi ? hi : x; }

// Tile t of all, to its sequence and its number there. With ends, sequence b's tiles are numbered from e_b units / size + b on, which leaves each at least as many numbers as
// it has tiles, and none shared: the largest b whose first number is at most t, by 64 probes at once. Rows behind the last sequence are one more.
template <int kSize> __device__ __forceinline__ int first_tile(const int* cu, int tiles_each, int units, int b) {
    if (!cu) return b * tiles_each;
    const long long e = b ? cu[b] : 0;
    return (int)cut(e * units / kSize, 0, 1 << 30) + b;
}
template <int kSize> __device__ __forceinline__ int find_sequence(const int* cu, int sequences, int tiles_each, int units, int t, int& tile) {
    if (!cu) { const int b = t / tiles_each; tile = t - b * tiles_each; return b; }
    const auto first = [&](int b) { return first_tile<kSize>(cu, tiles_each, units, b); };
    int lo = 0, hi = sequences;
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64, probe = lo + (lane_id() + 1) * step;
        const bool at_most = probe <= hi && first(probe <= hi ? probe : hi) <= t;
        lo += __builtin_popcountll(__ballot(at_most)) * step;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    lo = uniform(lo < sequences ? lo : sequences);
    tile = t - uniform(first(lo));
    return lo;
}
__device__ __forceinline__ Span span_of(const int* cu, int sequences, int each, long long rows, int b, const Operand3& x) {
    if (!cu) return { b, (long long)b * each, b < sequences ? each : 0, b * x.batch };
    const long long first = b ? cut(cu[b], 0, rows) : 0, end = b < sequences ? cut(cu[b + 1], first, rows) : rows;
    return { b, first, (int)(end - first), first * x.row };
}
// (keys that a sequence has, of those that it has room for)
__device__ __forceinline__ int keys_of(const AttentionArgs& d, const Span& k) {
    if (k.b >= d.sequences) return 0;
    return d.k_lens ? (int)cut(d.k_lens[k.b], 0, k.n) : k.n;
}

// A block's key head, part and number of its tile: heads of a tile lie beside each other, so that eight heads' keys and values are in the caches of one of the 8 XCDs each, to which blocks are
// dealt in turn; heads that share a line of the cache are on one XCD (64 sequences of 600 to 1024, 8 heads of 32, both ways: 262 us, with neighbours on different ones 271). (In 32 bits: a division in 64 takes the scalar unit a thousand cycles, and there are several.)
struct BlockPlace { int head, part; unsigned number; };
__device__ __forceinline__ BlockPlace place_of(const AttentionArgs& d) {
    const unsigned dealt = blockIdx.x + blockIdx.y * gridDim.x, set = (8u << d.line_heads) - 1;
    const unsigned id = (dealt & ~set) | (dealt & 7) << d.line_heads | (dealt & set) >> 3, rest = id / (unsigned)d.k_heads, number = d.parts == 1 ? rest : rest / (unsigned)d.parts;
    return { (int)(id - rest * d.k_heads), (int)(rest - number * d.parts), number };
}

// ---------------------------------------------------------------- shared memory
// Rows of kPitch bytes; the 16-byte piece c of row r lies at c ^ spread(r). 64 banks give 256 bytes a clock: 16 rows' pieces of one number are in different
// banks, and so are four rows' pieces of four neighbouring numbers, which a transposing read takes from 32 lanes (both measured without conflicts; a spread over eight rows takes twice
// as long). What depends on the lane is made once; the rest is constant offsets.
template <int kD> struct Tile {
    static constexpr int kPitch = kD <= 32 ? 64 : kD <= 64 ? 128 : 256, kPieces = kPitch / 16, kLines = 256 / kPitch;
    static __device__ __forceinline__ int spread(int r) { return (((r & 3) / kLines) << 2 | ((r >> 2) & 3)) & (kPieces - 1); }
};
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }
// 16 (4) bytes a lane from base + off to LDS at `to` + 16 (4) lane: `to` is the same in all lanes. Nothing waits for it but a vmcnt of the caller's.
__device__ __forceinline__ void to_lds16(uint32_t to, uint32_t off, const char* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(uint32_t to, uint32_t off, const char* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" :: "s"(to), "v"(off), "s"(base) : "memory", "m0");
}
// All of the wave's loads have landed, and every wave is here.
__device__ __forceinline__ void arrive() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                    // vmcnt 0, lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

typedef __attribute__((address_space(3))) const char* Shared;
// A wave's places in a tile: of its lane's row as an operand, and of the columns of 16 rows.
template <int kD> struct Places {
    using L = Tile<kD>;
    uint32_t row[kD / 16], column[kD / 32][2];
    __device__ __forceinline__ Places(uint32_t tile) {
        const int lane = lane_id(), half = lane >> 5, r = lane & 31, i = lane & 15;
#pragma unroll
        for (int s = 0; s < kD / 16; s++) row[s] = tile + r * L::kPitch + (((2 * s + half) ^ L::spread(r)) << 4);
#pragma unroll
        for (int t = 0; t < kD / 32; t++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const int k = 8 * b + 4 * half + (i >> 2), piece = 4 * t + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                column[t][b] = tile + k * L::kPitch + ((piece ^ L::spread(k)) << 4) + 8 * (i & 1);
            }
    }
    // columns 16 step + 8 half on of the lane's row of 32, from row `first`, of the tile `at` bytes on
    __device__ __forceinline__ v4u row_piece(int at, int first, int step) const {
        return *(__attribute__((address_space(3))) const v4u*)((Shared)row[step] + (at + first * L::kPitch));
    }
    // of 16 rows from `first` on, 8 rows of column 32 tile + lane % 32: rows 4 half .. and 8 + 4 half ..
    __device__ __forceinline__ v4u column_piece(int at, int first, int tile) const {
        v2u r[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
            r[b] = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)((Shared)column[tile][b] + (at + first * L::kPitch))));
        return v4u{ r[0].x, r[0].y, r[1].x, r[1].y };
    }
    // between two buffers whose addresses differ in one bit
    __device__ __forceinline__ void toggle_rows(int bit) {
#pragma unroll
        for (uint32_t& x : row) x ^= bit;
    }
    __device__ __forceinline__ void toggle_columns(int bit) {
#pragma unroll
        for (auto& x : column) { x[0] ^= bit; x[1] ^= bit; }
    }
};
// Rows of a matrix into a tile of kTile rows: each wave of four takes a quarter, 16 bytes a lane and load. The lane's row in the tile and its piece's byte there, of load i:
template <int kD, int kTile> struct Loads {
    using L = Tile<kD>;
    static constexpr int kEach = kTile * L::kPieces / 256;                 // loads a wave
    static __device__ __forceinline__ int slot(int i) { return (uniform(threadIdx.x >> 6) * kEach + i) * 64 + lane_id(); }
    static __device__ __forceinline__ int row(int i) { return slot(i) / L::kPieces; }
    static __device__ __forceinline__ int byte(int i, int D) {
        const int piece = (slot(i) % L::kPieces) ^ L::spread(row(i));
        return 16 * (8 * piece < D ? piece : 0);                           // past a head's end: any values of the row
    }
    // offset(i): of load i from `base`
    template <class F> static __device__ __forceinline__ void run(uint32_t to, const char* base, F offset) {
#pragma unroll
        for (int i = 0; i < kEach; i++) to_lds16(to + 1024 * (uniform(threadIdx.x >> 6) * kEach + i), offset(i), base);
    }
};
// ... of consecutive rows `stride` bytes apart, `n` of them there (past the end the last one again)
template <int kD, int kTile> struct RowLoads : Loads<kD, kTile> {
    using B = Loads<kD, kTile>;
    uint32_t off[B::kEach];
    int stride, D;
    __device__ __forceinline__ RowLoads(long long stride_, int D_) : stride((int)stride_), D(D_) {
#pragma unroll
        for (int i = 0; i < B::kEach; i++) off[i] = (uint32_t)B::row(i) * (uint32_t)stride + B::byte(i, D);
    }
    // load i of a whole tile
    __device__ __forceinline__ void piece(uint32_t to, const char* base, int i) const { to_lds16(to + 1024 * (uniform(threadIdx.x >> 6) * B::kEach + i), off[i], base); }
    __device__ __forceinline__ void load(uint32_t to, const char* base, int n) const {
        if (n >= kTile) B::run(to, base, [&](int i) { return off[i]; });
        else B::run(to, base, [&](int i) { const int r = B::row(i); return (uint32_t)(r < n ? r : n - 1) * (uint32_t)stride + B::byte(i, D); });
    }
};

// ---------------------------------------------------------------- rows in registers
// A row of a group's matrix: query and head, from a tile's first row
struct Row { int i, g; };
__device__ __forceinline__ Row row_at(const AttentionArgs& d, int i0, int g0, int x) {   // x rows after row (i0, g0), x + g0 < 2^16
    const int y = g0 + x, q = d.group_magic ? (int)__umulhi((unsigned)y, d.group_magic) : y;
    return { i0 + q, y - q * d.group };
}
// the lane's row as an operand: columns 16 step + 8 half .., 0 past D
template <int kD> __device__ __forceinline__ void load_row(v4u (&x)[kD / 16], const char* p, bool live, int D) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int s = 0; s < kD / 16; s++) {
        const int col = 16 * s + 8 * half;
        x[s] = live && col < D ? *(const v4u*)(p + 2 * col) : v4u{};
    }
}
template <class T> constexpr float kRest = std::is_same_v<T, f16> ? 2048.f : 1.f;   // what a result's rounding leaves is held times this: as large as the result
// a transposed result (32 kTiles columns of the lane's row) to memory, times f; with kRests what its rounding left
template <class T, int kD, bool kRests = false> __device__ __forceinline__ void store_row(char* p, const v16f (&x)[kD / 32], float f, bool live, int D) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int t = 0; t < kD / 32; t++)
#pragma unroll
        for (int a = 0; a < 2; a++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float y[2] = { x[t][8 * a + 2 * i] * f, x[t][8 * a + 2 * i + 1] * f };
                if constexpr (kRests) for (float& z : y) z = (z - (float)(T)z) * kRest<T>;
                w[i] = pack2<T>(y[0], y[1]);
            }
            const auto lo = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), hi = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            const int col = 32 * t + 16 * a + 8 * half;
            if (live && col < D) *(v4u*)(p + 2 * col) = v4u{ (uint32_t)lo[0], (uint32_t)hi[0], (uint32_t)lo[1], (uint32_t)hi[1] };
        }
}
// ... in 32 bits
template <int kD> __device__ __forceinline__ void store_floats(float* p, const v16f (&x)[kD / 32], float f, bool live, int D) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int t = 0; t < kD / 32; t++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
            const int col = 32 * t + 8 * a + 4 * half;
            if (live && col < D) *(float4*)(p + col) = make_float4(x[t][4 * a] * f, x[t][4 * a + 1] * f, x[t][4 * a + 2] * f, x[t][4 * a + 3] * f);
        }
}
// result register r of the lane is row 8 (r / 4) + 4 half + r % 4
__device__ __forceinline__ constexpr int result_row(int r) { return 8 * (r / 4) + r % 4; }
template <class T> __device__ __forceinline__ v4u packed(const v16f& x, int half16) {
    return v4u{ pack2<T>(x[8 * half16], x[8 * half16 + 1]), pack2<T>(x[8 * half16 + 2], x[8 * half16 + 3]), pack2<T>(x[8 * half16 + 4], x[8 * half16 + 5]),
                pack2<T>(x[8 * half16 + 6], x[8 * half16 + 7]) };
}

// ---------------------------------------------------------------- forward
// Four waves of 32 rows each go through keys and values 64 at a time, two buffers of each, which all of them read. The next stage's scores are made between this one's
// exponentials, so that the matrix unit is fed meanwhile. Causal, of what is not masked: 8192 tokens of 16 heads on 4 of 128 in 286 to 310 us, 890 to 960 TFLOP/s; seven sequences of 300
// to 4096 tokens, 32 heads on 8, in 373, 990 TFLOP/s, of which 297 are left when LDS reads, exponentials and loads are taken out: the matrix unit at the clock that the power leaves it, and
// masked halves of tiles. Heads of 32 are bound by their exponentials, one for 64 multiplications. Single tokens of 32 heads on 8 against 16 caches of 900 to 8192 keys: 66 us, 4.5 TB/s.
// float16: probabilities and their sum are held times 2^7, so that they are at most 2^15 (a maximum lags by 2^8) and those down to 2^-32 of a row's largest count: without, 60000 keys at 2^-25 of it,
// 2e-3 of the sum, came to twice that or to nothing.
template <class T> constexpr float kLift = std::is_same_v<T, f16> ? 7.f : 0.f;
template <class T, int kD> __global__ void __launch_bounds__(256, kD <= 32 ? 4 : kD <= 64 ? 3 : 2) k_attention(AttentionArgs d) {
    using L = Tile<kD>;
    constexpr int kTile = kKeys * L::kPitch;
    __shared__ alignas(2 * kTile) char lds[4 * kTile];     // keys, values; two of each
    const BlockPlace own_place = place_of(d);
    const int head = own_place.head, part = own_place.part;
    const unsigned number = own_place.number;
    if (number >= (unsigned)d.tiles) return;
    int tile;
    const int b = find_sequence<kRows>(d.cu_q, d.sequences, d.tiles_each, d.group, d.tiles - 1 - (int)number, tile);   // (a sequence's last rows, which see most keys, first)
    const Span qs = span_of(d.cu_q, d.sequences, d.q_each, d.q_rows, b, d.q);
    const long long rows = (long long)qs.n * d.group;
    if (tile < 0 || (long long)tile * kRows >= rows) return;
    const int kb = b < d.sequences ? b : 0;
    Span ks = span_of(d.cu_k, d.sequences, d.k_each, d.k_rows, kb, d.k);
    const int Lk = b < d.sequences ? keys_of(d, ks) : 0, off = Lk - qs.n;
    const long long v_start = d.cu_k ? ks.row * d.v.row : ks.b * d.v.batch;

    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), column = lane & 31, half = lane >> 5;
    const int r0 = tile * kRows + 32 * wave, i0 = r0 / d.group, g0 = r0 - i0 * d.group;
    const Row row = row_at(d, i0, g0, column);
    const bool live = row.i < qs.n;
    v4u q[kD / 16];
    load_row<kD>(q, d.q.p + qs.start + row.i * d.q.row + (head * d.group + row.g) * d.q.head, live, d.D);
    const int last = d.causal ? (row.i + off < Lk - 1 ? row.i + off : Lk - 1) : Lk - 1;                           // the last key that the lane's query sees
    const int wave_first = d.causal ? (i0 + off < Lk - 1 ? i0 + off : Lk - 1) : Lk - 1;                           // ... that each of the wave's does
    const int i_wave = (r0 + 31) / d.group, i_block = (tile * kRows + kRows - 1) / d.group;
    const int wave_last = d.causal ? (i_wave + off < Lk - 1 ? i_wave + off : Lk - 1) : Lk - 1;
    const int block_last = d.causal ? (i_block + off < Lk - 1 ? i_block + off : Lk - 1) : Lk - 1;
    const int all = block_last < 0 ? 0 : block_last / kKeys + 1;
    const int begin = d.parts == 1 ? 0 : all * part / d.parts, stages = d.parts == 1 ? all : all * (part + 1) / d.parts;   // (2^24 stages at most, 64 parts)

    // A stage is 64 keys. While its probabilities are made and summed up with the values, the next stage's scores are: products and the exponentials between them are
    // in an order that keeps both kinds of unit busy (a wave issues in order), with operands on their way two products ahead. Keys are loaded two stages ahead, values one.
    const char *kp = d.k.p + ks.start + head * d.k.head, *vp = d.v.p + v_start + head * d.v.head;
    const uint32_t lds0 = lds_address(lds);
    const RowLoads<kD, kKeys> key_loads(d.k.row, d.D), value_loads(d.v.row, d.D);
    const auto load_keys = [&](int s) { key_loads.load(lds0 + ((s - begin) & 1) * kTile, kp + (long long)s * kKeys * d.k.row, Lk - s * kKeys); };
    const auto load_values = [&](int s) { value_loads.load(lds0 + (2 + ((s - begin) & 1)) * kTile, vp + (long long)s * kKeys * d.v.row, Lk - s * kKeys); };
    constexpr int kPieces = 2 * Loads<kD, kKeys>::kEach;   // of both tiles' loads that a stage issues, between its first products where the tiles are whole
    constexpr int kScores = 2 * (kD / 16), kSums = 4 * (kD / 32), kAhead = kD <= 32 ? 2 : kD <= 64 ? 3 : 4;      // products of a stage, and how many operands come ahead of theirs
    const int full = wave_first < 0 ? 0 : (wave_first + 1) / kKeys;        // stages whose keys all of the wave's queries see
    const int own = wave_last < 0 ? 0 : wave_last / kKeys + 1, own_end = own < stages ? own : stages;
    Places<kD> places(lds0);
    const auto key_piece = [&](int at, int n) { return places.row_piece(at, 32 * (n & 1), n >> 1); };
    const auto value_piece = [&](int at, int n) { return places.column_piece(2 * kTile + at, 16 * (n / (kD / 32)), n % (kD / 32)); };
    const auto hide = [&](v16f& x, int j, int r, int s) { x[r] = 32 * j + result_row(r) <= last - s * kKeys - 4 * half ? x[r] : -NTC_INF; };

    v16f o[kD / 32] = {}, even[2], odd[2];                 // sums; scores of stages in turn
    // l: the sum of the probabilities as they are rounded, so that what rounding does to all values alike is in the products and in what they are divided by. (lse takes it too: it is off by
    // half a step at most, a probability's own rounding, and by that over the root of the keys as a rule.)
    float m = -NTC_INF, l = 0, most = -NTC_INF;
    const auto stage = [&](int s, v16f (&x)[2], v16f (&z)[2], auto key_at_, auto value_at_, auto masks_, auto more_, auto loads_) {
        constexpr bool kMasks = masks_.value, kMore = more_.value;         // of the next stage, whose scores z will be: they are masked, it is there
        constexpr bool kLoads = loads_.value;                              // the loads are this stage's own
        constexpr int kKeyAt = key_at_.value, kValueAt = value_at_.value;  // where the next stage's keys and this one's values are, from their places
        v4u f[kAhead + 1];
        if constexpr (kMore) {
#pragma unroll
            for (int n = 0; n < kAhead; n++) f[n] = key_piece(kKeyAt, n);
        }
        most = __builtin_fmaxf(most, other_half(most));
        const bool rises = most * d.c > m * d.c + 8.f;     // (m is -inf at first)
        if (__any(rises)) {
            const float next = rises ? most : m, by = m == next ? 1.f : fast_exp2((m - next) * d.c);
            m = next;
            l *= by;
#pragma unroll
            for (int t = 0; t < kD / 32; t++) o[t] *= by;
        }
        const float mc = (m == -NTC_INF ? 0.f : m * d.c) - kLift<T>;
        const char *key_base = nullptr, *value_base = nullptr;
        if constexpr (kLoads) {
            key_base = kp + (long long)(s + 2) * kKeys * d.k.row;
            value_base = vp + (long long)(s + 1) * kKeys * d.v.row;
        }
        uint32_t p[16];
        constexpr int kFirst = 10;                         // pairs of exponentials that lie between the next scores' products; the others lie between the sums'
        const auto exponentials = [&](int e) {             // of a pair
            const float a = fast_exp2(__builtin_fmaf(x[e / 8][2 * e % 16], d.c, -mc)), b = fast_exp2(__builtin_fmaf(x[e / 8][2 * e % 16 + 1], d.c, -mc));
            p[e] = pack2<T>(a, b);
            l = add2<T>(p[e], l);
        };
        if constexpr (kMore) {
            z[0] = z[1] = v16f{};
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < kScores; n++) {
                z[n & 1] = product<T>(f[n % (kAhead + 1)], q[n >> 1], z[n & 1]);
                f[(n + kAhead) % (kAhead + 1)] = n + kAhead < kScores ? key_piece(kKeyAt, n + kAhead) : value_piece(kValueAt, n + kAhead - kScores);
                if constexpr (kLoads) {                    // (keys where this stage's were, values where the last one's)
#pragma unroll
                    for (int i = kPieces * n / kScores; i < kPieces * (n + 1) / kScores; i++) {
                        if (i % 2 == 0) key_loads.piece(lds0 + kValueAt, key_base, i / 2);
                        else value_loads.piece(lds0 + 2 * kTile + kTile - kValueAt, value_base, i / 2);
                    }
                }
#pragma unroll
                for (int e = kFirst * n / kScores; e < kFirst * (n + 1) / kScores; e++) exponentials(e);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int n = 0; n < kAhead; n++) f[(n + kScores) % (kAhead + 1)] = value_piece(kValueAt, n);
#pragma unroll
            for (int e = 0; e < 16; e++) exponentials(e);
        }
        most = -NTC_INF;
#pragma unroll
        for (int n = 0; n < kSums; n++) {
            const int t = n % (kD / 32), h = n / (kD / 32);
            o[t] = product<T>(f[(n + kScores) % (kAhead + 1)], v4u{ p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3] }, o[t]);
            if (n + kAhead < kSums) f[(n + kAhead + kScores) % (kAhead + 1)] = value_piece(kValueAt, n + kAhead);
            if constexpr (kMore) {
                // (the rest of them, due a quarter of the products before theirs)
                constexpr int kRest = 16 - kFirst, kBy = kSums / 2 + kSums / 8;
#pragma unroll
                for (int e = kFirst + kRest * n / kBy; e < 16 && e < kFirst + kRest * (n + 1) / kBy; e++) exponentials(e);
#pragma unroll
                for (int e = 32 * n / kSums; e < 32 * (n + 1) / kSums; e++) {
                    if constexpr (kMasks) hide(z[e / 16], e / 16, e % 16, s + 1);
                    most = __builtin_fmaxf(most, z[e / 16][e % 16]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        asm volatile("" : "+v"(most), "+v"(l));            // (made here: the compiler would sink them behind the next barrier, between nothing)
    };
    if (begin < stages) {
        load_keys(begin);
        arrive();
        load_values(begin);
        if (begin + 1 < stages) load_keys(begin + 1);
        if (begin < own_end) {
            even[0] = even[1] = v16f{};
#pragma unroll
            for (int n = 0; n < kScores; n++) even[n & 1] = product<T>(key_piece(0, n), q[n >> 1], even[n & 1]);
            if (begin >= full) {
#pragma unroll
                for (int e = 0; e < 32; e++) hide(even[e / 16], e / 16, e % 16, begin);
            }
#pragma unroll
            for (int e = 0; e < 32; e++) most = __builtin_fmaxf(most, even[e / 16][e % 16]);
        }
    }
    const auto step = [&](int s) {
        arrive();
        if (s + 1 < stages) load_values(s + 1);
        if (s + 2 < stages) load_keys(s + 2);
    };
    const auto turn = [&] {                                // what was odd is even now
        even[0] = odd[0];
        even[1] = odd[1];
        places.toggle_rows(kTile);
        places.toggle_columns(kTile);
    };
    // (loops of their own, for the compiler: one loop over all kinds of stages moves the sums between registers each time)
    using Here = std::integral_constant<int, 0>;
    using There = std::integral_constant<int, kTile>;
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    int s = begin;
    const int end = full < own_end ? full : own_end;
    const int whole = Lk / kKeys < stages ? Lk / kKeys : stages;
    for (; s + 2 < end && s + 3 < whole; s += 2) {
        arrive();
        stage(s, even, odd, There{}, Here{}, no, yes, yes);
        arrive();
        stage(s + 1, odd, even, Here{}, There{}, no, yes, yes);
    }
    for (; s + 2 < end; s += 2) {
        step(s);
        stage(s, even, odd, There{}, Here{}, no, yes, no);
        step(s + 1);
        stage(s + 1, odd, even, Here{}, There{}, no, yes, no);
    }
    places.toggle_rows(kTile);
    if (s + 1 < end) { step(s); stage(s, even, odd, Here{}, Here{}, no, yes, no); turn(); s++; }
    for (; s + 1 < own_end; s++) { step(s); stage(s, even, odd, Here{}, Here{}, yes, yes, no); turn(); }
    if (s < own_end) { step(s); stage(s, even, odd, Here{}, Here{}, no, no, no); s++; }
    for (; s < stages; s++) step(s);
    l += other_half(l);
    if (last < begin * kKeys) {                            // (sees none of these: whatever keys and values of other rows hold, which probabilities of 0 multiply)
#pragma unroll
        for (int t = 0; t < kD / 32; t++) o[t] = v16f{};
    }
    // A row that sees no key has a sum of 0, and so has one whose scores are all -inf: that one is NaN, as its softmax is. (A part of it has a sum of -1: less than 0 together with others of its kind, 0
    // beside a part that has more.)
    const bool nothing = l == 0 && last >= begin * kKeys && begin < stages;
    const long long at = (qs.row + row.i) * d.q_heads + head * d.group + row.g;
    if (d.parts > 1) {
        const long long own = (long long)part * d.q_rows * d.q_heads + at;
        store_floats<kD>(d.part_sums + own * d.D, o, 1.f, live, d.D);
        if (live && half == 0) d.part_stats[own] = make_float2(m * d.c - kLift<T>, nothing ? -1.f : l);
        return;
    }
    const float f = nothing ? NTC_NAN : l == 0 ? 0.f : 1.f / l;
    store_row<T, kD>((char*)d.out + at * d.D * 2, o, f, live, d.D);
    if (d.rest) store_row<T, kD, true>((char*)d.rest + at * d.D * 2, o, f, live, d.D);
    if (d.lse && live && half == 0) d.lse[at] = nothing ? NTC_NAN : l == 0 ? -NTC_INF : (m * d.c - kLift<T> + fast_log2(l)) * kLn2;
}

// The parts of a row, joined by a wave: a lane takes a part's statistics first, then eight columns of every 64 / kPieces-th part.
template <class T, int kPieces> __global__ void __launch_bounds__(256) k_attention_join(AttentionArgs d) {
    constexpr int kGroups = 64 / kPieces;
    const int lane = lane_id(), piece = lane % kPieces, group = lane / kPieces, col = 8 * piece;
    const long long rows = d.q_rows * d.q_heads, row = block_number() * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const float2 st = lane < d.parts ? d.part_stats[lane * rows + row] : make_float2(-NTC_INF, 0.f);
    const auto larger = [](float a, float b) { return __builtin_fmaxf(a, b); };
    const auto add = [](float a, float b) { return a + b; };
    const float m = reduce64(st.x, larger), by = st.x == m ? 1.f : fast_exp2(st.x - m);                          // (no key at all: m is -inf, and what the part has is 0)
    const float l = reduce64(st.y * by, add);
    float sum[8] = {};
#pragma unroll 4
    for (int p0 = 0; p0 < d.parts; p0 += kGroups) {
        const int p = p0 + group;
        const float w = __shfl(by, p & 63);
        if (p >= d.parts || col >= d.D) continue;
        const float4 *of = (const float4*)(d.part_sums + (p * rows + row) * d.D + col), a = of[0], b = of[1];
        const float v[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] = __builtin_fmaf(v[i], w, sum[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int g = kPieces; g < 64; g *= 2) sum[i] += __shfl_xor(sum[i], g);
    if (group || col >= d.D) return;
    const float f = l < 0 ? NTC_NAN : l == 0 ? 0.f : 1.f / l;
    uint32_t out[4], rest[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y0 = sum[2 * i] * f, y1 = sum[2 * i + 1] * f;
        out[i] = pack2<T>(y0, y1);
        rest[i] = pack2<T>((y0 - (float)(T)y0) * kRest<T>, (y1 - (float)(T)y1) * kRest<T>);
    }
    const long long at = 2 * (row * d.D + col);
    *(v4u*)((char*)d.out + at) = v4u{ out[0], out[1], out[2], out[3] };
    if (d.rest) *(v4u*)((char*)d.rest + at) = v4u{ rest[0], rest[1], rest[2], rest[3] };
    if (d.lse && col == 0) d.lse[row] = l < 0 ? NTC_NAN : l == 0 ? -NTC_INF : (m + fast_log2(l)) * kLn2;
}

// ---------------------------------------------------------------- backward
// float16: the score's gradients, and probabilities of long rows, leave its range. They are multiplied by powers of two: probabilities by 2^14, the score's
// gradients by the largest that keeps 2 D max|dO| max|v|, which they cannot pass, within 2^15: for dq of the row's dO and its sequence's v, for dk of the sequence's both, so that what other sequences
// hold (and for dq, other rows' dO) does not decide what is left of them. A block takes the largest value of kExtentRows rows of v (first) or dO; who needs a sequence's joins its blocks'.
template <class T> __global__ void __launch_bounds__(256) k_attention_extent(AttentionArgs d) {
    __shared__ float parts[4];
    float to = 0;
    const unsigned pieces = d.D / 8;
    const long long block = block_number();
    const bool of_v = block < d.v_extents;
    const int number = (int)(of_v ? block : block - d.v_extents);
    if (!of_v && number >= d.do_extents) return;
    int tile;
    const int* cu = of_v ? d.cu_k : d.cu_q;
    const int b = find_sequence<kExtentRows>(cu, d.sequences, of_v ? d.v_extents_each : d.do_extents_each, 1, number, tile);
    if (b < d.sequences && tile >= 0) {
        const Operand3& of = of_v ? d.v : d.d_o;
        const Span span = of_v ? span_of(cu, d.sequences, d.k_each, d.k_rows, b, of) : span_of(cu, d.sequences, d.q_each, d.q_rows, b, of);
        const unsigned heads = of_v ? d.k_heads : d.q_heads;
        const long long left = (long long)(of_v ? keys_of(d, span) : span.n) - (long long)tile * kExtentRows;
        const unsigned all = (unsigned)cut(left, 0, kExtentRows) * heads * pieces;
        const char* p = of.p + span.start + (long long)tile * kExtentRows * of.row;
        typedef T v8 __attribute__((ext_vector_type(8)));
        for (unsigned x0 = threadIdx.x; x0 < all; x0 += 1024) {               // four loads of a thread on their way together
            v8 x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const unsigned own = x0 + 256 * k < all ? x0 + 256 * k : x0, y = own / pieces, r = y / heads;
                x[k] = *(const v8*)(p + r * of.row + (y - r * heads) * of.head + (own - y * pieces) * 16);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 8; i++) to = __builtin_fmaxf(to, __builtin_fabsf((float)x[k][i]));
        }
    }
    const auto most = [](float a, float b) { return __builtin_fmaxf(a, b); };
    to = reduce64(to, most);
    if (lane_id() == 0) parts[threadIdx.x >> 6] = to;
    __syncthreads();
    if (threadIdx.x == 0) (of_v ? d.extents_v : d.extents_do)[number] = most(most(parts[0], parts[1]), most(parts[2], parts[3]));
}
// A sequence's largest |v| (of n rows) or |dO|
__device__ __forceinline__ float extent_of(const float* extents, int first, int n) {
    float most = 0;
    for (int i = lane_id(); i < (n + kExtentRows - 1) / kExtentRows; i += 64) most = __builtin_fmaxf(most, extents[first + i]);
    return reduce64(most, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float extent_of_v(const AttentionArgs& d, int b, int n) { return extent_of(d.extents_v, first_tile<kExtentRows>(d.cu_k, d.v_extents_each, 1, b), n); }
__device__ __forceinline__ float extent_of_do(const AttentionArgs& d, int b, int n) { return extent_of(d.extents_do, first_tile<kExtentRows>(d.cu_q, d.do_extents_each, 1, b), n); }
// The power of two for the scores' gradients, as an exponent.
__device__ __forceinline__ int gradient_exponent(const AttentionArgs& d, float v, float d_o) {
    const float bound = 2.f * d.D * v * d_o;
    if (!(bound > 0) || bound > 3e38f) return 0;
    const int e = 14 - (int)((__float_as_uint(bound) >> 23) - 127);
    return e < -60 ? -60 : e > 60 ? 60 : e;
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }
template <class T> constexpr int kShift = std::is_same_v<T, f16> ? 14 : 0;      // probabilities are held times 2^kShift

// A row's dS add up to 0; rounded, they do not quite, and neither where the sum dO o is that of rounded probabilities. What they add up to, times a vector that is near
// the row's keys, is taken off: the error of dq is then one of the keys' differences from it, and keys with much in common keep their gradients' precision. The vector
// is the mean of the first stage's keys as the row weighs them (for a row that sees few keys, of all of them), and waits in dq's own place meanwhile. 1000 rows, keys of deviation 1 about a common mean of
// deviation 0, 1, 4 and 16, bfloat16: dq is off by 2.3e-3 of its size with any; without, by 2.4e-3, 3.1e-3, 8.8e-3 and 3.6e-2, in the same time.
// Rows as forward; three products for each key and row. 8192 tokens of 16 heads on 4 of 128, causal: 460 to 560 us, 740 to 900 TFLOP/s (the clock that a card's power leaves).
template <class T, int kD, bool kParts> __global__ void __launch_bounds__(256, kD <= 32 ? 4 : 2) k_attention_dq(AttentionArgs d) {
    using L = Tile<kD>;
    constexpr int kTile = kKeys * L::kPitch;
    __shared__ alignas(2 * kTile) char lds[4 * kTile];     // keys, values; two of each
    const BlockPlace own_place = place_of(d);
    const int head = own_place.head, part = kParts ? own_place.part : 0;
    const unsigned number = own_place.number;
    if (number >= (unsigned)d.tiles) return;
    int tile;
    const int b = find_sequence<kRows>(d.cu_q, d.sequences, d.tiles_each, d.group, d.tiles - 1 - (int)number, tile);
    const Span qs = span_of(d.cu_q, d.sequences, d.q_each, d.q_rows, b, d.q);
    const long long rows = (long long)qs.n * d.group;
    if (tile < 0 || (long long)tile * kRows >= rows) return;
    const int kb = b < d.sequences ? b : 0;
    Span ks = span_of(d.cu_k, d.sequences, d.k_each, d.k_rows, kb, d.k);
    const int Lk = b < d.sequences ? keys_of(d, ks) : 0, off = Lk - qs.n;
    const long long v_start = d.cu_k ? ks.row * d.v.row : ks.b * d.v.batch, do_start = d.cu_q ? qs.row * d.d_o.row : qs.b * d.d_o.batch;

    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), column = lane & 31, half = lane >> 5;
    const int r0 = tile * kRows + 32 * wave, i0 = r0 / d.group, g0 = r0 - i0 * d.group;
    const Row row = row_at(d, i0, g0, column);
    const bool live = row.i < qs.n;
    const int h = head * d.group + row.g;
    const long long at = (qs.row + row.i) * d.q_heads + h;
    v4u q[kD / 16], g[kD / 16];
    float delta = 0;
    {
        v4u o[kD / 16], rest[kD / 16];
        load_row<kD>(o, (const char*)d.out + at * d.D * 2, live, d.D);
        load_row<kD>(rest, (const char*)d.rest + at * d.D * 2, live, d.D);
        load_row<kD>(g, d.d_o.p + do_start + row.i * d.d_o.row + h * d.d_o.head, live, d.D);
        typedef T v8 __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int s = 0; s < kD / 16; s++) {
            const v8 a = __builtin_bit_cast(v8, o[s]), r = __builtin_bit_cast(v8, rest[s]), c = __builtin_bit_cast(v8, g[s]);
#pragma unroll
            for (int i = 0; i < 8; i++) delta = __builtin_fmaf(__builtin_fmaf((float)r[i], 1 / kRest<T>, (float)a[i]), (float)c[i], delta);
        }
    }
    load_row<kD>(q, d.q.p + qs.start + row.i * d.q.row + h * d.q.head, live, d.D);
    delta += other_half(delta);
    const float lse = live ? d.lse[at] * kLog2e : 0.f;
    int e = 0, e_sequence = 0;                             // of the row, and of its sequence
    if constexpr (std::is_same_v<T, f16>) {
        typedef T v8 __attribute__((ext_vector_type(8)));
        float most = 0;
#pragma unroll
        for (int s = 0; s < kD / 16; s++) {
            const v8 c = __builtin_bit_cast(v8, g[s]);
#pragma unroll
            for (int i = 0; i < 8; i++) most = __builtin_fmaxf(most, __builtin_fabsf((float)c[i]));
        }
        const float of_v = extent_of_v(d, b, Lk);
        e = gradient_exponent(d, of_v, __builtin_fmaxf(most, other_half(most)));
        e_sequence = gradient_exponent(d, of_v, extent_of_do(d, b, qs.n));
    }
    const float lse_up = lse - (float)e;                   // (2^e goes into the exponential: its argument is off by 2^-18 then)
    if (live && half == 0 && part == 0) {                               // as the keys' and values' gradients take them
        d.log_sums[at] = lse - kShift<T>;
        d.deltas[at] = delta * two_to(e_sequence) * two_to(-kShift<T>);
    }
    const int i_wave = (r0 + 31) / d.group, i_block = (tile * kRows + kRows - 1) / d.group;
    const int block_last = d.causal ? (i_block + off < Lk - 1 ? i_block + off : Lk - 1) : Lk - 1;
    const int all_stages = block_last < 0 || !d.dq ? 0 : block_last / kKeys + 1, each_stages = kParts ? (all_stages + d.parts - 1) / d.parts : all_stages;
    const int from = kParts ? min(part * each_stages, all_stages) : 0, stages = min(each_stages, all_stages - from), base = from * kKeys;
    // (the part's first key is number 0 from here on)
    const int Lp = Lk - base, top = Lp - 1, last = d.causal ? min(row.i + off - base, top) : top;
    const int wave_first = d.causal ? min(i0 + off - base, top) : top, wave_last = d.causal ? min(i_wave + off - base, top) : top;

    const char *kp = d.k.p + ks.start + head * d.k.head + (long long)base * d.k.row, *vp = d.v.p + v_start + head * d.v.head + (long long)base * d.v.row;
    const uint32_t lds0 = lds_address(lds);
    const RowLoads<kD, kKeys> key_loads(d.k.row, d.D), value_loads(d.v.row, d.D);
    const auto load = [&](int s) {
        key_loads.load(lds0 + (s & 1) * kTile, kp + (long long)s * kKeys * d.k.row, Lp - s * kKeys);
        value_loads.load(lds0 + (2 + (s & 1)) * kTile, vp + (long long)s * kKeys * d.v.row, Lp - s * kKeys);
    };
    const Places<kD> places(lds0);
    v16f dq[kD / 32] = {};
    float sum = 0;
    const auto none = [&] {                                // (a row that sees no key of these: as forward)
        if (last < 0) {
#pragma unroll
            for (int t = 0; t < kD / 32; t++) dq[t] = v16f{};
        }
    };
    constexpr int kScores = 2 * (kD / 16), kSums = 2 * (kD / 32), kAhead = 3;
    constexpr bool kBetween = kD <= 96;                    // (a wave's registers do not hold both halves of wider heads: 643 us where one after the other is 470; one wave to a SIMD, which has them, 595 where that is 560)
    // a stage at `at` in shared memory, in halves of 32 keys: the second half's scores are made between the first one's exponentials, the first one's sums between the second's
    const auto stage = [&](int s, auto at_, auto masks_) {
        constexpr int kAt = at_.value;
        constexpr bool kMasks = masks_.value;
        const auto row_piece = [&](int j, int n) { return places.row_piece(kAt + 2 * kTile * (n & 1), 32 * j, n >> 1); };        // keys and values in turn
        const auto column_piece = [&](int j, int n) { return places.column_piece(kAt, 32 * j + 16 * (n / (kD / 32)), n % (kD / 32)); };
        v4u p[2][2];
        const int seen = last - s * kKeys - 4 * half;
        const auto gradient = [&](const v16f& a, const v16f& c, int j, int r) {
            const float exponent = __builtin_fmaf(a[r], d.c, -lse_up), z = c[r] - delta;
            const bool in = !kMasks || 32 * j + result_row(r) <= seen;
            return fast_exp2(in ? exponent : -NTC_INF) * (in ? z : 0.f);
        };
        // n of `of` parts of a half's gradients, two at a time
        const auto gradients = [&](const v16f& a, const v16f& c, int j, int n, int of) {
#pragma unroll
            for (int r = 8 * n / of; r < 8 * (n + 1) / of; r++) {
                const uint32_t w = pack2<T>(gradient(a, c, j, 2 * r), gradient(a, c, j, 2 * r + 1));
                p[j][r / 4][r % 4] = w;
                sum = add2<T>(w, sum);
            }
        };
        v16f x = {}, y = {}, x2 = {}, y2 = {};
        v4u f[kAhead + 1];
#pragma unroll
        for (int n = 0; n < kAhead; n++) f[n] = row_piece(0, n);
        if constexpr (kD > 32) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 2 * kScores; n++) {
            const int m = n % kScores;
            if (n < kScores) { if (m & 1) y = product<T>(f[n % (kAhead + 1)], g[m >> 1], y); else x = product<T>(f[n % (kAhead + 1)], q[m >> 1], x); }
            else { if (m & 1) y2 = product<T>(f[n % (kAhead + 1)], g[m >> 1], y2); else x2 = product<T>(f[n % (kAhead + 1)], q[m >> 1], x2); }
            const int k = n + kAhead;
            f[k % (kAhead + 1)] = k < 2 * kScores ? row_piece(k / kScores, k % kScores) : column_piece(0, k - 2 * kScores);
            if (n >= kScores) gradients(x, y, 0, m, kScores);
            if constexpr (kD > 32) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < 2 * kSums; n++) {
            const int j = n / kSums, m = n % kSums, t = m % (kD / 32), a = m / (kD / 32), k = n + kAhead;
            dq[t] = product<T>(f[(n + 2 * kScores) % (kAhead + 1)], p[j][a], dq[t]);
            if (k < 2 * kSums) f[(k + 2 * kScores) % (kAhead + 1)] = column_piece(k / kSums, k % kSums);
            if (n < kSums) gradients(x2, y2, 1, n, kSums);
            if constexpr (kD > 32) __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" : "+v"(sum));
    };
    const auto step = [&](int s) {
        arrive();
        if (s + 1 < stages) load(s + 1);
    };
    const int full = wave_first < 0 ? 0 : (wave_first + 1) / kKeys, own = wave_last < 0 ? 0 : wave_last / kKeys + 1, own_end = own < stages ? own : stages, end = full < own_end ? full : own_end;
    using Here = std::integral_constant<int, 0>;
    using There = std::integral_constant<int, kTile>;
    if (stages) {
        load(0);
        step(0);
        if (own_end > 0 && part == 0) {
            v16f x[2] = {};
            float weight = 0;
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int i = 0; i < kD / 16; i++) x[j] = product<T>(places.row_piece(0, 32 * j, i), q[i], x[j]);
#pragma unroll
                for (int r = 0; r < 16; r++) x[j][r] = fast_exp2(32 * j + result_row(r) <= last - 4 * half ? __builtin_fmaf(x[j][r], d.c, kShift<T> - lse) : -NTC_INF);
            }
#pragma unroll
            for (int h4 = 0; h4 < 4; h4++) {
                const v4u w = packed<T>(x[h4 / 2], h4 & 1);
                weight = add2<T>(w.w, add2<T>(w.z, add2<T>(w.y, add2<T>(w.x, weight))));
#pragma unroll
                for (int t = 0; t < kD / 32; t++) dq[t] = product<T>(places.column_piece(0, 16 * h4, t), w, dq[t]);
            }
            weight += other_half(weight);
            none();
            store_row<T, kD>((char*)d.dq + at * d.D * 2, dq, weight > 0 ? 1.f / weight : 0.f, live, d.D);
#pragma unroll
            for (int t = 0; t < kD / 32; t++) dq[t] = v16f{};
        }
    }
    int s = 0;
    if constexpr (!kBetween) {
        for (; s < own_end; s++) {
            if (s) step(s);
            const int at = (s & 1) * kTile;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                v16f x = {}, y = {};
#pragma unroll
                for (int i = 0; i < kD / 16; i++) x = product<T>(places.row_piece(at, 32 * j, i), q[i], x);
#pragma unroll
                for (int i = 0; i < kD / 16; i++) y = product<T>(places.row_piece(at + 2 * kTile, 32 * j, i), g[i], y);
#pragma unroll
                for (int r = 0; r < 16; r++) x[r] = fast_exp2(__builtin_fmaf(x[r], d.c, -lse_up)) * (y[r] - delta);
                if (s * kKeys + 32 * j + 31 > wave_first) {
                    const int seen = last - s * kKeys - 32 * j - 4 * half;
#pragma unroll
                    for (int r = 0; r < 16; r++) x[r] = result_row(r) <= seen ? x[r] : 0.f;
                }
#pragma unroll
                for (int a = 0; a < 2; a++) {
                    const v4u p = packed<T>(x, a);
                    sum = add2<T>(p.w, add2<T>(p.z, add2<T>(p.y, add2<T>(p.x, sum))));
#pragma unroll
                    for (int t = 0; t < kD / 32; t++) dq[t] = product<T>(places.column_piece(at, 32 * j + 16 * a, t), p, dq[t]);
                }
            }
        }
    } else {
        for (; s + 1 < end; s += 2) {
            if (s) step(s);
            stage(s, Here{}, std::false_type{});
            step(s + 1);
            stage(s + 1, There{}, std::false_type{});
        }
        if (s < end) {
            if (s) step(s);
            stage(s, Here{}, std::false_type{});
            s++;
        }
        for (; s < own_end; s++) {
            if (s) step(s);
            if (s & 1) stage(s, There{}, std::true_type{});
            else stage(s, Here{}, std::true_type{});
        }
    }
    for (; s < stages; s++) if (s) step(s);
    sum += other_half(sum);
    none();
    if (kParts) {
        const long long all = d.q_rows * d.q_heads;
        store_floats<kD>(d.part_sums + (part * all + at) * d.D, dq, two_to(-e), live, d.D);
        if (live && half == 0) d.part_rests[part * all + at] = sum * two_to(-e);
        if (own_end == 0 && part == 0) store_row<T, kD>((char*)d.dq + at * d.D * 2, dq, 0.f, live, d.D);
        return;
    }
    if (own_end > 0 && live) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");             // (the vector was written by other lanes of the wave)
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        typedef T v4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int t = 0; t < kD / 32; t++)
#pragma unroll
            for (int a = 0; a < 4; a++) {
                const int col = 32 * t + 8 * a + 4 * half;
                const v4 near = col < d.D ? *(const v4*)((const char*)d.dq + (at * d.D + col) * 2) : v4{};
#pragma unroll
                for (int i = 0; i < 4; i++) dq[t][4 * a + i] = __builtin_fmaf(-sum, (float)near[i], dq[t][4 * a + i]);
            }
    }
    store_row<T, kD>((char*)d.dq + at * d.D * 2, dq, d.scale * two_to(-e), live && d.dq, d.D);
}

// The parts of dq added up, and what the vector near the keys takes off: eight columns to a thread.
template <class T> __global__ void __launch_bounds__(256) k_attention_dq_join(AttentionArgs d) {
    const long long rows = d.q_rows * d.q_heads, n = rows * d.D / 8, x = block_number() * 256 + threadIdx.x;
    if (x >= n) return;
    const long long row = x / (d.D / 8);
    char* to = (char*)d.dq + 16 * x;
    float sum[8] = {}, rest = 0;
#pragma unroll 4
    for (int p = 0; p < d.parts; p++) {
        const float4 *of = (const float4*)(d.part_sums + 8 * (p * n + x)), a = of[0], b = of[1];
        const float v[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += v[i];
        rest += d.part_rests[p * rows + row];
    }
    typedef T v8 __attribute__((ext_vector_type(8)));
    const v8 near = *(const v8*)to;
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = pack2<T>(__builtin_fmaf(-rest, (float)near[2 * i], sum[2 * i]) * d.scale, __builtin_fmaf(-rest, (float)near[2 * i + 1], sum[2 * i + 1]) * d.scale);
    *(v4u*)to = v4u{ out[0], out[1], out[2], out[3] };
}

// Keys and values of 32 columns a wave stay in registers, rows come 64 at a time, in steps of 32. While a step's probabilities and gradients are made and summed up with its
// rows' columns, the next step's scores are. With heads of 128 a wave has its SIMD to itself (404 registers): the order of its instructions is what keeps the units busy.
// Four products for each key and row. 8192 tokens of 16 heads on 4 of 128, causal, in two parts: 615 to 632 us, 870 to 895 TFLOP/s, and 14 for the parts' sum; 423 with LDS reads, exponentials and loads taken out.
template <class T, int kD> __global__ void __launch_bounds__(256, kD > 64 ? 1 : kD > 32 ? 2 : 3) k_attention_dkv(AttentionArgs d) {
    using L = Tile<kD>;
    constexpr int kStep = 64, kTile = kStep * L::kPitch, kBuffer = 2 * kTile, kBuffers = 3;
    __shared__ alignas(16) char lds[kBuffers * (kBuffer + 8 * kStep)];     // queries and gradients of kStep rows, three of each; then their log sums and deltas
    const BlockPlace own_place = place_of(d);
    const int head = own_place.head, part = own_place.part;
    const unsigned number = own_place.number;
    if (number >= (unsigned)d.tiles) return;
    int tile;
    const int b = find_sequence<kRows>(d.cu_k, d.sequences, d.tiles_each, 1, (int)number, tile);                      // (a sequence's first keys, which most queries see, first)
    const Span ks = span_of(d.cu_k, d.sequences, d.k_each, d.k_rows, b, d.k);
    if (tile < 0 || (long long)tile * kRows >= ks.n) return;
    const bool none = b >= d.sequences;
    const int Lk = none ? 0 : keys_of(d, ks);
    Span qs = span_of(d.cu_q, d.sequences, d.q_each, d.q_rows, none ? 0 : b, d.q);
    if (none) qs.n = 0;
    const int off = Lk - qs.n;
    const long long v_start = d.cu_k ? ks.row * d.v.row : ks.b * d.v.batch, do_start = d.cu_q ? qs.row * d.d_o.row : qs.b * d.d_o.batch;

    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), column = lane & 31, half = lane >> 5;
    const int k0 = tile * kRows + 32 * wave, key = k0 + column;
    const bool held = key < ks.n, live = key < Lk;
    v4u k[kD / 16], v[kD / 16];
    load_row<kD>(k, d.k.p + ks.start + key * d.k.row + head * d.k.head, live, d.D);
    load_row<kD>(v, d.v.p + v_start + key * d.v.row + head * d.v.head, live, d.D);
    int e = 0;
    if constexpr (std::is_same_v<T, f16>) if (qs.n) e = uniform(gradient_exponent(d, extent_of_v(d, b, Lk), extent_of_do(d, b, qs.n)));      // (without queries nothing has left them)
    const float up = two_to(e) * two_to(-kShift<T>);

    // Row r sees key j where r >= (j - off) G: the lane's first row, the wave's first whole one, and where wave and block start
    const int rows = qs.n * d.group;
    const auto first_row = [&](int j) { return d.causal && j > off ? (j - off) * d.group : 0; };
    const int lane_first = live ? first_row(key) : 1 << 30, wave_first = k0 + 31 < Lk ? first_row(k0 + 31) : 1 << 30;
    const int end = tile * kRows < Lk ? (rows + kStep - 1) / kStep : 0, first = end ? first_row(tile * kRows) / kStep : 0, all = end > first ? end - first : 0;
    const int start = first + (d.parts == 1 ? 0 : all * part / d.parts), stages = first + (d.parts == 1 ? all : all * (part + 1) / d.parts);
    const int wave_start = k0 < Lk ? first_row(k0) / kStep : stages, own = wave_start > start ? wave_start : start;

    const char *qp = d.q.p + qs.start + head * d.group * d.q.head, *gp = d.d_o.p + do_start + head * d.group * d.d_o.head;
    const long long at0 = qs.row * d.q_heads + head * d.group;
    const uint32_t lds0 = lds_address(lds);
    using RowsLoad = Loads<kD, kStep>;
    // a row's place: x rows after head g0 of a query
    const auto place = [&](int g0, int x, long long row, long long head_) {
        const Row r = row_at(d, 0, g0, x);
        return (uint32_t)r.i * (uint32_t)row + (uint32_t)r.g * (uint32_t)head_;
    };
    const int each = kStep / d.group;
    const bool whole = each * d.group == kStep;            // every stage starts with a query: its rows' places are the same each time
    uint32_t q_off[RowsLoad::kEach], g_off[RowsLoad::kEach], sum_off;
#pragma unroll
    for (int i = 0; i < RowsLoad::kEach; i++) {
        q_off[i] = place(0, RowsLoad::row(i), d.q.row, d.q.head) + RowsLoad::byte(i, d.D);
        g_off[i] = place(0, RowsLoad::row(i), d.d_o.row, d.d_o.head) + RowsLoad::byte(i, d.D);
    }
    sum_off = place(0, lane, 4ll * d.q_heads, 4);
    int to_buffer = 0;                                     // of the next load
    const auto load = [&](int s) {
        const int r0 = s * kStep, n = rows - r0, i0 = whole ? s * each : r0 / d.group, g0 = r0 - i0 * d.group;
        const uint32_t to = lds0 + to_buffer * kBuffer, to_sums = lds0 + kBuffers * kBuffer + to_buffer * 8 * kStep + 4 * kStep * wave;
        const char *qb = qp + i0 * d.q.row, *gb = gp + i0 * d.d_o.row, *sums = (const char*)((wave ? d.deltas : d.log_sums) + at0 + (long long)i0 * d.q_heads);
        if (whole && n >= kStep) {
            RowsLoad::run(to, qb, [&](int i) { return q_off[i]; });
            RowsLoad::run(to + kTile, gb, [&](int i) { return g_off[i]; });
            if (wave < 2) to_lds4(to_sums, sum_off, sums);
        } else {                                           // past the end the last one again
            const auto row = [&](int r) { return r < n ? r : n - 1; };
            RowsLoad::run(to, qb, [&](int i) { return place(g0, row(RowsLoad::row(i)), d.q.row, d.q.head) + RowsLoad::byte(i, d.D); });
            RowsLoad::run(to + kTile, gb, [&](int i) { return place(g0, row(RowsLoad::row(i)), d.d_o.row, d.d_o.head) + RowsLoad::byte(i, d.D); });
            if (wave < 2) to_lds4(to_sums, place(g0, row(lane), 4ll * d.q_heads, 4), sums);
        }
        to_buffer = to_buffer == kBuffers - 1 ? 0 : to_buffer + 1;
    };

    Places<kD> places(lds0);                               // rows: of the buffer of the next step; columns and sums: of this one's
    uint32_t at_sums = lds0 + kBuffers * kBuffer + 16 * half;
    constexpr int kScores = 2 * (kD / 16), kSums = 4 * (kD / 32), kAhead = 3;
    constexpr bool kNext = kD > 32;                     // the next step's scores are made between this one's exponentials (not where these outweigh the products: several waves take turns then)
    const auto row_piece = [&](int j, int n) { return places.row_piece((n & 1) * kTile, 32 * j, n >> 1); };                 // queries and gradients in turn
    const auto column_piece = [&](int j, int n) {                                                                          // gradients for dv, then queries for dk
        const int m = n % (kSums / 2);
        return places.column_piece(n < kSums / 2 ? kTile : 0, 32 * j + 16 * (m / (kD / 32)), m % (kD / 32));
    };
    typedef float v4f __attribute__((ext_vector_type(4)));
    const auto sums_of = [&](int which, int j, int a) { return *(__attribute__((address_space(3))) const v4f*)((Shared)at_sums + (4 * kStep * which + 128 * j + 32 * a)); };
    v16f dk[kD / 32] = {}, dv[kD / 32] = {}, x, y;         // x, y: scores and dO v of the step
    const auto scores = [&](int j, v16f& to_x, v16f& to_y) {
        to_x = to_y = v16f{};
#pragma unroll
        for (int n = 0; n < kScores; n++) {
            if (n & 1) to_y = product<T>(row_piece(j, n), v[n >> 1], to_y);
            else to_x = product<T>(row_piece(j, n), k[n >> 1], to_x);
        }
    };
    constexpr int kPieces = 2 * RowsLoad::kEach;           // loads of a stage, which the first step of one issues between its products where it can
    // step j of the stage from row r0 on; the next step's rows are the places' rows from row 32 `next` on
    const auto step = [&](int r0, auto j_, auto masks_, auto loads_) {
        constexpr int j = j_.value, next = 1 - j;
        constexpr bool kMasks = masks_.value, kLoads = loads_.value;
        uint32_t to = 0;
        const char *qb = nullptr, *gb = nullptr;
        if constexpr (kLoads) {
            const int i0 = (r0 / kStep + 2) * each;
            to = lds0 + to_buffer * kBuffer + 1024 * (wave * RowsLoad::kEach);
            qb = qp + i0 * d.q.row;
            gb = gp + i0 * d.d_o.row;
            if (wave < 2) to_lds4(lds0 + kBuffers * kBuffer + to_buffer * 8 * kStep + 4 * kStep * wave, sum_off, (const char*)((wave ? d.deltas : d.log_sums) + at0 + (long long)i0 * d.q_heads));
            to_buffer = to_buffer == kBuffers - 1 ? 0 : to_buffer + 1;
        }
        v4u f[kAhead + 1];
        v4f sum[4], delta[4];
        v16f p, x2 = {}, y2 = {};
        const int lo = lane_first - r0 - 32 * j - 4 * half, hi = rows - r0 - 32 * j - 4 * half;
        const auto seen = [&](int r) { return result_row(r) >= lo && result_row(r) < hi; };
        v4u pp[2], zz[2];
        if constexpr (kNext) {
#pragma unroll
            for (int i = 0; i < kAhead; i++) f[i] = row_piece(next, i);
        } else scores(j, x, y);
#pragma unroll
        for (int a = 0; a < 4; a++) sum[a] = sums_of(0, j, a);
#pragma unroll
        for (int a = 0; a < 4; a++) delta[a] = sums_of(1, j, a);
        if constexpr (kNext) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kScores; n++) {
            if (!kNext) f[(n + kAhead) % (kAhead + 1)] = n + kAhead < kScores ? v4u{} : column_piece(j, n + kAhead - kScores);
            else if (n & 1) y2 = product<T>(f[n % (kAhead + 1)], v[n >> 1], y2);
            else x2 = product<T>(f[n % (kAhead + 1)], k[n >> 1], x2);
            if (kNext) f[(n + kAhead) % (kAhead + 1)] = n + kAhead < kScores ? row_piece(next, n + kAhead) : column_piece(j, n + kAhead - kScores);
            if constexpr (kLoads) {
#pragma unroll
                for (int i = kPieces * n / kScores; i < kPieces * (n + 1) / kScores; i++) {
                    if (i % 2 == 0) to_lds16(to + 1024 * (i / 2), q_off[i / 2], qb);
                    else to_lds16(to + kTile + 1024 * (i / 2), g_off[i / 2], gb);
                }
            }
#pragma unroll
            for (int r = 16 * n / kScores; r < 16 * (n + 1) / kScores; r++) {
                const float exponent = __builtin_fmaf(x[r], d.c, -sum[r / 4][r % 4]);
                p[r] = fast_exp2(!kMasks || seen(r) ? exponent : -NTC_INF);
                if (r % 8 == 7) pp[r / 8] = packed<T>(p, r / 8);
            }
            if constexpr (kNext) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < kSums; n++) {
            const int m = n % (kSums / 2), t = m % (kD / 32), a = m / (kD / 32);
            if (n < kSums / 2) dv[t] = product<T>(f[(n + kScores) % (kAhead + 1)], pp[a], dv[t]);
            else dk[t] = product<T>(f[(n + kScores) % (kAhead + 1)], zz[a], dk[t]);
            if (n + kAhead < kSums) f[(n + kAhead + kScores) % (kAhead + 1)] = column_piece(j, n + kAhead);
            if (n < kSums / 2) {
#pragma unroll
                for (int r = 16 * n / (kSums / 2); r < 16 * (n + 1) / (kSums / 2); r++) {
                    const float z = __builtin_fmaf(y[r], up, -delta[r / 4][r % 4]);
                    p[r] *= !kMasks || seen(r) ? z : 0.f;
                    if (r % 8 == 7) zz[r / 8] = packed<T>(p, r / 8);
                }
            }
            if constexpr (kNext) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (kNext) { x = x2; y = y2; }
    };
    int buffer = 0;
    const auto stage = [&](int s, auto masks, auto loads) {
        using First = std::integral_constant<int, 0>;
        using Second = std::integral_constant<int, 1>;
        step(s * kStep, First{}, masks, loads);
        const int on = buffer == kBuffers - 1 ? -(kBuffers - 1) : 1;
        if constexpr (!kNext) step(s * kStep, Second{}, masks, std::false_type{});
#pragma unroll
        for (uint32_t& at : places.row) at += on * kBuffer;
        if constexpr (kNext) step(s * kStep, Second{}, masks, std::false_type{});
#pragma unroll
        for (auto& at : places.column) { at[0] += on * kBuffer; at[1] += on * kBuffer; }
        at_sums += on * 8 * kStep;
        buffer += on;
    };
    // a stage's rows are free once every wave is past it, which the next but one's barrier says: three buffers
    const auto turn = [&](int s) {
        arrive();
        if (s + 2 < stages) load(s + 2);
    };
    if (start < stages) {
        load(start);
        if (start + 1 < stages) load(start + 1);
    }
    int s = start;
    for (; s < own && s < stages; s++) {                   // (no row of these sees a key of the wave)
        turn(s);
        const int on = buffer == kBuffers - 1 ? -(kBuffers - 1) : 1;
#pragma unroll
        for (uint32_t& at : places.row) at += on * kBuffer;
#pragma unroll
        for (auto& at : places.column) { at[0] += on * kBuffer; at[1] += on * kBuffer; }
        at_sums += on * 8 * kStep;
        buffer += on;
    }
    if (s < stages) {
        turn(s);
        if constexpr (kNext) scores(0, x, y);
        const int clear = (wave_first + kStep - 1) / kStep, tail = rows / kStep;          // stages from `clear` up to `tail` need no mask
        bool arrived = true;
        while (s < stages) {
            for (; s < stages && (s < clear || s >= tail); s++) {
                if (!arrived) turn(s);
                arrived = false;
                stage(s, std::true_type{}, std::false_type{});
            }
            if (whole && kNext) {
                if (arrived && s + 2 < stages && s >= clear && s + 2 < tail) { stage(s, std::false_type{}, std::false_type{}); s++; arrived = false; }
                for (; s + 2 < stages && s >= clear && s + 2 < tail; s++) {
                    arrive();
                    stage(s, std::false_type{}, std::true_type{});
                }
            }
            for (; s < stages && s >= clear && s < tail; s++) {
                if (!arrived) turn(s);
                arrived = false;
                stage(s, std::false_type{}, std::false_type{});
            }
        }
    }
    if (!live) {
#pragma unroll
        for (int t = 0; t < kD / 32; t++) { dk[t] = v16f{}; dv[t] = v16f{}; }
    }
    const long long at = (ks.row + key) * d.k_heads + head;
    if (d.parts > 1) {
        const long long each = d.k_rows * d.k_heads;
        store_floats<kD>(d.part_sums + (part * each + at) * d.D, dk, two_to(-e), held, d.D);
        store_floats<kD>(d.part_sums + ((d.parts + part) * each + at) * d.D, dv, 1.f, held, d.D);
        return;
    }
    store_row<T, kD>((char*)d.dk + at * d.D * 2, dk, d.scale * two_to(-e), held && d.dk, d.D);
    store_row<T, kD>((char*)d.dv + at * d.D * 2, dv, two_to(-kShift<T>), held && d.dv, d.D);
}

// The parts of dk (dv: second half of the grid) added up: eight columns to a thread.
template <class T> __global__ void __launch_bounds__(256) k_attention_sum(AttentionArgs d) {
    const long long n = d.k_rows * d.k_heads * d.D / 8, x = block_number() * 256 + threadIdx.x;
    if (x >= 2 * n) return;
    const int which = x >= n;
    const float f = which ? two_to(-kShift<T>) : d.scale;
    const long long at = 8 * (which ? x - n : x);
    char* to = (char*)(which ? d.dv : d.dk);
    if (!to) return;
    float sum[8] = {};
#pragma unroll 4
    for (int p = 0; p < d.parts; p++) {
        const float4 *of = (const float4*)(d.part_sums + 8 * n * (which * d.parts + p) + at), a = of[0], b = of[1];
        const float v[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += v[i];
    }
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = pack2<T>(sum[2 * i] * f, sum[2 * i + 1] * f);
    *(v4u*)(to + 2 * at) = v4u{ out[0], out[1], out[2], out[3] };
}

// ---------------------------------------------------------------- launches
const char* wrong_sizes(const ntc_attention_desc* d) {
    if (!d) return "no description";
    if (d->sequences < 0 || d->q_rows < 0 || d->k_rows < 0 || d->sequences >= 1 << 30) return "sequences and rows from 0 on are needed, fewer than 2^30 sequences";
    if (d->dtype != NTC_BF16 && d->dtype != NTC_F16) return "queries, keys and values are bfloat16 or float16";
    if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8) return "a head has a multiple of 8 elements, up to 128";
    if (d->k_heads < 1 || d->q_heads < 1 || d->q_heads % d->k_heads || d->q_heads / d->k_heads > 1024 || d->q_heads > 65536) return "query heads must be 1 to 1024 times the key heads, at most 65536";
    if (!(d->scale > 0) || !(d->scale < 1e30f)) return "scale must be a number above 0";
    if (d->q_rows * (d->q_heads / d->k_heads) >= (int64_t)1 << 30 || d->k_rows >= (int64_t)1 << 30) return "fewer than 2^30 keys, and queries times a group's heads, are needed";
    if (!d->cu_q && d->sequences && d->q_rows % d->sequences) return "without ends every sequence has as many queries";
    if (!d->cu_k && d->sequences && d->k_rows % d->sequences) return "without ends every sequence has as many keys";
    if (!d->sequences && ((d->q_rows && !d->cu_q) || (d->k_rows && !d->cu_k))) return "rows without a sequence";
    return nullptr;
}
const char* wrong(const ntc_attention_desc* d, bool back) {
    if (const char* w = wrong_sizes(d)) return w;
    const int64_t* s = &d->q_row_stride;
    for (int i = 0; i < 9; i++) if (s[i] < 0 || s[i] % 8 || (i % 3 == 0 && s[i] > 1 << 22) || (i % 3 == 1 && s[i] > 1 << 20)) return "strides are multiples of 8 elements from 0 on, of rows at most 2^22, of heads 2^20";
    if (back) {
        const int64_t* t = &d->do_row_stride;
        for (int i = 0; i < 3; i++) if (t[i] < 0 || t[i] % 8 || (i == 0 && t[i] > 1 << 22) || (i == 1 && t[i] > 1 << 20)) return "strides are multiples of 8 elements from 0 on, of rows at most 2^22, of heads 2^20";
    }
    if (d->q_rows && (!d->q || !d->o || (back && (!d->d_o || !d->lse || !d->o_rest || !d->workspace)))) return "null pointer";
    if (d->k_rows && (!d->k || !d->v)) return "null pointer";
    uintptr_t all = (uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->o | (uintptr_t)d->o_rest | (uintptr_t)d->workspace;
    if (back) all |= (uintptr_t)d->d_o | (uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv;
    if (all % 16) return "operands, results and the workspace start at a multiple of 16 bytes";
    return nullptr;
}
AttentionArgs args_of(const ntc_attention_desc* d) {
    AttentionArgs a = {};
    a.q = { (const char*)d->q, 2 * d->q_row_stride, 2 * d->q_head_stride, 2 * d->q_batch_stride };
    a.k = { (const char*)d->k, 2 * d->k_row_stride, 2 * d->k_head_stride, 2 * d->k_batch_stride };
    a.v = { (const char*)d->v, 2 * d->v_row_stride, 2 * d->v_head_stride, 2 * d->v_batch_stride };
    a.d_o = { (const char*)d->d_o, 2 * d->do_row_stride, 2 * d->do_head_stride, 2 * d->do_batch_stride };
    a.out = d->o; a.rest = d->o_rest; a.dq = d->dq; a.dk = d->dk; a.dv = d->dv;
    a.lse = d->lse;
    a.cu_q = d->cu_q; a.cu_k = d->cu_k; a.k_lens = d->k_lens;
    a.q_rows = d->q_rows; a.k_rows = d->k_rows;
    a.sequences = (int)d->sequences;
    a.q_each = d->sequences ? (int)(d->q_rows / d->sequences) : 0;
    a.k_each = d->sequences ? (int)(d->k_rows / d->sequences) : 0;
    a.q_heads = d->q_heads; a.k_heads = d->k_heads; a.group = d->q_heads / d->k_heads; a.D = d->head_dim; a.causal = d->causal != 0;
    a.group_magic = a.group > 1 ? (unsigned)((((uint64_t)1 << 32) + a.group - 1) / a.group) : 0;
    a.parts = 1;
    a.line_heads = a.k_heads % 4 == 0 && a.D <= 16 ? 2 : a.k_heads % 2 == 0 && a.D <= 32 ? 1 : 0;
    a.scale = d->scale;
    a.c = d->scale * kLog2e;
    return a;
}
// tiles of `size` of rows that lie in sequences (each at most a tile more than its share, one more for what is behind the last)
void set_tiles(const AttentionArgs& a, bool ends, int64_t each, int64_t rows, int64_t size, int& tiles_each, int& tiles) {
    tiles_each = (int)((each + size - 1) / size);
    tiles = (int)(ends ? rows / size + a.sequences + 1 : (int64_t)tiles_each * a.sequences);
}
void set_row_tiles(AttentionArgs& a) { set_tiles(a, a.cu_q, (int64_t)a.q_each * a.group, a.q_rows * a.group, kRows, a.tiles_each, a.tiles); }
void set_key_tiles(AttentionArgs& a) { set_tiles(a, a.cu_k, a.k_each, a.k_rows, kRows, a.tiles_each, a.tiles); }
void set_extents(AttentionArgs& a) {
    set_tiles(a, a.cu_k, a.k_each, a.k_rows, kExtentRows, a.v_extents_each, a.v_extents);
    set_tiles(a, a.cu_q, a.q_each, a.q_rows, kExtentRows, a.do_extents_each, a.do_extents);
}
size_t extents_size(const AttentionArgs& a) { return 4 * ((size_t)a.v_extents + a.do_extents); }
template <class F> void with_head(int dtype, int D, F f) {
    const auto go = [&](auto t) {
        if (D <= 32) f(t, std::integral_constant<int, 32>{});
        else if (D <= 64) f(t, std::integral_constant<int, 64>{});
        else if (D <= 96) f(t, std::integral_constant<int, 96>{});
        else f(t, std::integral_constant<int, 128>{});
    };
    if (dtype == NTC_BF16) go(bf16{});
    else go(f16{});
}
bool too_many(const AttentionArgs& a) { return (int64_t)a.tiles * a.k_heads * a.parts >= ((int64_t)1 << 31) - (1 << 22); }
// (whole sets of 8 << line_heads blocks)
dim3 grid_for(const AttentionArgs& a) { const int64_t set = 8 << a.line_heads; return grid_of(((int64_t)a.tiles * a.k_heads * a.parts + set - 1) / set * set); }
size_t rounded(size_t n) { return (n + 15) / 16 * 16; }

// Parts of a sum. Without them the longest block's sum holds the card up where blocks are few; with them their 32-bit results are written and read once more. In us: `each` a
// stage where `slots` blocks are on the card at once (a quarter less where they are not), a stage and a half to begin a block, blocks of avg stages spread over the slots; `join` for
// the second launch (queries' gradients: 10 with what their parts hold twice), 4.5 TB/s for what the parts write and read. 8192 rows of 16 heads of 128 on 4, keys' and values' gradients: 864 us in one part, 646 in two, 667 in four, 755 in eight;
// 16 tokens against caches of 900 to 8192 rows: 186 in one, 71 in four to sixteen, 79 in 32; queries'
// gradients of 1 to 27 rows of 16 heads on 4 by 10 times 10200 to 12000 keys, all with both directions: 553 in one, 300 in parts; of ragged rows whose sums are 20 stages, 36 in one and 40 in two.
// Lengths are on the card, so a sequence's sum is taken to be of average length: one that is far longer than the others is split too little (single tokens of 63 sequences of 100 keys and one of 65536, 32 heads on 8 of
// 128: 1212 us, where the long one alone takes 51), and a cache's room counts in full (16 caches with room for 8192 that hold 100 keys: 10.7 us in parts).
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int parts_of(int64_t blocks, int64_t stages, float slots, float each, bool half, int64_t part_bytes, float join = 5) {
    int best = 1;
    float least = 0;
    for (int p = 1; p <= 64 && p <= stages; p *= 2) {
        const float busy = (float)blocks * (stages * (half ? 0.5f : 1.f) + 1.5f * p) / slots, longest = 0.75f * ((float)ceil_div(stages, p) + 1.5f);
        const float cost = each * (busy > longest ? busy : longest) + (p > 1 ? join + 2.f * p * part_bytes / 4.5e6f : 0.f);
        if (p == 1 || cost < least) { best = p; least = cost; }
    }
    return best;
}
int forward_parts(const AttentionArgs& a) {
    const int64_t keys = a.sequences ? ceil_div(a.k_rows, a.sequences) : 0, queries = a.sequences ? a.q_rows / a.sequences : 0;
    return parts_of((int64_t)a.tiles * a.k_heads, ceil_div(keys, kKeys), a.D <= 32 ? 1024 : a.D <= 64 ? 768 : 512, a.D <= 64 ? 2.7f : 2.2f, a.causal && 2 * queries > keys, a.q_rows * a.q_heads * a.D * 4);
}
int query_parts(const AttentionArgs& a) {
    const int64_t keys = a.sequences ? ceil_div(a.k_rows, a.sequences) : 0, queries = a.sequences ? a.q_rows / a.sequences : 0;
    return parts_of((int64_t)a.tiles * a.k_heads, ceil_div(keys, kKeys), a.D <= 32 ? 1024 : 512, a.D <= 64 ? 3.f : 3.6f, a.causal && 2 * queries > keys, a.q_rows * a.q_heads * a.D * 4, 10);
}
int backward_parts(const AttentionArgs& a) {
    const int64_t keys = a.sequences ? ceil_div(a.k_rows, a.sequences) : 0, queries = a.sequences ? a.q_rows / a.sequences : 0;
    return parts_of((int64_t)a.tiles * a.k_heads, ceil_div(queries * a.group, 64), a.D <= 32 ? 768 : a.D <= 64 ? 512 : 256, a.D <= 64 ? 3.f : 2.4f, a.causal && 2 * keys > queries, a.k_rows * a.k_heads * a.D * 8);
}

}  // namespace
}  // namespace ntc_ops

using namespace ntc_ops;

extern "C" {

size_t ntc_op_attention_workspace(const ntc_attention_desc* d, int32_t backward) {
    if (wrong_sizes(d)) return 0;
    AttentionArgs a = args_of(d);
    if (!backward) {
        if (!d->q_rows) return 0;
        set_row_tiles(a);
        const int parts = forward_parts(a);
        return parts > 1 ? (size_t)parts * d->q_rows * d->q_heads * (8 + 4 * (size_t)d->head_dim) : 0;
    }
    if (d->dtype == NTC_F16) set_extents(a);
    const size_t n = d->q_rows ? 2 * rounded((size_t)d->q_rows * d->q_heads * 4) + rounded(extents_size(a)) : 0;
    size_t of_parts = 0;                                   // (dq's are joined before dk's and dv's are made)
    if (d->q_rows && d->k_rows) {
        set_row_tiles(a);
        if (const int parts = query_parts(a); parts > 1) of_parts = (size_t)parts * d->q_rows * d->q_heads * 4 * (d->head_dim + 1);
        set_key_tiles(a);
        if (const int parts = backward_parts(a); parts > 1) of_parts = std::max(of_parts, (size_t)parts * d->k_rows * d->k_heads * d->head_dim * 8);
    }
    return n + of_parts;
}

int ntc_op_attention(const ntc_attention_desc* d, void* stream, char* why, size_t cap) {
    if (const char* w = wrong(d, false)) return refuse(why, cap, w);
    if (!d->q_rows) return 0;
    AttentionArgs a = args_of(d);
    const hipStream_t s = (hipStream_t)stream;
    set_row_tiles(a);
    a.parts = forward_parts(a);
    if (a.parts > 1) {
        if (!d->workspace) return refuse(why, cap, "null workspace");
        a.part_sums = (float*)d->workspace;
        a.part_stats = (float2*)(a.part_sums + (size_t)a.parts * d->q_rows * d->q_heads * d->head_dim);
    }
    if (too_many(a)) return refuse(why, cap, "too many tiles of rows times heads: 2^31 at most");
    const dim3 grid = grid_for(a);
    with_head(d->dtype, d->head_dim, [&](auto t, auto h) {
        k_attention<decltype(t), h.value><<<grid, 256, 0, s>>>(a);
        if (a.parts > 1) k_attention_join<decltype(t), h.value == 96 ? 16 : h.value / 8><<<grid_of(ceil_div(d->q_rows * d->q_heads, 4)), 256, 0, s>>>(a);
    });
    return launched(why, cap);
}

int ntc_op_attention_backward(const ntc_attention_desc* d, void* stream, char* why, size_t cap) {
    if (const char* w = wrong(d, true)) return refuse(why, cap, w);
    const hipStream_t s = (hipStream_t)stream;
    AttentionArgs a = args_of(d);
    a.log_sums = (float*)d->workspace;
    a.deltas = (float*)((char*)d->workspace + rounded((size_t)d->q_rows * d->q_heads * 4));
    if (d->dtype == NTC_F16) set_extents(a);
    a.extents_v = (float*)((char*)a.deltas + rounded((size_t)d->q_rows * d->q_heads * 4));
    a.extents_do = a.extents_v + a.v_extents;
    a.part_sums = d->q_rows ? (float*)((char*)a.extents_v + rounded(extents_size(a))) : (float*)d->workspace;
    set_key_tiles(a);
    a.parts = d->q_rows && d->k_rows ? backward_parts(a) : 1;
    const int parts = a.parts;
    const bool keys_many = too_many(a);
    set_row_tiles(a);
    const int q_parts = d->q_rows && d->k_rows && d->dq ? query_parts(a) : 1;
    a.parts = q_parts;
    a.part_rests = a.part_sums + (size_t)q_parts * d->q_rows * d->q_heads * d->head_dim;
    if (keys_many || too_many(a)) return refuse(why, cap, "too many tiles of rows times heads: 2^31 at most");
    if (d->q_rows) {
        if (d->dtype == NTC_F16) k_attention_extent<f16><<<grid_of((int64_t)a.v_extents + a.do_extents), 256, 0, s>>>(a);
        const dim3 grid = grid_for(a);
        with_head(d->dtype, d->head_dim, [&](auto t, auto h) {
            if (a.parts == 1) { k_attention_dq<decltype(t), h.value, false><<<grid, 256, 0, s>>>(a); return; }
            k_attention_dq<decltype(t), h.value, true><<<grid, 256, 0, s>>>(a);
            k_attention_dq_join<decltype(t)><<<grid_of(ceil_div(d->q_rows * d->q_heads * (d->head_dim / 8), 256)), 256, 0, s>>>(a);
        });
        if (const int rc = launched(why, cap)) return rc;
    }
    if (!d->k_rows || (!d->dk && !d->dv)) return 0;
    set_key_tiles(a);
    a.parts = parts;
    const dim3 grid = grid_for(a);
    with_head(d->dtype, d->head_dim, [&](auto t, auto h) {
        k_attention_dkv<decltype(t), h.value><<<grid, 256, 0, s>>>(a);
        if (a.parts > 1) k_attention_sum<decltype(t)><<<grid_of(ceil_div(d->k_rows * d->k_heads * (d->head_dim / 4), 256)), 256, 0, s>>>(a);
    });
    return launched(why, cap);
}

}  // extern "C"
