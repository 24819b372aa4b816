// Device code object of the experts' computation between a dispatch and a combine on gfx950: products of every expert's rows with
// that expert's weights, their gradients and the gated activation between two of them.  All of them work on the rows as the
// dispatch lays them out, with the rows' counts on the device only.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/deep_ep_hip.h"
#include "ep_expert_args.h"

#define WAVE 64

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_byte;

__device__ __forceinline__ int lane_id() { return threadIdx.x & (WAVE - 1); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return ((int64_t)uniform((int)(v >> 32)) << 32) | (unsigned)uniform((int)v);
}
__device__ __forceinline__ int align_up(int x, int a) { return (x + a - 1) / a * a; }
__device__ __forceinline__ int ceil_div(int x, int a) { return (x + a - 1) / a; }

__device__ __forceinline__ int wave_inclusive_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);      // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);      // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);      // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // row_bcast:15 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // row_bcast:31 to rows 2 and 3
    return v;
}

// ---- the layout ---------------------------------------------------------------------------------------

// Rows of an expert; limit: up to where its rows are written (padding included where it is asked for).  Whatever the counts on the
// device say, no row lies outside the tensors.
struct ExpertRows {
    int start, count, limit;
};
__device__ __forceinline__ ExpertRows rows_of_expert(const EpExpertLayout& l, int e) {
    ExpertRows r;
    if (l.psum == nullptr) {
        r.start = 0;
        r.count = r.limit = l.num_rows;
        return r;
    }
    const int before = e > 0 ? l.psum[e - 1] : 0, end = l.psum[e];
    r.start = min(align_up(min(max(before, 0), l.num_rows), l.alignment), l.num_rows);
    const int last = min(max(end, r.start), l.num_rows);
    r.count = last - r.start;
    r.limit = r.count;
    if (l.zero_rows == EP_ZERO_PADDING) r.limit = min(align_up(last, l.alignment), l.num_rows) - r.start;
    if (l.zero_rows == EP_ZERO_ALL) r.limit = (e + 1 < l.num_experts ? min(align_up(last, l.alignment), l.num_rows) : l.num_rows) - r.start;
    return r;
}

// A tile of output rows: of which expert, and which of its rows.
struct RowTile {
    int expert, first;            // first row in the tensor
    int valid, limit;             // rows of the tile that are computed, rows that are written
};

// Tile number -> (expert, rows): every wave scans the experts' counts, 64 at a time.
template <int TM>
__device__ __forceinline__ int count_row_tiles(const EpExpertLayout& l) {
    int total = 0;
    for (int e0 = 0; e0 < l.num_experts; e0 += WAVE) {
        const int e = e0 + lane_id();
        const int tiles = e < l.num_experts ? ceil_div(rows_of_expert(l, e).limit, TM) : 0;
        total += __builtin_amdgcn_readlane(wave_inclusive_sum(tiles), WAVE - 1);
    }
    return total;
}
template <int TM>
__device__ __forceinline__ RowTile find_row_tile(const EpExpertLayout& l, int tile) {
    RowTile t = {0, 0, 0, 0};
    for (int e0 = 0; e0 < l.num_experts; e0 += WAVE) {
        const int e = e0 + lane_id();
        ExpertRows r = {0, 0, 0};
        if (e < l.num_experts) r = rows_of_expert(l, e);
        const int tiles = ceil_div(r.limit, TM), upto = wave_inclusive_sum(tiles);
        const int all = __builtin_amdgcn_readlane(upto, WAVE - 1);
        if (tile >= all) {
            tile -= all;
            continue;
        }
        const int at = __builtin_ctzll(__ballot(upto > tile));
        const int skip = (tile - __builtin_amdgcn_readlane(upto - tiles, at)) * TM;
        t.expert = e0 + at;
        t.first = __builtin_amdgcn_readlane(r.start, at) + skip;
        t.valid = min(max(__builtin_amdgcn_readlane(r.count, at) - skip, 0), TM);
        t.limit = min(__builtin_amdgcn_readlane(r.limit, at) - skip, TM);
        break;
    }
    return t;
}

// Workgroup -> tile.  Workgroups go round the eight XCDs, each with an L2 of its own: an XCD takes one stretch of the tiles, and
// within a stretch GROUP row tiles go through the column tiles together, so that what runs at once on an XCD reads few panels.
__device__ __forceinline__ bool tile_of_block(int row_tiles, int column_tiles, int group, int& row, int& column) {
    const int total = row_tiles * column_tiles, share = ceil_div(total, 8);
    const int at = (int)blockIdx.x >> 3, id = ((int)blockIdx.x & 7) * share + at;
    if (at >= share || id >= total) return false;
    const int g = id / (group * column_tiles), first = g * group, rows = min(group, row_tiles - first);
    const int in = id - g * group * column_tiles;
    column = in / rows;
    row = first + in - column * rows;
    return true;
}

// ---- tiles in LDS -----------------------------------------------------------------------------------------
//
// A step of the products covers 128 bytes of depth (64 BF16, 128 FP8).  An operand comes in one of two forms:
//   direct      [tile, depth] in memory: 128 bytes of every row of the tile.  Row r's 16-byte chunk c lies at chunk c ^ (r / 2 % 8) of
//               its 128 bytes in LDS, so that 16 rows' chunks of the same number, which a matrix instruction wants at once, lie in
//               different banks.
//   transposed  [depth, tile] in memory (BF16): 64 rows of 2 * tile bytes.  32-byte granule g of row r lies at g ^ (r % 4 + r / 8 % 2 * 4),
//               for the rows that one transposing read goes over.
// Memory goes to LDS without passing registers (buffer loads with the LDS bit: lane l's 16 bytes land at m0 + 16 l); the swizzle
// is in the addresses that the lanes fetch.  Reads behind the operand's end (rows and channels that do not exist) bring zeros.

constexpr unsigned OUTSIDE = 0x7ffffff0u;      // beyond the bytes of any buffer

__device__ __forceinline__ i32x4 buffer_of(const char* base, unsigned bytes) {
    const uint64_t at = (uint64_t)base;
    return i32x4{(int)(unsigned)at, (int)((unsigned)(at >> 32) & 0xffffu), (int)bytes, 0x00020000};
}

// (No register is written: nothing that the compiler could use before the data are there.  What was fetched is read behind
// wait_and_meet.)
__device__ __forceinline__ void fetch16(unsigned to, unsigned from, i32x4 buffer) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(from), "s"(buffer) : "memory");
}
__device__ __forceinline__ void fetch4(unsigned to, unsigned from, i32x4 buffer) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(from), "s"(buffer) : "memory");
}
// All but this wave's last PENDING fetches have arrived, and so has every wave of the workgroup, done with what it read from LDS.
template <int PENDING>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory");
}

template <int T, int WAVES, bool TRANSPOSED>
struct TileFetch {
    static constexpr int PIECES = T / 8;                                   // of 1 KiB, one fetch of a wave each
    static constexpr int MINE = PIECES < WAVES ? 1 : PIECES / WAVES;       // (fewer pieces than waves: some are fetched twice)
    unsigned from[MINE];
    const char* base;
    int64_t ld;
    unsigned bytes;               // direct: all rows of the tile; transposed: one row's from the tile's first column on
    int depth_bytes, chunk;       // direct
    int depth;                    // transposed

    __device__ __forceinline__ void init(const char* b, int64_t row_bytes, int tile_size, int depth_, int elem, int wave) {
        base = b;
        ld = row_bytes;
        depth = depth_;
        depth_bytes = depth_ * elem;
        const int lane = lane_id();
        if (!TRANSPOSED) {
            bytes = tile_size > 0 ? (unsigned)((tile_size - 1) * row_bytes + depth_bytes) : 0u;
            // (pieces of a wave are an even number apart: the same chunk of every row)
            chunk = (lane & 7) ^ (((wave % PIECES) * 4 + (lane >> 4)) & 7);
#pragma unroll
            for (int i = 0; i < MINE; ++i) from[i] = (unsigned)((piece(i, wave) * 8 + (lane >> 3)) * row_bytes + chunk * 16);
        } else {
            bytes = (unsigned)tile_size * 2;
            constexpr int LANES = T / 8;                                   // of a row
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int r = piece(i, wave) * (WAVE / LANES) + lane / LANES, at = lane % LANES;
                const int c = (((at >> 1) ^ ((r & 3) | ((r >> 3) & 1) << 2)) << 1) | (at & 1);
                from[i] = c * 8 < tile_size ? (unsigned)(r * row_bytes + c * 16) : OUTSIDE;
            }
        }
    }
    __device__ __forceinline__ static int piece(int i, int wave) { return (wave + i * WAVES) % PIECES; }

    // step `s` of the depth into the LDS at `to` (behind the last step: zeros)
    __device__ __forceinline__ void fetch(int s, unsigned to, int wave) const {
        if (!TRANSPOSED) {
            const int left = depth_bytes - s * 128;
            const i32x4 buffer = buffer_of(base + (int64_t)s * 128, left > 0 && bytes > 0 ? bytes - s * 128 : 0u);
            if (left >= 128) {
#pragma unroll
                for (int i = 0; i < MINE; ++i) fetch16(to + piece(i, wave) * 1024, from[i], buffer);
            } else {
#pragma unroll
                for (int i = 0; i < MINE; ++i) fetch16(to + piece(i, wave) * 1024, chunk * 16 < left ? from[i] : OUTSIDE, buffer);
            }
        } else {
            const int rows = min(depth - s * 64, 64);
            const i32x4 buffer = buffer_of(base + (int64_t)s * 64 * ld, rows > 0 ? (unsigned)((rows - 1) * ld) + bytes : 0u);
#pragma unroll
            for (int i = 0; i < MINE; ++i) fetch16(to + piece(i, wave) * 1024, from[i], buffer);
        }
    }
};

// The 16 rows from `first` on of a direct tile, 16 bytes a lane: row lane % 16, chunk half * 4 + lane / 16.
__device__ __forceinline__ u32x4 direct_fragment(const char* tile, int first, int half) {
    const int lane = lane_id(), r = lane & 15;
    return *(const u32x4*)(tile + (first + r) * 128 + (((half * 4 + (lane >> 4)) ^ (r >> 1)) << 4));
}
// The 16 columns from `first` on of a transposed tile, rows half * 32 + lane / 16 * 8 + (0 .. 7) of them: two transposing reads, each of
// which hands the lanes of a group of 16 the columns of the four 32-byte row pieces that the group reads.
template <int T>
__device__ __forceinline__ u32x4 transposed_fragment(const char* tile, int first, int half) {
    const int lane = lane_id(), j = (lane >> 2) & 3, b = lane >> 4;
    const int granule = (first >> 4) ^ (j | (b & 1) << 2);
    const lds_byte* at = (const lds_byte*)(tile + (half * 32 + b * 8 + j) * (T * 2) + granule * 32 + (lane & 3) * 8);
    typedef __attribute__((address_space(3))) i16x4* quad;
    union {
        i16x4 q[2];
        u32x4 v;
    } f;
    f.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((quad)at);
    f.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((quad)(at + 4 * T * 2));
    return f.v;
}

template <bool TRANSPOSED, int T>
__device__ __forceinline__ u32x4 fragment(const char* tile, int first, int half) {
    if (TRANSPOSED) return transposed_fragment<T>(tile, first, half);
    return direct_fragment(tile, first, half);
}

union Fragment8 {
    u32x4 half[2];
    i32x8 v;
};

// ---- low-rank adapters: numbers of a tile ------------------------------------------------------------------

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) v = min(v, __shfl_xor(v, d));
    return v;
}
constexpr int NO_ADAPTER = 0x7fffffff;
// The smallest number of the tile's rows above `last`; every wave finds it by itself.
template <int TM>
__device__ __forceinline__ int next_adapter(const int* of_row, int last) {
    int v = NO_ADAPTER;
#pragma unroll
    for (int i = 0; i < TM; i += WAVE) {
        const int r = i + lane_id();
        const int a = r < TM ? of_row[r] : NO_ADAPTER;
        v = min(v, a > last ? a : NO_ADAPTER);
    }
    return uniform(wave_min(v));
}
template <int TM>
__device__ __forceinline__ void note_adapters(const EpLoraArgs& l, int first, int valid, int* of_row, int threads) {
    for (int r = threadIdx.x; r < TM; r += threads) {
        const int a = r < valid ? l.adapter[first + r] : -1;
        of_row[r] = a >= 0 && a < l.num_adapters ? a : NO_ADAPTER;
    }
}

// ---- products ---------------------------------------------------------------------------------------------
//
// One workgroup computes TM x TN of the output, WR x WC waves a part each, in 32 bits.  The matrix instruction's first operand is
// the output's columns, its second the rows: a lane then holds four neighbouring columns of one row.
template <int TM, int TN, int WR, int WC, int STAGES, bool FP8, bool COLUMNS_T, bool ROWS_T, bool OUT32, bool LORA = false>
struct Gemm {
    static constexpr int WAVES = WR * WC, FM = TM / WR, FN = TN / WC, NR = FM / 16, NC = FN / 16;
    static constexpr int COLUMNS_BYTES = TN * 128, ROWS_BYTES = TM * 128, SF_BYTES = FP8 ? (TM < WAVE ? WAVE : TM) * 4 : 0;
    static constexpr int STAGE_BYTES = COLUMNS_BYTES + ROWS_BYTES + SF_BYTES;
    static constexpr int OUT_ELEM = OUT32 ? 4 : 2, OUT_ROW = FN * OUT_ELEM + 16, OUT_BYTES = WAVES * 16 * OUT_ROW;
    static constexpr int BLOCKS = (TN + 127) / 128, TABLE = EP_EXPERT_MAX_DEPTH_FP8 / 128;
    static constexpr int TABLE_BYTES = FP8 ? BLOCKS * TABLE * 4 : 0;
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES > OUT_BYTES ? STAGES * STAGE_BYTES : OUT_BYTES;
    typedef TileFetch<TN, WAVES, COLUMNS_T> ColumnsFetch;
    typedef TileFetch<TM, WAVES, ROWS_T> RowsFetch;
    static constexpr int FETCHES = ColumnsFetch::MINE + RowsFetch::MINE + (FP8 ? 1 : 0);       // of a wave and step
    static constexpr int STEP = FP8 ? 128 : 64;

    // rows .. rows + valid: what is computed, up to limit zeros are written; columns from column on
    __device__ __forceinline__ static void run(const EpGemmArgs& a, const char* rows, const char* columns, int valid, int limit,
                                               int num_columns, int depth, const float* rows_sf, const float* columns_sf, char* out,
                                               int first = 0, const char* up = nullptr) {
        __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
        __shared__ float table[FP8 ? BLOCKS * TABLE : 1];
        __shared__ int adapters[LORA ? TM : 1];
        const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
        const int first_row = (wave / WC) * FM, first_column = (wave % WC) * FN;
        const unsigned lds0 = (unsigned)(size_t)(lds_byte*)lds;
        const int steps = valid > 0 ? ceil_div(depth, STEP) : 0;

        f32x4 acc[NR][NC];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        ColumnsFetch cf;
        RowsFetch rf;
        cf.init(columns, a.columns_ld, min(num_columns, TN), depth, FP8 ? 1 : 2, wave);
        rf.init(rows, a.rows_ld, valid, depth, FP8 ? 1 : 2, wave);
        unsigned sf_from = 0, sf_bytes = 0;
        const int groups = ceil_div(depth, 128);
        constexpr int SF_PIECES = SF_BYTES / 256 > 0 ? SF_BYTES / 256 : 1;
        if (FP8) {
            const int r = (wave % SF_PIECES) * WAVE + lane;
            sf_from = r < valid ? (unsigned)(r * a.rows_sf_row * 4) : OUTSIDE;
            sf_bytes = valid > 0 ? (unsigned)((valid - 1) * a.rows_sf_row + 1) * 4u : 0u;
            for (int i = threadIdx.x; i < BLOCKS * groups; i += WAVES * WAVE) {
                const int b = i / groups, g = i - b * groups;
                if (b * 128 < num_columns) table[b * TABLE + g] = columns_sf[b * a.columns_sf_row + g * a.columns_sf_col];
            }
        }
        auto fetch = [&](int s, int stage) {
            const unsigned to = lds0 + stage * STAGE_BYTES;
            cf.fetch(s, to, wave);
            rf.fetch(s, to + COLUMNS_BYTES, wave);
            if (FP8) {
                const i32x4 buffer = buffer_of((const char*)(rows_sf + s * a.rows_sf_col), s < steps ? sf_bytes : 0u);
                fetch4(to + COLUMNS_BYTES + ROWS_BYTES + (wave % SF_PIECES) * 256, sf_from, buffer);
            }
        };

        auto multiply = [&](const char* at, const char* at_rows) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                u32x4 c[NC], r[NR];
#pragma unroll
                for (int j = 0; j < NC; ++j) c[j] = fragment<COLUMNS_T, TN>(at, first_column + j * 16, half);
#pragma unroll
                for (int i = 0; i < NR; ++i) r[i] = fragment<ROWS_T, TM>(at_rows, first_row + i * 16, half);
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < NC; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c[j]), __builtin_bit_cast(bf16x8, r[i]),
                                                                           acc[i][j], 0, 0, 0);
            }
        };

        if (steps > 0) {
#pragma unroll
            for (int s = 0; s < STAGES - 1; ++s) fetch(s, s);
        }
        if (LORA) add_adapters(a, lds + (STAGES - 1) * STAGE_BYTES, adapters, first, valid, num_columns, up, multiply);
        int stage = 0;
        for (int s = 0; s < steps; ++s) {
            wait_and_meet<(STAGES - 2) * FETCHES>();
            fetch(s + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
            const char* const at = lds + stage * STAGE_BYTES;
            const char* const at_rows = at + COLUMNS_BYTES;
            if (!FP8) {
                multiply(at, at_rows);
            } else {
                // a step is one group of channels: its products are summed by themselves, then scaled
                const float* const scales = (const float*)(at_rows + ROWS_BYTES);
                const float of_columns = table[first_column / 128 * TABLE + s];
                Fragment8 c[NC];
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int half = 0; half < 2; ++half) c[j].half[half] = direct_fragment(at, first_column + j * 16, half);
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    Fragment8 r;
                    r.half[0] = direct_fragment(at_rows, first_row + i * 16, 0);
                    r.half[1] = direct_fragment(at_rows, first_row + i * 16, 1);
                    const float scale = scales[first_row + i * 16 + (lane & 15)] * of_columns;
#pragma unroll
                    for (int j = 0; j < NC; ++j) {
                        const f32x4 sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(c[j].v, r.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[i][j][k] = __builtin_fmaf(sum[k], scale, acc[i][j][k]);
                    }
                }
            }
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        wait_and_meet<0>();      // (the last fetches, of zeros, land in LDS too)

        // 16 rows of a wave's part at a time through LDS, to leave as whole lines
        char* const mine = lds + wave * 16 * OUT_ROW;
        constexpr int LANES = FN * OUT_ELEM / 16, PASS = WAVE / LANES;      // lanes of a row, rows of a store
        const int piece = lane % LANES, column = first_column + piece * (16 / OUT_ELEM);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                char* const to = mine + (lane & 15) * OUT_ROW + (j * 16 + (lane >> 4) * 4) * OUT_ELEM;
                if (OUT32) *(f32x4*)to = acc[i][j];
                else *(bf16x4*)to = __builtin_convertvector(acc[i][j], bf16x4);
            }
            asm volatile("" ::: "memory");
#pragma unroll
            for (int p = 0; p < 16; p += PASS) {
                const int r16 = p + lane / LANES, r = first_row + i * 16 + r16;
                if (r16 >= 16 || r >= limit || column >= num_columns) continue;
                u32x4 v = *(const u32x4*)(mine + r16 * OUT_ROW + piece * 16);
                if (r >= valid) v = u32x4{0u, 0u, 0u, 0u};
                u32x4* const to = (u32x4*)(out + ((int64_t)r * a.out_ld + column) * OUT_ELEM);
                if (OUT32 && a.accumulate) {
                    const f32x4 sum = *(const f32x4*)to + __builtin_bit_cast(f32x4, v);
                    v = __builtin_bit_cast(u32x4, sum);
                }
                *to = v;
            }
            asm volatile("" ::: "memory");
        }
    }

    // The adapters' part, in front of the product's first step and in the LDS of its last stage, while the first ones are on their way: for
    // every adapter that rows of the tile have, 32 ranks at a time, a step of 64 channels.  The low-rank rows are sums in 32 bits; they
    // go in as two BF16, the rounded value and the rest, against the same column of `up` twice, which keeps 2^-17 of them.
    template <typename Multiply>
    __device__ __forceinline__ static void add_adapters(const EpGemmArgs& a, char* stage, int* of_row, int first, int valid, int num_columns,
                                                        const char* up, Multiply multiply) {
        constexpr int THREADS = WAVES * WAVE;
        const EpLoraArgs& l = a.lora;
        char* const to_columns = stage;
        char* const to_rows = stage + COLUMNS_BYTES;
        note_adapters<TM>(l, first, valid, of_row, THREADS);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        for (int number = next_adapter<TM>(of_row, -1); number != NO_ADAPTER; number = next_adapter<TM>(of_row, number)) {
            for (int r0 = 0; r0 < l.rank; r0 += 32) {
                for (int i = threadIdx.x; i < TM * 4; i += THREADS) {
                    const int r = i >> 2, c = i & 3, rank = r0 + c * 8;
                    bf16x8 high = {}, rest = {};
                    if (of_row[r] == number && rank < l.rank) {
                        f32x4 sum[2] = {};
                        for (int k = 0; k < l.chunks; ++k) {
                            const f32x4* const from = (const f32x4*)(l.low + (((int64_t)k * a.layout.num_rows + first + r) * l.rank + rank));
                            sum[0] += from[0];
                            sum[1] += from[1];
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float v = sum[j >> 2][j & 3];
                            high[j] = (__bf16)v;
                            rest[j] = (__bf16)(v - (float)high[j]);
                        }
                    }
                    const int key = (r >> 1) & 7;
                    *(bf16x8*)(to_rows + r * 128 + ((c ^ key) << 4)) = high;
                    *(bf16x8*)(to_rows + r * 128 + (((c + 4) ^ key) << 4)) = rest;
                }
                for (int i = threadIdx.x; i < TN * 4; i += THREADS) {
                    const int r = i >> 2, c = i & 3, rank = r0 + c * 8;
                    u32x4 v = {0u, 0u, 0u, 0u};
                    if (r < num_columns && rank < l.rank) v = *(const u32x4*)(up + number * l.up_adapter + r * l.up_ld + rank * 2);
                    const int key = (r >> 1) & 7;
                    *(u32x4*)(to_columns + r * 128 + ((c ^ key) << 4)) = v;
                    *(u32x4*)(to_columns + r * 128 + (((c + 4) ^ key) << 4)) = v;
                }
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                multiply(to_columns, to_rows);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
        }
    }

    // Rows of the layout times the weights of their expert: out[r, c] = sum_d rows[r, d] columns[e(r)][c, d]
    __device__ __forceinline__ static void rows_kernel(const EpGemmArgs& a, int group) {
        const int row_tiles = count_row_tiles<TM>(a.layout);
        int row, column;
        if (!tile_of_block(row_tiles, a.column_tiles, group, row, column)) return;
        const RowTile t = find_row_tile<TM>(a.layout, row);
        const int64_t c0 = (int64_t)column * TN;
        const char* const columns = a.columns + t.expert * a.columns_expert + (COLUMNS_T ? c0 * 2 : c0 * a.columns_ld);
        run(a, a.rows + t.first * a.rows_ld, columns, t.valid, t.limit, a.num_columns - (int)c0, a.depth,
            a.rows_sf + (FP8 ? t.first * a.rows_sf_row : 0), a.columns_sf + (FP8 ? t.expert * a.columns_sf_expert + c0 / 128 * a.columns_sf_row : 0),
            a.out + (t.first * a.out_ld + c0) * OUT_ELEM, t.first,
            LORA ? a.lora.up + t.expert * a.lora.up_expert + c0 * a.lora.up_ld : nullptr);
    }

    // Gradient of an expert's weights: out[e][r, c] = sum over the expert's rows d of rows[d, r] columns[d, c]
    __device__ __forceinline__ static void weights_kernel(const EpGemmArgs& a, int group) {
        int row, column;
        if (!tile_of_block(a.row_tiles * a.layout.num_experts, a.column_tiles, group, row, column)) return;
        const int e = row / a.row_tiles, r0 = (row - e * a.row_tiles) * TM, c0 = column * TN;
        const ExpertRows in = rows_of_expert(a.layout, e);
        const int count = uniform(in.count);
        const int64_t start = uniform(in.start);
        const int out_rows = min(a.num_out_rows - r0, TM);
        run(a, a.rows + start * a.rows_ld + (int64_t)r0 * 2, a.columns + start * a.columns_ld + (int64_t)c0 * 2, out_rows, out_rows,
            a.num_columns - c0, count, nullptr, nullptr, a.out + (e * a.out_expert + (int64_t)r0 * a.out_ld + c0) * OUT_ELEM);
    }
};

#define EP_GEMM_ROWS(NAME, TM, TN, WR, WC, STAGES, FP8, COLUMNS_T, GROUP)                                             \
    extern "C" __global__ __launch_bounds__(WR* WC* WAVE) void NAME(EpGemmArgs a) {                                   \
        Gemm<TM, TN, WR, WC, STAGES, FP8, COLUMNS_T, false, false>::rows_kernel(a, GROUP);                             \
    }
EP_GEMM_ROWS(ep_grouped_bf16, 128, 128, 2, 2, 2, false, false, 8)
EP_GEMM_ROWS(ep_grouped_fp8, 128, 128, 2, 2, 2, true, false, 8)
EP_GEMM_ROWS(ep_grouped_transposed_bf16, 128, 128, 2, 2, 2, false, true, 8)
extern "C" __global__ __launch_bounds__(256) void ep_grouped_lora_bf16(EpGemmArgs a) {
    Gemm<128, 128, 2, 2, 2, false, false, false, false, true>::rows_kernel(a, 8);
}
extern "C" __global__ __launch_bounds__(256) void ep_grouped_weights_bf16(EpGemmArgs a) {
    Gemm<128, 128, 2, 2, 2, false, true, true, false>::weights_kernel(a, 8);
}
extern "C" __global__ __launch_bounds__(256) void ep_grouped_weights_f32(EpGemmArgs a) {
    Gemm<128, 128, 2, 2, 2, false, true, true, true>::weights_kernel(a, 8);
}

// ---- low-rank adapters: rows times the first matrix ---------------------------------------------------------
//
// low[chunk][r] = scale[a] * sum over the chunk's channels of down[a][e] rows[r].  A workgroup has ROWS rows of an expert, a chunk of the
// depth, which its four waves share 128 channels at a time, and every `slots`-th of the adapters that its rows have: all rows are
// multiplied with an adapter's matrix, and the rows that have it keep what they get.  Operands go from memory straight to
// registers: nothing is used twice but by the neighbouring waves, out of the caches.
template <int ROWS, int RANKS>
__device__ __forceinline__ void lora_down_body(const EpGemmArgs& a) {
    constexpr int NR = ROWS / 16, NK = RANKS / 16, PARTS = EP_LORA_STEP / 128;
    __shared__ int of_row[ROWS];
    __shared__ __attribute__((aligned(16))) float sums[4][ROWS][RANKS + 4];
    const EpLoraArgs& l = a.lora;
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    int at = blockIdx.x;
    const int slot = at % l.slots;
    at /= l.slots;
    const int chunk = at % l.chunks, tile = at / l.chunks;
    const RowTile t = find_row_tile<ROWS>(a.layout, tile);
    if (t.valid <= 0) return;
    note_adapters<ROWS>(l, t.first, t.valid, of_row, 256);
    __syncthreads();
    const int begin = chunk * l.chunk_depth, end = min(begin + l.chunk_depth, a.depth);
    const char* const rows = a.rows + t.first * a.rows_ld;
    int n = 0;
    for (int number = next_adapter<ROWS>(of_row, -1); number != NO_ADAPTER; number = next_adapter<ROWS>(of_row, number)) {
        if (n++ % l.slots != slot) continue;
        const char* const down = l.down + number * l.down_adapter + t.expert * l.down_expert;
        f32x4 acc[NR][NK];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < NK; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = begin + wave * 32 * PARTS; k0 < end; k0 += 128 * PARTS) {
            u32x4 x[PARTS][NR], w[PARTS][NK];
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const int k = k0 + p * 32 + (lane >> 4) * 8;
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int r = i * 16 + (lane & 15);
                    x[p][i] = r < t.valid && k < end ? *(const u32x4*)(rows + r * a.rows_ld + (int64_t)k * 2) : u32x4{0u, 0u, 0u, 0u};
                }
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    const int r = j * 16 + (lane & 15);
                    w[p][j] = r < l.rank && k < end ? *(const u32x4*)(down + r * l.down_ld + (int64_t)k * 2) : u32x4{0u, 0u, 0u, 0u};
                }
            }
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < NK; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[p][j]),
                                                                            __builtin_bit_cast(bf16x8, x[p][i]), acc[i][j], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < NK; ++j) *(f32x4*)&sums[wave][i * 16 + (lane & 15)][j * 16 + (lane >> 4) * 4] = acc[i][j];
        __syncthreads();
        const float scale = l.scales != nullptr ? l.scales[number] : 1.0f;
        for (int i = threadIdx.x; i < ROWS * (RANKS / 4); i += 256) {
            const int r = i / (RANKS / 4), c = (i - r * (RANKS / 4)) * 4;
            if (of_row[r] != number || c >= l.rank) continue;
            const f32x4 sum = (*(const f32x4*)&sums[0][r][c] + *(const f32x4*)&sums[1][r][c]) + (*(const f32x4*)&sums[2][r][c] + *(const f32x4*)&sums[3][r][c]);
            *(f32x4*)(l.low + (((int64_t)chunk * a.layout.num_rows + t.first + r) * l.rank + c)) = sum * scale;
        }
        __syncthreads();
    }
}
#define EP_LORA_DOWN(ROWS, RANKS) \
    extern "C" __global__ __launch_bounds__(256) void ep_lora_down_##ROWS##_##RANKS(EpGemmArgs a) { lora_down_body<ROWS, RANKS>(a); }
EP_LORA_DOWN(16, 16)
EP_LORA_DOWN(16, 32)
EP_LORA_DOWN(16, 64)
EP_LORA_DOWN(32, 16)
EP_LORA_DOWN(32, 32)
EP_LORA_DOWN(32, 64)

// ---- a token's number at the rows that it was sent to --------------------------------------------------------

extern "C" __global__ __launch_bounds__(256) void ep_expand_fill(EpExpandIndexArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < a.num_out) a.out[i] = -1;
}
extern "C" __global__ __launch_bounds__(256) void ep_expand_token_index_rows(EpExpandIndexArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(i / a.topk), k = (int)(i - (int64_t)row * a.topk);
    if (row >= min(a.num_rows, a.psum_rank[a.num_ranks - 1])) return;
    const int* const m = a.metadata + (int64_t)row * (a.topk + 2);
    const int slot = m[k], token = m[a.topk];
    if (slot >= 0 && slot < a.num_out && token >= 0 && token < a.num_values) a.out[slot] = a.values[token];
}

// ---- the gated activation -----------------------------------------------------------------------------
//
// out = silu(gate) * up * weight, a lane eight channels, a wave 512 of a row.

__device__ __forceinline__ float bf16_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ void widen(const u32x4& d, float* f) {
    f[0] = bf16_lo(d.x), f[1] = bf16_hi(d.x), f[2] = bf16_lo(d.y), f[3] = bf16_hi(d.y);
    f[4] = bf16_lo(d.z), f[5] = bf16_hi(d.z), f[6] = bf16_lo(d.w), f[7] = bf16_hi(d.w);
}
__device__ __forceinline__ u32x4 round_bf16(const float* f) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (__bf16)f[i];
    return __builtin_bit_cast(u32x4, v);
}
// (hardware exponential and reciprocal, each a unit in the last place off; for large negative gates the exponential is infinite and the
// reciprocal 0, as it has to be)
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f)); }

__device__ __forceinline__ unsigned row16_umax(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x128, 0xf, 0xf, false));  // row_ror:8
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x124, 0xf, 0xf, false));  // row_ror:4
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x122, 0xf, 0xf, false));  // row_ror:2
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x121, 0xf, 0xf, false));  // row_ror:1
    return x;
}

// 0: not a row to write, 1: one to write zeros into, 2: a row of an expert
__device__ __forceinline__ int kind_of_row(const EpExpertLayout& l, int row) {
    if (l.psum == nullptr) return 2;
    // experts that end at or before the row, and where the last of them ends
    int before = 0, end = 0;
    for (int e0 = 0; e0 < l.num_experts; e0 += WAVE) {
        const int e = e0 + lane_id();
        const int p = e < l.num_experts ? l.psum[e] : 0x7fffffff;
        const int n = __popcll(__ballot(p <= row));
        if (n > 0) end = __builtin_amdgcn_readlane(p, n - 1);
        before += n;
        if (n < WAVE) break;
    }
    const int start = align_up(max(end, 0), l.alignment);
    if (row < start) return l.zero_rows != EP_ZERO_NONE ? 1 : 0;
    return before < l.num_experts ? 2 : l.zero_rows == EP_ZERO_ALL ? 1 : 0;
}

template <bool FP8>
__device__ __forceinline__ void swiglu_body(const EpSwigluArgs& a) {
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int64_t task = (int64_t)blockIdx.x * 4 + wave;
    const int per_row = ceil_div(a.num_parts, a.parts_per_task);
    const int row = uniform((int)(task / per_row)), first = uniform((int)(task - (int64_t)row * per_row)) * a.parts_per_task;
    if (row >= a.layout.num_rows) return;
    const int kind = kind_of_row(a.layout, row);
    if (kind == 0) return;
    const float weight = kind == 2 && a.weights != nullptr ? a.weights[row] : 1.0f;
    const u32x4* const h = (const u32x4*)(a.h + (int64_t)row * a.h_ld * 2);
    const int vectors = a.channels >> 3;
    for (int part = first; part < min(first + a.parts_per_task, a.num_parts); ++part) {
        const int v = part * WAVE + lane;
        const bool live = v < vectors;
        float out[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live && kind == 2) {
            float gate[8], up[8];
            widen(h[v], gate);
            // (the ups begin at a multiple of eight channels as the gates do)
            widen(h[vectors + v], up);
#pragma unroll
            for (int i = 0; i < 8; ++i) out[i] = gate[i] * sigmoid(gate[i]) * up[i] * weight;
        }
        if (!FP8) {
            if (live) ((u32x4*)(a.out + (int64_t)row * a.out_ld * 2))[v] = round_bf16(out);
            continue;
        }
        // the quantiser of the dispatch, of the unrounded values
        unsigned bits = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = max(bits, __float_as_uint(out[i]) & 0x7fffffffu);
        const float m = __uint_as_float(row16_umax(bits));
        const float amax = m < 1e-4f ? 1e-4f : m;
        const float inverse = (1.0f / amax) * 448.0f;
        unsigned q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(out[4 * i] * inverse, out[4 * i + 1] * inverse, 0, false);
            q[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(out[4 * i + 2] * inverse, out[4 * i + 3] * inverse, w, true);
        }
        if (amax != amax) q[0] = q[1] = 0x7f7f7f7fu;
        if (!live) continue;
        ((u32x2*)(a.out + (int64_t)row * a.out_ld))[v] = u32x2{q[0], q[1]};
        if ((lane & 15) == 0) a.sf[(int64_t)row * a.sf_row + (int64_t)(v >> 4) * a.sf_col] = kind == 2 ? amax / 448.0f : 0.0f;
    }
}
extern "C" __global__ __launch_bounds__(256) void ep_swiglu_bf16(EpSwigluArgs a) { swiglu_body<false>(a); }
extern "C" __global__ __launch_bounds__(256) void ep_swiglu_fp8(EpSwigluArgs a) { swiglu_body<true>(a); }

// Gradients: a wave has a row, whose gate weight's gradient is the sum over its channels.
extern "C" __global__ __launch_bounds__(256) void ep_swiglu_gradients(EpSwigluArgs a) {
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int64_t task = (int64_t)blockIdx.x * 4 + wave;
    if (task >= a.layout.num_rows) return;
    const int row = (int)task, kind = kind_of_row(a.layout, row);
    if (kind == 0) return;
    const float weight = kind == 2 && a.weights != nullptr ? a.weights[row] : 1.0f;
    const u32x4* const h = (const u32x4*)(a.h + (int64_t)row * a.h_ld * 2);
    const u32x4* const grad_out = (const u32x4*)(a.grad_out + (int64_t)row * a.grad_out_ld * 2);
    u32x4* const grad_h = (u32x4*)(a.grad_h + (int64_t)row * a.grad_h_ld * 2);
    const int vectors = a.channels >> 3;
    float of_weight = 0.f;
    for (int v = lane; v < vectors; v += WAVE) {
        float of_gate[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, of_up[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (kind == 2) {
            float gate[8], up[8], grad[8];
            widen(h[v], gate);
            widen(h[vectors + v], up);
            widen(grad_out[v], grad);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = sigmoid(gate[i]), silu = gate[i] * s;
                of_weight = __builtin_fmaf(grad[i] * silu, up[i], of_weight);
                const float g = grad[i] * weight;
                of_up[i] = g * silu;
                of_gate[i] = g * up[i] * s * (1.0f + gate[i] * (1.0f - s));
            }
        }
        grad_h[v] = round_bf16(of_gate);
        grad_h[vectors + v] = round_bf16(of_up);
    }
    if (a.grad_weights == nullptr) return;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) of_weight += __shfl_xor(of_weight, d);
    if (lane == 0) a.grad_weights[row] = of_weight;
}
