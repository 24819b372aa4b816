// Device code object of the experts' computation between a dispatch and a combine on gfx950: products of every expert's rows with
// that expert's weights, their gradients and the gated activation between two of them.  All of them work on the rows as the
// dispatch lays them out, with the rows' counts on the device only.
//
//   ep_grouped_{bf16,fp8,transposed,lora}_<rows>x<columns>   a tile of the product (transposed: with the transposed weights, lora: with adapters)
//   ep_grouped_split_*, ep_sum_splits*                       few tiles: in parts of the depth, and their sum
//   ep_grouped_weights_*, ep_grouped_split_weights, ep_sum_weights_*   gradients of the weights
//   ep_lora_down_*                                           rows times the adapters' first matrices
//   ep_expand_*                                              a number per token -> per row
//   ep_swiglu_*                                              the activation and its gradients
//
// Rates that bound them on an MI355X, measured with a large copy, a large read and large library products: 4.9 and 6.3 TB/s, 1400
// (BF16, 8192 cubed; 1600 at 16384) and 3000 TFLOP/s (FP8).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/deep_ep_hip.h"
#include "ep_expert_args.h"

#define WAVE 64
// Loads and stores of what is touched once: past the caches.
template <bool NT, typename T>
__device__ __forceinline__ void store(T* p, T v) {
    if (NT) __builtin_nontemporal_store(v, p);
    else *p = v;
}

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

// 0: not a row to write, 1: one to write zeros into, 2: a row of an expert
__device__ __forceinline__ int kind_of_row(const EpExpertLayout& l, int row, int& expert) {
    expert = 0;
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
    expert = before;
    return before < l.num_experts ? 2 : l.zero_rows == EP_ZERO_ALL ? 1 : 0;
}

// Workgroup -> tile.  Workgroups go round the eight XCDs, each with an L2 of its own: an XCD takes one stretch of the tiles, and
// within a stretch GROUP row tiles go through the column tiles together, so that what runs at once on an XCD reads few panels.
__device__ __forceinline__ bool tile_of_block(int block, int row_tiles, int column_tiles, int group, int& row, int& column) {
    const int total = row_tiles * column_tiles, share = ceil_div(total, 8);
    const int at = block >> 3, id = (block & 7) * share + at;
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
//               (without it every group of 16 lanes would read two banks eight times over)
//   transposed  [depth, tile] in memory (BF16): 64 rows of 2 * tile bytes.  32-byte granule g of row r lies at g ^ (r % 4 + r / 8 % 2 * 4),
//               for the rows that one transposing read goes over.
// Memory goes to LDS without passing registers (buffer loads with the LDS bit: lane l's 16 bytes land at m0 + 16 l); the swizzle
// is in the addresses that the lanes fetch.  Reads behind the operand's end (rows and channels that do not exist) bring zeros.

constexpr unsigned OUTSIDE = 0x7ffffff0u;      // beyond the bytes of any buffer

__device__ __forceinline__ i32x4 buffer_of(const char* base, unsigned bytes) {
    const uint64_t at = (uint64_t)base;
    return i32x4{(int)(unsigned)at, (int)((unsigned)(at >> 32) & 0xffffu), (int)bytes, 0x00020000};
}

// (rows and channels that do not exist come as zeros)
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t bounded(const char* base, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(buffer_t buffer, unsigned from) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer, (int)from, 0, 0));
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

    // Step `s` of the depth (behind the last step: zeros): its buffer, and its fetches.  Steps come in order.
    __device__ __forceinline__ i32x4 step(int s) {
        if (TRANSPOSED) {
            const int rows = min(depth - s * 64, 64);
            return buffer_of(base + (int64_t)s * 64 * ld, rows > 0 ? (unsigned)((rows - 1) * ld) + bytes : 0u);
        }
        const int left = depth_bytes - s * 128;
#pragma unroll
        for (int i = 0; i < MINE; ++i) from[i] = chunk * 16 < left ? from[i] : OUTSIDE;
        return buffer_of(base + (int64_t)s * 128, left > 0 && bytes > 0 ? bytes - s * 128 : 0u);
    }
    __device__ __forceinline__ void fetch(i32x4 buffer, int i, unsigned to, int wave) const { fetch16(to + piece(i, wave) * 1024, from[i], buffer); }
};

constexpr int MT = 16;         // rows and columns of a matrix instruction
// What a lane gives one over MT rows (or columns) of an operand, 16 bytes at a time: of row lane % MT, chunk
// q * (64 / MT) + lane / MT of the step's eight.
__device__ __forceinline__ u32x4 direct_fragment(const char* tile, int first, int q) {
    const int lane = lane_id(), r = lane % MT;
    return *(const u32x4*)(tile + (first + r) * 128 + (((q * (WAVE / MT) + lane / MT) ^ ((r >> 1) & 7)) << 4));
}
// The same of a transposed tile, columns from `first` on: two transposing reads, each of which hands the lanes of a group of 16 the columns
// of the four 32-byte row pieces that the group reads.
template <int T>
__device__ __forceinline__ u32x4 transposed_fragment(const char* tile, int first, int q) {
    const int lane = lane_id(), j = (lane >> 2) & 3;
    const int row = (q * (WAVE / MT) + lane / MT) * 8 + j;
    const int granule = (first >> 4) ^ (j | ((lane / MT) & 1) << 2);
    const lds_byte* at = (const lds_byte*)(tile + row * (T * 2) + granule * 32 + (lane & 3) * 8);
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
__device__ __forceinline__ u32x4 fragment(const char* tile, int first, int q) {
    if (TRANSPOSED) return transposed_fragment<T>(tile, first, q);
    return direct_fragment(tile, first, q);
}

// MT x MT sums, four a lane, += BF16 columns x BF16 rows
__device__ __forceinline__ f32x4 multiply_add(u32x4 c, u32x4 r, f32x4 sums) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c), __builtin_bit_cast(bf16x8, r), sums, 0, 0, 0);
}
// ... e4m3: two chunks of each.  The instruction's scales are set to 1: those of the groups are not powers of two.  Of eight neighbouring
// products it keeps what lies above 2^-13 of the power of two below the largest (measured with single products), the sum is in 32 bits.
union Chunks {
    u32x4 half[2];
    i32x8 v;
};
__device__ __forceinline__ f32x4 multiply_add_fp8(const Chunks& c, const Chunks& r, f32x4 sums) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(c.v, r.v, sums, 0, 0, 0, 0, 0, 0);
}

// The compiler keeps what is in front of this in front.
#define KEEP_ORDER() __builtin_amdgcn_sched_barrier(0)

// ---- low-rank adapters: numbers of a tile ------------------------------------------------------------------

constexpr int NO_ADAPTER = 0x7fffffff;
__device__ __forceinline__ int adapter_of(const EpLoraArgs& l, int64_t first, int row, int valid) {
    const int a = row < valid ? l.adapter[first + row] : -1;
    return a >= 0 && a < l.num_adapters ? a : NO_ADAPTER;
}
__device__ __forceinline__ int wave_min(int v) {
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));      // row_shr:1
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));      // row_shr:2
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));      // row_shr:4
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));      // row_shr:8
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));      // row_bcast:15 to rows 1 and 3
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));      // row_bcast:31 to rows 2 and 3
    return __builtin_amdgcn_readlane(v, WAVE - 1);
}
// The smallest number above `last` of a tile's rows, a wave's lanes holding 64 rows' numbers each time.
template <int N>
__device__ __forceinline__ int next_adapter(const int (&of_row)[N], int last) {
    int v = NO_ADAPTER;
#pragma unroll
    for (int i = 0; i < N; ++i) v = min(v, of_row[i] > last ? of_row[i] : NO_ADAPTER);
    return wave_min(v);
}

// Eight ranks of a low-rank row.
__device__ __forceinline__ void low_ranks(const EpGemmArgs& a, int64_t row, int rank, f32x4 (&sum)[2]) {
    sum[0] = sum[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < a.lora.chunks; ++k) {
        const f32x4* const from = (const f32x4*)(a.lora.low + ((k * (int64_t)a.layout.num_rows + row) * a.lora.rank + rank));
        sum[0] += from[0];
        sum[1] += from[1];
    }
}

// ---- products ---------------------------------------------------------------------------------------------
//
// y[m] = W[e(m)] x[m]: one workgroup computes TM x TN of the output, WR x WC waves a part each, in 32 bits, over the whole depth (or its
// part of it), and rounds once, to BF16.  The matrix instruction's first operand is the output's columns, its second the rows: a lane then
// holds four neighbouring columns of one row.
//
// Few rows: the time is the weights', read once, with two or three steps of up to 512 workgroups under way (366 rows of 160 experts, 5120 channels
// to 2048: 508 us, 6.1 TB/s).
// Many rows: the matrix units' behind their operands.  A step of 256 x 256 is 64 KB from the L2 and 64 BF16 (32 FP8) matrix instructions a wave.
// BF16 has room for two stages of the rows and three of the columns in LDS: 16384 rows, 8192 x 8192 weights run at 1320 TFLOP/s with two of both
// and at 1400 with the third; the matrix units are busy 72 % of the time then, at the clock that power leaves them.
// FP8: a step is a group of channels, summed by itself in 32 bits and scaled with the row's and the block's scale as it is added (3 % of the time).
// Its scales take 4 KB of the LDS, which a third stage of the columns would need to the last byte: 98304 rows, 7168 channels to 4096, at 1700 TFLOP/s, the matrix units busy 46 % of the time and
// the waves waiting for a stage 27 %.  Fetching the step after that into the L2 made it slower, matrix instructions of 32 x 32 were level.
template <int TM, int TN, int WR, int WC, int SR, int SC, bool FP8, bool COLUMNS_T, bool ROWS_T, bool OUT32, bool LORA = false,
          bool LOW_RANK = false>
struct Gemm {
    static constexpr int WAVES = WR * WC, FM = TM / WR, FN = TN / WC, NR = FM / MT, NC = FN / MT;
    static constexpr int Q = MT / 8, HQ = Q / 2;      // fragments of a step and of half of one
    static constexpr int COLUMNS_BYTES = TN * 128, ROWS_BYTES = TM * 128, SF_BYTES = FP8 ? (TM < WAVE ? WAVE : TM) * 4 : 0;
    static constexpr int STAGES_BYTES = SC * COLUMNS_BYTES + SR * (ROWS_BYTES + SF_BYTES), ROWS_AT = SC * COLUMNS_BYTES, SF_AT = ROWS_AT + SR * ROWS_BYTES;
    static_assert(SC == SR || SC == SR + 1, "stages of the two operands");
    static constexpr int OUT_ELEM = OUT32 ? 4 : 2, OUT_ROW = FN * OUT_ELEM + 16, OUT_BYTES = WAVES * MT * OUT_ROW;
    static constexpr int BLOCKS = (TN + 127) / 128, TABLE = EP_EXPERT_MAX_DEPTH_FP8 / 128;
    static constexpr int TABLE_BYTES = FP8 ? BLOCKS * TABLE * 4 : 0;
    static constexpr int LDS_BYTES = STAGES_BYTES > OUT_BYTES ? STAGES_BYTES : OUT_BYTES;
    typedef TileFetch<TN, WAVES, COLUMNS_T> ColumnsFetch;
    typedef TileFetch<TM, WAVES, ROWS_T> RowsFetch;
    static constexpr int FETCHES = ColumnsFetch::MINE + RowsFetch::MINE + (FP8 ? 1 : 0);       // of a wave and step
    static constexpr int STEP = FP8 ? 128 : 64;
    // Results past the caches: those of large tiles are more than the L2 holds next to the operands (gradients of 64 experts' weights of
    // 1536 x 2560 from 7147 rows 250 -> 186 us, the FP8 product of 98304 rows 3402 -> 3340; the others are level).
    static constexpr bool STREAM = ROWS_T || TM >= 256;
    // fetches that a wave may have left when the rows and columns of a step have to be there, `ahead` steps before the newest
    static constexpr int pending(int ahead) { return ahead * FETCHES + (SC > SR ? ColumnsFetch::MINE : 0); }

    // rows .. rows + valid: what is computed, up to limit zeros are written; columns from column on
    __device__ __forceinline__ static void run(const EpGemmArgs& a, const char* rows, const char* columns, int valid, int limit,
                                               int num_columns, int depth, const float* rows_sf, const float* columns_sf, char* out,
                                               int64_t out_ld, int64_t first = 0, const char* up = nullptr, int numbers = NO_ADAPTER) {
        __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
        __shared__ float table[FP8 ? BLOCKS * TABLE : 1];
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
        if constexpr (LOW_RANK) {
            // columns: the adapters' matrices one below the other, lane j of `numbers` has the number of the j-th
            const EpLoraArgs& l = a.lora;
            const int base = __builtin_amdgcn_readlane(numbers, 0);
            int last = base;
#pragma unroll
            for (int i = 0; i < TN / 8; ++i) {
                const int n = __builtin_amdgcn_readlane(numbers, i);
                last = n != NO_ADAPTER ? n : last;
            }
            cf.bytes = (unsigned)((last - base) * l.down_adapter + (l.rank - 1) * l.down_ld) + depth * 2;
#pragma unroll
            for (int i = 0; i < ColumnsFetch::MINE; ++i) {
                const int r = ColumnsFetch::piece(i, wave) * 8, j = r / l.rank;      // (eight ranks of one adapter)
                const int n = __builtin_amdgcn_readlane(numbers, j);
                cf.from[i] = n == NO_ADAPTER ? OUTSIDE
                                             : (unsigned)((n - base) * l.down_adapter + (r - j * l.rank + (lane >> 3)) * l.down_ld) + cf.chunk * 16;
            }
        }
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
        // What a step leaves free is filled at once: with the rows SR steps on (and their scales), then with the columns SC steps on.
        struct Fetches {
            i32x4 columns, rows, sf;
            unsigned to_columns, to_rows, to_sf;
        };
        // (in three shares: between the matrix instructions, the scalar unit's time does not show)
        auto begin_share = [&](Fetches& f, int share, int s_rows, int slot_rows, int s_columns, int slot_columns) {
            if (share == 0) {
                f.rows = rf.step(s_rows);
                f.to_rows = lds0 + ROWS_AT + slot_rows * ROWS_BYTES;
            } else if (share == 1) {
                f.columns = cf.step(s_columns);
                f.to_columns = lds0 + slot_columns * COLUMNS_BYTES;
            } else if (FP8) {
                f.sf = buffer_of((const char*)(rows_sf + s_rows * a.rows_sf_col), s_rows < steps ? sf_bytes : 0u);
                f.to_sf = lds0 + SF_AT + slot_rows * SF_BYTES + (wave % SF_PIECES) * 256;
            }
        };
        auto begin_fetch = [&](int s_rows, int slot_rows, int s_columns, int slot_columns) {
            Fetches f;
#pragma unroll
            for (int share = 0; share < 3; ++share) begin_share(f, share, s_rows, slot_rows, s_columns, slot_columns);
            return f;
        };
        constexpr int OF_ROWS = RowsFetch::MINE + (FP8 ? 1 : 0);
        auto fetch_one = [&](const Fetches& f, int i) {
            if (i < RowsFetch::MINE) rf.fetch(f.rows, i, f.to_rows, wave);
            else if (i < OF_ROWS) fetch4(f.to_sf, sf_from, f.sf);
            else cf.fetch(f.columns, i - OF_ROWS, f.to_columns, wave);
        };
        auto fetch_all = [&](const Fetches& f, int from) {
#pragma unroll
            for (int i = 0; i < FETCHES; ++i)
                if (i >= from) fetch_one(f, i);
        };
        int slot_rows = 0, slot_columns = 0;
        auto next = [](int slot, int of) { return slot == of - 1 ? 0 : slot + 1; };

        // BF16: half a step is READS fragments and PRODUCTS matrix instructions.  While half a step is multiplied, the other half's
        // fragments are read, and the step after next is fetched, one instruction at a time between the products.
        constexpr int READS = HQ * (NC + NR), PRODUCTS = HQ * NC * NR;
        constexpr int READ_SPAN = (PRODUCTS * 5 + 7) / 8;
        auto read_one = [&](u32x4 (&c)[HQ][NC], u32x4 (&r)[HQ][NR], int slot_rows, int slot_columns, int half, int i) {
            const int q = i / (NC + NR), k = i - q * (NC + NR);
            if (k < NC) c[q][k] = fragment<COLUMNS_T, TN>(lds + slot_columns * COLUMNS_BYTES, first_column + k * MT, half * HQ + q);
            else r[q][k - NC] = fragment<ROWS_T, TM>(lds + ROWS_AT + slot_rows * ROWS_BYTES, first_row + (k - NC) * MT, half * HQ + q);
        };
        auto multiply_one = [&](const u32x4 (&c)[HQ][NC], const u32x4 (&r)[HQ][NR], int at) {
            const int q = at / (NR * NC), i = at / NC % NR, j = at % NC;
            acc[i][j] = multiply_add(c[q][j], r[q][i], acc[i][j]);
        };

        if (steps > 0) {
            if (SC > SR) fetch_all(begin_fetch(0, 0, 0, 0), OF_ROWS);
#pragma unroll
            for (int s = 0; s < SR - 1; ++s) fetch_all(begin_fetch(s, s, s + SC - SR, s + SC - SR), 0);
        }
        // The adapters' part: here for few adapters, behind the product for many.
        bool by_row = false;
        if (LORA) {
            int of_row[(TM + WAVE - 1) / WAVE];
#pragma unroll
            for (int i = 0; i < (TM + WAVE - 1) / WAVE; ++i) of_row[i] = i * WAVE + lane < TM ? adapter_of(a.lora, first, i * WAVE + lane, valid) : NO_ADAPTER;
            const int few = a.lora.rank / ceil_div(a.lora.rank, 32);
            int number = next_adapter(of_row, -1);
            for (int i = 0; i < few && number != NO_ADAPTER; ++i) number = next_adapter(of_row, number);
            by_row = number != NO_ADAPTER;
            if (!by_row) {
                add_adapters(a, lds + (SC - 1) * COLUMNS_BYTES, lds + ROWS_AT + (SR - 1) * ROWS_BYTES, of_row, first, valid, num_columns, up, [&] {
                    u32x4 c[HQ][NC], r[HQ][NR];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int i = 0; i < READS; ++i) read_one(c, r, SR - 1, SC - 1, half, i);
#pragma unroll
                        for (int i = 0; i < PRODUCTS; ++i) multiply_one(c, r, i);
                    }
                });
                // Rows of the tile without an adapter had zeros in its step.  Where it holds infinities or NaN these are no zeros any more, nor is
                // the rest of an infinite low-rank row: such a wave's rows take their own adapters only, behind the product.
                float probe = 0.f;
#pragma unroll
                for (int i = 0; i < NR * NC * 4; ++i) probe = __builtin_fmaf(acc[i / (NC * 4)][i / 4 % NC][i % 4], 0.f, probe);
                by_row = __ballot(probe != probe) != 0;
                if (by_row) {
#pragma unroll
                    for (int i = 0; i < NR * NC; ++i) acc[i / NC][i % NC] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
        }
        if (steps > 0 && !(FP8 && NR >= 4)) fetch_all(begin_fetch(SR - 1, SR - 1, SC - 1, SC - 1), 0);
        if constexpr (!FP8) {
            u32x4 c[2][HQ][NC], r[2][HQ][NR];
            // a wave whose rows do not exist only fetches: the other wave of its SIMD has the matrix unit to itself
            const bool active = first_row < valid;
            if (steps > 0) {
                wait_and_meet<pending(SR - 1)>();
#pragma unroll
                for (int i = 0; i < READS; ++i) read_one(c[0], r[0], 0, 0, 0, i);
            }
            for (int s = 0; s < steps; ++s) {
                Fetches f;
                if (active) {
#pragma unroll
                    for (int p = 0; p < PRODUCTS; ++p) {
#pragma unroll
                        for (int share = 0; share < 2; ++share)
                            if (p == (share + 1) * PRODUCTS / 3) begin_share(f, share, s + SR, slot_rows, s + SC, slot_columns);
                        // (early: they have arrived before the wave waits for the others)
#pragma unroll
                        for (int i = 0; i < READS; ++i)
                            if (i * READ_SPAN / READS == p) read_one(c[1], r[1], slot_rows, slot_columns, 1, i);
                        multiply_one(c[0], r[0], p);
                        KEEP_ORDER();
                    }
                }
                if (!active) f = begin_fetch(s + SR, slot_rows, s + SC, slot_columns);
                slot_rows = next(slot_rows, SR);
                slot_columns = next(slot_columns, SC);
                KEEP_ORDER();
                wait_and_meet<pending(SR - 2)>();
                KEEP_ORDER();
                if (active) {
#pragma unroll
                    for (int p = 0; p < PRODUCTS; ++p) {
#pragma unroll
                        for (int i = 0; i < FETCHES; ++i)
                            if (i * PRODUCTS / FETCHES == p) fetch_one(f, i);
#pragma unroll
                        for (int i = 0; i < READS; ++i)
                            if (i * PRODUCTS / READS == p) read_one(c[0], r[0], slot_rows, slot_columns, 0, i);
                        multiply_one(c[1], r[1], p);
                        KEEP_ORDER();
                    }
                } else {
                    fetch_all(f, 0);
                }
            }
        } else {
            // FP8: a step is one group of channels, whose products are summed by themselves, then scaled.
            const float* const of_block = &table[first_column / 128 * TABLE];
            auto read_columns = [&](Chunks (&c)[HQ], int slot_columns, int j) {
#pragma unroll
                for (int q = 0; q < Q; ++q) c[q / 2].half[q % 2] = direct_fragment(lds + slot_columns * COLUMNS_BYTES, first_column + j * MT, q);
            };
            auto read_row = [&](Chunks (&r)[HQ], float& scale, int slot_rows, int i) {
#pragma unroll
                for (int q = 0; q < Q; ++q) r[q / 2].half[q % 2] = direct_fragment(lds + ROWS_AT + slot_rows * ROWS_BYTES, first_row + i * MT, q);
                scale = ((const float*)(lds + SF_AT + slot_rows * SF_BYTES))[first_row + i * MT + lane % MT];
            };
            auto multiply = [&](const Chunks (&c)[HQ], const Chunks (&r)[HQ]) {
                f32x4 sum = {};
#pragma unroll
                for (int q = 0; q < HQ; ++q) sum = multiply_add_fp8(c[q], r[q], sum);
                return sum;
            };
            auto add_scaled = [&](f32x4& to, const f32x4& sum, float scale) {
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = __builtin_fmaf(sum[k], scale, to[k]);
            };
            if constexpr (NR >= 4) {
                // Rows of fragments are read two ahead; behind the last of them the waves meet, and while the last two rows are multiplied the
                // next step's first fragments are read.  The step after next is fetched meanwhile and in the next step's first rows.  Sums
                // are scaled DEPTH products behind.
                static_assert(NC >= 2, "a row's scale is needed until its last sum is scaled");
                constexpr int DEPTH = NC < 4 ? NC : 4, LAST = (NR - 2) * NC;
                const bool active = first_row < valid;
                constexpr int SPREAD = 2 * NC + (LAST < 2 * NC ? LAST : 2 * NC);
                auto fetch_at = [&](const Fetches& f, int place) {
#pragma unroll
                    for (int i = 0; i < FETCHES; ++i)
                        if (i * SPREAD / FETCHES == place) fetch_one(f, i);
                };
                // (of a step's fetches those in front of the next step's first row)
                constexpr int AT_ONCE = (2 * NC * FETCHES + SPREAD - 1) / SPREAD;
                Chunks c[NC][HQ], r[4][HQ];
                float scales[4];
                static_assert(SC == SR, "what is pending below");
                Fetches f;
                if (steps > 0) {
                    f = begin_fetch(SR - 1, SR - 1, SC - 1, SC - 1);
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) fetch_one(f, i);
                    if (!active) fetch_all(f, AT_ONCE);
                    wait_and_meet<(SR - 2) * FETCHES + AT_ONCE>();
#pragma unroll
                    for (int j = 0; j < NC; ++j) read_columns(c[j], 0, j);
                    read_row(r[0], scales[0], 0, 0);
                    read_row(r[1], scales[1], 0, 1);
                }
                for (int s = 0; s < steps; ++s) {
                    const float of_columns = of_block[s];
                    f32x4 sums[DEPTH];
                    // product p: of row i and column j; the last two rows column by column, so that the columns' fragments are free one by one
                    auto row_of = [](int p) { return p < LAST ? p / NC : NR - 2 + (p - LAST) % 2; };
                    auto column_of = [](int p) { return p < LAST ? p % NC : (p - LAST) / 2; };
                    auto scale_one = [&](int p) {
                        if (p >= 0) add_scaled(acc[row_of(p)][column_of(p)], sums[p % DEPTH], scales[row_of(p) % 4] * of_columns);
                    };
                    if (active) {
#pragma unroll
                        for (int p = 0; p < LAST; ++p) {
                            fetch_at(f, p + 2 * NC);
                            // (the fetches in flight are done with `f`)
                            constexpr int FROM = SPREAD - 2 * NC < LAST ? SPREAD - 2 * NC : LAST - 1;
#pragma unroll
                            for (int share = 0; share < 3; ++share)
                                if (p == FROM + share * (LAST - FROM) / 3) begin_share(f, share, s + SR, slot_rows, s + SC, slot_columns);
                            if (p % NC == 0 && p / NC + 2 < NR) read_row(r[(p / NC + 2) % 4], scales[(p / NC + 2) % 4], slot_rows, p / NC + 2);
                            scale_one(p - DEPTH);
                            sums[p % DEPTH] = multiply(c[column_of(p)], r[row_of(p) % 4]);
                            KEEP_ORDER();
                        }
                    }
                    if (!active) f = begin_fetch(s + SR, slot_rows, s + SC, slot_columns);
                    slot_rows = next(slot_rows, SR);
                    slot_columns = next(slot_columns, SC);
                    KEEP_ORDER();
                    wait_and_meet<pending(SR - 2)>();
                    KEEP_ORDER();
                    if (active) {
#pragma unroll
                        for (int p = LAST; p < NR * NC; ++p) {
                            fetch_at(f, p - LAST);
                            scale_one(p - DEPTH);
                            sums[p % DEPTH] = multiply(c[column_of(p)], r[row_of(p) % 4]);
                            if ((p - LAST) % 2 == 1) read_columns(c[column_of(p)], slot_columns, column_of(p));
                            if (p == LAST + 1) read_row(r[0], scales[0], slot_rows, 0);
                            if (p == LAST + 3) read_row(r[1], scales[1], slot_rows, 1);
                            KEEP_ORDER();
                        }
#pragma unroll
                        for (int p = NR * NC - DEPTH; p < NR * NC; ++p) scale_one(p);
                    } else {
                        fetch_all(f, 0);
                    }
                }
            } else {
                int free_rows = 0, free_columns = 0;
                for (int s = 0; s < steps; ++s) {
                    wait_and_meet<pending(SR - 2)>();
                    if (s > 0) fetch_all(begin_fetch(s - 1 + SR, free_rows, s - 1 + SC, free_columns), 0);
                    const float of_columns = of_block[s];
                    Chunks c[NC][HQ];
#pragma unroll
                    for (int j = 0; j < NC; ++j) read_columns(c[j], slot_columns, j);
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        Chunks r[HQ];
                        float scale;
                        read_row(r, scale, slot_rows, i);
#pragma unroll
                        for (int j = 0; j < NC; ++j) add_scaled(acc[i][j], multiply(c[j], r), scale * of_columns);
                    }
                    free_rows = slot_rows, free_columns = slot_columns;
                    slot_rows = next(slot_rows, SR);
                    slot_columns = next(slot_columns, SC);
                }
            }
        }
        wait_and_meet<0>();      // (the last fetches, of zeros, land in LDS too)
        if (LORA && by_row) add_adapters_by_row(a, acc, up, first, valid, first_row, first_column, num_columns);

        // MT rows of a wave's part at a time through LDS, to leave as whole lines
        char* const mine = lds + wave * MT * OUT_ROW;
        constexpr int LANES = FN * OUT_ELEM / 16, PASS = WAVE / LANES;      // lanes of a row, rows of a store
        const int piece = lane % LANES, column = first_column + piece * (16 / OUT_ELEM);
        int segment = 0, of_segment = NO_ADAPTER;      // of the adapters' ranks: which adapter's this lane stores
        if constexpr (LOW_RANK) {
            segment = column / a.lora.rank;
            of_segment = __shfl(numbers, segment);
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                // four neighbouring columns of row lane % MT
                char* const to = mine + lane % MT * OUT_ROW + (j * MT + lane / MT * 4) * OUT_ELEM;
                if (OUT32) *(f32x4*)to = acc[i][j];
                else *(bf16x4*)to = __builtin_convertvector(acc[i][j], bf16x4);
            }
            asm volatile("" ::: "memory");
#pragma unroll
            for (int p = 0; p < MT; p += PASS) {
                const int in = p + lane / LANES, r = first_row + i * MT + in;
                if (in >= MT || r >= limit || column >= num_columns) continue;
                u32x4 v = *(const u32x4*)(mine + in * OUT_ROW + piece * 16);
                if (r >= valid) v = u32x4{0u, 0u, 0u, 0u};
                u32x4* const to = (u32x4*)(out + (r * out_ld + column) * OUT_ELEM);
                if constexpr (LOW_RANK) {
                    // only the rows that have the adapter
                    const int mine = adapter_of(a.lora, first, r, valid);
                    if (mine == NO_ADAPTER || mine != of_segment) continue;
                    const float scale = a.lora.scales != nullptr ? a.lora.scales[mine] : 1.0f;
                    *(f32x4*)((float*)out + (int64_t)r * a.lora.rank + (column - segment * a.lora.rank)) = __builtin_bit_cast(f32x4, v) * scale;
                    continue;
                }
                if (OUT32 && a.accumulate && a.partial == nullptr) {
                    const f32x4 sum = *(const f32x4*)to + __builtin_bit_cast(f32x4, v);
                    v = __builtin_bit_cast(u32x4, sum);
                }
                store<STREAM>(to, v);
            }
            asm volatile("" ::: "memory");
        }
    }

    // Few adapters: in front of the product's first step and in the LDS of its last stage, while the first ones are on their way.  For
    // every adapter that rows of the tile have, 32 ranks at a time, a step of 64 channels.  The low-rank rows are sums in 32 bits; they
    // go in as two BF16, the rounded value and the rest, against the same column of `up` twice, which keeps 2^-17 of them.
    // A step is 4 to 10 us of a tile, as much as about one rank of add_adapters_by_row.  8192 rows, 4096 x 4096 weights, in us, this / by row:
    // 16 ranks, 4 adapters 239 / 305, 16 355 / 357, 64 680 / 486; 64 ranks, 6 adapters 350 / 726, 12 (24 steps) 491 / 820.
    template <typename Multiply>
    __device__ __forceinline__ static void add_adapters(const EpGemmArgs& a, char* to_columns, char* to_rows, const int (&of_row)[(TM + WAVE - 1) / WAVE],
                                                        int64_t first, int valid, int num_columns, const char* up, Multiply multiply) {
        constexpr int THREADS = WAVES * WAVE, MINE = (TM * 4 + THREADS - 1) / THREADS;
        const EpLoraArgs& l = a.lora;
        int mine[MINE];           // adapters of the rows that this thread brings
#pragma unroll
        for (int n = 0; n < MINE; ++n) {
            const int r = (threadIdx.x + n * THREADS) >> 2;
            mine[n] = r < TM ? adapter_of(l, first, r, valid) : NO_ADAPTER;
        }
        for (int number = next_adapter(of_row, -1); number != NO_ADAPTER; number = next_adapter(of_row, number)) {
            for (int r0 = 0; r0 < l.rank; r0 += 32) {
#pragma unroll
                for (int n = 0; n < MINE; ++n) {
                    const int i = threadIdx.x + n * THREADS, r = i >> 2, c = i & 3, rank = r0 + c * 8;
                    if (r >= TM) continue;
                    bf16x8 high = {}, rest = {};
                    if (mine[n] == number && rank < l.rank) {
                        f32x4 sum[2];
                        low_ranks(a, first + r, rank, sum);
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
                multiply();
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
        }
    }
    // Many adapters: behind the product, lane by lane with the row's own adapter, eight ranks at a time and four columns of a sum together.  The
    // time goes by the ranks and not by the number of adapters.
    __device__ __forceinline__ static void add_adapters_by_row(const EpGemmArgs& a, f32x4 (&acc)[NR][NC], const char* up, int64_t first,
                                                               int valid, int first_row, int first_column, int num_columns) {
        const EpLoraArgs& l = a.lora;
        const int lane = lane_id();
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int row = first_row + i * MT + lane % MT, number = adapter_of(l, first, row, valid);
            if (number == NO_ADAPTER) continue;
            const char* const mine = up + number * l.up_adapter;
            for (int rank = 0; rank < l.rank; rank += 8) {
                f32x4 low[2];
                low_ranks(a, first + row, rank, low);
#pragma unroll
                for (int j = 0; j < NC; ++j) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int column = first_column + j * MT + lane / MT * 4 + g;
                        if (column >= num_columns) continue;
                        const bf16x8 w = *(const bf16x8*)(mine + column * l.up_ld + rank * 2);
                        float sum = acc[i][j][g];
#pragma unroll
                        for (int k = 0; k < 8; ++k) sum = __builtin_fmaf(low[k >> 2][k & 3], (float)w[k], sum);
                        acc[i][j][g] = sum;
                    }
                }
            }
        }
    }

    // Rows of the layout times the weights of their expert: out[r, c] = sum_d rows[r, d] columns[e(r)][c, d].  SPLIT: of a part of
    // the depth, in 32 bits; ep_sum_splits adds the parts.
    template <bool SPLIT>
    __device__ __forceinline__ static void rows_kernel(const EpGemmArgs& a, int group, int block = blockIdx.x) {
        const int row_tiles = count_row_tiles<TM>(a.layout);
        int row, column, part = 0;
        if (!tile_of_block(block, row_tiles, SPLIT ? a.column_tiles * a.splits : a.column_tiles, group, row, column)) return;
        const RowTile t = find_row_tile<TM>(a.layout, row);
        int64_t d0 = 0;
        int depth = a.depth, limit = t.limit;
        char* out = a.out;
        if (SPLIT) {
            part = column % a.splits;
            column /= a.splits;
            d0 = (int64_t)part * a.split_depth;
            depth = min(a.split_depth, depth - (int)d0);
            limit = t.valid;
            out = (char*)(a.partial + (int64_t)part * a.layout.num_rows * a.num_columns);
        }
        const int64_t c0 = (int64_t)column * TN, out_ld = SPLIT ? a.num_columns : a.out_ld;
        const char* const columns = a.columns + t.expert * a.columns_expert +
                                    (COLUMNS_T ? c0 * 2 + d0 * a.columns_ld : c0 * a.columns_ld + d0 * (FP8 ? 1 : 2));
        run(a, a.rows + t.first * a.rows_ld + d0 * (FP8 ? 1 : 2), columns, t.valid, limit, a.num_columns - (int)c0, depth,
            a.rows_sf + (FP8 ? t.first * a.rows_sf_row + d0 / 128 * a.rows_sf_col : 0),
            a.columns_sf + (FP8 ? t.expert * a.columns_sf_expert + c0 / 128 * a.columns_sf_row + d0 / 128 * a.columns_sf_col : 0),
            out + (t.first * out_ld + c0) * OUT_ELEM, out_ld, t.first,
            LORA ? a.lora.up + t.expert * a.lora.up_expert + c0 * a.lora.up_ld : nullptr);
    }

    // Gradient of an expert's weights: out[e][r, c] = sum over the expert's rows d of rows[d, r] columns[d, c]
    // SPLIT: of a part of the expert's rows; ep_sum_weights adds the parts.
    template <bool SPLIT>
    __device__ __forceinline__ static void weights_kernel(const EpGemmArgs& a, int group) {
        int row, column, part = 0;
        const int column_tiles = SPLIT ? a.column_tiles * a.splits : a.column_tiles;
        // Every XCD has a stretch of each expert's tiles: experts have as many rows as they are popular.  Eight experts' weights of 2048 x 4096
        // from 16000 rows, level 204 us (an XCD with an expert to itself 210), of Zipf(1.2) popularity 216 (542); 64 experts' of 1536 x 2560 from
        // 28000 rows, level 250 (235), of Zipf(0.6) 254 (278).
        const int of_expert = align_up(a.row_tiles * column_tiles, 8), e = blockIdx.x / of_expert;
        if (e >= a.layout.num_experts || !tile_of_block(blockIdx.x - e * of_expert, a.row_tiles, column_tiles, group, row, column)) return;
        if (SPLIT) {
            part = column % a.splits;
            column /= a.splits;
        }
        const int r0 = row * TM, c0 = column * TN;
        const ExpertRows in = rows_of_expert(a.layout, e);
        int count = uniform(in.count);
        int64_t start = uniform(in.start);
        char* out = a.out;
        int64_t out_expert = a.out_expert, out_ld = a.out_ld;
        if (SPLIT) {
            const int share = align_up(ceil_div(count, a.splits), STEP), from = min(part * share, count);
            start += from;
            count = min(count - from, share);
            out_ld = a.num_columns;
            out_expert = (int64_t)a.num_out_rows * out_ld;
            out = (char*)(a.partial + (int64_t)part * a.layout.num_experts * out_expert);
        }
        const int out_rows = min(a.num_out_rows - r0, TM);
        run(a, a.rows + start * a.rows_ld + (int64_t)r0 * 2, a.columns + start * a.columns_ld + (int64_t)c0 * 2, out_rows, out_rows,
            a.num_columns - c0, count, nullptr, nullptr, out + (e * out_expert + (int64_t)r0 * out_ld + c0) * OUT_ELEM, out_ld);
    }
};

#define EP_GEMM_ROWS(NAME, TM, TN, WR, WC, SR, SC, FP8, COLUMNS_T, GROUP)                                         \
    extern "C" __global__ __launch_bounds__(WR* WC* WAVE) void NAME(EpGemmArgs a) {                                   \
        Gemm<TM, TN, WR, WC, SR, SC, FP8, COLUMNS_T, false, false>::rows_kernel<false>(a, GROUP);                 \
    }
typedef Gemm<64, 128, 2, 2, 3, 3, false, false, false, true> SplitBf16;
typedef Gemm<64, 128, 2, 2, 3, 3, true, false, false, true> SplitFp8;
extern "C" __global__ __launch_bounds__(256) void ep_grouped_split_bf16(EpGemmArgs a) { SplitBf16::rows_kernel<true>(a, 1); }
extern "C" __global__ __launch_bounds__(256) void ep_grouped_split_fp8(EpGemmArgs a) { SplitFp8::rows_kernel<true>(a, 1); }
#define EP_GEMM_LORA(NAME, TM, TN, WR, WC, SR, SC, GROUP)                                                         \
    extern "C" __global__ __launch_bounds__(WR* WC* WAVE) void NAME(EpGemmArgs a) {                                   \
        Gemm<TM, TN, WR, WC, SR, SC, false, false, false, false, true>::rows_kernel<false>(a, GROUP);             \
    }
#define EP_GEMM_WEIGHTS(NAME, TM, TN, WR, WC, SR, SC, OUT32, SPLIT, GROUP)                                        \
    extern "C" __global__ __launch_bounds__(WR* WC* WAVE) void NAME(EpGemmArgs a) {                                   \
        Gemm<TM, TN, WR, WC, SR, SC, false, true, true, OUT32>::weights_kernel<SPLIT>(a, GROUP);                         \
    }
EP_GEMM_ROWS(ep_grouped_bf16_32x64, 32, 64, 1, 4, 4, 4, false, false, 4)
EP_GEMM_ROWS(ep_grouped_bf16_64x128, 64, 128, 2, 2, 3, 3, false, false, 1)
EP_GEMM_ROWS(ep_grouped_bf16_64x256, 64, 256, 1, 8, 3, 3, false, false, 1)
EP_GEMM_ROWS(ep_grouped_bf16_128x256, 128, 256, 2, 4, 3, 3, false, false, 1)
EP_GEMM_ROWS(ep_grouped_bf16_256x256, 256, 256, 4, 2, 2, 3, false, false, 8)
EP_GEMM_ROWS(ep_grouped_fp8_32x64, 32, 64, 1, 4, 4, 4, true, false, 4)
EP_GEMM_ROWS(ep_grouped_fp8_64x128, 64, 128, 2, 2, 3, 3, true, false, 1)
EP_GEMM_ROWS(ep_grouped_fp8_64x256, 64, 256, 1, 8, 3, 3, true, false, 1)
EP_GEMM_ROWS(ep_grouped_fp8_128x256, 128, 256, 2, 4, 3, 3, true, false, 1)
EP_GEMM_ROWS(ep_grouped_fp8_256x256, 256, 256, 2, 4, 2, 2, true, false, 8)
EP_GEMM_ROWS(ep_grouped_transposed_64x128, 64, 128, 2, 2, 3, 3, false, true, 1)
EP_GEMM_ROWS(ep_grouped_transposed_64x256, 64, 256, 1, 8, 3, 3, false, true, 1)
EP_GEMM_ROWS(ep_grouped_transposed_128x256, 128, 256, 2, 4, 3, 3, false, true, 1)
EP_GEMM_ROWS(ep_grouped_transposed_256x256, 256, 256, 2, 4, 2, 3, false, true, 8)
EP_GEMM_LORA(ep_grouped_lora_32x64, 32, 64, 1, 4, 4, 4, 4)
EP_GEMM_LORA(ep_grouped_lora_64x128, 64, 128, 2, 2, 3, 3, 1)
EP_GEMM_LORA(ep_grouped_lora_64x256, 64, 256, 1, 8, 3, 3, 1)
EP_GEMM_LORA(ep_grouped_lora_128x256, 128, 256, 2, 4, 3, 3, 1)
EP_GEMM_LORA(ep_grouped_lora_256x256, 256, 256, 4, 2, 2, 3, 8)
EP_GEMM_WEIGHTS(ep_grouped_weights_bf16_128x128, 128, 128, 2, 4, 2, 2, false, false, 4)
EP_GEMM_WEIGHTS(ep_grouped_weights_bf16_256x256, 256, 256, 2, 4, 2, 3, false, false, 4)
EP_GEMM_WEIGHTS(ep_grouped_weights_f32_128x128, 128, 128, 2, 4, 2, 2, true, false, 4)
EP_GEMM_WEIGHTS(ep_grouped_weights_f32_256x256, 256, 256, 2, 4, 2, 3, true, false, 4)
EP_GEMM_WEIGHTS(ep_grouped_split_weights, 128, 128, 2, 4, 2, 2, true, true, 4)

// ---- low-rank adapters: rows times the first matrix ---------------------------------------------------------
//
// low[chunk][r] = scale[a] * sum over the chunk's channels of down[a][e] rows[r].  A workgroup has 16 rows of an expert, a chunk of the
// depth, which its four waves share 64 or 128 channels at a time, and every `slots`-th of the adapters that its rows have: all rows are
// multiplied with an adapter's matrix, and the rows that have it keep what they get.  Operands go from memory straight to
// registers: nothing is used twice but by the neighbouring waves, out of the caches.  Beside a product in parts it hides behind the weights: 61 rows
// of 32 adapters, 7168 channels to 4096, 16 ranks: 23.5 us, the product alone 17.2.
template <int RANKS>
__device__ __forceinline__ void lora_down_body(const EpGemmArgs& a, int block) {
    constexpr int ROWS = 16, NK = RANKS / 16, PARTS = RANKS > 32 ? 2 : 4;
    __shared__ __attribute__((aligned(16))) float sums[4][ROWS][RANKS + 4];
    const EpLoraArgs& l = a.lora;
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    int at = block;
    const int slot = at % l.slots;
    at /= l.slots;
    const int chunk = at % l.chunks, tile = at / l.chunks;
    const RowTile t = find_row_tile<ROWS>(a.layout, tile);
    if (t.valid <= 0) return;
    // every wave: the rows' adapters, and of each the first row that has it
    const int of_row = lane < ROWS ? adapter_of(l, t.first, lane, t.valid) : NO_ADAPTER;
    bool leads = of_row != NO_ADAPTER;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) leads = leads && !(lane > i && __builtin_amdgcn_readlane(of_row, i) == of_row);
    const int begin = chunk * l.chunk_depth, end = min(begin + l.chunk_depth, a.depth);
    const buffer_t x_buffer = bounded(a.rows + t.first * a.rows_ld, (unsigned)((t.valid - 1) * a.rows_ld) + a.depth * 2);
    int n = 0;
    for (uint64_t leaders = __ballot(leads); leaders != 0; leaders &= leaders - 1) {
        if (n++ % l.slots != slot) continue;
        const int number = __builtin_amdgcn_readlane(of_row, __builtin_ctzll(leaders));
        const buffer_t w_buffer = bounded(l.down + number * l.down_adapter + t.expert * l.down_expert, (unsigned)((l.rank - 1) * l.down_ld) + a.depth * 2);
        f32x4 acc[NK];
#pragma unroll
        for (int j = 0; j < NK; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (a turn's operands are on their way while the one before is multiplied)
        u32x4 x[2][PARTS], w[2][PARTS][NK];
        auto load = [&](int k0, u32x4 (&x)[PARTS], u32x4 (&w)[PARTS][NK]) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const int k = k0 + p * 32 + (lane >> 4) * 8;
                x[p] = load16(x_buffer, k < end ? (unsigned)((lane & 15) * a.rows_ld) + k * 2 : OUTSIDE);
#pragma unroll
                for (int j = 0; j < NK; ++j) w[p][j] = load16(w_buffer, k < end ? (unsigned)((j * 16 + (lane & 15)) * l.down_ld) + k * 2 : OUTSIDE);
            }
        };
        auto multiply = [&](const u32x4 (&x)[PARTS], const u32x4 (&w)[PARTS][NK]) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int j = 0; j < NK; ++j) acc[j] = multiply_add(w[p][j], x[p], acc[j]);
        };
        constexpr int TURN = 128 * PARTS;
        const int k0 = begin + wave * 32 * PARTS;
        load(k0, x[0], w[0]);
        for (int k = k0; k < end; k += 2 * TURN) {
            load(k + TURN, x[1], w[1]);
            multiply(x[0], w[0]);
            load(k + 2 * TURN, x[0], w[0]);
            multiply(x[1], w[1]);
        }
#pragma unroll
        for (int j = 0; j < NK; ++j) *(f32x4*)&sums[wave][lane & 15][j * 16 + (lane >> 4) * 4] = acc[j];
        __syncthreads();
        const float scale = l.scales != nullptr ? l.scales[number] : 1.0f;
        for (int i = threadIdx.x; i < ROWS * (RANKS / 4); i += 256) {
            const int r = i / (RANKS / 4), c = (i - r * (RANKS / 4)) * 4;
            if (__shfl(of_row, r) != number || c >= l.rank) continue;
            const f32x4 sum = (*(const f32x4*)&sums[0][r][c] + *(const f32x4*)&sums[1][r][c]) + (*(const f32x4*)&sums[2][r][c] + *(const f32x4*)&sums[3][r][c]);
            *(f32x4*)(l.low + (((int64_t)chunk * a.layout.num_rows + t.first + r) * l.rank + c)) = sum * scale;
        }
        __syncthreads();
    }
}
#define EP_LORA_DOWN(RANKS) \
    extern "C" __global__ __launch_bounds__(256) void ep_lora_down_##RANKS(EpGemmArgs a) { lora_down_body<RANKS>(a, blockIdx.x); }
EP_LORA_DOWN(16)
EP_LORA_DOWN(32)
EP_LORA_DOWN(64)

// Many rows: the same sums as a product of 64 rows with the matrices of as many adapters as have 64 ranks together.
typedef Gemm<64, 64, 4, 1, 3, 3, false, false, false, true, false, true> LowRank;
extern "C" __global__ __launch_bounds__(256) void ep_lora_down_rows(EpGemmArgs a) {
    const EpLoraArgs& l = a.lora;
    const int chunk = blockIdx.x % l.chunks;
    const RowTile t = find_row_tile<64>(a.layout, blockIdx.x / l.chunks);
    if (t.valid <= 0) return;
    const int of_row[1] = {adapter_of(l, t.first, lane_id(), t.valid)};
    const int64_t begin = (int64_t)chunk * l.chunk_depth;
    const int depth = min(l.chunk_depth, a.depth - (int)begin);
    EpGemmArgs low = a;
    low.columns_ld = l.down_ld;
    int number = next_adapter(of_row, -1);
    while (number != NO_ADAPTER) {
        const int first = number;
        int numbers = NO_ADAPTER, count = 0;
        for (; count < l.together && number != NO_ADAPTER; ++count) {
            if (lane_id() == count) numbers = number;
            number = next_adapter(of_row, number);
        }
        LowRank::run(low, a.rows + t.first * a.rows_ld + begin * 2, l.down + first * l.down_adapter + t.expert * l.down_expert + begin * 2, t.valid, t.valid,
                     count * l.rank, depth, nullptr, nullptr, (char*)(l.low + ((int64_t)chunk * a.layout.num_rows + t.first) * l.rank), 0, t.first, nullptr,
                     numbers);
        __syncthreads();          // (the next ones' fetches go where rows may still be on their way out)
    }
}

// Few tiles: the product in parts of the depth does not need the low-rank rows, ep_sum_splits joins both.  One launch for the two.
#define EP_LORA_SPLIT(RANKS)                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void ep_grouped_split_lora_##RANKS(EpGemmArgs a) {                   \
        const int behind = (int)blockIdx.x - ((int)gridDim.x - a.lora.blocks);                                        \
        if (behind < 0) SplitBf16::rows_kernel<true>(a, 1, blockIdx.x);                                               \
        else lora_down_body<RANKS>(a, behind);                                                                    \
    }
EP_LORA_SPLIT(16)
EP_LORA_SPLIT(32)
EP_LORA_SPLIT(64)

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

// ---- parts of a depth, added -----------------------------------------------------------------------------

// Always in the same order: the parts are in 32 bits and rounded once, behind the sum.  Of rows: a lane has eight columns of one, and adds what the
// row's adapter makes of its low-rank row.
template <bool LORA>
__device__ __forceinline__ void sum_splits_body(const EpGemmArgs& a) {
    const int vectors = a.num_columns >> 3, per_row = ceil_div(vectors, WAVE);
    const int64_t task = (int64_t)blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);
    const int row = uniform((int)(task / per_row)), v = (int)(task - (int64_t)row * per_row) * WAVE + lane_id();
    if (row >= a.layout.num_rows) return;
    int expert = 0;
    const int kind = kind_of_row(a.layout, row, expert);
    if (kind == 0) return;
    f32x4 sum[2] = {};
    if (kind == 2) {
        const int number = LORA ? uniform(adapter_of(a.lora, row, 0, 1)) : NO_ADAPTER;
        // (a lane has a rank of the low-rank row)
        float low = 0.f;
        if (LORA && number != NO_ADAPTER && lane_id() < a.lora.rank) {
#pragma unroll 4
            for (int k = 0; k < a.lora.chunks; ++k) low += a.lora.low[(k * (int64_t)a.layout.num_rows + row) * a.lora.rank + lane_id()];
        }
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s) {
            const f32x4* const from = (const f32x4*)(a.partial + ((int64_t)s * a.layout.num_rows + row) * a.num_columns) + 2 * (v < vectors ? v : 0);
            sum[0] += from[0];
            sum[1] += from[1];
        }
        if (LORA && number != NO_ADAPTER) {
            const char* const up = a.lora.up + number * a.lora.up_adapter + expert * a.lora.up_expert + (v < vectors ? v : 0) * 8 * a.lora.up_ld;
            for (int rank = 0; rank < a.lora.rank; rank += 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bf16x8 w = *(const bf16x8*)(up + i * a.lora.up_ld + rank * 2);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float of_rank = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(low), rank + k));
                        sum[i >> 2][i & 3] = __builtin_fmaf(of_rank, (float)w[k], sum[i >> 2][i & 3]);
                    }
                }
            }
        }
    }
    if (v >= vectors) return;
    bf16x8 out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (__bf16)sum[i >> 2][i & 3];
    *((bf16x8*)(a.out + row * a.out_ld * 2) + v) = out;
}
// Parts of an expert's rows: a lane has four weights.
template <bool OUT32>
__device__ __forceinline__ void sum_weights_body(const EpGemmArgs& a) {
    const int64_t of_expert = (int64_t)a.num_out_rows * a.num_columns, all = of_expert * a.layout.num_experts;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= all) return;
    f32x4 sum = {};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) sum += *(const f32x4*)(a.partial + s * all + at);
    const int64_t e = at / of_expert, in = at - e * of_expert, r = in / a.num_columns, c = in - r * a.num_columns;
    const int64_t to = e * a.out_expert + r * a.out_ld + c;
    if (OUT32) {
        f32x4* const out = (f32x4*)((float*)a.out + to);
        *out = a.accumulate ? *out + sum : sum;
    } else {
        *(bf16x4*)((__bf16*)a.out + to) = __builtin_convertvector(sum, bf16x4);
    }
}
extern "C" __global__ __launch_bounds__(256) void ep_sum_weights_bf16(EpGemmArgs a) { sum_weights_body<false>(a); }
extern "C" __global__ __launch_bounds__(256) void ep_sum_weights_f32(EpGemmArgs a) { sum_weights_body<true>(a); }

extern "C" __global__ __launch_bounds__(256) void ep_sum_splits(EpGemmArgs a) { sum_splits_body<false>(a); }
extern "C" __global__ __launch_bounds__(256) void ep_sum_splits_lora(EpGemmArgs a) { sum_splits_body<true>(a); }

// ---- the gated activation -----------------------------------------------------------------------------
//
// out = gate * sigmoid(gate) * up * weight in 32 bits, rounded once; a lane has eight channels, a wave 512 of a row, and 16 lanes a group of
// the quantiser, whose largest value goes round them without LDS.  Bound by memory, everything past the caches: 98304 rows of 2048 channels to e4m3
// in 172 us, 5.8 TB/s.  A wave takes several parts of a row when there are rows enough, the next one's operands on their way meanwhile: with one
// part a wave 180 us (BF16 190 and 198).

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
// 1 / (1 + exp(-x)).  The hardware's exponential (of two) and reciprocal are each a unit in the last place off, and a large gate's argument
// loses some to its rounding: of 201 million e4m3 values (98304 x 2048) 398 fall on a border's other side than in 64 bits, and 394 with
// the rounding given back as a factor and a step of Newton's behind the reciprocal, for 192 us instead of 172.
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}

__device__ __forceinline__ unsigned row16_umax(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x128, 0xf, 0xf, false));  // row_ror:8
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x124, 0xf, 0xf, false));  // row_ror:4
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x122, 0xf, 0xf, false));  // row_ror:2
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x121, 0xf, 0xf, false));  // row_ror:1
    return x;
}

template <bool FP8>
__device__ __forceinline__ void swiglu_body(const EpSwigluArgs& a) {
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int64_t task = (int64_t)blockIdx.x * 4 + wave;
    const int per_row = ceil_div(a.num_parts, a.parts_per_task);
    const int row = uniform((int)(task / per_row)), first = uniform((int)(task - (int64_t)row * per_row)) * a.parts_per_task;
    if (row >= a.layout.num_rows) return;
    const u32x4* const h = (const u32x4*)(a.h + (int64_t)row * a.h_ld * 2);
    // (the ups begin at a multiple of eight channels as the gates do)
    const int vectors = a.channels >> 3, end = min(first + a.parts_per_task, a.num_parts);
    // the first part is on its way while the row is looked up
    u32x4 next[2];
    auto fetch = [&](int part) {
        const int v = part * WAVE + lane;
        if (v >= vectors) return;
        next[0] = __builtin_nontemporal_load(h + v);
        next[1] = __builtin_nontemporal_load(h + vectors + v);
    };
    fetch(first);
    const float of_row = a.weights != nullptr ? a.weights[row] : 1.0f;
    int expert;
    const int kind = kind_of_row(a.layout, row, expert);
    if (kind == 0) return;
    for (int part = first; part < end; ++part) {
        const int v = part * WAVE + lane;
        const bool live = v < vectors;
        float out[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const u32x4 now[2] = {next[0], next[1]};
        if (part + 1 < end) fetch(part + 1);
        if (live && kind == 2) {
            float gate[8], up[8];
            widen(now[0], gate);
            widen(now[1], up);
#pragma unroll
            for (int i = 0; i < 8; ++i) out[i] = gate[i] * sigmoid(gate[i]) * up[i] * of_row;
        }
        if constexpr (!FP8) {
            if (live) store<true>((u32x4*)(a.out + (int64_t)row * a.out_ld * 2) + v, round_bf16(out));
        } else {
            // the quantiser of the dispatch, of the unrounded values
            unsigned bits = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) bits = max(bits, __float_as_uint(out[i]) & 0x7fffffffu);
            const float m = __uint_as_float(row16_umax(bits));
            const float amax = m < 1e-4f ? 1e-4f : m;
            const float inverse = 448.0f / amax;
            unsigned q[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int w = __builtin_amdgcn_cvt_pk_fp8_f32(out[4 * i] * inverse, out[4 * i + 1] * inverse, 0, false);
                q[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(out[4 * i + 2] * inverse, out[4 * i + 3] * inverse, w, true);
            }
            if (amax != amax) q[0] = q[1] = 0x7f7f7f7fu;
            if (!live) continue;
            store<true>((u32x2*)(a.out + (int64_t)row * a.out_ld) + v, u32x2{q[0], q[1]});
            if ((lane & 15) == 0) a.sf[(int64_t)row * a.sf_row + (int64_t)(v >> 4) * a.sf_col] = kind == 2 ? amax / 448.0f : 0.0f;
        }
    }
}
extern "C" __global__ __launch_bounds__(256) void ep_swiglu_bf16(EpSwigluArgs a) { swiglu_body<false>(a); }
extern "C" __global__ __launch_bounds__(256) void ep_swiglu_fp8(EpSwigluArgs a) { swiglu_body<true>(a); }

// Gradients: a wave has a row, whose gate weight's gradient is the sum over its channels.
extern "C" __global__ __launch_bounds__(256) void ep_swiglu_gradients(EpSwigluArgs a) {
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    const int64_t task = (int64_t)blockIdx.x * 4 + wave;
    if (task >= a.layout.num_rows) return;
    int expert;
    const int row = (int)task, kind = kind_of_row(a.layout, row, expert);
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
            widen(__builtin_nontemporal_load(h + v), gate);
            widen(__builtin_nontemporal_load(h + vectors + v), up);
            widen(__builtin_nontemporal_load(grad_out + v), grad);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = sigmoid(gate[i]), silu = gate[i] * s;
                of_weight = __builtin_fmaf(grad[i] * silu, up[i], of_weight);
                const float g = grad[i] * weight;
                of_up[i] = g * silu;
                of_gate[i] = g * up[i] * s * (1.0f + gate[i] * (1.0f - s));
            }
        }
        store<true>(grad_h + v, round_bf16(of_gate));
        store<true>(grad_h + vectors + v, round_bf16(of_up));
    }
    if (a.grad_weights == nullptr) return;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) of_weight += __shfl_xor(of_weight, d);
    if (lane == 0) a.grad_weights[row] = of_weight;
}
