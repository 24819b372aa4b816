// Host side of the experts' computation (ep_experts.hip): argument contracts of its C entries and the launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <mutex>

#include "ep_expert_args.h"
#include "ep_host.h"

namespace {

// Tiles of the products: output rows, output columns, threads of a workgroup.
struct Tile {
    int rows, columns, threads;
};
constexpr Tile kTiles[] = {{32, 64, 256}, {64, 128, 256}, {64, 256, 512}, {128, 256, 512}, {256, 256, 512}};
enum { kTile32, kTile64, kTile64Wide, kTile128, kTile256, kNumTiles };
constexpr int kKindBf16 = 0, kKindFp8 = 1, kKindLora = 2, kKindTransposed = 3;

struct ExpertKernels {
    hipModule_t module = nullptr;
    int device = -1;
    hipFunction_t rows[4][kNumTiles];             // [kKind*][kTiles]
    hipFunction_t split[2], split_lora[3], sum_splits, sum_splits_lora, split_weights, sum_weights[2];
    hipFunction_t weights[2][2];                  // [BF16, float32][128 x 128, 256 x 256]
    hipFunction_t swiglu[2], swiglu_grad, lora_down[3], lora_down_rows, expand_fill, expand_rows;
};
ExpertKernels g_k;
std::mutex g_mutex;

// (contracts are checked before: they need no GPU)
const ExpertKernels& kernels() {
    ep_load_expert_kernels(nullptr);
    int cur = -1;
    HIP_CHECK(hipGetDevice(&cur));
    EP_HOST_ASSERT(cur == g_k.device and "the kernels were loaded on another device");
    return g_k;
}

template <class A>
void launch(hipFunction_t fn, int64_t grid, unsigned block, void* stream, A& args) {
    EP_HOST_ASSERT(grid > 0 and grid * block <= UINT32_MAX);
    void* params[] = {&args};
    HIP_CHECK(hipModuleLaunchKernel(fn, (unsigned)grid, 1, 1, block, 1, 1, 0, (hipStream_t)stream, params, nullptr));
}

// Rows whose channels are contiguous and start on 16 bytes.
bool row_major(const ep_tensor_t& t) {
    if (not present(t) or t.ndim != 2 or t.size[0] < 0 or t.size[1] <= 0) return false;
    const int64_t elem = elem_size(t.dtype);
    if (t.size[1] != 1 and t.stride[1] != 1) return false;
    if (t.size[0] > 1 and (t.stride[0] < t.size[1] or t.stride[0] * elem % 16 != 0)) return false;
    return ((uintptr_t)t.data & 15) == 0;
}
// Every value of a matrix has a place of its own.
bool apart(const ep_tensor_t& t) {
    const int inner = t.size[0] > 1 and (t.size[1] <= 1 or t.stride[0] < t.stride[1]) ? 0 : 1, outer = 1 - inner;
    return (t.size[inner] <= 1 or t.stride[inner] > 0) and (t.size[outer] <= 1 or t.stride[outer] >= t.size[inner] * t.stride[inner]);
}
int64_t row_stride(const ep_tensor_t& t) { return t.size[0] > 1 ? t.stride[0] : (t.size[1] + 15) / 16 * 16; }

// Bytes of a tile's rows are counted in 31 bits.
constexpr int64_t kMaxRowBytes = 4 << 20;
bool addressable(const ep_tensor_t& t) { return row_stride(t) * elem_size(t.dtype) <= kMaxRowBytes; }

EpExpertLayout layout_of(const ep_tensor_t& psum, int num_experts, int alignment, int zero_rows, int64_t rows) {
    EP_HOST_ASSERT(num_experts > 0 and alignment > 0);
    EP_HOST_ASSERT(zero_rows >= EP_ZERO_NONE and zero_rows <= EP_ZERO_ALL);
    EP_HOST_ASSERT(rows + alignment <= INT32_MAX - 1024);      // (rounded up to tiles too)
    if (present(psum)) {
        EP_HOST_ASSERT(psum.ndim == 1 and psum.dtype == EP_DTYPE_I32 and contiguous(psum));
        EP_HOST_ASSERT(psum.size[0] == num_experts);
    } else {
        EP_HOST_ASSERT(num_experts == 1);
    }
    EpExpertLayout l{};
    l.psum = (const int*)psum.data;
    l.num_experts = num_experts;
    l.alignment = alignment;
    l.num_rows = (int)rows;
    l.zero_rows = zero_rows;
    return l;
}

// Row tiles of all experts are at most this many: every expert with rows begins a tile of its own.
int64_t row_tiles_bound(int64_t rows, int num_experts, int tile) {
    return num_experts == 1 ? ceil_div(rows, tile) : rows / tile + std::min<int64_t>(num_experts, rows);
}

// Rows of an expert on average, were the padding as much as it can be: the counts are known on the device only.  That is right for tensors of the
// dispatch's worst-case size; exact ones hold half of it, so that their tiles are counted low, and just above a whole round of them another tile would
// be faster.  Which of the two the tensors are is not known here.  With half of the padding for means above 64, in us, this / that:
//   exact: 16384 rows of 8 experts, 4096 to 2048, alignment 128, adapters 328 / 319; 7147 of 64, 2560 to 1536, alignment 32, with gradients
//   441 / 418; 8481 of 16, 2560 to 512, alignment 128 45 / 38; 12288 of 64, 4096 to 2048, alignment 128 level
//   worst-case: 12288 of 64, 4096 to 2048, alignment 128 279 / 330; 8192 of 32, 2048 to 2560, alignment 64 114 / 129; 4096 of 16, 4096 to 2048,
//   alignment 128 97 / 104
int64_t mean_rows(int64_t rows, int num_experts, int alignment) {
    return ceil_div(std::max<int64_t>(rows - (int64_t)(alignment - 1) * num_experts, std::min<int64_t>(rows, num_experts)), num_experts);
}

// Rows up to which the low-rank rows are made in tiles of 16 (lora_plan), in one launch with the parts of a product.
constexpr int64_t kFewLoraRows = 1024;

// How a product of rows is launched: its tile, and in how many parts of the depth.
struct Plan {
    int tile, splits, split_depth;
};
// Rounds of the chip's 256 CUs times what a round takes, in hundredths of one of 256 x 256 tiles.  Measured in us, BF16, tiles of 64 x 128
// (two workgroups a CU) / 64 x 256 / 128 x 256 / 256 x 256:
//   one expert, 7168 channels to 2048, 1500 rows 94 61 75 126, 3000 rows 115 125 84 130, 6000 rows 228 197 166 140, 12000 rows 444 385 277 296
//   8 experts, 4096 to 2048, 1500 rows 50 41 48 77, 3000 84 74 51 76, 6000 151 143 100 86, 12000 341 273 207 172, 16384 416 398 275 261
//   64 experts, 2560 to 1536, 7147 rows 162 160 124 121, of Zipf(0.6) popularity 161 163 146 131
//   32 experts, 4096 to 4096, 3500 rows 309 240 199 281, 6000 rows 521 456 257 311
// (the last two are bound by the weights).  Experts end inside a tile, half of one on average.
Plan plan_rows(int64_t rows, int num_experts, int alignment, int64_t depth, int64_t columns, bool transposed, bool adapters) {
    const int64_t mean = mean_rows(rows, num_experts, alignment);
    const int64_t cost[kNumTiles] = {0, 55, 48, 62, 100}, slots[kNumTiles] = {512, 512, 256, 256, 256};
    int64_t tiles[kNumTiles], best = INT64_MAX;
    Plan p{kTile256, 1, 0};
    for (int t = kTile64; t < kNumTiles; ++t) {
        const int64_t high = kTiles[t].rows, wide = ceil_div(columns, kTiles[t].columns);
        tiles[t] = num_experts == 1 ? ceil_div(rows, high) * wide : std::max<int64_t>(num_experts, num_experts * (2 * mean + high) / (2 * high)) * wide;
        const int64_t time = ceil_div(tiles[t], slots[t]) * cost[t];
        // (of equals the larger tile where its rows are there, the smaller where they are not)
        if (time < best or (time == best and mean > 64)) {
            best = time;
            p.tile = t;
        }
    }
    // half a round of wide tiles: as many bytes of weights in flight with twice the workgroups (32 experts of 8 rows, 4096 channels to 2048,
    // 122 -> 108 us)
    if (p.tile == kTile64Wide and tiles[kTile64Wide] <= 256) p.tile = kTile64;
    if (transposed) return p;
    // Less than a round of 64 x 128 tiles: smaller ones, or the depth in parts, whose sum is a launch of its own and as many times 32 bits of the
    // result.  In us, 32 x 64 / 64 x 128 in 2, 4, 8, 16 parts:
    //   2048 channels to 2048, 64 rows (16 tiles of 64 x 128) 10 / 12 10 11 11, 256 rows (64) 11 / 14 14 16 16
    //   4096 to 2048, 64 rows (16) 17 / 17 13 15 14, 128 rows (32) 17 / 17 13 14 17, 256 rows (64) 18 / 18 19 20 27
    //   7168 to 4096, 64 rows (32) 27 / 25 18 18 20, 128 rows (64) 28 / 26 25 28 34, 256 rows (128) 38 / 41 44 50 62
    // and FP8 the same.  Beside adapters 32 x 64 tiles need a launch of their own too, for the low-rank rows, and the parts do not:
    //   2048 to 2048, 64 rows (16) 29 / 16 14 14 14, 7168 to 4096, 64 rows (32) 53 / 31 25 25 28, 256 rows (128) 63 / 55 64 68 79
    if (tiles[kTile64] < 256) {
        const bool one_launch = adapters and rows <= kFewLoraRows;
        const int64_t few = tiles[kTile64], parts = std::clamp<int64_t>(128 / few, one_launch ? 2 : 4, 16);
        const bool split = one_launch or (few <= 64 and depth >= std::max<int64_t>(2560, 80 * few));
        const int64_t steps = ceil_div(depth, 128);
        p.split_depth = (int)(ceil_div(steps, split ? std::min(parts, std::max<int64_t>(1, steps / 2)) : 1) * 128);
        p.splits = (int)ceil_div(depth, p.split_depth);
        p.tile = p.splits > 1 ? kTile64 : kTile32;
    }
    return p;
}

// The gradient of weights: tiles of 256 x 256 as soon as they fill the chip; where those of 128 x 128 do not either and rows are many, rows
// in parts of 600 at least (8192 rows, one expert's 1024 x 1024: 74 -> 34 us; 1024 of each of eight experts, 512 x 512, in two parts: 15 -> 18).
struct WeightsPlan {
    bool large;
    int splits;
};
WeightsPlan plan_weights(int64_t rows, int num_experts, int alignment, int64_t out_rows, int64_t out_columns) {
    WeightsPlan p{num_experts * ceil_div(out_rows, 256) * ceil_div(out_columns, 256) >= 256, 1};
    const int64_t tiles = num_experts * ceil_div(out_rows, 128) * ceil_div(out_columns, 128);
    if (not p.large and tiles < 256)
        p.splits = (int)std::clamp<int64_t>(512 / tiles, 1, std::clamp<int64_t>(mean_rows(rows, num_experts, alignment) / 600, 1, 32));
    return p;
}

}  // namespace

void ep_load_expert_kernels(const char* dir) {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (g_k.module != nullptr) return;
    const std::string path = ep_code_object_path(dir, "ep_experts.hsaco");
    int ndev = 0;
    HIP_CHECK(hipGetDeviceCount(&ndev));
    if (ndev <= 0) throw EpError{"no HIP device visible: the EP kernels only run on a gfx950 GPU"};
    HIP_CHECK(hipGetDevice(&g_k.device));
    hipModule_t m;
    HIP_CHECK(hipModuleLoad(&m, path.c_str()));
    auto get = [&](hipFunction_t& fn, const char* name) { HIP_CHECK(hipModuleGetFunction(&fn, m, name)); };
    const char* kinds[] = {"bf16", "fp8", "lora", "transposed"};
    for (int k = 0; k < 4; ++k) {
        for (int t = 0; t < kNumTiles; ++t) {
            if (k == kKindTransposed and t == kTile32) continue;
            get(g_k.rows[k][t], format("ep_grouped_%s_%dx%d", kinds[k], kTiles[t].rows, kTiles[t].columns).c_str());
        }
    }
    for (int k = 0; k < 2; ++k) get(g_k.split[k], format("ep_grouped_split_%s", kinds[k]).c_str());
    for (int i = 0; i < 3; ++i) get(g_k.split_lora[i], format("ep_grouped_split_lora_%d", 16 << i).c_str());
    get(g_k.sum_splits, "ep_sum_splits");
    get(g_k.split_weights, "ep_grouped_split_weights");
    get(g_k.sum_weights[0], "ep_sum_weights_bf16");
    get(g_k.sum_weights[1], "ep_sum_weights_f32");
    get(g_k.sum_splits_lora, "ep_sum_splits_lora");
    for (int i = 0; i < 3; ++i) get(g_k.lora_down[i], format("ep_lora_down_%d", 16 << i).c_str());
    get(g_k.lora_down_rows, "ep_lora_down_rows");
    get(g_k.expand_fill, "ep_expand_fill");
    get(g_k.expand_rows, "ep_expand_token_index_rows");
    const char* outs[] = {"bf16", "f32"};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j)
            get(g_k.weights[i][j], format("ep_grouped_weights_%s_%dx%d", outs[i], 128 << j, 128 << j).c_str());
    get(g_k.swiglu[0], "ep_swiglu_bf16");
    get(g_k.swiglu[1], "ep_swiglu_fp8");
    get(g_k.swiglu_grad, "ep_swiglu_gradients");
    g_k.module = m;
}

extern "C" {

// How the rows times the adapters' first matrices are split: rows of a workgroup's tile, chunks of the depth, workgroups that share the
// adapters of a tile; 512 workgroups in all, two a CU, where there are so many.
struct LoraPlan {
    int rows, chunks, chunk_depth, slots;
};
// Up to kFewLoraRows tiles of 16 rows, adapter by adapter; more: 64 rows and as many adapters as have 64 ranks at once.  One expert, 4096 channels to
// 4096, 16 ranks, in us, 4 / 32 adapters: 128 rows 27 / 28 (the other 32 / 59), 512 rows 65 / 73 (60 / 92), 2048 rows 86 / 162 (81 / 148),
// 4096 rows 144 / 281 (134 / 217).
static LoraPlan lora_plan(int64_t rows, int num_experts, int64_t depth) {
    LoraPlan p{};
    p.rows = rows <= kFewLoraRows ? 16 : 64;
    const int64_t tiles = std::max<int64_t>(1, row_tiles_bound(rows, num_experts, p.rows));
    p.slots = p.rows == 16 ? (int)std::clamp<int64_t>(ceil_div(512, tiles), 1, std::min<int64_t>(p.rows, std::max<int64_t>(rows, 1))) : 1;
    const int64_t steps = ceil_div(depth, EP_LORA_STEP), chunks = std::clamp<int64_t>(ceil_div(512, tiles * p.slots), 1, std::min<int64_t>(steps, 16));
    p.chunk_depth = (int)(ceil_div(steps, chunks) * EP_LORA_STEP);
    p.chunks = (int)ceil_div(depth, p.chunk_depth);
    return p;
}

// The arguments of a product of rows, checked.
static EpGemmArgs linear_args(const ep_grouped_linear_args_t* args) {
    const ep_tensor_t &x = args->x, &w = args->weight, &out = args->out;
    EP_HOST_ASSERT(args->workspace_bytes >= 0 and (args->workspace != nullptr or args->workspace_bytes == 0));
    EP_HOST_ASSERT(((uintptr_t)args->workspace & 15) == 0);
    EP_HOST_ASSERT(row_major(x) and addressable(x));
    EP_HOST_ASSERT(row_major(w) and addressable(w) and w.dtype == x.dtype);
    const bool fp8 = x.dtype == EP_DTYPE_FP8_E4M3, transposed = args->transpose_weight != 0;
    EP_HOST_ASSERT(fp8 or x.dtype == EP_DTYPE_BF16);
    EP_HOST_ASSERT(not (fp8 and transposed));
    const int64_t rows = x.size[0], depth = x.size[1], columns = w.size[transposed ? 1 : 0];
    EP_HOST_ASSERT(w.size[transposed ? 0 : 1] == depth);
    EP_HOST_ASSERT(depth % (fp8 ? 16 : 8) == 0 and columns > 0 and columns % 8 == 0);
    EP_HOST_ASSERT(depth <= INT32_MAX / 2 and columns <= INT32_MAX / 2);
    EP_HOST_ASSERT(args->num_experts == 1 or (args->weight_expert_stride >= 0 and args->weight_expert_stride * elem_size(w.dtype) % 16 == 0));
    EP_HOST_ASSERT(row_major(out) and out.dtype == EP_DTYPE_BF16);
    EP_HOST_ASSERT(out.size[0] == rows and out.size[1] == columns);
    EpGemmArgs g{};
    g.layout = layout_of(args->psum_num_recv_tokens_per_expert, args->num_experts, args->expert_alignment, args->zero_rows, rows);
    g.rows = (const char*)x.data;
    g.columns = (const char*)w.data;
    g.rows_ld = row_stride(x) * elem_size(x.dtype);
    g.columns_ld = row_stride(w) * elem_size(w.dtype);
    g.columns_expert = args->weight_expert_stride * elem_size(w.dtype);
    g.out = (char*)out.data;
    g.out_ld = row_stride(out);
    g.depth = (int)depth;
    g.num_columns = (int)columns;
    EP_HOST_ASSERT(fp8 == present(args->x_sf) and fp8 == present(args->weight_sf));
    if (fp8) {
        const ep_tensor_t &sf = args->x_sf, &wsf = args->weight_sf;
        EP_HOST_ASSERT(depth <= EP_EXPERT_MAX_DEPTH_FP8);
        EP_HOST_ASSERT(sf.ndim == 2 and sf.dtype == EP_DTYPE_F32 and sf.size[0] == rows and sf.size[1] == ceil_div(depth, 128));
        EP_HOST_ASSERT(sf.stride[0] >= 0 and sf.stride[1] >= 0 and (rows <= 1 or sf.stride[0] * 4 <= kMaxRowBytes));
        EP_HOST_ASSERT(wsf.ndim == 2 and wsf.dtype == EP_DTYPE_F32);
        EP_HOST_ASSERT(wsf.size[0] == ceil_div(columns, 128) and wsf.size[1] == ceil_div(depth, 128));
        g.rows_sf = (const float*)sf.data;
        g.columns_sf = (const float*)wsf.data;
        g.rows_sf_row = rows > 1 ? sf.stride[0] : 1;
        g.rows_sf_col = sf.stride[1];
        g.columns_sf_row = wsf.stride[0];
        g.columns_sf_col = wsf.stride[1];
        g.columns_sf_expert = args->weight_sf_expert_stride;
    }
    return g;
}

// The launches of a product of rows; `workspace`: where the parts of a split depth go, if there is room.
static void launch_rows(EpGemmArgs& g, int kind, const LoraPlan* lora, void* workspace, int64_t workspace_bytes, void* stream) {
    const EpExpertLayout& l = g.layout;
    Plan p = plan_rows(l.num_rows, l.num_experts, l.alignment, g.depth, g.num_columns, kind == kKindTransposed, kind == kKindLora);
    const ExpertKernels& k = kernels();
    if (p.splits > 1 and (int64_t)p.splits * l.num_rows * g.num_columns * 4 > workspace_bytes) p = Plan{kTile32, 1, 0};
    const Tile& t = kTiles[p.tile];
    g.column_tiles = (int)ceil_div(g.num_columns, t.columns);
    g.splits = p.splits;
    g.split_depth = p.split_depth;
    g.partial = p.splits > 1 ? (float*)workspace : nullptr;
    const int64_t row_tiles = row_tiles_bound(l.num_rows, l.num_experts, t.rows);
    EP_HOST_ASSERT(row_tiles <= INT32_MAX / (8 * (int64_t)g.column_tiles * p.splits));
    const int64_t blocks = align_up(row_tiles * g.column_tiles * p.splits, 8);
    const int ranks = g.lora.rank <= 16 ? 0 : g.lora.rank <= 32 ? 1 : 2;
    // (few rows' low-rank rows come with the parts of the product, in one launch)
    const bool together = lora != nullptr and lora->rows == 16 and p.splits > 1;
    if (lora != nullptr and not together) launch(lora->rows == 16 ? k.lora_down[ranks] : k.lora_down_rows, g.lora.blocks, 256, stream, g);
    if (p.splits == 1) {
        launch(k.rows[kind][p.tile], blocks, t.threads, stream, g);
        return;
    }
    if (together) launch(k.split_lora[ranks], g.lora.blocks + blocks, t.threads, stream, g);
    else launch(k.split[kind == kKindFp8 ? 1 : 0], blocks, t.threads, stream, g);
    launch(lora != nullptr ? k.sum_splits_lora : k.sum_splits, ceil_div((int64_t)l.num_rows * ceil_div(g.num_columns, 512), 4), 256, stream, g);
}

int64_t ep_grouped_linear_workspace_bytes(int64_t num_rows, int num_experts, int expert_alignment, int64_t depth, int64_t num_columns, int adapters) {
    if (num_rows <= 0 or num_rows > INT32_MAX or num_experts <= 0 or expert_alignment <= 0 or depth <= 0 or depth > INT32_MAX / 2 or num_columns <= 0 or
        num_columns > INT32_MAX / 2)
        return 0;
    const Plan p = plan_rows(num_rows, num_experts, expert_alignment, depth, num_columns, false, adapters != 0);
    return p.splits > 1 ? (int64_t)p.splits * num_rows * num_columns * 4 : 0;
}

int ep_grouped_linear(const ep_grouped_linear_args_t* args) {
    return guarded([&] {
        EP_HOST_ASSERT(args != nullptr);
        EpGemmArgs g = linear_args(args);
        if (g.layout.num_rows == 0) return;
        launch_rows(g, args->x.dtype == EP_DTYPE_FP8_E4M3 ? kKindFp8 : args->transpose_weight ? kKindTransposed : kKindBf16, nullptr,
                    args->workspace, args->workspace_bytes, args->stream);
    });
}

int64_t ep_grouped_lora_workspace_bytes(int64_t num_rows, int num_experts, int64_t depth, int rank) {
    if (num_rows < 0 or num_rows > INT32_MAX or num_experts <= 0 or depth <= 0 or depth > INT32_MAX / 2 or rank <= 0 or rank > EP_LORA_MAX_RANK) return -1;
    return lora_plan(num_rows, num_experts, depth).chunks * num_rows * rank * 4;
}

int ep_grouped_lora_linear(const ep_grouped_lora_args_t* args) {
    return guarded([&] {
        EP_HOST_ASSERT(args != nullptr);
        EpGemmArgs g = linear_args(&args->linear);
        EP_HOST_ASSERT(args->linear.x.dtype == EP_DTYPE_BF16 and args->linear.transpose_weight == 0);
        const ep_tensor_t &down = args->lora_a, &up = args->lora_b, &idx = args->adapter_idx, &scales = args->scales;
        EP_HOST_ASSERT(row_major(down) and down.dtype == EP_DTYPE_BF16 and addressable(down));
        EP_HOST_ASSERT(row_major(up) and up.dtype == EP_DTYPE_BF16 and addressable(up));
        const int64_t rank = down.size[0];
        EP_HOST_ASSERT(rank > 0 and rank % 8 == 0 and rank <= EP_LORA_MAX_RANK);
        EP_HOST_ASSERT(down.size[1] == g.depth and up.size[0] == g.num_columns and up.size[1] == rank);
        EP_HOST_ASSERT(args->num_adapters > 0);
        for (const int64_t stride : {args->lora_a_adapter_stride, args->lora_a_expert_stride, args->lora_b_adapter_stride, args->lora_b_expert_stride})
            EP_HOST_ASSERT(stride >= 0 and stride % 8 == 0);
        EP_HOST_ASSERT(present(idx) and idx.ndim == 1 and idx.dtype == EP_DTYPE_I32 and contiguous(idx) and idx.size[0] == g.layout.num_rows);
        if (present(scales)) {
            EP_HOST_ASSERT(scales.ndim == 1 and scales.dtype == EP_DTYPE_F32 and contiguous(scales) and scales.size[0] == args->num_adapters);
        }
        const LoraPlan plan = lora_plan(g.layout.num_rows, g.layout.num_experts, g.depth);
        const int64_t bytes = (int64_t)plan.chunks * g.layout.num_rows * rank * 4;
        EP_HOST_ASSERT(bytes == 0 or (args->workspace != nullptr and ((uintptr_t)args->workspace & 15) == 0));
        EP_HOST_ASSERT(args->workspace_bytes >= bytes);
        if (g.layout.num_rows == 0) return;
        EpLoraArgs& l = g.lora;
        l.adapter = (const int*)idx.data;
        l.down = (const char*)down.data;
        l.up = (const char*)up.data;
        l.down_ld = row_stride(down) * 2;
        l.down_adapter = args->lora_a_adapter_stride * 2;
        l.down_expert = args->lora_a_expert_stride * 2;
        l.up_ld = row_stride(up) * 2;
        l.up_adapter = args->lora_b_adapter_stride * 2;
        l.up_expert = args->lora_b_expert_stride * 2;
        l.scales = (const float*)scales.data;
        l.low = (float*)args->workspace;
        l.num_adapters = args->num_adapters;
        l.rank = (int)rank;
        l.chunks = plan.chunks;
        l.chunk_depth = plan.chunk_depth;
        l.slots = plan.slots;
        const int64_t blocks = row_tiles_bound(g.layout.num_rows, g.layout.num_experts, plan.rows) * plan.chunks * plan.slots;
        EP_HOST_ASSERT(blocks <= INT32_MAX / 2);
        l.blocks = (int)blocks;
        // (one buffer of 31 bits has to reach all of them)
        const bool near = (int64_t)l.num_adapters * l.down_adapter + 64 * l.down_ld < INT32_MAX;
        l.together = near ? (int)(64 / rank) : 1;
        launch_rows(g, kKindLora, &plan, args->linear.workspace, args->linear.workspace_bytes, args->linear.stream);
    });
}

int ep_expand_token_index(const ep_tensor_t* values, const ep_tensor_t* src_metadata, const ep_tensor_t* psum_num_recv_tokens_per_rank,
                          const ep_tensor_t* out, void* stream) {
    return guarded([&] {
        EP_HOST_ASSERT(values != nullptr and src_metadata != nullptr and psum_num_recv_tokens_per_rank != nullptr and out != nullptr);
        const ep_tensor_t &v = *values, &m = *src_metadata, &psum = *psum_num_recv_tokens_per_rank, &o = *out;
        for (const ep_tensor_t* t : {&v, &m, &psum, &o})
            EP_HOST_ASSERT(present(*t) and t->dtype == EP_DTYPE_I32 and contiguous(*t) and t->size[0] <= INT32_MAX);
        EP_HOST_ASSERT(v.ndim == 1 and m.ndim == 2 and psum.ndim == 1 and o.ndim == 1);
        EP_HOST_ASSERT(m.size[1] > 2 and m.size[1] <= INT32_MAX and psum.size[0] > 0);
        EpExpandIndexArgs e{};
        e.metadata = (const int*)m.data;
        e.psum_rank = (const int*)psum.data;
        e.values = (const int*)v.data;
        e.out = (int*)o.data;
        e.num_rows = (int)m.size[0];
        e.num_ranks = (int)psum.size[0];
        e.topk = (int)m.size[1] - 2;
        e.num_values = (int)v.size[0];
        e.num_out = (int)o.size[0];
        if (e.num_out == 0) return;
        const ExpertKernels& k = kernels();
        launch(k.expand_fill, ceil_div(e.num_out, 256), 256, stream, e);
        if (e.num_rows > 0) launch(k.expand_rows, ceil_div((int64_t)e.num_rows * e.topk, 256), 256, stream, e);
    });
}

int ep_grouped_weight_grad(const ep_grouped_weight_grad_args_t* args) {
    return guarded([&] {
        EP_HOST_ASSERT(args != nullptr);
        const ep_tensor_t &grad = args->grad, &x = args->x, &out = args->out;
        EP_HOST_ASSERT(args->workspace_bytes >= 0 and (args->workspace != nullptr or args->workspace_bytes == 0));
        EP_HOST_ASSERT(((uintptr_t)args->workspace & 15) == 0);
        EP_HOST_ASSERT(row_major(grad) and grad.dtype == EP_DTYPE_BF16 and addressable(grad));
        EP_HOST_ASSERT(row_major(x) and x.dtype == EP_DTYPE_BF16 and addressable(x));
        EP_HOST_ASSERT(x.size[0] == grad.size[0] and x.size[1] % 8 == 0 and grad.size[1] % 8 == 0);
        const bool f32 = out.dtype == EP_DTYPE_F32;
        EP_HOST_ASSERT(row_major(out) and (f32 or out.dtype == EP_DTYPE_BF16));
        EP_HOST_ASSERT(out.size[0] == grad.size[1] and out.size[1] == x.size[1]);
        EP_HOST_ASSERT(f32 or args->accumulate == 0);
        EP_HOST_ASSERT(args->num_experts == 1 or
                       (args->out_expert_stride >= out.size[0] * row_stride(out) and args->out_expert_stride * elem_size(out.dtype) % 16 == 0));
        EpGemmArgs g{};
        g.layout = layout_of(args->psum_num_recv_tokens_per_expert, args->num_experts, args->expert_alignment, 0, x.size[0]);
        g.rows = (const char*)grad.data;
        g.columns = (const char*)x.data;
        g.rows_ld = row_stride(grad) * 2;
        g.columns_ld = row_stride(x) * 2;
        g.out = (char*)out.data;
        g.out_ld = row_stride(out);
        g.out_expert = args->out_expert_stride;
        g.num_columns = (int)x.size[1];
        g.num_out_rows = (int)grad.size[1];
        const int experts = g.layout.num_experts;
        WeightsPlan p = plan_weights(g.layout.num_rows, experts, g.layout.alignment, g.num_out_rows, g.num_columns);
        const int64_t bytes = (int64_t)p.splits * experts * g.num_out_rows * g.num_columns * 4;
        if (p.splits > 1 and bytes > args->workspace_bytes) p.splits = 1;
        const int tile = p.large ? 256 : 128;
        g.column_tiles = (int)ceil_div(g.num_columns, tile);
        g.row_tiles = (int)ceil_div(g.num_out_rows, tile);
        g.splits = p.splits;
        g.partial = p.splits > 1 ? (float*)args->workspace : nullptr;
        g.accumulate = args->accumulate != 0;
        EP_HOST_ASSERT((int64_t)g.row_tiles * p.splits <= INT32_MAX / (16 * (int64_t)g.column_tiles));
        const int64_t blocks = experts * align_up((int64_t)g.row_tiles * g.column_tiles * p.splits, 8);
        const ExpertKernels& k = kernels();
        launch(p.splits > 1 ? k.split_weights : k.weights[f32 ? 1 : 0][p.large ? 1 : 0], blocks, 512, args->stream, g);
        if (p.splits > 1) launch(k.sum_weights[f32 ? 1 : 0], ceil_div((int64_t)experts * g.num_out_rows * g.num_columns, 1024), 256, args->stream, g);
    });
}

int64_t ep_grouped_weight_grad_workspace_bytes(int64_t num_rows, int num_experts, int expert_alignment, int64_t out_rows, int64_t out_columns) {
    if (num_rows <= 0 or num_rows > INT32_MAX or num_experts <= 0 or expert_alignment <= 0 or out_rows <= 0 or out_rows > INT32_MAX / 2 or
        out_columns <= 0 or out_columns > INT32_MAX / 2)
        return 0;
    const WeightsPlan p = plan_weights(num_rows, num_experts, expert_alignment, out_rows, out_columns);
    return p.splits > 1 ? (int64_t)p.splits * num_experts * out_rows * out_columns * 4 : 0;
}

static EpSwigluArgs swiglu_args(const ep_tensor_t& h, const ep_tensor_t& weights, const ep_tensor_t& psum, int num_experts, int alignment,
                                int zero_rows) {
    EP_HOST_ASSERT(row_major(h) and h.dtype == EP_DTYPE_BF16 and h.size[1] % 16 == 0 and h.size[1] <= INT32_MAX / 2);
    EpSwigluArgs s{};
    s.layout = layout_of(psum, num_experts, alignment, zero_rows, h.size[0]);
    s.h = (const char*)h.data;
    s.h_ld = row_stride(h);
    s.channels = (int)(h.size[1] / 2);
    if (present(weights)) {
        EP_HOST_ASSERT(weights.ndim == 1 and weights.dtype == EP_DTYPE_F32 and weights.size[0] == h.size[0] and contiguous(weights));
        s.weights = (const float*)weights.data;
    }
    s.num_parts = (int)ceil_div(s.channels, 512);
    return s;
}

int ep_swiglu(const ep_swiglu_args_t* args) {
    return guarded([&] {
        EP_HOST_ASSERT(args != nullptr);
        const ep_tensor_t &out = args->out, &sf = args->out_sf;
        EpSwigluArgs s = swiglu_args(args->h, args->weights, args->psum_num_recv_tokens_per_expert, args->num_experts, args->expert_alignment,
                                     args->zero_rows);
        const bool fp8 = out.dtype == EP_DTYPE_FP8_E4M3;
        EP_HOST_ASSERT(present(out) and out.ndim == 2 and (fp8 or out.dtype == EP_DTYPE_BF16));
        EP_HOST_ASSERT(out.size[0] == args->h.size[0] and out.size[1] == s.channels);
        EP_HOST_ASSERT(out.stride[1] == 1 and (out.size[0] <= 1 or (out.stride[0] >= out.size[1] and out.stride[0] % 8 == 0)));
        EP_HOST_ASSERT(((uintptr_t)out.data & (fp8 ? 7 : 15)) == 0);
        s.out = (char*)out.data;
        s.out_ld = row_stride(out);
        EP_HOST_ASSERT(fp8 == present(sf));
        if (fp8) {
            EP_HOST_ASSERT(sf.ndim == 2 and sf.dtype == EP_DTYPE_F32 and sf.size[0] == out.size[0] and sf.size[1] == ceil_div(s.channels, 128));
            EP_HOST_ASSERT(apart(sf));
            s.sf = (float*)sf.data;
            s.sf_row = sf.stride[0];
            s.sf_col = sf.stride[1];
        }
        if (s.layout.num_rows == 0) return;
        s.parts_per_task = (int)std::clamp<int64_t>((int64_t)s.layout.num_rows * s.num_parts / 8192, 1, s.num_parts);
        const int64_t tasks = (int64_t)s.layout.num_rows * ceil_div(s.num_parts, s.parts_per_task);
        launch(kernels().swiglu[fp8 ? 1 : 0], ceil_div(tasks, 4), 256, args->stream, s);
    });
}

int ep_swiglu_grad(const ep_swiglu_grad_args_t* args) {
    return guarded([&] {
        EP_HOST_ASSERT(args != nullptr);
        const ep_tensor_t &grad = args->grad, &grad_h = args->grad_h, &grad_weights = args->grad_weights;
        EpSwigluArgs s = swiglu_args(args->h, args->weights, args->psum_num_recv_tokens_per_expert, args->num_experts, args->expert_alignment,
                                     args->zero_rows);
        EP_HOST_ASSERT(row_major(grad) and grad.dtype == EP_DTYPE_BF16);
        EP_HOST_ASSERT(grad.size[0] == args->h.size[0] and grad.size[1] == s.channels);
        EP_HOST_ASSERT(row_major(grad_h) and grad_h.dtype == EP_DTYPE_BF16);
        EP_HOST_ASSERT(grad_h.size[0] == args->h.size[0] and grad_h.size[1] == args->h.size[1]);
        s.grad_out = (const char*)grad.data;
        s.grad_out_ld = row_stride(grad);
        s.grad_h = (char*)grad_h.data;
        s.grad_h_ld = row_stride(grad_h);
        if (present(grad_weights)) {
            EP_HOST_ASSERT(grad_weights.ndim == 1 and grad_weights.dtype == EP_DTYPE_F32 and grad_weights.size[0] == grad.size[0]);
            EP_HOST_ASSERT(contiguous(grad_weights));
            s.grad_weights = (float*)grad_weights.data;
        }
        if (s.layout.num_rows == 0) return;
        launch(kernels().swiglu_grad, ceil_div(s.layout.num_rows, 4), 256, args->stream, s);
    });
}

}  // extern "C"
