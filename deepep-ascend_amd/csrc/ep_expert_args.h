// Kernel argument blocks of ep_experts.hip, shared with its host side (ep_experts.cpp).
#pragma once
#include <stdint.h>

#define EP_EXPERT_MAX_DEPTH_FP8 32768      // channels of an FP8 row: the scales of a column block fit a table in LDS

#define EP_LORA_STEP 512                   // channels that a workgroup of ep_lora_down_* goes through at a time

// Rows of the expert-major layout: expert e has rows [align(psum[e - 1]), psum[e]); psum == nullptr: one expert has all rows.
struct EpExpertLayout {
    const int* psum;
    int num_experts, alignment, num_rows;
    int zero_rows;                // EP_ZERO_*: which rows of no expert are written, as zeros
};

// Low-rank adapters beside a product: out[r] += up[a][e] low[r], low[r] = scale[a] down[a][e] rows[r] with a = adapter[r].
struct EpLoraArgs {
    const int* adapter;           // [rows]; outside [0, num_adapters): none
    const char *down, *up;        // BF16: [rank, depth] and [columns, rank] of adapter 0 and expert 0
    int64_t down_ld, down_adapter, down_expert, up_ld, up_adapter, up_expert;     // bytes
    const float* scales;          // [num_adapters] or nullptr
    float* low;                   // [chunks, rows, rank]: sums over the chunks of the depth
    int num_adapters, rank, chunks;
    int chunk_depth, slots;       // of what makes them: channels of a chunk, workgroups that share a tile's adapters,
    int blocks;                   // and workgroups in all
    int together;                 // adapters that are multiplied at once where rows are many
};

// out[r, c] = sum_d rows[r, d] columns[c, d] over a tile of output rows and output columns.
struct EpGemmArgs {
    EpExpertLayout layout;
    const char *rows, *columns;   // operand of the output's rows, operand of its columns
    int64_t rows_ld, columns_ld;  // bytes between rows of the two in memory
    int64_t columns_expert;       // bytes between experts
    const float *rows_sf, *columns_sf;
    int64_t rows_sf_row, rows_sf_col, columns_sf_row, columns_sf_col, columns_sf_expert;      // floats
    char* out;
    int64_t out_ld, out_expert;   // elements
    int depth;                    // channels that are summed over (weight gradient: the expert's rows, found on the device)
    int num_columns;              // channels of the output
    int num_out_rows;             // weight gradient: rows of the output of one expert
    int column_tiles, row_tiles;  // (row_tiles: weight gradient)
    int accumulate;               // weight gradient in 32 bits: added to what is there
    int splits, split_depth;      // the depth in so many parts (of split_depth channels), sums of each in `partial`
    float* partial;               // [splits, rows, num_columns]
    EpLoraArgs lora;
};

struct EpExpandIndexArgs {
    const int* metadata;          // [rows, topk + 2]
    const int* psum_rank;         // [ranks]
    const int* values;
    int* out;
    int num_rows, num_ranks, topk, num_values, num_out;
};

struct EpSwigluArgs {
    EpExpertLayout layout;
    const char* h;                // [rows, 2 * channels] BF16: gates, then ups
    int64_t h_ld;                 // elements
    const float* weights;         // [rows] or nullptr
    char* out;                    // [rows, channels] BF16 or e4m3fn
    int64_t out_ld;               // elements
    float* sf;                    // [rows, ceil(channels / 128)]
    int64_t sf_row, sf_col;
    // gradients
    const char* grad_out;         // [rows, channels] BF16
    int64_t grad_out_ld;
    char* grad_h;                 // [rows, 2 * channels] BF16
    int64_t grad_h_ld;
    float* grad_weights;          // [rows] or nullptr
    int channels;
    int num_parts, parts_per_task;  // parts of 512 channels of a row
};
