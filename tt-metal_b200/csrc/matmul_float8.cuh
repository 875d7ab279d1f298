// What the float8 matmul, its quantiser and the experts' MLP share.
#pragma once
#include "float8.cuh"

namespace ttb {

// Quantised activations in scratch (layout: float8.cuh).
struct F8Activation {
    uint8_t *codes;      // [blocks of 128 columns][rows_padded][128]
    float *scales;       // [rows_padded][scale_pitch]
    int64_t rows_padded;
    int64_t scale_pitch;
};

inline int64_t f8_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline bool f8_misaligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }
// Scratch of quantised rows; advances `at`.
inline F8Activation f8_place(uint8_t *base, int64_t &at, int64_t rows, int64_t cols) {
    F8Activation a;
    a.rows_padded = f8_rows_padded(rows);
    a.scale_pitch = f8_scale_pitch(cols);
    a.codes = base + at;
    at = f8_up(at + a.rows_padded * f8_blocks(cols) * kF8Block, 1024);
    a.scales = reinterpret_cast<float *>(base + at);
    at = f8_up(at + a.rows_padded * a.scale_pitch * 4, 1024);
    return a;
}

// bfloat16 rows that a kernel quantises itself: row r is row_of[r] of `ptr` (null: r itself).
struct F8Rows {
    const uint16_t *ptr;
    const int32_t *row_of;
    int64_t row_pitch;   // row-major: elements of a row; tiled: elements of a row of tiles
    bool tiled;
};

struct F8Weight {
    const void *codes;   // [experts, N, K], row-major
    const float *scales; // [experts, ceil(N / 128), ceil(K / 128)]
};

// act(x w^T + bias) of all rows with one weight, or of runs of rows with an expert's weight each.
struct F8Matmul {
    F8Activation a;
    F8Rows x;                // few rows: instead of `a`, where its ptr is not null
    bool early;              // weights and offsets are complete before the kernel before lets this one start
    F8Weight w[2];           // the second: the up projection of a gated pair
    int64_t rows, K, N;
    int experts;             // 0: one weight for all rows
    const int32_t *offsets;  // [experts + 1], device: rows offsets[e] .. offsets[e + 1] - 1 are expert e's
    int act;
    // either a plain result
    void *out;
    int out_dtype;
    bool out_row_major;
    const uint16_t *bias;    // bfloat16 [N], or the first row of a tiled [32, N]; may be null
    bool bias_row_major;
    // or act(x w0^T) * (x w1^T), quantised again
    bool gated;
    F8Activation h;
    // scratch for tiles whose K range several blocks share
    int32_t *tickets;   // kF8TicketBytes, zero when the kernel starts and when it ends
    float *partials;    // f8_partial_bytes, no particular contents
};
constexpr int kF8MaxExperts = 1024;
constexpr int64_t kF8TicketBytes = 8192;
int64_t f8_partial_bytes(int64_t rows);
int32_t launch_matmul_float8(const F8Matmul &p, cudaStream_t stream);
// Whether the kernel for these row counts quantises the activations itself.
bool f8_quantises_itself(int64_t rows, int64_t experts);

// Whether the blocks of 128 values of the rows count in 31 bits, as launch_quantize_operand needs it.
inline bool f8_blocks_count(int64_t rows, int64_t K) { return rows * f8_blocks(K) <= INT32_MAX; }
// Quantises [outer, H, K] bfloat16 rows into `out`: row r to row r, or (pos) to the rows pos[r * k + j] >= 0. `early`: lets the next kernel start at once, else
// when all that came before this one has ended.
int32_t launch_quantize_operand(const void *a, bool row_major, int64_t outer, int64_t H, int64_t K, const F8Activation &out, const int32_t *pos, int k,
                                bool early, cudaStream_t stream);

}  // namespace ttb
