// Quantisation to float8 codes with block scales (float8.cuh has the format).
//
// Weights and tensors a user keeps: codes row-major [outer, H, W], scales [outer, ceil(H / block_rows), ceil(W / 128)]. Activations of
// a matmul: the operand layout of float8.cuh in scratch. Sixteen lanes hold the 128 values of a row's block, eight each, so that the
// largest value needs four shuffles and every access is 16 bytes wide. Bound by HBM: each value is read once and its code written once.
#include "epilogue.cuh"
#include "float8.cuh"
#include "matmul_float8.cuh"
#include "sm100_ptx.cuh"

namespace ttb {
namespace {

struct Source {
    const void *ptr;
    int64_t pitch;      // elements between rows (row-major), tiles per tile row (tiled)
    int64_t slab;       // elements between matrices
    bool tiled, vector; // vector: eight neighbours of a row are 16-byte aligned
};

// Columns c .. c + 7 of a row; what lies behind W is zero.
template <typename T>
__device__ __forceinline__ void load8(const Source &s, int64_t o, int64_t row, int64_t c, int64_t W, float (&v)[8]) {
    const T *p = reinterpret_cast<const T *>(s.ptr) + o * s.slab + (s.tiled ? tiled_offset(row, c, s.pitch) : row * s.pitch + c);
    if (s.vector && c + 8 <= W) {
        if (sizeof(T) == 4) {
            const float4 a = __ldcg(reinterpret_cast<const float4 *>(p)), b = __ldcg(reinterpret_cast<const float4 *>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = __ldcg(reinterpret_cast<const uint4 *>(p));
            const uint32_t h[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = __uint_as_float(h[j] << 16);
                v[2 * j + 1] = __uint_as_float(h[j] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float x = 0.0f;
        if (c + j < W) {
            if (sizeof(T) == 4) x = reinterpret_cast<const float *>(p)[j];
            else x = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p)[j] << 16);
        }
        v[j] = x;
    }
}

__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
    return m;
}
__device__ __forceinline__ float amax16lanes(float m) {
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}

__device__ __forceinline__ void store_codes8(uint8_t *dst, int64_t c, int64_t W, uint2 q, bool vector) {
    if (vector && c + 8 <= W) {
        *reinterpret_cast<uint2 *>(dst) = q;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (c + j < W) dst[j] = (uint8_t)((j < 4 ? q.x >> (8 * j) : q.y >> (8 * (j - 4))) & 0xffu);
}

// One scale for 128 values of a row.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(Source src, uint8_t *codes, float *scales, int64_t rows, int64_t H, int64_t W, bool vector_out) {
    const int64_t blocks = f8_blocks(W);
    const int sub = threadIdx.x & 15;
    // (all lanes of a warp take part in the shuffles)
    const int64_t total = rows * blocks, step = (int64_t)gridDim.x * 16;
    for (int64_t first = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 5) * 2; first < total; first += step) {
        const int64_t i = first + ((threadIdx.x >> 4) & 1);
        const int64_t r = i / blocks, b = i - r * blocks, o = r / H;
        const int64_t c = b * kF8Block + sub * 8;
        float v[8] = {};
        if (i < total) load8<T>(src, o, r - o * H, c, W, v);
        const float scale = f8_scale(amax16lanes(amax8(v)));
        if (i < total) {
            store_codes8(codes + r * W + c, c, W, f8_pack8(v, scale), vector_out);
            if (sub == 0) scales[i] = scale;
        }
    }
}

// One scale for a block of 128 x 128: a thread block each, 32 values a thread. (256 threads with 64 values, 100 registers, took 30 us for 4096 x 4096 fp32.)
template <typename T>
__global__ void __launch_bounds__(512, 2) quantize_blocks_kernel(Source src, uint8_t *codes, float *scales, int64_t H, int64_t W, bool vector_out) {
    __shared__ float red[16];
    const int64_t wb = f8_blocks(W), hb = f8_blocks(H);
    const int64_t i = blockIdx.x, o = i / (hb * wb), h0 = (i / wb % hb) * kF8Block, c = i % wb * kF8Block + (threadIdx.x & 15) * 8;
    const int r0 = threadIdx.x >> 4;
    float v[4][8], m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = h0 + r0 + 32 * j;
        if (r < H) {
            load8<T>(src, o, r, c, W, v[j]);
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[j][q] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, amax8(v[j]));
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) m = fmaxf(m, red[j]);
    const float scale = f8_scale(m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = h0 + r0 + 32 * j;
        if (r < H) store_codes8(codes + (o * H + r) * W + c, c, W, f8_pack8(v[j], scale), vector_out);
    }
    if (threadIdx.x == 0) scales[i] = scale;
}

// Activations into the operand layout. Without `pos` row r goes to row r; with it to the rows pos[r * k + j] (-1: nowhere).
__global__ void __launch_bounds__(256) quantize_operand_kernel(Source src, int64_t rows, int64_t H, int64_t K, F8Activation out, const int32_t *pos, int k,
                                                               bool early) {
    if (early) ptx::grid_dep_launch();
    ptx::grid_dep_wait();
    if (!early) ptx::grid_dep_launch();
    const int64_t blocks = f8_blocks(K);
    const int sub = threadIdx.x & 15;
    const int64_t total = rows * blocks, step = (int64_t)gridDim.x * 16;
    for (int64_t first = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 5) * 2; first < total; first += step) {
        const int64_t i = first + ((threadIdx.x >> 4) & 1);
        const int64_t r = i / blocks, b = i - r * blocks, o = r / H;
        const int64_t c = b * kF8Block + sub * 8;
        float v[8] = {};
        if (i < total) load8<uint16_t>(src, o, r - o * H, c, K, v);
        const float scale = f8_scale(amax16lanes(amax8(v)));
        if (i >= total) continue;
        const uint2 q = f8_pack8(v, scale);
        for (int j = 0; j < k; ++j) {
            const int64_t to = pos ? pos[r * k + j] : r;
            if (to < 0) continue;
            *reinterpret_cast<uint2 *>(out.codes + f8_act_offset(out.rows_padded, b, to, sub * 8)) = q;
            if (sub == 0) out.scales[to * out.scale_pitch + b] = scale;
        }
    }
}

Source make_source(const void *ptr, int dtype, bool row_major, int64_t H, int64_t W) {
    Source s;
    s.ptr = ptr;
    s.tiled = !row_major;
    s.pitch = row_major ? W : (W + 31) / 32;
    s.slab = row_major ? H * W : round_up32(H) * round_up32(W);
    s.vector = (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && (!row_major || W % (dtype == TTB_FLOAT32 ? 4 : 8) == 0);
    return s;
}

}  // namespace

int32_t launch_quantize_operand(const void *a, bool row_major, int64_t outer, int64_t H, int64_t K, const F8Activation &out, const int32_t *pos, int k,
                                bool early, cudaStream_t stream) {
    const int64_t rows = outer * H, want = (rows * f8_blocks(K) + 15) / 16;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(want < 148 * 8 ? (want > 0 ? want : 1) : 148 * 8));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, quantize_operand_kernel, make_source(a, TTB_BFLOAT16, row_major, H, K), rows, H, K, out, pos, k, early));
    TTB_LAUNCH_CHECK("quantize_operand");
    return TTB_OK;
}

}  // namespace ttb

using ttb::fail;

extern "C" int32_t ttb_quantize_float8(const void *src, int32_t src_dtype, int32_t src_row_major, void *codes, void *scales, int64_t outer, int64_t H,
                                       int64_t W, int32_t block_rows, void *stream) {
    if (!src || !codes || !scales) return fail(TTB_E_INVALID, "ttb_quantize_float8: null pointer");
    if (src_dtype != TTB_FLOAT32 && src_dtype != TTB_BFLOAT16) return fail(TTB_E_UNSUPPORTED, "ttb_quantize_float8: the source must be float32 or bfloat16");
    if (block_rows != 1 && block_rows != ttb::kF8Block) return fail(TTB_E_INVALID, "ttb_quantize_float8: block_rows must be 1 or 128, got %d", block_rows);
    if (outer <= 0 || H <= 0 || W <= 0) return fail(TTB_E_INVALID, "ttb_quantize_float8: the extents must be positive");
    const int64_t limit = int64_t(1) << 40;
    if ((double)outer * (double)H * (double)W > (double)limit)
        return fail(TTB_E_UNSUPPORTED, "ttb_quantize_float8: too many elements");
    if ((reinterpret_cast<uintptr_t>(src) & (src_dtype == TTB_FLOAT32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(scales) & 3))
        return fail(TTB_E_INVALID, "ttb_quantize_float8: misaligned pointer");
    const ttb::Source s = ttb::make_source(src, src_dtype, src_row_major != 0, H, W);
    const bool vector_out = (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && W % 8 == 0;
    if (block_rows == 1) {
        const int64_t want = (outer * H * ttb::f8_blocks(W) + 15) / 16;
        const unsigned grid = (unsigned)(want < 148 * 64 ? want : 148 * 64);
        auto kernel = src_dtype == TTB_FLOAT32 ? ttb::quantize_rows_kernel<float> : ttb::quantize_rows_kernel<uint16_t>;
        kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(s, (uint8_t *)codes, (float *)scales, outer * H, H, W, vector_out);
    } else {
        const int64_t blocks = outer * ttb::f8_blocks(H) * ttb::f8_blocks(W);
        if (blocks > INT32_MAX) return fail(TTB_E_UNSUPPORTED, "ttb_quantize_float8: too many blocks");
        auto kernel = src_dtype == TTB_FLOAT32 ? ttb::quantize_blocks_kernel<float> : ttb::quantize_blocks_kernel<uint16_t>;
        kernel<<<(unsigned)blocks, 512, 0, (cudaStream_t)stream>>>(s, (uint8_t *)codes, (float *)scales, H, W, vector_out);
    }
    TTB_LAUNCH_CHECK("quantize_float8");
    return TTB_OK;
}
