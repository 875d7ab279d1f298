// Quantisation to float8 codes with block scales (float8.cuh has the format).
//
// Weights and tensors a user keeps: codes row-major [outer, H, W], scales [outer, ceil(H / block_rows), ceil(W / 128)]. Activations of
// a matmul: the operand layout of float8.cuh in scratch. Sixteen lanes hold the 128 values of a row's block, eight each, so that the
// largest value needs four shuffles and every access is 16 bytes wide. Each value is read once and its code written once; bound by instructions (190 for 256 values
// at 72 % of the issue slots), which keeps fp32 at 5.2 and bfloat16 at 3.2 to 3.8 TB/s (8192 x 8192: 65 and 53 to 63 us).
#include "epilogue.cuh"
#include "float8.cuh"
#include "matmul_float8.cuh"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>

namespace ttb {
namespace {

struct Source {
    const void *ptr;
    int64_t pitch;      // elements between rows (row-major), tiles per tile row (tiled)
    int64_t slab;       // elements between matrices
    bool tiled, vector; // vector: eight neighbours of a row are 16-byte aligned
};

// Columns c .. c + 7 of a row as they lie in memory; what lies behind W is zero.
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ const T *place_of(const Source &s, int64_t o, int64_t row, int64_t c) {
    return reinterpret_cast<const T *>(s.ptr) + o * s.slab + (s.tiled ? tiled_offset(row, c, s.pitch) : row * s.pitch + c);
}
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const Source &s, int64_t o, int64_t row, int64_t c) {   // all there and aligned
    const uint4 *p = reinterpret_cast<const uint4 *>(place_of<T>(s, o, row, c));
    Raw8<T> v;
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
        const uint4 a = __ldcg(p + j);
        v.w[4 * j] = a.x; v.w[4 * j + 1] = a.y; v.w[4 * j + 2] = a.z; v.w[4 * j + 3] = a.w;
    }
    return v;
}
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const Source &s, int64_t o, int64_t row, int64_t c, int64_t W) {
    if (s.vector && c + 8 <= W) return load8<T>(s, o, row, c);
    constexpr int N = 2 * sizeof(T);   // words
    const T *p = place_of<T>(s, o, row, c);
    Raw8<T> v;
    constexpr int per = 8 / N;   // values of a word
#pragma unroll
    for (int j = 0; j < N; ++j) {
        v.w[j] = 0;
#pragma unroll
        for (int q = 0; q < per; ++q)
            if (c + j * per + q < W) {
                if (sizeof(T) == 4) v.w[j] = reinterpret_cast<const uint32_t *>(p)[j];
                else v.w[j] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[2 * j + q] << (16 * q);
            }
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void values8(const Raw8<T> &r, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (sizeof(T) == 4) v[j] = __uint_as_float(r.w[j % (2 * sizeof(T))]);
        else v[j] = __uint_as_float(j & 1 ? r.w[j / 2] & 0xffff0000u : r.w[j / 2] << 16);
    }
}

// The largest magnitude; a NaN counts nothing.
template <typename T>
__device__ __forceinline__ float amax8(const Raw8<T> &r) {
    if (sizeof(T) == 2) {
        __nv_bfloat162 m[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = r.w[j] & 0x7fff7fffu;
            m[j] = *reinterpret_cast<const __nv_bfloat162 *>(&w);
        }
        const __nv_bfloat162 a = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
        return fmaxf(fmaxf(__low2float(a), __high2float(a)), 0.0f);   // (0: all are NaN)
    }
    float v[8], m = 0.0f;
    values8(r, v);
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

// The blocks of 128 values of the rows of [outer, H, W], sixteen lanes each, two a warp, are dealt out to the warps round by round. Which matrix, row and block a
// lane's next one is follows from the last one's by additions (64-bit divisions for each cost as much as its codes). The launchers keep the blocks below 2^31.
struct RowWalk {
    uint32_t i, b, h, o, step, step_b, step_h, step_o, total, blocks, H;
    __device__ RowWalk(int64_t rows, int64_t H_, int64_t W) : total((uint32_t)(rows * f8_blocks(W))), blocks((uint32_t)f8_blocks(W)), H((uint32_t)H_) {
        step = gridDim.x * 16;
        i = blockIdx.x * 16 + (threadIdx.x >> 4);
        split(i, b, h, o);
        split(step, step_b, step_h, step_o);
    }
    __device__ void split(uint32_t x, uint32_t &block, uint32_t &in, uint32_t &out) const {
        const uint32_t row = x / blocks;
        block = x - row * blocks;
        out = row / H;
        in = row - out * H;
    }
    __device__ bool here() const { return i < total; }
    __device__ bool warp_here() const { return i - ((threadIdx.x >> 4) & 1) < total; }   // (all lanes of a warp take part in the shuffles)
    __device__ void next() {
        i += step;
        b += step_b;
        h += step_h;
        o += step_o;
        if (b >= blocks) { b -= blocks; ++h; }
        if (h >= H) { h -= H; ++o; }
    }
};

// One scale for 128 values of a row. The values of the next block are on their way while this one's codes are made.
template <typename T>
__global__ void __launch_bounds__(256, 6) quantize_rows_kernel(Source src, uint8_t *codes, float *scales, int64_t rows, int64_t H, int64_t W, bool vector_out) {
    const int sub = threadIdx.x & 15;
    RowWalk at(rows, H, W);
    auto load = [&]() { return at.here() ? load8<T>(src, at.o, at.h, (int64_t)at.b * kF8Block + sub * 8, W) : Raw8<T>{}; };
    Raw8<T> raw = load();
    while (at.warp_here()) {
        const uint32_t i = at.i;
        const int64_t r = (int64_t)at.o * H + at.h, c = (int64_t)at.b * kF8Block + sub * 8;
        float v[8];
        values8(raw, v);
        const float m = amax8(raw);
        at.next();
        raw = load();
        const float scale = f8_scale(amax16lanes(m));
        if (i < at.total) {
            store_codes8(codes + r * W + c, c, W, f8_pack8(v, scale), vector_out);
            if (sub == 0) scales[i] = scale;
        }
    }
}

// One scale for a block of 128 x 128: a thread block each, 32 values a thread. (256 threads with 64 values, 100 registers, took 30 us for 4096 x 4096 fp32.)
template <typename T>
__global__ void __launch_bounds__(512, sizeof(T) == 4 ? 2 : 3) quantize_blocks_kernel(Source src, uint8_t *codes, float *scales, int64_t H, int64_t W, bool vector_out) {
    __shared__ float red[16];
    const uint32_t wb = (uint32_t)f8_blocks(W), hb = (uint32_t)f8_blocks(H), i = blockIdx.x, row = i / wb;   // (the launcher keeps the blocks below 2^31)
    const int64_t o = row / hb, h0 = (int64_t)(row - row / hb * hb) * kF8Block, c = (int64_t)(i - row * wb) * kF8Block + (threadIdx.x & 15) * 8;
    const int r0 = threadIdx.x >> 4;
    Raw8<T> raw[4];
    float m = 0.0f;
    if (src.vector && h0 + kF8Block <= H && c + 8 <= W) {
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = load8<T>(src, o, h0 + r0 + 32 * j, c);
    } else {
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
            const int64_t r = h0 + r0 + 32 * j;
            const Raw8<T> x = r < H ? load8<T>(src, o, r, c, W) : Raw8<T>{};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q == j) raw[q] = x;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, amax8(raw[j]));
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
        float v[8];
        values8(raw[j], v);
        if (r < H) store_codes8(codes + (o * H + r) * W + c, c, W, f8_pack8(v, scale), vector_out);
    }
    if (threadIdx.x == 0) scales[i] = scale;
}

// Activations into the operand layout. Without `pos` row r goes to row r; with it to the rows pos[r * k + j] (-1: nowhere).
__global__ void __launch_bounds__(256, 6) quantize_operand_kernel(Source src, int64_t rows, int64_t H, int64_t K, F8Activation out, const int32_t *pos, int k,
                                                               bool early) {
    if (early) ptx::grid_dep_launch();
    ptx::grid_dep_wait();
    if (!early) ptx::grid_dep_launch();
    const int sub = threadIdx.x & 15;
    RowWalk at(rows, H, K);
    auto load = [&]() { return at.here() ? load8<uint16_t>(src, at.o, at.h, (int64_t)at.b * kF8Block + sub * 8, K) : Raw8<uint16_t>{}; };
    Raw8<uint16_t> raw = load();
    while (at.warp_here()) {
        const uint32_t i = at.i;
        const int64_t r = (int64_t)at.o * H + at.h, b = at.b;
        float v[8];
        values8(raw, v);
        const float m = amax8(raw);
        at.next();
        raw = load();
        const float scale = f8_scale(amax16lanes(m));
        if (i >= at.total) continue;
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
    cfg.gridDim = dim3((unsigned)(want < 148 * 6 ? (want > 0 ? want : 1) : 148 * 6));
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
    const int64_t row_blocks = block_rows == 1 ? outer * H : outer * ttb::f8_blocks(H), blocks = row_blocks * ttb::f8_blocks(W);
    if (outer * H > INT32_MAX || blocks > INT32_MAX) return fail(TTB_E_UNSUPPORTED, "ttb_quantize_float8: too many blocks");
    if (block_rows == 1) {
        const int64_t want = (blocks + 15) / 16;
        const unsigned grid = (unsigned)(want < 148 * 6 ? want : 148 * 6);
        auto kernel = src_dtype == TTB_FLOAT32 ? ttb::quantize_rows_kernel<float> : ttb::quantize_rows_kernel<uint16_t>;
        kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(s, (uint8_t *)codes, (float *)scales, outer * H, H, W, vector_out);
    } else {
        auto kernel = src_dtype == TTB_FLOAT32 ? ttb::quantize_blocks_kernel<float> : ttb::quantize_blocks_kernel<uint16_t>;
        kernel<<<(unsigned)blocks, 512, 0, (cudaStream_t)stream>>>(s, (uint8_t *)codes, (float *)scales, H, W, vector_out);
    }
    TTB_LAUNCH_CHECK("quantize_float8");
    return TTB_OK;
}
