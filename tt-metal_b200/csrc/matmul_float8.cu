// Matmul of float8 operands with block scales: out[m, n] = act(sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} a[m, k] w[n, k] + bias[n]), for all
// rows with one weight or for runs of rows with an expert's weight each (a grouped matmul), optionally as a gated pair whose product is quantised
// again for the next matmul.
//
// A tile is 128 rows x W blocks of 128 weight rows (output columns). Per block of 128 K values
//   * one warp fetches the operands: the weight's 128 x 128 bytes straight from the row-major tensor with a 128-byte-swizzled tensor map, the rows'
//     codes with one contiguous copy (they are kept in the operand layout, float8.cuh);
//   * one warp issues four tcgen05.mma (kind::f8f6f4, 128 x 128 W x 32) into one of two tensor memory accumulators;
//   * eight warps add the finished accumulator, times the two scales, to fp32 sums in registers while the MMAs fill the other. A thread holds one row
//     and 64 W columns, so the scales are one number a block and thread.
// The tensor cores' own chain of additions is thus 128 products long whatever K is.
// Every mbarrier wait is bounded; a wait that runs out raises a status word instead of hanging.
#include <cuda.h>

#include "epilogue.cuh"
#include "matmul_float8.cuh"
#include "sm100_ptx.cuh"

namespace ttb {
unsigned barrier_limit_kcycles();
int32_t status_word_address(int **out);
int32_t tensor_map_encoder(void **out);
namespace {

using namespace ptx;

constexpr int BM = 128;
constexpr int kMaxStages = 12;
constexpr int kEpiWarps = 8, kProducerWarp = 8, kMmaWarp = 9, kThreads = 32 * 10;
constexpr int kSmemLimit = 232448 - 1024;   // the rest: static shared memory
constexpr int kMaxExperts = 1024;

struct alignas(64) Args {
    CUtensorMap wmap[2];
    const float *sw[2];
    F8Activation a, h;
    const int32_t *offsets;
    const uint16_t *bias;
    void *out;
    int64_t N;
    int rows, experts, Kb, Nb, ct;   // ct: column tiles
    int a_rows, stages, stage_bytes; // rows of a stage's activations (a multiple of 8); the ring
    int act, out_dtype, out_row_major, bias_row_major, out_aligned;   // out_aligned: bytes that a store may have
    unsigned wait_limit;
    int *status;
};

__device__ __forceinline__ long long wait_clocks(const Args &p) { return (long long)p.wait_limit << 10; }

// K-major operand with the 128-byte swizzle: rows of 128 bytes, eight rows form a 1024-byte atom in which 16-byte chunk c of row r lies at c ^ r.
__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor for kind::f8f6f4, both operands e4m3 and K-major, fp32 accumulator.
__host__ __device__ constexpr uint32_t instr_desc_e4m3(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

__device__ __forceinline__ void mma_e4m3_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// A tile of the launch: rows [lo, hi) of expert e, kept as rows base .. base + 127 (base: a multiple of eight, at most lo), column tile c.
struct Tile {
    int e, lo, hi, base, c;
};

__device__ __forceinline__ int row_tiles(int lo, int hi) { return hi > lo ? (hi - (lo & ~7) + BM - 1) / BM : 0; }

// Tile t of the launch. Row tiles vary fastest (up to 16 of them), so that blocks that run together share weights.
__device__ __forceinline__ Tile tile_of(const Args &p, const int *off, const int *cum, int t) {
    Tile s;
    int lo = 0, hi = p.rows;
    s.e = 0;
    if (p.experts) {
        int a = 0, b = p.experts;   // the last expert with cum[e] <= t
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if (cum[m] <= t) a = m; else b = m;
        }
        s.e = a;
        t -= cum[a];
        lo = off[a];
        hi = off[a + 1];
    }
    const int rt = row_tiles(lo, hi), per = 16 * p.ct;
    const int group = t / per, in = t - group * per, height = min(16, rt - group * 16);
    const int r = group * 16 + in % height;
    s.c = in / height;
    s.base = (lo & ~7) + r * BM;
    s.lo = max(lo, s.base);
    s.hi = min(hi, s.base + BM);
    return s;
}

// 16 columns from n on of one row.
__device__ __forceinline__ void store16(const Args &p, int64_t row, int64_t n, const float *v) {
    const int64_t width = p.out_row_major ? p.N : ((p.N + 31) & ~(int64_t)31);
    if (n >= width) return;
    const int64_t off = p.out_row_major ? row * p.N + n : tiled_offset(row, n, width >> 5);
    if (p.out_dtype == TTB_FLOAT32) {
        float *o = reinterpret_cast<float *>(p.out) + off;
        if (p.out_aligned >= 16 && n + 16 <= width) {
#pragma unroll
            for (int q = 0; q < 4; ++q) reinterpret_cast<float4 *>(o)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (n + j < width) o[j] = v[j];
        }
    } else {
        uint16_t *o = reinterpret_cast<uint16_t *>(p.out) + off;
        if (p.out_aligned >= 16 && n + 16 <= width) {
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = (uint32_t)f32_to_bf16_bits(v[2 * j]) | ((uint32_t)f32_to_bf16_bits(v[2 * j + 1]) << 16);
            reinterpret_cast<uint4 *>(o)[0] = make_uint4(h[0], h[1], h[2], h[3]);
            reinterpret_cast<uint4 *>(o)[1] = make_uint4(h[4], h[5], h[6], h[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (n + j < width) o[j] = f32_to_bf16_bits(v[j]);
        }
    }
}

template <int ACT, int NC>
__device__ __forceinline__ void finish_row(const Args &p, int64_t row, int64_t n0, float (&acc)[NC]) {
#pragma unroll
    for (int q = 0; q < NC; q += 16) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int64_t n = n0 + q + j;
            float b = 0.0f;
            if (p.bias && n < p.N) b = p.bias_row_major ? __uint_as_float((uint32_t)__ldg(p.bias + n) << 16) : bias_at(p.bias, n);
            v[j] = apply_activation_t<ACT>(acc[q + j] + b);
        }
        store16(p, row, n0 + q, v);
        asm volatile("" ::: "memory");   // (keeps the compiler from fetching all groups' bias values at once)
    }
}

// act(g) * u of one row's 64 columns, quantised with the scale of all 128: the warp with the other 64 exchanges its largest magnitudes through `red` (a
// barrier of the two warps, in bounded waits like every other). Returns false where that ran out.
template <int ACT>
__device__ __forceinline__ bool finish_gated(const Args &p, int row, bool valid, int c, int half, int lane_row, float (&acc)[128], float (*red)[BM], uint32_t bar,
                                             volatile int *abort_flag) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
        acc[j] = apply_activation_t<ACT>(acc[j]) * acc[64 + j];
        m = fmaxf(m, fabsf(acc[j]));
    }
    auto meet = [&](uint32_t parity) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
        return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, 55, wait_clocks(p)));
    };
    red[half][lane_row] = m;
    if (!meet(0)) return false;
    const float scale = f8_scale(fmaxf(m, red[half ^ 1][lane_row]));
    if (!meet(1)) return false;   // (the next tile writes `red` again)
    if (!valid) return true;
#pragma unroll
    for (int q = 0; q < 64; q += 16) {
        float v[8], u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = acc[q + j];
            u[j] = acc[q + 8 + j];
        }
        const uint2 x = f8_pack8(v, scale), y = f8_pack8(u, scale);
        *reinterpret_cast<uint4 *>(p.h.codes + f8_act_offset(p.h.rows_padded, c, row, half * 64 + q)) = make_uint4(x.x, x.y, y.x, y.y);
    }
    if (half == 0) p.h.scales[row * p.h.scale_pitch + c] = scale;
    return true;
}

// W: weight blocks per tile. GATED: the two blocks are the same rows of the two weights.
template <int W, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) matmul_float8_kernel(const __grid_constant__ Args p) {
    static_assert(!GATED || W == 2, "a gated tile takes a block of either weight");
    constexpr int NC = 64 * W;   // columns of an epilogue thread
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 6];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_word;
    __shared__ int tiles_word;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    uint8_t *after = smem + p.stages * p.stage_bytes;
    float (*red)[BM] = reinterpret_cast<float (*)[BM]>(after);
    int *off = reinterpret_cast<int *>(after + (GATED ? 2 * BM * 4 : 0));
    int *cum = off + p.experts + 1;
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto done = [&](int s) { return bar0 + 8u * (kMaxStages + s); };   // the MMAs of the stage have read it and its accumulator is complete
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * kMaxStages + b); };
    auto pair = [&](int quad) { return bar0 + 8u * (2 * kMaxStages + 2 + quad); };
    volatile int *abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(done(s), 1);
        }
        for (int b = 0; b < 2; ++b) mbar_init(acc_empty(b), kEpiWarps);
        for (int q = 0; q < 4; ++q) mbar_init(pair(q), 2);
        abort_word = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&tmem_slot), 256 * W);
        tmem_relinquish();
    }
    grid_dep_wait();
    grid_dep_launch();
    if (p.experts) {
        for (int i = threadIdx.x; i <= p.experts; i += kThreads) off[i] = p.offsets[i];
        __syncthreads();
        if (warp == 0) {
            int run = 0;
            for (int i = 0; i < p.experts; i += 32) {
                int x = i + lane < p.experts ? row_tiles(off[i + lane], off[i + lane + 1]) * p.ct : 0, sum = x;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += y;
                }
                if (i + lane < p.experts) cum[i + lane] = run + sum - x;
                run += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (lane == 0) tiles_word = run;
        }
    } else if (threadIdx.x == 0) {
        tiles_word = row_tiles(0, p.rows) * p.ct;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    const int tiles = tiles_word;

    if (warp == kProducerWarp) {
        const bool leader = elect_one();
        fence_proxy_async_global();   // the activations were written by ordinary stores of the kernel before
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const Tile T = tile_of(p, off, cum, t);
            const uint32_t a_bytes = (uint32_t)(((T.hi + 7) & ~7) - T.base) * kF8Block;
            for (int kb = 0; kb < p.Kb; ++kb) {
                if (!__all_sync(0xffffffffu, mbar_wait(done(s), ph ^ 1, abort_flag, p.status, 51, wait_clocks(p)))) { ok = false; break; }
                if (leader) {
                    const uint32_t dst = sbase + (uint32_t)(s * p.stage_bytes), w_dst = dst + (uint32_t)(p.a_rows * kF8Block);
                    mbar_arrive_expect_tx(full(s), a_bytes + W * kF8BlockBytes);
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        tma_load_3d_plain(w_dst + j * kF8BlockBytes, &p.wmap[GATED ? j : 0], kb * kF8Block, (GATED ? T.c : T.c * W + j) * kF8Block, T.e, full(s));
                    bulk_g2s_plain(dst, p.a.codes + ((int64_t)kb * p.a.rows_padded + T.base) * kF8Block, a_bytes, full(s));
                }
                if (++s == p.stages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == kMmaWarp) {
        const bool leader = elect_one();
        constexpr uint32_t idesc = instr_desc_e4m3(BM, 128 * W);
        int s = 0, n = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x)
            for (int kb = 0; kb < p.Kb; ++kb, ++n) {
                const int buf = n & 1;
                if (!__all_sync(0xffffffffu, mbar_wait(acc_empty(buf), (uint32_t)(((n >> 1) & 1) ^ 1), abort_flag, p.status, 52, wait_clocks(p))) ||
                    !__all_sync(0xffffffffu, mbar_wait(full(s), ph, abort_flag, p.status, 53, wait_clocks(p)))) { ok = false; break; }
                tc_fence_after_sync();
                if (leader) {
                    const uint32_t src = sbase + (uint32_t)(s * p.stage_bytes);
                    const uint64_t a = smem_desc_sw128(src), b = smem_desc_sw128(src + (uint32_t)(p.a_rows * kF8Block));
#pragma unroll
                    for (int k = 0; k < 4; ++k)   // 32 bytes of K further: two 16-byte units in the descriptor's address
                        mma_e4m3_ss(tmem_base + (uint32_t)(buf * 128 * W), a + 2 * k, b + 2 * k, idesc, k > 0);
                    mma_commit(done(s));
                }
                if (++s == p.stages) { s = 0; ph ^= 1; }
            }
    } else {
        const int quad = warp & 3, half = warp >> 2;
        const int lane_row = quad * 32 + lane;
        int s = 0, n = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const Tile T = tile_of(p, off, cum, t);
            const int row = T.base + lane_row;
            const bool valid = row >= T.lo && row < T.hi;
            const bool warp_valid = T.base + quad * 32 < T.hi;
            const float *sa = p.a.scales + (int64_t)min(row, T.hi - 1) * p.a.scale_pitch;
            const float *sw0, *sw1;
            if (GATED) {
                sw0 = p.sw[0] + ((int64_t)T.e * p.Nb + T.c) * p.Kb;
                sw1 = p.sw[1] + ((int64_t)T.e * p.Nb + T.c) * p.Kb;
            } else {
                sw0 = sw1 = p.sw[0] + ((int64_t)T.e * p.Nb + min(T.c * W + (W == 2 ? half : 0), p.Nb - 1)) * p.Kb;
            }
            // columns of the accumulator: 64 of either weight (gated), else NC neighbours
            const uint32_t col0 = GATED ? half * 64 : half * NC;
            float acc[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
            for (int kb = 0; kb < p.Kb; ++kb, ++n) {
                const int buf = n & 1;
                const float x = __ldcg(sa + kb), f0 = x * __ldg(sw0 + kb), f1 = GATED ? x * __ldg(sw1 + kb) : f0;
                if (!__all_sync(0xffffffffu, mbar_wait(done(s), ph, abort_flag, p.status, 54, wait_clocks(p)))) { ok = false; break; }
                tc_fence_after_sync();
                if (warp_valid) {
                    const uint32_t t0 = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * 128 * W);
#pragma unroll
                    for (int q = 0; q < NC; q += 32) {
                        uint32_t r0[16], r1[16];
                        const uint32_t c = GATED ? (q / 64) * 128 + half * 64 + (q & 63) : col0 + q;
                        tmem_ld16(t0 + c, r0);
                        tmem_ld16(t0 + c + 16, r1);
                        tmem_ld_wait();
                        const float f = GATED && q >= 64 ? f1 : f0;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            acc[q + j] = fmaf(__uint_as_float(r0[j]), f, acc[q + j]);
                            acc[q + 16 + j] = fmaf(__uint_as_float(r1[j]), f, acc[q + 16 + j]);
                        }
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(buf));
                if (++s == p.stages) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            if constexpr (GATED) {
                TTB_DISPATCH_ACT(p.act, ok = finish_gated<ACT>(p, row, valid, T.c, half, lane_row, acc, red, pair(quad), abort_flag));
            } else {
                if (valid) TTB_DISPATCH_ACT(p.act, (finish_row<ACT, NC>(p, row, (int64_t)T.c * 128 * W + half * NC, acc)));
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        // A wait ran out: give copies and MMAs still in flight a bounded time to finish before the block's memory is released.
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 256 * W);
    }
}

// [experts, N, K] bytes, 128 x 128 boxes with the 128-byte swizzle; rows and K values behind the end are zeros.
int32_t make_map(const void *codes, int64_t experts, int64_t N, int64_t K, CUtensorMap &map) {
    using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    void *fn = nullptr;
    if (int32_t rc = tensor_map_encoder(&fn)) return rc;
    const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)N, (cuuint64_t)experts};
    const cuuint64_t strides[2] = {(cuuint64_t)K, (cuuint64_t)(N * K)};
    const cuuint32_t box[3] = {kF8Block, kF8Block, 1}, estr[3] = {1, 1, 1};
    const CUresult r = reinterpret_cast<EncodeFn>(fn)(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(codes), dims, strides, box, estr,
                                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TTB_E_CUDA, "cuTensorMapEncodeTiled failed with %d for a float8 weight", (int)r);
    return TTB_OK;
}

template <int W, bool GATED>
int32_t launch(const Args &p, int grid, int smem, int dev, cudaStream_t stream) {
    static Once once[64];
    if (int32_t rc = once[dev].run([&]() -> int32_t {
            TTB_CUDA_TRY(cudaFuncSetAttribute(matmul_float8_kernel<W, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
            return TTB_OK;
        }))
        return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, matmul_float8_kernel<W, GATED>, p));
    TTB_LAUNCH_CHECK("matmul_float8");
    return TTB_OK;
}

}  // namespace

int32_t launch_matmul_float8(const F8Matmul &m, cudaStream_t stream) {
    Args p;
    const int64_t experts = m.experts ? m.experts : 1;
    if (m.experts > kMaxExperts) return fail(TTB_E_UNSUPPORTED, "ttb_experts_mlp_float8: at most %d experts", kMaxExperts);
    if (int32_t rc = make_map(m.w[0].codes, experts, m.N, m.K, p.wmap[0])) return rc;
    p.wmap[1] = p.wmap[0];
    if (m.gated)
        if (int32_t rc = make_map(m.w[1].codes, experts, m.N, m.K, p.wmap[1])) return rc;
    p.sw[0] = m.w[0].scales;
    p.sw[1] = m.w[1].scales;
    p.a = m.a; p.h = m.h;
    p.offsets = m.offsets; p.bias = m.bias; p.out = m.out; p.N = m.N;
    p.rows = (int)m.rows; p.experts = m.experts;
    p.Kb = (int)f8_blocks(m.K); p.Nb = (int)f8_blocks(m.N);
    const int W = m.gated ? 2 : 1;
    p.ct = m.gated ? p.Nb : (p.Nb + W - 1) / W;
    p.a_rows = (int)(f8_rows_padded(m.rows) < BM ? f8_rows_padded(m.rows) : BM);
    p.stage_bytes = p.a_rows * kF8Block + W * kF8BlockBytes;
    const int extra = (m.gated ? 2 * BM * 4 : 0) + (m.experts ? 4 * (2 * m.experts + 1) : 0) + 1024;
    p.stages = (kSmemLimit - extra) / p.stage_bytes;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    p.act = m.act; p.out_dtype = m.out_dtype; p.out_row_major = m.out_row_major; p.bias_row_major = m.bias_row_major;
    // 16 neighbouring columns of a row start at a multiple of this many bytes
    p.out_aligned = 0;
    if (!m.gated && (reinterpret_cast<uintptr_t>(m.out) & 15) == 0 && (!m.out_row_major || m.N * (m.out_dtype == TTB_FLOAT32 ? 4 : 2) % 16 == 0)) p.out_aligned = 16;
    p.wait_limit = barrier_limit_kcycles();
    if (int32_t rc = status_word_address(&p.status)) return rc;
    int dev = 0, sms = 0;
    TTB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: device index %d is out of range", dev);
    TTB_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const int64_t most = (f8_rows_padded(m.rows) / BM + 1 + m.experts) * (int64_t)p.ct;   // an upper bound for a grouped matmul
    if (most > INT32_MAX / 2) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: too many output tiles");
    const int grid = most < sms ? (int)most : sms, smem = p.stages * p.stage_bytes + extra;
    return m.gated ? launch<2, true>(p, grid, smem, dev, stream) : launch<1, false>(p, grid, smem, dev, stream);
}

}  // namespace ttb

using ttb::fail;

namespace {
constexpr int64_t kMaxExtent = int64_t(1) << 24;   // rows, K and N: tile coordinates and row indexes stay far inside 32 bits

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

bool misaligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// Scratch of quantised rows; advances `at`.
ttb::F8Activation place(uint8_t *base, int64_t &at, int64_t rows, int64_t cols) {
    ttb::F8Activation a;
    a.rows_padded = ttb::f8_rows_padded(rows);
    a.scale_pitch = ttb::f8_scale_pitch(cols);
    a.codes = base + at;
    at = up(at + a.rows_padded * ttb::f8_blocks(cols) * ttb::kF8Block, 1024);
    a.scales = reinterpret_cast<float *>(base + at);
    at = up(at + a.rows_padded * a.scale_pitch * 4, 1024);
    return a;
}
}  // namespace

extern "C" {

int64_t ttb_linear_float8_workspace_bytes(int64_t rows, int64_t K, int64_t N) {
    if (rows <= 0 || K <= 0 || N <= 0 || rows > kMaxExtent || K > kMaxExtent || N > kMaxExtent) return -1;
    int64_t at = 0;
    place(nullptr, at, rows, K);
    return at;
}

int32_t ttb_linear_float8(const void *a, const void *w_codes, const void *w_scales, const void *bias, void *out, int32_t out_dtype, int64_t rows, int64_t K,
                          int64_t N, int32_t activation, int32_t flags, void *workspace, int64_t workspace_bytes, void *stream) {
    if (!a || !w_codes || !w_scales || !out) return fail(TTB_E_INVALID, "ttb_linear_float8: null tensor pointer");
    if (out_dtype != TTB_BFLOAT16 && out_dtype != TTB_FLOAT32) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: output must be bfloat16 or float32");
    if (flags & ~(TTB_MM_A_ROW_MAJOR | TTB_MM_OUT_ROW_MAJOR | TTB_MM_BIAS_ROW_MAJOR)) return fail(TTB_E_INVALID, "ttb_linear_float8: unknown flags %d", flags);
    if (activation < TTB_ACT_NONE || activation > TTB_ACT_SILU) return fail(TTB_E_INVALID, "ttb_linear_float8: unknown activation %d", activation);
    const int64_t need = ttb_linear_float8_workspace_bytes(rows, K, N);
    if (need < 0) return fail(TTB_E_INVALID, "ttb_linear_float8: rows, K and N must be between 1 and 2^24");
    if (K % 16) return fail(TTB_E_INVALID, "ttb_linear_float8: K must be a multiple of 16 (got %lld)", (long long)K);
    const bool a_rm = flags & TTB_MM_A_ROW_MAJOR, out_rm = flags & TTB_MM_OUT_ROW_MAJOR;
    if ((!a_rm || !out_rm) && rows % 32) return fail(TTB_E_INVALID, "ttb_linear_float8: tiled tensors have a multiple of 32 rows (got %lld)", (long long)rows);
    if (misaligned(a, 16) || misaligned(w_codes, 16) || misaligned(w_scales, 4) || misaligned(out, out_dtype == TTB_FLOAT32 ? 4 : 2) || (bias && misaligned(bias, 2)))
        return fail(TTB_E_INVALID, "ttb_linear_float8: activations and codes must be 16-byte aligned, the other tensors as their elements");
    if (!ttb::workspace_serves(workspace, workspace_bytes, need)) return fail(TTB_E_WORKSPACE, "ttb_linear_float8: needs %lld bytes of 256-byte aligned workspace", (long long)need);
    ttb::F8Matmul m = {};
    int64_t at = 0;
    m.a = place(static_cast<uint8_t *>(workspace), at, rows, K);
    m.w[0] = {w_codes, static_cast<const float *>(w_scales)};
    m.rows = rows; m.K = K; m.N = N;
    m.act = activation;
    m.out = out; m.out_dtype = out_dtype; m.out_row_major = out_rm;
    m.bias = static_cast<const uint16_t *>(bias);
    m.bias_row_major = flags & TTB_MM_BIAS_ROW_MAJOR;
    if (int32_t rc = ttb::launch_quantize_operand(a, a_rm, 1, rows, K, m.a, nullptr, 1, nullptr, 0, (cudaStream_t)stream)) return rc;
    return ttb::launch_matmul_float8(m, (cudaStream_t)stream);
}

}  // extern "C"
