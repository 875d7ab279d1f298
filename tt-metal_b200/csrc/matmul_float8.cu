// Matmul of float8 operands with block scales: out[m, n] = act(sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} a[m, k] w[n, k] + bias[n]), for all
// rows with one weight or for runs of rows with an expert's weight each (a grouped matmul), optionally as a gated pair whose product is quantised
// again for the next matmul.
//
// A tile is 128 rows x W blocks of 128 weight rows (output columns). Per block of 128 K values
//   * one warp fetches the operands: the weight's 128 x 128 bytes straight from the row-major tensor with a 128-byte-swizzled tensor map, the rows'
//     codes with one contiguous copy (they are kept in the operand layout, float8.cuh);
//   * one of two warps issues four tcgen05.mma (kind::f8f6f4, 128 x 128 W x 32) into one of 4 / W tensor memory accumulators (waits, four MMAs and a commit
//     take an issuing thread some 650 clocks, a block's MMAs 256 W);
//   * eight warps add the finished accumulator, times the two scales, to fp32 sums in registers while the MMAs fill the others. A thread holds one row
//     and 64 W columns, so the scales are one number a block and thread.
// The tensor cores' own chain of additions is thus 128 products long whatever K is.
// Blocks take whole tiles round by round; the tiles left after the last whole round form one list of (tile, K block) units, which is dealt out evenly.
// The blocks that share a tile leave their fp32 sums in scratch and take a ticket; the last one adds them in block order (so results
// repeat bit for bit) and finishes the rows. No block waits for another. A block's range ends with the first part of a tile, whose other parts are the
// beginnings of other blocks' ranges: it mostly finds them all there and adds them to its sums in registers.
// What bounds it (2048 x 8192 x 28672, 477 us in a graph with the quantiser, 2017 TFLOP/s; 551 us and 1745 TFLOP/s in a loop of seconds, at 1500 MHz under the power
// limit): a block's copies, 48 KB for a unit of 128 x 256 x 128 or 61 B per clock and SM (331 us
// by themselves), with the MMAs 398, and the turns of an accumulator, of which two alternate. A tile's results take 3 us to store (fp32 6), and a unit 0.5.
// Every mbarrier wait is bounded; a wait that runs out raises a status word instead of hanging.
#include "float8_tiles.cuh"

namespace ttb {
unsigned barrier_limit_kcycles();
int32_t status_word_address(int **out);
int32_t tensor_map_encoder(void **out);
int stream_blocks();
int32_t launch_matmul_float8_few(const f8::Args &p, int act, int W, int R, bool gated, int grid, int smem, int dev, cudaStream_t stream);
namespace {

using namespace f8;
using namespace ptx;

// 32 bytes, one sector.
__device__ __forceinline__ void load_partial8(const float *src, float (&v)[8]) {
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(src)
                 : "memory");
}
__device__ __forceinline__ void store_partial8(float *dst, const float *v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

// Eight warps add up, with 64 W columns a thread. (Sixteen with half as many were no faster: 2048 x 8192 x 28672 523 us against 556.)
constexpr int kAddWarps = 8, kFetchWarp = kAddWarps, kIssueWarp = kFetchWarp + 1, kHandWarp = kIssueWarp + kIssuers, kManyThreads = 32 * (kHandWarp + 1);
// Registers a thread: of the 384 x 168 that the block is launched with, the adding warps of the two-block tiles take 216 each (128 sums, 32 values on their way
// from tensor memory) and leave 72 to the other four.
constexpr int kRegs = 168, kAddRegs = 216, kOtherRegs = 72;
static_assert(kAddWarps * kAddRegs + 4 * kOtherRegs == (kAddWarps + 4) * kRegs, "a warpgroup that asks for more than the block holds waits for good");

// W: weight blocks per tile. GATED: the two blocks are the same rows of the two weights.
template <int ACT, int W, bool GATED>
__global__ void __maxnreg__(kRegs) matmul_float8_kernel(const __grid_constant__ Args p) {
    static_assert(!GATED || W == 2, "a gated tile takes a block of either weight");
    constexpr int NC = 64 * W;      // columns of an adding thread
    constexpr int NB = 4 / W;       // accumulators: all of tensor memory
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 11];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_word;
    __shared__ int tiles_word;
    __shared__ volatile int ticket, pending, progress;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    uint8_t *after = smem + p.stages * p.stage_bytes;
    float (*red)[BM] = reinterpret_cast<float (*)[BM]>(after);
    int *off = reinterpret_cast<int *>(after + (GATED ? 2 * BM * 4 : 0));
    int *cum = off + p.experts + 1;
    const uint32_t bar0 = smem_u32(bars);
    auto pair = [&](int quad) { return bar0 + 8u * (2 * kMaxStages + 4 + quad); };
    const uint32_t all_bar = bar0 + 8u * (2 * kMaxStages + 8), handed_bar = all_bar + 8, told_bar = handed_bar + 8;
    volatile int *abort_flag = &abort_word;
    const Ring ring = {sbase, bar0, bar0 + 8u * kMaxStages, bar0 + 8u * (2 * kMaxStages), abort_flag, &progress};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(ring.full(s), 1);
            mbar_init(ring.done(s), 1);
        }
        for (int b = 0; b < NB; ++b) mbar_init(ring.acc_empty(b), kAddWarps);
        for (int q = 0; q < 4; ++q) mbar_init(pair(q), 2);
        mbar_init(all_bar, kAddWarps);
        mbar_init(handed_bar, kAddWarps);
        mbar_init(told_bar, 1);
        abort_word = progress = 0;
        fence_mbar_init();
    }
    if (warp == kIssueWarp) {
        tmem_alloc(smem_u32(&tmem_slot), 512);
        tmem_relinquish();
    }
    // The kernel before may still run (programmatic dependency): what is read before grid_dep_wait - the weights and the experts' row ranges - was written
    // before that kernel let this one start.
    if (!p.early) grid_dep_wait();
    count_tiles(p, off, cum, &tiles_word);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    Walk walk(p, tiles_word);
    Segment seg;

    if (warp >= kAddWarps) {
        if (W == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kFetchWarp) {
            fetch<W, GATED, false, false>(p, ring, walk, off, cum);
        } else if (warp < kIssueWarp + kIssuers) {
            issue_mmas<NB, true>(p, ring, walk, off, cum, warp - kIssueWarp, [&](uint32_t src, int buf, const Tile &) {
                const uint64_t a = smem_desc_sw128(src), b = smem_desc_sw128(src + (uint32_t)(p.a_rows * kF8Block));
#pragma unroll
                for (int k = 0; k < 4; ++k)   // 32 bytes of K further: two 16-byte units in the descriptor's address
                    mma_e4m3_ss(tmem_base + (uint32_t)(buf * 128 * W), a + 2 * k, b + 2 * k, instr_desc_e4m3(BM, 128 * W), k > 0);
            });
        } else {
            hand_over<ACT, W, GATED, false>(p, handed_bar, told_bar, &pending, ring, walk, off, cum);
        }
    } else {
        if (W == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAddRegs));
        grid_dep_wait();
        const int quad = warp & 3, part = warp >> 2;   // 32 rows, half of the columns
        const int lane_row = quad * 32 + lane;
        // accumulator column of sum j: 64 of either weight (gated), else NC neighbours
        auto column = [&](int j) { return GATED ? (j / 64) * 128 + part * 64 + (j & 63) : part * NC + j; };
        Meeting meet = {pair(quad), 0, abort_flag}, meet_all = {all_bar, 0, abort_flag};
        int s = 0, n = 0;
        uint32_t ph = 0;
        bool ok = true;
        // scales of a segment's first blocks: of this thread's row four blocks at a time, of the weight (the same for all threads) lane l that of block 32 i + l; both
        // one step ahead, and the next segment's before this one's rows are finished
        struct Scales {
            const float *sa, *sw0, *sw1;
            float4 xa, xa_next;
            float w0, w0_next, w1, w1_next;
        };
        auto load_a = [&](const float *sa, int kb) { return kb < p.a.scale_pitch ? __ldcg(reinterpret_cast<const float4 *>(sa + kb)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f); };
        auto load_w = [&](const float *sw, int kb) { return kb + lane < p.Kb ? __ldg(sw + kb + lane) : 0.0f; };
        auto scales_of = [&](const Segment &g, const Tile &T) {
            Scales c;
            c.sa = p.a.scales + (int64_t)max(min(T.base + lane_row, T.hi - 1), T.lo) * p.a.scale_pitch;
            const int64_t wrow = (int64_t)T.e * p.Nb + (GATED ? T.c : min(T.c * W + (W == 2 ? part : 0), p.Nb - 1));
            c.sw0 = p.sw[0] + wrow * p.Kb;
            c.sw1 = GATED ? p.sw[1] + wrow * p.Kb : nullptr;
            c.xa = load_a(c.sa, g.kb0 & ~3);
            c.xa_next = load_a(c.sa, (g.kb0 & ~3) + 4);
            c.w0 = load_w(c.sw0, g.kb0 & ~31);
            c.w0_next = load_w(c.sw0, (g.kb0 & ~31) + 32);
            c.w1 = GATED ? load_w(c.sw1, g.kb0 & ~31) : 0.0f;
            c.w1_next = GATED ? load_w(c.sw1, (g.kb0 & ~31) + 32) : 0.0f;
            return c;
        };
        Segment handed = {-1, 0, 0};   // the shared tile that the hand-over warp has
        bool more = walk.next(seg);
        Tile next_tile = {};
        Scales next_scales = {};
        if (more) {
            next_tile = tile_of(p, off, cum, seg.tile);
            next_scales = scales_of(seg, next_tile);
        }
        while (ok && more) {
            const Segment now = seg;
            const Tile T = next_tile;
            Scales c = next_scales;
            const int row = T.base + lane_row;
            const bool valid = row >= T.lo && row < T.hi;
            const bool warp_valid = T.base + quad * 32 < T.hi && T.base + quad * 32 + 32 > T.lo;
            float acc[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
            for (int kb = now.kb0; kb < now.kb1; ++kb, ++n) {
                const int buf = n % NB;
                const float x = (kb & 2) ? ((kb & 1) ? c.xa.w : c.xa.z) : ((kb & 1) ? c.xa.y : c.xa.x);
                const float f0 = x * __shfl_sync(0xffffffffu, c.w0, kb & 31), f1 = GATED ? x * __shfl_sync(0xffffffffu, c.w1, kb & 31) : f0;
                if ((kb & 3) == 3) {
                    c.xa = c.xa_next;
                    c.xa_next = load_a(c.sa, kb + 5);
                    if ((kb & 31) == 31) {
                        c.w0 = c.w0_next;
                        c.w0_next = load_w(c.sw0, kb + 33);
                        if (GATED) {
                            c.w1 = c.w1_next;
                            c.w1_next = load_w(c.sw1, kb + 33);
                        }
                    }
                }
                if (!__all_sync(0xffffffffu, mbar_wait(ring.done(s), ph, abort_flag, p.status, 54, wait_clocks(p)))) { ok = false; break; }
                tc_fence_after_sync();
                auto free = [&]() {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(ring.acc_empty(buf));
                };
                if (warp_valid) add_accumulator<NC, GATED>(tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * 128 * W), f0, f1, acc, column, free);
                else free();
                if (++s == p.stages) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            more = walk.next(seg);
            if (more) {
                next_tile = tile_of(p, off, cum, seg.tile);
                next_scales = scales_of(seg, next_tile);
            }
            if (now.kb1 - now.kb0 < p.Kb) {
                // ---- a shared tile ----
                const Sharing sh(walk, now);
                const int tile_floats = p.partial_rows * 128 * W, mine = lane_row * (128 * W);
                const bool last_segment = !more;
                bool all_here = false;
                if ((int)blockIdx.x == sh.c0 && last_segment) {
                    // The first of the sharers, which comes to this tile at the end of its range: the others mostly have been here long ago.
                    if (threadIdx.x == 0) ticket = read_tickets(p.tickets + sh.q);
                    if (!meet_all(p)) { ok = false; break; }
                    all_here = ticket == sh.c1 - sh.c0;
                    if (!meet_all(p)) { ok = false; break; }   // (`ticket` is written again)
                }
                if (all_here) {
                    if (threadIdx.x == 0) p.tickets[sh.q] = 0;
                    if (valid) {
#pragma unroll 1
                        for (int b = sh.c0 + 1; b <= sh.c1; ++b) {
                            const float *src = sh.part(p, b, tile_floats) + mine;
#pragma unroll
                            for (int j = 0; j < NC; j += 32) {
                                float v[4][8];
#pragma unroll
                                for (int i = 0; i < 4; ++i) load_partial8(src + column(j + 8 * i), v[i]);
#pragma unroll
                                for (int i = 0; i < 4; ++i)
#pragma unroll
                                    for (int e = 0; e < 8; ++e) acc[j + 8 * i + e] += v[i][e];
                            }
                        }
                    }
                } else {
                    if (valid) {
                        float *dst = sh.part(p, (int)blockIdx.x, tile_floats) + mine;
#pragma unroll
                        for (int j = 0; j < NC; j += 8) store_partial8(dst + column(j), acc + j);
                    }
                    if (!last_segment) {   // the hand-over warp sees to the rest while the next segment runs
                        __syncwarp();
                        if (lane == 0) mbar_arrive(handed_bar);
                        handed = now;
                        continue;
                    }
                    if (!meet_all(p)) { ok = false; break; }
                    if (threadIdx.x == 0) ticket = take_ticket(p.tickets + sh.q);
                    if (!meet_all(p)) { ok = false; break; }
                    if (ticket != sh.c1 - sh.c0) continue;
                    if (threadIdx.x == 0) p.tickets[sh.q] = 0;
                    // the last one adds them: row after row, each by a whole warp
                    auto part_of = [&](int block) { return sh.part(p, block, tile_floats); };
                    const int r_end = T.hi - T.base, r0 = T.lo - T.base + warp;
                    add_parts<ACT, W, GATED, 4, 2, kAddWarps>(p, part_of, sh.c0, sh.c1, r0, r_end, T.base, T.c, lane);
                    continue;
                }
            }
            if constexpr (GATED) {
                ok = finish_gated<ACT>(p, row, valid, T.c, part, lane_row, acc, red, meet);
            } else {
                if (valid) finish_row<ACT, NC>(p, row, (int64_t)T.c * 128 * W + part * NC, acc);
            }
        }
        if (ok && !more && handed.tile >= 0 && __all_sync(0xffffffffu, mbar_wait(told_bar, 0, abort_flag, p.status, 61, wait_clocks(p))) && pending >= 0) {
            const Sharing sh(walk, handed);
            const Tile T = tile_of(p, off, cum, handed.tile);
            if (threadIdx.x == 0) p.tickets[sh.q] = 0;
            auto part_of = [&](int block) { return sh.part(p, block, p.partial_rows * 128 * W); };
            add_parts<ACT, W, GATED, 4, 2, kAddWarps>(p, part_of, sh.c0, sh.c1, T.lo - T.base + warp, T.hi - T.base, T.base, T.c, lane);
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
    if (warp == kIssueWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
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

template <int ACT, int W, bool GATED>
int32_t launch(const Args &p, int grid, int smem, int dev, cudaStream_t stream) {
    static Once once[64];
    if (int32_t rc = once[dev].run([&]() -> int32_t {
            TTB_CUDA_TRY(cudaFuncSetAttribute(matmul_float8_kernel<ACT, W, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
            return TTB_OK;
        }))
        return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kManyThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, matmul_float8_kernel<ACT, W, GATED>, p));
    TTB_LAUNCH_CHECK("matmul_float8");
    return TTB_OK;
}

}  // namespace

static int partial_rows(int64_t rows) { return rows >= BM - 31 ? BM : (int)(f8_rows_padded(rows) + 31) / 32 * 32; }
int64_t f8_partial_bytes(int64_t rows) { return 2 * (int64_t)stream_blocks() * partial_rows(rows) * 128 * 2 * 4; }

// All rows, or what an expert has on average.
static int64_t mean_rows(int64_t rows, int64_t experts) {
    const int64_t hit = rows < experts ? rows : experts;
    return experts ? (rows + hit - 1) / hit : rows;
}
// Rows of a tile. The experts' MLP in a graph, us, tiles of 32 / 64 / 128 rows:
//  * 64 experts of 2048 x 1024, chosen evenly: 16 rows each 88 / 93 / 116, 24 rows 93 to 101 / 101 / 117, 32 rows 112 / 105 / 118, 56 rows 141 / 127 / 124, 64 rows 142 / 133 / 126;
//  * 8 experts of 4096 x 14336, chosen evenly: 24 rows 233 / 240 / 262, 32 rows 238 / 248 / 263, 48 rows 414 / 270 / 270, 56 rows 376 / 280 / 269, 64 rows 351 / 290 / 271.
// The mean says little where some experts are chosen far more often than others, and the larger tile is then the better one from smaller means on: 8 experts with 24 rows
// on average and 75 at most 247 / 240 / 208, 32 and 99: 350 / 310 / 268, 56 and 197: 456 / 363 / 256.
static int rows_per_tile(int64_t rows, int64_t experts) {
    const int64_t mean = mean_rows(rows, experts);
    return mean <= (experts ? 24 : 32) ? 32 : mean <= (experts ? 56 : 64) ? 64 : BM;
}
// Up to 8 rows a plain matmul is one launch, quantising its rows itself, and so is the gated one up to 4 rows an expert. That saves a launch where latency counts and costs
// time with several rows, which every block quantises again for each of its tiles (in a graph, us, itself / by the quantiser's kernel): 1 x 4096 x 1024 9.4 / 9.7, 8 x 4096 x
// 1024 10.2 / 9.9, 1 x 8192 x 8192 20.1 / 21.2, 8 x 8192 x 8192 22.3 / 21.8, 8 x 4544 x 4672 15.9 / 13.4, 16 x 8192 x 8192 28.6 / 21.5; the experts' MLP, 1 row on 8 of 64 experts of
// 2048 x 1024 30.0 / 28.4, 4 rows an expert 84.0 / 81.6 (chosen unevenly 62.9 / 54.1), of 8 of 4096 x 14336 218 / 222, 6 rows an expert 221 / 218.
bool f8_quantises_itself(int64_t rows, int64_t experts) { return mean_rows(rows, experts) <= (experts ? 4 : 8); }

// Weight blocks per tile of a plain matmul. Two make the longer unit of work; which is better goes by the whole rounds over the multiprocessors (us, one / two
// blocks a tile):
//  * many rows: a round of two-block tiles takes 1.47 times as long as one of one-block tiles. 512 x 8192 x 8192 60.0 / 49.1, 350 x 8192 x 8192 58.5 / 45.9, 2048 x
//    4096 x 4096 70.0 / 57.4, but 512 x 4096 x 4096 21.1 / 28.5, 1024 x 4544 x 4672 42.2 / 55.0, 2048 x 4544 x 4672 79.5 / 85.1;
//  * 9 to 64 rows: where one-block tiles are more than a round. 32 x 8192 x 28672 55.1 / 44.7, but 32 x 4544 x 18176 23.1 / 24.0, 32 x 28672 x 8192 49.7 / 51.0;
//  * up to 8 rows (quantised by the kernel itself, whose warps do that once a tile): from 1000 one-block units on. 1 x 8192 x 28672 46.9 / 40.8, 1 x 4096 x 4096
//    11.3 / 10.0, but 1 x 8192 x 1024 9.3 / 10.2, 1 x 4096 x 1024 8.4 / 9.0.
static int weight_blocks(const F8Matmul &m, int R, int64_t sms) {
    const int64_t hit = m.experts ? (m.rows < m.experts ? m.rows : m.experts) : 1, row_tiles = hit * ((m.rows / hit + R - 1) / R), nb = f8_blocks(m.N);
    const int64_t one = row_tiles * nb, two = row_tiles * ((nb + 1) / 2);
    if (m.x.ptr) return one * f8_blocks(m.K) >= 1000 ? 2 : 1;
    if (R < BM) return one > sms ? 2 : 1;
    return (two + sms - 1) / sms * 147 < (one + sms - 1) / sms * 100 ? 2 : 1;
}

int32_t launch_matmul_float8(const F8Matmul &m, cudaStream_t stream) {
    Args p;
    const int64_t experts = m.experts ? m.experts : 1;
    if (m.experts > kF8MaxExperts) return fail(TTB_E_UNSUPPORTED, "ttb_experts_mlp_float8: at most %d experts", kF8MaxExperts);
    if (int32_t rc = make_map(m.w[0].codes, experts, m.N, m.K, p.wmap[0])) return rc;
    p.wmap[1] = p.wmap[0];
    if (m.gated)
        if (int32_t rc = make_map(m.w[1].codes, experts, m.N, m.K, p.wmap[1])) return rc;
    p.sw[0] = m.w[0].scales;
    p.sw[1] = m.w[1].scales;
    p.a = m.a; p.h = m.h;
    p.x = m.x; p.K = m.K;
    p.early = m.early;
    p.row_mask = m.x.ptr ? 0 : 7;
    p.offsets = m.offsets; p.bias = m.bias; p.out = m.out; p.N = m.N;
    p.rows = (int)m.rows; p.experts = m.experts;
    p.Kb = (int)f8_blocks(m.K); p.Nb = (int)f8_blocks(m.N);
    const int sms = stream_blocks();
    const int R = rows_per_tile(m.rows, m.experts), W = m.gated ? 2 : weight_blocks(m, R, sms);
    // Where tiles are shared (units a block takes at least; units that sharing has to save): the hand-over costs what a few units of few rows take, and some 40
    // of many rows, whose parts are larger (us, shared / whole: 32 x 8192 x 8192 21.8 / 27.1, 32 x 8192 x 28672 49.4 / 44.4 with 15 of 64 units to save, 96 x 18176 x
    // 4544 35.6 / 53.5, 128 x 28672 x 8192 65.7 / 83.7, 128 x 8192 x 20000 58.6 / 43.7 with 30 of 64, 256 x 28672 x 8192 101 / 93 with 30 of 224).
    p.stream_min = R < BM ? 4 : 16;
    p.stream_gain = m.x.ptr ? 8 : p.Kb / 3 > (R < BM ? 8 : 40) ? p.Kb / 3 : R < BM ? 8 : 40;
    p.tickets = m.tickets;
    p.partials = m.partials;
    p.partial_rows = partial_rows(m.rows);
    p.ct = m.gated ? p.Nb : (p.Nb + W - 1) / W;
    p.tile_rows = m.x.ptr ? kQuantRows : R;
    p.a_rows = (int)(f8_rows_padded(m.rows) < p.tile_rows ? f8_rows_padded(m.rows) : p.tile_rows);
    p.stage_bytes = p.a_rows * kF8Block + W * kF8BlockBytes;
    const int extra = (R < BM ? p.tile_rows * 128 * W * 4 : m.gated ? 2 * BM * 4 : 0) + (m.experts ? 4 * (2 * m.experts + 1) : 0) + 1024;
    p.stages = (kSmemLimit - extra) / p.stage_bytes;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    if (R >= BM) p.stages &= ~1;   // (matmul_float8.cu: FULL_FIRST)
    if (p.stages < (R < BM ? (W * R > 64 ? 2 : 4) : 4 / W)) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: no room for the ring");
    p.out_dtype = m.out_dtype; p.out_row_major = m.out_row_major; p.bias_row_major = m.bias_row_major;
    // 16 neighbouring columns of a row start at a multiple of this many bytes (0: stores by element)
    p.out_aligned = 0;
    for (int bytes = 16; bytes <= 32 && !m.gated; bytes *= 2)
        if (reinterpret_cast<uintptr_t>(m.out) % bytes == 0 && (!m.out_row_major || m.N * (m.out_dtype == TTB_FLOAT32 ? 4 : 2) % bytes == 0)) p.out_aligned = bytes;
    p.wait_limit = barrier_limit_kcycles();
    if (int32_t rc = status_word_address(&p.status)) return rc;
    int dev = 0;
    TTB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: device index %d is out of range", dev);
    if (sms * 16 > kF8TicketBytes) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: too many multiprocessors");
    const int64_t most = (f8_rows_padded(m.rows) / p.tile_rows + 1 + m.experts) * (int64_t)p.ct;   // an upper bound for a grouped matmul
    if (most > INT32_MAX / 2 || (uint64_t)sms * sms * p.Kb > 0xffffffffu) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: too many output tiles");
    const int grid = most * p.Kb / p.stream_min < sms ? (int)(most * p.Kb / p.stream_min > most ? most * p.Kb / p.stream_min : most) : sms, smem = p.stages * p.stage_bytes + extra;
    if (R < BM) return launch_matmul_float8_few(p, m.act, W, R, m.gated, grid, smem, dev, stream);
    TTB_DISPATCH_ACT(m.act, return m.gated ? (launch<ACT, 2, true>(p, grid, smem, dev, stream)) : W == 2 ? (launch<ACT, 2, false>(p, grid, smem, dev, stream)) : (launch<ACT, 1, false>(p, grid, smem, dev, stream)));
    return TTB_OK;
}

}  // namespace ttb

using ttb::fail;

namespace {
// The head of the workspace is that of ttb_matmul: arrival counters, of which the float8 kernels use the first kF8TicketBytes, and its accumulation tiles, which
// they leave alone.
constexpr int64_t kWorkspaceHead = 65536 + (int64_t(16) << 20);
constexpr int64_t kMaxExtent = int64_t(1) << 24;   // rows, K and N: tile coordinates and row indexes stay far inside 32 bits
}  // namespace

extern "C" {

int64_t ttb_linear_float8_workspace_bytes(int64_t rows, int64_t K, int64_t N) {
    if (rows <= 0 || K <= 0 || N <= 0 || rows > kMaxExtent || K > kMaxExtent || N > kMaxExtent) return -1;
    int64_t at = kWorkspaceHead + ttb::f8_partial_bytes(rows);
    if (!ttb::f8_quantises_itself(rows, 0)) ttb::f8_place(nullptr, at, rows, K);
    return at;
}

int32_t ttb_linear_float8(const void *a, const void *w_codes, const void *w_scales, const void *bias, void *out, int32_t out_dtype, int64_t rows, int64_t K,
                          int64_t N, int32_t activation, int32_t flags, void *workspace, int64_t workspace_bytes, void *stream) {
    if (!a || !w_codes || !w_scales || !out) return fail(TTB_E_INVALID, "ttb_linear_float8: null tensor pointer");
    if (out_dtype != TTB_BFLOAT16 && out_dtype != TTB_FLOAT32) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: output must be bfloat16 or float32");
    if (flags & ~(TTB_MM_A_ROW_MAJOR | TTB_MM_OUT_ROW_MAJOR | TTB_MM_BIAS_ROW_MAJOR | TTB_MM_WORKSPACE_ZEROED | TTB_MM_WEIGHTS_RESIDENT)) return fail(TTB_E_INVALID, "ttb_linear_float8: unknown flags %d", flags);
    if (activation < TTB_ACT_NONE || activation > TTB_ACT_SILU) return fail(TTB_E_INVALID, "ttb_linear_float8: unknown activation %d", activation);
    const int64_t need = ttb_linear_float8_workspace_bytes(rows, K, N);
    if (need < 0) return fail(TTB_E_INVALID, "ttb_linear_float8: rows, K and N must be between 1 and 2^24");
    if (K % 16) return fail(TTB_E_INVALID, "ttb_linear_float8: K must be a multiple of 16 (got %lld)", (long long)K);
    if (!ttb::f8_blocks_count(rows, K)) return fail(TTB_E_UNSUPPORTED, "ttb_linear_float8: too many blocks of 128 activations");
    const bool a_rm = flags & TTB_MM_A_ROW_MAJOR, out_rm = flags & TTB_MM_OUT_ROW_MAJOR;
    if ((!a_rm || !out_rm) && rows % 32) return fail(TTB_E_INVALID, "ttb_linear_float8: tiled tensors have a multiple of 32 rows (got %lld)", (long long)rows);
    if (ttb::f8_misaligned(a, 16) || ttb::f8_misaligned(w_codes, 16) || ttb::f8_misaligned(w_scales, 4) || ttb::f8_misaligned(out, out_dtype == TTB_FLOAT32 ? 4 : 2) ||
        (bias && ttb::f8_misaligned(bias, 2)))
        return fail(TTB_E_INVALID, "ttb_linear_float8: activations and codes must be 16-byte aligned, the other tensors as their elements");
    if (!ttb::workspace_serves(workspace, workspace_bytes, need)) return fail(TTB_E_WORKSPACE, "ttb_linear_float8: needs %lld bytes of 256-byte aligned workspace", (long long)need);
    ttb::F8Matmul m = {};
    m.tickets = static_cast<int32_t *>(workspace);
    m.partials = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kWorkspaceHead);
    int64_t at = kWorkspaceHead + ttb::f8_partial_bytes(rows);
    m.a = ttb::f8_place(static_cast<uint8_t *>(workspace), at, rows, K);
    m.w[0] = {w_codes, static_cast<const float *>(w_scales)};
    m.rows = rows; m.K = K; m.N = N;
    m.act = activation;
    m.out = out; m.out_dtype = out_dtype; m.out_row_major = out_rm;
    m.bias = static_cast<const uint16_t *>(bias);
    m.bias_row_major = flags & TTB_MM_BIAS_ROW_MAJOR;
    if (!(flags & TTB_MM_WORKSPACE_ZEROED)) TTB_CUDA_TRY(cudaMemsetAsync(workspace, 0, ttb::kF8TicketBytes, (cudaStream_t)stream));
    const bool early = flags & TTB_MM_WEIGHTS_RESIDENT;
    if (ttb::f8_quantises_itself(rows, 0)) {
        m.a = {};
        m.x = {static_cast<const uint16_t *>(a), nullptr, a_rm ? K : (K + 31) / 32 * 1024, !a_rm};
        m.early = early;
    } else {
        // (a quantiser that does not let the matmul start at once lets it when all that came before has ended)
        if (int32_t rc = ttb::launch_quantize_operand(a, a_rm, 1, rows, K, m.a, nullptr, 1, early, (cudaStream_t)stream)) return rc;
        m.early = true;
    }
    return ttb::launch_matmul_float8(m, (cudaStream_t)stream);
}

}  // extern "C"
