// The float8 matmul for tiles of at most 32 or 64 rows (decode batches, experts with few tokens); matmul_float8.cu has the formulas and the rule.
//
// "Swap-AB": the MMA's M dimension (128 TMEM lanes) runs over weight rows (output columns), its N dimension over the tile's rows, so that neither the MMAs
// nor the eight warps that keep the sums spend time on rows that are not there. A thread has one output column and up to 64 rows; the rows' scales sit in the
// warp's lanes and go round by shuffles. Finished sums pass through shared memory, from which whole warps finish row after row: whole lines to memory, and
// little code, which runs cold once or twice a launch (a thread per row, as the other kernel has it, took 3 to 5 us to store 32 rows of 256 columns).
// Tiles are shared between blocks as float8_tiles.cuh has it. Bound by the weight's bytes: 1 x 8192 x 28672 40.8 us, 5.8 TB/s; 32 x 8192 x 28672 44.4 us; 32 rows on
// eight experts of 4096 x 14336 218 to 231 us, 6.1 to 6.5 TB/s; small ones by the launch and a hand-over of 2 to 4 us (1 x 4096 x 1024 8.4 us).
//
// Tiles of 8 rows: four more warps quantise the block's rows straight into the operand (QUANT), so that a call is one launch. (For 32 rows the quantising took
// four times as long as the weights, and a kernel of its own, which this one overlaps, is the better way.)
#include "float8_tiles.cuh"

namespace ttb {
namespace {

using namespace f8;
using namespace ptx;

__host__ __device__ constexpr int few_accumulators(int W, int R) { return W * R > 64 ? 2 : 4; }   // (at most as many as the ring has stages: issue_mmas)
constexpr int kQuantWarp0 = 12, kQuantWarps = 4;
constexpr int kScaleSlots = kMaxStages + 4;   // a row scale is read until the sums have it: at most 4 units behind the MMAs, which are at most the ring behind
constexpr int few_threads(bool quant) { return 32 * (quant ? kQuantWarp0 + kQuantWarps : 12); }

// A quantising warp takes the units of every fourth stage, of at most kQuantRows rows: 16 lanes have 128 values of a row, the loads run one unit of the warp's
// ahead. (Stages, not units, are dealt out: a wait for a phase's parity means something only to a warp that has waited for the stage's phase before it. Dealt by
// units, with five stages, a warp could overtake another's MMAs by a whole round of the ring, and did: the block left with copies under way.)
__device__ __forceinline__ void quantise(const Args &p, const Ring &ring, uint8_t *smem, uint32_t ready0, float *scales, Walk walk, const int *off, const int *cum, int which) {
    grid_dep_wait();
    const int lane = threadIdx.x & 31, sub = lane & 15, r0 = lane >> 4;
    const int64_t step = p.x.tiled ? 4096 : kF8Block;   // elements between blocks of 128 columns
    const int col = p.x.tiled ? (sub >> 2) * 1024 + ((sub >> 1) & 1) * 256 + (sub & 1) * 8 : sub * 8;
    Segment seg;
    int n = 0;   // unit at the segment's beginning
    while (walk.next(seg)) {
        const Tile T = tile_of(p, off, cum, seg.tile);
        const int rows = T.hi - T.base, end = n + seg.kb1 - seg.kb0;
        const uint16_t *src[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int row = min(T.base + r0 + 2 * i, T.hi - 1);
            if (p.x.row_of) row = __ldcg(p.x.row_of + row);
            src[i] = p.x.ptr + col + (p.x.tiled ? (int64_t)(row >> 5) * p.x.row_pitch + ((row >> 4) & 1) * 512 + (row & 15) * 16 : (int64_t)row * p.x.row_pitch);
        }
        auto load = [&](int i, int unit) {   // (K is a multiple of 16: eight values are all there or none)
            const int kb = seg.kb0 + unit - n;
            return r0 + 2 * i < rows && unit < end && (int64_t)kb * kF8Block + sub * 8 < p.K ? __ldcg(reinterpret_cast<const uint4 *>(src[i] + kb * step)) : make_uint4(0, 0, 0, 0);
        };
        auto mine = [&](int unit) {   // the warp's first unit from this one on
            while (unit % p.stages % kQuantWarps != which) ++unit;
            return unit;
        };
        int unit = mine(n);
        uint4 next[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) next[i] = load(i, unit);
        while (unit < end) {
            const int s = unit % p.stages, slot = unit % kScaleSlots;
            const uint32_t parity = (uint32_t)((unit / p.stages) & 1) ^ 1;
            unit = mine(unit + 1);
            uint4 now[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                now[i] = next[i];
                next[i] = load(i, unit);
            }
            if (!__all_sync(0xffffffffu, mbar_wait(ring.done(s), parity, ring.abort_flag, p.status, 57, wait_clocks(p)))) return;
            uint8_t *const stage = smem + s * p.stage_bytes;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (2 * i >= rows) break;   // (the same for all lanes)
                const uint32_t h[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
                float v[8], m = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[2 * j] = __uint_as_float(h[j] << 16);
                    v[2 * j + 1] = __uint_as_float(h[j] & 0xffff0000u);
                    m = fmaxf(m, fmaxf(fabsf(v[2 * j]), fabsf(v[2 * j + 1])));
                }
#pragma unroll
                for (int d = 8; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
                const float scale = f8_scale(m);
                const int r = r0 + 2 * i;
                if (r < rows) {
                    *reinterpret_cast<uint2 *>(stage + r * kF8Block + (((sub >> 1) ^ (r & 7)) << 4) + (sub & 1) * 8) = f8_pack8(v, scale);
                    if (sub == 0) scales[slot * 32 + r] = scale;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(ring.full(s));
                mbar_arrive(ready0 + 8u * slot);
            }
        }
        n = end;
    }
}

// W: weight blocks per tile (GATED: the same block of either weight). R: rows per tile at most. (At R = 32 128 registers a thread in any case: blocks of the
// quantiser in front of the next launch then fit beside this one's and are there when it ends.)
template <int ACT, int W, int R, bool GATED, bool QUANT>
__global__ void __launch_bounds__(R == 32 ? 512 : 384, 1) matmul_float8_few_kernel(const __grid_constant__ Args p) {
    static_assert(!GATED || W == 2, "a gated tile takes a block of either weight");
    static_assert(!QUANT || (R == 32 && kQuantRows == 8), "half a warp has every other row of a tile, four at most");
    constexpr int NR = R * W / 2;             // rows of an epilogue thread: all of them of weight block `half`, or half of the rows of the one block
    constexpr int NX = NR > 32 ? 2 : 1;       // registers that hold a scale of each
    constexpr bool ADD = R <= 32;
    constexpr int RU = QUANT ? 1 : R == 32 ? 2 : 4 / W, BU = QUANT ? 8 / W : R == 32 ? 4 / W : 4;   // rows and blocks whose parts a warp adds at a time
    constexpr int NB = few_accumulators(W, R), kTmemCols = NB * W * R;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + NB + 3 + kScaleSlots];
    __shared__ float scales[QUANT ? kScaleSlots * 32 : 1];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_word;
    __shared__ int tiles_word;
    __shared__ volatile int ticket, pending, progress;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *sums = reinterpret_cast<float *>(smem + p.stages * p.stage_bytes);   // [tile_rows][128 W]
    int *off = reinterpret_cast<int *>(sums + p.tile_rows * 128 * W);
    int *cum = off + p.experts + 1;
    const uint32_t bar0 = smem_u32(bars);
    volatile int *abort_flag = &abort_word;
    const Ring ring = {smem_u32(smem), bar0, bar0 + 8u * kMaxStages, bar0 + 8u * (2 * kMaxStages), abort_flag, &progress};
    const uint32_t all_bar = bar0 + 8u * (2 * kMaxStages + NB), handed_bar = all_bar + 8, told_bar = handed_bar + 8, ready0 = told_bar + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(ring.full(s), QUANT ? 2 : 1);
            mbar_init(ring.done(s), 1);
        }
        for (int b = 0; b < NB; ++b) mbar_init(ring.acc_empty(b), kEpiWarps);
        mbar_init(all_bar, kEpiWarps);
        mbar_init(handed_bar, kEpiWarps);
        mbar_init(told_bar, 1);
        for (int i = 0; i < kScaleSlots; ++i) mbar_init(ready0 + 8u * i, 1);
        abort_word = progress = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    if (!p.early) grid_dep_wait();
    // (what is read before grid_dep_wait: see matmul_float8.cu)
    count_tiles(p, off, cum, &tiles_word);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    Walk walk(p, tiles_word);

    if (warp == kProducerWarp) {
        fetch<W, GATED, true, QUANT>(p, ring, walk, off, cum);
    } else if (warp >= kMmaWarp && warp < kMmaWarp + kIssuers) {
        issue_mmas<NB, false>(p, ring, walk, off, cum, warp - kMmaWarp, [&](uint32_t src, int buf, const Tile &T) {
            const uint64_t x = smem_desc_sw128(src), w = smem_desc_sw128(src + (uint32_t)(p.a_rows * kF8Block));
            const uint32_t idesc = instr_desc_e4m3(128, (T.hi - T.base + 15) & ~15);
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k)   // 32 bytes of K further: two 16-byte units in the descriptor's address
                    mma_e4m3_ss(tmem_base + (uint32_t)((buf * W + j) * R), w + j * (kF8BlockBytes >> 4) + 2 * k, x + 2 * k, idesc, k > 0);
        });
    } else if (QUANT && warp >= kQuantWarp0) {
        quantise(p, ring, smem, ready0, scales, walk, off, cum, warp - kQuantWarp0);
    } else if (warp >= kMmaWarp + kIssuers) {
        hand_over<ACT, W, GATED, ADD>(p, handed_bar, told_bar, &pending, ring, walk, off, cum);
    } else {
        grid_dep_wait();
        const int quad = warp & 3, half = warp >> 2;
        const int first_row = W == 1 ? half * NR : 0, block = W == 1 ? 0 : half;   // of this thread's sums
        Meeting meet = {all_bar, 0, abort_flag};
        Segment seg, handed = {-1, 0, 0};   // the shared tile that the hand-over warp has
        int s = 0, n = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok && walk.next(seg)) {
            const Tile T = tile_of(p, off, cum, seg.tile);
            const int rows = T.hi - T.base;
            // scales: lane l has those of row first_row + l (and + 32), for four blocks where they lie in scratch; and the weight block's for K block 32 i + l,
            // one step ahead
            const float *sa[NX];
#pragma unroll
            for (int i = 0; i < NX; ++i) sa[i] = QUANT ? nullptr : p.a.scales + (int64_t)max(min(T.base + first_row + i * 32 + (lane & (NR - 1)), T.hi - 1), T.lo) * p.a.scale_pitch;
            const float *const sw = p.sw[GATED ? half : 0] + ((int64_t)T.e * p.Nb + (GATED ? T.c : min(T.c * W + block, p.Nb - 1))) * p.Kb;
            auto load_a = [&](int i, int kb) { return !QUANT && kb < p.a.scale_pitch ? __ldcg(reinterpret_cast<const float4 *>(sa[i] + kb)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f); };
            auto load_w = [&](int kb) { return kb + lane < p.Kb ? __ldg(sw + kb + lane) : 0.0f; };
            float4 xa[NX], xa_next[NX];
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                xa[i] = load_a(i, seg.kb0 & ~3);
                xa_next[i] = load_a(i, (seg.kb0 & ~3) + 4);
            }
            float w0 = load_w(seg.kb0 & ~31), w0_next = load_w((seg.kb0 & ~31) + 32);
            float acc[NR];
#pragma unroll
            for (int j = 0; j < NR; ++j) acc[j] = 0.0f;
            for (int kb = seg.kb0; kb < seg.kb1; ++kb, ++n) {
                const int buf = n % NB;
                const float w = __shfl_sync(0xffffffffu, w0, kb & 31);
                float f[NX];
                if (QUANT) {
                    if (!__all_sync(0xffffffffu, mbar_wait(ready0 + 8u * (n % kScaleSlots), (uint32_t)((n / kScaleSlots) & 1), abort_flag, p.status, 58, wait_clocks(p)))) { ok = false; break; }
                    f[0] = w * scales[(n % kScaleSlots) * 32 + first_row + (lane & (NR - 1))];
                }
#pragma unroll
                for (int i = 0; i < NX && !QUANT; ++i) f[i] = w * ((kb & 2) ? ((kb & 1) ? xa[i].w : xa[i].z) : ((kb & 1) ? xa[i].y : xa[i].x));
                if ((kb & 3) == 3) {
#pragma unroll
                    for (int i = 0; i < NX; ++i) {
                        xa[i] = xa_next[i];
                        xa_next[i] = load_a(i, kb + 5);
                    }
                    if ((kb & 31) == 31) {
                        w0 = w0_next;
                        w0_next = load_w(kb + 33);
                    }
                }
                if (!__all_sync(0xffffffffu, mbar_wait(ring.done(s), ph, abort_flag, p.status, 54, wait_clocks(p)))) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t t0 = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)((buf * W + block) * R + first_row);
#pragma unroll
                for (int q = 0; q < NR; q += 32) {
                    uint32_t r[2][16];
                    if (first_row + q < rows) {
                        tmem_ld16(t0 + q, r[0]);
                        if (NR > 16 && first_row + q + 16 < rows) tmem_ld16(t0 + q + 16, r[1]);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[q + j] = fmaf(__uint_as_float(r[0][j]), __shfl_sync(0xffffffffu, f[q / 32], j), acc[q + j]);
                        if (NR > 16 && first_row + q + 16 < rows)
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                acc[(q + 16 + j) & (NR - 1)] = fmaf(__uint_as_float(r[1][j]), __shfl_sync(0xffffffffu, f[q / 32], 16 + j), acc[(q + 16 + j) & (NR - 1)]);
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(ring.acc_empty(buf));
                if (++s == p.stages) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            // the tile's sums, [row][128 W]
#pragma unroll
            for (int j = 0; j < NR; ++j)
                if (first_row + j < rows) sums[(first_row + j) * (128 * W) + block * 128 + quad * 32 + lane] = acc[j];
            const bool shared_tile = seg.kb1 - seg.kb0 < p.Kb, last_segment = walk.u >= walk.u_end;
            const int r0 = T.lo - T.base + warp;
            if (!shared_tile) {
                if (!meet(p)) { ok = false; break; }
#pragma unroll 1
                for (int r = r0; r < rows; r += kEpiWarps) {
                    float4 v[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) v[j] = *reinterpret_cast<const float4 *>(sums + r * (128 * W) + j * 128 + lane * 4);
                    finish_row_warp<ACT, W, GATED>(p, T.base + r, T.c, lane, v);
                }
            } else {
                const Sharing sh(walk, seg);
                const int tile_floats = p.partial_rows * 128 * W;
                auto part_of = [&](int b) { return sh.part(p, b, tile_floats); };
                // The first of the sharers comes to this tile at the end of its range: the others mostly have been here long ago.
                const bool first = (int)blockIdx.x == sh.c0 && last_segment;
                if (first && threadIdx.x == 0) ticket = read_tickets(p.tickets + sh.q);
                if (!meet(p)) { ok = false; break; }
                if (first && ticket == sh.c1 - sh.c0) {
                    if (threadIdx.x == 0) p.tickets[sh.q] = 0;
                    add_parts<ACT, W, GATED, RU, BU, kEpiWarps>(p, part_of, sh.c0, sh.c1, r0, rows, T.base, T.c, lane, sums);
                } else {
                    float *const part = part_of((int)blockIdx.x) + lane * 4;
#pragma unroll 4
                    for (int r = r0; r < rows; r += kEpiWarps)
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            *reinterpret_cast<float4 *>(part + r * (128 * W) + j * 128) = *reinterpret_cast<const float4 *>(sums + r * (128 * W) + j * 128 + lane * 4);
                    if (!last_segment) {   // the hand-over warp sees to the rest while the next segment runs
                        __syncwarp();
                        if (lane == 0) mbar_arrive(handed_bar);
                        handed = seg;
                    } else {
                        if (!meet(p)) { ok = false; break; }
                        if (threadIdx.x == 0) ticket = take_ticket(p.tickets + sh.q);
                        if (!meet(p)) { ok = false; break; }
                        if (ticket == sh.c1 - sh.c0) {   // the last one adds them
                            if (threadIdx.x == 0) p.tickets[sh.q] = 0;
                            add_parts<ACT, W, GATED, RU, BU, kEpiWarps>(p, part_of, sh.c0, sh.c1, r0, rows, T.base, T.c, lane);
                        }
                    }
                }
            }
            if (!meet(p)) { ok = false; break; }   // (the next tile's sums take the place of these)
        }
        if (!ADD && ok && handed.tile >= 0 && __all_sync(0xffffffffu, mbar_wait(told_bar, 0, abort_flag, p.status, 61, wait_clocks(p))) && pending >= 0) {
            const Sharing sh(walk, handed);
            const Tile T = tile_of(p, off, cum, handed.tile);
            if (threadIdx.x == 0) p.tickets[sh.q] = 0;
            auto part_of = [&](int b) { return sh.part(p, b, p.partial_rows * 128 * W); };
            add_parts<ACT, W, GATED, RU, BU, kEpiWarps>(p, part_of, sh.c0, sh.c1, T.lo - T.base + warp, T.hi - T.base, T.base, T.c, lane);
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
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <int ACT, int W, int R, bool GATED, bool QUANT>
int32_t launch(const Args &p, int grid, int smem, int dev, cudaStream_t stream) {
    static Once once[64];
    if (int32_t rc = once[dev].run([&]() -> int32_t {
            TTB_CUDA_TRY(cudaFuncSetAttribute(matmul_float8_few_kernel<ACT, W, R, GATED, QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
            return TTB_OK;
        }))
        return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(few_threads(QUANT));
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, matmul_float8_few_kernel<ACT, W, R, GATED, QUANT>, p));
    TTB_LAUNCH_CHECK("matmul_float8_few");
    return TTB_OK;
}

template <int ACT, bool QUANT>
int32_t launch_act(const Args &p, int W, int R, bool gated, int grid, int smem, int dev, cudaStream_t stream) {
    if (R == 32) {
        if (gated) return launch<ACT, 2, 32, true, QUANT>(p, grid, smem, dev, stream);
        return W == 2 ? launch<ACT, 2, 32, false, QUANT>(p, grid, smem, dev, stream) : launch<ACT, 1, 32, false, QUANT>(p, grid, smem, dev, stream);
    }
    if constexpr (!QUANT) {
        if (gated) return launch<ACT, 2, 64, true, false>(p, grid, smem, dev, stream);
        return W == 2 ? launch<ACT, 2, 64, false, false>(p, grid, smem, dev, stream) : launch<ACT, 1, 64, false, false>(p, grid, smem, dev, stream);
    }
    return fail(TTB_E_UNSUPPORTED, "matmul_float8_few: no kernel quantises tiles of %d rows itself", R);
}

}  // namespace

// `extra` bytes of shared memory behind the ring, `p.stages` of which the caller has fitted into kSmemLimit.
int32_t launch_matmul_float8_few(const Args &p, int act, int W, int R, bool gated, int grid, int smem, int dev, cudaStream_t stream) {
    TTB_DISPATCH_ACT(act, return p.x.ptr ? (launch_act<ACT, true>(p, W, R, gated, grid, smem, dev, stream)) : (launch_act<ACT, false>(p, W, R, gated, grid, smem, dev, stream)));
    return TTB_OK;
}

}  // namespace ttb
