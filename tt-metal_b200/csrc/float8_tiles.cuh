// What the float8 matmul kernels (matmul_float8.cu, matmul_float8_few.cu) share: the list of tiles and how blocks share it, the fetching and issuing warps,
// the hand-over of shared tiles, and the finishing of rows.
#pragma once
#include <cuda.h>

#include "epilogue.cuh"
#include "matmul_float8.cuh"
#include "sm100_ptx.cuh"

namespace ttb {
namespace f8 {


using namespace ptx;

constexpr int kMaxStages = 12;
constexpr int kEpiWarps = 8, kProducerWarp = 8, kMmaWarp = 9, kIssuers = 2;
constexpr int kQuantRows = 8;               // rows of a tile whose kernel quantises them itself
constexpr int kSmemLimit = 232448 - 3072;   // the rest: static shared memory

struct alignas(64) Args {
    CUtensorMap wmap[2];
    const float *sw[2];
    F8Activation a, h;
    F8Rows x;                        // where the kernel quantises the activations itself
    bool early;                      // the weights and the experts' row ranges may be read before the kernel before has ended
    const int32_t *offsets;
    const uint16_t *bias;
    void *out;
    int64_t N, K;
    int rows, experts, Kb, Nb, ct;   // ct: column tiles
    int tile_rows, row_mask;         // rows of a tile; tiles start at a row that has none of these bits (7 where the activations lie in scratch in whole atoms)
    int a_rows, stages, stage_bytes; // rows of a stage's activations (a multiple of 8); the ring
    int stream_min, stream_gain;     // units a block takes at least of the shared tiles; rounds' units that sharing has to save
    int *tickets;
    float *partials;
    int partial_rows;                // of a tile (a multiple of 32)
    int out_dtype, out_row_major, bias_row_major, out_aligned;   // out_aligned: bytes that a store may have
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

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { return (uint32_t)f32_to_bf16_bits(lo) | ((uint32_t)f32_to_bf16_bits(hi) << 16); }

// a += r * f of two neighbours in one instruction (f holds the factor twice).
__device__ __forceinline__ void fma_pair(float &a0, float &a1, uint32_t r0, uint32_t r1, uint64_t f) {
    asm("{\n\t"
        ".reg .b64 a, r;\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "mov.b64 r, {%2, %3};\n\t"
        "fma.rn.f32x2 a, r, %4, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t"
        "}"
        : "+f"(a0), "+f"(a1)
        : "r"(r0), "r"(r1), "l"(f));
}

// Adds an accumulator's NC columns, times f0 (gated: the second half times f1), to the sums, 32 at a time, the next 32 on their way meanwhile. column(j): that of
// sum j; free() is called as soon as the accumulator may be written again.
template <int NC, bool GATED, typename C, typename F>
__device__ __forceinline__ void add_accumulator(uint32_t t0, float f0, float f1, float (&acc)[NC], C column, F free) {
    uint32_t r[2][32];
    auto load = [&](int q, uint32_t (&v)[32]) {
        uint32_t lo[16], hi[16];
        tmem_ld16(t0 + column(q), lo);
        tmem_ld16(t0 + column(q + 16), hi);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            v[j] = lo[j];
            v[16 + j] = hi[j];
        }
    };
    load(0, r[0]);
    tmem_ld_wait();
#pragma unroll
    for (int q = 0; q < NC; q += 32) {
        if (q + 32 < NC) load(q + 32, r[(q / 32 + 1) & 1]);
        else free();
        const float factor = GATED && q >= NC / 2 ? f1 : f0;
        const uint64_t f = f8_two(factor, factor);
#pragma unroll
        for (int j = 0; j < 32; j += 2) fma_pair(acc[q + j], acc[q + j + 1], r[(q / 32) & 1][j], r[(q / 32) & 1][j + 1], f);
        if (q + 32 < NC) tmem_ld_wait();
    }
}

// A tile of the launch: rows [lo, hi) of expert e, kept as rows base .. base + tile_rows - 1 (base: at most lo), column tile c.
struct Tile {
    int e, lo, hi, base, c;
};

__device__ __forceinline__ int row_tiles(const Args &p, int lo, int hi) { return hi > lo ? (hi - (lo & ~p.row_mask) + p.tile_rows - 1) / p.tile_rows : 0; }

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
    const int rt = row_tiles(p, lo, hi), per = 16 * p.ct;
    const int group = t / per, in = t - group * per, height = min(16, rt - group * 16);
    const int r = group * 16 + in % height;
    s.c = in / height;
    s.base = (lo & ~p.row_mask) + r * p.tile_rows;
    s.lo = max(lo, s.base);
    s.hi = min(hi, s.base + p.tile_rows);
    return s;
}

// How many tiles the launch has; fills off[experts + 1] (first row of each expert) and cum[experts] (first tile). Called by all threads; `word` is written by
// one of them and read after the next barrier.
__device__ __forceinline__ void count_tiles(const Args &p, int *off, int *cum, int *word) {
    const int lane = threadIdx.x & 31;
    if (p.experts) {
        for (int i = threadIdx.x; i <= p.experts; i += blockDim.x) off[i] = __ldcg(p.offsets + i);
        __syncthreads();
        if (threadIdx.x < 32) {
            int run = 0;
            for (int i = 0; i < p.experts; i += 32) {
                int x = i + lane < p.experts ? row_tiles(p, off[i + lane], off[i + lane + 1]) * p.ct : 0, sum = x;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += y;
                }
                if (i + lane < p.experts) cum[i + lane] = run + sum - x;
                run += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (lane == 0) *word = run;
        }
    } else if (threadIdx.x == 0) {
        *word = row_tiles(p, 0, p.rows) * p.ct;
    }
}

// A block's work: whole tiles first, first + grid, ..; then the units [u, u_end) of the shared tiles.
struct Segment {
    int tile, kb0, kb1;
};
struct Walk {
    int tile, whole, grid, u, u_end, Kb;
    int sharers, units;   // blocks that the shared tiles are dealt out to, their units

    __device__ Walk(const Args &p, int tiles) : Walk(p, tiles, (int)gridDim.x, (int)blockIdx.x) {}
    __device__ Walk(const Args &p, int tiles, int blocks, int block) {
        Kb = p.Kb;
        grid = blocks;
        const int left = tiles % grid;
        whole = tiles - left;
        units = left * Kb;
        sharers = min(grid, max(left, units / p.stream_min));
        // not where a round of whole tiles is about as long
        if (left == 0 || Kb - (units + sharers - 1) / max(sharers, 1) < p.stream_gain) {
            whole = tiles;
            units = sharers = 0;
        }
        tile = block;
        u = block < sharers ? first_unit(block) : 0;
        u_end = block < sharers ? first_unit(block + 1) : 0;
    }
    // (the launcher keeps the products below 2^32; 64-bit divisions took a microsecond a piece where a hand-over waits for them)
    __device__ int first_unit(int block) const { return (int)((uint32_t)block * (uint32_t)units / (uint32_t)sharers); }
    __device__ int block_of(int unit) const { return (int)((((uint32_t)unit + 1) * (uint32_t)sharers - 1) / (uint32_t)units); }   // the last block with first_unit <= unit
    __device__ bool next(Segment &s) {
        if (tile < whole) {
            s.tile = tile;
            s.kb0 = 0;
            s.kb1 = Kb;
            tile += grid;
            return true;
        }
        if (u >= u_end) return false;
        const int q = u / Kb;
        s.tile = whole + q;
        s.kb0 = u - q * Kb;
        s.kb1 = min(Kb, s.kb0 + (u_end - u));
        u += s.kb1 - s.kb0;
        return true;
    }
};

// The ring's barriers: full (operands are there), done (the MMAs have read them and their accumulator is complete); acc_empty (an accumulator may be written).
struct Ring {
    uint32_t sbase, full0, done0, acc0;
    volatile int *abort_flag;
    volatile int *progress;   // the unit that is fetched, at most the ring's stages ahead of the adding warps
    __device__ uint32_t full(int s) const { return full0 + 8u * s; }
    __device__ uint32_t done(int s) const { return done0 + 8u * s; }
    __device__ uint32_t acc_empty(int b) const { return acc0 + 8u * b; }
    __device__ uint32_t stage(const Args &p, int s) const { return sbase + (uint32_t)(s * p.stage_bytes); }
};

// The fetching warp. A stage: the rows' codes [a_rows][128], then W weight blocks [128][128].
// ONCE: a weight is mostly read by one block only. QUANT: the block quantises its rows itself.
template <int W, bool GATED, bool ONCE, bool QUANT>
__device__ __forceinline__ void fetch(const Args &p, const Ring &ring, Walk walk, const int *off, const int *cum) {
    const bool leader = elect_one();
    const uint64_t policy = ONCE ? l2_policy_evict_first() : 0;
    Segment seg;
    auto a_bytes = [&](const Tile &T) { return QUANT ? 0u : (uint32_t)(((T.hi + 7) & ~7) - T.base) * kF8Block; };
    auto fetch_weights = [&](int s, const Tile &T, int kb) {
        mbar_arrive_expect_tx(ring.full(s), a_bytes(T) + W * kF8BlockBytes);
        const uint32_t dst = ring.stage(p, s) + (uint32_t)(p.a_rows * kF8Block);
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (ONCE) tma_load_3d(dst + j * kF8BlockBytes, &p.wmap[GATED ? j : 0], kb * kF8Block, (GATED ? T.c : T.c * W + j) * kF8Block, T.e, ring.full(s), policy);
            else tma_load_3d_plain(dst + j * kF8BlockBytes, &p.wmap[GATED ? j : 0], kb * kF8Block, (GATED ? T.c : T.c * W + j) * kF8Block, T.e, ring.full(s));
    };
    // the weights of the first stages, before the activations exist
    int ahead = 0;
    for (Walk w = walk; p.early && ahead < p.stages && w.next(seg);) {
        const Tile T = tile_of(p, off, cum, seg.tile);
        for (int kb = seg.kb0; kb < seg.kb1 && ahead < p.stages; ++kb, ++ahead)
            if (leader) fetch_weights(ahead, T, kb);
    }
    grid_dep_wait();
    grid_dep_launch();   // (not before: a kernel that this lets start may rely on all that came before this one)
    fence_proxy_async_global();   // the activations were written by ordinary stores of the kernel before
    int s = 0, n = 0;
    uint32_t ph = 0;
    while (walk.next(seg)) {
        const Tile T = tile_of(p, off, cum, seg.tile);
        for (int kb = seg.kb0; kb < seg.kb1; ++kb, ++n) {
            if (n >= ahead) {
                if (!__all_sync(0xffffffffu, mbar_wait(ring.done(s), ph ^ 1, ring.abort_flag, p.status, 51, wait_clocks(p)))) return;
                if (leader) {
                    fetch_weights(s, T, kb);
                    *ring.progress = n;
                }
            }
            if (!QUANT && leader) bulk_g2s_plain(ring.stage(p, s), p.a.codes + ((int64_t)kb * p.a.rows_padded + T.base) * kF8Block, a_bytes(T), ring.full(s));
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
    }
}

// Issuing warp `which` of kIssuers: every kIssuers-th unit. The ring has to have NB stages or more: the wait for a free accumulator says that the unit NB before
// is over, and with it the stage's last use, whoever issued that; without it the parity of the wait for the stage would mean nothing. FULL_FIRST: the ring has an even
// number of stages, so that a stage is always the same warp's, and the waits may come the other way round. issue(stage address, accumulator, tile) issues the unit's MMAs.
template <int NB, bool FULL_FIRST, typename F>
__device__ __forceinline__ void issue_mmas(const Args &p, const Ring &ring, Walk walk, const int *off, const int *cum, int which, F issue) {
    grid_dep_wait();   // (the bounded waits are not to count the time of the kernel before)
    const bool leader = elect_one();
    Segment seg;
    int s = 0, n = 0;
    uint32_t ph = 0;
    while (walk.next(seg)) {
        const Tile T = tile_of(p, off, cum, seg.tile);
        for (int kb = seg.kb0; kb < seg.kb1; ++kb, ++n) {
            if (n % kIssuers == which) {
                const int buf = n % NB;
                const uint32_t acc_parity = (uint32_t)(((n / NB) & 1) ^ 1);
                auto wait_full = [&]() { return (bool)__all_sync(0xffffffffu, mbar_wait(ring.full(s), ph, ring.abort_flag, p.status, 53, wait_clocks(p))); };
                // (what mostly comes last is waited for last)
                if ((FULL_FIRST && !wait_full()) || !__all_sync(0xffffffffu, mbar_wait(ring.acc_empty(buf), acc_parity, ring.abort_flag, p.status, 52, wait_clocks(p))) ||
                    (!FULL_FIRST && !wait_full()))
                    return;
                tc_fence_after_sync();
                if (leader) {
                    issue(ring.stage(p, s), buf, T);
                    mma_commit(ring.done(s));
                }
            }
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
    }
}

// The blocks c0 .. c1 that share a tile, and where each leaves its sums: a block has a slot for the tile that its range starts in and one for the tile that it
// ends in.
struct Sharing {
    int q, c0, c1;
    bool c0_ends_here;   // (the others' ranges all start in the tile)
    __device__ Sharing(const Walk &w, const Segment &s) : q(s.tile - w.whole), c0(w.block_of(q * w.Kb)), c1(w.block_of(q * w.Kb + w.Kb - 1)), c0_ends_here(w.first_unit(c0) < q * w.Kb) {}
    __device__ float *part(const Args &p, int block, int tile_floats) const { return p.partials + (int64_t)(2 * block + (block == c0 && c0_ends_here ? 1 : 0)) * tile_floats; }
};

// The warps of `bar` meet (in bounded waits like every other). Returns false where that ran out.
struct Meeting {
    uint32_t bar, phase;
    volatile int *abort_flag;
    __device__ bool operator()(const Args &p) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
        const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, phase, abort_flag, p.status, 55, wait_clocks(p)));
        phase ^= 1;
        return ok;
    }
};

constexpr int BM = 128;   // rows of a block's part of a tile in the many-rows kernels

// 32 bytes, a whole sector.
__device__ __forceinline__ void store8(void *dst, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// 16 columns from n on of one row.
__device__ __forceinline__ void store16(const Args &p, int64_t row, int64_t n, const float *v) {
    const int64_t width = p.out_row_major ? p.N : ((p.N + 31) & ~(int64_t)31);
    if (n >= width) return;
    const int64_t off = p.out_row_major ? row * p.N + n : tiled_offset(row, n, width >> 5);
    uint32_t h[16];
    const bool whole = n + 16 <= width;
    if (p.out_dtype == TTB_FLOAT32) {
        float *o = reinterpret_cast<float *>(p.out) + off;
#pragma unroll
        for (int j = 0; j < 16; ++j) h[j] = __float_as_uint(v[j]);
        if (p.out_aligned >= 32 && whole) {
            store8(o, h);
            store8(o + 8, h + 8);
        } else if (p.out_aligned >= 16 && whole) {
#pragma unroll
            for (int q = 0; q < 4; ++q) reinterpret_cast<uint4 *>(o)[q] = make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (n + j < width) o[j] = v[j];
        }
    } else {
        uint16_t *o = reinterpret_cast<uint16_t *>(p.out) + off;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
        if (p.out_aligned >= 32 && whole) {
            store8(o, h);
        } else if (p.out_aligned >= 16 && whole) {
            reinterpret_cast<uint4 *>(o)[0] = make_uint4(h[0], h[1], h[2], h[3]);
            reinterpret_cast<uint4 *>(o)[1] = make_uint4(h[4], h[5], h[6], h[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (n + j < width) o[j] = f32_to_bf16_bits(v[j]);
        }
    }
}

// The activation. (apply_activation_t's relu makes a NaN zero: the other matmuls keep that.)
template <int ACT>
__device__ __forceinline__ float activate(float v) {
    return ACT == TTB_ACT_RELU ? (v <= 0.0f ? 0.0f : v) : apply_activation_t<ACT>(v);
}

// 16 columns from n on: bias, activation, store.
template <int ACT>
__device__ __forceinline__ void finish16(const Args &p, int64_t row, int64_t n, float *v) {
    if (p.bias && n < p.N) {
        const uint16_t *b = p.bias + (p.bias_row_major ? n : tiled_offset(0, n, p.N >> 5));   // (16 columns of the first tile row are neighbours)
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (n + j < p.N) v[j] += __uint_as_float((uint32_t)__ldg(b + j) << 16);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = activate<ACT>(v[j]);
    store16(p, row, n, v);
}

// A thread's columns of a whole tile. With an activation 16 at a time in a loop that shifts the sums down: 128 inlined activations are up to 60 KB of code, which
// runs cold once a tile (a 350 x 4544 x 4672 launch with gelu: 39 us against 21 without finishing its tiles).
template <int ACT, int NC>
__device__ __forceinline__ void finish_row(const Args &p, int64_t row, int64_t n0, float (&acc)[NC]) {
    if (!p.out_row_major && n0 + NC > p.N) {   // columns that only pad a tile: a NaN or an infinity of the row times the zeros behind the weight's last row is a NaN
#pragma unroll
        for (int j = 0; j < NC; ++j)
            if (n0 + j >= p.N) acc[j] = 0.0f;
    }
    if constexpr (ACT == TTB_ACT_NONE) {
#pragma unroll
        for (int q = 0; q < NC; q += 16) finish16<ACT>(p, row, n0 + q, acc + q);
    } else {
#pragma unroll 1
        for (int q = 0; q < NC; q += 16) {
            finish16<ACT>(p, row, n0 + q, acc);
#pragma unroll
            for (int j = 0; j + 16 < NC; ++j) acc[j] = acc[j + 16];
        }
    }
}

// act(g) * u; silu with a division that is right to 2 units in the last place, like the exponential (where 1 + exp(-g) passes 2^126 the result, less than 2^-119 of u,
// becomes 0). The fast exponential would be off by a part of 2^-24 that grows with |g|.
template <int ACT>
__device__ __forceinline__ float gate(float g, float u) {
    if (ACT == TTB_ACT_SILU) return __fdividef(g, 1.0f + expf(-g)) * u;
    return activate<ACT>(g) * u;
}

// act(g) * u of one row's 64 columns from part * 64 on, quantised with the scale of all 128: the two warps of the rows exchange their largest magnitudes
// through `red`.
template <int ACT>
__device__ __forceinline__ bool finish_gated(const Args &p, int row, bool valid, int c, int part, int lane_row, float (&acc)[128], float (*red)[BM], Meeting &meet) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
        acc[j] = gate<ACT>(acc[j], acc[64 + j]);
        m = fmaxf(m, fabsf(acc[j]));
    }
    red[part][lane_row] = m;
    if (!meet(p)) return false;
    const float scale = f8_scale(fmaxf(m, red[part ^ 1][lane_row]));
    if (!meet(p)) return false;   // (the next tile writes `red` again)
    if (!valid) return true;
    const F8Codes codes(scale);
#pragma unroll
    for (int q = 0; q < 64; q += 16)
        *reinterpret_cast<uint4 *>(p.h.codes + f8_act_offset(p.h.rows_padded, c, row, part * 64 + q)) =
            make_uint4(codes.four(acc + q), codes.four(acc + q + 4), codes.four(acc + q + 8), codes.four(acc + q + 12));
    if (part == 0) p.h.scales[row * p.h.scale_pitch + c] = scale;
    return true;
}

// Four columns from n (a multiple of four) on of one row.
template <int ACT>
__device__ __forceinline__ void finish4(const Args &p, int64_t row, int64_t n, float4 s) {
    const int64_t width = p.out_row_major ? p.N : (p.N + 31) & ~(int64_t)31;
    if (n >= width) return;
    float v[4] = {s.x, s.y, s.z, s.w};
    if (p.bias) {
        const uint16_t *b = p.bias + (p.bias_row_major ? n : tiled_offset(0, n, p.N >> 5));   // (first tile row: the pitch does not count)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) v[j] += __uint_as_float((uint32_t)b[j] << 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = n + j < p.N ? activate<ACT>(v[j]) : 0.0f;   // (as in finish_row)
    const int64_t off = p.out_row_major ? row * p.N + n : tiled_offset(row, n, width >> 5);
    const bool f32 = p.out_dtype == TTB_FLOAT32;
    if (p.out_aligned >= 16 && n + 4 <= width) {
        if (f32) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.out) + off) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.out) + off) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < width) {
            if (f32) reinterpret_cast<float *>(p.out)[off + j] = v[j];
            else reinterpret_cast<uint16_t *>(p.out)[off + j] = f32_to_bf16_bits(v[j]);
        }
}

// One row of a tile by a whole warp: lane l has columns 4 l .. 4 l + 3 of each of the W weight blocks.
template <int ACT, int W, bool GATED>
__device__ __forceinline__ void finish_row_warp(const Args &p, int row, int c, int lane, const float4 (&s)[W]) {
    if constexpr (GATED) {
        const float h[4] = {gate<ACT>(s[0].x, s[W - 1].x), gate<ACT>(s[0].y, s[W - 1].y), gate<ACT>(s[0].z, s[W - 1].z), gate<ACT>(s[0].w, s[W - 1].w)};
        float m = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float scale = f8_scale(m);
        *reinterpret_cast<uint32_t *>(p.h.codes + f8_act_offset(p.h.rows_padded, c, row, lane * 4)) = F8Codes(scale).four(h);
        if (lane == 0) p.h.scales[row * p.h.scale_pitch + c] = scale;
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j) finish4<ACT>(p, row, ((int64_t)c * W + j) * kF8Block + lane * 4, s[j]);
    }
}

// One more arrival. Releases what this thread has seen written (the other threads' stores are ordered before by the meeting of the warps) and acquires what
// the earlier arrivals released; a fence in every thread cost 20 us a shared tile here, beside the copies in flight.
__device__ __forceinline__ int take_ticket(int *counter) {
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    return old;
}

__device__ __forceinline__ int read_tickets(const int *counter) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
    return v;
}

// Adds the parts of blocks c0 .. c1 of the rows r0, r0 + STEP, .. below r_end, in block order, and finishes the rows: RU rows and BU blocks at a time, all loads
// of which are under way together. (Little code on purpose: it runs once a shared tile, mostly with cold instruction caches. Eight rows at a time of 16 a
// warp, with the activation chosen row by row, took 25 us longer.)
// `own`: null, or the part of c0, which its block still has in shared memory, [row][128 W].
template <int ACT, int W, bool GATED, int RU, int BU, int STEP, typename F>
__device__ __forceinline__ void add_parts(const Args &p, F part_of, int c0, int c1, int r0, int r_end, int base, int c, int lane, const float *own = nullptr) {
#pragma unroll 1
    for (int r = r0; r < r_end; r += STEP * RU) {
        float4 sum[RU][W];
#pragma unroll
        for (int i = 0; i < RU; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                sum[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (own && r + STEP * i < r_end) sum[i][j] = *reinterpret_cast<const float4 *>(own + (r + STEP * i) * (128 * W) + j * 128 + lane * 4);
            }
#pragma unroll 1
        for (int b0 = own ? c0 + 1 : c0; b0 <= c1; b0 += BU) {
            float4 v[BU][RU][W];
#pragma unroll
            for (int b = 0; b < BU; ++b) {
                const float *const part = part_of(min(b0 + b, c1)) + lane * 4;
#pragma unroll
                for (int i = 0; i < RU; ++i)
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        v[b][i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (b0 + b <= c1 && r + STEP * i < r_end) v[b][i][j] = __ldcg(reinterpret_cast<const float4 *>(part + (r + STEP * i) * (128 * W) + j * 128));
                    }
            }
#pragma unroll
            for (int b = 0; b < BU; ++b)
#pragma unroll
                for (int i = 0; i < RU; ++i)
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        sum[i][j].x += v[b][i][j].x; sum[i][j].y += v[b][i][j].y; sum[i][j].z += v[b][i][j].z; sum[i][j].w += v[b][i][j].w;
                    }
        }
#pragma unroll
        for (int i = 0; i < RU; ++i)
            if (r + STEP * i < r_end) finish_row_warp<ACT, W, GATED>(p, base + r + STEP * i, c, lane, sum[i]);
    }
}

// mbar_wait for what lies any number of units ahead: the limit is for the time in which no unit is fetched. (A wait with one limit for all of it would run out in a
// sound launch that is longer than the limit. The fetching warp has the time to say where it is: a store a unit in the adding warps cost 4 % of 2048 rows on experts,
// one in the issuing warps 1 % of 2048 x 8192 x 28672.)
__device__ __forceinline__ bool wait_while_units_pass(const Ring &ring, uint32_t bar, uint32_t parity, int *status, int code, long long limit) {
    if (mbar_try_wait(bar, parity)) return true;
    int at = *ring.progress;
    long long t0 = clock64();
    for (uint32_t spin = 1;; ++spin) {
        if (mbar_try_wait_suspend(bar, parity, 4000u)) return true;
        if ((spin & 7u) == 0u) {
            if (*ring.abort_flag) return false;
            if (*ring.progress != at) {
                at = *ring.progress;
                t0 = clock64();
            } else if (clock64() - t0 > limit) {
                *ring.abort_flag = 1;
                atomicCAS(status, 0, code);
                return false;
            }
        }
    }
}

// The warp that takes the ticket for the one shared tile that is not its block's last segment (a range is at most a tile long), while the next segment runs:
// `handed` says that its part is written. Where all parts are there with it, it finishes the tile itself if it has few rows (ADD), else the adding warps do it after
// their last segment (`pending`: the tile, or -1; then `told`): one warp alone took 126 x 18272 x 6376 from 47 to 83 us.
template <int ACT, int W, bool GATED, bool ADD>
__device__ __forceinline__ void hand_over(const Args &p, uint32_t handed, uint32_t told, volatile int *pending, const Ring &ring, Walk walk, const int *off, const int *cum) {
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    Segment seg;
    while (walk.next(seg)) {
        if (seg.kb1 - seg.kb0 == p.Kb || walk.u >= walk.u_end) continue;
        if (!__all_sync(0xffffffffu, wait_while_units_pass(ring, handed, 0, p.status, 56, wait_clocks(p)))) return;
        const Sharing sh(walk, seg);
        int last = 0;
        if (lane == 0) last = take_ticket(p.tickets + sh.q) == sh.c1 - sh.c0;
        if constexpr (!ADD) {
            if (lane == 0) {
                *pending = last ? seg.tile : -1;
                mbar_arrive(told);
            }
            return;
        }
        if (!__shfl_sync(0xffffffffu, last, 0)) return;
        __syncwarp();   // what lane 0 acquired with its ticket, the parts, is ordered before the other lanes' reads by this, not by the shuffle
        if (lane == 0) p.tickets[sh.q] = 0;
        const Tile T = tile_of(p, off, cum, seg.tile);
        auto part_of = [&](int block) { return sh.part(p, block, p.partial_rows * 128 * W); };
        add_parts<ACT, W, GATED, 1, 4 / W, 1>(p, part_of, sh.c0, sh.c1, T.lo - T.base, T.hi - T.base, T.base, T.c, lane);
        return;
    }
}

}  // namespace f8
}  // namespace ttb
