// Mixture of experts: the router (scores, groups, top-k, weights) and the experts' gated MLP on float8 weights.
//
// Router. A warp takes a row. An expert's choice value is its logit where that orders the scores (no bias, no sum over a group: the order is then that of exact
// scores, also where they saturate in 64 bits), else score + bias, first in 32 bits and, for the rows where two values that decide lie closer than that tells, again
// in 64: the choice is a whole number and has to be that of 64-bit values. Ties go to the lowest index. Bound by instructions, not by the logits' bytes: 8191 rows of 128
// with bias and 4 of 8 groups, top 6, 19.3 us, 1490 warp instructions a row at 61 % of the issue slots; by logits alone 9.5 us and 780. (All rows in 64 bits: 22 us.)
//
// The MLP y[t] = sum_j p[t, j] * down_e( q(act(gate_e x) * (up_e x)) ), e = ids[t, j], runs as
//   plan      every assignment (t, j) gets a row, sorted by expert and then by t * k + j, with no room between the experts (the matmul's row tiles start at
//             a multiple of eight rows and leave the rows before an expert's first alone);
//   quantise  each token once, written to its k rows in the operand layout;
//   gated     matmul of both weights, product and quantisation in the epilogue;
//   down      matmul, fp32 rows;
//   combine   the weighted sum of a token's rows, in the order of j.
// Sums, weights and the rows between down and combine are fp32; no atomics on numbers, so results repeat bit for bit.
#include "epilogue.cuh"
#include "matmul_float8.cuh"
#include "sm100_ptx.cuh"

#include <math_constants.h>

namespace ttb {
namespace {

using namespace ptx;

constexpr int kMaxExperts = kF8MaxExperts, kMaxTopK = 32, kMaxGroups = 32;
constexpr int kRouteWarps = 4;

struct RouteArgs {
    const void *logits;
    const float *bias;     // [E] or null
    float *weights;
    int32_t *experts;
    int64_t rows, H;
    int E, k, groups, top_groups;
    bool bf16, row_major, sigmoid, sum_of_two, renormalize;
    float scale;
};

__device__ __forceinline__ void best_of_warp(double &v, int &i) {   // the largest value, the lowest index among equals
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        const double w = __shfl_xor_sync(0xffffffffu, v, d);
        const int j = __shfl_xor_sync(0xffffffffu, i, d);
        if (w > v || (w == v && j < i)) { v = w; i = j; }
    }
}
// The same for 32-bit values, as two integer reductions: a larger value has the larger ordered().
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);   // (one zero)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ void best_of_warp(float &v, int &i) {
    const uint32_t u = ordered(v), top = __reduce_max_sync(0xffffffffu, u);
    i = __reduce_min_sync(0xffffffffu, u == top ? i : kMaxExperts);
    v = from_ordered(top);
}

// The chosen experts of one row, one a lane: lane j keeps the j-th (index E: none). `x`: this lane's logits, `key`: choice values (-inf: not to be chosen).
// MARGIN: also says whether no two values that decide something lie within `eps` of each other.
template <typename K, int V, bool MARGIN>
__device__ __forceinline__ bool choose(const RouteArgs &p, const float (&x)[V], K (&key)[V], K eps, K *mine, int lane, int &my_id, float &my_x, float &first) {
    const K none = -CUDART_INF_F;
    bool sure = true;
    if (p.groups > 1) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * 32 + lane < p.E) mine[i * 32 + lane] = key[i];
        __syncwarp();
        const int size = p.E / p.groups;
        K v = none;
        if (lane < p.groups) {
            K second = none;
            for (int i = 0; i < size; ++i) {
                const K c = mine[lane * size + i];
                if (c > v) { second = v; v = c; }
                else if (c > second) second = c;
            }
            if (p.sum_of_two && second > none) v += second;
        }
        uint32_t kept = 0;
        K last = none;
        for (int g = 0; g <= p.top_groups && g < p.groups; ++g) {   // (one more than is kept, for the margin)
            const bool free = lane < p.groups && !(kept >> lane & 1);
            K b = free ? v : none;
            int i = free ? lane : 64;
            best_of_warp(b, i);
            if (g == p.top_groups) {
                if (MARGIN) sure = sure && (b == none || last - b > 2 * eps);
                break;
            }
            if (i < 32) kept |= 1u << i;
            last = b;
            if (!MARGIN && g + 1 == p.top_groups) break;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = i * 32 + lane;
            if (e < p.E && !(kept >> (e / size) & 1)) key[i] = none;
        }
        __syncwarp();   // (`mine` may be written again)
    }
    my_id = p.E;
    my_x = first = 0.0f;
    K last = none;
    for (int j = 0; j <= p.k; ++j) {
        if (!MARGIN && j == p.k) break;
        K b = none;
        int id = kMaxExperts;
        float bx = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (key[i] > b) { b = key[i]; id = i * 32 + lane; bx = x[i]; }
        const int own = id;
        best_of_warp(b, id);
        if (b == none) break;   // nothing is left
        if (MARGIN && j > 0) sure = sure && last - b > eps;
        last = b;
        if (j == p.k) break;
        bx = __shfl_sync(0xffffffffu, bx, id & 31);
        if (own == id) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i * 32 + lane == id) key[i] = none;
        }
        if (lane == j) { my_id = id; my_x = bx; }
        first = j == 0 ? bx : fmaxf(first, bx);
    }
    return sure;
}

// V: logits per lane.
template <int V>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteArgs p) {
    extern __shared__ double choice_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * kRouteWarps + warp;
    if (r >= p.rows) return;
    const int64_t o = r / p.H, h = r - o * p.H;
    float x[V];
    bool nan = false;
    float most = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i * 32 + lane;
        x[i] = -CUDART_INF_F;
        if (e < p.E) {
            const int64_t at = p.row_major ? r * p.E + e : o * (((p.H + 31) & ~(int64_t)31) * ((p.E + 31) & ~31)) + tiled_offset(h, e, (p.E + 31) >> 5);
            x[i] = p.bf16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p.logits)[at] << 16) : reinterpret_cast<const float *>(p.logits)[at];
            nan |= x[i] != x[i] || (x[i] == CUDART_INF_F && !p.sigmoid);   // (inf - inf in the softmax)
            most = fmaxf(most, x[i]);
        }
    }
    nan = __any_sync(0xffffffffu, nan);
    most = from_ordered(__reduce_max_sync(0xffffffffu, ordered(most)));
    const bool by_score = p.bias != nullptr || (p.groups > 1 && p.sum_of_two);
    double *const mine = choice_smem + (size_t)warp * p.E;
    // exp's argument; among infinite logits, whose softmax is NaN, those come first all the same
    auto below = [&](auto v) { return v == most ? decltype(v)(0) : v - decltype(v)(most); };
    auto is_free = [&](int i) { return i * 32 + lane < p.E && x[i] > -CUDART_INF_F; };   // (false for a NaN)
    int my_id;
    float my_x, first, key[V];
    bool sure;
    if (!by_score) {   // the logits order the scores
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = is_free(i) ? x[i] : -CUDART_INF_F;
        sure = choose<float, V, false>(p, x, key, 0.0f, reinterpret_cast<float *>(mine), lane, my_id, my_x, first);
    } else {
        // In 32 bits first. A score is off by at most 2^-20 of 1 (exp, a sum of up to 1024 terms, a division), the sum with the bias by 2^-24 of itself.
        float total = 1.0f, size = 1.0f;
        if (!p.sigmoid) {
            total = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (is_free(i)) total += expf(below(x[i]));
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            key[i] = -CUDART_INF_F;
            if (is_free(i)) {
                const float s = p.sigmoid ? 1.0f / (1.0f + expf(-x[i])) : expf(below(x[i])) / total, b = p.bias ? p.bias[i * 32 + lane] : 0.0f;
                key[i] = s + b == s + b ? s + b : -CUDART_INF_F;
                if (fabsf(b) < CUDART_INF_F) size = fmaxf(size, fabsf(b));
            }
        }
        size = from_ordered(__reduce_max_sync(0xffffffffu, ordered(size)));
        sure = choose<float, V, true>(p, x, key, size * 0x1p-18f, reinterpret_cast<float *>(mine), lane, my_id, my_x, first);
    }
    double total = 1.0;
    if (!p.sigmoid && (!sure || !p.renormalize)) {
        total = 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (is_free(i)) total += exp(below((double)x[i]));
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    auto score = [&](float v) { return p.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp(below((double)v)) / total; };
    if (!sure) {   // two values next to each other: again in 64 bits
        double key64[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            key64[i] = -CUDART_INF;
            if (is_free(i)) {
                const double s = score(x[i]) + (p.bias ? (double)p.bias[i * 32 + lane] : 0.0);
                if (s == s) key64[i] = s;
            }
        }
        choose<double, V, false>(p, x, key64, 0.0, mine, lane, my_id, my_x, first);
    }
    double w = 0.0;   // (the softmax's denominator drops out of shares)
    if (my_id < p.E) w = p.renormalize && !p.sigmoid ? exp((double)my_x - (by_score ? (double)most : (double)first)) : score(my_x);
    if (p.renormalize) {
        double sum = w;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (sum != 0.0) w /= sum;
    }
    if (lane < p.k) {
        p.experts[r * p.k + lane] = my_id;
        p.weights[r * p.k + lane] = my_id < p.E ? (nan ? CUDART_NAN_F : (float)(w * (double)p.scale)) : 0.0f;
    }
}

// Block e: the rows of expert e. ids outside [0, E) get no row. row_of: the row of the activations (of a tiled tensor: with its padding) that a row is from.
// Every block looks through all ids, eight neighbours a thread (so that the loads of 8192 are under way together): first for those of the experts before e, whose
// rows come first, then for its own. (One id a thread and step took 51 us for 16384 assignments.)
constexpr int kPlanThreads = 1024, kPlanIds = 8;
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t *ids, int64_t assignments, int E, int k, int H, int Hp, int32_t *offsets, int32_t *pos, int32_t *row_of,
                                                            int32_t *zero, int zeros) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int warp_sum[2][32];
    const int e = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = e * kPlanThreads + threadIdx.x; i < zeros; i += gridDim.x * kPlanThreads) zero[i] = 0;
    const bool vector = (reinterpret_cast<uintptr_t>(ids) & 15) == 0;
    auto load = [&](int64_t i, int (&x)[kPlanIds]) {   // behind the end: -1
        if (vector && i + kPlanIds <= assignments) {
#pragma unroll
            for (int q = 0; q < kPlanIds; q += 4) {
                const int4 v = __ldcg(reinterpret_cast<const int4 *>(ids + i + q));
                x[q] = v.x; x[q + 1] = v.y; x[q + 2] = v.z; x[q + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int q = 0; q < kPlanIds; ++q) x[q] = i + q < assignments ? __ldcg(ids + i + q) : -1;
        }
    };
    constexpr int64_t step = kPlanThreads * kPlanIds;
    int below = 0, x[kPlanIds];
    for (int64_t i = (int64_t)threadIdx.x * kPlanIds; i < assignments; i += step) {
        load(i, x);
#pragma unroll
        for (int q = 0; q < kPlanIds; ++q) {
            below += x[q] >= 0 && x[q] < e;
            if (e == 0 && i + q < assignments && (x[q] < 0 || x[q] >= E)) pos[i + q] = -1;
        }
    }
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) warp_sum[0][warp] = below;
    __syncthreads();
    int next = __reduce_add_sync(0xffffffffu, warp_sum[0][lane]);
    if (threadIdx.x == 0) offsets[e] = next;
    int buf = 1;
    for (int64_t i0 = 0; i0 < assignments; i0 += step, buf ^= 1) {
        const int64_t i = i0 + (int64_t)threadIdx.x * kPlanIds;
        if (assignments > step || i0 > 0) load(i, x);   // (else they are there still)
        else if (i >= assignments) load(i, x);
        int mine = 0;
#pragma unroll
        for (int q = 0; q < kPlanIds; ++q) mine += x[q] == e;
        int before = mine;   // rows of e up to and with this thread's
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before += y;
        }
        if (lane == 31) warp_sum[buf][warp] = before;
        __syncthreads();   // (the other buffer is free again: whoever reads it has come here)
        const int s = warp_sum[buf][lane];
        int at = next + before - mine + __reduce_add_sync(0xffffffffu, lane < warp ? s : 0);
        next += __reduce_add_sync(0xffffffffu, s);
#pragma unroll
        for (int q = 0; q < kPlanIds; ++q)
            if (x[q] == e && i + q < assignments) {
                const int row = (int)((i + q) / k);
                pos[i + q] = at;
                row_of[at++] = row / H * Hp + row % H;
            }
    }
    if (e == E - 1 && threadIdx.x == 0) offsets[E] = next;
}

// out[t] = sum_j weights[t, j] * y[pos[t, j]], four columns a thread; rows that only pad a tile are zero.
__global__ void __launch_bounds__(256) combine_kernel(const float *y, const int32_t *pos, const float *weights, uint16_t *out, int64_t outer, int64_t H, int64_t Hp,
                                                      int64_t hidden, int64_t width, int k, bool row_major) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t quads = width / 4, total = outer * Hp * quads;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t pr = i / quads, c = (i - pr * quads) * 4, o = pr / Hp, h = pr - o * Hp;
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (h < H && c < hidden) {
            const int64_t r = o * H + h;
            for (int j0 = 0; j0 < k; j0 += 4) {   // four of the token's rows under way together
                int32_t at[4];
                float w[4];
                float4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    at[j] = j0 + j < k ? __ldcg(pos + r * k + j0 + j) : -1;
                    w[j] = j0 + j < k ? weights[r * k + j0 + j] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at[j] >= 0) v[j] = __ldcg(reinterpret_cast<const float4 *>(y + (int64_t)at[j] * hidden + c));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at[j] >= 0) {
                        s.x = fmaf(w[j], v[j].x, s.x); s.y = fmaf(w[j], v[j].y, s.y); s.z = fmaf(w[j], v[j].z, s.z); s.w = fmaf(w[j], v[j].w, s.w);
                    }
            }
        }
        uint16_t *dst = out + (row_major ? pr * width + c : o * Hp * width + tiled_offset(h, c, width >> 5));
        *reinterpret_cast<uint2 *>(dst) = make_uint2((uint32_t)f32_to_bf16_bits(s.x) | ((uint32_t)f32_to_bf16_bits(s.y) << 16),
                                                     (uint32_t)f32_to_bf16_bits(s.z) | ((uint32_t)f32_to_bf16_bits(s.w) << 16));
    }
}

template <typename... P, typename... A>
int32_t launch_dependent(void (*kernel)(P...), unsigned grid, unsigned block, cudaStream_t stream, const char *name, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
    TTB_LAUNCH_CHECK(name);
    return TTB_OK;
}

template <int V>
int32_t launch_route(const RouteArgs &p, cudaStream_t stream) {
    const int64_t blocks = (p.rows + kRouteWarps - 1) / kRouteWarps;
    const size_t smem = p.groups > 1 ? (size_t)kRouteWarps * p.E * 8 : 0;
    route_kernel<V><<<(unsigned)blocks, 32 * kRouteWarps, smem, stream>>>(p);
    TTB_LAUNCH_CHECK("route");
    return TTB_OK;
}

// Scratch of the experts' MLP.
struct Scratch {
    int64_t assignments;
    int32_t *offsets, *pos, *row_of;
    F8Activation x, h;
    float *y;
    int32_t *gated_tickets, *down_tickets;   // neighbours, cleared together
    float *partials;                         // of either matmul, one after the other
    int64_t bytes;
};
Scratch lay_out(uint8_t *base, int64_t rows, int64_t experts, int64_t k, int64_t hidden, int64_t ffn) {
    Scratch s;
    s.assignments = rows * k;
    int64_t at = 0;
    s.offsets = reinterpret_cast<int32_t *>(base + at);
    at = f8_up(at + 4 * (experts + 1), 1024);
    s.pos = reinterpret_cast<int32_t *>(base + at);
    at = f8_up(at + 4 * s.assignments, 1024);
    s.row_of = reinterpret_cast<int32_t *>(base + at);
    at = f8_up(at + 4 * s.assignments, 1024);
    s.x = f8_quantises_itself(s.assignments, experts) ? F8Activation{} : f8_place(base, at, s.assignments, hidden);
    s.h = f8_place(base, at, s.assignments, ffn);
    s.y = reinterpret_cast<float *>(base + at);
    at = f8_up(at + s.assignments * hidden * 4, 1024);
    s.gated_tickets = reinterpret_cast<int32_t *>(base + at);
    s.down_tickets = reinterpret_cast<int32_t *>(base + at + kF8TicketBytes);
    at += 2 * kF8TicketBytes;
    s.partials = reinterpret_cast<float *>(base + at);
    at += f8_partial_bytes(s.assignments);
    s.bytes = at;
    return s;
}
constexpr int64_t kMaxExtent = int64_t(1) << 24;
bool in_range(int64_t v) { return v > 0 && v <= kMaxExtent; }

}  // namespace
}  // namespace ttb

using ttb::fail;

extern "C" {

int32_t ttb_route_to_experts(const void *logits, int32_t logits_dtype, const void *bias, void *weights, void *experts, int64_t outer, int64_t H, int64_t E,
                             int32_t k, int32_t score, int32_t groups, int32_t top_groups, int32_t group_score, int32_t renormalize, float scale, int32_t flags,
                             void *stream) {
    const char *who = "ttb_route_to_experts";
    if (!logits || !weights || !experts) return fail(TTB_E_INVALID, "%s: null tensor pointer", who);
    if (logits_dtype != TTB_FLOAT32 && logits_dtype != TTB_BFLOAT16) return fail(TTB_E_UNSUPPORTED, "%s: the logits must be float32 or bfloat16", who);
    if (flags & ~TTB_MM_A_ROW_MAJOR) return fail(TTB_E_INVALID, "%s: unknown flags %d", who, flags);
    if (outer <= 0 || H <= 0 || outer > INT32_MAX || H > INT32_MAX || outer * H > INT32_MAX) return fail(TTB_E_INVALID, "%s: the row count must be between 1 and 2^31 - 1", who);
    if (E < 1 || E > ttb::kMaxExperts) return fail(TTB_E_UNSUPPORTED, "%s: between 1 and %d experts, got %lld", who, ttb::kMaxExperts, (long long)E);
    if (k < 1 || k > ttb::kMaxTopK || k > E) return fail(TTB_E_INVALID, "%s: k must be between 1 and the number of experts, at most %d, got %d", who, ttb::kMaxTopK, k);
    if (score != TTB_SCORE_SOFTMAX && score != TTB_SCORE_SIGMOID) return fail(TTB_E_INVALID, "%s: unknown score %d", who, score);
    if (groups < 1 || groups > ttb::kMaxGroups || E % groups) return fail(TTB_E_INVALID, "%s: the experts must divide into 1 to %d groups of one size", who, ttb::kMaxGroups);
    if (top_groups < 1 || top_groups > groups) return fail(TTB_E_INVALID, "%s: top_groups must be between 1 and the number of groups", who);
    if (k > E / groups * top_groups) return fail(TTB_E_INVALID, "%s: %d groups of %lld experts have no %d to choose", who, top_groups, (long long)(E / groups), k);
    if (group_score != TTB_GROUP_MAX && group_score != TTB_GROUP_TOP2_SUM) return fail(TTB_E_INVALID, "%s: unknown group score %d", who, group_score);
    if (ttb::f8_misaligned(logits, logits_dtype == TTB_FLOAT32 ? 4 : 2) || (bias && ttb::f8_misaligned(bias, 4)) || ttb::f8_misaligned(weights, 4) || ttb::f8_misaligned(experts, 4))
        return fail(TTB_E_INVALID, "%s: misaligned tensor", who);
    ttb::RouteArgs p;
    p.logits = logits; p.bias = (const float *)bias; p.weights = (float *)weights; p.experts = (int32_t *)experts;
    p.rows = outer * H; p.H = H; p.E = (int)E; p.k = k; p.groups = groups; p.top_groups = top_groups;
    p.bf16 = logits_dtype == TTB_BFLOAT16; p.row_major = flags & TTB_MM_A_ROW_MAJOR; p.sigmoid = score == TTB_SCORE_SIGMOID;
    p.sum_of_two = group_score == TTB_GROUP_TOP2_SUM; p.renormalize = renormalize != 0; p.scale = scale;
    const cudaStream_t s = (cudaStream_t)stream;
    if (E <= 32) return ttb::launch_route<1>(p, s);
    if (E <= 64) return ttb::launch_route<2>(p, s);
    if (E <= 128) return ttb::launch_route<4>(p, s);
    if (E <= 256) return ttb::launch_route<8>(p, s);
    return ttb::launch_route<32>(p, s);
}

int64_t ttb_experts_mlp_float8_workspace_bytes(int64_t rows, int64_t experts, int64_t k, int64_t hidden, int64_t ffn) {
    using ttb::in_range;
    if (!in_range(rows) || experts < 1 || experts > ttb::kMaxExperts || k < 1 || k > ttb::kMaxTopK || !in_range(rows * k) || !in_range(hidden) || !in_range(ffn)) return -1;
    return ttb::lay_out(nullptr, rows, experts, k, hidden, ffn).bytes;
}

int32_t ttb_experts_mlp_float8(const void *x, const void *ids, const void *weights, const void *gate_codes, const void *gate_scales, const void *up_codes,
                               const void *up_scales, const void *down_codes, const void *down_scales, void *out, int64_t outer, int64_t H, int64_t experts,
                               int32_t k, int64_t hidden, int64_t ffn, int32_t activation, int32_t flags, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "ttb_experts_mlp_float8";
    if (!x || !ids || !weights || !gate_codes || !gate_scales || !up_codes || !up_scales || !down_codes || !down_scales || !out)
        return fail(TTB_E_INVALID, "%s: null tensor pointer", who);
    if (flags & ~(TTB_MM_A_ROW_MAJOR | TTB_MM_OUT_ROW_MAJOR)) return fail(TTB_E_INVALID, "%s: unknown flags %d", who, flags);
    if (activation < TTB_ACT_NONE || activation > TTB_ACT_SILU) return fail(TTB_E_INVALID, "%s: unknown activation %d", who, activation);
    if (!ttb::in_range(outer) || !ttb::in_range(H)) return fail(TTB_E_INVALID, "%s: rows must be between 1 and 2^24", who);
    const int64_t rows = outer * H, need = ttb_experts_mlp_float8_workspace_bytes(rows, experts, k, hidden, ffn);
    if (need < 0)
        return fail(TTB_E_INVALID, "%s: between 1 and 2^24 rows times k, hidden and ffn sizes of at most 2^24, 1 to %d experts and k of 1 to %d", who, ttb::kMaxExperts, ttb::kMaxTopK);
    if (hidden % 16 || ffn % 16) return fail(TTB_E_INVALID, "%s: the hidden and ffn sizes must be multiples of 16 (got %lld, %lld)", who, (long long)hidden, (long long)ffn);
    if (!ttb::f8_blocks_count(rows, hidden)) return fail(TTB_E_UNSUPPORTED, "%s: too many blocks of 128 activations", who);
    for (const void *p : {x, gate_codes, up_codes, down_codes, (const void *)out})
        if (ttb::f8_misaligned(p, 16)) return fail(TTB_E_INVALID, "%s: activations, codes and the result must be 16-byte aligned", who);
    for (const void *p : {ids, weights, gate_scales, up_scales, down_scales})
        if (ttb::f8_misaligned(p, 4)) return fail(TTB_E_INVALID, "%s: misaligned tensor", who);
    if (!ttb::workspace_serves(workspace, workspace_bytes, need)) return fail(TTB_E_WORKSPACE, "%s: needs %lld bytes of 256-byte aligned workspace", who, (long long)need);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool x_rm = flags & TTB_MM_A_ROW_MAJOR, out_rm = flags & TTB_MM_OUT_ROW_MAJOR;
    const ttb::Scratch w = ttb::lay_out(static_cast<uint8_t *>(workspace), rows, experts, k, hidden, ffn);
    if (int32_t rc = ttb::launch_dependent(ttb::plan_kernel, (unsigned)experts, ttb::kPlanThreads, s, "plan", (const int32_t *)ids, w.assignments, (int)experts, (int)k, (int)H,
                                           (int)(x_rm ? H : ttb::round_up32(H)), w.offsets, w.pos, w.row_of, w.gated_tickets, (int)(2 * ttb::kF8TicketBytes / 4)))
        return rc;
    ttb::F8Matmul m = {};
    if (ttb::f8_quantises_itself(w.assignments, experts)) {
        m.x = {static_cast<const uint16_t *>(x), w.row_of, x_rm ? hidden : (hidden + 31) / 32 * 1024, !x_rm};
    } else {
        if (int32_t rc = ttb::launch_quantize_operand(x, x_rm, outer, H, hidden, w.x, w.pos, k, false, s)) return rc;
        m.a = w.x;
        m.early = true;   // (the quantiser waits for the plan before it lets the matmul start)
    }
    m.w[0] = {gate_codes, (const float *)gate_scales};
    m.w[1] = {up_codes, (const float *)up_scales};
    m.rows = w.assignments; m.K = hidden; m.N = ffn;
    m.experts = (int)experts; m.offsets = w.offsets;
    m.act = activation;
    m.gated = true; m.h = w.h;
    m.tickets = w.gated_tickets; m.partials = w.partials;
    if (int32_t rc = ttb::launch_matmul_float8(m, s)) return rc;
    ttb::F8Matmul d = {};
    d.a = w.h;
    d.early = true;   // (so does the gated matmul)
    d.w[0] = {down_codes, (const float *)down_scales};
    d.rows = w.assignments; d.K = ffn; d.N = hidden;
    d.experts = (int)experts; d.offsets = w.offsets;
    d.act = TTB_ACT_NONE;
    d.tickets = w.down_tickets; d.partials = w.partials;
    d.out = w.y; d.out_dtype = TTB_FLOAT32; d.out_row_major = true;
    if (int32_t rc = ttb::launch_matmul_float8(d, s)) return rc;
    const int64_t Hp = out_rm ? H : ttb::round_up32(H), width = out_rm ? hidden : ttb::round_up32(hidden);
    const int64_t want = (outer * Hp * (width / 4) + 255) / 256;
    return ttb::launch_dependent(ttb::combine_kernel, (unsigned)(want < 148 * 32 ? want : 148 * 32), 256, s, "combine", (const float *)w.y, (const int32_t *)w.pos,
                                 (const float *)weights, (uint16_t *)out, outer, H, Hp, hidden, width, (int)k, out_rm);
}

}  // extern "C"
