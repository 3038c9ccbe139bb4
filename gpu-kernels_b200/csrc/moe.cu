// moe.cu — the mixture-of-experts layer around the experts' products: the top-k router
// (weights, experts, the row of each token's choice in expert order, row offsets), the
// movement of token rows to expert order and back, and the gradients of all of them.
//
// Measured: router of 16 tokens, 64 experts, one launch, 4.1 us; 16381 tokens, 256 experts, 8
// choices with a bias 32.8 us in two launches (27 and 9 alone), its bytes would take 3.  The
// choice is bound by latency: 256 CTAs keep 27 of an SM's 64 warp slots busy, an instruction
// of a warp takes 11.6 cycles (2.9 in fixed latencies, 1.7 in warp reductions and shuffles,
// 1.5 in loads), and 59 % of the cycles issue one.  Ranking every expert exactly, with a sort
// in each lane, took 31 us where this took 28.
// Dispatch, combine and its gradient of 8191 tokens x 8 x 2048: 47, 48 and 94 us = 6.4, 6.3
// and 6.1 TB/s of a copy's 6.55.
//
// Every result is computed in a fixed order, so it has the same bits on every call: rows
// are numbered by counting bits, never by the order in which atomics arrive.
#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"
#include "ptx.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace moe {

constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 32;          // one choice per lane of the token's warp
constexpr int kMaxTokens = 1 << 20;
constexpr int kRouteThreads = 512;    // at 42 registers, three CTAs an SM
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kMaxChunks = 256;

// Tokens per CTA of the router ("chunk").  Up to 64 tokens are one chunk and one launch.
// More are cut into chunks of 32, or of the least multiple of 32 that makes no more than
// kMaxChunks chunks: one wave of CTAs.
static int chunk_tokens(int T) {
    if (T <= 64) return 64;
    return 32 * ((T + 32 * kMaxChunks - 1) / (32 * kMaxChunks));
}

// Clusters of 8 chunks add their counts up in distributed shared memory, so that the
// second kernel, where every CTA sums all earlier counts, reads at most 32 x E of them and
// not 256 x E (which took it 15 us for 256 experts).
constexpr int kClusterChunks = 8;

struct RouteParams {
    const void *logits;
    const float *bias;
    float *weights;
    int *experts, *rows, *m_offsets;
    int *counts;  // [clusters][E] choices of each expert by cluster of chunks
    int *before;  // [chunks][E] choices in earlier chunks of the same cluster
    int T, E, k, chunk, chunks;
    int sigmoid, renormalize;
    float scale;
};

template <typename T>
__device__ __forceinline__ float to_float(T v) {
    return Type16<T>::load(&v);
}
template <>
__device__ __forceinline__ float to_float<float>(float v) {
    return v;
}

// 1 / (1 + exp(-x)), each step one IEEE operation: the score also ranks the experts when a
// bias is added to it, so its rounding is the plain formula's.
// The reciprocal is the correctly rounded one, so it has the bits of the division.
__device__ __forceinline__ float sigmoid(float x) { return __frcp_rn(__fadd_rn(1.0f, expf(-x))); }

// A number whose signed order is the floats' order (both zeros alike, a NaN at one of the
// ends); kMasked is below every float that is not NaN.
constexpr int kMasked = INT_MIN;
__device__ __forceinline__ int order_key(float v) {
    const int u = __float_as_int(__fadd_rn(v, 0.0f));
    return u ^ ((u >> 31) & 0x7fffffff);
}

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Sorted choice: each lane sorts its own keys once (equal keys stay in the order of their
// experts); every round then takes the highest of the lanes' first keys, the lowest expert
// among equal ones, and the lane that won moves up its next key.  Lane j returns choice j.
template <int NI>
__device__ __forceinline__ int choose_sorted(int (&key)[NI], int k, int lane) {
    int at[NI];  // which of the lane's experts
#pragma unroll
    for (int i = 0; i < NI; i++) at[i] = i;
    // neighbours change places only when the later key is higher: a stable sort
#pragma unroll
    for (int round = 0; round < NI; round++)
#pragma unroll
        for (int i = round & 1; i + 1 < NI; i += 2) {
            const bool swap = key[i + 1] > key[i];
            const int a = key[i], b = key[i + 1], x = at[i], y = at[i + 1];
            key[i] = max(a, b);
            key[i + 1] = min(a, b);
            at[i] = swap ? y : x;
            at[i + 1] = swap ? x : y;
        }
    uint32_t order = 0;  // the sorted places, four bits each
#pragma unroll
    for (int i = 0; i < NI; i++) order |= (uint32_t)at[i] << (4 * i);
    int expert = -1;
    for (int j = 0; j < k; j++) {
        const int top = __reduce_max_sync(0xffffffffu, key[0]);
        if (top == kMasked) break;
        const uint32_t e = key[0] == top ? (uint32_t)lane + 32u * (order & 15u) : 0xffffffffu;
        const uint32_t first = __reduce_min_sync(0xffffffffu, e);
        if (lane == j) expert = (int)first;
        const bool won = e == first;
#pragma unroll
        for (int i = 0; i + 1 < NI; i++) key[i] = won ? key[i + 1] : key[i];
        key[NI - 1] = won ? kMasked : key[NI - 1];
        order = won ? order >> 4 : order;
    }
    return expert;
}

// One warp chooses the experts of token t: lane l holds logits l, l + 32, ...  An expert whose
// logit is -inf or NaN is masked; when only masked ones are left the choice is -1.
//
// Most experts are far from being chosen, and an exact score costs some 40 instructions, so
// the ranks are first taken approximately (fast exponential and reciprocal, within 1e-6 of
// the score).  The k-th highest of the lanes' highest ranks cannot be above the token's k-th
// highest rank; what reaches it, less a margin for both errors, are the candidates.  If they
// are at most one a lane, only they are ranked exactly, one each, in the order of their
// experts, and k rounds of "highest key, lowest lane" choose among them.  Otherwise, and
// where the token has fewer than k experts left, every expert is ranked exactly and sorted.
template <typename T, int NI, bool SIGMOID>
__device__ __forceinline__ int choose(const RouteParams &p, int t, int lane, const float (&bias)[NI], int *slots,
                                      float &weight) {
    const T *l = static_cast<const T *>(p.logits) + (int64_t)t * p.E;
    const bool biased = SIGMOID && p.bias;
    float v[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = lane + 32 * i;
        v[i] = e < p.E ? to_float<T>(l[e]) : -INFINITY;
        if (!(v[i] > -INFINITY)) v[i] = -INFINITY;
    }
    auto exact_key = [&](float x, float b) {
        float rank = x;
        if (biased) rank = __fadd_rn(sigmoid(x > -INFINITY ? x : 0.0f), b);
        const int key = rank == rank ? max(order_key(rank), kMasked + 1) : kMasked + 1;  // a NaN bias ranks last
        return x > -INFINITY ? key : kMasked;
    };
    int expert = -1;
    bool done = false;
    if constexpr (NI > 1) {
        float near[NI], best = -INFINITY;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            near[i] = v[i];
            if (biased) near[i] = v[i] > -INFINITY ? __fdividef(1.0f, 1.0f + __expf(-v[i])) + bias[i] : -INFINITY;
            best = fmaxf(best, near[i]);
        }
        int high = order_key(best), kth = kMasked;
        for (int j = 0; j < p.k; j++) {
            kth = __reduce_max_sync(0xffffffffu, high);
            if (high == kth) high = kMasked;
        }
        float bound = __int_as_float(kth ^ ((kth >> 31) & 0x7fffffff));  // order_key's inverse
        if (biased) bound -= 4e-6f + fabsf(bound) * 0x1p-21f;
        int n = 0;
        uint32_t take = 0;
#pragma unroll
        for (int i = 0; i < NI; i++) take |= (near[i] >= bound && v[i] > -INFINITY ? 1u : 0u) << i;
        n = __reduce_add_sync(0xffffffffu, __popc(take));
        if (kth != kMasked && n >= p.k && n <= 32) {
            int base = 0;
#pragma unroll
            for (int i = 0; i < NI; i++) {  // by expert: i, then lane
                const uint32_t with = __ballot_sync(0xffffffffu, (take >> i) & 1u);
                if ((take >> i) & 1u) slots[base + __popc(with & ((1u << lane) - 1u))] = lane + 32 * i;
                base += __popc(with);
            }
            __syncwarp();
            const int mine = lane < n ? slots[lane] : 0;
            __syncwarp();
            int key = lane < n ? exact_key(to_float<T>(l[mine]), biased ? p.bias[mine] : 0.0f) : kMasked;
            for (int j = 0; j < p.k; j++) {
                const int top = __reduce_max_sync(0xffffffffu, key);
                const int winner = __ffs(__ballot_sync(0xffffffffu, key == top)) - 1;
                const int e = __shfl_sync(0xffffffffu, mine, winner);
                if (lane == j) expert = e;
                if (lane == winner) key = kMasked;
            }
            done = true;
        }
    }
    if (!done) {
        int key[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) key[i] = exact_key(v[i], bias[i]);
        expert = choose_sorted<NI>(key, p.k, lane);
    }
    const float logit = expert >= 0 ? to_float<T>(l[expert]) : -INFINITY;
    float score = 0.0f, total = 1.0f;
    if constexpr (SIGMOID) {
        score = expert >= 0 ? sigmoid(logit) : 0.0f;
        if (p.renormalize) total = warp_sum(score);
    } else {
        float m = v[0];
#pragma unroll
        for (int i = 1; i < NI; i++) m = fmaxf(m, v[i]);
        m = warp_max(m);
        if (m == -INFINITY) m = 0.0f;  // nothing to choose: every exponential is zero
        score = expert >= 0 ? expf(logit - m) : 0.0f;
        if (p.renormalize) {
            total = warp_sum(score);
        } else {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NI; i++) s += expf(v[i] - m);
            total = warp_sum(s);
        }
    }
    weight = expert >= 0 && !(total == 0.0f) ? score / total * p.scale : 0.0f;
    return expert;
}

// Shared memory: the choices of the chunk's tokens as bits, bits[e][word of 32 tokens].
// The row of (token, expert) is the expert's first row, plus its choices in earlier chunks,
// plus the bits set before the token: no order of arrival enters.
__device__ __forceinline__ void number_rows(const RouteParams &p, int t0, int n, int words, const uint32_t *bits,
                                            const int *base) {
    for (int i = threadIdx.x; i < n * p.k; i += kRouteThreads) {
        const int t = i / p.k;
        const int64_t at = (int64_t)t0 * p.k + i;
        const int e = p.experts[at];
        int r = -1;
        if (e >= 0) {
            const uint32_t *b = bits + e * words;
            r = base[e];
            for (int w = 0; w < (t >> 5); w++) r += __popc(b[w]);
            r += __popc(b[t >> 5] & ((1u << (t & 31)) - 1u));
        }
        p.rows[at] = r;
    }
}

// First rows from the experts' totals: one warp scans up to 256 counts.
__device__ __forceinline__ void scan_totals(const int *total, int *first, int E, int lane) {
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
        const int e = e0 + lane, c = e < E ? total[e] : 0;
        int s = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        if (e < E) first[e] = carry + s - c;
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) first[E] = carry;
}

// Choice, one CTA per chunk of tokens.  With a single chunk (a decode step) the same CTA
// numbers the rows too: one launch in all.
template <typename T, int NI, bool SIGMOID>
__global__ void __launch_bounds__(kRouteThreads, 3) moe_route_kernel(const RouteParams p) {
    extern __shared__ uint32_t bits[];  // [E][words]
    __shared__ int total[kMaxExperts], first[kMaxExperts + 1], slots[kRouteWarps][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int words = p.chunk / 32;
    const int t0 = blockIdx.x * p.chunk, n = max(0, min(p.chunk, p.T - t0));
    for (int i = threadIdx.x; i < p.E * words; i += kRouteThreads) bits[i] = 0u;
    __syncthreads();
    float bias[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) bias[i] = p.bias && lane + 32 * i < p.E ? p.bias[lane + 32 * i] : 0.0f;
    for (int t = warp; t < n; t += kRouteWarps) {
        float w;
        const int e = choose<T, NI, SIGMOID>(p, t0 + t, lane, bias, slots[warp], w);
        if (lane < p.k) {
            const int64_t at = (int64_t)(t0 + t) * p.k + lane;
            p.weights[at] = w;
            p.experts[at] = e;
            if (e >= 0) atomicOr(&bits[e * words + (t >> 5)], 1u << (t & 31));
        }
    }
    __syncthreads();
    for (int e = warp; e < p.E; e += kRouteWarps) {
        int c = 0;
        for (int w = lane; w < words; w += 32) c += __popc(bits[e * words + w]);
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) total[e] = c;
    }
    if (p.chunks > 1) {
        __syncwarp();  // barrier.cluster is .aligned
        cluster_sync();
        const int rank = blockIdx.x % kClusterChunks, cluster = blockIdx.x / kClusterChunks;
        const int per = (p.E + kClusterChunks - 1) / kClusterChunks;  // this CTA's experts
        if ((int)threadIdx.x < per && rank * per + (int)threadIdx.x < p.E) {
            const int e = rank * per + threadIdx.x;
            int c[kClusterChunks], sum = 0;
#pragma unroll
            for (int q = 0; q < kClusterChunks; q++) c[q] = ld_cluster_s32(map_to_cta(smem_u32(&total[e]), q));
#pragma unroll
            for (int q = 0; q < kClusterChunks; q++) {
                p.before[(int64_t)(cluster * kClusterChunks + q) * p.E + e] = sum;
                sum += c[q];
            }
            p.counts[(int64_t)cluster * p.E + e] = sum;
        }
        __syncwarp();
        cluster_sync();  // the others may still read this CTA's counts
        return;
    }
    __syncthreads();
    if (warp == 0) scan_totals(total, first, p.E, lane);
    __syncthreads();
    for (int e = threadIdx.x; e <= p.E; e += kRouteThreads) p.m_offsets[e] = first[e];
    number_rows(p, t0, n, words, bits, first);
}

// Rows of every chunk, once all counts are known: each CTA adds up the clusters' counts (at
// most 32 x 256 numbers out of L2), so no grid-wide scan is needed between the launches.
__global__ void __launch_bounds__(kRouteThreads) moe_rows_kernel(const RouteParams p) {
    extern __shared__ uint32_t bits[];  // [E][words]
    __shared__ int part_total[kRouteThreads], part_before[kRouteThreads];
    __shared__ int total[kMaxExperts], base[kMaxExperts + 1];
    const int words = p.chunk / 32;
    const int t0 = blockIdx.x * p.chunk, n = min(p.chunk, p.T - t0);
    for (int i = threadIdx.x; i < p.E * words; i += kRouteThreads) bits[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n * p.k; i += kRouteThreads) {
        const int e = p.experts[(int64_t)t0 * p.k + i], t = i / p.k;
        if (e >= 0) atomicOr(&bits[e * words + (t >> 5)], 1u << (t & 31));
    }
    const int parts = kRouteThreads / p.E;  // at least two threads an expert
    const int clusters = (p.chunks + kClusterChunks - 1) / kClusterChunks, own = blockIdx.x / kClusterChunks;
    const int e = threadIdx.x % p.E, part = threadIdx.x / p.E;
    int all = 0, before = 0;
    if (part < parts)
#pragma unroll 16
        for (int c = part; c < clusters; c += parts) {
            const int v = p.counts[(int64_t)c * p.E + e];
            all += v;
            if (c < own) before += v;
        }
    if (part == 0) before += p.before[(int64_t)blockIdx.x * p.E + e];
    part_total[threadIdx.x] = all;
    part_before[threadIdx.x] = before;
    __syncthreads();
    if (threadIdx.x < p.E) {
        int a = 0;
        for (int q = 0; q < parts; q++) a += part_total[q * p.E + threadIdx.x];
        total[threadIdx.x] = a;
    }
    __syncthreads();
    if (threadIdx.x < 32) scan_totals(total, base, p.E, threadIdx.x);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= p.E; i += kRouteThreads) p.m_offsets[i] = base[i];
    __syncthreads();
    if (threadIdx.x < p.E) {
        int b = base[threadIdx.x];
        for (int q = 0; q < parts; q++) b += part_before[q * p.E + threadIdx.x];
        base[threadIdx.x] = b;
    }
    __syncthreads();
    number_rows(p, t0, n, words, bits, base);
}

// Gradient of the logits, one warp a token.  With p the scores, c the chosen experts and
// d_j = scale * dweight_j:
//   renormalised:  ds_j = (d_j - sum_i q_i d_i) / S,  q = p / S, S = sum of the chosen p
//   softmax:       dl_e = p_e (ds_e - sum_i p_i ds_i)    (ds_e = 0 for experts not chosen)
//   sigmoid:       dl_e = ds_e p_e (1 - p_e)
// Renormalised softmax needs no sum over all experts: the chosen ones' share p_j / S is the
// softmax over them alone, and dl_j = q_j (d_j - sum_i q_i d_i).
template <typename T, int NI>
__global__ void __launch_bounds__(256) moe_route_backward_kernel(const T *logits, const float *dweights,
                                                                 const int *experts, T *dlogits, int n_tokens, int E,
                                                                 int k, int use_sigmoid, int renormalize, float scale) {
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= n_tokens) return;
    const T *l = logits + (int64_t)t * E;
    float v[NI], g[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = lane + 32 * i;
        v[i] = e < E ? to_float<T>(l[e]) : -INFINITY;
        if (!(v[i] > -INFINITY)) v[i] = -INFINITY;
        g[i] = 0.0f;
    }
    int expert = -1;
    float d = 0.0f, lv = -INFINITY;
    if (lane < k) {
        expert = experts[(int64_t)t * k + lane];
        if (expert >= E) expert = -1;
        if (expert >= 0) {
            d = dweights[(int64_t)t * k + lane] * scale;
            lv = to_float<T>(l[expert]);
        }
    }
    float mine = 0.0f;  // lane j: the gradient of choice j's logit (softmax without renormalising: ds_j)
    float m = 0.0f, total = 1.0f, dot = 0.0f;
    if (use_sigmoid) {
        const float s = expert >= 0 ? sigmoid(lv) : 0.0f;
        float ds = d;
        if (renormalize) {
            total = warp_sum(s);
            const float q = total > 0.0f ? s / total : 0.0f;
            dot = warp_sum(q * d);
            ds = total > 0.0f ? (d - dot) / total : 0.0f;
        }
        mine = expert >= 0 ? ds * s * (1.0f - s) : 0.0f;
    } else {
        m = v[0];
#pragma unroll
        for (int i = 1; i < NI; i++) m = fmaxf(m, v[i]);
        m = warp_max(m);
        if (m == -INFINITY) m = 0.0f;
        const float s = expert >= 0 ? expf(lv - m) : 0.0f;
        if (renormalize) {
            total = warp_sum(s);
        } else {
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < NI; i++) z += expf(v[i] - m);
            total = warp_sum(z);
        }
        const float q = total > 0.0f ? s / total : 0.0f;
        dot = warp_sum(q * d);
        mine = renormalize ? q * (d - dot) : d;
    }
    for (int j = 0; j < k; j++) {
        const int e = __shfl_sync(0xffffffffu, expert, j);
        const float x = __shfl_sync(0xffffffffu, mine, j);
#pragma unroll
        for (int i = 0; i < NI; i++)
            if (e == lane + 32 * i) g[i] = x;
    }
    T *dl = dlogits + (int64_t)t * E;
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = lane + 32 * i;
        float x = g[i];
        if (!use_sigmoid && !renormalize) {
            const float q = total > 0.0f ? expf(v[i] - m) / total : 0.0f;
            x = q * (x - dot);
        }
        if (e < E) {
            if constexpr (sizeof(T) == 4)
                dl[e] = x;
            else
                dl[e] = Type16<T>::round(x);
        }
    }
}

// ---------------------------------------------------------------------------------------
// Movement of rows.  All of it is bound by memory: 16 bytes a thread, the loads of a token's
// rows issued together, sums in fp32 in the order of the choices.
// ---------------------------------------------------------------------------------------
constexpr int kMoveThreads = 256;

// Threads of one token's row: whole warps, up to the CTA.  Rows narrower than the CTA share
// it between tokens; wider ones take several CTAs ("slabs").
struct MoveShape {
    int vecs;     // 16-byte vectors of a row
    int lanes;    // threads per token and slab
    int tokens;   // tokens per CTA
    int slabs;    // CTAs per row
};
static MoveShape move_shape(int K) {
    MoveShape s;
    s.vecs = K / 8;
    s.lanes = std::min(kMoveThreads, (s.vecs + 31) / 32 * 32);
    s.tokens = kMoveThreads / s.lanes;
    s.slabs = (s.vecs + s.lanes - 1) / s.lanes;
    return s;
}

struct MoveParams {
    const uint4 *x;         // dispatch: token rows; combine: expert rows
    const uint4 *dy;        // combine backward
    const uint4 *residual;  // combine, may be null
    uint4 *out;
    const int *rows;        // [T, k]
    const float *weights;   // [T, k], null: all ones
    const int *m_offsets;   // [E + 1]
    float *dweights;        // [T, k]
    int T, k, E;
    MoveShape s;
};

// Rows that no choice owns (there are some when tokens were masked) are zeroed.
__device__ __forceinline__ void zero_spare_rows(const MoveParams &p) {
    const int total = p.T * p.k;
    const int used = min(max(p.m_offsets[p.E], 0), total);
    for (int64_t r = used + (int64_t)blockIdx.x; r < total; r += gridDim.x)
        for (int c = threadIdx.x; c < p.s.vecs; c += kMoveThreads)
            p.out[r * p.s.vecs + c] = make_uint4(0u, 0u, 0u, 0u);
}

__global__ void __launch_bounds__(kMoveThreads) moe_dispatch_kernel(const MoveParams p) {
    const int slab = blockIdx.x % p.s.slabs, block = blockIdx.x / p.s.slabs;
    const int in_cta = threadIdx.x / p.s.lanes;
    const int64_t t = (int64_t)block * p.s.tokens + in_cta;
    const int c = slab * p.s.lanes + threadIdx.x - in_cta * p.s.lanes;
    const int total = p.T * p.k;
    if (in_cta < p.s.tokens && t < p.T && c < p.s.vecs) {
        const uint4 v = p.x[t * p.s.vecs + c];
        for (int j = 0; j < p.k; j++) {
            const int r = p.rows[t * p.k + j];
            if (r >= 0 && r < total) p.out[(int64_t)r * p.s.vecs + c] = v;
        }
    }
    zero_spare_rows(p);
}

template <typename T>
__global__ void __launch_bounds__(kMoveThreads) moe_combine_kernel(const MoveParams p) {
    const int slab = blockIdx.x % p.s.slabs, block = blockIdx.x / p.s.slabs;
    const int in_cta = threadIdx.x / p.s.lanes;
    const int64_t t = (int64_t)block * p.s.tokens + in_cta;
    const int c = slab * p.s.lanes + threadIdx.x - in_cta * p.s.lanes;
    if (in_cta >= p.s.tokens || t >= p.T || c >= p.s.vecs) return;
    const int total = p.T * p.k;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    uint4 res = make_uint4(0u, 0u, 0u, 0u);
    if (p.residual) res = p.residual[t * p.s.vecs + c];
    for (int j0 = 0; j0 < p.k; j0 += 4) {
        uint4 v[4];
        float w[4];
        bool live[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = j0 + j < p.k ? p.rows[t * p.k + j0 + j] : -1;
            live[j] = r >= 0 && r < total;
            v[j] = make_uint4(0u, 0u, 0u, 0u);
            w[j] = 0.0f;
            if (live[j]) {
                v[j] = p.x[(int64_t)r * p.s.vecs + c];
                w[j] = p.weights ? p.weights[t * p.k + j0 + j] : 1.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (live[j]) {
                float f[8];
                unpack8<T>(v[j], f);
#pragma unroll
                for (int i = 0; i < 8; i++) acc[i] = fmaf(w[j], f[i], acc[i]);
            }
    }
    if (p.residual) {
        float f[8];
        unpack8<T>(res, f);
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] += f[i];
    }
    p.out[t * p.s.vecs + c] = pack8<T>(acc);
}

// drows[r] = w dy and dweight = <rows[r], dy>: the CTA's threads of a token walk its row
// together (every slab), then their dot products are summed in a fixed tree.
template <typename T>
__global__ void __launch_bounds__(kMoveThreads) moe_combine_backward_kernel(const MoveParams p) {
    __shared__ float part[kMoveThreads / 32][4];
    const int in_cta = threadIdx.x / p.s.lanes, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * p.s.tokens + in_cta;
    const bool on = in_cta < p.s.tokens && t < p.T;
    const int c0 = threadIdx.x - in_cta * p.s.lanes;
    const int total = p.T * p.k, warps = p.s.lanes / 32;
    for (int j0 = 0; j0 < p.k; j0 += 4) {
        float dot[4] = {0.f, 0.f, 0.f, 0.f}, w[4];
        int64_t at[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = on && j0 + j < p.k ? p.rows[t * p.k + j0 + j] : -1;
            at[j] = r >= 0 && r < total ? (int64_t)r * p.s.vecs : -1;
            w[j] = at[j] >= 0 ? p.weights[t * p.k + j0 + j] : 0.0f;
        }
        if (on)
            for (int c = c0; c < p.s.vecs; c += p.s.lanes) {
                const uint4 raw = p.dy[t * p.s.vecs + c];
                uint4 v[4];
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = at[j] >= 0 ? p.x[at[j] + c] : make_uint4(0u, 0u, 0u, 0u);
                float g[8];
                unpack8<T>(raw, g);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (at[j] >= 0) {
                        float f[8], o[8];
                        unpack8<T>(v[j], f);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            dot[j] = fmaf(f[i], g[i], dot[j]);
                            o[i] = w[j] * g[i];
                        }
                        p.out[at[j] + c] = pack8<T>(o);
                    }
            }
#pragma unroll
        for (int j = 0; j < 4; j++) dot[j] = warp_sum(dot[j]);
        __syncthreads();  // the previous round's sums have been read
        if (lane == 0)
#pragma unroll
            for (int j = 0; j < 4; j++) part[warp][j] = dot[j];
        __syncthreads();
        if (on && c0 < 4 && j0 + c0 < p.k) {
            float s = 0.0f;
            for (int q = 0; q < warps; q++) s += part[in_cta * warps + q][c0];
            p.dweights[t * p.k + j0 + c0] = s;
        }
    }
    zero_spare_rows(p);
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
template <typename Kernel, typename... Args>
static int launch(Kernel kern, int grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    kern<<<grid, threads, smem, stream>>>(args...);
    count_launch();
    return cuda_status(cudaGetLastError());
}

template <typename Kernel, typename... Args>
static int launch_cluster(Kernel kern, int cluster, int grid, int threads, size_t smem, cudaStream_t stream,
                          Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return NVFP4_ERR_CUDA;
    count_launch();
    return cuda_status(cudaGetLastError());
}

// The bits of the largest chunk.  The limit is set once per kernel and device, to this size:
// it is shared by all threads, so a call that set its own could lower it under another's
// launch.
constexpr int kMaxBitBytes = kMaxExperts * (kMaxTokens / kMaxChunks / 32) * 4;
template <typename Kernel>
static int allow_bits(Kernel kern, std::atomic<bool> *configured) {
    DeviceInfo di;
    int st = device_info(&di);
    if (st) return st;
    if (configured[di.device]) return NVFP4_OK;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBitBytes) != cudaSuccess)
        return NVFP4_ERR_CUDA;
    configured[di.device] = true;
    return NVFP4_OK;
}

template <typename T, int NI, bool SIGMOID>
static int route_t(const RouteParams &p, cudaStream_t s) {
    auto kern = moe_route_kernel<T, NI, SIGMOID>;
    const size_t smem = (size_t)p.E * (p.chunk / 32) * 4;
    static std::atomic<bool> configured[64] = {}, configured_rows[64] = {};
    int st = smem > 32768 ? allow_bits(kern, configured) : NVFP4_OK;
    if (!st && smem > 32768) st = allow_bits(moe_rows_kernel, configured_rows);
    if (st) return st;
    if (p.chunks == 1) return launch(kern, 1, kRouteThreads, smem, s, p);
    const int grid = (p.chunks + kClusterChunks - 1) / kClusterChunks * kClusterChunks;
    st = launch_cluster(kern, kClusterChunks, grid, kRouteThreads, smem, s, p);
    if (st) return st;
    return launch(moe_rows_kernel, p.chunks, kRouteThreads, smem, s, p);
}

template <typename T, bool SIGMOID>
static int route_e(const RouteParams &p, cudaStream_t s) {
    if (p.E <= 32) return route_t<T, 1, SIGMOID>(p, s);
    if (p.E <= 64) return route_t<T, 2, SIGMOID>(p, s);
    if (p.E <= 128) return route_t<T, 4, SIGMOID>(p, s);
    return route_t<T, 8, SIGMOID>(p, s);
}

template <typename T>
static int route(const RouteParams &p, cudaStream_t s) {
    return p.sigmoid ? route_e<T, true>(p, s) : route_e<T, false>(p, s);
}

template <typename T, int NI>
static int route_backward_t(const void *logits, const float *dw, const int *experts, void *dl, int n, int E, int k,
                            int sg, int rn, float scale, cudaStream_t s) {
    return launch(moe_route_backward_kernel<T, NI>, (n + 7) / 8, 256, 0, s, static_cast<const T *>(logits), dw, experts,
        static_cast<T *>(dl), n, E, k, sg, rn, scale);
}

template <typename T>
static int route_backward(const void *logits, const float *dw, const int *experts, void *dl, int n, int E, int k,
                          int sg, int rn, float scale, cudaStream_t s) {
    if (E <= 32) return route_backward_t<T, 1>(logits, dw, experts, dl, n, E, k, sg, rn, scale, s);
    if (E <= 64) return route_backward_t<T, 2>(logits, dw, experts, dl, n, E, k, sg, rn, scale, s);
    if (E <= 128) return route_backward_t<T, 4>(logits, dw, experts, dl, n, E, k, sg, rn, scale, s);
    return route_backward_t<T, 8>(logits, dw, experts, dl, n, E, k, sg, rn, scale, s);
}

static bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Sizes that dispatch, combine and their gradients share.
static int move_sizes(int T, int k, int K) {
    if (T < 0 || T > kMaxTokens || k < 1 || k > kMaxTopK || K < 8 || K % 8) return NVFP4_ERR_SHAPE;
    if ((int64_t)T * k > INT_MAX) return NVFP4_ERR_SHAPE;
    const MoveShape s = move_shape(K);
    if ((int64_t)((T + s.tokens - 1) / s.tokens) * s.slabs > INT_MAX) return NVFP4_ERR_SHAPE;
    return NVFP4_OK;
}

}  // namespace moe
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

size_t nvfp4_moe_route_workspace_size(int T, int E) {
    if (T < 0 || T > moe::kMaxTokens || E < 1 || E > moe::kMaxExperts) return 0;
    const int c = moe::chunk_tokens(T), chunks = std::max(1, (T + c - 1) / c);
    const int clusters = (chunks + moe::kClusterChunks - 1) / moe::kClusterChunks;
    return (size_t)clusters * (moe::kClusterChunks + 1) * E * sizeof(int);
}

int nvfp4_moe_route(const void *logits, int dtype, const float *bias, int T, int E, int top_k, int scoring,
                    int renormalize, float scale, float *weights, int32_t *experts, int32_t *rows, int32_t *m_offsets,
                    void *workspace, size_t workspace_bytes, void *stream) {
    if (dtype < NVFP4_BF16 || dtype > NVFP4_F32 || scoring < NVFP4_SCORE_SOFTMAX || scoring > NVFP4_SCORE_SIGMOID)
        return NVFP4_ERR_INVALID;
    if (T < 0 || T > moe::kMaxTokens || E < 1 || E > moe::kMaxExperts || top_k < 1 || top_k > moe::kMaxTopK ||
        top_k > E)
        return NVFP4_ERR_SHAPE;
    if (!m_offsets || (T && (!logits || !weights || !experts || !rows))) return NVFP4_ERR_INVALID;
    if (bias && scoring != NVFP4_SCORE_SIGMOID) return NVFP4_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(logits) & (dtype == NVFP4_F32 ? 3u : 1u)) || !moe::aligned4(bias) ||
        !moe::aligned4(weights) || !moe::aligned4(experts) || !moe::aligned4(rows) || !moe::aligned4(m_offsets) ||
        !moe::aligned4(workspace))
        return NVFP4_ERR_ALIGN;
    moe::RouteParams p;
    p.chunk = moe::chunk_tokens(T);
    p.chunks = std::max(1, (T + p.chunk - 1) / p.chunk);
    if (p.chunks > 1 && (!workspace || workspace_bytes < nvfp4_moe_route_workspace_size(T, E)))
        return NVFP4_ERR_WORKSPACE;
    DeviceInfo di;
    int st = device_info(&di);
    if (st) return st;
    p.logits = logits;
    p.bias = bias;
    p.weights = weights;
    p.experts = experts;
    p.rows = rows;
    p.m_offsets = m_offsets;
    p.counts = static_cast<int *>(workspace);
    p.before = p.counts + (int64_t)((p.chunks + moe::kClusterChunks - 1) / moe::kClusterChunks) * E;
    p.T = T;
    p.E = E;
    p.k = top_k;
    p.sigmoid = scoring == NVFP4_SCORE_SIGMOID;
    p.renormalize = renormalize != 0;
    p.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16) return moe::route<__nv_bfloat16>(p, s);
    if (dtype == NVFP4_F16) return moe::route<__half>(p, s);
    return moe::route<float>(p, s);
}

int nvfp4_moe_route_backward(const float *dweights, const void *logits, int dtype, const int32_t *experts, int T,
                             int E, int top_k, int scoring, int renormalize, float scale, void *dlogits,
                             void *stream) {
    if (dtype < NVFP4_BF16 || dtype > NVFP4_F32 || scoring < NVFP4_SCORE_SOFTMAX || scoring > NVFP4_SCORE_SIGMOID)
        return NVFP4_ERR_INVALID;
    if (T < 0 || T > moe::kMaxTokens || E < 1 || E > moe::kMaxExperts || top_k < 1 || top_k > moe::kMaxTopK ||
        top_k > E)
        return NVFP4_ERR_SHAPE;
    if (T && (!logits || !dweights || !experts || !dlogits)) return NVFP4_ERR_INVALID;
    const uintptr_t mask = dtype == NVFP4_F32 ? 3u : 1u;
    if ((reinterpret_cast<uintptr_t>(logits) & mask) || (reinterpret_cast<uintptr_t>(dlogits) & mask) ||
        !moe::aligned4(dweights) || !moe::aligned4(experts))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    int st = device_info(&di);
    if (st) return st;
    if (T == 0) return NVFP4_OK;
    const int sg = scoring == NVFP4_SCORE_SIGMOID, rn = renormalize != 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == NVFP4_BF16)
        return moe::route_backward<__nv_bfloat16>(logits, dweights, experts, dlogits, T, E, top_k, sg, rn, scale, s);
    if (dtype == NVFP4_F16)
        return moe::route_backward<__half>(logits, dweights, experts, dlogits, T, E, top_k, sg, rn, scale, s);
    return moe::route_backward<float>(logits, dweights, experts, dlogits, T, E, top_k, sg, rn, scale, s);
}

int nvfp4_moe_dispatch(const void *X, const int32_t *rows, const int32_t *m_offsets, int T, int E, int top_k, int K,
                       void *X_rows, void *stream) {
    if (E < 1 || E > moe::kMaxExperts) return NVFP4_ERR_SHAPE;
    int st = moe::move_sizes(T, top_k, K);
    if (st) return st;
    if (T && (!X || !rows || !m_offsets || !X_rows)) return NVFP4_ERR_INVALID;
    if (!aligned16(X) || !aligned16(X_rows) || !moe::aligned4(rows) || !moe::aligned4(m_offsets))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    moe::MoveParams p = {};
    p.x = static_cast<const uint4 *>(X);
    p.out = static_cast<uint4 *>(X_rows);
    p.rows = rows;
    p.m_offsets = m_offsets;
    p.T = T;
    p.k = top_k;
    p.E = E;
    p.s = moe::move_shape(K);
    return moe::launch(moe::moe_dispatch_kernel, (T + p.s.tokens - 1) / p.s.tokens * p.s.slabs,
                                        moe::kMoveThreads, 0, static_cast<cudaStream_t>(stream), p);
}

int nvfp4_moe_combine(const void *X_rows, int dtype, const int32_t *rows, const float *weights, const void *residual,
                      int T, int top_k, int K, void *Y, void *stream) {
    if (dtype != NVFP4_BF16 && dtype != NVFP4_F16) return NVFP4_ERR_INVALID;
    int st = moe::move_sizes(T, top_k, K);
    if (st) return st;
    if (T && (!X_rows || !rows || !Y)) return NVFP4_ERR_INVALID;
    if (!aligned16(X_rows) || !aligned16(Y) || !aligned16(residual) || !moe::aligned4(rows) || !moe::aligned4(weights))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    moe::MoveParams p = {};
    p.x = static_cast<const uint4 *>(X_rows);
    p.out = static_cast<uint4 *>(Y);
    p.residual = static_cast<const uint4 *>(residual);
    p.rows = rows;
    p.weights = weights;
    p.T = T;
    p.k = top_k;
    p.s = moe::move_shape(K);
    const int grid = (T + p.s.tokens - 1) / p.s.tokens * p.s.slabs;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == NVFP4_BF16
               ? moe::launch(moe::moe_combine_kernel<__nv_bfloat16>, grid, moe::kMoveThreads, 0, s, p)
               : moe::launch(moe::moe_combine_kernel<__half>, grid, moe::kMoveThreads, 0, s, p);
}

int nvfp4_moe_combine_backward(const void *dY, const void *X_rows, int dtype, const int32_t *rows,
                               const float *weights, const int32_t *m_offsets, int T, int E, int top_k, int K,
                               void *dX_rows, float *dweights, void *stream) {
    if (dtype != NVFP4_BF16 && dtype != NVFP4_F16) return NVFP4_ERR_INVALID;
    if (E < 1 || E > moe::kMaxExperts) return NVFP4_ERR_SHAPE;
    int st = moe::move_sizes(T, top_k, K);
    if (st) return st;
    if (T && (!dY || !X_rows || !rows || !weights || !m_offsets || !dX_rows || !dweights)) return NVFP4_ERR_INVALID;
    if (!aligned16(dY) || !aligned16(X_rows) || !aligned16(dX_rows) || !moe::aligned4(rows) ||
        !moe::aligned4(weights) || !moe::aligned4(m_offsets) || !moe::aligned4(dweights))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (T == 0) return NVFP4_OK;
    moe::MoveParams p = {};
    p.x = static_cast<const uint4 *>(X_rows);
    p.dy = static_cast<const uint4 *>(dY);
    p.out = static_cast<uint4 *>(dX_rows);
    p.rows = rows;
    p.weights = weights;
    p.m_offsets = m_offsets;
    p.dweights = dweights;
    p.T = T;
    p.k = top_k;
    p.E = E;
    p.s = moe::move_shape(K);
    const int grid = (T + p.s.tokens - 1) / p.s.tokens;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == NVFP4_BF16 ? moe::launch(moe::moe_combine_backward_kernel<__nv_bfloat16>, grid,
                                                              moe::kMoveThreads, 0, s, p)
                               : moe::launch(moe::moe_combine_backward_kernel<__half>, grid,
                                                              moe::kMoveThreads, 0, s, p);
}

}  // extern "C"
