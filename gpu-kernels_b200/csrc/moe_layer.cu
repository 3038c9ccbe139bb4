// moe_layer.cu — a whole mixture-of-experts layer for the few tokens of a decode step, bound
// by streaming the chosen experts' weights once.
//
//   y[t] = residual[t] + sum_j w[t, j] W2_e ( silu(W1_e x[t]) * (W3_e x[t]) ),  e = e(t, j)
//
// Several rows an expert are another file's (streamed(), below).  Here there are two launches:
// the router (moe.cu, which also clears this kernel's counters), and one
// cooperative kernel for the experts and the weighted sum, where six kernels and their gaps
// took longer than the weights of small experts do.
//
// The work is a list of units of 16 weight rows: first all of W13 (8 gate rows with their 8 up
// rows, so SwiGLU stays in a thread), then all of W2, each by active expert; experts without a
// token are not in it, and one with more than 16 has each unit once for every 16 rows, side by
// side, so that the weights come from memory once.  CTAs take the units in turn.  A W2 unit
// waits for its expert's hidden rows alone (a counter an expert), not for the grid.  The rows'
// results are left in fp32, and the warp that brings a block of 16 columns its last part forms
// the weighted sum there, in the order of the choices: the same bits every time.
//
// Warps: 0-7 multiply, 8 watches the hidden rows' counters, 9-14 add the parts up and hand them
// on, a unit each in turn (the stores and the counter of one unit take 5 us under load, longer
// than the weights of a short one).  A stage is 512 elements of 16 weight rows.  Each
// multiplying warp has one of its own: when it has read its stage it copies the next weights
// there itself, one tensor copy, and brings the tokens' (hidden) rows by cp.async while they
// are on their way, so its latencies run under the other warps' stages and nothing is handed
// from warp to warp but sums.  The weights run on into W2 while its hidden rows are still being
// made.  For each chunk of 32 elements lanes 4g .. 4g + 3 read 64 bytes of row g, which is
// mma.m16n8k16's A fragment with the chunk's elements permuted, and the tokens are read with
// the same permutation, so nothing is shuffled.  The products are tiny (8 token columns a
// tile); the tensor core only has to keep up with memory.
//
// The weights are seen as [block of 64 elements][row][64] so that a box is eight whole swizzled
// tiles of 8 rows by 128 bytes for each half of the rows.  Elements past the last whole block
// come beside the last stage's blocks, from a second view that knows the row's end.
//
// Measured, both launches, on the GPU: one token by 2 of 8 experts of 4096 x 14336 112 us (6.3
// TB/s), 8 tokens by 6 of 64 of 2048 x 2048 124 us (6.3), 13 by 6 of 64 of 2056 x 1408, whose
// rows begin anywhere in a 128-byte line, 132 to 139 us (5.4), one by 8 of 128 of 2048 x 768 28 us:
// there it is bound by the router's launch (5 us), the first weights (3.5), the way from the
// last W13 weights to the last hidden rows (4.5) and from the last W2 weights to the sum (4.5).
//
// On the way, the first two of these: pieces of 16 bytes by cp.async 3.6 TB/s whatever the
// depth; a bulk copy for each of the 16 rows 2.8 and 2.8 (82 cycles to issue one); every warp a
// part of each stage 4.4 and 3.9; tokens by bulk copies of another warp, which then came after
// the weights, 4.6 and 3.5; all weights copied by one lane, 0.4 us a stage, 5.5 and 5.4; stages
// described by a warp of their own, 500 cycles each, 6.2 and 6.3 but 4.6 instead of 5.8 for 256
// experts of 2048 x 768.
#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"
#include "linear.cuh"
#include "moe.cuh"
#include "moe_products.cuh"
#include "ptx.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace moe_layer {

constexpr int kWarps = 8;                  // that multiply, at most: one a stage
constexpr int kMaxTiles = 2;               // of 8 token columns
constexpr int kSets = 4;                   // of parts
constexpr int kEpiWarps = 6;               // that add them up
constexpr int kWatchWarp = kWarps, kEpiWarp = kWarps + 1;
constexpr int kThreads = 32 * (kEpiWarp + kEpiWarps);
constexpr int kMaxRows = 8 * kMaxTiles;    // of a unit
constexpr int kMaxTokens = 64;             // one launch of the router
constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 32;
constexpr int kMaxSize = 1 << 20;          // of K and F
constexpr int kSegment = 512;              // elements of a row in a stage
constexpr int kBlocks = kSegment / 64;
constexpr int kBlockBytes = 16 * 128;      // 64 elements of 16 rows
constexpr int kTokenRows = 8;              // of a stage: a second tile's rows take the first one's place
constexpr int kMaxStages = kWarps;
constexpr int kSmem = 228 * 1000;          // ring, parts, a row of zeros, the choices; the tables are static

struct Params {
    const void *x, *w13, *w2, *residual;
    void *y;
    int64_t ldx;
    const float *weights;      // [T, k]
    const int *rows;           // [T, k]
    const int *m_offsets;      // [E + 1]
    int *up_done;              // [E] finished units of an expert's hidden rows
    int *col_done;             // [column blocks] finished units
    void *h;                   // [T k, hp]
    float *part;               // [T k, K]
    int T, E, k, K, F, hp;
    int stages, stage_bytes;   // of the ring
    int tail;                  // a stage has room for a block past its eight
    int pitch;                 // bytes between token rows: eight lanes read different banks
    KernelCtl ctl;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *tmap, uint32_t bar, int32_t x, int32_t y,
                                            int32_t z, int32_t w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
// A counter in shared memory that only goes up, and the bounded wait for it to reach `want`.
__device__ __forceinline__ void count_release(int *c, int n) {
    asm volatile("red.release.cta.shared::cta.add.s32 [%0], %1;" ::"r"(smem_u32(c)), "r"(n) : "memory");
}
__device__ __forceinline__ bool count_reached(const int *c, int want) {
    int v;
    asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(c)) : "memory");
    return v - want >= 0;
}
__device__ __forceinline__ bool count_wait(const int *c, int want, uint64_t timeout_ns, volatile int *abort) {
    if (count_reached(c, want)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t i = 1;; i++) {
        if (count_reached(c, want)) return true;
        if ((i & 63) == 0 && (*abort || global_timer_ns() - t0 > timeout_ns)) return false;
    }
}
__device__ __forceinline__ bool warp_count_wait(const int *c, int want, uint64_t timeout_ns, volatile int *abort,
                                                int lane) {
    int ok = 1;
    if (lane == 0) ok = count_wait(c, want, timeout_ns, abort);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();  // what lane 0 has acquired, for all
    return ok != 0;
}
__device__ __forceinline__ void add_release(int *p) {
    asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(p) : "memory");
}
__device__ __forceinline__ int add_acquire_release(int *p) {
    int v;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int load_acquire(const int *p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// What a unit is, and a stage of it.
struct Unit {
    bool up;                       // of W13
    int a, idx, n, row0;           // active expert, its unit, the rows that take part and the first one
};
struct Stage {
    Unit unit;
    int number;                    // of the unit, among the CTA's
    int row, block, blocks, rest;  // weight: row, first block of 64 elements, whole blocks, elements past them
    bool first, last;              // the warp's first and last stage in the unit
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    moe_layer_kernel(const __grid_constant__ CUtensorMap map13, const __grid_constant__ CUtensorMap tail13,
                     const __grid_constant__ CUtensorMap map2, const __grid_constant__ CUtensorMap tail2, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
    __shared__ short act_e[kMaxExperts], act_row[kMaxExperts], act_n[kMaxExperts];
    __shared__ int n_active, n_groups;  // experts, and sixteens of their rows
    __shared__ short act_g[kMaxExperts + 1];  // sixteens of rows before
    __shared__ uint64_t bars[kMaxStages];
    __shared__ int parted[kSets], taken[kSets], hidden;  // counters
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;  // fragment row / column, and quarter of 32 elements
    const uint32_t bar_full = smem_u32(bars);

    // shared memory: the ring, the parts [set][warp][tile][lane], a row of zeros, the choices
    const int tiles_cap = min(kMaxTiles, (p.T + 7) / 8), choices = p.T * p.k;
    float4 *sums = reinterpret_cast<float4 *>(smem + p.stages * p.stage_bytes);
    uint8_t *zeros = reinterpret_cast<uint8_t *>(sums + kSets * kWarps * tiles_cap * 32);
    float *choice_weight = reinterpret_cast<float *>(zeros + p.pitch);
    int16_t *choice_row = reinterpret_cast<int16_t *>(choice_weight + choices);
    uint16_t *row_token = reinterpret_cast<uint16_t *>(choice_row + choices);

    // ---- active experts and the rows' tokens
    if (threadIdx.x == 0) {
        prefetch_tmap(&map13);
        prefetch_tmap(&map2);
        abort_word = 0;
        for (int i = 0; i < p.stages; i++) mbar_init(bar_full + 8 * i, 1);
        for (int i = 0; i < kSets; i++) parted[i] = taken[i] = 0;
        hidden = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        int at[kMaxExperts / 32 + 1];  // row offsets of experts lane, lane + 32, ...
#pragma unroll
        for (int i = 0; i < kMaxExperts / 32; i++) at[i] = p.m_offsets[min(i * 32 + lane, p.E)];
        at[kMaxExperts / 32] = p.m_offsets[p.E];
        int n = 0, sixteens = 0;
#pragma unroll
        for (int i = 0; i < kMaxExperts / 32; i++) {
            int end = __shfl_down_sync(0xffffffffu, at[i], 1);
            const int next = __shfl_sync(0xffffffffu, at[i + 1], 0);
            if (lane == 31) end = next;
            const uint32_t live = __ballot_sync(0xffffffffu, end > at[i]);
            if (end > at[i]) {
                const int slot = n + __popc(live & ((1u << lane) - 1u));
                act_e[slot] = (short)(i * 32 + lane);
                act_row[slot] = (short)at[i];
                act_n[slot] = (short)(end - at[i]);
            }
            const int own = (end - at[i] + kMaxRows - 1) / kMaxRows;
            int upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            if (own) act_g[n + __popc(live & ((1u << lane) - 1u)) + 1] = (short)(sixteens + upto);
            n += __popc(live);
            sixteens += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) {
            n_active = n;
            n_groups = sixteens;
            act_g[0] = 0;
        }
    } else {
        for (int i = threadIdx.x - 32; i < choices; i += kThreads - 32) {
            const int r = p.rows[i];
            choice_row[i] = (int16_t)r;
            choice_weight[i] = p.weights[i];
            if (r >= 0) row_token[r] = (uint16_t)(i / p.k);
        }
    }
    for (int i = threadIdx.x; i * 4 < p.pitch; i += kThreads) reinterpret_cast<int *>(zeros)[i] = 0;
    __syncthreads();

    const T *x = static_cast<const T *>(p.x);
    T *h = static_cast<T *>(p.h);
    const int units_up = p.F / 8, units_down = (p.K + 15) / 16;
    const int total_up = n_groups * units_up, total = total_up + n_groups * units_down;
    const int first = (int)blockIdx.x, stride = (int)gridDim.x;
    const uint64_t tmo = p.ctl.wait_timeout_ns;
    const uint32_t stage_bytes = p.stage_bytes;
    // A reduction's stages, by their first element: up to eight whole blocks of 64, the last one
    // with the elements past them
    auto stages_of = [](int red) { return max(1, ((red & ~63) + kSegment - 1) / kSegment); };

    // The CTA's units, by number: of W13's and then of W2's, by expert, by the expert's unit, by
    // sixteens of its rows.  a: the active expert of a unit before, or 0.
    const int n_ups = first < total_up ? (total_up - first + stride - 1) / stride : 0;
    const int n_units = first < total ? (total - first + stride - 1) / stride : 0;
    const int stages_up = stages_of(p.K), stages_down = stages_of(p.F);
    auto unit_at = [&](int number, int a) {
        Unit r;
        r.up = number < n_ups;
        const int per = r.up ? units_up : units_down, v = first + number * stride - (r.up ? 0 : total_up);
        while (act_g[a + 1] * per <= v) a++;
        const int at = v - act_g[a] * per, sixteens = act_g[a + 1] - act_g[a];
        r.a = a;
        r.idx = sixteens == 1 ? at : at / sixteens;
        const int part = at - r.idx * sixteens;
        r.n = min(kMaxRows, act_n[a] - part * kMaxRows);
        r.row0 = act_row[a] + part * kMaxRows;
        return r;
    };

    // y of 16 columns once all their parts are there (or none is to come)
    auto combine = [&](int col0) {
        const int cols = min(16, p.K - col0) / 4;  // 4 or 2 pieces of 4
        for (int i = lane; i < p.T * 4; i += 32) {
            const int t = i >> 2, c = i & 3;
            if (c >= cols) continue;
            const int64_t at = (int64_t)t * p.K + col0 + c * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j0 = 0; j0 < p.k; j0 += 8) {
                float4 v[8];
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int r = j0 + j < p.k ? choice_row[t * p.k + j0 + j] : -1;
                    w[j] = r >= 0 ? choice_weight[t * p.k + j0 + j] : 0.0f;
                    v[j] = r >= 0 ? __ldcg(reinterpret_cast<const float4 *>(p.part + (int64_t)r * p.K + col0 + c * 4))
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    s.x = fmaf(w[j], v[j].x, s.x);
                    s.y = fmaf(w[j], v[j].y, s.y);
                    s.z = fmaf(w[j], v[j].z, s.z);
                    s.w = fmaf(w[j], v[j].w, s.w);
                }
            }
            if (p.residual) {
                const uint2 r = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.residual) + at);
                const float2 a = Type16<T>::unpack(r.x), b = Type16<T>::unpack(r.y);
                s.x += a.x;
                s.y += a.y;
                s.z += b.x;
                s.w += b.y;
            }
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.y) + at) =
                make_uint2(Type16<T>::pack(s.x, s.y), Type16<T>::pack(s.z, s.w));
        }
    };
    if (total == 0) {  // no token has an expert
        constexpr int kAll = kThreads / 32;
        for (int b = (int)blockIdx.x * kAll + warp; b < units_down; b += (int)gridDim.x * kAll) combine(b * 16);
        return;
    }

    if (warp >= kEpiWarp) {
        // ---- the parts of the units in turn
        // which of a unit's rows a lane's fragments hold: the order in which eight lanes read two
        // rows of a swizzled tile from different banks
        const int r = (g >> 1) | ((g & 1) << 2);
        const int parts_up = min(stages_up, p.stages), parts_down = min(stages_down, p.stages);
        int a = 0;
        for (int i = warp - kEpiWarp; i < n_units; i += kEpiWarps) {
            const int set = i % kSets;
            if (i >= n_ups && i - kEpiWarps < n_ups) a = 0;  // W2's units begin with the first expert
            const Unit un = unit_at(i, a);
            a = un.a;
            // the unit's parts, its first stage's warp, and the parts that the set has got by then
            const int parts = un.up ? parts_up : parts_down;
            const int from_warp = (min(i, n_ups) * stages_up + max(0, i - n_ups) * stages_down) % p.stages;
            auto of_set = [&](int n) { return n > set ? (n - 1 - set) / kSets + 1 : 0; };  // its units among n
            const int ups = of_set(min(i + 1, n_ups));
            const int want = ups * parts_up + (of_set(i + 1) - ups) * parts_down;
            if (!warp_count_wait(&parted[set], want, tmo, abort_flag, lane)) {
                if (lane == 0) report_timeout(abort_flag, p.ctl.status);
                break;
            }
            float4 sum[kMaxTiles];
#pragma unroll
            for (int i = 0; i < kMaxTiles; i++) {
                if (i * 8 >= un.n) break;
                const float4 *from = sums + (set * kWarps * tiles_cap + i) * 32 + lane;
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int w = 0, at = from_warp; w < parts; w++) {  // in the order of the stages
                    const float4 o = from[at * tiles_cap * 32];
                    at = at + 1 == p.stages ? 0 : at + 1;
                    s.x += o.x;
                    s.y += o.y;
                    s.z += o.z;
                    s.w += o.w;
                }
                sum[i] = s;
            }
            __syncwarp();
            if (lane == 0) count_release(&taken[set], 1);  // other parts may take their place
#pragma unroll
            for (int i = 0; i < kMaxTiles; i++) {
                if (i * 8 >= un.n) break;
                const float4 s = sum[i];
                const int c = i * 8 + 2 * q;  // s.x, s.z: column c, rows r and r + 8; s.y, s.w: column c + 1
                if (un.up) {
                    T *to = h + (int64_t)(un.row0 + c) * p.hp + un.idx * 8 + r;
                    if (c < un.n) to[0] = Type16<T>::round(s.x * linear::sigma(s.x) * s.z);
                    if (c + 1 < un.n) to[p.hp] = Type16<T>::round(s.y * linear::sigma(s.y) * s.w);
                } else {
                    const int row = un.idx * 16 + r;
                    float *to = p.part + (int64_t)(un.row0 + c) * p.K + row;
                    if (c < un.n && row < p.K) to[0] = s.x;
                    if (c < un.n && row + 8 < p.K) to[8] = s.z;
                    if (c + 1 < un.n && row < p.K) to[p.K] = s.y;
                    if (c + 1 < un.n && row + 8 < p.K) to[p.K + 8] = s.w;
                }
            }
            __syncwarp();
            int last = 0;
            if (lane == 0) {
                if (un.up) add_release(p.up_done + act_e[un.a]);
                else last = add_acquire_release(p.col_done + un.idx) == n_groups - 1;
            }
            last = __shfl_sync(0xffffffffu, last, 0);
            __syncwarp();  // what lane 0 has acquired, for all
            if (last) combine(un.idx * 16);
            __syncwarp();
        }
        return;
    }

    if (warp == kWatchWarp) {
        // ---- which experts' hidden rows are there, by all CTAs of the grid
        if (lane == 0 && n_units > 0) {
            const uint64_t t0 = global_timer_ns();
            for (int a = 0; a < n_active; a++) {
                const int *done = p.up_done + act_e[a];
                const int want = units_up * (act_g[a + 1] - act_g[a]);
                while (load_acquire(done) < want)
                    if (*abort_flag || global_timer_ns() - t0 > tmo) {
                        report_timeout(abort_flag, p.ctl.status);
                        return;
                    }
                count_release(&hidden, 1);
            }
        }
        return;
    }

    // ---- the products: every p.stages-th of the CTA's stages
    if (warp >= p.stages) return;
    uint8_t *weights = smem + warp * stage_bytes, *rows = weights + (kBlocks + p.tail) * kBlockBytes;
    const int wr = (g >> 1) | ((g & 1) << 2);  // the weight row of this lane's fragments
    const uint8_t *even = weights + wr * 128 + ((q ^ wr) << 4), *odd = weights + wr * 128 + (((4 + q) ^ wr) << 4);
    const uint32_t full = bar_full + 8 * warp;
    // The warp's next stage: unit `number`, stage `at` of it, which may be past the unit's.
    int number = 0, at = warp, expert = 0;
    auto next_stage = [&](Stage &s) {
        for (;;) {
            const int stages = number < n_ups ? stages_up : stages_down;
            if (at < stages || number >= n_units) break;
            at -= stages;
            number++;
            if (number == n_ups) expert = 0;
        }
        if (number >= n_units) return false;
        s.unit = unit_at(number, expert);
        expert = s.unit.a;
        s.number = number;
        const int e = act_e[s.unit.a], red = s.unit.up ? p.K : p.F, stages = s.unit.up ? stages_up : stages_down;
        s.row = s.unit.up ? e * 2 * p.F + (s.unit.idx >> 1) * 32 + (s.unit.idx & 1) * 8 : e * p.K + s.unit.idx * 16;
        s.block = at * kBlocks;
        s.blocks = min(kBlocks, red / 64 - s.block);
        s.rest = at == stages - 1 ? red & 63 : 0;
        s.first = at < p.stages;
        s.last = at + p.stages >= stages;
        at += p.stages;
        return true;
    };
    auto copy_weights = [&](const Stage &s) {
        if (lane == 0) {
            const uint32_t dst = smem_u32(weights);
            mbar_arrive_expect_tx(full, ((s.blocks > 0 ? kBlocks : 0) + (s.rest ? 1 : 0)) * kBlockBytes);
            if (s.blocks > 0) {  // blocks past the last are filled with zeros
                if (s.unit.up) tma_load_4d(dst, &map13, full, 0, s.row, 0, s.block);
                else linear::tma_load_3d(dst, &map2, full, 0, s.row, s.block);
            }
            if (s.rest) {
                const int k = (s.unit.up ? p.K : p.F) & ~63;
                if (s.unit.up) linear::tma_load_3d(dst + kBlocks * kBlockBytes, &tail13, full, k, s.row, 0);
                else tma_load_2d(dst + kBlocks * kBlockBytes, &tail2, full, k, s.row);
            }
        }
        __syncwarp();
    };
    // eight of the unit's rows, the stage's elements of them; lane r knows where row r is
    auto bring = [&](const Stage &s, int tile) {
        const int n = s.blocks * 64 + s.rest, rows_here = min(8, s.unit.n - tile * 8);
        const T *mine = nullptr;
        if (lane < rows_here) {
            const int row = s.unit.row0 + tile * 8 + lane;
            mine = (s.unit.up ? x + row_token[row] * p.ldx : h + (int64_t)row * p.hp) + s.block * 64;
        }
        const uint32_t to = smem_u32(rows) + lane * 16;
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const T *from = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(mine), r));
            if (r >= rows_here) break;
#pragma unroll
            for (int c = 0; c < 3; c++)  // at most 575 elements
                if (c * 256 + lane * 8 < n) copy16(to + r * p.pitch + c * 512, from + c * 256 + lane * 8);
        }
    };
    float acc[kMaxTiles][2][4];
    Stage stage;
    bool ok = true, brought = false, more = next_stage(stage), flying = more;  // the rows; the weights
    int phase = 0;
    if (more) copy_weights(stage);
    while (more) {
        if (!brought) {
            if (!stage.unit.up) ok = warp_count_wait(&hidden, stage.unit.a + 1, tmo, abort_flag, lane);
            if (!ok) break;
            bring(stage, 0);
        }
        Stage next;
        more = next_stage(next);
        if (stage.first)
#pragma unroll
            for (int t = 0; t < kMaxTiles; t++)
#pragma unroll
                for (int j = 0; j < 8; j++) acc[t][j >> 2][j & 3] = 0.0f;
        ok = linear::warp_wait_parity(full, phase, tmo, abort_flag, lane);
        if (!ok) break;
        phase ^= 1;
        flying = false;
#pragma unroll
        for (int t = 0; t < kMaxTiles; t++) {
            if (t * 8 >= stage.unit.n) break;
            if (t) {
                __syncwarp();  // the first tile's rows have been read
                bring(stage, t);
            }
            copies_wait();
            __syncwarp();
            const uint8_t *column = (t * 8 + g < stage.unit.n ? rows + g * p.pitch : zeros) + q * 16;
            auto chunk = [&](const uint8_t *w, const uint8_t *b) {
                const uint4 wa = *reinterpret_cast<const uint4 *>(w), wb = *reinterpret_cast<const uint4 *>(w + 1024);
                const uint4 v = *reinterpret_cast<const uint4 *>(b);
                mma<T>(acc[t][0], wa.x, wb.x, wa.y, wb.y, v.x, v.y);
                mma<T>(acc[t][1], wa.z, wb.z, wa.w, wb.w, v.z, v.w);
            };
            if (stage.blocks == kBlocks) {
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    chunk(even + b * kBlockBytes, column + b * 128);
                    chunk(odd + b * kBlockBytes, column + b * 128 + 64);
                }
            } else {
                for (int b = 0; b < stage.blocks; b++) {
                    chunk(even + b * kBlockBytes, column + b * 128);
                    chunk(odd + b * kBlockBytes, column + b * 128 + 64);
                }
            }
            if (stage.rest)  // the weights past the row's end are zeros, the tokens' row is read no further
#pragma unroll
                for (int half = 0; half < 2; half++)
                    if (half * 32 < stage.rest) {
                        const bool in = half * 32 + q * 8 < stage.rest;
                        chunk((half ? odd : even) + kBlocks * kBlockBytes,
                              in ? column + stage.blocks * 128 + half * 64 : zeros);
                    }
        }
        __syncwarp();
        const bool last = stage.last;
        const int unit = stage.number, columns = stage.unit.n;
        brought = false;
        if (more) {
            stage = next;
            copy_weights(stage);
            flying = true;
            // hidden rows that are not there yet wait for others, this warp's own parts among them
            brought = stage.unit.up || count_reached(&hidden, stage.unit.a + 1);
            brought = __shfl_sync(0xffffffffu, (int)brought, 0) != 0;
            __syncwarp();  // what lane 0 has acquired, for all
            if (brought) bring(stage, 0);
        }
        if (last) {
            const int set = unit % kSets;
            ok = warp_count_wait(&taken[set], unit / kSets, tmo, abort_flag, lane);
            if (!ok) break;
            float4 *to = sums + (set * kWarps + warp) * tiles_cap * 32 + lane;
#pragma unroll
            for (int t = 0; t < kMaxTiles; t++)
                if (t * 8 < columns)
                    to[t * 32] = make_float4(acc[t][0][0] + acc[t][1][0], acc[t][0][1] + acc[t][1][1],
                                             acc[t][0][2] + acc[t][1][2], acc[t][0][3] + acc[t][1][3]);
            __syncwarp();
            if (lane == 0) count_release(&parted[set], 1);
        }
    }
    if (!ok) {  // let the copies in flight land before the memory goes
        volatile int never = 0;
        __syncwarp();
        if (lane == 0) {
            report_timeout(abort_flag, p.ctl.status);
            if (flying) wait_parity(full, phase, p.ctl.drain_timeout_ns, &never);
        }
        copies_wait();
        __syncwarp();
    }
}

// ------------------------------------------------------------------------- host side
// Whether the kernel above takes the layer, or two products by row group (moe_products.cu).  An
// expert's rows are brought to every unit, so few of them: up to 8 tokens, one tile at most, or
// four rows on average.  Beyond 8 tokens units of two stages and more, since a unit's sums take
// longer than one stage's weights.  us, this kernel and the products: 1 token by 2 of 8 experts
// of 512 x 1024 16 and 20, 7 by 2 of 16 of 648 x 288 20 and 21, 8 by 8 of 8 of 2048 x 4096 76 and
// 89; 16 by 2 73 and 83, by 4 88 and 87, by 8 105 and 89; 32 by 8 of 256 of 2048 x 768 (2.9
// stages a unit) 263 and 264, 40 by 4 of 60 of 1024 x 704 (2.0) 72 and 66, 64 by 4 of 256 of 768 x
// 512 (1.6) 114 and 98.
static bool streamed(int T, int E, int k, int K, int F) {
    const int64_t ups = F / 8, downs = (K + 15) / 16, units = ups + downs;
    const int64_t stages = ups * ((K + kSegment - 1) / kSegment) + downs * ((F + kSegment - 1) / kSegment);
    return T <= 8 || (T * k <= 4 * E && 4 * stages >= 9 * units);
}

struct Layout {
    size_t weights, experts, rows, offsets, counters, h, part, parts, x_rows, bytes;
    int n_counters, hp;
};
static Layout layout(int T, int E, int k, int K, int F) {
    Layout l;
    size_t n = 0;
    auto take = [&](size_t bytes) {
        const size_t at = n;
        n += (bytes + 255) & ~(size_t)255;
        return at;
    };
    const size_t R = (size_t)T * k;
    const bool one = streamed(T, E, k, K, F);
    l.hp = one ? (F + 63) & ~63 : F;  // one kernel: whole 128-byte lines, no two rows share one
    l.n_counters = one ? E + (K + 15) / 16 : 0;
    l.weights = take(R * 4);
    l.experts = take(R * 4);
    l.rows = take(R * 4);
    l.offsets = take((size_t)(E + 1) * 4);
    l.counters = take((size_t)l.n_counters * 4);
    l.h = take(R * l.hp * 2);
    l.part = take(R * K * 4 * (one ? 1 : moe_products::kMaxParts));
    l.parts = take(one ? 0 : (size_t)E * ((K + moe_products::kTile - 1) / moe_products::kTile));
    l.x_rows = take(one ? 0 : R * K * 2);
    l.bytes = n;
    return l;
}

// The weight's views: boxes of 8 blocks of 64 elements by 16 rows (W13: 8 gate rows and the 8
// up rows 16 further on), and of the elements past the last whole block.  Without such a part
// its view is not used, and the other stands in for it.
template <typename T>
static int map_weights(CUtensorMap *map, CUtensorMap *tail, const void *w, int64_t rows, int red, bool pairs) {
    const uint64_t row = (uint64_t)red * 2, whole = red / 64;
    const uint64_t n = (uint64_t)rows - (pairs ? 16 : 0);
    int st = NVFP4_OK;
    if (pairs) {
        const uint64_t dims[4] = {64, n, 2, whole}, strides[3] = {row, 16 * row, 128};
        const uint32_t box[4] = {64, 8, 2, kBlocks};
        const uint64_t tdims[3] = {(uint64_t)red, n, 2}, tstrides[2] = {row, 16 * row};
        const uint32_t tbox[3] = {64, 8, 2};
        if (whole) st = encode_tiled(map, linear::tma_type<T>(), 4, w, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
        if (!st && red % 64)
            st = encode_tiled(tail, linear::tma_type<T>(), 3, w, tdims, tstrides, tbox, CU_TENSOR_MAP_SWIZZLE_128B);
    } else {
        const uint64_t dims[3] = {64, n, whole}, strides[2] = {row, 128};
        const uint32_t box[3] = {64, 16, kBlocks};
        const uint64_t tdims[2] = {(uint64_t)red, n}, tstrides[1] = {row};
        const uint32_t tbox[2] = {64, 16};
        if (whole) st = encode_tiled(map, linear::tma_type<T>(), 3, w, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
        if (!st && red % 64)
            st = encode_tiled(tail, linear::tma_type<T>(), 2, w, tdims, tstrides, tbox, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (!whole) *map = *tail;
    if (red % 64 == 0) *tail = *map;
    return st;
}

template <typename T>
static int launch(const Params &p, const DeviceInfo &di, cudaStream_t s) {
    auto kern = moe_layer_kernel<T>;
    CUtensorMap map13, tail13, map2, tail2;
    int st = map_weights<T>(&map13, &tail13, p.w13, (int64_t)p.E * 2 * p.F, p.K, true);
    if (!st) st = map_weights<T>(&map2, &tail2, p.w2, (int64_t)p.E * p.K, p.F, false);
    if (st) return st;
    static std::atomic<bool> configured[64] = {};
    if (!configured[di.device].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeCooperative;  // its blocks wait for each other
    attr.val.cooperative = 1;
    cfg.gridDim = dim3((unsigned)di.sm_count);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, map13, tail13, map2, tail2, p) != cudaSuccess) return NVFP4_ERR_CUDA;
    count_launch();
    return cuda_status(cudaGetLastError());
}

static int check_sizes(int T, int E, int k, int K, int F) {
    if (T < 0 || T > kMaxTokens || E < 1 || E > kMaxExperts || k < 1 || k > kMaxTopK || k > E) return NVFP4_ERR_SHAPE;
    if (K < 8 || K % 8 || F < 16 || F % 16 || K > kMaxSize || F > kMaxSize) return NVFP4_ERR_SHAPE;
    return (int64_t)E * 2 * F > INT_MAX || (int64_t)E * K > INT_MAX ? NVFP4_ERR_SHAPE : NVFP4_OK;
}

}  // namespace moe_layer
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

size_t nvfp4_moe_layer_workspace_size(int T, int E, int top_k, int K, int F) {
    if (T < 1 || moe_layer::check_sizes(T, E, top_k, K, F)) return 0;
    return moe_layer::layout(T, E, top_k, K, F).bytes;
}

int nvfp4_moe_layer(const void *X, int64_t ldx, const void *logits, int logits_dtype, const float *bias,
                    const void *W13, const void *W2, const void *residual, void *Y, int T, int E, int top_k, int K,
                    int F, int scoring, int renormalize, float scale, int dtype, void *workspace,
                    size_t workspace_bytes, void *stream) {
    if (dtype != NVFP4_BF16 && dtype != NVFP4_F16) return NVFP4_ERR_INVALID;
    int st = moe_layer::check_sizes(T, E, top_k, K, F);
    if (st) return st;
    if (ldx < K || ldx % 8) return NVFP4_ERR_SHAPE;
    if (!W13 || !W2 || (T && (!X || !logits || !Y))) return NVFP4_ERR_INVALID;
    if (!aligned16(X) || !aligned16(W13) || !aligned16(W2) || !aligned16(residual) || !aligned16(Y) ||
        (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return NVFP4_ERR_ALIGN;
    const size_t need = nvfp4_moe_layer_workspace_size(T, E, top_k, K, F);
    if (T && (!workspace || workspace_bytes < need)) return NVFP4_ERR_WORKSPACE;
    if (T == 0) return NVFP4_OK;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    const moe_layer::Layout l = moe_layer::layout(T, E, top_k, K, F);
    moe_layer::Params p = {};
    p.x = X;
    p.w13 = W13;
    p.w2 = W2;
    p.residual = residual;
    p.y = Y;
    p.ldx = ldx;
    p.weights = reinterpret_cast<float *>(ws + l.weights);
    p.rows = reinterpret_cast<int *>(ws + l.rows);
    p.m_offsets = reinterpret_cast<int *>(ws + l.offsets);
    p.up_done = reinterpret_cast<int *>(ws + l.counters);
    p.col_done = p.up_done + E;
    p.h = ws + l.h;
    p.part = reinterpret_cast<float *>(ws + l.part);
    int *experts = reinterpret_cast<int *>(ws + l.experts);
    p.T = T;
    p.E = E;
    p.k = top_k;
    p.K = K;
    p.F = F;
    p.hp = l.hp;
    // the router's checks of its own arguments come before any launch
    st = moe::route_tokens(logits, logits_dtype, bias, T, E, top_k, scoring, renormalize, scale,
                           const_cast<float *>(p.weights), experts, const_cast<int *>(p.rows),
                           const_cast<int *>(p.m_offsets), nullptr, 0, p.up_done, l.n_counters, stream);
    if (st) return st;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!moe_layer::streamed(T, E, top_k, K, F)) {
        moe_products::Args a = {};
        a.x = X;
        a.w13 = W13;
        a.w2 = W2;
        a.residual = residual;
        a.y = Y;
        a.ldx = ldx;
        a.weights = p.weights;
        a.experts = experts;
        a.rows = p.rows;
        a.m_offsets = p.m_offsets;
        a.x_rows = ws + l.x_rows;
        a.h = p.h;
        a.part = p.part;
        a.parts = ws + l.parts;
        a.T = T;
        a.E = E;
        a.k = top_k;
        a.K = K;
        a.F = F;
        a.dtype = dtype;
        return moe_products::run(a, di, s);
    }
    const int tiles = std::min(moe_layer::kMaxTiles, (T + 7) / 8);
    p.tail = K % 64 || F % 64;
    p.pitch = (moe_layer::kSegment + 64 * p.tail) * 2 + 64;
    p.stage_bytes =
        ((moe_layer::kBlocks + p.tail) * moe_layer::kBlockBytes + moe_layer::kTokenRows * p.pitch + 1023) & ~1023;
    const int beside = 1024 + moe_layer::kSets * moe_layer::kWarps * tiles * 512 + p.pitch + 8 * T * top_k;
    p.stages = std::min(moe_layer::kMaxStages, (moe_layer::kSmem - beside) / p.stage_bytes);
    if ((st = kernel_ctl(&p.ctl))) return st;
    return dtype == NVFP4_BF16 ? moe_layer::launch<__nv_bfloat16>(p, di, s) : moe_layer::launch<__half>(p, di, s);
}

}  // extern "C"
