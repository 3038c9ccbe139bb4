// moe_layer.cu — a whole mixture-of-experts layer for the few tokens of a decode step, bound
// by streaming the chosen experts' weights once.
//
//   y[t] = residual[t] + sum_j w[t, j] W2_e ( silu(W1_e x[t]) * (W3_e x[t]) ),  e = e(t, j)
//
// Two launches: the router (moe.cu, which also clears this kernel's counters), and one
// cooperative kernel for the experts and the weighted sum, where six kernels and their gaps
// took longer than the weights of small experts do.
//
// The work is a list of units of 16 weight rows: first all of W13 (8 gate rows with their 8 up
// rows, so SwiGLU stays in a thread), then all of W2, each by active expert; experts without a
// token are not in it.  Groups of warps take the units in turn, the warps of a group share a
// unit's reduction and add their parts up in shared memory in order.  Where W2's units begin a
// group waits for its expert's hidden rows alone (a counter an expert), not for the grid.  The
// rows' results are left in fp32, and the warp that brings a block of 16 columns its last
// part forms the weighted sum there, in the order of the choices: the same bits every time.
//
// Weights go through a ring of shared memory that belongs to each thread alone: it copies its
// own 16-byte pieces asynchronously and reads them back itself, so the stream needs no
// barrier, and it runs on across units and into W2 while its hidden rows are still being made.
// A piece is 8 elements of a row; lanes 4g .. 4g + 3 hold row g, which is mma.m16n8k16's A
// fragment with the reduction's elements permuted, and the tokens are read with the same
// permutation, so nothing is shuffled.  The products are tiny (8 token columns a tile); the
// tensor core only has to keep up with memory.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "linear.cuh"
#include "moe.cuh"
#include "ptx.cuh"
#include "types16.cuh"

namespace nvfp4 {
namespace moe_layer {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTokens = 32;             // rows of an expert, so at most four tiles of 8 columns
constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 32;
constexpr int kSlots = 6;                  // ring: 16 KB each
constexpr int kSlotBytes = kThreads * 32;
constexpr int kMaxTiles = kMaxTokens / 8;

struct Params {
    const void *x, *w13, *w2, *residual;
    void *y;
    int64_t ldx;
    const float *weights;      // [T, k]
    const int *rows;           // [T, k]
    const int *m_offsets;      // [E + 1]
    int *up_done;              // [E] finished tiles of an expert's hidden rows
    int *col_done;             // [column blocks] finished tiles
    void *h;                   // [T k, hp]
    float *part;               // [T k, K]
    int T, E, k, K, F, hp;
    int group;                 // warps of a group
    KernelCtl ctl;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void group_barrier(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) moe_layer_kernel(const Params p) {
    extern __shared__ uint8_t smem[];
    __shared__ int act_e[kMaxExperts], act_row[kMaxExperts], act_n[kMaxExperts];
    __shared__ uint16_t row_token[kMaxTokens * kMaxTopK];
    __shared__ int n_active, n_tiles, ready[kWarps];
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;  // fragment row / column, and quarter of 32 elements
    const int in_group = warp % p.group, group = warp / p.group, groups = kWarps / p.group;
    const int bar = 1 + group, bar_threads = p.group * 32;

    // ---- active experts and the rows' tokens
    if (threadIdx.x == 0) abort_word = 0;
    if (warp == 0) {
        int n = 0, tiles = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane;
            int r0 = 0, r1 = 0;
            if (e < p.E) {
                r0 = p.m_offsets[e];
                r1 = p.m_offsets[e + 1];
            }
            const uint32_t live = __ballot_sync(0xffffffffu, r1 > r0);
            if (r1 > r0) {
                const int at = n + __popc(live & ((1u << lane) - 1u));
                act_e[at] = e;
                act_row[at] = r0;
                act_n[at] = r1 - r0;
            }
            n += __popc(live);
            tiles += __reduce_add_sync(0xffffffffu, (r1 - r0 + 7) / 8);
        }
        if (lane == 0) {
            n_active = n;
            n_tiles = tiles;
        }
    } else {
        for (int i = threadIdx.x - 32; i < p.T * p.k; i += kThreads - 32) {
            const int r = p.rows[i];
            if (r >= 0) row_token[r] = (uint16_t)(i / p.k);
        }
    }
    __syncthreads();

    const T *x = static_cast<const T *>(p.x);
    T *h = static_cast<T *>(p.h);
    const int units_up = p.F / 8, units_down = (p.K + 15) / 16;
    const int total_up = n_active * units_up, total = total_up + n_active * units_down;
    const int first = group * (int)gridDim.x + (int)blockIdx.x, stride = groups * (int)gridDim.x;

    // y of 16 columns once all their parts are there (or none is to come)
    auto combine = [&](int col0) {
        const int cols = min(16, p.K - col0) / 4;  // 4 or 2 pieces of 4
        for (int i = lane; i < p.T * 4; i += 32) {
            const int t = i >> 2, c = i & 3;
            if (c >= cols) continue;
            const int64_t at = (int64_t)t * p.K + col0 + c * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j = 0; j < p.k; j++) {
                const int r = p.rows[t * p.k + j];
                if (r < 0) continue;
                const float w = p.weights[t * p.k + j];
                const float4 v = __ldcg(reinterpret_cast<const float4 *>(p.part + (int64_t)r * p.K + col0 + c * 4));
                s.x = fmaf(w, v.x, s.x);
                s.y = fmaf(w, v.y, s.y);
                s.z = fmaf(w, v.z, s.z);
                s.w = fmaf(w, v.w, s.w);
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
        for (int b = (int)blockIdx.x * kWarps + warp; b < units_down; b += (int)gridDim.x * kWarps) combine(b * 16);
        return;
    }

    // ---- the stream of weights: this thread's pieces of rows g and g + 8 of each unit
    const uint32_t ring = smem_u32(smem) + threadIdx.x * 16;
    int iu = first, ic = in_group, i_chunks = 0, i_red = 0, i_slot = 0;
    const T *pa = nullptr, *pb = nullptr;  // null: past the weight's rows
    auto open = [&]() {
        if (iu < total_up) {
            const int a = iu / units_up, f = iu - a * units_up;
            i_red = p.K;
            pa = static_cast<const T *>(p.w13) +
                 ((int64_t)act_e[a] * 2 * p.F + (f >> 1) * 32 + (f & 1) * 8 + g) * p.K + q * 8;
            pb = pa + (int64_t)16 * p.K;
        } else if (iu < total) {
            const int a = (iu - total_up) / units_down, row = (iu - total_up - a * units_down) * 16 + g;
            i_red = p.F;
            const T *w = static_cast<const T *>(p.w2) + ((int64_t)act_e[a] * p.K + row) * p.F + q * 8;
            pa = row < p.K ? w : nullptr;
            pb = row + 8 < p.K ? w + (int64_t)8 * p.F : nullptr;
        }
        i_chunks = (i_red + 31) / 32;
    };
    auto issue = [&]() {
        while (iu < total && ic >= i_chunks) {  // a unit with fewer chunks than the group has warps may have none here
            iu += stride;
            ic = in_group;
            open();
        }
        if (iu < total) {
            const bool in = ic * 32 + q * 8 < i_red;
            const uint32_t dst = ring + i_slot * kSlotBytes;
            const bool live_a = in && pa, live_b = in && pb;
            copy16(dst, live_a ? pa + ic * 32 : static_cast<const T *>(p.w13), live_a);
            copy16(dst + kThreads * 16, live_b ? pb + ic * 32 : static_cast<const T *>(p.w13), live_b);
            ic += p.group;
        }
        copy_commit();
        i_slot = i_slot + 1 == kSlots ? 0 : i_slot + 1;
    };
    open();
    for (int s = 0; s < kSlots; s++) issue();

    // ---- the units
    float4 *sums = reinterpret_cast<float4 *>(smem + kSlots * kSlotBytes);  // [2][warp][tile][lane]
    const int tiles_cap = (p.T + 7) / 8;
    int slot = 0, parity = 0, have = -1, turn = 0;
    for (int u = first; u < total; u += stride, parity ^= 1, turn++) {
        const bool up = u < total_up;
        const int per = up ? units_up : units_down, v = up ? u : u - total_up, a = v / per, idx = v - a * per;
        const int n = act_n[a], row0 = act_row[a], tiles = (n + 7) / 8;
        const int red = up ? p.K : p.F, chunks = (red + 31) / 32;
        if (!up && have != a) {
            // the expert's hidden rows, by all groups of the grid
            if (in_group == 0 && lane == 0) {
                const int want = units_up * tiles;
                int ok = 1;
                if (load_acquire(p.up_done + act_e[a]) < want) {
                    const uint64_t t0 = global_timer_ns();
                    while (load_acquire(p.up_done + act_e[a]) < want) {
                        if (*abort_flag || global_timer_ns() - t0 > p.ctl.wait_timeout_ns) {
                            report_timeout(abort_flag, p.ctl.status);
                            ok = 0;
                            break;
                        }
                    }
                }
                ready[group] = ok;
            }
            group_barrier(bar, bar_threads);
            const int ok = ready[group];
            group_barrier(bar, bar_threads);
            if (!ok) break;
            have = a;
        }
        auto accumulate = [&](auto tiles_const) {
            constexpr int NT = decltype(tiles_const)::value;
            float acc[NT][4];
            const T *col[NT];
#pragma unroll
            for (int i = 0; i < NT; i++) {
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
                const int c = i * 8 + g;
                col[i] = c >= n ? nullptr
                                : (up ? x + row_token[row0 + c] * p.ldx : h + (int64_t)(row0 + c) * p.hp) + q * 8;
            }
            for (int c = in_group; c < chunks; c += p.group) {
                const bool in = c * 32 + q * 8 < red;
                uint4 b[NT];
#pragma unroll
                for (int i = 0; i < NT; i++)
                    b[i] = in && col[i] ? *reinterpret_cast<const uint4 *>(col[i] + c * 32) : make_uint4(0u, 0u, 0u, 0u);
                copy_wait<kSlots - 1>();
                uint4 wa, wb;
                const uint32_t src = ring + slot * kSlotBytes;
                ld_shared_v4(src, wa.x, wa.y, wa.z, wa.w);
                ld_shared_v4(src + kThreads * 16, wb.x, wb.y, wb.z, wb.w);
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    mma<T>(acc[i], wa.x, wb.x, wa.y, wb.y, b[i].x, b[i].y);
                    mma<T>(acc[i], wa.z, wb.z, wa.w, wb.w, b[i].z, b[i].w);
                }
                issue();  // the pieces are in registers: their slot takes the next ones
                slot = slot + 1 == kSlots ? 0 : slot + 1;
            }
            float4 *mine = sums + ((parity * kWarps + warp) * tiles_cap) * 32 + lane;
#pragma unroll
            for (int i = 0; i < NT; i++)
                if (i < tiles_cap) mine[i * 32] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        };
        if (tiles == 1) accumulate(std::integral_constant<int, 1>());
        else if (tiles == 2) accumulate(std::integral_constant<int, 2>());
        else accumulate(std::integral_constant<int, 4>());
        group_barrier(bar, bar_threads);
        // a warp a tile adds the parts up, another one for each unit; the sums' other half takes
        // the next unit's parts meanwhile
        for (int i = 0; i < tiles; i++) {
            if ((turn + i) % p.group != in_group) continue;
            const float4 *from = sums + ((parity * kWarps + group * p.group) * tiles_cap + i) * 32 + lane;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < p.group; w++) {
                const float4 o = from[w * tiles_cap * 32];
                s.x += o.x;
                s.y += o.y;
                s.z += o.z;
                s.w += o.w;
            }
            const int c = i * 8 + 2 * q;  // s.x, s.z: column c, rows g and g + 8; s.y, s.w: column c + 1
            if (up) {
                T *to = h + (int64_t)(row0 + c) * p.hp + idx * 8 + g;
                if (c < n) to[0] = Type16<T>::round(s.x * linear::sigma(s.x) * s.z);
                if (c + 1 < n) to[p.hp] = Type16<T>::round(s.y * linear::sigma(s.y) * s.w);
                __syncwarp();
                if (lane == 0) {
                    __threadfence();
                    atomicAdd(p.up_done + act_e[a], 1);
                }
            } else {
                const int row = idx * 16 + g;
                float *to = p.part + (int64_t)(row0 + c) * p.K + row;
                if (c < n && row < p.K) to[0] = s.x;
                if (c < n && row + 8 < p.K) to[8] = s.z;
                if (c + 1 < n && row < p.K) to[p.K] = s.y;
                if (c + 1 < n && row + 8 < p.K) to[p.K + 8] = s.w;
                __syncwarp();
                int last = 0;
                if (lane == 0) {
                    __threadfence();
                    last = atomicAdd(p.col_done + idx, 1) == n_tiles - 1;
                    __threadfence();
                }
                if (__shfl_sync(0xffffffffu, last, 0)) combine(idx * 16);
            }
            __syncwarp();
        }
    }
    copy_wait<0>();
}

// ------------------------------------------------------------------------- host side
struct Layout {
    size_t weights, experts, rows, offsets, counters, h, part, bytes;
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
    l.hp = (F + 63) & ~63;  // whole 128-byte lines: no two rows share one
    l.n_counters = E + (K + 15) / 16;
    l.weights = take(R * 4);
    l.experts = take(R * 4);
    l.rows = take(R * 4);
    l.offsets = take((size_t)(E + 1) * 4);
    l.counters = take((size_t)l.n_counters * 4);
    l.h = take(R * l.hp * 2);
    l.part = take(R * K * 4);
    l.bytes = n;
    return l;
}

// Warps of a group: all of a CTA's where a reduction is long enough for each to have 4 chunks
// of 32, so that the units are spread over the GPU most evenly.
static int group_warps(int K, int F) {
    const int chunks = std::min(K, F) / 32;
    return chunks >= 64 ? 16 : chunks >= 32 ? 8 : 4;
}

template <typename T>
static int launch(const Params &p, const DeviceInfo &di, cudaStream_t s) {
    auto kern = moe_layer_kernel<T>;
    const int tiles = (p.T + 7) / 8;
    const int bytes = kSlots * kSlotBytes + 2 * kWarps * tiles * 512;
    static int configured[64] = {};
    if (!configured[di.device]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kSlots * kSlotBytes + 2 * kWarps * kMaxTiles * 512) != cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeCooperative;  // its blocks wait for each other
    attr.val.cooperative = 1;
    cfg.gridDim = dim3((unsigned)di.sm_count);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return NVFP4_ERR_CUDA;
    count_launch();
    return cuda_status(cudaGetLastError());
}

static int check_sizes(int T, int E, int k, int K, int F) {
    if (T < 0 || T > kMaxTokens || E < 1 || E > kMaxExperts || k < 1 || k > kMaxTopK || k > E) return NVFP4_ERR_SHAPE;
    if (K < 8 || K % 8 || F < 16 || F % 16 || K > (1 << 20) || F > (1 << 20)) return NVFP4_ERR_SHAPE;
    return NVFP4_OK;
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
    p.T = T;
    p.E = E;
    p.k = top_k;
    p.K = K;
    p.F = F;
    p.hp = l.hp;
    p.group = moe_layer::group_warps(K, F);
    // the router's checks of its own arguments come before any launch
    st = moe::route_tokens(logits, logits_dtype, bias, T, E, top_k, scoring, renormalize, scale,
                           const_cast<float *>(p.weights), reinterpret_cast<int *>(ws + l.experts),
                           const_cast<int *>(p.rows), const_cast<int *>(p.m_offsets), nullptr, 0,
                           p.up_done, l.n_counters, stream);
    if (st) return st;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if ((st = kernel_ctl(&p.ctl))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == NVFP4_BF16 ? moe_layer::launch<__nv_bfloat16>(p, di, s) : moe_layer::launch<__half>(p, di, s);
}

}  // extern "C"
