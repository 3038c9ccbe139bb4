// linear_decode.cu — the 16-bit linear layer, or its input gradient, for few tokens (a decode
// step): bound by streaming the weights once.
//
// One CTA multiplies 128 weight rows (the MMA's M) by the tokens (its N, a multiple of 16)
// over a part of the reduction; a cluster of up to 8 CTAs splits the reduction of a tile, so
// that a weight with few rows still occupies every SM.  The parts meet in distributed shared
// memory: each CTA leaves its fp32 partial tile there, and after one cluster barrier the
// CTAs add disjoint pieces of it in the order of the parts (the same bits every time) and
// run the epilogue on them.  No workspace, no atomics, no second launch.
//
// The ring is sized so that two CTAs share an SM: the prologue and the reduction of one run
// under the loads of another, and as a programmatic dependent the next forward call's set-up
// runs under this one's end (one token, N=K=4096, 12.4 -> 9.4 us a call).  Measured, M = 1, on
// the GPU: N=K=4096 7.4 us with the weight left in L2 by the call before, 9.6 us from memory
// (3.5 TB/s); N=14336 K=4096 22.3 us (5.3), N=28672 K=8192 74 us (6.3 of a copy's 6.55): bound
// by the weights' bytes, and for the smaller ones by what a launch, the first loads and the
// cluster's sum take.
//
// Warps: 0 TMA producer, 1 MMA issue and TMEM owner, 2-5 read the accumulator out; all six
// reduce.
#include <algorithm>
#include <climits>

#include "linear.cuh"

namespace nvfp4 {
namespace linear {

constexpr int kDecThreads = 192;
constexpr int kDecMaxStages = 8;
constexpr int kDecMaxSplits = 8;
constexpr int kDecBarBytes = 256;
constexpr int kDecSmem = 112 * 1024;  // two CTAs an SM

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Eight consecutive features of a token: the cluster's partial sums added in order.
__device__ __forceinline__ void sum_parts(uint32_t addr, int splits, float (&v)[8]) {
    float4 a[kDecMaxSplits], b[kDecMaxSplits];
#pragma unroll
    for (int s = 0; s < kDecMaxSplits; s++)
        if (s < splits) {
            const uint32_t at = map_to_cta(addr, s);
            a[s] = ld_cluster_f4(at);
            b[s] = ld_cluster_f4(at + 16);
        }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < kDecMaxSplits; s++)
        if (s < splits) {
            v[0] += a[s].x;
            v[1] += a[s].y;
            v[2] += a[s].z;
            v[3] += a[s].w;
            v[4] += b[s].x;
            v[5] += b[s].y;
            v[6] += b[s].z;
            v[7] += b[s].w;
        }
}

template <typename T>
__device__ __forceinline__ void add_bias(const void *bias, int64_t at, float (&v)[8]) {
    if (!bias) return;
    const T *b = static_cast<const T *>(bias) + at;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += Type16<T>::load(b + i);
}

template <typename T>
__device__ __forceinline__ void add_row(const void *residual, int64_t at, float (&v)[8]) {
    if (!residual) return;
    float r[8];
    unpack8<T>(*reinterpret_cast<const uint4 *>(static_cast<const T *>(residual) + at), r);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += r[i];
}

template <typename T>
__device__ __forceinline__ void put8(void *dst, int64_t at, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(static_cast<T *>(dst) + at) = pack8<T>(v);
}

template <typename T, int FORM>
__global__ void __launch_bounds__(kDecThreads)
    linear_decode_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                         const Params p) {
    constexpr bool kBf16 = !std::is_same<T, __half>::value, kAmn = FORM == kDgrad;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t slot = kTileBytes + (uint32_t)p.ncap * 128u;  // weight rows, then tokens
    const uint32_t bars = (uint32_t)p.stages * slot;
    const uint32_t bar_full = base + bars, bar_empty = bar_full + 8 * kDecMaxStages;
    const uint32_t bar_acc = bar_empty + 8 * kDecMaxStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(base_ptr + bars + 16 * kDecMaxStages + 8);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float *part = reinterpret_cast<float *>(base_ptr);  // [tokens][128], in the ring's place at the end

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = p.splits, split = (int)cluster_ctarank();
    const int tile = blockIdx.x / splits;
    const uint32_t tmem_cols = p.ncap <= 32 ? 32u : p.ncap <= 64 ? 64u : 128u;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        mbar_init(bar_acc, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    __syncwarp();
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), tmem_cols);
        tmem_relinquish();
    }
    const int n_f = (p.features + 127) / 128;
    const int nkb = (p.red + kBlockK - 1) / kBlockK;
    const int kb0 = (int)((int64_t)nkb * split / splits), kb1 = (int)((int64_t)nkb * (split + 1) / splits);
    // As a programmatic dependent (plan_decode) the set-up above runs while the previous kernel
    // finishes; nothing of global memory is read or written before it has.
    grid_dependency_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint64_t tmo = p.ctl.wait_timeout_ns;

    // Tiles are numbered over the groups that have rows: the others' weights are not read.
    int g = p.m_offsets ? -1 : 0, f = tile;
    if (p.m_offsets) {
        int nth = tile / n_f;
        f = tile - nth * n_f;
        for (int b = 0; b < p.groups && g < 0; b += 32) {
            int a = 0, z = 0;
            if (b + lane < p.groups) group_rows(p.m_offsets, b + lane, p.m_total, a, z);
            uint32_t live = __ballot_sync(0xffffffffu, z > a);
            const int n = __popc(live);
            if (nth < n) {
                for (; nth; nth--) live &= live - 1;
                g = b + __ffs(live) - 1;
            } else {
                nth -= n;
            }
        }
    }
    int r0 = 0, r1 = 0;
    if (g >= 0) group_rows(p.m_offsets, g, p.m_total, r0, r1);
    const int rows = r1 - r0, n16 = (rows + 15) & ~15;

    if (rows > 0) {  // the same for every CTA of the cluster
        if (warp == 0) {
            if (elect_one()) {
                const uint32_t bytes = kTileBytes + (uint32_t)n16 * 128u;
                uint32_t stage = 0, phase = 0, issued = 0, parity = 0;
                bool ok = true;
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!wait_parity(bar_empty + 8 * stage, phase ^ 1, tmo, abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        ok = false;
                        break;
                    }
                    const uint32_t bar = bar_full + 8 * stage, dA = base + stage * slot;
                    mbar_arrive_expect_tx(bar, bytes);
                    issued |= 1u << stage;
                    parity = (parity & ~(1u << stage)) | (phase << stage);
                    if constexpr (kAmn) {
                        tma_load_3d(dA, &tmap_a, bar, f * 128, kb * kBlockK, g);
                        tma_load_3d(dA + 8192, &tmap_a, bar, f * 128 + 64, kb * kBlockK, g);
                    } else {
                        tma_load_3d(dA, &tmap_a, bar, kb * kBlockK, f * 128, g);
                    }
                    for (int c = 0; c < n16; c += 16)
                        tma_load_2d(dA + kTileBytes + c * 128, &tmap_b, bar, kb * kBlockK, r0 + c);
                    if (++stage == (uint32_t)p.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                grid_launch_dependents();  // all loads issued: the next kernel may set itself up
                // the MMAs' last arrivals have to come before the CTA ends
                for (int s = 0; ok && s < p.stages; s++) {
                    if (!wait_parity(bar_empty + 8 * stage, phase ^ 1, tmo, abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        ok = false;
                    }
                    if (++stage == (uint32_t)p.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) {
                    volatile int never = 0;
                    for (int s = 0; s < p.stages; s++)
                        if (issued & (1u << s))
                            wait_parity(bar_full + 8 * s, (parity >> s) & 1, p.ctl.drain_timeout_ns, &never);
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            if (elect_one()) {
                const uint32_t idesc = idesc_f16(kBf16, kAmn, false, 128, (uint32_t)n16);
                const uint64_t a_desc = operand_desc<kAmn>(base), b_desc = operand_desc<false>(base + kTileBytes);
                uint32_t stage = 0, phase = 0;
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!spin_parity(bar_full + 8 * stage, phase, tmo, abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        break;
                    }
                    tc_fence_after();
                    const uint64_t a = a_desc + (uint64_t)(stage * (slot >> 4));
                    const uint64_t b = b_desc + (uint64_t)(stage * (slot >> 4));
                    const int steps = min(4, (p.red - kb * kBlockK + 15) / 16);
                    for (int j = 0; j < steps; j++)
                        mma_f16(tmem_base, a + j * kStep16<kAmn>, b + j * kStep16<false>, idesc,
                                kb != kb0 || j != 0 ? 1u : 0u);
                    mma_commit(bar_empty + 8 * stage);
                    if (++stage == (uint32_t)p.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                mma_commit(bar_acc);  // after an abort too: what was issued has then finished
            }
            __syncwarp();
        } else {
            // every MMA has read its slot, so the ring's memory takes the partial tile
            if (!warp_wait_parity(bar_acc, 0, tmo, abort_flag, lane)) {
                if (lane == 0) report_timeout(abort_flag, p.ctl.status);
            }
            tc_fence_after();
            const int quarter = warp & 3;
            const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16);
            for (int c = 0; c < n16; c += 16) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(acc + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; i++) part[(c + i) * 128 + quarter * 32 + lane] = __uint_as_float(r[i]);
            }
            tc_fence_before();
        }
        if (splits > 1) warp_cluster_sync();
        else __syncthreads();

        // each CTA of the cluster finishes its share of the tokens, whole rows of the tile
        const int share = (rows + splits - 1) / splits, t0 = min(rows, split * share), t1 = min(rows, t0 + share);
        const uint32_t part_addr = base;
        const int feat0 = f * 128;
        if (p.act == kActSwiglu) {
            for (int i = t0 * 8 + (int)threadIdx.x; i < t1 * 8; i += kDecThreads) {
                const int t = i >> 3, c = i & 7;  // 8 of the tile's 64 outputs
                const int gf = (c >> 1) * 32 + (c & 1) * 8;
                if (feat0 + gf >= p.features) continue;
                float gate[8], up[8];
                sum_parts(part_addr + (t * 128 + gf) * 4, splits, gate);
                sum_parts(part_addr + (t * 128 + gf + 16) * 4, splits, up);
                add_bias<T>(p.bias, (int64_t)g * p.features + feat0 + gf, gate);
                add_bias<T>(p.bias, (int64_t)g * p.features + feat0 + gf + 16, up);
                if (p.z) {
                    put8<T>(p.z, (int64_t)(r0 + t) * p.features + feat0 + gf, gate);
                    put8<T>(p.z, (int64_t)(r0 + t) * p.features + feat0 + gf + 16, up);
                }
                const int64_t at = (int64_t)(r0 + t) * p.out_cols + feat0 / 2 + c * 8;
#pragma unroll
                for (int k = 0; k < 8; k++) gate[k] = gate[k] * sigma(gate[k]) * up[k];
                add_row<T>(p.residual, at, gate);
                put8<T>(p.y, at, gate);
            }
        } else {
            for (int i = t0 * 16 + (int)threadIdx.x; i < t1 * 16; i += kDecThreads) {
                const int t = i >> 4, c = (i & 15) * 8;
                if (feat0 + c >= p.features) continue;
                float v[8];
                sum_parts(part_addr + (t * 128 + c) * 4, splits, v);
                add_bias<T>(p.bias, (int64_t)g * p.features + feat0 + c, v);
                const int64_t at = (int64_t)(r0 + t) * p.out_cols + feat0 + c;
                if (p.z) put8<T>(p.z, at, v);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (p.act == kActRelu) v[k] = act<kActRelu>(v[k]);
                    if (p.act == kActSilu) v[k] = act<kActSilu>(v[k]);
                    if (p.act == kActGeluTanh) v[k] = act<kActGeluTanh>(v[k]);
                }
                add_row<T>(p.residual, at, v);
                put8<T>(p.y, at, v);
            }
        }
        if (splits > 1) warp_cluster_sync();  // the others may still read this CTA's part
    }
    if (p.m_offsets) {  // rows outside every group are zero
        int lo, hi, unused;
        group_rows(p.m_offsets, 0, p.m_total, lo, unused);
        group_rows(p.m_offsets, p.groups - 1, p.m_total, unused, hi);
        const int outside = lo + p.m_total - hi;
        for (int i = blockIdx.x; i < outside; i += gridDim.x) {
            const int64_t row = i < lo ? i : hi + (i - lo);
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            for (int c = threadIdx.x; c < p.out_cols / 8; c += kDecThreads)
                reinterpret_cast<uint4 *>(static_cast<T *>(p.y) + row * p.out_cols)[c] = zero;
            if (p.z)
                for (int c = threadIdx.x; c < p.features / 8; c += kDecThreads)
                    reinterpret_cast<uint4 *>(static_cast<T *>(p.z) + row * p.features)[c] = zero;
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, tmem_cols);
    }
}

void plan_decode(int form, int groups, int m_total, int features, int red, int sm_count, Plan *plan) {
    const int n_f = (features + 127) / 128;
    const int64_t tiles = (int64_t)n_f * std::min(groups, m_total);
    const int nkb = (red + kBlockK - 1) / kBlockK;
    plan->decode = 1;
    // split while every CTA still fits on the GPU at once (two an SM) and has 4 slots to load
    plan->splits = 1;
    while (plan->splits < kDecMaxSplits && tiles * plan->splits * 2 <= 2 * sm_count && nkb >= plan->splits * 8)
        plan->splits *= 2;
    // use_decode() keeps the grid within two CTAs an SM, so all of them are resident at once
    plan->tiles = tiles * plan->splits;
    const int slot = kTileBytes + ((m_total + 15) & ~15) * 128;
    plan->stages = std::max(2, std::min(kDecMaxStages, (kDecSmem - 1024 - kDecBarBytes) / slot));
    // The forward form only.  A programmatic dependent inside the gradient's launches is what
    // once stopped a stream (linear.cu), so the input gradient waits its turn.
    plan->programmatic = form == kForward;
}

template <typename T, int FORM>
int decode_product(const void *X, int64_t ldx, const void *W, Params p, const Plan &plan, int red, const DeviceInfo &di,
                   cudaStream_t s) {
    if (p.m_total > kDecodeTokens) return NVFP4_ERR_SHAPE;
    if (plan.tiles > INT_MAX) return NVFP4_ERR_SHAPE;
    p.red = red;
    p.ncap = (p.m_total + 15) & ~15;
    p.splits = plan.splits;
    p.stages = plan.stages;
    const int smem = p.stages * (kTileBytes + p.ncap * 128) + kDecBarBytes + 1024;
    CUtensorMap a, b;
    int st = FORM == kDgrad ? map_weight<T>(&a, W, p.groups, red, p.features, 64)
                            : map_weight<T>(&a, W, p.groups, p.features, red, 128);
    if (!st) st = map_rows<T>(&b, X, p.m_total, red, ldx, 16);
    if (st) return st;
    auto kern = linear_decode_kernel<T, FORM>;
    static int configured[64] = {};
    if (!configured[di.device]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kDecSmem) != cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)plan.tiles);
    cfg.blockDim = dim3(kDecThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = plan.programmatic ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kern, a, b, p) != cudaSuccess) return NVFP4_ERR_CUDA;
    count_launch();
    return cuda_status(cudaGetLastError());
}

#define INSTANCE(T, FORM) \
    template int decode_product<T, FORM>(const void *, int64_t, const void *, Params, const Plan &, int, \
                                         const DeviceInfo &, cudaStream_t)
INSTANCE(__nv_bfloat16, kForward);
INSTANCE(__half, kForward);
INSTANCE(__nv_bfloat16, kDgrad);
INSTANCE(__half, kDgrad);
#undef INSTANCE

}  // namespace linear
}  // namespace nvfp4
