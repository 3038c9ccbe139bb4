// moe_products.cu — moe_layer where its experts have several rows each: the tokens' rows put in
// expert order, W13's product with SwiGLU in its epilogue (nvfp4_linear), and here W2's product
// with fp32 results and their weighted sum.
//
// Bound by the weights' bytes.  An expert's rows, 64 at most, are the MMA's N, so each weight is
// read once.  The list of all 64-element slots of the reduction, by active expert, tile of 128
// weight rows and slot, is cut into equal pieces, one a CTA, two CTAs an SM: whatever the number
// of experts and tiles, all SMs read the same number of bytes.  A tile that is cut leaves parts,
// in an order that follows from the sizes alone; the sum adds them in that order, so the same
// inputs give the same bits.
//
// The results stay in fp32 up to the sum: rounded to 16 bits, as the rows of a product by
// itself are, they would add as much error as the hidden rows' rounding does (bf16, 32 tokens by
// 8 of 8 experts: 0.0029 of the output's norm against 0.0024, where the output's own rounding
// alone is 0.0017).
//
// Measured, all launches on the GPU: 32 tokens by 2 of 8 of 4096 x 14336 442 us (6.4 TB/s of a
// copy's 6.55), 64 by 6 of 64 of 2048 x 2048 266 (6.1), 64 by 8 of 8 of 2048 x 4096 103 (3.9: the
// router 8, W13 52, W2 28, the sum 6 and the launches' gaps; their bytes would take 61).
//
// Warps: 0 TMA producer, 1 MMA issue and TMEM owner, 2-5 write the accumulators out, under the
// next tile's loads and products.
#include <algorithm>
#include <atomic>
#include <climits>

#include "linear.cuh"
#include "moe_products.cuh"

namespace nvfp4 {
namespace moe_products {

using namespace linear;

constexpr int kThreads = 192;
constexpr int kResident = 2;        // CTAs an SM
constexpr int kMaxStages = 8;
constexpr int kRing = 108 * 1024;   // of a CTA
constexpr int kMinSlots = 4;        // of a CTA's piece, if there are as many
constexpr int kExperts = kMaxGroups;
constexpr int kGatherThreads = 256;
constexpr int kSumThreads = 256;
constexpr int kSumTokens = kSumThreads / 32;  // of a CTA: 32 threads of 4 columns each

// How the reduction's slots are cut into pieces.  A tile has at most kMaxParts of them: no more
// pieces than 3 a tile are made, none of less than kMinSlots.
struct Cut {
    int64_t slots, pieces;
    int per;     // slots of a tile
    bool small;  // products of slots and pieces are 32-bit numbers, whose division is short
    __device__ __forceinline__ Cut(int active, int tiles, int per_tile, int ctas) : per(per_tile) {
        slots = (int64_t)active * tiles * per;
        pieces = max((int64_t)1, min(min((int64_t)ctas, slots / kMinSlots), (int64_t)active * tiles * 3));
        small = (slots + 1) * pieces < ((int64_t)1 << 32);
    }
    __device__ __forceinline__ int64_t begin(int64_t piece) const {
        return small ? (uint32_t)(slots * piece) / (uint32_t)pieces : slots * piece / pieces;
    }
    __device__ __forceinline__ int piece_of(int64_t slot) const {
        const int64_t n = (slot + 1) * pieces - 1;
        return (int)(small ? (uint32_t)n / (uint32_t)slots : n / slots);
    }
};

__global__ void __launch_bounds__(kGatherThreads)
    gather_kernel(const uint4 *x, int64_t ld, const int *rows, uint4 *out, int k, int total, int vecs) {
    const int choice = blockIdx.y, c = blockIdx.x * kGatherThreads + threadIdx.x;
    const int r = rows[choice];
    if (c < vecs && r >= 0 && r < total) out[(int64_t)r * vecs + c] = __ldg(x + choice / k * ld + c);
}

struct DownParams {
    const int *m_offsets;
    float *part;
    uint8_t *parts;  // [E][tiles]: how many a tile has
    int E, R, K, F;
    int stages, ncap, ctas;
    KernelCtl ctl;
};

template <typename T>
__global__ void __launch_bounds__(kThreads, kResident)
    down_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_h,
                const DownParams p) {
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ uint64_t bars[2 * kMaxStages + 5];
    __shared__ short act_e[kExperts], act_row[kExperts], act_n[kExperts];
    __shared__ int n_active, abort_word;
    __shared__ uint32_t tmem_at;
    volatile int *abort_flag = &abort_word;
    const uint32_t slot_bytes = kTileBytes + (uint32_t)p.ncap * 128u;  // weight rows, then the expert's rows
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kMaxStages;
    const uint32_t acc_full = bar_empty + 8 * kMaxStages, acc_empty = acc_full + 16, bar_done = acc_empty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t tmem_cols = p.ncap <= 16 ? 32u : p.ncap <= 32 ? 64u : 128u;  // two accumulators
    const uint64_t tmo = p.ctl.wait_timeout_ns;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxStages; i++) {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 4);
        }
        mbar_init(bar_done, 1);
        abort_word = 0;
        fence_barrier_init();
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_h);
    }
    __syncwarp();
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_at), tmem_cols);
        tmem_relinquish();
    } else if (warp == 2) {
        int n = 0;
        for (int b = 0; b < p.E; b += 32) {
            int r0 = 0, r1 = 0;
            if (b + lane < p.E) group_rows(p.m_offsets, b + lane, p.R, r0, r1);
            const uint32_t live = __ballot_sync(0xffffffffu, r1 > r0);
            if (r1 > r0) {
                const int at = n + __popc(live & ((1u << lane) - 1u));
                act_e[at] = (short)(b + lane);
                act_row[at] = (short)r0;
                act_n[at] = (short)min(r1 - r0, p.ncap);
            }
            n += __popc(live);
        }
        if (lane == 0) n_active = n;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    const int tiles = (p.K + 127) / 128;
    const Cut cut(n_active, tiles, (p.F + kBlockK - 1) / kBlockK, p.ctas);
    const bool mine = cut.slots > 0 && blockIdx.x < cut.pieces;
    const int64_t i0 = mine ? cut.begin(blockIdx.x) : 0, i1 = mine ? cut.begin((int64_t)blockIdx.x + 1) : 0;
    // the tile that a slot belongs to, by active expert and tile, and the slot in it
    const int64_t tile0 = !mine ? 0 : i0 >> 31 ? i0 / cut.per : (uint32_t)i0 / (uint32_t)cut.per;
    const int a0 = (int)(tile0 / tiles), f0 = (int)(tile0 - (int64_t)a0 * tiles);
    const int s0 = (int)(i0 - tile0 * cut.per);

    if (warp == 0) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0, parity = 0;
            int a = a0, f = f0, s = s0;
            bool ok = true;
            for (int64_t i = i0; i < i1; i++) {
                if (!wait_parity(bar_empty + 8 * stage, phase ^ 1, tmo, abort_flag)) {
                    report_timeout(abort_flag, p.ctl.status);
                    ok = false;
                    break;
                }
                const uint32_t bar = bar_full + 8 * stage, to = base + stage * slot_bytes;
                const int n16 = (act_n[a] + 15) & ~15;
                mbar_arrive_expect_tx(bar, kTileBytes + (uint32_t)n16 * 128u);
                issued |= 1u << stage;
                parity = (parity & ~(1u << stage)) | (phase << stage);
                tma_load_3d(to, &tmap_w, bar, s * kBlockK, f * 128, act_e[a]);
                for (int c = 0; c < n16; c += 16)
                    tma_load_2d(to + kTileBytes + c * 128, &tmap_h, bar, s * kBlockK, act_row[a] + c);
                if (++stage == (uint32_t)p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
                if (++s == cut.per) {
                    s = 0;
                    if (++f == tiles) {
                        f = 0;
                        a++;
                    }
                }
            }
            // the MMAs' last arrivals have to come before the CTA ends
            for (int j = 0; ok && j < p.stages; j++) {
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
                for (int j = 0; j < p.stages; j++)
                    if (issued & (1u << j))
                        wait_parity(bar_full + 8 * j, (parity >> j) & 1, p.ctl.drain_timeout_ns, &never);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint64_t a_desc = operand_desc<false>(base), b_desc = operand_desc<false>(base + kTileBytes);
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, idesc = 0;
            int a = a0, f = f0, s = s0;
            for (int64_t i = i0; i < i1; i++) {
                const bool first = i == i0 || s == 0;
                if (first) {
                    if (!wait_parity(acc_empty + 8 * acc, acc_phase ^ 1, tmo, abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        break;
                    }
                    idesc = idesc_f16(kBf16, false, false, 128, (uint32_t)((act_n[a] + 15) & ~15));
                }
                if (!spin_parity(bar_full + 8 * stage, phase, tmo, abort_flag)) {
                    report_timeout(abort_flag, p.ctl.status);
                    break;
                }
                tc_fence_after();
                const uint64_t da = a_desc + (uint64_t)(stage * (slot_bytes >> 4));
                const uint64_t db = b_desc + (uint64_t)(stage * (slot_bytes >> 4));
                const int steps = min(4, (p.F - s * kBlockK + 15) / 16);
                for (int j = 0; j < steps; j++)
                    mma_f16(tmem + acc * p.ncap, da + j * kStep16<false>, db + j * kStep16<false>, idesc,
                            !first || j != 0 ? 1u : 0u);
                mma_commit(bar_empty + 8 * stage);
                if (++stage == (uint32_t)p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
                const bool last = i + 1 == i1 || s + 1 == cut.per;
                if (last) {
                    mma_commit(acc_full + 8 * acc);
                    acc ^= 1;
                    if (!acc) acc_phase ^= 1;
                }
                if (++s == cut.per) {
                    s = 0;
                    if (++f == tiles) {
                        f = 0;
                        a++;
                    }
                }
            }
            // after an abort too: nothing is in flight when the accumulators are given back
            volatile int never = 0;
            mma_commit(bar_done);
            if (!wait_parity(bar_done, 0, p.ctl.drain_timeout_ns, &never)) report_timeout(abort_flag, p.ctl.status);
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3;
        uint32_t acc = 0, acc_phase = 0;
        int a = a0, f = f0, s = s0;
        for (int64_t i = i0; i < i1;) {
            const int n = (int)min(i1 - i, (int64_t)(cut.per - s));  // slots of this tile
            if (!warp_wait_parity(acc_full + 8 * acc, acc_phase, tmo, abort_flag, lane)) {
                if (lane == 0) report_timeout(abort_flag, p.ctl.status);
                break;
            }
            tc_fence_after();
            const int part = (int)blockIdx.x - cut.piece_of(i - s), feature = f * 128 + quarter * 32 + lane;
            if (s + n == cut.per && quarter == 0 && lane == 0) p.parts[act_e[a] * tiles + f] = (uint8_t)(part + 1);
            float *to = p.part + ((int64_t)part * p.R + act_row[a]) * p.K + feature;
            const int rows = act_n[a];
            const uint32_t from = tmem + acc * p.ncap + ((uint32_t)(quarter * 32) << 16);
            for (int c = 0; c < rows; c += 16) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(from + c, r);
                tmem_ld_wait();
                if (feature < p.K)
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c + j < rows) to[(int64_t)(c + j) * p.K] = __uint_as_float(r[j]);
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + 8 * acc);
            acc ^= 1;
            if (!acc) acc_phase ^= 1;
            i += n;
            s = 0;
            if (++f == tiles) {
                f = 0;
                a++;
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, tmem_cols);
    }
}

struct SumParams {
    const float *part, *weights;
    const uint8_t *parts;
    const int *experts, *rows;
    const void *residual;
    void *y;
    int T, k, R, K;
};

// 128 columns (a tile's) of kSumTokens tokens.
template <typename T>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const SumParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tile = blockIdx.x;
    const int t = blockIdx.y * kSumTokens + warp, col = tile * 128 + lane * 4;
    if (t >= p.T) return;
    int row = -1, count = 0;  // of the token's choice `lane`
    float weight = 0.0f;
    if (lane < p.k) {
        row = p.rows[t * p.k + lane];
        weight = p.weights[t * p.k + lane];
        const int expert = p.experts[t * p.k + lane];
        if (row >= 0 && row < p.R) count = p.parts[expert * (int)gridDim.x + tile];
    }
    const bool in = col < p.K;
    const int64_t at = (int64_t)t * p.K + col;
    uint2 res = make_uint2(0u, 0u);
    if (p.residual && in) res = *reinterpret_cast<const uint2 *>(static_cast<const T *>(p.residual) + at);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < p.k; j0 += 8) {
        float4 v[8][2];
        float w[8];
        int n[8], r[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            r[j] = __shfl_sync(0xffffffffu, row, j0 + j);
            n[j] = __shfl_sync(0xffffffffu, count, j0 + j);
            w[j] = __shfl_sync(0xffffffffu, weight, j0 + j);
#pragma unroll
            for (int i = 0; i < 2; i++)
                v[j][i] = in && i < n[j] ? *reinterpret_cast<const float4 *>(p.part + ((int64_t)i * p.R + r[j]) * p.K + col)
                                         : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float4 o = make_float4(v[j][0].x + v[j][1].x, v[j][0].y + v[j][1].y, v[j][0].z + v[j][1].z,
                                   v[j][0].w + v[j][1].w);
            for (int i = 2; in && i < n[j]; i++) {
                const float4 u = *reinterpret_cast<const float4 *>(p.part + ((int64_t)i * p.R + r[j]) * p.K + col);
                o.x += u.x;
                o.y += u.y;
                o.z += u.z;
                o.w += u.w;
            }
            if (n[j]) {
                s.x = fmaf(w[j], o.x, s.x);
                s.y = fmaf(w[j], o.y, s.y);
                s.z = fmaf(w[j], o.z, s.z);
                s.w = fmaf(w[j], o.w, s.w);
            }
        }
    }
    if (!in) return;
    if (p.residual) {
        const float2 lo = Type16<T>::unpack(res.x), hi = Type16<T>::unpack(res.y);
        s.x += lo.x;
        s.y += lo.y;
        s.z += hi.x;
        s.w += hi.y;
    }
    *reinterpret_cast<uint2 *>(static_cast<T *>(p.y) + at) =
        make_uint2(Type16<T>::pack(s.x, s.y), Type16<T>::pack(s.z, s.w));
}

template <typename T>
static int run_t(const Args &a, const DeviceInfo &di, cudaStream_t s) {
    const int R = a.T * a.k, vecs = a.K / 8;
    gather_kernel<<<dim3((unsigned)((vecs + kGatherThreads - 1) / kGatherThreads), (unsigned)R), kGatherThreads, 0, s>>>(
        static_cast<const uint4 *>(a.x), a.ldx / 8, a.rows, static_cast<uint4 *>(a.x_rows), a.k, R, vecs);
    count_launch();
    int st = cuda_status(cudaGetLastError());
    if (!st)
        st = nvfp4_linear(a.x_rows, a.K, a.w13, nullptr, nullptr, a.h, nullptr, a.m_offsets, a.E, R, 2 * a.F, a.K,
                          NVFP4_ACT_SWIGLU, a.dtype, s);
    if (st) return st;

    DownParams d = {};
    d.m_offsets = a.m_offsets;
    d.part = a.part;
    d.parts = a.parts;
    d.E = a.E;
    d.R = R;
    d.K = a.K;
    d.F = a.F;
    d.ncap = (a.T + 15) & ~15;  // a token chooses an expert once
    d.stages = std::min(kMaxStages, kRing / (kTileBytes + d.ncap * 128));
    d.ctas = kResident * di.sm_count;
    if ((st = kernel_ctl(&d.ctl))) return st;
    CUtensorMap w, h;
    if ((st = map_weight<T>(&w, a.w2, a.E, a.K, a.F, 128))) return st;
    if ((st = map_rows<T>(&h, a.h, R, a.F, a.F, 16))) return st;
    auto kern = down_kernel<T>;
    static std::atomic<bool> configured[64] = {};
    if (!configured[di.device].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing + 1024) != cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device].store(true, std::memory_order_release);
    }
    kern<<<(unsigned)d.ctas, kThreads, d.stages * (kTileBytes + d.ncap * 128) + 1024, s>>>(w, h, d);
    count_launch();
    if ((st = cuda_status(cudaGetLastError()))) return st;

    SumParams m = {};
    m.part = a.part;
    m.parts = a.parts;
    m.weights = a.weights;
    m.experts = a.experts;
    m.rows = a.rows;
    m.residual = a.residual;
    m.y = a.y;
    m.T = a.T;
    m.k = a.k;
    m.R = R;
    m.K = a.K;
    sum_kernel<T><<<dim3((unsigned)((a.K + 127) / 128), (unsigned)((a.T + kSumTokens - 1) / kSumTokens)), kSumThreads, 0,
                    s>>>(m);
    count_launch();
    return cuda_status(cudaGetLastError());
}

int run(const Args &a, const DeviceInfo &di, cudaStream_t stream) {
    return a.dtype == NVFP4_BF16 ? run_t<__nv_bfloat16>(a, di, stream) : run_t<__half>(a, di, stream);
}

}  // namespace moe_products
}  // namespace nvfp4
