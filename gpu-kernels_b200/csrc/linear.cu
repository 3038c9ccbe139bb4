// linear.cu — the persistent CTA-pair kernel of the 16-bit linear layers: forward with a
// fused epilogue, input gradient and weight gradient, dense or grouped by expert.
//
// A cluster of two CTAs computes 256 features x up to 256 tokens with
// tcgen05.mma.cta_group::2 (kind::f16, fp32 accumulators).  Each CTA stages its 128
// features and its half of the tokens by TMA into a ring of slots of 64 reduction elements:
// 6 of 32 KB for 256 tokens, up to 10 for smaller token tiles in the same memory.  Two
// accumulators of 256 columns fill the tensor memory, so the epilogue of one tile runs under
// the MMAs of the next; or, for "wide" tiles, one tile of up to 512 tokens uses both: each A
// tile is then read once for twice the tokens, which pays where there is one round of tiles to
// run, or a long reduction (token_tile).
//
// Launched in plain stream order, as all kernels of the gradient are, the split-reduction
// kernel's input gradient among them: as programmatic dependents of each other they gained
// nothing (415 us a step of 64 experts either way) and stopped for good once in about 10^5
// steps, none of their bounded waits running.  The cause was not found.
//
// Large products are held by the power cap.  Calls in turn with the library's 16-bit product,
// with pauses / kept busy for seconds, us: 8192^3 with residual 797/849 (1.38/1.30 PFLOP/s)
// against 812/782 without; 8192 x 28672 x 8192 2903/2949 against 2967/2748; of 4096 x 14336 x
// 4096 the input gradient 380/377 against 370/366, the weight gradient 353 against 366.  Small
// tiles are held by L2: a CTA takes about 98 GB/s whatever the number of slots.  The barriers
// of a slot have CTA scope: announcing each CTA's own bytes on the leader's barrier with
// cluster-scope arrivals, and acquiring at cluster scope, took 1416 us for 8192^3.
//
// Warps: 0 TMA producer, 1 MMA issue (leader CTA) and TMEM owner, 2-9 epilogue, 10 (wgrad)
// clears the rows past a group's end in its last slot.
#include <algorithm>
#include <climits>

#include "linear.cuh"

namespace nvfp4 {
namespace linear {

constexpr int kMaxStages = 12;
constexpr int kRingBytes = 6 * 2 * kTileBytes;  // p.stages slots of A (16 KB) and B (bt * 64 bytes)
constexpr int kEpiWarps = 8;
constexpr int kTailWarp = 2 + kEpiWarps;
constexpr int kThreads = 32 * (kTailWarp + 1);
constexpr int kMaxTokens = 256;  // of a tile
constexpr int kAccCols = 256;

constexpr int kBox = 32 * 64;  // wgrad: 32 rows x 32 columns; two a warp, one of them in what the ring leaves
constexpr int kOffStage = kRingBytes;  // per epilogue warp 2 KB: 32 tokens x 32 features
constexpr int kStageWarp = 32 * 64;
constexpr int kOffBar = kOffStage + kEpiWarps * kStageWarp;
constexpr int kBarBytes = 512;
constexpr int kOffTables = kOffBar + kBarBytes;
constexpr int kSmem = kOffTables + 3 * (kMaxGroups + 1) * 4 + 1024;
static_assert(kSmem <= 232448, "shared memory budget");

struct Tile {
    int group, f;     // group and feature tile (256 features)
    int row0, rows;   // forward / dgrad: first token row and tokens of the tile; wgrad: the group's rows
    int col;          // wgrad: column tile
};

// One 32-token x 32-feature piece of the accumulator (a warp's lane quarter): fragments to
// outputs.  v[q][i] packs nothing yet: feature quarter q (l/4 + 8q), tokens 8i + 2(l%4), +1.
template <typename T, int ACT>
__device__ __forceinline__ void store_piece(const Params &p, uint32_t (&ra)[16], uint32_t (&rb)[16], uint32_t stage,
                                            const float (&bias)[4], int row0, int n_rows, int feat0, int lane) {
    constexpr bool kGlu = ACT == kActSwiglu;
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            ra[4 * i + e] = __float_as_uint(__uint_as_float(ra[4 * i + e]) + bias[0]);
            ra[4 * i + 2 + e] = __float_as_uint(__uint_as_float(ra[4 * i + 2 + e]) + bias[1]);
            rb[4 * i + e] = __float_as_uint(__uint_as_float(rb[4 * i + e]) + bias[2]);
            rb[4 * i + 2 + e] = __float_as_uint(__uint_as_float(rb[4 * i + 2 + e]) + bias[3]);
        }
    }
    auto pk = [&](const uint32_t *r) { return Type16<T>::pack(__uint_as_float(r[0]), __uint_as_float(r[1])); };
    // staging: 64 bytes a token, its 16-byte chunks permuted by the token so that the eight
    // rows of a matrix, and the eight lanes of a read, each touch all banks once
    const int mj = lane >> 3, mi = lane & 7;
    auto stage64 = [&](int i) {  // matrix mj = features 8 mj.., tokens 8 i + mi
        const int t = 8 * i + mi;
        return stage + t * 64 + ((mj ^ ((t >> 1) & 3)) << 4);
    };
    auto copy_out64 = [&](void *dst, int cols, int f0) {
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const int t = it * 8 + (lane >> 2), c = lane & 3;
            uint32_t a, b, cc, d;
            ld_shared_v4(stage + t * 64 + ((c ^ ((t >> 1) & 3)) << 4), a, b, cc, d);
            if (t < n_rows && f0 + c * 8 < cols)
                *reinterpret_cast<uint4 *>(static_cast<T *>(dst) + (int64_t)(row0 + t) * cols + f0 + c * 8) =
                    make_uint4(a, b, cc, d);
        }
        __syncwarp();
    };
    if (p.z) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            stmatrix_x4_trans(stage64(i), pk(ra + 4 * i), pk(ra + 4 * i + 2), pk(rb + 4 * i), pk(rb + 4 * i + 2));
        copy_out64(p.z, p.features, feat0);
    }
    if constexpr (!kGlu) {
        if (p.residual) {
#pragma unroll
            for (int it = 0; it < 4; it++) {
                const int t = it * 8 + (lane >> 2), c = lane & 3;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (t < n_rows && feat0 + c * 8 < p.out_cols)
                    v = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) +
                                                         (int64_t)(row0 + t) * p.out_cols + feat0 + c * 8);
                st_shared_v4(stage + t * 64 + ((c ^ ((t >> 1) & 3)) << 4), v.x, v.y, v.z, v.w);
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                o[e] = act<ACT>(__uint_as_float(ra[4 * i + e]));
                o[4 + e] = act<ACT>(__uint_as_float(rb[4 * i + e]));
            }
            if (p.residual) {
                uint32_t w[4];
                ldmatrix_x4_trans(stage64(i), w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float2 f = Type16<T>::unpack(w[q]);
                    o[2 * q] += f.x;
                    o[2 * q + 1] += f.y;
                }
            }
            stmatrix_x4_trans(stage64(i), Type16<T>::pack(o[0], o[1]), Type16<T>::pack(o[2], o[3]),
                              Type16<T>::pack(o[4], o[5]), Type16<T>::pack(o[6], o[7]));
        }
        copy_out64(p.y, p.out_cols, feat0);
    } else {
        // lanes 0-15 of the quarter are gate features, 16-31 up: 16 output features, 32 bytes
        // a token; two token groups a matrix instruction
        const int f0 = feat0 >> 1;
        auto stage32 = [&](int i) {
            const int t = 8 * (i + (mj >> 1)) + mi;
            return stage + t * 32 + (((mj & 1) ^ ((t >> 2) & 1)) << 4);
        };
        if (p.residual) {
#pragma unroll
            for (int it = 0; it < 2; it++) {
                const int t = it * 16 + (lane >> 1), c = lane & 1;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (t < n_rows && f0 + c * 8 < p.out_cols)
                    v = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) +
                                                         (int64_t)(row0 + t) * p.out_cols + f0 + c * 8);
                st_shared_v4(stage + t * 32 + ((c ^ ((t >> 2) & 1)) << 4), v.x, v.y, v.z, v.w);
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float o[8];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float g = __uint_as_float(ra[4 * (i + h) + e]), u = __uint_as_float(rb[4 * (i + h) + e]);
                    o[4 * h + e] = g * sigma(g) * u;
                }
            if (p.residual) {
                uint32_t w[4];
                ldmatrix_x4_trans(stage32(i), w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float2 f = Type16<T>::unpack(w[q]);
                    o[2 * q] += f.x;
                    o[2 * q + 1] += f.y;
                }
            }
            stmatrix_x4_trans(stage32(i), Type16<T>::pack(o[0], o[1]), Type16<T>::pack(o[2], o[3]),
                              Type16<T>::pack(o[4], o[5]), Type16<T>::pack(o[6], o[7]));
        }
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 2; it++) {
            const int t = it * 16 + (lane >> 1), c = lane & 1;
            uint32_t a, b, cc, d;
            ld_shared_v4(stage + t * 32 + ((c ^ ((t >> 2) & 1)) << 4), a, b, cc, d);
            if (t < n_rows && f0 + c * 8 < p.out_cols)
                *reinterpret_cast<uint4 *>(static_cast<T *>(p.y) + (int64_t)(row0 + t) * p.out_cols + f0 + c * 8) =
                    make_uint4(a, b, cc, d);
        }
        __syncwarp();
    }
}

template <typename T, int FORM>
__device__ __forceinline__ void store_act(const Params &p, uint32_t (&ra)[16], uint32_t (&rb)[16], uint32_t stage,
                                          const float (&bias)[4], int row0, int n_rows, int feat0, int lane) {
    switch (FORM == kForward ? p.act : (int)kActNone) {
        case kActRelu: store_piece<T, kActRelu>(p, ra, rb, stage, bias, row0, n_rows, feat0, lane); break;
        case kActSilu: store_piece<T, kActSilu>(p, ra, rb, stage, bias, row0, n_rows, feat0, lane); break;
        case kActGeluTanh: store_piece<T, kActGeluTanh>(p, ra, rb, stage, bias, row0, n_rows, feat0, lane); break;
        case kActSwiglu: store_piece<T, kActSwiglu>(p, ra, rb, stage, bias, row0, n_rows, feat0, lane); break;
        default: store_piece<T, kActNone>(p, ra, rb, stage, bias, row0, n_rows, feat0, lane);
    }
}

template <typename T, int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_d, const Params p) {
    constexpr bool kAmn = FORM != kForward, kBmn = FORM == kWgrad;
    constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const int n_stages = p.stages;
    const int subs_max = FORM == kWgrad ? 1 : 1 + p.wide, tile_tokens = p.bt * subs_max;
    const uint32_t sub_bytes = (uint32_t)p.bt * 64u;  // this CTA's half of bt tokens
    const uint32_t slot = kTileBytes + sub_bytes * subs_max;  // a slot: A, then B
    const uint32_t sA = base, sB = base + kTileBytes;
    const uint32_t bar_full = base + kOffBar;            // [stages], leader's used: both CTAs' data
    const uint32_t bar_empty = bar_full + 8 * kMaxStages;   // [stages]
    const uint32_t bar_tail = bar_empty + 8 * kMaxStages;   // [stages] wgrad: a group's last slot has landed
    const uint32_t bar_ready = bar_tail + 8 * kMaxStages;   // [stages] wgrad: that slot is cleared in both CTAs
    const uint32_t bar_acc_full = bar_ready + 8 * kMaxStages;
    const uint32_t bar_acc_empty = bar_acc_full + 16;
    const uint32_t bar_drain = bar_acc_empty + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(base_ptr + kOffBar + (4 * kMaxStages + 5) * 8);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    static_assert((4 * kMaxStages + 5) * 8 + 8 <= kBarBytes, "barrier region");
    int *g_r0 = reinterpret_cast<int *>(base_ptr + kOffTables);
    int *g_r1 = g_r0 + kMaxGroups + 1;
    int *g_t0 = g_r1 + kMaxGroups + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const int n_f = (p.features + 255) / 256;
    const int n_c = FORM == kWgrad ? (p.out_cols + p.bt - 1) / p.bt : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < n_stages; s++) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
            mbar_init(bar_tail + 8 * s, 1);
            mbar_init(bar_ready + 8 * s, 2);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(bar_acc_full + 8 * b, 1);
            mbar_init(bar_acc_empty + 8 * b, 2 * kEpiWarps);
        }
        mbar_init(bar_drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    __syncwarp();
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);
        tmem_relinquish_pair();
    }
    if (warp == 2)
        build_tables(p.m_offsets, p.groups, p.m_total, FORM == kWgrad ? 0 : tile_tokens, FORM == kWgrad ? n_f * n_c : n_f,
                     lane, g_r0, g_r1, g_t0);
    tc_fence_before();
    warp_cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint64_t tmo = p.ctl.wait_timeout_ns;
    const int n_tiles = g_t0[p.groups];

    // Strips of p.strip feature tiles sweep a group's tokens (wgrad: columns) together, the
    // features fastest: the pairs that run at the same time share both operands in L2.
    auto tile_at = [&](int t) {
        Tile ti;
        int lo = 0, hi = p.groups - 1;  // the last group with g_t0[g] <= t
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (g_t0[mid] <= t) lo = mid; else hi = mid - 1;
        }
        ti.group = lo;
        const int r0 = g_r0[lo], n = g_r1[lo] - r0;
        const int others = FORM == kWgrad ? n_c : (n + tile_tokens - 1) / tile_tokens;
        const int local = t - g_t0[lo], per_strip = p.strip * others;
        const int s = local / per_strip, f0 = s * p.strip, fs = min(p.strip, n_f - f0), rem = local - s * per_strip;
        if (FORM == kWgrad) {  // the columns fastest: 2-3 % faster than the features at 4096 x 14336 x 4096
            ti.col = rem % others;
            ti.f = f0 + rem / others;
            ti.row0 = r0;
            ti.rows = n;
        } else {
            const int o = rem / fs;
            ti.col = 0;
            ti.f = f0 + rem % fs;
            ti.row0 = r0 + o * tile_tokens;
            ti.rows = min(tile_tokens, n - o * tile_tokens);
        }
        return ti;
    };
    auto blocks_of = [&](const Tile &ti) {
        return ((FORM == kWgrad ? ti.rows : p.red) + kBlockK - 1) / kBlockK;
    };
    // Parts of a tile (two for a wide one with more than bt tokens), the tokens of each, and
    // its MMA columns: the tokens rounded up to 32, the step of N for a CTA pair (multiples of
    // 16 are for one CTA alone).  Each CTA holds half of them; the rounding's rows are loaded
    // but never stored.
    auto subs_of = [&](const Tile &ti) { return FORM != kWgrad && ti.rows > p.bt ? 2 : 1; };
    auto sub_rows = [&](const Tile &ti, int s) { return s ? ti.rows - p.bt : min(ti.rows, p.bt); };
    auto width_of = [&](const Tile &ti, int s) { return FORM == kWgrad ? p.bt : (sub_rows(ti, s) + 31) & ~31; };
    // wgrad: reduction rows past the group's end belong to the next group; the last slot's
    // are cleared unless the MMA's 16-row steps end exactly with the group
    auto dirty_tail = [&](const Tile &ti) { return FORM == kWgrad && (ti.rows & 15) != 0; };

    if (warp == 0) {
        // ------------------------------------------------------------ producer (both CTAs)
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0;
            uint32_t tail_mask = 0, tail_parity = 0;  // tail barriers used; parity of their next phase
            const uint32_t lead_full = map_to_cta(bar_full, 0), own_tail = map_to_cta(bar_tail, rank);
            bool ok = true;
            for (int t = pair; ok && t < n_tiles; t += num_pairs) {
                const Tile ti = tile_at(t);
                const int nkb = blocks_of(ti);
                const int f0 = ti.f * 256 + (int)rank * 128;
                const int b0 = FORM == kWgrad ? ti.col * p.bt + (int)rank * (p.bt / 2)
                                              : ti.row0 + (int)rank * (width_of(ti, 0) / 2);
                const int subs = subs_of(ti);
                const int b1 = subs == 2 ? ti.row0 + p.bt + (int)rank * (width_of(ti, 1) / 2) : 0;
                const uint32_t tx_bytes = kTileBytes + sub_bytes * subs;
                for (int kb = 0; kb < nkb; kb++) {
                    if (!wait_parity(bar_empty + 8 * stage, phase ^ 1, tmo, abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        ok = false;
                        break;
                    }
                    const bool tail = kb == nkb - 1 && dirty_tail(ti);
                    // both CTAs' copies complete on the leader's barrier; a slot to be cleared
                    // lands on each CTA's own tail barrier instead
                    const uint32_t bar = tail ? own_tail + 8 * stage : lead_full + 8 * stage;
                    if (tail) {
                        if (rank == 0) mbar_arrive(bar_full + 8 * stage);
                        mbar_arrive_expect_tx(bar_tail + 8 * stage, tx_bytes);
                        tail_mask |= 1u << stage;
                        tail_parity ^= 1u << stage;
                        issued_mask &= ~(1u << stage);
                    } else {
                        if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, 2 * tx_bytes);
                        issued_mask |= 1u << stage;
                        issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    }
                    const uint32_t dA = sA + stage * slot, dB = sB + stage * slot;
                    const int k0 = kb * kBlockK;
                    if constexpr (FORM == kForward) {
                        tma_load_3d_pair(dA, &tmap_a, bar, k0, f0, ti.group);
                        tma_load_2d_pair(dB, &tmap_b, bar, k0, b0);
                        if (subs == 2) tma_load_2d_pair(dB + sub_bytes, &tmap_b, bar, k0, b1);
                    } else if constexpr (FORM == kDgrad) {
                        tma_load_3d_pair(dA, &tmap_a, bar, f0, k0, ti.group);
                        tma_load_3d_pair(dA + 8192, &tmap_a, bar, f0 + 64, k0, ti.group);
                        tma_load_2d_pair(dB, &tmap_b, bar, k0, b0);
                        if (subs == 2) tma_load_2d_pair(dB + sub_bytes, &tmap_b, bar, k0, b1);
                    } else {
                        tma_load_2d_pair(dA, &tmap_a, bar, f0, ti.row0 + k0);
                        tma_load_2d_pair(dA + 8192, &tmap_a, bar, f0 + 64, ti.row0 + k0);
                        for (int c = 0; c < p.bt / 2; c += 64)
                            tma_load_2d_pair(dB + c * 128, &tmap_b, bar, b0 + c, ti.row0 + k0);
                    }
                    if (++stage == (uint32_t)n_stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // The MMAs release slots with arrivals that the tensor core sends, to the other CTA
            // too, whenever they complete; no thread's barrier orders them.  Take in the last
            // ones: one that came after this CTA's end would arrive on a barrier of the next
            // CTA here.
            for (int s = 0; ok && s < n_stages; s++) {
                if (!wait_parity(bar_empty + 8 * stage, phase ^ 1, tmo, abort_flag)) {
                    report_timeout(abort_flag, p.ctl.status);
                    ok = false;
                }
                if (++stage == (uint32_t)n_stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) {  // let the copies in flight land before the memory goes
                volatile int never = 0;
                for (int s = 0; s < n_stages; s++) {
                    if (rank == 0 && (issued_mask & (1u << s)))
                        wait_parity(bar_full + 8 * s, (issued_parity >> s) & 1, p.ctl.drain_timeout_ns, &never);
                    if (tail_mask & (1u << s))
                        wait_parity(bar_tail + 8 * s, ((tail_parity >> s) & 1) ^ 1, p.ctl.drain_timeout_ns, &never);
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issue (leader)
        if (rank == 0 && elect_one()) {
            const uint32_t empty0 = map_to_cta(bar_empty, 0), empty1 = map_to_cta(bar_empty, 1);
            const uint32_t accf0 = map_to_cta(bar_acc_full, 0), accf1 = map_to_cta(bar_acc_full, 1);
            const uint64_t a_desc = operand_desc<kAmn>(sA), b_desc = operand_desc<kBmn>(sB);
            uint32_t stage = 0, phase = 0, ready_parity = 0;
            int local = 0;  // accumulators handed over so far: buffer local & 1, its use local / 2
            bool ok = true, any = false;
            for (int t = pair; ok && t < n_tiles; t += num_pairs) {
                const Tile ti = tile_at(t);
                const int nkb = blocks_of(ti), subs = subs_of(ti);
                // a wide launch uses both accumulators in every tile
                for (int s = 0; s < subs_max && ok; s++)
                    if (!spin_parity(bar_acc_empty + 8 * ((local + s) & 1), (((local + s) >> 1) & 1) ^ 1, tmo,
                                     abort_flag)) {
                        report_timeout(abort_flag, p.ctl.status);
                        ok = false;
                    }
                if (!ok) break;
                tc_fence_after();
                const uint32_t d0 = tmem_base + (local & 1) * kAccCols, d1 = tmem_base + kAccCols;
                const uint32_t idesc0 = idesc_f16(kBf16, kAmn, kBmn, 256, (uint32_t)width_of(ti, 0));
                const uint32_t idesc1 = subs == 2 ? idesc_f16(kBf16, kAmn, kBmn, 256, (uint32_t)width_of(ti, 1)) : 0u;
                const int red = FORM == kWgrad ? ti.rows : p.red;
                for (int kb = 0; kb < nkb; kb++) {
                    bool landed = spin_parity(bar_full + 8 * stage, phase, tmo, abort_flag);
                    if (landed && kb == nkb - 1 && dirty_tail(ti)) {
                        landed = wait_parity_cluster(bar_ready + 8 * stage, (ready_parity >> stage) & 1, tmo, abort_flag);
                        ready_parity ^= 1u << stage;
                    }
                    if (!landed) {
                        report_timeout(abort_flag, p.ctl.status);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t a = a_desc + (uint64_t)(stage * (slot >> 4));
                    const uint64_t b = b_desc + (uint64_t)(stage * (slot >> 4));
                    any = true;
                    if ((kb + 1) * kBlockK <= red) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            mma_f16_pair(d0, a + j * kStep16<kAmn>, b + j * kStep16<kBmn>, idesc0,
                                         (kb | j) != 0 ? 1u : 0u);
                    } else {  // what is left, in steps of 16 (zeros past the end)
                        const int steps = (red - kb * kBlockK + 15) / 16;
                        for (int j = 0; j < steps; j++)
                            mma_f16_pair(d0, a + j * kStep16<kAmn>, b + j * kStep16<kBmn>, idesc0,
                                         (kb | j) != 0 ? 1u : 0u);
                    }
                    if (subs == 2) {
                        const uint64_t b2 = b + (sub_bytes >> 4);
                        const int steps = min(4, (red - kb * kBlockK + 15) / 16);
                        for (int j = 0; j < steps; j++)
                            mma_f16_pair(d1, a + j * kStep16<kAmn>, b2 + j * kStep16<kBmn>, idesc1,
                                         (kb | j) != 0 ? 1u : 0u);
                    }
                    mma_commit_pair(empty0 + 8 * stage);
                    mma_commit_pair(empty1 + 8 * stage);
                    if (++stage == (uint32_t)n_stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                for (int s = 0; s < subs_max; s++, local++) {
                    mma_commit_pair(accf0 + 8 * (local & 1));
                    mma_commit_pair(accf1 + 8 * (local & 1));
                }
            }
            // likewise the epilogues' last arrivals, the other CTA's among them
            for (int s = 0; ok && s < 2; s++)
                if (!spin_parity(bar_acc_empty + 8 * ((local + s) & 1), (((local + s) >> 1) & 1) ^ 1, tmo, abort_flag)) {
                    report_timeout(abort_flag, p.ctl.status);
                    ok = false;
                }
            if (!ok && any) {
                volatile int never = 0;
                mma_commit_pair(map_to_cta(bar_drain, 0));
                wait_parity(bar_drain, 0, p.ctl.drain_timeout_ns, &never);
            }
        }
    } else if (warp == kTailWarp) {
        // ------------------------------------------------------------ tail of a group (wgrad)
        // Both operands' rows past the group's end are set to zero (the next group's rows
        // may hold anything, infinities included), up to the 16-row step the MMA reads.
        if constexpr (FORM == kWgrad) {
            uint32_t slots = 0, parity = 0;  // slots used so far; parity of each tail barrier
            bool ok = true;
            for (int t = pair; ok && t < n_tiles; t += num_pairs) {
                const Tile ti = tile_at(t);
                slots += (uint32_t)blocks_of(ti);
                if (!dirty_tail(ti)) continue;
                const uint32_t stage = (slots - 1) % (uint32_t)n_stages;
                if (!warp_wait_parity(bar_tail + 8 * stage, (parity >> stage) & 1, tmo, abort_flag, lane)) {
                    if (lane == 0) report_timeout(abort_flag, p.ctl.status);
                    ok = false;
                    break;
                }
                parity ^= 1u << stage;
                const int valid = (ti.rows - 1) % kBlockK + 1, end = (valid + 15) & ~15;
                const int per = (end - valid) * 8;  // 16-byte pieces of one 64-column chunk
                for (int i = lane; i < per; i += 32) {
                    const uint32_t at = (uint32_t)(valid * 128 + i * 16) + stage * slot;
                    st_shared_v4(sA + at, 0u, 0u, 0u, 0u);
                    st_shared_v4(sA + 8192 + at, 0u, 0u, 0u, 0u);
                    for (int c = 0; c < p.bt / 2; c += 64) st_shared_v4(sB + c * 128 + at, 0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_to_cta(bar_ready + 8 * stage, 0));
                __syncwarp();
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue (warps 2..9, both CTAs)
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lead_acc_empty = map_to_cta(bar_acc_empty, 0);
        const uint32_t stage = base + kOffStage - (FORM == kWgrad ? kTileBytes : 0) +
                               (warp - 2) * (FORM == kWgrad ? 2 * kBox : kStageWarp);
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        int local = 0;
        uint32_t boxes = 0;
        bool ok = true;
        for (int t = pair; ok && t < n_tiles; t += num_pairs) {
            const Tile ti = tile_at(t);
            const int feat0 = ti.f * 256 + (int)rank * 128 + quarter * 32;
            float bias[4] = {0.f, 0.f, 0.f, 0.f};
            if (FORM == kForward && p.bias) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int f = feat0 + 8 * q + (lane >> 2);
                    if (f < p.features)
                        bias[q] = Type16<T>::load(static_cast<const T *>(p.bias) + (int64_t)ti.group * p.features + f);
                }
            }
            for (int sub = 0; sub < subs_max; sub++, local++) {
                const uint32_t buf = local & 1, use = local >> 1;
                if (!warp_wait_parity(bar_acc_full + 8 * buf, use & 1, tmo, abort_flag, lane)) {
                    if (lane == 0) report_timeout(abort_flag, p.ctl.status);
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem_base + lane_base + buf * kAccCols;
                if constexpr (FORM != kWgrad) {
                    const int rows = sub < subs_of(ti) ? sub_rows(ti, sub) : 0;
                    for (int c = half * 32; c < rows; c += 64) {
                        uint32_t ra[16], rb[16];
                        tmem_ld_16x256b_x4(acc + c, ra);
                        tmem_ld_16x256b_x4(acc + (16u << 16) + c, rb);
                        tmem_ld_wait();
                        if (feat0 >= p.features) continue;
                        store_act<T, FORM>(p, ra, rb, stage, bias, ti.row0 + sub * p.bt + c, rows - c, feat0, lane);
                    }
                } else {
                    // a lane is a row of dW: 32 rows x 32 columns at a time through shared memory,
                    // in the 64-byte swizzle, and out as one box that the tensor map clips to the
                    // group's rows and columns
                    const int cols = min(p.bt, p.out_cols - ti.col * p.bt);
                    for (int c = half * 32; c < cols; c += 64) {
                        uint32_t r[32];
                        tmem_ld_32x32b_x32(acc + c, r);
                        tmem_ld_wait();
                        if (feat0 >= p.features) continue;
                        uint32_t v[16];
#pragma unroll
                        for (int i = 0; i < 16; i++)  // a group without rows: its gradient is zero
                            v[i] = ti.rows > 0 ? Type16<T>::pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])) : 0u;
                        const uint32_t box = stage + (boxes++ & 1) * kBox;
                        if (lane == 0) bulk_wait_group_read<1>();  // the box's last store has read it
                        __syncwarp();
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            st_shared_v4(box + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4), v[4 * q], v[4 * q + 1],
                                         v[4 * q + 2], v[4 * q + 3]);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_3d(&tmap_d, box, ti.col * p.bt + c, feat0, ti.group);
                            bulk_commit_group();
                        }
                        __syncwarp();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_cta_release(lead_acc_empty + 8 * buf);
                __syncwarp();
            }
        }
        if constexpr (FORM != kWgrad)
            if (p.m_offsets) {  // rows outside every group (tokens that were not routed) are zero
                const int lo = g_r0[0], hi = g_r1[p.groups - 1], outside = lo + p.m_total - hi;
                for (int i = (int)blockIdx.x * kEpiWarps + warp - 2; i < outside; i += (int)gridDim.x * kEpiWarps) {
                    const int64_t row = i < lo ? i : hi + (i - lo);
                    auto clear = [&](void *dst, int cols) {
                        uint4 *d = reinterpret_cast<uint4 *>(static_cast<T *>(dst) + row * cols);
                        for (int c = lane; c < cols / 8; c += 32) d[c] = make_uint4(0u, 0u, 0u, 0u);
                    };
                    clear(p.y, p.out_cols);
                    if (p.z) clear(p.z, p.features);
                }
            }
        if (FORM == kWgrad && lane == 0) bulk_wait_group<0>();  // stores done before the memory goes
        __syncwarp();
    }

    __syncwarp();
    tc_fence_before();
    warp_cluster_sync();  // no CTA leaves while its peer may still signal it
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ------------------------------------------------------------------------- host side
template <typename T, int FORM>
static int launch_pair(const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &d, Params p, const Plan &plan,
                       const DeviceInfo &di, cudaStream_t stream) {
    auto kern = linear_pair_kernel<T, FORM>;
    static int configured[64] = {};
    if (!configured[di.device]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
            return NVFP4_ERR_CUDA;
        configured[di.device] = 1;
    }
    if (plan.tiles > INT_MAX) return NVFP4_ERR_SHAPE;
    p.stages = plan.stages;
    p.strip = 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(plan.tiles, di.sm_count / 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    if (cudaLaunchKernelEx(&cfg, kern, a, b, d, p) != cudaSuccess) return NVFP4_ERR_CUDA;
    count_launch();
    return cuda_status(cudaGetLastError());
}

// Tokens of a tile.  A slot of 64 reduction elements costs a pair about 150 ns for its 256
// features plus 1.07 ns a token (measured from 32 to 256 tokens, N = K = 4096), so few wide
// tiles win, unless their number fills the last round of pairs badly.
//   dense: the M tokens in n equal tiles, n chosen by rounds x cost (by the eight sizes that a
//     tile can have, so the choice takes as long for a million tokens as for a thousand);
//     or in wide tiles: two parts that share the A tile, up to 512 tokens, whose epilogue,
//     about 20 ns a token, no other tile's MMAs hide.  They pay for one round, us without /
//     with: M=333 N=14344 K=4104 70.4/54.6, M=450 78.1/65.3; M=385 N=14344 K=2056 37.1/32.1.
//     More rounds expose an epilogue each, in calls with pauses: 8192^3 with residual 797/910,
//     8192 x 28672 x 8192 2903/3464, 3000 x 8192 x 8192 319/396, 4096 x 6144 x 6144 267/304;
//     kept busy for seconds, under the power cap, 849/870, 2949/2922, 332/328, 252/252.  With
//     reductions of 200 slots and more the epilogue is 5 % of a tile and the A tiles' second
//     reading costs as much: the input gradient of 4096 x 14336 x 4096 390/396 with pauses and
//     392/375 without, 2048 x 8192 x 14336 380/385 and 402/373.  There they are taken if they
//     fill the rounds as well as the narrow ones (8192 x 4096 x 14336, 7 rounds of 256 tokens
//     against 4 of 512: 701/814 and 734/743).
//   groups (their rows are known on the device only): up to twice the mean rows, so that
//     most groups are one tile or 256-token tiles; a tile's MMAs follow its own rows.  Wide
//     tiles were slower or the same (64 experts of 4096 x 2048, 512 rows each, 537/590 us).
constexpr int kWideSlots = 200;
struct TokenTile {
    int bt, wide;
};
static TokenTile token_tile(int64_t m, int groups, int n_f, int pairs, int red) {
    TokenTile best = {kMaxTokens, 0};
    if (groups > 1) {
        best.bt = 32;
        while (best.bt < kMaxTokens && (int64_t)best.bt * groups < 2 * m) best.bt *= 2;
        return best;
    }
    double least = 1e300;
    int64_t narrow = 0;  // rounds x tokens of the best tiles of one part
    const int nkb = (red + kBlockK - 1) / kBlockK;
    const int64_t n0 = (m + kMaxTokens - 1) / kMaxTokens;
    for (int wide = 0; wide <= 1; wide++)
        for (int bt = kMaxTokens; bt >= 32; bt -= 32) {  // down to a quarter of the fewest tiles' tokens
            const int64_t n = (m + bt - 1) / bt;
            if (n > 4 * n0) break;
            if (wide && n == 1) continue;
            const int tokens = bt * (1 + wide);
            const int64_t tiles = (m + tokens - 1) / tokens * n_f, rounds = (tiles + pairs - 1) / pairs;
            if (wide && rounds > 1 && (nkb < kWideSlots || rounds * tokens > narrow)) continue;
            const double cost =
                (double)rounds * nkb * (150.0 + 1.07 * tokens) + (wide ? rounds : 1) * 20.0 * tokens;
            if (cost < least) {
                least = cost;
                best = {bt, wide};
                if (!wide) narrow = rounds * tokens;
            }
        }
    return best;
}

// Whether the split-reduction kernel takes a forward product or an input gradient (at most
// kDecodeTokens rows).  It wins where 256-feature tiles are too few to stream the weights on
// every SM, or the reduction is long; with more tokens its tiles re-read them more often, and
// the persistent kernel, without a reduction between CTAs, does.  The input gradient gives way
// earlier: it is launched in plain order (plan_decode).  Measured with weights that are not
// in L2, us, this kernel / persistent (features x reduction):
//   forward         1 token 4096 x 4096 9.9/20.7, 14336 x 4096 22.8/27.0, 28672 x 8192 73.0/80.8;
//                   64 tokens 4096 x 4096 15.8/20.7, 14336 x 4096 24.8/28.8, 28672 x 8192
//                   79.9/84.1; 128 tokens 1024 x 4096 12.3/20.8, 4096 x 4096 21.2/20.8, 8192 x
//                   4096 23.4/22.3, 4096 x 16384 37.3/61.7, 8192 x 2048 17.6/14.6
//   input gradient  1 token 4096 x 4096 12.5/20.7; 64 tokens 4096 x 4096 18.6/20.7, 14336 x 4096
//                   26.9/24.8; 128 tokens 4096 x 4096 24.8/20.7, 4096 x 16384 39.7/61.7
//   groups          8 of 2048 x 2048, 64 rows 10.7/14.7; 64 of them 87.0/84.8
static bool use_decode(int form, int m, int groups, int n_f, int red) {
    if (m > kDecodeTokens) return false;
    const int64_t tiles = (int64_t)n_f * std::min(groups, m);
    if (m <= 32) return tiles <= 128;
    if (m <= 64) return tiles <= (form == kForward ? 128 : 37);
    return tiles <= 32 && red >= (form == kForward ? 4096 : 8192);
}

Plan make_plan(int form, int groups, bool ragged, int m_total, int features, int red, int sm_count) {
    Plan plan = {};
    const int n_f = (features + 255) / 256, pairs = sm_count / 2;
    if (form == kWgrad) {
        // 256 x 256 tiles, or 256 x 128 where the others would leave half the pairs idle: a
        // tile's time is its tokens' (8192 tokens, N = K = 1024: 52 us in 16 tiles, 39 in 32;
        // but 4096 tokens, N = K = 2048: 36 in 64, 42 in 128)
        plan.bt = (int64_t)groups * n_f * ((red + 255) / 256) * 2 <= pairs ? 128 : 256;
        plan.tiles = (int64_t)groups * n_f * ((red + plan.bt - 1) / plan.bt);
    } else {
        if (use_decode(form, m_total, groups, n_f, red)) {
            plan_decode(form, groups, m_total, features, red, sm_count, &plan);
            return plan;
        }
        const TokenTile tt = token_tile(m_total, groups, n_f, pairs, red);
        plan.bt = tt.bt;
        plan.wide = tt.wide;
        plan.tiles = ((m_total + plan.bt - 1) / plan.bt + (ragged ? groups : 0)) * (int64_t)n_f;
    }
    const int ring = kRingBytes - (form == kWgrad ? kTileBytes : 0);
    plan.stages = std::min(kMaxStages, ring / (kTileBytes + plan.bt * 64 * (1 + plan.wide)));
    return plan;
}

template <typename T>
static int forward_t(const void *X, int64_t ldx, const void *W, Params p, int K, const DeviceInfo &di,
                     cudaStream_t s) {
    const Plan plan = make_plan(kForward, p.groups, p.m_offsets, p.m_total, p.features, K, di.sm_count);
    if (plan.decode) return decode_product<T, kForward>(X, ldx, W, p, plan, K, di, s);
    p.bt = plan.bt;
    p.wide = plan.wide;
    p.red = K;
    CUtensorMap a, b;
    int st = map_weight<T>(&a, W, p.groups, p.features, K, 128);
    if (!st) st = map_rows<T>(&b, X, p.m_total, K, ldx, p.bt / 2);
    if (st) return st;
    return launch_pair<T, kForward>(a, b, b, p, plan, di, s);
}

template <typename T>
static int dgrad_t(const void *dZ, const void *W, Params p, int N, const DeviceInfo &di, cudaStream_t s) {
    const Plan plan = make_plan(kDgrad, p.groups, p.m_offsets, p.m_total, p.features, N, di.sm_count);
    if (plan.decode) return decode_product<T, kDgrad>(dZ, N, W, p, plan, N, di, s);
    p.bt = plan.bt;
    p.wide = plan.wide;
    p.red = N;
    CUtensorMap a, b;
    int st = map_weight<T>(&a, W, p.groups, N, p.features, 64);
    if (!st) st = map_rows<T>(&b, dZ, p.m_total, N, N, p.bt / 2);
    if (st) return st;
    return launch_pair<T, kDgrad>(a, b, b, p, plan, di, s);
}

template <typename T>
static int wgrad_t(const void *dZ, const void *X, int64_t ldx, Params p, const DeviceInfo &di, cudaStream_t s) {
    const Plan plan = make_plan(kWgrad, p.groups, p.m_offsets, p.m_total, p.features, p.out_cols, di.sm_count);
    p.bt = plan.bt;
    CUtensorMap a, b, d;
    int st = map_rows<T>(&a, dZ, std::max(p.m_total, 1), p.features, p.features, 64);
    if (!st) st = map_rows<T>(&b, X, std::max(p.m_total, 1), p.out_cols, ldx, 64);
    if (!st) st = map_gradient<T>(&d, p.y, p.groups, p.features, p.out_cols);
    if (st) return st;
    return launch_pair<T, kWgrad>(a, b, d, p, plan, di, s);
}

// Sizes and pointers that the entry points have in common.
static int check_sizes(int groups, const int *m_offsets, int M, int N, int K, int dtype) {
    if (dtype != NVFP4_BF16 && dtype != NVFP4_F16) return NVFP4_ERR_INVALID;
    if (groups < 1 || (groups > 1 && !m_offsets)) return NVFP4_ERR_INVALID;
    if (groups > kMaxGroups || M < 0 || N < 8 || N % 8 || K < 8 || K % 8) return NVFP4_ERR_SHAPE;
    if (M > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return NVFP4_ERR_SHAPE;
    if ((int64_t)N * K > ((int64_t)1 << 40) / 2) return NVFP4_ERR_SHAPE;  // a tensor map's strides are below 2^40
    if (reinterpret_cast<uintptr_t>(m_offsets) & 3u) return NVFP4_ERR_ALIGN;
    return NVFP4_OK;
}

}  // namespace linear
}  // namespace nvfp4

using namespace nvfp4;

extern "C" {

int nvfp4_linear(const void *X, int64_t ldx, const void *W, const void *bias, const void *residual, void *Y, void *Z,
                 const int32_t *m_offsets, int groups, int M, int N, int K, int activation, int dtype, void *stream) {
    int st = linear::check_sizes(groups, m_offsets, M, N, K, dtype);
    if (st) return st;
    if (activation < NVFP4_ACT_NONE || activation > NVFP4_ACT_SWIGLU) return NVFP4_ERR_INVALID;
    if (activation == NVFP4_ACT_SWIGLU && N % 32) return NVFP4_ERR_SHAPE;
    if (ldx < K || ldx % 8) return NVFP4_ERR_SHAPE;
    if (!W || (M && (!X || !Y))) return NVFP4_ERR_INVALID;
    if (!aligned16(X) || !aligned16(W) || !aligned16(Y) || !aligned16(Z) || !aligned16(residual) ||
        (reinterpret_cast<uintptr_t>(bias) & 1u))
        return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (M == 0) return NVFP4_OK;
    linear::Params p = {};
    p.y = Y;
    p.z = Z;
    p.bias = bias;
    p.residual = residual;
    p.m_offsets = m_offsets;
    p.groups = groups;
    p.m_total = M;
    p.features = N;
    p.out_cols = activation == NVFP4_ACT_SWIGLU ? N / 2 : N;
    p.act = activation;
    if ((st = kernel_ctl(&p.ctl))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == NVFP4_BF16 ? linear::forward_t<__nv_bfloat16>(X, ldx, W, p, K, di, s)
                               : linear::forward_t<__half>(X, ldx, W, p, K, di, s);
}

int nvfp4_linear_dgrad(const void *dZ, const void *W, void *dX, const int32_t *m_offsets, int groups, int M, int N,
                       int K, int dtype, void *stream) {
    int st = linear::check_sizes(groups, m_offsets, M, N, K, dtype);
    if (st) return st;
    if (!W || (M && (!dZ || !dX))) return NVFP4_ERR_INVALID;
    if (!aligned16(dZ) || !aligned16(W) || !aligned16(dX)) return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    if (M == 0) return NVFP4_OK;
    linear::Params p = {};
    p.y = dX;
    p.m_offsets = m_offsets;
    p.groups = groups;
    p.m_total = M;
    p.features = K;
    p.out_cols = K;
    if ((st = kernel_ctl(&p.ctl))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == NVFP4_BF16 ? linear::dgrad_t<__nv_bfloat16>(dZ, W, p, N, di, s)
                               : linear::dgrad_t<__half>(dZ, W, p, N, di, s);
}

int nvfp4_linear_wgrad(const void *dZ, const void *X, int64_t ldx, void *dW, const int32_t *m_offsets, int groups,
                       int M, int N, int K, int dtype, void *stream) {
    int st = linear::check_sizes(groups, m_offsets, M, N, K, dtype);
    if (st) return st;
    if (ldx < K || ldx % 8) return NVFP4_ERR_SHAPE;
    if (!dW || (M && (!dZ || !X))) return NVFP4_ERR_INVALID;
    if (!aligned16(dZ) || !aligned16(X) || !aligned16(dW)) return NVFP4_ERR_ALIGN;
    DeviceInfo di;
    if ((st = device_info(&di))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M == 0)  // no token: the gradient is zero
        return cuda_status(cudaMemsetAsync(dW, 0, (size_t)groups * N * K * 2, s));
    linear::Params p = {};
    p.y = dW;
    p.m_offsets = m_offsets;
    p.groups = groups;
    p.m_total = M;
    p.features = N;
    p.out_cols = K;
    if ((st = kernel_ctl(&p.ctl))) return st;
    return dtype == NVFP4_BF16 ? linear::wgrad_t<__nv_bfloat16>(dZ, X, ldx, p, di, s)
                               : linear::wgrad_t<__half>(dZ, X, ldx, p, di, s);
}

}  // extern "C"
